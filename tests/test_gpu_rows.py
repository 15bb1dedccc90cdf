"""The row operators on the GPU against their definitions in 64 bits (tests/rows_ref.py): layer norm over
folded leaves, its gradient, checkpoints in 8 bits, activations and their gradient."""
import importlib.util
import math
import os

import pytest
import torch

import ext_mpi_collectives_amd as emac
import rows_ref as ref

pytestmark = pytest.mark.gpu

CODE = {torch.float32: emac.FLOAT, torch.bfloat16: emac.BF16, torch.float16: emac.HALF}
KINDS = {"silu": emac.SILU, "gelu": emac.GELU, "gelu_tanh": emac.GELU_TANH}
TYPES = list(ref.TYPES)


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def rnd(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def matrix(rows, cols, t, gen=None, pad=0, off=0, scale=1.0):
    """rows x cols inside a larger buffer of a known value: `off` elements into it, rows `pad` apart."""
    buf = torch.full((off + rows * (cols + pad) + 8,), 7.0, device="cuda").to(t)
    m = buf[off:off + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    if gen is not None:
        m.copy_(torch.randn(rows, cols, device="cuda", generator=gen) * scale)
    return m, buf


def edges_kept(m, buf, value=7.0):
    """Nothing of a matrix's buffer but the matrix was written."""
    copy = buf.clone()
    view = torch.as_strided(copy, m.shape, m.stride(), m.storage_offset())
    view.fill_(value)
    return bool((copy == value).all())


def go(*handles, stream=None):
    for h in handles:
        emac.set_stream(h, (stream or torch.cuda.current_stream()).cuda_stream)
        emac.start(h)
    for h in handles:
        emac.wait(h)
        emac.done(h)


SIZES = [(1, 1), (3, 2), (5, 7), (1, 8), (33, 127), (4, 128), (17, 129), (7, 512), (5, 513), (9, 1000), (600, 1024), (3, 2047),
         (5, 2049), (2, 4096), (515, 4100), (3, 8191), (2, 10000), (3, 16384), (4, 16385), (2, 32768), (2, 65535)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("size", range(len(SIZES)))
def test_layernorm(size, t):
    rows, cols = SIZES[size]
    dt, gen = ref.TYPES[t], rnd(size)
    nsrc = [1, 2, 1, 4, 8, 1, 16, 3][size % 8]
    pad, off = [(0, 0), (3, 1), (8, 0), (1, 5)][size % 4]
    wt = dt if size % 3 else torch.float32
    srcs = [matrix(rows, cols, dt, gen, pad, off)[0] for _ in range(nsrc)]
    res = matrix(rows, cols, dt, gen, 2, 3, 2.0)[0] if size % 2 else None
    w = torch.randn(cols, device="cuda", generator=gen).to(wt) if size % 5 else None
    b = torch.randn(cols, device="cuda", generator=gen).to(wt) if size % 7 else None
    (y, ybuf), (s, sbuf) = matrix(rows, cols, dt, pad=1, off=1), matrix(rows, cols, dt, pad=pad)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    (q, qbuf), scale = matrix(rows, cols, torch.int8, pad=5, off=3), torch.empty(rows, -(-cols // 128), device="cuda")
    go(emac.layernorm_init(rows, cols, CODE[dt], [x.data_ptr() for x in srcs], y.data_ptr(), src_stride=srcs[0].stride(0),
                           y_stride=y.stride(0), residual=None if res is None else res.data_ptr(),
                           residual_stride=0 if res is None else res.stride(0), weight=None if w is None else w.data_ptr(),
                           bias=None if b is None else b.data_ptr(), wdtype=CODE[wt], eps=1e-5, sum=s.data_ptr(),
                           sum_stride=s.stride(0), mean=mean.data_ptr(), rstd=rstd.data_ptr(), q=q.data_ptr(),
                           q_stride=q.stride(0), scale=scale.data_ptr()))
    x = ref.fold(srcs, res)
    assert torch.equal(s, x)
    rq, rscale = ref.save8(x)
    assert torch.equal(q, rq) and torch.equal(scale, rscale)
    rmean, rrstd, ry, by = ref.layernorm(x, w, b, 1e-5)
    bmean, brstd = ref.stats_bounds(x, rrstd)
    ref.close(mean, rmean, bmean)
    ref.close(rstd, rrstd, rrstd * brstd)
    ref.close(y, ry, by)
    assert edges_kept(y, ybuf) and edges_kept(s, sbuf) and edges_kept(q, qbuf, 7)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("saved", [False, True])
@pytest.mark.parametrize("size", range(len(SIZES)))
def test_layernorm_grad(size, saved, t):
    rows, cols = SIZES[size]
    dt, gen = ref.TYPES[t], rnd(100 + size)
    nsrc = [1, 2, 1, 5, 1, 16][size % 6]
    pad, off = [(0, 0), (3, 1), (8, 0), (1, 5)][size % 4]
    wt, gt = (dt if size % 3 else torch.float32), (dt if size % 2 else torch.float32)
    dys = [matrix(rows, cols, dt, gen, pad, off)[0] for _ in range(nsrc)]
    x = matrix(rows, cols, dt, gen, pad, off, 3.0)[0]
    dsum = matrix(rows, cols, dt, gen, 1, 1)[0] if size % 2 else None
    w = torch.randn(cols, device="cuda", generator=gen).to(wt) if size % 5 else None
    b = torch.randn(cols, device="cuda", generator=gen).to(wt) if size % 7 else None
    q, scale = ref.save8(x)
    xv = ref.restore8(q, scale) if saved else x.float()
    m64, r64 = x.double().mean(1), (x.double().var(1, unbiased=False) + 1e-5).rsqrt()
    mean, rstd = m64.float(), r64.float()
    (dx, dxbuf), (y, ybuf) = matrix(rows, cols, dt, pad=3, off=2), matrix(rows, cols, dt, pad=1)
    dw, db = torch.full((cols + 1,), 7.0, device="cuda").to(gt), torch.full((cols + 1,), 7.0, device="cuda").to(gt)
    kw = {"q": q.data_ptr(), "scale": scale.data_ptr()} if saved else {"x": x.data_ptr(), "x_stride": x.stride(0)}
    go(emac.layernorm_grad_init(rows, cols, CODE[dt], [d.data_ptr() for d in dys], mean.data_ptr(), rstd.data_ptr(),
                                dy_stride=dys[0].stride(0), weight=None if w is None else w.data_ptr(), wdtype=CODE[wt],
                                bias=None if b is None else b.data_ptr(), dsum=None if dsum is None else dsum.data_ptr(),
                                dsum_stride=0 if dsum is None else dsum.stride(0), dx=dx.data_ptr(), dx_stride=dx.stride(0),
                                dweight=dw.data_ptr(), dbias=db.data_ptr(), gdtype=CODE[gt], y=y.data_ptr(),
                                y_stride=y.stride(0), **kw))
    g = dys[0].float()
    for d in dys[1:]:
        g = g + d.float()
    rdx, bdx, rdw, bdw, rdb, bdb = ref.layernorm_grad(g, xv, mean, rstd, w, dsum)
    ref.close(dx, rdx, bdx)
    ref.close(dw[:cols], rdw, bdw)
    ref.close(db[:cols], rdb, bdb)
    xh = (xv.double() - mean.double()[:, None]) * rstd.double()[:, None]
    ry = xh * (1.0 if w is None else w.double()) + (0.0 if b is None else b.double())
    by = 8 * ref.U * ((xh.abs() + rstd.double()[:, None] * (xv.double().abs() + mean.double().abs()[:, None])) *
                      (1.0 if w is None else w.double().abs()) + (0.0 if b is None else b.double().abs()))
    ref.close(y, ry, by)
    assert float(dw[cols]) == 7 and float(db[cols]) == 7 and edges_kept(dx, dxbuf) and edges_kept(y, ybuf)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(2000, 96), (4099, 256), (5000, 1024), (1500, 4096), (40, 20000)])
def test_layernorm_grad_many_rows(rows, cols, t):
    """More rows than workgroups: the column sums over several rows of a workgroup and the partial rows;
    the same bits twice; added to with accumulate; only the column sums; only dx."""
    dt, gen = ref.TYPES[t], rnd(rows)
    dy, x = matrix(rows, cols, dt, gen)[0], matrix(rows, cols, dt, gen)[0]
    mean, rstd = x.float().mean(1), (x.float().var(1, unbiased=False) + 1e-5).rsqrt()
    rdx, bdx, rdw, bdw, rdb, bdb = ref.layernorm_grad(dy, x, mean, rstd, None, None)
    out = []
    for _ in range(2):
        dx, dw, db = torch.empty_like(x), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
        h = emac.layernorm_grad_init(rows, cols, CODE[dt], [dy.data_ptr()], mean.data_ptr(), rstd.data_ptr(), x=x.data_ptr(),
                                     dx=dx.data_ptr(), dweight=dw.data_ptr(), dbias=db.data_ptr(), gdtype=emac.FLOAT)
        go(h)
        out.append((dx, dw, db))
    for k, (r, bnd) in enumerate(((rdx, bdx), (rdw, bdw), (rdb, bdb))):
        ref.close(out[0][k], r, bnd)
        assert torch.equal(out[0][k], out[1][k])
    dw, db = torch.full((cols,), 2.0, device="cuda"), torch.full((cols,), -1.0, device="cuda")
    go(emac.layernorm_grad_init(rows, cols, CODE[dt], [dy.data_ptr()], mean.data_ptr(), rstd.data_ptr(), x=x.data_ptr(),
                                dweight=dw.data_ptr(), dbias=db.data_ptr(), gdtype=emac.FLOAT, accumulate=True))
    assert torch.equal(dw, 2.0 + out[0][1]) and torch.equal(db, -1.0 + out[0][2])
    dx, db = torch.empty_like(x), torch.empty(cols, device="cuda")
    go(emac.layernorm_grad_init(rows, cols, CODE[dt], [dy.data_ptr()], mean.data_ptr(), rstd.data_ptr(), x=x.data_ptr(), dx=dx.data_ptr()),
       emac.layernorm_grad_init(rows, cols, CODE[dt], [dy.data_ptr()], mean.data_ptr(), rstd.data_ptr(), x=x.data_ptr(),
                                dbias=db.data_ptr(), gdtype=emac.FLOAT))
    assert torch.equal(dx, out[0][0]) and torch.equal(db, out[0][2])


WIDTHS = [(70001, 5), (70000, 40), (33333, 72), (9001, 264), (3000, 1300), (1025, 4096), (700, 5000), (600, 5121), (550, 8192), (600, 10001),
          (520, 12290), (510, 13000), (515, 16384), (260, 16387), (300, 20001), (257, 32773), (270, 33000), (5, 65529)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nsrc", [1, 3])
@pytest.mark.parametrize("rows,cols", WIDTHS)
def test_forward_and_gradient_over_many_rows(rows, cols, nsrc, t):
    """Every width's kernels with more rows than workgroups: the norm with a checkpoint, then its gradient
    from x and from the checkpoint, the checkpoint's with the norm's output again."""
    dt, gen = ref.TYPES[t], rnd(rows + nsrc)
    src = [torch.randn(rows, cols, device="cuda", generator=gen).to(dt) for _ in range(nsrc)]
    w, b = (torch.randn(cols, device="cuda", generator=gen).to(dt) for _ in range(2))
    x, y, y2, dx, dx8 = (torch.empty_like(src[0]) for _ in range(5))
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    q, scale = torch.empty(rows, cols, dtype=torch.int8, device="cuda"), torch.empty(rows, -(-cols // 128), device="cuda")
    dw, db, dw8, db8 = (torch.empty(cols, device="cuda") for _ in range(4))
    go(emac.layernorm_init(rows, cols, CODE[dt], [v.data_ptr() for v in src], y.data_ptr(), weight=w.data_ptr(), bias=b.data_ptr(), sum=x.data_ptr(),
                           mean=mean.data_ptr(), rstd=rstd.data_ptr(), q=q.data_ptr(), scale=scale.data_ptr()))
    assert torch.equal(x, ref.fold(src))
    rq, rscale = ref.save8(x)
    assert torch.equal(q, rq) and torch.equal(scale, rscale)
    _, rrstd, ry, by = ref.layernorm(x, w, b, 1e-5)
    ref.close(y, ry, by)
    ref.close(rstd, rrstd, rrstd * ref.stats_bounds(x, rrstd)[1])
    kw = dict(weight=w.data_ptr(), gdtype=emac.FLOAT)
    dys = [v.data_ptr() for v in src]  # any rows do as gradients
    go(emac.layernorm_grad_init(rows, cols, CODE[dt], dys, mean.data_ptr(), rstd.data_ptr(), x=x.data_ptr(), dx=dx.data_ptr(), dweight=dw.data_ptr(),
                                dbias=db.data_ptr(), **kw),
       emac.layernorm_grad_init(rows, cols, CODE[dt], dys, mean.data_ptr(), rstd.data_ptr(), q=q.data_ptr(), scale=scale.data_ptr(), dx=dx8.data_ptr(),
                                dweight=dw8.data_ptr(), dbias=db8.data_ptr(), dsum=x.data_ptr(), bias=b.data_ptr(), y=y2.data_ptr(), **kw))
    g = src[0].float()
    for v in src[1:]:
        g = g + v.float()
    xq = ref.restore8(rq, rscale)
    for xv, o, ow, ob, ds in ((x, dx, dw, db, None), (xq, dx8, dw8, db8, x)):
        rdx, bdx, rdw, bdw, rdb, bdb = ref.layernorm_grad(g, xv, mean, rstd, w, ds)
        ref.close(o, rdx, bdx)
        ref.close(ow, rdw, bdw)
        ref.close(ob, rdb, bdb)
    xh = (xq.double() - mean.double()[:, None]) * rstd.double()[:, None]
    exh = 8 * ref.U * (xh.abs() + rstd.double()[:, None] * (xq.double().abs() + mean.double().abs()[:, None]))
    ref.close(y2, xh * w.double() + b.double(), exh * w.double().abs() + 8 * ref.U * b.double().abs())


@pytest.mark.parametrize("cols,t", [(200, "f32"), (1000, "f32"), (5000, "f32")])
def test_layernorm_grad_by_differences(cols, t):
    """The change of L = sum(y r) along a direction of x, w and b, by central differences of the forward
    kernel, against the gradient kernel's. A step h leaves h^2/6 of the third derivative (the values
    here are O(1): under 1e-4 at h = 2^-6) and the roundings of y, 4 U |y||r| per element in the root
    of their number, over 2h."""
    rows, gen, h = 6, rnd(cols), 2.0 ** -6
    x, r, vx = (torch.randn(rows, cols, device="cuda", generator=gen) for _ in range(3))
    w, b, vw, vb = (torch.randn(cols, device="cuda", generator=gen) for _ in range(4))
    mean, rstd, y = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty_like(x)

    def loss(k):
        xx, ww, bb = x + k * vx, w + k * vw, b + k * vb
        go(emac.layernorm_init(rows, cols, emac.FLOAT, [xx.data_ptr()], y.data_ptr(), weight=ww.data_ptr(), bias=bb.data_ptr(),
                               mean=mean.data_ptr(), rstd=rstd.data_ptr()))
        return float((y.double() * r.double()).sum())

    change = (loss(h) - loss(-h)) / (2 * h)
    loss(0.0)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    go(emac.layernorm_grad_init(rows, cols, emac.FLOAT, [r.data_ptr()], mean.data_ptr(), rstd.data_ptr(), x=x.data_ptr(),
                                weight=w.data_ptr(), dx=dx.data_ptr(), dweight=dw.data_ptr(), dbias=db.data_ptr()))
    slope = float((dx.double() * vx).sum() + (dw.double() * vw).sum() + (db.double() * vb).sum())
    n = rows * cols
    size = float((y.double().abs() * r.abs()).sum())
    noise = 4 * ref.U * size / math.sqrt(n) / h + 1e-3 * math.sqrt(n)
    assert abs(change - slope) < noise, (change, slope, noise)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (2, 127), (5, 128), (4, 129), (70, 64), (3, 300), (65, 8192), (17, 8200), (2, 100003)])
def test_save_and_restore(rows, cols, t):
    dt, gen = ref.TYPES[t], rnd(cols)
    x = matrix(rows, cols, dt, gen, 3, 1)[0]
    x[:, ::53] *= 40
    x[0] = 0
    (q, qbuf), scale = matrix(rows, cols, torch.int8, pad=1, off=1), torch.empty(rows, -(-cols // 128), device="cuda")
    back, bbuf = matrix(rows, cols, dt, pad=2, off=1)
    go(emac.save8_init(rows, cols, CODE[dt], x.data_ptr(), q.data_ptr(), scale.data_ptr(), x_stride=x.stride(0), q_stride=q.stride(0)))
    go(emac.restore8_init(rows, cols, CODE[dt], q.data_ptr(), scale.data_ptr(), back.data_ptr(), q_stride=q.stride(0), x_stride=back.stride(0)))
    rq, rscale = ref.save8(x)
    assert torch.equal(q, rq) and torch.equal(scale, rscale)
    assert torch.equal(back, ref.restore8(rq, rscale).to(dt))
    assert edges_kept(q, qbuf, 7) and edges_kept(back, bbuf)
    a = torch.zeros(rows, -(-cols // 128) * 128, device="cuda")
    a[:, :cols] = x.float().abs()
    a = a.view(rows, -1, 128).amax(2).repeat_interleave(128, 1)[:, :cols].double()
    ref.close(back, x.double(), a * (1 / 254 + 5 * ref.U) + 2.0 ** -107)  # tests/test_rows_cpu.py counts them


@pytest.mark.parametrize("t", TYPES)
def test_save_of_special_values(t):
    """Infinities, NaN, the type's largest and smallest values, subnormal blocks, both zeros."""
    dt = ref.TYPES[t]
    x = torch.randn(8, 300, device="cuda", generator=rnd(1)).to(dt)
    f = torch.finfo(dt)
    x[0, 3], x[1, 130], x[2, 299] = math.inf, -math.inf, math.nan
    x[3, 7], x[3, 8], x[4, 200] = f.max, f.min, f.smallest_normal
    x[5], x[6, :128] = ref.SMALLEST[dt], -0.0
    q, scale, back = torch.empty(8, 300, dtype=torch.int8, device="cuda"), torch.empty(8, 3, device="cuda"), torch.empty_like(x)
    go(emac.save8_init(8, 300, CODE[dt], x.data_ptr(), q.data_ptr(), scale.data_ptr()))
    go(emac.restore8_init(8, 300, CODE[dt], q.data_ptr(), scale.data_ptr(), back.data_ptr()))
    rq, rscale = ref.save8(x)
    assert torch.equal(q, rq) and torch.equal(scale.nan_to_num(-1), rscale.nan_to_num(-1))
    nan = torch.zeros(8, 300, dtype=torch.bool, device="cuda")
    nan[0, :128], nan[1, 128:256], nan[2, 256:] = True, True, True
    assert torch.equal(back.isnan(), nan)
    want = ref.restore8(rq, rscale).to(dt)
    assert torch.equal(back[~nan], want[~nan]) and float(back[3, 7]) == float(want[3, 7])


def test_layernorm_of_special_rows():
    """A row of one value (variance 0), rows with an infinity or a NaN beside others, which keep theirs."""
    x = torch.randn(6, 777, device="cuda", generator=rnd(2))
    x[1], x[2, 5], x[3, 9], x[4] = 2.5, math.inf, math.nan, 0
    y, mean, rstd = torch.empty_like(x), torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
    go(emac.layernorm_init(6, 777, emac.FLOAT, [x.data_ptr()], y.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr()))
    assert bool(y[2].isnan().all()) and bool(y[3].isnan().all())
    rmean, rrstd, ry, by = ref.layernorm(x, None, None, 1e-5)
    keep = [0, 1, 4, 5]
    ref.close(y[keep], ry[keep], by[keep])
    assert bool((y[4] == 0).all())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("gate", [False, True])
def test_act_and_grad(gate, kind, t):
    for k, (rows, cols) in enumerate([(1, 1), (3, 5), (2, 128), (9, 129), (130, 70), (3, 1000), (40, 4097), (2, 20000)]):
        dt, gen = ref.TYPES[t], rnd(7 * k)
        pad = [0, 3, 8, 1][k % 4]
        n = 2 if gate else 1
        ab = matrix(rows, n * cols, dt, gen, pad, k % 3, 3.0)[0]
        a, b = ab[:, :cols], ab[:, cols:] if gate else None
        dh = matrix(rows, cols, dt, gen, pad, 1)[0]
        h, hbuf = matrix(rows, cols, dt, pad=1, off=1)
        (qa, qbuf), sa = matrix(rows, cols, torch.int8, pad=3, off=1), torch.empty(rows, -(-cols // 128), device="cuda")
        qb, sb = torch.full((rows, cols + 3), 7, dtype=torch.int8, device="cuda")[:, :cols], torch.empty_like(sa)
        dab, dbuf = matrix(rows, n * cols, dt, pad=pad, off=1)
        da, db = dab[:, :cols], dab[:, cols:] if gate else None
        h2 = torch.empty(rows, cols, dtype=dt, device="cuda")
        go(emac.act_init(rows, cols, CODE[dt], KINDS[kind], a.data_ptr(), h.data_ptr(), a_stride=a.stride(0), h_stride=h.stride(0),
                         b=b.data_ptr() if gate else None, b_stride=b.stride(0) if gate else 0, qa=qa.data_ptr(), sa=sa.data_ptr(),
                         qb=qb.data_ptr() if gate else None, sb=sb.data_ptr() if gate else None, q_stride=cols + 3))
        go(emac.act_grad_init(rows, cols, CODE[dt], KINDS[kind], dh.data_ptr(), qa.data_ptr(), sa.data_ptr(), da.data_ptr(),
                              dh_stride=dh.stride(0), da_stride=da.stride(0), qb=qb.data_ptr() if gate else None,
                              sb=sb.data_ptr() if gate else None, db=db.data_ptr() if gate else None,
                              db_stride=db.stride(0) if gate else 0, q_stride=cols + 3, h=h2.data_ptr()))
        rqa, rsa = ref.save8(a)
        assert torch.equal(qa, rqa) and torch.equal(sa, rsa)
        v, _, bv, _ = ref.act(kind, a)
        ra = ref.restore8(rqa, rsa)
        rv, slope, brv, bslope = ref.act(kind, ra)
        one = torch.ones(1, dtype=torch.float64, device="cuda")
        fb, rb = (b.double(), ref.restore8(*ref.save8(b)).double()) if gate else (one, one)
        if gate:
            rqb, rsb = ref.save8(b)
            assert torch.equal(qb, rqb) and torch.equal(sb, rsb)
        g, u = dh.double(), 4 * ref.U
        ref.close(h, v * fb, (bv + u * v.abs()) * fb.abs())
        ref.close(h2, rv * rb, (brv + u * rv.abs()) * rb.abs())
        ref.close(da, g * slope * rb, g.abs() * rb.abs() * (bslope + u * slope.abs()))
        if gate:
            ref.close(db, g * rv, g.abs() * (brv + u * rv.abs()))
        assert edges_kept(h, hbuf) and edges_kept(qa, qbuf, 7) and edges_kept(dab, dbuf)


@pytest.mark.parametrize("kind", list(KINDS))
def test_act_at_its_ends(kind):
    """Far tails, zeros and the largest values: no NaN where the function has a value."""
    a = torch.tensor([[0.0, -0.0, 1e-30, -1e-30, 10.0, -10.0, 40.0, -40.0, 100.0, -100.0, 1e4, -1e4, 1e20, -1e20, 3e38, -3e38]], device="cuda")
    h = torch.empty_like(a)
    go(emac.act_init(1, 16, emac.FLOAT, KINDS[kind], a.data_ptr(), h.data_ptr()))
    assert not bool(h.isnan().any())
    assert torch.equal(h[0, 6::2], a[0, 6::2])
    assert bool((h[0, 9::2] == 0).all()) and bool((h[0, 5::2] <= 0).all())
    v, _, bv, _ = ref.act(kind, a[:, :8])
    ref.close(h[:, :8], v, bv)
    x = torch.tensor([[math.inf, math.nan, 1.0]], device="cuda")
    for t in ref.TYPES.values():
        xt, ht = x.to(t), torch.empty_like(x.to(t))
        go(emac.act_init(1, 3, CODE[t], KINDS[kind], xt.data_ptr(), ht.data_ptr()))
        assert float(ht[0, 0]) == math.inf and math.isnan(float(ht[0, 1])) and 0.7 < float(ht[0, 2]) < 0.9
    da, dh = torch.empty_like(a), torch.ones_like(a)
    for j in range(16):  # each value a block of its own, restored to within a rounding
        q, s = torch.full((1, 1), 127 if a[0, j] > 0 else -127, dtype=torch.int8, device="cuda"), (a[:, j:j + 1].abs() / 127).contiguous()
        go(emac.act_grad_init(1, 1, emac.FLOAT, KINDS[kind], dh[:, j:].data_ptr(), q.data_ptr(), s.data_ptr(), da[:, j:].data_ptr()))
    assert not bool(da.isnan().any())
    assert torch.equal(da[0, 8::2], torch.ones(4, device="cuda")) and bool((da[0, 9::2].abs() == 0).all())


def test_act_without_checkpoint_and_checkpoint_alone():
    a, b = torch.randn(5, 999, device="cuda").half(), torch.randn(5, 999, device="cuda").half()
    h, h2 = torch.empty_like(a), torch.empty_like(a)
    qa, sa, qb, sb = (torch.empty(5, 999, dtype=torch.int8, device="cuda"), torch.empty(5, 8, device="cuda"),
                      torch.empty(5, 999, dtype=torch.int8, device="cuda"), torch.empty(5, 8, device="cuda"))
    go(emac.act_init(5, 999, emac.HALF, emac.SILU, a.data_ptr(), h.data_ptr(), b=b.data_ptr()),
       emac.act_init(5, 999, emac.HALF, emac.SILU, a.data_ptr(), b=b.data_ptr(), qa=qa.data_ptr(), sa=sa.data_ptr(), qb=qb.data_ptr(), sb=sb.data_ptr()))
    assert torch.equal(qb, ref.save8(b)[0]) and torch.equal(qa, ref.save8(a)[0])
    go(emac.act_init(5, 999, emac.HALF, emac.SILU, a.data_ptr(), h2.data_ptr(), b=b.data_ptr(), qa=qa.data_ptr(), sa=sa.data_ptr(), qb=qb.data_ptr(),
                     sb=sb.data_ptr()))
    assert torch.equal(h, h2)


def test_in_place():
    """An output over an input of its type: sum over the residual, y over a leaf, dx over dy, da over dh."""
    rows, cols = 300, 1030
    gen = rnd(3)
    src, res = (torch.randn(rows, cols, device="cuda", generator=gen).bfloat16() for _ in range(2))
    y, s = torch.empty_like(src), torch.empty_like(src)
    q, sc = torch.empty(rows, cols, dtype=torch.int8, device="cuda"), torch.empty(rows, 9, device="cuda")
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    go(emac.layernorm_init(rows, cols, emac.BF16, [src.data_ptr()], y.data_ptr(), residual=res.data_ptr(), sum=s.data_ptr(), q=q.data_ptr(),
                           scale=sc.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr()))
    src2, res2 = src.clone(), res.clone()
    go(emac.layernorm_init(rows, cols, emac.BF16, [src2.data_ptr()], src2.data_ptr(), residual=res2.data_ptr(), sum=res2.data_ptr()))
    assert torch.equal(src2, y) and torch.equal(res2, s)
    dw = torch.empty(cols, device="cuda")
    dx, dy2, dw2 = torch.empty_like(src), src.clone(), torch.empty_like(dw)
    go(emac.layernorm_grad_init(rows, cols, emac.BF16, [src.data_ptr()], mean.data_ptr(), rstd.data_ptr(), x=s.data_ptr(), dx=dx.data_ptr(),
                                dweight=dw.data_ptr(), gdtype=emac.FLOAT),
       emac.layernorm_grad_init(rows, cols, emac.BF16, [dy2.data_ptr()], mean.data_ptr(), rstd.data_ptr(), x=s.data_ptr(), dx=dy2.data_ptr(),
                                dweight=dw2.data_ptr(), gdtype=emac.FLOAT))
    assert torch.equal(dx, dy2) and torch.equal(dw, dw2)
    da, dh2 = torch.empty_like(src), src.clone()
    go(emac.act_grad_init(rows, cols, emac.BF16, emac.GELU, src.data_ptr(), q.data_ptr(), sc.data_ptr(), da.data_ptr()),
       emac.act_grad_init(rows, cols, emac.BF16, emac.GELU, dh2.data_ptr(), q.data_ptr(), sc.data_ptr(), dh2.data_ptr()))
    assert torch.equal(da, dh2)


@pytest.mark.parametrize("cols", [9, 129, 130, 519, 521, 1031, 4097, 8193])
def test_in_place_at_odd_widths(cols):
    """In place where the row's last vector is not whole and may lie in another wave than the one before."""
    rows, gen = 500, rnd(cols)
    a, b, dh, res = (torch.randn(rows, cols, device="cuda", generator=gen).bfloat16() for _ in range(4))
    nb = -(-cols // 128)
    q, q2, q3 = (torch.empty(rows, cols, dtype=torch.int8, device="cuda") for _ in range(3))
    s, s2, s3 = (torch.empty(rows, nb, device="cuda") for _ in range(3))
    h, da, db = torch.empty_like(a), torch.empty_like(a), torch.empty_like(a)
    code, silu = emac.BF16, emac.SILU
    go(emac.act_init(rows, cols, code, silu, a.data_ptr(), h.data_ptr(), b=b.data_ptr(), qa=q.data_ptr(), sa=s.data_ptr(), qb=q2.data_ptr(), sb=s2.data_ptr()),
       emac.act_grad_init(rows, cols, code, silu, dh.data_ptr(), q.data_ptr(), s.data_ptr(), da.data_ptr(), qb=q2.data_ptr(), sb=s2.data_ptr(), db=db.data_ptr()))
    a2, dh2, db2 = a.clone(), dh.clone(), torch.empty_like(a)
    go(emac.act_init(rows, cols, code, silu, a2.data_ptr(), a2.data_ptr(), b=b.data_ptr(), qa=q3.data_ptr(), sa=s3.data_ptr(), qb=q2.data_ptr(), sb=s2.data_ptr()),
       emac.act_grad_init(rows, cols, code, silu, dh2.data_ptr(), q.data_ptr(), s.data_ptr(), dh2.data_ptr(), qb=q2.data_ptr(), sb=s2.data_ptr(), db=db2.data_ptr()))
    assert torch.equal(a2, h) and torch.equal(q3, q) and torch.equal(s3, s) and torch.equal(dh2, da) and torch.equal(db2, db)
    x, res2, mean, rstd, y = torch.empty_like(a), res.clone(), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty_like(a)
    go(emac.layernorm_init(rows, cols, code, [a.data_ptr()], y.data_ptr(), residual=res.data_ptr(), sum=x.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr()),
       emac.layernorm_init(rows, cols, code, [a.data_ptr()], residual=res2.data_ptr(), sum=res2.data_ptr()))
    assert torch.equal(x, ref.fold([a], res)) and torch.equal(res2, x)
    y2, dx, dy2, dw, dw2 = a.clone(), torch.empty_like(a), dh.clone(), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    go(emac.layernorm_init(rows, cols, code, [y2.data_ptr()], y2.data_ptr(), residual=res.data_ptr()))
    assert torch.equal(y2, y)
    for g, o, w in ((dh, dx, dw), (dy2, dy2, dw2)):
        go(emac.layernorm_grad_init(rows, cols, code, [g.data_ptr()], mean.data_ptr(), rstd.data_ptr(), x=x.data_ptr(), dx=o.data_ptr(), dsum=g.data_ptr(),
                                    dweight=w.data_ptr(), gdtype=emac.FLOAT))
    assert torch.equal(dy2, dx) and torch.equal(dw2, dw)


def test_in_place_wide_gradient():
    """Rows wider than the registers hold: the column sums are taken before dx replaces dy."""
    rows, cols = 9, 20001
    dy, x = (torch.randn(rows, cols, device="cuda", generator=rnd(4)) for _ in range(2))
    mean, rstd = x.mean(1), (x.var(1, unbiased=False) + 1e-5).rsqrt()
    dx, dy2 = torch.empty_like(x), dy.clone()
    dw, dw2 = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    for g, o, w in ((dy, dx, dw), (dy2, dy2, dw2)):
        go(emac.layernorm_grad_init(rows, cols, emac.FLOAT, [g.data_ptr()], mean.data_ptr(), rstd.data_ptr(), x=x.data_ptr(), dx=o.data_ptr(),
                                    dweight=w.data_ptr()))
    assert torch.equal(dx, dy2) and torch.equal(dw, dw2)


def test_no_rows():
    """Nothing is touched; a gradient's sums over no rows are zeros, or what was there with accumulate."""
    y = torch.full((4,), 7.0, device="cuda")
    dw, db, kept = torch.full((40,), 7.0, device="cuda"), torch.full((40,), 7.0, device="cuda").bfloat16(), torch.full((40,), 7.0, device="cuda")
    go(emac.layernorm_init(0, 40, emac.FLOAT, [None], y.data_ptr()), emac.save8_init(0, 40, emac.FLOAT, None, None, None),
       emac.restore8_init(0, 40, emac.FLOAT, None, None, None), emac.act_init(0, 40, emac.FLOAT, emac.GELU, None),
       emac.act_grad_init(0, 40, emac.FLOAT, emac.GELU, None, None, None, None))
    go(emac.layernorm_grad_init(0, 40, emac.BF16, [None], None, None, dweight=dw.data_ptr(), gdtype=emac.FLOAT),
       emac.layernorm_grad_init(0, 40, emac.BF16, [None], None, None, dbias=db.data_ptr()),
       emac.layernorm_grad_init(0, 40, emac.BF16, [None], None, None, dweight=kept.data_ptr(), gdtype=emac.FLOAT, accumulate=True))
    assert bool((dw == 0).all()) and bool((db == 0).all()) and bool((kept == 7).all()) and bool((y == 7).all())


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_offsets_past_32_bits(t):
    """Rows more than 2^31 elements apart."""
    dt, rows, cols, ld = ref.TYPES[t], 3, 700, (1 << 30) + 5
    buf = torch.empty((rows - 1) * ld + cols, dtype=dt, device="cuda")
    x = torch.as_strided(buf, (rows, cols), (ld, 1))
    x.copy_(torch.randn(rows, cols, device="cuda", generator=rnd(5)))
    qbuf = torch.empty(2 * (1 << 31) + cols, dtype=torch.int8, device="cuda")
    q = torch.as_strided(qbuf, (rows, cols), (1 << 31, 1))
    scale = torch.empty(rows, 6, device="cuda")
    y, mean, rstd = torch.empty(rows, cols, dtype=dt, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    go(emac.layernorm_init(rows, cols, CODE[dt], [x.data_ptr()], y.data_ptr(), src_stride=ld, mean=mean.data_ptr(), rstd=rstd.data_ptr(),
                           q=q.data_ptr(), q_stride=1 << 31, scale=scale.data_ptr()))
    rq, rscale = ref.save8(x.contiguous())
    assert torch.equal(q, rq) and torch.equal(scale, rscale)
    _, _, ry, by = ref.layernorm(x, None, None, 1e-5)
    ref.close(y, ry, by)
    dy, dw = torch.randn(rows, cols, device="cuda", generator=rnd(6)).to(dt), torch.empty(cols, device="cuda")
    rdx, bdx, rdw, bdw, _, _ = ref.layernorm_grad(dy, ref.restore8(rq, rscale), mean, rstd, None, None)
    go(emac.layernorm_grad_init(rows, cols, CODE[dt], [dy.data_ptr()], mean.data_ptr(), rstd.data_ptr(), q=q.data_ptr(), q_stride=1 << 31,
                                scale=scale.data_ptr(), dx=x.data_ptr(), dx_stride=ld, dweight=dw.data_ptr(), gdtype=emac.FLOAT))
    ref.close(x, rdx, bdx)
    ref.close(dw, rdw, bdw)
    go(emac.restore8_init(rows, cols, CODE[dt], q.data_ptr(), scale.data_ptr(), x.data_ptr(), q_stride=1 << 31, x_stride=ld))
    assert torch.equal(x, ref.restore8(rq, rscale).to(dt))


def test_more_blocks_than_one_grid_dimension():
    """2^28 and a few blocks, of one column each: 127 or -127, and back to the value's own bits."""
    rows = (1 << 28) + 37
    x = torch.randn(rows, 1, dtype=torch.bfloat16, device="cuda", generator=rnd(8))
    x[x == 0] = 1
    q, scale, back = torch.empty(rows, 1, dtype=torch.int8, device="cuda"), torch.empty(rows, 1, device="cuda"), torch.empty_like(x)
    go(emac.save8_init(rows, 1, emac.BF16, x.data_ptr(), q.data_ptr(), scale.data_ptr()),
       emac.restore8_init(rows, 1, emac.BF16, q.data_ptr(), scale.data_ptr(), back.data_ptr()))
    assert torch.equal(q, (x.sign() * 127).to(torch.int8)) and torch.equal(back, x)


def test_one_training_step_as_used():
    """The operators in a row on one stream, as a tensor-parallel block uses them: 8 ranks' partial rows
    folded onto the residual stream and normed with a checkpoint, a gated activation with checkpoints,
    its gradient, the partial gradients folded through the norm's; the fold by the Allreduce handle of
    the same leaves gives the same bits as the norm's own."""
    R, rows, cols, wide = 8, 384, 1024, 2560
    gen = rnd(8)
    parts = [torch.randn(rows, cols, device="cuda", generator=gen) for _ in range(R)]
    res = torch.randn(rows, cols, device="cuda", generator=gen)
    w, b = torch.randn(cols, device="cuda", generator=gen), torch.randn(cols, device="cuda", generator=gen)
    W = torch.randn(cols, 2 * wide, device="cuda", generator=gen) / 32
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    y, y2, x = torch.empty_like(res), torch.empty_like(res), torch.empty_like(res)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    q, sc = torch.empty(rows, cols, dtype=torch.int8, device="cuda"), torch.empty(rows, 8, device="cuda")
    folded = torch.empty_like(res)
    ab = torch.empty(rows, 2 * wide, device="cuda")
    a, bb = ab[:, :wide], ab[:, wide:]
    h, dh = torch.empty(rows, wide, device="cuda"), torch.randn(rows, wide, device="cuda", generator=gen)
    qa, qb = (torch.empty(rows, wide, dtype=torch.int8, device="cuda") for _ in range(2))
    sa, sb = (torch.empty(rows, wide // 128, device="cuda") for _ in range(2))
    dab = torch.empty_like(ab)
    dyp = [torch.empty(rows, cols, device="cuda") for _ in range(2)]
    dx, dw, db = torch.empty_like(res), torch.empty_like(w), torch.empty_like(b)
    ops = {
        "fold": emac.fold_init([p.data_ptr() for p in parts], [folded.data_ptr()], rows * cols, emac.FLOAT),
        "norm2": emac.layernorm_init(rows, cols, emac.FLOAT, [folded.data_ptr()], y2.data_ptr(), residual=res.data_ptr(), weight=w.data_ptr(), bias=b.data_ptr()),
        "norm": emac.layernorm_init(rows, cols, emac.FLOAT, [p.data_ptr() for p in parts], y.data_ptr(), residual=res.data_ptr(), weight=w.data_ptr(),
                                    bias=b.data_ptr(), sum=x.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr(), q=q.data_ptr(), scale=sc.data_ptr()),
        "act": emac.act_init(rows, wide, emac.FLOAT, emac.SILU, a.data_ptr(), h.data_ptr(), b=bb.data_ptr(), a_stride=2 * wide, b_stride=2 * wide,
                             qa=qa.data_ptr(), sa=sa.data_ptr(), qb=qb.data_ptr(), sb=sb.data_ptr()),
        "dact": emac.act_grad_init(rows, wide, emac.FLOAT, emac.SILU, dh.data_ptr(), qa.data_ptr(), sa.data_ptr(), dab.data_ptr(), qb=qb.data_ptr(),
                                   sb=sb.data_ptr(), db=dab[:, wide:].data_ptr(), da_stride=2 * wide, db_stride=2 * wide),
        "dnorm": emac.layernorm_grad_init(rows, cols, emac.FLOAT, [d.data_ptr() for d in dyp], mean.data_ptr(), rstd.data_ptr(), q=q.data_ptr(),
                                          scale=sc.data_ptr(), weight=w.data_ptr(), dx=dx.data_ptr(), dweight=dw.data_ptr(), dbias=db.data_ptr()),
    }
    for k in ops.values():
        emac.set_stream(k, s.cuda_stream)
    with torch.cuda.stream(s):
        for k in ("fold", "norm2", "norm"):
            emac.start(ops[k])
        torch.mm(y, W, out=ab)
        emac.start(ops["act"])
        emac.start(ops["dact"])
        torch.mm(dab[:, :wide], W[:, :wide].t().contiguous(), out=dyp[0])
        torch.mm(dab[:, wide:], W[:, wide:].t().contiguous(), out=dyp[1])
        emac.start(ops["dnorm"])
    for k in ops.values():
        emac.wait(k)
    assert torch.equal(y, y2) and torch.equal(x, ref.fold(parts, res))
    _, _, ry, by = ref.layernorm(x, w, b, 1e-5)
    ref.close(y, ry, by)
    xq = ref.restore8(*ref.save8(x))
    rdx, bdx, rdw, bdw, rdb, bdb = ref.layernorm_grad(dyp[0] + dyp[1], xq, mean, rstd, w, None)
    ref.close(dx, rdx, bdx)
    ref.close(dw, rdw, bdw)
    ref.close(db, rdb, bdb)
    for k in ops.values():
        emac.done(k)


def test_captured_and_replayed():
    """Starts captured into a graph and replayed with new inputs, eager work and eager Starts of other
    handles between the replays; two graphs of two handles on the same inputs."""
    rows, cols = 700, 1536
    x, dy = torch.empty(rows, cols, device="cuda"), torch.empty(rows, cols, device="cuda")
    s = torch.cuda.Stream()

    def make():
        o = {k: torch.empty(rows, cols, device="cuda") for k in ("y", "dx")}
        o.update(q=torch.empty(rows, cols, dtype=torch.int8, device="cuda"), sc=torch.empty(rows, 12, device="cuda"), mean=torch.empty(rows, device="cuda"),
                 rstd=torch.empty(rows, device="cuda"), dw=torch.empty(cols, device="cuda"), db=torch.empty(cols, device="cuda"))
        p = {k: v.data_ptr() for k, v in o.items()}
        f = emac.layernorm_init(rows, cols, emac.FLOAT, [x.data_ptr()], p["y"], mean=p["mean"], rstd=p["rstd"], q=p["q"], scale=p["sc"])
        g = emac.layernorm_grad_init(rows, cols, emac.FLOAT, [dy.data_ptr()], p["mean"], p["rstd"], q=p["q"], scale=p["sc"], dx=p["dx"], dweight=p["dw"],
                                     dbias=p["db"])
        return o, (f, g)

    (o1, h1), (o2, h2), (eager, he) = make(), make(), make()
    graphs = []
    for hs in (h1, h2):
        for h in hs:
            emac.set_stream(h, s.cuda_stream)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            for h in hs:
                emac.start(h)
        graphs.append(gr)
    for h in he:
        emac.set_stream(h, torch.cuda.current_stream().cuda_stream)
    for k in range(4):
        gen = rnd(50 + k)
        x.copy_(torch.randn(rows, cols, device="cuda", generator=gen))
        dy.copy_(torch.randn(rows, cols, device="cuda", generator=gen))
        for o in (o1, o2, eager):
            for v in o.values():
                v.zero_()
        graphs[0].replay()
        for h in he:
            emac.start(h)
        graphs[1].replay()
        torch.cuda.synchronize()
        for name in eager:
            assert torch.equal(o1[name], eager[name]) and torch.equal(o2[name], eager[name]), (k, name)
        assert float(eager["dw"].abs().max()) > 0
    del graphs
    for h in h1 + h2 + he:
        emac.done(h)


def test_streams():
    """The handle's own stream (made when first needed), the default stream, and a change of streams."""
    x = torch.randn(64, 512, device="cuda")
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    h = emac.layernorm_init(64, 512, emac.FLOAT, [x.data_ptr()], y.data_ptr())
    assert emac.test(h) == 1 and emac.wait(h) == 0
    emac.start(h)
    emac.wait(h)
    own = emac.stream(h)
    assert own and emac.test(h) == 1
    want = y.clone()
    s = torch.cuda.Stream()
    for stream in (0, s.cuda_stream, 0):
        y.zero_()
        torch.cuda.synchronize()
        emac.set_stream(h, stream)
        emac.start(h)
        assert (emac.stream(h) or 0) == stream
        emac.wait(h)
        assert torch.equal(y, want)
    emac.start_legs(h, emac.LEG_STAGE)  # no leg of it
    with pytest.raises(emac.ExtMpiError):
        emac.start_legs(h, emac.LEG_ALL | emac.LEG_STEP(0))
    emac.done(h)
    with pytest.raises(emac.ExtMpiError):
        emac.start(h)


ARG, UNSUPPORTED = emac.ERROR_ARG, emac.ERROR_UNSUPPORTED


def refused(code, f, *a, **kw):
    with pytest.raises(emac.ExtMpiError) as e:
        f(*a, **kw)
    assert e.value.code == code, (e.value.code, code)


def test_an_earlier_error_of_the_program_is_not_a_starts():
    x = torch.randn(4, 256, device="cuda", generator=rnd(3))
    y, q, scale, dw = torch.empty_like(x), torch.empty(4, 256, dtype=torch.int8, device="cuda"), torch.empty(4, 2, device="cuda"), torch.empty(256, device="cuda")
    mean, rstd = torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    hs = [emac.layernorm_init(4, 256, emac.FLOAT, [x.data_ptr()], y.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr()),
          emac.layernorm_grad_init(4, 256, emac.FLOAT, [x.data_ptr()], mean.data_ptr(), rstd.data_ptr(), x=x.data_ptr(), dweight=dw.data_ptr()),
          emac.save8_init(4, 256, emac.FLOAT, x.data_ptr(), q.data_ptr(), scale.data_ptr()),
          emac.act_init(4, 256, emac.FLOAT, emac.SILU, x.data_ptr(), y.data_ptr())]
    stream = torch.cuda.current_stream().cuda_stream
    for h in hs:
        emac.set_stream(h, stream)
    assert emac.lib().hipSetDevice(9999) != 0  # refused, and remembered by the runtime
    try:
        for h in hs:
            emac.start(h)
    finally:
        emac.lib().hipGetLastError()
    for h in hs:
        emac.wait(h)
        emac.done(h)
    assert torch.equal(q, ref.save8(x)[0])


def test_refusals_of_memory():
    x, y = torch.randn(64, 256, device="cuda"), torch.empty(64, 256, device="cuda")
    v, q, sc = torch.empty(300, device="cuda"), torch.empty(64, 256, dtype=torch.int8, device="cuda"), torch.empty(64, 2, device="cuda")
    host = torch.empty(64, 256)
    X, Y, V, Q, S = (t.data_ptr() for t in (x, y, v, q, sc))
    F = emac.FLOAT
    ln, gr = emac.layernorm_init, emac.layernorm_grad_init
    refused(ARG, ln, 64, 256, F, [host.data_ptr()], Y)
    refused(ARG, ln, 64, 256, F, [X], host.data_ptr())
    refused(ARG, ln, 64, 256, F, [X + 2], Y)                      # not at an element
    refused(ARG, ln, 64, 256, F, [None], Y)
    refused(ARG, ln, 64, 256, F, [X], None)                       # no output
    refused(ARG, ln, 64, 256, F, [X], Y, src_stride=255)
    refused(ARG, ln, 64, 256, F, [X], Y, y_stride=-1)
    refused(ARG, ln, 64, 256, F, [X], Y, q=Q)                     # a checkpoint without scales
    refused(ARG, ln, 64, 256, F, [X], Y, q=Q, scale=S, q_stride=255)
    refused(ARG, ln, 64, 256, F, [X], Y, eps=-1.0)
    refused(ARG, ln, 64, 256, F, [X], Y, eps=math.nan)
    refused(ARG, ln, 64, 256, F, [X], Y, eps=math.inf)
    refused(ARG, ln, 32, 256, F, [X], X + 1024)                   # overlaps its input, not in place
    refused(ARG, ln, 32, 128, F, [X], X, src_stride=256, y_stride=128)
    refused(ARG, ln, 64, 256, F, [X], Y, sum=Y)                   # two outputs in one place
    refused(ARG, ln, 64, 256, F, [X], Y, mean=V, rstd=V + 4)
    refused(ARG, ln, 64, 256, F, [X], Y, weight=Y)
    refused(ARG, gr, 64, 256, F, [X], V, V, dx=Y)                 # neither x nor a checkpoint
    refused(ARG, gr, 64, 256, F, [X], V, V, x=X, q=Q, scale=S, dx=Y)
    refused(ARG, gr, 64, 256, F, [X], V, V, q=Q, dx=Y)
    refused(ARG, gr, 64, 256, F, [X], V, V, x=X)                  # no output
    refused(ARG, gr, 64, 256, F, [X], None, V, x=X, dx=Y)
    refused(ARG, gr, 64, 256, F, [X], V, V, x=X, dx=Y, dweight=V)
    refused(ARG, gr, 64, 256, F, [X], V, V, x=X, dx=Y, y=X)       # y is no in-place output
    refused(ARG, emac.save8_init, 64, 256, F, X, X, S)
    refused(ARG, emac.save8_init, 64, 256, F, X, Q, None)
    refused(ARG, emac.restore8_init, 64, 256, F, Q, S, Q)
    act, dact = emac.act_init, emac.act_grad_init
    refused(ARG, act, 64, 256, F, emac.SILU, X)                   # no output
    refused(ARG, act, 64, 256, F, emac.SILU, X, Y, b=X, qa=Q, sa=S)  # the gate's checkpoint is missing
    refused(ARG, act, 64, 256, F, emac.SILU, X, Y, qb=Q, sb=S)
    refused(ARG, act, 64, 256, F, 3, X, Y)
    refused(ARG, dact, 64, 256, F, emac.SILU, X, Q, S, None)
    refused(ARG, dact, 64, 256, F, emac.SILU, X, Q, S, Y, qb=Q, sb=S)
    refused(ARG, dact, 64, 256, F, emac.SILU, X, Q, None, Y)
    # the halves of one matrix's rows are not an overlap
    ab = torch.randn(64, 512, device="cuda")
    h = act(64, 256, F, emac.SILU, ab.data_ptr(), ab[:, 256:].data_ptr(), a_stride=512, h_stride=512)
    emac.done(h)
    refused(ARG, act, 64, 256, F, emac.SILU, ab.data_ptr(), ab[:, 255:].data_ptr(), a_stride=512, h_stride=512)


def gradient(dys, x, mean, rstd, dx=None, gt=torch.float32, **kw):
    """dx (a new matrix unless given), dweight and dbias in type gt, of contiguous rows."""
    rows, cols = x.shape
    dx = torch.empty_like(x) if dx is None else dx
    dw, db = torch.empty(cols, dtype=gt, device="cuda"), torch.empty(cols, dtype=gt, device="cuda")
    go(emac.layernorm_grad_init(rows, cols, CODE[x.dtype], [d.data_ptr() for d in dys], mean.data_ptr(), rstd.data_ptr(), x=x.data_ptr(), dx=dx.data_ptr(),
                                dweight=dw.data_ptr(), dbias=db.data_ptr(), gdtype=CODE[gt], **kw))
    return dx, dw, db


@pytest.mark.parametrize("nsrc", [1, 2])
@pytest.mark.parametrize("rows,cols", [(300, 5), (300, 64), (1001, 131), (333, 200), (70001, 40), (1025, 512)])
def test_rows_past_the_last_add_nothing(rows, cols, nsrc):
    """Rows side by side in a workgroup that the last workgroup does not fill, and an infinity in the last
    row: its column's sum is that infinity, all others are finite."""
    gen = rnd(rows + cols)
    x, dy = (torch.randn(rows, cols, device="cuda", generator=gen) for _ in range(2))
    mean, rstd = x.mean(1), (x.var(1, unbiased=False) + 1e-5).rsqrt()
    x[-1, 3], dy[-1, 3] = math.inf, 1.0
    _, dw, db = gradient([dy] * nsrc, x, mean, rstd)
    want = torch.zeros(cols, dtype=torch.bool, device="cuda")
    want[3] = True
    assert torch.equal(dw == math.inf, want) and torch.equal(dw.isfinite(), ~want) and bool(db.isfinite().all())


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("nsrc", [1, 2])
@pytest.mark.parametrize("rows,cols", [(5, 7), (29, 1024), (200, 300), (300, 5), (300, 64), (1001, 131), (333, 200), (70001, 40), (1025, 512), (700, 1000),
                                       (600, 4099), (300, 9000), (9, 20001), (400, 20001)])
def test_dx_over_x(rows, cols, nsrc, t):
    """dx in place of x: the same bits as beside it, where the last row's dx overflows its type and dweight's
    columns do not (fp16: g about 2^12 at an rstd of 2^9 gives 2^21 where 2^16 overflows; g xh is about 2^12 in
    32 bits)."""
    dt, gen = ref.TYPES[t], rnd(rows + cols + nsrc)
    x = torch.randn(rows, cols, device="cuda", generator=gen).to(dt)
    dys = [torch.randn(rows, cols, device="cuda", generator=gen).to(dt) for _ in range(nsrc)]
    mean, rstd = x.float().mean(1), (x.float().var(1, unbiased=False) + 1e-5).rsqrt()
    x[-1] /= 512
    mean[-1], rstd[-1] = mean[-1] / 512, rstd[-1] * 512
    dys[0][-1] *= 4096
    kept = gradient(dys, x, mean, rstd)
    x2 = x.clone()
    over = gradient(dys, x2, mean, rstd, dx=x2)
    if t == "f16":
        assert bool(kept[0][-1].isinf().any())
    assert bool(kept[1].isfinite().all()) and bool(kept[2].isfinite().all())
    for a, b in zip(over, kept):
        assert torch.equal(a, b)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nsrc", [1, 2])
@pytest.mark.parametrize("rows,cols", [(20, 5), (300, 7), (40, 100), (600, 100), (50, 129), (500, 500), (30, 1024), (600, 1027), (500, 5000), (400, 9001),
                                       (300, 13000), (8, 20001), (300, 20001)])
def test_rows_with_a_large_mean(rows, cols, nsrc, t):
    """Rows a thousand deviations from zero. (x - mean) * rstd is off by a rounding of the difference and one of the
    product, 2 U of its own size (3 U are counted): no rounding is of the size of x or of mean * rstd. From a checkpoint too,
    whose restored values are fixed to the bit."""
    dt, gen = ref.TYPES[t], rnd(rows + cols)
    x = (torch.randn(rows, cols, device="cuda", generator=gen) + 1000).to(dt)
    dys = [torch.randn(rows, cols, device="cuda", generator=gen).to(dt) for _ in range(nsrc)]
    w = torch.randn(cols, device="cuda", generator=gen)
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    q, scale = torch.empty(rows, cols, dtype=torch.int8, device="cuda"), torch.empty(rows, -(-cols // 128), device="cuda")
    go(emac.layernorm_init(rows, cols, CODE[dt], [x.data_ptr()], y.data_ptr(), weight=w.data_ptr(), wdtype=emac.FLOAT, mean=mean.data_ptr(),
                           rstd=rstd.data_ptr(), q=q.data_ptr(), scale=scale.data_ptr()))
    rmean, _, ry, by = ref.layernorm(x, w, None, 1e-5)
    ref.close(y, ry, by)
    ref.close(mean, rmean, ref.stats_bounds(x, rstd.double())[0])
    rq, rscale = ref.save8(x)
    assert torch.equal(q, rq) and torch.equal(scale, rscale)
    g = dys[0].float()
    for d in dys[1:]:
        g = g + d.float()
    for xv, kw in ((x, {"x": x.data_ptr()}), (ref.restore8(rq, rscale), {"q": q.data_ptr(), "scale": scale.data_ptr()})):
        dx, dw, db = torch.empty_like(x), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
        go(emac.layernorm_grad_init(rows, cols, CODE[dt], [d.data_ptr() for d in dys], mean.data_ptr(), rstd.data_ptr(), dx=dx.data_ptr(),
                                    dweight=dw.data_ptr(), dbias=db.data_ptr(), weight=w.data_ptr(), wdtype=emac.FLOAT, gdtype=emac.FLOAT, **kw))
        rdx, bdx, rdw, bdw, rdb, bdb = ref.layernorm_grad(g, xv, mean, rstd, w, None, exh=3 * ref.U)
        ref.close(dx, rdx, bdx)
        ref.close(dw, rdw, bdw)
        ref.close(db, rdb, bdb)


def test_the_most_blocks():
    """As many blocks as are taken, of one column each."""
    rows = emac.BLOCKS8_MAX
    x = torch.randint(0, 2, (rows, 1), dtype=torch.int8, device="cuda", generator=rnd(9)).mul_(2).sub_(1)
    t = x.to(torch.bfloat16)
    q, scale = torch.empty(rows, 1, dtype=torch.int8, device="cuda"), torch.empty(rows, 1, device="cuda")
    go(emac.save8_init(rows, 1, emac.BF16, t.data_ptr(), q.data_ptr(), scale.data_ptr()))
    assert torch.equal(q, x.mul_(127))
    t.zero_()
    go(emac.restore8_init(rows, 1, emac.BF16, q.data_ptr(), scale.data_ptr(), t.data_ptr()))
    assert torch.equal(t.to(torch.int8).mul_(127), x)


@pytest.mark.parametrize("name", ["norm_prefill", "grad_batch"])
def test_a_pass_of_the_cases_follows_the_current_stream(name):
    """perf/operators.py: handles prepared on one stream, a pass under another, behind a late producer of its inputs."""
    spec = importlib.util.spec_from_file_location("operators_own", os.path.join(os.path.dirname(emac.HERE), "perf", "operators.py"))
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    ops.own = True
    state = ops.prepare(next(c for c in ops.listed() if c["name"] == name), 1)
    want = {k: v.clone() for k, v in ops.run(state).items()}
    src = state["in"]["src" if name == "norm_prefill" else "dy"][0]
    kept = src.clone()
    src.zero_()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(200_000_000)
        src.copy_(kept)
        got = {k: v.clone() for k, v in ops.run(state).items()}
    s.synchronize()
    for k in want:
        assert torch.equal(got[k], want[k])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("w32", [False, True])
@pytest.mark.parametrize("rows,cols", WIDTHS)
def test_one_leaf_over_many_rows(rows, cols, w32, t):
    """One leaf, more rows than workgroups, against the definitions: the norm with a residual (and without weights, one
    leaf alone), its gradient with dsum from x and from the checkpoint, without the norm's output again."""
    dt, gen = ref.TYPES[t], rnd(rows + cols + w32)
    wt = torch.float32 if w32 else dt
    src, res, dy, dsum = (torch.randn(rows, cols, device="cuda", generator=gen).to(dt) for _ in range(4))
    w, b = (torch.randn(cols, device="cuda", generator=gen).to(wt) for _ in range(2))
    x, y = torch.empty_like(src), torch.empty_like(src)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    kw = dict(mean=mean.data_ptr(), rstd=rstd.data_ptr())
    for r in (None, res):
        ww, bb = (None, None) if r is None else (w, b)
        more = {} if r is None else dict(residual=r.data_ptr(), sum=x.data_ptr(), weight=w.data_ptr(), bias=b.data_ptr(), wdtype=CODE[wt])
        go(emac.layernorm_init(rows, cols, CODE[dt], [src.data_ptr()], y.data_ptr(), **kw, **more))
        want = ref.fold([src], r)
        assert r is None or torch.equal(x, want)
        rmean, rrstd, ry, by = ref.layernorm(want, ww, bb, 1e-5)
        bmean, brstd = ref.stats_bounds(want, rrstd)
        ref.close(mean, rmean, bmean)
        ref.close(rstd, rrstd, rrstd * brstd)
        ref.close(y, ry, by)
        del want, ry, by
    q, scale = ref.save8(x)
    dx, dw, db = torch.empty_like(x), torch.empty(cols, dtype=wt, device="cuda"), torch.empty(cols, dtype=wt, device="cuda")
    for xv, kw in ((x, {"x": x.data_ptr()}), (ref.restore8(q, scale), {"q": q.data_ptr(), "scale": scale.data_ptr()})):
        for o in (dx, dw, db):
            o.fill_(7.0)
        go(emac.layernorm_grad_init(rows, cols, CODE[dt], [dy.data_ptr()], mean.data_ptr(), rstd.data_ptr(), weight=w.data_ptr(), wdtype=CODE[wt],
                                    dsum=dsum.data_ptr(), dx=dx.data_ptr(), dweight=dw.data_ptr(), dbias=db.data_ptr(), gdtype=CODE[wt], **kw))
        rdx, bdx, rdw, bdw, rdb, bdb = ref.layernorm_grad(dy, xv, mean, rstd, w, dsum, exh=3 * ref.U)
        ref.close(dx, rdx, bdx)
        ref.close(dw, rdw, bdw)
        ref.close(db, rdb, bdb)
        del rdx, bdx, rdw, bdw, rdb, bdb


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(3, 5), (40, 300), (700, 300), (600, 4100), (20, 20000), (300, 20000)])
def test_added_to_in_16_bits(rows, cols, t):
    """accumulate with gradients in 16 bits: what was there and the sum are added in 32 bits and rounded once."""
    dt, gen = ref.TYPES[t], rnd(rows)
    x, dy = (torch.randn(rows, cols, device="cuda", generator=gen).to(dt) for _ in range(2))
    mean, rstd = x.float().mean(1), (x.float().var(1, unbiased=False) + 1e-5).rsqrt()
    dw0, db0 = ((torch.randn(cols, device="cuda", generator=gen) * 20).to(dt) for _ in range(2))
    dw, db = dw0.clone(), db0.clone()
    go(emac.layernorm_grad_init(rows, cols, CODE[dt], [dy.data_ptr()], mean.data_ptr(), rstd.data_ptr(), x=x.data_ptr(), dweight=dw.data_ptr(),
                                dbias=db.data_ptr(), accumulate=True))
    _, _, rdw, bdw, rdb, bdb = ref.layernorm_grad(dy, x, mean, rstd, None, None, exh=3 * ref.U)
    for got, was, r, bound in ((dw, dw0, rdw, bdw), (db, db0, rdb, bdb)):
        ref.close(got, was.double() + r, bound + ref.U * (was.double().abs() + r.abs() + bound))


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("kind", list(KINDS))
def test_act_at_its_ends_in_16_bits(kind, t):
    """Far tails and the largest values: the definition where it is in reach of the type, a itself far above zero, zero
    far below it, a slope of 1 and of 0 there."""
    dt = ref.TYPES[t]
    top = float(torch.finfo(dt).max)
    a = torch.tensor([[0.0, -0.0, 1e-4, -1e-4, 3.0, -3.0, 9.0, -9.0, 14.0, -14.0, 40.0, -40.0, 100.0, -100.0, 1e4, -1e4, top, -top]], device="cuda").to(dt)
    n = a.shape[1]
    h, da, dh = torch.empty_like(a), torch.empty_like(a), torch.ones_like(a)
    go(emac.act_init(1, n, CODE[dt], KINDS[kind], a.data_ptr(), h.data_ptr()))
    v, _, bv, _ = ref.act(kind, a[:, :12])
    ref.close(h[:, :12], v, bv)
    assert torch.equal(h[0, 12::2], a[0, 12::2]) and bool((h[0, 13::2] == 0).all())
    back = torch.empty(1, n, device="cuda")
    for j in range(n):  # each value a block of its own
        one = a[:, j:j + 1].float()
        q, s = ref.save8(one)
        back[:, j:j + 1] = ref.restore8(q, s)
        go(emac.act_grad_init(1, 1, CODE[dt], KINDS[kind], dh[:, j:].data_ptr(), q.data_ptr(), s.data_ptr(), da[:, j:].data_ptr()))
    _, slope, _, bslope = ref.act(kind, back[:, :12])
    ref.close(da[:, :12], slope, bslope + 4 * ref.U * slope.abs())
    assert bool((da[0, 12::2] == 1).all()) and bool((da[0, 13::2] == 0).all())
