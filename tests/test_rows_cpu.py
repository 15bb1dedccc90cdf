"""The row operators without a GPU: refusals that come before any device is asked for, the test of two
matrices for shared bytes, and the oracle's own checkpoint against the definition in 64 bits."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

import ext_mpi_collectives_amd as emac
import rows_ref as ref

ARG, UNSUPPORTED = emac.ERROR_ARG, emac.ERROR_UNSUPPORTED


def code_of(f, *a, **kw):
    with pytest.raises(emac.ExtMpiError) as e:
        f(*a, **kw)
    return e.value.code


CALLS = [
    (lambda r, c, t: emac.layernorm_init(r, c, t, [64], 64)),
    (lambda r, c, t: emac.layernorm_grad_init(r, c, t, [64], 64, 64, x=64, dx=64)),
    (lambda r, c, t: emac.save8_init(r, c, t, 64, 64, 64)),
    (lambda r, c, t: emac.restore8_init(r, c, t, 64, 64, 64)),
    (lambda r, c, t: emac.act_init(r, c, t, emac.GELU, 64, 64)),
    (lambda r, c, t: emac.act_grad_init(r, c, t, emac.GELU, 64, 64, 64, 64)),
]


@pytest.mark.parametrize("call", range(len(CALLS)))
def test_refusals_before_the_device(call):
    f = CALLS[call]
    assert code_of(f, -1, 8, emac.FLOAT) == ARG
    assert code_of(f, 1, 0, emac.FLOAT) == ARG
    assert code_of(f, 1, -8, emac.FLOAT) == ARG
    assert code_of(f, 1, 8, 6) == ARG and code_of(f, 1, 8, -1) == ARG
    for t in (emac.DOUBLE, emac.LONG, emac.INT):
        assert code_of(f, 1, 8, t) == UNSUPPORTED
    assert code_of(f, 1, (1 << 30) + 1, emac.FLOAT) == UNSUPPORTED
    if call < 2:
        assert code_of(f, 1, emac.ROW_COLS_MAX + 1, emac.FLOAT) == UNSUPPORTED
    if not torch.cuda.is_available():
        assert code_of(f, 1, 8, emac.FLOAT) == emac.ERROR_DEVICE  # and no answer from the CPU


def test_null_descriptors():
    L, h = emac.lib(), ctypes.c_int(-1)
    for name, desc in (("layernorm", emac.LayernormDesc), ("layernorm_grad", emac.LayernormGradDesc), ("act", emac.ActDesc),
                       ("act_grad", emac.ActGradDesc)):
        f = getattr(L, f"ext_mpi_amd_{name}_init")
        assert f(None, ctypes.byref(h)) == ARG
        assert f(ctypes.byref(desc()), None) == ARG
    assert L.ext_mpi_amd_save8_init(1, 8, emac.FLOAT, None, 0, None, 0, None, None) == ARG
    with pytest.raises(ValueError):
        emac.layernorm_init(1, 8, emac.FLOAT, [], 64)
    with pytest.raises(ValueError):
        emac.layernorm_init(1, 8, emac.FLOAT, [64] * 17, 64)


def test_the_allreduce_handles_refuse_the_new_types():
    for t in (emac.BF16, emac.HALF):
        assert code_of(emac.plan_describe, 2, 64, t, "6;1 -2 2", 0) == ARG


def test_shared_bytes():
    """Against the sets of bytes themselves."""
    f = emac.lib().ext_mpi_amd_check_rows_share
    f.argtypes = [ctypes.c_long] * 8
    f.restype = ctypes.c_int
    cells = lambda p, rows, ln, ld: {p + r * ld + k for r in range(rows) for k in range(ln)}  # noqa: E731
    for rows_a in (1, 2, 5):
        for rows_b in (1, 2, 5):
            for len_a in (1, 3, 8):
                for len_b in (1, 4, 8):
                    for b in range(0, 70):
                        a, ld = 20, 8
                        shared = bool(cells(a, rows_a, len_a, ld) & cells(b, rows_b, len_b, ld))
                        got = bool(f(a, rows_a, len_a, ld, b, rows_b, len_b, ld))
                        assert got or not shared, (rows_a, rows_b, len_a, len_b, b)
                        if rows_a == rows_b == 5 and len_a + len_b <= ld and not shared:
                            assert not got, (len_a, len_b, b)  # interleaved rows are told apart
    assert f(0, 4, 8, 16, 8, 4, 8, 32) == 1   # other strides that cross: refused
    assert f(0, 4, 8, 16, 4096, 4, 8, 32) == 0


def test_oracle_checkpoint():
    """The oracle's bytes are the nearest of the definition's values, its scale within a rounding. Beyond the
    half step a / 254: 127 / a and its product with x are off by U each of up to 127 steps, 2 U a; 1 / 127
    and its product with a by U each, 2 U a; the restored product by U a."""
    for t in ref.TYPES.values():
        x = (torch.randn(7, 300, generator=torch.Generator().manual_seed(1)) * 3).to(t)
        x[2], x[3, 5] = 0, 1000.0
        q, s = ref.save8(x)
        back = ref.restore8(q, s).double()
        a = torch.zeros(7, 384).double()
        a[:, :300] = x.double().abs()
        a = a.view(7, 3, 128).amax(2)
        assert bool(((s.double() * 127 - a).abs() <= 3 * ref.U * a + 2.0 ** -99).all())
        lim = a.repeat_interleave(128, 1)[:, :300] * (1 / 254 + 5 * ref.U) + 2.0 ** -107
        assert bool(((back - x.double()).abs() <= lim).all())
        assert int(q.abs().max()) == 127 and not bool(q[2].any())
    x = torch.ones(1, 256)
    x[0, 3] = math.nan
    q, s = ref.save8(x)
    assert math.isnan(float(s[0, 0])) and not bool(q[0, :128].any()) and float(s[0, 1]) > 0


def test_struct_layouts():
    """The ctypes structures are the header's, byte for byte (8-byte pointers and longs, 4-byte ints)."""
    assert ctypes.sizeof(emac.LayernormDesc) == 16 + 16 + 16 * 8 + 15 * 8
    assert ctypes.sizeof(emac.LayernormGradDesc) == 16 + 24 + 16 * 8 + 18 * 8
    assert ctypes.sizeof(emac.ActDesc) == 24 + 11 * 8
    assert ctypes.sizeof(emac.ActGradDesc) == 24 + 13 * 8


@pytest.fixture(scope="module")
def host_check(tmp_path_factory):
    """tests/rows_host_check.c over the engine's own sources."""
    here = os.path.dirname(os.path.abspath(__file__))
    src, exe = os.path.join(here, "..", "ext_mpi_collectives_amd", "csrc"), str(tmp_path_factory.mktemp("rows") / "check")
    units = [os.path.join(src, f"{u}.c") for u in ("engine", "engine_rows", "engine_tune", "engine_node", "engine_comm", "engine_ipc", "engine_join", "plan", "layout")]
    subprocess.run(["gcc", "-O1", "-g", "-std=gnu11", "-w", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + os.path.join(src, "..", "..", "include"), "-I" + src,
                    "-o", exe, os.path.join(here, "rows_host_check.c"), *units, "-no-pie", "-Wl,--unresolved-symbols=ignore-all"], check=True)

    def run(what):
        r = subprocess.run([exe, what], capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, r.stdout + r.stderr
    return run


def test_the_default_stream_of_another_device(host_check):
    """Start, Test, Wait, set_stream and Done of a handle on its device's default stream, another device current."""
    host_check("default_stream")


def test_a_stream_of_another_device_is_refused(host_check):
    """The handle keeps the stream it had."""
    host_check("other_stream")


def test_eps_is_a_floats(host_check):
    """An eps that a float takes for 0 or for an infinity is refused, like a negative one."""
    host_check("eps")


@pytest.mark.parametrize("call", range(2, len(CALLS)))
def test_the_most_columns_and_blocks(call):
    """Checkpoints and activations: the header's limits are the last sizes that are not refused as too large."""
    f, t = CALLS[call], emac.FLOAT
    text = open(os.path.join(os.path.dirname(emac.HERE), "include", "ext_mpi_amd.h")).read()
    assert "#define EXT_MPI_AMD_COLS8_MAX (1L << 30)" in text and "#define EXT_MPI_AMD_BLOCKS8_MAX ((1L << 31) - 4096)" in text
    assert (emac.COLS8_MAX, emac.BLOCKS8_MAX) == (1 << 30, (1 << 31) - 4096)
    for cols in (1, 127, 128, 129, 1000, emac.COLS8_MAX):
        most = emac.BLOCKS8_MAX // -(-cols // 128)
        assert code_of(f, most + 1, cols, t) == UNSUPPORTED
        assert code_of(f, 1 << 40, cols, t) == UNSUPPORTED
        assert code_of(f, most, cols, t) != UNSUPPORTED  # no device, or no memory at the addresses
    assert code_of(f, 1, emac.COLS8_MAX + 1, t) == UNSUPPORTED


def test_the_normal_tail():
    """The polynomial that GELU's kernels take for erfcx(|a| / sqrt 2) / 2, against it. In 64 bits it is off by the fit
    alone, 1.6e-7 (the figure beside the kernel; 2.7 U). In 32 bits, with a reciprocal within a step, 1 + c a and its
    reciprocal put 3 U into t, and t P'(t) / P(t) is under 2.6: 7.8 U; eight multiply-adds round at most 8 U of the sum of
    the terms' magnitudes, which is under 1.7 P: 13.6 U; one product more: 25.1 U with the fit."""
    f = emac.lib().ext_mpi_amd_check_gelu_tail
    f.argtypes, f.restype = [ctypes.c_int], ctypes.c_double
    at, c = f(0), [f(k) for k in range(1, 9)]
    a = torch.linspace(0, 12 * math.sqrt(2), 400001, dtype=torch.float64)
    want = torch.special.erfcx(a / math.sqrt(2)) / 2

    def tail(t):
        p = torch.full_like(t, c[0])
        for k in c[1:]:
            p = p * t + k
        return p * t

    assert float((tail(1 / (1 + at * a)) / want - 1).abs().max()) < 1.6e-7
    b = a.float()
    want = torch.special.erfcx(b.double() / math.sqrt(2)) / 2
    assert float((tail(1 / (1 + at * b)).double() / want - 1).abs().max()) < 25.1 * ref.U


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_a_fold_of_16_bits_is_a_value_error(dt):
    """The call with the code of bfloat16 or half raises what is a ValueError and an ExtMpiError."""
    for f in (lambda t: emac.fold_init([64], [64], 8, t), lambda t: emac.node_allreduce_init([64], [64], 8, t),
              lambda t: emac.allreduce_init(64, 64, 8, t, 0), lambda t: emac.node_comm_allreduce_init([64], [64], 8, t, 0),
              lambda t: emac.plan_describe(2, 64, t, "6;1 -2 2", 0), lambda t: emac.comm_program(2, 0, 64, t)):
        with pytest.raises(ValueError):
            f(emac.dtype_code(dt))
        assert code_of(f, emac.dtype_code(dt)) == ARG
