"""W8A8 entry points: what they refuse, without a GPU (nothing is launched)."""
import pytest

from vllm_rs_amd import _lib, ops

P = 4096  # a pointer that nothing reads
BF16, F16, F32 = 0, 1, 2


def refused(fn, *args):
    L = _lib.load()
    L.vra_clear_error()
    getattr(L, fn)(*args)
    msg = L.vra_last_error().decode()
    L.vra_clear_error()
    return msg


@pytest.mark.parametrize("args, why", [
    ((P, P, P, -1, 64, BF16, 0), "rows >= 0"), ((P, P, P, 1, 0, BF16, 0), "columns"), ((P, P, P, 1, 131073, BF16, 0), "columns"),
    ((P, P, P, 1, 64, F32, 0), "dtype"), ((P, P, P, 1, 64, 7, 0), "dtype"), ((None, P, P, 1, 64, BF16, 0), "null"), ((P, None, P, 1, 64, F16, 0), "null"),
    ((P, P, None, 1, 64, BF16, 0), "null"), ((P + 1, P, P, 1, 64, BF16, 0), "multiple"), ((P, P, P + 2, 1, 64, BF16, 0), "multiple")])
def test_rows(args, why):
    assert why in refused("vra_quant_rows_i8", *args)


def test_norms():
    ok = [P, P, P, P, 1, 64, 1e-5, BF16, 0]
    for i in range(4):
        assert "null" in refused("vra_rms_norm_i8", *ok[:i], None, *ok[i + 1:])
    assert "multiple" in refused("vra_rms_norm_i8", P, P + 1, P, P, 1, 64, 1e-5, BF16, 0)
    assert "dtype" in refused("vra_rms_norm_i8", P, P, P, P, 1, 64, 1e-5, F32, 0)
    ok = [P] * 6 + [1, 64, 1e-5, F16, 0]
    for i in range(6):
        assert "null" in refused("vra_add_rms_norm_i8", *ok[:i], None, *ok[i + 1:])
    for i in (0, 1, 2, 3, 5):
        assert "multiple" in refused("vra_add_rms_norm_i8", *ok[:i], P + 1, *ok[i + 1:])
    assert "columns" in refused("vra_add_rms_norm_i8", *[P] * 6, 1, 200000, 1e-5, F16, 0)


def test_products():
    def gemm(x=P, xs=P, w=P, ws=P, bias=None, residual=None, out=P, work=None, m=4, k=64, n=32, dt=BF16):
        return refused("vra_w8a8_gemm", x, xs, w, ws, bias, residual, out, work, m, k, n, dt, 0)

    for name in ("x", "xs", "w", "ws", "out"):
        assert "null" in gemm(**{name: None})
    for bad in (dict(m=-1), dict(k=0), dict(n=0), dict(k=131072), dict(n=(1 << 24) + 1)):
        assert "131071" in gemm(**bad)
    assert "dtype" in gemm(dt=3)
    for bad in (dict(xs=P + 2), dict(ws=P + 1), dict(bias=P + 1), dict(residual=P + 1), dict(out=P + 1), dict(out=P + 2, dt=F32), dict(bias=P + 2, dt=F32)):
        assert "multiple" in gemm(**bad)
    assert "workspace" in gemm(work=P + 8)

    def pair(x=P, xs=P, g=P, sg=P, u=P, su=P, out=P, work=None, m=4, k=64, n=32, dt=BF16):
        return refused("vra_w8a8_gate_up_silu", x, xs, g, sg, u, su, out, work, m, k, n, dt, 0)

    for name in ("x", "xs", "g", "sg", "u", "su", "out"):
        assert "null" in pair(**{name: None})
    assert "dtype" in pair(dt=F32)
    assert "131071" in pair(k=140000)
    assert "multiple" in pair(su=P + 2) and "workspace" in pair(work=P + 4)


def test_no_rows_is_no_work():
    for fn, args in (("vra_quant_rows_i8", (None, None, None, 0, 64, BF16, 0)), ("vra_rms_norm_i8", (None,) * 4 + (0, 64, 1e-5, BF16, 0)),
                     ("vra_add_rms_norm_i8", (None,) * 6 + (0, 64, 1e-5, BF16, 0)), ("vra_w8a8_gemm", (None,) * 8 + (0, 64, 32, BF16, 0)),
                     ("vra_w8a8_gate_up_silu", (None,) * 8 + (0, 64, 32, BF16, 0))):
        assert refused(fn, *args) == ""


def test_workspace_size():
    assert ops.lib().vra_w8a8_workspace_bytes() >= 16


def code(kind, size, slices=1):
    return slices << 16 | kind << 8 | size


def test_named_kernels():
    def on(kernel, pair=False, x=P, bias=None, work=None, m=40, k=1024, n=512):
        return refused("vra_w8a8_gemm_on", kernel, x, P, P, P, P if pair else None, P if pair else None, bias, None, P, work, m, k, n, BF16, 0)

    for bad in (code(0, 0), code(0, 0x12), code(0, 0x22, 3), code(3, 0), code(1, 3), code(1, 8), code(1, 4, 3), code(2, 0x11), code(2, 0x44, 2), code(2, 0x12, 16), -1, 0):
        assert "no such kernel" in on(bad, work=P)
    assert "no such kernel" in on(code(1, 1, 2))  # slices without a workspace
    assert "no such kernel" in on(code(1, 1), m=65) and "no such kernel" in on(code(1, 4), m=33)
    assert "no such kernel" in on(code(1, 1), pair=True) and "no such kernel" in on(code(0, 0x11), pair=True, bias=P)
    assert "no such kernel" in on(code(2, 0x22), k=1000) and "no such kernel" in on(code(2, 0x22), x=P + 4) and "no such kernel" in on(code(1, 2), k=1000)
    assert "no such kernel" in on(code(1, 1, 8), work=P, k=1008)  # runs without a step
    assert "no such kernel" in on(code(2, 0x12, 2), work=P, m=8192, n=8192)  # more tiles than the workspace has counters for
    assert "null" in on(code(0, 0x11), x=None)


def test_kernel_choice():
    pick = lambda pair, m, k, n, ws=1: _lib.load().vra_w8a8_kernel(pair, m, k, n, ws)
    kind = lambda c: c >> 8 & 255
    assert pick(0, 0, 64, 64) == 0 and pick(0, 1, 131072, 64) == 0 and pick(1, 5, 64, 0) == 0
    for m in (1, 4, 16, 17, 64, 65, 150, 1021, 8192):
        for k, n in ((4096, 6144), (14336, 4096), (3584, 32000), (128, 64), (16, 1), (1000, 300)):
            for pair in (0, 1):
                c, alone = pick(pair, m, k, n), pick(pair, m, k, n, 0)
                assert alone >> 16 == 1 and c >> 16 in (1, 2, 4, 8)
                if k % 16:
                    assert kind(c) == (0 if m > 64 else kind(c)) < 2
                else:
                    assert kind(c) == (1 if m <= 16 else 2 if m > 64 else kind(c))
    assert pick(0, 8192, 14336, 4096) == code(2, 0x44) and pick(0, 1, 14336, 4096) == code(1, 1) and pick(0, 16, 3584, 32000) == code(1, 4)
    assert pick(0, 64, 14336, 4096) >> 16 > 1 and pick(0, 64, 14336, 4096, 0) >> 16 == 1
