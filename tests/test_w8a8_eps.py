"""The RMS norms with 8-bit output: rows of zeros whatever eps is, and the eps that they refuse."""
import numpy as np
import pytest

from tests import w8a8_plain as plain
from tests.util import BF16, F16, rng
from vllm_rs_amd import _lib, ops


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6])
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("cols", [1, 7, 333, 1024, 4096, 9000, 33000])
def test_rows_of_zeros(cols, dt, eps):
    """padding rows (zeros, zeros of both signs, a sum that cancels) between others: codes 0 and scale 0; the others as the definition has them"""
    r, eps = rng(cols + dt), float(np.float32(eps))
    x, w = plain.to(r.standard_normal((5, cols)), dt), plain.to(1 + 0.2 * r.standard_normal(cols), dt)
    x[1], x[3] = 0, plain.to(np.where(np.arange(cols) % 2, -0.0, 0.0), dt)
    zero = [1, 3]
    q, s = ops.rms_norm_i8(ops.dev(x), ops.dev(w), 5, cols, eps, dt)
    check(x, w, eps, dt, q.numpy(np.int8, (5, cols)), s.numpy(np.float32, (5,)), zero)
    res = np.zeros_like(x)
    res[4] = x[4] ^ 0x8000  # x + residual = 0
    h, q, s = ops.add_rms_norm_i8(ops.dev(x), ops.dev(res), ops.dev(w), 5, cols, eps, dt)
    hb = h.numpy(np.uint16, (5, cols))
    assert not (hb[4] & 0x7FFF).any()
    check(hb, w, eps, dt, q.numpy(np.int8, (5, cols)), s.numpy(np.float32, (5,)), zero + [4])


def check(h, w, eps, dt, q, s, zero):
    assert not q[zero].any() and (s[zero] == 0.0).all(), f"scales of zero rows: {s[zero]}"
    rest = [t for t in range(len(h)) if t not in zero]
    ref, want = plain.rms_norm(h[rest], w, eps, dt)
    assert np.array_equal(q[rest], ref)
    plain.assert_within(s[rest].astype(np.float64), want, plain.SCALE * np.abs(want) + 2.0 ** -149, "scales")


@pytest.mark.parametrize("eps", [-1e-6, -1.0, float("nan"), float("-inf")])
def test_refused(eps):
    """(null pointers: without the refusal there is another one, and no launch)"""
    L = _lib.load()
    for fn, pointers in (("vra_rms_norm_i8", 4), ("vra_add_rms_norm_i8", 6)):
        L.vra_clear_error()
        getattr(L, fn)(*[None] * pointers, 1, 64, eps, BF16, 0)
        assert "eps" in L.vra_last_error().decode()
        L.vra_clear_error()
        getattr(L, fn)(*[None] * pointers, 1, 64, 0.0, BF16, 0)
        assert "null" in L.vra_last_error().decode()
        L.vra_clear_error()
