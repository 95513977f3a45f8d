"""The W8A8 operators from their definitions in 64 bits, and the bounds of their kernels' errors (numpy)."""
import numpy as np

from oracle import oracle as orc

BF16, F16, F32 = 0, 1, 2
U = 2.0 ** -24  # half a step of f32, relative
HALF_STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: U}  # a rounding's error, relative
LOWEST = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -150}  # ... below the normal range, absolute


def to(x, dt):
    return x.astype(np.float32) if dt == F32 else orc.to_dt(np.ascontiguousarray(x, np.float32), dt)


def wide(bits, dt):
    return np.asarray(bits, np.float64) if dt == F32 else orc.from_dt(bits, dt).astype(np.float64)


def codes(p):
    """p [rows, cols] in 64 bits (products as f32 holds them) -> (q, max |p|); rows that are not finite: codes 0, NaN"""
    a = np.abs(p).max(1, initial=0.0)
    fine = np.isfinite(p).all(1)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        t = 127.0 * p / a[:, None]
    q = np.where((fine & (a > 0))[:, None], np.rint(t), 0.0)
    return q.astype(np.int8), np.where(fine, a, np.nan)


def quant_rows(x, dt):
    q, a = codes(wide(x, dt))
    return q, a / 127.0


def rms_norm(h, weight, eps, dt):
    f = wide(h, dt)
    with np.errstate(over="ignore", invalid="ignore"):
        p = (f * wide(weight, dt)[None, :]).astype(np.float32).astype(np.float64)
        mean = (f * f).sum(1) / f.shape[1]
    q, a = codes(p)
    return q, a / 127.0 / np.sqrt(mean + eps)


SCALE = 1.01 * U  # error of a scale, relative: it is formed in 64 bits and rounded once


def gemm(x, xs, w, ws, bias, residual, dt):
    """(result in 64 bits, bound of the error of a result rounded once to dt)"""
    acc = x.astype(np.float64) @ w.astype(np.float64).T  # below 2^53: exact
    y = acc * xs.astype(np.float64)[:, None] * ws.astype(np.float64)[None, :]
    mag = np.abs(y)
    for extra in (None if bias is None else wide(bias, dt)[None, :], None if residual is None else wide(residual, dt)):
        if extra is not None:
            y = y + extra
            mag = mag + np.abs(extra)
    # the sum's conversion and two products, one rounding for each addition; then the result's own
    off = 5.0 * U * mag
    return y, off + HALF_STEP[dt] * (np.abs(y) + off) * 1.01 + LOWEST[dt]


def gate_up_silu(x, xs, wg, sg, wu, su, dt):
    g, u = (gemm(x, xs, w, s, None, None, F32)[0] for w, s in ((wg, sg), (wu, su)))
    with np.errstate(over="ignore"):
        y = g / (1.0 + np.exp(-g)) * u
    # g and u three roundings each; the error of g moves the exponential by |g| times as much; the exponential two steps, sum, quotient and product one rounding each
    off = (3.0 + 3.0 + 3.0 * np.abs(g) + 4.0 + 3.0) * U * np.abs(y)
    return y, off + HALF_STEP[dt] * (np.abs(y) + off) * 1.01 + LOWEST[dt]


def assert_within(got, ref, bound, name):
    fine = np.isfinite(ref)
    assert np.array_equal(fine, np.isfinite(got)), f"{name}: finite in other places"
    far = np.abs(got - ref)[fine] / bound[fine]
    assert far.size == 0 or far.max() <= 1.0, f"{name}: {far.max():.3f} of the bound, {int((far > 1).sum())} values beyond it"
