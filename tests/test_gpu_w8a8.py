"""W8A8 operators on the GPU against their definitions in 64 bits (tests/w8a8_plain.py)."""
import ctypes as C

import numpy as np
import pytest

from tests import w8a8_plain as plain
from tests.util import BF16, F16, F32, rng
from vllm_rs_amd import ops

pytestmark = pytest.mark.gpu
EPS = float(np.float32(1e-5))  # (the argument is a float)
GUARD = 77  # bytes behind every output that have to stay


class Guarded(ops.DevBuf):
    """an output with bytes in front of it (`shift`) and behind it that no call may write"""

    def __init__(self, nbytes, shift=0):
        super().__init__(nbytes + shift + GUARD)
        self.n, self.shift = nbytes, shift
        self.fill_bytes(0xA5)

    @property
    def at(self):
        return self.ptr + self.shift

    def take(self, dtype, shape):
        raw = self.numpy(np.uint8, (self.n + self.shift + GUARD,))
        assert (raw[:self.shift] == 0xA5).all() and (raw[self.shift + self.n:] == 0xA5).all(), "written outside the output"
        return raw[self.shift:self.shift + self.n].copy().view(dtype).reshape(shape)


class Shifted(ops.DevBuf):
    """an input that begins `shift` bytes behind a multiple of 256"""

    def __init__(self, array, shift=0):
        array = np.ascontiguousarray(array)
        super().__init__(array=np.concatenate([np.zeros(shift, np.uint8), array.reshape(-1).view(np.uint8)]))
        self.at = self.ptr + shift


def rows_of(kind, x, dt, residual=None, weight=None, shift=0, in_place=None):
    """one call -> (h or None, q, scales)"""
    L, (T, H) = ops.lib(), x.shape
    q, sc = Guarded(T * H, shift), Guarded(T * 4)
    xd = Shifted(x, 2 * shift)
    if kind == "quant":
        L.vra_quant_rows_i8(xd.at, q.at, sc.at, T, H, dt, 0)
        h = None
    elif kind == "norm":
        wd = Shifted(weight, 2 * shift)
        L.vra_rms_norm_i8(xd.at, wd.at, q.at, sc.at, T, H, EPS, dt, 0)
        h = None
    else:
        wd, rd, h = Shifted(weight, 2 * shift), Shifted(residual, 2 * shift), Guarded(T * H * 2, 2 * shift)
        to = {None: h, "x": xd, "residual": rd}[in_place]
        L.vra_add_rms_norm_i8(xd.at, rd.at, wd.at, to.at, q.at, sc.at, T, H, EPS, dt, 0)
    ops.check_error()
    if kind == "add":
        h = h.take(np.uint16, (T, H)) if in_place is None else to.numpy(np.uint8, (to.nbytes,))[2 * shift:].copy().view(np.uint16).reshape(T, H)
    return h, q.take(np.int8, (T, H)), sc.take(np.float32, (T,))


def check_rows(kind, x, dt, got, residual=None, weight=None):
    h, q, sc = got
    if kind == "add":
        with np.errstate(over="ignore"):
            x = plain.to(plain.wide(x, dt).astype(np.float32) + plain.wide(residual, dt).astype(np.float32), dt)
        assert np.array_equal(h, x), "the sum"
    ref, want = plain.quant_rows(x, dt) if kind == "quant" else plain.rms_norm(x, weight, EPS, dt)
    assert np.array_equal(q, ref), f"codes: {int((q != ref).sum())} of {q.size} differ"
    plain.assert_within(sc.astype(np.float64), want, plain.SCALE * np.abs(want) + 2.0 ** -149, "scales")


def some_rows(r, rows, cols, dt):
    x = r.standard_normal((rows, cols)) * np.exp(r.standard_normal((rows, 1)) * 3)
    x *= 1 + 24 * (r.random(cols) < 0.01)
    if rows > 2:
        x[1] = 0  # a padded row
    return plain.to(x, dt)


# widths at the edges of a vector, of what 64 .. 1024 threads keep in registers, and past it
WIDTHS = [1, 2, 7, 8, 9, 63, 64, 512, 513, 519, 520, 1001, 1024, 1032, 2047, 2048, 2056, 4096, 4103, 4104, 5632, 8191, 8192, 8193, 8200, 14336, 16391, 16392, 18944, 24576, 24584, 32768, 32776, 131072]


@pytest.mark.parametrize("kind", ["quant", "norm", "add"])
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("cols", WIDTHS)
def test_rows(kind, dt, cols):
    r = rng(cols * 7 + dt)
    rows = 5 if cols < 20000 else 3
    x, res, w = some_rows(r, rows, cols, dt), some_rows(r, rows, cols, dt), plain.to(1 + 0.2 * r.standard_normal(cols), dt)
    check_rows(kind, x, dt, rows_of(kind, x, dt, res, w), res, w)


@pytest.mark.parametrize("kind", ["quant", "norm", "add"])
@pytest.mark.parametrize("rows", [1, 3, 4, 66, 1021])
@pytest.mark.parametrize("cols, shift", [(1000, 1), (4096, 3), (333, 0), (16384, 5)])
def test_rows_that_begin_anywhere(kind, rows, cols, shift):
    r = rng(rows + cols)
    x, res, w = some_rows(r, rows, cols, BF16), some_rows(r, rows, cols, BF16), plain.to(1 + 0.2 * r.standard_normal(cols), BF16)
    check_rows(kind, x, BF16, rows_of(kind, x, BF16, res, w, shift), res, w)


@pytest.mark.parametrize("kind", ["quant", "norm", "add"])
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("cols", [1024, 1031, 1032, 4096, 4104, 8192, 8203, 16384, 16400, 24576])
def test_many_rows(kind, dt, cols):
    r = rng(cols + dt)
    x, res, w = some_rows(r, 513, cols, dt), some_rows(r, 513, cols, dt), plain.to(1 + 0.2 * r.standard_normal(cols), dt)
    check_rows(kind, x, dt, rows_of(kind, x, dt, res, w), res, w)


@pytest.mark.parametrize("in_place", ["x", "residual"])
@pytest.mark.parametrize("cols", [777, 4096, 40000])
def test_sum_in_place(in_place, cols):
    r = rng(cols)
    x, res, w = some_rows(r, 4, cols, F16), some_rows(r, 4, cols, F16), plain.to(1 + 0.2 * r.standard_normal(cols), F16)
    check_rows("add", x, F16, rows_of("add", x, F16, res, w, in_place=in_place), res, w)


@pytest.mark.parametrize("dt", [BF16, F16])
def test_halves_and_their_neighbours(dt):
    """quotients that are halves (ties to even), and the nearest representable values on both sides of them, at many maxima"""
    r = rng(5)
    rows = []
    for a in [127.0, 254.0, 1.984375, 63.5, 3.0, 100.0, 255.0, 1.0, 0.0078125 * 127] + list(np.exp(r.standard_normal(40))):
        a = float(plain.wide(plain.to(np.array([a]), dt), dt)[0])
        half = np.array([s * a * (2 * i + 1) / 254 for i in range(127) for s in (1, -1)])
        bits = plain.to(half, dt)
        near = np.concatenate([bits, (bits + 1).astype(np.uint16), (bits - 1).astype(np.uint16)])
        keep = np.abs(plain.wide(near, dt)) <= a
        rows.append(np.concatenate([plain.to(np.array([a]), dt), np.where(keep, near, 0)]))
    x = np.stack(rows).astype(np.uint16)
    check_rows("quant", x, dt, rows_of("quant", x, dt))
    w = plain.to(np.ones(x.shape[1]), dt)
    check_rows("norm", x, dt, rows_of("norm", x, dt, None, w), None, w)
    w = plain.to(np.exp(r.standard_normal(x.shape[1])), dt)
    check_rows("norm", x, dt, rows_of("norm", x, dt, None, w), None, w)


@pytest.mark.parametrize("kind", ["quant", "norm"])
def test_ends_of_the_range(kind):
    r = rng(8)
    base = r.standard_normal((9, 300)) / 4
    scale = [2.0 ** -133, 2.0 ** -127, 2.0 ** -120, 2.0 ** -62, 2.0 ** -58, 2.0 ** 58, 2.0 ** 62, 2.0 ** 120, 2.0 ** 127]
    x = plain.to(base * np.array(scale)[:, None], BF16)
    w = plain.to(np.ones(300), BF16)
    h, q, sc = rows_of(kind, x, BF16, None, w)
    ref, want = plain.quant_rows(x, BF16) if kind == "quant" else plain.rms_norm(x, w, EPS, BF16)
    assert np.array_equal(q, ref)
    plain.assert_within(sc.astype(np.float64), want, plain.SCALE * np.abs(want) + 2.0 ** -149, "scales")
    x = plain.to(np.array([[65504.0, -65504.0, 6e-8, 0.0], [6e-8, -6e-8, 1.2e-7, 0.0]]), F16)
    check_rows("quant", x, F16, rows_of("quant", x, F16))


@pytest.mark.parametrize("cols", [5, 640, 9000, 33000])
def test_rows_that_are_not_finite(cols):
    r = rng(cols)
    for dt, kind, put in ((BF16, "quant", np.inf), (F16, "quant", np.nan), (BF16, "norm", -np.inf), (F16, "add", np.nan), (BF16, "norm", np.nan)):
        x, res, w = some_rows(r, 5, cols, dt), some_rows(r, 5, cols, dt), plain.to(np.ones(cols), dt)
        bad = np.array([put], np.float32)
        x[2, cols - 1] = plain.to(bad, dt)[0]
        _, q, sc = rows_of(kind, x, dt, res, w)
        assert np.isnan(sc[2]) and not q[2].any() and np.isfinite(np.delete(sc, 2)).all()
        keep = [0, 1, 3, 4]
        _, q1, sc1 = rows_of(kind, x[keep], dt, res[keep], w)
        assert np.array_equal(q[keep], q1) and np.array_equal(sc[keep], sc1)  # a row's result does not depend on its neighbours
    x, w = some_rows(r, 5, cols, BF16), plain.to(np.ones(cols), BF16)
    x[2, cols - 1] = plain.to(np.array([1e25], np.float32), BF16)[0]  # its square is past 32 bits, and the row in order
    check_rows("norm", x, BF16, rows_of("norm", x, BF16, None, w), None, w)
    w[0] = plain.to(np.array([3e38], np.float32), BF16)[0]
    x[2, 0] = plain.to(np.array([7.0], np.float32), BF16)[0]
    x[3, 0] = 0
    _, q, sc = rows_of("norm", x, BF16, None, w)  # a product past it, a weight beside a zero
    assert np.isnan(sc[2]) and not q[2].any() and np.isfinite(sc[3])
    w[0], x[2, 0] = 0, plain.to(np.array([np.inf], np.float32), BF16)[0]
    _, q, sc = rows_of("norm", x, BF16, None, w)
    assert np.isnan(sc[2]) and not q[2].any()


def part_of(buf, at, n, dtype):
    """n elements of a device buffer from element `at` on"""
    out = np.empty(n, dtype)
    ops.lib().vra_device_sync()
    ops.lib().vra_memcpy_d2h(out.ctypes.data, buf.ptr + at * out.itemsize, out.nbytes, 0)
    ops.lib().vra_device_sync()
    return out


def test_more_rows_than_a_launch_takes():
    r, T, H = rng(3), (1 << 20) + 37, 3
    x, res, w = plain.to(r.standard_normal((T, H)), BF16), plain.to(r.standard_normal((T, H)), BF16), plain.to(1 + 0.2 * r.standard_normal(H), BF16)
    for kind in ("quant", "add"):
        check_rows(kind, x, BF16, rows_of(kind, x, BF16, res, w), res, w)


# ---------------------------------------------------------------- products
def some_codes(r, rows, cols):
    q = np.clip(np.rint(r.standard_normal((rows, cols)) * 40), -128, 127).astype(np.int8)
    return q, ((0.5 + r.random(rows)) / 40).astype(np.float32)


def product(r, M, K, N, dt, bias=False, residual=False, pair=False, shift=0, work=None, in_place=False, tensors=None):
    """(got, ref, bound) of one call"""
    L = ops.lib()
    if tensors is None:
        x, xs = some_codes(r, M, K)
        w, ws = some_codes(r, N, K)
        tensors = [x, xs, w, ws / np.float32(K ** 0.5)]
        if pair:
            w2, ws2 = some_codes(r, N, K)
            tensors += [w2, ws2 / np.float32(K ** 0.5)]
    dev = [Shifted(t, shift if t.dtype == np.int8 else 4 * shift) for t in tensors]
    size = 4 if dt == F32 else 2
    out = Guarded(M * N * size, size * shift)
    b = plain.to(r.standard_normal(N), dt) if bias else None
    res = plain.to(r.standard_normal((M, N)), dt) if residual else None
    bd, rd = None if b is None else Shifted(b, size * shift), None if res is None else Shifted(res, size * shift)
    work = None if work is None else work.ptr
    if pair:
        L.vra_w8a8_gate_up_silu(*[d.at for d in dev], out.at, work, M, K, N, dt, 0)
    else:
        to = rd if in_place else out
        L.vra_w8a8_gemm(*[d.at for d in dev], bd and bd.at, rd and rd.at, to.at, work, M, K, N, dt, 0)
    ops.check_error()
    kind = np.float32 if dt == F32 else np.uint16
    got = rd.numpy(np.uint8, (rd.nbytes,))[size * shift:].copy().view(kind).reshape(M, N) if in_place else out.take(kind, (M, N))
    ref, bound = plain.gate_up_silu(*tensors, dt) if pair else plain.gemm(*tensors, b, res, dt)
    return got, ref, bound


def check_product(r, M, K, N, dt, **kw):
    got, ref, bound = product(r, M, K, N, dt, **kw)
    plain.assert_within(plain.wide(got, dt), ref, bound, f"{M} x {N}, K = {K}, {kw}")
    return got


@pytest.fixture(scope="module")
def work():
    return ops.DevBuf(ops.lib().vra_w8a8_workspace_bytes()).zero()


ROWS = [1, 2, 5, 16, 17, 32, 33, 48, 64, 65, 100, 128, 129, 200, 256, 257, 300]


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("M", ROWS)
def test_gemm(dt, M, work):
    r = rng(M + dt)
    # whole steps, K that ends inside one, inside a vector, shorter than either; columns that end inside every unit
    for i, (K, N) in enumerate([(1024, 512), (4096, 272), (144, 130), (2064, 100), (1000, 36), (17, 3), (1, 1), (130, 1), (15, 64), (128, 1003), (896, 2100)]):
        check_product(r, M, K, N, dt, bias=i % 2 == 0, residual=i % 3 == 0, work=work)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("M", ROWS)
def test_gate_up_silu(dt, M, work):
    r = rng(3 * M + dt)
    for K, N in [(1024, 512), (4096, 144), (144, 130), (2064, 100), (1000, 36), (17, 3), (1, 1), (128, 1003), (896, 1100)]:
        check_product(r, M, K, N, dt, pair=True, work=work)


KERNELS = [(1, c, s) for c in (1, 2, 4, 8) for s in (1, 2, 8)] + [(2, t, s) for t in (0x12, 0x22, 0x32, 0x24) for s in (1, 2, 4, 8)] + [(2, 0x34, 1), (2, 0x44, 1)] + [(0, t, s) for t in (0x11, 0x22) for s in (1, 2, 4, 8)] + [(0, 0x44, 1)]


@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("kind, size, slices", KERNELS)
def test_named_kernels(kind, size, slices, pair, work):
    """every kernel at the edges of its tiles, in K steps of 128 (one, an odd number, a part behind them, 16 of the last), against 64-row tiles of the kernel for any alignment:
    the same bits; that one, and its own, against the definition"""
    L, r = ops.lib(), rng(size * 8 + slices)
    blocks = 16 if kind == 1 else size // 16 * 64
    rows = [1, 15, 16, 17, 33, 48, 64] if kind == 1 else [1, blocks - 1, blocks, blocks + 1, 2 * blocks + 3]
    for i, M in enumerate(rows):
        for j, (K, N) in enumerate([(1024, 300), (1168, 257), (1408, 64), (2032, 516), (3216, 8)] if kind == 1 or slices > 1 else [(128, 300), (16, 257), (384, 64), (496, 516), (656, 8)]):
            K += 3 * (j < 4 and kind == 0 or j % 2 and (kind, size) == (1, 2 if pair else 1))
            dt = [BF16, F16, BF16 if pair else F32][(i + j) % 3]
            x, xs = some_codes(r, M, K)
            w, ws = some_codes(r, N, K)
            w2, ws2 = some_codes(r, N, K)
            bias, res = plain.to(r.standard_normal(N), dt), plain.to(r.standard_normal((M, N)), dt)
            d = [ops.dev(t) for t in (x, xs, w, ws, w2, ws2, bias, res)]
            kind_np, size_np = (np.float32, 4) if dt == F32 else (np.uint16, 2)
            got = []
            for code in (0x10011, slices << 16 | kind << 8 | size):
                out = Guarded(M * N * size_np)
                L.vra_w8a8_gemm_on(code, *[t.ptr for t in d[:4]], *([t.ptr for t in d[4:6]] if pair else [None, None]), None if pair or j % 2 else d[6].ptr,
                                   None if pair or i % 2 else d[7].ptr, out.at, work.ptr, M, K, N, dt, 0)
                if code != 0x10011 and L.vra_last_error().decode():
                    assert "no such kernel" in L.vra_last_error().decode()
                    mt = (M + 15) // 16  # only what the table of kernels lacks: few rows beyond a size's blocks
                    assert kind == 1 and (mt > (4 if size <= 2 else 2 if size == 4 else 1) or (size == 1) == pair and size in (1, 8) or size == 8 and not pair)
                    L.vra_clear_error()
                    got.append(got[0])
                    continue
                ops.check_error()
                got.append(out.take(kind_np, (M, N)))
            assert np.array_equal(got[0], got[1]), f"{M} x {N}, K = {K}"
            if kind == 0 or i == j == 1:
                ref, bound = plain.gate_up_silu(x, xs, w, ws, w2, ws2, dt) if pair else plain.gemm(x, xs, w, ws, None if j % 2 else bias, None if i % 2 else res, dt)
                plain.assert_within(plain.wide(got[0], dt), ref, bound, f"any alignment, {M} x {N}, K = {K}")


@pytest.mark.parametrize("M, K, N", [(1, 512, 96), (8, 1024, 64), (40, 256, 200), (150, 640, 300), (300, 384, 520)])
@pytest.mark.parametrize("shift", [1, 4, 8])
def test_tensors_that_begin_anywhere(M, K, N, shift, work):
    r = rng(M + shift)
    for pair in (False, True):
        check_product(r, M, K, N, BF16, bias=not pair, residual=not pair, pair=pair, shift=shift, work=work)
    check_product(r, M, K, N, F32, bias=True, residual=True, shift=shift, work=work)


@pytest.mark.parametrize("M, K, N", [(1, 4096, 128), (24, 8192, 256), (100, 8192, 512), (256, 2048, 1024), (600, 1024, 640)])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_residual_in_place(M, K, N, dt, work):
    check_product(rng(M), M, K, N, dt, bias=True, residual=True, in_place=True, work=work)


@pytest.mark.parametrize("M", [1, 3, 20, 40, 130, 520])
def test_largest_sums(M, work):
    """-128 everywhere, the longest K: 2147467264, below 2^31; and the other sign"""
    K, N = 131071, 24
    for v in (-128, 127):
        x, w = np.full((M, K), -128, np.int8), np.full((N, K), v, np.int8)
        one = np.ones(max(M, N), np.float32)
        got, ref, bound = product(rng(1), M, K, N, F32, tensors=[x, one[:M], w, one[:N]], work=work)
        assert ref[0, 0] == -128.0 * v * K
        plain.assert_within(got.astype(np.float64), ref, bound, "sums")


@pytest.mark.parametrize("M, K, N", [(1, 14336, 512), (16, 4096, 256), (32, 14336, 300), (64, 8192, 1024), (100, 14336, 512), (150, 4100, 640), (256, 16384, 512), (700, 4096, 256)])
@pytest.mark.parametrize("pair", [False, True])
def test_the_workspace_changes_no_bit(M, K, N, pair, work):
    L, r = ops.lib(), rng(M)
    x, xs = some_codes(r, M, K)
    w, ws = some_codes(r, N, K)
    t = [x, xs, w, ws] + ([w[::-1].copy(), ws] if pair else [])
    dt = BF16 if pair else F32
    first = product(rng(2), M, K, N, dt, pair=pair, tensors=t)[0]
    for _ in range(3):  # and is left as it was found
        assert np.array_equal(product(rng(2), M, K, N, dt, pair=pair, tensors=t, work=work)[0], first)


def test_rows_do_not_depend_on_each_other(work):
    """a row's bits in any batch, on whichever kernel it falls"""
    r, K, N = rng(4), 2048, 768
    x, xs = some_codes(r, 400, K)
    w, ws = some_codes(r, N, K)
    whole = product(r, 400, K, N, BF16, tensors=[x, xs, w, ws], work=work)[0]
    for m in (1, 4, 16, 30, 64, 150, 399):
        assert np.array_equal(product(r, m, K, N, BF16, tensors=[x[:m], xs[:m], w, ws], work=work)[0], whole[:m])


@pytest.mark.parametrize("M", [2, 40, 300])
def test_scales_that_are_zero_or_nan(M, work):
    r, K, N = rng(6), 512, 128
    x, xs = some_codes(r, M, K)
    w, ws = some_codes(r, N, K)
    xs[0], xs[1] = 0.0, np.nan
    got = plain.wide(product(r, M, K, N, BF16, tensors=[x, xs, w, ws], work=work)[0], BF16)
    assert (got[0] == 0).all() and np.isnan(got[1]).all() and np.isfinite(got[2:]).all()


def test_more_tiles_than_a_launch_takes():
    """2^28 rows of one element: the launch is cut behind 2^22 tiles of 64 rows; the last rows of the first part and the second part"""
    L, M, cut = ops.lib(), (1 << 28) + 70, 1 << 28
    x, xs, res, out = ops.DevBuf(M), ops.DevBuf(M * 4), ops.DevBuf(M * 2), Guarded(M * 2)
    L.vra_fill_hash_u32(x.ptr, M // 4, 3, 0)
    L.vra_memset(x.ptr + M // 4 * 4, 5, M % 4, 0)
    L.vra_fill_normal(xs.ptr, M, 4, 0.0, 1.0, F32, 0)
    L.vra_fill_normal(res.ptr, M, 5, 0.0, 1.0, BF16, 0)
    w, ws = np.full((1, 1), -77, np.int8), np.full(1, 0.01, np.float32)
    wd, sd = ops.dev(w), ops.dev(ws)
    L.vra_w8a8_gemm(x.ptr, xs.ptr, wd.ptr, sd.ptr, None, res.ptr, out.at, None, M, 1, 1, BF16, 0)
    ops.check_error()
    for at, n in ((0, 500), (cut - 300, 370)):
        ref, bound = plain.gemm(part_of(x, at, n, np.int8)[:, None], part_of(xs, at, n, np.float32), w, ws, None, part_of(res, at, n, np.uint16)[:, None], BF16)
        plain.assert_within(plain.wide(part_of(out, at, n, np.uint16)[:, None], BF16), ref, bound, f"rows from {at}")
    assert (part_of(out, 2 * M, GUARD, np.uint8) == 0xA5).all()


def test_wrappers():
    """the Python entry points, as a feed-forward block uses them together: each step against its definition on the step's own inputs"""
    r, T, H, F = rng(11), 37, 512, 1376
    x, res, w = some_rows(r, T, H, BF16), some_rows(r, T, H, BF16), plain.to(1 + 0.2 * r.standard_normal(H), BF16)
    wg, sg = some_codes(r, F, H)
    wu, su = some_codes(r, F, H)
    wd, sd = some_codes(r, H, F)
    p = ops.W8A8()
    h, q, s = ops.add_rms_norm_i8(ops.dev(x), ops.dev(res), ops.dev(w), T, H, EPS)
    act = p.gate_up_silu(q, s, ops.dev(wg), ops.dev(sg), ops.dev(wu), ops.dev(su), T, H, F)
    aq, asc = ops.quant_rows_i8(act, T, F)
    out = p.gemm(aq, asc, ops.dev(wd), ops.dev(sd), T, F, H, residual=h)
    hb, qb, sb = h.numpy(np.uint16, (T, H)), q.numpy(np.int8, (T, H)), s.numpy(np.float32, (T,))
    check_rows("add", x, BF16, (hb, qb, sb), res, w)
    ab = act.numpy(np.uint16, (T, F))
    plain.assert_within(plain.wide(ab, BF16), *plain.gate_up_silu(qb, sb, wg, sg, wu, su, BF16), "pair")
    check_rows("quant", ab, BF16, (None, aq.numpy(np.int8, (T, F)), asc.numpy(np.float32, (T,))))
    plain.assert_within(plain.wide(out.numpy(np.uint16, (T, H)), BF16),
                        *plain.gemm(aq.numpy(np.int8, (T, F)), asc.numpy(np.float32, (T,)), wd, sd, None, hb, BF16), "down")
    q2, s2 = ops.rms_norm_i8(h, ops.dev(w), T, H, EPS)
    assert np.array_equal(q2.numpy(np.int8, (T, H)), qb) and np.array_equal(s2.numpy(np.float32, (T,)), sb)


# ---------------------------------------------------------------- streams and graphs
class Block:
    """a feed-forward block of T rows on caller-owned buffers: add + norm, gate / up pair, rows to 8 bits, down with the residual"""

    def __init__(self, T, seed, H=1024, F=2816):
        self.L, self.T, self.H, self.F, self.r = ops.lib(), T, H, F, rng(seed)
        codes = lambda *s: ops.dev(self.r.integers(-127, 128, s).astype(np.int8))
        ones = lambda n, v: ops.dev(np.full(n, v, np.float32))
        self.b = dict(x=ops.DevBuf(T * H * 2), res=ops.dev(self.rows()), w=ops.dev(plain.to(1 + 0.2 * self.r.standard_normal(H), BF16)), h=ops.DevBuf(T * H * 2),
                      q=ops.DevBuf(T * H), s=ops.DevBuf(T * 4), wg=codes(F, H), wu=codes(F, H), sg=ones(F, 4e-4), act=ops.DevBuf(T * F * 2), aq=ops.DevBuf(T * F),
                      sa=ops.DevBuf(T * 4), wd=codes(H, F), sd=ones(H, 3e-4), out=ops.DevBuf(T * H * 2), ws=ops.DevBuf(self.L.vra_w8a8_workspace_bytes()).zero())
        self.refill()

    def rows(self):
        return plain.to(self.r.standard_normal((self.T, self.H)), BF16)

    def refill(self):
        x = self.rows()
        self.L.vra_memcpy_h2d(self.b["x"].ptr, x.ctypes.data, x.nbytes, 0)
        self.L.vra_device_sync()

    def __call__(self, stream):
        p = {k: v.ptr for k, v in self.b.items()}
        T, H, F = self.T, self.H, self.F
        self.L.vra_add_rms_norm_i8(p["x"], p["res"], p["w"], p["h"], p["q"], p["s"], T, H, EPS, BF16, stream)
        self.L.vra_w8a8_gate_up_silu(p["q"], p["s"], p["wg"], p["sg"], p["wu"], p["sg"], p["act"], p["ws"], T, H, F, BF16, stream)
        self.L.vra_quant_rows_i8(p["act"], p["aq"], p["sa"], T, F, BF16, stream)
        self.L.vra_w8a8_gemm(p["aq"], p["sa"], p["wd"], p["sd"], None, p["h"], p["out"], p["ws"], T, F, H, BF16, stream)
        ops.check_error()

    def take(self):
        """the result; the buffer is cleared behind it"""
        out = self.b["out"].numpy(np.uint16, (self.T, self.H))
        self.b["out"].zero()
        self.L.vra_device_sync()
        return out


class Graph:
    """what `body(stream)` launches, captured once (the HIP runtime that the library has loaded)"""

    def __init__(self, stream, body):
        self.hip, self.stream, self.exec = C.CDLL("libamdhip64.so.7"), C.c_void_p(stream), C.c_void_p()
        graph = C.c_void_p()
        assert self.hip.hipStreamBeginCapture(self.stream, 2) == 0  # hipStreamCaptureModeRelaxed
        body(stream)
        assert self.hip.hipStreamEndCapture(self.stream, C.byref(graph)) == 0 and graph.value
        assert self.hip.hipGraphInstantiate(C.byref(self.exec), graph, None, None, C.c_size_t(0)) == 0
        assert self.hip.hipGraphDestroy(graph) == 0

    def replay(self):
        assert self.hip.hipGraphLaunch(self.exec, self.stream) == 0

    def close(self):
        assert self.hip.hipGraphExecDestroy(self.exec) == 0


@pytest.mark.parametrize("T", [1, 12, 40, 130, 600])
def test_graph(T):
    block, stream = Block(T, T), ops.lib().vra_stream_create()
    graph = Graph(stream, block)  # (the first call of these kernels may be a captured one)
    for _ in range(4):
        block.refill()
        block(stream)
        want = block.take()
        graph.replay()
        got = block.take()
        assert np.array_equal(got, want) and want.any()
    graph.close()
    ops.lib().vra_stream_destroy(stream)


@pytest.mark.parametrize("T", [1, 40, 200])
def test_two_streams(T):
    """two blocks at once, a workspace each; one of them as a graph"""
    L = ops.lib()
    blocks, streams = [Block(T, s) for s in (1, 2)], [L.vra_stream_create() for _ in range(2)]
    want = []
    for b, s in zip(blocks, streams):
        b(s)
        want.append(b.take())
    graph = Graph(streams[1], blocks[1])
    for _ in range(10):
        blocks[0](streams[0])
        graph.replay()
    for b, w in zip(blocks, want):
        assert np.array_equal(b.take(), w) and w.any()
    graph.close()
    for s in streams:
        L.vra_stream_destroy(s)
