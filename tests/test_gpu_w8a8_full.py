"""W8A8 products at the sizes that serving meets: whole chips of workgroups, many K steps, many tile rows and columns, operands past 4 GiB; and every kernel that such sizes
may be given to, by its name.  All kernels give the same bits: each against 64 x 64 tiles of the kernel for any alignment, and that one, at sampled rows, against the definition."""
import numpy as np
import pytest

from tests import w8a8_plain as plain
from tests.test_gpu_w8a8 import GUARD, Guarded, part_of
from tests.util import BF16, F16, F32, rng
from vllm_rs_amd import ops

pytestmark = pytest.mark.gpu
FEW, TILE, ANY = 1, 2, 0
PLAIN = 1 << 16 | ANY << 8 | 0x11


def code(kind, size, slices=1):
    return slices << 16 | kind << 8 | size


def size_of(dt):
    return 4 if dt == F32 else 2


def kind_of(dt):
    return np.float32 if dt == F32 else np.uint16


def some_bytes(n, seed):
    """n random 8-bit integers on the device, all 256 values"""
    b = ops.DevBuf((n + 3) // 4 * 4)
    ops.lib().vra_fill_hash_u32(b.ptr, (n + 3) // 4, seed, 0)
    return b


class Product:
    """operands on the device; `rows` of them on the host"""

    def __init__(self, seed, pair, M, K, N, dt, bias=False, residual=False):
        r, L = rng(seed), ops.lib()
        self.pair, self.M, self.K, self.N, self.dt = pair, M, K, N, dt
        self.x, self.w = some_bytes(M * K, 1000 + seed), [some_bytes(N * K, 2000 + seed + i) for i in range(1 + pair)]
        scale = 1.0 / (74.0 * K ** 0.5)  # results of about one
        self.xs, self.ws = (0.5 + r.random(M)).astype(np.float32), [((0.5 + r.random(N)) * scale / 74.0).astype(np.float32) for _ in range(1 + pair)]
        self.bias = plain.to(r.standard_normal(N), dt) if bias else None
        self.dev = [ops.dev(self.xs)] + [ops.dev(s) for s in self.ws] + [ops.dev(self.bias) if bias else None]
        self.res = None
        if residual:
            self.res = ops.DevBuf(M * N * size_of(dt))
            L.vra_fill_normal(self.res.ptr, M * N, 3000 + seed, 0.0, 1.0, dt, 0)

    def __call__(self, work, kernel=None, in_place=False):
        """the output's buffer; kernel None: the public entry"""
        L, b = ops.lib(), self.dev[-1]
        out = Guarded(self.M * self.N * size_of(self.dt))
        if in_place:
            L.vra_memcpy_d2d(out.at, self.res.ptr, out.n, 0)
        res = None if self.res is None else out.at if in_place else self.res.ptr
        xs, ws = self.dev[0].ptr, [d.ptr for d in self.dev[1:-1]]
        tail = (work.ptr, self.M, self.K, self.N, self.dt, 0)
        if kernel is not None:
            up = (self.w[1].ptr, ws[1]) if self.pair else (None, None)
            L.vra_w8a8_gemm_on(kernel, self.x.ptr, xs, self.w[0].ptr, ws[0], *up, b and b.ptr, res, out.at, *tail)
        elif self.pair:
            L.vra_w8a8_gate_up_silu(self.x.ptr, xs, self.w[0].ptr, ws[0], self.w[1].ptr, ws[1], out.at, *tail)
        else:
            L.vra_w8a8_gemm(self.x.ptr, xs, self.w[0].ptr, ws[0], b and b.ptr, res, out.at, *tail)
        ops.check_error()
        return out

    def take(self, out):
        return out.take(kind_of(self.dt), (self.M, self.N))

    def rows(self, out, rows, cols=None):
        """(rows of the result, the definition's, bounds); cols: a range of columns, the whole width without"""
        M, K, N, dt = self.M, self.K, self.N, self.dt
        c0, c1 = cols or (0, N)
        x = np.stack([part_of(self.x, t * K, K, np.int8) for t in rows])
        got = np.stack([part_of(out, t * N + c0, c1 - c0, kind_of(dt)) for t in rows])
        res = None if self.res is None else np.stack([part_of(self.res, t * N + c0, c1 - c0, kind_of(dt)) for t in rows])
        refs = []
        for a in range(c0, c1, 2048):  # columns by blocks: the 64-bit copies stay small
            e = min(a + 2048, c1)
            w = [part_of(b, a * K, (e - a) * K, np.int8).reshape(e - a, K) for b in self.w]
            if self.pair:
                refs.append(plain.gate_up_silu(x, self.xs[rows], w[0], self.ws[0][a:e], w[1], self.ws[1][a:e], dt))
            else:
                refs.append(plain.gemm(x, self.xs[rows], w[0], self.ws[0][a:e], None if self.bias is None else self.bias[a:e],
                                       None if res is None else res[:, a - c0:e - c0], dt))
        return plain.wide(got, dt), np.concatenate([f[0] for f in refs], 1), np.concatenate([f[1] for f in refs], 1)


@pytest.fixture(scope="module")
def work():
    return ops.DevBuf(ops.lib().vra_w8a8_workspace_bytes()).zero()


TILES = [code(TILE, t) for t in (0x12, 0x22, 0x32, 0x24, 0x34, 0x44)]


def sliced(*sizes_and_slices):
    return [code(TILE, t, s) for t, s in sizes_and_slices]


@pytest.mark.parametrize("pair, M, K, N, dt, kernels", [
    (0, 3063, 3584, 2600, BF16, TILES),                                                    # three prompts: 12 to 48 tile rows, 11 to 21 tile columns
    (1, 3063, 3584, 4736, BF16, TILES),
    (0, 4100, 1168, 8200, F16, TILES),                                                     # more 256 x 256 tiles than CUs, K off 128
    (1, 2100, 2064, 9000, F16, TILES),
    (0, 1030, 4096, 6144, F32, TILES),
    (0, 600, 16384, 2576, BF16, sliced((0x12, 4), (0x22, 4), (0x32, 4), (0x24, 4))),      # slices of K over a full chip
    (1, 400, 6160, 1500, F16, sliced((0x12, 2), (0x22, 2), (0x32, 2), (0x24, 2))),
    (0, 256, 14336, 4096, F32, sliced((0x12, 4), (0x22, 4), (0x24, 4), (0x22, 8))),
    (0, 4096, 4099, 4100, BF16, [code(ANY, 0x22), code(ANY, 0x44)]),                       # rows that begin anywhere
    (1, 3000, 2741, 2300, F16, [code(ANY, 0x22), code(ANY, 0x44)]),
    (0, 500, 8193, 1003, F32, [code(ANY, 0x11, 4), code(ANY, 0x22, 8)]),
    (0, 16, 3584, 32000, F32, [code(FEW, c) for c in (1, 2, 4)]),                          # few rows
    (0, 32, 14336, 4096, BF16, [code(FEW, 1, 4), code(FEW, 2, 8), code(FEW, 4, 8)]),
    (0, 64, 1168, 20000, F16, [code(FEW, 1), code(FEW, 2)]),
    (1, 16, 4096, 14336, BF16, [code(FEW, c) for c in (2, 4, 8)]),
    (1, 32, 14336, 4096, F16, [code(FEW, 2, 2), code(FEW, 4, 4)]),
    (1, 64, 3600, 9000, BF16, [code(FEW, 2)]),
    (0, 33, 3585, 20001, BF16, [code(FEW, 1)]),
    (1, 50, 4385, 9001, F16, [code(FEW, 2)]),
])
def test_full_grids(pair, M, K, N, dt, kernels, work):
    p = Product(M + K, pair, M, K, N, dt, bias=not pair and dt != BF16, residual=not pair)
    out = p(work, PLAIN)
    rows = sorted({0, 1, M // 2, M - 2, M - 1} | set(rng(M).integers(0, M, 12).tolist()))
    plain.assert_within(*p.rows(out, rows), f"any alignment, {M} x {N}, K = {K}")
    want = p.take(out)
    for kernel in [None] + kernels:
        got = p.take(p(work, kernel))
        assert np.array_equal(got, want), f"{'the public entry' if kernel is None else hex(kernel)}: {int((got != want).sum())} of {want.size} differ"


@pytest.mark.parametrize("M, K, N, dt, kernels", [(1030, 400, 2600, BF16, TILES), (1030, 400, 2600, F32, TILES), (520, 4096, 1500, F16, sliced((0x22, 4), (0x32, 2))),
                                                  (1030, 403, 2600, F16, [code(ANY, t) for t in (0x11, 0x22, 0x44)]), (16, 3584, 9000, F16, [code(FEW, 4)]),
                                                  (30, 8192, 500, BF16, [code(FEW, 4, 8)])])
def test_residual_in_place_on_named_kernels(M, K, N, dt, kernels, work):
    p = Product(M + N, False, M, K, N, dt, bias=True, residual=True)
    want = p.take(p(work, PLAIN))
    for kernel in [None] + kernels:
        assert np.array_equal(p.take(p(work, kernel, in_place=True)), want), "the public entry" if kernel is None else hex(kernel)


@pytest.mark.parametrize("kernel", TILES + sliced((0x12, 8), (0x22, 8), (0x32, 8), (0x24, 8)))
def test_largest_sums_on_tiles(kernel, work):
    """-128 everywhere and the longest K of a kernel with whole vectors: 2147221504, below 2^31; and the other sign"""
    L, M, K, N = ops.lib(), 260, 131056, 132
    x, w, one, out = ops.DevBuf(M * K), ops.DevBuf(N * K), ops.dev(np.ones(M, np.float32)), ops.DevBuf(M * N * 4)
    x.fill_bytes(0x80)
    for byte, v in ((0x80, -128), (0x7F, 127)):
        w.fill_bytes(byte)
        out.fill_bytes(0xFF)
        L.vra_w8a8_gemm_on(kernel, x.ptr, one.ptr, w.ptr, one.ptr, None, None, None, None, out.ptr, work.ptr, M, K, N, F32, 0)
        ops.check_error()
        assert (out.numpy(np.float32, (M, N)) == np.float32(-128.0 * v * K)).all()


@pytest.mark.parametrize("dt", [BF16, F16])
def test_a_block_from_16_bit_weights(dt):
    """weights and their scales made by the rows' entry, and a feed-forward block on them: each step against its definition on the step's own inputs"""
    r, T, H, F, eps = rng(21), 37, 512, 1376, float(np.float32(1e-5))
    x, res, norm_w = (plain.to(t, dt) for t in (r.standard_normal((T, H)), r.standard_normal((T, H)), 1 + 0.2 * r.standard_normal(H)))
    w16 = {"gate": plain.to(r.standard_normal((F, H)) / 20, dt), "up": plain.to(r.standard_normal((F, H)) / 20, dt), "down": plain.to(r.standard_normal((H, F)) / 30, dt)}
    w16["down"][3] = 0  # a channel that is off
    dev = {k: ops.quant_rows_i8(ops.dev(v), *v.shape, dt) for k, v in w16.items()}
    host = {k: (dev[k][0].numpy(np.int8, v.shape), dev[k][1].numpy(np.float32, (len(v),))) for k, v in w16.items()}
    for k, v in w16.items():
        q, s = plain.quant_rows(v, dt)
        assert np.array_equal(host[k][0], q)
        plain.assert_within(host[k][1].astype(np.float64), s, plain.SCALE * s + 2.0 ** -149, k)
    p = ops.W8A8()
    h, q, s = ops.add_rms_norm_i8(ops.dev(x), ops.dev(res), ops.dev(norm_w), T, H, eps, dt)
    act = p.gate_up_silu(q, s, *dev["gate"], *dev["up"], T, H, F, dtype=dt)
    aq, a_s = ops.quant_rows_i8(act, T, F, dt)
    out = p.gemm(aq, a_s, *dev["down"], T, F, H, residual=h, dtype=dt)
    hb, qb, sb = h.numpy(np.uint16, (T, H)), q.numpy(np.int8, (T, H)), s.numpy(np.float32, (T,))
    ab, aqb, asb = act.numpy(np.uint16, (T, F)), aq.numpy(np.int8, (T, F)), a_s.numpy(np.float32, (T,))
    assert np.array_equal(qb, plain.rms_norm(hb, norm_w, eps, dt)[0]) and np.array_equal(aqb, plain.quant_rows(ab, dt)[0])
    plain.assert_within(plain.wide(ab, dt), *plain.gate_up_silu(qb, sb, *host["gate"], *host["up"], dt), "pair")
    got = out.numpy(np.uint16, (T, H))
    plain.assert_within(plain.wide(got, dt), *plain.gemm(aqb, asb, *host["down"], None, hb, dt), "down")
    assert np.array_equal(got[:, 3], hb[:, 3])


# ---------------------------------------------------------------- past 4 GiB and 2^31 elements
@pytest.mark.parametrize("M, K", [(1, 12288), (40, 12288), (300, 12288), (3, 12289)])
def test_weights_past_4_gib(M, K, work):
    N = 400010
    p = Product(M, False, M, K, N, BF16, bias=True)
    out = p(work)
    rows, last = sorted({0, M // 2, M - 1}), (1 << 32) // K  # the column whose row of weights holds byte 2^32
    for cols in ((0, 64), (last // 2 - 30, last // 2 + 30), (last - 40, last + 40), (N - 70, N)):
        plain.assert_within(*p.rows(out, rows, cols), f"columns {cols}")
    assert (part_of(out, 2 * M * N, GUARD, np.uint8) == 0xA5).all()


@pytest.mark.parametrize("K, N, pair", [(12288, 24, 0), (12288, 24, 1), (12289, 24, 0)])
def test_rows_past_4_gib(K, N, pair, work):
    M = 400010
    p = Product(N, pair, M, K, N, F16, residual=not pair)
    out = p(work)
    last = (1 << 32) // K
    plain.assert_within(*p.rows(out, [0, 255, last // 2, last // 2 + 1, last - 1, last, last + 1, 350000, M - 257, M - 1]), "rows")
    assert (part_of(out, 2 * M * N, GUARD, np.uint8) == 0xA5).all()


@pytest.mark.parametrize("K, pair", [(16, 0), (16, 1), (17, 0)])
def test_output_past_2_31_elements(K, pair, work):
    M, N = 70001, 33000
    p = Product(K, pair, M, K, N, BF16, bias=not pair, residual=not pair)
    out = p(work)
    last = (1 << 31) // N
    plain.assert_within(*p.rows(out, [0, 1, last // 2, last // 2 + 1, last - 1, last, last + 1, 66000, M - 200, M - 1]), "rows")
    assert (part_of(out, 2 * M * N, GUARD, np.uint8) == 0xA5).all()


@pytest.mark.parametrize("cols", [32776, 32768])
@pytest.mark.parametrize("kind", ["quant", "add"])
def test_rows_to_8_bits_past_2_31_elements(kind, cols):
    L, T, dt, eps = ops.lib(), 70001, BF16, float(np.float32(1e-5))
    x, q, s = ops.DevBuf(T * cols * 2), Guarded(T * cols), Guarded(T * 4)
    L.vra_fill_normal(x.ptr, T * cols, 5, 0.0, 1.0, dt, 0)
    if kind == "quant":
        L.vra_quant_rows_i8(x.ptr, q.at, s.at, T, cols, dt, 0)
    else:
        res, h, w = ops.DevBuf(T * cols * 2), Guarded(T * cols * 2), plain.to(1 + 0.2 * rng(1).standard_normal(cols), dt)
        L.vra_fill_normal(res.ptr, T * cols, 6, 0.0, 1.0, dt, 0)
        wd = ops.dev(w)
        L.vra_add_rms_norm_i8(x.ptr, res.ptr, wd.ptr, h.at, q.at, s.at, T, cols, eps, dt, 0)
    ops.check_error()
    scales = s.take(np.float32, (T,))
    for t in (0, 1, 32767, 32768, (1 << 31) // cols - 1, (1 << 31) // cols, (1 << 31) // cols + 1, T - 1):
        xb = part_of(x, t * cols, cols, np.uint16)[None]
        if kind == "add":
            xb = plain.to(plain.wide(xb, dt).astype(np.float32) + plain.wide(part_of(res, t * cols, cols, np.uint16)[None], dt).astype(np.float32), dt)
            assert np.array_equal(part_of(h, t * cols, cols, np.uint16), xb[0])
        ref, want = plain.quant_rows(xb, dt) if kind == "quant" else plain.rms_norm(xb, w, eps, dt)
        assert np.array_equal(part_of(q, t * cols, cols, np.int8), ref[0]), f"row {t}"
        plain.assert_within(scales[t:t + 1].astype(np.float64), want, plain.SCALE * np.abs(want) + 2.0 ** -149, f"scale of row {t}")
    assert (part_of(q, T * cols, GUARD, np.uint8) == 0xA5).all()
