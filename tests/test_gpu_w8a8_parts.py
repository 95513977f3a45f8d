"""W8A8 products of more rows than a launch takes, on named kernels: cut in parts as the public entry cuts them."""
import numpy as np
import pytest

from tests import w8a8_plain as plain
from tests.test_gpu_w8a8 import GUARD, Guarded, part_of
from tests.util import BF16, rng
from vllm_rs_amd import ops

pytestmark = pytest.mark.gpu
MOST = 1 << 28  # rows of a part where there is one column of tiles


# the last size at which one launch held 2^32 threads is 2^30 - 64 rows for 64 x 64 tiles of 256 threads, 2^29 - 64 for 64 x 128 of 512; near 2^31 rows the tiles' rows leave 32 bits
@pytest.mark.parametrize("kernel, M, K, N, pair", [(0x10011, (1 << 30) + 70, 1, 1, 0), (0x10011, (1 << 29) + 70, 1, 33, 1), (0x10012, (1 << 29) + 70, 16, 1, 0), (0x10022, (1 << 29) + 70, 1, 1, 0),
                                                   (0x10044, (1 << 31) - 1, 1, 1, 0), (0x10022, (1 << 31) - 1, 1, 1, 0), (None, (1 << 31) - 1, 1, 1, 0)])
def test_more_rows_than_a_launch_takes(kernel, M, K, N, pair):
    L, r = ops.lib(), rng(K)
    if kernel is not None and K == 16:
        kernel |= 0x200
    x, xs, out = ops.DevBuf(M * K + 4), ops.DevBuf(M * 4), Guarded(M * N * 2)
    L.vra_fill_hash_u32(x.ptr, (M * K + 3) // 4, 3, 0)
    L.vra_fill_normal(xs.ptr, M, 4, 0.0, 1.0, 2, 0)
    res = None if pair else ops.DevBuf(M * N * 2)
    if not pair:
        L.vra_fill_normal(res.ptr, M * N, 5, 0.0, 1.0, BF16, 0)
    w, ws = [r.integers(-128, 128, (N, K)).astype(np.int8) for _ in range(2)], [(0.5 + r.random(N)).astype(np.float32) / 100 for _ in range(2)]
    wd, sd = [ops.dev(t) for t in w], [ops.dev(t) for t in ws]
    if kernel is None:
        L.vra_w8a8_gemm(x.ptr, xs.ptr, wd[0].ptr, sd[0].ptr, None, res.ptr, out.at, None, M, K, N, BF16, 0)
    else:
        L.vra_w8a8_gemm_on(kernel, x.ptr, xs.ptr, wd[0].ptr, sd[0].ptr, wd[1].ptr if pair else None, sd[1].ptr if pair else None, None, res and res.ptr, out.at, None, M, K, N, BF16, 0)
    ops.check_error()
    n = 400
    for at in [0, M - n] + [c - n // 2 for c in range(MOST, M - n, MOST)]:
        xh, sh = part_of(x, at * K, n * K, np.int8).reshape(n, K), part_of(xs, at, n, np.float32)
        rh = None if pair else part_of(res, at * N, n * N, np.uint16).reshape(n, N)
        ref, bound = plain.gate_up_silu(xh, sh, w[0], ws[0], w[1], ws[1], BF16) if pair else plain.gemm(xh, sh, w[0], ws[0], None, rh, BF16)
        plain.assert_within(plain.wide(part_of(out, at * N, n * N, np.uint16).reshape(n, N), BF16), ref, bound, f"rows from {at}")
    assert (part_of(out, 2 * M * N, GUARD, np.uint8) == 0xA5).all()
