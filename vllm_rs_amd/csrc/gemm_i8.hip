// gemm_i8.hip — the C entry points of the 8-bit integer products (gemm_i8.cuh), and which kernel a product runs on.
#include "gemm_i8.cuh"

#include <algorithm>

namespace {

// a kernel: kind << 8 | its size, and the slices of K << 16
enum { I8_ANY = 0, I8_FEW = 1, I8_TILE = 2 };
struct Choice {
  int kind, size, slices;  // few: virtual columns / 16 of a workgroup; tile, any: rows / 64 * 16 + virtual columns / 64
};

// whether rows of x and w may be read 16 bytes at a time from where they begin
bool in_sixteens(const GemmI8Args& a) { return ((uintptr_t)a.x | (uintptr_t)a.w[0] | (uintptr_t)a.w[1] | (uintptr_t)a.K) % 16 == 0; }

int64_t over(int64_t a, int64_t b) { return (a + b - 1) / b; }

int64_t few_tiles(int N, bool pair, int C) { return over(N, pair ? C * 8 : C * 16); }
bool few_has(bool pair, int M, int C) {
  const int MT = (M + 15) / 16;
  return pair ? (C == 2 && MT <= 4) || (C == 4 && MT <= 2) || (C == 8 && MT == 1) : (C == 1 || C == 2 ? MT <= 4 : C == 4 && MT <= 2);
}
int64_t tile_count(int M, int N, bool pair, int t) { return over(M, (t >> 4) * 64) * over(N, (t & 15) * (pair ? 32 : 64)); }
bool any_has(int t) { return t == 0x11 || t == 0x22 || t == 0x44; }
int64_t tile_bytes(int t) { return (t >> 4) * (t & 15) * 16384; }  // of its sums
bool tile_has(int t) { return t == 0x12 || t == 0x22 || t == 0x32 || t == 0x24 || t == 0x34 || t == 0x44; }
// whether `slices` runs of K have a step each and meet within the workspace
bool slices_fit(int slices, int K, int64_t tiles, int64_t tile_bytes) {
  return slices == 1 || ((slices == 2 || slices == 4 || slices == 8) && slices <= K / 128 && tiles <= I8_WS_TILES && tiles * slices * tile_bytes <= (int64_t)I8_WS_PARTIAL_BYTES);
}
int64_t few_bytes(bool pair, int M, int C) { return (int64_t)((M + 15) / 16) * C * 1024; }  // of a workgroup's sums

// Times in us, fitted to 2018 (few) and 2957 (tile) measured ones: 1..64 and 17..8192 rows, 27 products of K = 992..18944 and 192..32000 columns, weights from memory; the
// choice by them is 0.65 % behind the best one of the same times on average and 17 % at most (411 of 472 products, the others chose what was not measured; none was held out).  Rows that are no whole lines of 128 bytes cost more on every way.
// few: what the busiest CU reads, at 36 GB/s, and the weights at 7.0 TB/s, the longer of them and a quarter of the other; the slices' meeting, for each of them and for each MB that they write and read
double few_us(bool pair, int M, int N, int K, int C, int slices) {
  const double wgs = (double)few_tiles(N, pair, C) * slices, t = pair ? 2 : 1;
  const double cu = (double)over((int64_t)wgs, 256) * (16.0 * C + M) * K / slices / 35.9e3 * (K % 128 ? 1.14 : 1.0);
  const double chip = t * N * K / 7.03e6 * (K % 128 ? 1.53 : 1.0);
  return 2.73 + (slices > 1 ? 0.92 + slices * (0.175 + 0.596 * over(M, 16) * 16 * N * t * 8e-6) : 0.0) + std::max(cu, chip) + 0.235 * std::min(cu, chip);
}
// tile: as in gemm_rows_tile (gemm_rows.cuh): rounds of 256 workgroups (64 x 128 on few: two a CU), for each a fixed time and one for each K step, the last round's between that of few workgroups
// and of all, less by the share `rows` of it where the last tile row is not full; never quicker than the weights' way through memory; and the slices' meeting
double tile_us(bool pair, int M, int N, int K, int t, int slices) {
  const int64_t wgs = tile_count(M, N, pair, t) * slices;
  const bool deep = t == 0x12 && wgs <= 256;
  struct Times { int tile; double t0, round, one, half, full, rows, meet, slice, mb; };
  static const Times times[7] = {{0x12, 3.1, 2.72, 0.474, 0.745, 0.693, 0.0, 0.0, 0.87, 0.164}, {0x22, 0.5, 4.25, 0.510, 0, 0.524, 0.466, 0.0, 0.77, 0.203},
                                 {0x32, 0.7, 4.41, 0.610, 0, 0.689, 0.151, 0.0, 0.97, 0.176}, {0x24, 0.0, 5.58, 0.771, 0, 0.858, 0.32, 0.0, 1.28, 0.155},
                                 {0x34, 0.7, 6.53, 0.821, 0, 1.080, 0.289, 0, 0, 0}, {0x44, 0.0, 8.78, 0.984, 0, 1.374, 0.517, 0, 0, 0},
                                 {0x12, 1.6, 2.53, 0.388, 0, 0.433, 0.207, 0.34, 0.53, 0.25}};
  const Times* c = &times[6];
  if (!deep)
    for (c = times; c->tile != t;) c++;
  const int bm = (t >> 4) * 64, bn = (t & 15) * 64, slots = t == 0x12 && !deep ? 512 : 256;
  const double full = (double)(wgs / slots), rem = (double)(wgs % slots), steps = (double)over(K, 128) / slices, rows = (double)M / over(M, bm);
  double last = rem > 0 ? c->one + (c->full - c->one) * rem / slots : 0.0;
  if (slots == 512 && rem > 0) last = rem <= 256 ? c->one : c->half + (c->full - c->half) * (rem - 256) / 256;
  const double fill = (1.0 - c->rows + c->rows * (bn + rows) / (bn + bm)) * (K % 128 ? 1.35 : 1.0);
  const double us = std::max(c->t0 + (full + (rem > 0)) * c->round + steps * fill * (full * c->full + last), 3.0 + (pair ? 2.0 : 1.0) * N * K / 6.3e6);
  return slices == 1 ? us : us + c->meet + c->slice * slices + c->mb * wgs * rows * bn * 8e-6;
}
// rows that begin anywhere, 1913 times of 176 products, 1..8192 rows, the choice 2.5 % behind the best of these on average, 39 % at most (4 rows x 5632 + 5632, K = 2001): the same forms.  any: 64 x 64 and 128 x 128 two workgroups a CU, a K step's time a
// constant and one for each of the CU's workgroups
double few_any_us(bool pair, int M, int N, int K, int slices) {
  const double t = pair ? 2 : 1, wgs = (double)over(N, 16);
  const double us = 3.2 + t * N * K / 8.9e6 + wgs * M * K / 9.4e6 + (double)over((int64_t)wgs * slices, 256) * (16.0 * t + M) * K / slices / 15.1e3;
  return slices == 1 ? us : us + 1.54 + slices * (0.04 + 0.67 * over(M, 16) * 16 * N * t * 8e-6);
}
double any_us(bool pair, int M, int N, int K, int t, int slices) {
  struct Times { int slots; double t0, round, one, each, meet, slice, mb; };
  static const Times times[3] = {{512, 3.0, 0.9, 0.322, 0.372, 0.65, 0.78, 0.276}, {512, 7.5, 0.0, 0.026, 1.07, 0.0, 1.56, 0.202}, {256, 1.5, 9.9, 2.26, 0.05, 0, 0, 0}};
  const Times& c = times[t == 0x11 ? 0 : t == 0x22 ? 1 : 2];
  const int64_t wgs = tile_count(M, N, pair, t) * slices;
  const double steps = (double)over(K, 128) / slices, full = (double)(wgs / c.slots), rem = (double)(wgs % c.slots);
  double us = c.t0 + full * (c.round + steps * (c.one + c.each * c.slots / 256));
  if (rem > 0) us += c.round + steps * (c.one + c.each * std::max(1.0, rem / 256));
  if (slices > 1) us += c.meet + c.slice * slices + c.mb * wgs * ((double)M / over(M, (t >> 4) * 64)) * (t & 15) * 64 * 8e-6;
  return std::max(us, 3.0 + (pair ? 2.0 : 1.0) * N * K / 5.0e6);
}

Choice choose(bool pair, int M, int N, int K, bool workspace, bool sixteens) {
  Choice best = {};
  double us = 0.0;
  auto offer = [&](int kind, int size, int slices, double v) {
    if (us == 0.0 || v < us) best = Choice{kind, size, slices}, us = v;
  };
  for (int slices = 1; slices <= (workspace ? 8 : 1); slices *= 2) {
    if (!sixteens) {
      const int one = pair ? 2 : 1;
      if (M <= 64 && slices_fit(slices, K, few_tiles(N, pair, one), few_bytes(pair, M, one))) offer(I8_FEW, one, slices, few_any_us(pair, M, N, K, slices));
      for (const int t : {0x11, 0x22, 0x44})
        if (t <= 0x22 ? slices_fit(slices, K, tile_count(M, N, pair, t), tile_bytes(t)) : slices == 1) offer(I8_ANY, t, slices, any_us(pair, M, N, K, t, slices));
      continue;
    }
    if (M <= 64)
      for (int C = 1; C <= 8; C *= 2)
        if (few_has(pair, M, C) && slices_fit(slices, K, few_tiles(N, pair, C), few_bytes(pair, M, C))) offer(I8_FEW, C, slices, few_us(pair, M, N, K, C, slices));
    if (M > 16)
      for (const int t : {0x12, 0x22, 0x32, 0x24, 0x34, 0x44})
        if (t <= 0x32 ? slices_fit(slices, K, tile_count(M, N, pair, t), tile_bytes(t)) : slices == 1) offer(I8_TILE, t, slices, tile_us(pair, M, N, K, t, slices));
  }
  return best;
}

template <bool PAIR, int MT, int C, bool ANY>
void few(const GemmI8Args& a, void* ws, int slices, hipStream_t st) {
  // (one row block of 16 columns: two steps at once pay, as a wave has little else in flight: 1 x 4096, K = 14336 12.9 us, 14.6 without; 32 rows 25.3 / 22.0)
  constexpr int U = MT == 1 && C == 1 ? 2 : 1;
  gemm_i8_few_kernel<PAIR, MT, C, U, ANY><<<(unsigned)(few_tiles(a.N, PAIR, C) * slices), I8_NW * 64, 0, st>>>(a, ws, slices);
}
template <bool PAIR, int C, bool ANY>
void few_rows(const GemmI8Args& a, void* ws, int slices, hipStream_t st) {
  constexpr int most = C <= 2 ? 4 : C == 4 ? 2 : 1;  // (few_has)
  if (a.M <= 16) return few<PAIR, 1, C, ANY>(a, ws, slices, st);
  if constexpr (most >= 2)
    if (a.M <= 32) return few<PAIR, 2, C, ANY>(a, ws, slices, st);
  if constexpr (most >= 4) a.M <= 48 ? few<PAIR, 3, C, ANY>(a, ws, slices, st) : few<PAIR, 4, C, ANY>(a, ws, slices, st);
}

// launches on up to 160 KB of LDS
template <auto KERNEL>
void launch_lds(unsigned grid, int threads, size_t lds, const GemmI8Args& a, const GemmI8Tiles& g, hipStream_t st) {
  static uint64_t attr_devs = 0;  // function attributes belong to the device current at the call
  int dev = 0;
  (void)hipGetDevice(&dev);
  if (!((__atomic_load_n(&attr_devs, __ATOMIC_RELAXED) >> (dev & 63)) & 1)) {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    __atomic_fetch_or(&attr_devs, (uint64_t)1 << (dev & 63), __ATOMIC_RELAXED);
  }
  KERNEL<<<grid, threads, lds, st>>>(a, g);
}
template <bool PAIR, int BM, int BN>
GemmI8Tiles tiles_of(const GemmI8Args& a, void* ws, int slices) {
  constexpr int BC = PAIR ? BN / 2 : BN;
  return {ws, (a.M + BM - 1) / BM, (a.N + BC - 1) / BC, slices};
}
template <bool PAIR, int BM, int BN, bool DEEP>
void tile(const GemmI8Args& a, void* ws, int slices, hipStream_t st) {
  using G = GrTile<BM, BN, DEEP>;
  const GemmI8Tiles g = tiles_of<PAIR, BM, BN>(a, ws, slices);
  launch_lds<gemm_i8_tile_kernel<PAIR, BM, BN, DEEP>>((unsigned)(g.MT * g.NT * slices), 512, (size_t)G::S * G::KP * G::STG, a, g, st);
}
template <bool PAIR, int BM, int BN, int NT, int D>
void any(const GemmI8Args& a, void* ws, int slices, hipStream_t st) {
  const GemmI8Tiles g = tiles_of<PAIR, BM, BN>(a, ws, slices);
  launch_lds<gemm_i8_any_kernel<PAIR, BM, BN, NT, D>>((unsigned)(g.MT * g.NT * slices), NT, (size_t)2 * (BM + BN) * 128, a, g, st);
}

template <bool PAIR>
void run(const GemmI8Args& a, void* ws, const Choice& c, hipStream_t st) {
  const bool sixteens = in_sixteens(a);
  if (c.kind == I8_FEW) {
    constexpr int one = PAIR ? 2 : 1;
    if (!sixteens) return few_rows<PAIR, one, true>(a, ws, c.slices, st);
    if (c.size == 2) return few_rows<PAIR, 2, false>(a, ws, c.slices, st);
    if (c.size == 4) return few_rows<PAIR, 4, false>(a, ws, c.slices, st);
    return few_rows<PAIR, PAIR ? 8 : 1, false>(a, ws, c.slices, st);
  }
  if (c.kind == I8_TILE) {
    if (c.size == 0x44) return tile<PAIR, 256, 256, false>(a, ws, c.slices, st);
    if (c.size == 0x34) return tile<PAIR, 192, 256, false>(a, ws, c.slices, st);
    if (c.size == 0x24) return tile<PAIR, 128, 256, false>(a, ws, c.slices, st);
    if (c.size == 0x32) return tile<PAIR, 192, 128, false>(a, ws, c.slices, st);
    if (c.size == 0x22) return tile<PAIR, 128, 128, false>(a, ws, c.slices, st);
    // 64 x 128: two K steps a phase where every workgroup has a CU to itself, otherwise two workgroups a CU (gemm_rows_launch)
    if (tile_count(a.M, a.N, PAIR, 0x12) * c.slices <= 256) return tile<PAIR, 64, 128, true>(a, ws, c.slices, st);
    return tile<PAIR, 64, 128, false>(a, ws, c.slices, st);
  }
  if (c.size == 0x44) return any<PAIR, 256, 256, 512, 1>(a, ws, c.slices, st);
  if (c.size == 0x22) return any<PAIR, 128, 128, 256, 2>(a, ws, c.slices, st);
  any<PAIR, 64, 64, 256, 2>(a, ws, c.slices, st);
}

// a launch stays within 2^32 threads, and the rows of its tiles within 2^31: 2^22 tiles of 64 x 64 (2^31 threads on the kernels that take most for a result: 64 x 32 of 256, 64 x 64 of 512);
// what has slices has few tiles and is not cut.  kernel_of(part): the kernel of each part
template <class F>
void in_parts(GemmI8Args a, bool pair, void* ws, hipStream_t st, F kernel_of) {
  const int64_t most = std::max<int64_t>((((int64_t)1 << 22) / (a.N / 64 + 1) * 64) & ~(int64_t)255, 256);
  while (a.M > 0) {
    GemmI8Args part = a;
    part.M = (int)std::min<int64_t>(a.M, most);
    const Choice c = kernel_of(part);
    if (pair) run<true>(part, ws, c, st);
    else run<false>(part, ws, c, st);
    const size_t by = (size_t)part.M * a.N * (a.dtype == VRA_F32 ? 4 : 2);
    a.x += (size_t)part.M * a.K, a.xs += part.M, a.out = static_cast<char*>(a.out) + by, a.M -= part.M;
    if (a.residual) a.residual = static_cast<const char*>(a.residual) + by;
  }
}
void launch(const GemmI8Args& a, bool pair, void* ws, hipStream_t st) {
  const bool sixteens = in_sixteens(a);
  in_parts(a, pair, ws, st, [&](const GemmI8Args& part) { return choose(pair, part.M, a.N, a.K, ws != nullptr, sixteens); });
}

bool product_ok(const char* who, const GemmI8Args& a, bool pair, const void* workspace) {
  if (a.M < 0 || a.K <= 0 || a.K > 131071 || a.N <= 0 || a.N > 1 << 24) {
    vra_set_error("%s: m >= 0, 1 <= k <= 131071 (sums of 32 bits), 1 <= n <= 2^24 (m=%d k=%d n=%d)", who, a.M, a.K, a.N);
    return false;
  }
  const bool f32 = a.dtype == VRA_F32;
  if (a.dtype != VRA_BF16 && a.dtype != VRA_F16 && !(f32 && !pair)) {
    vra_set_error("%s: dtype must be bf16/f16%s", who, pair ? "" : "/f32");
    return false;
  }
  if (a.M == 0) return true;
  if (!a.x || !a.xs || !a.out || !a.w[0] || !a.ws[0] || (pair && (!a.w[1] || !a.ws[1]))) {
    vra_set_error("%s: null pointer", who);
    return false;
  }
  if (((uintptr_t)a.xs | (uintptr_t)a.ws[0] | (uintptr_t)a.ws[1]) % 4 || ((uintptr_t)a.bias | (uintptr_t)a.residual | (uintptr_t)a.out) % (f32 ? 4 : 2)) {
    vra_set_error("%s: a pointer that is not a multiple of its elements' size", who);
    return false;
  }
  if ((uintptr_t)workspace % 16) {
    vra_set_error("%s: the workspace begins at a multiple of 16", who);
    return false;
  }
  return true;
}

}  // namespace

extern "C" size_t vra_w8a8_workspace_bytes(void) { return I8_WS_BYTES; }

extern "C" void vra_w8a8_gemm(const int8_t* x, const float* x_scales, const int8_t* w, const float* w_scales, const void* bias, const void* residual, void* out,
                              void* workspace, int32_t m, int32_t k, int32_t n, int32_t dtype, int64_t stream) {
  const GemmI8Args a = {x, x_scales, {w, nullptr}, {w_scales, nullptr}, bias, residual, out, m, n, k, dtype};
  if (product_ok("vra_w8a8_gemm", a, false, workspace)) launch(a, false, workspace, as_stream(stream));
}
extern "C" void vra_w8a8_gate_up_silu(const int8_t* x, const float* x_scales, const int8_t* w_gate, const float* s_gate, const int8_t* w_up, const float* s_up,
                                      void* out, void* workspace, int32_t m, int32_t k, int32_t n, int32_t dtype, int64_t stream) {
  const GemmI8Args a = {x, x_scales, {w_gate, w_up}, {s_gate, s_up}, nullptr, nullptr, out, m, n, k, dtype};
  if (product_ok("vra_w8a8_gate_up_silu", a, true, workspace)) launch(a, true, workspace, as_stream(stream));
}

extern "C" int32_t vra_w8a8_kernel(int32_t pair, int32_t m, int32_t k, int32_t n, int32_t has_workspace) {
  if (m <= 0 || k <= 0 || k > 131071 || n <= 0 || n > 1 << 24) return 0;
  const Choice c = choose(pair != 0, m, n, k, has_workspace != 0, k % 16 == 0);
  return c.slices << 16 | c.kind << 8 | c.size;
}
extern "C" void vra_w8a8_gemm_on(int32_t kernel, const int8_t* x, const float* x_scales, const int8_t* w, const float* w_scales, const int8_t* w_up, const float* s_up,
                                 const void* bias, const void* residual, void* out, void* workspace, int32_t m, int32_t k, int32_t n, int32_t dtype, int64_t stream) {
  const bool pair = w_up != nullptr;
  const GemmI8Args a = {x, x_scales, {w, w_up}, {w_scales, s_up}, bias, residual, out, m, n, k, dtype};
  if (!product_ok("vra_w8a8_gemm_on", a, pair, workspace) || m == 0) return;
  const Choice c = {kernel >> 8 & 255, kernel & 255, kernel >> 16};
  bool has = !(pair && (bias || residual)) && c.slices >= 1 && (c.slices == 1 || workspace);
  if (c.kind == I8_FEW) {
    has = has && few_has(pair, m, c.size) && slices_fit(c.slices, k, few_tiles(n, pair, c.size), few_bytes(pair, m, c.size)) && (in_sixteens(a) || c.size == (pair ? 2 : 1));
  } else if (c.kind == I8_TILE) {
    has = has && tile_has(c.size) && in_sixteens(a) && (c.size <= 0x32 ? slices_fit(c.slices, k, tile_count(m, n, pair, c.size), tile_bytes(c.size)) : c.slices == 1);
  } else {
    has = has && c.kind == I8_ANY && any_has(c.size) && (c.size <= 0x22 ? slices_fit(c.slices, k, tile_count(m, n, pair, c.size), tile_bytes(c.size)) : c.slices == 1);
  }
  VRA_CHECK_ARG(has, "vra_w8a8_gemm_on: no such kernel for this product");
  in_parts(a, pair, workspace, as_stream(stream), [&](const GemmI8Args&) { return c; });
}
