// gemm_i8.cuh — products of 8-bit integers with a scale a row (token) and a scale a column (channel):
//   out[m, n] = round( xs[m] ws[n] sum_k x[m, k] w[n, k]  + bias[n] + residual[m, n] ),   pair: round( silu(g) u ), g and u such products.
// Sums are 32-bit integers (K <= 131071: |sum| <= 128 128 K < 2^31): exact, the same in any order, so no split of K changes a bit.  The scales, the bias and
// the residual are applied in f32, with one rounding at the end.  Weights are row-major [n, K] as checkpoints hold them.
// Weights = A, rows of x = B of v_mfma_i32_16x16x64_i8 (16 bytes of a row a lane; a lane's result: 4 consecutive columns of one row), at the bf16 instruction's
// clocks for twice the K: every byte of an operand costs what it costs the 16-bit kernels (gemm_rows.cuh).
#pragma once
#include <type_traits>

#include "gemm_rows.cuh"

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a1 __attribute__((aligned(1)));  // 16 bytes anywhere

// (the forms and hazards of common.cuh's 16-bit instructions: tied accumulator; mfma_i8_ready: operands not written by VALU within two wait states)
__device__ __forceinline__ void mfma_i8(i32x4& acc, u32x4 a, u32x4 b) {
  asm volatile("s_nop 1\n\tv_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+v"(acc) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mfma_i8_ready(i32x4& acc, u32x4 a, u32x4 b) {
  asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+v"(acc) : "v"(a), "v"(b));
}
__device__ __forceinline__ i32x4 zero_acc_i8() {
  i32x4 z = {0, 0, 0, 0};
  asm volatile("" : "+v"(z));
  return z;
}

struct GemmI8Args {
  const int8_t* x;
  const float* xs;
  const int8_t* w[2];  // pair: gate, up
  const float* ws[2];
  const void* bias;
  const void* residual;  // (may be out: a lane reads an element before it writes it)
  void* out;
  int M, N, K;  // pair: N columns of each tensor
  int dtype;    // of out, bias and residual
};

struct PlainF32 {};  // VRA_F32 as a type of the epilogue

// what stands behind the sums g (and u) of an element
template <bool PAIR>
__device__ __forceinline__ float i8_value(int g, int u, float xs, float gs, float us) {
  float v = (float)g * xs * gs;
  if (PAIR) {
    // silu(v) u = v u / (1 + exp(-v)); below zero exp(v / 2) goes to both factors: exp(-v) would end at v = -88, where bf16 still holds the result.  The hardware's
    // exp2 and reciprocal, a step each and |v| / 2 steps by the exponent's rounding: a 16-bit result's own rounding is 2^12 (f16) and 2^15 times as coarse
    const float h = __builtin_amdgcn_exp2f(-0.72134752f * fabsf(v)), s = v < 0.f ? h : 1.0f;
    v = v * s * __builtin_amdgcn_rcpf(fmaf(h, h, 1.0f)) * ((float)u * xs * us * s);
  }
  asm("" : "+v"(v));  // (the last product is not drawn into a conversion to f16, here or there: the bits are the same in all kernels)
  return v;
}

// rows begin anywhere: 16 bytes at a multiple of an element
typedef f32x4 f32x4_a4 __attribute__((aligned(4)));
typedef u32x2 u32x2_a2 __attribute__((aligned(2)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
// columns n .. n + 3 (those within N) of a row of 16- or 32-bit elements as they are stored; the others are left alone
template <class One, class V>
__device__ __forceinline__ void i8_four(const void* row, int n, int N, V& v) {
  typedef typename std::conditional<sizeof(One) == 4, f32x4_a4, u32x2_a2>::type Anywhere;
  const One* const h = static_cast<const One*>(row) + n;
  if (n + 4 <= N) v = *reinterpret_cast<const Anywhere*>(h);
  else if (n < N) {
    v = V{};
#pragma unroll
    for (int e = 0; e < 3; e++)
      if (n + e < N) {
        if constexpr (sizeof(One) == 4) v[e] = h[e];
        else v[e >> 1] |= (uint32_t)h[e] << (e & 1 ? 16 : 0);
      }
  }
}
// A wave's R blocks of 16 rows x 64 virtual columns: lane (r16, q4) holds columns 4 q4 .. + 3 of the four tiles of a block (acc[block][tile]), of its row r16.  m: that row in
// block 0; n0: the wave's first column.  What is read of rows and columns is asked for together, the residual two blocks ahead;
// 16-bit results trade places between a row's four lanes and go out 16 bytes a lane.
template <class T, bool PAIR, int R>
__device__ __forceinline__ void i8_store_rows(const GemmI8Args& a, int m, int n0, int q4, const i32x4 (&acc)[R][4]) {
  constexpr int NJ = PAIR ? 2 : 4;
  constexpr bool F32 = std::is_same<T, PlainF32>::value;
  typedef typename std::conditional<F32, f32x4, u32x2>::type Four;
  typedef typename std::conditional<F32, float, uint16_t>::type One;
  const int M = a.M, N = a.N;
  float gs[NJ][4], us[NJ][4], xs[R];
  Four bias[NJ], res[2][NJ];
  auto scales = [&](const float* p, int n, float (&f)[4]) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    i8_four<float>(p, n, N, v);
#pragma unroll
    for (int e = 0; e < 4; e++) f[e] = v[e];
  };
  auto fetch = [&](int i) {
    const One* const row = static_cast<const One*>(a.residual) + (size_t)min(m + i * 16, M - 1) * N;
#pragma unroll
    for (int j = 0; j < NJ; j++) i8_four<One>(row, n0 + j * 16 + q4 * 4, N, res[i & 1][j]);
  };
  const bool has_res = !PAIR && a.residual, has_bias = !PAIR && a.bias;
  if (has_res) {
    fetch(0);
    if (R > 1) fetch(1);
  }
#pragma unroll
  for (int j = 0; j < NJ; j++) {
    const int n = n0 + j * 16 + q4 * 4;
    scales(a.ws[0], n, gs[j]);
    if (PAIR) scales(a.ws[1], n, us[j]);
    if (has_bias) i8_four<One>(a.bias, n, N, bias[j]);
  }
#pragma unroll
  for (int i = 0; i < R; i++) xs[i] = a.xs[min(m + i * 16, M - 1)];
  auto add = [&](float (&y)[4], const Four& v) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if constexpr (F32) y[e] += v[e];
      else y[e] += T::to_f32((uint16_t)(v[e >> 1] >> (e & 1 ? 16 : 0)));
    }
  };
#pragma unroll
  for (int i = 0; i < R; i++) {
    float y[NJ][4];
#pragma unroll
    for (int j = 0; j < NJ; j++) {
#pragma unroll
      for (int e = 0; e < 4; e++) y[j][e] = i8_value<PAIR>(acc[i][PAIR ? 2 * j : j][e], acc[i][PAIR ? 2 * j + 1 : j][e], xs[i], gs[j][e], PAIR ? us[j][e] : 0.f);
      if (has_bias) add(y[j], bias[j]);
      if (has_res) add(y[j], res[i & 1][j]);
    }
    if (has_res && i + 2 < R) fetch(i + 2);
    const bool in = m + i * 16 < M;
    One* const row = static_cast<One*>(a.out) + (size_t)(m + i * 16) * N;
    if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < NJ; j++) {
        const int n = n0 + j * 16 + q4 * 4;
        if (in && n + 4 <= N) *reinterpret_cast<f32x4_a4*>(row + n) = f32x4{y[j][0], y[j][1], y[j][2], y[j][3]};
        else if (in)
#pragma unroll
          for (int e = 0; e < 3; e++)
            if (n + e < N) row[n + e] = y[j][e];
      }
    } else {
      u32x2 v[NJ];
#pragma unroll
      for (int j = 0; j < NJ; j++) v[j] = u32x2{T::pack2(y[j][0], y[j][1]), T::pack2(y[j][2], y[j][3])};
      gr_gather_columns(v);
#pragma unroll
      for (int h = 0; h < NJ / 2; h++) {
        const int n = n0 + q4 * (NJ * 4) + h * 8;
        const u32x4 p = {v[2 * h][0], v[2 * h][1], v[2 * h + 1][0], v[2 * h + 1][1]};
        if (in && n + 8 <= N) *reinterpret_cast<u32x4_a2*>(row + n) = p;
        else if (in)
#pragma unroll
          for (int e = 0; e < 7; e++)
            if (n + e < N) row[n + e] = (uint16_t)(p[e >> 1] >> (e & 1 ? 16 : 0));
      }
    }
  }
}
template <bool PAIR, int R>
__device__ __forceinline__ void i8_store_rows(const GemmI8Args& a, int m, int n0, int q4, const i32x4 (&acc)[R][4]) {
  if (a.dtype == VRA_BF16) i8_store_rows<BF16, PAIR, R>(a, m, n0, q4, acc);
  else if (PAIR || a.dtype == VRA_F16) i8_store_rows<F16, PAIR, R>(a, m, n0, q4, acc);
  else if constexpr (!PAIR) i8_store_rows<PlainF32, PAIR, R>(a, m, n0, q4, acc);
}

// 16 bytes of a row of K from byte k on (k a multiple of 16), zeros behind the row's end; any address, nothing beyond the row is read
__device__ __forceinline__ u32x4 i8_load16(const int8_t* row, int k, int K) {
  u32x4 v = {0u, 0u, 0u, 0u};
  if (k + 16 <= K) return *reinterpret_cast<const u32x4_a1*>(row + k);
  if (k < K) {
    const int left = K - k;
    if (K >= 16) {  // the row's last 16 bytes, the first of them shifted out
      const u32x4 t = *reinterpret_cast<const u32x4_a1*>(row + K - 16);
      const int d = (16 - left) >> 2, b = (16 - left) & 3;
      uint32_t s[8];
#pragma unroll
      for (int i = 0; i < 8; i++) s[i] = i < 4 ? t[i] : 0u;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t lo = d == 0 ? s[i] : d == 1 ? s[i + 1] : d == 2 ? s[i + 2] : s[i + 3], hi = d == 0 ? s[i + 1] : d == 1 ? s[i + 2] : d == 2 ? s[i + 3] : s[i + 4];
        v[i] = __builtin_amdgcn_alignbyte(hi, lo, b);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 15; e++)
        if (e < left) v[e >> 2] |= (uint32_t)(uint8_t)row[k + e] << (8 * (e & 3));
    }
  }
  return v;
}

// ---------------------------------------------------------------- few rows (decode)
// Where the K slices of a product meet: the sums of every slice, and a counter for each wave of a tile (a line each), zero between calls.
#define I8_WS_TILES 1024
#define I8_WS_PARTIALS ((size_t)I8_WS_TILES * 8 * 64)
#define I8_WS_PARTIAL_BYTES ((size_t)32 << 20)
#define I8_WS_BYTES (I8_WS_PARTIALS + I8_WS_PARTIAL_BYTES)

// A wave stores its V sums a lane of slice z and counts itself; the last of the `slices` waves of the same place of the tile adds the others' sums to its own, sets the counter back and
// returns true.  Nobody waits for anybody, and where slices end together their waves share the work.  Sums go through memory with agent scope (sc1: the L2s of the XCDs are
// not coherent); a wave's stores are acknowledged before it counts itself, and the last one reads behind all counts.  It asks for several slices at a time: one after the other they were
// 0.8 .. 1.7 us each, and a workgroup's waves waited for its last (150 x 3584, K = 18944, four slices of 128 x 128: 29.4 us, so 28.0; 32 x 512, K = 14336, eight slices: 8.9, 7.6).
template <int V, int THREADS>
__device__ __forceinline__ bool i8_meet(int (&v)[V], void* ws, int tile, int tiles, int z, int slices) {
  static_assert(V % 4 == 0, "16 bytes a lane");
  constexpr int B = V <= 16 ? 4 : V <= 32 ? 3 : 2;  // slices in flight
  const int tid = threadIdx.x;
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(static_cast<char*>(ws) + I8_WS_PARTIALS, 0, (int)I8_WS_PARTIAL_BYTES, 0x00020000u);
  auto at = [&](int s, int i) { return (uint32_t)(((s * tiles + tile) * (V / 4) + i) * THREADS + tid) * 16u; };
#pragma unroll
  for (int i = 0; i < V / 4; i++)
    __builtin_amdgcn_raw_buffer_store_b128(u32x4{(uint32_t)v[4 * i], (uint32_t)v[4 * i + 1], (uint32_t)v[4 * i + 2], (uint32_t)v[4 * i + 3]}, r, at(z, i), 0, 16);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  uint32_t* const count = static_cast<uint32_t*>(ws) + (tile * 8 + (tid >> 6)) * 16;
  uint32_t before = 0u;
  if ((tid & 63) == 0) before = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  before = __builtin_amdgcn_readfirstlane(before);
  asm volatile("" ::: "memory");
  if (before != (uint32_t)slices - 1u) return false;
  for (int s0 = 1; s0 < slices; s0 += B) {
    u32x4 p[B][V / 4];
#pragma unroll
    for (int b = 0; b < B; b++) {
      const int s = z + s0 + b, o = s0 + b < slices ? (s >= slices ? s - slices : s) : z;  // (behind the last: its own again, not added)
#pragma unroll
      for (int i = 0; i < V / 4; i++) p[b][i] = __builtin_amdgcn_raw_buffer_load_b128(r, at(o, i), 0, 16);
    }
#pragma unroll
    for (int b = 0; b < B; b++)
      if (s0 + b < slices)
#pragma unroll
        for (int i = 0; i < V; i++) v[i] += (int)p[b][i >> 2][i & 3];
  }
  if ((tid & 63) == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return true;
}

#define I8_NW 8
// Bound: the weights' way through memory.  A workgroup takes 16 C virtual columns (pair: gate and up blocks of 16 in turn), all MT 16 rows and one of `slices` runs of
// K; its eight waves take the run's steps of 128 in turn, straight into registers, U of them asked for at once.  The waves' sums meet in LDS, the slices' in the workspace.  ANY: rows that begin anywhere, or K off 16.
template <bool PAIR, int MT, int C, int U, bool ANY>
__global__ __launch_bounds__(I8_NW * 64) void gemm_i8_few_kernel(const GemmI8Args a, void* ws, int slices) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int NW = I8_NW;
  constexpr int CO = PAIR ? C / 2 : C, FOURS = MT * CO * 64;  // four results a thread
  static_assert(FOURS <= NW * 64, "a thread has one four");
  __shared__ __attribute__((aligned(16))) int part[NW * MT * C * 256];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int M = a.M, N = a.N, K = a.K, tile = (int)blockIdx.x / slices, z = (int)blockIdx.x - tile * slices, n0 = tile * CO * 16;
  // a lane's two pieces of a step: one of each half, so that a request is for 64 bytes of a row.  It meets fewer lines than one for 128 where rows do not begin with one (pieces side by side / so:
  // pair 11 x 9216, K = 9264 49.9 / 47.4 us, 11 x 17024, K = 4384 26.9 / 24.2; whole lines 1 % slower, and with the form by K 7 %, for its registers)
  const int8_t* wp[C];
  const int8_t* xp[MT];
#pragma unroll
  for (int c = 0; c < C; c++) wp[c] = (PAIR && (c & 1) ? a.w[1] : a.w[0]) + (size_t)min(n0 + (PAIR ? c >> 1 : c) * 16 + r16, N - 1) * K + q4 * 16;
#pragma unroll
  for (int i = 0; i < MT; i++) xp[i] = a.x + (size_t)min(i * 16 + r16, M - 1) * K + q4 * 16;
  u32x4 w[U][C][2], x[U][MT][2];
  auto load = [&](int u, int step) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int at = step * 128 + h * 64;
#pragma unroll
      for (int c = 0; c < C; c++) w[u][c][h] = ANY ? (u32x4)*reinterpret_cast<const u32x4_a1*>(wp[c] + at) : *reinterpret_cast<const u32x4*>(wp[c] + at);
#pragma unroll
      for (int i = 0; i < MT; i++)
        if (i * 16 + r16 < M) x[u][i][h] = ANY ? (u32x4)*reinterpret_cast<const u32x4_a1*>(xp[i] + at) : *reinterpret_cast<const u32x4*>(xp[i] + at);
    }
  };
  i32x4 acc[MT][C];
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int c = 0; c < C; c++) acc[i][c] = zero_acc_i8();
  auto product = [&](int u) {
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int c = 0; c < C; c++) mfma_i8(acc[i][c], w[u][c][h], x[u][i][h]);
  };
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int i = 0; i < MT; i++) x[u][i][0] = x[u][i][1] = u32x4{0u, 0u, 0u, 0u};  // (rows beyond M)
  // the epilogue's operands: thread t has columns 4 (t / 16 % 4) .. + 3 of block t / 64 % CO, row t % 16 of row block t / (64 CO)
  const int m = tid / (64 * CO) * 16 + r16, n = n0 + (tid >> 6) % CO * 16 + q4 * 4;
  const bool mine = tid < FOURS && m < M && n < N, f32 = a.dtype == VRA_F32;
  const size_t row = (size_t)m * N;
  float xs = 0.f;
  f32x4 gs = {}, us = {}, bias4 = {}, res4 = {};
  u32x2 bias2 = {}, res2 = {};
  if (mine) {
    xs = a.xs[m];
    i8_four<float>(a.ws[0], n, N, gs);
    if (PAIR) i8_four<float>(a.ws[1], n, N, us);
    else if (f32) {
      if (a.bias) i8_four<float>(a.bias, n, N, bias4);
      if (a.residual) i8_four<float>(static_cast<const float*>(a.residual) + row, n, N, res4);
    } else {
      if (a.bias) i8_four<uint16_t>(a.bias, n, N, bias2);
      if (a.residual) i8_four<uint16_t>(static_cast<const uint16_t*>(a.residual) + row, n, N, res2);
    }
  }
  // steps of 128 of the run, begun at another place in every workgroup: rows of a power of two bytes lie on the same channels of the memory, and all workgroups would ask for the same
  // of them at a time (pair 1 x 14336, K = 4096, in order / so: 24.9 / 22.0 us; K = 3584: no difference)
  const int whole = K >> 7, s0 = (int)((int64_t)whole * z / slices), len = (int)((int64_t)whole * (z + 1) / slices) - s0, turn = len ? tile * 5 % len : 0;
  auto place = [&](int s) { return s0 + (s + turn < len ? s + turn : s + turn - len); };
  for (int s = wave; s < len; s += NW * U) {
#pragma unroll
    for (int u = 0; u < U; u++)
      if (s + u * NW < len) load(u, place(s + u * NW));
#pragma unroll
    for (int u = 0; u < U; u++)
      if (s + u * NW < len) product(u);
  }
  if ((K & 127) && z == slices - 1 && wave == whole % NW) {  // what K leaves behind whole steps; a chunk beyond it counts nothing, as its x is zero
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int k = whole * 128 + h * 64 + q4 * 16;
#pragma unroll
      for (int c = 0; c < C; c++) w[0][c][h] = i8_load16(wp[c] - q4 * 16, k, K);
#pragma unroll
      for (int i = 0; i < MT; i++) x[0][i][h] = i8_load16(xp[i] - q4 * 16, k, K);
    }
    product(0);
  }
  VRA_MFMA_DRAIN();
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int c = 0; c < C; c++) *reinterpret_cast<i32x4*>(&part[((wave * MT + i) * C + c) * 256 + lane * 4]) = acc[i][c];
  __syncthreads();
  if (wave * 64 >= FOURS) return;
  int sums[PAIR ? 8 : 4];
  const int b = tid >> 6;  // block (row block, column block) of the results; its sums are in blocks of C a row block
  const int* const p = &part[(PAIR ? b * 2 : b) * 256 + lane * 4];
  i32x4 g = {0, 0, 0, 0}, u = {0, 0, 0, 0};
#pragma unroll
  for (int v = 0; v < NW; v++) {
    g += *reinterpret_cast<const i32x4*>(p + v * MT * C * 256);
    if (PAIR) u += *reinterpret_cast<const i32x4*>(p + v * MT * C * 256 + 256);
  }
  if (slices > 1) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      sums[e] = g[e];
      if (PAIR) sums[4 + e] = u[e];
    }
    if (!i8_meet<PAIR ? 8 : 4, FOURS>(sums, ws, tile, (int)gridDim.x / slices, z, slices)) return;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      g[e] = sums[e];
      if (PAIR) u[e] = sums[4 + e];
    }
  }
  if (!mine) return;
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; e++) y[e] = i8_value<PAIR>(g[e], u[e], xs, gs[e], us[e]);
  if (f32) {
    float* const to = static_cast<float*>(a.out) + row + n;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (a.bias) y[e] += bias4[e];
      if (a.residual) y[e] += res4[e];
    }
    if (n + 4 <= N) *reinterpret_cast<f32x4_a4*>(to) = f32x4{y[0], y[1], y[2], y[3]};
    else
#pragma unroll
      for (int e = 0; e < 3; e++)
        if (n + e < N) to[e] = y[e];
    return;
  }
  auto store = [&](auto t) {
    using T = decltype(t);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (!PAIR && a.bias) y[e] += T::to_f32((uint16_t)(bias2[e >> 1] >> (e & 1 ? 16 : 0)));
      if (!PAIR && a.residual) y[e] += T::to_f32((uint16_t)(res2[e >> 1] >> (e & 1 ? 16 : 0)));
    }
    uint16_t* const to = static_cast<uint16_t*>(a.out) + row + n;
    if (n + 4 <= N) *reinterpret_cast<u32x2_a2*>(to) = u32x2{T::pack2(y[0], y[1]), T::pack2(y[2], y[3])};
    else
#pragma unroll
      for (int e = 0; e < 3; e++)
        if (n + e < N) to[e] = T::from_f32(y[e]);
  };
  if (a.dtype == VRA_BF16) store(BF16{});
  else store(F16{});
#endif
}

// ---------------------------------------------------------------- many rows (prompts, larger batches)
// The loop, the two groups of waves and the LDS layout of gemm_rows.cuh, whose K step of 64 16-bit elements is 128 bytes of a row as one of 128 here is: the same requests,
// LDS reads and clocks, twice the products.  Bound: as there, the chip's power at 256 x 256, what a CU gets past L2 below it.
// K any multiple of 16: in the last step a chunk of x beyond K is taken as zeros, so what stands in its place of w (the next row's bytes) counts nothing; the
// tensors' descriptors end with their last row, nothing behind it is read.
// slices > 1: a tile's K steps in as many runs, a workgroup each, that meet in the workspace (i8_meet).
struct GemmI8Tiles {
  void* ws;
  int MT, NT, slices;
};

// PAIR: virtual columns, gate and up interleaved in blocks of 16
template <bool PAIR, int BM, int BN, bool DEEP>
__global__ __launch_bounds__(512, 2) void gemm_i8_tile_kernel(const GemmI8Args a, const GemmI8Tiles g) {
#ifdef __HIP_DEVICE_COMPILE__
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  using G = GrTile<BM, BN, DEEP>;
  constexpr int H = G::H, KP = G::KP, S = G::S, NX = G::NX, STG = G::STG, EX = G::EX, EW = G::EW, D = EX + EW;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wg = wave >> 2, cw = (wave & 3) % G::CW, rw = (wave & 3) / G::CW, r16 = lane & 15, q4 = lane >> 4;
  // the tile and its run of K steps.  slices (1, 2, 4, 8): a place of K belongs to 8 / slices XCDs (ids mod 8), which read that part of x and w only; within it contiguous runs of
  // the tiles' order go to one XCD each
  const int tiles = g.MT * g.NT, z = (int)blockIdx.x % g.slices, id = (int)blockIdx.x / g.slices, P = 8 / g.slices, q = tiles / P, r = tiles % P, p = id % P;
  const int lin = p * q + min(p, r) + id / P;
  int mt, nt;
  gr_tile_of(lin, g.MT, g.NT, mt, nt);
  const int K = a.K, KT = (K + 127) >> 7, ks0 = (int)((int64_t)KT * z / g.slices), ks1 = (int)((int64_t)KT * (z + 1) / g.slices);
  const int m0 = mt * BM, n0 = nt * (PAIR ? BN / 2 : BN), rows = min(a.M - m0, BM), cols = min(a.N - n0, PAIR ? BN / 2 : BN);  // (n0: of each tensor)
  const int8_t* const x = a.x + (size_t)m0 * K;
  const int8_t* const w0 = a.w[0] + (size_t)n0 * K;
  const int8_t* const w1 = PAIR ? a.w[1] + (size_t)n0 * K : w0;
  // (pair: virtual block f is of tensor f & 1.  A wave requests the blocks 2 wave and 2 wave + 1 of a 256-column tile, block wave of a 128-column one)
  const int8_t* const wlo = PAIR && EW == 2 && (wave & 1) ? w1 : w0;
  const int8_t* const whi = PAIR && EW == 4 ? w1 : wlo;
  const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(x), 0, rows * K, 0x00020000u);
  const __amdgpu_buffer_rsrc_t rlo = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(wlo), 0, cols * K, 0x00020000u);
  const __amdgpu_buffer_rsrc_t rhi = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(whi), 0, cols * K, 0x00020000u);
  const int sr = lane >> 3, sc = (lane & 7) ^ sr;
  auto upper = [&](int e) { return EX == 4 ? e < 2 : e == 0 || (e == 1 && wave < 4); };
  auto xrow8 = [&](int e) {
    if (H == 1) return (wave * EX + e) * 8;
    if (EX == 4) return (wave < 4 ? wave : wave + 4) * 16 + (e >> 1) * 64 + (e & 1) * 8;
    const int i = wave < 4 ? (upper(e) ? wave * 2 + e : 8 + wave) : (upper(e) ? 4 + wave : (wave - 4) * 2 + e - 1);
    return i / 6 * 96 + i % 6 * 8 + (upper(e) ? 0 : 48);
  };
  uint32_t vx[EX], vw[EW];
#pragma unroll
  for (int e = 0; e < EX; e++) vx[e] = (uint32_t)min(xrow8(e) + sr, rows - 1) * (uint32_t)K + (uint32_t)sc * 16u;
#pragma unroll
  for (int e = 0; e < EW; e++) {
    const int r8 = (wave * EW + e) * 8;
    vw[e] = (uint32_t)min((PAIR ? (r8 >> 5) * 16 + (r8 & 15) : r8) + sr, cols - 1) * (uint32_t)K + (uint32_t)sc * 16u;
  }
  typedef __attribute__((address_space(3))) void* lds_ptr;
  // requests of K step ks (beyond the run: its last step again, never read) into the buffer at byte `o`
  auto stage_x = [&](int o, int ks, int e0, int e1) {
    const uint32_t so = (uint32_t)min(ks, ks1 - 1) * 128u;
#pragma unroll
    for (int e = e0; e < e1; e++) __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_ptr)(smem + o + xrow8(e) * 128), 16, vx[e], so, 0, 0);
  };
  auto stage_half = [&](int o, int ks, bool up) {
#pragma unroll
    for (int e = 0; e < EX; e++)
      if (upper(e) == up) stage_x(o, ks, e, e + 1);
  };
  auto stage_w = [&](int o, int ks) {
    const uint32_t so = (uint32_t)min(ks, ks1 - 1) * 128u;
#pragma unroll
    for (int e = 0; e < EW; e++) {
      unsigned char* const d = smem + o + G::XB * 2048 + (wave * EW + e) * 1024;
      if (e < EW / 2) __builtin_amdgcn_raw_ptr_buffer_load_lds(rlo, (lds_ptr)d, 16, vw[e], so, 0, 0);
      else __builtin_amdgcn_raw_ptr_buffer_load_lds(rhi, (lds_ptr)d, 16, vw[e], so, 0, 0);
    }
  };
  const int row0 = wg * (BM / 2) + rw * (BM / 2 / G::RW);  // the wave's first row in the tile
  const int c0 = r16 * 128 + (q4 ^ (r16 & 7)) * 16, c1 = c0 ^ 64;
  const unsigned char* const xb = smem + row0 * 128;
  const unsigned char* const wb = smem + G::XB * 2048 + cw * 4 * 2048;
  u32x4 xa[KP * NX][2], wa[KP * 4][2];
  auto read_x = [&](int o, int h, int k = 0) {
#pragma unroll
    for (int i = 0; i < NX; i++) {
      xa[k * NX + i][0] = *reinterpret_cast<const u32x4*>(xb + o + c0 + (h * NX + i) * 2048);
      xa[k * NX + i][1] = *reinterpret_cast<const u32x4*>(xb + o + c1 + (h * NX + i) * 2048);
    }
  };
  auto read_w = [&](int o, int k = 0) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      wa[k * 4 + j][0] = *reinterpret_cast<const u32x4*>(wb + o + c0 + j * 2048);
      wa[k * 4 + j][1] = *reinterpret_cast<const u32x4*>(wb + o + c1 + j * 2048);
    }
  };
  i32x4 acc[H * NX][4];
#pragma unroll
  for (int i = 0; i < H * NX; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j] = zero_acc_i8();
  // (a wave's 64 columns, a phase's rows: nothing of them in the matrix, no MFMAs)
  const bool in_c = (PAIR ? cw * 32 : cw * 64) < cols, in = in_c && row0 < rows, in1 = H == 2 && in_c && row0 + NX * 16 < rows;
  auto compute = [&](auto HH, int ks) {  // K steps ks .. ks + KP - 1, those of them within the run
    constexpr int h = decltype(HH)::value;
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(H == 2 ? D : (S - 2) * KP * D) : "memory");
#pragma unroll
    for (int k = 0; k < KP; k++)
      if ((ks + k) * 128 + 128 > K) {  // (the last step of a K off 128, or an H = 2 step behind an odd number of them)
#pragma unroll
        for (int kc = 0; kc < 2; kc++) {
          const bool beyond = (ks + k) * 128 + kc * 64 + q4 * 16 >= K;
#pragma unroll
          for (int i = 0; i < NX; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) xa[k * NX + i][kc][e] = beyond ? 0u : xa[k * NX + i][kc][e];
        }
        asm volatile("s_nop 1");
      }
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if (h ? in1 : in) {
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int k = 0; k < KP; k++) {
        if (k && ks + k >= ks1) break;
#pragma unroll
        for (int kc = 0; kc < 2; kc++)
#pragma unroll
          for (int i = 0; i < NX; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) mfma_i8_ready(acc[h * NX + i][j], wa[k * 4 + j][kc], xa[k * NX + i][kc]);
      }
      __builtin_amdgcn_s_setprio(0);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
  };
  auto no_scalar_loads = [] {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    __builtin_amdgcn_sched_barrier(0);
  };
  using C0 = std::integral_constant<int, 0>;
  using C1 = std::integral_constant<int, 1>;
  if constexpr (H == 2) {
    stage_half(0, 0, true);
    stage_w(0, 0);
    stage_half(0, 0, false);
    stage_half(STG, 1, true);
    stage_w(STG, 1);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(D) : "memory");
    __builtin_amdgcn_s_barrier();
    if (wg == 1) __builtin_amdgcn_s_barrier();  // the second group runs one barrier behind the first
    auto step = [&](auto B, int ks) {
      constexpr int o = decltype(B)::value * STG;
      read_w(o);
      __builtin_amdgcn_sched_barrier(0);
      read_x(o, 0);
      stage_half(STG - o, ks + 1, false);
      compute(C0{}, ks);
      read_x(o, 1);
      stage_half(o, ks + 2, true);
      stage_w(o, ks + 2);
      compute(C1{}, ks);
    };
    no_scalar_loads();
    for (int ks = 0; ks < KT; ks += 2) {
      step(C0{}, ks);
      step(C1{}, ks + 1);
    }
  } else {
#pragma unroll
    for (int s = 0; s < (S - 1) * KP; s++) stage_x(s * STG, ks0 + s, 0, EX), stage_w(s * STG, ks0 + s);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 2) * KP * D) : "memory");
    __builtin_amdgcn_s_barrier();
    if (wg == 1) __builtin_amdgcn_s_barrier();
    no_scalar_loads();
    int o = 0, p = (S - 1) * KP * STG;  // buffers of this phase and of the one before it
    for (int ks = ks0; ks < ks1; ks += KP) {
#pragma unroll
      for (int k = 0; k < KP; k++) read_w(o + k * STG, k), read_x(o + k * STG, 0, k);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < KP; k++) {
        stage_x(p + k * STG, ks + (S - 1) * KP + k, 0, EX);
        stage_w(p + k * STG, ks + (S - 1) * KP + k);
      }
      compute(C0{}, ks);
      p = o;
      o = o == (S - 1) * KP * STG ? 0 : o + KP * STG;
    }
  }
  if (wg == 0) __builtin_amdgcn_s_barrier();
  // (the requests beyond the run still write LDS: they end before the workgroup does)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  VRA_MFMA_DRAIN();
  if constexpr (H == 1) {
    if (g.slices > 1) {
      if (!in) return;
      int v[NX * 16];
#pragma unroll
      for (int i = 0; i < NX * 16; i++) v[i] = acc[i >> 4][i >> 2 & 3][i & 3];
      if (!i8_meet<NX * 16, 512>(v, g.ws, lin, tiles, z, g.slices)) return;
#pragma unroll
      for (int i = 0; i < NX * 16; i++) acc[i >> 4][i >> 2 & 3][i & 3] = v[i];
    }
  }
  i8_store_rows<PAIR, H * NX>(a, m0 + row0 + r16, n0 + (PAIR ? cw * 32 : cw * 64), q4, acc);
#endif
}

// ---------------------------------------------------------------- many rows, any K, any alignment
// Rows that begin anywhere cannot go to LDS by themselves: they come through registers, 16 bytes at any address a load, D K steps of 128 ahead of the one in
// LDS (one step of 64 ahead: 777 x 1003, K = 2741 31 us, nearly all of it waiting; so 17).  Bound: those loads, which take two turns of a CU's 64 bytes a clock where they are
// off 16 bytes, beside LDS (8192 x 6144, K = 4097: 128 x 128 362 us, 256 x 256 248: half the loads a product, one step ahead for want of registers).  A wave has 64 virtual columns and R blocks of 16 rows; LDS as above, two
// buffers.  PAIR: virtual columns, gate and up interleaved in blocks of 16.
template <bool PAIR, int BM, int BN, int NT, int D>
__global__ __launch_bounds__(NT, 2) void gemm_i8_any_kernel(const GemmI8Args a, const GemmI8Tiles g) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int CW = BN / 64, RW = NT / 64 / CW, R = BM / RW / 16, RL = NT / 8, XE = BM / RL, WE = BN / RL, STG = (BM + BN) * 128;  // RL rows a round of loads
  static_assert(RL % 32 == 0 && R * RW * 16 == BM && XE * RL == BM && WE * RL == BN, "whole rounds");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), cw = wave % CW, rw = wave / CW;
  const int tiles = g.MT * g.NT, z = (int)blockIdx.x % g.slices, lin = (int)blockIdx.x / g.slices;
  int mt, nt;
  gr_tile_of(lin, g.MT, g.NT, mt, nt);
  const int K = a.K, KT = (K + 127) >> 7, ks0 = (int)((int64_t)KT * z / g.slices), ks1 = (int)((int64_t)KT * (z + 1) / g.slices);
  const int m0 = mt * BM, n0 = nt * (PAIR ? BN / 2 : BN);
  // piece e of a thread: 16-byte chunk tid & 7 of row (tid >> 3) + RL e
  const int ch = tid & 7, r8 = tid >> 3;
  const int8_t* const x = a.x + (size_t)m0 * K;
  const int8_t* const w = (PAIR && (r8 & 16) ? a.w[1] : a.w[0]) + (size_t)n0 * K;
  uint32_t xo[XE], wo[WE];
#pragma unroll
  for (int e = 0; e < XE; e++) xo[e] = (uint32_t)min(r8 + RL * e, a.M - 1 - m0) * (uint32_t)K;
#pragma unroll
  for (int e = 0; e < WE; e++) {
    const int v = r8 + RL * e;
    wo[e] = (uint32_t)min(PAIR ? (v >> 5) * 16 + (v & 15) : v, a.N - 1 - n0) * (uint32_t)K;
  }
  const int slot = r8 * 128 + ((ch ^ (r8 & 7)) * 16);
  u32x4 xr[D][XE], wr[D][WE];
  auto load = [&](int b, int ks) __attribute__((always_inline)) {
    if (ks >= ks1) return;
    const uint32_t k = (uint32_t)ks * 128u + ch * 16u;
    if (ks * 128 + 128 <= K) {
#pragma unroll
      for (int e = 0; e < XE; e++) xr[b][e] = *reinterpret_cast<const u32x4_a1*>(x + (xo[e] + k));
#pragma unroll
      for (int e = 0; e < WE; e++) wr[b][e] = *reinterpret_cast<const u32x4_a1*>(w + (wo[e] + k));
    } else {
#pragma unroll
      for (int e = 0; e < XE; e++) xr[b][e] = i8_load16(x + xo[e], (int)k, K);
#pragma unroll
      for (int e = 0; e < WE; e++) wr[b][e] = i8_load16(w + wo[e], (int)k, K);
    }
  };
  auto put = [&](int b, int o) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < XE; e++) *reinterpret_cast<u32x4*>(smem + o + slot + e * (RL * 128)) = xr[b][e];
#pragma unroll
    for (int e = 0; e < WE; e++) *reinterpret_cast<u32x4*>(smem + o + BM * 128 + slot + e * (RL * 128)) = wr[b][e];
  };
  const int c0 = r16 * 128 + (q4 ^ (r16 & 7)) * 16;
  i32x4 acc[R][4];
#pragma unroll
  for (int i = 0; i < R; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j] = zero_acc_i8();
  // K step ks is in buffer b; the registers hold step ks + 1 (D = 2: set 1 - b) and, on its way, step ks + 2
  auto step = [&](auto B, int ks) __attribute__((always_inline)) {
    constexpr int b = decltype(B)::value, o = b * STG, set = D == 2 ? 1 - b : 0;
    if (ks < ks1) {
#pragma unroll
      for (int kc = 0; kc < 2; kc++) {
        u32x4 wa[4];
#pragma unroll
        for (int j = 0; j < 4; j++) wa[j] = *reinterpret_cast<const u32x4*>(smem + o + BM * 128 + (c0 ^ (kc * 64)) + (cw * 4 + j) * 2048);
#pragma unroll
        for (int i0 = 0; i0 < R; i0 += 4) {
          u32x4 xa[R < 4 ? R : 4];
#pragma unroll
          for (int i = 0; i < (R < 4 ? R : 4); i++) xa[i] = *reinterpret_cast<const u32x4*>(smem + o + (c0 ^ (kc * 64)) + (rw * R + i0 + i) * 2048);
#pragma unroll
          for (int i = 0; i < (R < 4 ? R : 4); i++)
#pragma unroll
            for (int j = 0; j < 4; j++) mfma_i8(acc[i0 + i][j], wa[j], xa[i]);
        }
      }
    }
    if (ks + 1 < ks1) put(set, STG - o);
    load(set, ks + 1 + D);
    __syncthreads();
  };
  load(0, ks0);
  if (D == 2) load(D - 1, ks0 + 1);
  put(0, 0);
  load(0, ks0 + D);
  __syncthreads();
  for (int ks = ks0; ks < ks1; ks += 2) {
    step(std::integral_constant<int, 0>{}, ks);
    step(std::integral_constant<int, 1>{}, ks + 1);
  }
  VRA_MFMA_DRAIN();
  if constexpr (R <= 4) {
    if (g.slices > 1) {
      int v[R * 16];
#pragma unroll
      for (int i = 0; i < R * 16; i++) v[i] = acc[i >> 4][i >> 2 & 3][i & 3];
      if (!i8_meet<R * 16, NT>(v, g.ws, lin, tiles, z, g.slices)) return;
#pragma unroll
      for (int i = 0; i < R * 16; i++) acc[i >> 4][i >> 2 & 3][i & 3] = v[i];
    }
  }
  i8_store_rows<PAIR, R>(a, m0 + rw * R * 16 + r16, n0 + (PAIR ? cw * 32 : cw * 64), q4, acc);
#endif
}
