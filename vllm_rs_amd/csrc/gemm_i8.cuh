// gemm_i8.cuh — products of 8-bit integers with a scale a row (token) and a scale a column (channel):
//   out[m, n] = round( xs[m] ws[n] sum_k x[m, k] w[n, k]  + bias[n] + residual[m, n] ),   pair: round( silu(g) u ), g and u such products.
// Sums are 32-bit integers (K <= 131071: |sum| <= 128 128 K < 2^31): exact, the same in any order, so no split of K changes a bit.  The scales, the bias and
// the residual are applied in f32, with one rounding at the end.  Weights are row-major [n, K] as checkpoints hold them.
// Weights = A, rows of x = B of v_mfma_i32_16x16x64_i8 (16 bytes of a row a lane; a lane's result: 4 consecutive columns of one row), at the bf16 instruction's
// clocks for twice the K: every byte of an operand costs what it costs the 16-bit kernels (gemm_rows.cuh).
#pragma once
#include "common.cuh"

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

// four consecutive columns n .. n + 3 (those within N) of row m
template <class T>
__device__ __forceinline__ void load4(float (&f)[4], const void* p, size_t at, int n, int N, bool whole) {
  const uint16_t* const h = static_cast<const uint16_t*>(p) + at;
  if (whole) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(h);
#pragma unroll
    for (int e = 0; e < 4; e++) f[e] = T::to_f32((uint16_t)(v[e >> 1] >> (e & 1 ? 16 : 0)));
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) f[e] = n + e < N ? T::to_f32(h[e]) : 0.f;
  }
}
struct PlainF32 {};  // (VRA_F32 as a type of the epilogue)
template <>
__device__ __forceinline__ void load4<PlainF32>(float (&f)[4], const void* p, size_t at, int n, int N, bool whole) {
  const float* const h = static_cast<const float*>(p) + at;
  if (whole) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(h);
#pragma unroll
    for (int e = 0; e < 4; e++) f[e] = v[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) f[e] = n + e < N ? h[e] : 0.f;
  }
}
template <class T>
__device__ __forceinline__ void store4(const float (&f)[4], void* p, size_t at, int n, int N, bool whole) {
  uint16_t* const h = static_cast<uint16_t*>(p) + at;
  if (whole) *reinterpret_cast<u32x2*>(h) = u32x2{T::pack2(f[0], f[1]), T::pack2(f[2], f[3])};
  else
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (n + e < N) h[e] = T::from_f32(f[e]);
}
template <>
__device__ __forceinline__ void store4<PlainF32>(const float (&f)[4], void* p, size_t at, int n, int N, bool whole) {
  float* const h = static_cast<float*>(p) + at;
  if (whole) *reinterpret_cast<f32x4*>(h) = f32x4{f[0], f[1], f[2], f[3]};
  else
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (n + e < N) h[e] = f[e];
}

// whether four columns at a multiple of 4 may be read and written at once, in all rows
__host__ __device__ __forceinline__ bool i8_whole_fours(const GemmI8Args& a) {
  const uintptr_t all = (uintptr_t)a.out | (uintptr_t)a.residual | (uintptr_t)a.bias;
  return a.N % 4 == 0 && all % (a.dtype == VRA_F32 ? 16 : 8) == 0;
}

// sums g (and u) of columns n .. n + 3 of row m -> what is stored there
template <bool PAIR>
__device__ __forceinline__ void i8_values(const GemmI8Args& a, float xs, int n, i32x4 g, i32x4 u, float (&y)[4]) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const int c = min(n + e, a.N - 1);
    float v = (float)g[e] * xs * a.ws[0][c];
    if (PAIR) {
      // silu(v) u = v u / (1 + exp(-v)); below zero exp(v / 2) goes to both factors: exp(-v) would end at v = -88, where bf16 still holds the result
      const float h = expf(-0.5f * fabsf(v)), s = v < 0.f ? h : 1.0f;
      v = v * s / (1.0f + h * h) * ((float)u[e] * xs * a.ws[1][c] * s);
    }
    y[e] = v;
  }
}
template <class T, bool PAIR>
__device__ __forceinline__ void i8_store(const GemmI8Args& a, int m, int n, bool whole, i32x4 g, i32x4 u) {
  if (m >= a.M || n >= a.N) return;
  whole = whole && n + 4 <= a.N;
  const size_t at = (size_t)m * a.N + n;
  float y[4], f[4];
  i8_values<PAIR>(a, a.xs[m], n, g, u, y);
  if (!PAIR && a.bias) {
    load4<T>(f, a.bias, n, n, a.N, whole);
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] += f[e];
  }
  if (!PAIR && a.residual) {
    load4<T>(f, a.residual, at, n, a.N, whole);
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] += f[e];
  }
  store4<T>(y, a.out, at, n, a.N, whole);
}

// ---------------------------------------------------------------- any K, any alignment
// 64 rows x 64 columns (pair: 32 gate and 32 up columns, interleaved in blocks of 16) a workgroup of four waves, 32 x 32 each; steps of 64 k through two
// buffers of LDS, filled through registers by loads of 16 bytes at any address (bytes one by one where K ends inside them).
template <class T, bool PAIR>
__global__ __launch_bounds__(256) void gemm_i8_any_kernel(const GemmI8Args a, int cols) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int P = 80;  // bytes from row to row in LDS
  __shared__ __attribute__((aligned(16))) unsigned char buf[2][2][64 * P];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, q4 = lane >> 4;
  const int K = a.K, mt = (int)blockIdx.x / cols, m0 = mt * 64, n0 = ((int)blockIdx.x - mt * cols) * (PAIR ? 32 : 64);
  const int row = tid >> 2, chunk = (tid & 3) * 16;
  // (virtual column `row` of a pair: block row / 16, of tensor block & 1)
  const int col = min(n0 + (PAIR ? (row >> 5) * 16 + (row & 15) : row), a.N - 1);
  const int8_t* const xp = a.x + (size_t)min(m0 + row, a.M - 1) * K;
  const int8_t* const wp = (PAIR && (row & 16) ? a.w[1] : a.w[0]) + (size_t)col * K;
  auto load16 = [&](const int8_t* p, int k) {
    u32x4 v = {0u, 0u, 0u, 0u};
    if (k + 16 <= K) return *reinterpret_cast<const u32x4_a1*>(p + k);
#pragma unroll
    for (int e = 0; e < 15; e++)
      if (k + e < K) v[e >> 2] |= (uint32_t)(uint8_t)p[k + e] << (8 * (e & 3));
    return (u32x4_a1)v;
  };
  auto put = [&](int b, u32x4 x, u32x4 w) {
    *reinterpret_cast<u32x4*>(&buf[b][0][row * P + chunk]) = x;
    *reinterpret_cast<u32x4*>(&buf[b][1][row * P + chunk]) = w;
  };
  i32x4 acc[2][2];
#pragma unroll
  for (int i = 0; i < 4; i++) acc[i >> 1][i & 1] = zero_acc_i8();
  const int xr = (wave >> 1) * 32, wr = (wave & 1) * 32;
  put(0, load16(xp, chunk), load16(wp, chunk));
  __syncthreads();
  for (int k = 0, b = 0; k < K; k += 64, b ^= 1) {
    u32x4 nx = {}, nw = {};
    const bool more = k + 64 < K;
    if (more) nx = load16(xp, k + 64 + chunk), nw = load16(wp, k + 64 + chunk);
    u32x4 xf[2], wf[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      xf[i] = *reinterpret_cast<const u32x4*>(&buf[b][0][(xr + i * 16 + r16) * P + q4 * 16]);
      wf[i] = *reinterpret_cast<const u32x4*>(&buf[b][1][(wr + i * 16 + r16) * P + q4 * 16]);
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < 2; j++) mfma_i8(acc[i][j], wf[j], xf[i]);
    if (more) put(b ^ 1, nx, nw);
    __syncthreads();
  }
  VRA_MFMA_DRAIN();
  const bool whole = i8_whole_fours(a);
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int m = m0 + xr + i * 16 + r16;
    if (PAIR) i8_store<T, true>(a, m, n0 + (wr >> 1) + q4 * 4, whole, acc[i][0], acc[i][1]);
    else
#pragma unroll
      for (int j = 0; j < 2; j++) i8_store<T, false>(a, m, n0 + wr + j * 16 + q4 * 4, whole, acc[i][j], acc[i][j]);
  }
#endif
}
