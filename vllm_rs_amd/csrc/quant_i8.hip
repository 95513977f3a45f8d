// quant_i8.hip — rows of 16-bit activations to 8-bit integers with a scale a row, alone and behind the RMS norm (with or without the residual's addition):
// what stands ahead of the products of gemm_i8.hip.
//
//   p = x (alone), x w or round(x + residual) w (norm),  a = max |p|,  q = rint(127 p / a),  scale = a / 127 [ / sqrt(mean(h^2) + eps) ]
//
// The norm's factor is the same for a whole row: it is in the scale, and not in q.  Products of two 16-bit floats are exact in f32, and a quotient within the
// f32 division's error of a half is decided by its exact remainder: q is the definition's, bit for bit, whatever the order of the sums.
// Bound: memory.  A row is read once and kept in registers as it came (the sum as it is stored) between the reduction and the quotients.
#include <type_traits>

#include "common.cuh"

namespace {

// rows begin anywhere: 16 bytes at a multiple of 2, 8 at any
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef u32x2 u32x2_a1 __attribute__((aligned(1)));

struct RowsI8Args {
  const uint16_t* x;
  const uint16_t* residual;
  const uint16_t* weight;
  uint16_t* h_out;  // (may be x or residual: a thread reads its elements before it writes them)
  int8_t* q;
  float* scales;
  int rows, cols;
  float eps;
};

enum { QI_PLAIN, QI_NORM, QI_ADD_NORM };

// eight elements; TAIL: the first n of them, zeros behind
template <bool TAIL>
__device__ __forceinline__ u32x4 load8(const uint16_t* p, int n) {
  if (!TAIL) return *reinterpret_cast<const u32x4_a2*>(p);
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < 7; e++)
    if (e < n) v[e >> 1] |= (uint32_t)p[e] << (e & 1 ? 16 : 0);
  return v;
}

// sum and maximum over the T threads of a row, in all of them
template <int T, bool SUM>
__device__ __forceinline__ void row_reduce(double& sum, uint32_t& top) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    if (SUM) sum += __shfl_xor(sum, o, 64);
    top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  }
  if constexpr (T > 64) {
    __shared__ double sums[T / 64];
    __shared__ uint32_t tops[T / 64];
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum, tops[threadIdx.x >> 6] = top;
    __syncthreads();
    sum = sums[0], top = tops[0];
#pragma unroll
    for (int w = 1; w < T / 64; w++) sum += sums[w], top = max(top, tops[w]);
  }
}

// T threads a row.  V > 0: rows of up to 8 T V elements, kept in registers; V = 0: longer ones, read twice
template <class DT, int MODE, int T, int V>
__global__ __launch_bounds__(T < 256 ? 256 : T) void rows_i8_kernel(const RowsI8Args a) {
  constexpr bool NORM = MODE != QI_PLAIN, ADD = MODE == QI_ADD_NORM;
  const int tid = T < 256 ? threadIdx.x % T : threadIdx.x, row = T < 256 ? blockIdx.x * (256 / T) + threadIdx.x / T : blockIdx.x;
  if (T < 256 && row >= a.rows) return;  // (whole waves: a row of 64 threads has no barrier)
  const int cols = a.cols, whole = cols & ~7, n = cols & 7;
  const bool has_tail = n && tid == T - 1;  // the elements behind the last eight
  const size_t at = (size_t)row * cols;
  u32x4 keep[V ? V : 1], wk[V ? V : 1], keep_t, wk_t;
  double sum = 0.0;  // (squares of bf16 leave f32's range at 2^64; an f64 multiply-add runs at the f32 rate)
  uint32_t top = 0u;  // |p| as bits: ordered as the values are, infinities and NaN above all others
  auto first = [&](auto tail, int c, u32x4& kept, u32x4& wv) {
    constexpr bool TL = decltype(tail)::value;
    u32x4 v = load8<TL>(a.x + at + c, n);
    float f[8];
    if (NORM) wv = load8<TL>(a.weight + c, n);
    if (ADD) {
      float r[8];
      unpack8<DT>(v, f);
      unpack8<DT>(load8<TL>(a.residual + at + c, n), r);
#pragma unroll
      for (int e = 0; e < 8; e++) f[e] += r[e];
      v = pack8<DT>(f);
      if (!TL) *reinterpret_cast<u32x4_a2*>(a.h_out + at + c) = v;
      else
#pragma unroll
        for (int e = 0; e < 7; e++)
          if (e < n) a.h_out[at + c + e] = (uint16_t)(v[e >> 1] >> (e & 1 ? 16 : 0));
    }
    kept = v;
    unpack8<DT>(v, f);
    if (NORM) {
      float w[8];
      unpack8<DT>(wv, w);
#pragma unroll
      for (int e = 0; e < 8; e++) sum = fma((double)f[e], (double)f[e], sum), f[e] *= w[e];
    }
#pragma unroll
    for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
  };
  if constexpr (V > 0) {
#pragma unroll
    for (int i = 0; i < V; i++)
      if ((tid + i * T) * 8 < whole) first(std::false_type{}, (tid + i * T) * 8, keep[i], wk[i]);
  } else {
    for (int c = tid * 8; c < whole; c += T * 8) first(std::false_type{}, c, keep[0], wk[0]);
  }
  if (has_tail) first(std::true_type{}, whole, keep_t, wk_t);
  row_reduce<T, NORM>(sum, top);
  // a row that is not finite in 32 bits: codes 0 and scale NaN, which makes NaN of all that is computed from it
  const bool finite = top < 0x7f800000u && sum < (double)INFINITY;  // (an infinity or NaN times a weight of zero is in the sum)
  const float amax = __uint_as_float(top);
  if (tid == 0) {
    const double s = (double)amax / 127.0;
    a.scales[row] = finite ? (float)(NORM ? s / sqrt(sum / cols + (double)a.eps) : s) : __uint_as_float(0x7fc00000u);
  }
  // the range's ends are moved to its middle, by a power of two: neither 127 / a nor 127 p overflows, no remainder is lost below the normal range
  const float shift = amax < 0x1p-60f ? 0x1p64f : amax > 0x1p60f ? 0x1p-64f : 1.0f;
  const float as = amax * shift, inv = finite && top ? 127.0f / as : 0.f;
  auto second = [&](auto tail, int c, const u32x4& v, const u32x4& wv) {
    constexpr bool TL = decltype(tail)::value;
    float f[8], r[8];
    unpack8<DT>(v, f);
    if (NORM) {
      float w[8];
      unpack8<DT>(wv, w);
#pragma unroll
      for (int e = 0; e < 8; e++) f[e] *= w[e];
    }
    bool close = false;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      f[e] = finite ? f[e] * shift : 0.f;
      const float t = f[e] * inv;  // |t| <= 127 (1 + 2^-22): off by less than 2^-15
      r[e] = rintf(t);
      close |= fabsf(t - r[e]) > 0.5f - 0x1p-14f;
    }
    if (close) {
      // 127 p = hi + lo exactly; d = hi - r a is exact: |d| is about a / 2, a multiple of both units and within 24 bits of the larger one.  2 |d + lo| against a
      // says on which side of the half the quotient lies
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float hi = 127.0f * f[e], lo = fmaf(127.0f, f[e], -hi), d = fmaf(-r[e], as, hi);
        const float up = d > 0.f ? 1.f : -1.f, over = fmaf(2.0f, fabsf(d), -as) + 2.0f * up * lo;
        if (over > 0.f || (over == 0.f && ((int)r[e] & 1))) r[e] += up;
      }
    }
    u32x2 o = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; e++) o[e >> 2] |= ((uint32_t)(int)r[e] & 0xffu) << (8 * (e & 3));
    int8_t* const to = a.q + at + c;
    if (!TL) *reinterpret_cast<u32x2_a1*>(to) = o;
    else
#pragma unroll
      for (int e = 0; e < 7; e++)
        if (e < n) to[e] = (int8_t)(o[e >> 2] >> (8 * (e & 3)));
  };
  if constexpr (V > 0) {
#pragma unroll
    for (int i = 0; i < V; i++)
      if ((tid + i * T) * 8 < whole) second(std::false_type{}, (tid + i * T) * 8, keep[i], wk[i]);
  } else {
    for (int c = tid * 8; c < whole; c += T * 8) {
      const u32x4 v = load8<false>((ADD ? a.h_out : a.x) + at + c, 8);  // (the sum: this thread's own stores)
      second(std::false_type{}, c, v, NORM ? load8<false>(a.weight + c, 8) : v);
    }
  }
  if (has_tail) second(std::true_type{}, whole, keep_t, wk_t);
}

template <class DT, int MODE>
void launch(RowsI8Args a, hipStream_t st) {
  const int most = 1 << 20;  // rows of a launch: within 2^32 threads
  for (; a.rows > most; a.rows -= most) {
    RowsI8Args part = a;
    part.rows = most;
    launch<DT, MODE>(part, st);
    const size_t by = (size_t)most * a.cols;
    a.x += by, a.q += by, a.scales += most;
    if (MODE == QI_ADD_NORM) a.residual += by, a.h_out += by;
  }
  if (a.cols <= 2048) rows_i8_kernel<DT, MODE, 64, 4><<<(a.rows + 3) / 4, 256, 0, st>>>(a);
  else if (a.cols <= 8192) rows_i8_kernel<DT, MODE, 256, 4><<<a.rows, 256, 0, st>>>(a);
  else if (a.cols <= 32768) rows_i8_kernel<DT, MODE, 1024, 4><<<a.rows, 1024, 0, st>>>(a);
  else rows_i8_kernel<DT, MODE, 1024, 0><<<a.rows, 1024, 0, st>>>(a);
}

template <int MODE>
void rows_i8(const char* who, const RowsI8Args& a, int dtype, int64_t stream) {
  VRA_CHECK_ARG(a.rows >= 0 && a.cols > 0 && a.cols <= 131072, "%s: rows >= 0 and 1..131072 columns (rows=%d columns=%d)", who, a.rows, a.cols);
  VRA_CHECK_ARG(dtype == VRA_BF16 || dtype == VRA_F16, "%s: dtype must be bf16/f16", who);
  if (a.rows == 0) return;
  VRA_CHECK_ARG(a.x && a.q && a.scales && (MODE == QI_PLAIN || a.weight) && (MODE != QI_ADD_NORM || (a.residual && a.h_out)), "%s: null pointer", who);
  VRA_CHECK_ARG((((uintptr_t)a.x | (uintptr_t)a.residual | (uintptr_t)a.weight | (uintptr_t)a.h_out) & 1) == 0 && ((uintptr_t)a.scales & 3) == 0,
                "%s: a pointer that is not a multiple of its elements' size", who);
  dtype == VRA_BF16 ? launch<BF16, MODE>(a, as_stream(stream)) : launch<F16, MODE>(a, as_stream(stream));
}

}  // namespace

extern "C" void vra_quant_rows_i8(const void* x, int8_t* q, float* scales, int32_t rows, int32_t cols, int32_t dtype, int64_t stream) {
  rows_i8<QI_PLAIN>("vra_quant_rows_i8", RowsI8Args{static_cast<const uint16_t*>(x), nullptr, nullptr, nullptr, q, scales, rows, cols, 0.f}, dtype, stream);
}
extern "C" void vra_rms_norm_i8(const void* x, const void* weight, int8_t* q, float* scales, int32_t tokens, int32_t hidden, float eps, int32_t dtype,
                                int64_t stream) {
  rows_i8<QI_NORM>("vra_rms_norm_i8", RowsI8Args{static_cast<const uint16_t*>(x), nullptr, static_cast<const uint16_t*>(weight), nullptr, q, scales, tokens, hidden, eps},
                   dtype, stream);
}
extern "C" void vra_add_rms_norm_i8(const void* x, const void* residual, const void* weight, void* h_out, int8_t* q, float* scales, int32_t tokens,
                                    int32_t hidden, float eps, int32_t dtype, int64_t stream) {
  rows_i8<QI_ADD_NORM>("vra_add_rms_norm_i8", RowsI8Args{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(residual), static_cast<const uint16_t*>(weight),
                                                         static_cast<uint16_t*>(h_out), q, scales, tokens, hidden, eps}, dtype, stream);
}
