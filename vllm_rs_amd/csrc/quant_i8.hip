// quant_i8.hip — rows of 16-bit activations to 8-bit integers with a scale a row, alone and behind the RMS norm (with or without the residual's addition):
// what stands ahead of the products of gemm_i8.hip.
//
//   p = x (alone), x w or round(x + residual) w (norm),  a = max |p|,  q = rint(127 p / a),  scale = a / 127 [ / sqrt(mean(h^2) + eps) ]
//
// The norm's factor is the same for a whole row: it is in the scale, and not in q.  Products of two 16-bit floats are exact in f32, and a quotient within the
// f32 division's error of a half is decided by its exact remainder: q is the definition's, bit for bit, whatever the order of the sums.
// Bound: memory, and close behind it the vector instructions, 12 an element without a norm and 18 with one (8192 x 4096 bf16: sum and norm 44.6 us = 5.3 TB/s, norm 23.5 = 4.3;
// 3063 x 18944 f16 38.0 = 4.6).  A row is read once and kept in registers as it came (the sum as it is stored) between the reduction and the quotients.
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
  double sum = 0.0;  // (squares of bf16 leave f32's range at 2^64)
  uint32_t top = 0u;  // |p| as bits: ordered as the values are, infinities and NaN above all others
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 top2 = {0, 0};  // the same of the elements as they are stored (no norm), two at a time
  auto first = [&](auto tail, int c, u32x4& kept, u32x4& wv) __attribute__((always_inline)) {
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
    if (NORM) {
      float w[8];
      unpack8<DT>(v, f);
      unpack8<DT>(wv, w);
#pragma unroll
      for (int e = 0; e < 8; e++) sum = fma((double)f[e], (double)f[e], sum), f[e] *= w[e];
#pragma unroll
      for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) top2 = __builtin_elementwise_max(top2, __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu));
    }
  };
  if constexpr (V > 0) {
#pragma unroll
    for (int i = 0; i < V; i++)
      if ((tid + i * T) * 8 < whole) first(std::false_type{}, (tid + i * T) * 8, keep[i], wk[i]);
  } else {
    for (int c = tid * 8; c < whole; c += T * 8) first(std::false_type{}, c, keep[0], wk[0]);
  }
  if (has_tail) first(std::true_type{}, whole, keep_t, wk_t);
  if (!NORM) top = __float_as_uint(DT::to_f32(max(top2[0], top2[1])));
  row_reduce<T, NORM>(sum, top);
  // a row that is not finite in 32 bits: codes 0 and scale NaN, which makes NaN of all that is computed from it
  const bool finite = top < 0x7f800000u && sum < (double)INFINITY;  // (an infinity or NaN times a weight of zero is in the sum)
  const float amax = __uint_as_float(top);
  if (tid == 0) {
    const double s = (double)amax / 127.0;
    // (nothing but zeros: 0, also where eps = 0 makes the norm 0 / 0)
    a.scales[row] = !finite ? __uint_as_float(0x7fc00000u) : top == 0u ? 0.f : (float)(NORM ? s / sqrt(sum / cols + (double)a.eps) : s);
  }
  // the lower end of the range is moved up by a power of two: 127 / a does not overflow, no remainder is lost below the normal range
  const bool tiny = __builtin_amdgcn_readfirstlane(amax < 0x1p-60f);
  const float as = tiny ? amax * 0x1p64f : amax, inv = top ? 127.0f / as : 0.f;
  auto second = [&](auto tail, int c, u32x4 v, u32x4 wv) __attribute__((always_inline)) {
    constexpr bool TL = decltype(tail)::value;
    constexpr float WHOLE = 12582912.0f;  // 1.5 2^23: a sum with it is a whole number, rounded to even, whose lowest byte is the 8-bit integer
    float f[8], r[8], far = 0.f;
    unpack8<DT>(v, f);
    if (NORM) {
      float w[8];
      unpack8<DT>(wv, w);
#pragma unroll
      for (int e = 0; e < 8; e++) f[e] *= w[e];
    }
    if (tiny)
#pragma unroll
      for (int e = 0; e < 8; e++) f[e] *= 0x1p64f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float t = f[e] * inv;  // |t| <= 127 (1 + 2^-22): off by less than 2^-15
      r[e] = t + WHOLE;
      far = fmaxf(far, fabsf(t - (r[e] - WHOLE)));
    }
    if (far > 0.5f - 0x1p-14f) {
      // 127 p = hi + lo exactly; d = hi - r a is exact: |d| is about a / 2, a multiple of both units and within 24 bits of the larger one.  2 |d + lo| against a
      // says on which side of the half the quotient lies.  (127 p of the range's upper end: both moved down)
      const float down = as > 0x1p60f ? 0x1p-64f : 1.0f, ad = as * down;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float p = f[e] * down, q = r[e] - WHOLE, hi = 127.0f * p, lo = fmaf(127.0f, p, -hi), d = fmaf(-q, ad, hi);
        const float up = d > 0.f ? 1.f : -1.f, over = fmaf(2.0f, fabsf(d), -ad) + 2.0f * up * lo;
        if (over > 0.f || (over == 0.f && ((int)q & 1))) r[e] += up;
      }
    }
    u32x2 o;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(r[4 * h + 1]), __float_as_uint(r[4 * h]), 0x0c0c0400u);
      const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(r[4 * h + 3]), __float_as_uint(r[4 * h + 2]), 0x0c0c0400u);
      o[h] = finite ? lo | hi << 16 : 0u;
    }
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
  // Threads of a row and the eights each keeps.  Few rows (two workgroups a CU at most): as many threads as there are eights, the row is one round trip (16 x 14336: 256 threads 9.2 us,
  // 512 5.7, 1024 4.5).  Many: two eights and more a thread, so that the barrier and the reduction stand behind more requests (8192 x 4096: 512 threads 27.9 us, 256 23.5; 8192 x 1024: 256 threads
  // 11.8, one wave 9.6), beyond 8192 as many as keep their registers (4096 x 14336, no norm: 1024 threads 43.5 us, 512 39.6; norm and sum: 75.3 / 78.1)
  const int whole = a.cols & ~7;
  const bool many = a.rows > 512;
  auto go = [&](auto t, auto v) {
    constexpr int T = decltype(t)::value, V = decltype(v)::value;
    rows_i8_kernel<DT, MODE, T, V><<<T == 64 ? (a.rows + 3) / 4 : a.rows, T == 64 ? 256 : T, 0, st>>>(a);
  };
#define QI_KERNEL(T, V) go(std::integral_constant<int, T>{}, std::integral_constant<int, V>{})
  if (whole <= (many ? 1024 : 512)) QI_KERNEL(64, 2);
  else if (!many && whole <= 2048) QI_KERNEL(256, 1);
  else if (!many && whole <= 4096) QI_KERNEL(512, 1);
  else if (!many && whole <= 8192) QI_KERNEL(1024, 1);
  else if (whole <= 4096) QI_KERNEL(256, 2);
  else if (whole <= 8192) QI_KERNEL(512, 2);
  else if (many && MODE == QI_PLAIN && whole <= 16384) QI_KERNEL(512, MODE == QI_PLAIN ? 4 : 2);
  else if (whole <= 16384) QI_KERNEL(1024, 2);
  else if (whole <= 24576) QI_KERNEL(1024, 3);
  else if (whole <= 32768) QI_KERNEL(1024, 4);
  else QI_KERNEL(1024, 0);
#undef QI_KERNEL
}

template <int MODE>
void rows_i8(const char* who, const RowsI8Args& a, int dtype, int64_t stream) {
  VRA_CHECK_ARG(a.rows >= 0 && a.cols > 0 && a.cols <= 131072, "%s: rows >= 0 and 1..131072 columns (rows=%d columns=%d)", who, a.rows, a.cols);
  VRA_CHECK_ARG(dtype == VRA_BF16 || dtype == VRA_F16, "%s: dtype must be bf16/f16", who);
  VRA_CHECK_ARG(a.eps >= 0.f, "%s: eps must be 0 or above (eps=%g)", who, (double)a.eps);  // (NaN is neither; with less a finite row could have the scale of one that is not)
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
