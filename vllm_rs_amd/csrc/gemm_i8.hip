// gemm_i8.hip — the C entry points of the 8-bit integer products (gemm_i8.cuh).
#include "gemm_i8.cuh"

#include <algorithm>

namespace {

template <class F>
void with_type(int dtype, const F& f) {
  if (dtype == VRA_BF16) f(BF16{});
  else if (dtype == VRA_F16) f(F16{});
  else f(PlainF32{});
}

template <bool PAIR>
void launch(GemmI8Args a, void* workspace, hipStream_t st) {
  // a launch stays within 2^32 threads: 2^22 tiles of 64 x 64
  const int64_t most = std::max<int64_t>(((int64_t)1 << 22) / (a.N / 64 + 1) * 64 & ~(int64_t)255, 256);
  for (; a.M > most; a.M -= (int)most) {
    GemmI8Args part = a;
    part.M = (int)most;
    launch<PAIR>(part, workspace, st);
    const size_t by = (size_t)most * a.N * (a.dtype == VRA_F32 ? 4 : 2);
    a.x += (size_t)most * a.K, a.xs += most, a.out = static_cast<char*>(a.out) + by;
    if (a.residual) a.residual = static_cast<const char*>(a.residual) + by;
  }
  with_type(a.dtype, [&](auto t) {
    const int cols = (a.N + (PAIR ? 31 : 63)) / (PAIR ? 32 : 64);
    gemm_i8_any_kernel<decltype(t), PAIR><<<(unsigned)((a.M + 63) / 64 * cols), 256, 0, st>>>(a, cols);
  });
}

bool product_ok(const char* who, const GemmI8Args& a, const void* workspace, int tensors) {
  if (a.M < 0 || a.K <= 0 || a.K > 131071 || a.N <= 0) {
    vra_set_error("%s: m >= 0, 1 <= k <= 131071 (sums of 32 bits), n >= 1 (m=%d k=%d n=%d)", who, a.M, a.K, a.N);
    return false;
  }
  const bool f32 = a.dtype == VRA_F32;
  if (a.dtype != VRA_BF16 && a.dtype != VRA_F16 && !(f32 && tensors == 1)) {
    vra_set_error("%s: dtype must be bf16/f16%s", who, tensors == 1 ? "/f32" : "");
    return false;
  }
  if (a.M == 0) return true;
  bool null = !a.x || !a.xs || !a.out;
  uintptr_t words = (uintptr_t)a.xs;
  for (int t = 0; t < tensors; t++) null |= !a.w[t] || !a.ws[t], words |= (uintptr_t)a.ws[t];
  if (null) {
    vra_set_error("%s: null pointer", who);
    return false;
  }
  if (words % 4 || ((uintptr_t)a.bias | (uintptr_t)a.residual | (uintptr_t)a.out) % (f32 ? 4 : 2)) {
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

extern "C" size_t vra_w8a8_workspace_bytes(void) { return 16; }

extern "C" void vra_w8a8_gemm(const int8_t* x, const float* x_scales, const int8_t* w, const float* w_scales, const void* bias, const void* residual, void* out,
                              void* workspace, int32_t m, int32_t k, int32_t n, int32_t dtype, int64_t stream) {
  const GemmI8Args a = {x, x_scales, {w, nullptr}, {w_scales, nullptr}, bias, residual, out, m, n, k, dtype};
  if (product_ok("vra_w8a8_gemm", a, workspace, 1) && m) launch<false>(a, workspace, as_stream(stream));
}
extern "C" void vra_w8a8_gate_up_silu(const int8_t* x, const float* x_scales, const int8_t* w_gate, const float* s_gate, const int8_t* w_up, const float* s_up,
                                      void* out, void* workspace, int32_t m, int32_t k, int32_t n, int32_t dtype, int64_t stream) {
  const GemmI8Args a = {x, x_scales, {w_gate, w_up}, {s_gate, s_up}, nullptr, nullptr, out, m, n, k, dtype};
  if (product_ok("vra_w8a8_gate_up_silu", a, workspace, 2) && m) launch<true>(a, workspace, as_stream(stream));
}
