// Internal entries and device functions shared by the training kernels (arguments already validated).
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

// fp32 on the CUDA cores (train_simt.cu)
int dice_internal_simt_linear(const void* a, int64_t n_rows, int k_dim, const void* w, int n_slabs, int n_dim,
                              const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, void* out,
                              uint32_t* status, cudaStream_t s);
int dice_internal_simt_dgrad(const void* dy, int64_t n_rows, int n_dim, const void* w, int n_slabs, int k_dim,
                             const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, void* dx,
                             uint32_t* status, cudaStream_t s);
int dice_internal_simt_wgrad(const void* dy, const void* x, int64_t n_rows, int n_dim, int k_dim,
                             const int32_t* seg_offsets, int n_slabs, int gate_up, void* dw, void* dw_up,
                             uint32_t* status, cudaStream_t s);

// bf16 on the tensor cores (train_gemm.cu)
int dice_internal_tc_dgrad(const void* dy, int64_t n_rows, int n_dim, const void* w, int n_slabs, int k_dim,
                           const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, void* dx, uint32_t* status,
                           cudaStream_t s);
int dice_internal_tc_wgrad(const void* dy, const void* x, int64_t n_rows, int n_dim, int k_dim, const int32_t* seg_offsets,
                           int n_slabs, int gate_up, void* dw, void* dw_up, uint32_t* status, cudaStream_t s);

// the forward product with the activation and what is kept in its epilogue, and the second product's input gradient with
// the activation's backward pass in its epilogue (see train_gemm.cu); pointers as in the public entry points
int dice_internal_tc_keep(const void* rows, int64_t n_rows, int hidden, int ffn, int act, int keep, const void* w1, int n_slabs,
                          const int32_t* seg_offsets, int n_seg, void* pre, void* a, void* codes, float* scales,
                          uint32_t* status, cudaStream_t s);
int dice_internal_tc_back(const void* d_out, int64_t n_rows, int hidden, int ffn, int act, int keep, const void* w2, int n_slabs,
                          const int32_t* seg_offsets, const void* kept, const float* scales, void* d_pre, void* a,
                          uint32_t* status, cudaStream_t s);

constexpr int kKeepGroup = 128;               // columns of a kept argument that share a scale
constexpr float kKeepFloor = 7.888609e-31f;   // 2^-100: the smallest group maximum a scale is made from

// ---- activation functions and their derivatives, fp32 ------------------------------
// gelu_tanh(p) = p/2 (1 + tanh(u)) = p sigmoid(2u), u = sqrt(2/pi) (p + 0.044715 p^3): the sigmoid form has no
// cancellation for negative p.  EXACT (fp32 tensors) uses the correctly rounded division and expf; the other form
// (16-bit tensors, whose rounding is 2^-9) the fast ones, good to about 2^-21.
template <bool EXACT>
__device__ __forceinline__ float sigmoid_t(float x) {
  if (EXACT) return 1.0f / (1.0f + expf(-x));
  return __fdividef(1.0f, 1.0f + __expf(-x));
}
constexpr float kGeluTwoC = 1.5957691216057308f;  // 2 sqrt(2 / pi)
template <bool EXACT>
__device__ __forceinline__ float gelu_t(float p) {
  return p * sigmoid_t<EXACT>(kGeluTwoC * fmaf(0.044715f * p * p, p, p));
}
// value and derivative
template <bool EXACT>
__device__ __forceinline__ void gelu_grad_t(float p, float& a, float& da) {
  const float s = sigmoid_t<EXACT>(kGeluTwoC * fmaf(0.044715f * p * p, p, p));
  a = p * s;
  da = fmaf(a * (1.0f - s), kGeluTwoC * fmaf(3.0f * 0.044715f * p, p, 1.0f), s);
}
template <bool EXACT>
__device__ __forceinline__ void silu_grad_t(float g, float& a, float& da) {
  const float s = sigmoid_t<EXACT>(g);
  a = g * s;
  da = s * fmaf(g, 1.0f - s, 1.0f);
}

// ---- 8-bit codes ---------------------------------------------------------------------
// code = rn(x * (top / most)), read back as code * (most / top); `most` is the group's largest magnitude, at least
// 2^-100 (so that top / most is finite and an all-zero group reads back as zeros).
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float keep_top(int keep) { return keep == DICE_KEEP_INT8 ? 127.0f : 448.0f; }
// the stored scale of a group and the factor its values are multiplied by; an infinity or a NaN in the group makes
// the scale NaN, and with it every value that is read back
__device__ __forceinline__ void keep_scale(float most, float top, float& scale, float& factor) {
  most = max_nan(most, kKeepFloor);
  factor = __fdiv_rn(top, most);
  scale = most <= 3.402823466e+38f ? __fdiv_rn(most, top) : __int_as_float(0x7fc00000);
}
// four codes in a word
template <int KEEP>
__device__ __forceinline__ uint32_t keep_codes4(float a, float b, float c, float d) {
  if (KEEP == DICE_KEEP_INT8) {
    // adding 1.5 * 2^23 rounds to an integer (ties to even) and leaves it in the low byte; the conversion instruction
    // would take the pipe of exp and reciprocal, which the activation needs.  What a NaN gives is never read (its
    // scale is NaN).
    // (__fadd_rn: fused with the caller's multiplication the sum would round once, and ties elsewhere.)
    const float kRound = 12582912.0f;
    return __byte_perm(__byte_perm(__float_as_uint(__fadd_rn(a, kRound)), __float_as_uint(__fadd_rn(b, kRound)), 0x0040),
                       __byte_perm(__float_as_uint(__fadd_rn(c, kRound)), __float_as_uint(__fadd_rn(d, kRound)), 0x0040), 0x5410);
  }
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}
template <int KEEP>
__device__ __forceinline__ void keep_read4(uint32_t w, float scale, float* v) {
  if (KEEP == DICE_KEEP_INT8) {
    // the byte plus 128 becomes the low mantissa bits of 2^23: exact, and again without the conversion instruction
    const uint32_t biased = w ^ 0x80808080u;
    const uint32_t kBase = 0x4b000000u;
    v[0] = (__uint_as_float(__byte_perm(biased, kBase, 0x7540)) - 8388736.0f) * scale;
    v[1] = (__uint_as_float(__byte_perm(biased, kBase, 0x7541)) - 8388736.0f) * scale;
    v[2] = (__uint_as_float(__byte_perm(biased, kBase, 0x7542)) - 8388736.0f) * scale;
    v[3] = (__uint_as_float(__byte_perm(biased, kBase, 0x7543)) - 8388736.0f) * scale;
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t h2;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(w >> (16 * i))));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
      v[2 * i] = f.x * scale;
      v[2 * i + 1] = f.y * scale;
    }
  }
}
