// Internal entries and device functions shared by the training kernels (arguments already validated).
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

// fp32 on the CUDA cores (train_simt.cu): few rows, or no scratch
int dice_internal_simt_linear(const void* a, int64_t n_rows, int k_dim, const void* w, int n_slabs, int n_dim,
                              const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, void* out,
                              uint32_t* status, cudaStream_t s);
int dice_internal_simt_dgrad(const void* dy, int64_t n_rows, int n_dim, const void* w, int n_slabs, int k_dim,
                             const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, void* dx,
                             uint32_t* status, cudaStream_t s);
int dice_internal_simt_wgrad(const void* dy, const void* x, int64_t n_rows, int n_dim, int k_dim,
                             const int32_t* seg_offsets, int n_slabs, int gate_up, void* dw, void* dw_up,
                             uint32_t* status, cudaStream_t s);

// the values of an fp32 product (kind: DICE_PRODUCT_*) that are not finite, made again if `non_finite` says that there are any
int dice_internal_f32_repair(int kind, const void* a, const void* b, int64_t n_rows, int n_dim, int k_dim, int n_slabs,
                             const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, int gate_up, void* out,
                             void* out_up, const unsigned int* non_finite, cudaStream_t s);

// bf16 input gradient of at most kThinTotal rows, on the CUDA cores (train_thin.cu)
constexpr int kThinTotal = 4;
int dice_internal_thin_dgrad(const void* dy, int64_t n_rows, int n_dim, const void* w, int n_slabs, int k_dim,
                             const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, void* dx, uint32_t* status,
                             cudaStream_t s);

// bf16 on the tensor cores (train_gemm.cu)
size_t dice_internal_split_bytes(int64_t n_rows, int n_dim, int k_dim, int n_slabs, bool weight_gradient);
int dice_internal_tc_dgrad(const void* dy, int64_t n_rows, int n_dim, const void* w, int n_slabs, int k_dim,
                           const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, void* dx, void* scratch,
                           size_t scratch_bytes, uint32_t* status, cudaStream_t s);
int dice_internal_tc_wgrad(const void* dy, const void* x, int64_t n_rows, int n_dim, int k_dim, const int32_t* seg_offsets,
                           int n_slabs, int gate_up, void* dw, void* dw_up, void* scratch, size_t scratch_bytes, uint32_t* status,
                           cudaStream_t s);

// fp32 on the tensor cores, as six products of bf16 planes: scratch that it takes (0: not there), and the product
size_t dice_internal_f32_bytes(int kind, int64_t n_rows, int n_dim, int k_dim, int n_slabs);
int dice_internal_f32_product(int kind, const void* a, const void* b, int64_t n_rows, int n_dim, int k_dim, int n_slabs,
                              const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, int gate_up, void* out,
                              void* out_up, void* scratch, size_t scratch_bytes, uint32_t* status, cudaStream_t s);

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

// where what was kept may start: codes are read eight at a time, an argument in its own type 16 bytes at a time
inline bool kept_aligned(const void* kept, int keep) {
  return (reinterpret_cast<uintptr_t>(kept) & (keep == DICE_KEEP_NONE ? 15u : 7u)) == 0;
}

// ---- two fp32 values --------------------------------------------------------------
// The functions below work on two values at a time, in one of two forms that round alike: `f32x2` is a register pair for
// Blackwell's two-wide multiplies and adds, half the instructions where those are what bounds a kernel (the products'
// epilogues); `two` is two plain registers, which the row-wise kernels take: bounded by memory, they lose more to the
// moves in and out of pairs than they gain (activation's backward pass at 32768 x 4608: 229 us plain, 239 two-wide).
typedef uint64_t f32x2;
struct two {
  float x, y;
};
template <typename V>
__device__ __forceinline__ V pair(float lo, float hi) {
  if constexpr (sizeof(V) == sizeof(f32x2) && !__is_class(V)) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
  } else {
    return V{lo, hi};
  }
}
template <typename V>
__device__ __forceinline__ V both(float v) { return pair<V>(v, v); }
__device__ __forceinline__ two halves(f32x2 v) {
  two r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ two halves(two v) { return v; }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ two mul2(two a, two b) { return {__fmul_rn(a.x, b.x), __fmul_rn(a.y, b.y)}; }
__device__ __forceinline__ two add2(two a, two b) { return {__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)}; }
__device__ __forceinline__ two fma2(two a, two b, two c) { return {__fmaf_rn(a.x, b.x, c.x), __fmaf_rn(a.y, b.y, c.y)}; }
template <typename V>
__device__ __forceinline__ V most2(V v, float most) {
  const two f = halves(v);
  return pair<V>(fminf(f.x, most), fminf(f.y, most));
}
template <typename V>
__device__ __forceinline__ V bf16_pair(uint32_t w) { return pair<V>(bf16lo_to_f32(w), bf16hi_to_f32(w)); }
template <typename V>
__device__ __forceinline__ uint32_t to_bf16(V v) {
  const two f = halves(v);
  return pack_bf16x2(f.x, f.y);
}

// ---- activation functions and their derivatives, fp32 ------------------------------
// gelu_tanh(p) = p/2 (1 + tanh(u)) = p sigmoid(2u), u = sqrt(2/pi) (p + 0.044715 p^3): the sigmoid form has no
// cancellation for negative p.  EXACT (fp32 tensors) uses the correctly rounded division and expf; the other form
// (16-bit tensors, whose rounding is 2^-9) the hardware's exp2 and reciprocal, good to about 2^-21.
template <bool EXACT, typename V>
__device__ __forceinline__ V sigmoid2(V x) {
  if (EXACT) {
    const two v = halves(x);
    return pair<V>(1.0f / (1.0f + expf(-v.x)), 1.0f / (1.0f + expf(-v.y)));
  }
  two t = halves(mul2(x, both<V>(-1.4426950408889634f)));  // -log2(e) x
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t.y));
  t = halves(add2(pair<V>(t.x, t.y), both<V>(1.0f)));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(t.x));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(t.y));
  return pair<V>(t.x, t.y);
}
constexpr float kGeluTwoC = 1.5957691216057308f;  // 2 sqrt(2 / pi)
template <bool EXACT, typename V>
__device__ __forceinline__ V gelu_sigmoid2(V p) {
  return sigmoid2<EXACT>(mul2(both<V>(kGeluTwoC), fma2(mul2(mul2(both<V>(0.044715f), p), p), p, p)));
}
template <bool EXACT, typename V>
__device__ __forceinline__ V gelu2(V p) {
  return mul2(p, gelu_sigmoid2<EXACT>(p));
}
template <bool EXACT, typename V>
__device__ __forceinline__ V swiglu2(V g, V u) {
  return mul2(mul2(g, sigmoid2<EXACT>(g)), u);
}
// value a and derivative
template <bool EXACT, typename V>
__device__ __forceinline__ V gelu_grad2(V p, V& a) {
  const V s = gelu_sigmoid2<EXACT>(p), one = both<V>(1.0f);
  a = mul2(p, s);
  // (the square may be beyond the range; 1 - s, which it meets, is 0 or a is long before)
  const V inner = mul2(both<V>(kGeluTwoC), add2(most2(mul2(mul2(both<V>(3.0f * 0.044715f), p), p), 1e30f), one));
  return fma2(mul2(a, fma2(s, both<V>(-1.0f), one)), inner, s);
}
template <bool EXACT, typename V>
__device__ __forceinline__ V silu_grad2(V g, V& a) {
  const V s = sigmoid2<EXACT>(g), one = both<V>(1.0f);
  a = mul2(g, s);
  return mul2(s, fma2(g, fma2(s, both<V>(-1.0f), one), one));
}
// the argument's gradient from the activation's (da): SwiGLU g, u -> their gradients, GELU g -> its; and the activation
template <bool EXACT, int ACT, typename V>
__device__ __forceinline__ V act_backward2(V da, V& g, V& u) {
  V a;
  if (ACT == DICE_ACT_SWIGLU) {
    const V slope = silu_grad2<EXACT>(g, a), act = a;
    g = mul2(mul2(da, u), slope);
    a = mul2(act, u);
    u = mul2(da, act);
  } else {
    g = mul2(da, gelu_grad2<EXACT>(g, a));
  }
  return a;
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
// four values (already times the factor) as codes in a word
template <int KEEP, typename V>
__device__ __forceinline__ uint32_t keep_codes4(V ab, V cd) {
  if (KEEP == DICE_KEEP_INT8) {
    // adding 1.5 * 2^23 rounds to an integer (ties to even) and leaves it in the low byte; the conversion instruction
    // would take the pipe of exp and reciprocal, which the activation needs.  What a NaN gives is never read (its
    // scale is NaN).
    // (Scalar additions: the compiler joins a two-wide one with the caller's multiplication, and the sum would round once.)
    const float kRound = 12582912.0f;
    const two x = halves(ab), y = halves(cd);
    return __byte_perm(__byte_perm(__float_as_uint(__fadd_rn(x.x, kRound)), __float_as_uint(__fadd_rn(x.y, kRound)), 0x0040),
                       __byte_perm(__float_as_uint(__fadd_rn(y.x, kRound)), __float_as_uint(__fadd_rn(y.y, kRound)), 0x0040), 0x5410);
  }
  const two x = halves(ab), y = halves(cd);
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x.y), "f"(x.x));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y.y), "f"(y.x));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}
// and back, times the scale
template <int KEEP, typename V>
__device__ __forceinline__ void keep_read4(uint32_t w, V scale, V& ab, V& cd) {
  if (KEEP == DICE_KEEP_INT8) {
    // the byte plus 128 becomes the low mantissa bits of 2^23: exact, and again without the conversion instruction
    const uint32_t biased = w ^ 0x80808080u, base = 0x4b000000u;
    const V off = both<V>(-8388736.0f);
    ab = mul2(add2(pair<V>(__uint_as_float(__byte_perm(biased, base, 0x7540)), __uint_as_float(__byte_perm(biased, base, 0x7541))), off), scale);
    cd = mul2(add2(pair<V>(__uint_as_float(__byte_perm(biased, base, 0x7542)), __uint_as_float(__byte_perm(biased, base, 0x7543))), off), scale);
  } else {
    uint32_t lo, hi;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"(static_cast<uint16_t>(w)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"(static_cast<uint16_t>(w >> 16)));
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo)), y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    ab = mul2(pair<V>(x.x, x.y), scale);
    cd = mul2(pair<V>(y.x, y.y), scale);
  }
}
