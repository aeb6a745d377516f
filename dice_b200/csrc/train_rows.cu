// The row-wise operators of the training step, each one pass over its data:
//
//   act_keep          a = act(p), and p itself in 8 bits for the backward pass (128 columns share a scale)
//   act_backward      dp = da * act'(p), a = act(p) again, p read back from its 8 bits
//   combine_backward  the gradient of out[t] = w0 y[pos0] + w1 y[pos1]: rows w_s dout[t], weights <dout[t], y[pos_s]>
//
// All three are bounded by HBM: 16 bytes (bf16) or 32 bytes (fp32) per lane and access, eight columns a lane.  For
// the activation, 16 lanes own one group of 128 columns, so that the group's maximum is four shuffles; with SwiGLU
// the same 16 lanes own the group's gate and its up columns, which the packed order puts 128 columns apart.
//
// Measured on a B200 whose copies reach 6.55 TB/s, two sets of inputs in turn: act_keep (int8, SwiGLU, 32768 x 4608) moves
// 1217 MB in 203 us = 6.0 TB/s (235 us before one division served four quotients and both groups' maxima shared their
// shuffles: it issues about 20 instructions an element and was bounded by them); act_backward 1519 MB in 228 us = 6.7 TB/s
// (906 MB of them written; a memset, which only writes, takes 244 us for as many); combine_backward (16384 tokens x 1152)
// 189 MB in 31.5 us = 6.0 TB/s.
#include "train.cuh"

namespace {

constexpr int kThreadsRows = 256;
constexpr int kHalfWarps = kThreadsRows / 16;

// eight neighbouring values in their storage type, and as four times two fp32
template <typename T>
struct Vec8;
template <>
struct Vec8<__nv_bfloat16> {
  uint4 v;
  __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = ldg_stream16(p); }
  __device__ __forceinline__ void get(two (&f)[4]) const {
    f[0] = bf16_pair<two>(v.x); f[1] = bf16_pair<two>(v.y); f[2] = bf16_pair<two>(v.z); f[3] = bf16_pair<two>(v.w);
  }
  // largest magnitude (NaN if there is one)
  __device__ __forceinline__ float most() const {
    uint32_t m = v.x & 0x7fff7fffu;
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(v.y & 0x7fff7fffu));
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(v.z & 0x7fff7fffu));
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(v.w & 0x7fff7fffu));
    return max_nan(bf16lo_to_f32(m), bf16hi_to_f32(m));
  }
};
template <>
struct Vec8<float> {
  uint4 v[2];
  __device__ __forceinline__ void zero() { v[0] = v[1] = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load(const float* p) {
    v[0] = ldg_stream16(p);
    v[1] = ldg_stream16(p + 4);
  }
  __device__ __forceinline__ void get(two (&f)[4]) const {
    f[0] = pair<two>(__uint_as_float(v[0].x), __uint_as_float(v[0].y));
    f[1] = pair<two>(__uint_as_float(v[0].z), __uint_as_float(v[0].w));
    f[2] = pair<two>(__uint_as_float(v[1].x), __uint_as_float(v[1].y));
    f[3] = pair<two>(__uint_as_float(v[1].z), __uint_as_float(v[1].w));
  }
  __device__ __forceinline__ float most() const {
    const float* f = reinterpret_cast<const float*>(v);
    float m = fabsf(f[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(f[i]));
    return m;
  }
};
__device__ __forceinline__ void put8(__nv_bfloat16* p, const two (&f)[4]) {
  stg_stream16(p, make_uint4(to_bf16(f[0]), to_bf16(f[1]), to_bf16(f[2]), to_bf16(f[3])));
}
__device__ __forceinline__ void put8(float* p, const two (&f)[4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const two x = halves(f[2 * i]), y = halves(f[2 * i + 1]);
    stg_stream16(p + 4 * i, make_uint4(__float_as_uint(x.x), __float_as_uint(x.y), __float_as_uint(y.x), __float_as_uint(y.y)));
  }
}

// The largest magnitudes of a half-warp's one or two groups of 128, from its lanes' own; of two bf16 groups, both at once.
template <bool BOTH, typename T>
__device__ __forceinline__ void group_most(float& g, float& u) {
  const unsigned mask = 0xffffu << (threadIdx.x & 16);
  if constexpr (BOTH && sizeof(T) == 2) {
    uint32_t m = (__float_as_uint(g) >> 16) | (__float_as_uint(u) & 0xffff0000u);
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(__shfl_xor_sync(mask, m, off)));
    g = bf16lo_to_f32(m);
    u = bf16hi_to_f32(m);
  } else {
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) {
      g = max_nan(g, __shfl_xor_sync(mask, g, off));
      if (BOTH) u = max_nan(u, __shfl_xor_sync(mask, u, off));
    }
  }
}

// The factors of the groups (all 16 lanes), whose scales one lane each stores.  One division a lane makes all four
// quotients: lanes 0-3 the first group's factor, 4-7 its scale, 8-11 and 12-15 the second group's.
template <bool BOTH, int KEEP>
__device__ __forceinline__ void group_factors(float g, float u, float* scales, float& factor_g, float& factor_u) {
  const int lane = threadIdx.x & 15;
  const unsigned mask = 0xffffu << (threadIdx.x & 16);
  const float top = keep_top(KEEP);
  float most = BOTH && (lane & 8) ? u : g;
  const bool finite = most <= 3.402823466e+38f;
  most = max_nan(most, kKeepFloor);
  const bool scale = lane & 4;
  const float q = __fdiv_rn(scale ? most : top, scale ? top : most);
  factor_g = __shfl_sync(mask, q, 0, 16);
  factor_u = BOTH ? __shfl_sync(mask, q, 8, 16) : 0.f;
  if (lane == 4 || (BOTH && lane == 12)) scales[lane >> 3] = finite ? q : __int_as_float(0x7fc00000);
}

template <int KEEP>
__device__ __forceinline__ void put_codes(const two (&f)[4], float factor, uint8_t* codes) {
  const two k = both<two>(factor);
  *reinterpret_cast<uint2*>(codes) =
      make_uint2(keep_codes4<KEEP>(mul2(f[0], k), mul2(f[1], k)), keep_codes4<KEEP>(mul2(f[2], k), mul2(f[3], k)));
}

struct ActParams {
  const void* in;        // keep: pre; backward: da
  const void* kept;      // backward: codes, or pre
  const float* kept_scales;
  void* a;               // may be NULL (backward)
  uint8_t* codes;
  float* scales;
  void* d_pre;
  int64_t n_rows;
  int ffn, cols, groups_in, blocks;  // cols: of the argument; groups_in: scales of a row; blocks: units of 16 lanes a row
  int rows_per_cta;
};

template <typename T, int ACT, int KEEP>
__global__ void __launch_bounds__(kThreadsRows) act_keep_kernel(const ActParams p) {
  constexpr bool EXACT = sizeof(T) == 4, GLU = ACT == DICE_ACT_SWIGLU;
  const int hw = threadIdx.x >> 4, lane = threadIdx.x & 15;
  pdl_trigger();
  pdl_wait();
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * p.rows_per_cta;
  const int64_t left = p.n_rows - row0;
  const int items = static_cast<int>(left < p.rows_per_cta ? left : p.rows_per_cta) * p.blocks;
  int b = hw % p.blocks;
  int64_t row = row0 + hw / p.blocks;
  for (int it = hw; it < items; it += kHalfWarps, b += kHalfWarps) {
    for (; b >= p.blocks; b -= p.blocks) ++row;
    const int col = b * kKeepGroup + lane * 8;  // of the activation
    const bool ok = col < p.ffn;
    const int64_t at = row * p.cols + (GLU ? b * 2 * kKeepGroup + lane * 8 : col);  // of the argument
    Vec8<T> v, u;
    v.zero();
    u.zero();
    if (ok) {
      v.load(static_cast<const T*>(p.in) + at);
      if (GLU) u.load(static_cast<const T*>(p.in) + at + kKeepGroup);
    }
    two g[4], h[4], a[4];
    v.get(g);
    if (GLU) u.get(h);
    if (KEEP != DICE_KEEP_NONE) {
      float mg = v.most(), mu = GLU ? u.most() : 0.f, fg, fu;
      group_most<GLU, T>(mg, mu);
      group_factors<GLU, KEEP>(mg, mu, p.scales + row * p.groups_in + (GLU ? 2 * b : b), fg, fu);
      // the packed order's filling columns get codes too (of zero)
      if (GLU || ok) put_codes<KEEP>(g, fg, p.codes + at);
      if (GLU) put_codes<KEEP>(h, fu, p.codes + at + kKeepGroup);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = GLU ? swiglu2<EXACT>(g[i], h[i]) : gelu2<EXACT>(g[i]);
    if (ok) put8(static_cast<T*>(p.a) + row * p.ffn + col, a);
  }
}

// the kept argument of eight columns, read back
template <typename T, int KEEP>
struct Kept8;
template <typename T>
struct Kept8<T, DICE_KEEP_NONE> {
  Vec8<T> v;
  __device__ __forceinline__ void load(const void* base, int64_t at, const float*) { v.load(static_cast<const T*>(base) + at); }
  __device__ __forceinline__ void get(two (&f)[4]) const { v.get(f); }
};
template <typename T, int KEEP>
struct Kept8 {
  uint2 w;
  float scale;
  __device__ __forceinline__ void load(const void* base, int64_t at, const float* sc) {
    w = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(base) + at);
    scale = *sc;
  }
  __device__ __forceinline__ void get(two (&f)[4]) const {
    keep_read4<KEEP>(w.x, both<two>(scale), f[0], f[1]);
    keep_read4<KEEP>(w.y, both<two>(scale), f[2], f[3]);
  }
};

template <typename T, int ACT, int KEEP>
__global__ void __launch_bounds__(kThreadsRows) act_backward_kernel(const ActParams p) {
  constexpr bool EXACT = sizeof(T) == 4, GLU = ACT == DICE_ACT_SWIGLU;
  const int hw = threadIdx.x >> 4, lane = threadIdx.x & 15;
  pdl_trigger();
  pdl_wait();
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * p.rows_per_cta;
  const int64_t left = p.n_rows - row0;
  const int items = static_cast<int>(left < p.rows_per_cta ? left : p.rows_per_cta) * p.blocks;
  int b = hw % p.blocks;
  int64_t row = row0 + hw / p.blocks;
  for (int it = hw; it < items; it += kHalfWarps, b += kHalfWarps) {
    for (; b >= p.blocks; b -= p.blocks) ++row;
    const int col = b * kKeepGroup + lane * 8;
    const int64_t at = row * p.cols + (GLU ? b * 2 * kKeepGroup + lane * 8 : col);
    T* d_pre = static_cast<T*>(p.d_pre) + at;
    if (col >= p.ffn) {
      if (GLU) {  // the packed order's filling columns: their gradient is zero
        const two z[4] = {};
        put8(d_pre, z);
        put8(d_pre + kKeepGroup, z);
      }
      continue;
    }
    const float* sc = KEEP == DICE_KEEP_NONE ? nullptr : p.kept_scales + row * p.groups_in + (GLU ? 2 * b : b);
    Vec8<T> d;
    Kept8<T, KEEP> kg, ku;
    d.load(static_cast<const T*>(p.in) + row * p.ffn + col);
    kg.load(p.kept, at, sc);
    if (GLU) ku.load(p.kept, at + kKeepGroup, sc + 1);
    two da[4], g[4], u[4], a[4];
    d.get(da);
    kg.get(g);
    if (GLU) ku.get(u);
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = act_backward2<EXACT, ACT>(da[i], g[i], u[i]);
    put8(d_pre, g);
    if (GLU) put8(d_pre + kKeepGroup, u);
    if (p.a != nullptr) put8(static_cast<T*>(p.a) + row * p.ffn + col, a);
  }
}

template <typename T, int ACT, int KEEP>
cudaError_t launch_act(const ActParams& p, bool backward, unsigned grid, cudaStream_t s) {
  return backward ? dice_launch(act_backward_kernel<T, ACT, KEEP>, dim3(grid), dim3(kThreadsRows), 0, s, p)
                  : dice_launch(act_keep_kernel<T, ACT, KEEP>, dim3(grid), dim3(kThreadsRows), 0, s, p);
}
template <typename T, int ACT>
cudaError_t launch_act(int keep, const ActParams& p, bool backward, unsigned grid, cudaStream_t s) {
  switch (keep) {
    case DICE_KEEP_INT8: return launch_act<T, ACT, DICE_KEEP_INT8>(p, backward, grid, s);
    case DICE_KEEP_E4M3: return launch_act<T, ACT, DICE_KEEP_E4M3>(p, backward, grid, s);
    default: return launch_act<T, ACT, DICE_KEEP_NONE>(p, backward, grid, s);
  }
}

int run_act(ActParams p, int act, int keep, int dtype, bool backward, cudaStream_t s) {
  p.blocks = (p.ffn + kKeepGroup - 1) / kKeepGroup;
  p.groups_in = act == DICE_ACT_SWIGLU ? 2 * p.blocks : p.blocks;
  p.cols = act == DICE_ACT_SWIGLU ? 2 * p.blocks * kKeepGroup : p.ffn;
  // a CTA's share: 64 units of 16 lanes (four passes) where a row has fewer
  p.rows_per_cta = 64 / p.blocks > 1 ? 64 / p.blocks : 1;
  const int64_t grid = (p.n_rows + p.rows_per_cta - 1) / p.rows_per_cta;
  if (grid > 0x7fffffffLL) return DICE_ERR_LIMIT;
  const unsigned g = static_cast<unsigned>(grid);
  cudaError_t err;
  if (dtype == DICE_BF16)
    err = act == DICE_ACT_SWIGLU ? launch_act<__nv_bfloat16, DICE_ACT_SWIGLU>(keep, p, backward, g, s)
                                 : launch_act<__nv_bfloat16, DICE_ACT_GELU_TANH>(keep, p, backward, g, s);
  else
    err = act == DICE_ACT_SWIGLU ? launch_act<float, DICE_ACT_SWIGLU>(keep, p, backward, g, s)
                                 : launch_act<float, DICE_ACT_GELU_TANH>(keep, p, backward, g, s);
  return err == cudaSuccess ? DICE_OK : DICE_ERR_CUDA;
}

// ---- gradient of the combine ---------------------------------------------------------
// One warp per token: dout[t] is read once for its two rows.
template <typename T>
__global__ void __launch_bounds__(256)
combine_backward_kernel(const T* dout, const T* rows_out, const int32_t* pos, const float* weights, int64_t n_tokens,
                        int64_t n_rows, int hidden, T* d_rows, float* d_weights) {
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  pdl_trigger();
  pdl_wait();
  if (t >= n_tokens) return;
  const int2 pp = *reinterpret_cast<const int2*>(pos + 2 * t);
  const float2 w = *reinterpret_cast<const float2*>(weights + 2 * t);
  const bool ok0 = pp.x >= 0 && pp.x < n_rows, ok1 = pp.y >= 0 && pp.y < n_rows;
  const T* src = dout + t * hidden;
  const int64_t o0 = static_cast<int64_t>(pp.x) * hidden, o1 = static_cast<int64_t>(pp.y) * hidden;
  two d0 = {0.f, 0.f}, d1 = {0.f, 0.f};
  const two w0 = both<two>(w.x), w1 = both<two>(w.y);
  for (int c = lane * 8; c < hidden; c += 256) {
    Vec8<T> d, y0, y1;
    y0.zero();
    y1.zero();
    d.load(src + c);
    if (ok0) y0.load(rows_out + o0 + c);
    if (ok1) y1.load(rows_out + o1 + c);
    two f[4], y[4], r[4];
    d.get(f);
    if (ok0) {
      y0.get(y);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        d0 = fma2(f[i], y[i], d0);
        r[i] = mul2(w0, f[i]);
      }
      put8(d_rows + o0 + c, r);
    }
    if (ok1) {
      y1.get(y);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        d1 = fma2(f[i], y[i], d1);
        r[i] = mul2(w1, f[i]);
      }
      put8(d_rows + o1 + c, r);
    }
  }
  float s0 = halves(d0).x + halves(d0).y, s1 = halves(d1).x + halves(d1).y;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    s0 += __shfl_xor_sync(0xffffffffu, s0, off);
    s1 += __shfl_xor_sync(0xffffffffu, s1, off);
  }
  if (lane == 0) *reinterpret_cast<float2*>(d_weights + 2 * t) = make_float2(s0, s1);
}

int check_act(int64_t n_rows, int ffn, int act, int keep, int dtype) {
  DICE_CHECK_ARG(act == DICE_ACT_SWIGLU || act == DICE_ACT_GELU_TANH, DICE_ERR_ARG);
  DICE_CHECK_ARG(keep == DICE_KEEP_NONE || keep == DICE_KEEP_INT8 || keep == DICE_KEEP_E4M3, DICE_ERR_ARG);
  DICE_CHECK_ARG(n_rows >= 0 && ffn > 0, DICE_ERR_ARG);
  DICE_CHECK_ARG(dice_dtype_size(dtype) != 0, DICE_ERR_DTYPE);
  DICE_CHECK_ARG(ffn % 8 == 0, DICE_ERR_SHAPE);
  DICE_CHECK_ARG(ffn <= (1 << 24) && n_rows < 0x7fffff00LL, DICE_ERR_LIMIT);
  return DICE_OK;
}

}  // namespace

extern "C" int dice_act_keep(const void* pre, int64_t n_rows, int ffn, int act, int keep, int dtype, void* a, void* codes,
                             float* scales, void* stream) {
  const int rc = check_act(n_rows, ffn, act, keep, dtype);
  if (rc != DICE_OK) return rc;
  if (n_rows == 0) return DICE_OK;
  DICE_CHECK_ARG(pre && a && (keep == DICE_KEEP_NONE || (codes && scales)), DICE_ERR_ARG);
  DICE_CHECK_ARG(dice_aligned16(pre) && dice_aligned16(a) && dice_aligned16(codes), DICE_ERR_ALIGN);
  ActParams p = {};
  p.in = pre;
  p.a = a;
  p.codes = static_cast<uint8_t*>(codes);
  p.scales = scales;
  p.n_rows = n_rows;
  p.ffn = ffn;
  return run_act(p, act, keep, dtype, false, static_cast<cudaStream_t>(stream));
}

extern "C" int dice_act_backward(const void* da, const void* kept, const float* scales, int64_t n_rows, int ffn, int act,
                                 int keep, int dtype, void* d_pre, void* a, void* stream) {
  const int rc = check_act(n_rows, ffn, act, keep, dtype);
  if (rc != DICE_OK) return rc;
  if (n_rows == 0) return DICE_OK;
  DICE_CHECK_ARG(da && kept && d_pre && (keep == DICE_KEEP_NONE || scales), DICE_ERR_ARG);
  DICE_CHECK_ARG(dice_aligned16(da) && kept_aligned(kept, keep) && dice_aligned16(d_pre) && dice_aligned16(a), DICE_ERR_ALIGN);
  ActParams p = {};
  p.in = da;
  p.kept = kept;
  p.kept_scales = scales;
  p.d_pre = d_pre;
  p.a = a;
  p.n_rows = n_rows;
  p.ffn = ffn;
  return run_act(p, act, keep, dtype, true, static_cast<cudaStream_t>(stream));
}

extern "C" int dice_combine_backward(const void* dout, const void* rows_out, const int32_t* pos, const float* weights,
                                     int64_t n_tokens, int64_t n_rows, int hidden, int dtype, void* d_rows,
                                     float* d_weights, void* stream) {
  DICE_CHECK_ARG(n_tokens >= 0 && n_rows >= 0 && hidden > 0, DICE_ERR_ARG);
  DICE_CHECK_ARG(dice_dtype_size(dtype) != 0, DICE_ERR_DTYPE);
  DICE_CHECK_ARG(hidden % 8 == 0, DICE_ERR_SHAPE);
  DICE_CHECK_ARG(n_tokens < 0x3fffff00LL && n_rows < 0x7fffff00LL, DICE_ERR_LIMIT);
  if (n_tokens == 0) return DICE_OK;
  DICE_CHECK_ARG(dout && pos && weights && d_weights && (n_rows == 0 || (rows_out && d_rows)), DICE_ERR_ARG);
  DICE_CHECK_ARG(dice_aligned16(dout) && dice_aligned16(rows_out) && dice_aligned16(d_rows), DICE_ERR_ALIGN);
  DICE_CHECK_ARG((reinterpret_cast<uintptr_t>(pos) & 7u) == 0 && (reinterpret_cast<uintptr_t>(weights) & 7u) == 0 &&
                     (reinterpret_cast<uintptr_t>(d_weights) & 7u) == 0,
                 DICE_ERR_ALIGN);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>((n_tokens + 7) / 8));
  const cudaError_t err =
      dtype == DICE_BF16
          ? dice_launch(combine_backward_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, static_cast<const __nv_bfloat16*>(dout),
                        static_cast<const __nv_bfloat16*>(rows_out), pos, weights, n_tokens, n_rows, hidden,
                        static_cast<__nv_bfloat16*>(d_rows), d_weights)
          : dice_launch(combine_backward_kernel<float>, grid, dim3(256), 0, s, static_cast<const float*>(dout),
                        static_cast<const float*>(rows_out), pos, weights, n_tokens, n_rows, hidden,
                        static_cast<float*>(d_rows), d_weights);
  return err == cudaSuccess ? DICE_OK : DICE_ERR_CUDA;
}
