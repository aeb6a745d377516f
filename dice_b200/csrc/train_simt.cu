// Products grouped by expert on the CUDA cores, for the training step's fp32 form (the tensor cores would round
// fp32 operands to tf32) in its three directions:
//
//   NT  out[r, n] = sum_k a[r, k] w[seg(r)][n, k]        the forward product (nn.Linear weights)
//   NN  dx[r, k]  = sum_n dy[r, n] w[seg(r)][n, k]       its input gradient
//   TN  dw[s][n, k] = sum_{r in seg s} dy[r, n] x[r, k]  its weight gradient
//
// 128 x 128 output tile per CTA, 16-deep shared-memory slices in two buffers (the next slice is loaded into
// registers while the present one is multiplied), 8 x 8 fp32 accumulators per thread.  Segments are ragged: each
// CTA finds its own on the device.
#include "common.cuh"
#include "train.cuh"

namespace {

constexpr int TM = 128, TN = 128, TK = 16;
constexpr int kMaxSegSimt = 256;
enum { MODE_NT = 0, MODE_NN = 1, MODE_TN = 2 };

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  return make_float4(bf16lo_to_f32(v.x), bf16hi_to_f32(v.x), bf16lo_to_f32(v.y), bf16hi_to_f32(v.y));
}
__device__ __forceinline__ void store4(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float* v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

// One thread's share (two groups of 4) of a 128 x 16 operand slice.  KMAJOR: the reduction index is contiguous in
// memory ([mn][k]), the thread holds 8 reduction elements of one row; else ([k][mn]) it holds columns c .. c+3 and
// c+64 .. c+67 of one reduction row.  mn_valid / k_valid: what is left of the operand from the slice's corner.
template <typename T, bool KMAJOR>
__device__ __forceinline__ void load_slice(const T* base, int64_t ld, int mn_valid, int64_t k_valid, float4 (&v)[2]) {
  v[0] = v[1] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (KMAJOR) {
    const int r = threadIdx.x >> 1, k = (threadIdx.x & 1) * 8;
    if (r < mn_valid) {
      const T* p = base + static_cast<int64_t>(r) * ld + k;
      if (k < k_valid) v[0] = load4(p);
      if (k + 4 < k_valid) v[1] = load4(p + 4);
    }
  } else {
    const int k = threadIdx.x >> 4, c = (threadIdx.x & 15) * 4;
    if (k < k_valid) {
      const T* p = base + static_cast<int64_t>(k) * ld + c;
      if (c < mn_valid) v[0] = load4(p);
      if (c + 64 < mn_valid) v[1] = load4(p + 64);
    }
  }
}
template <bool KMAJOR>
__device__ __forceinline__ void put_slice(float (*s)[TM + 4], const float4 (&v)[2]) {
  if (KMAJOR) {
    const int r = threadIdx.x >> 1, k = (threadIdx.x & 1) * 8;
    s[k + 0][r] = v[0].x; s[k + 1][r] = v[0].y; s[k + 2][r] = v[0].z; s[k + 3][r] = v[0].w;
    s[k + 4][r] = v[1].x; s[k + 5][r] = v[1].y; s[k + 6][r] = v[1].z; s[k + 7][r] = v[1].w;
  } else {
    const int k = threadIdx.x >> 4, c = (threadIdx.x & 15) * 4;
    *reinterpret_cast<float4*>(&s[k][c]) = v[0];
    *reinterpret_cast<float4*>(&s[k][c + 64]) = v[1];
  }
}

struct SimtParams {
  const void* a;   // NT: rows, NN / TN: dy
  const void* b;   // NT / NN: w, TN: x
  void* out;
  void* out_up;    // TN with gate_up: the up gradients
  const int* seg_offsets;
  const int* seg_slab;
  int n_seg, n_slabs;
  int64_t n_rows;
  int m_cols;      // TN: output rows per slab (dy columns)
  int n_cols;      // output columns
  int red;         // NT / NN: reduction length
  int gate_up;     // TN: 0, or ffn: output rows are packed gate / up blocks
  uint32_t* status;
};

template <typename T, int MODE>
__global__ void __launch_bounds__(256) simt_grouped_kernel(const SimtParams p) {
  __shared__ __align__(16) float As[2][TK][TM + 4];
  __shared__ __align__(16) float Bs[2][TK][TN + 4];
  __shared__ int s_seg, s_row0, s_rows;
  pdl_trigger();
  pdl_wait();
  if (threadIdx.x == 0) {
    int found = -1, row0 = 0, rows = 0;
    bool ok = true;
    if (MODE == MODE_TN) {
      found = blockIdx.z;
      row0 = p.seg_offsets[found];
      rows = p.seg_offsets[found + 1] - row0;
      ok = row0 >= 0 && rows >= 0 && static_cast<int64_t>(row0) + rows <= p.n_rows;
    } else {
      int run = 0;
      for (int s = 0; s < p.n_seg && found < 0 && ok; ++s) {
        const int beg = p.seg_offsets[s], cnt = p.seg_offsets[s + 1] - beg;
        ok = beg >= 0 && cnt >= 0 && static_cast<int64_t>(beg) + cnt <= p.n_rows;
        const int nb = ok ? (cnt + TM - 1) / TM : 0;
        if (ok && static_cast<int>(blockIdx.x) < run + nb) {
          found = s;
          row0 = beg + (static_cast<int>(blockIdx.x) - run) * TM;
          rows = beg + cnt - row0;
        }
        run += nb;
      }
      if (found >= 0 && p.seg_slab != nullptr) {
        found = p.seg_slab[found];  // -1: rows that belong to no expert
        ok = found < p.n_slabs;
      }
    }
    if (!ok) {
      found = -1;
      if (p.status != nullptr) atomicCAS(p.status, 0u, DICE_STATUS_BAD_SEGMENTS);
    }
    s_seg = found; s_row0 = row0; s_rows = rows;
  }
  __syncthreads();
  if (s_seg < 0) return;
  const int slab = s_seg, row0 = s_row0, seg_rows = s_rows;
  const int col0 = blockIdx.y * TN;

  const T* a = static_cast<const T*>(p.a);
  const T* b = static_cast<const T*>(p.b);
  int64_t lda, ldb, red;   // strides and reduction length
  int m_valid;
  const int n_valid = p.n_cols - col0;
  constexpr bool kA = MODE != MODE_TN, kB = MODE == MODE_NT;  // which operands have the reduction contiguous
  if (MODE == MODE_TN) {
    lda = p.m_cols; ldb = p.n_cols; red = seg_rows;
    a += static_cast<int64_t>(row0) * lda + static_cast<int64_t>(blockIdx.x) * TM;
    b += static_cast<int64_t>(row0) * ldb + col0;
    m_valid = p.m_cols - static_cast<int>(blockIdx.x) * TM;
  } else {
    lda = red = p.red;
    a += static_cast<int64_t>(row0) * lda;
    m_valid = seg_rows;
    if (MODE == MODE_NT) {
      ldb = p.red;
      b += (static_cast<int64_t>(slab) * p.n_cols + col0) * ldb;
    } else {
      ldb = p.n_cols;
      b += static_cast<int64_t>(slab) * p.red * ldb + col0;
    }
  }
  const int64_t a_step = kA ? TK : static_cast<int64_t>(TK) * lda;
  const int64_t b_step = kB ? TK : static_cast<int64_t>(TK) * ldb;

  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  float acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = 0.f;

  float4 av[2], bv[2];
  load_slice<T, kA>(a, lda, m_valid, red, av);
  load_slice<T, kB>(b, ldb, n_valid, red, bv);
  put_slice<kA>(As[0], av);
  put_slice<kB>(Bs[0], bv);
  __syncthreads();
  int buf = 0;
  for (int64_t k0 = 0; k0 < red; k0 += TK) {
    const bool more = k0 + TK < red;
    if (more) {
      a += a_step;
      b += b_step;
      load_slice<T, kA>(a, lda, m_valid, red - k0 - TK, av);
      load_slice<T, kB>(b, ldb, n_valid, red - k0 - TK, bv);
    }
#pragma unroll
    for (int k = 0; k < TK; ++k) {
      float ar[8], br[8];
      *reinterpret_cast<float4*>(ar) = *reinterpret_cast<const float4*>(&As[buf][k][ty * 4]);
      *reinterpret_cast<float4*>(ar + 4) = *reinterpret_cast<const float4*>(&As[buf][k][ty * 4 + 64]);
      *reinterpret_cast<float4*>(br) = *reinterpret_cast<const float4*>(&Bs[buf][k][tx * 4]);
      *reinterpret_cast<float4*>(br + 4) = *reinterpret_cast<const float4*>(&Bs[buf][k][tx * 4 + 64]);
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(ar[i], br[j], acc[i][j]);
    }
    if (more) {
      put_slice<kA>(As[buf ^ 1], av);
      put_slice<kB>(Bs[buf ^ 1], bv);
      __syncthreads();
      buf ^= 1;
    }
  }

  T* out = static_cast<T*>(p.out);
  if (MODE == MODE_TN) {
    if (p.gate_up == 0) {
      out += (static_cast<int64_t>(slab) * p.m_cols + static_cast<int64_t>(blockIdx.x) * TM) * p.n_cols;
    } else {
      // a tile is one 128-row block of the packed order: even blocks are gate rows, odd ones the matching up rows
      if (blockIdx.x & 1) out = static_cast<T*>(p.out_up);
      const int r0 = static_cast<int>(blockIdx.x >> 1) * TM;
      out += (static_cast<int64_t>(slab) * p.gate_up + r0) * p.n_cols;
      m_valid = p.gate_up - r0;
    }
  } else {
    out += static_cast<int64_t>(row0) * p.n_cols;
  }
  out += col0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = ty * 4 + (i & 3) + (i >> 2) * 64;
    if (r >= m_valid) continue;
    T* o = out + static_cast<int64_t>(r) * p.n_cols;
    if (tx * 4 < n_valid) store4(o + tx * 4, acc[i]);
    if (tx * 4 + 64 < n_valid) store4(o + tx * 4 + 64, acc[i] + 4);
  }
}

template <int MODE>
int launch_simt(const SimtParams& p, int64_t gx, int dtype, cudaStream_t s) {
  const int64_t gy = (static_cast<int64_t>(p.n_cols) + TN - 1) / TN;
  if (gx > 0x7fffffffLL || gy > 65535) return DICE_ERR_LIMIT;
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy), MODE == MODE_TN ? p.n_slabs : 1);
  const cudaError_t err = dtype == DICE_F32
                              ? dice_launch(simt_grouped_kernel<float, MODE>, grid, dim3(256), 0, s, p)
                              : dice_launch(simt_grouped_kernel<__nv_bfloat16, MODE>, grid, dim3(256), 0, s, p);
  return err == cudaSuccess ? DICE_OK : DICE_ERR_CUDA;
}

}  // namespace

int dice_internal_simt_linear(const void* a, int64_t n_rows, int k_dim, const void* w, int n_slabs, int n_dim,
                              const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, int dtype, void* out,
                              uint32_t* status, cudaStream_t s) {
  SimtParams p = {a, w, out, nullptr, seg_offsets, seg_slab, n_seg, n_slabs, n_rows, 0, n_dim, k_dim, 0, status};
  return launch_simt<MODE_NT>(p, (n_rows + TM - 1) / TM + n_seg, dtype, s);
}

int dice_internal_simt_dgrad(const void* dy, int64_t n_rows, int n_dim, const void* w, int n_slabs, int k_dim,
                             const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, int dtype, void* dx,
                             uint32_t* status, cudaStream_t s) {
  SimtParams p = {dy, w, dx, nullptr, seg_offsets, seg_slab, n_seg, n_slabs, n_rows, 0, k_dim, n_dim, 0, status};
  return launch_simt<MODE_NN>(p, (n_rows + TM - 1) / TM + n_seg, dtype, s);
}

int dice_internal_simt_wgrad(const void* dy, const void* x, int64_t n_rows, int n_dim, int k_dim,
                             const int32_t* seg_offsets, int n_slabs, int gate_up, int dtype, void* dw, void* dw_up,
                             uint32_t* status, cudaStream_t s) {
  SimtParams p = {dy, x, dw, dw_up, seg_offsets, nullptr, n_slabs, n_slabs, n_rows, n_dim, k_dim, 0, gate_up, status};
  return launch_simt<MODE_TN>(p, (n_dim + TM - 1) / TM, dtype, s);
}
