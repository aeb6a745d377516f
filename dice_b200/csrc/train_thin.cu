// Input gradient of a product grouped by expert for a handful of bf16 rows (single tokens, at most kThinTotal rows in all):
//   dx[r, k] = sum_n dy[r, n] w[seg(r)][n, k]
//
// Bound: reading the weights of the experts that have rows, 21 MB for one token's two rows at 1152 -> 4608. The
// tensor-core kernel needs tensor memory, barriers, two tensor maps and a chain of dependent k-blocks for what is a
// matrix-vector product: 12.0 us a call, against 8.9 here (of which the
// host needs 8). From five rows on it is the faster one (8 rows of one expert 11.0 us). A CTA streams 128 columns: 16 threads hold a weight
// row's piece (8 columns, 16 bytes each), 16 times four rows at once, and use every value for the up to 2 rows of the
// tile; sums are fp32. Threads' parts are added in shared memory, and the CTAs of a cluster that share the reduction add
// theirs in the first one's registers, in a fixed order.
#include "train.cuh"
#include "umma.cuh"  // sm_count_cached

namespace {

constexpr int kRows = 2, kCols = 128, kJoinRows = 2;  // rows of a tile, its columns, rows whose parts are joined at a time

struct ThinParams {
  const __nv_bfloat16* dy;
  const __nv_bfloat16* w;
  __nv_bfloat16* dx;
  const int* seg_offsets;
  const int* seg_slab;
  int n_seg, n_slabs, n_rows, n_dim, k_dim;
  uint32_t* status;
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__global__ void __launch_bounds__(256, 3) thin_dgrad_kernel(const ThinParams p) {
  __shared__ __align__(16) float sums[kRows * kCols];
  __shared__ __align__(16) float parts[16 * kJoinRows * kCols];
  __shared__ int s_slab, s_row0, s_rows;
  pdl_trigger();
  pdl_wait();
  if (threadIdx.x == 0) {
    int slab = -1, row0 = 0, rows = 0, run = 0;
    bool ok = true, found = false;
    for (int s = 0; s < p.n_seg && !found && ok; ++s) {
      const int beg = p.seg_offsets[s], end = p.seg_offsets[s + 1];
      ok = beg >= 0 && end >= beg && end <= p.n_rows;
      const int tiles = ok ? (end - beg + kRows - 1) / kRows : 0;
      if (static_cast<int>(blockIdx.x) < run + tiles) {
        found = true;
        slab = p.seg_slab != nullptr ? p.seg_slab[s] : s;  // -1: rows of no expert
        row0 = beg + (static_cast<int>(blockIdx.x) - run) * kRows;
        rows = end - row0 < kRows ? end - row0 : kRows;
        ok = slab < p.n_slabs;
      }
      run += tiles;
    }
    if (!ok) {
      slab = -1;
      if (p.status != nullptr) atomicCAS(p.status, 0u, DICE_STATUS_BAD_SEGMENTS);
    }
    s_slab = slab; s_row0 = row0; s_rows = rows;
  }
  __syncthreads();
  if (s_slab < 0) return;  // (all of a cluster: its CTAs have the same tile)
  const int rows = s_rows, col0 = blockIdx.y * kCols;
  const int c = (threadIdx.x & 15) * 8, n0 = static_cast<int>(threadIdx.x >> 4) * 4;
  const __nv_bfloat16* a = p.dy + static_cast<int64_t>(s_row0) * p.n_dim;
  const __nv_bfloat16* w = p.w + static_cast<int64_t>(s_slab) * p.n_dim * p.k_dim + col0 + c;

  f32x2 acc[kRows][4];
#pragma unroll
  for (int r = 0; r < kRows; ++r)
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[r][q] = 0;
  if (col0 + c < p.k_dim) {
#pragma unroll 2
    for (int n = blockIdx.z * 64 + n0; n < p.n_dim; n += static_cast<int>(gridDim.z) * 64) {  // (n_dim is a multiple of 8)
      uint4 x[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] = ldg_stream16(w + static_cast<int64_t>(n + q) * p.k_dim);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (r < rows) {
          const uint2 y2 = *reinterpret_cast<const uint2*>(a + static_cast<int64_t>(r) * p.n_dim + n);
          const float y[4] = {bf16lo_to_f32(y2.x), bf16hi_to_f32(y2.x), bf16lo_to_f32(y2.y), bf16hi_to_f32(y2.y)};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x2 yy = both<f32x2>(y[q]);
            acc[r][0] = fma2(yy, bf16_pair<f32x2>(x[q].x), acc[r][0]);
            acc[r][1] = fma2(yy, bf16_pair<f32x2>(x[q].y), acc[r][1]);
            acc[r][2] = fma2(yy, bf16_pair<f32x2>(x[q].z), acc[r][2]);
            acc[r][3] = fma2(yy, bf16_pair<f32x2>(x[q].w), acc[r][3]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int r0 = 0; r0 < kRows; r0 += kJoinRows) {
    if (r0 < rows) {
#pragma unroll
      for (int r = 0; r < kJoinRows; ++r) {
        float* at = parts + ((threadIdx.x >> 4) * kJoinRows + r) * kCols + c;
        *reinterpret_cast<ulonglong2*>(at) = make_ulonglong2(acc[r0 + r][0], acc[r0 + r][1]);
        *reinterpret_cast<ulonglong2*>(at + 4) = make_ulonglong2(acc[r0 + r][2], acc[r0 + r][3]);
      }
      __syncthreads();
      {  // 2 rows x 128 columns: one of them a thread
        const int i = threadIdx.x;
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) t += parts[k * kJoinRows * kCols + i];
        sums[r0 * kCols + i] = t;
      }
      __syncthreads();
    }
  }
  static_assert(kJoinRows * kCols == 256, "a value a thread");
  if (gridDim.z > 1) cluster_sync();
  if (blockIdx.z == 0) {
    for (int i = threadIdx.x * 2; i < rows * kCols; i += 512) {
      float t0 = sums[i], t1 = sums[i + 1];
      const uint32_t here = static_cast<uint32_t>(__cvta_generic_to_shared(sums + i));
      for (uint32_t other = 1; other < gridDim.z; ++other) {
        uint32_t there;
        float y0, y1;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(other));
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(y0), "=f"(y1) : "r"(there));
        t0 += y0;
        t1 += y1;
      }
      const int col = col0 + i % kCols;
      if (col < p.k_dim)
        *reinterpret_cast<uint32_t*>(p.dx + static_cast<int64_t>(s_row0 + i / kCols) * p.k_dim + col) = pack_bf16x2(t0, t1);
    }
  }
  if (gridDim.z > 1) cluster_sync();  // nobody leaves while its sums may be read
}

}  // namespace

int dice_internal_thin_dgrad(const void* dy, int64_t n_rows, int n_dim, const void* w, int n_slabs, int k_dim,
                             const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, void* dx, uint32_t* status,
                             cudaStream_t s) {
  const int64_t cols = (static_cast<int64_t>(k_dim) + kCols - 1) / kCols;
  if (cols > 65535) return DICE_ERR_LIMIT;
  ThinParams p = {static_cast<const __nv_bfloat16*>(dy), static_cast<const __nv_bfloat16*>(w), static_cast<__nv_bfloat16*>(dx),
                  seg_offsets, seg_slab, n_seg, n_slabs, static_cast<int>(n_rows), n_dim, k_dim, status};
  // as many CTAs to a tile's reduction (at most 8) as fill the GPU's slots about once, each with at least two rounds
  const int64_t slots = 3ll * dice_umma::sm_count_cached();
  unsigned shares = 1;
  while (shares < 8 && 2 * shares * n_rows * cols <= slots + slots / 4 && n_dim >= 256 * static_cast<int>(shares)) shares *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(n_rows), static_cast<unsigned>(cols), shares);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = shares;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dice_pdl_enabled() ? 2 : 1;
  dice_count_launch();
  return cudaLaunchKernelEx(&cfg, thin_dgrad_kernel, p) == cudaSuccess ? DICE_OK : DICE_ERR_CUDA;
}
