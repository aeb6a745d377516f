// Products grouped by expert on the CUDA cores, for the training step's fp32 form where few rows meet a weight (from 96
// rows a slab on, train_gemm.cu makes six tensor-core products of it), in its three directions:
//
//   NT  out[r, n] = sum_k a[r, k] w[seg(r)][n, k]        the forward product (nn.Linear weights)
//   NN  dx[r, k]  = sum_n dy[r, n] w[seg(r)][n, k]       its input gradient
//   TN  dw[s][n, k] = sum_{r in seg s} dy[r, n] x[r, k]  its weight gradient
//
// Bound: the fp32 pipe (74 TFLOP/s nominal; measured 50 for NT and NN and 59.5 for TN at 4096^3, 33 and 47 at 1024 rows
// through 8 experts, 4608 x 1152, where a fifth of the rows that the tiles hold do not exist).  Every thread holds 8 x 8 sums and multiplies with two-wide fused
// multiply-adds, which leaves issue slots to the shared-memory reads; the next two slices of the operands are copied
// into shared memory asynchronously while the present one is multiplied (staging one slice in registers instead left
// the pipe idle a third of the time).  An operand whose reduction index is contiguous is transposed on its way, four
// bytes a copy.  Segments are ragged, and each CTA finds its own on the device.
//
// NT and NN have few rows in a segment and a long reduction: 64 x 64 tiles (an expert with 130 rows fills 3 of them
// to 68 %, but 2 tiles of 128 rows to 51 %), and a CTA's four groups of 64 threads each sum every fourth slice of the
// reduction, added up in shared memory at the end (1024 rows through 8 experts, 4608 -> 1152: 180 tiles alone would
// leave most of the GPU's warp slots empty).  Where even that leaves slots empty or a nearly empty last wave, the 2 to 8
// CTAs of a cluster share a tile's reduction in the same way and the first adds up what the others hold in shared
// memory.  The order of all these sums is fixed.  A tile with at most 12 rows (single tokens) is bounded by reading the
// weights: its CTA forgoes the tiling and streams them, every value used for the rows there are.  TN has many tiles and a short reduction: 128 x 128 tiles, one group.
#include "train.cuh"
#include "umma.cuh"  // sm_count_cached

namespace {

constexpr int WM = 128, WN = 128, WK = 16;           // TN: tile and slice
constexpr int TM = 64, TN = 64, TK = 8, GROUPS = 4;  // NT, NN: tile, slice, groups that share the reduction
enum { MODE_NT = 0, MODE_NN = 1 };

static_assert(TK == 8, "sizes are multiples of 8, so a reduction is a whole number of slices");
constexpr int kRing = 3;  // slices in shared memory: one being multiplied, two on their way

// asynchronous copy of BYTES (4 or 16); zeros where !ok (nothing is read then)
template <int BYTES>
__device__ __forceinline__ void copy_async(float* dst, const float* src, bool ok) {
  const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(ok ? 16 : 0) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory"); }
__device__ __forceinline__ void store4(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}


// 8 x 8 sums of one slice: rows ra .. ra+3 and ra+STEP .. of A (HALF: the first four only), columns likewise of B
template <int DEPTH, int WIDTH, int STEP, bool HALF = false>
__device__ __forceinline__ void multiply(const float (*As)[WIDTH + 4], const float (*Bs)[WIDTH + 4], int ra, int cb,
                                         f32x2 (&acc)[8][4]) {
#pragma unroll
  for (int k = 0; k < DEPTH; ++k) {
    float ar[8];
    f32x2 br[4];
    *reinterpret_cast<float4*>(ar) = *reinterpret_cast<const float4*>(&As[k][ra]);
    if (!HALF) *reinterpret_cast<float4*>(ar + 4) = *reinterpret_cast<const float4*>(&As[k][ra + STEP]);
    *reinterpret_cast<ulonglong2*>(br) = *reinterpret_cast<const ulonglong2*>(&Bs[k][cb]);
    *reinterpret_cast<ulonglong2*>(br + 2) = *reinterpret_cast<const ulonglong2*>(&Bs[k][cb + STEP]);
#pragma unroll
    for (int i = 0; i < (HALF ? 4 : 8); ++i) {
      const f32x2 a2 = both<f32x2>(ar[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = fma2(a2, br[j], acc[i][j]);
    }
  }
}
__device__ __forceinline__ void store_tile_row(float* o, const f32x2 (&acc)[4], int c0, int step, int n_valid) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c = c0 + h * step;
    if (c < n_valid) {
      const two lo = halves(acc[2 * h]), hi = halves(acc[2 * h + 1]);
      const float v[4] = {lo.x, lo.y, hi.x, hi.y};
      store4(o + c, v);
    }
  }
}

// One thread's share of a group's 64 x 8 operand slice.  KMAJOR: the reduction index is contiguous in memory
// ([mn][k]); eight lanes copy a row's eight elements (one 32-byte sector), into eight banks.  Else ([k][mn]).  Rows and
// columns that do not exist repeat the last one that does (their sums are not stored); the reduction is a whole number of
// slices (sizes are multiples of 8), so nothing needs a zero.
template <bool KMAJOR>
__device__ __forceinline__ void copy_slice(float (*s)[TM + 4], const float* base, int ld, int mn_valid, int t) {
  if (KMAJOR) {
    const int k = t & 7, r = t >> 3;
#pragma unroll
    for (int h = 0; h < 8; ++h) {
      const int row = r + 8 * h < mn_valid ? r + 8 * h : mn_valid - 1;
      copy_async<4>(&s[k][r + 8 * h], base + static_cast<uint32_t>(row) * static_cast<uint32_t>(ld) + k, true);
    }
  } else {
    const int k = t >> 4, c = (t & 15) * 4, col = c < mn_valid ? c : mn_valid - 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) copy_async<16>(&s[k + 4 * h][c], base + static_cast<int64_t>(k + 4 * h) * ld + col, true);
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
  int shares;      // TN: CTAs that share a tile
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The CTAs of a cluster that share a tile: the first adds the others' 8 x 8 sums to its own, in their order, out of their
// shared memory (32 pairs a thread, `step` apart from `place`).  Called by all threads; `active` ones hold sums.  True in
// the first CTA.
__device__ __forceinline__ bool cluster_total(f32x2 (&acc)[8][4], f32x2* place, int step, unsigned rank, unsigned size, bool active) {
  if (rank != 0 && active) {
#pragma unroll
    for (int i = 0; i < 32; ++i) place[i * step] = acc[i >> 2][i & 3];
  }
  cluster_sync();
  if (rank == 0 && active) {
    const uint32_t here = static_cast<uint32_t>(__cvta_generic_to_shared(place));
    for (uint32_t other = 1; other < size; ++other) {
      uint32_t there;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(other));
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        f32x2 y;
        asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(y) : "r"(there + i * step * 8));
        acc[i >> 2][i & 3] = add2(acc[i >> 2][i & 3], y);
      }
    }
  }
  cluster_sync();  // nobody leaves while its sums may be read
  return rank == 0;
}

struct Slices {
  float a[kRing][TK][TM + 4], b[kRing][TK][TN + 4];
};
constexpr int kRowsSmem = GROUPS * sizeof(Slices);
static_assert(kRowsSmem >= 2 * TM * TN * sizeof(float) && kRowsSmem >= (12 + 16 * 8) * TN * sizeof(float),
              "sums are exchanged in place of the slices");

// A tile of at most kThinRows rows: every thread sums over its own part of the reduction, straight from memory, and the
// parts are added in shared memory (`sums`, [ROWS][64] of them at its front at the end).  NN: 16 threads hold a weight
// row's 64 columns, 16 times four rows at once.  NT: a warp holds four weight rows (columns of the output), its lanes four
// elements of each.  Either way a value of the few rows is used for four of the weight's.
constexpr int kThinRows = 12;  // (8 slabs of 4608 x 1152: 4 rows 65 us, 12 rows 106, 16 rows 145; half a tile takes 129)
template <int MODE, int ROWS>
__device__ __forceinline__ void thin_tile(const float* a, int64_t lda, const float* w, int64_t ldb, int rows, int n_valid, int red,
                                          int share, int shares, float* sums) {
  float acc[ROWS][4] = {};
  if (MODE == MODE_NN) {
    const int c = (threadIdx.x & 15) * 4, n0 = static_cast<int>(threadIdx.x >> 4);
    if (c < n_valid) {
      for (int n = (share * 16 + n0) * 4; n < red; n += shares * 64) {  // (red is a multiple of 8)
        float4 x[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) x[q] = *reinterpret_cast<const float4*>(w + (n + q) * ldb + c);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          if (r < rows) {
            const float4 y = *reinterpret_cast<const float4*>(a + r * lda + n);
            const float ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              acc[r][0] = fmaf(ys[q], x[q].x, acc[r][0]);
              acc[r][1] = fmaf(ys[q], x[q].y, acc[r][1]);
              acc[r][2] = fmaf(ys[q], x[q].z, acc[r][2]);
              acc[r][3] = fmaf(ys[q], x[q].w, acc[r][3]);
            }
          }
        }
      }
    }
    // the 16 parts, a few rows at a time (all of 12 would not fit)
    constexpr int kRows = ROWS % 8 == 0 ? 8 : ROWS % 4 == 0 ? 4 : ROWS;
#pragma unroll
    for (int r0 = 0; r0 < ROWS; r0 += kRows) {
      float* part = sums + ROWS * TN;
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        *reinterpret_cast<float4*>(&part[(n0 * kRows + r) * TN + c]) = make_float4(acc[r0 + r][0], acc[r0 + r][1], acc[r0 + r][2], acc[r0 + r][3]);
      __syncthreads();
      for (int i = threadIdx.x; i < kRows * TN; i += 64 * GROUPS) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) t += part[k * kRows * TN + i];
        sums[r0 * TN + i] = t;
      }
      __syncthreads();
    }
  } else {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int c = warp * 4; c < n_valid; c += 8 * GROUPS) {  // (n_valid is a multiple of 8)
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[r][q] = 0.f;
      for (int k = (share * 32 + lane) * 4; k < red; k += shares * 128) {
        float4 x[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) x[q] = *reinterpret_cast<const float4*>(w + (c + q) * ldb + k);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          if (r < rows) {
            const float4 y = *reinterpret_cast<const float4*>(a + r * lda + k);
#pragma unroll
            for (int q = 0; q < 4; ++q)
              acc[r][q] = fmaf(y.x, x[q].x, fmaf(y.y, x[q].y, fmaf(y.z, x[q].z, fmaf(y.w, x[q].w, acc[r][q]))));
          }
        }
      }
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (r < rows) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            for (int off = 16; off > 0; off >>= 1) acc[r][q] += __shfl_xor_sync(0xffffffffu, acc[r][q], off);
          }
          if (lane == 0) *reinterpret_cast<float4*>(&sums[r * TN + c]) = make_float4(acc[r][0], acc[r][1], acc[r][2], acc[r][3]);
        }
      }
    }
    __syncthreads();
  }
}

template <int MODE>
__global__ void __launch_bounds__(64 * GROUPS, 2) simt_rows_kernel(const SimtParams p) {
  constexpr bool kB = MODE == MODE_NT;  // B has the reduction contiguous (A always has)
  extern __shared__ __align__(16) uint8_t smem_rows[];
  Slices* slices = reinterpret_cast<Slices*>(smem_rows);
  __shared__ int s_slab, s_row0, s_rows;
  pdl_trigger();
  pdl_wait();
  if (threadIdx.x == 0) {
    int slab = -1, row0 = 0, rows = 0, run = 0;
    bool ok = true, found = false;
    for (int s = 0; s < p.n_seg && !found && ok; ++s) {
      const int beg = p.seg_offsets[s], end = p.seg_offsets[s + 1];
      ok = beg >= 0 && end >= beg && end <= p.n_rows;
      const int nb = ok ? (end - beg + TM - 1) / TM : 0;
      if (static_cast<int>(blockIdx.x) < run + nb) {
        found = true;
        slab = p.seg_slab != nullptr ? p.seg_slab[s] : s;  // -1: rows of no expert
        row0 = beg + (static_cast<int>(blockIdx.x) - run) * TM;
        rows = end - row0;
        ok = slab < p.n_slabs;
      }
      run += nb;
    }
    if (!ok) {
      slab = -1;
      if (p.status != nullptr) atomicCAS(p.status, 0u, DICE_STATUS_BAD_SEGMENTS);
    }
    s_slab = slab; s_row0 = row0; s_rows = rows;
  }
  __syncthreads();
  if (s_slab < 0) return;
  const int row0 = s_row0, m_valid = s_rows < TM ? s_rows : TM;
  const int col0 = blockIdx.y * TN, n_valid = p.n_cols - col0 < TN ? p.n_cols - col0 : TN;
  const int group = threadIdx.x >> 6, t = threadIdx.x & 63;
  const int ra = (t >> 3) * 4, cb = (t & 7) * 4;

  const int64_t lda = p.red, ldb = kB ? p.red : p.n_cols;
  const float* a = static_cast<const float*>(p.a) + static_cast<int64_t>(row0) * lda;
  const float* b = static_cast<const float*>(p.b) + (kB ? (static_cast<int64_t>(s_slab) * p.n_cols + col0) * ldb
                                               : static_cast<int64_t>(s_slab) * p.red * ldb + col0);
  if (m_valid <= kThinRows) {
    float* sums = reinterpret_cast<float*>(slices);
    if (m_valid <= 2) thin_tile<MODE, 2>(a, lda, b, ldb, m_valid, n_valid, p.red, blockIdx.z, gridDim.z, sums);
    else if (m_valid <= 8) thin_tile<MODE, 8>(a, lda, b, ldb, m_valid, n_valid, p.red, blockIdx.z, gridDim.z, sums);
    else thin_tile<MODE, kThinRows>(a, lda, b, ldb, m_valid, n_valid, p.red, blockIdx.z, gridDim.z, sums);
    if (gridDim.z > 1) cluster_sync();
    if (blockIdx.z == 0) {
      float* out = static_cast<float*>(p.out) + static_cast<int64_t>(row0) * p.n_cols + col0;
      for (int i = threadIdx.x; i < m_valid * TN; i += 64 * GROUPS) {
        float t = sums[i];
        const uint32_t here = static_cast<uint32_t>(__cvta_generic_to_shared(sums + i));
        for (uint32_t other = 1; other < gridDim.z; ++other) {
          uint32_t there;
          float y;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(other));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(y) : "r"(there));
          t += y;
        }
        if (i % TN < n_valid) out[static_cast<int64_t>(i / TN) * p.n_cols + i % TN] = t;
      }
    }
    if (gridDim.z > 1) cluster_sync();
    return;
  }
  const int64_t b_slice = kB ? TK : static_cast<int64_t>(TK) * ldb;
  const int sharing = GROUPS * static_cast<int>(gridDim.z), share = static_cast<int>(blockIdx.z) * GROUPS + group;
  a += static_cast<int64_t>(share) * TK;
  b += share * b_slice;
  int64_t left = static_cast<int64_t>(p.red) - share * TK;  // of the reduction, from this group's slice on

  f32x2 acc[8][4] = {};
  Slices& mine = slices[group];
  auto fetch = [&](int buf) {
    if (left > 0) {
      copy_slice<true>(mine.a[buf], a, p.red, m_valid, t);
      copy_slice<kB>(mine.b[buf], b, kB ? p.red : p.n_cols, n_valid, t);
      a += sharing * TK;
      b += sharing * b_slice;
      left -= sharing * TK;
    }
    copies_commit();
  };
  int todo = left > 0 ? static_cast<int>((left + sharing * TK - 1) / (sharing * TK)) : 0;
  fetch(0);
  fetch(1);
  for (int buf = 0; todo > 0; --todo) {
    copies_wait();
    asm volatile("bar.sync %0, 64;" ::"r"(group + 1) : "memory");  // the slice is there, the one before it is done with
    fetch(buf == 0 ? kRing - 1 : buf - 1);
    if (m_valid > TM / 2) multiply<TK, TM, 32>(mine.a[buf], mine.b[buf], ra, cb, acc);
    else multiply<TK, TM, 32, true>(mine.a[buf], mine.b[buf], ra, cb, acc);  // (32 rows a slab: 152 -> 129 us)
    buf = buf == kRing - 1 ? 0 : buf + 1;
  }

  // groups 2 and 3 hand their sums to 0 and 1, then 1 to 0
  f32x2* sums = reinterpret_cast<f32x2*>(slices);
#pragma unroll
  for (int half = GROUPS / 2; half >= 1; half >>= 1) {
    __syncthreads();
    if (group >= half && group < 2 * half) {
#pragma unroll
      for (int i = 0; i < 32; ++i) sums[(group - half) * (TM * TN / 2) + i * 64 + t] = acc[i >> 2][i & 3];
    }
    __syncthreads();
    if (group < half) {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        acc[i >> 2][i & 3] = add2(acc[i >> 2][i & 3], sums[group * (TM * TN / 2) + i * 64 + t]);
      }
    }
  }
  if (gridDim.z > 1) {
    if (blockIdx.z != 0) __syncthreads();  // (their last exchange in the same place)
    if (!cluster_total(acc, sums + t, 64, blockIdx.z, gridDim.z, group == 0)) return;
  }
  if (group != 0) return;
  float* out = static_cast<float*>(p.out) + static_cast<int64_t>(row0) * p.n_cols + col0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = ra + (i & 3) + (i >> 2) * 32;
    if (r < m_valid) store_tile_row(out + static_cast<int64_t>(r) * p.n_cols, acc[i], cb, 32, n_valid);
  }
}

// one thread's share of a 128 x 16 slice: columns c .. c+3 and c+64 .. c+67 of one reduction row
__device__ __forceinline__ void copy_wide(float (*s)[WM + 4], const float* base, int64_t ld, int mn_valid, int k_valid) {
  const int k = threadIdx.x >> 4, c = (threadIdx.x & 15) * 4;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const bool ok = k < k_valid && c + 64 * h < mn_valid;
    copy_async<16>(&s[k][c + 64 * h], ok ? base + static_cast<int64_t>(k) * ld + c + 64 * h : base, ok);
  }
}

struct WideSlices {
  float a[kRing][WK][WM + 4], b[kRing][WK][WN + 4];
};
constexpr int kWideSmem = sizeof(WideSlices) > WM * WN * sizeof(float) ? sizeof(WideSlices) : WM * WN * sizeof(float);

__global__ void __launch_bounds__(256, 2) simt_wgrad_kernel(const SimtParams p) {
  extern __shared__ __align__(16) uint8_t smem_wide[];
  WideSlices& sl = *reinterpret_cast<WideSlices*>(smem_wide);
  pdl_trigger();
  pdl_wait();
  const int slab = blockIdx.z;
  const int row0 = p.seg_offsets[slab], end = p.seg_offsets[slab + 1];
  if (row0 < 0 || end < row0 || end > p.n_rows) {
    if (threadIdx.x == 0 && p.status != nullptr) atomicCAS(p.status, 0u, DICE_STATUS_BAD_SEGMENTS);
    return;
  }
  // the CTAs of a cluster take every shares-th slice of the reduction
  const int shares = p.shares, share = static_cast<int>(blockIdx.x) % shares, block = static_cast<int>(blockIdx.x) / shares;
  const int m0 = block * WM, col0 = blockIdx.y * WN;
  const int n_valid = p.n_cols - col0;
  int m_valid = p.m_cols - m0;
  const float* a = static_cast<const float*>(p.a) + static_cast<int64_t>(row0) * p.m_cols + m0;
  const float* b = static_cast<const float*>(p.b) + static_cast<int64_t>(row0) * p.n_cols + col0;
  int left = end - row0 - share * WK;
  a += static_cast<int64_t>(share) * WK * p.m_cols;
  b += static_cast<int64_t>(share) * WK * p.n_cols;

  const int ra = (threadIdx.x >> 4) * 4, cb = (threadIdx.x & 15) * 4;
  f32x2 acc[8][4] = {};
  auto fetch = [&](int buf) {
    if (left > 0) {
      copy_wide(sl.a[buf], a, p.m_cols, m_valid, left);
      copy_wide(sl.b[buf], b, p.n_cols, n_valid, left);
      a += static_cast<int64_t>(shares) * WK * p.m_cols;
      b += static_cast<int64_t>(shares) * WK * p.n_cols;
      left -= shares * WK;
    }
    copies_commit();
  };
  int todo = left > 0 ? (left + shares * WK - 1) / (shares * WK) : 0;
  fetch(0);
  fetch(1);
  for (int buf = 0; todo > 0; --todo) {
    copies_wait();
    __syncthreads();  // the slice is there, the one before it is done with
    fetch(buf == 0 ? kRing - 1 : buf - 1);
    multiply<WK, WM, 64>(sl.a[buf], sl.b[buf], ra, cb, acc);
    buf = buf == kRing - 1 ? 0 : buf + 1;
  }

  if (shares > 1) {
    __syncthreads();  // the slices are done with
    if (!cluster_total(acc, reinterpret_cast<f32x2*>(smem_wide) + threadIdx.x, 256, share, shares, true)) return;
  }

  float* out = static_cast<float*>(p.out);
  if (p.gate_up == 0) {
    out += (static_cast<int64_t>(slab) * p.m_cols + m0) * p.n_cols + col0;
  } else {
    // a tile is one 128-row block of the packed order: even blocks are gate rows, odd ones the matching up rows
    if (block & 1) out = static_cast<float*>(p.out_up);
    const int r0 = (block >> 1) * WM;
    out += (static_cast<int64_t>(slab) * p.gate_up + r0) * p.n_cols + col0;
    m_valid = p.gate_up - r0;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = ra + (i & 3) + (i >> 2) * 64;
    if (r < m_valid) store_tile_row(out + static_cast<int64_t>(r) * p.n_cols, acc[i], cb, 64, n_valid);
  }
}

// ---- values of a product by planes that are not finite ------------------------------------
// An fp32 product on the tensor cores is made of products of bf16 planes, among which an infinity meets zeros (inf * 0) and
// large finite values may overflow to infinities of both signs: NaN where the sum of the products themselves is an infinity,
// or even a number.  If the product's epilogues saw a value that is not finite, every 64 x 64 tile that holds one is
// multiplied again from the operands, one fused multiply-add after the other, and those values alone are replaced: the
// others keep their bits, whatever their neighbours hold.  Without such a value this launch reads one word (2 to 3 us
// of a product's 25 and more: 8 x 128 rows, 4608 x 1152, weight gradient 93 -> 95 us); with one, the time of its tiles at some 10 TFLOP/s is of no account.
struct RepairParams {
  const float* a;
  const float* b;
  float* out;
  float* out_up;
  const int* seg_offsets;
  const int* seg_slab;
  const unsigned int* non_finite;
  int64_t n_rows, a_row, a_red, b_col, b_red, b_slab;  // distances: rows and reduction of a, columns and reduction of b, slabs of b
  int n_seg, n_slabs, m_cols, n_cols, red, gate_up;
  bool wgrad;
};
constexpr int RT = 64, RK = 16;

__global__ void __launch_bounds__(256) f32_repair_kernel(const RepairParams p) {
  __shared__ float as[RK][RT + 1], bs[RK][RT + 1];
  __shared__ int s_seg, s_row0, s_rows;
  pdl_trigger();
  pdl_wait();
  if (*p.non_finite == 0u) return;
  const int64_t col_tiles = (static_cast<int64_t>(p.n_cols) + RT - 1) / RT, m_tiles = (p.m_cols + RT - 1) / RT;
  for (int64_t t = blockIdx.x;; t += gridDim.x) {
    const int64_t m_tile = t / col_tiles;
    const int col0 = static_cast<int>(t - m_tile * col_tiles) * RT;
    if (p.wgrad) {
      if (m_tile >= m_tiles * p.n_slabs) return;
    } else {
      __syncthreads();
      if (threadIdx.x == 0) {
        int64_t run = 0;
        s_seg = -1;
        for (int s = 0; s < p.n_seg && s_seg < 0; ++s) {
          const int beg = p.seg_offsets[s], end = p.seg_offsets[s + 1];
          if (beg < 0 || end < beg || end > p.n_rows) break;  // (a product of such segments was not made)
          const int64_t tiles = (static_cast<int64_t>(end) - beg + RT - 1) / RT;
          if (m_tile < run + tiles) {
            s_seg = s;
            s_row0 = beg + static_cast<int>(m_tile - run) * RT;
            s_rows = end - s_row0;
          }
          run += tiles;
        }
      }
      __syncthreads();
      if (s_seg < 0) return;
    }
    // the tile's operands, and the place of its first value
    const int seg = p.wgrad ? static_cast<int>(m_tile / m_tiles) : s_seg;
    const int slab = !p.wgrad && p.seg_slab != nullptr ? p.seg_slab[seg] : seg;
    if (slab < 0 || slab >= p.n_slabs) continue;  // rows of no expert
    int m0, m_valid, red = p.red;
    const float* a = p.a;
    const float* b = p.b + slab * p.b_slab + col0 * p.b_col;
    float* out = p.out;
    if (p.wgrad) {
      m0 = static_cast<int>(m_tile - seg * m_tiles) * RT;
      m_valid = p.m_cols - m0;
      const int beg = p.seg_offsets[seg], end = p.seg_offsets[seg + 1];
      if (beg < 0 || end < beg || end > p.n_rows) return;
      red = end - beg;
      a += m0 * p.a_row + beg * p.a_red;
      b = p.b + beg * p.b_red + col0 * p.b_col;
      if (p.gate_up == 0) {
        out += (static_cast<int64_t>(slab) * p.m_cols + m0) * p.n_cols + col0;
      } else {  // 128 rows of gate, 128 of up in turn: a tile is half of one of them
        const int r0 = m0 / 256 * 128 + m0 % 128;
        if (m0 & 128) out = p.out_up;
        out += (static_cast<int64_t>(slab) * p.gate_up + r0) * p.n_cols + col0;
        m_valid = p.gate_up - r0;
      }
    } else {
      m0 = s_row0;
      m_valid = s_rows;
      a += m0 * p.a_row;
      out += static_cast<int64_t>(m0) * p.n_cols + col0;
    }
    m_valid = m_valid < RT ? m_valid : RT;
    const int n_valid = p.n_cols - col0 < RT ? p.n_cols - col0 : RT;
    const int r0 = static_cast<int>(threadIdx.x >> 4) * 4, c0 = static_cast<int>(threadIdx.x & 15) * 4;
    unsigned again = 0;  // which of this thread's 4 x 4 values
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = r0 + (i >> 2), c = c0 + (i & 3);
      if (r < m_valid && c < n_valid && !isfinite(out[static_cast<int64_t>(r) * p.n_cols + c])) again |= 1u << i;
    }
    if (!__syncthreads_or(again != 0)) continue;
    float acc[16] = {};
    for (int k0 = 0; k0 < red; k0 += RK) {
      __syncthreads();
      for (int i = threadIdx.x; i < RK * RT; i += 256) {
        const int k = i / RT, m = i % RT;
        const bool in = k0 + k < red;
        as[k][m] = in && m < m_valid ? a[m * p.a_row + (k0 + k) * p.a_red] : 0.f;
        bs[k][m] = in && m < n_valid ? b[m * p.b_col + (k0 + k) * p.b_red] : 0.f;
      }
      __syncthreads();
      const int depth = red - k0 < RK ? red - k0 : RK;
      for (int k = 0; k < depth; ++k) {
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = fmaf(as[k][r0 + (i >> 2)], bs[k][c0 + (i & 3)], acc[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (again >> i & 1) out[static_cast<int64_t>(r0 + (i >> 2)) * p.n_cols + c0 + (i & 3)] = acc[i];
  }
}

// both kernels use more shared memory than the default limit; set once per device and kernel
template <typename K>
bool allow_smem(K kernel, int bytes, bool (&done)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (!done[dev]) done[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
  return done[dev];
}

int launch_cluster(void (*kernel)(SimtParams), dim3 grid, int threads, int smem, dim3 cluster, const SimtParams& p, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster.x;
  attr[0].val.clusterDim.y = cluster.y;
  attr[0].val.clusterDim.z = cluster.z;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dice_pdl_enabled() ? 2 : 1;
  dice_count_launch();
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? DICE_OK : DICE_ERR_CUDA;
}

// CTAs that share a tile's reduction: as many (a power of two, at most 8) as give every one of the GPU's CTA slots five
// tiles, while each of a CTA's groups keeps at least four slices.  Measured without / with sharing: 11 rows in 3 of 4
// experts, 4608 -> 1152: 161 / 76 us; 1024 rows through 8 experts, the whole FFN step: 1782 / 1674 us.  Rows are counted
// as if every segment filled half a tile more than it has.
int shares_of(const SimtParams& p, int64_t col_tiles) {
  const int64_t tiles = (p.n_rows / TM + (p.n_seg + 1) / 2 + 1) * col_tiles, slots = 2ll * dice_umma::sm_count_cached();
  int shares = 1;
  while (shares < 8 && tiles * shares < 5 * slots && p.red >= 2 * shares * GROUPS * TK * 4) shares *= 2;
  return shares;
}

template <int MODE>
int launch_rows(const SimtParams& p, cudaStream_t s) {
  const int64_t gx = (p.n_rows + TM - 1) / TM + p.n_seg, gy = (static_cast<int64_t>(p.n_cols) + TN - 1) / TN;
  if (gx > 0x7fffffffLL || gy > 65535) return DICE_ERR_LIMIT;
  static bool done[64];
  if (!allow_smem(simt_rows_kernel<MODE>, kRowsSmem, done)) return DICE_ERR_CUDA;
  const unsigned shares = static_cast<unsigned>(shares_of(p, gy));
  return launch_cluster(simt_rows_kernel<MODE>, dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy), shares), 64 * GROUPS,
                        kRowsSmem, dim3(1, 1, shares), p, s);
}

}  // namespace

int dice_internal_simt_linear(const void* a, int64_t n_rows, int k_dim, const void* w, int n_slabs, int n_dim,
                              const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, void* out,
                              uint32_t* status, cudaStream_t s) {
  SimtParams p = {a, w, out, nullptr, seg_offsets, seg_slab, n_seg, n_slabs, n_rows, 0, n_dim, k_dim, 0, status};
  return launch_rows<MODE_NT>(p, s);
}

int dice_internal_simt_dgrad(const void* dy, int64_t n_rows, int n_dim, const void* w, int n_slabs, int k_dim,
                             const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, void* dx,
                             uint32_t* status, cudaStream_t s) {
  SimtParams p = {dy, w, dx, nullptr, seg_offsets, seg_slab, n_seg, n_slabs, n_rows, 0, k_dim, n_dim, 0, status};
  return launch_rows<MODE_NN>(p, s);
}

int dice_internal_simt_wgrad(const void* dy, const void* x, int64_t n_rows, int n_dim, int k_dim,
                             const int32_t* seg_offsets, int n_slabs, int gate_up, void* dw, void* dw_up,
                             uint32_t* status, cudaStream_t s) {
  SimtParams p = {dy, x, dw, dw_up, seg_offsets, nullptr, n_slabs, n_slabs, n_rows, n_dim, k_dim, 0, gate_up, status};
  const int64_t gm = (static_cast<int64_t>(n_dim) + WM - 1) / WM, gy = (static_cast<int64_t>(k_dim) + WN - 1) / WN;
  if (gy > 65535) return DICE_ERR_LIMIT;
  // as many CTAs to a tile (a power of two, at most 8) as fill the GPU's slots once, each with eight slices or more of an
  // average segment
  const int64_t tiles = gm * gy * n_slabs, slots = 2ll * dice_umma::sm_count_cached();
  p.shares = 1;
  while (p.shares < 8 && 2 * p.shares * tiles <= slots && n_rows >= 16ll * p.shares * WK * n_slabs) p.shares *= 2;
  static bool done[64];
  if (!allow_smem(simt_wgrad_kernel, kWideSmem, done)) return DICE_ERR_CUDA;
  return launch_cluster(simt_wgrad_kernel, dim3(static_cast<unsigned>(gm * p.shares), static_cast<unsigned>(gy), static_cast<unsigned>(n_slabs)),
                        256, kWideSmem, dim3(p.shares, 1, 1), p, s);
}

int dice_internal_f32_repair(int kind, const void* a, const void* b, int64_t n_rows, int n_dim, int k_dim, int n_slabs,
                             const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, int gate_up, void* out,
                             void* out_up, const unsigned int* non_finite, cudaStream_t s) {
  RepairParams p = {};
  p.a = static_cast<const float*>(a);
  p.b = static_cast<const float*>(b);
  p.out = static_cast<float*>(out);
  p.out_up = static_cast<float*>(out_up);
  p.seg_offsets = seg_offsets;
  p.seg_slab = seg_slab;
  p.non_finite = non_finite;
  p.n_rows = n_rows;
  p.n_seg = n_seg;
  p.n_slabs = n_slabs;
  p.gate_up = gate_up;
  if (kind == DICE_PRODUCT_WGRAD) {  // a = dy, b = x: rows are the reduction
    p.wgrad = true;
    p.m_cols = n_dim;
    p.n_cols = k_dim;
    p.a_row = p.b_col = 1;
    p.a_red = n_dim;
    p.b_red = k_dim;
  } else {
    const bool linear = kind == DICE_PRODUCT_LINEAR;
    p.n_cols = linear ? n_dim : k_dim;
    p.red = linear ? k_dim : n_dim;
    p.a_row = p.red;
    p.a_red = 1;
    p.b_col = linear ? k_dim : 1;  // w [n_dim, k_dim]
    p.b_red = linear ? 1 : k_dim;
    p.b_slab = static_cast<int64_t>(n_dim) * k_dim;
  }
  const int sms = dice_umma::sm_count_cached();
  if (sms <= 0) return DICE_ERR_CUDA;
  return dice_launch(f32_repair_kernel, dim3(static_cast<unsigned>(2 * sms)), dim3(256), 0, s, p) == cudaSuccess ? DICE_OK : DICE_ERR_CUDA;
}
