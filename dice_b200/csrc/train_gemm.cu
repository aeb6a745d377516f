// The gradients of the products grouped by expert on the tensor cores, with CTA pairs (tcgen05 cta_group::2):
//
//   NN  dx[r, k] = sum_n dy[r, n] w[slab][n, k]              input gradient: reduction over a slab's rows
//   TN  dw[s][n, k] = sum_{r in seg s} dy[r, n] x[r, k]      weight gradient: reduction over a segment's rows
//
// The pair computes a 256 x 256 tile as in grouped_gemm_pair.cu (each CTA brings 128 rows of A and half of the B
// columns, the leader issues, each CTA keeps 128 rows of the result).  What differs is the operands: where the
// reduction is not the contiguous dimension (w and x as B, dy as A of the weight gradient) the tile stays as it lies
// in memory, 64 reduction rows of 64 columns (128 bytes, 128-byte swizzle) per TMA box, and the matrix instruction
// reads it "MN-major"; nothing is transposed.
//
// A weight gradient's reduction is ragged.  Its last k-block may reach into the next segment (or behind the tensor, or
// into rows that hold anything): the instructions stop at the last 16 rows that the segment touches, and the up to
// 15 rows of those that are not the segment's are zeroed in shared memory, in both operands, since a zero in one
// would not silence a NaN in the other.  For such a block each CTA's copies complete on a barrier of its own; a warp
// waits there, zeroes, makes the zeros visible to the asynchronous proxy and completes the copies' bytes on the leader's
// "full" barrier in their place.  All other blocks go from the copies to the tensor cores directly.  (The leader expects
// both CTAs' bytes; a peer that announced its own with a cluster-scope arrival cost twice the time of a block.)
//
// Few tiles and a long reduction: the pairs that would idle take a share of the reduction each (split).  Every epilogue
// warp files its part of the sum in fp32; the last one to arrive at a part adds them up in the order of the shares, so
// the result does not depend on who was last.
#include <cuda.h>

#include "train.cuh"
#include "umma_pair.cuh"

using namespace dice_umma;

namespace {

enum { MODE_NN = 1, MODE_TN = 2 };

constexpr int PM = 256;
constexpr int kStagesT = 6;
constexpr int kStageBytesT = 32768;  // 128 rows (or columns) x 64 of each operand
constexpr int kOperandBytes = 16384;
constexpr int kBoxBytes = 8192;      // 64 reduction rows x 128 bytes
constexpr int kThreadsT = 352;       // warp 0 loader, 1 tensor-core issue, 2..9 epilogue, 10 ragged ends
constexpr int kStageStore = 2048;    // per epilogue warp, as in grouped_gemm_pair.cu
constexpr int kSmemT = kStagesT * kStageBytesT + kAuxBytes + kEpilogueWarps * kStageStore + 1024;
constexpr int kSplitFloats = 4 * 32 * 32;  // an epilogue warp's part of a tile: 4 chunks of 32 rows x 32 columns
constexpr int kMinSplitBlocks = 4;         // k-blocks of a share, at least

struct TrainGemm {
  const int* seg_offsets;
  const int* seg_slab;
  int n_seg, n_slabs;
  int n_rows;
  int red_blocks;   // NN: k-blocks of the reduction
  int n_mblk;       // TN: row tiles of a slab's gradient
  int n_nblk;       // column tiles
  int n_cols;       // output columns
  int m_rows;       // TN: output rows of a slab
  int gate_up;      // TN: 0, or ffn: the rows are packed gate / up blocks and go to two tensors
  __nv_bfloat16* out;
  __nv_bfloat16* out_up;
  float* split_ws;  // NULL: no split.  [pair][cta][epilogue warp][kSplitFloats]
  unsigned int* split_count;  // zero on entry: [tile][cta][epilogue warp]
  uint32_t* status;
};

// Shared-memory operand descriptor of an MN-major tile: boxes of 64 reduction rows x 128 bytes with the 128-byte
// swizzle; 8 reduction rows are 1024 bytes apart, the next 64 columns 8192.
__device__ __forceinline__ uint64_t make_mn_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(kBoxBytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}
// bytes of a ragged end accounted for on the leader's barrier, in the place of the copies (whose bytes the leader expects)
__device__ __forceinline__ void mbar_complete_tx_cluster(uint32_t cluster_addr, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cluster.shared::cluster.b64 [%0], %1;" ::"r"(cluster_addr), "r"(bytes) : "memory");
}
// orders the zeroing before that (release), and after it in the issuing warp (acquire)
__device__ __forceinline__ void fence_cluster() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <int MODE>
__global__ void __launch_bounds__(kThreadsT, 1)
train_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const TrainGemm p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* aux = smem + kStagesT * kStageBytesT;
  uint64_t* bars = reinterpret_cast<uint64_t*>(aux);
  const uint32_t full_bar = smem_u32(bars);                                 // [kStagesT] used in the leader
  const uint32_t empty_bar = smem_u32(bars + kStagesT);                     // [kStagesT] in both CTAs
  const uint32_t tail_bar = smem_u32(bars + 2 * kStagesT);                  // [kStagesT] in both CTAs (TN)
  const uint32_t acc_full_bar = smem_u32(bars + 3 * kStagesT);              // [kAccStages] in both CTAs
  const uint32_t acc_empty_bar = smem_u32(bars + 3 * kStagesT + kAccStages);  // used in the leader
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 3 * kStagesT + 2 * kAccStages);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  int* s_split = reinterpret_cast<int*>(tmem_slot + 2);
  int* s_seg_off = reinterpret_cast<int*>(tmem_slot + 4);
  int* s_mprefix = s_seg_off + (kMaxSeg + 1);  // NN: first row tile of every segment
  const uint32_t tiles_smem = smem_u32(smem);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta_rank = cluster_cta_rank();
  const bool leader = cta_rank == 0;
  const int64_t pair_id = blockIdx.x >> 1;
  const int64_t n_pairs = gridDim.x >> 1;

  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStagesT; ++s) {
      mbar_init(full_bar + 8 * s, 1);
      mbar_init(empty_bar + 8 * s, 1);
      mbar_init(tail_bar + 8 * s, 1);
    }
    for (int a = 0; a < kAccStages; ++a) {
      mbar_init(acc_full_bar + 8 * a, 1);
      mbar_init(acc_empty_bar + 8 * a, 2 * kEpilogueWarps);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc_pair(smem_u32(tmem_slot), kTmemCols);
  pdl_wait();

  for (int i = threadIdx.x; i <= p.n_seg; i += kThreadsT) s_seg_off[i] = p.seg_offsets[i];
  __syncthreads();
  if (threadIdx.x == 0) {
    int run = 0, most = 0;
    bool ok = s_seg_off[0] >= 0;
    for (int s = 0; s < p.n_seg; ++s) {
      const int cnt = s_seg_off[s + 1] - s_seg_off[s];
      // (the difference of two non-negative offsets does not overflow; a negative one is found first)
      ok = ok && s_seg_off[s + 1] >= 0 && cnt >= 0;
      s_mprefix[s] = run;
      bool has_weights = true;
      if (MODE == MODE_NN && p.seg_slab != nullptr) {
        has_weights = p.seg_slab[s] >= 0;  // slab -1: rows of no expert
        ok = ok && p.seg_slab[s] < p.n_slabs;
      }
      if (ok) {
        run += (cnt > 0 && has_weights) ? (cnt + PM - 1) / PM : 0;
        most = cnt > most ? cnt : most;
      }
    }
    ok = ok && s_seg_off[p.n_seg] <= p.n_rows;
    if (MODE == MODE_TN) run = p.n_seg * p.n_mblk;
    if (!ok) {
      run = 0;
      if (p.status != nullptr) atomicCAS(p.status, 0u, DICE_STATUS_BAD_SEGMENTS);
    }
    s_mprefix[p.n_seg] = run;
    // shares of the reduction: as many as there are pairs for every tile, if each is long enough
    int split = 1;
    if (p.split_ws != nullptr && run > 0) {
      const int64_t per_tile = n_pairs / (static_cast<int64_t>(run) * p.n_nblk);
      const int blocks = MODE == MODE_NN ? p.red_blocks : (most + BK - 1) / BK;
      split = static_cast<int>(per_tile < blocks / kMinSplitBlocks ? per_tile : blocks / kMinSplitBlocks);
      if (split < 1) split = 1;
    }
    *s_split = split;
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_barrier();
  tc_fence_after_sync();

  const uint32_t tmem_base = *tmem_slot;
  const int split = *s_split;
  const int64_t total = static_cast<int64_t>(s_mprefix[p.n_seg]) * p.n_nblk * split;

  // work item t -> tile, share of the reduction, this CTA's rows
  struct Tile {
    int64_t tile;
    int share, nb, mb, slab, row0, rows_valid, kb0, kb1, n_mma, last_rows;
    bool zero;  // TN: a segment without rows, whose gradient is written as zeros (by the first share)
  };
  auto decode = [&](int64_t t, int& seg) {
    Tile ti;
    ti.tile = split == 1 ? t : t / split;
    ti.share = split == 1 ? 0 : static_cast<int>(t - ti.tile * split);
    const int m = static_cast<int>(ti.tile / p.n_nblk);
    ti.nb = static_cast<int>(ti.tile - static_cast<int64_t>(m) * p.n_nblk);
    int blocks;
    if (MODE == MODE_NN) {
      while (m >= s_mprefix[seg + 1]) ++seg;
      ti.mb = m - s_mprefix[seg];
      ti.row0 = s_seg_off[seg] + ti.mb * PM + static_cast<int>(cta_rank) * BM;
      ti.rows_valid = s_seg_off[seg + 1] - ti.row0;
      ti.slab = p.seg_slab != nullptr ? p.seg_slab[seg] : seg;
      blocks = p.red_blocks;
      ti.last_rows = BK;
    } else {
      seg = m / p.n_mblk;
      ti.mb = m - seg * p.n_mblk;
      ti.slab = seg;
      ti.row0 = ti.mb * PM + static_cast<int>(cta_rank) * BM;  // of the gradient
      ti.rows_valid = p.m_rows - ti.row0;
      const int cnt = s_seg_off[seg + 1] - s_seg_off[seg];
      blocks = (cnt + BK - 1) / BK;
      ti.last_rows = cnt - (blocks - 1) * BK;
    }
    ti.zero = blocks == 0;
    ti.kb0 = static_cast<int>(static_cast<int64_t>(blocks) * ti.share / split);
    ti.kb1 = static_cast<int>(static_cast<int64_t>(blocks) * (ti.share + 1) / split);
    if (ti.kb1 < blocks) ti.last_rows = BK;
    int n_valid = p.n_cols - ti.nb * BN;
    if (n_valid > BN) n_valid = BN;
    ti.n_mma = (n_valid + 31) & ~31;  // half of the columns come from each CTA
    return ti;
  };

  if (warp == 0) {
    // ---------------- loader (both CTAs) ----------------
    int stage = 0, seg = 0;
    uint32_t phase = 0;
    bool alive = true;
    for (int64_t t = pair_id; alive && t < total; t += n_pairs) {
      const Tile ti = decode(t, seg);
      const int half = ti.n_mma / 2;
      const int col0 = ti.nb * BN + static_cast<int>(cta_rank) * half;  // this CTA's B columns
      const int b_boxes = half > 64 ? 2 : 1;
      const uint32_t bytes = kOperandBytes + b_boxes * kBoxBytes;
      const int ragged = MODE == MODE_TN ? ti.last_rows & 15 : 0;
      for (int kb = ti.kb0; kb < ti.kb1; ++kb) {
        if (!mbar_wait(empty_bar + 8 * stage, phase ^ 1u, abort_flag, p.status, DICE_STATUS_WAIT_SMEM_EMPTY)) {
          alive = false;
          break;
        }
        const uint32_t a_dst = tiles_smem + stage * kStageBytesT, b_dst = a_dst + kOperandBytes;
        const uint32_t leader_full = map_to_cta(full_bar + 8 * stage, 0);
        if (elect_one()) {
          if (leader) mbar_expect_tx(full_bar + 8 * stage, 2 * bytes);
          if (MODE == MODE_NN) {
            tma_load_2d_pair(a_dst, &tm_a, kb * BK, ti.row0, leader_full);
            for (int j = 0; j < b_boxes; ++j)
              tma_load_3d_pair(b_dst + j * kBoxBytes, &tm_b, col0 + 64 * j, kb * BK, ti.slab, leader_full);
          } else {
            const int row = s_seg_off[seg] + kb * BK;
            uint32_t bar = leader_full;
            if (ragged != 0 && kb == ti.kb1 - 1) {
              bar = tail_bar + 8 * stage;
              mbar_expect_tx(bar, bytes);
              bar = map_to_cta(bar, cta_rank);
            }
            for (int j = 0; j < 2; ++j) tma_load_2d_pair(a_dst + j * kBoxBytes, &tm_a, ti.row0 + 64 * j, row, bar);
            for (int j = 0; j < b_boxes; ++j) tma_load_2d_pair(b_dst + j * kBoxBytes, &tm_b, col0 + 64 * j, row, bar);
          }
        }
        __syncwarp();
        if (++stage == kStagesT) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    // ---------------- tensor-core issue (leader only) ----------------
    if (leader) {
      int stage = 0, acc = 0, seg = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool alive = true;
      for (int64_t t = pair_id; alive && t < total; t += n_pairs) {
        const Tile ti = decode(t, seg);
        if (ti.kb0 == ti.kb1) continue;
        // both operands' majors: A is K-major in NN, MN-major in TN; B is MN-major
        const uint32_t idesc = make_instr_desc(PM, ti.n_mma) | (MODE == MODE_TN ? 1u << 15 : 0u) | (1u << 16);
        if (!mbar_wait(acc_empty_bar + 8 * acc, acc_phase ^ 1u, abort_flag, p.status, DICE_STATUS_WAIT_ACC_EMPTY)) break;
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
        for (int kb = ti.kb0; kb < ti.kb1; ++kb) {
          if (!mbar_wait(full_bar + 8 * stage, phase, abort_flag, p.status, DICE_STATUS_WAIT_SMEM_FULL)) {
            alive = false;
            break;
          }
          int steps = BK / UMMA_K;
          if (MODE == MODE_TN && kb == ti.kb1 - 1) {
            steps = (ti.last_rows + UMMA_K - 1) / UMMA_K;
            if (ti.last_rows & 15) fence_cluster();
          }
          tc_fence_after_sync();
          const uint32_t a_addr = tiles_smem + stage * kStageBytesT;
          const uint64_t a_desc = MODE == MODE_NN ? make_operand_desc(a_addr) : make_mn_desc(a_addr);
          const uint64_t b_desc = make_mn_desc(a_addr + kOperandBytes);
          // 16 reduction elements further: 32 bytes along a K-major row, 16 rows of 128 bytes in an MN-major box
          constexpr uint64_t kStepA = MODE == MODE_NN ? 2 : 128, kStepB = 128;
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < BK / UMMA_K; ++kk)
              if (kk < steps)
                umma_bf16_pair(d_tmem, a_desc + kk * kStepA, b_desc + kk * kStepB, idesc,
                               static_cast<uint32_t>(kb != ti.kb0 || kk != 0));
            umma_commit_pair(empty_bar + 8 * stage);
          }
          __syncwarp();
          if (++stage == kStagesT) { stage = 0; phase ^= 1u; }
        }
        if (!alive) break;
        if (elect_one()) umma_commit_pair(acc_full_bar + 8 * acc);
        __syncwarp();
        if (++acc == kAccStages) { acc = 0; acc_phase ^= 1u; }
      }
    }
  } else if (warp == 10) {
    // ---------------- ragged ends of a weight gradient's reduction (both CTAs) ----------------
    if (MODE == MODE_TN) {
      int seg = 0;
      uint32_t tail_phase = 0;  // one bit per slot
      int slot = 0;             // slot of the tile's first block
      for (int64_t t = pair_id; t < total; t += n_pairs) {
        const Tile ti = decode(t, seg);
        const int blocks = ti.kb1 - ti.kb0;
        const int valid = ti.last_rows;
        if (blocks > 0 && (valid & 15) != 0) {
          const int stage = (slot + blocks - 1) % kStagesT;
          if (!mbar_wait(tail_bar + 8 * stage, (tail_phase >> stage) & 1u, abort_flag, p.status, DICE_STATUS_WAIT_SMEM_FULL)) break;
          tail_phase ^= 1u << stage;
          // rows [valid, next multiple of 16) of the four boxes (a row's 128 bytes are permuted within the row only)
          const int rows = 16 - (valid & 15);
          uint8_t* base = smem + stage * kStageBytesT + valid * 128;
          for (int i = lane; i < rows * 8; i += 32)
#pragma unroll
            for (int b = 0; b < 4; ++b) *reinterpret_cast<uint4*>(base + b * kBoxBytes + i * 16) = make_uint4(0, 0, 0, 0);
          fence_async_smem();
          fence_cluster();
          __syncwarp();
          if (lane == 0)
            mbar_complete_tx_cluster(map_to_cta(full_bar + 8 * stage, 0), kOperandBytes + (ti.n_mma > 128 ? 2 : 1) * kBoxBytes);
        }
        slot = (slot + blocks) % kStagesT;
      }
    }
  } else {
    // ---------------- epilogue (both CTAs, each over its own 128 rows) ----------------
    const int quad = warp & 3;
    const int half = (warp - 2) >> 2;
    int acc = 0, seg = 0;
    uint32_t acc_phase = 0;
    for (int64_t t = pair_id; t < total; t += n_pairs) {
      const Tile ti = decode(t, seg);
      if (ti.zero && ti.share != 0) continue;
      const bool summed = ti.kb0 != ti.kb1;  // this share has something in tensor memory
      if (summed) {
        if (!mbar_wait(acc_full_bar + 8 * acc, acc_phase, abort_flag, p.status, DICE_STATUS_WAIT_ACC_FULL)) break;
        tc_fence_after_sync();
      }
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(acc * BN);
      const int col0 = ti.nb * BN;
      int n_valid = p.n_cols - col0;
      if (n_valid > BN) n_valid = BN;

      // rows of the output this lane stores pieces of (see store_chunk): NULL beyond the segment or the gradient
      __nv_bfloat16* dst_rows[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rr = quad * 32 + i * 8 + (lane >> 2);
        dst_rows[i] = nullptr;
        if (rr < ti.rows_valid) {
          if (MODE == MODE_NN) {
            dst_rows[i] = p.out + static_cast<int64_t>(ti.row0 + rr) * p.n_cols + col0;
          } else if (p.gate_up == 0) {
            dst_rows[i] = p.out + (static_cast<int64_t>(ti.slab) * p.m_rows + ti.row0 + rr) * p.n_cols + col0;
          } else {
            // a pair's tile is a 128-row block of gate rows (leader) and its block of up rows (peer)
            const int r = ti.mb * BM + rr;
            if (r < p.gate_up)
              dst_rows[i] = (leader ? p.out : p.out_up) + (static_cast<int64_t>(ti.slab) * p.gate_up + r) * p.n_cols + col0;
          }
        }
      }
      uint4* stage_buf = reinterpret_cast<uint4*>(aux + kAuxBytes + (warp - 2) * kStageStore);
      // 32 columns of 32 rows: a lane holds a row, the stores cover 64-byte pieces of rows
      auto store_chunk = [&](const float (&v)[32], int c) {
        const int swz = (lane >> 1) & 3;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          stage_buf[lane * 4 + (j ^ swz)] =
              make_uint4(pack_bf16x2(v[8 * j + 0], v[8 * j + 1]), pack_bf16x2(v[8 * j + 2], v[8 * j + 3]),
                         pack_bf16x2(v[8 * j + 4], v[8 * j + 5]), pack_bf16x2(v[8 * j + 6], v[8 * j + 7]));
        __syncwarp();
        const int piece = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rr = i * 8 + (lane >> 2);
          const uint4 val = stage_buf[rr * 4 + (piece ^ ((rr >> 1) & 3))];
          if (dst_rows[i] != nullptr && piece * 8 < n_valid - c) *reinterpret_cast<uint4*>(dst_rows[i] + c + piece * 8) = val;
        }
        __syncwarp();
      };

      bool store = true;
      const bool shared_tile = split > 1 && !ti.zero;
      const int64_t part = (static_cast<int64_t>(cta_rank) * kEpilogueWarps + (warp - 2)) * kSplitFloats;
      constexpr int64_t kPairFloats = 2ll * kEpilogueWarps * kSplitFloats;
      if (shared_tile) {
        float* mine = p.split_ws + (ti.tile * split + ti.share) * kPairFloats + part + lane;
        for (int c = half * 32; c < n_valid; c += 64) {
          uint32_t a[32];
          if (summed) {
            tmem_ld32(taddr + c, a);
            tmem_ld_wait();
          }
          float* dst = mine + (c >> 6) * 1024;
#pragma unroll
          for (int j = 0; j < 32; ++j) dst[j * 32] = summed ? __uint_as_float(a[j]) : 0.f;
        }
        __threadfence();
        __syncwarp();
        unsigned int before = 0;
        if (lane == 0) before = atomicAdd(&p.split_count[(ti.tile * 2 + cta_rank) * kEpilogueWarps + (warp - 2)], 1u);
        store = __shfl_sync(0xffffffffu, before, 0) == static_cast<unsigned int>(split - 1);
        __threadfence();
      }
      if (store) {
        const float* parts = shared_tile ? p.split_ws + ti.tile * split * kPairFloats + part + lane : nullptr;
        for (int c = half * 32; c < n_valid; c += 64) {
          float v[32];
          if (shared_tile) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0.f;
            const float* src = parts + (c >> 6) * 1024;
            for (int s = 0; s < split; ++s, src += kPairFloats) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] += __ldcg(src + j * 32);
            }
          } else if (summed) {
            uint32_t a[32];
            tmem_ld32(taddr + c, a);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(a[j]);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0.f;
          }
          store_chunk(v, c);
        }
      }
      if (summed) {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_cta(acc_empty_bar + 8 * acc, 0));
        if (++acc == kAccStages) { acc = 0; acc_phase ^= 1u; }
      }
    }
  }

  // ---------------- teardown ----------------
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag != 0) {
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    __syncthreads();
  }
  cluster_barrier();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

// CTA pairs of this kernel that can be resident at once (cached per device); 0 on error
template <int MODE>
int resident_pairs_train() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (cached[dev] == 0) {
    if (cudaFuncSetAttribute(train_gemm_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemT) != cudaSuccess) return 0;
    const int sms = sm_count_cached();
    if (sms <= 0) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(sms & ~1), 1, 1);
    cfg.blockDim = dim3(kThreadsT, 1, 1);
    cfg.dynamicSmemBytes = kSmemT;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, train_gemm_kernel<MODE>, &cfg) != cudaSuccess || n <= 0) return 0;
    cached[dev] = n < sms / 2 ? n : sms / 2;
  }
  return cached[dev];
}

template <int MODE>
int launch_train(const CUtensorMap& tm_a, const CUtensorMap& tm_b, const TrainGemm& p, int64_t most_tiles, int pairs,
                 cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  const int64_t use = most_tiles < pairs && p.split_ws == nullptr ? most_tiles : pairs;
  cfg.gridDim = dim3(static_cast<unsigned>(2 * use), 1, 1);
  cfg.blockDim = dim3(kThreadsT, 1, 1);
  cfg.dynamicSmemBytes = kSmemT;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dice_pdl_enabled() ? 2 : 1;
  dice_count_launch();
  return cudaLaunchKernelEx(&cfg, train_gemm_kernel<MODE>, tm_a, tm_b, p) == cudaSuccess ? DICE_OK : DICE_ERR_CUDA;
}

}  // namespace

int dice_internal_tc_dgrad(const void* dy, int64_t n_rows, int n_dim, const void* w, int n_slabs, int k_dim,
                           const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, void* dx, uint32_t* status,
                           cudaStream_t s) {
  const int pairs = resident_pairs_train<MODE_NN>();
  if (pairs <= 0) return DICE_ERR_CUDA;
  CUtensorMap tm_a, tm_b;
  int rc = encode_map(&tm_a, dy, static_cast<uint64_t>(n_rows), static_cast<uint64_t>(n_dim), BM);
  if (rc == DICE_OK)
    rc = encode_map3(&tm_b, w, static_cast<uint64_t>(n_slabs), static_cast<uint64_t>(n_dim), static_cast<uint64_t>(k_dim), BK);
  if (rc != DICE_OK) return rc;
  TrainGemm p = {};
  p.seg_offsets = seg_offsets;
  p.seg_slab = seg_slab;
  p.n_seg = n_seg;
  p.n_slabs = n_slabs;
  p.n_rows = static_cast<int>(n_rows);
  p.red_blocks = (n_dim + BK - 1) / BK;
  p.n_nblk = (k_dim + BN - 1) / BN;
  p.n_cols = k_dim;
  p.out = static_cast<__nv_bfloat16*>(dx);
  p.status = status;
  return launch_train<MODE_NN>(tm_a, tm_b, p, ((n_rows + PM - 1) / PM + n_seg) * p.n_nblk, pairs, s);
}

int dice_internal_tc_wgrad(const void* dy, const void* x, int64_t n_rows, int n_dim, int k_dim, const int32_t* seg_offsets,
                           int n_slabs, int gate_up, void* dw, void* dw_up, uint32_t* status, cudaStream_t s) {
  const int pairs = resident_pairs_train<MODE_TN>();
  if (pairs <= 0) return DICE_ERR_CUDA;
  CUtensorMap tm_a, tm_b;
  // without rows no operand is read; the maps still want one
  const uint64_t map_rows = n_rows > 0 ? static_cast<uint64_t>(n_rows) : 1;
  int rc = encode_map(&tm_a, n_rows > 0 ? dy : dw, map_rows, static_cast<uint64_t>(n_dim), BK);
  if (rc == DICE_OK) rc = encode_map(&tm_b, n_rows > 0 ? x : dw, map_rows, static_cast<uint64_t>(k_dim), BK);
  if (rc != DICE_OK) return rc;
  TrainGemm p = {};
  p.seg_offsets = seg_offsets;
  p.n_seg = n_slabs;
  p.n_slabs = n_slabs;
  p.n_rows = static_cast<int>(n_rows);
  p.n_mblk = (n_dim + PM - 1) / PM;
  p.m_rows = n_dim;
  p.n_nblk = (k_dim + BN - 1) / BN;
  p.n_cols = k_dim;
  p.gate_up = gate_up;
  p.out = static_cast<__nv_bfloat16*>(dw);
  p.out_up = static_cast<__nv_bfloat16*>(dw_up);
  p.status = status;
  return launch_train<MODE_TN>(tm_a, tm_b, p, static_cast<int64_t>(n_slabs) * p.n_mblk * p.n_nblk, pairs, s);
}
