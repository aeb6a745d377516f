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
// Bound: the tensor cores, and in calls that follow each other the GPU's power; an instruction takes the same time for
// K-major and MN-major operands (512 cycles a k-block, measured with all operands in shared memory).  Eight segments of 4096
// rows, 9216 x 1024 and 9216 x 1152 (4.5 tiles of columns), PFLOP/s of one call after a pause / of calls for a second, at SM
// clocks of 1.1-1.24 of 1.97 GHz under the power cap: NN 1.48 / 1.24 and 1.38 / 1.17, TN 1.47 / 1.24 and 1.43 / 1.19, cuBLAS
// (all rows, one weight) 1.50 / 1.25 and 1.47 / 1.21.  So the half tile costs 3 to 7 %, the power 16 %.  A weight gradient
// of few rows is bounded by writing it (777 rows, 16 x 1792 x 7168: 411 MB in 111 us = 3.7 TB/s, memset 3.8).
//
// A weight gradient's reduction is ragged.  Its last k-block may reach into the next segment (or behind the tensor, or
// into rows that hold anything): the instructions stop at the last 16 rows that the segment touches, and the up to
// 15 rows of those that are not the segment's are zeroed in shared memory, in both operands, since a zero in one
// would not silence a NaN in the other.  For such a block each CTA's copies complete on a barrier of its own; a warp
// waits there, zeroes, makes the zeros visible to the asynchronous proxy and completes the copies' bytes on the leader's
// "full" barrier in their place.  All other blocks go from the copies to the tensor cores directly.  (The leader expects
// both CTAs' bytes; a peer that announced its own with a cluster-scope arrival cost twice the time of a block.)
//
// Two products have the activation in their epilogue, so that neither its argument nor its gradient passes through
// memory in 16 bits between two kernels:
//   NT + EPI_KEEP  the first forward product (rows and weights as they lie): a warp pair holds a row's 128 columns of a
//                  group in registers, rounds them to bf16, makes the group's scale, and writes the activation and the
//                  8-bit codes.  SwiGLU's packed order makes a 256-column tile one group of gate and one of up columns.
//   NN + EPI_BACK  the second product's input gradient: every column's gradient meets the codes of its argument in fp32
//                  and leaves as the argument's gradient, beside the activation for the weight gradient behind it.
// The activation, its argument and the argument's gradient are rounded to bf16 here because the next product's tensor-core
// operands are bf16 (a second plane of 8 more bits would double that product).  A result of the second product is then
// off by the roundings of the activation and its own, 2.4e-3 of its norm against 1.7e-3 for its own alone.
//
// fp32 operands (PLANES 3) come as three bf16 planes each, x = hi + 2^-8 mid + 2^-16 lo exactly (8 bits of the mantissa a
// plane), and a product is six: hi hi, hi mid, mid hi, mid mid, hi lo, lo hi; what is left out is below 2^-25 of it.  The
// accumulator in tensor memory is cut, not rounded, after every instruction, so it is emptied after every k-block of 64 into
// fp32 registers that round, and within a block the small products come first: those of 2^-16, then, the sum scaled by 2^-8
// as the first of them is added, those of 2^-8, then, scaled again, hi hi.  The planes hold their bits at hi's own
// magnitude, since bf16 ends where fp32 does: unscaled, mid and lo of values below 2^-110 would have lost their last bits
// there, which a large factor on the other side makes visible (fp32's own subnormals, below 2^-126, have their bits in mid
// and lo: their products are good to 2^-8).  Six instructions for one leave ~220 TFLOP/s, three times the CUDA cores' 74.
// An infinity in an operand (times a zero plane), or planes' products that overflow to infinities of both signs, leave a NaN
// where the sum may be an infinity or a number: an epilogue that sees a value that is not finite says so, and the CUDA cores
// make those values again (dice_internal_f32_repair).
//
// A bf16 product's accumulator is cut after every 16 of the reduction too, always towards zero, by up to 2^-23 of the sum so
// far.  Over 32768 of the reduction (512 k-blocks) that is at most 2^-12 of a sum whose terms have one sign, an eighth of
// half a step of the bf16 result, but it grows with the length: 2^21 rows would lose 2^-6.  Products that may be longer
// (LONG: weight gradients of more than 32768 rows, input gradients of more than 32768 columns of dy) empty the accumulator
// every 512 k-blocks into fp32 registers that round, as planes do every one (65536 rows, 8 x 9216 x 1152: 973 -> 1000 us;
// 2304 x 1152: 356 -> 333; 131072 rows, 4608 x 1152: 1610 -> 1760; the same without a cut, so not the emptying).  The
// products with the activation in their epilogue, which reduce over the hidden dimension, are not cut up: 32768 is beyond
// any hidden dimension known.
//
// Few tiles: they are made half as wide if that keeps more pairs busy (one token's two rows, 1152 -> 4608: 36 tiles of
// 256 columns, 72 of 128; 80 tiles on 74 pairs are two rounds, and so are 144 of half the width).  Fewer still, and a long
// reduction: the pairs that would idle take a share of the reduction each (split).  Every epilogue warp files its part of
// the sum in fp32; the last one to arrive at a part adds them up in the order of the shares, so the result does not depend
// on who was last.
#include <cuda.h>

#include "train.cuh"
#include "umma_pair.cuh"

using namespace dice_umma;

namespace {

enum { MODE_NT = 0, MODE_NN = 1, MODE_TN = 2 };
enum { EPI_PLAIN = 0, EPI_KEEP = 1, EPI_BACK = 2 };

constexpr int PM = 256;
// Operand ring slots and, per epilogue warp, staging buffers of 32 rows x 64 bytes.  The activation's epilogues write (and
// read) several bytes for every one of a plain product, so they give a ring slot for two more buffers and let the copy
// unit store them (see Stager).
constexpr int stages_of(int epi, int planes = 1) { return planes == 3 ? 2 : epi == EPI_PLAIN ? 6 : 5; }
constexpr int buffers_of(int epi) { return epi == EPI_PLAIN ? 1 : 3; }
constexpr int kStageBytesT = 32768;  // 128 rows (or columns) x 64 of each operand
constexpr int kOperandBytes = 16384;
constexpr int kBoxBytes = 8192;      // 64 reduction rows x 128 bytes
// warp 0 loader, 1 tensor-core issue, 2..9 epilogue, TN: 10 ragged ends
constexpr int threads_of(int mode) { return 32 * (2 + kEpilogueWarps + (mode == MODE_TN ? 1 : 0)); }
constexpr int kStageStore = 2048;    // per epilogue warp, as in grouped_gemm_pair.cu
constexpr int kExchangeBytes = 4096;  // EPI_KEEP, SwiGLU: group maxima, [2 tiles][2 halves][gate, up][128 rows]
constexpr int smem_of(int epi, int planes) {
  return stages_of(epi, planes) * planes * kStageBytesT + kAuxBytes + kEpilogueWarps * buffers_of(epi) * kStageStore + kExchangeBytes + 1024;
}
constexpr int kSplitFloats = 4 * 32 * 32;  // an epilogue warp's part of a tile: 4 chunks of 32 rows x 32 columns
constexpr int kBand = 8;                   // TN: row tiles of a band, and the elements of x from which there are
constexpr int64_t kBandElems = 32 << 20;   // bands (see decode)
constexpr int kMinSplitBlocks = 4;         // k-blocks of a share, at least
constexpr int kLongBlocks = 512;           // k-blocks of a chain (see LONG)
constexpr int kMaxSplit = 16;              // the last warp reads the shares one after the other

struct TrainGemm {
  const int* seg_offsets;
  const int* seg_slab;
  int n_seg, n_slabs;
  int n_rows;
  int red_blocks;   // NN: k-blocks of the reduction
  int n_mblk;       // TN: row tiles of a slab's gradient
  int n_cols;       // output columns
  int m_rows;       // TN: output rows of a slab
  int a_plane, b_plane;  // PLANES 3: rows (NN: slabs of w) from one plane of an operand to the next
  int gate_up;      // TN: 0, or ffn: the rows are packed gate / up blocks and go to two tensors
  __nv_bfloat16* out;
  __nv_bfloat16* out_up;
  float* split_ws;  // NULL: no split.  [pair][cta][epilogue warp][kSplitFloats]
  unsigned int* split_count;  // zero on entry: [tile][cta][epilogue warp]
  uint32_t* status;
  // EPI_KEEP and EPI_BACK: `out` is d_pre (EPI_BACK) or pre (EPI_KEEP that keeps it), its rows are arg_cols wide
  int ffn, arg_cols, groups;
  __nv_bfloat16* act_out;
  const void* kept;             // EPI_BACK: codes or pre
  const float* kept_scales;
  int kept_wide;                // its rows are whole pieces of 32 bytes
  unsigned int* non_finite;     // PLANES 3: set where a result is (see dice_internal_f32_repair)
  uint8_t* codes;               // EPI_KEEP
  int codes_tma;                // its rows are whole pieces of 16 bytes
  float* scales;
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
// D = A B + 2^-8 D
__device__ __forceinline__ void umma_bf16_pair_scaled(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.eq.b32 p, 0, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p, 8;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc)
      : "memory");
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
// Wait for a ragged end.  Any number of tiles without one may lie between it and the last, so the limit is on a standstill:
// it starts anew whenever the loader has filled another slot (its own waits are bounded one by one).
__device__ __noinline__ bool mbar_wait_behind(uint32_t bar, uint32_t parity, volatile uint32_t* filled, volatile uint32_t* abort_flag,
                                              uint32_t* status) {
  uint64_t t0 = global_timer_ns();
  uint32_t seen = *filled, spins = 0;
  while (!mbar_try_wait(bar, parity)) {
    if ((++spins & 127u) != 0) continue;
    if (*abort_flag != 0) return false;
    const uint32_t now = *filled;
    const uint64_t t = global_timer_ns();
    if (now != seen) {
      seen = now;
      t0 = t;
    } else if (t - t0 > kWaitLimitNs) {
      if (status != nullptr) atomicCAS(status, 0u, DICE_STATUS_WAIT_SMEM_FULL);
      *abort_flag = 1;
      __threadfence_block();
      return false;
    }
  }
  return true;
}
// orders the zeroing before that (release), and after it in the issuing warp (acquire)
__device__ __forceinline__ void fence_cluster() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// Stores of 32 rows of 64 bytes that a warp holds one row per lane.  They go through shared memory, laid out as the 64-byte
// swizzle wants it.  If all 32 rows exist (a segment's last tile may have fewer) and BUFS > 1, the copy unit stores them as
// one box, clipped to the tensor's columns; a few buffers in turn, of which the one about to be written is no longer read.
// Else lane l takes piece (l & 3) of rows (l >> 2) + 8 i, so that an instruction covers whole 64-byte pieces:
// `put(i, piece, v)` stores one.  An SM's memory path handles so many lines a cycle; a chunk's three outputs cost it
// 48 + 48 + 96 this way and 48 + 0 + 0 by the copy unit, beside the operands' 128 a k-block.
template <int BUFS>
struct Stager {
  uint8_t* buffers;
  int lane, next, row0;
  bool whole;
  template <typename F>
  __device__ __forceinline__ void store(const uint4 (&mine)[4], const CUtensorMap* map, int c, F put) {
    const int swz = (lane >> 1) & 3;
    if (BUFS > 1) {
      // the copies that may still read: with the copy unit all but the oldest buffer's, else none
      if (lane == 0) {
        if (whole && map != nullptr) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(BUFS - 1) : "memory");
        else asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      }
      __syncwarp();
    }
    uint4* buf = reinterpret_cast<uint4*>(buffers + next * kStageStore);
#pragma unroll
    for (int j = 0; j < 4; ++j) buf[lane * 4 + (j ^ swz)] = mine[j];
    if (BUFS > 1 && whole && map != nullptr) {
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)),
                     "r"(c), "r"(row0), "r"(smem_u32(buf))
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
      next = next == BUFS - 1 ? 0 : next + 1;
      return;
    }
    __syncwarp();
    const int piece = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rr = i * 8 + (lane >> 2);
      put(i, piece, buf[rr * 4 + (piece ^ ((rr >> 1) & 3))]);
    }
    __syncwarp();
  }
  // before the buffers go: everything has been read and written
  __device__ __forceinline__ void finish() {
    if (BUFS > 1 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
};
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// EPI_KEEP: one tile of the first product, by one of the two warps that share 32 rows.  SwiGLU: the tile's columns are
// 128 gate and 128 up columns of the same 128 activations, a warp takes 64 of them, and the two warps exchange their parts
// of the groups' maxima; GELU: the tile is two groups, a warp takes one.  Columns behind ffn count as zeros.
template <int ACT, int KEEP, typename Fetch, typename Store, typename Staging>
__device__ __forceinline__ void keep_tile(const TrainGemm& p, int nb, int quad, int half, int lane, int row, bool row_ok,
                                          const int64_t (&dst_row)[4], Staging& stager, const CUtensorMap* tm_out,
                                          const CUtensorMap* tm_act, const CUtensorMap* tm_codes, float* exchange, uint32_t bar,
                                          uint32_t phase, volatile uint32_t* abort_flag, Fetch fetch, Store store_bf16) {
  constexpr bool GLU = ACT == DICE_ACT_SWIGLU, CODES = KEEP == DICE_KEEP_INT8 || KEEP == DICE_KEEP_E4M3;
  // this warp's first activation column, and how many of its 64 (GELU: 128) exist
  const int act0 = GLU ? nb * 128 + half * 64 : nb * 256 + half * 128;
  int valid = p.ffn - act0;
  valid = valid < 0 ? 0 : (valid > (GLU ? 64 : 128) ? (GLU ? 64 : 128) : valid);
  // four chunks of 32 columns of the argument, rounded to bf16: SwiGLU gate, gate, up, up; GELU four in a row
  uint32_t w[4][16];
  uint32_t most2[2] = {0u, 0u};  // largest magnitudes, two bf16 each: gate and up (GELU: the first)
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int left = valid - (GLU ? (q & 1) : q) * 32;
    if (left > 0) {
      float v[32];
      fetch(GLU ? (q >> 1) * 128 + half * 64 + (q & 1) * 32 : half * 128 + q * 32, v);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        w[q][j] = 2 * j < left ? pack_bf16x2(v[2 * j], v[2 * j + 1]) : 0u;  // (valid is a multiple of 8)
        if (CODES) {
          uint32_t& m = most2[GLU ? q >> 1 : 0];
          asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[q][j] & 0x7fff7fffu));
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) w[q][j] = 0u;
    }
  }
  float scale[2], factor[2];
  if (CODES) {
    float most[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) most[g] = max_nan(bf16lo_to_f32(most2[g]), bf16hi_to_f32(most2[g]));
    if (GLU) {
      // two buffers in turn: a warp writes the next tile's only after the other has read this one's predecessor
      float* buf = exchange + phase * 512;
      const int r = quad * 32 + lane;
      buf[half * 256 + r] = most[0];
      buf[half * 256 + 128 + r] = most[1];
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
      // (should the other warp have given up, the values below are of no use, but nothing waits for them)
      mbar_wait(bar, phase, abort_flag, p.status, DICE_STATUS_WAIT_ACC_FULL);
      most[0] = max_nan(most[0], buf[(half ^ 1) * 256 + r]);
      most[1] = max_nan(most[1], buf[(half ^ 1) * 256 + 128 + r]);
    }
#pragma unroll
    for (int g = 0; g < (GLU ? 2 : 1); ++g) keep_scale(most[g], keep_top(KEEP), scale[g], factor[g]);
    if (row_ok && (GLU || valid > 0))
      p.scales[static_cast<int64_t>(row) * p.groups + nb * 2 + half] = GLU && half ? scale[1] : scale[0];
  }
  // the activation
#pragma unroll
  for (int q = 0; q < (GLU ? 2 : 4); ++q) {
    if (valid > q * 32) {
      uint4 o[4];
      uint32_t* ow = reinterpret_cast<uint32_t*>(o);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const f32x2 x = bf16_pair<f32x2>(w[q][j]);
        ow[j] = to_bf16(GLU ? swiglu2<false>(x, bf16_pair<f32x2>(w[q + 2][j])) : gelu2<false>(x));
      }
      store_bf16(o, tm_act, p.act_out, p.ffn, act0 + q * 32, valid - q * 32);
    }
  }
  // what is kept: SwiGLU all 64 gate and 64 up columns (the filling ones are zeros), GELU those that exist
  if (KEEP == DICE_KEEP_NONE) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int left = GLU ? 32 : valid - q * 32;
      if (left > 0) {
        uint4 o[4];
        uint32_t* ow = reinterpret_cast<uint32_t*>(o);
#pragma unroll
        for (int j = 0; j < 16; ++j) ow[j] = w[q][j];
        store_bf16(o, tm_out, p.out, p.arg_cols, GLU ? nb * 256 + (q >> 1) * 128 + half * 64 + (q & 1) * 32 : act0 + q * 32, left);
      }
    }
  } else if (CODES) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {  // 64 codes each
      const int left = GLU ? 64 : valid - g * 64;
      if (left > 0) {
        const f32x2 f = both<f32x2>(GLU ? factor[g] : factor[0]);
        uint4 o[4];
        uint32_t* ow = reinterpret_cast<uint32_t*>(o);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const uint32_t lo = w[2 * g + (j >> 3)][(j & 7) * 2], hi = w[2 * g + (j >> 3)][(j & 7) * 2 + 1];
          ow[j] = keep_codes4<KEEP>(mul2(bf16_pair<f32x2>(lo), f), mul2(bf16_pair<f32x2>(hi), f));
        }
        const int c = GLU ? nb * 256 + g * 128 + half * 64 : act0 + g * 64;
        stager.store(o, GLU || p.codes_tma ? tm_codes : nullptr, c, [&](int i, int piece, const uint4& v) {
          if (dst_row[i] < 0) return;
          uint8_t* dst = p.codes + dst_row[i] * p.arg_cols + c + piece * 16;
          // a row of GELU codes may start on 8 bytes only, and end in the middle of a piece
          if (GLU || (piece * 16 + 16 <= left && (p.arg_cols & 15) == 0)) {
            *reinterpret_cast<uint4*>(dst) = v;
          } else {
            if (piece * 16 < left) *reinterpret_cast<uint2*>(dst) = make_uint2(v.x, v.y);
            if (piece * 16 + 8 < left) *reinterpret_cast<uint2*>(dst + 8) = make_uint2(v.z, v.w);
          }
        });
      }
    }
  }
}

// 32 bytes in one load.  A lane holds a row of its own, so a load touches 32 lines whatever its width, and those lines
// are what the memory path of an SM has too few of beside the operands' copies and the matrix instructions' reads (the
// product of 32768 x 1152 x 4608 took 564 us with 16-byte loads and a scale for every 32 columns, 535 us like this; 16
// epilogue warps in the place of 8, with stores of 32 bytes a lane, took 588).
__device__ __forceinline__ void ld_32bytes(const void* p, uint4& a, uint4& b) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
               : "l"(p));
}

// 32 columns of a row's kept argument
template <int KEEP>
struct KeptChunk {
  static constexpr int kVecs = KEEP == DICE_KEEP_NONE ? 4 : 2, kCols = 32 / kVecs;
  uint4 v[kVecs];
  // at: element offset of the first column; n_left: columns that exist (a multiple of 8); wide: rows of whole 32 bytes
  __device__ __forceinline__ void load(const TrainGemm& p, int64_t at, int n_left, bool ok) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) v[i] = make_uint4(0, 0, 0, 0);
    if (!ok) return;
    const uint8_t* src = static_cast<const uint8_t*>(p.kept) + at * (KEEP == DICE_KEEP_NONE ? 2 : 1);
    if (p.kept_wide && n_left >= 32) {
#pragma unroll
      for (int i = 0; i < kVecs; i += 2) ld_32bytes(src + i * 16, v[i], v[i + 1]);
    } else {  // the ragged end of a row, or rows that start on 8 bytes
#pragma unroll
      for (int i = 0; i < 2 * kVecs; ++i) {
        if (i * kCols / 2 < n_left) {
          const uint2 w = *reinterpret_cast<const uint2*>(src + i * 8);
          uint4& x = v[i >> 1];
          if (i & 1) { x.z = w.x; x.w = w.y; }
          else { x.x = w.x; x.y = w.y; }
        }
      }
    }
  }
  // columns 8 g .. 8 g + 7
  __device__ __forceinline__ void get8(int g, f32x2 scale, f32x2 (&f)[4]) const {
    if (KEEP == DICE_KEEP_NONE) {
      const uint4 x = v[KEEP == DICE_KEEP_NONE ? g : 0];
      f[0] = bf16_pair<f32x2>(x.x); f[1] = bf16_pair<f32x2>(x.y); f[2] = bf16_pair<f32x2>(x.z); f[3] = bf16_pair<f32x2>(x.w);
    } else {
      const uint4 x = v[g >> 1];
      keep_read4<KEEP>(g & 1 ? x.z : x.x, scale, f[0], f[1]);
      keep_read4<KEEP>(g & 1 ? x.w : x.y, scale, f[2], f[3]);
    }
  }
};

// What an EPI_BACK warp holds of a row's kept argument: 32 columns, and the scales of their group.  A warp's share of a
// tile is 128 columns of the activation's gradient, a group.
template <int ACT, int KEEP>
struct BackChunk {
  static constexpr bool GLU = ACT == DICE_ACT_SWIGLU;
  KeptChunk<KEEP> g, u;
  float scale_g, scale_u;
  __device__ __forceinline__ void load(const TrainGemm& p, int col, int row, bool ok) {
    const int64_t at = static_cast<int64_t>(row) * p.arg_cols + (GLU ? col + col / kKeepGroup * kKeepGroup : col);
    const int n_left = GLU ? 32 : p.ffn - col;
    g.load(p, at, n_left, ok);
    if (GLU) u.load(p, at + kKeepGroup, n_left, ok);
  }
  __device__ __forceinline__ void load_first(const TrainGemm& p, int nb, int half, int row, bool ok) {
    const int col = nb * BN + half * 128;
    ok = ok && col < (GLU ? p.arg_cols / 2 : p.ffn);
    scale_g = scale_u = 0.f;
    if (KEEP != DICE_KEEP_NONE && ok) {
      const float* sc = p.kept_scales + static_cast<int64_t>(row) * p.groups + col / kKeepGroup * (GLU ? 2 : 1);
      scale_g = sc[0];
      if (GLU) scale_u = sc[1];
    }
    load(p, col, row, ok);
  }
};

// EPI_BACK: a warp's 128 columns of one tile of the activation's gradient, 32 at a time, with SwiGLU up to the end of the
// packed order's last block (whose filling columns get gradient zero)
template <int ACT, int KEEP, typename Fetch, typename Store>
__device__ __forceinline__ void back_tile(const TrainGemm& p, int nb, int half, int row, bool row_ok, BackChunk<ACT, KEEP>& kept,
                                          const CUtensorMap* tm_out, const CUtensorMap* tm_act, Fetch fetch, Store store_bf16) {
  constexpr bool GLU = ACT == DICE_ACT_SWIGLU;
  const int end = GLU ? p.arg_cols / 2 : p.ffn;
  for (int h = 0; h < 128; h += 32) {
    const int c = half * 128 + h, col = nb * BN + c, left = p.ffn - col;  // activation columns from here on (none: only filling)
    if (col >= end) break;
    float v[32];
    if (left > 0) fetch(c, v);
    if (left < 32) {
      // columns behind ffn: whatever the product left there, the gradient is zero
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = j < left ? v[j] : 0.f;
    }
    uint4 og[4], ou[4], oa[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x2 x[4], u[4], a[4];
      kept.g.get8(g, both<f32x2>(kept.scale_g), x);
      if (GLU) kept.u.get8(g, both<f32x2>(kept.scale_u), u);
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = act_backward2<false, ACT>(pair<f32x2>(v[g * 8 + 2 * i], v[g * 8 + 2 * i + 1]), x[i], u[i]);
      og[g] = make_uint4(to_bf16(x[0]), to_bf16(x[1]), to_bf16(x[2]), to_bf16(x[3]));
      if (GLU) ou[g] = make_uint4(to_bf16(u[0]), to_bf16(u[1]), to_bf16(u[2]), to_bf16(u[3]));
      oa[g] = make_uint4(to_bf16(a[0]), to_bf16(a[1]), to_bf16(a[2]), to_bf16(a[3]));
    }
    if (h + 32 < 128 && col + 32 < end) kept.load(p, col + 32, row, row_ok);  // on its way while this chunk is stored
    const int at = GLU ? col + col / kKeepGroup * kKeepGroup : col;
    store_bf16(og, tm_out, p.out, p.arg_cols, at, GLU ? 32 : left);
    if (GLU) store_bf16(ou, tm_out, p.out, p.arg_cols, at + kKeepGroup, 32);
    if (left > 0) store_bf16(oa, tm_act, p.act_out, p.ffn, col, left);
  }
}

template <int MODE, int EPI, int ACT, int KEEP, int PLANES, bool LONG>
__global__ void __launch_bounds__(threads_of(MODE), 1)
train_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                  const __grid_constant__ CUtensorMap tm_out, const __grid_constant__ CUtensorMap tm_act,
                  const __grid_constant__ CUtensorMap tm_codes, const TrainGemm p) {
  constexpr int kStagesT = stages_of(EPI, PLANES), kSlotBytes = PLANES * kStageBytesT;
  // the accumulator is emptied into the epilogue's registers after every chain of k-blocks, not once a tile
  constexpr bool kChains = PLANES == 3 || LONG;
  constexpr int kChain = PLANES == 3 ? 1 : kLongBlocks;
  static_assert(!kChains || EPI == EPI_PLAIN, "plain products");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* aux = smem + kStagesT * kSlotBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(aux);
  const uint32_t full_bar = smem_u32(bars);                                 // [kStagesT] used in the leader
  const uint32_t empty_bar = smem_u32(bars + kStagesT);                     // [kStagesT] in both CTAs
  const uint32_t tail_bar = smem_u32(bars + 2 * kStagesT);                  // [kStagesT] in both CTAs (TN)
  const uint32_t acc_full_bar = smem_u32(bars + 3 * kStagesT);              // [kAccStages] in both CTAs
  const uint32_t acc_empty_bar = smem_u32(bars + 3 * kStagesT + kAccStages);  // used in the leader
  const uint32_t xchg_bar = smem_u32(bars + 3 * kStagesT + 2 * kAccStages);  // [4] EPI_KEEP: a quadrant's two warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 3 * kStagesT + 2 * kAccStages + 4);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  int* s_split = reinterpret_cast<int*>(tmem_slot + 2);  // shares of the reduction; columns of a tile
  volatile uint32_t* filled = tmem_slot + 4;             // TN: slots that the loader has filled so far
  int* s_seg_off = reinterpret_cast<int*>(tmem_slot + 5);
  int* s_mprefix = s_seg_off + (kMaxSeg + 1);  // NT, NN: first row tile of every segment
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
    for (int q = 0; q < 4; ++q) mbar_init(xchg_bar + 8 * q, 2);
    *abort_flag = 0;
    *filled = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc_pair(smem_u32(tmem_slot), kTmemCols);
  pdl_wait();

  for (int i = threadIdx.x; i <= p.n_seg; i += threads_of(MODE)) s_seg_off[i] = p.seg_offsets[i];
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
    // narrow tiles take about 0.65 of a wide one's time each
    const int64_t wide_waves = (static_cast<int64_t>(run) * ((p.n_cols + BN - 1) / BN) + n_pairs - 1) / n_pairs;
    const int64_t narrow_waves = (static_cast<int64_t>(run) * ((p.n_cols + BN / 2 - 1) / (BN / 2)) + n_pairs - 1) / n_pairs;
    const int bn = EPI == EPI_PLAIN && 13 * narrow_waves < 20 * wide_waves ? BN / 2 : BN;
    if (EPI == EPI_PLAIN && p.split_ws != nullptr && run > 0) {
      const int64_t per_tile = n_pairs / (static_cast<int64_t>(run) * ((p.n_cols + bn - 1) / bn));
      const int blocks = MODE != MODE_TN ? p.red_blocks : (most + BK - 1) / BK;
      split = static_cast<int>(per_tile < blocks / kMinSplitBlocks ? per_tile : blocks / kMinSplitBlocks);
      split = split < 1 ? 1 : (split > kMaxSplit ? kMaxSplit : split);
    }
    s_split[0] = split;
    s_split[1] = bn;
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_barrier();
  tc_fence_after_sync();

  const uint32_t tmem_base = *tmem_slot;
  const int split = EPI == EPI_PLAIN ? s_split[0] : 1, bn = EPI == EPI_PLAIN ? s_split[1] : BN;
  const int n_nblk = (p.n_cols + bn - 1) / bn;
  const int64_t total = static_cast<int64_t>(s_mprefix[p.n_seg]) * n_nblk * split;

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
    const int m = static_cast<int>(ti.tile / n_nblk);
    ti.nb = static_cast<int>(ti.tile - static_cast<int64_t>(m) * n_nblk);
    int blocks;
    if (MODE != MODE_TN) {
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
      const int cnt = s_seg_off[seg + 1] - s_seg_off[seg];
      if (static_cast<int64_t>(cnt) * p.n_cols > kBandElems) {
        // x's segment is more than half of L2: row after row of tiles would read all of it from memory for every two or
        // three.  In bands of 8 row tiles, down a band's columns, the tiles that run at one time read few columns of
        // either operand: 8192 rows, 8192 x 8192 748 -> 704 us; 8 x 4096 rows, 1024 x 9216 456 -> 416.  Where the
        // segment stays in L2 the rows' order is the better one by 1 to 7 %: 16 x 2048 rows, 1792 x 7168 603 -> 648.
        const int in_slab = ti.mb * n_nblk + ti.nb;
        const int band = in_slab / (kBand * n_nblk), in_band = in_slab - band * kBand * n_nblk;
        const int tall = p.n_mblk - band * kBand < kBand ? p.n_mblk - band * kBand : kBand;
        ti.nb = in_band / tall;
        ti.mb = band * kBand + in_band - ti.nb * tall;
      }
      ti.slab = seg;
      ti.row0 = ti.mb * PM + static_cast<int>(cta_rank) * BM;  // of the gradient
      ti.rows_valid = p.m_rows - ti.row0;
      blocks = (cnt + BK - 1) / BK;
      ti.last_rows = cnt - (blocks - 1) * BK;
    }
    ti.zero = blocks == 0;
    ti.kb0 = static_cast<int>(static_cast<int64_t>(blocks) * ti.share / split);
    ti.kb1 = static_cast<int>(static_cast<int64_t>(blocks) * (ti.share + 1) / split);
    if (ti.kb1 < blocks) ti.last_rows = BK;
    int n_valid = p.n_cols - ti.nb * bn;
    if (n_valid > bn) n_valid = bn;
    ti.n_mma = (n_valid + 31) & ~31;  // half of the columns come from each CTA
    return ti;
  };

  if (warp == 0) {
    // ---------------- loader (both CTAs) ----------------
    int stage = 0, seg = 0;
    uint32_t phase = 0, n_filled = 0;
    bool alive = true;
    for (int64_t t = pair_id; alive && t < total; t += n_pairs) {
      const Tile ti = decode(t, seg);
      const int half = ti.n_mma / 2;
      const int col0 = ti.nb * bn + static_cast<int>(cta_rank) * half;  // this CTA's B columns
      const int b_boxes = half > 64 ? 2 : 1;
      const uint32_t bytes = PLANES * (kOperandBytes + b_boxes * kBoxBytes);
      const int ragged = MODE == MODE_TN ? ti.last_rows & 15 : 0;
      for (int kb = ti.kb0; kb < ti.kb1; ++kb) {
        if (!mbar_wait(empty_bar + 8 * stage, phase ^ 1u, abort_flag, p.status, DICE_STATUS_WAIT_SMEM_EMPTY)) {
          alive = false;
          break;
        }
        const uint32_t slot_smem = tiles_smem + stage * kSlotBytes;
        const uint32_t leader_full = map_to_cta(full_bar + 8 * stage, 0);
        ++n_filled;
        if (elect_one()) {
          if (MODE == MODE_TN) *filled = n_filled;
          if (leader) mbar_expect_tx(full_bar + 8 * stage, 2 * bytes);
          uint32_t bar = leader_full;
          if (MODE == MODE_TN && ragged != 0 && kb == ti.kb1 - 1) {
            bar = tail_bar + 8 * stage;
            mbar_expect_tx(bar, bytes);
            bar = map_to_cta(bar, cta_rank);
          }
#pragma unroll
          for (int pl = 0; pl < PLANES; ++pl) {
            const uint32_t a_dst = slot_smem + pl * kStageBytesT, b_dst = a_dst + kOperandBytes;
            const int a_off = pl * p.a_plane, b_off = pl * p.b_plane;
            if (MODE == MODE_TN) {
              const int row = s_seg_off[seg] + kb * BK;
              for (int j = 0; j < 2; ++j) tma_load_2d_pair(a_dst + j * kBoxBytes, &tm_a, ti.row0 + 64 * j, row + a_off, bar);
              for (int j = 0; j < b_boxes; ++j) tma_load_2d_pair(b_dst + j * kBoxBytes, &tm_b, col0 + 64 * j, row + b_off, bar);
            } else {
              tma_load_2d_pair(a_dst, &tm_a, kb * BK, ti.row0 + a_off, bar);
              for (int j = 0; j < b_boxes; ++j) {
                if (MODE == MODE_NT)
                  tma_load_2d_pair(b_dst + j * kBoxBytes, &tm_b, kb * BK, ti.slab * p.arg_cols + col0 + 64 * j + b_off, bar);
                else
                  tma_load_3d_pair(b_dst + j * kBoxBytes, &tm_b, col0 + 64 * j, kb * BK, ti.slab + b_off, bar);
              }
            }
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
        // both operands' majors: A is MN-major in TN, B in NN and TN
        const uint32_t idesc = make_instr_desc(PM, ti.n_mma) | (MODE == MODE_TN ? 1u << 15 : 0u) | (MODE != MODE_NT ? 1u << 16 : 0u);
        if (!kChains) {
          if (!mbar_wait(acc_empty_bar + 8 * acc, acc_phase ^ 1u, abort_flag, p.status, DICE_STATUS_WAIT_ACC_EMPTY)) break;
        }
        for (int kb = ti.kb0; kb < ti.kb1; ++kb) {
          const int in_chain = kChains ? (kb - ti.kb0) % kChain : kb - ti.kb0;
          if (kChains && in_chain == 0 &&  // every chain has an accumulator of its own
              !mbar_wait(acc_empty_bar + 8 * acc, acc_phase ^ 1u, abort_flag, p.status, DICE_STATUS_WAIT_ACC_EMPTY)) {
            alive = false;
            break;
          }
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
          const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
          const uint32_t slot_smem = tiles_smem + stage * kSlotBytes;
          // 16 reduction elements further: 32 bytes along a K-major row, 16 rows of 128 bytes in an MN-major box
          constexpr uint64_t kStepA = MODE != MODE_TN ? 2 : 128, kStepB = MODE == MODE_NT ? 2 : 128;
          const bool chain_ends = kChains && (in_chain == kChain - 1 || kb == ti.kb1 - 1);
          constexpr int kProducts = PLANES == 3 ? 6 : 1;
          // (planes scaled by 2^16 together, by 2^8, by 1: the sum is brought to the next one's scale on the way)
          constexpr int kPlaneA[6] = {PLANES == 3 ? 2 : 0, 0, 1, 1, 0, 0}, kPlaneB[6] = {0, 2, 1, 0, 1, 0};
          if (elect_one()) {
#pragma unroll
            for (int q = 0; q < kProducts; ++q) {
              const uint32_t a_addr = slot_smem + kPlaneA[q] * kStageBytesT;
              const uint32_t b_addr = slot_smem + kPlaneB[q] * kStageBytesT + kOperandBytes;
              const uint64_t a_desc = MODE != MODE_TN ? make_operand_desc(a_addr) : make_mn_desc(a_addr);
              const uint64_t b_desc = MODE == MODE_NT ? make_operand_desc(b_addr) : make_mn_desc(b_addr);
#pragma unroll
              for (int kk = 0; kk < BK / UMMA_K; ++kk)
                if (kk < steps) {
                  if (PLANES == 3 && kk == 0 && (q == 3 || q == 5))
                    umma_bf16_pair_scaled(d_tmem, a_desc, b_desc, idesc);
                  else
                    umma_bf16_pair(d_tmem, a_desc + kk * kStepA, b_desc + kk * kStepB, idesc,
                                   static_cast<uint32_t>(in_chain != 0 || q != 0 || kk != 0));
                }
            }
            umma_commit_pair(empty_bar + 8 * stage);
            if (chain_ends) umma_commit_pair(acc_full_bar + 8 * acc);
          }
          __syncwarp();
          if (++stage == kStagesT) { stage = 0; phase ^= 1u; }
          if (chain_ends && ++acc == kAccStages) { acc = 0; acc_phase ^= 1u; }
        }
        if (!alive) break;
        if (!kChains) {
          if (elect_one()) umma_commit_pair(acc_full_bar + 8 * acc);
          __syncwarp();
          if (++acc == kAccStages) { acc = 0; acc_phase ^= 1u; }
        }
      }
    }
  } else if (warp == 2 + kEpilogueWarps) {
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
          if (!mbar_wait_behind(tail_bar + 8 * stage, (tail_phase >> stage) & 1u, filled, abort_flag, p.status)) break;
          tail_phase ^= 1u << stage;
          // rows [valid, next multiple of 16) of the four boxes (a row's 128 bytes are permuted within the row only)
          const int rows = 16 - (valid & 15);
          uint8_t* base = smem + stage * kSlotBytes + valid * 128;
          for (int i = lane; i < rows * 8; i += 32)
#pragma unroll
            for (int b = 0; b < 4 * PLANES; ++b) *reinterpret_cast<uint4*>(base + b * kBoxBytes + i * 16) = make_uint4(0, 0, 0, 0);
          fence_async_smem();
          fence_cluster();
          __syncwarp();
          if (lane == 0)
            mbar_complete_tx_cluster(map_to_cta(full_bar + 8 * stage, 0), PLANES * (kOperandBytes + (ti.n_mma > 128 ? 2 : 1) * kBoxBytes));
        }
        slot = (slot + blocks) % kStagesT;
      }
    }
  } else {
    // ---------------- epilogue (both CTAs, each over its own 128 rows) ----------------
    const int quad = warp & 3;
    const int half = (warp - 2) >> 2;  // which of the quadrant's warps: its share of the columns
    int acc = 0, seg = 0;
    uint32_t acc_phase = 0, xchg_phase = 0;
    Stager<buffers_of(EPI)> stager = {aux + kAuxBytes + (warp - 2) * buffers_of(EPI) * kStageStore, lane, 0, 0, false};
    for (int64_t t = pair_id; t < total; t += n_pairs) {
      const Tile ti = decode(t, seg);
      if (ti.zero && ti.share != 0) continue;
      const bool summed = ti.kb0 != ti.kb1;  // this share has something in tensor memory
      BackChunk<ACT, KEEP> kept;
      if (EPI == EPI_BACK) kept.load_first(p, ti.nb, half, ti.row0 + quad * 32 + lane, quad * 32 + lane < ti.rows_valid);
      f32x2 sums[kChains ? 4 : 1][16];  // this lane's row of the tile, columns half * 32 + 64 i ..
      if (kChains) {
        bool alive = true;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) sums[kChains ? i : 0][j] = 0;
        for (int kb = ti.kb0; kb < ti.kb1; kb += kChain) {
          if (!mbar_wait(acc_full_bar + 8 * acc, acc_phase, abort_flag, p.status, DICE_STATUS_WAIT_ACC_FULL)) {
            alive = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t t0 = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(acc * BN + half * 32);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (half * 32 + 64 * i < ti.n_mma) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t a[16];
                tmem_ld16(t0 + 64 * i + 16 * h, a);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  f32x2& sum = sums[kChains ? i : 0][8 * h + j];
                  sum = add2(sum, pair<f32x2>(__uint_as_float(a[2 * j]), __uint_as_float(a[2 * j + 1])));
                }
              }
            }
          }
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(map_to_cta(acc_empty_bar + 8 * acc, 0));
          if (++acc == kAccStages) { acc = 0; acc_phase ^= 1u; }
        }
        if (!alive) break;
      } else if (summed) {
        if (!mbar_wait(acc_full_bar + 8 * acc, acc_phase, abort_flag, p.status, DICE_STATUS_WAIT_ACC_FULL)) break;
        tc_fence_after_sync();
      }
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(acc * BN);
      const int col0 = ti.nb * bn;
      int n_valid = p.n_cols - col0;
      if (n_valid > bn) n_valid = bn;

      // the rows of the output that this lane stores pieces of (store_transposed): -1 beyond the segment or the gradient
      int64_t dst_row[4];
      bool up_rows = false;  // TN with gate_up: the peer's rows are the up projection's
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rr = quad * 32 + i * 8 + (lane >> 2);
        dst_row[i] = -1;
        if (rr < ti.rows_valid) {
          if (MODE != MODE_TN) {
            dst_row[i] = ti.row0 + rr;
          } else if (p.gate_up == 0) {
            dst_row[i] = static_cast<int64_t>(ti.slab) * p.m_rows + ti.row0 + rr;
          } else {
            // a pair's tile is a 128-row block of gate rows (leader) and its block of up rows (peer)
            const int r = ti.mb * BM + rr;
            up_rows = !leader;
            if (r < p.gate_up) dst_row[i] = static_cast<int64_t>(ti.slab) * p.gate_up + r;
          }
        }
      }
      stager.row0 = ti.row0 + quad * 32;
      stager.whole = ti.rows_valid >= quad * 32 + 32;
      // 32 bf16 columns from column c of a tensor with ld columns, of which n_left exist
      auto store_bf16 = [&](const uint4 (&w)[4], const CUtensorMap* map, __nv_bfloat16* base, int64_t ld, int c, int n_left) {
        stager.store(w, map, c, [&](int i, int piece, const uint4& v) {
          if (dst_row[i] >= 0 && piece * 8 < n_left) *reinterpret_cast<uint4*>(base + dst_row[i] * ld + c + piece * 8) = v;
        });
      };

      bool store = true;
      const bool shared_tile = split > 1 && !ti.zero;
      const int64_t part = (static_cast<int64_t>(cta_rank) * kEpilogueWarps + (warp - 2)) * kSplitFloats;
      constexpr int64_t kPairFloats = 2ll * kEpilogueWarps * kSplitFloats;
      if (shared_tile) {
        float* mine = p.split_ws + (ti.tile * split + ti.share) * kPairFloats + part + lane;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = half * 32 + 64 * i;
          if (c >= n_valid) break;
          float* dst = mine + i * 1024;
          if (kChains) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const two v = halves(sums[kChains ? i : 0][j]);
              dst[2 * j * 32] = v.x;
              dst[(2 * j + 1) * 32] = v.y;
            }
          } else {
            uint32_t a[32];
            if (summed) {
              tmem_ld32(taddr + c, a);
              tmem_ld_wait();
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) dst[j * 32] = summed ? __uint_as_float(a[j]) : 0.f;
          }
        }
        __threadfence();
        __syncwarp();
        unsigned int before = 0;
        if (lane == 0) before = atomicAdd(&p.split_count[(ti.tile * 2 + cta_rank) * kEpilogueWarps + (warp - 2)], 1u);
        store = __shfl_sync(0xffffffffu, before, 0) == static_cast<unsigned int>(split - 1);
        __threadfence();
      }
      const float* parts = shared_tile ? p.split_ws + ti.tile * split * kPairFloats + part + lane : nullptr;
      // 32 columns of the tile from column c on, of this lane's row
      auto fetch = [&](int c, float (&v)[32]) {
        if (shared_tile) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0.f;
          const float* src = parts + (c >> 6) * 1024;
#pragma unroll 2
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
      };

      if (kChains) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = half * 32 + 64 * i;
          if (!store || c >= n_valid) break;
          float v[32];
          if (shared_tile) {
            fetch(c, v);
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const two x = halves(sums[kChains ? i : 0][j]);
              v[2 * j] = x.x;
              v[2 * j + 1] = x.y;
            }
          }
          if (PLANES == 1) {
            const uint4 w[4] = {pack8(v), pack8(v + 8), pack8(v + 16), pack8(v + 24)};
            store_bf16(w, nullptr, up_rows ? p.out_up : p.out, p.n_cols, col0 + c, n_valid - c);
            continue;
          }
          float zero = 0.f;  // NaN if one of the values is not finite
#pragma unroll
          for (int j = 0; j < 32; ++j) zero = fmaf(v[j], 0.f, zero);
          if (zero != 0.f && quad * 32 + lane < ti.rows_valid) *static_cast<volatile unsigned int*>(p.non_finite) = 1u;
          float* const base = reinterpret_cast<float*>(up_rows ? p.out_up : p.out);
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // 16 columns are 64 bytes
            uint4 w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              w[j] = make_uint4(__float_as_uint(v[16 * h + 4 * j]), __float_as_uint(v[16 * h + 4 * j + 1]),
                                __float_as_uint(v[16 * h + 4 * j + 2]), __float_as_uint(v[16 * h + 4 * j + 3]));
            const int at = c + 16 * h, n_left = n_valid - at;
            stager.store(w, nullptr, 0, [&](int r, int piece, const uint4& x) {
              if (dst_row[r] >= 0 && piece * 4 < n_left)
                *reinterpret_cast<uint4*>(base + dst_row[r] * p.n_cols + col0 + at + piece * 4) = x;
            });
          }
        }
      } else if (EPI == EPI_PLAIN) {
        for (int c = half * 32; store && c < n_valid; c += 64) {
          float v[32];
          fetch(c, v);
          const uint4 w[4] = {pack8(v), pack8(v + 8), pack8(v + 16), pack8(v + 24)};
          store_bf16(w, nullptr, up_rows ? p.out_up : p.out, p.n_cols, col0 + c, n_valid - c);
        }
      } else if (EPI == EPI_KEEP) {
        keep_tile<ACT, KEEP>(p, ti.nb, quad, half, lane, ti.row0 + quad * 32 + lane, quad * 32 + lane < ti.rows_valid, dst_row,
                             stager, &tm_out, &tm_act, &tm_codes,
                             reinterpret_cast<float*>(aux + kAuxBytes + kEpilogueWarps * buffers_of(EPI) * kStageStore),
                             xchg_bar + 8 * quad, xchg_phase, abort_flag, fetch, store_bf16);
        xchg_phase ^= 1u;
      } else {
        back_tile<ACT, KEEP>(p, ti.nb, half, ti.row0 + quad * 32 + lane, quad * 32 + lane < ti.rows_valid, kept, &tm_out, &tm_act,
                             fetch, store_bf16);
      }
      if (!kChains && summed) {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_cta(acc_empty_bar + 8 * acc, 0));
        if (++acc == kAccStages) { acc = 0; acc_phase ^= 1u; }
      }
    }
    stager.finish();
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
template <int MODE, int EPI = EPI_PLAIN, int ACT = 0, int KEEP = 0, int PLANES = 1, bool LONG = false>
int resident_pairs_train() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (cached[dev] == 0) {
    if (cudaFuncSetAttribute(train_gemm_kernel<MODE, EPI, ACT, KEEP, PLANES, LONG>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_of(EPI, PLANES)) != cudaSuccess) return 0;
    const int sms = sm_count_cached();
    if (sms <= 0) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(sms & ~1), 1, 1);
    cfg.blockDim = dim3(threads_of(MODE), 1, 1);
    cfg.dynamicSmemBytes = smem_of(EPI, PLANES);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, train_gemm_kernel<MODE, EPI, ACT, KEEP, PLANES, LONG>, &cfg) != cudaSuccess || n <= 0) return 0;
    cached[dev] = n < sms / 2 ? n : sms / 2;
  }
  return cached[dev];
}

template <int MODE, int EPI = EPI_PLAIN, int ACT = 0, int KEEP = 0, int PLANES = 1, bool LONG = false>
int launch_train(const CUtensorMap& tm_a, const CUtensorMap& tm_b, const CUtensorMap* stores, const TrainGemm& p,
                 int64_t most_tiles, int pairs, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  const int64_t use = most_tiles < pairs && p.split_ws == nullptr ? most_tiles : pairs;
  cfg.gridDim = dim3(static_cast<unsigned>(2 * use), 1, 1);
  cfg.blockDim = dim3(threads_of(MODE), 1, 1);
  cfg.dynamicSmemBytes = smem_of(EPI, PLANES);
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
  return cudaLaunchKernelEx(&cfg, train_gemm_kernel<MODE, EPI, ACT, KEEP, PLANES, LONG>, tm_a, tm_b, stores[0], stores[1], stores[2], p) == cudaSuccess ? DICE_OK : DICE_ERR_CUDA;
}

int64_t col_tiles(int cols, int width) { return (static_cast<int64_t>(cols) + width - 1) / width; }

// scratch of a split: the counters (zeroed here), then every pair's sums
size_t counter_bytes(int pairs) { return (static_cast<size_t>(pairs) * 2 * kEpilogueWarps * sizeof(unsigned int) + 255) / 256 * 256; }
size_t split_bytes(int pairs) { return counter_bytes(pairs) + static_cast<size_t>(pairs) * 2 * kEpilogueWarps * kSplitFloats * sizeof(float); }
int use_scratch(TrainGemm& p, void* scratch, size_t scratch_bytes, int pairs, cudaStream_t s) {
  if (scratch == nullptr) return DICE_OK;
  if (scratch_bytes < split_bytes(pairs)) return DICE_ERR_SCRATCH;
  if (!dice_aligned16(scratch)) return DICE_ERR_ALIGN;
  if (cudaMemsetAsync(scratch, 0, counter_bytes(pairs), s) != cudaSuccess) return DICE_ERR_CUDA;
  p.split_count = static_cast<unsigned int*>(scratch);
  p.split_ws = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + counter_bytes(pairs));
  return DICE_OK;
}

}  // namespace

// What a split can use: 0 where it would not be made.  A weight gradient's tiles are known here; an input gradient's
// depend on the segments, of which at least the rows' own number of tiles exists (a quarter of the pairs at most, so that
// uneven segments still leave room).  Shares are at least four k-blocks of 64, so the reduction has to have eight.
size_t dice_internal_split_bytes(int64_t n_rows, int n_dim, int k_dim, int n_slabs, bool weight_gradient) {
  const int pairs = sm_count_cached() / 2;
  if (pairs <= 0 || n_rows == 0) return 0;
  const int64_t cols = col_tiles(k_dim, BN / 2);
  if (weight_gradient) {
    const int64_t tiles = static_cast<int64_t>(n_slabs) * ((n_dim + PM - 1) / PM) * cols;
    return 2 * tiles <= pairs && n_rows >= 2 * kMinSplitBlocks * BK ? split_bytes(pairs) : 0;
  }
  return 4 * ((n_rows + PM - 1) / PM) * cols <= pairs && n_dim >= 2 * kMinSplitBlocks * BK ? split_bytes(pairs) : 0;
}

int dice_internal_tc_dgrad(const void* dy, int64_t n_rows, int n_dim, const void* w, int n_slabs, int k_dim,
                           const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, void* dx, void* scratch,
                           size_t scratch_bytes, uint32_t* status, cudaStream_t s) {
  const bool is_long = n_dim > kLongBlocks * BK;
  const int pairs = is_long ? resident_pairs_train<MODE_NN, EPI_PLAIN, 0, 0, 1, true>() : resident_pairs_train<MODE_NN>();
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
  p.n_cols = k_dim;
  p.out = static_cast<__nv_bfloat16*>(dx);
  p.status = status;
  const CUtensorMap no_stores[3] = {tm_a, tm_a, tm_a};  // a plain epilogue stores from registers
  if ((rc = use_scratch(p, scratch, scratch_bytes, pairs, s)) != DICE_OK) return rc;
  const int64_t tiles = ((n_rows + PM - 1) / PM + n_seg) * col_tiles(k_dim, BN / 2);
  return is_long ? launch_train<MODE_NN, EPI_PLAIN, 0, 0, 1, true>(tm_a, tm_b, no_stores, p, tiles, pairs, s)
                 : launch_train<MODE_NN>(tm_a, tm_b, no_stores, p, tiles, pairs, s);
}

int dice_internal_tc_wgrad(const void* dy, const void* x, int64_t n_rows, int n_dim, int k_dim, const int32_t* seg_offsets,
                           int n_slabs, int gate_up, void* dw, void* dw_up, void* scratch, size_t scratch_bytes, uint32_t* status,
                           cudaStream_t s) {
  const bool is_long = n_rows > kLongBlocks * BK;
  const int pairs = is_long ? resident_pairs_train<MODE_TN, EPI_PLAIN, 0, 0, 1, true>() : resident_pairs_train<MODE_TN>();
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
  p.n_cols = k_dim;
  p.gate_up = gate_up;
  p.out = static_cast<__nv_bfloat16*>(dw);
  p.out_up = static_cast<__nv_bfloat16*>(dw_up);
  p.status = status;
  const CUtensorMap no_stores[3] = {tm_a, tm_a, tm_a};  // a plain epilogue stores from registers
  if ((rc = use_scratch(p, scratch, scratch_bytes, pairs, s)) != DICE_OK) return rc;
  const int64_t tiles = static_cast<int64_t>(n_slabs) * p.n_mblk * col_tiles(k_dim, BN / 2);
  return is_long ? launch_train<MODE_TN, EPI_PLAIN, 0, 0, 1, true>(tm_a, tm_b, no_stores, p, tiles, pairs, s)
                 : launch_train<MODE_TN>(tm_a, tm_b, no_stores, p, tiles, pairs, s);
}

namespace {

template <int ACT, int KEEP>
int run_keep(const CUtensorMap& tm_a, const CUtensorMap& tm_b, const CUtensorMap* st, const TrainGemm& p, cudaStream_t s) {
  const int pairs = resident_pairs_train<MODE_NT, EPI_KEEP, ACT, KEEP>();
  if (pairs <= 0) return DICE_ERR_CUDA;
  return launch_train<MODE_NT, EPI_KEEP, ACT, KEEP>(tm_a, tm_b, st, p, ((p.n_rows + PM - 1ll) / PM + p.n_seg) * col_tiles(p.n_cols, BN), pairs, s);
}
template <int ACT, int KEEP>
int run_back(const CUtensorMap& tm_a, const CUtensorMap& tm_b, const CUtensorMap* st, const TrainGemm& p, cudaStream_t s) {
  const int pairs = resident_pairs_train<MODE_NN, EPI_BACK, ACT, KEEP>();
  if (pairs <= 0) return DICE_ERR_CUDA;
  return launch_train<MODE_NN, EPI_BACK, ACT, KEEP>(tm_a, tm_b, st, p, ((p.n_rows + PM - 1ll) / PM + p.n_seg) * col_tiles(p.n_cols, BN), pairs, s);
}
template <int ACT>
int run_epilogue(bool back, int keep, const CUtensorMap& tm_a, const CUtensorMap& tm_b, const CUtensorMap* st, const TrainGemm& p, cudaStream_t s) {
  switch (keep) {
    case DICE_KEEP_INT8: return back ? run_back<ACT, DICE_KEEP_INT8>(tm_a, tm_b, st, p, s) : run_keep<ACT, DICE_KEEP_INT8>(tm_a, tm_b, st, p, s);
    case DICE_KEEP_NOTHING: return run_keep<ACT, DICE_KEEP_NOTHING>(tm_a, tm_b, st, p, s);  // (a backward pass has something)
    case DICE_KEEP_E4M3: return back ? run_back<ACT, DICE_KEEP_E4M3>(tm_a, tm_b, st, p, s) : run_keep<ACT, DICE_KEEP_E4M3>(tm_a, tm_b, st, p, s);
    default: return back ? run_back<ACT, DICE_KEEP_NONE>(tm_a, tm_b, st, p, s) : run_keep<ACT, DICE_KEEP_NONE>(tm_a, tm_b, st, p, s);
  }
}

void set_argument(TrainGemm& p, int ffn, int act) {
  const int blocks = (ffn + kKeepGroup - 1) / kKeepGroup;
  p.ffn = ffn;
  p.arg_cols = act == DICE_ACT_SWIGLU ? 2 * blocks * kKeepGroup : ffn;
  p.groups = act == DICE_ACT_SWIGLU ? 2 * blocks : blocks;
}

}  // namespace

int dice_internal_tc_keep(const void* rows, int64_t n_rows, int hidden, int ffn, int act, int keep, const void* w1, int n_slabs,
                          const int32_t* seg_offsets, int n_seg, void* pre, void* a, void* codes, float* scales,
                          uint32_t* status, cudaStream_t s) {
  TrainGemm p = {};
  set_argument(p, ffn, act);
  CUtensorMap tm_a, tm_b, stores[3];
  int rc = encode_map(&tm_a, rows, static_cast<uint64_t>(n_rows), static_cast<uint64_t>(hidden), BM);
  if (rc == DICE_OK)
    rc = encode_map(&tm_b, w1, static_cast<uint64_t>(n_slabs) * static_cast<uint64_t>(p.arg_cols), static_cast<uint64_t>(hidden), BK);
  // what is stored: pre (if it is kept), the activation, the codes
  if (rc == DICE_OK) rc = encode_store_map(&stores[1], a, n_rows, ffn, 2);
  stores[0] = stores[2] = stores[1];
  p.codes_tma = p.arg_cols % 16 == 0;
  if (rc == DICE_OK && keep == DICE_KEEP_NONE) rc = encode_store_map(&stores[0], pre, n_rows, p.arg_cols, 2);
  if (rc == DICE_OK && (keep == DICE_KEEP_INT8 || keep == DICE_KEEP_E4M3) && p.codes_tma) rc = encode_store_map(&stores[2], codes, n_rows, p.arg_cols, 1);
  if (rc != DICE_OK) return rc;
  p.seg_offsets = seg_offsets;
  p.n_seg = n_seg;
  p.n_slabs = n_slabs;
  p.n_rows = static_cast<int>(n_rows);
  p.red_blocks = (hidden + BK - 1) / BK;
  p.n_cols = p.arg_cols;
  p.out = static_cast<__nv_bfloat16*>(pre);
  p.act_out = static_cast<__nv_bfloat16*>(a);
  p.codes = static_cast<uint8_t*>(codes);
  p.scales = scales;
  p.status = status;
  return act == DICE_ACT_SWIGLU ? run_epilogue<DICE_ACT_SWIGLU>(false, keep, tm_a, tm_b, stores, p, s)
                                : run_epilogue<DICE_ACT_GELU_TANH>(false, keep, tm_a, tm_b, stores, p, s);
}

int dice_internal_tc_back(const void* d_out, int64_t n_rows, int hidden, int ffn, int act, int keep, const void* w2, int n_slabs,
                          const int32_t* seg_offsets, const void* kept, const float* scales, void* d_pre, void* a,
                          uint32_t* status, cudaStream_t s) {
  TrainGemm p = {};
  set_argument(p, ffn, act);
  CUtensorMap tm_a, tm_b, stores[3];
  int rc = encode_map(&tm_a, d_out, static_cast<uint64_t>(n_rows), static_cast<uint64_t>(hidden), BM);
  if (rc == DICE_OK)
    rc = encode_map3(&tm_b, w2, static_cast<uint64_t>(n_slabs), static_cast<uint64_t>(hidden), static_cast<uint64_t>(ffn), BK);
  if (rc == DICE_OK) rc = encode_store_map(&stores[0], d_pre, n_rows, p.arg_cols, 2);
  if (rc == DICE_OK) rc = encode_store_map(&stores[1], a, n_rows, ffn, 2);
  if (rc != DICE_OK) return rc;
  stores[2] = stores[1];
  p.seg_offsets = seg_offsets;
  p.n_seg = n_slabs;
  p.n_slabs = n_slabs;
  p.n_rows = static_cast<int>(n_rows);
  p.red_blocks = (hidden + BK - 1) / BK;
  p.n_cols = ffn;
  p.out = static_cast<__nv_bfloat16*>(d_pre);
  p.act_out = static_cast<__nv_bfloat16*>(a);
  p.kept = kept;
  p.kept_scales = scales;
  p.kept_wide = (reinterpret_cast<uintptr_t>(kept) & 31) == 0 && static_cast<int64_t>(p.arg_cols) * (keep == DICE_KEEP_NONE ? 2 : 1) % 32 == 0;
  p.status = status;
  return act == DICE_ACT_SWIGLU ? run_epilogue<DICE_ACT_SWIGLU>(true, keep, tm_a, tm_b, stores, p, s)
                                : run_epilogue<DICE_ACT_GELU_TANH>(true, keep, tm_a, tm_b, stores, p, s);
}

// ---- fp32 operands ------------------------------------------------------------------
namespace {

// x -> three planes of bf16, x == hi + 2^-8 mid + 2^-16 lo for every finite x, the smallest included.  A plane is the
// nearest to what the planes before it leave, times 2^8 for each of them.  Two tensors in one launch, eight values a thread.
// Rounded to nearest, which halves what the next plane has to hold twice over; the largest values, which would round to an
// infinity, are cut (what a cut leaves is below 2^-7 of the value: times 2^8 it is still finite).
__device__ __forceinline__ uint32_t nearest_plane(float x) {
  const uint32_t near = static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(x))) << 16;
  return (near & 0x7f800000u) == 0x7f800000u ? __float_as_uint(x) & 0xffff0000u : near;
}
struct PlaneJob {
  const float* x;
  __nv_bfloat16* planes;
  int64_t n;  // values (a multiple of 8), also the distance of the planes
};
__global__ void __launch_bounds__(256) split_planes_kernel(const PlaneJob first, const PlaneJob second, unsigned int* non_finite) {
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == 0 && threadIdx.x == 0) *non_finite = 0u;
  int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8;
  const bool in_first = i < first.n;
  if (!in_first) i -= first.n;
  const PlaneJob& job = in_first ? first : second;
  if (i >= job.n) return;
  const uint4 lo4 = ldg_stream16(job.x + i), hi4 = ldg_stream16(job.x + i + 4);
  const uint32_t raw[8] = {lo4.x, lo4.y, lo4.z, lo4.w, hi4.x, hi4.y, hi4.z, hi4.w};
  uint32_t plane[3][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = __uint_as_float(raw[j]);
    // a value that is not finite stays as it is, alone (a NaN whose payload is cut away would be an infinity)
    const bool finite = (raw[j] & 0x7f800000u) != 0x7f800000u;
    plane[0][j] = finite ? nearest_plane(x) : static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(x))) << 16;
    const float rest = finite ? (x - __uint_as_float(plane[0][j])) * 256.0f : 0.f;
    plane[1][j] = nearest_plane(rest);
    plane[2][j] = nearest_plane((rest - __uint_as_float(plane[1][j])) * 256.0f);
  }
#pragma unroll
  for (int q = 0; q < 3; ++q)
    stg_stream16(job.planes + q * job.n + i, make_uint4((plane[q][0] >> 16) | plane[q][1], (plane[q][2] >> 16) | plane[q][3],
                                                        (plane[q][4] >> 16) | plane[q][5], (plane[q][6] >> 16) | plane[q][7]));
}

constexpr size_t kFlagBytes = 256;  // at the scratch's end: whether a result is not finite
size_t plane_bytes(int64_t n) { return (static_cast<size_t>(n) * 6 + 255) / 256 * 256; }

}  // namespace

// Scratch of an fp32 product on the tensor cores: both operands' planes, and a split's parts.  0: the CUDA cores are the
// better place.  Where a weight takes part, making its planes has to be paid by enough rows of a slab, and three launches'
// worth of latency by enough work; a weight gradient's operands are the rows themselves.  Measured, CUDA cores / tensor
// cores, 8 slabs of 4608 x 1152: input gradient 64 rows a slab 155 / 183 us, 128 rows 287 / 185; weight gradient 32 rows
// 71 / 77, 64 rows 111 / 83.  One slab, 1000 rows, 512 x 256 (2^27 multiplications): 16 / 28; 4 slabs of 2000 rows, 256 x
// 512 (2^30): 69 / 27.
constexpr int kF32Rows = 96, kF32WgradRows = 48;
constexpr int64_t kF32Work = 1ll << 28;
size_t dice_internal_f32_bytes(int kind, int64_t n_rows, int n_dim, int k_dim, int n_slabs) {
  const int64_t limit = 0x7fffff00LL / 3;
  if (n_rows >= limit || static_cast<int64_t>(n_slabs) * n_dim >= limit) return 0;
  const int64_t w = static_cast<int64_t>(n_slabs) * n_dim * k_dim;
  if (kind == DICE_PRODUCT_WGRAD) {
    if (n_rows < kF32WgradRows * static_cast<int64_t>(n_slabs)) return 0;
    return plane_bytes(n_rows * n_dim) + plane_bytes(n_rows * k_dim) +
           dice_internal_split_bytes(n_rows, n_dim, k_dim, n_slabs, true) + kFlagBytes;
  }
  if (n_rows < kF32Rows * static_cast<int64_t>(n_slabs) || n_rows < kF32Work / (static_cast<int64_t>(n_dim) * k_dim)) return 0;
  const int a_cols = kind == DICE_PRODUCT_DGRAD ? n_dim : k_dim;
  const int out_cols = kind == DICE_PRODUCT_DGRAD ? k_dim : n_dim;
  return plane_bytes(n_rows * a_cols) + plane_bytes(w) + dice_internal_split_bytes(n_rows, a_cols, out_cols, n_slabs, false) + kFlagBytes;
}

// a, b: what the kind multiplies (forward rows and w, input gradient dy and w, weight gradient dy and x)
int dice_internal_f32_product(int kind, const void* a, const void* b, int64_t n_rows, int n_dim, int k_dim, int n_slabs,
                              const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, int gate_up, void* out,
                              void* out_up, void* scratch, size_t scratch_bytes, uint32_t* status, cudaStream_t s) {
  if (scratch_bytes < dice_internal_f32_bytes(kind, n_rows, n_dim, k_dim, n_slabs)) return DICE_ERR_SCRATCH;
  if (!dice_aligned16(scratch)) return DICE_ERR_ALIGN;
  const bool wgrad = kind == DICE_PRODUCT_WGRAD;
  const int64_t a_n = n_rows * (kind == DICE_PRODUCT_LINEAR ? k_dim : n_dim);
  const int64_t b_n = wgrad ? n_rows * k_dim : static_cast<int64_t>(n_slabs) * n_dim * k_dim;
  uint8_t* at = static_cast<uint8_t*>(scratch);
  const PlaneJob ja = {static_cast<const float*>(a), reinterpret_cast<__nv_bfloat16*>(at), a_n};
  at += plane_bytes(a_n);
  const PlaneJob jb = {static_cast<const float*>(b), reinterpret_cast<__nv_bfloat16*>(at), b_n};
  at += plane_bytes(b_n);
  const int64_t blocks = ((a_n + b_n) / 8 + 255) / 256;
  if (blocks > 0x7fffffffLL) return DICE_ERR_LIMIT;

  TrainGemm p = {};
  p.seg_offsets = seg_offsets;
  p.seg_slab = seg_slab;
  p.n_seg = n_seg;
  p.n_slabs = n_slabs;
  p.n_rows = static_cast<int>(n_rows);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_up = static_cast<__nv_bfloat16*>(out_up);
  p.status = status;
  p.a_plane = static_cast<int>(n_rows);
  CUtensorMap tm_a, tm_b;
  const uint64_t rows3 = 3 * static_cast<uint64_t>(n_rows), slabs3 = 3 * static_cast<uint64_t>(n_slabs);
  int rc, pairs;
  size_t split = 0;
  if (kind == DICE_PRODUCT_LINEAR) {
    rc = encode_map(&tm_a, ja.planes, rows3, static_cast<uint64_t>(k_dim), BM);
    if (rc == DICE_OK) rc = encode_map(&tm_b, jb.planes, slabs3 * static_cast<uint64_t>(n_dim), static_cast<uint64_t>(k_dim), BK);
    p.b_plane = n_slabs * n_dim;
    p.arg_cols = p.n_cols = n_dim;
    p.red_blocks = (k_dim + BK - 1) / BK;
    pairs = resident_pairs_train<MODE_NT, EPI_PLAIN, 0, 0, 3>();
    split = dice_internal_split_bytes(n_rows, k_dim, n_dim, n_slabs, false);
  } else if (kind == DICE_PRODUCT_DGRAD) {
    rc = encode_map(&tm_a, ja.planes, rows3, static_cast<uint64_t>(n_dim), BM);
    if (rc == DICE_OK) rc = encode_map3(&tm_b, jb.planes, slabs3, static_cast<uint64_t>(n_dim), static_cast<uint64_t>(k_dim), BK);
    p.b_plane = n_slabs;
    p.n_cols = k_dim;
    p.red_blocks = (n_dim + BK - 1) / BK;
    pairs = resident_pairs_train<MODE_NN, EPI_PLAIN, 0, 0, 3>();
    split = dice_internal_split_bytes(n_rows, n_dim, k_dim, n_slabs, false);
  } else {
    rc = encode_map(&tm_a, ja.planes, rows3, static_cast<uint64_t>(n_dim), BK);
    if (rc == DICE_OK) rc = encode_map(&tm_b, jb.planes, rows3, static_cast<uint64_t>(k_dim), BK);
    p.b_plane = static_cast<int>(n_rows);
    p.n_mblk = (n_dim + PM - 1) / PM;
    p.m_rows = n_dim;
    p.n_cols = k_dim;
    p.gate_up = gate_up;
    pairs = resident_pairs_train<MODE_TN, EPI_PLAIN, 0, 0, 3>();
    split = dice_internal_split_bytes(n_rows, n_dim, k_dim, n_slabs, true);
  }
  if (rc != DICE_OK) return rc;
  if (pairs <= 0) return DICE_ERR_CUDA;
  if (split > 0 && (rc = use_scratch(p, at, split, pairs, s)) != DICE_OK) return rc;
  p.non_finite = reinterpret_cast<unsigned int*>(at + split);
  if (dice_launch(split_planes_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, ja, jb, p.non_finite) != cudaSuccess)
    return DICE_ERR_CUDA;
  const CUtensorMap no_stores[3] = {tm_a, tm_a, tm_a};
  const int64_t tiles = (wgrad ? static_cast<int64_t>(n_slabs) * p.n_mblk : (n_rows + PM - 1) / PM + n_seg) * col_tiles(p.n_cols, BN / 2);
  if (kind == DICE_PRODUCT_LINEAR) rc = launch_train<MODE_NT, EPI_PLAIN, 0, 0, 3>(tm_a, tm_b, no_stores, p, tiles, pairs, s);
  else if (kind == DICE_PRODUCT_DGRAD) rc = launch_train<MODE_NN, EPI_PLAIN, 0, 0, 3>(tm_a, tm_b, no_stores, p, tiles, pairs, s);
  else rc = launch_train<MODE_TN, EPI_PLAIN, 0, 0, 3>(tm_a, tm_b, no_stores, p, tiles, pairs, s);
  if (rc != DICE_OK) return rc;
  return dice_internal_f32_repair(kind, a, b, n_rows, n_dim, k_dim, n_slabs, seg_offsets, seg_slab, n_seg, gate_up, out, out_up,
                                  p.non_finite, s);
}
