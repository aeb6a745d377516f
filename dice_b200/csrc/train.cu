// Entry points of the expert FFN's training step: the gradients of the products grouped by expert, and the whole
// forward and backward pass over expert-sorted rows.  Arguments are checked here, and the kernel is chosen: train_gemm.cu
// (tensor cores, bf16 and fp32), train_simt.cu (fp32 of few rows), train_thin.cu (bf16 input gradients of single tokens),
// train_rows.cu (row-wise operators); the second forward product in bf16 is the eval path's.
#include "train.cuh"

namespace {

constexpr int kMaxSegTrain = 256;

// what every grouped product asks of its sizes
int check_product(int64_t n_rows, int n_dim, int k_dim, int n_slabs, int n_seg, int dtype) {
  DICE_CHECK_ARG(n_rows >= 0 && n_dim > 0 && k_dim > 0 && n_slabs > 0 && n_seg >= 0, DICE_ERR_ARG);
  DICE_CHECK_ARG(dice_dtype_size(dtype) != 0, DICE_ERR_DTYPE);
  DICE_CHECK_ARG(n_dim % 8 == 0 && k_dim % 8 == 0, DICE_ERR_SHAPE);
  DICE_CHECK_ARG(n_seg <= kMaxSegTrain && n_rows < 0x7fffff00LL && n_dim <= (1 << 24) && k_dim <= (1 << 22) &&
                     static_cast<int64_t>(n_slabs) * n_dim < 0x7fffff00LL && static_cast<int64_t>(n_slabs) * k_dim < 0x7fffff00LL,
                 DICE_ERR_LIMIT);
  return DICE_OK;
}

}  // namespace

extern "C" size_t dice_grouped_scratch_bytes(int64_t n_rows, int n_dim, int k_dim, int n_slabs, int product, int dtype) {
  if (product < DICE_PRODUCT_DGRAD || product > DICE_PRODUCT_LINEAR || n_rows <= 0 ||
      check_product(n_rows, n_dim, k_dim, n_slabs, 0, dtype) != DICE_OK)
    return 0;
  if (dtype == DICE_F32) return dice_internal_f32_bytes(product, n_rows, n_dim, k_dim, n_slabs);
  if (product == DICE_PRODUCT_LINEAR || (product == DICE_PRODUCT_DGRAD && n_rows <= kThinTotal)) return 0;
  return dice_internal_split_bytes(n_rows, n_dim, k_dim, n_slabs, product == DICE_PRODUCT_WGRAD);
}

extern "C" int dice_grouped_dgrad(const void* dy, int64_t n_rows, int n_dim, const void* w, int n_slabs, int k_dim,
                                  const int32_t* seg_offsets, const int32_t* seg_slab, int n_seg, int dtype, void* dx,
                                  void* scratch, size_t scratch_bytes, uint32_t* status, void* stream) {
  const int rc = check_product(n_rows, n_dim, k_dim, n_slabs, n_seg, dtype);
  if (rc != DICE_OK) return rc;
  DICE_CHECK_ARG(seg_slab != nullptr || n_seg <= n_slabs, DICE_ERR_ARG);
  if (n_rows == 0 || n_seg == 0) return DICE_OK;
  DICE_CHECK_ARG(dy && w && seg_offsets && dx, DICE_ERR_ARG);
  DICE_CHECK_ARG(dice_aligned16(dy) && dice_aligned16(w) && dice_aligned16(dx), DICE_ERR_ALIGN);
  if (dtype == DICE_BF16 && n_rows <= kThinTotal)
    return dice_internal_thin_dgrad(dy, n_rows, n_dim, w, n_slabs, k_dim, seg_offsets, seg_slab, n_seg, dx, status,
                                    static_cast<cudaStream_t>(stream));
  // a product that has no use for scratch takes whatever it is given, and leaves it alone
  if (dice_grouped_scratch_bytes(n_rows, n_dim, k_dim, n_slabs, DICE_PRODUCT_DGRAD, dtype) == 0) scratch = nullptr;
  if (dtype == DICE_BF16)
    return dice_internal_tc_dgrad(dy, n_rows, n_dim, w, n_slabs, k_dim, seg_offsets, seg_slab, n_seg, dx, scratch,
                                  scratch_bytes, status, static_cast<cudaStream_t>(stream));
  if (scratch != nullptr)
    return dice_internal_f32_product(DICE_PRODUCT_DGRAD, dy, w, n_rows, n_dim, k_dim, n_slabs, seg_offsets, seg_slab, n_seg, 0, dx,
                                     nullptr, scratch, scratch_bytes, status, static_cast<cudaStream_t>(stream));
  return dice_internal_simt_dgrad(dy, n_rows, n_dim, w, n_slabs, k_dim, seg_offsets, seg_slab, n_seg, dx, status,
                                  static_cast<cudaStream_t>(stream));
}

extern "C" int dice_grouped_wgrad(const void* dy, const void* x, int64_t n_rows, int n_dim, int k_dim,
                                  const int32_t* seg_offsets, int n_slabs, int gate_up, int dtype, void* dw, void* dw_up,
                                  void* scratch, size_t scratch_bytes, uint32_t* status, void* stream) {
  const int rc = check_product(n_rows, n_dim, k_dim, n_slabs, n_slabs, dtype);
  if (rc != DICE_OK) return rc;
  DICE_CHECK_ARG(gate_up >= 0, DICE_ERR_ARG);
  DICE_CHECK_ARG(gate_up == 0 || (gate_up % 8 == 0 && static_cast<int64_t>(n_dim) == dice_w13_rows(gate_up)), DICE_ERR_SHAPE);
  DICE_CHECK_ARG(seg_offsets && dw && (gate_up == 0 || dw_up) && (n_rows == 0 || (dy && x)), DICE_ERR_ARG);
  DICE_CHECK_ARG(dice_aligned16(dy) && dice_aligned16(x) && dice_aligned16(dw) && dice_aligned16(dw_up), DICE_ERR_ALIGN);
  if (dice_grouped_scratch_bytes(n_rows, n_dim, k_dim, n_slabs, DICE_PRODUCT_WGRAD, dtype) == 0) scratch = nullptr;
  if (dtype == DICE_BF16)
    return dice_internal_tc_wgrad(dy, x, n_rows, n_dim, k_dim, seg_offsets, n_slabs, gate_up, dw, dw_up, scratch,
                                  scratch_bytes, status, static_cast<cudaStream_t>(stream));
  if (scratch != nullptr)
    return dice_internal_f32_product(DICE_PRODUCT_WGRAD, dy, x, n_rows, n_dim, k_dim, n_slabs, seg_offsets, nullptr, n_slabs, gate_up,
                                     dw, dw_up, scratch, scratch_bytes, status, static_cast<cudaStream_t>(stream));
  return dice_internal_simt_wgrad(dy, x, n_rows, n_dim, k_dim, seg_offsets, n_slabs, gate_up, dw, dw_up, status,
                                  static_cast<cudaStream_t>(stream));
}

extern "C" int dice_grouped_ffn_train(const void* rows_in, int64_t n_rows, int hidden, int ffn, int act, int keep, int dtype,
                                      const void* w1, const void* w2, int n_slabs, const int32_t* seg_offsets, int n_seg,
                                      void* pre, void* a, void* codes, float* scales, void* rows_out, void* scratch,
                                      size_t scratch_bytes, uint32_t* status, void* stream) {
  DICE_CHECK_ARG(act == DICE_ACT_SWIGLU || act == DICE_ACT_GELU_TANH, DICE_ERR_ARG);
  DICE_CHECK_ARG(ffn > 0 && n_seg <= n_slabs, DICE_ERR_ARG);
  const int64_t cols = act == DICE_ACT_SWIGLU ? dice_w13_rows(ffn) : ffn;
  DICE_CHECK_ARG(cols <= (1 << 22), DICE_ERR_LIMIT);
  int rc = check_product(n_rows, static_cast<int>(cols), hidden, n_slabs, n_seg, dtype);
  if (rc == DICE_OK) rc = check_product(n_rows, hidden, ffn, n_slabs, n_seg, dtype);
  if (rc != DICE_OK) return rc;
  if (n_rows == 0 || n_seg == 0) return DICE_OK;
  DICE_CHECK_ARG(rows_in && w1 && w2 && seg_offsets && a && rows_out, DICE_ERR_ARG);
  // bf16 keeps the first product in its epilogue: `pre` is written only when it is what is kept
  DICE_CHECK_ARG(pre || (dtype == DICE_BF16 && keep != DICE_KEEP_NONE), DICE_ERR_ARG);
  DICE_CHECK_ARG(dice_aligned16(rows_in) && dice_aligned16(w1) && dice_aligned16(w2) && dice_aligned16(pre) &&
                     dice_aligned16(a) && dice_aligned16(rows_out),
                 DICE_ERR_ALIGN);
  DICE_CHECK_ARG(keep == DICE_KEEP_NONE || keep == DICE_KEEP_INT8 || keep == DICE_KEEP_E4M3 || keep == DICE_KEEP_NOTHING, DICE_ERR_ARG);
  DICE_CHECK_ARG(keep == DICE_KEEP_NONE || keep == DICE_KEEP_NOTHING || (codes && scales), DICE_ERR_ARG);
  DICE_CHECK_ARG(dice_aligned16(codes), DICE_ERR_ALIGN);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == DICE_BF16) {
    rc = dice_internal_tc_keep(rows_in, n_rows, hidden, ffn, act, keep, w1, n_slabs, seg_offsets, n_seg, pre, a, codes, scales,
                               status, s);
    if (rc != DICE_OK) return rc;
    return dice_grouped_gemm(a, n_rows, ffn, w2, n_slabs, hidden, seg_offsets, nullptr, n_seg, DICE_EPI_STORE, rows_out,
                             hidden, hidden, 0, status, stream);
  }
  auto linear = [&](const void* in, int k_dim, const void* w, int n_dim, void* out) {
    if (scratch != nullptr && dice_internal_f32_bytes(DICE_PRODUCT_LINEAR, n_rows, n_dim, k_dim, n_slabs) > 0)
      return dice_internal_f32_product(DICE_PRODUCT_LINEAR, in, w, n_rows, n_dim, k_dim, n_slabs, seg_offsets, nullptr, n_seg, 0,
                                       out, nullptr, scratch, scratch_bytes, status, s);
    return dice_internal_simt_linear(in, n_rows, k_dim, w, n_slabs, n_dim, seg_offsets, nullptr, n_seg, out, status, s);
  };
  if ((rc = linear(rows_in, hidden, w1, static_cast<int>(cols), pre)) != DICE_OK) return rc;
  if ((rc = dice_act_keep(pre, n_rows, ffn, act, keep == DICE_KEEP_NOTHING ? DICE_KEEP_NONE : keep, dtype, a, codes, scales, stream)) != DICE_OK) return rc;
  return linear(a, ffn, w2, hidden, rows_out);
}

extern "C" int dice_grouped_ffn_backward(const void* d_out, const void* rows_in, const void* kept, const float* scales,
                                         int64_t n_rows, int hidden, int ffn, int act, int keep, int dtype, const void* w1,
                                         const void* w2, int n_slabs, const int32_t* seg_offsets, void* da, void* d_pre,
                                         void* a, void* d_rows, void* dw1, void* dw1_up, void* dw2, void* scratch,
                                         size_t scratch_bytes, uint32_t* status, void* stream) {
  DICE_CHECK_ARG(act == DICE_ACT_SWIGLU || act == DICE_ACT_GELU_TANH, DICE_ERR_ARG);
  DICE_CHECK_ARG(ffn > 0, DICE_ERR_ARG);
  const bool glu = act == DICE_ACT_SWIGLU;
  const int64_t cols = glu ? dice_w13_rows(ffn) : ffn;
  DICE_CHECK_ARG(cols <= (1 << 22), DICE_ERR_LIMIT);
  int rc = check_product(n_rows, hidden, ffn, n_slabs, n_slabs, dtype);
  if (rc == DICE_OK) rc = check_product(n_rows, static_cast<int>(cols), hidden, n_slabs, n_slabs, dtype);
  if (rc != DICE_OK) return rc;
  DICE_CHECK_ARG(seg_offsets && (!dw1 || (dw2 && (!glu || dw1_up))), DICE_ERR_ARG);
  DICE_CHECK_ARG(keep == DICE_KEEP_NONE || keep == DICE_KEEP_INT8 || keep == DICE_KEEP_E4M3, DICE_ERR_ARG);
  // a gradient whose pointer is NULL is not made, and without any there is nothing to do
  if (n_rows > 0 && (d_rows || dw2)) {
    DICE_CHECK_ARG(d_out && rows_in && kept && w1 && w2 && d_pre && a && (keep == DICE_KEEP_NONE || scales), DICE_ERR_ARG);
    DICE_CHECK_ARG(da || dtype == DICE_BF16, DICE_ERR_ARG);  // bf16: the activation's gradient stays in the epilogue
    DICE_CHECK_ARG(dice_aligned16(d_out) && kept_aligned(kept, keep) && dice_aligned16(w2) && dice_aligned16(d_pre) && dice_aligned16(a),
                   DICE_ERR_ALIGN);
    if (dtype == DICE_BF16) {
      rc = dice_internal_tc_back(d_out, n_rows, hidden, ffn, act, keep, w2, n_slabs, seg_offsets, kept, scales, d_pre, a, status,
                                 static_cast<cudaStream_t>(stream));
      if (rc != DICE_OK) return rc;
    } else {
      if ((rc = dice_grouped_dgrad(d_out, n_rows, hidden, w2, n_slabs, ffn, seg_offsets, nullptr, n_slabs, dtype, da,
                                   scratch, scratch_bytes, status, stream)) != DICE_OK)
        return rc;
      if ((rc = dice_act_backward(da, kept, scales, n_rows, ffn, act, keep, dtype, d_pre, a, stream)) != DICE_OK) return rc;
    }
  }
  const int c = static_cast<int>(cols);
  if (dw2 &&
      (rc = dice_grouped_wgrad(d_out, a, n_rows, hidden, ffn, seg_offsets, n_slabs, 0, dtype, dw2, nullptr,
                               scratch, scratch_bytes, status, stream)) != DICE_OK)
    return rc;
  if (d_rows &&
      (rc = dice_grouped_dgrad(d_pre, n_rows, c, w1, n_slabs, hidden, seg_offsets, nullptr, n_slabs, dtype, d_rows,
                               scratch, scratch_bytes, status, stream)) != DICE_OK)
    return rc;
  if (!dw1) return DICE_OK;
  return dice_grouped_wgrad(d_pre, rows_in, n_rows, c, hidden, seg_offsets, n_slabs, glu ? ffn : 0, dtype, dw1, dw1_up,
                            scratch, scratch_bytes, status, stream);
}
