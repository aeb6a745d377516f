"""The expert FFN's training passes element by element: every tensor between their products is read back and compared with
64 bits, and every product with the tensors that it was made of (bounds as test_train_ops_gpu derives them)."""
import pytest
import torch
from test_train_ops_gpu import D, U, _act64, _check_product, _ffn_inputs, _gen, _parts, _read

from dice_b200 import _lib, ops

pytestmark = pytest.mark.gpu

# segments that end inside a group of 32 rows and on one, in the first and the second CTA of a pair's tile, and beyond it
COUNTS = [64, 33, 0, 31, 133, 1, 290]


def _ffn64(p, act, ffn):
    """act_columns of an argument in 64 bits -> which columns exist"""
    exists = torch.ones(p.shape[1], dtype=torch.bool, device=p.device)
    if act == "swiglu":
        exists[:] = False
        at = _parts(p, ffn)[2]
        exists[at] = exists[at + 128] = True
    return exists


@pytest.mark.parametrize("ffn", [64, 264, 392, 512, 1032])
@pytest.mark.parametrize("keep", ["int8", "e4m3", None])
@pytest.mark.parametrize("act", ["swiglu", "gelu_tanh"])
def test_forward_is_its_parts_bit_for_bit(cuda_device, act, keep, ffn):
    """bf16: the first product's epilogue leaves what grouped_gemm and act_keep leave after each other."""
    gen = _gen(30)
    h = 264
    rows, _, w1, w2, seg = _ffn_inputs(gen, COUNTS, h, ffn, act, torch.bfloat16, cuda_device)
    status = ops.device_status(cuda_device)
    out, kept = ops.grouped_ffn_train(rows, w1, w2, seg, act, ffn, keep=keep)
    pre = ops.grouped_gemm(rows, w1, seg, ops.EPI_STORE, w1.shape[1], status)
    a, kept2 = ops.act_keep(pre, act, ffn, keep=keep)
    assert torch.equal(kept.codes.view(torch.uint8), kept2.codes.view(torch.uint8))
    assert kept.scales is None if keep is None else torch.equal(kept.scales, kept2.scales)
    assert torch.equal(out, ops.grouped_gemm(a, w2, seg, ops.EPI_STORE, h, status))
    ops.check_status(status)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ffn", [64, 264, 392, 512, 1032])
@pytest.mark.parametrize("keep", ["int8", "e4m3", None])
@pytest.mark.parametrize("act", ["swiglu", "gelu_tanh"])
def test_backward_element_by_element(cuda_device, act, keep, ffn, dtype):
    """d_pre and the activation against 64 bits, from what was kept: the activation's gradient has the product's bound
    (it stays in fp32), which the slope carries on, the slope its own, and the result half a step.  Then each gradient
    against the product of these very tensors.  Rows before and behind the segments stay as they were."""
    gen = _gen(31)
    h, front, back = 264, 3, 40
    counts = [front, *COUNTS, back]
    rows, d_out, w1, w2, seg = _ffn_inputs(gen, counts, h, ffn, act, dtype, cuda_device)
    w1, w2, seg = w1[1:-1].contiguous(), w2[1:-1].contiguous(), seg[1:-1].contiguous()
    n, e, cols = rows.shape[0], len(COUNTS), w1.shape[1]
    _, kept = ops.grouped_ffn_train(rows, w1, w2, seg, act, ffn, keep=keep)
    full = lambda *s: torch.full(s, -7.0, dtype=dtype, device=cuda_device)  # noqa: E731
    da, d_pre, a, d_rows = full(n, ffn), full(n, cols), full(n, ffn), full(n, h)
    dw1, dw1_up, dw2 = full(e, ffn, h), full(e, ffn, h) if act == "swiglu" else None, full(e, h, ffn)
    lib, code = _lib.load(), ops._dtype_code(rows)
    held = [torch.empty(max(16, max(lib.dice_grouped_scratch_bytes(n, i, j, e, prod, code) for i, j in ((h, ffn), (cols, h))
                                    for prod in (ops.PRODUCT_DGRAD, ops.PRODUCT_WGRAD))), dtype=torch.uint8, device=cuda_device)]
    status = ops.device_status(cuda_device)
    ops._lib.check(lib.dice_grouped_ffn_backward(
        d_out.data_ptr(), rows.data_ptr(), kept.codes.data_ptr(), ops._ptr(kept.scales), n, h, ffn, ops.ACT_CODES[act],
        ops.KEEP_CODES[keep], code, w1.data_ptr(), w2.data_ptr(), e, seg.data_ptr(), da.data_ptr(), d_pre.data_ptr(),
        a.data_ptr(), d_rows.data_ptr(), dw1.data_ptr(), ops._ptr(dw1_up), dw2.data_ptr(), held[0].data_ptr(), held[0].numel(),
        status.data_ptr(), torch.cuda.current_stream().cuda_stream), "dice_grouped_ffn_backward")
    ops.check_status(status)
    inside = torch.zeros(n, dtype=torch.bool, device=cuda_device)
    inside[front:n - back] = True
    for t in (d_rows,) if dtype == torch.float32 else (d_rows, d_pre, a):  # (fp32: the scratch goes by rows, not by segments)
        assert bool((t[~inside] == -7).all())
    at = front
    for s, c in enumerate(COUNTS):
        cut = slice(at, at + c)
        at += c
        if c == 0:
            assert bool((dw2[s] == 0).all()) and bool((dw1[s] == 0).all()) and (dw1_up is None or bool((dw1_up[s] == 0).all()))
            continue
        x, g, b1, b2 = rows[cut].to(D), d_out[cut].to(D), w1[s].to(D), w2[s].to(D)
        p = _read(kept)[cut]
        ref_a, slopes, err, errs = _act64(p, act, ffn)
        assert bool(((a[cut].to(D) - ref_a).abs() <= U[dtype] * ref_a.abs() + 2 * err + 1e-36).all())
        da64, da_err = g @ b2, (h + 1) * 2.0 ** -23 * (g.abs() @ b2.abs())
        if dtype == torch.float32:  # (the kernel's own da is rounded to fp32)
            da_err = da_err + 2.0 ** -24 * da64.abs()
        exists = _ffn64(p, act, ffn)
        assert bool((d_pre[cut][:, ~exists] == 0).all())
        got = _parts(d_pre[cut].to(D), ffn)[:2] if act == "swiglu" else (d_pre[cut].to(D),)
        for have, slope, er in zip(got, slopes, errs):
            want = da64 * slope
            bound = (1 + 2.0 ** -7) * (slope.abs() + 2 * er) * da_err + U[dtype] * want.abs() + 2 * da64.abs() * er + 1e-36
            assert bool(((have - want).abs() <= bound).all()), float(((have - want).abs() / bound).max())
        dp, ac = d_pre[cut].to(D), a[cut].to(D)
        _check_product(d_rows[cut], dp @ b1, dp.abs() @ b1.abs(), cols, dtype)
        _check_product(dw2[s], g.T @ ac, g.abs().T @ ac.abs(), c, dtype)
        want, mass = dp.T @ x, dp.abs().T @ x.abs()
        if act == "swiglu":
            cols_at = _parts(p, ffn)[2]
            _check_product(dw1[s], want[cols_at], mass[cols_at], c, dtype)
            _check_product(dw1_up[s], want[cols_at + 128], mass[cols_at + 128], c, dtype)
        else:
            _check_product(dw1[s], want, mass, c, dtype)


@pytest.mark.parametrize("act", ["swiglu", "gelu_tanh"])
@pytest.mark.parametrize("keep", ["int8", None])
def test_bf16_step_as_far_as_its_roundings(cuda_device, act, keep):
    """Against 64 bits from the kept argument on, each result carries two roundings to bf16 (of the tensor that its product
    is made of, and its own): each moves a norm by at most 2^-8 / sqrt(3) of it, since a rounding is spread evenly over half
    a step at most; together sqrt(2) of that, 3.2e-3, with a tenth for the fp32 sums and chance."""
    gen = _gen(32)
    counts, h, ffn = [300, 0, 700], 384, 1032
    rows, d_out, w1, w2, seg = _ffn_inputs(gen, counts, h, ffn, act, torch.bfloat16, cuda_device)
    out, kept = ops.grouped_ffn_train(rows, w1, w2, seg, act, ffn, keep=keep)
    d_rows, dw1, dw2 = ops.grouped_ffn_backward(d_out, rows, kept, w1, w2, seg, act, ffn)
    tol, at = 1.1 * 2 ** 0.5 * 2.0 ** -8 / 3 ** 0.5, 0
    for s, c in enumerate(counts):
        cut = slice(at, at + c)
        at += c
        if c == 0:
            continue
        x, g, b1, b2 = rows[cut].to(D), d_out[cut].to(D), w1[s].to(D), w2[s].to(D)
        p = _read(kept)[cut]
        ref_a, slopes, _, _ = _act64(p, act, ffn)
        da = g @ b2
        dp = torch.zeros_like(p)
        if act == "swiglu":
            cols = _parts(p, ffn)[2]
            dp[:, cols], dp[:, cols + 128] = da * slopes[0], da * slopes[1]
        else:
            dp = da * slopes[0]
        pairs = [(d_rows[cut], dp @ b1), (dw2[s], g.T @ ref_a)]
        full = dp.T @ x
        pairs += [(dw1[0][s], full[cols]), (dw1[1][s], full[cols + 128])] if act == "swiglu" else [(dw1[s], full)]
        pre = (x @ b1.T).to(torch.bfloat16).to(D)
        pairs.append((out[cut], _act64(pre, act, ffn)[0] @ b2.T))
        for got, ref in pairs:
            assert float((got.to(D) - ref).norm() / ref.norm()) <= tol
