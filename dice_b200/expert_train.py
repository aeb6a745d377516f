"""The expert part of the block's training step on the kernels: differentiable forms of "gather rows by expert,
expert FFN, gate-weighted sum" (models.py:313-320) and of the shared expert (models.py:355-357), used by
``SparseMoeBlock`` when it was built with ``train_kernels=True``.

What is kept for the backward pass of the first product is its result in 8 bits (``keep`` "int8" / "e4m3") or as it
is (None); the gathered rows are gathered again.  The experts' weights are stacked once per forward call, since the
optimizer changes them between calls.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import ops


def _first_order_only() -> None:
    """The kernels' gradients have no graph.  With create_graph=True one would be left out silently, since the saved
    tensors, not the incoming gradient, carry it."""
    if torch.is_grad_enabled():
        raise RuntimeError("train_kernels offers no gradients of gradients (create_graph=True)")


def _stack(act: str, ffn: int, dtype: torch.dtype, params: Sequence[torch.Tensor]):
    """Expert parameters, expert by expert (gate, up, down or fc1, fc2), as the kernels' stacked weights."""
    if act == "swiglu":
        gate, up, down = params[0::3], params[1::3], params[2::3]
        w1 = torch.empty((len(gate), ops.w13_rows(ffn), gate[0].shape[1]), dtype=dtype, device=gate[0].device)
        for slab, g, u in zip(w1, gate, up):
            ops.pack_w13(g.to(dtype), u.to(dtype), out=slab)
        return w1, torch.stack([p.to(dtype) for p in down])
    fc1, fc2 = params[0::2], params[1::2]
    return torch.stack([p.to(dtype) for p in fc1]), torch.stack([p.to(dtype) for p in fc2])


def _ffn_grads(ctx, d_out, rows, kept, w1, w2, seg, want_rows: bool, needs: Sequence[bool]):
    """The rows' gradient (None unless wanted) and the parameters', one each in their order; no product is made for
    gradients that nobody needs (frozen experts)."""
    n_firsts = 2 if ctx.act == "swiglu" else 1  # matrices of the first product
    per = n_firsts + 1
    want_w1, want_w2 = any(n for i, n in enumerate(needs) if i % per != n_firsts), any(needs[n_firsts::per])
    d_rows, dw1, dw2 = ops.grouped_ffn_backward(d_out, rows, kept, w1, w2, seg, ctx.act, ctx.ffn, want_rows=want_rows,
                                                want_w1=want_w1, want_w2=want_w2)
    stacks = [*(dw1 if ctx.act == "swiglu" and want_w1 else [dw1] * n_firsts), dw2]
    grads = [stacks[i % per][i // per].to(dt) if need else None for i, (need, dt) in enumerate(zip(needs, ctx.param_dtypes))]
    return d_rows, grads


def without_grad(*tensors: torch.Tensor):
    """Under torch.no_grad() autograd functions still see which inputs require gradients; without that, nothing is kept."""
    return tensors if torch.is_grad_enabled() else tuple(t.detach() for t in tensors)


class RoutedExperts(torch.autograd.Function):
    """``y[t] = sum_s weights[t, s] * expert[idx[t, s]](x[t])`` with gradients for ``x``, ``weights`` and every expert
    parameter.  ``x [N, h]`` bf16 or fp32, ``idx`` int64 ``[N, 2]``, ``weights`` fp32 ``[N, 2]``."""

    @staticmethod
    def forward(ctx, x, idx, weights, act: str, ffn: int, keep: Optional[str], *params):
        per_expert = 3 if act == "swiglu" else 2
        n_experts = len(params) // per_expert
        n = x.shape[0]
        x, weights = x.contiguous(), weights.contiguous()
        w1, w2 = _stack(act, ffn, x.dtype, params)
        pos, seg, _ = ops.permute_plan(idx.reshape(-1), n_experts)
        rows = ops.permute_rows(x, pos, 2)
        trains = any(ctx.needs_input_grad)
        rows_out, kept = ops.grouped_ffn_train(rows, w1, w2, seg, act, ffn, keep=keep, want_kept=trains)
        pos = pos.view(n, 2)
        y = ops.unpermute_combine(rows_out, pos[:, 0], rows_out, pos[:, 1], weights[:, 0], weights[:, 1], n)
        if trains:
            ctx.save_for_backward(x, pos, seg, weights, rows_out, w1, w2, *kept)
        ctx.act, ctx.ffn, ctx.param_dtypes = act, ffn, [p.dtype for p in params]
        return y

    @staticmethod
    def backward(ctx, dy):
        _first_order_only()
        x, pos, seg, weights, rows_out, w1, w2, codes, scales = ctx.saved_tensors
        n = x.shape[0]
        d_out, d_weights = ops.combine_backward(dy.contiguous(), rows_out, pos, weights)
        want_x, needs = ctx.needs_input_grad[0], ctx.needs_input_grad[6:]
        if not (want_x or any(needs)):
            return (None, None, d_weights, None, None, None, *[None] * len(needs))
        rows = ops.permute_rows(x, pos.view(-1), 2)
        d_rows, grads = _ffn_grads(ctx, d_out, rows, ops.KeptAct(codes, scales), w1, w2, seg, want_x, needs)
        dx = ops.unpermute_combine(d_rows, pos[:, 0], d_rows, pos[:, 1], None, None, n) if want_x else None
        return (dx, None, d_weights, None, None, None, *grads)


class DenseExpert(torch.autograd.Function):
    """One expert over all rows of ``x [N, h]`` (the block's shared expert)."""

    @staticmethod
    def forward(ctx, x, act: str, ffn: int, keep: Optional[str], *params):
        x = x.contiguous()
        w1, w2 = _stack(act, ffn, x.dtype, params)
        seg = torch.zeros(2, dtype=torch.int32, device=x.device)
        seg[1:].fill_(x.shape[0])
        trains = any(ctx.needs_input_grad)
        y, kept = ops.grouped_ffn_train(x, w1, w2, seg, act, ffn, keep=keep, want_kept=trains)
        if trains:
            ctx.save_for_backward(x, seg, w1, w2, *kept)
        ctx.act, ctx.ffn, ctx.param_dtypes = act, ffn, [p.dtype for p in params]
        return y

    @staticmethod
    def backward(ctx, dy):
        _first_order_only()
        x, seg, w1, w2, codes, scales = ctx.saved_tensors
        dx, grads = _ffn_grads(ctx, dy.contiguous(), x, ops.KeptAct(codes, scales), w1, w2, seg, ctx.needs_input_grad[0],
                               ctx.needs_input_grad[4:])
        return (dx, None, None, None, *grads)
