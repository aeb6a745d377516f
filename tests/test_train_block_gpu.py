"""A SparseMoeBlock that trains its experts on the kernels against the same block in 64 bits and plain torch."""
import copy

import pytest
import torch

from dice_b200 import ops
from dice_b200.moe_block import ParaMode, SparseMoeBlock

pytestmark = pytest.mark.gpu
D = torch.float64


def _block(h, e, ratio, dev, **kw):
    torch.manual_seed(0)
    blk = SparseMoeBlock(h, ratio, e, 2, pretraining_tp=1, layer_idx=0, total_layers=1, para_mode=ParaMode(), train_kernels=True,
                         **kw).to(dev).train()
    return blk


def _reference(blk, x, dy):
    """Output and gradients in 64 bits by the block's plain training path."""
    ref = copy.deepcopy(blk).double()
    ref.train_kernels = False
    xr = x.detach().double().requires_grad_()
    y = ref(xr)
    y.backward(dy.double())
    return y.detach(), xr.grad, {k: p.grad for k, p in ref.named_parameters()}


def _far(got, ref):
    n = float(ref.norm())
    return float((got.to(D) - ref).norm()) / n if n else float(got.to(D).norm())


@pytest.mark.parametrize("act,shared,renorm", [("swiglu", True, False), ("gelu_tanh", False, True)])
@pytest.mark.parametrize("shape,h,e", [((1, 1), 64, 4), ((2, 67), 136, 8)])
def test_fp32_step(cuda_device, act, shared, renorm, shape, h, e):
    """Nothing is rounded on the way but to fp32.  The sums have at most 4h = 544 terms (the gate's gradient sums the two
    rows' dot products): 64 units of 2^-24 cover the square roots of all of them many times over in norm."""
    blk = _block(h, e, 4, cuda_device, expert_act=act, shared_expert=shared, train_keep=None)
    blk.gate.norm_topk_prob = renorm
    x = torch.randn(*shape, h, device=cuda_device, requires_grad=True)
    dy = torch.randn(*shape, h, device=cuda_device)
    y = blk(x)
    y.backward(dy)
    y_ref, dx_ref, grads = _reference(blk, x, dy)
    tol = 64 * 2.0 ** -24
    assert _far(y, y_ref) <= tol and _far(x.grad, dx_ref) <= tol
    for k, p in blk.named_parameters():
        g = p.grad if p.grad is not None else torch.zeros_like(p)
        r = grads[k] if grads[k] is not None else torch.zeros_like(p, dtype=D)
        assert g.dtype == p.dtype
        assert _far(g, r) <= (tol if "gate.weight" not in k else 20 * tol), k
    ops.check_status(ops.device_status(cuda_device))


@pytest.mark.parametrize("keep", ["int8", "e4m3", None])
@pytest.mark.parametrize("act", ["swiglu", "gelu_tanh"])
def test_bf16_step_under_autocast(cuda_device, keep, act):
    """Parameters and activations in fp32, products in bf16.  Up to eight roundings to bf16 (2^-8 each at most, as norms:
    operands, argument, activation, two gradients, outputs) lie on the way to a gradient; an argument kept in 8 bits is
    off by at most half a step: 1/254 of its group's maximum, which for normal values is below 4.5 of their deviation
    (int8: 1.8 %), or 2^-4 (e4m3).  The slopes carry that on at a factor of at most 1.2."""
    blk = _block(192, 8, 2, cuda_device, expert_act=act, train_keep=keep)
    x = torch.randn(3, 80, 192, device=cuda_device, requires_grad=True)
    dy = torch.randn(3, 80, 192, device=cuda_device)
    # the gate in fp32 (outside autocast it would be): the reference then routes alike
    gate = blk.gate.forward
    blk.gate.forward = lambda z: torch.autocast("cuda", enabled=False)(gate)(z)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = blk(x)
    y.backward(dy)
    del blk.gate.forward
    y_ref, dx_ref, grads = _reference(blk, x, dy)
    tol = 8 * 2.0 ** -8 + 1.2 * {"int8": 0.018, "e4m3": 2.0 ** -4, None: 0.0}[keep]
    assert y.dtype == torch.float32 and _far(y, y_ref) <= 8 * 2.0 ** -8 and _far(x.grad, dx_ref) <= tol
    for k, p in blk.named_parameters():
        assert p.grad.dtype == torch.float32 and _far(p.grad, grads[k]) <= tol, (k, _far(p.grad, grads[k]))


def test_parameters_may_change_between_calls_in_any_way(cuda_device):
    """An optimizer's in-place step, a write through .data (which no version counter sees) and a replaced parameter all
    reach the next forward call; gradients add up over two backward calls."""
    blk = _block(64, 4, 2, cuda_device, train_keep=None, shared_expert=False)
    x = torch.randn(1, 40, 64, device=cuda_device)
    y0 = blk(x).detach()
    with torch.no_grad():
        for e in blk.experts:
            e.down_proj.weight.data.mul_(2.0)
    y1 = blk(x).detach()
    assert _far(y1, 2 * y0.double()) <= 1e-6
    blk.experts[0].down_proj.weight = torch.nn.Parameter(torch.zeros_like(blk.experts[0].down_proj.weight))
    assert not torch.equal(blk(x), y1)
    for _ in range(2):
        blk(x).sum().backward()
    g = blk.experts[1].up_proj.weight.grad.clone()
    blk.zero_grad()
    blk(x).sum().backward()
    assert _far(g, 2 * blk.experts[1].up_proj.weight.grad.double()) <= 1e-6


def test_frozen_experts_and_inputs(cuda_device):
    blk = _block(64, 4, 2, cuda_device)
    for p in blk.experts[2].parameters():
        p.requires_grad_(False)
    blk(torch.randn(1, 40, 64, device=cuda_device)).sum().backward()
    assert all(p.grad is None for p in blk.experts[2].parameters())
    assert all(p.grad is not None for p in blk.experts[1].parameters())


def test_step_in_a_graph(cuda_device):
    blk = _block(128, 4, 2, cuda_device)
    params = list(blk.parameters())
    x = torch.randn(2, 33, 128, device=cuda_device, requires_grad=True)

    def step():
        with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
            y = blk(x)
        return [y.detach(), *torch.autograd.grad(y, [x, *params], torch.ones_like(y))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(2):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            params[0].mul_(1.01)
        g.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_memory_kept_in_8_bits(cuda_device):
    """Between forward and backward the kept argument takes half the bytes of bf16."""
    held = {}
    x = torch.randn(1, 4096, 256, device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    for keep in ("int8", None):
        blk = _block(256, 8, 4, cuda_device, shared_expert=False, train_keep=keep).to(torch.bfloat16)
        blk(x)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = blk(x)
        held[keep] = torch.cuda.memory_allocated() - before
        del y, blk
    cols = 2 * 8 * 256 // 2  # gate and up columns of a 1024-wide expert
    rows = 2 * 4096
    assert held[None] - held["int8"] >= rows * cols * (2 - 1 - 4 / 128) * 0.99


def test_no_tokens_and_retained_graphs(cuda_device):
    blk = _block(64, 4, 2, cuda_device, train_keep=None)
    x = torch.zeros(0, 5, 64, device=cuda_device, requires_grad=True)
    blk.gate.alpha = 0.0  # (the auxiliary loss is a mean over tokens)
    y = blk(x)
    assert y.shape == (0, 5, 64)
    y.sum().backward()
    assert x.grad.shape == x.shape and bool((blk.experts[0].up_proj.weight.grad == 0).all())
    x = torch.randn(1, 9, 64, device=cuda_device, requires_grad=True)
    y = blk(x).sum()
    first = torch.autograd.grad(y, [x, *blk.experts.parameters()], retain_graph=True)
    second = torch.autograd.grad(y, [x, *blk.experts.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with torch.no_grad():
        assert torch.equal(blk(x), blk(x))
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        torch.autograd.grad(blk(x).sum(), x, create_graph=True)
