"""How far a training step of the block is from 64 bits, beside the torch loop's, and the choice of fp32."""
import copy

import pytest
import torch

from dice_b200 import ops
from dice_b200.moe_block import ParaMode, SparseMoeBlock

pytestmark = pytest.mark.gpu
D = torch.float64


def _far(got, ref):
    return float((got.detach().to(D) - ref).norm() / ref.norm())


def _setup(dev, act, **kw):
    torch.manual_seed(0)
    blk = SparseMoeBlock(192, 2, 8, 2, 1, 0, 1, ParaMode(), expert_act=act, train_kernels=True, **kw).to(dev).train()
    # the gate in fp32, so that every form routes alike
    forward = blk.gate.forward
    blk.gate.forward = lambda z: torch.autocast("cuda", enabled=False)(forward)(z.float())
    x = torch.randn(3, 160, 192, device=dev)
    return blk, x, torch.randn_like(x)


def _reference(blk, x, dy):
    """In 64 bits by the block's torch loop, with the gate's own decisions"""
    gate = blk.gate.forward
    del blk.gate.forward
    ref = copy.deepcopy(blk).double()
    blk.gate.forward = gate
    ref.train_kernels = False
    xr = x.double().requires_grad_()
    y = ref(xr)
    y.backward(dy.double())
    return {"y": y.detach(), "x": xr.grad, **{k: p.grad for k, p in ref.named_parameters()}}


def _step(blk, x, dy):
    blk.zero_grad()
    xx = x.clone().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = blk(xx)
    y.backward(dy)
    return {"y": y.detach(), "x": xx.grad, **{k: p.grad.clone() for k, p in blk.named_parameters()}}


@pytest.mark.parametrize("act", ["swiglu", "gelu_tanh"])
def test_bf16_step_is_about_as_near_as_the_loop(cuda_device, act):
    """The kernels round to bf16 at the products' operands and results; the loop there and, with SwiGLU, at every operation
    between them.  The kernels have one rounding of their own: the output's gradient, which they take in bf16 and the loop
    weights in fp32 first.  It moves a norm by at most 2^-8 / sqrt(3) and is independent of the others, so squares add up;
    a twentieth for chance.  (The gate's gradient hangs on one dot product a token and expert: half more is allowed.)"""
    blk, x, dy = _setup(cuda_device, act)
    ref = _reference(blk, x, dy)
    kernels = _step(blk, x, dy)
    blk.train_kernels = False
    loop = _step(blk, x, dy)
    for k, r in ref.items():
        most = (_far(loop[k], r) ** 2 + 2.0 ** -16 / 3) ** 0.5
        assert _far(kernels[k], r) <= (1.5 if "gate.weight" in k else 1.05) * most, (k, _far(kernels[k], r), _far(loop[k], r))


@pytest.mark.parametrize("act", ["swiglu", "gelu_tanh"])
def test_fp32_by_choice(cuda_device, act):
    """Under autocast, in fp32 all the same: the bound of test_train_block_gpu's fp32 step."""
    blk, x, dy = _setup(cuda_device, act, train_dtype=torch.float32)
    ref, got = _reference(blk, x, dy), _step(blk, x, dy)
    for k, r in ref.items():
        assert got[k].dtype == torch.float32
        assert _far(got[k], r) <= (64 if "gate.weight" not in k else 20 * 64) * 2.0 ** -24, (k, _far(got[k], r))
    ops.check_status(ops.device_status(cuda_device))


def test_fp32_by_choice_of_bf16_parameters(cuda_device):
    """A bf16 block: parameters, inputs and results are bf16, nothing between them is; a gradient carries its own rounding
    (2^-8 / sqrt(3) of its norm at most, a tenth for chance) and the output's gradient none."""
    blk, x, dy = _setup(cuda_device, "swiglu", train_dtype=torch.float32)
    blk, x, dy = blk.to(torch.bfloat16), x.to(torch.bfloat16), dy.to(torch.bfloat16)
    del blk.gate.forward
    gate = copy.deepcopy(blk.gate).float()
    blk.gate.forward = lambda z: gate(z.float())
    ref = copy.deepcopy(blk).double()
    ref.train_kernels = False
    ref.gate.forward = lambda z: tuple(t.double() if t is not None and t.is_floating_point() else t for t in gate(z.float()))
    xr = x.double().requires_grad_()
    ref(xr).backward(dy.double())
    xx = x.clone().requires_grad_()
    blk(xx).backward(dy)
    want = dict(ref.named_parameters())
    for k, p in blk.named_parameters():
        if "gate.weight" in k:
            continue
        assert p.grad.dtype == torch.bfloat16 and _far(p.grad, want[k].grad) <= 1.1 * 2.0 ** -8 / 3 ** 0.5, k
