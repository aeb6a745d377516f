"""Refusals of the training operators that need no GPU: the C ABI's host-side checks and the Python layer's."""
import pytest
import torch

from dice_b200 import _lib, ops
from dice_b200.moe_block import ParaMode, SparseMoeBlock


def test_c_abi_refuses_on_the_host():
    lib = _lib.load()
    P = 1 << 20  # a pointer that is aligned and never followed: every call below is refused before a launch
    dgrad = lambda n_rows=4, n=64, k=32, slabs=2, segs=2, dt=0, dy=P, w=P, out=P, seg=P, slab=None: lib.dice_grouped_dgrad(  # noqa: E731
        dy, n_rows, n, w, slabs, k, seg, slab, segs, dt, out, None, 0, None, None)
    assert dgrad(n=60) == -2 and dgrad(k=36) == -2
    assert dgrad(dt=7) == -3
    assert dgrad(segs=300, slabs=300) == -7 and dgrad(n_rows=1 << 31) == -7
    assert dgrad(segs=3) == -1  # more segments than slabs and no table that names their slabs
    assert dgrad(dy=None) == -1 and dgrad(dy=P + 8) == -4
    assert dgrad(n_rows=-1) == -1
    assert dgrad(n_rows=0, dy=None, w=None, out=None, seg=None) == 0
    wgrad = lambda n_rows=4, n=256, k=32, slabs=2, gu=0, dt=0, dw=P, up=P: lib.dice_grouped_wgrad(  # noqa: E731
        P, P, n_rows, n, k, P, slabs, gu, dt, dw, up, None, 0, None, None)
    assert wgrad(n=60) == -2 and wgrad(gu=200) == -2 and wgrad(gu=100) == -2  # 200 takes 512 packed columns; 100 is no multiple of 8
    assert wgrad(gu=128, up=None) == -1 and wgrad(dw=P + 4) == -4 and wgrad(slabs=257) == -7 and wgrad(gu=-1) == -1
    # no scratch without rows, for sizes that are refused, for an unknown product; fp32 planes take 6 bytes a value
    assert lib.dice_grouped_scratch_bytes(0, 4096, 64, 1, 0, 0) == 0 and lib.dice_grouped_scratch_bytes(0, 4096, 64, 1, 1, 1) == 0
    assert lib.dice_grouped_scratch_bytes(100, 60, 64, 1, 0, 0) == 0 and lib.dice_grouped_scratch_bytes(5000, 64, 64, 1, 3, 1) == 0
    assert lib.dice_grouped_scratch_bytes(4, 4096, 64, 1, 0, 1) == 0  # few rows: the CUDA cores
    assert lib.dice_grouped_scratch_bytes(5120, 512, 256, 2, 1, 1) >= 6 * 5120 * (512 + 256)
    assert lib.dice_grouped_scratch_bytes(5120, 512, 256, 2, 2, 1) >= 6 * (5120 * 256 + 2 * 512 * 256)
    keep = lambda ffn=64, act=0, kp=1, dt=0, codes=P, scales=P: lib.dice_act_keep(P, 4, ffn, act, kp, dt, P, codes, scales, None)  # noqa: E731
    assert keep(ffn=60) == -2 and keep(act=5) == -1 and keep(kp=9) == -1 and keep(dt=3) == -3
    assert keep(codes=None) == -1 and keep(scales=None) == -1 and keep(codes=P + 8) == -4
    back = lambda ffn=64, kp=1, scales=P, d_pre=P: lib.dice_act_backward(P, P, scales, 4, ffn, 0, kp, 0, d_pre, None, None)  # noqa: E731
    assert back(ffn=4) == -2 and back(scales=None) == -1 and back(d_pre=None) == -1 and back(d_pre=P + 2) == -4
    comb = lambda h=64, dt=0, pos=P, dw=P, tokens=4: lib.dice_combine_backward(P, P, pos, P, tokens, 8, h, dt, P, dw, None)  # noqa: E731
    assert comb(h=60) == -2 and comb(dt=9) == -3 and comb(pos=None) == -1 and comb(pos=P + 4) == -4 and comb(dw=P + 4) == -4
    assert comb(tokens=0, pos=None) == 0
    train = lambda act=0, h=64, ffn=64, segs=2, kp=1: lib.dice_grouped_ffn_train(  # noqa: E731
        P, 4, h, ffn, act, kp, 0, P, P, 2, P, segs, None, P, P, P, P, None, 0, None, None)
    assert train(act=7) == -1 and train(h=60) == -2 and train(ffn=12) == -2 and train(segs=3) == -1
    assert train(kp=0) == -1  # no buffer for the first product, which is what would be kept
    assert train(kp=5) == -1
    backward = lambda act=0, up=P, dw2=P, h=64: lib.dice_grouped_ffn_backward(  # noqa: E731
        P, P, P, P, 4, h, 64, act, 1, 0, P, P, 2, P, P, P, P, P, P, up, dw2, None, 0, None, None)
    assert backward(act=9) == -1 and backward(up=None) == -1 and backward(dw2=None) == -1 and backward(h=20) == -2


def test_cpu_tensors_are_refused():
    z, seg = torch.zeros(4, 64), torch.tensor([0, 4], dtype=torch.int32)
    w = torch.zeros(1, 64, 64)
    for call in (
        lambda: ops.grouped_dgrad(z, w, seg),
        lambda: ops.grouped_wgrad(z, z, seg),
        lambda: ops.act_keep(z, "gelu_tanh", 64),
        lambda: ops.act_backward(z, ops.KeptAct(z, None), "gelu_tanh", 64),
        lambda: ops.combine_backward(z, z, torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)),
        lambda: ops.grouped_ffn_train(z, w, w, seg, "gelu_tanh", 64),
        lambda: ops.grouped_ffn_backward(z, z, ops.KeptAct(z, None), w, w, seg, "gelu_tanh", 64),
    ):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    with pytest.raises(ValueError, match="int8"):
        ops.act_keep(z, "gelu_tanh", 64, keep="int4")
    with pytest.raises(ValueError, match="unknown activation"):
        ops.act_columns("relu", 64)
    assert ops.act_columns("swiglu", 130) == 512 and ops.act_columns("gelu_tanh", 136) == 136


def test_block_refusals():
    with pytest.raises(ValueError, match="train_keep"):
        SparseMoeBlock(32, 4, 8, 2, 1, 0, 1, ParaMode(), train_kernels=True, train_keep="fp4")
    with pytest.raises(ValueError, match="two experts per token"):
        SparseMoeBlock(32, 4, 8, 1, 1, 0, 1, ParaMode(), train_kernels=True)
    blk = SparseMoeBlock(32, 4, 8, 2, 1, 0, 1, ParaMode(), train_kernels=True).train()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        blk(torch.zeros(1, 4, 32))


def test_a_block_without_train_kernels_trains_as_before():
    torch.manual_seed(0)
    blk = SparseMoeBlock(32, 2, 4, 2, 1, 0, 1, ParaMode()).train()
    x = torch.randn(2, 5, 32, requires_grad=True)
    blk(x).sum().backward()
    assert x.grad is not None and blk.gate.weight.grad is not None and not blk.train_kernels


def test_result_that_shares_memory_with_an_operand():
    z = torch.zeros(10, 64)
    ops._check_out(z[:5], z[5:], torch.zeros(4))
    for out, operand in ((z, z), (z[:5], z[4:]), (z[2:4], z), (z, z.view(-1)[64:72])):
        with pytest.raises(ValueError, match="shares memory"):
            ops._check_out(out, torch.zeros(4), operand)
