"""What the training path asks of a block and of its callers, as far as no GPU is needed."""
import inspect

import pytest
import torch

from dice_b200 import ops
from dice_b200.moe_block import ParaMode, SparseMoeBlock


def _block(k=2, **kw):
    return SparseMoeBlock(32, 2, 4, k, 1, 0, 1, ParaMode(), **kw).train()


@pytest.mark.parametrize("k", [1, 4])
def test_kernels_switched_on_after_construction(k):
    """The kernels gather rows two to a token: with four, they would read behind the tokens."""
    blk = _block(k)
    blk.train_kernels = True
    with pytest.raises(ValueError, match="two experts per token"):
        blk(torch.zeros(1, 3, 32))
    blk = _block()
    blk.train_kernels = True
    blk.gate.top_k = k
    with pytest.raises(ValueError, match="two experts per token"):
        blk(torch.zeros(1, 3, 32))
    blk = _block()
    blk.train_kernels = True
    blk.para_mode = ParaMode(ep=True)
    with pytest.raises(ValueError, match="expert parallelism"):
        blk(torch.zeros(1, 3, 32))


def test_block_without_the_attributes():
    """A block restored from a pickle of before train_kernels existed has neither attribute; it trains as it did."""
    blk = _block()
    del blk.__dict__["train_kernels"], blk.__dict__["train_keep"]
    x = torch.randn(1, 3, 32, requires_grad=True)
    blk(x).sum().backward()
    assert x.grad is not None


def test_float64_is_refused():
    """The default loop computes in 64 bits; the kernels have 32 at most and do not pretend otherwise."""
    with pytest.raises(TypeError, match="float64"):
        _block(train_kernels=True).double()(torch.zeros(1, 3, 32, dtype=torch.float64))
    blk = _block(train_kernels=True)
    blk.experts[1].double()
    with pytest.raises(TypeError, match="float64"):
        blk(torch.zeros(1, 3, 32))
    blk = _block(train_kernels=True)
    blk.shared_experts.double()
    with pytest.raises(TypeError, match="float64"):
        blk(torch.zeros(1, 3, 32))
    assert _block().double()(torch.zeros(1, 3, 32, dtype=torch.float64)).dtype == torch.float64


def test_nothing_is_quantised_unasked():
    assert _block(train_kernels=True).train_keep is None
    assert inspect.signature(ops.grouped_ffn_train).parameters["keep"].default is None


def test_single_tokens_ask_for_no_scratch():
    class Lib:
        asked = 0

        def dice_grouped_scratch_bytes(self, *args):
            self.asked += 1
            return 1 << 20

    lib = Lib()
    for rows in range(1, 5):
        assert ops._split_bytes(lib, rows, 9216, 1152, 8, ops.PRODUCT_DGRAD, ops.DICE_BF16) == 0
    assert lib.asked == 0
    assert ops._split_bytes(lib, 5, 9216, 1152, 8, ops.PRODUCT_DGRAD, ops.DICE_BF16) == 1 << 20


def test_train_dtype():
    assert _block().train_dtype is None
    with pytest.raises(ValueError, match="train_dtype"):
        _block(train_kernels=True, train_dtype=torch.float16)
    blk = _block()
    del blk.__dict__["train_dtype"]  # as a block pickled before it existed
    assert blk.train_dtype is None
