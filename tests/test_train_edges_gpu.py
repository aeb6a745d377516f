"""The training operators where a gradient is not wanted, an argument is at its limit or a value at the end of its range.

Bounds are those of test_train_ops_gpu: half a step of the type for a rounding, K 2^-23 of the products' magnitudes for a
sum of K in fp32.
"""
import pytest
import torch

from dice_b200 import _lib, ops
from dice_b200.moe_block import ParaMode, SparseMoeBlock

pytestmark = pytest.mark.gpu
D = torch.float64


def _block(dev, act, dtype, **kw):
    torch.manual_seed(0)
    blk = SparseMoeBlock(64, 2, 4, 2, 1, 0, 1, ParaMode(), expert_act=act, train_kernels=True, **kw)
    return blk.to(dev, dtype).train()


def _launches(fn):
    before = _lib.load().dice_kernel_launches()
    out = fn()
    return out, _lib.load().dice_kernel_launches() - before


# ---- gradients that nobody needs -----------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ["swiglu", "gelu_tanh"])
def test_frozen_weights_cost_no_products(cuda_device, act, dtype):
    """With every expert frozen the backward pass makes the rows' gradients alone: two weight gradients fewer for the
    routed and two for the shared experts.  With inputs that need none, the rows' own."""
    x = torch.randn(1, 200, 64, device=cuda_device, dtype=dtype)
    dy = torch.randn_like(x)
    blk = _block(cuda_device, act, dtype)
    firsts = [n for n, _ in blk.named_parameters() if "expert" in n and ("gate_proj" in n or "up_proj" in n or "fc1" in n)]
    seconds = [n for n, _ in blk.named_parameters() if "expert" in n and n not in firsts]

    def step(frozen, want_x):
        params = dict(blk.named_parameters())
        for n, p in params.items():
            p.requires_grad_(n not in frozen)
            p.grad = None
        xx = x.clone().requires_grad_(want_x)
        y = blk(xx)
        _, n_launches = _launches(lambda: y.backward(dy))
        return n_launches, xx.grad, {n: p.grad for n, p in params.items()}

    full, dx, grads = step([], True)
    for frozen, want_x, fewer in [(firsts + seconds, True, 4), (firsts, True, 2), (seconds, True, 0), ([], False, 3),
                                  (firsts, False, 5)]:
        n_launches, dx2, grads2 = step(frozen, want_x)
        if dtype == torch.bfloat16:  # (fp32 has further launches for its operands)
            assert n_launches == full - fewer, (frozen, want_x)
        else:
            assert n_launches <= full - fewer
        assert torch.equal(dx, dx2) if want_x else dx2 is None
        for n, g in grads2.items():
            assert g is None if n in frozen else torch.equal(g, grads[n]), n
    # the gate alone: its weights' gradient needs the combine's, and no product
    n_launches, _, grads2 = step(firsts + seconds, False)
    assert n_launches == 1 and torch.equal(grads2["gate.weight"], grads["gate.weight"])


def test_ffn_backward_of_what_is_wanted(cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=gen, device=cuda_device).to(torch.bfloat16)  # noqa: E731
    rows, d_out, w1, w2 = rand(90, 64), rand(90, 64), rand(2, 256, 64), rand(2, 64, 128)
    seg = torch.tensor([0, 50, 90], dtype=torch.int32, device=cuda_device)
    _, kept = ops.grouped_ffn_train(rows, w1, w2, seg, "swiglu", 128)
    back = lambda **kw: ops.grouped_ffn_backward(d_out, rows, kept, w1, w2, seg, "swiglu", 128, **kw)  # noqa: E731
    d_rows, (gate, up), dw2 = back()
    assert back(want_rows=False, want_w1=False, want_w2=False) == (None, None, None)
    a = back(want_w1=False, want_w2=False)
    assert torch.equal(a[0], d_rows) and a[1] is None and a[2] is None
    a = back(want_rows=False, want_w1=False)
    assert a[0] is None and a[1] is None and torch.equal(a[2], dw2)
    a = back(want_rows=False, want_w2=False)  # dw2 comes along
    assert a[0] is None and torch.equal(a[1][0], gate) and torch.equal(a[1][1], up) and torch.equal(a[2], dw2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ["swiglu", "gelu_tanh"])
@pytest.mark.parametrize("ffn", [64, 200, 392])
def test_nothing_kept_where_nothing_follows(cuda_device, act, dtype, ffn):
    gen = torch.Generator(device="cuda").manual_seed(2)
    rand = lambda *s: torch.randn(*s, generator=gen, device=cuda_device).to(dtype)  # noqa: E731
    cols = ops.act_columns(act, ffn)
    rows, w1, w2 = rand(333, 72), rand(3, cols, 72), rand(3, 72, ffn)
    seg = torch.tensor([0, 300, 300, 333], dtype=torch.int32, device=cuda_device)
    for keep in (None, "int8", "e4m3"):
        out, kept = ops.grouped_ffn_train(rows, w1, w2, seg, act, ffn, keep=keep)
        out2, nothing = ops.grouped_ffn_train(rows, w1, w2, seg, act, ffn, keep=keep, want_kept=False)
        assert kept is not None and nothing is None and torch.equal(out, out2)
    ops.check_status(ops.device_status(cuda_device))


@pytest.mark.parametrize("keep", [None, "int8"])
def test_no_grad_in_training_mode_keeps_nothing(cuda_device, keep, monkeypatch):
    """The same bits as with gradients, and no kept argument."""
    blk = _block(cuda_device, "swiglu", torch.bfloat16, train_keep=keep)
    x = torch.randn(1, 100, 64, device=cuda_device, dtype=torch.bfloat16)
    want, real = blk(x).detach(), ops.grouped_ffn_train
    wanted = []

    def spy(*args, **kw):
        wanted.append(kw["want_kept"])
        return real(*args, **kw)

    monkeypatch.setattr(ops, "grouped_ffn_train", spy)
    with torch.no_grad():
        assert torch.equal(blk(x), want)
    assert wanted == [False, False]
    blk(x).sum().backward()
    assert wanted[2:] == [True, True]


# ---- scratch ------------------------------------------------------------------------------


def test_scratch_that_is_not_needed(cuda_device):
    """A product for which the size query says 0 leaves any scratch alone, whatever its size; one that has a use for
    scratch refuses too little."""
    lib = _lib.load()
    gen = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=gen, device=cuda_device).to(torch.bfloat16)  # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream
    n, k = 9216, 64
    for rows, needs in [(1, False), (4, False), (5, True), (300, True), (20000, False)]:
        assert (lib.dice_grouped_scratch_bytes(rows, n, k, 1, ops.PRODUCT_DGRAD, ops.DICE_BF16) > 0) == needs, rows
    small = torch.full((1024,), 7, dtype=torch.uint8, device=cuda_device)

    def dgrad(rows, scratch, n_bytes):
        dy, seg, out = rand(rows, n), torch.tensor([0, rows], dtype=torch.int32, device=cuda_device), None
        w = rand(1, n, k)
        out = torch.empty(rows, k, dtype=torch.bfloat16, device=cuda_device)
        rc = lib.dice_grouped_dgrad(dy.data_ptr(), rows, n, w.data_ptr(), 1, k, seg.data_ptr(), None, 1, ops.DICE_BF16,
                                    out.data_ptr(), scratch.data_ptr(), n_bytes, None, stream)
        return rc, out, ops.grouped_dgrad(dy, w, seg)

    for rows in (1, 4, 20000):
        rc, out, want = dgrad(rows, small, 1024)
        assert rc == 0 and torch.equal(out, want)
    assert dgrad(300, small, 1024)[0] < 0
    # a weight gradient with as many tiles as SM pairs, or a short reduction
    for rows, nn, kk in [(3000, 2048, 2056), (100, 64, 64)]:
        assert lib.dice_grouped_scratch_bytes(rows, nn, kk, 1, ops.PRODUCT_WGRAD, ops.DICE_BF16) == 0
        dy, x, seg = rand(rows, nn), rand(rows, kk), torch.tensor([0, rows], dtype=torch.int32, device=cuda_device)
        dw = torch.empty(1, nn, kk, dtype=torch.bfloat16, device=cuda_device)
        rc = lib.dice_grouped_wgrad(dy.data_ptr(), x.data_ptr(), rows, nn, kk, seg.data_ptr(), 1, 0, ops.DICE_BF16,
                                    dw.data_ptr(), None, small.data_ptr(), 1024, None, stream)
        assert rc == 0 and torch.equal(dw, ops.grouped_wgrad(dy, x, seg))
    assert bool((small == 7).all())


# ---- kept codes that are a part of a tensor ----------------------------------------------------


@pytest.mark.parametrize("keep", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ffn", [72, 136, 328])
def test_kept_codes_that_start_on_8_bytes(cuda_device, keep, dtype, ffn):
    """Rows of GELU codes are a multiple of 8 bytes long, and so is the start of a slice of them."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    rand = lambda *s: torch.randn(*s, generator=gen, device=cuda_device).to(dtype)  # noqa: E731
    rows, d_out, da, w1, w2 = rand(67, 64), rand(66, 64), rand(66, ffn), rand(2, ffn, 64), rand(2, 64, ffn)
    _, kept = ops.act_keep(rand(67, ffn), "gelu_tanh", ffn, keep=keep)
    part = ops.KeptAct(kept.codes[1:], kept.scales[1:])
    assert part.codes.data_ptr() % 16 == 8 and part.codes.is_contiguous()
    whole = ops.KeptAct(*(t.clone() for t in part))
    for a, b in zip(ops.act_backward(da, part, "gelu_tanh", ffn), ops.act_backward(da, whole, "gelu_tanh", ffn)):
        assert torch.equal(a, b)
    seg = torch.tensor([0, 40, 66], dtype=torch.int32, device=cuda_device)
    back = lambda k: ops.grouped_ffn_backward(d_out, rows[1:], k, w1, w2, seg, "gelu_tanh", ffn)  # noqa: E731
    assert all(torch.equal(a, b) for a, b in zip(back(part), back(whole)))
    out = ops.KeptAct(torch.empty(66 * ffn + 4, dtype=part.codes.dtype, device=cuda_device)[4:].view(66, ffn), part.scales)
    with pytest.raises(RuntimeError, match="aligned"):
        ops.act_backward(da, out, "gelu_tanh", ffn)


# ---- memory of the results ---------------------------------------------------------------------


def test_uninitialised_memory_is_filled_if_asked(cuda_device):
    """Deterministic algorithms fill what is left uninitialised with NaN (torch's own rule for torch.empty)."""
    dy, w = torch.ones(9, 64, device=cuda_device), torch.ones(1, 64, 72, device=cuda_device)
    seg = torch.tensor([2, 7], dtype=torch.int32, device=cuda_device)
    ops.grouped_dgrad(dy, w, seg)  # (its memory goes back to the cache, with 64 in it)
    torch.use_deterministic_algorithms(True)
    try:
        dx = ops.grouped_dgrad(dy, w, seg)
    finally:
        torch.use_deterministic_algorithms(False)
    assert bool(torch.isnan(dx[:2]).all()) and bool(torch.isnan(dx[7:]).all()) and bool((dx[2:7] == 64).all())


def test_dispatch_modes_see_the_allocations(cuda_device):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    x = torch.ones(9, 64, device=cuda_device)
    with Seen() as seen:
        ops.act_keep(x, "gelu_tanh", 64)
    assert sum("empty" in n for n in seen.names) == 3


# ---- fp32 over all of its range -------------------------------------------------------------------


def _check_f32(got, a, b, of_mass=0.0):
    """a, b in 64 bits; K 2^-23 of the magnitudes and half a step of the result, as test_train_ops_gpu derives it, and
    ``of_mass`` of the magnitudes"""
    ref, mass = a @ b, a.abs() @ b.abs()
    err, bound = (got.to(D) - ref).abs(), 2.0 ** -24 * ref.abs() + ((a.shape[1] + 1) * 2.0 ** -23 + of_mass) * mass
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("low,high", [(-126, 120), (-112, 100), (-100, 100), (100, -112), (120, -126)])
def test_fp32_planes_at_the_end_of_the_range(cuda_device, low, high):
    """Values whose last bits lie below what bf16 can hold, met by factors that bring them back into sight."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    rows, n, k = 440, 1032, 712
    seg = torch.tensor([0, 200, 200, 440], dtype=torch.int32, device=cuda_device)
    rand = lambda *s, e: (torch.randn(*s, generator=gen, device=cuda_device, dtype=D) * 2.0 ** e).float()  # noqa: E731
    dy, x, w = rand(rows, n, e=low), rand(rows, k, e=high), rand(3, n, k, e=high)
    for product in (ops.PRODUCT_DGRAD, ops.PRODUCT_WGRAD):
        assert ops._split_bytes(_lib.load(), rows, n, k, 3, product, ops.DICE_F32) >= 6 * rows * n
    dx, dw = ops.grouped_dgrad(dy, w, seg), ops.grouped_wgrad(dy, x, seg)
    w1 = w.transpose(1, 2).contiguous()
    _, kept = ops.grouped_ffn_train(dy, w1, torch.zeros_like(w), seg, "gelu_tanh", k)
    for s, (beg, end) in enumerate([(0, 200), (200, 200), (200, 440)]):
        a, b, g = dy[beg:end].to(D), w[s].to(D), x[beg:end].to(D)
        _check_f32(dx[beg:end], a, b)
        _check_f32(dw[s], a.T, g)
        _check_f32(kept.codes[beg:end], a, b)


def test_fp32_subnormals(cuda_device):
    """Subnormals have their bits in the second and the third plane, whose products with the other operand's second and
    third (at most 2^-9 and 2^-17 of it, what rounding to 8 and to 16 bits leaves) are left out: 2^-8 covers both.  The
    first plane alone, and any flush to zero, would be off by all of it."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    rows, n, k = 440, 1032, 712
    seg = torch.tensor([0, 440], dtype=torch.int32, device=cuda_device)
    rand = lambda *s, e: (torch.randn(*s, generator=gen, device=cuda_device, dtype=D) * 2.0 ** e).float()  # noqa: E731
    dy, x, w = rand(rows, n, e=-141), rand(rows, k, e=120), rand(1, n, k, e=120)
    _check_f32(ops.grouped_dgrad(dy, w, seg), dy.to(D), w[0].to(D), of_mass=2.0 ** -8)
    _check_f32(ops.grouped_wgrad(dy, x, seg)[0], dy.to(D).T, x.to(D), of_mass=2.0 ** -8)
    # a call without scratch is on the CUDA cores, and exact
    out = torch.empty(rows, k, device=cuda_device)
    rc = _lib.load().dice_grouped_dgrad(dy.data_ptr(), rows, n, w.data_ptr(), 1, k, seg.data_ptr(), None, 1, ops.DICE_F32,
                                        out.data_ptr(), None, 0, None, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    _check_f32(out, dy.to(D), w[0].to(D))


def test_one_small_value_among_ordinary_ones(cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(6)
    dy = torch.randn(300, 1032, generator=gen, device=cuda_device)
    dy[:, 7] = (dy[:, 7].double() * 2.0 ** -122).float()
    w = torch.zeros(1, 1032, 1160, device=cuda_device)
    w[0, 7] = (torch.randn(1160, generator=gen, device=cuda_device, dtype=D) * 2.0 ** 118).float()
    seg = torch.tensor([0, 300], dtype=torch.int32, device=cuda_device)
    assert ops._split_bytes(_lib.load(), 300, 1032, 1160, 1, ops.PRODUCT_DGRAD, ops.DICE_F32) > 0
    _check_f32(ops.grouped_dgrad(dy, w, seg), dy.to(D), w[0].to(D))


def _products(dy, x, w, seg):
    """dx, dw and the forward product (rows dy) of one call each"""
    w1 = w.transpose(1, 2).contiguous()
    _, kept = ops.grouped_ffn_train(dy, w1, torch.zeros_like(w), seg, "gelu_tanh", w.shape[2])
    return ops.grouped_dgrad(dy, w, seg), ops.grouped_wgrad(dy, x, seg), kept.codes


@pytest.mark.parametrize("rows,n,k", [(40, 1032, 712), (440, 1032, 712), (513, 2048, 72), (3000, 264, 328)])
def test_fp32_infinities_stay_infinities(cuda_device, rows, n, k):
    """Whether few rows or many (CUDA cores, or planes on the tensor cores): an infinity meets factors that are not zero and
    stays one, of the right sign; with its like of the other sign, or a zero, it is NaN; nothing else changes a bit."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    cut = rows * 3 // 5
    seg = torch.tensor([0, cut, cut, rows - 1], dtype=torch.int32, device=cuda_device)  # the last row is nobody's
    dy, x, w = (torch.randn(*s, generator=gen, device=cuda_device) for s in ((rows, n), (rows, k), (3, n, k)))
    want = _products(dy, x, w, seg)
    inf = float("inf")
    dy2, x2, w2 = dy.clone(), x.clone(), w.clone()
    dy2[1, 3], dy2[cut, 4], dy2[cut, 5], dy2[rows - 1] = inf, inf, inf, inf
    w2[0, 3, 9], w2[0, 6, 11], x2[2, 13], x2[rows - 1] = 0.0, -inf, -inf, float("nan")
    w2[1] = float("nan")  # an expert without rows
    got = _products(dy2, x2, w2, seg)
    ref64 = []
    for a, b in (((dy2, w2),) * 2):
        ref64.append(torch.cat([dy2[:cut].double() @ w2[0].double(), dy2[cut:rows - 1].double() @ w2[2].double()]))
    dw64 = torch.stack([dy2[:cut].double().T @ x2[:cut].double(), torch.zeros(n, k, device=cuda_device, dtype=D),
                        dy2[cut:rows - 1].double().T @ x2[cut:rows - 1].double()])
    for g, ref, clean in ((got[0][:rows - 1], ref64[0], want[0][:rows - 1]), (got[1], dw64, want[1]),
                          (got[2][:rows - 1], ref64[1], want[2][:rows - 1])):
        odd = ~torch.isfinite(ref)
        assert 0 < int(odd.sum()) < odd.numel()
        assert torch.equal(torch.isnan(g), torch.isnan(ref)) and torch.equal(g[odd].nan_to_num(7.0), ref[odd].float().nan_to_num(7.0))
        same = ~odd
        if g.shape == got[0][:rows - 1].shape and g is not got[1]:
            same[:, 9] = False  # (the weight that was set to zero)
            same[:cut, 9] = False
        assert torch.equal(g[same], clean[same])
    # and without the infinities again: the clean bits (nothing stays of the call before)
    assert all(torch.equal(a[:rows - 1], b[:rows - 1]) for a, b in zip(_products(dy, x, w, seg), want))
    ops.check_status(ops.device_status(cuda_device))


@pytest.mark.parametrize("rows", [40, 600])
def test_fp32_products_that_overflow(cuda_device, rows):
    """Finite values whose products overflow in one direction: an infinity, as fp32 sums give it, not NaN; a neighbour
    whose values fit keeps every bit."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    n, k = 1032, 712
    seg = torch.tensor([0, rows], dtype=torch.int32, device=cuda_device)
    dy, x, w = (torch.rand(*s, generator=gen, device=cuda_device) + 0.5 for s in ((rows, n), (rows, k), (1, n, k)))
    want = _products(dy, x, w, seg)
    dy2, x2, w2 = dy.clone(), x.clone(), w.clone()
    dy2[5] *= 2.0 ** 90
    w2[0, :, 7] *= -2.0 ** 90
    x2[:, 11] *= -2.0 ** 127  # times dy[5]: beyond the range whatever the rest
    x2[:, 11] = x2[:, 11].clamp(min=-3e38)
    dx, dw, fwd = _products(dy2, x2, w2, seg)
    for g, clean in ((dx, want[0]), (fwd, want[2])):
        assert bool((g[5, 7] == -float("inf")).all()) and bool(torch.isfinite(g[5, :7]).all()) and bool(torch.isfinite(g[:5, 7]).all())
        others = torch.ones_like(g, dtype=torch.bool)
        others[5], others[:, 7] = False, False
        assert torch.equal(g[others], clean[others])
    assert bool((dw[0, :, 11] == -float("inf")).all()) and bool(torch.isfinite(dw[0, :, :11]).all())


@pytest.mark.parametrize("ffn", [200, 328])
def test_fp32_infinities_with_gate_and_up_apart(cuda_device, ffn):
    gen = torch.Generator(device="cuda").manual_seed(10)
    cols, k = ops.w13_rows(ffn), 328
    seg = torch.tensor([0, 300, 500], dtype=torch.int32, device=cuda_device)
    dy, x = (torch.randn(500, c, generator=gen, device=cuda_device) for c in (cols, k))
    dy[7, 130], dy[400, 3], x[310, 17] = float("inf"), -float("inf"), float("inf")
    packed = ops.grouped_wgrad(dy, x, seg).unflatten(1, (-1, 2, 128))
    gate, up = ops.grouped_wgrad(dy, x, seg, gate_up=ffn)
    for got, part in ((gate, 0), (up, 1)):
        want = packed[:, :, part].flatten(1, 2)[:, :ffn]
        assert torch.equal(got.nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0))
    ref = torch.stack([dy[:300].double().T @ x[:300].double(), dy[300:].double().T @ x[300:].double()]).unflatten(1, (-1, 2, 128))
    assert torch.equal(torch.isnan(packed), torch.isnan(ref)) and torch.equal(torch.isinf(packed), torch.isinf(ref))


def test_fp32_infinities_in_a_graph(cuda_device):
    """Captured without an infinity, replayed with one and without again."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    dy, w = torch.randn(300, 1032, generator=gen, device=cuda_device), torch.randn(1, 1032, 1160, generator=gen, device=cuda_device)
    seg = torch.tensor([0, 300], dtype=torch.int32, device=cuda_device)
    clean = ops.grouped_dgrad(dy, w, seg)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx = ops.grouped_dgrad(dy, w, seg)
    for value in (float("inf"), 1.0, float("inf"), 1.0):
        before = dy[3, 3].clone()
        dy[3, 3] *= value
        graph.replay()
        torch.cuda.synchronize()
        assert bool(torch.isinf(dx[3]).all()) == (value != 1.0) and not bool(torch.isnan(dx).any())
        dx2 = dx.clone()
        dx2[3] = clean[3]
        assert torch.equal(dx2, clean)
        dy[3, 3] = before


# ---- long calls ---------------------------------------------------------------------------------------


def test_ragged_end_behind_a_second_of_work(cuda_device):
    """The first segment's reduction is whole, the second one's is not: the warp that zeroes ragged ends has nothing to do
    for over a second (2.8e14 multiply-adds' operations at some 220 TFLOP/s), which is no reason to give up."""
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("takes 80 GB")
    gen = torch.Generator(device="cuda").manual_seed(12)
    rows, n = 32768, 65536
    dy, x = (torch.randn(rows + 5, n, generator=gen, device=cuda_device) for _ in range(2))
    seg = torch.tensor([0, rows, rows + 5], dtype=torch.int32, device=cuda_device)
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    dw = ops.grouped_wgrad(dy, x, seg)
    stop.record()
    ops.check_status(ops.device_status(cuda_device))
    assert start.elapsed_time(stop) > 1000
    at = torch.arange(0, n, 4099, device=cuda_device)
    for s, (beg, end) in enumerate([(0, rows), (rows, rows + 5)]):
        _check_f32(dw[s][at][:, at], dy[beg:end, at].to(D).T.contiguous(), x[beg:end, at].to(D))
    del dw, dy, x
    torch.cuda.empty_cache()


def _sums_of_one_sign(dev, rows, n, k):
    """Values of one sign with all their 8 bits: a sum that is cut after every few products falls behind.  The second
    operand's columns have factors of their own, so that the results' roundings differ from column to column."""
    gen = torch.Generator(device="cuda").manual_seed(13)
    rand = lambda *s: torch.rand(*s, generator=gen, device=dev) + 1  # noqa: E731
    return rand(rows, n).to(torch.bfloat16), (rand(rows, k) * rand(1, k)).to(torch.bfloat16)


def _check_sums_of_one_sign(got, ref):
    """Half a step of the result (2^-8 of the value), 2^-12 of it for the accumulator's cuts over at most 32768 of the
    reduction (2048 instructions of up to 2^-23 each), and roundings to nearest of 2^-24 for every chain of 32768 and every
    share (fewer than 128): 2^-17.  In the mean the first averages out: roundings spread over +-2^-8 have a deviation of
    2^-8 / sqrt(3), of which four, over the square root of the number of columns, are allowed."""
    err = (got.to(D) - ref) / ref
    assert bool((err.abs() <= 2.0 ** -8 + 2.0 ** -12 + 2.0 ** -17).all()), float(err.abs().max())
    assert abs(float(err.mean())) <= 2.0 ** -12 + 2.0 ** -17 + 4 * 2.0 ** -8 / (3 * ref.shape[1]) ** 0.5, float(err.mean())


@pytest.mark.parametrize("counts,n,k", [([1 << 21], 264, 136), ([700001, 0, 13, 1 << 20], 136, 264), ([32768, 32769], 264, 328)])
@pytest.mark.parametrize("scratch", [True, False])
def test_long_sums_of_one_sign(cuda_device, counts, n, k, scratch):
    """A bf16 weight gradient over many rows: the error does not grow with them."""
    rows = sum(counts)
    dy, x = _sums_of_one_sign(cuda_device, rows, n, k)
    seg = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device=cuda_device)
    if scratch:
        dw = ops.grouped_wgrad(dy, x, seg)
    else:
        dw = torch.empty(len(counts), n, k, dtype=torch.bfloat16, device=cuda_device)
        rc = _lib.load().dice_grouped_wgrad(dy.data_ptr(), x.data_ptr(), rows, n, k, seg.data_ptr(), len(counts), 0, ops.DICE_BF16,
                                            dw.data_ptr(), None, None, 0, None, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
    beg = 0
    for s, c in enumerate(counts):
        ref = torch.zeros(n, k, dtype=D, device=cuda_device)
        for at in range(beg, beg + c, 1 << 18):
            end = min(at + (1 << 18), beg + c)
            ref += dy[at:end].to(D).T @ x[at:end].to(D)
        if c:
            _check_sums_of_one_sign(dw[s], ref)
        else:
            assert bool((dw[s] == 0).all())
        beg += c
    ops.check_status(ops.device_status(cuda_device))


def test_long_input_gradient_of_one_sign(cuda_device):
    dy, w = _sums_of_one_sign(cuda_device, 300, 1 << 19, 8)[0], _sums_of_one_sign(cuda_device, 1 << 19, 136, 8)[0]
    seg = torch.tensor([0, 300], dtype=torch.int32, device=cuda_device)
    ref = dy.to(D) @ w.to(D)
    for scratch in (True, False):
        dx = torch.empty(300, 136, dtype=torch.bfloat16, device=cuda_device)
        if scratch:
            ops.grouped_dgrad(dy, w.unsqueeze(0), seg, out=dx)
        else:
            rc = _lib.load().dice_grouped_dgrad(dy.data_ptr(), 300, 1 << 19, w.data_ptr(), 1, 136, seg.data_ptr(), None, 1,
                                                ops.DICE_BF16, dx.data_ptr(), None, 0, None, torch.cuda.current_stream().cuda_stream)
            assert rc == 0
        _check_sums_of_one_sign(dx, ref)


# ---- activation at the end of the range -------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ["swiglu", "gelu_tanh"])
@pytest.mark.parametrize("keep", ["int8", "e4m3", None])
def test_slopes_of_large_arguments(cuda_device, dtype, act, keep):
    """Far out an activation is the identity or zero: slope 1 or 0, not infinity times zero."""
    magnitudes = torch.tensor([2.0 ** e for e in (5, 8, 20, 60, 64, 65, 66, 90, 127)], dtype=D)
    for big in magnitudes.tolist():
        pre = torch.zeros(2, ops.act_columns(act, 128), dtype=dtype, device=cuda_device)
        pre[0, :128], pre[1, :128] = big, -big
        if act == "swiglu":
            pre[:, 128:] = 0.5
        a, kept = ops.act_keep(pre, act, 128, keep=keep)
        d_pre, a2 = ops.act_backward(torch.ones(2, 128, dtype=dtype, device=cuda_device), kept, act, 128)
        unit = 0.5 if act == "swiglu" else 1.0
        # the 8-bit codes' scale and factor are rounded to fp32: 2^-22, and half a step of the type
        for got, want in ((a[0], unit * big), (a2[0], unit * big), (d_pre[0, :128], unit)):
            assert bool(((got.to(D) - want).abs() <= (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -21) * want).all()), big
        # below zero: e^-32 of 2^5 at most
        for got in (a[1], a2[1], d_pre[1, :128]):
            assert bool((got.to(D).abs() <= 2.0 ** 5 * 2.0 ** -46).all()), big


@pytest.mark.parametrize("big", [2.0 ** 65, 2.0 ** 100])
def test_slopes_of_large_arguments_in_the_product(cuda_device, big):
    """The same in the second product's epilogue: one column of each expert's argument is large."""
    gen = torch.Generator(device="cuda").manual_seed(14)
    h, ffn, n = 64, 264, 70
    rows = torch.zeros(n, h, device=cuda_device, dtype=torch.bfloat16)
    rows[:, 0] = 1
    w1 = torch.zeros(1, ffn, h, device=cuda_device, dtype=torch.bfloat16)
    w1[0, 5, 0], w1[0, 200, 0] = big, -big
    w2 = torch.randn(1, h, ffn, generator=gen, device=cuda_device).to(torch.bfloat16)
    d_out = torch.randn(n, h, generator=gen, device=cuda_device).to(torch.bfloat16)
    seg = torch.tensor([0, n], dtype=torch.int32, device=cuda_device)
    _, kept = ops.grouped_ffn_train(rows, w1, w2, seg, "gelu_tanh", ffn)
    d_rows, dw1, dw2 = ops.grouped_ffn_backward(d_out, rows, kept, w1, w2, seg, "gelu_tanh", ffn)
    want = (d_out.to(D) @ w2[0].to(D))[:, 5].sum()  # slope 1; column 200: slope 0
    mass = (d_out.to(D).abs() @ w2[0].to(D).abs())[:, 5].sum()
    assert abs(float(dw1[0, 5, 0].to(D) - want)) <= 2.0 ** -8 * float(want.abs()) + (2.0 ** -8 + 200 * 2.0 ** -23) * float(mass)
    assert float(dw1[0, 200, 0]) == 0.0 and bool(torch.isfinite(dw1).all()) and bool(torch.isfinite(d_rows).all())


# ---- calls at the limits of what is documented ---------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("per_expert", [1, 3, 100])
def test_as_many_experts_as_there_may_be(cuda_device, dtype, per_expert):
    gen = torch.Generator(device="cuda").manual_seed(15)
    e, h, ffn = 256, 64, 72
    rows = e * per_expert
    rand = lambda *s: torch.randn(*s, generator=gen, device=cuda_device).to(dtype)  # noqa: E731
    x, d_out, w1, w2 = rand(rows, h), rand(rows, h), rand(e, ffn, h), rand(e, h, ffn)
    seg = torch.arange(0, rows + 1, per_expert, dtype=torch.int32, device=cuda_device)
    half = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[dtype]
    dx, dw = ops.grouped_dgrad(x, w2, seg), ops.grouped_wgrad(d_out, x, seg)
    a, b, g = (t.to(D).view(e, -1, t.shape[-1]) for t in (x, w2, d_out))
    for got, p, q, n in ((dx.view(e, -1, ffn), a, b, h), (dw, g.transpose(1, 2), a, per_expert)):
        ref, mass = p @ q, p.abs() @ q.abs()
        assert bool(((got.to(D) - ref).abs() <= half * ref.abs() + (n + 1) * 2.0 ** -23 * mass).all())
    out, kept = ops.grouped_ffn_train(x, w1, w2, seg, "gelu_tanh", ffn)
    grads = ops.grouped_ffn_backward(d_out, x, kept, w1, w2, seg, "gelu_tanh", ffn)
    p = kept.codes.to(D).view(e, -1, ffn)
    act = torch.nn.functional.gelu(p, approximate="tanh")
    for got, ref in ((out, (act @ w2.to(D).transpose(1, 2)).flatten(0, 1)), (grads[2], g.transpose(1, 2) @ act)):
        assert float((got.to(D) - ref).norm() / ref.norm()) <= (6 if dtype == torch.bfloat16 else 64) * half  # (as test_train_ops_gpu and test_train_block_gpu)
    with pytest.raises(RuntimeError, match="documented maximum"):
        ops.grouped_wgrad(d_out[:1], x[:1], torch.zeros(258, dtype=torch.int32, device=cuda_device))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ["swiglu", "gelu_tanh"])
@pytest.mark.parametrize("keep", [None, "int8"])
def test_the_smallest_ffn(cuda_device, dtype, act, keep):
    """Eight columns everywhere, one row in the last of three experts."""
    gen = torch.Generator(device="cuda").manual_seed(16)
    rand = lambda *s: torch.randn(*s, generator=gen, device=cuda_device).to(dtype)  # noqa: E731
    x, d_out, w1, w2 = rand(1, 8), rand(1, 8), rand(3, ops.act_columns(act, 8), 8), rand(3, 8, 8)
    seg = torch.tensor([0, 0, 0, 1], dtype=torch.int32, device=cuda_device)
    out, kept = ops.grouped_ffn_train(x, w1, w2, seg, act, 8, keep=keep)
    d_rows, dw1, dw2 = ops.grouped_ffn_backward(d_out, x, kept, w1, w2, seg, act, 8)
    a = w1[2].to(D).requires_grad_()
    b, xx = w2[2].to(D).requires_grad_(), x.to(D).requires_grad_()
    pre = (xx @ a.T)
    if act == "swiglu":
        mid = torch.nn.functional.silu(pre[:, :8]) * pre[:, 128:136]
    else:
        mid = torch.nn.functional.gelu(pre, approximate="tanh")
    want = mid @ b.T
    want.backward(d_out.to(D))
    # five roundings on the way at most, and int8's half step of the largest of the group: 1/254 of it, for 8 values of
    # which the others may be smaller by any factor, so against the largest result
    tol = {torch.bfloat16: 8 * 2.0 ** -8, torch.float32: 64 * 2.0 ** -24}[dtype] + (0.05 if keep else 0)
    gate_up = [a.grad[:8], a.grad[128:136]] if act == "swiglu" else [a.grad]
    for got, ref in [(out, want), (d_rows, xx.grad), (dw2[2], b.grad), *zip(dw1 if act == "swiglu" else [dw1], gate_up)]:
        got = got[2] if got.dim() == 3 else got
        assert float((got.to(D) - ref.detach()).abs().max()) <= tol * float(ref.detach().abs().max()) + 1e-30
    assert bool((dw2[:2] == 0).all()) and all(bool((t[:2] == 0).all()) for t in (dw1 if act == "swiglu" else [dw1]))


def test_fp32_slab_table_on_the_tensor_cores(cuda_device):
    """Segments that share a slab, one without an expert (its rows hold NaN), an infinity in a shared slab."""
    gen = torch.Generator(device="cuda").manual_seed(17)
    counts, slab, n, k = [150, 60, 40, 250], [1, 0, -1, 1], 1032, 712
    seg = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device=cuda_device)
    dy, w = torch.randn(500, n, generator=gen, device=cuda_device), torch.randn(2, n, k, generator=gen, device=cuda_device)
    assert ops._split_bytes(_lib.load(), 500, n, k, 2, ops.PRODUCT_DGRAD, ops.DICE_F32) > 0
    dy[210:250] = float("nan")
    table = torch.tensor(slab, dtype=torch.int32, device=cuda_device)
    out = torch.full((500, k), -7.0, device=cuda_device)
    clean = ops.grouped_dgrad(dy, w, seg, seg_slab=table, out=out).clone()
    w2 = w.clone()
    w2[1, 100, 200] = float("inf")
    got = ops.grouped_dgrad(dy, w2, seg, seg_slab=table)
    at = 0
    for c, s in zip(counts, slab):
        cut = slice(at, at + c)
        at += c
        if s < 0:
            assert bool((clean[cut] == -7).all())
            continue
        _check_f32(clean[cut], dy[cut].to(D), w[s].to(D))
        others = torch.arange(k, device=cuda_device) != 200
        assert torch.equal(got[cut][:, others], clean[cut][:, others])
        if s == 1:
            assert torch.equal(got[cut][:, 200], torch.sign(dy[cut][:, 100]) * float("inf"))
        else:
            assert torch.equal(got[cut], clean[cut])


@pytest.mark.parametrize("rows", [33000, 70001])
def test_long_weight_gradient_with_gate_and_up_apart(cuda_device, rows):
    """More than 32768 rows take the form that empties its accumulator: the same bits packed and apart, and 64 bits'."""
    gen = torch.Generator(device="cuda").manual_seed(18)
    ffn, k = 136, 72
    cols = ops.w13_rows(ffn)
    dy, x = (torch.randn(rows, c, generator=gen, device=cuda_device).to(torch.bfloat16) for c in (cols, k))
    seg = torch.tensor([0, 32800, 32800, rows], dtype=torch.int32, device=cuda_device)
    packed = ops.grouped_wgrad(dy, x, seg)
    gate, up = ops.grouped_wgrad(dy, x, seg, gate_up=ffn)
    parts = packed.unflatten(1, (-1, 2, 128))
    assert torch.equal(gate, parts[:, :, 0].flatten(1, 2)[:, :ffn]) and torch.equal(up, parts[:, :, 1].flatten(1, 2)[:, :ffn])
    for s, (beg, end) in enumerate([(0, 32800), (32800, 32800), (32800, rows)]):
        a, b = dy[beg:end].to(D).T, x[beg:end].to(D)
        ref, mass = a @ b, a.abs() @ b.abs()
        assert bool(((packed[s].to(D) - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -12 * mass).all())


def test_two_fp32_calls_at_once(cuda_device):
    """Planes, the word for values that are not finite and shared reductions are each call's own."""
    gen = torch.Generator(device="cuda").manual_seed(19)
    seg = torch.tensor([0, 700], dtype=torch.int32, device=cuda_device)
    ins = [[torch.randn(*s, generator=gen, device=cuda_device) for s in ((700, 1032), (700, 72), (1, 1032, 712))] for _ in range(2)]
    ins[1][0][3, 3] = float("inf")
    call = lambda i: (ops.grouped_dgrad(ins[i][0], ins[i][2], seg), ops.grouped_wgrad(ins[i][0], ins[i][1], seg))  # noqa: E731
    want = [call(0), call(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in range(2):
        for pair in got[i]:
            assert all(torch.equal(a.nan_to_num(7.0, 8.0, 9.0), b.nan_to_num(7.0, 8.0, 9.0)) for a, b in zip(pair, want[i]))
