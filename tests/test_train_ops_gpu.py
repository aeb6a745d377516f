"""The training operators against plain implementations in 64 bits.

Bounds.  u(t) = half a step of type t (bf16 2^-8, fp32 2^-24).  A sum of K products in fp32 is off by at most
K 2^-23 sum|a b| (twice the usual bound K 2^-24: the tensor cores may cut where the CUDA cores round; fp32 operands in
three bf16 planes leave out less than 2^-25 of a product, and K counts from 1, so K + 1 covers it), and rounding it to
type t adds u(t) of the value.  The sigmoid of z is off by at most delta = (8 + 4 |z|) 2^-23 of its value: expf's
and the division's few units plus the argument's own rounding, which exp multiplies by |z|.
"""
import math

import pytest
import torch

from dice_b200 import ops

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TYPES = [torch.bfloat16, torch.float32]
D = torch.float64


def _seg(counts, dev, start=0):
    out = [start]
    for c in counts:
        out.append(out[-1] + c)
    return torch.tensor(out, dtype=torch.int32, device=dev)


def _randn(gen, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _check_product(got, ref, mass, length, dtype):
    """``mass``: the sum of the products' magnitudes"""
    bound = U[dtype] * ref.abs() + (length + 1) * 2.0 ** -23 * mass + 1e-38
    err = (got.to(D) - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


# counts per expert, n, k
SHAPES = [
    ([1], 8, 8),
    ([0, 1, 0], 64, 72),
    ([3, 0, 130, 1], 200, 136),
    ([129, 64, 63, 65, 0], 128, 256),
    ([0, 0, 300], 264, 1160),
    ([16, 48, 17, 31] * 8, 72, 328),
    ([1000, 1, 23], 520, 384),
    ([257, 255], 1152, 648),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,n,k", SHAPES)
def test_dgrad(cuda_device, counts, n, k, dtype):
    gen = _gen(1)
    rows, e = sum(counts), len(counts)
    dy, w = _randn(gen, rows, n, dtype=dtype), _randn(gen, e, n, k, dtype=dtype, scale=0.02)
    seg = _seg(counts, cuda_device)
    dx = ops.grouped_dgrad(dy, w, seg)
    r = 0
    for s, c in enumerate(counts):
        a, b = dy[r:r + c].to(D), w[s].to(D)
        _check_product(dx[r:r + c], a @ b, a.abs() @ b.abs(), n, dtype)
        r += c
    ops.check_status(ops.device_status(cuda_device))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,n,k", SHAPES)
def test_wgrad(cuda_device, counts, n, k, dtype):
    gen = _gen(2)
    rows, e = sum(counts), len(counts)
    dy, x = _randn(gen, rows, n, dtype=dtype), _randn(gen, rows, k, dtype=dtype)
    dw = ops.grouped_wgrad(dy, x, _seg(counts, cuda_device))
    assert dw.shape == (e, n, k)
    r = 0
    for s, c in enumerate(counts):
        a, b = dy[r:r + c].to(D).T, x[r:r + c].to(D)
        _check_product(dw[s], a @ b, a.abs() @ b.abs(), c, dtype)
        r += c
    ops.check_status(ops.device_status(cuda_device))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,n,k", [
    ([1], 9216, 64), ([2, 0, 1], 4608, 264), ([300], 2048, 72), ([129, 3], 1160, 520),   # shared by the input gradient
    ([6000], 72, 64), ([3001, 0, 700], 136, 264), ([1100], 264, 328),                      # and by the weight gradient
    ([1, 1], 1152, 4608),                                                                   # narrow tiles, nothing shared
    ([8, 5, 1, 9], 328, 1160), ([2] * 16, 1032, 264), ([12, 13, 32, 33, 76], 520, 264),     # fp32: tiles of few rows
])
def test_long_reductions_and_few_tiles(cuda_device, counts, n, k, dtype):
    """Few tiles: the reduction is shared, and added up in a fixed order."""
    gen = _gen(16)
    rows, e = sum(counts), len(counts)
    dy, x, w = _randn(gen, rows, n, dtype=dtype), _randn(gen, rows, k, dtype=dtype), _randn(gen, e, n, k, dtype=dtype, scale=0.02)
    seg = _seg(counts, cuda_device)
    dx, dw = ops.grouped_dgrad(dy, w, seg), ops.grouped_wgrad(dy, x, seg)
    r = 0
    for s, c in enumerate(counts):
        a, b, g = dy[r:r + c].to(D), w[s].to(D), x[r:r + c].to(D)
        _check_product(dx[r:r + c], a @ b, a.abs() @ b.abs(), n, dtype)
        _check_product(dw[s], a.T @ g, a.abs().T @ g.abs(), c, dtype)
        r += c
    for _ in range(5):
        assert torch.equal(dx, ops.grouped_dgrad(dy, w, seg)) and torch.equal(dw, ops.grouped_wgrad(dy, x, seg))
    ops.check_status(ops.device_status(cuda_device))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ffn", [8, 64, 128, 136, 320, 1152])
def test_wgrad_gate_up(cuda_device, ffn, dtype):
    """The packed rows' gradient written apart is that of the packed form, bit for bit."""
    gen = _gen(3)
    counts = [40, 0, 97]
    cols = ops.w13_rows(ffn)
    dy, x = _randn(gen, sum(counts), cols, dtype=dtype), _randn(gen, sum(counts), 72, dtype=dtype)
    seg = _seg(counts, cuda_device)
    packed = ops.grouped_wgrad(dy, x, seg).unflatten(1, (-1, 2, 128))
    gate, up = ops.grouped_wgrad(dy, x, seg, gate_up=ffn)
    assert torch.equal(gate, packed[:, :, 0].flatten(1, 2)[:, :ffn])
    assert torch.equal(up, packed[:, :, 1].flatten(1, 2)[:, :ffn])


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_outside_the_segments(cuda_device, dtype):
    """Rows before the first and behind the last segment are neither read nor written, whatever they hold; a NaN or an
    infinity in one expert's rows or weights reaches no other expert."""
    gen = _gen(4)
    counts, n, k = [5, 0, 70, 13], 136, 264
    seg = _seg(counts, cuda_device, start=3)
    rows = int(seg[-1]) + 20
    dy, x = _randn(gen, rows, n, dtype=dtype), _randn(gen, rows, k, dtype=dtype)
    w = _randn(gen, 4, n, k, dtype=dtype)
    want_dx, want_dw = ops.grouped_dgrad(dy, w, seg), ops.grouped_wgrad(dy, x, seg)
    for bad in (float("nan"), float("inf")):
        dy2, x2, w2 = dy.clone(), x.clone(), w.clone()
        for t in (dy2, x2):
            t[:3] = bad
            t[int(seg[-1]):] = bad
            t[int(seg[2]):int(seg[3])] = bad  # the third expert's rows
        w2[1] = bad  # an expert without rows
        out = torch.full((rows, k), -7.0, dtype=dtype, device=cuda_device)
        dx = ops.grouped_dgrad(dy2, w2, seg, out=out)
        dw = ops.grouped_wgrad(dy2, x2, seg)
        fine = torch.ones(rows, dtype=torch.bool, device=cuda_device)
        fine[:3] = fine[int(seg[-1]):] = fine[int(seg[2]):int(seg[3])] = False
        assert torch.equal(dx[fine], want_dx[fine])
        assert bool((dx[:3] == -7).all()) and bool((dx[int(seg[-1]):] == -7).all())
        assert not bool(torch.isfinite(dx[int(seg[2]):int(seg[3])]).any())
        assert torch.equal(dw[[0, 1, 3]], want_dw[[0, 1, 3]])
        assert not bool(torch.isfinite(dw[2]).any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(8, 8), (1160, 136), (4608, 2056)])
def test_dgrad_of_single_tokens(cuda_device, dtype, n, k):
    """One to four rows: together, apart, beside rows of no expert that hold NaN, through a table of slabs."""
    gen = _gen(20)
    w = _randn(gen, 3, n, k, dtype=dtype, scale=0.1)
    for offsets, slab in [([0, 1], [2]), ([0, 0, 2, 2], None), ([0, 1, 1, 2], None), ([0, 4], [1]), ([0, 3, 4, 4], None),
                          ([1, 2, 2, 3], [0, -1, 2]), ([0, 1, 2, 4], [1, -1, 1])]:
        rows = 4 if offsets[0] else offsets[-1]
        dy = _randn(gen, rows, n, dtype=dtype)
        fine = torch.zeros(rows, dtype=torch.bool, device=cuda_device)
        seg = torch.tensor(offsets, dtype=torch.int32, device=cuda_device)
        table = None if slab is None else torch.tensor(slab, dtype=torch.int32, device=cuda_device)
        slabs = slab if slab is not None else range(3)
        for s, beg, end in zip(slabs, offsets, offsets[1:]):
            fine[beg:end] = s >= 0
        dy[~fine] = float("nan")
        out = torch.full((rows, k), -7.0, dtype=dtype, device=cuda_device)
        ops.grouped_dgrad(dy, w if slab is not None or len(offsets) == 4 else w[:len(offsets) - 1], seg, seg_slab=table, out=out)
        assert bool((out[~fine] == -7).all())
        for s, beg, end in zip(slabs, offsets, offsets[1:]):
            if s >= 0 and end > beg:
                a, b = dy[beg:end].to(D), w[s].to(D)
                _check_product(out[beg:end], a @ b, a.abs() @ b.abs(), n, dtype)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    ops.grouped_dgrad(dy, w, torch.tensor([0, 2, 1, 4], dtype=torch.int32, device=cuda_device), status=status)
    with pytest.raises(RuntimeError, match="segment offsets"):
        ops.check_status(status)


@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows_at_all(cuda_device, dtype):
    seg = torch.zeros(4, dtype=torch.int32, device=cuda_device)
    dy, x = torch.empty(0, 64, dtype=dtype, device=cuda_device), torch.empty(0, 72, dtype=dtype, device=cuda_device)
    w = torch.ones(3, 64, 72, dtype=dtype, device=cuda_device)
    assert ops.grouped_dgrad(dy, w, seg).shape == (0, 72)
    assert bool((ops.grouped_wgrad(dy, x, seg) == 0).all())
    dy, x = torch.full((5, 64), float("nan"), dtype=dtype, device=cuda_device), torch.ones(5, 72, dtype=dtype, device=cuda_device)
    assert bool((ops.grouped_wgrad(dy, x, seg) == 0).all())  # rows, but none of them any expert's
    assert ops.grouped_wgrad(dy[:0], x[:0], seg, gate_up=None).shape == (3, 64, 72)
    with pytest.raises(AssertionError):
        ops.grouped_wgrad(dy, x, seg, gate_up=-8)
    with pytest.raises(RuntimeError, match="unsupported shape"):
        ops.grouped_wgrad(dy, x, seg, gate_up=64)  # 64 gate rows take 256 packed columns
    with pytest.raises(RuntimeError, match="invalid argument"):
        ops.grouped_dgrad(dy, w[:2], seg)  # three segments, two slabs, no table
    with pytest.raises(RuntimeError, match="not 16-byte aligned"):
        ops.grouped_dgrad(dy, w, seg, out=torch.empty(5 * 72 + 1, dtype=dtype, device=cuda_device)[1:].view(5, 72))
    a, kept = ops.act_keep(dy[:0], "gelu_tanh", 64)
    assert a.shape == (0, 64) and kept.codes.shape == (0, 64)
    d, w2 = ops.combine_backward(dy[:0], dy[:0], torch.empty(0, 2, dtype=torch.int32, device=cuda_device),
                                 torch.empty(0, 2, device=cuda_device))
    assert d.shape == (0, 64) and w2.shape == (0, 2)


@pytest.mark.parametrize("dtype", TYPES)
def test_dgrad_slab_table(cuda_device, dtype):
    """Segments name their slab, some share one, -1 means rows of no expert."""
    gen = _gen(5)
    counts, slab = [10, 33, 7, 40], [1, 0, -1, 1]
    n, k = 72, 136
    dy, w = _randn(gen, sum(counts), n, dtype=dtype), _randn(gen, 2, n, k, dtype=dtype)
    seg = _seg(counts, cuda_device)
    out = torch.full((sum(counts), k), -7.0, dtype=dtype, device=cuda_device)
    ops.grouped_dgrad(dy, w, seg, seg_slab=torch.tensor(slab, dtype=torch.int32, device=cuda_device), out=out)
    r = 0
    for c, s in zip(counts, slab):
        if s < 0:
            assert bool((out[r:r + c] == -7).all())
        else:
            a, b = dy[r:r + c].to(D), w[s].to(D)
            _check_product(out[r:r + c], a @ b, a.abs() @ b.abs(), n, dtype)
        r += c


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offsets", [[0, 9, 5], [0, 4, 11], [-1, 4, 10], [0, 4, 2 ** 31 - 1]])
def test_bad_segments_are_reported(cuda_device, dtype, offsets):
    seg = torch.tensor(offsets, dtype=torch.int32, device=cuda_device)
    dy, x = torch.ones(10, 64, dtype=dtype, device=cuda_device), torch.ones(10, 72, dtype=dtype, device=cuda_device)
    w = torch.ones(2, 64, 72, dtype=dtype, device=cuda_device)
    for call in (lambda s: ops.grouped_dgrad(dy, w, seg, status=s), lambda s: ops.grouped_wgrad(dy, x, seg, status=s)):
        status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
        call(status)
        with pytest.raises(RuntimeError, match="segment offsets"):
            ops.check_status(status)


@pytest.mark.parametrize("dtype", TYPES)
def test_bad_slab_is_reported(cuda_device, dtype):
    dy, w = torch.ones(10, 64, dtype=dtype, device=cuda_device), torch.ones(2, 64, 72, dtype=dtype, device=cuda_device)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    ops.grouped_dgrad(dy, w, _seg([10], cuda_device), status=status,
                      seg_slab=torch.tensor([2], dtype=torch.int32, device=cuda_device))
    with pytest.raises(RuntimeError, match="segment offsets"):
        ops.check_status(status)


# ---- activation ---------------------------------------------------------------------


def _parts(x, ffn):
    cols = torch.arange(ffn, device=x.device)
    at = cols // 128 * 256 + cols % 128
    return x[:, at], x[:, at + 128], at


def _act64(p, act, ffn):
    """value, derivatives (one or two), and bounds on their errors, in 64 bits"""
    if act == "swiglu":
        g, u, _ = _parts(p, ffn)
        delta = (8 + 4 * g.abs()) * 2.0 ** -23
        s = torch.sigmoid(g)
        slope = s * (1 + g * (1 - s))
        return g * s * u, (u * slope, g * s), 2 * delta * (g * s * u).abs(), (
            3 * delta * u.abs() * s * (1 + g.abs()), 2 * delta * (g * s).abs())
    c = 2 * math.sqrt(2 / math.pi)
    z = c * (p + 0.044715 * p ** 3)
    delta = (8 + 4 * z.abs()) * 2.0 ** -23
    s = torch.sigmoid(z)
    dz = c * (1 + 3 * 0.044715 * p ** 2)
    return p * s, (s + p * s * (1 - s) * dz,), 2 * delta * (p * s).abs(), (4 * delta * s * (1 + p.abs() * dz),)


def _codes32(x, keep):
    """The definition in fp32, step by step: (codes, scales)"""
    r, c = x.shape
    groups = (c + 127) // 128
    # a tensor: by a number torch would multiply with the reciprocal, which rounds twice
    top = torch.full((r, groups), 127.0 if keep == "int8" else 448.0, device=x.device)
    g = torch.nn.functional.pad(x.float(), (0, groups * 128 - c)).view(r, groups, 128)
    most = g.abs().amax(2).clamp(min=2.0 ** -100)
    q = g * (top / most)[:, :, None]
    q = q.round().to(torch.int8) if keep == "int8" else q.to(torch.float8_e4m3fn)
    return q.view(r, -1)[:, :c], most / top


def _read(kept):
    if kept.scales is None:
        return kept.codes.to(D)
    return kept.codes.to(D) * kept.scales.repeat_interleave(128, 1)[:, :kept.codes.shape[1]].to(D)


def _argument(gen, rows, act, ffn, dtype, scale=1.5):
    pre = _randn(gen, rows, ops.act_columns(act, ffn), dtype=dtype, scale=scale)
    if act == "swiglu":
        pre.unflatten(1, (-1, 2, 128))[:, -1, :, (ffn - 1) % 128 + 1:] = 0
    return pre


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["swiglu", "gelu_tanh"])
@pytest.mark.parametrize("keep", ["int8", "e4m3", None])
@pytest.mark.parametrize("rows,ffn", [(1, 8), (3, 128), (37, 1000), (130, 264), (2, 9000), (513, 64)])
def test_act_keep_and_backward(cuda_device, dtype, act, keep, rows, ffn):
    gen = _gen(6)
    pre = _argument(gen, rows, act, ffn, dtype)
    a, kept = ops.act_keep(pre, act, ffn, keep=keep)
    ref, _, err, _ = _act64(pre.to(D), act, ffn)
    assert bool(((a.to(D) - ref).abs() <= U[dtype] * ref.abs() + 1.01 * err + 1e-36).all())
    if keep is None:
        assert kept.codes is pre or torch.equal(kept.codes, pre)
    else:
        codes, scales = _codes32(pre, keep)
        assert torch.equal(kept.scales, scales)
        assert torch.equal(kept.codes.view(torch.uint8), codes.contiguous().view(torch.uint8))
        # the largest values are off by at most half a step of the 8-bit type: 1/254 of the group's maximum (int8), 2^-4
        # of the value or half the smallest subnormal, 2^-10, times the scale (e4m3); the factor's own rounding adds 2^-23
        far = (_read(kept) - pre.to(D)).abs()
        sc = scales.repeat_interleave(128, 1)[:, :pre.shape[1]].to(D)
        bound = 0.5 * sc * 1.001 if keep == "int8" else torch.maximum(2.0 ** -4 * pre.to(D).abs(), 2.0 ** -10 * sc) * 1.001
        assert bool((far <= bound).all())
    da = _randn(gen, rows, ffn, dtype=dtype)
    d_pre, a2 = ops.act_backward(da, kept, act, ffn)
    p = _read(kept)
    # code * scale is rounded to fp32 once (2^-24 of p), which moves value and slope by less than delta of theirs
    ref, slopes, err, errs = _act64(p, act, ffn)
    assert bool(((a2.to(D) - ref).abs() <= U[dtype] * ref.abs() + 2 * err + 1e-36).all())
    if act == "swiglu":
        dg, du, at = _parts(d_pre.to(D), ffn)
        rest = torch.ones(d_pre.shape[1], dtype=torch.bool, device=cuda_device)
        rest[at] = rest[at + 128] = False
        assert bool((d_pre[:, rest] == 0).all())
        got = (dg, du)
    else:
        got = (d_pre.to(D),)
    for g, slope, e in zip(got, slopes, errs):
        want = da.to(D) * slope
        assert bool(((g - want).abs() <= U[dtype] * want.abs() + 2 * da.to(D).abs() * e + 1e-36).all())
    d_pre2, none = ops.act_backward(da, kept, act, ffn, want_act=False)
    assert none is None and torch.equal(d_pre, d_pre2)


@pytest.mark.parametrize("act", ["swiglu", "gelu_tanh"])
def test_act_backward_against_differences(cuda_device, act):
    """Central differences of the fp32 forward pass: step h, error at most h^2/6 times the third derivative (below 3)
    plus the values' rounding, 4 * 2^-24 * |a| / h."""
    gen = _gen(7)
    ffn, h = 136, 2.0 ** -6
    pre = _argument(gen, 9, act, ffn, torch.float32, scale=1.0)
    one = torch.ones(9, ffn, device=cuda_device)
    d_pre, a = ops.act_backward(one, ops.KeptAct(pre, None), act, ffn)
    parts = [slice(None)] if act != "swiglu" else [0, 1]
    for part in parts:
        step = torch.zeros_like(pre)
        (step.unflatten(1, (-1, 2, 128))[:, :, part] if act == "swiglu" else step)[...] = h
        up, dn = ops.act_keep(pre + step, act, ffn, keep=None)[0], ops.act_keep(pre - step, act, ffn, keep=None)[0]
        diff = (up.double() - dn.double()) / (2 * h)
        got = d_pre.double() if act != "swiglu" else _parts(d_pre.double(), ffn)[part]
        scale = 1.0 if act != "swiglu" else _parts(pre.double(), ffn)[1].abs() + 1
        assert bool(((diff - got).abs() <= 0.5 * h * h * scale + 2.0 ** -21 * (a.abs().double() + 1) / h).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("keep", ["int8", "e4m3"])
def test_groups_that_are_special(cuda_device, dtype, keep):
    """All zeros, the smallest values, the largest, an infinity, a NaN: each in a group of its own."""
    pre = torch.zeros(6, 256, dtype=dtype, device=cuda_device)
    pre[1, :128] = torch.finfo(dtype).tiny
    pre[2, :128] = torch.finfo(dtype).max
    pre[3, 5] = float("inf")
    pre[4, 127] = float("nan")
    pre[5, 0], pre[5, 1] = 2.0 ** -99, -2.0 ** -101
    pre[:, 128:] = 1.0
    a, kept = ops.act_keep(pre, "gelu_tanh", 256, keep=keep)
    back = _read(kept)
    assert bool((back[0, :128] == 0).all()) and bool((back[1, :128] == 0).all())
    assert bool(((back[2, :128] - pre[2, :128].to(D)).abs() <= 2.0 ** -22 * pre[2, :128].to(D)).all())
    assert bool(torch.isnan(kept.scales[3:5, 0]).all()) and bool(torch.isfinite(kept.scales[:, 1]).all())
    assert bool(torch.isfinite(kept.scales[[0, 1, 2, 5]]).all())
    assert float(back[5, 0]) == pytest.approx(2.0 ** -99, rel=2.0 ** -22)
    assert bool(((back[:, 128:] - 1).abs() <= 2.0 ** -22).all())
    da = torch.ones(6, 256, dtype=dtype, device=cuda_device)
    d_pre, _ = ops.act_backward(da, kept, "gelu_tanh", 256)
    assert bool(torch.isnan(d_pre[3:5, :128]).all()) and bool(torch.isfinite(d_pre[[0, 1, 5]]).all())
    assert bool(torch.isfinite(d_pre[3:5, 128:]).all())


def test_filling_columns_are_not_read(cuda_device):
    gen = _gen(8)
    pre = _argument(gen, 5, "swiglu", 136, torch.bfloat16)
    bad = pre.clone()
    bad.unflatten(1, (-1, 2, 128))[:, -1, :, 8:] = float("nan")
    (a, kept), (a2, kept2) = ops.act_keep(pre, "swiglu", 136), ops.act_keep(bad, "swiglu", 136)
    assert torch.equal(a, a2) and torch.equal(kept.codes, kept2.codes) and torch.equal(kept.scales, kept2.scales)


# ---- combine ----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,h", [(1, 8), (1, 1152), (7, 264), (300, 1160), (33, 2056)])
def test_combine_backward(cuda_device, dtype, tokens, h):
    gen = _gen(9)
    dout, y = _randn(gen, tokens, h, dtype=dtype), _randn(gen, 2 * tokens, h, dtype=dtype)
    pos = torch.randperm(2 * tokens, generator=gen, device=cuda_device).to(torch.int32).view(tokens, 2)
    w = torch.rand(tokens, 2, generator=gen, device=cuda_device)
    d_rows, d_w = ops.combine_backward(dout, y, pos, w)
    for s in range(2):
        want = w[:, s:s + 1].to(D) * dout.to(D)
        assert bool(((d_rows[pos[:, s].long()].to(D) - want).abs() <= (U[dtype] + 2.0 ** -24) * want.abs() + 1e-40).all())
        prods = dout.to(D) * y[pos[:, s].long()].to(D)
        assert bool(((d_w[:, s].to(D) - prods.sum(1)).abs() <= (h + 1) * 2.0 ** -24 * prods.abs().sum(1)).all())
    # what the forward kernel computes is what this is the gradient of
    out = ops.unpermute_combine(y, pos[:, 0], y, pos[:, 1], w[:, 0], w[:, 1], tokens)
    want = (w.to(D).unsqueeze(2) * y.to(D)[pos.long()]).sum(1)
    mass = (w.to(D).unsqueeze(2) * y.to(D)[pos.long()]).abs().sum(1)
    assert bool(((out.to(D) - want).abs() <= U[dtype] * want.abs() + 2.0 ** -22 * mass).all())


def test_combine_backward_positions_without_a_row(cuda_device):
    gen = _gen(10)
    dout, y = _randn(gen, 3, 64, dtype=torch.bfloat16), _randn(gen, 4, 64, dtype=torch.bfloat16)
    pos = torch.tensor([[0, -1], [4, 3], [1, 2 ** 31 - 1]], dtype=torch.int32, device=cuda_device)
    d_rows, d_w = ops.combine_backward(dout, y, pos, torch.ones(3, 2, device=cuda_device))
    assert torch.equal(d_rows[[0, 3, 1]], dout)
    assert d_w[0, 1] == 0 and d_w[1, 0] == 0 and d_w[2, 1] == 0 and bool((d_w[[0, 1, 2], [0, 1, 0]] != 0).all())


# ---- calls as a program makes them ----------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_inputs(cuda_device, dtype):
    gen = _gen(11)
    counts = [20, 31]
    wide = _randn(gen, 51, 400, dtype=dtype)
    dy, x = wide[:, 8:208:1], wide.flip(0)[:, 64:200]
    w = _randn(gen, 136, 200, 2, dtype=dtype).permute(2, 1, 0)
    seg = _seg(counts, cuda_device)
    assert torch.equal(ops.grouped_dgrad(dy, w, seg), ops.grouped_dgrad(dy.contiguous(), w.contiguous(), seg))
    assert torch.equal(ops.grouped_wgrad(dy, x, seg), ops.grouped_wgrad(dy.contiguous(), x.contiguous(), seg))
    a, kept = ops.act_keep(dy, "gelu_tanh", 200)
    a2, kept2 = ops.act_keep(dy.contiguous(), "gelu_tanh", 200)
    assert torch.equal(a, a2) and torch.equal(kept.codes, kept2.codes)
    one = torch.ones(1, 1, dtype=dtype, device=cuda_device).expand(51, 200)
    assert torch.equal(ops.act_backward(one, kept, "gelu_tanh", 200)[0], ops.act_backward(one.contiguous(), kept, "gelu_tanh", 200)[0])


def _ffn_inputs(gen, counts, h, ffn, act, dtype, dev):
    e, rows = len(counts), sum(counts)
    if act == "swiglu":
        w1 = torch.stack([ops.pack_w13(_randn(gen, ffn, h, dtype=dtype, scale=0.1), _randn(gen, ffn, h, dtype=dtype, scale=0.1))
                          for _ in range(e)])
    else:
        w1 = _randn(gen, e, ffn, h, dtype=dtype, scale=0.1)
    return _randn(gen, rows, h, dtype=dtype), _randn(gen, rows, h, dtype=dtype), w1, _randn(gen, e, h, ffn, dtype=dtype, scale=0.1), _seg(counts, dev)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["swiglu", "gelu_tanh"])
@pytest.mark.parametrize("keep", ["int8", "e4m3", None])
@pytest.mark.parametrize("counts,h,ffn", [([1], 64, 64), ([0, 33, 300, 0, 7], 200, 264), ([128, 0, 256], 384, 512),
                                          ([5, 1, 8, 2, 70, 12, 9], 136, 1032), ([1, 3], 1792, 7168), ([200, 100, 0, 250], 264, 2056)])
def test_ffn_forward_and_backward(cuda_device, dtype, act, keep, counts, h, ffn):
    """The whole pass against 64 bits, fed with the kernel's own kept argument.  Norm bounds: every rounding to the type
    on the way moves its tensor by at most u of each value, and a product carries relative errors of its factors on; five
    such steps (argument, activation, its gradient, argument's gradient, output) and the fp32 sums stay below 6 u plus
    2^-24 times the longest sum's square root times 4."""
    gen = _gen(12)
    rows, d_out, w1, w2, seg = _ffn_inputs(gen, counts, h, ffn, act, dtype, cuda_device)
    out, kept = ops.grouped_ffn_train(rows, w1, w2, seg, act, ffn, keep=keep)
    d_rows, dw1, dw2 = ops.grouped_ffn_backward(d_out, rows, kept, w1, w2, seg, act, ffn)
    tol = 6 * U[dtype] + 4 * 2.0 ** -24 * math.sqrt(max(ffn, max(counts)))
    far = lambda got, ref: float((got.to(D) - ref).norm() / ref.norm()) if ref.norm() > 0 else float(got.to(D).norm())  # noqa: E731
    r = 0
    for s, c in enumerate(counts):
        x, g, a1, a2 = rows[r:r + c].to(D), d_out[r:r + c].to(D), w1[s].to(D), w2[s].to(D)
        pre = (x @ a1.T).to(dtype).to(D)
        p = _read(kept)[r:r + c]
        ref_a, slopes, _, _ = _act64(p, act, ffn)
        da = g @ a2
        if act == "swiglu":
            d_pre = torch.zeros_like(p)
            at = _parts(p, ffn)[2]
            d_pre[:, at], d_pre[:, at + 128] = da * slopes[0], da * slopes[1]
        else:
            d_pre = da * slopes[0]
        refs = [(d_rows[r:r + c], d_pre @ a1), (dw2[s], g.T @ ref_a), (out[r:r + c], _act64(pre, act, ffn)[0] @ a2.T)]
        full = d_pre.T @ x
        if act == "swiglu":
            refs += [(dw1[0][s], full[at]), (dw1[1][s], full[at + 128])]
        else:
            refs += [(dw1[s], full)]
        if c:
            for got, ref in refs:
                assert far(got, ref) <= tol, (s, far(got, ref), tol)
            if keep is not None:  # what is kept is the first product, in 8 bits
                assert far(_read(kept)[r:r + c], pre) <= 2.0 ** -4
        else:
            assert bool((dw2[s] == 0).all())
        r += c
    ops.check_status(ops.device_status(cuda_device))


def test_what_is_kept_is_the_operators_own(cuda_device):
    """The pass is its parts: first product, act_keep, second product; and backwards."""
    gen = _gen(13)
    counts, h, ffn = [100, 3, 0, 290], 256, 392
    for act in ("swiglu", "gelu_tanh"):
        rows, d_out, w1, w2, seg = _ffn_inputs(gen, counts, h, ffn, act, torch.bfloat16, cuda_device)
        status = ops.device_status(cuda_device)
        out, kept = ops.grouped_ffn_train(rows, w1, w2, seg, act, ffn, keep="int8")
        pre = ops.grouped_gemm(rows, w1, seg, ops.EPI_STORE, w1.shape[1], status)
        a, kept2 = ops.act_keep(pre, act, ffn, keep="int8")
        assert torch.equal(kept.codes, kept2.codes) and torch.equal(kept.scales, kept2.scales)
        assert torch.equal(out, ops.grouped_gemm(a, w2, seg, ops.EPI_STORE, h, status))


@pytest.mark.parametrize("counts,n,k", [([700, 1, 0, 300], 1032, 1160), ([97, 95, 96], 1152, 4608), ([2000, 30], 264, 520)])
def test_fp32_on_the_tensor_cores(cuda_device, counts, n, k):
    """Sizes that take the six products of bf16 planes: as near to 64 bits as fp32 sums are, element by element, over
    magnitudes from 2^-40 to 2^40 in one operand's rows, and with the largest values."""
    gen = _gen(19)
    rows, e = sum(counts), len(counts)
    dy, x = _randn(gen, rows, n, dtype=torch.float32), _randn(gen, rows, k, dtype=torch.float32)
    w = _randn(gen, e, n, k, dtype=torch.float32)
    dy *= torch.exp2(torch.randint(-40, 41, (rows, 1), generator=gen, device=cuda_device).float())
    dy[5, 7], x[5, :] = torch.finfo(torch.float32).max, 0.25  # would round to an infinity in 16 bits
    seg = _seg(counts, cuda_device)
    for product in (ops.PRODUCT_DGRAD, ops.PRODUCT_WGRAD):
        assert ops._split_bytes(ops._lib.load(), rows, n, k, e, product, ops.DICE_F32) >= 6 * rows * n
    w[0, 7, :] = 0.125
    dx, dw = ops.grouped_dgrad(dy, w, seg), ops.grouped_wgrad(dy, x, seg)
    r = 0
    for s, c in enumerate(counts):
        a, b, g = dy[r:r + c].to(D), w[s].to(D), x[r:r + c].to(D)
        _check_product(dx[r:r + c], a @ b, a.abs() @ b.abs(), n, torch.float32)
        _check_product(dw[s], a.T @ g, a.abs().T @ g.abs(), c, torch.float32)
        r += c
    # without scratch the CUDA cores do it: another order of sums, the same bounds
    lib, out = ops._lib.load(), torch.empty_like(dx)
    ops._lib.check(lib.dice_grouped_dgrad(dy.data_ptr(), rows, n, w.data_ptr(), e, k, seg.data_ptr(), None, e, ops.DICE_F32,
                                          out.data_ptr(), None, 0, None, torch.cuda.current_stream().cuda_stream), "dgrad")
    r = 0
    for s, c in enumerate(counts):
        a, b = dy[r:r + c].to(D), w[s].to(D)
        _check_product(out[r:r + c], a @ b, a.abs() @ b.abs(), n, torch.float32)
        r += c
    # a scratch that is too small is refused
    small = torch.empty(1024, dtype=torch.uint8, device=cuda_device)
    with pytest.raises(RuntimeError, match="scratch"):
        ops._lib.check(lib.dice_grouped_dgrad(dy.data_ptr(), rows, n, w.data_ptr(), e, k, seg.data_ptr(), None, e, ops.DICE_F32,
                                              out.data_ptr(), small.data_ptr(), 1024, None, torch.cuda.current_stream().cuda_stream), "dgrad")


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_rows_on_the_tensor_cores(cuda_device, dtype):
    """As test_rows_outside_the_segments, at sizes where fp32 is on the tensor cores too: NaN and infinities around the
    segments, in a neighbour and in unused weights change no other bit."""
    gen = _gen(21)
    counts, n, k = [301, 0, 205, 90], 1032, 1160
    seg = _seg(counts, cuda_device, start=5)
    rows = int(seg[-1]) + 9
    dy, x, w = (_randn(gen, *sh, dtype=dtype) for sh in ((rows, n), (rows, k), (4, n, k)))
    want_dx, want_dw = ops.grouped_dgrad(dy, w, seg), ops.grouped_wgrad(dy, x, seg)
    for bad in (float("nan"), float("inf")):
        dy2, x2, w2 = dy.clone(), x.clone(), w.clone()
        for t in (dy2, x2):
            t[:5] = t[int(seg[-1]):] = t[int(seg[2]):int(seg[3])] = bad
        w2[1] = bad
        out = torch.full((rows, k), -7.0, dtype=dtype, device=cuda_device)
        dx, dw = ops.grouped_dgrad(dy2, w2, seg, out=out), ops.grouped_wgrad(dy2, x2, seg)
        for s in (0, 3):
            assert torch.equal(dx[int(seg[s]):int(seg[s + 1])], want_dx[int(seg[s]):int(seg[s + 1])])
        assert bool((dx[:5] == -7).all()) and bool((dx[int(seg[-1]):] == -7).all())
        assert not bool(torch.isfinite(dx[int(seg[2]):int(seg[3])]).any())
        assert torch.equal(dw[[0, 1, 3]], want_dw[[0, 1, 3]]) and not bool(torch.isfinite(dw[2]).any())


def test_wgrad_whose_tiles_go_in_bands(cuda_device):
    """A segment whose second operand does not stay in L2 takes its tiles in another order; the one beside it does not."""
    gen = _gen(18)
    counts, n, k = [4100, 70], 2328, 8264  # 10 row tiles: a band of 8 and one of 2
    dy, x = _randn(gen, sum(counts), n, dtype=torch.bfloat16), _randn(gen, sum(counts), k, dtype=torch.bfloat16)
    dw = ops.grouped_wgrad(dy, x, _seg(counts, cuda_device))
    r = 0
    for s, c in enumerate(counts):
        a, b = dy[r:r + c].to(D).T, x[r:r + c].to(D)
        _check_product(dw[s], a @ b, a.abs() @ b.abs(), c, torch.bfloat16)
        r += c


@pytest.mark.parametrize("dtype", TYPES)
def test_offsets_past_32_bits(cuda_device, dtype):
    """Tensors of more than 2^31 elements: the first and the last rows against 64 bits (products) and against calls on these
    rows alone (the row-wise operators, which go row by row whatever their number)."""
    gen = _gen(17)
    rows, wide, narrow = 240000, 9216, 64
    assert rows * wide > 2 ** 31
    cut = [slice(0, 300), slice(rows - 300, rows)]
    seg = torch.tensor([0, 300, rows - 300, rows], dtype=torch.int32, device=cuda_device)
    dy, w = _randn(gen, rows, narrow, dtype=dtype), _randn(gen, 3, narrow, wide, dtype=dtype, scale=0.1)
    dx = ops.grouped_dgrad(dy, w, seg)
    for c, e in zip(cut, (0, 2)):
        a, b = dy[c].to(D), w[e].to(D)
        _check_product(dx[c], a @ b, a.abs() @ b.abs(), narrow, dtype)
    dw = ops.grouped_wgrad(dx, dy, seg)  # its wide operand read back
    for c, e in zip(cut, (0, 2)):
        a, b = dx[c].to(D).T, dy[c].to(D)
        _check_product(dw[e], a @ b, a.abs() @ b.abs(), 300, dtype)
    ffn = wide // 2
    a, kept = ops.act_keep(dx, "swiglu", ffn, keep="int8")
    parts = [dx[c].clone() for c in cut]
    del dx
    d_pre, a2 = ops.act_backward(a, kept, "swiglu", ffn)
    for c, part in zip(cut, parts):
        a_c, kept_c = ops.act_keep(part, "swiglu", ffn, keep="int8")
        assert torch.equal(a[c], a_c) and torch.equal(kept.codes[c], kept_c.codes) and torch.equal(kept.scales[c], kept_c.scales)
        d_c, a2_c = ops.act_backward(a_c, kept_c, "swiglu", ffn)
        assert torch.equal(d_pre[c], d_c) and torch.equal(a2[c], a2_c)


def test_other_stream_and_two_calls_at_once(cuda_device):
    gen = _gen(14)
    counts, h, ffn = [200, 0, 311], 128, 256
    ins = [_ffn_inputs(gen, counts, h, ffn, "swiglu", torch.bfloat16, cuda_device) for _ in range(2)]

    def step(i):
        rows, d_out, w1, w2, seg = ins[i]
        out, kept = ops.grouped_ffn_train(rows, w1, w2, seg, "swiglu", ffn)
        d_rows, dw1, dw2 = ops.grouped_ffn_backward(d_out, rows, kept, w1, w2, seg, "swiglu", ffn)
        return [out, d_rows, *dw1, dw2]

    want = [step(0), step(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    few = [(_randn(gen, 900, 72, dtype=torch.bfloat16), _randn(gen, 900, 64, dtype=torch.bfloat16)) for _ in range(2)]
    one = _seg([900], cuda_device)  # a shared reduction has scratch, each call its own
    want_few = [ops.grouped_wgrad(*f, one) for f in few]
    for _ in range(5):
        got_few = []
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got_few.append([ops.grouped_wgrad(*few[i], one) for _ in range(4)])
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for gs, w in zip(got_few, want_few) for g in gs)
    for _ in range(5):
        got = []
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append(step(i))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_captured_and_replayed(cuda_device):
    """Two graphs of the same calls on different buffers, replayed in turn and with new contents."""
    gen = _gen(15)
    counts, h, ffn = [70, 1, 0, 130], 136, 200
    ins = [_ffn_inputs(gen, counts, h, ffn, "gelu_tanh", torch.bfloat16, cuda_device) for _ in range(2)]
    ops.device_status(cuda_device)

    def step(i):
        rows, d_out, w1, w2, seg = ins[i]
        out, kept = ops.grouped_ffn_train(rows, w1, w2, seg, "gelu_tanh", ffn, keep="e4m3")
        d_rows, dw1, dw2 = ops.grouped_ffn_backward(d_out, rows, kept, w1, w2, seg, "gelu_tanh", ffn)
        return [out, d_rows, dw1, dw2]

    step(0)
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
    for turn in range(3):
        for i in range(2):
            ins[i][0].copy_(_randn(gen, sum(counts), h, dtype=torch.bfloat16))
            # other segments of the same number of rows
            ins[i][4].copy_(_seg([10 * turn, 201 - 10 * turn - 5, 5, 0], cuda_device))
        want = [step(0), step(1)]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, w))
