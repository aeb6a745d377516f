"""The operators of the expert FFN's training step, as calls that can be timed and compared.

``run`` makes one call: with ``own`` false in elementary torch operations, in 32 bits; with ``own`` true through
``dice_b200.ops``.  The operators, for rows sorted by expert (segment ``s`` = rows ``[seg[s], seg[s+1])``):

* ``dgrad``    ``dx[r] = dy[r] @ w[seg(r)]``: the input gradient of a matrix product grouped by expert
* ``wgrad``    ``dw[s] = dy[seg s].T @ x[seg s]``: its weight gradient (zero for an expert without rows)
* ``keep``     the activation function and, beside it, its argument in 8 bits: groups of 128 columns share a scale
* ``unkeep``   the activation's gradient from those 8 bits, and the activation again for the weight gradient behind it
* ``combine``  the gradient of the gate-weighted sum of a token's two rows, for the rows and for the gate weights
* ``step``     all of an expert FFN's forward and backward pass over sorted rows, made of these

SwiGLU arguments come in the packed order of the first product's weights: 128 gate columns, their 128 up columns,
the next 128 gate columns and so on, filled up with zeros.
"""
import math

import numpy as np
import torch

own = False

GROUP = 128
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one token at a time (its two routed rows) through the second product: the latency end
        dict(name="dgrad_token", op="dgrad", rows=2, experts=8, n=1152, k=4608, dtype="bf16", skew=0.0),
        # 64 images of 256 tokens in a 1152-wide block: the gradient that leaves the first (gate and up) product
        dict(name="dgrad_batch", op="dgrad", rows=32768, experts=8, n=9216, k=1152, dtype="bf16", skew=0.0),
        # few rows on many wide experts, unevenly routed: most of the work is writing the gradients
        dict(name="wgrad_few_rows", op="wgrad", rows=777, experts=16, n=1792, k=7168, dtype="bf16", skew=1.2, gate_up=0),
        # the 64 images again: gradients of gate and up weights
        dict(name="wgrad_batch", op="wgrad", rows=32768, experts=8, n=9216, k=1152, dtype="bf16", skew=0.0, gate_up=4608),
        # keeping the SwiGLU argument of the 64 images
        dict(name="keep_batch", op="keep", rows=32768, ffn=4608, act="swiglu", keep="int8", dtype="bf16"),
        # a short ragged remainder in fp32, width not a whole number of groups
        dict(name="keep_ragged_f32", op="keep", rows=37, ffn=1000, act="gelu_tanh", keep="e4m3", dtype="f32"),
        # a wider block (expert width 4 x 1792), half the tokens, kept as e4m3
        dict(name="unkeep_wide", op="unkeep", rows=16384, ffn=7168, act="swiglu", keep="e4m3", dtype="bf16"),
        # one image of 256 tokens, two-matrix experts
        dict(name="unkeep_image", op="unkeep", rows=512, ffn=4608, act="gelu_tanh", keep="int8", dtype="bf16"),
        # one token: latency
        dict(name="combine_token", op="combine", tokens=1, hidden=1152, dtype="bf16"),
        # 64 images of 256 tokens
        dict(name="combine_batch", op="combine", tokens=16384, hidden=1152, dtype="bf16"),
        # the whole FFN of the 64 images, argument kept in 8 bits
        dict(name="step_batch", op="step", rows=32768, experts=8, hidden=1152, ffn=4608, act="swiglu", keep="int8", dtype="bf16", skew=0.0),
        # two images of 256 tokens in fp32, nothing rounded: the parity configuration
        dict(name="step_f32", op="step", rows=1024, experts=8, hidden=1152, ffn=4608, act="gelu_tanh", keep="none", dtype="f32", skew=0.0),
    ]


def _log_int(rng, lo, hi, of=1):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))) // of * of))


def draw(rng):
    most_bytes = max(work(c)["bytes"] for c in listed())
    most_flops = max(work(c)["flops"] for c in listed())
    while True:
        op = rng.choice(["dgrad", "dgrad", "wgrad", "wgrad", "keep", "unkeep", "combine", "step", "step"])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        case = dict(op=op, dtype=dtype)
        if op == "combine":
            case.update(tokens=_log_int(rng, 1, 16384), hidden=_log_int(rng, 64, 2048, 8))
        else:
            case.update(rows=_log_int(rng, 1, 32768))
        if op in ("dgrad", "wgrad"):
            case.update(n=_log_int(rng, 64, 9216, 8), k=_log_int(rng, 64, 7168, 8))
            if op == "wgrad":
                case["gate_up"] = 0
                if rng.random() < 0.4:
                    case["gate_up"] = ffn = _log_int(rng, 64, 4608, 8)
                    case["n"] = _packed(ffn)
        if op in ("keep", "unkeep", "step"):
            case.update(ffn=_log_int(rng, 64, 7168, 8), act=rng.choice(["swiglu", "gelu_tanh"]), keep=rng.choice(["int8", "e4m3"]))
        if op == "step":
            case.update(hidden=_log_int(rng, 64, 1792, 8))
            # the fp32 step rounds nothing on its way, 8-bit codes included
            case["keep"] = "none" if dtype == "f32" else rng.choice(["int8", "e4m3", "none"])
        if op in ("dgrad", "wgrad", "step"):
            case.update(experts=rng.choice([1, 2, 5, 8, 16, 32]), skew=rng.choice([0.0, 0.0, 1.2]))
        w = work(case)
        # fp32 products run on the CUDA cores: a twentieth of the work takes as long
        if w["bytes"] <= most_bytes and w["flops"] <= (most_flops if dtype == "bf16" else most_flops / 20):
            return case


def _packed(ffn):
    """Columns of a packed SwiGLU argument."""
    return 2 * GROUP * ((ffn + GROUP - 1) // GROUP)


def _argument_cols(case):
    return _packed(case["ffn"]) if case["act"] == "swiglu" else case["ffn"]


def work(case):
    op, es = case["op"], 2 if case["dtype"] == "bf16" else 4
    if op == "combine":
        t, h = case["tokens"], case["hidden"]
        return dict(bytes=t * h * es * 5 + t * 2 * 12, flops=6 * t * h)
    rows = case["rows"]
    if op in ("dgrad", "wgrad"):
        n, k, e = case["n"], case["k"], case["experts"]
        slabs = min(e, rows) if op == "dgrad" else e  # every expert's gradient is written
        return dict(bytes=(rows * (n + k) + slabs * n * k) * es, flops=2 * rows * n * k)
    ffn, cols = case["ffn"], (2 if case["act"] == "swiglu" else 1) * case["ffn"]
    kept = cols * es if case["keep"] == "none" else cols + 4 * -(-cols // GROUP)
    if op == "keep":
        return dict(bytes=rows * (cols * es + ffn * es + kept), flops=20 * rows * ffn)
    if op == "unkeep":
        return dict(bytes=rows * (2 * ffn * es + cols * es + kept), flops=30 * rows * ffn)
    h, e = case["hidden"], case["experts"]
    products = rows * h * (cols + ffn)
    return dict(bytes=(4 * rows * h + 2 * e * h * (cols + ffn)) * es + 2 * rows * kept, flops=6 * products)


def _segments(case, rng):
    """Rows per expert for independent routing decisions, even or Zipf-skewed over experts in random order."""
    e, rows = case["experts"], case["rows"]
    p = 1.0 / np.arange(1, e + 1) ** case["skew"]
    counts = rng.multinomial(rows, rng.permutation(p / p.sum()))
    return counts


def _expert_weights(gen, e, out, inp, dtype):
    return (torch.randn(e, out, inp, generator=gen, device="cuda") * 0.02).to(dtype)


def _pack(gate, up):
    """[..., F, h] gate and up rows -> the packed order, zero rows behind them."""
    f = gate.shape[-2]
    fill = _packed(f) // 2 - f
    pair = [torch.nn.functional.pad(w, (0, 0, 0, fill)).unflatten(-2, (-1, 1, GROUP)) for w in (gate, up)]
    return torch.cat(pair, dim=-3).flatten(-4, -2).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    s = dict(case=case)
    if case["op"] == "combine":
        t, h = case["tokens"], case["hidden"]
        s["dout"] = normal(t, h, scale=0.01)
        s["rows_out"] = normal(2 * t, h)
        s["pos"] = torch.randperm(2 * t, generator=gen, device="cuda").to(torch.int32).view(t, 2)
        top = torch.rand(t, 1, generator=gen, device="cuda") * 0.5 + 0.5
        s["weights"] = torch.cat([top, 1 - top], dim=1) * 0.9
        return s
    rows = case["rows"]
    if "experts" in case:
        counts = _segments(case, rng)
        s["longest"] = int(counts.max())
        s["seg"] = torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32, device="cuda")
    if case["op"] == "dgrad":
        s["dy"] = normal(rows, case["n"], scale=0.01)
        s["w"] = _expert_weights(gen, case["experts"], case["n"], case["k"], dtype)
    elif case["op"] == "wgrad":
        s["dy"] = normal(rows, case["n"], scale=0.01)
        s["x"] = normal(rows, case["k"])
    elif case["op"] == "keep":
        s["pre"] = normal(rows, _argument_cols(case))
        if case["act"] == "swiglu":
            s["pre"].unflatten(1, (-1, 2, GROUP))[:, -1, :, case["ffn"] - _packed(case["ffn"]) // 2 + GROUP:] = 0
    elif case["op"] == "unkeep":
        pre = normal(rows, _argument_cols(case))
        if case["act"] == "swiglu":
            pre.unflatten(1, (-1, 2, GROUP))[:, -1, :, case["ffn"] - _packed(case["ffn"]) // 2 + GROUP:] = 0
        s["codes"], s["scales"] = _to_codes(pre.float(), case["keep"])
        s["da"] = normal(rows, case["ffn"], scale=0.01)
    else:
        e, h, f = case["experts"], case["hidden"], case["ffn"]
        s["rows"], s["dout"] = normal(rows, h), normal(rows, h, scale=0.01)
        if case["act"] == "swiglu":
            s["w1"] = _pack(_expert_weights(gen, e, f, h, dtype), _expert_weights(gen, e, f, h, dtype))
        else:
            s["w1"] = _expert_weights(gen, e, f, h, dtype)
        s["w2"] = _expert_weights(gen, e, h, f, dtype)
    return s


# ---- the plain form ----------------------------------------------------------------


def _to_codes(x, keep):
    """x [R, C] in fp32 -> codes [R, C] and a scale for each row's 128 columns.

    The largest magnitude of a group (at least 2^-100) becomes the format's largest value; the codes are rounded to
    nearest, ties to even."""
    r, c = x.shape
    groups = -(-c // GROUP)
    # a tensor: by a number torch would multiply with the reciprocal, which rounds twice
    top = torch.full((r, groups), 127.0 if keep == "int8" else 448.0, device=x.device)
    x = torch.nn.functional.pad(x, (0, groups * GROUP - c)).view(r, groups, GROUP)
    most = x.abs().amax(dim=2).clamp(min=2.0 ** -100)
    q = x * (top / most).unsqueeze(2)
    q = q.round().to(torch.int8) if keep == "int8" else q.to(torch.float8_e4m3fn)
    return q.view(r, groups * GROUP)[:, :c].contiguous(), most / top


def _from_codes(codes, scales):
    if scales is None:
        return codes.float()
    c = codes.shape[1]
    return codes.float() * scales.repeat_interleave(GROUP, dim=1)[:, :c]


def _gate_up(x, ffn):
    """The gate and the up columns of packed ones."""
    pair = x.unflatten(1, (-1, 2, GROUP))
    return pair[:, :, 0].flatten(1)[:, :ffn], pair[:, :, 1].flatten(1)[:, :ffn]


def _activate(pre, act, ffn):
    if act == "swiglu":
        g, u = _gate_up(pre, ffn)
        return g * torch.sigmoid(g) * u
    return pre * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (pre + 0.044715 * pre * pre * pre))


def _activate_backward(da, pre, act, ffn):
    """Gradient of the argument (packed for SwiGLU) and the activation."""
    if act == "swiglu":
        g, u = _gate_up(pre, ffn)
        sig = torch.sigmoid(g)
        dg, du = da * u * sig * (1 + g * (1 - sig)), da * g * sig
        fill = _packed(ffn) // 2 - ffn
        pair = [torch.nn.functional.pad(d, (0, fill)).unflatten(1, (-1, 1, GROUP)) for d in (dg, du)]
        return torch.cat(pair, dim=2).flatten(1), g * sig * u
    c = 2 * math.sqrt(2 / math.pi)
    sig = torch.sigmoid(c * (pre + 0.044715 * pre * pre * pre))
    return da * (sig + pre * sig * (1 - sig) * c * (1 + 3 * 0.044715 * pre * pre)), pre * sig


def _places(s):
    """For every row its place in a table of one equally long block for each expert."""
    seg = s["seg"].long()
    rows = torch.arange(s["case"]["rows"], device=seg.device)
    expert = torch.searchsorted(seg[1:], rows, right=True)
    return expert * s["longest"] + rows - seg[expert]


def _blocks(s, x, places):
    e, longest = s["case"]["experts"], s["longest"]
    table = torch.zeros(e * longest, x.shape[1], dtype=torch.float32, device=x.device)
    table[places] = x.float()
    return table.view(e, longest, x.shape[1])


def _grouped(s, x, w, places):
    """x[r] @ w[seg(r)]"""
    return torch.bmm(_blocks(s, x, places), w.float()).flatten(0, 1)[places]


def _grouped_outer(s, dy, x, places):
    return torch.bmm(_blocks(s, dy, places).transpose(1, 2), _blocks(s, x, places))


def _split(dw, ffn):
    """Packed weight gradients -> those of gate and up."""
    pair = dw.unflatten(1, (-1, 2, GROUP))
    return pair[:, :, 0].flatten(1, 2)[:, :ffn], pair[:, :, 1].flatten(1, 2)[:, :ffn]


def run(state):
    s, case = state, state["case"]
    op, dtype = case["op"], TYPES[case["dtype"]]
    if own:
        return _run_own(s, case)
    if op == "combine":
        dout, pos = s["dout"].float(), s["pos"].long()
        d_rows = torch.empty_like(s["rows_out"])
        d_rows[pos.view(-1)] = (s["weights"].unsqueeze(2) * dout.unsqueeze(1)).flatten(0, 1).to(dtype)
        d_weights = (s["rows_out"].float()[pos] * dout.unsqueeze(1)).sum(dim=2)
        return dict(d_rows=d_rows, d_weights=d_weights)
    if op == "dgrad":
        return dict(dx=_grouped(s, s["dy"], s["w"], _places(s)).to(dtype))
    if op == "wgrad":
        dw = _grouped_outer(s, s["dy"], s["x"], _places(s)).to(dtype)
        if not case["gate_up"]:
            return dict(dw=dw)
        gate, up = _split(dw, case["gate_up"])
        return dict(gate=gate.contiguous(), up=up.contiguous())
    act, ffn = case["act"], case["ffn"]
    if op == "keep":
        pre = s["pre"].float()
        codes, scales = _to_codes(pre, case["keep"])
        return dict(a=_activate(pre, act, ffn).to(dtype), codes=codes, scales=scales)
    if op == "unkeep":
        d_pre, a = _activate_backward(s["da"].float(), _from_codes(s["codes"], s["scales"]), act, ffn)
        return dict(d_pre=d_pre.to(dtype), a=a.to(dtype))
    places = _places(s)
    # what is kept is the product in the operators' type
    pre = _grouped(s, s["rows"], s["w1"].transpose(1, 2), places).to(dtype).float()
    rows_out = _grouped(s, _activate(pre, act, ffn), s["w2"].transpose(1, 2), places)
    kept = (pre, None) if case["keep"] == "none" else _to_codes(pre, case["keep"])
    da = _grouped(s, s["dout"], s["w2"], places)
    d_pre, a = _activate_backward(da, _from_codes(*kept), act, ffn)
    dw2 = _grouped_outer(s, s["dout"], a, places)
    d_rows = _grouped(s, d_pre, s["w1"], places)
    dw1 = _grouped_outer(s, d_pre, s["rows"], places).to(dtype)
    dw1 = tuple(d.contiguous() for d in _split(dw1, ffn)) if act == "swiglu" else dw1
    return dict(rows_out=rows_out.to(dtype), d_rows=d_rows.to(dtype), dw1=dw1, dw2=dw2.to(dtype))


# ---- the framework's calls -------------------------------------------------------------


def _run_own(s, case):
    from dice_b200 import ops

    op = case["op"]
    if op == "combine":
        d_rows, d_weights = ops.combine_backward(s["dout"], s["rows_out"], s["pos"], s["weights"])
        return dict(d_rows=d_rows, d_weights=d_weights)
    if op == "dgrad":
        return dict(dx=ops.grouped_dgrad(s["dy"], s["w"], s["seg"]))
    if op == "wgrad":
        if not case["gate_up"]:
            return dict(dw=ops.grouped_wgrad(s["dy"], s["x"], s["seg"]))
        gate, up = ops.grouped_wgrad(s["dy"], s["x"], s["seg"], gate_up=case["gate_up"])
        return dict(gate=gate, up=up)
    act, ffn = case["act"], case["ffn"]
    if op == "keep":
        a, kept = ops.act_keep(s["pre"], act, ffn, keep=case["keep"])
        return dict(a=a, codes=kept.codes, scales=kept.scales)
    if op == "unkeep":
        d_pre, a = ops.act_backward(s["da"], ops.KeptAct(s["codes"], s["scales"]), act, ffn)
        return dict(d_pre=d_pre, a=a)
    keep = None if case["keep"] == "none" else case["keep"]
    rows_out, kept = ops.grouped_ffn_train(s["rows"], s["w1"], s["w2"], s["seg"], act, ffn, keep=keep)
    d_rows, dw1, dw2 = ops.grouped_ffn_backward(s["dout"], s["rows"], kept, s["w1"], s["w2"], s["seg"], act, ffn)
    return dict(rows_out=rows_out, d_rows=d_rows, dw1=dw1, dw2=dw2)


# ---- the definition, in 64 bits ---------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    f64 = torch.float64

    def swiglu_parts(x, ffn):
        cols = torch.arange(ffn, device=x.device)
        at = cols // GROUP * (2 * GROUP) + cols % GROUP
        return x[..., at], x[..., at + GROUP], at

    def gelu_inner(x):
        return math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)

    def value(x, act, ffn):
        if act == "swiglu":
            g, u, _ = swiglu_parts(x, ffn)
            return u * g / (1 + torch.exp(-g))
        return 0.5 * x * (1 + torch.tanh(gelu_inner(x)))

    def gradient(da, x, act, ffn):
        if act == "swiglu":
            g, u, at = swiglu_parts(x, ffn)
            ex = torch.exp(-g)
            d = torch.zeros_like(x)
            d[..., at] = da * u * (1 / (1 + ex) + g * ex / (1 + ex) ** 2)
            d[..., at + GROUP] = da * g / (1 + ex)
            return d
        t = torch.tanh(gelu_inner(x))
        return da * (0.5 * (1 + t) + 0.5 * x * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * x ** 2))

    def scale_of(x, keep):
        r, c = x.shape
        top = 127.0 if keep == "int8" else 448.0
        parts = [x[:, i:i + GROUP].abs().max(dim=1).values for i in range(0, c, GROUP)]
        return torch.stack(parts, dim=1).clamp(min=2.0 ** -100) / top

    def read_back(x, keep):
        """x after its stay in 8 bits"""
        if keep == "none":
            return x
        scale = scale_of(x, keep)
        for i in range(scale.shape[1]):
            part, sc = x[:, i * GROUP:(i + 1) * GROUP], scale[:, i:i + 1]
            q = torch.round(part / sc) if keep == "int8" else (part / sc).float().to(torch.float8_e4m3fn).to(f64)
            x[:, i * GROUP:(i + 1) * GROUP] = q * sc
        return x

    if op == "combine":
        dout, rows_out, w = s["dout"].to(f64), s["rows_out"].to(f64), s["weights"].to(f64)
        d_rows, d_weights = torch.zeros_like(rows_out), torch.zeros_like(w)
        for k in range(2):
            at = s["pos"][:, k].long()
            d_rows.index_copy_(0, at, w[:, k:k + 1] * dout)
            d_weights[:, k] = torch.einsum("th,th->t", dout, rows_out[at])
        return dict(d_rows=d_rows, d_weights=d_weights)
    if op in ("dgrad", "wgrad"):
        seg = s["seg"].tolist()
        dy = s["dy"].to(f64)
        if op == "dgrad":
            dx = torch.zeros(case["rows"], case["k"], dtype=f64, device=dy.device)
            for e in range(case["experts"]):
                if seg[e + 1] > seg[e]:
                    dx[seg[e]:seg[e + 1]] = dy[seg[e]:seg[e + 1]] @ s["w"][e].to(f64)
            return dict(dx=dx)
        x = s["x"].to(f64)
        dw = torch.stack([dy[seg[e]:seg[e + 1]].T @ x[seg[e]:seg[e + 1]] for e in range(case["experts"])])
        if not case["gate_up"]:
            return dict(dw=dw)
        gate, up, _ = swiglu_parts(dw.transpose(1, 2), case["gate_up"])
        return dict(gate=gate.transpose(1, 2), up=up.transpose(1, 2))
    act, ffn = case["act"], case["ffn"]
    if op == "keep":
        pre = s["pre"].to(f64)
        return dict(a=value(pre, act, ffn), codes=None, scales=scale_of(pre, case["keep"]))
    if op == "unkeep":
        pre = s["codes"].to(f64)
        for i in range(s["scales"].shape[1]):
            pre[:, i * GROUP:(i + 1) * GROUP] *= s["scales"][:, i:i + 1].to(f64)
        return dict(d_pre=gradient(s["da"].to(f64), pre, act, ffn), a=value(pre, act, ffn))
    seg, dtype = s["seg"].tolist(), TYPES[case["dtype"]]
    h, cols = case["hidden"], _argument_cols(case)
    rows_out = torch.zeros(case["rows"], h, dtype=f64, device="cuda")
    d_rows = torch.zeros_like(rows_out)
    dw1 = torch.zeros(case["experts"], cols, h, dtype=f64, device="cuda")
    dw2 = torch.zeros(case["experts"], h, ffn, dtype=f64, device="cuda")
    for e in range(case["experts"]):
        if seg[e + 1] == seg[e]:
            continue
        x, dout = s["rows"][seg[e]:seg[e + 1]].to(f64), s["dout"][seg[e]:seg[e + 1]].to(f64)
        w1, w2 = s["w1"][e].to(f64), s["w2"][e].to(f64)
        pre = x @ w1.T
        pre = pre.to(dtype).to(f64) if dtype != torch.float32 else pre
        rows_out[seg[e]:seg[e + 1]] = value(pre, act, ffn) @ w2.T
        pre = read_back(pre, case["keep"])
        d_pre = gradient(dout @ w2, pre, act, ffn)
        dw2[e] = dout.T @ value(pre, act, ffn)
        d_rows[seg[e]:seg[e + 1]] = d_pre @ w1
        dw1[e] = d_pre.T @ x
    if act == "swiglu":
        gate, up, _ = swiglu_parts(dw1.transpose(1, 2), ffn)
        dw1 = (gate.transpose(1, 2), up.transpose(1, 2))
    return dict(rows_out=rows_out, d_rows=d_rows, dw1=dw1, dw2=dw2)
