"""Device operations of the MoE block: thin wrappers that hand torch CUDA
tensors (device memory + stream only) to the C-ABI kernels.

Every function requires CUDA tensors and the built native library; there is no
CPU or PyTorch fallback.  Names follow the reference's vocabulary: *rows* are
the (token, slot) rows of ``ep_fwd.py:100-111``, *segments* the per-expert runs
of expert-sorted rows.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib

DICE_BF16, DICE_F32 = 0, 1
ACT_SWIGLU, ACT_GELU_TANH = 0, 1
EPI_STORE, EPI_GELU_TANH, EPI_SWIGLU = 0, 1, 2
ACT_CODES = {"swiglu": ACT_SWIGLU, "gelu_tanh": ACT_GELU_TANH}


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return DICE_BF16
    if t.dtype == torch.float32:
        return DICE_F32
    raise TypeError(f"dice_b200 kernels take bfloat16 or float32 tensors, got {t.dtype}")


def _require_cuda(*tensors: Optional[torch.Tensor]) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError(
                "dice_b200 operations run on CUDA tensors only (no CPU fallback); got a tensor on " + str(t.device)
            )


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream() -> int:
    """Raw handle of torch's current stream on the current device."""
    if _raw_stream is not None:  # much cheaper than building a Stream object
        return _raw_stream(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


_stream_objects = {}


def current_stream_object() -> "torch.cuda.Stream":
    """torch's current stream as a Stream object, looked up by its raw handle
    (``torch.cuda.current_stream()`` itself costs several microseconds per call,
    which adds up on the per-layer path of the asynchronous exchange)."""
    if _raw_stream is None:
        return torch.cuda.current_stream()
    dev = torch.cuda.current_device()
    key = (dev, _raw_stream(dev))
    obj = _stream_objects.get(key)
    if obj is None:
        if len(_stream_objects) > 64:
            _stream_objects.clear()
        obj = _stream_objects[key] = torch.cuda.current_stream()
    return obj


def no_grad(fn):
    """``@torch.no_grad()`` that costs nothing when gradients are already off
    (the block's forward enters the no-grad region once; the functions below
    it keep the reference's decorators without paying for them again)."""
    import functools

    @functools.wraps(fn)
    def wrapper(*args, **kwargs):
        if torch.is_grad_enabled():
            with torch.no_grad():
                return fn(*args, **kwargs)
        return fn(*args, **kwargs)

    return wrapper


def check_status(status: torch.Tensor, what: str = "dice_b200 kernel") -> None:
    """Read a device status word (synchronises) and raise if a kernel's bounded
    wait expired."""
    code = int(status.item())
    if code != 0:
        msg = _lib.load().dice_status_message(code).decode()
        status.zero_()
        raise RuntimeError(f"{what}: device status {code}: {msg}")


class _StatusWord:
    """The status word every kernel of this process reports to on one device,
    with a pinned host mirror that is refreshed by asynchronous copies."""

    def __init__(self, device: torch.device):
        self.dev = torch.zeros(1, dtype=torch.int32, device=device)
        self.host = torch.zeros(1, dtype=torch.int32).pin_memory()
        self.event = torch.cuda.Event()
        self.pending = False


_status_words = {}


def _status_word(device) -> _StatusWord:
    device = torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    word = _status_words.get(device)
    if word is None:
        word = _status_words[device] = _StatusWord(device)
    return word


def device_status(device) -> torch.Tensor:
    """The int32 status word shared by the kernels this package launches on
    ``device`` (the first failure wins; see ``dice_status_message``)."""
    return _status_word(device).dev


def poll_status(device=None) -> None:
    """Look at the device status word WITHOUT synchronising: raise if the copy
    enqueued by an earlier call has landed and shows a failure (an expired
    wait, an exchange buffer that was too small, a peer that gave up), then
    enqueue the next copy on the current stream.  Called once per model
    forward and per sampling step by the block and by ``ep_set_step`` /
    ``ep_cache_clear``, so a failure surfaces within a step or two instead of
    turning into silently wrong images."""
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    if torch.cuda.is_current_stream_capturing():
        return
    word = _status_word(device)
    if word.pending:
        if not word.event.query():
            return
        word.pending = False
        code = int(word.host[0])
        if code != 0:
            word.dev.zero_()
            word.host.zero_()
            raise RuntimeError(f"dice_b200 kernels reported device status {code}: "
                               + _lib.load().dice_status_message(code).decode())
    with torch.cuda.device(device):
        word.host.copy_(word.dev, non_blocking=True)
        word.event.record()
    word.pending = True


# --------------------------------------------------------------------------- #
# router
# --------------------------------------------------------------------------- #


def router_top2(
    x2d: torch.Tensor, w_gate: torch.Tensor, renorm: bool = False, want_logits: bool = False,
    status: Optional[torch.Tensor] = None, want_chunks: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """Fused gate: returns ``(topk_idx int64 [N,2], topk_weight fp32 [N,2],
    hist int32 [E], logits or None)``; replaces ``MoEGate.forward``
    (models.py:179-217) and the ``bincount`` of ep_fwd.py:70.

    With ``want_chunks`` (bf16 only) the third result is instead the
    per-128-token histogram table ``int32 [ceil(N/128), E]`` that
    :func:`permute_plan_chunked` consumes."""
    _require_cuda(x2d, w_gate)
    assert x2d.dim() == 2 and w_gate.dim() == 2 and x2d.shape[1] == w_gate.shape[1]
    assert x2d.dtype == w_gate.dtype, "router weight must have the activation dtype"
    x2d = x2d.contiguous()
    w_gate = w_gate.contiguous()
    n, h = x2d.shape
    e = w_gate.shape[0]
    idx = torch.empty((n, 2), dtype=torch.int64, device=x2d.device)
    w = torch.empty((n, 2), dtype=torch.float32, device=x2d.device)
    hist = chunks = None
    if want_chunks:
        chunks = torch.empty(((n + 127) // 128, e), dtype=torch.int32, device=x2d.device)
    else:
        hist = torch.empty((e,), dtype=torch.int32, device=x2d.device)
    logits = torch.empty((n, e), dtype=x2d.dtype, device=x2d.device) if want_logits else None
    lib = _lib.load()
    _lib.check(
        lib.dice_router_top2(
            _ptr(x2d), _ptr(w_gate), n, h, e, _dtype_code(x2d), int(renorm), _ptr(idx), _ptr(w), _ptr(hist),
            _ptr(chunks), _ptr(logits), _ptr(status), _stream(),
        ),
        "dice_router_top2",
    )
    return idx, w, (chunks if want_chunks else hist), logits


def top2_from_logits(logits: torch.Tensor, renorm: bool = False):
    """Selection stage only (softmax + top-2 of models.py:186-196)."""
    _require_cuda(logits)
    logits = logits.contiguous()
    n, e = logits.shape
    idx = torch.empty((n, 2), dtype=torch.int64, device=logits.device)
    w = torch.empty((n, 2), dtype=torch.float32, device=logits.device)
    hist = torch.empty((e,), dtype=torch.int32, device=logits.device)
    lib = _lib.load()
    _lib.check(
        lib.dice_top2_from_logits(_ptr(logits), n, e, _dtype_code(logits), int(renorm), _ptr(idx), _ptr(w), _ptr(hist), _stream()),
        "dice_top2_from_logits",
    )
    return idx, w, hist


# --------------------------------------------------------------------------- #
# permutation
# --------------------------------------------------------------------------- #


def permute_plan(flat_idx: torch.Tensor, n_experts: int, want_order: bool = False):
    """Stable counting sort of rows by expert.  Returns ``(pos int32 [R],
    seg_offsets int32 [E+1], order int32 [R] or None)`` where ``pos[r]`` is the
    sorted position of row ``r`` (the inverse of the reference's
    ``flat_expert_indices.argsort()``, ep_fwd.py:100) and ``order`` is that
    argsort itself."""
    _require_cuda(flat_idx)
    assert flat_idx.dtype == torch.int64 and flat_idx.dim() == 1
    flat_idx = flat_idx.contiguous()
    r = flat_idx.shape[0]
    lib = _lib.load()
    nbytes = lib.dice_permute_scratch_bytes(r, n_experts)
    scratch = torch.empty((max(nbytes, 4) // 4,), dtype=torch.int32, device=flat_idx.device)
    pos = torch.empty((r,), dtype=torch.int32, device=flat_idx.device)
    order = torch.empty((r,), dtype=torch.int32, device=flat_idx.device) if want_order else None
    seg = torch.empty((n_experts + 1,), dtype=torch.int32, device=flat_idx.device)
    _lib.check(
        lib.dice_permute_plan(_ptr(flat_idx), r, n_experts, _ptr(scratch), scratch.numel() * 4, _ptr(pos), _ptr(order),
                              _ptr(seg), _stream()),
        "dice_permute_plan",
    )
    return pos, seg, order


def permute_plan_chunked(flat_idx: torch.Tensor, chunk_hist: torch.Tensor, n_experts: int, world: int = 1,
                         x2d: Optional[torch.Tensor] = None, k: int = 2, want_order: bool = False):
    """The plan in one launch from the router's per-128-token histograms
    (``router_top2(..., want_chunks=True)``), ordered by expert id (``world``
    1) or by ``(owner rank, local slot)`` of the round-robin placement
    (``world`` > 1, etrim.py:23-24).  With ``x2d`` the row gather of
    :func:`permute_rows` is part of the same kernel.  Returns ``(pos, seg_offsets,
    order or None, rows or None)``."""
    _require_cuda(flat_idx, chunk_hist, x2d)
    assert flat_idx.dtype == torch.int64 and flat_idx.dim() == 1 and flat_idx.is_contiguous()
    assert chunk_hist.dtype == torch.int32 and chunk_hist.is_contiguous()
    r = flat_idx.shape[0]
    assert chunk_hist.numel() == (r + 255) // 256 * n_experts
    dev = flat_idx.device
    pos = torch.empty((r,), dtype=torch.int32, device=dev)
    order = torch.empty((r,), dtype=torch.int32, device=dev) if want_order else None
    seg = torch.empty((n_experts + 1,), dtype=torch.int32, device=dev)
    rows, h, code = None, 0, 0
    if x2d is not None:
        assert x2d.is_contiguous() and x2d.shape[0] * k == r
        h, code = x2d.shape[1], _dtype_code(x2d)
        rows = torch.empty((r, h), dtype=x2d.dtype, device=dev)
    _lib.check(
        _lib.load().dice_permute_plan_chunked(_ptr(flat_idx), _ptr(chunk_hist), r, n_experts, world, _ptr(pos), _ptr(order),
                                              _ptr(seg), _ptr(x2d), k, h, code, _ptr(rows), _stream()),
        "dice_permute_plan_chunked",
    )
    return pos, seg, order, rows


# the chunked plan adds the whole per-chunk table up in every CTA: beyond this size use the three-pass plan
PLAN_CHUNKED_MAX_INTS = 16384


def permute_rows(x2d: torch.Tensor, pos: torch.Tensor, k: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[pos[t*k+s]] = x[t]`` — the row gather of ep_fwd.py:107-111."""
    _require_cuda(x2d, pos, out)
    x2d = x2d.contiguous()
    n, h = x2d.shape
    assert pos.dtype == torch.int32 and pos.numel() == n * k
    if out is None:
        out = torch.empty((n * k, h), dtype=x2d.dtype, device=x2d.device)
    assert out.is_contiguous() and out.shape[1] == h and out.shape[0] >= n * k and out.dtype == x2d.dtype
    _lib.check(
        _lib.load().dice_permute_rows(_ptr(x2d), _ptr(pos), n, k, h, _dtype_code(x2d), _ptr(out), _stream()),
        "dice_permute_rows",
    )
    return out


def unpermute_combine(
    src0: torch.Tensor,
    idx0: Optional[torch.Tensor],
    src1: Optional[torch.Tensor],
    idx1: Optional[torch.Tensor],
    w0: Optional[torch.Tensor],
    w1: Optional[torch.Tensor],
    n_tokens: int,
    addend: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    resid: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    tokens_per_sample: int = 1,
) -> torch.Tensor:
    """``y[t] = w0[t]*src0[idx0[t]] + w1[t]*src1[idx1[t]] + addend[t]`` and
    ``out[t] = resid[t] + gate[t // tokens_per_sample] * y[t]`` (residual and
    gate optional: the DiT block's ``x + gate_mlp * moe(...)``, models.py:519).

    ``idx*`` and ``w*`` may be strided 1-D views (e.g. ``pos[0::2]``); the two
    weight views must share one stride.  Replaces ep_fwd.py:172-195."""
    _require_cuda(src0, idx0, src1, idx1, w0, w1, addend, out, resid, gate)
    h = src0.shape[1]
    assert src0.is_contiguous() and (src1 is None or (src1.is_contiguous() and src1.dtype == src0.dtype))
    for i in (idx0, idx1):
        assert i is None or (i.dtype == torch.int32 and i.dim() == 1 and i.shape[0] == n_tokens)
    w_stride = 1
    for w in (w0, w1):
        if w is not None:
            assert w.dtype == torch.float32 and w.dim() == 1 and w.shape[0] == n_tokens
            w_stride = w.stride(0) if n_tokens > 1 else 1
    if w0 is not None and w1 is not None and n_tokens > 1:
        assert w0.stride(0) == w1.stride(0)
    if addend is not None:
        assert addend.is_contiguous() and addend.shape == (n_tokens, h) and addend.dtype == src0.dtype
    if resid is not None:
        assert resid.is_contiguous() and resid.shape == (n_tokens, h) and resid.dtype == src0.dtype
    if gate is not None:
        assert gate.is_contiguous() and gate.dim() == 2 and gate.shape[1] == h and gate.dtype == src0.dtype
        assert gate.shape[0] * tokens_per_sample >= n_tokens
    if out is None:
        out = torch.empty((n_tokens, h), dtype=src0.dtype, device=src0.device)
    assert out.is_contiguous() and out.shape == (n_tokens, h) and out.dtype == src0.dtype
    s0 = idx0.stride(0) if (idx0 is not None and n_tokens > 1) else 1
    s1 = idx1.stride(0) if (idx1 is not None and n_tokens > 1) else 1
    _lib.check(
        _lib.load().dice_unpermute_combine(
            _ptr(src0), _ptr(idx0), s0, _ptr(src1), _ptr(idx1), s1, _ptr(w0), _ptr(w1), w_stride, _ptr(addend),
            _ptr(resid), _ptr(gate), tokens_per_sample, n_tokens, h, _dtype_code(src0), _ptr(out), _stream(),
        ),
        "dice_unpermute_combine",
    )
    return out


def ln_modulate(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, eps: float = 1e-6,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``LayerNorm(x) * (1 + scale[:, None]) + shift[:, None]`` in one pass
    (``modulate(self.norm2(x), shift_mlp, scale_mlp)``, models.py:75-76, :494,
    :519).  ``x`` is ``[B, T, h]``, ``shift`` / ``scale`` are ``[B, h]`` of
    the same dtype (bf16 or fp32); statistics in fp32."""
    _require_cuda(x, shift, scale)
    assert x.dim() == 3 and shift.shape == (x.shape[0], x.shape[2]) and scale.shape == shift.shape
    assert shift.dtype == x.dtype and scale.dtype == x.dtype
    x, shift, scale = x.contiguous(), shift.contiguous(), scale.contiguous()
    b, t, h = x.shape
    out_dtype = out_dtype or x.dtype
    out = torch.empty((b, t, h), dtype=out_dtype, device=x.device)
    code_out = DICE_BF16 if out_dtype == torch.bfloat16 else DICE_F32
    assert out_dtype in (torch.bfloat16, torch.float32)
    _lib.check(
        _lib.load().dice_ln_modulate(_ptr(x), _ptr(shift), _ptr(scale), b * t, h, t, float(eps), _dtype_code(x), code_out,
                                     _ptr(out), _stream()),
        "dice_ln_modulate",
    )
    return out


# --------------------------------------------------------------------------- #
# expert weights and the grouped FFN
# --------------------------------------------------------------------------- #


def w13_rows(ffn: int) -> int:
    return int(_lib.load().dice_w13_rows(ffn))


def pack_w13(gate_proj: torch.Tensor, up_proj: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Interleave ``gate_proj``/``up_proj`` ([F, h] each, models.py:246-247)
    in 128-row blocks for the SwiGLU epilogue."""
    _require_cuda(gate_proj, up_proj, out)
    gate_proj, up_proj = gate_proj.contiguous(), up_proj.contiguous()
    f, h = gate_proj.shape
    assert up_proj.shape == (f, h) and up_proj.dtype == gate_proj.dtype
    rows = w13_rows(f)
    if out is None:
        out = torch.empty((rows, h), dtype=gate_proj.dtype, device=gate_proj.device)
    assert out.shape == (rows, h) and out.is_contiguous()
    _lib.check(
        _lib.load().dice_pack_w13(_ptr(gate_proj), _ptr(up_proj), h, f, _dtype_code(gate_proj), _ptr(out), _stream()),
        "dice_pack_w13",
    )
    return out


def grouped_gemm(
    a: torch.Tensor,
    w: torch.Tensor,
    seg_offsets: torch.Tensor,
    epilogue: int,
    n_out: int,
    status: torch.Tensor,
    seg_slab: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    reserve_sms: int = 0,
) -> torch.Tensor:
    """One grouped GEMM stage on the tensor cores (bf16):
    ``out[r] = epilogue(a[r] @ w[slab(seg(r))].T)``."""
    _require_cuda(a, w, seg_offsets, status, seg_slab, out)
    assert a.dtype == torch.bfloat16 and w.dtype == torch.bfloat16 and a.is_contiguous() and w.is_contiguous()
    assert w.dim() == 3 and a.dim() == 2 and w.shape[2] == a.shape[1]
    assert seg_offsets.dtype == torch.int32 and status.dtype == torch.int32
    n_rows, k_dim = a.shape
    n_slabs, w_rows, _ = w.shape
    n_seg = seg_offsets.numel() - 1
    if out is None:
        out = torch.empty((n_rows, n_out), dtype=torch.bfloat16, device=a.device)
    assert out.dim() == 2 and out.stride(1) == 1 and out.shape[0] >= n_rows
    _lib.check(
        _lib.load().dice_grouped_gemm(
            _ptr(a), n_rows, k_dim, _ptr(w), n_slabs, w_rows, _ptr(seg_offsets), _ptr(seg_slab), n_seg, epilogue,
            _ptr(out), out.stride(0), n_out, reserve_sms, _ptr(status), _stream(),
        ),
        "dice_grouped_gemm",
    )
    return out


def _event_handle(event: Optional[torch.cuda.Event]):
    """The cudaEvent_t behind a torch event (torch creates it at the first record)."""
    if event is None:
        return None
    handle = event.cuda_event
    handle = getattr(handle, "value", handle)
    if not handle:
        raise RuntimeError("the event has never been recorded: torch has not created its CUDA event yet")
    return handle


def grouped_ffn(
    rows: torch.Tensor,
    w1: torch.Tensor,
    w2: torch.Tensor,
    seg_offsets: torch.Tensor,
    act: str,
    ffn: int,
    status: Optional[torch.Tensor] = None,
    seg_slab: Optional[torch.Tensor] = None,
    inter: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    reserve_sms: int = 0,
    shared=None,
    rows_done: Optional[torch.Tensor] = None,
    first_gemm_done: Optional[torch.cuda.Event] = None,
):
    """Expert FFN over expert-sorted rows (ep_fwd.py:199-211; models.py:368-376).

    ``w1``: packed gate/up ``[S, w13_rows(F), h]`` (swiglu) or fc1 ``[S, F, h]``
    (gelu_tanh); ``w2``: ``[S, h, F]``.  bf16 runs on the tensor cores, fp32 on
    the CUDA cores.  ``reserve_sms`` SMs are left to kernels of other streams
    (the side-stream pushes of the asynchronous exchange).

    ``shared = (tokens [N, h], w1 [1, ..., h], w2 [1, h, Fs], Fs)`` (bf16 only)
    runs the block's shared expert over all tokens inside the same two
    launches; the result is then ``(rows_out, shared_out)``.

    ``rows_done`` (bf16 only): zeroed int32 counters, one per 256-row block of
    the output, that the second GEMM raises as blocks complete (a return push
    on another stream follows them); ``first_gemm_done``: an event recorded
    between the two GEMMs (that push's stream waits for it)."""
    _require_cuda(rows, w1, w2, seg_offsets, status, seg_slab, inter, out, rows_done)
    assert rows.is_contiguous() and w1.is_contiguous() and w2.is_contiguous()
    assert seg_offsets.dtype == torch.int32
    n_rows, h = rows.shape
    n_slabs = w1.shape[0]
    n_seg = seg_offsets.numel() - 1
    assert w2.shape == (n_slabs, h, ffn) and w1.shape[2] == h
    if inter is None:
        inter = torch.empty((max(n_rows, 1), ffn), dtype=rows.dtype, device=rows.device)
    if out is None:
        out = torch.empty((n_rows, h), dtype=rows.dtype, device=rows.device)
    assert inter.is_contiguous() and out.is_contiguous() and inter.shape[1] == ffn and inter.shape[0] >= n_rows
    lib = _lib.load()
    if rows.dtype == torch.bfloat16:
        assert status is not None and status.dtype == torch.int32
        sx = sw1 = sw2 = s_inter = s_out = None
        n_shared = s_ffn = 0
        if shared is not None:
            sx, sw1, sw2, s_ffn = shared
            _require_cuda(sx, sw1, sw2)
            assert sx.is_contiguous() and sx.dtype == rows.dtype and sx.shape[1] == h
            assert sw1.is_contiguous() and sw2.is_contiguous() and sw2.shape == (1, h, s_ffn) and sw1.shape[0] == 1
            n_shared = sx.shape[0]
            s_inter = torch.empty((max(n_shared, 1), s_ffn), dtype=rows.dtype, device=rows.device)
            s_out = torch.empty((n_shared, h), dtype=rows.dtype, device=rows.device)
        _lib.check(
            lib.dice_grouped_ffn(
                _ptr(rows), n_rows, h, ffn, ACT_CODES[act], _ptr(w1), _ptr(w2), n_slabs, _ptr(seg_offsets),
                _ptr(seg_slab), n_seg, _ptr(inter), _ptr(out), _ptr(sx), n_shared, s_ffn, _ptr(sw1), _ptr(sw2),
                _ptr(s_inter), _ptr(s_out), reserve_sms, _ptr(rows_done),
                _event_handle(first_gemm_done), _ptr(status), _stream(),
            ),
            "dice_grouped_ffn",
        )
        return (out, s_out) if shared is not None else out
    assert shared is None, "the shared expert rides along in the bf16 kernel only"
    assert rows_done is None, "block counters are the bf16 kernel's"
    if rows.dtype == torch.float32:
        _lib.check(
            lib.dice_grouped_ffn_f32(
                _ptr(rows), n_rows, h, ffn, ACT_CODES[act], _ptr(w1), _ptr(w2), n_slabs, _ptr(seg_offsets),
                _ptr(seg_slab), n_seg, _ptr(inter), _ptr(out), _stream(),
            ),
            "dice_grouped_ffn_f32",
        )
    else:
        raise TypeError(f"unsupported dtype {rows.dtype}")
    return out


def grouped_ffn_combine(rows: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, seg_offsets: torch.Tensor, act: str,
                        ffn: int, order: torch.Tensor, flat_weights: torch.Tensor, status: torch.Tensor,
                        reserve_sms: int = 0) -> torch.Tensor:
    """Expert FFN over expert-sorted rows with the gate-weighted combine
    (models.py:377-381) inside the second GEMM's epilogue: returns ``[N, h]``
    token rows, ``out[t] = sum_s w[t, s] * ffn(row(t, s))``.  bf16, two rows
    per token; ``order`` is the plan's sorted-position -> flat-row map,
    ``flat_weights`` the fp32 top-2 weights viewed flat."""
    _require_cuda(rows, w1, w2, seg_offsets, order, flat_weights, status)
    assert rows.dtype == torch.bfloat16 and rows.is_contiguous() and w1.is_contiguous() and w2.is_contiguous()
    n_rows, h = rows.shape
    assert n_rows % 2 == 0 and order.dtype == torch.int32 and order.numel() == n_rows
    assert flat_weights.dtype == torch.float32 and flat_weights.is_contiguous() and flat_weights.numel() == n_rows
    n_slabs = w1.shape[0]
    inter = torch.empty((max(n_rows, 1), ffn), dtype=rows.dtype, device=rows.device)
    out = torch.empty((n_rows // 2, h), dtype=rows.dtype, device=rows.device)
    _lib.check(
        _lib.load().dice_grouped_ffn_combine(
            _ptr(rows), n_rows, h, ffn, ACT_CODES[act], _ptr(w1), _ptr(w2), n_slabs, _ptr(seg_offsets), None,
            seg_offsets.numel() - 1, _ptr(inter), _ptr(order), _ptr(flat_weights), 2, _ptr(out), reserve_sms, _ptr(status),
            _stream(),
        ),
        "dice_grouped_ffn_combine",
    )
    return out


def shared_expert_can_ride() -> bool:
    """Whether the grouped-FFN launches can carry the shared expert as an extra
    problem (the CTA-pair kernel can; ``DICE_GEMM_PAIR=0`` selects the
    one-CTA-per-tile kernel, which cannot)."""
    import os

    return os.environ.get("DICE_GEMM_PAIR", "1") != "0"


# --------------------------------------------------------------------------- #
# the training step: gradients of the grouped products, 8-bit kept activations
# --------------------------------------------------------------------------- #

KEEP_CODES = {None: 0, "int8": 1, "e4m3": 2}
KEEP_NOTHING = 3  # no backward pass will follow
KEEP_DTYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
KEEP_GROUP = 128  # columns that share a scale


class KeptAct(NamedTuple):
    """What the forward pass keeps of an activation's argument: ``codes`` int8 or float8_e4m3fn ``[R, C]`` with fp32
    ``scales [R, ceil(C / 128)]`` (the value is ``code * scale``), or the argument itself with ``scales`` None."""

    codes: torch.Tensor
    scales: Optional[torch.Tensor]

    @property
    def keep(self) -> Optional[str]:
        return None if self.scales is None else "int8" if self.codes.dtype == torch.int8 else "e4m3"


# The small calls of a training step are bounded by the host: one token's gradients cost the GPU a few microseconds, and
# every torch.empty with keyword arguments two, every look-up of a device half of one.  Hence one comparison per tensor,
# written out, allocations through torch's own short path where it exists, and widths computed here.
# That path goes past dispatch modes and past the filling of uninitialised memory that deterministic algorithms may ask
# for, so it is not taken where either is on.
_empty_cuda = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None)
_dispatch_modes = getattr(torch._C, "_len_torch_dispatch_stack", None)
_deterministic = getattr(torch._C, "_get_deterministic_algorithms", torch.are_deterministic_algorithms_enabled)
if _dispatch_modes is None:
    _empty_cuda = None


def _new(shape: Tuple[int, ...], dtype: torch.dtype, index: int) -> torch.Tensor:
    """An uninitialised contiguous tensor on the current device, which is number ``index``."""
    if _empty_cuda is not None and not _deterministic() and not _dispatch_modes():
        stride = (shape[1], 1) if len(shape) == 2 else (shape[1] * shape[2], shape[2], 1)
        return _empty_cuda(shape, stride, dtype)
    return torch.empty(shape, dtype=dtype, device=torch.device("cuda", index))


def _one_device(*tensors: Optional[torch.Tensor]) -> int:
    """The number of the CUDA device that all these tensors are on."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and (index < 0 or t.get_device() != index):
            _require_cuda(*tensors)
            raise RuntimeError(f"all tensors of a call must be on one device, got {tensors[0].device} and {t.device}")
    return index


# Launches go to the current device's current stream, so a call on another device's tensors makes that device current.
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _stream_of(index: int) -> int:
    return _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


def _status_ptr(status: Optional[torch.Tensor], index: int) -> int:
    if status is None:
        word = _status_by_index.get(index)
        if word is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("call dice_b200.ops.device_status(device) once before capturing a graph")
            word = _status_by_index[index] = device_status(torch.device("cuda", index)).data_ptr()
        return word
    assert status.dtype == torch.int32 and status.numel() >= 1
    return status.data_ptr()


_status_by_index = {}  # device number -> address of its status word, which lives as long as the process


PRODUCT_DGRAD, PRODUCT_WGRAD, PRODUCT_LINEAR = 0, 1, 2
THIN_ROWS = 4  # as kThinTotal of csrc/train.cuh


def _split_bytes(lib, n_rows: int, n_dim: int, k_dim: int, n_slabs: int, product: int, code: int) -> int:
    """dice_grouped_scratch_bytes; bf16 products with more tiles than any GPU has SM pairs for are not asked about, nor
    the input gradients of few rows, which have a kernel of their own."""
    if code == DICE_BF16:
        col_tiles = (k_dim + 127) // 128
        if product == PRODUCT_WGRAD:
            few = 2 * n_slabs * ((n_dim + 255) // 256) * col_tiles <= 128
        else:
            few = product == PRODUCT_DGRAD and n_rows > THIN_ROWS and 4 * ((n_rows + 255) // 256) * col_tiles <= 128
        if not few:
            return 0
    return lib.dice_grouped_scratch_bytes(n_rows, n_dim, k_dim, n_slabs, product, code)


def _split_scratch(index: int, n_bytes: int) -> Tuple[Optional[torch.Tensor], Optional[int], int]:
    """A product's scratch (the tensor, which the caller holds until the launch, its address and its size)."""
    if n_bytes == 0:
        return None, None, 0
    scratch = _new((1, n_bytes), torch.uint8, index)
    return scratch, scratch.data_ptr(), n_bytes


def _check_segments(seg_offsets: torch.Tensor) -> int:
    assert seg_offsets.dtype == torch.int32 and seg_offsets.dim() == 1 and seg_offsets.is_contiguous()
    assert seg_offsets.numel() >= 1, "seg_offsets holds one offset more than there are segments"
    return seg_offsets.numel() - 1


def _check_out(out: torch.Tensor, *operands: torch.Tensor) -> None:
    """The kernels write ``out`` while they still read their (contiguous) operands."""
    begin = out.data_ptr()
    end = begin + out.numel() * out.element_size()
    for t in operands:
        if t.data_ptr() < end and begin < t.data_ptr() + t.numel() * t.element_size():
            raise ValueError("out shares memory with an operand")


def act_columns(act: str, ffn: int) -> int:
    """Columns of an activation's argument: ``ffn``, or the packed gate / up width of SwiGLU (``w13_rows(ffn)``)."""
    if act == "swiglu":
        return (ffn + 127) // 128 * 256
    if act not in ACT_CODES:
        raise ValueError(f"unknown activation {act!r}")
    return ffn


def grouped_dgrad(dy: torch.Tensor, w: torch.Tensor, seg_offsets: torch.Tensor, status: Optional[torch.Tensor] = None,
                  seg_slab: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Input gradient of :func:`grouped_gemm`: ``dx[r] = dy[r] @ w[slab(seg(r))]`` with ``dy [R, N]``,
    ``w [S, N, K]`` (bf16 or fp32).  Rows of no segment are left as they are in ``out`` (uninitialised without it), which
    shares no memory with the operands."""
    index = _one_device(dy, w, seg_offsets, status, seg_slab, out)
    if index != _current_device():
        with torch.cuda.device(index):
            return grouped_dgrad(dy, w, seg_offsets, status, seg_slab, out)
    assert dy.dim() == 2 and w.dim() == 3 and w.dtype == dy.dtype
    n_seg = _check_segments(seg_offsets)
    assert seg_slab is None or (seg_slab.dtype == torch.int32 and seg_slab.is_contiguous() and seg_slab.numel() == n_seg)
    code = _dtype_code(dy)
    dy, w = dy.contiguous(), w.contiguous()
    n_rows, n_dim = dy.shape
    n_slabs, w_rows, k_dim = w.shape
    assert w_rows == n_dim
    if out is None:
        out = _new((n_rows, k_dim), dy.dtype, index)
    else:
        _check_out(out, dy, w)
    assert out.is_contiguous() and out.shape == (n_rows, k_dim) and out.dtype == dy.dtype
    lib = _lib.load()
    held, scratch, n_bytes = _split_scratch(index, _split_bytes(lib, n_rows, n_dim, k_dim, n_slabs, PRODUCT_DGRAD, code))
    _lib.check(
        lib.dice_grouped_dgrad(dy.data_ptr(), n_rows, n_dim, w.data_ptr(), n_slabs, k_dim, seg_offsets.data_ptr(),
                               _ptr(seg_slab), n_seg, code, out.data_ptr(), scratch, n_bytes, _status_ptr(status, index),
                               _stream_of(index)),
        "dice_grouped_dgrad",
    )
    return out


def grouped_wgrad(dy: torch.Tensor, x: torch.Tensor, seg_offsets: torch.Tensor, status: Optional[torch.Tensor] = None,
                  gate_up: Optional[int] = None):
    """Weight gradient of :func:`grouped_gemm`: ``dw[s] = dy[seg s].T @ x[seg s]`` ``[S, N, K]`` in the rows' type, zero
    for a segment without rows.  ``gate_up=ffn``: ``dy`` has the packed gate / up columns of :func:`pack_w13`, and the
    result is the pair of gradients ``[S, ffn, K]`` of the gate and the up projections."""
    index = _one_device(dy, x, seg_offsets, status)
    if index != _current_device():
        with torch.cuda.device(index):
            return grouped_wgrad(dy, x, seg_offsets, status, gate_up)
    assert dy.dim() == 2 and x.dim() == 2 and x.dtype == dy.dtype
    n_slabs = _check_segments(seg_offsets)
    assert n_slabs >= 1
    assert gate_up is None or gate_up > 0
    code = _dtype_code(dy)
    dy, x = dy.contiguous(), x.contiguous()
    n_rows, n_dim = dy.shape
    x_rows, k_dim = x.shape
    assert x_rows == n_rows
    shape = (n_slabs, gate_up or n_dim, k_dim)
    dw = _new(shape, dy.dtype, index)
    dw_up = _new(shape, dy.dtype, index) if gate_up else None
    lib = _lib.load()
    held, scratch, n_bytes = _split_scratch(index, _split_bytes(lib, n_rows, n_dim, k_dim, n_slabs, PRODUCT_WGRAD, code))
    _lib.check(
        lib.dice_grouped_wgrad(dy.data_ptr(), x.data_ptr(), n_rows, n_dim, k_dim, seg_offsets.data_ptr(), n_slabs,
                               gate_up or 0, code, dw.data_ptr(), _ptr(dw_up), scratch, n_bytes, _status_ptr(status, index),
                               _stream_of(index)),
        "dice_grouped_wgrad",
    )
    return (dw, dw_up) if gate_up else dw


def _groups(cols: int) -> int:
    return (cols + KEEP_GROUP - 1) // KEEP_GROUP


def _check_kept(codes: torch.Tensor, scales: Optional[torch.Tensor], n_rows: int, cols: int, dtype: torch.dtype) -> int:
    """The keep code of what was kept for ``n_rows`` rows of ``cols`` columns."""
    assert codes.shape == (n_rows, cols) and codes.is_contiguous()
    if scales is None:
        assert codes.dtype == dtype
        return 0
    assert scales.dtype == torch.float32 and scales.is_contiguous() and scales.shape == (n_rows, _groups(cols))
    if codes.dtype == torch.int8:
        return 1
    if codes.dtype != torch.float8_e4m3fn:
        raise TypeError(f"codes are int8 or float8_e4m3fn, got {codes.dtype}")
    return 2


def _check_keep(keep: Optional[str]) -> None:
    if keep not in KEEP_CODES:
        raise ValueError(f"keep is None, 'int8' or 'e4m3', got {keep!r}")


def act_keep(pre: torch.Tensor, act: str, ffn: int, keep: Optional[str] = "int8") -> Tuple[torch.Tensor, KeptAct]:
    """The activation ``a [R, ffn]`` of ``pre`` (SwiGLU: packed gate / up columns ``[R, w13_rows(ffn)]``; GELU:
    ``[R, ffn]``) and, in the same pass, ``pre`` in 8 bits for :func:`act_backward`: every row's 128 columns share a
    scale.  ``keep=None`` keeps ``pre`` itself."""
    _check_keep(keep)
    index = _one_device(pre)
    if index != _current_device():
        with torch.cuda.device(index):
            return act_keep(pre, act, ffn, keep)
    cols = act_columns(act, ffn)
    assert pre.dim() == 2
    code = _dtype_code(pre)
    pre = pre.contiguous()
    n_rows, pre_cols = pre.shape
    assert pre_cols == cols
    a = _new((n_rows, ffn), pre.dtype, index)
    if keep is None:
        kept, codes_ptr, scales_ptr = KeptAct(pre, None), None, None
    else:
        kept = KeptAct(_new((n_rows, cols), KEEP_DTYPES[keep], index), _new((n_rows, _groups(cols)), torch.float32, index))
        codes_ptr, scales_ptr = kept.codes.data_ptr(), kept.scales.data_ptr()
    _lib.check(
        _lib.load().dice_act_keep(pre.data_ptr(), n_rows, ffn, ACT_CODES[act], KEEP_CODES[keep], code, a.data_ptr(), codes_ptr,
                                  scales_ptr, _stream_of(index)),
        "dice_act_keep",
    )
    return a, kept


def act_backward(da: torch.Tensor, kept: KeptAct, act: str, ffn: int, want_act: bool = True):
    """Backward pass of :func:`act_keep`: ``(d_pre, a)`` from the activation's gradient ``da [R, ffn]`` and what was
    kept; ``a`` is the activation of the kept argument (None without ``want_act``), which the second product's weight
    gradient needs."""
    codes, scales = kept
    index = _one_device(da, codes, scales)
    if index != _current_device():
        with torch.cuda.device(index):
            return act_backward(da, kept, act, ffn, want_act)
    cols = act_columns(act, ffn)
    assert da.dim() == 2
    code = _dtype_code(da)
    n_rows, da_cols = da.shape
    assert da_cols == ffn
    keep = _check_kept(codes, scales, n_rows, cols, da.dtype)
    da = da.contiguous()
    d_pre = _new((n_rows, cols), da.dtype, index)
    a = _new((n_rows, ffn), da.dtype, index) if want_act else None
    _lib.check(
        _lib.load().dice_act_backward(da.data_ptr(), codes.data_ptr(), _ptr(scales), n_rows, ffn, ACT_CODES[act], keep, code,
                                      d_pre.data_ptr(), _ptr(a), _stream_of(index)),
        "dice_act_backward",
    )
    return d_pre, a


def combine_backward(dout: torch.Tensor, rows_out: torch.Tensor, pos: torch.Tensor, weights: torch.Tensor):
    """Gradient of the gate-weighted sum of a token's two rows (:func:`unpermute_combine`): ``d_rows [R, h]`` with
    ``d_rows[pos[t, s]] = weights[t, s] * dout[t]`` and ``d_weights [N, 2]`` fp32 ``= <dout[t], rows_out[pos[t, s]]>``.
    ``pos`` int32 ``[N, 2]`` names no row twice (a plan's); rows that it does not name are left uninitialised, a
    position outside ``rows_out`` has gradient 0."""
    index = dout.get_device()
    if index < 0 or rows_out.get_device() != index or pos.get_device() != index or weights.get_device() != index:
        _one_device(dout, rows_out, pos, weights)
    if index != _current_device():
        with torch.cuda.device(index):
            return combine_backward(dout, rows_out, pos, weights)
    assert dout.dim() == 2 and rows_out.dim() == 2
    n_tokens, h = dout.shape
    n_rows, row_cols = rows_out.shape
    dtype = dout.dtype
    assert row_cols == h and rows_out.dtype == dtype
    assert pos.dtype == torch.int32 and pos.shape == (n_tokens, 2)
    assert weights.dtype == torch.float32 and weights.shape == (n_tokens, 2)
    code = _dtype_code(dout)
    dout, rows_out, pos, weights = dout.contiguous(), rows_out.contiguous(), pos.contiguous(), weights.contiguous()
    d_rows = _new((n_rows, h), dtype, index)
    d_weights = _new((n_tokens, 2), torch.float32, index)
    rc = _lib.load().dice_combine_backward(dout.data_ptr(), rows_out.data_ptr(), pos.data_ptr(), weights.data_ptr(), n_tokens,
                                           n_rows, h, code, d_rows.data_ptr(), d_weights.data_ptr(), _stream_of(index))
    if rc:
        _lib.check(rc, "dice_combine_backward")
    return d_rows, d_weights


def _check_ffn(rows, w1, w2, seg_offsets, act, ffn):
    cols = act_columns(act, ffn)
    assert rows.dim() == 2 and w1.dim() == 3 and w2.dim() == 3
    n_slabs, h = w1.shape[0], rows.shape[1]
    assert w1.shape == (n_slabs, cols, h) and w2.shape == (n_slabs, h, ffn)
    assert w1.dtype == rows.dtype and w2.dtype == rows.dtype and w1.is_contiguous() and w2.is_contiguous()
    assert _check_segments(seg_offsets) == n_slabs, "one segment per expert"
    return n_slabs, h, cols


def grouped_ffn_train(rows: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, seg_offsets: torch.Tensor, act: str, ffn: int,
                      status: Optional[torch.Tensor] = None, keep: Optional[str] = None, want_kept: bool = True):
    """:func:`grouped_ffn` for training: ``(rows_out, kept)``, where ``kept`` is the activation's argument as it is
    (``keep`` None) or in 8 bits ("int8" or "e4m3"), for :func:`grouped_ffn_backward`; None without ``want_kept``, when no
    backward pass will follow.  The first product is rounded to the rows' type before the activation, and the activation
    before the second product (and the argument's gradient in the backward pass): in bf16 a result is 2.4e-3 of its norm
    from 64 bits, where its own rounding alone is 1.7e-3.  fp32 rows and weights have fp32's precision throughout (three
    bf16 planes an operand on the tensor cores, or the CUDA cores where few rows meet a weight)."""
    _check_keep(keep)
    index = _one_device(rows, w1, w2, seg_offsets, status)
    if index != _current_device():
        with torch.cuda.device(index):
            return grouped_ffn_train(rows, w1, w2, seg_offsets, act, ffn, status, keep, want_kept)
    code = _dtype_code(rows)
    n_slabs, h, cols = _check_ffn(rows, w1, w2, seg_offsets, act, ffn)
    rows = rows.contiguous()
    n_rows, dt = rows.shape[0], rows.dtype
    # bf16 makes the activation and the 8-bit codes in the first product's epilogue
    pre = _new((n_rows, cols), dt, index) if (keep is None and want_kept) or code == DICE_F32 else None
    a = _new((n_rows, ffn), dt, index)
    rows_out = _new((n_rows, h), dt, index)
    codes = scales = kept = None
    if not want_kept:
        keep_code = KEEP_NOTHING
    elif keep is None:
        keep_code, kept = KEEP_CODES[None], KeptAct(pre, None)
    else:
        keep_code = KEEP_CODES[keep]
        codes, scales = kept = KeptAct(_new((n_rows, cols), KEEP_DTYPES[keep], index),
                                       _new((n_rows, _groups(cols)), torch.float32, index))
    lib = _lib.load()
    held, scratch, n_bytes = _split_scratch(index, 0 if code == DICE_BF16 else max(
        _split_bytes(lib, n_rows, n, k, n_slabs, PRODUCT_LINEAR, code) for n, k in ((cols, h), (h, ffn))))
    _lib.check(
        lib.dice_grouped_ffn_train(
            rows.data_ptr(), n_rows, h, ffn, ACT_CODES[act], keep_code, code, w1.data_ptr(), w2.data_ptr(), n_slabs,
            seg_offsets.data_ptr(), n_slabs, _ptr(pre), a.data_ptr(), _ptr(codes), _ptr(scales), rows_out.data_ptr(), scratch,
            n_bytes, _status_ptr(status, index), _stream_of(index),
        ),
        "dice_grouped_ffn_train",
    )
    return rows_out, kept


def grouped_ffn_backward(d_out: torch.Tensor, rows: torch.Tensor, kept: KeptAct, w1: torch.Tensor, w2: torch.Tensor,
                         seg_offsets: torch.Tensor, act: str, ffn: int, status: Optional[torch.Tensor] = None,
                         want_rows: bool = True, want_w1: bool = True, want_w2: bool = True):
    """Backward pass of :func:`grouped_ffn_train` from what it kept: ``(d_rows, dw1, dw2)``; for SwiGLU ``dw1`` is the
    pair of the gate and the up projections' gradients ``[S, ffn, h]``.  A gradient that is not wanted is not made, and
    None in its place (dw2 comes along where dw1 is wanted)."""
    codes, scales = kept
    index = _one_device(d_out, rows, codes, scales, w1, w2, seg_offsets, status)
    if index != _current_device():
        with torch.cuda.device(index):
            return grouped_ffn_backward(d_out, rows, kept, w1, w2, seg_offsets, act, ffn, status, want_rows, want_w1, want_w2)
    code = _dtype_code(rows)
    n_slabs, h, cols = _check_ffn(rows, w1, w2, seg_offsets, act, ffn)
    n_rows, dt = rows.shape[0], rows.dtype
    assert d_out.shape == rows.shape and d_out.dtype == dt
    keep = _check_kept(codes, scales, n_rows, cols, dt)
    d_out, rows = d_out.contiguous(), rows.contiguous()
    want_w2 = want_w2 or want_w1
    if not (want_rows or want_w2):
        return None, None, None
    da = _new((n_rows, ffn), dt, index) if code == DICE_F32 else None  # bf16: stays in the product's epilogue
    d_pre, a = _new((n_rows, cols), dt, index), _new((n_rows, ffn), dt, index)
    d_rows = _new((n_rows, h), dt, index) if want_rows else None
    dw2 = _new((n_slabs, h, ffn), dt, index) if want_w2 else None
    dw1 = _new((n_slabs, ffn, h), dt, index) if want_w1 else None
    dw1_up = _new((n_slabs, ffn, h), dt, index) if want_w1 and act == "swiglu" else None
    lib = _lib.load()
    held, scratch, n_bytes = _split_scratch(index, max(
        _split_bytes(lib, n_rows, n, k, n_slabs, product, code) if made else 0
        for n, k, product, made in ((h, ffn, PRODUCT_DGRAD, code == DICE_F32), (h, ffn, PRODUCT_WGRAD, want_w2),
                                    (cols, h, PRODUCT_DGRAD, want_rows), (cols, h, PRODUCT_WGRAD, want_w1))))
    _lib.check(
        lib.dice_grouped_ffn_backward(
            d_out.data_ptr(), rows.data_ptr(), codes.data_ptr(), _ptr(scales), n_rows, h, ffn, ACT_CODES[act], keep, code,
            w1.data_ptr(), w2.data_ptr(), n_slabs, seg_offsets.data_ptr(), _ptr(da), d_pre.data_ptr(), a.data_ptr(),
            _ptr(d_rows), _ptr(dw1), _ptr(dw1_up), _ptr(dw2), scratch, n_bytes, _status_ptr(status, index),
            _stream_of(index),
        ),
        "dice_grouped_ffn_backward",
    )
    return d_rows, (dw1 if dw1_up is None else (dw1, dw1_up)), dw2
