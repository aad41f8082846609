"""The operators of a decode step around the expert layers: new keys and values go into a paged cache
with the position rotation applied, one new token per sequence attends over that cache, the residual
is added and normalised, and the logits get their penalties, biases and grammar masks.

The reference leaves these to stock PyTorch (attention, norms and rotation of its model files,
modeling_olmoe.py:300-618, 1120-1200; greedy argmax in tools/benchmark_e2e_grid.py:325-420).  All of
them run on the current stream, allocate only what they return (and scratch), and never synchronise,
so they can be captured in a CUDA graph.  There is no CPU path: tensors must live on a CUDA device.
Nor is there a backward pass: where gradients are recorded, inputs that require one are refused.

Pages.  ``k_pages`` and ``v_pages`` are ``[num_pages, page_size, num_kv_heads, head_dim]`` with any
strides that are multiples of 16 bytes and the head's dimensions side by side; fastest is one where a head's tokens of a page
are, too (allocate ``[num_pages, num_kv_heads, page_size, head_dim]`` and pass ``.transpose(1, 2)``).  They hold the
rows' type (fp16 or bf16) or ``torch.float8_e4m3fn`` with one scale per head.  Token ``i`` of sequence ``b`` is in page
``block_table[b, i // page_size]``.  ``status`` is an optional int32 tensor of one element, zero
at first: a page, position or length that does not fit sets it (``raise_on_status``).
"""
from __future__ import annotations

import struct
from typing import Optional

import torch

from . import _native

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2, torch.float8_e4m3fn: 3}
_ROWS = (torch.float16, torch.bfloat16)
_LOGIT_TYPES = (torch.float16, torch.bfloat16, torch.float32)
# the structs of include/trismoe_b200.h, field by field (packing bytes takes a third of the time of a ctypes structure)
_PAGED_KV = struct.Struct("@2Q6q3Qq8iQ")
_APPEND = struct.Struct("@3Q6q6Q8i")
_ATTENTION = struct.Struct("@Q2q4Qq3if")
_NORM = struct.Struct("@6Q4q5if")
_LOGITS = struct.Struct("@11Q5q6i")
_NO_GRADIENT = "an input requires a gradient, and there is none: call it under torch.no_grad(), or with detached tensors"
# (device, sizes) -> a byte seen as many, whose like is the scratch of a call; None where there is none to have
_scratch: dict = {}


def _fail(what: str, why: str):
    raise RuntimeError(f"trismoe_b200 {what}: {why}")


def _same_device(what: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> torch.device:
    index = first.get_device()
    if index < 0:
        _native.require_cuda(first, what)
    grad = torch.is_grad_enabled()
    if grad and first.requires_grad:
        _fail(what, _NO_GRADIENT)
    for t in others:
        if t is not None:
            if t.get_device() != index:
                _fail(what, "all tensors must live on one CUDA device")
            if grad and t.requires_grad:
                _fail(what, _NO_GRADIENT)
    return first.device


def _want(what: str, name: str, t: torch.Tensor, dtype, shape: tuple) -> int:
    """Address of a contiguous tensor of that type and shape."""
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        _fail(what, f"{name} must be contiguous {dtype} of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _matrix(what: str, name: str, t: torch.Tensor, dtype, rows: int, columns: Optional[int] = None) -> tuple:
    """Address, row stride and columns of a matrix whose rows lie side by side in themselves."""
    shape = t.shape
    if len(shape) != 2 or t.dtype is not dtype or shape[0] != rows or (columns is not None and shape[1] != columns) or (t.stride(1) != 1 and shape[1] > 1):
        _fail(what, f"{name} must be {dtype} [{rows}, {'any' if columns is None else columns}] with a row side by side, got {t.dtype} {tuple(shape)}")
    return t.data_ptr(), t.stride(0), shape[1]


def _new_like(t: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Contiguous, of t's shape and device, and t's type unless told otherwise (torch.empty with those spelled out takes twice as long)."""
    return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


def _launch(what: str, name: str, dev: torch.device, *structs: bytes) -> None:
    """Calls an entry point of the library on the device's current stream."""
    entry = getattr(_native._lib or _native.load(), name)
    if dev.index == torch._C._cuda_getDevice():
        status = entry(*structs, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            status = entry(*structs, _native.stream_of(dev))
    if status:
        _native.check(status, what)


def _cache(what: str, k_pages, v_pages, block_table, k_scale, v_scale, status) -> tuple:
    """The cache as the library takes it, and (dtype, heads, head_dim, sequences, table width, page size) of it."""
    shape, dtype = k_pages.shape, k_pages.dtype
    if len(shape) != 4 or shape != v_pages.shape or dtype is not v_pages.dtype or dtype not in _DTYPES:
        _fail(what, "k_pages and v_pages must have the same type and shape [num_pages, page_size, num_kv_heads, head_dim]")
    pages, page_size, heads, dim = shape
    k0, k1, k2, k3 = k_pages.stride()
    v0, v1, v2, v3 = v_pages.stride()
    if k3 != 1 or v3 != 1:
        _fail(what, "the dimensions of a head must be side by side")
    if block_table.dim() != 2 or block_table.dtype is not torch.int32:
        _fail(what, "block_table must be int32 [sequences, pages]")
    sequences, width = block_table.shape
    t0, t1 = block_table.stride()
    if t1 != 1 and width > 1:
        _fail(what, "block_table must have the pages of a sequence side by side")
    if (k_scale is not None or v_scale is not None) and dtype is not torch.float8_e4m3fn:
        _fail(what, "scales belong to e4m3 pages")
    packed = _PAGED_KV.pack(
        k_pages.data_ptr(), v_pages.data_ptr(), k0, k1, k2, v0, v1, v2,
        0 if k_scale is None else _want(what, "k_scale", k_scale, torch.float32, (heads,)),
        0 if v_scale is None else _want(what, "v_scale", v_scale, torch.float32, (heads,)),
        block_table.data_ptr(), t0, sequences, width, pages, page_size, heads, dim,
        _DTYPES[dtype], 0, 0 if status is None else _want(what, "status", status, torch.int32, (1,)))
    return packed, (dtype, heads, dim, sequences, width, page_size)


def raise_on_status(status: torch.Tensor, what: str = "paged cache") -> None:
    """Reads a status word (waits for the GPU), and raises if an operator has set it."""
    word = int(status.item())
    if word:
        raise RuntimeError(f"trismoe_b200 {what}: a kernel reported {_native.STATUS_NAMES.get(word, word)} "
                           "(a page, position or length outside the cache, its block table or the rotation tables)")


def append_paged_kv(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    block_table: torch.Tensor, positions: torch.Tensor, sequences: Optional[torch.Tensor] = None, *,
                    cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, interleaved: bool = False,
                    k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None, return_key: bool = False,
                    status: Optional[torch.Tensor] = None):
    """Rotates queries and keys by their positions and writes keys and values to the cache.

    ``q`` [tokens, q heads, head_dim] (or None), ``k`` and ``v`` [tokens, kv heads, head_dim]: views into one projection's output are
    fine.  Token ``t`` belongs to sequence ``sequences[t]`` (int32; default: ``t``, of which the block table must have as many) and stands at ``positions[t]`` (int32 or
    int64; negative: padding, not written).  ``cos`` and ``sin`` [positions, rotary_dim / 2] in fp32 rotate the first ``rotary_dim``
    dimensions, pairs ``(i, i + rotary_dim / 2)`` or, ``interleaved``, ``(2 i, 2 i + 1)``; None: no rotation.  e4m3 pages get
    ``x / scale``, saturated.  Tokens of one call must have different places.  Returns the rotated queries (None without ``q``),
    with ``return_key`` a pair with the rotated keys."""
    what = "append_paged_kv"
    dev = _same_device(what, k, v, q, k_pages, v_pages, block_table, positions, sequences, cos, sin, k_scale, v_scale, status)
    cache, (_, cache_heads, cache_dim, table_sequences, _, _) = _cache(what, k_pages, v_pages, block_table, k_scale, v_scale, status)
    shape, dtype = k.shape, k.dtype
    if len(shape) != 3 or v.shape != shape or dtype not in _ROWS or v.dtype is not dtype:
        _fail(what, "k and v must be fp16 or bf16 [tokens, num_kv_heads, head_dim]")
    tokens, heads, dim = shape
    if heads != cache_heads or dim != cache_dim:
        _fail(what, f"k {tuple(shape)} does not fit pages of num_kv_heads {cache_heads} and head_dim {cache_dim}")
    wide = positions.dtype is torch.int64
    at = _want(what, "positions", positions, torch.int64 if wide else torch.int32, (tokens,))
    if sequences is not None:
        sequence_at = _want(what, "sequences", sequences, torch.int32, (tokens,))
    elif tokens <= table_sequences:
        sequence_at = 0
    else:
        _fail(what, f"{tokens} tokens without sequences do not fit a block table of {table_sequences} sequences")
    k0, k1, k2 = k.stride()
    v0, v1, v2 = v.stride()
    q_at = q0 = q1 = q_heads = out_at = 0
    q2, q_out, k_out = 1, None, None
    if q is not None:
        if q.dim() != 3 or q.dtype is not dtype or q.shape[0] != tokens or q.shape[2] != dim:
            _fail(what, "q must be [tokens, q heads, head_dim] in the keys' type")
        q_at, q_heads = q.data_ptr(), q.shape[1]
        q0, q1, q2 = q.stride()
        q_out = _new_like(q)
        out_at = q_out.data_ptr()
    if (k2 != 1 or v2 != 1 or q2 != 1) and dim > 1:
        _fail(what, "the dimensions of a head must be side by side")
    rows = half = cos_at = sin_at = 0
    if cos is not None or sin is not None:
        if cos is None or sin is None or cos.dim() != 2 or cos.shape != sin.shape or not (cos.is_contiguous() and sin.is_contiguous()) \
                or cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
            _fail(what, "cos and sin go together, contiguous fp32 [positions, rotary_dim / 2] each")
        rows, half = cos.shape
        cos_at, sin_at = cos.data_ptr(), sin.data_ptr()
    if return_key:
        k_out = _new_like(k)
    args = _APPEND.pack(q_at, k.data_ptr(), v.data_ptr(), q0, q1, k0, k1, v0, v1, cos_at, sin_at, at, sequence_at, out_at,
                        0 if k_out is None else k_out.data_ptr(), tokens, q_heads, 2 * half, rows, wide, bool(interleaved), _DTYPES[dtype], 0)
    _launch(what, "tris_paged_kv_append", dev, cache, args)
    return (q_out, k_out) if return_key else q_out


def paged_decode_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, *,
                           softmax_scale: Optional[float] = None, window: Optional[int] = None, k_scale: Optional[torch.Tensor] = None,
                           v_scale: Optional[torch.Tensor] = None, return_lse: bool = False, status: Optional[torch.Tensor] = None):
    """Attention of one new token per sequence over a paged cache that holds its key and value already.

    ``q`` [sequences, q heads, head_dim] in fp16 or bf16; query head ``h`` reads key/value head ``h // (q heads / kv heads)``.
    ``lengths`` (int32 [sequences]) counts the cached tokens, the new one included; with ``window`` only the last ``window`` of them are
    attended to.  ``softmax_scale`` defaults to ``head_dim ** -0.5``.  A sequence of length 0 gives zeros.  Returns
    [sequences, q heads, head_dim] in q's type, with ``return_lse`` a pair with the natural logarithm of the softmax's sum (fp32
    [sequences, q heads], -inf for length 0)."""
    what = "paged_decode_attention"
    dev = _same_device(what, q, k_pages, v_pages, block_table, lengths, k_scale, v_scale, status)
    shape, dtype = q.shape, q.dtype
    if len(shape) != 3 or dtype not in _ROWS:
        _fail(what, "q must be fp16 or bf16 [sequences, q heads, head_dim]")
    batch, heads, dim = shape
    q0, q1, q2 = q.stride()
    if q2 != 1 and dim > 1:
        _fail(what, "the dimensions of a head must be side by side")
    cache, sizes = _cache(what, k_pages, v_pages, block_table, k_scale, v_scale, status)
    if sizes[2] != dim or sizes[3] != batch:
        _fail(what, f"q {tuple(shape)} does not fit pages of head_dim {sizes[2]} and a block table of {sizes[3]} sequences")
    lengths_at = _want(what, "lengths", lengths, torch.int32, (batch,))
    window = max(-1, min(window or 0, 2 ** 31 - 1))  # as a 32-bit number; no cache is longer
    key = (dev.index, heads, window, sizes)
    like, ws_at, ws_bytes = _scratch.get(key, False), 0, 0
    known = like is not False
    if not known:
        with torch.cuda.device(dev):
            capturing = torch.cuda.is_current_stream_capturing()  # what is allocated now belongs to a graph
            need = int(_native.load().tris_paged_decode_attention_workspace_bytes(cache, heads, window))
        like = torch.empty((1,), dtype=torch.uint8, device=dev).expand(need) if need else None
    if like is not None:
        ws = _new_like(like)
        ws_at, ws_bytes = ws.data_ptr(), ws.numel()
    out, lse = _new_like(q), None
    if return_lse:
        lse = torch.empty((batch, heads), dtype=torch.float32, device=dev)
    args = _ATTENTION.pack(q.data_ptr(), q0, q1, lengths_at, out.data_ptr(), 0 if lse is None else lse.data_ptr(), ws_at, ws_bytes,
                           heads, window, _DTYPES[dtype], dim ** -0.5 if softmax_scale is None else softmax_scale)
    _launch(what, "tris_paged_decode_attention", dev, cache, args)
    if not known and not capturing:  # a call that was refused says nothing of what the next one needs
        if len(_scratch) >= 4096:  # block tables may grow for ever
            _scratch.clear()
        _scratch[key] = like
    return (out, lse) if return_lse else out


def _norm(what: str, x, residual, weight, eps: float, group_size: Optional[int]):
    dev = _same_device(what, x, residual, weight)
    shape, dtype = x.shape, x.dtype
    if not shape or dtype not in _ROWS:
        _fail(what, "x must be fp16 or bf16 [..., hidden]")
    hidden = shape[-1]
    weight_at = _want(what, "weight", weight, dtype, (hidden,))
    x2, h = x, None
    if len(shape) != 2 or x.stride(1) != 1:
        x2 = x.reshape(-1, hidden).contiguous()
    r_at = r_stride = h_at = scales_at = 0
    if residual is not None:
        if residual.shape != shape or residual.dtype is not dtype:
            _fail(what, "residual must have x's shape and type")
        r2, h = residual, _new_like(x)
        if len(shape) != 2 or residual.stride(1) != 1:
            r2 = residual.reshape(-1, hidden).contiguous()
        r_at, r_stride, h_at = r2.data_ptr(), r2.stride(0), h.data_ptr()
    group, scales = hidden, None
    if group_size is None:
        y = _new_like(x)
    else:
        group = group_size or hidden
        if hidden == 0 or group < 0 or hidden % group:
            _fail(what, f"groups of {group} columns do not divide rows of {hidden}")
        y = _new_like(x, torch.float8_e4m3fn)
        scales = torch.empty(shape[:-1] + (hidden // group,), dtype=torch.float32, device=dev)
        scales_at = scales.data_ptr()
    args = _NORM.pack(x2.data_ptr(), r_at, weight_at, h_at, y.data_ptr(), scales_at, x2.stride(0), r_stride, hidden, hidden, x2.shape[0],
                      hidden, group, _DTYPES[dtype], _DTYPES[y.dtype], eps)
    _launch(what, "tris_add_rms_norm", dev, args)
    return y, scales, h


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-5):
    """``h = residual + x`` and ``y = h / sqrt(mean(h ** 2) + eps) * weight`` over the last dimension, in fp32, rounded once each.
    Returns ``(y, h)`` in x's type; without a residual ``(y, None)``."""
    y, _, h = _norm("add_rms_norm", x, residual, weight, eps, None)
    return y, h


def add_rms_norm_e4m3(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-5, *, group_size: int = 0):
    """The same with y in 8 bits: returns ``(values, scales, h)`` with ``y = values * scales``, values in ``torch.float8_e4m3fn`` and a scale
    (fp32 [..., groups], the group's largest magnitude / 448) for each ``group_size`` columns, a multiple of 16 - or 0: for each row."""
    return _norm("add_rms_norm_e4m3", x, residual, weight, eps, group_size)


def apply_logit_controls(logits: torch.Tensor, *, tokens: Optional[torch.Tensor] = None, token_lengths: Optional[torch.Tensor] = None,
                         prompt_lengths: Optional[torch.Tensor] = None, repetition: Optional[torch.Tensor] = None,
                         presence: Optional[torch.Tensor] = None, frequency: Optional[torch.Tensor] = None,
                         bias_ids: Optional[torch.Tensor] = None, bias_values: Optional[torch.Tensor] = None,
                         allowed: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Logits [rows, vocab] (fp16, bf16 or fp32) as the choice of a token sees them, in fp32.  Each control is optional, in this order:

    * ``repetition`` [rows] > 0: logits of tokens in ``tokens[b, :token_lengths[b]]`` are divided by it where positive, else multiplied;
    * ``frequency``, ``presence`` [rows]: ``z -= frequency * n + presence * (n > 0)``, n counting the token in the history from
      ``prompt_lengths[b]`` on (None: in all of it);
    * ``bias_ids`` (int32), ``bias_values`` (fp32) [rows, n]: ``z += value``; negative ids are skipped, repeated ones add up;
    * ``allowed`` int32 [rows, ceil(vocab / 32)]: ``z = -inf`` where bit ``v % 32`` of word ``v // 32`` is 0, whatever the logit was.

    ``tokens`` is int32 [rows, any]; ids outside the vocabulary are skipped.  ``out`` may be fp32 logits themselves."""
    what = "apply_logit_controls"
    dev = _same_device(what, logits, tokens, token_lengths, prompt_lengths, repetition, presence, frequency, bias_ids, bias_values, allowed, out)
    shape, dtype = logits.shape, logits.dtype
    if len(shape) != 2 or dtype not in _LOGIT_TYPES or (logits.stride(1) != 1 and shape[1] > 1):
        _fail(what, "logits must be fp16, bf16 or fp32 [rows, vocab] with a row's logits side by side")
    rows, vocab = shape
    if out is None:
        out = _new_like(logits, torch.float32)
    elif out.dtype is not torch.float32 or out.shape != shape or (vocab > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < vocab):
        _fail(what, "out must be fp32 of the logits' shape with a row side by side, and the next one behind it")

    if tokens is None and (repetition is not None or presence is not None or frequency is not None):
        _fail(what, "penalties need tokens")
    if (tokens is None) != (token_lengths is None):
        _fail(what, "tokens and token_lengths go together")
    if (bias_ids is None) != (bias_values is None):
        _fail(what, "bias_ids and bias_values go together")
    tok = tok_stride = history = ids = values = bias_stride = biases = mask = mask_stride = 0
    if tokens is not None:
        tok, tok_stride, history = _matrix(what, "tokens", tokens, torch.int32, rows)
    if bias_ids is not None:
        ids, bias_stride, biases = _matrix(what, "bias_ids", bias_ids, torch.int32, rows)
        values, value_stride, _ = _matrix(what, "bias_values", bias_values, torch.float32, rows, biases)
        if biases and rows > 1 and bias_stride != value_stride:
            _fail(what, "bias_ids and bias_values must have the same stride")
    if allowed is not None:
        mask, mask_stride, _ = _matrix(what, "allowed", allowed, torch.int32, rows, (vocab + 31) // 32)
    each, f32, i32 = (rows,), torch.float32, torch.int32
    args = _LOGITS.pack(logits.data_ptr(), out.data_ptr(), tok,
                        0 if token_lengths is None else _want(what, "token_lengths", token_lengths, i32, each),
                        0 if prompt_lengths is None else _want(what, "prompt_lengths", prompt_lengths, i32, each),
                        0 if repetition is None else _want(what, "repetition", repetition, f32, each),
                        0 if presence is None else _want(what, "presence", presence, f32, each),
                        0 if frequency is None else _want(what, "frequency", frequency, f32, each),
                        ids, values, mask, logits.stride(0), out.stride(0), tok_stride, bias_stride, mask_stride,
                        rows, vocab, history, biases, _DTYPES[dtype], 0)
    _launch(what, "tris_logit_controls", dev, args)
    return out
