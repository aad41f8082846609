"""The operators of a decode step around the expert layers: new keys and values go into a paged cache
with the position rotation applied, one new token per sequence attends over that cache, the residual
is added and normalised, and the logits get their penalties, biases and grammar masks.

The reference leaves these to stock PyTorch (attention, norms and rotation of its model files,
modeling_olmoe.py:300-618, 1120-1200; greedy argmax in tools/benchmark_e2e_grid.py:325-420).  All of
them run on the current stream, allocate only what they return (and scratch), and never synchronise,
so they can be captured in a CUDA graph.  There is no CPU path: tensors must live on a CUDA device.

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
# the structs of include/trismoe_b200.h, field by field (packing bytes takes a third of the time of a ctypes structure)
_PAGED_KV = struct.Struct("@2Q6q3Qq8iQ")
_APPEND = struct.Struct("@3Q6q6Q8i")
_ATTENTION = struct.Struct("@Q2q4Qq3if")
_NORM = struct.Struct("@6Q4q5if")
_LOGITS = struct.Struct("@11Q5q6i")
_workspace_bytes: dict = {}


def _fail(what: str, why: str):
    raise RuntimeError(f"trismoe_b200 {what}: {why}")


def _same_device(what: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> torch.device:
    _native.require_cuda(first, what)
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            _fail(what, "all tensors must live on one CUDA device")
    return first.device


def _want(what: str, name: str, t: torch.Tensor, dtype, *shape) -> int:
    """Address of a contiguous tensor of that type and shape."""
    if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
        _fail(what, f"{name} must be contiguous {dtype} of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _cache(what: str, k_pages, v_pages, block_table, k_scale, v_scale, status) -> bytes:
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype or k_pages.dtype not in _DTYPES:
        _fail(what, "k_pages and v_pages must have the same type and shape [num_pages, page_size, num_kv_heads, head_dim]")
    pages, page_size, heads, dim = k_pages.shape
    ks, vs, e4m3 = k_pages.stride(), v_pages.stride(), k_pages.dtype == torch.float8_e4m3fn
    if ks[3] != 1 or vs[3] != 1:
        _fail(what, "the dimensions of a head must be side by side")
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        _fail(what, "block_table must be int32 [sequences, pages] with the pages of a sequence side by side")
    if (k_scale is not None or v_scale is not None) and not e4m3:
        _fail(what, "scales belong to e4m3 pages")
    return _PAGED_KV.pack(
        k_pages.data_ptr(), v_pages.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
        0 if k_scale is None else _want(what, "k_scale", k_scale, torch.float32, heads),
        0 if v_scale is None else _want(what, "v_scale", v_scale, torch.float32, heads),
        block_table.data_ptr(), block_table.stride(0), block_table.shape[0], block_table.shape[1], pages, page_size, heads, dim,
        _DTYPES[k_pages.dtype], 0, 0 if status is None else _want(what, "status", status, torch.int32, 1))


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
    fine.  Token ``t`` belongs to sequence ``sequences[t]`` (int32; default: ``t``) and stands at ``positions[t]`` (int32 or
    int64; negative: padding, not written).  ``cos`` and ``sin`` [positions, rotary_dim / 2] in fp32 rotate the first ``rotary_dim``
    dimensions, pairs ``(i, i + rotary_dim / 2)`` or, ``interleaved``, ``(2 i, 2 i + 1)``; None: no rotation.  e4m3 pages get
    ``x / scale``, saturated.  Tokens of one call must have different places.  Returns the rotated queries (None without ``q``),
    with ``return_key`` a pair with the rotated keys."""
    what = "append_paged_kv"
    dev = _same_device(what, k, v, q, k_pages, v_pages, block_table, positions, sequences, cos, sin, k_scale, v_scale, status)
    if k.dim() != 3 or v.shape != k.shape or k.dtype not in _ROWS or v.dtype != k.dtype or (k_pages.dim() == 4 and k.shape[1:] != k_pages.shape[2:]):
        _fail(what, "k and v must be fp16 or bf16 [tokens, num_kv_heads, head_dim] of the cache")
    tokens, kv_heads, dim = k.shape
    if q is not None and (q.dim() != 3 or q.dtype != k.dtype or q.shape[0] != tokens or q.shape[2] != dim):
        _fail(what, "q must be [tokens, q heads, head_dim] in the keys' type")
    if positions.dtype not in (torch.int32, torch.int64):
        _fail(what, "positions must be int32 or int64")
    _want(what, "positions", positions, positions.dtype, tokens)
    if sequences is not None:
        _want(what, "sequences", sequences, torch.int32, tokens)
    rotary, rows = 0, 0
    if (cos is None) != (sin is None):
        _fail(what, "cos and sin go together")
    if cos is not None:
        if cos.dim() != 2:
            _fail(what, "cos and sin must be [positions, rotary_dim / 2]")
        rows, rotary = cos.shape[0], 2 * cos.shape[1]
        _want(what, "cos", cos, torch.float32, rows, rotary // 2)
        _want(what, "sin", sin, torch.float32, rows, rotary // 2)
    ks, vs, qs = k.stride(), v.stride(), (0, 0, 1) if q is None else q.stride()
    if tokens and (ks[2] != 1 or vs[2] != 1 or qs[2] != 1):
        _fail(what, "the dimensions of a head must be side by side")
    cache = _cache(what, k_pages, v_pages, block_table, k_scale, v_scale, status)
    q_out = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=dev)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=dev) if return_key else None
    args = _APPEND.pack(
        0 if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1],
        0 if cos is None else cos.data_ptr(), 0 if cos is None else sin.data_ptr(), positions.data_ptr(),
        0 if sequences is None else sequences.data_ptr(), 0 if q is None else q_out.data_ptr(), 0 if k_out is None else k_out.data_ptr(),
        tokens, 0 if q is None else q.shape[1], rotary, rows, positions.dtype == torch.int64, bool(interleaved), _DTYPES[k.dtype], 0)
    lib = _native.load()
    with _native.on_device(dev):
        _native.check(lib.tris_paged_kv_append(cache, args, _native.stream_of(dev)), what)
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
    if q.dim() != 3 or q.dtype not in _ROWS or q.stride(2) != 1:
        _fail(what, "q must be fp16 or bf16 [sequences, q heads, head_dim] with the dimensions of a head side by side")
    batch, heads, dim = q.shape
    cache = _cache(what, k_pages, v_pages, block_table, k_scale, v_scale, status)
    if k_pages.shape[3] != dim or block_table.shape[0] != batch:
        _fail(what, f"q {tuple(q.shape)} does not fit pages of head_dim {k_pages.shape[3]} and a block table of {block_table.shape[0]} sequences")
    lengths_ptr = _want(what, "lengths", lengths, torch.int32, batch)
    lib = _native.load()
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty((batch, heads), dtype=torch.float32, device=dev) if return_lse else None
    with _native.on_device(dev):
        key = (dev.index, heads, k_pages.shape[2], dim)
        need = _workspace_bytes.get(key)
        if need is None:
            need = int(lib.tris_paged_decode_attention_workspace_bytes(cache, heads))
            if need:
                _workspace_bytes[key] = need
        ws = torch.empty((need,), dtype=torch.uint8, device=dev)
        args = _ATTENTION.pack(q.data_ptr(), q.stride(0), q.stride(1), lengths_ptr, out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                               ws.data_ptr(), need, heads, int(window or 0), _DTYPES[q.dtype],
                               dim ** -0.5 if softmax_scale is None else float(softmax_scale))
        _native.check(lib.tris_paged_decode_attention(cache, args, _native.stream_of(dev)), what)
    return (out, lse) if return_lse else out


def _norm(what: str, x, residual, weight, eps: float, group_size: Optional[int]):
    dev = _same_device(what, x, residual, weight)
    if x.dim() < 1 or x.dtype not in _ROWS:
        _fail(what, "x must be fp16 or bf16 [..., hidden]")
    hidden = x.shape[-1]
    _want(what, "weight", weight, x.dtype, hidden)
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        _fail(what, "residual must have x's shape and type")
    x2 = x if x.dim() == 2 and x.stride(1) == 1 else x.reshape(-1, hidden).contiguous()
    r2 = residual
    if residual is not None and not (residual.dim() == 2 and residual.stride(1) == 1):
        r2 = residual.reshape(-1, hidden).contiguous()
    rows = x2.shape[0]
    h = torch.empty(x.shape, dtype=x.dtype, device=dev) if residual is not None else None
    if group_size is None:
        y, scales, group = torch.empty(x.shape, dtype=x.dtype, device=dev), None, hidden
    else:
        group = int(group_size) or hidden
        if hidden == 0 or group < 0 or hidden % group:
            _fail(what, f"groups of {group} columns do not divide rows of {hidden}")
        y = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=dev)
        scales = torch.empty(x.shape[:-1] + (hidden // group,), dtype=torch.float32, device=dev)
    args = _NORM.pack(x2.data_ptr(), 0 if r2 is None else r2.data_ptr(), weight.data_ptr(), 0 if h is None else h.data_ptr(), y.data_ptr(),
                      0 if scales is None else scales.data_ptr(), x2.stride(0), 0 if r2 is None else r2.stride(0), hidden, hidden, rows, hidden,
                      group, _DTYPES[x.dtype], _DTYPES[y.dtype], eps)
    lib = _native.load()
    with _native.on_device(dev):
        _native.check(lib.tris_add_rms_norm(args, _native.stream_of(dev)), what)
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
    if logits.dim() != 2 or logits.dtype not in _DTYPES or logits.dtype == torch.float8_e4m3fn or (logits.shape[1] > 1 and logits.stride(1) != 1):
        _fail(what, "logits must be fp16, bf16 or fp32 [rows, vocab] with a row's logits side by side")
    rows, vocab = logits.shape
    if out is None:
        out = torch.empty((rows, vocab), dtype=torch.float32, device=dev)
    elif out.dtype != torch.float32 or out.shape != logits.shape or (vocab > 1 and out.stride(1) != 1):
        _fail(what, "out must be fp32 of the logits' shape with a row side by side")

    def matrix(name, t, dtype, columns=None):
        if t is None:
            return 0, 0, 0
        if t.dim() != 2 or t.dtype != dtype or t.shape[0] != rows or (columns is not None and t.shape[1] != columns) or (t.shape[1] > 1 and t.stride(1) != 1):
            _fail(what, f"{name} must be {dtype} [rows, {'any' if columns is None else columns}] with a row side by side, got {t.dtype} {tuple(t.shape)}")
        return t.data_ptr(), t.stride(0), t.shape[1]

    def column(name, t, dtype=torch.float32):
        return 0 if t is None else _want(what, name, t, dtype, rows)

    if tokens is None and (repetition is not None or presence is not None or frequency is not None):
        _fail(what, "penalties need tokens")
    if (tokens is None) != (token_lengths is None):
        _fail(what, "tokens and token_lengths go together")
    if (bias_ids is None) != (bias_values is None):
        _fail(what, "bias_ids and bias_values go together")
    tok, tok_stride, history = matrix("tokens", tokens, torch.int32)
    ids, id_stride, biases = matrix("bias_ids", bias_ids, torch.int32)
    values, value_stride, _ = matrix("bias_values", bias_values, torch.float32, biases)
    if ids and biases and id_stride != value_stride:
        _fail(what, "bias_ids and bias_values must have the same stride")
    mask, mask_stride, _ = matrix("allowed", allowed, torch.int32, (vocab + 31) // 32)
    args = _LOGITS.pack(logits.data_ptr(), out.data_ptr(), tok, column("token_lengths", token_lengths, torch.int32),
                        column("prompt_lengths", prompt_lengths, torch.int32), column("repetition", repetition), column("presence", presence),
                        column("frequency", frequency), ids, values, mask, logits.stride(0), out.stride(0), tok_stride, id_stride, mask_stride,
                        rows, vocab, history, biases, _DTYPES[logits.dtype], 0)
    lib = _native.load()
    with _native.on_device(dev):
        _native.check(lib.tris_logit_controls(args, _native.stream_of(dev)), what)
    return out
