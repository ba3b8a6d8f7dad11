"""Serving operators around a 4-bit paged key/value cache, on torch tensors.

What a prompt and the decode tokens of a batch of sequences need besides the
projections (the C ABI's serving operators, include/frcuda.h; no reference
counterpart: the reference forwarder keeps one sequence's fp32 cache in NumPy,
flatrun/model/qwen2.py:1527-1614):

  qk_norm_rope          bias, norms of query and key heads, position rotation
  rope_tables_scaled    the rotation's tables, also for long contexts
  kv_cache_q4           an empty 4-bit paged cache
  kv_append_q4          keys and values of tokens into it
  kv_read_q4            and back
  attention_decode_q4   one query token a sequence over its cached tokens
  attention_prefill     causal attention of whole packed prompts

A step of a batch: ``qk_norm_rope``, then ``kv_append_q4`` of the new tokens,
then ``attention_decode_q4`` with lengths that count them; a prompt attends
through ``attention_prefill`` and is appended for the tokens that follow.

Every call is enqueued on the current stream of its tensors' device and
returns without waiting; positions, slots, tables and lengths are read on the
device, so calls can be captured in a CUDA graph and replayed with new ones
(pass ``out=`` to keep the results in place).  Arguments that do not fit raise
ValueError before anything is launched.  Inference only: tensors that require
gradients, outputs among them, are refused while gradients are recorded, and so are
tensors with forward-mode tangents.
"""

from __future__ import annotations

import ctypes
import math
import struct

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib

_TYPE = {torch.float32: _lib.FRC_F32, torch.float16: _lib.FRC_F16, torch.bfloat16: _lib.FRC_BF16}
_BLOCK = 16  # tokens of a cache block


# The records of frc_serving_call (include/frcuda.h): one ctypes argument in
# place of two dozen, which cost a quarter of a microsecond each.
_ROPE = (0, struct.Struct("qqQqqqqqQQQdQQqqqQQqQqQq"))
_APPEND = (1, struct.Struct("qQqqQqqqQqqqqQ"))
_READ = (2, struct.Struct("qQQqqqqqQqqQqq"))
_DECODE = (3, struct.Struct("qQqqQqqQqqQqqqqdQqQqq"))
_PREFILL = (4, struct.Struct("qQqqQqqQqqQQqqqqqqdqQqq"))

# The current device, and the raw handle of a device's current stream: as
# torch.cuda.current_device() and torch.cuda.current_stream(i).cuda_stream,
# without a Python object each.
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda i: torch.cuda.current_stream(i).cuda_stream)


def _need(cond: bool, what: str) -> None:
    if not cond:
        raise ValueError(what)


def _launch(device: int, op, *args) -> None:
    """The operator with `device` current, on its current stream."""
    lib = _lib._lib or _lib.load()
    number, record = op
    if device == _current_device():
        rc = lib.frc_serving_call(number, record.pack(*args), record.size, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = lib.frc_serving_call(number, record.pack(*args), record.size, _raw_stream(device))
    if rc == _lib.FRC_ERR_INVALID:
        raise ValueError(_lib.last_error(lib))
    if rc:
        _lib.check(rc)


def _device(first, *others) -> int:
    """The CUDA device that all tensors are on."""
    i = first.get_device()
    for t in others:
        if t.get_device() != i:
            raise ValueError(f"tensors on different devices: {first.device} and {t.device}")
    if i < 0 or not first.is_cuda:
        raise ValueError(f"tensors must be on a CUDA device, not {first.device}")
    return i


def _no_grad(*tensors) -> None:
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("the operator has no backward pass: call it under torch.no_grad()")
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError("the operator has no forward-mode derivative: its results would have no tangents")


def _index(t: torch.Tensor, name: str, dtype: torch.dtype, shape) -> None:
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}")


def _rows(t: torch.Tensor, name: str, shape, dtype: torch.dtype):
    """Strides of the rows and heads of a (rows, heads, head_dim) tensor with contiguous channels."""
    if t.shape != shape or t.dtype != dtype:
        raise ValueError(f"{name} must be a {dtype} tensor of shape {tuple(shape)}, not {t.dtype} {tuple(t.shape)}")
    rows, heads, channels = t.stride()
    if channels != 1 and shape[2] > 1 and t.numel():
        raise ValueError(f"the channels of {name} must be contiguous")
    return rows, heads


# ---- position rotation ----------------------------------------------------------------
def rope_tables_scaled(rot: int, theta: float, max_pos: int, scaling: dict | None = None):
    """cos and sin tables [max_pos][rot / 2] in fp32 of the rotation by
    position * theta^(-2 i / rot), with the angles in 64 bits, so that far
    positions keep their phase.  `scaling` stretches them for long contexts:

    * ``{"type": "linear", "factor": s}``: positions / s;
    * ``{"type": "ntk", "factor": s}``: theta * s^(rot / (rot - 2)), which
      stretches the slowest pair by s and leaves the fastest;
    * ``{"type": "yarn", "factor": s, "original_max_position": n}``
      (``beta_fast`` 32, ``beta_slow`` 1, ``attention_factor`` 0.1 ln s + 1):
      pairs that turn more than beta_fast times in n positions stay, those below
      beta_slow turns are divided by s, a linear ramp between; cos and sin
      times the attention factor (Peng et al. 2023, arXiv 2309.00071);
    * ``{"type": "llama3", "factor": s, "original_max_position": n}``
      (``low_freq_factor`` 1, ``high_freq_factor`` 4): the same with the ramp
      linear in the number of turns.
    """
    _need(rot > 0 and rot % 2 == 0 and max_pos > 0 and theta > 0, "rot must be even and max_pos and theta positive")
    inv = float(theta) ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    magnitude = 1.0
    if scaling is not None:
        kind, s = scaling.get("type"), float(scaling.get("factor", 0.0))
        _need(kind in ("linear", "ntk", "yarn", "llama3"), f"unknown rope scaling {kind!r}")
        _need(s >= 1.0, "rope scaling needs a factor of at least 1")
        if kind == "linear":
            inv = inv / s
        elif kind == "ntk":
            _need(rot > 2, "ntk scaling needs more than one pair")
            inv = (theta * s ** (rot / (rot - 2))) ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
        else:
            n = float(scaling.get("original_max_position", 0))
            _need(n > 0, f"{kind} scaling needs original_max_position")
            turns = n * inv / (2 * math.pi)
            if kind == "yarn":
                fast, slow = float(scaling.get("beta_fast", 32)), float(scaling.get("beta_slow", 1))
                _need(fast > slow > 0, "yarn scaling needs beta_fast > beta_slow > 0")
                _need(theta > 1, "yarn scaling needs theta above 1")

                def pair(r):  # the (fractional) pair that turns r times in n positions
                    return rot * math.log(n / (r * 2 * math.pi)) / (2 * math.log(theta))

                low = max(math.floor(pair(fast)), 0)
                high = min(math.ceil(pair(slow)), rot - 1)
                ramp = np.clip((np.arange(rot // 2) - low) / max(high - low, 1e-3), 0.0, 1.0)
                inv = inv * (1 - ramp) + inv / s * ramp
                magnitude = float(scaling.get("attention_factor", 0.1 * math.log(s) + 1.0))
            else:
                lo, hi = float(scaling.get("low_freq_factor", 1)), float(scaling.get("high_freq_factor", 4))
                _need(hi > lo > 0, "llama3 scaling needs high_freq_factor > low_freq_factor > 0")
                keep = np.clip((turns - lo) / (hi - lo), 0.0, 1.0)
                inv = inv * keep + inv / s * (1 - keep)
    angle = np.arange(max_pos, dtype=np.float64)[:, None] * inv
    return (np.cos(angle) * magnitude).astype(np.float32), (np.sin(angle) * magnitude).astype(np.float32)


def qk_norm_rope(qkv, heads: int, kv_heads: int, cos, sin, positions, *, bias=None, q_norm=None, k_norm=None,
                 eps: float = 1e-6, interleaved: bool = False, out_dtype=None, out=None):
    """Queries, keys and values of tokens, ready for attention, in one pass.

    `qkv` (tokens, (heads + 2 kv_heads) * head_dim): rows [q | k | v], which
    get `bias`, norms of each query and key head (weights `q_norm`, `k_norm` of
    head_dim, RMS with `eps`) and the rotation at `positions` (int32) by
    `cos` and `sin` (max_pos, rot / 2), fp32; rot may be less than head_dim.
    Pairs are (i, i + rot / 2), or (2 i, 2 i + 1) if `interleaved`.  Rows whose
    position is outside the tables are padding: their outputs are left as they
    are (zeros where this call makes the outputs).

    Returns q (tokens, heads, head_dim), k and v (tokens, kv_heads, head_dim)
    in `out_dtype` (default: qkv's); `out` = (q, k, v) to write to: the three
    parts of qkv itself, or tensors that share no memory with it or each
    other.
    """
    in_type = _TYPE.get(qkv.dtype)
    if qkv.dim() != 2 or in_type is None:
        raise ValueError("qkv must be a 2-D fp32, fp16 or bf16 tensor")
    if heads <= 0 or kv_heads <= 0:
        raise ValueError("heads and kv_heads must be positive")
    tokens, n = qkv.shape
    row, column = qkv.stride()
    hd, rest = divmod(n, heads + 2 * kv_heads)
    if rest:
        raise ValueError(f"rows of {n} do not hold {heads} + 2 * {kv_heads} heads")
    if hd <= 0 or hd % 2 or hd > 256:
        raise ValueError(f"head_dim must be even and at most 256, not {hd}")
    if column != 1:
        raise ValueError("the rows of qkv must be contiguous")
    if (cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32 or
            not cos.is_contiguous() or not sin.is_contiguous() or cos.shape[0] == 0):
        raise ValueError("cos and sin must be contiguous fp32 tensors of one shape (max_pos, rot / 2)")
    max_pos, pairs = cos.shape
    if 2 * pairs > hd:
        raise ValueError(f"the tables rotate {2 * pairs} of {hd} channels")
    _index(positions, "positions", torch.int32, (tokens,))
    _no_grad(qkv, cos, sin)
    p_bias = p_q = p_k = 0
    if bias is not None:
        p_bias = _weight(bias, "bias", n, qkv)
    if q_norm is not None:
        p_q = _weight(q_norm, "q_norm", hd, qkv)
    if k_norm is not None:
        p_k = _weight(k_norm, "k_norm", hd, qkv)
    if out is None:
        dtype = out_dtype or qkv.dtype
        if dtype not in _TYPE:
            raise ValueError(f"out_dtype must be fp32, fp16 or bf16, not {dtype}")
        out = tuple(torch.zeros((tokens, h, hd), dtype=dtype, device=qkv.device) for h in (heads, kv_heads, kv_heads))
    elif len(out) != 3:
        raise ValueError("out must be (q, k, v)")
    q, k, v = out
    dtype = q.dtype
    if dtype not in _TYPE or (out_dtype is not None and out_dtype != dtype):
        raise ValueError("out has another type than out_dtype, or not fp32, fp16 or bf16")
    shape = (tokens, kv_heads, hd)
    _no_grad(q, k, v)
    q_row = _packed(q, "out q", (tokens, heads, hd), dtype)
    k_row = _packed(k, "out k", shape, dtype)
    v_row = _packed(v, "out v", shape, dtype)
    _launch(_device(qkv, cos, sin, positions, q, k, v), _ROPE, in_type, _TYPE[dtype], qkv.data_ptr(),
            row if tokens > 1 else n, tokens, heads, kv_heads, hd, p_bias, p_q, p_k, eps, cos.data_ptr(), sin.data_ptr(),
            max_pos, 2 * pairs, 1 if interleaved else 0, positions.data_ptr(), q.data_ptr(), q_row, k.data_ptr(), k_row,
            v.data_ptr(), v_row)
    return out


def _weight(t, name: str, size: int, beside) -> int:
    _index(t, name, torch.float32, (size,))
    _no_grad(t)
    if t.get_device() != beside.get_device():
        raise ValueError(f"tensors on different devices: {beside.device} and {t.device}")
    return t.data_ptr()


def _packed(t, name: str, shape, dtype) -> int:
    """Row stride of a (rows, heads, head_dim) output with contiguous heads."""
    row, head = _rows(t, name, shape, dtype)
    rows, heads, hd = shape
    if rows == 0:
        return heads * hd
    if head != hd and heads > 1:
        raise ValueError(f"the heads of {name} must be contiguous")
    if rows == 1:
        return heads * hd
    if row < heads * hd:
        raise ValueError(f"the rows of {name} overlap")
    return row


# ---- the cache ------------------------------------------------------------------------
def kv_cache_q4(pages: int, page_size: int, kv_heads: int, head_dim: int, device="cuda") -> torch.Tensor:
    """A 4-bit cache of `pages` pages of `page_size` tokens (a multiple of 16):
    a uint8 tensor (pages, kv_heads, page_size / 16, 20 * head_dim), zeroed
    (zeros stand for zeros).  head_dim is 64 or 128."""
    _need(pages > 0 and kv_heads > 0, "pages and kv_heads must be positive")
    _need(page_size > 0 and page_size % _BLOCK == 0, f"page_size must be a multiple of {_BLOCK}, not {page_size}")
    _need(head_dim in (64, 128), f"head_dim must be 64 or 128, not {head_dim}")
    return torch.zeros((pages, kv_heads, page_size // _BLOCK, 20 * head_dim), dtype=torch.uint8, device=device)


def _cache(cache) -> tuple[int, int, int, int]:
    shape = cache.shape
    if len(shape) == 4 and cache.dtype == torch.uint8 and cache.is_contiguous():
        pages, kv_heads, blocks, nbytes = shape
        if pages and kv_heads and blocks and (nbytes == 20 * 128 or nbytes == 20 * 64):
            return pages, kv_heads, blocks * _BLOCK, nbytes // 20
    raise ValueError("the cache must be a contiguous uint8 tensor (pages, kv_heads, page_size / 16, 20 * head_dim), "
                     "head_dim 64 or 128")


def kv_append_q4(cache, k, v, slots) -> None:
    """Quantise keys and values (tokens, kv_heads, head_dim) into `slots`
    (int64, page * page_size + offset) of the cache.  Slots outside the cache
    are skipped (use -1 for padding rows); the others of one call must differ."""
    pages, nkv, page, hd = _cache(cache)
    dtype = _TYPE.get(k.dtype)
    if dtype is None:
        raise ValueError(f"keys must be fp32, fp16 or bf16, not {k.dtype}")
    tokens = k.shape[0] if k.dim() else 0
    shape = (tokens, nkv, hd)
    k_row, k_head = _rows(k, "k", shape, k.dtype)
    v_row, v_head = _rows(v, "v", shape, k.dtype)
    _index(slots, "slots", torch.int64, (tokens,))
    _no_grad(k, v)
    _launch(_device(cache, k, v, slots), _APPEND, dtype, k.data_ptr(), k_row, k_head, v.data_ptr(), v_row, v_head,
            tokens, slots.data_ptr(), nkv, hd, pages, page, cache.data_ptr())


def kv_read_q4(cache, slots, *, dtype=None, out=None):
    """Keys and values (tokens, kv_heads, head_dim) that the cache holds in
    `slots`, in `dtype` (default fp32) or into `out` = (k, v).  Rows whose slot
    is outside the cache are left as they are (zeros where this call makes
    the outputs)."""
    pages, nkv, page, hd = _cache(cache)
    if slots.dim() != 1:
        raise ValueError("slots must have one dimension")
    tokens = slots.shape[0]
    _index(slots, "slots", torch.int64, (tokens,))
    shape = (tokens, nkv, hd)
    if out is None:
        dtype = dtype or torch.float32
        if dtype not in _TYPE:
            raise ValueError(f"dtype must be fp32, fp16 or bf16, not {dtype}")
        out = tuple(torch.zeros(shape, dtype=dtype, device=cache.device) for _ in range(2))
    if len(out) != 2 or out[0].dtype not in _TYPE or dtype not in (None, out[0].dtype):
        raise ValueError("out must be (k, v) in fp32, fp16 or bf16, of the type asked for")
    k, v = out
    _no_grad(k, v)
    k_row, k_head = _rows(k, "out k", shape, k.dtype)
    v_row, v_head = _rows(v, "out v", shape, k.dtype)
    if tokens and (min(k_row, v_row) <= 0 < tokens - 1 or min(k_head, v_head) <= 0 < nkv - 1):
        raise ValueError("the rows or heads of out overlap")
    _launch(_device(cache, slots, k, v), _READ, _TYPE[k.dtype], cache.data_ptr(), slots.data_ptr(), tokens, nkv, hd,
            pages, page, k.data_ptr(), k_row, k_head, v.data_ptr(), v_row, v_head)
    return out


# ---- attention ----------------------------------------------------------------------------
_workspace_bytes: dict = {}  # by head_dim


def _decode_q4_workspace(batch: int, nh: int, nkv: int, hd: int) -> int:
    if hd not in _workspace_bytes:
        ws = ctypes.c_size_t()
        _lib.check(_lib.load().frc_attention_decode_q4_workspace(batch, nh, nkv, hd, ctypes.byref(ws)))
        _workspace_bytes[hd] = int(ws.value)
    return _workspace_bytes[hd]


def _decode_q4_kernels(batch: int, nh: int, nkv: int, room: int) -> int:
    """Kernels that attention_decode_q4 launches for tables of `room` tokens: the second joins what several CTAs have
    of a head, and a CTA takes eight places (of 32 tokens, and one more a sequence, KV head and eight query heads)."""
    units = batch * nkv * -(-nh // nkv // 8)
    return 1 if batch == 0 or units * (-(-room // 32) + 1) <= 8 else 2


def attention_decode_q4(q, cache, block_table, lengths, *, scale: float | None = None, out=None):
    """Attention of one query token a sequence over the 4-bit cache.

    `q` (batch, heads, head_dim), fp32, fp16 or bf16, heads a multiple of the
    cache's; sequence b's tokens 0 .. lengths[b] - 1 lie in pages
    block_table[b] (int32, (batch, max_pages)), the t-th in entry
    t // page_size.  `scale` defaults to head_dim^-1/2.  Page numbers outside
    the cache hide their tokens, lengths are held to what the table covers, and
    a sequence without tokens gives zeros.  Returns (batch, heads, head_dim) in
    q's type, into `out` where given (q itself, or apart from it).
    """
    pages, nkv, page, hd = _cache(cache)
    dtype = _TYPE.get(q.dtype)
    if q.dim() != 3 or dtype is None:
        raise ValueError("q must be (batch, heads, head_dim) in fp32, fp16 or bf16")
    batch, nh, _ = q.shape
    shape = (batch, nh, hd)
    q_seq, q_head = _rows(q, "q", shape, q.dtype)
    if nh == 0 or nh % nkv:
        raise ValueError(f"{nh} query heads are not a multiple of the cache's {nkv}")
    if block_table.dim() != 2:
        raise ValueError("block_table must be (batch, max_pages)")
    max_pages = block_table.shape[1]
    _index(block_table, "block_table", torch.int32, (batch, max_pages))
    _index(lengths, "lengths", torch.int32, (batch,))
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=q.device)
    o_seq, o_head = _rows(out, "out", shape, q.dtype)
    if batch and (o_seq <= 0 < batch - 1 or o_head <= 0 < nh - 1):
        raise ValueError("the rows or heads of out overlap")
    _no_grad(q, out)
    device = _device(q, cache, block_table, lengths, out)
    nbytes = _decode_q4_workspace(batch, nh, nkv, hd)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    _launch(device, _DECODE, dtype, q.data_ptr(), q_seq, q_head, cache.data_ptr(), pages,
            page, block_table.data_ptr(), max_pages, max_pages, lengths.data_ptr(), batch, nh, nkv, hd,
            hd ** -0.5 if scale is None else scale, ws.data_ptr(), nbytes, out.data_ptr(), o_seq, o_head)
    return out


def attention_prefill(q, k, v, cu_q, cu_k=None, *, causal: bool = True, scale: float | None = None, out=None):
    """Attention of whole prompts, packed one after the other.

    `q` (tokens, heads, head_dim), `k` and `v` (key tokens, kv_heads,
    head_dim), fp16 or bf16, head_dim 64 or 128, heads a multiple of kv_heads;
    sequence b is rows cu_q[b] .. cu_q[b + 1] of q and cu_k[b] .. cu_k[b + 1] of
    k and v (int32, batch + 1 ends that do not fall; `cu_k` defaults to `cu_q`).
    Causal: the last query of a sequence sees all its keys, each earlier one a
    key less, so a prompt may go on behind tokens that came before.  A query that
    sees no key gives zeros; rows of no sequence are left as they are (zeros
    where this call makes the output).  `scale` defaults to head_dim^-1/2.  `out`
    shares no memory with q, k and v.
    """
    if q.dim() != 3 or q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("q must be (tokens, heads, head_dim), fp16 or bf16")
    if k.dim() != 3:
        raise ValueError("k must be (tokens, kv_heads, head_dim)")
    tokens, nh, hd = q.shape
    tokens_k, nkv, _ = k.shape
    if hd not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, not {hd}")
    dtype, shape, shape_k = q.dtype, (tokens, nh, hd), (tokens_k, nkv, hd)
    strides = [_rows(q, "q", shape, dtype), _rows(k, "k", shape_k, dtype), _rows(v, "v", shape_k, dtype)]
    if nkv == 0 or nh == 0 or nh % nkv:
        raise ValueError(f"{nh} query heads are not a multiple of {nkv} key heads")
    if cu_k is None:
        cu_k = cu_q
    if cu_q.dim() != 1 or cu_q.shape[0] < 1:
        raise ValueError("cu_q must hold batch + 1 ends")
    _index(cu_q, "cu_q", torch.int32, cu_q.shape)
    _index(cu_k, "cu_k", torch.int32, cu_q.shape)
    if out is None:
        out = torch.zeros(shape, dtype=dtype, device=q.device)
    strides.append(_rows(out, "out", shape, dtype))
    at = [q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()]
    (q_row, q_head), (k_row, k_head), (v_row, v_head), (o_row, o_head) = strides
    if (at[0] | at[1] | at[2] | at[3]) & 15 or (q_row | q_head | k_row | k_head | v_row | v_head | o_row | o_head) & 7:
        for t, (row, head), p, name in zip((q, k, v, out), strides, at, ("q", "k", "v", "out")):
            if (p % 16 or row % 8 or head % 8) and t.numel():
                raise ValueError(f"{name} must be 16-byte aligned, with row and head strides that are multiples of 8")
    if tokens and (o_row <= 0 < tokens - 1 or o_head <= 0 < nh - 1):
        raise ValueError("the rows or heads of out overlap")
    if at[3] in at[:3] and tokens:
        raise ValueError("out must not be q, k or v: they are read while its rows are written")
    _no_grad(q, k, v, out)
    _launch(_device(q, k, v, cu_q, cu_k, out), _PREFILL, _TYPE[dtype], at[0], q_row, q_head, at[1], k_row, k_head,
            at[2], v_row, v_head, cu_q.data_ptr(), cu_k.data_ptr(), cu_q.shape[0] - 1, tokens, tokens_k, nh, nkv, hd,
            hd ** -0.5 if scale is None else scale, 1 if causal else 0, at[3], o_row, o_head)
    return out


__all__ = ["qk_norm_rope", "rope_tables_scaled", "kv_cache_q4", "kv_append_q4", "kv_read_q4", "attention_decode_q4",
           "attention_prefill"]
