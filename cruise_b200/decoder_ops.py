"""The decoder operators on CUDA tensors (over the C ABI of include/cruise_decoder.h).

The pieces of one decode step around the paged cache, for any number of rows
and any context length: :func:`rotate_store` (head norms, rotation, paged
store), :func:`paged_attention` (one new token per row) and :func:`choose`
(logit rules and the greedy choice).  ``EpochEngine.decoder_step`` is the whole
step for the engine's four rows.

Calls run on the current stream of their tensors' device, queue their kernels
and return without waiting; they may be captured into a CUDA graph.  They keep
no state between calls.  They are inference operators: a tensor that requires
a gradient is refused while gradients are recorded.  Arguments that do not fit
raise ``ValueError``, failures of the library :class:`DecoderOpError`.  There is
no fallback without the built library.
"""

from __future__ import annotations

import functools
import math

import torch

from . import _lib

_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_HALF = (torch.bfloat16, torch.float16)
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


class DecoderOpError(RuntimeError):
    """A decoder operator's status other than invalid arguments (a CUDA error code)."""

    def __init__(self, code: int, message: str) -> None:
        super().__init__(f"decoder operator failed ({code}): {message}")
        self.code = code


def _done(rc: int) -> None:
    if rc != 0:
        message = _lib.load().cruise_decoder_last_error().decode()
        if rc == -1:
            raise ValueError(message)
        raise DecoderOpError(rc, message)


def _need(condition: bool, message: str) -> None:
    if not condition:
        raise ValueError(message)


def _same_device(device: torch.device, **tensors) -> None:
    for name, tensor in tensors.items():
        if tensor is None:
            continue
        if not isinstance(tensor, torch.Tensor) or tensor.device != device:
            raise ValueError(f"{name} must be a tensor on {device}")
        if tensor.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient: the decoder operators are for inference")


def _cuda_device(tensor, name: str) -> torch.device:
    if not isinstance(tensor, torch.Tensor) or not tensor.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return tensor.device


def _vector(tensor, name: str, dtype: torch.dtype, count: int) -> None:
    if tensor.dtype != dtype or tensor.dim() != 1 or tensor.shape[0] != count or (count > 1 and tensor.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous {dtype} vector of {count}")


def _row_stride(tensor, width: int) -> int:
    """Elements between rows; a single row's stride is its width (torch leaves any value there)."""
    return tensor.stride(0) if tensor.shape[0] > 1 else max(width, 1)


def _heads(tensor, name: str, rows: int, heads: int, d: int, dtype: torch.dtype) -> int:
    """Row stride of [rows, heads, d] with adjacent heads."""
    if tensor.dtype != dtype or tuple(tensor.shape) != (rows, heads, d):
        raise ValueError(f"{name} must be {dtype} [{rows}, {heads}, {d}]")
    if rows and (tensor.stride(2) != 1 or (heads > 1 and tensor.stride(1) != d)):
        raise ValueError(f"{name}: the heads of a row must lie next to one another")
    return _row_stride(tensor, heads * d)


def _caches(key, value, d: int | None = None):
    """Block stride of two paged caches [blocks, block_size, kv heads, d]."""
    _need(key.dim() == 4 and value.shape == key.shape and value.dtype == key.dtype and key.dtype in _HALF,
          "key_cache and value_cache must be bf16 or fp16 [blocks, block_size, kv_heads, head_dim] of one shape")
    blocks, block, nkv, width = key.shape
    _need(min(key.shape) > 0, "the caches must not be empty")
    inner = (nkv * width, width, 1)
    for name, cache in (("key_cache", key), ("value_cache", value)):
        for axis in (1, 2, 3):
            if key.shape[axis] > 1 and cache.stride(axis) != inner[axis - 1]:
                raise ValueError(f"{name}: the slots of a block must be contiguous")
    if blocks > 1:
        _need(key.stride(0) == value.stride(0), "key_cache and value_cache must have one block stride")
    return key.stride(0) if blocks > 1 else block * nkv * width


def _index(device: torch.device) -> int:
    return device.index if device.index is not None else torch.cuda.current_device()


def rotate_store(qkv: torch.Tensor, position: torch.Tensor, slot: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                 key_cache: torch.Tensor, value_cache: torch.Tensor, *, num_heads: int,
                 q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Norms of queries and keys per head (with ``q_norm`` and ``k_norm``), the
    position rotation and the write into the paged cache, in one pass.

    ``qkv`` [tokens, (num_heads + 2 kv_heads) d] bf16 or fp16 holds query, key
    and value heads; ``cos`` and ``sin`` [rows, rotary] (bf16 or fp32, both halves
    written out as in :func:`cruise_b200.engine.rope_tables`) the rotation by
    ``position`` int64 [tokens]; ``slot`` int32 [tokens] the cache slot of each
    token (block * block_size + offset; outside the cache: not stored, and two
    tokens must not share one).  The caches [blocks, block_size, kv_heads, d] are
    updated in place.  A token whose position lies outside the tables is not
    stored and gets zeros.  Returns the rotated queries [tokens, num_heads, d]
    (``out``)."""
    device = _cuda_device(qkv, "qkv")
    _same_device(device, qkv=qkv, position=position, slot=slot, cos=cos, sin=sin, key_cache=key_cache,
                 value_cache=value_cache, q_norm=q_norm, k_norm=k_norm, out=out)
    block_stride = _caches(key_cache, value_cache)
    blocks, block, nkv, d = key_cache.shape
    dtype = qkv.dtype
    width = (num_heads + 2 * nkv) * d
    _need(dtype == key_cache.dtype, "qkv and the caches must have one type")
    _need(num_heads > 0 and qkv.dim() == 2 and qkv.shape[1] == width,
          f"qkv must be [tokens, {width}] for {num_heads} query and {nkv} KV heads of {d}")
    tokens = qkv.shape[0]
    _need(qkv.stride(1) == 1 or tokens == 0, "qkv rows must be contiguous")
    _vector(position, "position", torch.int64, tokens)
    _vector(slot, "slot", torch.int32, tokens)
    _need(cos.dim() == 2 and cos.shape == sin.shape and cos.dtype == sin.dtype and cos.dtype in (torch.bfloat16, torch.float32)
          and cos.is_contiguous() and sin.is_contiguous(), "cos and sin must be contiguous bf16 or fp32 [rows, rotary]")
    _need((q_norm is None) == (k_norm is None), "pass both norm weights or neither")
    if q_norm is not None:
        _vector(q_norm, "q_norm", dtype, d)
        _vector(k_norm, "k_norm", dtype, d)
    if out is None:
        out = torch.empty((tokens, num_heads, d), dtype=dtype, device=device)
    q_stride = _heads(out, "out", tokens, num_heads, d, dtype)
    index = _index(device)
    _done(_lib.load().cruise_decoder_rotate_store(
        qkv.data_ptr(), _row_stride(qkv, width), tokens, num_heads, nkv, d, _CODES[dtype], position.data_ptr(),
        slot.data_ptr(), None if q_norm is None else q_norm.data_ptr(), None if k_norm is None else k_norm.data_ptr(),
        eps, cos.data_ptr(), sin.data_ptr(), _CODES[cos.dtype], cos.shape[0], cos.shape[1], out.data_ptr(), q_stride,
        key_cache.data_ptr(), value_cache.data_ptr(), blocks, block, block_stride, index, _raw_stream(index)))
    return out


@functools.lru_cache(maxsize=1024)
def _attention_workspace(rows: int, nq: int, nkv: int, d: int, capacity: int, device: int) -> int:
    need = _lib.load().cruise_decoder_attention_workspace(rows, nq, nkv, d, capacity, device)
    if need < 0:
        _done(-1)
    return need


def paged_attention(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor,
                    seq_len: torch.Tensor, *, scale: float | None = None, out: torch.Tensor | None = None,
                    lse: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per row over the paged cache, split over the
    length and joined.

    ``q`` [rows, heads, d]; row r attends to its positions t < ``seq_len[r]``
    (int32 [rows]), position t in block ``block_table[r, t // block_size]`` (int32
    [rows, width]) of the caches [blocks, block_size, kv_heads, d].  Query heads
    share KV heads in order; ``scale`` is 1 / sqrt(d) by default.  Positions whose
    block lies outside the cache are left out; a row with no position left gets
    zeros.  Returns the outputs [rows, heads, d] (``out``); ``lse`` fp32
    [rows, heads] receives the logarithm of each softmax's sum (-inf for a row
    with no position), which joins outputs over further keys."""
    device = _cuda_device(q, "q")
    _same_device(device, q=q, key_cache=key_cache, value_cache=value_cache, block_table=block_table, seq_len=seq_len,
                 out=out, lse=lse)
    block_stride = _caches(key_cache, value_cache)
    blocks, block, nkv, d = key_cache.shape
    _need(q.dim() == 3 and q.shape[2] == d and q.shape[1] % nkv == 0 and q.shape[1] > 0,
          f"q must be [rows, a multiple of {nkv} heads, {d}]")
    rows, nq = q.shape[0], q.shape[1]
    dtype = key_cache.dtype
    q_stride = _heads(q, "q", rows, nq, d, dtype)
    _need(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == rows
          and (block_table.shape[1] < 2 or block_table.stride(1) == 1),
          f"block_table must be int32 [{rows}, width] with contiguous rows")
    table = block_table.shape[1]
    _vector(seq_len, "seq_len", torch.int32, rows)
    if out is None:
        out = torch.empty((rows, nq, d), dtype=dtype, device=device)
    out_stride = _heads(out, "out", rows, nq, d, dtype)
    if lse is not None:
        _need(lse.dtype == torch.float32 and tuple(lse.shape) == (rows, nq) and lse.is_contiguous(),
              f"lse must be contiguous fp32 [{rows}, {nq}]")
    index = _index(device)
    need = _attention_workspace(rows, nq, nkv, d, table * block, index)
    # from torch's allocator on this stream, so calls on other streams and captured graphs have their own
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _done(_lib.load().cruise_decoder_attention(
        q.data_ptr(), q_stride, rows, nq, nkv, d, _CODES[dtype], key_cache.data_ptr(), value_cache.data_ptr(), blocks,
        block, block_stride, block_table.data_ptr() if table else None, _row_stride(block_table, table), table,
        seq_len.data_ptr(), 1.0 / math.sqrt(d) if scale is None else scale, out.data_ptr(), out_stride,
        None if lse is None else lse.data_ptr(), None if workspace is None else workspace.data_ptr(), need, index,
        _raw_stream(index)))
    return out


def choose(logits: torch.Tensor, *, history: torch.Tensor | None = None, prompt_len: torch.Tensor | None = None,
           history_len: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
           frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
           bias_token: torch.Tensor | None = None, bias_value: torch.Tensor | None = None,
           bias_len: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
           active: torch.Tensor | None = None, processed: torch.Tensor | None = None,
           out: torch.Tensor | None = None, append: bool = False) -> torch.Tensor:
    """Bias, penalties for repeated tokens and a grammar mask on the logits, and
    the greedy token, in one pass.

    Per token of ``logits`` [rows, vocab] (fp32, bf16 or fp16), in fp32 and in
    this order: plus its ``bias_value`` (lists ``bias_token`` int32 / ``bias_value``
    fp32 [rows, width], the first ``bias_len[r]`` entries, tokens strictly
    increasing); when in the row's history, divided (x > 0) or multiplied by
    ``repetition[r]``; minus ``frequency[r]`` times its occurrences in the output,
    minus ``presence[r]`` when it occurs there; -inf when its bit of ``allowed``
    (int32 [rows, ceil(vocab / 32)], bit n % 32 of word n // 32) is 0.  The history
    int32 [rows, width] holds ``history_len[r]`` tokens, the first
    ``prompt_len[r]`` of them the prompt; ids outside the vocabulary do not count.

    Returns int64 [rows] (``out``): the first maximum above -inf; -1 where no
    token is left; -2 where a processed value is NaN or +inf.  Rows with
    ``active[r]`` 0 give -1 and write nothing else.  ``processed`` fp32
    [rows, vocab] receives the processed logits (it may be the fp32 logits
    themselves).  ``append`` also writes a chosen token to
    ``history[r, history_len[r]]`` where that is inside the tensor; the caller
    advances ``history_len``."""
    device = _cuda_device(logits, "logits")
    _same_device(device, logits=logits, history=history, prompt_len=prompt_len, history_len=history_len,
                 repetition=repetition, frequency=frequency, presence=presence, bias_token=bias_token,
                 bias_value=bias_value, bias_len=bias_len, allowed=allowed, active=active, processed=processed, out=out)
    _need(logits.dim() == 2 and logits.shape[1] > 0 and logits.dtype in _CODES
          and (logits.shape[1] == 1 or logits.stride(1) == 1),
          "logits must be fp32, bf16 or fp16 [rows, vocab] with contiguous rows")
    rows, vocab = logits.shape
    history_stride = history_width = 0
    if history is not None:
        _need(prompt_len is not None and history_len is not None, "a history needs prompt_len and history_len")
        _need(history.dtype == torch.int32 and history.dim() == 2 and history.shape[0] == rows and history.shape[1] > 0
              and (history.shape[1] == 1 or history.stride(1) == 1),
              f"history must be int32 [{rows}, width] with contiguous rows")
        _vector(prompt_len, "prompt_len", torch.int32, rows)
        _vector(history_len, "history_len", torch.int32, rows)
        history_width = history.shape[1]
        history_stride = _row_stride(history, history_width)
        _need(rows < 2 or history_stride >= history_width, "the rows of history must not overlap")
    else:
        _need(prompt_len is None and history_len is None and not append and repetition is None and frequency is None
              and presence is None, "penalties, lengths and append need a history")
    for name, vector in (("repetition", repetition), ("frequency", frequency), ("presence", presence)):
        if vector is not None:
            _vector(vector, name, torch.float32, rows)
    bias_stride = bias_width = 0
    if bias_token is not None:
        _need(bias_value is not None and bias_len is not None, "a bias list needs bias_value and bias_len")
        _need(bias_token.dtype == torch.int32 and bias_value.dtype == torch.float32 and bias_token.dim() == 2
              and bias_token.shape[0] == rows and bias_token.shape[1] > 0 and bias_token.shape == bias_value.shape
              and bias_token.is_contiguous() and bias_value.is_contiguous(),
              f"bias_token int32 and bias_value fp32 must be contiguous [{rows}, width]")
        _vector(bias_len, "bias_len", torch.int32, rows)
        bias_stride = bias_width = bias_token.shape[1]
    else:
        _need(bias_value is None and bias_len is None, "bias_value and bias_len need bias_token")
    allowed_stride = 0
    if allowed is not None:
        words = (vocab + 31) // 32
        _need(allowed.dtype == torch.int32 and tuple(allowed.shape) == (rows, words)
              and (words == 1 or allowed.stride(1) == 1),
              f"allowed must be int32 [{rows}, {words}] with contiguous rows")
        allowed_stride = _row_stride(allowed, words)
    if active is not None:
        _vector(active, "active", torch.int32, rows)
    processed_stride = 0
    if processed is not None:
        _need(processed.dtype == torch.float32 and processed.shape == logits.shape
              and (vocab == 1 or processed.stride(1) == 1),
              f"processed must be fp32 [{rows}, {vocab}] with contiguous rows")
        processed_stride = _row_stride(processed, vocab)
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=device)
    else:
        _vector(out, "out", torch.int64, rows)
    index = _index(device)

    def ptr(tensor):
        return None if tensor is None else tensor.data_ptr()

    _done(_lib.load().cruise_decoder_choose(
        logits.data_ptr(), _row_stride(logits, vocab), rows, vocab, _CODES[logits.dtype], ptr(active), ptr(history),
        history_stride, history_width, ptr(prompt_len), ptr(history_len), ptr(repetition), ptr(frequency),
        ptr(presence), ptr(bias_token), ptr(bias_value), bias_stride, bias_width, ptr(bias_len), ptr(allowed),
        allowed_stride, ptr(processed), processed_stride, out.data_ptr(), 1 if append else 0, index,
        _raw_stream(index)))
    return out
