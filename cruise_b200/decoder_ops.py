"""The decoder operators on CUDA tensors (over the C ABI of include/cruise_decoder.h).

The pieces of one decode step around the paged cache, for any number of rows
and any context length: :func:`rotate_store` (head norms, rotation, paged
store), :func:`paged_attention` (one new token per row) and :func:`choose`
(logit rules and the greedy choice).  ``EpochEngine.decoder_step`` is the whole
step for the engine's four rows.

Calls run on the current stream of their tensors' device, queue their kernels
and return without waiting; they may be captured into a CUDA graph.  They keep
no state between calls.  They are inference operators: a tensor that requires
a gradient is refused while gradients are recorded, and one that carries a
forward-mode tangent; ``torch.compile`` runs them between its graphs.  Arguments that do not fit
raise ``ValueError``, failures of the library :class:`DecoderOpError`.  There is
no fallback without the built library.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib


class DecoderOpError(RuntimeError):
    """A decoder operator's failure other than invalid arguments (a CUDA error code)."""

    def __init__(self, code: int, message: str) -> None:
        super().__init__(f"decoder operator failed ({code}): {message}")
        self.code = code


def _bound():
    """The extension module that checks the tensors and calls the library."""
    try:
        from . import _decoder_bind
    except ImportError as exc:
        raise RuntimeError("the decoder operators' extension module is missing: build it with "
                           "`python -m cruise_b200.build` (there is no fallback)") from exc
    lib = _lib.load()
    names = ("rotate_store", "attention", "attention_workspace", "choose", "last_error")
    _decoder_bind.bind(*(ctypes.cast(getattr(lib, f"cruise_decoder_{name}"), ctypes.c_void_p).value for name in names),
                       DecoderOpError)
    return _decoder_bind


_bind = _bound()


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
    return _bind.rotate_store(qkv, position, slot, cos, sin, key_cache, value_cache, num_heads, q_norm, k_norm, eps, out)


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
    return _bind.paged_attention(q, key_cache, value_cache, block_table, seq_len, scale, out, lse)


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
    fp32 [rows, width], the first ``bias_len[r]`` entries, tokens
    increasing; entries of one token add up); when in the row's history, divided (x > 0) or multiplied by
    ``repetition[r]``; when it occurs in the output, minus ``frequency[r]`` times
    its occurrences there and minus ``presence[r]``; -inf when its bit of ``allowed``
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
    return _bind.choose(logits, history, prompt_len, history_len, repetition, frequency, presence, bias_token,
                        bias_value, bias_len, allowed, active, processed, out, append)
