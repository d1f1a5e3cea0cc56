"""The host-loop route: an epoch driven from the host, one decoder call per
token (the reference's host runner, ``RunHostCase`` in
``history/attempts/g4c-attempt69e-r4-b4-resident-epoch-storage-guard/host/g4c_b4_epoch_runner.cpp:245-382``).

Each step calls the 9-in / 4-out decoder ABI (``EpochEngine.decoder_step``),
copies the logits to the host and decides there what the resident epoch
decides on the device: the greedy token (first maximum, non-finite logits
fail), the position progress check, the next slot (-1 at capacity), EOS and
the finish reasons.  It is the baseline of the resident epoch: both compute
the same tokens, KV and accounting, and the epoch saves the per-token host
round trips.

:class:`RuledChoice` in the place of the greedy choice leaves the logits on the
device and chooses there under each row's logit rules (penalties for repeated
tokens, biases, a grammar mask), which the resident epoch does not take.
"""

from __future__ import annotations

from typing import TYPE_CHECKING, Callable, Sequence

import numpy as np

from .model_config import BATCH, MAX_STEPS

if TYPE_CHECKING:
    import torch

FINISH_NONE, FINISH_EOS, FINISH_MAX_STEPS, FINISH_EMPTY, FINISH_ALREADY_FINISHED = 0, 1, 2, 4, 5


class HostLoopError(RuntimeError):
    """The runner's failure codes: 22 an inactive row moved, 23 non-finite
    logits or no position progress, 24 no slot for the next position."""

    def __init__(self, code: int, message: str) -> None:
        super().__init__(f"host loop failed ({code}): {message}")
        self.code = code


def first_max(logits_row: np.ndarray) -> int | None:
    """Index of the first maximum; None when any value is not finite."""
    if not np.isfinite(logits_row).all():
        return None
    return int(np.argmax(logits_row))   # numpy returns the first occurrence


def row_slot(block_table: np.ndarray, block_size: int, row: int, position: int) -> int:
    blocks = block_table.reshape(BATCH, -1)
    if position < 0 or position >= block_size * blocks.shape[1]:
        return -1
    return int(blocks[row, position // block_size]) * block_size + position % block_size


class RuledChoice:
    """The rows' tokens under logit rules, chosen on the device
    (:func:`cruise_b200.decoder_ops.choose`); the rows' histories stay there and
    grow with each choice.

    ``prompts``: the rows' tokens so far (they count for ``repetition``);
    ``capacity``: the longest history (the wider, the slower where rows are many:
    :func:`~cruise_b200.decoder_ops.choose` is planned by it).  ``repetition``, ``frequency``,
    ``presence``: a number, or one per row.  ``bias``: per row a dict of token to
    bias, or None.  ``allowed``: int32 bit masks [rows, ceil(vocab / 32)] on the
    device (replace or rewrite them between steps as a grammar advances).

    Calling it with logits [rows, vocab] on the device and the rows' active
    flags returns the tokens, int64 on the host: -1 where no token is left or the
    row is inactive, -2 where a processed logit is NaN or +inf."""

    def __init__(self, vocab: int, prompts: Sequence[Sequence[int]], capacity: int, *, device: int = 0,
                 repetition: float | Sequence[float] = 1.0, frequency: float | Sequence[float] = 0.0,
                 presence: float | Sequence[float] = 0.0, bias: Sequence[dict[int, float] | None] | None = None,
                 allowed: torch.Tensor | None = None) -> None:
        import torch

        rows = len(prompts)
        lengths = [len(p) for p in prompts]
        if capacity < 1 or max(lengths, default=0) > capacity:
            raise ValueError(f"a prompt of {max(lengths, default=0)} tokens does not fit a history of {capacity}")
        if bias is not None and len(bias) != rows:
            raise ValueError(f"{len(bias)} bias lists for {rows} rows")
        cuda = torch.device("cuda", device)

        def per_row(value) -> torch.Tensor:
            values = [float(value)] * rows if np.isscalar(value) else [float(v) for v in value]
            if len(values) != rows:
                raise ValueError(f"{len(values)} values for {rows} rows")
            return torch.tensor(values, dtype=torch.float32, device=cuda)

        history = torch.zeros((rows, capacity), dtype=torch.int32)
        for r, prompt in enumerate(prompts):
            history[r, : len(prompt)] = torch.tensor(list(prompt), dtype=torch.int32)
        self.vocab = vocab
        self.rules = dict(repetition=per_row(repetition), frequency=per_row(frequency), presence=per_row(presence))
        self.history = history.to(cuda)
        self.prompt_len = torch.tensor(lengths, dtype=torch.int32, device=cuda)
        self.history_len = self.prompt_len.clone()
        self.allowed = allowed
        lists = [sorted((entry or {}).items()) for entry in (bias or [])]
        width = max((len(entry) for entry in lists), default=0)
        if width:
            pad = [entry + [(vocab, 0.0)] * (width - len(entry)) for entry in lists]
            self.rules["bias_token"] = torch.tensor([[t for t, _ in e] for e in pad], dtype=torch.int32, device=cuda)
            self.rules["bias_value"] = torch.tensor([[v for _, v in e] for e in pad], dtype=torch.float32, device=cuda)
            self.rules["bias_len"] = torch.tensor([len(e) for e in lists], dtype=torch.int32, device=cuda)

    def __call__(self, logits: torch.Tensor, active) -> np.ndarray:
        import torch

        from . import decoder_ops

        flags = torch.as_tensor(np.asarray(active, dtype=np.int32), device=self.history.device)
        token = decoder_ops.choose(logits, history=self.history, prompt_len=self.prompt_len,
                                   history_len=self.history_len, allowed=self.allowed, active=flags, append=True,
                                   **self.rules)
        # (a full history keeps its length: what comes after no longer counts)
        self.history_len = torch.where(token >= 0, self.history_len + 1, self.history_len).clamp_(max=self.history.shape[1])
        return token.cpu().numpy()


def host_loop_epoch(step: Callable, inputs: dict, block_size: int, capacity: int,
                    choose: Callable | None = None) -> tuple[np.ndarray, np.ndarray]:
    """One epoch of ``inputs`` (the 8-in epoch ABI: token, position, seq_len,
    slot, active, block_table, control) as K host-driven decoder calls.
    ``step(token, position, seq_len, slot, active, block_table)`` returns
    (logits f32 [4, V], next_position i64 [4]).  ``choose(logits, active)`` (a
    :class:`RuledChoice`) gives the rows' tokens where it is not the first
    maximum; a negative one fails the loop (23).  Returns the token history
    i64 [8][4] and the runner's control words i32[28] (status 0; generation
    words 0, the runner does not report them)."""
    control = np.asarray(inputs["control"], dtype=np.int32)
    max_steps = int(control[0])
    eos = [int(v) for v in control[1:1 + BATCH]]
    token = np.array(inputs["token"], dtype=np.int64).reshape(BATCH)
    position = np.array(inputs["position"], dtype=np.int64).reshape(BATCH)
    length = np.array(inputs["seq_len"], dtype=np.int32).reshape(BATCH)
    slot = np.array(inputs["slot"], dtype=np.int32).reshape(BATCH)
    active = np.array(inputs["active"], dtype=np.int32).reshape(BATCH)
    block_table = np.array(inputs["block_table"], dtype=np.int32).reshape(-1)
    initial = active.copy()
    executed = [0] * BATCH
    reason = [FINISH_NONE] * BATCH
    for r in range(BATCH):
        if initial[r] == 0:
            reason[r] = FINISH_EMPTY if length[r] == 0 else FINISH_ALREADY_FINISHED
    history = np.full((MAX_STEPS, BATCH), -1, dtype=np.int64)
    calls = 0
    while calls < max_steps and active.any():
        before = active.copy()
        logits, next_position = step(token, position, length, slot, active, block_table)
        chosen = choose(logits, before) if choose is not None else None
        for r in range(BATCH):
            if before[r] == 0:
                if next_position[r] != position[r]:
                    raise HostLoopError(22, f"inactive row {r} moved")
                continue
            if chosen is None:
                generated = first_max(logits[r])
            else:
                generated = int(chosen[r]) if chosen[r] >= 0 else None
            if generated is None or next_position[r] != position[r] + 1:
                raise HostLoopError(23, f"row {r}: non-finite logits or no position progress" if chosen is None else
                                    f"row {r}: no token to choose, non-finite logits or no position progress")
            history[calls, r] = generated
            executed[r] += 1
            token[r] = generated
            length[r] = next_position[r] + 1
            if next_position[r] == capacity:
                slot[r] = -1
            else:
                slot[r] = row_slot(block_table, block_size, r, int(next_position[r]))
                if slot[r] < 0:
                    raise HostLoopError(24, f"row {r}: no slot for position {int(next_position[r])}")
            if generated == eos[r]:
                active[r] = 0
                reason[r] = FINISH_EOS
        position = next_position.astype(np.int64).copy()
        calls += 1
    for r in range(BATCH):
        if initial[r] == 1 and reason[r] == FINISH_NONE:
            reason[r] = FINISH_MAX_STEPS
    out = np.zeros(28, dtype=np.int32)
    out[0] = max_steps
    out[4] = calls
    for r in range(BATCH):
        out[6 + r] = eos[r]
        out[10 + r] = initial[r]
        out[14 + r] = executed[r]
        out[18 + r] = reason[r]
    out[22] = int(np.count_nonzero(initial))
    out[23] = int(np.count_nonzero(active))
    return history, out
