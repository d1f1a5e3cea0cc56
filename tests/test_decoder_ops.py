"""Refusals of the decoder operators (cruise_b200.decoder_ops, include/cruise_decoder.h)
that need no GPU: the C entries check their arguments before any CUDA call, the
Python calls before the library."""

from __future__ import annotations

import pytest
import torch

from cruise_b200 import _lib, decoder_ops

A = 1 << 20   # made-up device addresses, far apart and 16-byte aligned; a refused call never follows them


def at(i: int) -> int:
    return A * (1 + 64 * i)


ROTATE = dict(qkv=at(0), qkv_stride=512, tokens=4, num_heads=4, num_kv_heads=2, head_dim=64, dtype=0, position=at(1),
              slot=at(2), q_norm=None, k_norm=None, eps=1e-6, rope_cos=at(3), rope_sin=at(4), rope_dtype=0,
              rope_rows=32, rotary=64, q_out=at(5), q_stride=256, key_cache=at(6), value_cache=at(7), num_blocks=8,
              block_size=16, block_stride=2048, device=0, stream=None)
ATTEND = dict(q=at(0), q_stride=256, rows=4, num_heads=4, num_kv_heads=2, head_dim=64, dtype=0, key_cache=at(1),
              value_cache=at(2), num_blocks=8, block_size=16, block_stride=2048, block_table=at(3), table_stride=2,
              table_width=2, seq_len=at(4), scale=0.125, out=at(5), out_stride=256, lse=None, workspace=None,
              workspace_bytes=0, device=0, stream=None)
CHOOSE = dict(logits=at(0), logits_stride=100, rows=4, vocab=100, dtype=2, active=None, history=at(1),
              history_stride=10, history_width=10, prompt_len=at(2), history_len=at(3), repetition=None,
              frequency=None, presence=None, bias_token=None, bias_value=None, bias_stride=0, bias_width=0,
              bias_len=None, allowed=None, allowed_stride=0, processed=None, processed_stride=0, token=at(4), append=1,
              device=0, stream=None)


def call(name: str, arguments: dict) -> tuple[int, str]:
    lib = _lib.load()
    rc = getattr(lib, name)(*arguments.values())
    return rc, lib.cruise_decoder_last_error().decode()


@pytest.mark.parametrize("change, reason", [
    (dict(tokens=-1), "tokens"), (dict(num_heads=0), "heads"), (dict(head_dim=96), "head size"),
    (dict(dtype=2), "dtype"), (dict(rope_dtype=1), "rope dtype"), (dict(rotary=24), "multiple of 16"),
    (dict(rotary=80), "head size"), (dict(rope_rows=0), "rows"), (dict(q_norm=at(8)), "both norm weights"),
    (dict(num_blocks=0), "blocks"), (dict(num_blocks=1 << 30), "below 2^31"), (dict(qkv_stride=504), "stride"),
    (dict(q_stride=257), "multiples of 8"), (dict(block_stride=1024), "stride"), (dict(qkv=None), "NULL"),
    (dict(slot=None), "NULL"), (dict(qkv=at(0) + 8), "aligned"), (dict(q_out=at(0) + 64), "overlap"),
    (dict(key_cache=at(0)), "overlap"), (dict(key_cache=at(7)), "must not be one"), (dict(q_out=at(6) + 2048), "overlap"),
])
def test_rotate_store_refuses(change, reason):
    rc, why = call("cruise_decoder_rotate_store", {**ROTATE, **change})
    assert rc == -1 and reason in why and why.startswith("cruise_decoder_rotate_store"), (rc, why)


@pytest.mark.parametrize("change, reason", [
    (dict(rows=-1), "rows"), (dict(num_heads=5), "multiple"), (dict(head_dim=32), "head size"),
    (dict(dtype=2), "dtype"), (dict(num_blocks=0), "blocks"), (dict(table_width=-1), "tables"),
    (dict(table_width=1 << 28, table_stride=1 << 28), "capacity"),
    (dict(rows=1, num_heads=1, num_kv_heads=1, table_width=(2 ** 31 - 200) // 16, table_stride=1 << 28), "capacity"),
    (dict(rows=8, num_heads=8, num_kv_heads=8, table_width=(2 ** 31 - 320) // 16, table_stride=1 << 28, q_stride=512,
          out_stride=512, block_stride=8192), "passes 2^31"),
    (dict(rows=1 << 20, table_width=1 << 20, table_stride=1 << 20), "passes 2^31"),
    (dict(table_stride=1), "stride"), (dict(q_stride=252), "stride"), (dict(out_stride=260), "multiples of 8"),
    (dict(num_blocks=1 << 20, block_stride=1 << 16), "2^35"), (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(out=None), "NULL"),
    (dict(block_table=None), "NULL"), (dict(q=at(0) + 2), "aligned"), (dict(out=at(0)), "overlap"),
    (dict(out=at(2) + 4096), "overlap"), (dict(lse=at(5) + 16), "overlap"), (dict(lse=at(4)), "overlap"),
    (dict(table_width=1 << 16, table_stride=1 << 16), "workspace"),
    (dict(table_width=1 << 16, table_stride=1 << 16, workspace=at(9), workspace_bytes=64), "workspace"),
    (dict(table_width=1 << 16, table_stride=1 << 16, workspace=at(1) - 4096, workspace_bytes=1 << 40), "workspace must not"),
])
def test_attention_refuses(change, reason):
    if "workspace" in reason:   # long rows are split whatever the device, and the pieces need room
        lib, a = _lib.load(), {**ATTEND, **change}
        assert lib.cruise_decoder_attention_workspace(a["rows"], a["num_heads"], a["num_kv_heads"], a["head_dim"],
                                                      a["table_width"] * a["block_size"], a["device"]) > 64
    rc, why = call("cruise_decoder_attention", {**ATTEND, **change})
    if torch.cuda.is_available() or "workspace" not in reason:
        assert rc == -1 and reason in why, (rc, why)
    else:   # the workspace is asked of the device
        assert rc != 0, why


@pytest.mark.parametrize("change, reason", [
    (dict(rows=-1), "rows"), (dict(rows=70000), "rows"), (dict(vocab=0), "logits"), (dict(vocab=(1 << 20) + 1), "logits"),
    (dict(vocab=1000000, logits_stride=1000000, history_width=30000, history_stride=30000), "entries"),
    (dict(history_width=1 << 30, history_stride=1 << 30), "entries"),
    (dict(bias_token=at(6), bias_value=at(7), bias_len=at(8), bias_width=(1 << 30) - 10, bias_stride=1 << 30), "entries"),
    (dict(dtype=3), "dtype"), (dict(logits_stride=99), "stride"), (dict(history_width=11), "history"),
    (dict(history_len=None), "history"), (dict(history=None), "need a history"),
    (dict(history=None, append=0, presence=at(6)), "need a history"),
    (dict(bias_token=at(6)), "bias list"),
    (dict(bias_token=at(6), bias_value=at(7), bias_len=at(8), bias_width=4, bias_stride=3), "bias list"),
    (dict(allowed=at(6), allowed_stride=3), "stride"), (dict(processed=at(6), processed_stride=99), "stride"),
    (dict(processed=at(0) + 64, processed_stride=100), "overlap"),
    (dict(processed=at(0), processed_stride=104), "overlap"), (dict(processed=at(1) - 64, processed_stride=100), "overlap"),
    (dict(token=at(1)), "overlap"), (dict(allowed=at(4) - 32, allowed_stride=4), "overlap"), (dict(token=None), "NULL"), (dict(logits=None), "NULL"),
    (dict(logits=at(0) + 2), "aligned"), (dict(token=at(4) + 4), "aligned"),
])
def test_choose_refuses(change, reason):
    rc, why = call("cruise_decoder_choose", {**CHOOSE, **change})
    assert rc == -1 and reason in why, (rc, why)


def test_nothing_to_do_succeeds_without_a_device():
    for name, arguments, empty in (("cruise_decoder_rotate_store", ROTATE, "tokens"),
                                   ("cruise_decoder_attention", ATTEND, "rows"), ("cruise_decoder_choose", CHOOSE, "rows")):
        assert call(name, {**arguments, empty: 0}) == (0, "")


def test_workspace_is_planned_on_the_host():
    lib = _lib.load()
    assert lib.cruise_decoder_attention_workspace(4, 28, 4, 128, 256, 0) == 0
    assert lib.cruise_decoder_attention_workspace(4, 28, 4, 128, 1 << 17, 0) > 0
    assert lib.cruise_decoder_attention_workspace(4, 28, 3, 128, 256, 0) == -1
    assert "multiple" in lib.cruise_decoder_last_error().decode()
    assert lib.cruise_decoder_attention_workspace(4, 28, 4, 96, 256, 0) == -1


def test_last_error_is_the_calling_threads():
    import threading

    assert call("cruise_decoder_choose", {**CHOOSE, "vocab": 0})[0] == -1
    seen = []
    thread = threading.Thread(target=lambda: seen.append(_lib.load().cruise_decoder_last_error()))
    thread.start()
    thread.join()
    assert seen == [b""] and _lib.load().cruise_decoder_last_error() != b""


def test_python_calls_refuse_cpu_tensors():
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    ints = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="q must be a CUDA tensor"):
        decoder_ops.paged_attention(x, cache, cache, torch.zeros(2, 1, dtype=torch.int32), ints)
    with pytest.raises(ValueError, match="qkv must be a CUDA tensor"):
        decoder_ops.rotate_store(x.view(2, -1), ints.long(), ints, x[0], x[0], cache, cache, num_heads=1)
    with pytest.raises(ValueError, match="logits must be a CUDA tensor"):
        decoder_ops.choose(torch.zeros(2, 10))
    with pytest.raises(ValueError, match="logits must be a CUDA tensor"):
        decoder_ops.choose([[0.0]])


def test_a_cuda_failure_is_an_exception_with_its_code():
    error = decoder_ops.DecoderOpError(700, "why")
    assert error.code == 700 and isinstance(error, RuntimeError) and "why" in str(error)


def test_the_python_calls_use_the_loaded_library():
    assert decoder_ops._bind.bind is not None
    with pytest.raises(ValueError, match="NULL"):
        decoder_ops._bind.bind(0, 0, 0, 0, 0, RuntimeError)
    with pytest.raises(TypeError, match="arguments"):
        decoder_ops._bind.choose(1, 2)
    with pytest.raises(ValueError, match="logits must be a CUDA tensor"):   # still bound
        decoder_ops.choose(torch.zeros(1, 1))
