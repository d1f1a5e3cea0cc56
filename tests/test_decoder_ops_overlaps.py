"""The C entries of the decoder operators refuse outputs that overlap what the
call reads, before any launch (no GPU needed); arrays that only lie between one
another pass this check."""

from __future__ import annotations

import pytest
import torch

from test_decoder_ops import CHOOSE, ROTATE, at, call

NORMS = dict(q_norm=at(8), k_norm=at(9))
# rotate_store's sizes: qkv 4 rows of 512, q_out 4 of 256, caches 8 blocks of 2048 elements (4096 bytes), tables of 4096 bytes


@pytest.mark.parametrize("change", [
    dict(q_out=at(1)), dict(q_out=at(1) - 2032), dict(position=at(5) + 1024), dict(slot=at(5) + 2044), dict(q_out=at(2)),
    dict(q_out=at(3) + 4080), dict(q_out=at(4)), dict(rope_sin=at(5) + 16), dict(q_out=at(8) + 112, **NORMS),
    dict(q_out=at(9), **NORMS), dict(position=at(6) + 32760), dict(slot=at(7) + 4), dict(rope_cos=at(6) + 64),
    dict(rope_sin=at(7)), dict(q_norm=at(6), k_norm=at(9)), dict(q_norm=at(8), k_norm=at(7) + 32752),
    dict(qkv=at(6) + 32752),
])
def test_rotate_store_refuses_outputs_over_inputs(change):
    rc, why = call("cruise_decoder_rotate_store", {**ROTATE, **change})
    assert rc == -1 and "overlap" in why, (rc, why)


@pytest.mark.parametrize("change", [
    dict(value_cache=at(6) + 16), dict(value_cache=at(6) + 4096), dict(value_cache=at(6) - 4080), dict(key_cache=at(7) + 7 * 4096),
    dict(value_cache=at(6) + 4080, block_stride=4096), dict(value_cache=at(6) + 4112, block_stride=4096),
    dict(value_cache=at(6) - 8192 * 3 - 16, block_stride=4096), dict(value_cache=at(6) + 64, num_blocks=1),
])
def test_rotate_store_refuses_caches_over_one_another(change):
    rc, why = call("cruise_decoder_rotate_store", {**ROTATE, **change})
    assert rc == -1 and "blocks of the two caches" in why, (rc, why)


@pytest.mark.parametrize("change", [
    dict(value_cache=at(6) + 4096, block_stride=4096), dict(value_cache=at(6) - 4096, block_stride=4096),
    dict(value_cache=at(6) + 8192 * 5 + 4096, block_stride=4096), dict(value_cache=at(6) + 8 * 4096),
    dict(value_cache=at(6) - 8 * 4096), dict(value_cache=at(6) + 4096, num_blocks=1), dict(value_cache=at(6) + 5000 * 16, block_stride=1 << 15),
])
def test_rotate_store_takes_caches_that_alternate(change):
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: the call would launch")
    rc, why = call("cruise_decoder_rotate_store", {**ROTATE, **change})
    assert rc > 0, why   # no device: past every check


# choose's sizes: logits 4 rows of 100 fp32, history 4 of 10, vectors of 4, processed 1600 bytes, token 32
EVERY = dict(processed=at(5), processed_stride=100, active=at(6), repetition=at(7), frequency=at(8), presence=at(9),
             bias_token=at(10), bias_value=at(11), bias_len=at(12), bias_width=5, bias_stride=6, allowed=at(13), allowed_stride=4)


@pytest.mark.parametrize("name", ["active", "repetition", "frequency", "presence", "bias_token", "bias_value", "bias_len",
                                  "allowed", "prompt_len", "history_len"])
@pytest.mark.parametrize("output, last", [("token", 28), ("processed", 1596), ("history", 156)])
def test_choose_refuses_outputs_over_inputs(name, output, last):
    base = {**CHOOSE, **EVERY}
    for off in (0, last):
        rc, why = call("cruise_decoder_choose", {**base, name: base[output] + off})
        assert rc == -1 and "overlap" in why, (rc, why)
    rc, why = call("cruise_decoder_choose", {**base, output: base[name] + 8})
    assert rc == -1 and "overlap" in why, (rc, why)


def test_choose_takes_neighbours_and_a_history_it_only_reads():
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: the call would launch")
    for change in (dict(active=at(4) + 32), dict(repetition=at(5) + 1600), dict(presence=at(1) + 160),
                   dict(append=0, history_len=at(1) + 8), dict(repetition=at(9), presence=at(9)), dict(processed=at(0))):
        rc, why = call("cruise_decoder_choose", {**CHOOSE, **EVERY, **change})
        assert rc > 0, why   # no device: past every check


def test_the_capacity_s_limit_is_the_one_that_is_named():
    from cruise_b200 import _lib

    workspace = _lib.load().cruise_decoder_attention_workspace
    assert workspace(1, 1, 1, 64, 2 ** 31 - 257, 0) > 0
    assert workspace(1, 1, 1, 64, 2 ** 31 - 256, 0) == -1
    assert "below 2^31 - 256" in _lib.load().cruise_decoder_last_error().decode()
