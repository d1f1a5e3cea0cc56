"""The C entries of the decoder operators refuse outputs that overlap what the
call reads, before any launch (no GPU needed); arrays that only lie between one
another pass this check."""

from __future__ import annotations

import pytest
import torch

from test_decoder_ops import ROTATE, at, call

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
