"""The host loop's choice hook (cruise_b200.host_loop) on the CPU, driven by the
oracle's decoder step: first maxima through the hook are the plain loop, a
negative choice fails it, inactive rows' choices are not read."""

from __future__ import annotations

import numpy as np
import pytest

from cruise_b200.host_loop import HostLoopError, first_max, host_loop_epoch
from oracle.decoder import OracleDecoder
from oracle.epoch import OracleEpochController
from oracle.model import TINY, seeded_weights
from scenario import decode_inputs, make_scenario, prefill_epochs
from test_host_loop import OracleStep


def _run(choose):
    sc = make_scenario(vocab=TINY.vocab, seed=2, active_rows=(1, 0, 1, 1), k=4)
    controller = OracleEpochController(OracleDecoder(TINY, seeded_weights(TINY, seed=0)))
    for prefill in prefill_epochs(sc, TINY.block_size, TINY.vocab):
        controller.run(**prefill)
    return host_loop_epoch(OracleStep(controller), decode_inputs(sc, TINY.block_size), TINY.block_size, TINY.capacity, choose=choose)


def test_first_maxima_through_the_hook_are_the_plain_loop():
    seen = []

    def choose(logits, active):
        seen.append(np.asarray(active).copy())
        return np.array([first_max(row) if on else -1 for row, on in zip(logits, active)])

    for got, want in zip(_run(choose), _run(None)):
        np.testing.assert_array_equal(got, want)
    assert seen and not any(flags[1] for flags in seen)


@pytest.mark.parametrize("bad", [-1, -2])
def test_a_negative_choice_fails_the_loop(bad):
    with pytest.raises(HostLoopError) as err:
        _run(lambda logits, active: np.array([5, 5, bad, 5]))
    assert err.value.code == 23 and "row 2" in str(err.value)
