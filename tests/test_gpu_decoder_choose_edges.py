"""choose on values at the border of its definition: infinite logits and
negative, infinite and NaN penalties, against the definition step by step."""

from __future__ import annotations

import math

import pytest
import torch

from decoder_reference import choose_reference
from test_gpu_decoder_ops import check_choose, choose_case

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _device(cuda_ok):
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("vocab, pad", [(1, 0), (37, 1), (5003, 2), (50257, 0), (152064, 1)])
def test_infinite_logits_under_a_negative_repetition(vocab, pad, dtype):
    """+inf over a negative factor is -inf: the row has a choice, unless a +inf
    outside the history or a NaN is left."""
    rows = 9
    case = choose_case(rows, vocab, dtype, bias=0, mask=False, seed=60, pad=pad)
    first, last, mid = 0, vocab - 1, vocab // 2
    case["history"][:, :3] = torch.tensor([first, last, mid], dtype=torch.int32, device="cuda")
    case["history_len"][:] = 3
    case["prompt_len"][:] = torch.tensor([0, 1, 2, 3, 3, 0, 0, 0, 0], dtype=torch.int32, device="cuda")
    case["repetition"][:] = -1.5
    case["repetition"][1] = -0.0
    case["repetition"][5] = 1.5
    logits = case["logits"]
    logits[0, first] = logits[1, last] = logits[2, mid] = math.inf   # in vectors, before them and behind them
    logits[3, [first, last, mid]] = math.inf
    logits[4, [first, last, mid]] = math.inf
    logits[4, vocab // 3] = math.inf       # not in the history (but for one token)
    logits[5, mid] = math.inf              # a positive factor leaves it
    logits[6, mid] = math.nan
    logits[7] = math.inf
    case["active"] = torch.tensor([1] * 8 + [0], dtype=torch.int32, device="cuda")
    token = check_choose(case).tolist()
    check_choose(case, processed=False, append=False)
    if vocab > 37:
        assert min(token[:4]) >= 0 and token[4:8] == [-2] * 4


def test_infinite_logits_under_a_negative_repetition_in_place():
    from cruise_b200.decoder_ops import choose

    case = choose_case(4, 20011, FP32, seed=61)
    case["repetition"][:] = -1.2
    for r in range(4):
        n = int(case["history_len"][r])
        at = case["history"][r, :n].long()
        case["logits"][r, at[(at >= 0) & (at < 20011)]] = math.inf
    x32, token32 = choose_reference(**case, dtype=FP32)
    assert torch.equal(choose(**case, processed=case["logits"]), token32)
    same = (case["logits"] == x32) | (case["logits"].isnan() & x32.isnan())
    assert same.all()


def test_penalties_that_are_not_finite_act_on_the_tokens_they_are_for():
    """frequency and presence change tokens that occur in the output, repetition
    those of the history, and no others: infinite and NaN ones too."""
    from cruise_b200.decoder_ops import choose

    case = choose_case(7, 3001, FP32, bias=0, mask=True, seed=62)
    case["history_len"][:] = 20
    case["prompt_len"][:] = 5
    for r, (name, value) in enumerate([("frequency", math.inf), ("frequency", -math.inf), ("frequency", math.nan),
                                       ("presence", math.inf), ("presence", math.nan), ("repetition", math.inf),
                                       ("repetition", math.nan)]):
        case[name][r] = value
    check_choose(case)
    room = torch.empty(7, 3001, device="cuda")
    token = choose(**case, processed=room)
    for r in range(7):
        output = case["history"][r, 5:20].long()
        output = output[(output >= 0) & (output < 3001)]
        untouched = torch.ones(3001, dtype=torch.bool, device="cuda")
        seen = case["history"][r, :20].long()
        untouched[seen[(seen >= 0) & (seen < 3001)]] = False
        allowed = (case["allowed"][r, torch.arange(3001, device="cuda") >> 5] >> (torch.arange(3001, device="cuda") & 31)) & 1 != 0
        assert torch.equal(room[r][untouched & allowed], case["logits"][r][untouched & allowed])
        if r in (0, 3):   # an infinite penalty bans what was said
            assert (room[r][output] == -math.inf).all() and int(token[r]) not in output.tolist() and token[r] >= 0


@pytest.mark.parametrize("rows, vocab, cap", [(70, 152064, 13001), (40, 100003, 32768), (3, 390000, 20000)])
def test_histories_far_wider_than_what_they_hold(rows, vocab, cap):
    """Tensors so wide that a row takes sixteen CTAs however many rows there are;
    their rows hold a few tokens, some hold all the tensor has."""
    case = choose_case(rows, vocab, BF16, cap=cap, seed=63)
    case["history_len"][:] = torch.arange(rows, device="cuda") % 50
    case["history_len"][rows - 1] = cap - 1
    case["prompt_len"][:] = case["history_len"] // 2
    token = check_choose(case, processed=False, append=False)
    tight = dict(case)
    narrow = int(case["history_len"][:-1].max())
    tight["history"] = case["history"][:, :max(narrow, 1)].contiguous()
    from cruise_b200.decoder_ops import choose

    assert torch.equal(choose(**tight)[:-1], token[:-1])
