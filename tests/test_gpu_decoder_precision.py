"""paged_attention keeps its probabilities in more bits than the cache's type:
outputs against 64 bits with bounds that have no rounding of the probabilities
in them, and weak keys beside a dominating one.

The second product takes a probability p (at most 1) as two terms of the cache's
type, hi = round(c p (1 - 2 u)) and lo = round(c p - hi), u half a step of the
type relative to the value, c a power of two (1 in bf16, 2^15 in fp16).  hi is at
most u off its argument, so 0 <= c p - hi <= 3 u c p, and lo's own rounding is at
most u of that: the pair is at most 3 u^2 p off, and in fp16 half the smallest
step, 2^-25 / 2^15 = 2^-40, where lo falls below the type's normal range.
"""

from __future__ import annotations

import math

import pytest
import torch

from decoder_reference import U32, attention_reference, floor, unit
from test_gpu_decoder_ops import attend_case

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _device(cuda_ok):
    yield
    torch.cuda.synchronize()


def tight_bound(q, key, value, table, lens):
    """The bound of attention_reference with 3 u^2 and 2^-40 in the place of the
    probabilities' rounding u and its floor."""
    rows, nq, d = q.shape
    block, nkv = key.shape[1], key.shape[2]
    group, u, scale = nq // nkv, unit(q.dtype), 1.0 / math.sqrt(d)
    out = attention_reference(q, key, value, table, lens)[0]
    bound = torch.zeros_like(out)
    for r, n in enumerate(lens.tolist()):
        if n == 0:
            continue
        t = torch.arange(n, device=q.device)
        pages = table[r].long()[t // block]
        k, v = key[pages, t % block].double(), value[pages, t % block].double()
        for h in range(nkv):
            heads = slice(h * group, (h + 1) * group)
            qh = q[r, heads].double()
            ds = (d + 8) * 2 * U32 * scale * (qh.abs() @ k[:, h].abs().T).amax(1, keepdim=True)
            weight = torch.softmax(scale * qh @ k[:, h].T, dim=1) @ v[:, h].abs()
            err = weight * (3 * u * u + (n + 64) * 2 * U32 + torch.expm1(2 * ds)) + n * 2.0 ** -40 * v[:, h].abs().amax()
            bound[r, heads] = err + u * (out[r, heads].abs() + err) + floor(q.dtype)
    return out, bound


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lens, nq, nkv, d, width", [
    ([16, 3, 0, 1], 14, 2, 128, 1),            # a warp for each unit
    ([31, 64, 1, 0], 24, 2, 64, 4),            # four warps
    ([250, 44, 0, 131], 28, 4, 128, 16),       # eight
    ([256, 257, 300], 16, 1, 128, None),       # a cluster, 16 heads a unit
    ([513, 0, 1, 900, 64], 7, 1, 128, 2000),   # split over all CTAs
    ([700, 20, 300], 32, 2, 64, 2000),
])
def test_outputs_have_no_rounding_of_the_probabilities(lens, nq, nkv, d, width, dtype):
    from cruise_b200.decoder_ops import paged_attention

    case = attend_case(lens, nq, nkv, d, dtype, width=width, seed=50 + len(lens))
    got = paged_attention(*case.values()).double()
    want, bound = tight_bound(*case.values())
    excess = (got - want).abs() - bound
    assert float(excess.max()) <= 0, f"{int((excess > 0).sum())} of {excess.numel()} outputs pass the bound"


@pytest.mark.parametrize("rows, heads, d, length, width", [
    (600, 8, 64, 131072, 8192),    # whole rows for a CTA of the split form: 32768 keys for a warp
    (3, 16, 128, 2048, 128),       # clusters
    (1, 1, 64, 256, 16),
])
def test_weak_keys_beside_a_dominating_one_count(rows, heads, d, length, width):
    """Key 0 has score 18 and value 0, the others score 0 and value 1, so the
    output is N w / (1 + N w) with w = e^-18 = 2^-25.97, under half of fp16's
    smallest step.  Scores are exact up to the factor log2 e (2 U32 of 26); the
    chains of sums are at most the warp's length / 64 steps of 16 keys, for the
    numerator and for the sum, and the joins of up to 16 parts."""
    from cruise_b200.decoder_ops import paged_attention

    key = torch.zeros(length // 16, 16, 1, d, dtype=FP16, device="cuda")
    value = torch.ones_like(key)
    key[0, 0, 0, 0] = 1
    value[0, 0] = 0
    q = torch.zeros(rows, heads, d, dtype=FP16, device="cuda")
    q[..., 0] = 18
    table = torch.arange(width, dtype=torch.int32, device="cuda").expand(rows, width).contiguous()
    lens = torch.full((rows,), length, dtype=torch.int32, device="cuda")
    lse = torch.empty(rows, heads, device="cuda")
    out = paged_attention(q, key, value, table, lens, scale=1.0, lse=lse).double()
    weak = (length - 1) * math.exp(-18)
    want = weak / (1 + weak)
    sums = 2 * (length // 64 + 80) * 2 * U32 + 4 * 26 * U32
    bound = want * sums + unit(FP16) * want * (1 + sums) + floor(FP16) + length * 2.0 ** -40
    assert float((out - want).abs().max()) <= bound, (float((out - want).abs().max()) / want, bound / want)
    # the sum's chain, in fp32: weak keys next to 1 lose at most half a step of it each
    assert float((lse.double() - (18 + math.log1p(weak))).abs().max()) <= sums + 4 * U32 * 19


def test_infinite_values_stay_infinite():
    """No part of a probability is zero or negative where the probability is not:
    an infinite value gives an infinite output, also for p = 1 and p = 1/2."""
    from cruise_b200.decoder_ops import paged_attention

    for dtype in (BF16, FP16):
        for lens in ([1, 2, 40], [1, 2, 200]):
            case = attend_case(lens, 4, 2, 64, dtype, seed=51)
            case["key_cache"].zero_()   # equal weights, exact in the type for lengths 1 and 2
            page = case["block_table"][:, 0]
            case["value_cache"][page[0], 0, 0, 5] = math.inf
            case["value_cache"][page[1], 1, 1, 6] = -math.inf
            case["value_cache"][page[2], 7, 0, 7] = math.inf
            out = paged_attention(*case.values())
            assert (out[0, :2, 5] == math.inf).all() and (out[1, 2:, 6] == -math.inf).all() and (out[2, :2, 7] == math.inf).all()
            assert int(torch.isfinite(out).sum()) == out.numel() - 6
