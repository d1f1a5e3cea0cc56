"""The decoder operators (cruise_b200.decoder_ops) on the GPU against their
definitions in 64 bits (decoder_reference), with bounds that count the
kernels' roundings; their edges (empty rows, bad blocks and slots, NaN in
masked places, strides, far offsets); streams and CUDA graphs; and a run of
the three as a decode loop uses them."""

from __future__ import annotations

import math

import pytest
import torch

from decoder_reference import U32, attention_reference, choose_reference, rotate_reference

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _device(cuda_ok):
    yield
    torch.cuda.synchronize()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=FP32):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def within(got, want, bound, what):
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    if got.numel() == 0:
        return
    excess = (got - want).abs() - bound
    assert float(excess.max()) <= 0, f"{what}: {float((got - want).abs().max()):.3g} off, bound passed by {float(excess.max()):.3g}"


# ---- rotate_store ------------------------------------------------------------------

def rope(rows, rotary, dtype):
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * (
        1e6 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary))
    angle = torch.cat((angle, angle), dim=1)
    return angle.cos().to(dtype), angle.sin().to(dtype)


def rotate_case(tokens, nq, nkv, d, dtype, *, rotary=None, tables=BF16, norm=False, block=16, seed=0, rows=600):
    g = gen(seed)
    blocks = -(-tokens // block) + 2
    cos, sin = rope(rows, rotary or d, tables)
    case = dict(qkv=randn(g, tokens, (nq + 2 * nkv) * d, dtype=dtype),
                position=torch.randint(0, rows, (tokens,), device="cuda", generator=g),
                slot=torch.randperm(blocks * block, device="cuda", generator=g)[:tokens].int(),
                cos=cos, sin=sin, key_cache=randn(g, blocks, block, nkv, d, dtype=dtype),
                value_cache=randn(g, blocks, block, nkv, d, dtype=dtype))
    keep = dict(num_heads=nq)
    if norm:
        keep.update(q_norm=1 + randn(g, d, dtype=dtype) / 8, k_norm=1 + randn(g, d, dtype=dtype) / 8, eps=1e-5)
    return case, keep


def check_rotate(case, keep, out=None):
    from cruise_b200.decoder_ops import rotate_store

    key0, value0 = case["key_cache"].clone(), case["value_cache"].clone()
    blocks, block, nkv, d = key0.shape
    nq = keep["num_heads"]
    q = rotate_store(*case.values(), **keep, out=out)
    z, bound, v = rotate_reference(case["qkv"], case["position"], case["cos"], case["sin"], nq, nkv, d,
                                   keep.get("q_norm"), keep.get("k_norm"), keep.get("eps", 1e-6))
    within(q, z[:, :nq], bound[:, :nq], "q")
    position, slot = case["position"], case["slot"].long()
    stored = (slot >= 0) & (slot < blocks * block) & (position >= 0) & (position < case["cos"].shape[0])
    key, value = case["key_cache"].reshape(-1, nkv, d), case["value_cache"].reshape(-1, nkv, d)
    within(key[slot[stored]], z[stored][:, nq:], bound[stored][:, nq:], "k")
    assert torch.equal(value[slot[stored]].double(), v[stored])
    untouched = torch.ones(blocks * block, dtype=torch.bool, device="cuda")
    untouched[slot[stored]] = False
    assert torch.equal(key[untouched], key0.reshape(-1, nkv, d)[untouched])
    assert torch.equal(value[untouched], value0.reshape(-1, nkv, d)[untouched])
    return q


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens, nq, nkv, d, rotary, tables, norm", [
    (1, 1, 1, 64, 64, BF16, False), (4, 28, 4, 128, 128, BF16, False), (4, 28, 4, 128, 128, FP32, True),
    (3, 9, 3, 64, 32, FP32, True), (7, 5, 5, 128, 16, BF16, True), (333, 6, 1, 64, 48, BF16, True),
    (1000, 28, 4, 128, 64, FP32, True), (2777, 3, 1, 128, 128, BF16, False),
])
def test_rotate_store(tokens, nq, nkv, d, rotary, tables, norm, dtype):
    check_rotate(*rotate_case(tokens, nq, nkv, d, dtype, rotary=rotary, tables=tables, norm=norm, seed=tokens))


def test_rotate_store_leaves_out_padded_tokens():
    case, keep = rotate_case(9, 4, 2, 64, BF16, norm=True, seed=3)
    case["slot"][2], case["slot"][5], case["slot"][6] = -1, case["key_cache"].shape[0] * 16, 2 ** 31 - 1
    case["position"][1], case["position"][7], case["position"][8] = -1, case["cos"].shape[0], 2 ** 40
    q = check_rotate(case, keep)
    assert not q[[1, 7, 8]].any()


def test_rotate_store_strided_rows_and_blocks():
    case, keep = rotate_case(37, 7, 1, 128, FP16, norm=True, seed=4, block=24)
    wide = torch.full((37, case["qkv"].shape[1] + 40), float("nan"), dtype=FP16, device="cuda")
    wide[:, 8:-32] = case["qkv"]
    case["qkv"] = wide[:, 8:-32]
    both = torch.stack((case["key_cache"], case["value_cache"]), dim=1)   # [blocks, 2, ...]: K and V of a block together
    case["key_cache"], case["value_cache"] = both[:, 0], both[:, 1]
    room = torch.zeros(37, 9, 128, dtype=FP16, device="cuda")
    check_rotate(case, keep, out=room[:, 1:8])
    assert not room[:, 0].any() and not room[:, 8].any()


def test_rotate_store_zero_vector_and_far_positions():
    case, keep = rotate_case(5, 2, 1, 64, BF16, norm=True, seed=5, rows=131072, tables=FP32)
    case["qkv"][1] = 0
    case["position"][:] = torch.tensor([131071, 0, 131070, 65537, 1])
    q = check_rotate(case, keep)
    assert not q[1].any()


def test_rotate_store_past_32_bits():
    blocks, block, nkv, d = 8200, 512, 4, 128   # 2^31 elements and more per cache
    case, keep = rotate_case(4, 4, nkv, d, BF16, seed=6)
    case["key_cache"] = torch.zeros(blocks, block, nkv, d, dtype=BF16, device="cuda")
    case["value_cache"] = torch.zeros(blocks, block, nkv, d, dtype=BF16, device="cuda")
    case["slot"] = torch.tensor([0, blocks * block - 1, 4194304, 4194303], dtype=torch.int32, device="cuda")
    check_rotate(case, keep)


def test_rotate_store_without_tokens():
    case, keep = rotate_case(1, 4, 2, 64, BF16)
    from cruise_b200.decoder_ops import rotate_store

    case.update(qkv=case["qkv"][:0], position=case["position"][:0], slot=case["slot"][:0])
    assert rotate_store(*case.values(), **keep).shape == (0, 4, 64)


# ---- paged_attention ---------------------------------------------------------------

def attend_case(lens, nq, nkv, d, dtype, *, block=16, width=None, seed=0, loud=1.5):
    g = gen(seed)
    rows = len(lens)
    used = [-(-n // block) for n in lens]
    blocks = sum(used) + 3
    order = torch.randperm(blocks, device="cuda", generator=g).int()
    table = torch.full((rows, max(width or 0, max(used), 1)), -7, dtype=torch.int32, device="cuda")
    start = 0
    for r, n in enumerate(used):
        table[r, :n] = order[start:start + n]
        start += n
    return dict(q=randn(g, rows, nq, d, dtype=dtype) * loud, key_cache=randn(g, blocks, block, nkv, d, dtype=dtype),
                value_cache=randn(g, blocks, block, nkv, d, dtype=dtype), block_table=table,
                seq_len=torch.tensor(lens, dtype=torch.int32, device="cuda"))


def check_attend(case, **keep):
    from cruise_b200.decoder_ops import paged_attention

    rows, nq, d = case["q"].shape
    lse = torch.full((rows, nq), 5.0, device="cuda")
    out = paged_attention(*case.values(), lse=lse, **keep)
    again = paged_attention(*case.values(), **{k: v for k, v in keep.items() if k != "out"})
    want, want_lse, bound, lse_bound = attention_reference(*case.values(), scale=keep.get("scale"))
    within(out, want, bound, "out")
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    within(lse[~empty], want_lse[~empty], lse_bound[~empty], "lse")
    assert torch.equal(out, again)   # the split is fixed by the sizes: the same bits again
    return out


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lens, nq, nkv, d, block, width", [
    ([1], 1, 1, 64, 16, None),
    ([0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256], 28, 4, 128, 128, 2),
    ([200, 44, 0, 131], 28, 4, 128, 128, 2),
    ([5, 100, 40], 8, 8, 64, 24, None),
    ([511, 512, 300], 9, 1, 128, 64, 8),
    ([513, 0, 1, 2000, 64, 5000], 7, 1, 128, 16, None),
    ([3000, 1, 0, 777], 32, 8, 64, 24, None),
    ([1025] * 5, 16, 1, 64, 32, None),
    ([700, 20, 1300], 40, 2, 128, 128, None),      # 20 heads share a KV head: two units of 10
    ([900, 0, 4097], 33, 1, 64, 48, None),          # three units of 11
    ([1] * 150 + [2500], 4, 2, 64, 16, None),       # more rows than threads of a CTA
    ([0, 0, 0], 4, 2, 128, 128, 8),
    ([10000], 12, 4, 128, 128, 1024),               # a table far wider than the row
    ([1, 0, 127, 128, 129, 1000, 2048], 6, 2, 128, 64, None),   # ten CTAs a unit, more than some rows have tiles
    ([383, 384, 385, 0], 14, 2, 64, 32, None),
    ([256, 257, 300], 16, 1, 128, 16, None),
    ([16384, 5], 8, 1, 128, 128, None),
    ([1024] * 36 + [0], 28, 4, 128, 128, None),     # one CTA for each unit, and for each SM
    ([16, 3, 0, 1], 14, 2, 128, 16, 1),             # a warp for each unit
    ([1, 100, 33, 0, 17] * 40, 16, 4, 64, 16, 8),   # (more of them than run at once)
    ([31, 64, 1, 0], 24, 2, 64, 16, 4),             # four warps for each unit
    ([200, 500, 0, 1, 64, 65] * 30, 11, 1, 128, 24, None),
    ([513, 0, 1, 2000, 64, 5000], 7, 1, 128, 16, 2000),         # wide tables: units split over all CTAs
    ([3000, 1, 0, 777], 32, 8, 64, 24, 1000),
    ([1025] * 5, 16, 1, 64, 32, 600),
    ([700, 20, 1300], 40, 2, 128, 128, 150),
    ([900, 0, 4097], 33, 1, 64, 48, 400),
])
def test_paged_attention(lens, nq, nkv, d, block, width, dtype):
    check_attend(attend_case(lens, nq, nkv, d, dtype, block=block, width=width, seed=len(lens)))


def test_paged_attention_long_row():
    check_attend(attend_case([70001], 7, 1, 128, BF16, block=128, seed=1))


def test_paged_attention_sharp_and_scaled():
    check_attend(attend_case([600, 37], 8, 2, 64, FP16, seed=2, loud=12.0))
    check_attend(attend_case([600, 37], 8, 2, 64, BF16, seed=2), scale=-0.3)
    check_attend(attend_case([600, 37], 8, 2, 64, BF16, seed=2), scale=0.0)


@pytest.mark.parametrize("width", [4, 64, 2000])
def test_paged_attention_ignores_what_is_masked(width):
    """NaN and infinities behind a row's length, in blocks of nobody and behind
    invalid table entries do not reach the outputs."""
    case = attend_case([33, 1, 64, 0, 50], 6, 2, 64, BF16, block=16, width=width, seed=3)
    case["block_table"][4, 1] = -1
    case["block_table"][4, 2] = case["key_cache"].shape[0]
    clean = check_attend(case)
    used = torch.zeros(case["key_cache"].shape[:2], dtype=torch.bool, device="cuda")
    for r, n in enumerate([33, 1, 64, 0, 50]):
        for t in range(n):
            page = int(case["block_table"][r, t // 16])
            if 0 <= page < used.shape[0]:
                used[page, t % 16] = True
    for bad in (float("nan"), float("inf"), -float("inf")):
        case["key_cache"][~used] = bad
        case["value_cache"][~used] = bad
        from cruise_b200.decoder_ops import paged_attention

        assert torch.equal(paged_attention(*case.values()), clean)


@pytest.mark.parametrize("width", [2, 80, 2000])
def test_paged_attention_no_valid_block(width):
    case = attend_case([20, 30], 4, 2, 128, BF16, block=16, width=width, seed=4)
    case["block_table"][1] = -1
    out = check_attend(case)
    assert not out[1].any()


@pytest.mark.parametrize("width", [4, 64, 2000])
def test_paged_attention_propagates_what_is_attended(width):
    from cruise_b200.decoder_ops import paged_attention

    case = attend_case([40, 40, 40], 4, 2, 64, BF16, block=16, width=width, seed=5)
    at = case["block_table"][:, 1]
    case["key_cache"][at[0], 3, 0, 0] = float("nan")      # KV head 0 of row 0: heads 0 and 1
    case["value_cache"][at[1], 3, 1, 7] = float("inf")    # dimension 7 of heads 2 and 3 of row 1
    out = paged_attention(*case.values())
    assert torch.isnan(out[0, :2]).all() and torch.isfinite(out[0, 2:]).all()
    assert (out[1, 2:, 7] == math.inf).all() and torch.isfinite(out[1, :2]).all() and torch.isfinite(out[2]).all()


def test_paged_attention_length_past_the_table():
    case = attend_case([48, 20], 4, 2, 64, BF16, block=16, seed=6)
    want = check_attend(case)
    from cruise_b200.decoder_ops import paged_attention

    case["seq_len"] = torch.tensor([2 ** 31 - 1, 20], dtype=torch.int32, device="cuda")
    assert torch.equal(paged_attention(*case.values()), want)
    case["seq_len"] = torch.tensor([48, -3], dtype=torch.int32, device="cuda")
    out = paged_attention(*case.values())
    assert torch.equal(out[0], want[0]) and not out[1].any()


def test_paged_attention_strides():
    """Queries inside a qkv row, blocks of a cache that holds K and V together,
    a table inside a wider one, outputs inside a wider row."""
    case = attend_case([700, 33, 0, 128], 6, 2, 64, FP16, block=16, seed=7)
    qkv = torch.full((4, 10, 64), float("nan"), dtype=FP16, device="cuda")
    qkv[:, :6] = case["q"]
    both = torch.stack((case["key_cache"], case["value_cache"]), dim=1)
    wide = torch.full((4, case["block_table"].shape[1] + 5), 1 << 30, dtype=torch.int32, device="cuda")
    wide[:, 2:-3] = case["block_table"]
    room = torch.zeros(4, 8, 64, dtype=FP16, device="cuda")
    case.update(q=qkv[:, :6], key_cache=both[:, 0], value_cache=both[:, 1], block_table=wide[:, 2:-3])
    check_attend(case, out=room[:, 1:7])
    assert not room[:, 0].any() and not room[:, 7].any()


def test_paged_attention_past_32_bits():
    blocks, block, nkv, d = 8200, 512, 4, 128
    g = gen(8)
    key = torch.zeros(blocks, block, nkv, d, dtype=BF16, device="cuda")
    value = torch.zeros(blocks, block, nkv, d, dtype=BF16, device="cuda")
    table = torch.tensor([[blocks - 1, 0, 8192, 8191]], dtype=torch.int32, device="cuda")
    for page in table[0].tolist():
        key[page] = randn(g, block, nkv, d, dtype=BF16)
        value[page] = randn(g, block, nkv, d, dtype=BF16)
    check_attend(dict(q=randn(g, 1, 8, d, dtype=BF16), key_cache=key, value_cache=value, block_table=table,
                      seq_len=torch.tensor([2000], dtype=torch.int32, device="cuda")))


def test_paged_attention_lse_joins_parts():
    """Outputs over a row's halves, weighted by exp(lse), are the output over the row."""
    from cruise_b200.decoder_ops import paged_attention

    case = attend_case([640], 4, 2, 64, BF16, block=16, seed=9)
    lse = [torch.empty(1, 4, device="cuda") for _ in range(2)]
    parts = [paged_attention(case["q"], case["key_cache"], case["value_cache"], case["block_table"][:, 20 * i:20 * i + 20].contiguous(),
                             torch.tensor([320], dtype=torch.int32, device="cuda"), lse=lse[i]) for i in range(2)]
    weight = torch.softmax(torch.stack(lse).double(), dim=0)[..., None]
    want, _, bound, lse_bound = attention_reference(*case.values())
    joined = sum(w * p.double() for w, p in zip(weight, parts))
    # each half is off by its own bound and its rounding, its weight by its lse's error
    assert float(((joined - want).abs() - (3 * bound + 2 * lse_bound[..., None] + 2.0 ** -8 * want.abs().amax())).max()) <= 0


@pytest.mark.parametrize("width", [1, 4, 40])
def test_paged_attention_of_very_many_rows(width):
    """More rows than a grid's second dimension, sharing a few blocks (40 blocks of
    16 a row: split over all CTAs)."""
    from cruise_b200.decoder_ops import paged_attention

    g = gen(12)
    rows = 140001
    key, value = (randn(g, 9, 16, 1, 64, dtype=BF16) for _ in range(2))
    table = torch.randint(-1, 10, (rows, width), device="cuda", dtype=torch.int32, generator=g)
    lens = torch.randint(0, 33, (rows,), device="cuda", dtype=torch.int32, generator=g)
    q = randn(g, rows, 2, 64, dtype=BF16)
    out = paged_attention(q, key, value, table, lens)
    some = torch.cat([torch.arange(40), torch.arange(65520, 65560), torch.arange(131060, 131080), torch.arange(rows - 40, rows)]).cuda()
    want, _, bound, _ = attention_reference(q[some], key, value, table[some], lens[some])
    within(out[some], want, bound, "out")


def test_paged_attention_without_rows_or_columns():
    from cruise_b200.decoder_ops import paged_attention

    case = attend_case([3, 4], 4, 2, 64, BF16, seed=10)
    none = {**case, "q": case["q"][:0], "block_table": case["block_table"][:0], "seq_len": case["seq_len"][:0]}
    assert paged_attention(*none.values()).shape == (0, 4, 64)
    flat = {**case, "block_table": case["block_table"][:, :0]}
    assert not paged_attention(*flat.values()).any()


# ---- choose --------------------------------------------------------------------------

def choose_case(rows, vocab, dtype, *, cap=40, bias=5, mask=True, penal=True, seed=0, pad=0):
    g = gen(seed)
    logits = torch.full((rows, vocab + pad), float("nan"), dtype=dtype, device="cuda")
    logits[:, :vocab] = randn(g, rows, vocab, dtype=dtype) * 3
    case = dict(logits=logits[:, :vocab])
    if penal:
        small = torch.randint(0, vocab, (rows, 8), device="cuda", generator=g)
        case["history"] = small.gather(1, torch.randint(0, 8, (rows, cap), device="cuda", generator=g)).int()
        case["history"][:, ::5] = torch.randint(-3, vocab + 3, case["history"][:, ::5].shape, device="cuda", generator=g).int()
        case["history_len"] = torch.randint(0, cap, (rows,), device="cuda", generator=g).int()
        case["prompt_len"] = (case["history_len"] // 3).int()
        case["repetition"] = 0.7 + torch.rand(rows, device="cuda", generator=g)
        case["frequency"] = torch.rand(rows, device="cuda", generator=g) - 0.2
        case["presence"] = torch.rand(rows, device="cuda", generator=g) - 0.2
    if bias:
        n = min(bias, vocab)
        case["bias_token"] = torch.stack([torch.randperm(vocab, device="cuda", generator=g)[:n].sort().values
                                          for _ in range(rows)]).int()
        case["bias_value"] = randn(g, rows, n) * 4
        case["bias_len"] = torch.randint(0, n + 1, (rows,), device="cuda", generator=g).int()
    if mask:
        case["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), device="cuda", generator=g).int()
    return case


def check_choose(case, *, append=True, processed=True, out=None):
    from cruise_b200.decoder_ops import choose

    case = dict(case)
    reference = {k: v for k, v in case.items() if k != "logits"}
    x32, token32 = choose_reference(case["logits"], **reference, dtype=FP32)
    x64, _ = choose_reference(case["logits"], **reference)
    before = case["history"].clone() if "history" in case else None
    room = torch.full_like(x32, 3.0) if processed else None
    append = append and before is not None
    token = choose(**case, processed=room, append=append, out=out)
    assert torch.equal(token, token32)
    rows = range(len(token)) if case.get("active") is None else case["active"].nonzero()[:, 0].tolist()
    if processed:
        for r in range(len(token)):
            if r in rows:
                same = (room[r] == x32[r]) | (torch.isnan(room[r]) & torch.isnan(x32[r]))
                assert same.all(), f"row {r}: {int((~same).sum())} processed logits differ"
            else:
                assert (room[r] == 3.0).all()
        # against 64 bits: the bias' sum, the repetition's factor, and the frequency's product and
        # difference and the presence's difference are five roundings of values under `size`
        live = torch.tensor(list(rows), device="cuda", dtype=torch.long)
        a, b = room[live].double(), x64[live]
        fine = torch.isfinite(b)
        assert torch.equal(torch.isfinite(a), fine)
        size = 0.0 + b[fine].abs()
        size += 12.0 * 2 + 2 * case["history"].shape[1] if before is not None else 12.0
        assert float(((a[fine] - b[fine]).abs() - 5 * U32 * 2 * size).max()) <= 0 if fine.any() else True
    if before is not None:
        if append:
            for r in rows:
                end = int(case["history_len"][r])
                if token[r] >= 0 and 0 <= end < before.shape[1]:
                    before[r, end] = token[r]
        assert torch.equal(case["history"], before)
    return token


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("rows, vocab, pad", [
    (1, 1, 0), (3, 2, 1), (2, 31, 0), (5, 33, 0), (4, 500, 3), (1, 4096, 0), (7, 4099, 0), (300, 1001, 0),
    (4, 50257, 0), (2, 152064, 7), (1, 300000, 0), (2, 1000003, 0),
])
def test_choose(rows, vocab, pad, dtype):
    check_choose(choose_case(rows, vocab, dtype, seed=rows + vocab, pad=pad))


@pytest.mark.parametrize("penal, bias, mask", [(False, 0, False), (True, 0, False), (False, 3, False), (False, 0, True)])
def test_choose_single_rules(penal, bias, mask):
    case = choose_case(6, 5003, FP32, penal=penal, bias=bias, mask=mask, seed=11)
    check_choose(case)
    check_choose(case, processed=False, append=False)


def test_choose_neutral_penalties_leave_the_logits():
    from cruise_b200.decoder_ops import choose

    case = choose_case(3, 700, BF16, bias=0, mask=False, seed=12)
    case.update(repetition=torch.ones(3, device="cuda"), frequency=torch.zeros(3, device="cuda"), presence=None)
    room = torch.empty(3, 700, device="cuda")
    choose(**case, processed=room)
    assert torch.equal(room, case["logits"].float())


def test_choose_ties_take_the_lowest_token():
    logits = torch.zeros(3, 20011, device="cuda")
    logits[0, [19999, 7001, 12345]] = 2.0
    logits[2] = -0.0
    logits[2, 9000] = 0.0
    token = check_choose(dict(logits=logits))
    assert token.tolist() == [7001, 0, 0]


def test_choose_rows_without_a_choice():
    logits = randn(gen(13), 7, 3001)
    allowed = torch.full((7, 94), -1, dtype=torch.int32, device="cuda")
    allowed[0] = 0                                   # nothing allowed
    logits[1, 5] = float("nan")
    logits[2, 2999] = float("inf")
    logits[3] = -float("inf")                        # masked by the caller
    logits[4, 100] = float("nan")
    logits[4, 101] = float("inf")
    allowed[4, 3] &= ~((1 << 4) | (1 << 5))          # tokens 100 and 101 masked: their values do not matter
    logits[5] = torch.finfo(torch.float32).min       # a mask of the type's lowest value is still a value
    allowed[6] = 0
    allowed[6, 93] = 1 << 24                         # token 3000 alone, the last bit that counts
    token = check_choose(dict(logits=logits, allowed=allowed))
    assert token.tolist()[:4] == [-1, -2, -2, -1] and token[4] >= 0 and token.tolist()[5:] == [0, 3000]


def test_choose_bits_past_the_vocabulary_do_not_count():
    logits = randn(gen(14), 1, 40)
    allowed = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    allowed[0, 1] = -256                             # bits 40 to 63 only
    assert check_choose(dict(logits=logits, allowed=allowed)).tolist() == [-1]


def test_choose_infinite_bias():
    case = choose_case(2, 100, FP32, penal=False, mask=False, bias=2, seed=15)
    case["bias_token"] = torch.tensor([[3, 60], [3, 60]], dtype=torch.int32, device="cuda")
    case["bias_value"] = torch.tensor([[-math.inf, 50.0], [math.inf, 0.0]], device="cuda")
    case["bias_len"] = torch.tensor([2, 2], dtype=torch.int32, device="cuda")
    assert check_choose(case).tolist() == [60, -2]


def test_choose_inactive_rows_are_left_alone():
    case = choose_case(5, 2000, FP32, seed=16)
    case["active"] = torch.tensor([1, 0, 1, 0, 7], dtype=torch.int32, device="cuda")
    token = check_choose(case)
    assert token[1] == -1 and token[3] == -1


def test_choose_history_edges():
    """Full, empty and negative lengths, a prompt longer than the history, one
    token all over the history."""
    case = choose_case(6, 777, FP32, cap=9, bias=0, mask=False, seed=17)
    case["history"][3] = 5
    case["history_len"] = torch.tensor([9, 0, -4, 8, 20, 8], dtype=torch.int32, device="cuda")
    case["prompt_len"] = torch.tensor([3, 0, 0, 0, 2, 100], dtype=torch.int32, device="cuda")
    check_choose(case)


def test_choose_in_place():
    from cruise_b200.decoder_ops import choose

    case = choose_case(3, 5001, FP32, seed=18)
    x32, token32 = choose_reference(**case, dtype=FP32)
    assert torch.equal(choose(**case, processed=case["logits"]), token32)
    assert torch.equal(case["logits"], x32)


def test_choose_long_history():
    case = choose_case(2, 3000, FP32, cap=70000, bias=0, mask=False, seed=19)
    case["history"][0] = 17
    case["history_len"] = torch.tensor([69999, 65537], dtype=torch.int32, device="cuda")
    case["prompt_len"] = torch.tensor([100, 5], dtype=torch.int32, device="cuda")
    check_choose(case)


def test_choose_without_rows():
    from cruise_b200.decoder_ops import choose

    assert choose(torch.empty(0, 10, device="cuda")).shape == (0,)


# ---- refusals of the Python calls ------------------------------------------------------

def test_python_refusals():
    from cruise_b200.decoder_ops import choose, paged_attention, rotate_store

    case = attend_case([20, 3], 4, 2, 64, BF16, seed=20)

    def refused(match, call, **change):
        with pytest.raises(ValueError, match=match):
            call(**change)

    def attend(**change):
        paged_attention(**{**case, **change})

    refused("multiple of 2", attend, q=case["q"][:, :3])
    refused("must be torch.bfloat16", attend, q=case["q"].half())
    refused("next to one another", attend, q=case["q"].transpose(0, 1).contiguous().transpose(0, 1))
    refused("one shape", attend, value_cache=case["value_cache"][:-1])
    refused("contiguous", attend, key_cache=case["key_cache"].transpose(1, 2).contiguous().transpose(1, 2))
    refused("int32", attend, block_table=case["block_table"].long())
    refused("seq_len", attend, seq_len=case["seq_len"][:1])
    refused("lse", attend, lse=torch.empty(2, 3, device="cuda"))
    refused("on cuda", attend, block_table=case["block_table"].cpu())
    refused("overlap", attend, out=case["q"])
    refused("inference", attend, q=case["q"].float().to(BF16).requires_grad_())
    with torch.no_grad():
        attend(q=case["q"].clone().requires_grad_())
    refused("finite", attend, scale=math.nan)

    case2, keep = rotate_case(4, 4, 2, 64, BF16)

    def rotate(**change):
        rotate_store(**{**case2, **keep, **change})

    refused("qkv must be", rotate, num_heads=3)
    refused("both norm", rotate, q_norm=torch.ones(64, dtype=BF16, device="cuda"))
    refused("q_norm", rotate, q_norm=torch.ones(64, device="cuda"), k_norm=torch.ones(64, device="cuda"))
    refused("position", rotate, position=case2["position"].int())
    refused("slot", rotate, slot=case2["slot"].long())
    refused("cos and sin", rotate, cos=case2["cos"].half(), sin=case2["sin"].half())
    refused("one type", rotate, qkv=case2["qkv"].half())
    refused("multiple of 16", rotate, cos=case2["cos"][:, :24].contiguous(), sin=case2["sin"][:, :24].contiguous())
    odd = torch.empty(4 * 516, dtype=BF16, device="cuda").as_strided((4, 512), (516, 1))
    refused("multiples of 8", rotate, qkv=odd)

    case3 = choose_case(2, 100, FP32)

    def pick(**change):
        choose(**{**case3, **change})

    refused("need", pick, prompt_len=None)
    refused("need a history", pick, history=None, prompt_len=None, history_len=None)
    refused("bias_len", pick, bias_len=None)
    refused("allowed", pick, allowed=case3["allowed"][:, :3])
    refused("logits", pick, logits=case3["logits"].double())
    refused("processed", pick, processed=torch.empty(2, 100, dtype=BF16, device="cuda"))
    refused("out", pick, out=torch.empty(2, dtype=torch.int32, device="cuda"))
    refused("history", pick, history=case3["history"].long())


# ---- streams, graphs, threads -----------------------------------------------------------

def test_calls_follow_the_current_stream():
    from cruise_b200.decoder_ops import paged_attention

    case = attend_case([3000, 800], 8, 2, 64, BF16, seed=21)
    want = paged_attention(*case.values())
    late = torch.zeros_like(case["q"])
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        late.copy_(case["q"])          # the call has to wait for this on its stream
        got = paged_attention(late, *list(case.values())[1:])
    stream.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("width", [None, 2000])
def test_overlapping_calls_do_not_meet(width):
    """Two streams and two threads at once: each call has its own workspace."""
    import threading

    from cruise_b200.decoder_ops import paged_attention

    cases = [attend_case([9000 - 37 * i], 8, 2, 64, BF16, width=width, seed=22 + i) for i in range(4)]
    wants = [paged_attention(*c.values()) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(50):
                got = paged_attention(*cases[i].values())
                stream.synchronize()
                if not torch.equal(got, wants[i]):
                    bad.append(i)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_captured_attention_follows_its_inputs():
    """A captured call reads lengths, table and queries at replay; two graphs
    that replay at once on two streams do not share a workspace."""
    from cruise_b200.decoder_ops import paged_attention

    cases = [attend_case([2000, 17, 900], 8, 2, 64, BF16, width=2000, seed=30 + i) for i in range(2)]
    outs = [torch.empty_like(c["q"]) for c in cases]
    graphs = []
    for case, out in zip(cases, outs):
        paged_attention(*case.values(), out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged_attention(*case.values(), out=out)
        graphs.append(graph)
    for case in cases:
        case["seq_len"].copy_(torch.tensor([700, 0, 900]))
        case["q"].mul_(-1)
    wants = [paged_attention(*c.values()) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for out in outs:
            out.fill_(9)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, wants):
            assert torch.equal(out, want)


FIRST_CALLS = """
import torch
from cruise_b200.decoder_ops import choose, paged_attention

def captured_first(call, out):
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    graph.replay()
    torch.cuda.synchronize()
    got = out.clone()
    call()
    torch.cuda.synchronize()
    assert torch.equal(got, out)

cuda = dict(device="cuda")
key, value = (torch.randn(32, 16, 2, 64, **cuda).bfloat16() for _ in range(2))
for rows, width in ((2, 100), (2, 3000), (200, 20), (2, 1)):
    q = torch.randn(rows, 8, 64, **cuda).bfloat16()
    table = torch.randint(0, 32, (rows, width), dtype=torch.int32, **cuda)
    lens = torch.full((rows,), width * 16 - 5, dtype=torch.int32, **cuda)
    out = torch.empty_like(q)
    captured_first(lambda: paged_attention(q, key, value, table, lens, out=out), out)
logits, token = torch.randn(3, 50000, **cuda), torch.empty(3, dtype=torch.int64, **cuda)
captured_first(lambda: choose(logits, out=token), token)
assert torch.equal(token, logits.argmax(dim=1))
print("the same")
"""


def test_first_calls_may_be_captured():
    """In a fresh process: the first call of each form of attention and of choose
    inside a capture, where the library asks the device for its limits."""
    import pathlib
    import subprocess
    import sys

    root = pathlib.Path(__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "the same" in done.stdout, done.stderr[-2000:]


def test_captured_calls_behind_copies_memsets_and_joins():
    """Captured behind a memset, a copy and a join of two streams, each call
    still waits for what it reads."""
    from cruise_b200.decoder_ops import choose, paged_attention, rotate_store

    case = attend_case([700, 90], 8, 2, 64, BF16, seed=33)
    rot, keep = rotate_case(40, 4, 2, 64, BF16, seed=34)
    pick = dict(logits=randn(gen(35), 3, 5000))
    source = {name: t.clone() for name, t in (("q", case["q"]), ("qkv", rot["qkv"]), ("logits", pick["logits"]))}
    out = [torch.empty_like(case["q"]), torch.empty(40, 4, 64, dtype=BF16, device="cuda"), torch.empty(3, dtype=torch.int64, device="cuda")]

    def body(side):
        case["q"].zero_()
        paged_attention(*case.values(), out=out[0])            # behind a memset: uniform weights
        case["q"].copy_(source["q"])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            rot["qkv"].copy_(source["qkv"])
            rotate_store(*rot.values(), **keep, out=out[1])    # behind a copy, on another stream
            pick["logits"].copy_(source["logits"])
        torch.cuda.current_stream().wait_stream(side)
        choose(**pick, out=out[2])                             # behind a join
        paged_attention(*case.values(), out=out[0])

    side = torch.cuda.Stream()
    body(side)
    torch.cuda.synchronize()
    want = [t.clone() for t in out]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        body(side)
    for _ in range(5):
        for t in (*out, case["q"], rot["qkv"]):
            t.fill_(1)
        pick["logits"].fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for got, wanted in zip(out, want):
            assert torch.equal(got, wanted)


@pytest.mark.parametrize("width", [80, 2000])
def test_calls_one_after_another_wait_for_each_other(width):
    """A chain of calls that each read what the one before wrote, without a pause."""
    from cruise_b200.decoder_ops import paged_attention

    case = attend_case([900, 33, 128], 4, 2, 64, FP16, width=width, seed=36)
    slow = case["q"].clone()
    for _ in range(30):
        slow = paged_attention(slow, *list(case.values())[1:])
        torch.cuda.synchronize()
    fast = case["q"].clone()
    for _ in range(30):
        fast = paged_attention(fast, *list(case.values())[1:])
    assert torch.equal(fast, slow)


# ---- a run of the three, as a decode loop uses them ----------------------------------------

class DecodeLoop:
    """One attention layer between an embedding and a vocabulary projection:
    qkv = x W, rotate_store, paged_attention, logits = o U, choose."""

    def __init__(self, rows, vocab, nq, nkv, d, block, width, seed):
        g = gen(seed)
        self.nq = nq
        self.embed = randn(g, vocab, 64) / 2
        self.w = randn(g, 64, (nq + 2 * nkv) * d) / 8
        self.head = randn(g, nq * d, vocab) / 4
        self.cos, self.sin = rope(block * width, d, FP32)
        self.norm = [1 + randn(g, d, dtype=BF16) / 8 for _ in range(2)]
        order = torch.randperm(rows * width, device="cuda", generator=g).int()
        self.table = order.view(rows, width)
        self.key = torch.zeros(rows * width, block, nkv, d, dtype=BF16, device="cuda")
        self.value = torch.zeros_like(self.key)
        self.token = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
        self.position = torch.zeros(rows, dtype=torch.int64, device="cuda")
        self.history = torch.zeros(rows, block * width, dtype=torch.int32, device="cuda")
        self.history[:, 0] = self.token
        self.length = torch.ones(rows, dtype=torch.int32, device="cuda")
        self.prompt = torch.ones(rows, dtype=torch.int32, device="cuda")
        self.rules = dict(repetition=torch.full((rows,), 1.3, device="cuda"),
                          frequency=torch.full((rows,), 0.2, device="cuda"),
                          presence=torch.full((rows,), 0.1, device="cuda"),
                          allowed=torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), device="cuda", generator=g).int())
        self.rows = torch.arange(rows, device="cuda")
        self.block = block

    def step(self):
        from cruise_b200.decoder_ops import choose, paged_attention, rotate_store

        qkv = (self.embed[self.token] @ self.w).to(BF16)
        page = self.position // self.block
        slot = (self.table[self.rows, page].long() * self.block + self.position % self.block).int()
        q = rotate_store(qkv, self.position, slot, self.cos, self.sin, self.key, self.value, num_heads=self.nq,
                         q_norm=self.norm[0], k_norm=self.norm[1])
        out = paged_attention(q, self.key, self.value, self.table, (self.position + 1).int())
        logits = out.flatten(1).float() @ self.head
        choose(logits, history=self.history, prompt_len=self.prompt, history_len=self.length, **self.rules,
               append=True, out=self.token)
        self.position.add_(1)
        self.length.add_(1)
        return qkv, slot, q, out, logits


def test_decode_loop_of_the_three():
    loop = DecodeLoop(3, 3001, 6, 2, 64, 16, 40, seed=40)
    for i in range(20):
        history = loop.history.clone()
        length = loop.length.clone()
        qkv, slot, q, out, logits = loop.step()
        position = loop.position - 1
        z, bound, v = rotate_reference(qkv, position, loop.cos, loop.sin, 6, 2, 64, *loop.norm)
        within(q, z[:, :6], bound[:, :6], f"step {i}: q")
        within(loop.key.view(-1, 2, 64)[slot.long()], z[:, 6:], bound[:, 6:], f"step {i}: k")
        assert torch.equal(loop.value.view(-1, 2, 64)[slot.long()].double(), v)
        want, _, out_bound, _ = attention_reference(q, loop.key, loop.value, loop.table, loop.position)
        within(out, want, out_bound, f"step {i}: out")
        _, token = choose_reference(logits, history, loop.prompt, length, **loop.rules, dtype=FP32)
        assert torch.equal(loop.token, token) and (token >= 0).all()
        assert torch.equal(loop.history[loop.rows, length.long()].long(), token)


def test_captured_decode_loop_equals_the_eager_one():
    eager, captured = (DecodeLoop(3, 3001, 6, 2, 64, 16, 40, seed=41) for _ in range(2))
    for loop in (eager, captured):
        for _ in range(3):
            loop.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step()
    for _ in range(200):
        eager.step()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured.history, eager.history) and torch.equal(captured.position, eager.position)
    assert torch.equal(captured.key, eager.key) and torch.equal(captured.value, eager.value)
