"""Measured passes through the decoder operators on device tensors: head norms with
rotation and the paged-cache write (``rotate_store``), attention of one new
token per row over the paged cache (``paged_attention``), and the logit rules
with the greedy choice (``choose``).

A case is a dict of plain values; ``prepare`` makes its inputs from a seed,
``run`` makes one pass: the plain torch form, or with ``own`` true the calls a
decode loop makes of :mod:`cruise_b200.decoder_ops`.  ``exact`` gives the same
outputs from the definitions in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # The resident cohort's shape: 4 rows inside 256 positions, one layer of
        # the 7B preset.  Microseconds of work: latency counts.
        dict(name="attend 4 rows x 256", op="attend", rows=4, nq=28, nkv=4, d=128, block=128, min_len=44, max_len=256,
             empty=0, dtype="bf16"),
        # One user with a long context: a single row must fill the GPU.
        dict(name="attend 1 row x 131071", op="attend", rows=1, nq=28, nkv=4, d=128, block=128, min_len=131071,
             max_len=131071, empty=0, dtype="bf16"),
        # A mixed server: small pages, lengths from a few tokens to thousands, padded rows.
        dict(name="attend 64 ragged rows, pages of 16", op="attend", rows=64, nq=32, nkv=8, d=64, block=16, min_len=1,
             max_len=16384, empty=3, dtype="fp16"),
        # The large batch: cache bandwidth.
        dict(name="attend 256 rows x 4096", op="attend", rows=256, nq=28, nkv=4, d=128, block=128, min_len=1500,
             max_len=4096, empty=0, dtype="bf16"),
        # One decode step's tokens, no head norms (the 7B preset's layers).
        dict(name="rotate 4 tokens", op="rotate", tokens=4, nq=28, nkv=4, d=128, rotary=128, block=128, norm=False,
             tables="bf16", capacity=256, dtype="bf16"),
        # A chunk of a prompt with an odd token count, small heads, head norms.
        dict(name="rotate 333 tokens, head norms", op="rotate", tokens=333, nq=9, nkv=3, d=64, rotary=64, block=16,
             norm=True, tables="fp32", capacity=4096, dtype="fp16"),
        # Many prompts' tokens at once: memory bandwidth.
        dict(name="rotate 8192 tokens, head norms", op="rotate", tokens=8192, nq=28, nkv=4, d=128, rotary=128,
             block=128, norm=True, tables="bf16", capacity=32768, dtype="bf16"),
        # The smallest vocabulary of the tests, one row, no rule but a penalty.
        dict(name="choose 1 row x 4096", op="choose", rows=1, vocab=4096, dtype="fp32", history=33, bias=0, mask=False,
             processed=False),
        # The resident cohort's logits with a history of one row capacity.
        dict(name="choose 4 rows x 152064", op="choose", rows=4, vocab=152064, dtype="fp32", history=256, bias=16,
             mask=False, processed=False),
        # Structured output: half-precision logits, an odd vocabulary, a grammar mask.
        dict(name="choose 64 rows x 50257, grammar", op="choose", rows=64, vocab=50257, dtype="bf16", history=1000,
             bias=7, mask=True, processed=False),
        # A large batch whose processed logits feed a sampler: every rule, read and written.
        dict(name="choose 256 rows x 152064, all", op="choose", rows=256, vocab=152064, dtype="fp32", history=4096,
             bias=64, mask=True, processed=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(("attend", "attend", "rotate", "choose"))
    if op == "attend":
        nkv = rng.choice((1, 2, 4, 8))
        group = rng.choice((1, 2, 3, 4, 5, 6, 7, 8, 12, 16))
        d = rng.choice((64, 128))
        rows = _log_int(rng, 1, 256)
        # at most the largest listed case's cache bytes and products
        most = min(131072, 320_000_000 // (rows * nkv * d), 2_200_000_000 // (rows * nkv * group * d))
        max_len = _log_int(rng, 1, most)
        min_len = rng.choice((max_len, max(1, max_len // 2), 1))
        return dict(op=op, rows=rows, nq=nkv * group, nkv=nkv, d=d, block=rng.choice((16, 24, 32, 64, 128)),
                    min_len=min_len, max_len=max_len, empty=rng.choice((0, 0, min(2, rows - 1))),
                    dtype=rng.choice(("bf16", "fp16")))
    if op == "rotate":
        nkv = rng.choice((1, 2, 3, 4, 8))
        group = rng.choice((1, 2, 3, 4, 5, 7, 8))
        d = rng.choice((64, 128))
        return dict(op=op, tokens=_log_int(rng, 1, 8192), nq=nkv * group, nkv=nkv, d=d,
                    rotary=rng.choice((d, d, d // 2)), block=rng.choice((16, 24, 128)), norm=rng.choice((True, False)),
                    tables=rng.choice(("bf16", "fp32")), capacity=_log_int(rng, 16, 131072),
                    dtype=rng.choice(("bf16", "fp16")))
    vocab = _log_int(rng, 500, 152064)
    return dict(op=op, rows=_log_int(rng, 1, 256), vocab=vocab, dtype=rng.choice(("fp32", "bf16")),
                history=_log_int(rng, 1, 4096), bias=rng.choice((0, 1, 17, 64)), mask=rng.choice((True, False)),
                processed=rng.choice((True, False)))


def _lengths(case):
    """The case's lengths: spread geometrically from min_len to max_len, the last ``empty`` rows 0."""
    n = case["rows"] - case["empty"]
    lo, hi = case["min_len"], case["max_len"]
    lens = [int(round(lo * (hi / lo) ** (i / max(1, n - 1)))) if n > 1 else hi for i in range(n)]
    return lens + [0] * case["empty"]


def _rand(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = random.Random(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    s = {"op": op, "case": case}
    if op == "attend":
        rows, nkv, d, block = case["rows"], case["nkv"], case["d"], case["block"]
        lens = _lengths(case)
        host.shuffle(lens)
        per_row = -(-case["max_len"] // block)
        used = [-(-n // block) for n in lens]
        total = sum(used) + 3
        order = torch.randperm(total, device="cuda", generator=gen).to(torch.int32)
        # the row's blocks in allocation order, -1 past its last block
        first = torch.tensor([sum(used[:r]) for r in range(rows)], dtype=torch.int64, device="cuda")[:, None]
        count = torch.tensor(used, dtype=torch.int64, device="cuda")[:, None]
        column = torch.arange(per_row, device="cuda")[None, :]
        table = order[(first + column).clamp(max=total - 1)]
        s["table"] = torch.where(column < count, table, -1).contiguous()
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["key"] = torch.empty(total, block, nkv, d, dtype=dtype, device="cuda").normal_(generator=gen)
        s["value"] = torch.empty(total, block, nkv, d, dtype=dtype, device="cuda").normal_(generator=gen)
        s["q"] = (_rand(gen, rows, case["nq"], d) * 1.5).to(dtype)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(rows, case["nq"], dtype=torch.float32, device="cuda")
    elif op == "rotate":
        tokens, nq, nkv, d, rot = case["tokens"], case["nq"], case["nkv"], case["d"], case["rotary"]
        blocks = -(-tokens // case["block"]) + 2
        s["qkv"] = _rand(gen, tokens, (nq + 2 * nkv) * d).to(dtype)
        angles = torch.arange(case["capacity"], dtype=torch.float64, device="cuda")[:, None] * (
            1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot))[None, :]
        angles = torch.cat((angles, angles), dim=-1)
        s["cos"] = angles.cos().to(DTYPES[case["tables"]])
        s["sin"] = angles.sin().to(DTYPES[case["tables"]])
        s["position"] = torch.randint(0, case["capacity"], (tokens,), device="cuda", generator=gen)
        s["slot"] = torch.randperm(blocks * case["block"], device="cuda", generator=gen)[:tokens].to(torch.int32)
        s["key"] = _rand(gen, blocks, case["block"], nkv, d).to(dtype)
        s["value"] = _rand(gen, blocks, case["block"], nkv, d).to(dtype)
        s["wq"] = (1 + 0.1 * _rand(gen, d)).to(dtype) if case["norm"] else None
        s["wk"] = (1 + 0.1 * _rand(gen, d)).to(dtype) if case["norm"] else None
        s["out"] = torch.empty(tokens, nq, d, dtype=dtype, device="cuda")
    else:
        rows, vocab, cap = case["rows"], case["vocab"], case["history"] + 2
        s["logits"] = (_rand(gen, rows, vocab) * 3).to(dtype)
        # a running text: half of the history from a small set of repeated tokens
        common = torch.randint(0, vocab, (rows, 50), device="cuda", generator=gen)
        often = common.gather(1, torch.randint(0, 50, (rows, cap), device="cuda", generator=gen))
        rare = torch.randint(0, vocab, (rows, cap), device="cuda", generator=gen)
        coin = torch.rand(rows, cap, device="cuda", generator=gen) < 0.5
        s["history"] = torch.where(coin, often, rare).to(torch.int32)
        s["length"] = torch.randint((case["history"] + 1) // 2, case["history"] + 1, (rows,), device="cuda",
                                    generator=gen).to(torch.int32)
        s["prompt"] = (s["length"] // 3).to(torch.int32)
        s["repetition"] = 1.0 + 0.3 * torch.rand(rows, device="cuda", generator=gen)
        s["frequency"] = 0.5 * torch.rand(rows, device="cuda", generator=gen)
        s["presence"] = 0.5 * torch.rand(rows, device="cuda", generator=gen)
        s["bias_token"] = s["bias_value"] = s["bias_len"] = None
        if case["bias"]:
            nb = min(case["bias"], vocab)
            s["bias_token"] = torch.stack([torch.randperm(vocab, device="cuda", generator=gen)[:nb]
                                           for _ in range(rows)]).sort(dim=1).values.to(torch.int32)
            s["bias_value"] = _rand(gen, rows, nb) * 2
            s["bias_len"] = torch.randint(0, nb + 1, (rows,), device="cuda", generator=gen).to(torch.int32)
        s["allowed"] = None
        if case["mask"]:   # a grammar's bit mask: a few tokens to nearly all of them per row
            share = torch.rand(rows, 1, device="cuda", generator=gen)
            words = torch.zeros(rows, -(-vocab // 32), dtype=torch.int32, device="cuda")
            for bit in range(32):
                keep = torch.rand(words.shape, device="cuda", generator=gen) < share
                words |= torch.where(keep, torch.tensor(-(1 << 31) if bit == 31 else (1 << bit), dtype=torch.int32,
                                                        device="cuda"), 0)
            s["allowed"] = words
        s["token"] = torch.empty(rows, dtype=torch.int64, device="cuda")
        s["processed"] = (torch.empty(rows, vocab, dtype=torch.float32, device="cuda") if case["processed"] else None)
    return s


def run(s):
    if own:
        return _run_own(s)
    return {"attend": _plain_attend, "rotate": _plain_rotate, "choose": _plain_choose}[s["op"]](s)


def _run_own(s):
    from cruise_b200 import decoder_ops

    if s["op"] == "attend":
        decoder_ops.paged_attention(s["q"], s["key"], s["value"], s["table"], s["lens"], out=s["out"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if s["op"] == "rotate":
        decoder_ops.rotate_store(s["qkv"], s["position"], s["slot"], s["cos"], s["sin"], s["key"], s["value"],
                                 num_heads=s["case"]["nq"], q_norm=s["wq"], k_norm=s["wk"], eps=1e-6, out=s["out"])
        return {"q": s["out"], "key": s["key"], "value": s["value"]}
    decoder_ops.choose(s["logits"], history=s["history"], prompt_len=s["prompt"], history_len=s["length"],
                       repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                       bias_token=s["bias_token"], bias_value=s["bias_value"], bias_len=s["bias_len"],
                       allowed=s["allowed"], processed=s["processed"], out=s["token"], append=True)
    answer = {"token": s["token"], "history": s["history"]}
    if s["processed"] is not None:
        answer["processed"] = s["processed"]
    return answer


def _plain_attend(s):
    q, key, value, table, lens = s["q"], s["key"], s["value"], s["table"], s["lens"]
    rows, nq, d = q.shape
    block, nkv = key.shape[1], key.shape[2]
    t = torch.arange(s["case"]["max_len"], device=q.device)
    live = t[None, :] < lens[:, None]
    slot = torch.where(live, table.long()[:, t // block] * block + t % block, 0)
    k = key.view(-1, nkv, d)[slot].float().transpose(1, 2)      # [rows, nkv, t, d]
    v = value.view(-1, nkv, d)[slot].float().transpose(1, 2)
    qf = q.float().view(rows, nkv, nq // nkv, d)
    scores = torch.matmul(qf, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    scores = torch.where(live[:, None, None, :], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, v) / torch.where(total == 0, 1.0, total)
    lse = torch.log(total) + top
    return {"out": out.reshape(rows, nq, d).to(q.dtype), "lse": lse.reshape(rows, nq)}


def _plain_rotate(s):
    case = s["case"]
    nq, nkv, d, rot = case["nq"], case["nkv"], case["d"], case["rotary"]
    tokens = s["qkv"].shape[0]
    x = s["qkv"].view(tokens, nq + 2 * nkv, d)
    q, k, v = x[:, :nq].float(), x[:, nq:nq + nkv].float(), x[:, nq + nkv:]
    if s["wq"] is not None:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s["wq"].float()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * s["wk"].float()
    cos, sin = s["cos"][s["position"]].float()[:, None, :], s["sin"][s["position"]].float()[:, None, :]

    def rotate(y):
        turned, rest = y[..., :rot], y[..., rot:]
        half = torch.cat((-turned[..., rot // 2:], turned[..., :rot // 2]), dim=-1)
        return torch.cat((turned * cos + half * sin, rest), dim=-1).to(s["qkv"].dtype)

    slot = s["slot"].long()
    s["key"].view(-1, nkv, d)[slot] = rotate(k)
    s["value"].view(-1, nkv, d)[slot] = v
    return {"q": rotate(q), "key": s["key"], "value": s["value"]}


def _plain_choose(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    history = s["history"].long()
    at = torch.arange(history.shape[1], device=x.device)[None, :]
    in_prompt = at < s["prompt"][:, None]
    in_output = (at < s["length"][:, None]) & ~in_prompt
    # a spare last column takes what does not count
    ones = torch.ones_like(s["history"])
    prompt = torch.zeros(rows, vocab + 1, dtype=torch.int32, device=x.device).scatter_add_(
        1, torch.where(in_prompt, history, vocab), ones)[:, :vocab]
    count = torch.zeros(rows, vocab + 1, dtype=torch.int32, device=x.device).scatter_add_(
        1, torch.where(in_output, history, vocab), ones)[:, :vocab]
    if s["bias_token"] is not None:
        live = torch.arange(s["bias_token"].shape[1], device=x.device)[None, :] < s["bias_len"][:, None]
        x = x + torch.zeros(rows, vocab + 1, device=x.device).scatter_(
            1, torch.where(live, s["bias_token"].long(), vocab), s["bias_value"])[:, :vocab]
    seen = (prompt > 0) | (count > 0)
    repetition = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
    x = x - s["frequency"][:, None] * count
    x = x - s["presence"][:, None] * (count > 0)
    ids = torch.arange(vocab, device=x.device)
    if s["allowed"] is not None:
        x = torch.where(((s["allowed"][:, ids >> 5] >> (ids & 31)) & 1) != 0, x, -math.inf)
    broken = (torch.isnan(x) | (x == math.inf)).any(1)
    top = x.amax(1, keepdim=True)
    first = torch.where((x == top) & (x > -math.inf), ids, vocab).amin(1)
    token = torch.where(broken, -2, torch.where(first == vocab, -1, first))
    end = s["length"].long()[:, None]
    s["history"].scatter_(1, end, torch.where(token[:, None] >= 0, token[:, None], s["history"].gather(1, end).long())
                          .to(torch.int32))
    answer = {"token": token, "history": s["history"]}
    if s["processed"] is not None:
        answer["processed"] = x
    return answer


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        nq, nkv, d, block = case["nq"], case["nkv"], case["d"], case["block"]
        out = torch.zeros(case["rows"], nq, d, dtype=torch.float64, device="cuda")
        lse = torch.full((case["rows"], nq), -math.inf, dtype=torch.float64, device="cuda")
        for r, n in enumerate(s["lens"].tolist()):
            if n == 0:
                continue
            pages = s["table"][r, : -(-n // block)].long()
            k = s["key"][pages].reshape(-1, nkv, d)[:n].double()
            v = s["value"][pages].reshape(-1, nkv, d)[:n].double()
            for h in range(nkv):
                group = slice(h * nq // nkv, (h + 1) * nq // nkv)
                z = s["q"][r, group].double() @ k[:, h].T / math.sqrt(d)
                lse[r, group] = torch.logsumexp(z, dim=1)
                out[r, group] = torch.softmax(z, dim=1) @ v[:, h]
        return {"out": out, "lse": lse}
    if case["op"] == "rotate":
        nq, nkv, d, rot = case["nq"], case["nkv"], case["d"], case["rotary"]
        x = s["qkv"].double().reshape(-1, nq + 2 * nkv, d)
        y = x[:, : nq + nkv].clone()
        if case["norm"]:
            weight = torch.cat((s["wq"].double().expand(nq, d), s["wk"].double().expand(nkv, d)))
            y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / d + 1e-6) * weight
        c, z = s["cos"].double()[s["position"]], s["sin"].double()[s["position"]]
        h = rot // 2
        low, high = y[..., :h].clone(), y[..., h:rot].clone()
        y[..., :h] = low * c[:, None, :h] - high * z[:, None, :h]
        y[..., h:rot] = high * c[:, None, h:] + low * z[:, None, h:]
        key, value = s["key"].double(), s["value"].double()
        pages, inside = s["slot"].long() // case["block"], s["slot"].long() % case["block"]
        key[pages, inside] = y[:, nq:]
        value[pages, inside] = x[:, nq + nkv:]
        return {"q": y[:, :nq], "key": key, "value": value}
    if not case["processed"]:
        return None
    x = s["logits"].double()
    rows, vocab = x.shape
    length, prompt = s["length"].tolist(), s["prompt"].tolist()
    for r in range(rows):
        if s["bias_token"] is not None:
            n = int(s["bias_len"][r])
            x[r].index_add_(0, s["bias_token"][r, :n].long(), s["bias_value"][r, :n].double())
        output = torch.bincount(s["history"][r, prompt[r]:length[r]].long(), minlength=vocab).double()
        seen = torch.bincount(s["history"][r, :length[r]].long(), minlength=vocab) > 0
        rep = s["repetition"][r].double()
        x[r] = torch.where(seen, x[r] * torch.where(x[r] > 0, 1 / rep, rep), x[r])
        x[r] -= s["frequency"][r].double() * output + s["presence"][r].double() * output.clamp(max=1)
    if s["allowed"] is not None:
        for bit in range(32):
            column = torch.arange(bit, vocab, 32, device="cuda")
            gone = (s["allowed"][:, : column.numel()] >> bit) & 1 == 0
            x[:, column] = torch.where(gone, -math.inf, x[:, column])
    return {"token": None, "history": None, "processed": x}


def work(case):
    if case["op"] == "attend":
        tokens, width = sum(_lengths(case)), case["nkv"] * case["d"]
        vectors = case["rows"] * case["nq"] * (2 * case["d"] * 2 + 4)
        table = 4 * sum(-(-n // case["block"]) for n in _lengths(case)) + 4 * case["rows"]
        return {"bytes": tokens * width * 2 * 2 + vectors + table, "flops": 4.0 * tokens * case["nq"] * case["d"]}
    if case["op"] == "rotate":
        tokens, heads = case["tokens"], case["nq"] + 2 * case["nkv"]
        entry = 4 if case["tables"] == "fp32" else 2
        positions = min(tokens, case["capacity"])
        return {"bytes": tokens * heads * case["d"] * 2 * 2 + tokens * 12 + positions * case["rotary"] * 2 * entry,
                "flops": float(tokens * (case["nq"] + case["nkv"]) * case["d"] * (8 if case["norm"] else 4))}
    rows, vocab = case["rows"], case["vocab"]
    size = rows * vocab * (4 if case["dtype"] == "fp32" else 2)
    size += rows * (case["history"] * 3 // 4 * 4 + case["bias"] * 4 + 8 + 28)
    size += rows * vocab // 8 if case["mask"] else 0
    size += rows * vocab * 4 if case["processed"] else 0
    return {"bytes": size, "flops": 4.0 * rows * vocab}
