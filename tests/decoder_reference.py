"""The decoder operators' definitions in 64 bits, with a bound on what the
kernels' arithmetic may differ by, element for element.

u(t) = finfo(t).eps / 2 is half a step of t relative to the value: one rounding.
"""

from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24


def unit(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def floor(dtype: torch.dtype) -> float:
    """Half the smallest step: what a rounding loses at the bottom of the range."""
    info = torch.finfo(dtype)
    return info.tiny * info.eps / 2


def rotate_reference(qkv, position, cos, sin, nq, nkv, d, q_norm=None, k_norm=None, eps=1e-6):
    """(q and k heads [T, nq + nkv, d] after norm and rotation, their bound, v heads).

    Bound: the stored rounding u |z|, and before it the fp32 operations: the
    mean of d squares (at most 8 + log2 16 = 12 additions in a chain, d products),
    its reciprocal root (2 steps), two products with the vector and the weight,
    two products and a sum of the rotation: under 32 roundings in all, each
    relative 2^-24 to |y_i cos_i| + |y_j sin_j|."""
    x = qkv.double().reshape(qkv.shape[0], nq + 2 * nkv, d)
    y = x[:, : nq + nkv].clone()
    if q_norm is not None:
        y[:, :nq] *= q_norm.double() / (y[:, :nq].pow(2).mean(-1, keepdim=True) + eps).sqrt()
        y[:, nq:] *= k_norm.double() / (y[:, nq:].pow(2).mean(-1, keepdim=True) + eps).sqrt()
    rot = cos.shape[1]
    known = (position >= 0) & (position < cos.shape[0])
    at = torch.where(known, position, 0)
    c, s = cos.double()[at][:, None], sin.double()[at][:, None]
    h = rot // 2
    turned = torch.cat((-y[..., h:rot], y[..., :h]), dim=-1)
    z = torch.cat((y[..., :rot] * c + turned * s, y[..., rot:]), dim=-1)
    size = torch.cat(((y[..., :rot] * c).abs() + (turned * s).abs(), y[..., rot:].abs()), dim=-1)
    before = 32 * U32 * size
    bound = unit(qkv.dtype) * (z.abs() + before) + before + floor(qkv.dtype)
    z = torch.where(known[:, None, None], z, 0.0)
    return z, bound, x[:, nq + nkv:]


def attention_reference(q, key, value, table, lens, scale=None):
    """(out, lse, bound of out, bound of lse) in 64 bits, row by row.

    Bounds per row and head, with p the softmax and n positions: a score's fp32
    error is at most ds = (d + 8) 2^-23 scale sum |q||k| (d products and sums, the
    scale, log2 e); p moves by a factor e^(2 ds); it is rounded to the cache's
    type (u, at least its floor); the fp32 sums of n products add (n + 64) 2^-23;
    the quotient is rounded to the output's type."""
    rows, nq, d = q.shape
    block, nkv = key.shape[1], key.shape[2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    group, u = nq // nkv, unit(q.dtype)
    out = torch.zeros(rows, nq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((rows, nq), -math.inf, dtype=torch.float64, device=q.device)
    out_bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)
    capacity = table.shape[1] * block
    for r, n in enumerate(lens.tolist()):
        n = max(0, min(n, capacity))
        if n == 0:
            continue
        t = torch.arange(n, device=q.device)
        pages = table[r].long()[t // block]
        live = (pages >= 0) & (pages < key.shape[0])
        pages, t = pages[live], t[live]
        if pages.numel() == 0:
            continue
        k, v = key[pages, t % block].double(), value[pages, t % block].double()
        for h in range(nkv):
            heads = slice(h * group, (h + 1) * group)
            qh = q[r, heads].double()
            scores = scale * qh @ k[:, h].T
            ds = (d + 8) * 2 * U32 * abs(scale) * (qh.abs() @ k[:, h].abs().T).amax(1, keepdim=True)
            p = torch.softmax(scores, dim=1)
            out[r, heads] = p @ v[:, h]
            lse[r, heads] = torch.logsumexp(scores, dim=1)
            weight = p @ v[:, h].abs()
            sums = (pages.numel() + 64) * 2 * U32
            err = weight * (u + sums + torch.expm1(2 * ds)) + pages.numel() * floor(q.dtype) * v[:, h].abs().amax()
            out_bound[r, heads] = err + u * (out[r, heads].abs() + err) + floor(q.dtype)
            lse_bound[r, heads] = ds[:, 0] + sums + 4 * U32 * lse[r, heads].abs()
    return out, lse, out_bound, lse_bound


def choose_reference(logits, history=None, prompt_len=None, history_len=None, repetition=None, frequency=None,
                     presence=None, bias_token=None, bias_value=None, bias_len=None, allowed=None, active=None,
                     dtype=torch.float64):
    """(processed logits, token) row by row in ``dtype``: in fp32 every step is
    the kernel's own rounded operation, so both agree bit for bit."""
    x = logits.to(dtype).clone()
    rows, vocab = x.shape
    token = torch.full((rows,), -1, dtype=torch.int64, device=x.device)
    for r in range(rows):
        if bias_token is not None:
            for t, b in zip(bias_token[r, : bias_len[r]].tolist(), bias_value[r, : bias_len[r]]):
                if 0 <= t < vocab:
                    x[r, t] += b.to(dtype)
        if history is not None:
            n, p = int(history_len[r]), int(prompt_len[r])
            n = max(0, min(n, history.shape[1]))
            p = max(0, min(p, n))
            ids = history[r, :n].long()
            inside = (ids >= 0) & (ids < vocab)
            count = torch.bincount(ids[p:][inside[p:]], minlength=vocab)
            seen = torch.bincount(ids[inside], minlength=vocab) > 0
            one = lambda v, neutral: (torch.tensor(neutral) if v is None else v[r]).to(x.device, dtype)  # noqa: E731
            rep, freq, pres = one(repetition, 1.0), one(frequency, 0.0), one(presence, 0.0)
            x[r] = torch.where(seen, torch.where(x[r] > 0, x[r] / rep, x[r] * rep), x[r])
            x[r] = torch.where(count > 0, x[r] - freq * count.to(dtype), x[r])
            x[r] = torch.where(count > 0, x[r] - pres, x[r])
        if allowed is not None:
            ids = torch.arange(vocab, device=x.device)
            x[r] = torch.where(((allowed[r, ids >> 5] >> (ids & 31)) & 1) != 0, x[r], -math.inf)
        if active is not None and int(active[r]) == 0:
            continue
        if bool((torch.isnan(x[r]) | (x[r] == math.inf)).any()):
            token[r] = -2
        elif bool((x[r] > -math.inf).any()):
            token[r] = int((x[r] == x[r].max()).nonzero()[0])
    return x, token
