"""Plain 64-bit forms of the window, shared-prefix and beam operators, and the error bounds of the kernels.

Test infrastructure only: per-sequence loops over dense keys in float64 on whatever device the inputs are on.

Error bound of an attention output (``bound``).  With p the exact softmax weights over n visible keys, A =
sum p |v| and S = max over visible keys of sum_d |q_d k_d| / sqrt(D):

* a score is a sum of D products in 32 bits (at most one rounding per addition, taken as a whole step since the
  tensor cores may truncate): off by e_s <= (D + 4) 2^-23 S, which moves each weight by a factor e^(+-2 e_s)
  once numerator and denominator are counted;
* ex2.approx: 2^-22 relative on each weight, again twice;
* sums over n keys in 32 bits: at most n roundings of 2^-24 in numerator and denominator each;
* weights rounded to 16 bits before P V (tensor cores only): u_p = eps / 2 of the type;
* merged partials: a handful of 32-bit roundings, 16 * 2^-24;
* the output's own rounding: u = eps / 2 of the type, relative to the value.
"""

from __future__ import annotations

import math

import torch

PAGE = 16


def dense(pool, table_row, n):
    """(Hkv, n, D) float64: the first n keys of a table row; pages of -1 read as NaN."""
    pages = table_row[: (n + PAGE - 1) // PAGE].long()
    x = pool[pages.clamp(min=0)].double()
    x[pages < 0] = math.nan
    return x.permute(1, 0, 2, 3).reshape(pool.shape[1], -1, pool.shape[3])[:, :n]


def attention(q, k_pool, v_pool, tables, kv_lens, cu=None, positions=None, window=None, sinks=0):
    """(out, bound) in float64, both (Hq, T, D), for q (Hq, T, D).

    cu / positions None: one query per sequence at position kv_len - 1.  Only visible keys are touched.
    """
    hq, t, d = q.shape
    hkv = k_pool.shape[1]
    g = hq // hkv
    dev = q.device
    lens = kv_lens.tolist()
    cu = list(range(len(lens) + 1)) if cu is None else cu.tolist()
    out = torch.zeros(hq, t, d, dtype=torch.float64, device=dev)
    bound = torch.zeros_like(out)
    u = torch.finfo(q.dtype).eps / 2
    u_p = u if q.dtype != torch.float32 else 0.0
    for s, n in enumerate(lens):
        if cu[s + 1] == cu[s] or n == 0:
            continue
        tok = slice(cu[s], cu[s + 1])
        at = torch.full((1,), n - 1, device=dev) if positions is None else positions[tok].long()
        at = at[:, None]
        key = torch.arange(n, device=dev)[None, :]
        seen = key <= at
        if window is not None:
            seen &= (at - key < window) | (key < sinks)
        some = seen.any(0)
        if not some.any():
            continue
        k = dense(k_pool, tables[s], n)[:, some]
        v = dense(v_pool, tables[s], n)[:, some]
        seen = seen[:, some]
        rows = q[:, tok].double().reshape(hkv, -1, d)
        x = (rows @ k.transpose(1, 2) / math.sqrt(d)).view(hkv, g, -1, k.shape[1])
        x = x.masked_fill(~seen, -math.inf)
        p = torch.softmax(x, -1).nan_to_num(0.0)  # a row without a visible key: zeros
        o = (p.reshape(hkv, -1, k.shape[1]) @ v).view(hq, -1, d)
        a = (p.reshape(hkv, -1, k.shape[1]) @ v.abs()).view(hq, -1, d)
        big = (rows.abs() @ k.abs().transpose(1, 2) / math.sqrt(d)).view(hkv, g, -1, k.shape[1])
        big = big.masked_fill(~seen, 0.0).amax(-1).view(hq, -1, 1)
        count = seen.sum(-1).view(1, -1, 1)
        out[:, tok] = o
        e_s = (d + 4) * 2.0**-23 * big
        bound[:, tok] = a * (2 * e_s + 2 * 2.0**-22 + 2 * count * 2.0**-24 + 16 * 2.0**-24 + u_p) + u * o.abs() + 1e-30
    return out, bound


def check_attention(got, want, what=""):
    out, bound = want
    assert got.shape == out.shape, what
    assert torch.isfinite(got.float()).all(), f"{what}: not finite"
    # fp16 / bf16 have their own smallest step
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    over = (got.double() - out).abs() - bound - tiny
    worst = over.max().item() if over.numel() else -1.0
    assert worst <= 0, f"{what}: {worst:.3g} over the bound at {torch.nonzero(over > 0)[:4].tolist()}"


def beam_select(logits, scores, num_select, finished=None, eos=-1):
    """(tokens, parents, scores64) by a full sort in float64."""
    n, w = scores.shape
    v = logits.shape[1]
    x = logits.double()
    x = x - x.amax(1, keepdim=True)  # first, or logits of 1e38 swallow the logarithm of the sum
    total = scores.double().reshape(-1, 1) + (x - torch.exp(x).sum(1, keepdim=True).log())
    total[~torch.isfinite(scores.reshape(-1))] = -math.inf
    total = torch.where(torch.isnan(total) | (total == math.inf), torch.full_like(total, -math.inf), total)
    if finished is not None:
        for r in torch.nonzero(finished.reshape(-1))[:, 0].tolist():
            total[r] = -math.inf
            total[r, eos] = scores.reshape(-1)[r].double()
    total = total.reshape(n, w * v)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    return at[:, :num_select] % v, at[:, :num_select] // v, best[:, :num_select]


def beam_reorder(k_pools, v_pools, tables, kv_lens, parents):
    """New tables; copies in place in the given (cloned) pools.  Row by row, as the rule reads."""
    n, w = parents.shape
    new = tables.clone()
    moves = []
    for i in range(n):
        row0 = i * w
        kv = int(kv_lens[row0])
        full, fill = kv // PAGE, kv % PAGE
        par = parents[i].tolist()
        idle = [r for r in range(w) if r not in par]
        taken = set()
        for r in range(w):
            p = par[r]
            donor = p if p not in taken else idle.pop(0)
            taken.add(p)
            new[row0 + r, :full] = tables[row0 + p, :full]
            new[row0 + r, full:] = tables[row0 + donor, full:]
            if donor != p and fill:
                moves.append((int(tables[row0 + p, full]), int(tables[row0 + donor, full]), fill))
    for pool in [*k_pools, *v_pools]:
        old = pool.clone()
        for src, dst, fill in moves:
            pool[dst, :, :fill] = old[src, :, :fill]
    return new
