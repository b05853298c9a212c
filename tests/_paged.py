"""The paged operators by their definitions, on the CPU: whole numbers with
Python integers, everything else in 64 bits.  Shared by the paged tests."""
import math

import torch

NO_PAGE, PAGE_OOB, LENGTH, TOKEN_OOB = 0x4, 0x8, 0x10, 0x1


def plan_ref(lens, new, table, n_blocks, free, n_free, page, max_rows):
    """The plan of one step page by page: (slots, positions, reqs, row_lens, row_start, table,
    n_blocks, free, n_free, flags) as lists."""
    table, have, free = [list(r) for r in table], list(n_blocks), list(free)
    n_pages, max_blocks, flags = len(free), len(table[0]) if table else 0, 0

    def clamp(v, lo, hi):
        nonlocal flags
        if v < lo or v > hi:
            flags |= LENGTH
        return max(lo, min(hi, v))

    lens = [clamp(n, 0, max_blocks * page) for n in lens]
    new = [int(n > 0) for n in lens] if new is None else [clamp(w, 0, n) for w, n in zip(new, lens)]
    have = [clamp(h, 0, max_blocks) for h in have]
    n_free = clamp(n_free, 0, n_pages)
    need = [-(-n // page) for n in lens]
    for b, row in enumerate(table):
        for j in range(need[b], have[b]):
            if n_free < n_pages:
                free[n_free] = row[j]
                n_free += 1
            else:
                flags |= LENGTH
    for b, row in enumerate(table):
        keep = min(need[b], have[b])
        got = keep
        for j in range(have[b], need[b]):
            if n_free > 0:
                n_free -= 1
                row[j] = free[n_free]
                got = j + 1
            else:
                flags |= NO_PAGE
                row[j] = -1
        for j in range(need[b], max_blocks):
            row[j] = -1
        have[b] = got
        if any(not 0 <= p < n_pages for p in row[:got]):
            flags |= PAGE_OOB
    rows, start = [], [0]
    for b, n in enumerate(lens):
        for p in range(n - new[b], n):
            pg = table[b][p // page]
            rows.append((pg * page + p % page if 0 <= pg < n_pages else -1, p, b, p + 1))
        start.append(len(rows))
    if len(rows) > max_rows:
        flags |= LENGTH
    rows = rows[:max_rows] + [(-1, 0, 0, 0)] * (max_rows - len(rows))
    cols = [list(c) for c in zip(*rows)] if rows else [[], [], [], []]
    return (*cols, [min(s, max_rows) for s in start], table, have, free, n_free, flags)


def attention_ref(q, ck, cv, table, lens, reqs=None, scale=None):
    """(out, lse, bound) in 64 bits on the CPU.  bound[r, h, i] is what an f32 evaluation may be
    off by: with A = scale sum |q k| at its largest over the keys and n keys,
      - a score is a sum of head_dim products, each q scaled and rounded first: A (hd + 4) 2^-24;
      - the exponent s - m is rounded again, and e^ is good to 2^-22: |s - m| 2^-23 + 2^-22;
      - sums of n terms: n 2^-24 (the order is free), rescalings and joins: 64 2^-24;
    all relative to p, which enters the numerator (times |v|) and the denominator."""
    q, ck, cv = q.detach().double().cpu(), ck.detach().cpu(), cv.detach().cpu()
    table, lens = table.cpu().tolist(), lens.cpu().tolist()
    R, H, hd = q.shape
    P, S, Hk, _ = ck.shape
    scale = hd ** -0.5 if scale is None else scale
    reqs = list(range(R)) if reqs is None else reqs.cpu().tolist()
    out, lse, bound = torch.zeros(R, H, hd).double(), torch.full((R, H), -math.inf).double(), torch.zeros(R, H, hd).double()
    u = 2.0 ** -24
    for r in range(R):
        n = max(0, min(lens[r], len(table[0]) * S))
        if not 0 <= reqs[r] < len(table):
            continue
        slots = [(table[reqs[r]][j // S], j % S) for j in range(n)]
        slots = [(p, i) for p, i in slots if 0 <= p < P]
        if not slots:
            continue
        at = torch.tensor(slots)
        k, v = ck[at[:, 0], at[:, 1]].double(), cv[at[:, 0], at[:, 1]].double()   # [n, Hk, hd]
        k, v = (t.repeat_interleave(H // Hk, 1).transpose(0, 1) for t in (k, v))    # [H, n, hd]
        s = scale * torch.einsum("hd,hnd->hn", q[r], k)
        p = torch.softmax(s, -1)
        out[r] = torch.einsum("hn,hnd->hd", p, v)
        lse[r] = torch.logsumexp(s, -1)
        a = (scale * torch.einsum("hd,hnd->hn", q[r].abs(), k.abs())).amax(-1)
        spread = (s.amax(-1, keepdim=True) - s).clamp(max=100.0).amax(-1)  # e^-100 weighs nothing
        rel = a * (hd + 4) * u + spread * 2 * u + 4 * u + (len(slots) + 64) * u
        bound[r] = 2 * rel[:, None] * torch.einsum("hn,hnd->hd", p, v.abs())
    return out, lse, bound


def logprobs_ref(x, tokens, k):
    """(logprob, entropy, ids, top logprobs, bounds of the first two) in 64 bits on the CPU.  The bound:
    e^d is good to 2^-22 and d log2 e is rounded (|d| 2^-23, weighted by p: at most ln V on the
    average over the mass); a sum runs over at most V terms of which a thread adds V / 256 + 8 and
    joins 32 times; d and the two logarithms are rounded to f32."""
    x = x.detach().cpu().double()
    N, V = x.shape
    u = 2.0 ** -24
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    S = e.sum(-1)
    mean = torch.where(e > 0, e * d, 0.0).sum(-1) / S
    entropy = torch.log(S) - mean
    best = torch.sort(x + 0.0, dim=-1, descending=True, stable=True).indices[:, :k]
    top = d.gather(1, best) - torch.log(S)[:, None]
    lp = None
    if tokens is not None:
        lp = d.gather(1, tokens.cpu().long().clamp(0, V - 1)[:, None])[:, 0] - torch.log(S)
    rel = (4 + 2 * math.log(V) + V / 256 + 8 + 32) * u
    return lp, entropy, best.to(torch.int32), top, rel, 2 * rel * (1 - mean) + 4 * u * entropy.abs()
