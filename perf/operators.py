"""The operators of paged T3 serving as they are measured: their cases, their plain form and the calls of the library.

Four operators, in the order in which a decode step uses them:

  plan      block tables, slot maps and row positions from the lengths of the requests (``ops.paged_plan``)
  append    the QKV epilogue: bias, Q, and the K / V rows written into the pages (``ops.qkv_kv_append_paged``)
  attend    attention of one new token per row over the pages (``ops.paged_decode_attention``)
  logprobs  log probability of a given token, entropy and the most probable alternatives (``ops.token_logprobs``)

``own`` selects between the plain form (elementary torch operations in f32, rounded once at the end) and the
library's calls.
"""
from __future__ import annotations

import math
import random

import torch

own = False

F32, F16, BF16 = "float32", "float16", "bfloat16"
SIZE = {F32: 4, F16: 2, BF16: 2}


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # A decode step of a large server: 512 streams of up to T3's 8196 positions, one new token each, some streams
        # that have just ended and give their pages back.
        _plan("plan_step_512", 512, 16, 8196, "decode"),
        # The prefill of 64 utterances of 1024 tokens (65,536 rows).
        _plan("plan_prefill_64", 64, 16, 1024, "prefill"),
        # The engine as it is: one stream, one token, an f32 cache.
        _append("append_1", 1, 16, 16, 64, F32, F32),
        # The same prefill's K / V rows, written in bf16.
        _append("append_prefill_64", 65536, 16, 16, 64, F32, BF16),
        # One stream of about a thousand tokens on the engine's f32 cache: latency.
        _attend("attend_1", 1, 1000, 16, 16, 16, 64, F32, F32, "full"),
        # 64 streams of unequal length on an f16 cache (T3's 2048-token context).
        _attend("attend_64_ragged", 64, 2048, 16, 16, 16, 64, F32, F16, "ragged"),
        # 128 streams up to T3's longest position table, everything in bf16.
        _attend("attend_128_long", 128, 8196, 32, 16, 16, 64, BF16, BF16, "ragged"),
        # One long document with grouped heads of 128: only the split over the keys gives parallel work.
        _attend("attend_1_grouped", 1, 65537, 64, 32, 8, 128, BF16, BF16, "full"),
        # One row of T3's speech logits: latency.
        _logprobs("logprobs_1", 1, 6563, F32, 5),
        # The 256 streams of a batched decode step.
        _logprobs("logprobs_256", 256, 6563, F32, 8),
        # Scoring 8192 speech tokens that are given; rows of odd length in 16 bits.
        _logprobs("logprobs_8192", 8192, 6563, BF16, 1),
        # Scoring over the text vocabulary, with 20 alternatives.
        _logprobs("logprobs_text_2048", 2048, 50276, F16, 20),
    ]


def _plan(name, requests, page, context, phase):
    return {"name": name, "kind": "plan", "requests": requests, "page": page, "context": context, "phase": phase}


def _append(name, rows, heads, kv_heads, head_dim, in_type, cache_type):
    return {"name": name, "kind": "append", "rows": rows, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "in_type": in_type, "cache_type": cache_type}


def _attend(name, rows, context, page, heads, kv_heads, head_dim, q_type, cache_type, lengths):
    return {"name": name, "kind": "attend", "rows": rows, "context": context, "page": page, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "q_type": q_type, "cache_type": cache_type,
            "lengths": lengths}


def _logprobs(name, rows, vocab, logit_type, top):
    return {"name": name, "kind": "logprobs", "rows": rows, "vocab": vocab, "type": logit_type, "top": top}


def draw(rng):
    """One more case of the same ranges: sizes over their logarithm, odd ones among them."""
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(("plan", "append", "attend", "attend", "logprobs", "logprobs"))
    if kind == "plan":
        case = _plan("", size(1, 512), rng.choice((8, 16, 32, 64)), size(64, 8196), rng.choice(("decode", "prefill", "mixed")))
        case["requests"] = min(case["requests"], 512 * 512 * case["page"] // case["context"])
        if case["phase"] != "decode":  # at most the rows of the 64 x 1024 prefill
            case["requests"] = max(1, min(case["requests"], 65536 // case["context"]))
    elif kind == "append":
        kv_heads, group, hd = rng.choice((1, 2, 4, 8, 16)), rng.choice((1, 1, 2, 4)), rng.choice((64, 80, 128))
        in_type = rng.choice((F32, F32, BF16, F16))
        heads = kv_heads * group
        case = _append("", size(1, 65536), heads, kv_heads, hd, in_type,
                       rng.choice((F32, F16, BF16)) if in_type == F32 else in_type)
        case["rows"] = max(1, min(case["rows"], 65536 * 16 * 64 // max(heads * hd, kv_heads * hd * 2)))
    elif kind == "attend":
        kv_heads, group, hd = rng.choice((1, 2, 4, 8, 16)), rng.choice((1, 1, 2, 4, 8)), rng.choice((32, 64, 64, 80, 128))
        cache_type = rng.choice((F32, F16, BF16))
        q_type = rng.choice((F32, cache_type))
        heads = kv_heads * group
        rows, context = size(1, 256), size(1, 65537)
        most = 0.9 * 128 * 8196 * 16 * 64  # bytes of keys, as in the largest listed case
        context = max(1, min(context, int(most / (rows * heads * hd * SIZE[cache_type]))))
        case = _attend("", rows, context, rng.choice((1, 8, 16, 32, 64, 100)), heads, kv_heads, hd, q_type, cache_type,
                       rng.choice(("full", "ragged")))
    else:
        vocab, logit_type = size(97, 50276), rng.choice((F32, F16, BF16))
        most = 2 * 2048 * 50276 // (vocab * SIZE[logit_type])
        case = _logprobs("", max(1, min(size(1, 8192), most)), vocab, logit_type, rng.choice((0, 1, 2, 5, 8, 20)))
    del case["name"]
    return case


def _rng_of(case):
    """Lengths belong to the case, so that work() knows them; everything else comes from the seed."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _plan_lengths(case):
    """(tokens before the step, tokens after it, new tokens) of each request."""
    r, n, ctx = _rng_of(case), case["requests"], case["context"]
    before, after, new = [], [], []
    for _ in range(n):
        what = r.random()
        if case["phase"] == "prefill" or (case["phase"] == "mixed" and what < 0.25):
            b, a = 0, ctx if case["phase"] == "prefill" else r.randint(1, ctx)
            w = a
        elif what > 0.94:  # ended: the pages go back
            b, a, w = r.randint(1, ctx), 0, 0
        else:
            b = r.randint(0, ctx - 1)
            a, w = b + 1, 1
        before.append(b)
        after.append(a)
        new.append(w)
    return before, after, new


def _attend_lengths(case):
    if case["lengths"] == "full":
        return [case["context"]] * case["rows"]
    r = _rng_of(case)
    return [r.randint(1, case["context"]) for _ in range(case["rows"])]


def work(case):
    kind = case["kind"]
    if kind == "plan":
        _, _, new = _plan_lengths(case)
        n, blocks = case["requests"], -(-case["context"] // case["page"])
        state = 4 * (n * blocks + n + n * blocks + 1)          # table, counts, free list, its height
        return {"bytes": 2 * state + 8 * n + 4 * (n + 1) + 16 * max(1, sum(new)), "flops": 0}
    if kind == "append":
        qd, kd = case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
        si, sc = SIZE[case["in_type"]], SIZE[case["cache_type"]]
        row = (qd + 2 * kd) * si + qd * si + 2 * kd * sc + 4
        return {"bytes": case["rows"] * row + 4 * (qd + 2 * kd), "flops": case["rows"] * (qd + 2 * kd)}
    if kind == "attend":
        lens = _attend_lengths(case)
        qd, kd = case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
        blocks = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 2 * sum(lens) * kd * SIZE[case["cache_type"]] + 2 * case["rows"] * qd * SIZE[case["q_type"]]
                + 4 * (blocks + case["rows"]), "flops": 4 * sum(lens) * qd}
    rows, vocab = case["rows"], case["vocab"]
    return {"bytes": rows * (vocab * SIZE[case["type"]] + 12 + 8 * case["top"]), "flops": 6 * rows * vocab}


# ----------------------------------------------------------------- inputs --

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"plan": _prepare_plan, "append": _prepare_append, "attend": _prepare_attend,
            "logprobs": _prepare_logprobs}[case["kind"]](dict(case), g)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _prepare_plan(s, g):
    before, after, new = _plan_lengths(s)
    n, page = s["requests"], s["page"]
    blocks = -(-s["context"] // page)
    pages = n * blocks
    have = [-(-b // page) for b in before]
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    held = torch.arange(blocks, device="cuda")[None, :] < _ints(have)[:, None]
    table = torch.full((n, blocks), -1, dtype=torch.int32, device="cuda")
    used = sum(have)
    table[held] = ids[:used]
    free = torch.cat([ids[used:], torch.full((used,), -1, dtype=torch.int32, device="cuda")])
    rows = max(1, sum(new))
    s.update(seq_lens=_ints(after), n_new=_ints(new), table=table, n_blocks=_ints(have), free=free,
             n_free=_ints([pages - used]), max_rows=rows, err=_ints([0]))
    # the buffers that a serving loop keeps for the step's plan
    s["out"] = [torch.empty(rows, dtype=torch.int32, device="cuda") for _ in range(4)] + [
        torch.empty(n + 1, dtype=torch.int32, device="cuda"), torch.empty_like(table), torch.empty_like(s["n_blocks"]),
        torch.empty_like(free), torch.empty_like(s["n_free"])]
    return s


def _prepare_append(s, g):
    rows, page = s["rows"], 16
    qd, kd = s["heads"] * s["head_dim"], s["kv_heads"] * s["head_dim"]
    pages = -(-rows // page) + 3
    ct = getattr(torch, s["cache_type"])
    s["qkv"] = torch.randn(rows, qd + 2 * kd, generator=g, device="cuda").to(getattr(torch, s["in_type"]))
    s["bias"] = 0.1 * torch.randn(qd + 2 * kd, generator=g, device="cuda")
    shape = (pages, page, s["kv_heads"], s["head_dim"])
    s["cache_k"] = torch.zeros(shape, dtype=ct, device="cuda")
    s["cache_v"] = torch.zeros(shape, dtype=ct, device="cuda")
    # pages in any order, the rows of a page one behind the other
    order = torch.randperm(pages, generator=g, device="cuda")[:, None] * page + torch.arange(page, device="cuda")
    s["slots"] = order.reshape(-1)[:rows].to(torch.int32)
    s["err"] = _ints([0])
    return s


def _prepare_attend(s, g):
    lens = _attend_lengths(s)
    rows, page, hd = s["rows"], s["page"], s["head_dim"]
    blocks = -(-s["context"] // page)
    have = [-(-n // page) for n in lens]
    pages = sum(have) + 1
    ct, shape = getattr(torch, s["cache_type"]), (pages, page, s["kv_heads"], hd)
    s["q"] = (1.5 * torch.randn(rows, s["heads"], hd, generator=g, device="cuda")).to(getattr(torch, s["q_type"]))
    s["cache_k"] = torch.empty(shape, dtype=ct, device="cuda").normal_(generator=g)
    s["cache_v"] = torch.empty(shape, dtype=ct, device="cuda").normal_(generator=g)
    table = torch.full((rows, blocks), -1, dtype=torch.int32, device="cuda")
    held = torch.arange(blocks, device="cuda")[None, :] < _ints(have)[:, None]
    table[held] = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[:sum(have)]
    s.update(table=table, seq_lens=_ints(lens), err=_ints([0]))
    return s


def _prepare_logprobs(s, g):
    rows, vocab = s["rows"], s["vocab"]
    # a language model's logits: a wide bulk, and a given token that is often a probable one
    x = 2.5 * torch.randn(rows, vocab, generator=g, device="cuda")
    tok = torch.randint(0, vocab, (rows, 1), generator=g, device="cuda")
    x.scatter_add_(1, tok, 6.0 * torch.rand(rows, 1, generator=g, device="cuda"))
    s["logits"] = x.to(getattr(torch, s["type"]))
    s["tokens"] = tok.reshape(-1).to(torch.int32)
    s["err"] = _ints([0])
    return s


# ------------------------------------------------------------------ a pass --

def run(s):
    return {"plan": _run_plan, "append": _run_append, "attend": _run_attend, "logprobs": _run_logprobs}[s["kind"]](s)


def _run_plan(s):
    if own:
        from chatterbox_amdvulkan_b200 import ops
        return list(ops.paged_plan(s["seq_lens"], s["table"], s["n_blocks"], s["free"], s["n_free"], s["page"],
                                   n_new=s["n_new"], max_rows=s["max_rows"], out=s["out"], err=s["err"])[:9])
    page, table, free = s["page"], s["table"].long(), s["free"].long()
    lens, new, have, n_free = s["seq_lens"].long(), s["n_new"].long(), s["n_blocks"].long(), s["n_free"].long()
    need = (lens + page - 1) // page
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    freed = (col >= need[:, None]) & (col < have[:, None])
    fresh = (col >= have[:, None]) & (col < need[:, None])
    # released pages onto the stack, in the order of the table
    at = n_free + torch.cumsum(freed.reshape(-1), 0) - 1
    stack = torch.cat([free, free.new_zeros(1)])
    stack = stack.scatter(0, torch.where(freed.reshape(-1), at, free.numel()), table.reshape(-1))[:-1]
    top = n_free + freed.sum()
    # missing pages from its top, in the order of the table
    at = (top - torch.cumsum(fresh.reshape(-1), 0)).reshape(fresh.shape)
    got = torch.where(at >= 0, stack[at.clamp(min=0)], -1)
    table = torch.where(fresh, got, torch.where(col < need[:, None], table, -1))
    start = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    t = torch.arange(s["max_rows"], device=table.device)
    req = torch.searchsorted(start[1:], t, right=True).clamp(max=lens.numel() - 1)
    live = t < start[-1]
    pos = torch.where(live, lens[req] - new[req] + t - start[req], 0)
    slot = torch.where(live, table[req, pos // page] * page + pos % page, -1)
    out = (slot, pos, torch.where(live, req, 0), torch.where(live, pos + 1, 0), start, table, need, stack,
           top - fresh.sum())
    return [x.to(torch.int32) for x in out]


def _run_append(s):
    ck, cv = s["cache_k"], s["cache_v"]
    if own:
        from chatterbox_amdvulkan_b200 import ops
        q, _ = ops.qkv_kv_append_paged(s["qkv"], s["bias"], ck, cv, s["slots"], err=s["err"])
        return [q, ck, cv]
    kd = s["kv_heads"] * s["head_dim"]
    x = s["qkv"].float() + s["bias"]
    qd, at = x.shape[1] - 2 * kd, s["slots"].long()
    ck.view(-1, kd)[at] = x[:, qd:qd + kd].to(ck.dtype)
    cv.view(-1, kd)[at] = x[:, qd + kd:].to(cv.dtype)
    return [x[:, :qd].to(s["qkv"].dtype), ck, cv]


def _run_attend(s):
    if own:
        from chatterbox_amdvulkan_b200 import ops
        return ops.paged_decode_attention(s["q"], s["cache_k"], s["cache_v"], s["table"], s["seq_lens"], err=s["err"])
    rows, heads, hd = s["q"].shape
    hk = s["kv_heads"]
    at = s["table"].long().clamp(min=0)
    k = s["cache_k"][at].reshape(rows, -1, hk, hd).transpose(1, 2).float()
    q = s["q"].float().view(rows, hk, heads // hk, hd)
    x = (q @ k.transpose(2, 3)) * (1.0 / math.sqrt(hd))
    del k
    there = torch.arange(x.shape[-1], device=x.device)[None, :] < s["seq_lens"][:, None]
    x = x.masked_fill(~there[:, None, None, :], float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    v = s["cache_v"][at].reshape(rows, -1, hk, hd).transpose(1, 2).float()
    return ((p @ v) / p.sum(-1, keepdim=True)).view(rows, heads, hd).to(s["q"].dtype)


def _run_logprobs(s):
    if own:
        from chatterbox_amdvulkan_b200 import ops
        return list(ops.token_logprobs(s["logits"], s["tokens"], top_k=s["top"], err=s["err"])[:4])
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(-1)
    log_total = torch.log(total)
    lp = d.gather(1, s["tokens"].long()[:, None])[:, 0] - log_total
    entropy = log_total - (e * d).sum(-1) / total
    # the largest first, equal ones by their index: one whole number holds both
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * (1 << 32) + (x.shape[1] - 1 - torch.arange(x.shape[1], device=x.device))
    ids = torch.topk(key, s["top"], dim=-1).indices
    return [lp, entropy, ids.to(torch.int32), d.gather(1, ids) - log_total[:, None]]


# ----------------------------------------------------- 64 bits, by definition --

def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "append": _exact_append, "attend": _exact_attend,
            "logprobs": _exact_logprobs}[case["kind"]](s)


def _exact_plan(s):
    """The stack and the tables, page by page."""
    page = s["page"]
    table, have = s["table"].tolist(), s["n_blocks"].tolist()
    stack, height = s["free"].tolist(), s["n_free"].item()
    lens, new = s["seq_lens"].tolist(), s["n_new"].tolist()
    need = [-(-n // page) for n in lens]
    for b, row in enumerate(table):
        for j in range(need[b], have[b]):
            stack[height] = row[j]
            height += 1
            row[j] = -1
    for b, row in enumerate(table):
        for j in range(have[b], need[b]):
            height -= 1
            row[j] = stack[height]
    rows, start = [], [0]
    for b, n in enumerate(lens):
        for p in range(n - new[b], n):
            rows.append((table[b][p // page] * page + p % page, p, b, p + 1))
        start.append(len(rows))
    rows += [(-1, 0, 0, 0)] * (s["max_rows"] - len(rows))
    return [torch.tensor(v, dtype=torch.int32) for v in (*map(list, zip(*rows)), start, table, need, stack, [height])]


def _exact_append(s):
    x = s["qkv"].double() + s["bias"].double()
    kd = s["kv_heads"] * s["head_dim"]
    k, v = s["cache_k"].double(), s["cache_v"].double()
    at = s["slots"].long()
    k.view(-1, kd).index_copy_(0, at, x[:, -2 * kd:-kd])
    v.view(-1, kd).index_copy_(0, at, x[:, -kd:])
    return [x[:, :-2 * kd], k, v]


def _exact_attend(s):
    """Request by request, head by head of the cache."""
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group, page, table = s["heads"] // s["kv_heads"], s["page"], s["table"].long()
    for r, n in enumerate(s["seq_lens"].tolist()):
        pages = table[r, :-(-n // page)]
        k = s["cache_k"][pages].flatten(0, 1)[:n].double()
        v = s["cache_v"][pages].flatten(0, 1)[:n].double()
        for h in range(s["kv_heads"]):
            q = s["q"][r, h * group:(h + 1) * group].double()
            p = torch.softmax(q @ k[:, h].T / math.sqrt(s["head_dim"]), -1)
            out[r, h * group:(h + 1) * group] = p @ v[:, h]
    return out


def _exact_logprobs(s):
    lp, entropy, ids, alt = [], [], [], []
    for x, tok in zip(s["logits"].split(512), s["tokens"].long().split(512)):
        y = torch.log_softmax(x.double(), -1)
        lp.append(y.gather(1, tok[:, None])[:, 0])
        entropy.append(-(y.exp() * y).sum(-1))
        best = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[:, :s["top"]]
        ids.append(best.to(torch.int32))
        alt.append(y.gather(1, best))
    return [torch.cat(v) for v in (lp, entropy, ids, alt)]
