"""Cases of the cache-eviction operators: decode attention that scores the cached tokens,
differential decode attention, the 16-bit append, the selection of the tokens to keep and the
compaction of a paged cache.

A case is a dict of plain values; ``case["op"]`` names the operator. ``run`` computes it with
elementary torch operations in 32 bits (``own`` false) or through bpt's entry points (``own``
true). ``exact`` is the definition in 64 bits, sequence by sequence.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "kvq-decode_b200")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------ the cases

def _attend(name, **kw):
    c = dict(name=name, op="scored", dtype="fp16", batch=1, q_heads=32, kv_heads=8, head_dim=128,
             block_size=16, ctx=4096, lo=1.0, decay=1.0)
    c.update(kw)
    return c


def _diff(name, **kw):
    c = dict(name=name, op="diff", dtype="bf16", batch=1, heads=16, kv_heads=8, head_dim=64,
             block_size=16, ctx=4096, lo=1.0, decay=1.0, norm=True, scored=False)
    c.update(kw)
    return c


def _append(name, **kw):
    c = dict(name=name, op="append", dtype="fp16", batch=64, kv_heads=8, head_dim=128,
             block_size=16, new=1, slots=1024, state=True)
    c.update(kw)
    return c


def _select(name, **kw):
    c = dict(name=name, op="select", batch=1, kv_heads=8, slots=4096, lo=1.0, budget=1024,
             recent=64, sinks=4, zeros=0.1)
    c.update(kw)
    return c


def _compact(name, **kw):
    c = dict(name=name, op="compact", dtype="fp16", batch=1, kv_heads=8, head_dim=128,
             block_size=16, slots=4096, lo=1.0, budget=1024, recent=64, sinks=4, state=True)
    c.update(kw)
    return c


def listed():
    return [
        # one user's decode step over a short cache: latency
        _attend("scored b1 4k fp16"),
        # an ordinary ragged serving batch, scores that fade from step to step
        _attend("scored b8 16k bf16", dtype="bf16", batch=8, ctx=16384, lo=0.75, decay=0.9),
        # the largest: a full batch of long caches
        _attend("scored b16 32k fp16", batch=16, ctx=32768, lo=0.75, block_size=64),
        # a small differential layer, single user: latency
        _diff("diff b1 4k bf16"),
        # a long ragged batch of a wider differential model that is evicted too; odd group of 3
        _diff("diff b8 16k fp16 scored", dtype="fp16", batch=8, heads=12, kv_heads=4,
              head_dim=128, ctx=16384, lo=0.75, block_size=32, scored=True),
        # each decode step's own token, a batch of 64
        _append("append b64 one token"),
        # prompts that enter the cache
        _append("append b8 prompt 2048", dtype="bf16", batch=8, new=2048, slots=4096,
                block_size=64),
        # steady decoding: one page past the budget, every sequence of a batch
        _select("select b32 4k + a page", batch=32, slots=4112, budget=4096, recent=512),
        # a long prompt brought down to the budget
        _select("select b1 128k to 4k", slots=131072, budget=4096, recent=1024),
        _select("select b8 32k to 4k", batch=8, slots=32768, budget=4096, recent=1024, lo=0.5),
        # the moves that belong to the two kinds of selection
        _compact("compact b32 4k + a page", batch=32, slots=4112, budget=4096, recent=512),
        _compact("compact b8 32k to 4k", dtype="bf16", batch=8, slots=32768, budget=4096,
                 recent=1024, block_size=64, lo=0.5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["scored", "diff", "append", "select", "compact"])
    dtype = rng.choice(["fp16", "bf16"])
    batch = _log_int(rng, 1, 64)
    kv = rng.choice([1, 2, 4, 8])
    bs = rng.choice([16, 32, 64, 128, 256])
    lo = rng.choice([0.0, 0.5, 0.75, 1.0])
    if op in ("scored", "diff"):
        # at most 512k tokens of 8 heads of 128 channels
        most = min(131072, (1 << 19) * 8 // (batch * kv) // (2 if op == "diff" else 1))
        D = rng.choice([64, 128, 256] if op == "scored" else [64, 128])
        ctx = _log_int(rng, 1, max(16, most * 128 // D // 2 if D > 128 else most // 2))
        decay = rng.choice([1.0, 0.9, 0.0])
        if op == "scored":
            c = _attend("", dtype=dtype, batch=batch, q_heads=kv * rng.randint(1, 8),
                        kv_heads=kv, head_dim=D, block_size=bs, ctx=ctx, lo=lo, decay=decay)
        else:
            c = _diff("", dtype=dtype, batch=batch, heads=kv * rng.randint(1, 4), kv_heads=kv,
                      head_dim=D, block_size=bs, ctx=ctx, lo=lo, decay=decay,
                      norm=rng.random() < 0.7, scored=rng.random() < 0.5)
    elif op == "append":
        new = _log_int(rng, 1, max(2, 16384 // batch))
        c = _append("", dtype=dtype, batch=batch, kv_heads=kv, head_dim=rng.choice([64, 128, 256]),
                    block_size=bs, new=new, slots=new + _log_int(rng, 1, 2048),
                    state=rng.random() < 0.7)
    else:
        most = min(131072, (1 << 18) * 8 // (batch * kv) // 2)
        slots = _log_int(rng, 8, most)
        budget = _log_int(rng, 1, slots * 3 // 4)
        recent = rng.randint(0, budget // 2)
        sinks = rng.randint(0, min(8, budget - recent))
        if op == "select":
            c = _select("", batch=batch, kv_heads=kv, slots=slots, lo=lo, budget=budget,
                        recent=recent, sinks=sinks, zeros=rng.choice([0.0, 0.1, 0.9]))
        else:
            c = _compact("", dtype=dtype, batch=batch, kv_heads=kv,
                         head_dim=rng.choice([64, 128]), block_size=bs, slots=slots, lo=lo,
                         budget=budget, recent=recent, sinks=sinks, state=rng.random() < 0.7)
    del c["name"]
    return c


# ------------------------------------------------------------------------------ the inputs

def _lens(case, ctx, g):
    """Lengths U[lo ctx, ctx] of a batch; where lo is 0 an empty sequence and one of a token."""
    B, lo = case["batch"], int(case["lo"] * ctx)
    n = torch.randint(lo, ctx + 1, (B,), generator=g)
    if case["lo"] == 0.0 and B > 1:
        n[0] = 0
        n[-1] = 1
    return n


def _pages(lens, slots, block_size, g):
    """A table of random pages, every sequence with all its own: (block_table, num_blocks)."""
    B = lens.numel()
    per = (slots + block_size - 1) // block_size
    return torch.randperm(B * per, generator=g).to(torch.int32).reshape(B, per), B * per


def _scores(shape, zeros, dg):
    """Accumulated weights as a decode leaves them: spread over decades, the newest still 0."""
    s = torch.exp(2.0 * torch.randn(shape, generator=dg, device="cuda") - 5.0)
    return torch.where(torch.rand(shape, generator=dg, device="cuda") < zeros,
                       torch.zeros((), device="cuda"), s)


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    dg = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    B, H = case["batch"], case["kv_heads"]
    dt = DTYPES[case["dtype"]] if "dtype" in case else None

    def rand(*shape, dtype=dt):
        return torch.randn(*shape, generator=dg, device="cuda", dtype=dtype)

    s = {"case": case}
    if op in ("scored", "diff"):
        D, bs = case["head_dim"], case["block_size"]
        lens = _lens(case, case["ctx"], g)
        bt, nb = _pages(lens, case["ctx"], bs, g)
        T = bt.shape[1] * bs
        two = 2 if op == "diff" else 1
        heads = case["q_heads"] if op == "scored" else 2 * case["heads"]
        s.update(q=rand(B, heads, D), k=rand(nb, bs, two * H, D), v=rand(nb, bs, H, two * D),
                 bt=bt.cuda(), lens=lens.to(torch.int32).cuda())
        if op == "scored" or case["scored"]:
            s["scores"] = _scores((B, H, T), 0.1, dg)
        if op == "diff":
            s["lam"] = 0.2 + 0.5 * torch.rand(case["heads"], generator=dg, device="cuda")
            s["w"] = 1.0 + 0.1 * rand(2 * D, dtype=torch.float32) if case["norm"] else None
    elif op == "append":
        D, bs, S = case["head_dim"], case["block_size"], case["new"]
        start = torch.randint(0, case["slots"] - S + 1, (B,), generator=g)
        new = torch.full((B,), S) if S == 1 else torch.randint(S // 2, S + 1, (B,), generator=g)
        bt, nb = _pages(start, case["slots"], bs, g)
        s.update(k=rand(nb, bs, H, D), v=rand(nb, bs, H, D), kn=rand(B, S, H, D),
                 vn=rand(B, S, H, D), bt=bt.cuda(), start=start.to(torch.int32).cuda(),
                 new=new.to(torch.int32).cuda())
        if case["state"]:
            T = bt.shape[1] * bs
            s["scores"] = _scores((B, H, T), 0.1, dg)
            s["positions"] = torch.randint(0, 1 << 20, (B, H, T), generator=dg, device="cuda",
                                           dtype=torch.int32)
            s["next_pos"] = (start + 1000).to(torch.int32).cuda()
    else:
        T = case["slots"]
        lens = _lens(case, T, g)
        n = lens.cuda()
        # earlier evictions left the slots out of order: distinct positions below next_pos
        order = torch.rand(B, H, T, generator=dg, device="cuda")
        t = torch.arange(T, device="cuda")
        order = torch.where(t < n[:, None, None], order, 2.0)
        positions = torch.argsort(torch.argsort(order, dim=-1), dim=-1).to(torch.int32) + 7
        if case["sinks"]:
            positions = torch.where(positions < 7 + case["sinks"], positions - 7, positions)
        s.update(scores=_scores((B, H, T), case.get("zeros", 0.1), dg), positions=positions,
                 lens=lens.to(torch.int32).cuda(), next_pos=(n + 7).to(torch.int32))
        if op == "compact":
            D, bs = case["head_dim"], case["block_size"]
            bt, nb = _pages(lens, T, bs, g)
            s.update(k=rand(nb, bs, H, D), v=rand(nb, bs, H, D), bt=bt.cuda())
            s["moves"] = _select_plain(s, case)
    return s


# ------------------------------------------------------------------------------ plain forms

def _gather(cache, bt):
    """The slots of every sequence in 32 bits: [B, T, heads, channels]."""
    x = cache[bt.long()]
    return x.reshape(x.shape[0], -1, *x.shape[3:]).float()


def _softmax(x, valid):
    """Weights over the last axis where valid; nothing valid gives zeros."""
    x = torch.where(valid, x, float("-inf"))
    m = x.amax(dim=-1, keepdim=True)
    e = torch.exp(x - torch.where(m == float("-inf"), 0.0, m))
    total = e.sum(dim=-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


def _score_plain(scores, add, valid, decay):
    """Slots of valid tokens: decay * score + add; the others keep theirs. In place."""
    new = add if decay == 0 else decay * scores + add
    scores.copy_(torch.where(valid, new, scores))
    return scores


def _scored_plain(s, c):
    B, H, D = c["batch"], c["kv_heads"], c["head_dim"]
    k, v = _gather(s["k"], s["bt"]), _gather(s["v"], s["bt"])
    T = k.shape[1]
    valid = (torch.arange(T, device="cuda") < s["lens"][:, None])[:, None]        # [B, 1, T]
    q = s["q"].float().reshape(B, H, -1, D)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(D))             # [B, H, G, T]
    p = _softmax(x, valid[:, :, None])
    out = torch.matmul(p, v.permute(0, 2, 1, 3)).reshape(B, -1, D).to(s["q"].dtype)
    return {"out": out, "scores": _score_plain(s["scores"], p.sum(dim=2), valid, c["decay"])}


def _diff_plain(s, c):
    B, H, D = c["batch"], c["kv_heads"], c["head_dim"]
    G = c["heads"] // H
    k, v = _gather(s["k"], s["bt"]), _gather(s["v"], s["bt"])
    T = k.shape[1]
    valid = (torch.arange(T, device="cuda") < s["lens"][:, None])[:, None]
    q = s["q"].float().reshape(B, H, G, 2, D).transpose(2, 3)                     # [B, H, 2, G, D]
    kk = k.reshape(B, T, H, 2, D).permute(0, 2, 3, 4, 1)                          # [B, H, 2, D, T]
    p = _softmax(torch.matmul(q, kk) * (1.0 / math.sqrt(D)), valid[:, :, None, None])
    a = p[:, :, 0] - s["lam"].reshape(H, G, 1) * p[:, :, 1]                       # [B, H, G, T]
    o = torch.matmul(a, v.permute(0, 2, 1, 3))                                    # [B, H, G, 2D]
    if c["norm"]:
        o = o * torch.rsqrt(o.square().mean(dim=-1, keepdim=True) + 1e-5) * s["w"]
        o = o * 0.2
    r = {"out": o.reshape(B, H * G, 2 * D).to(s["q"].dtype)}
    if c["scored"]:
        r["scores"] = _score_plain(s["scores"], a.abs().sum(dim=2), valid, c["decay"])
    return r


def _append_plain(s, c):
    bs, S = c["block_size"], c["new"]
    t = torch.arange(S, device="cuda")
    b, i = torch.nonzero(t < s["new"][:, None], as_tuple=True)
    slot = s["start"].long()[b] + i
    page = s["bt"].long()[b, slot // bs]
    s["k"][page, slot % bs] = s["kn"][b, i]
    s["v"][page, slot % bs] = s["vn"][b, i]
    r = {"k": s["k"], "v": s["v"]}
    if c["state"]:
        s["scores"][b, :, slot] = 0.0
        s["positions"][b, :, slot] = (s["next_pos"][b] + i.to(torch.int32))[:, None]
        r.update(scores=s["scores"], positions=s["positions"])
    return r


def _select_plain(s, c):
    budget = c["budget"]
    scores, pos = s["scores"], s["positions"]
    B, H, T = scores.shape
    t = torch.arange(T, device="cuda")
    n = s["lens"][:, None, None]
    keep_by_rule = (pos < c["sinks"]) | (pos >= (s["next_pos"] - c["recent"])[:, None, None])
    key = torch.where(keep_by_rule, float("inf"), scores)
    key = torch.where(t < n, key, float("-inf"))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, t.expand(B, H, T))
    kept = (rank < budget) & (t < n)
    full = n > budget
    hole = full & ~kept & (t < budget)
    mover = full & kept & (t >= budget)
    counts = mover.sum(dim=-1)
    M = max(1, min(budget, T - budget))
    src = torch.full((B, H, M + 1), -1, dtype=torch.int32, device="cuda")
    dst = src.clone()
    slots = t.to(torch.int32).expand(B, H, T)
    # the i-th hole from the front takes the i-th mover from the back; place M is a bin
    at = torch.where(hole, hole.cumsum(-1) - 1, M)
    dst.scatter_(-1, at, slots)
    at = torch.where(mover, counts[..., None] - mover.cumsum(-1), M)
    src.scatter_(-1, at, slots)
    return {"src": src[..., :M].contiguous(), "dst": dst[..., :M].contiguous(),
            "counts": counts.to(torch.int32), "new_lens": s["lens"].clamp(max=budget)}


def _compact_plain(s, c):
    bs, m = c["block_size"], s["moves"]
    b, h, i = torch.nonzero(m["src"] >= 0, as_tuple=True)
    src, dst = m["src"][b, h, i].long(), m["dst"][b, h, i].long()
    bt = s["bt"].long()
    ps, pd = bt[b, src // bs], bt[b, dst // bs]
    s["k"][pd, dst % bs, h] = s["k"][ps, src % bs, h]
    s["v"][pd, dst % bs, h] = s["v"][ps, src % bs, h]
    r = {"k": s["k"], "v": s["v"]}
    if c["state"]:
        s["scores"][b, h, dst] = s["scores"][b, h, src]
        s["positions"][b, h, dst] = s["positions"][b, h, src]
        r.update(scores=s["scores"], positions=s["positions"])
    return r


# ------------------------------------------------------------------------------ bpt's calls

def _run_own(s, c):
    from bpt import diff, evict
    op = c["op"]
    if op == "scored":
        out = evict.paged_decode_attention_scored(s["q"], s["k"], s["v"], s["bt"], s["lens"],
                                                  s["scores"], decay=c["decay"])
        return {"out": out, "scores": s["scores"]}
    if op == "diff":
        out = diff.paged_decode_attention_diff(
            s["q"], s["k"], s["v"], s["bt"], s["lens"], s["lam"], norm_weight=s["w"],
            out_scale=0.2 if c["norm"] else 1.0, scores=s.get("scores"), decay=c["decay"])
        return {"out": out, "scores": s["scores"]} if c["scored"] else {"out": out}
    if op == "append":
        evict.append_tokens(s["k"], s["v"], s["kn"], s["vn"], s["new"], s["start"], s["bt"],
                            scores=s.get("scores"), positions=s.get("positions"),
                            next_pos=s.get("next_pos"))
    elif op == "select":
        m = evict.select_evictions(s["scores"], s["positions"], s["lens"], s["next_pos"],
                                   c["budget"], recent=c["recent"], sinks=c["sinks"])
        return {"src": m.src, "dst": m.dst, "counts": m.counts, "new_lens": m.new_lens}
    else:
        m = s["moves"]
        evict.compact_cache(s["k"], s["v"], s["bt"],
                            evict.EvictionMoves(m["src"], m["dst"], m["counts"], m["new_lens"]),
                            scores=s["scores"] if c["state"] else None,
                            positions=s["positions"] if c["state"] else None)
    r = {"k": s["k"], "v": s["v"]}
    if c["state"]:
        r.update(scores=s["scores"], positions=s["positions"])
    return r


_PLAIN = {"scored": _scored_plain, "diff": _diff_plain, "append": _append_plain,
          "select": _select_plain, "compact": _compact_plain}


def run(state):
    c = state["case"]
    if own:
        return _run_own(state, c)
    return _PLAIN[c["op"]](state, c)


# ------------------------------------------------------------------------------ the work

def work(case):
    c, op = case, case["op"]
    B, H = c["batch"], c["kv_heads"]
    if op in ("scored", "diff"):
        N = B * c["ctx"] * (1.0 + c["lo"]) / 2            # lengths are uniform in [lo, 1] ctx
        D, two = c["head_dim"], 2 if op == "diff" else 1
        heads = c["q_heads"] if op == "scored" else 2 * c["heads"]
        bytes_ = N * H * 2 * two * D * 2 + B * heads * D * 2 * 2 + N / c["block_size"] * 4 + 4 * B
        if op == "scored" or c["scored"]:
            bytes_ += N * H * 4 * (2 if c["decay"] else 1)
        flops = N * heads * (2 * D + 2 * two * D)
        return {"bytes": bytes_, "flops": flops}
    if op == "append":
        S = 1.0 if c["new"] == 1 else 0.75 * c["new"]     # new lengths are uniform in [S / 2, S]
        rows = B * S * H
        return {"bytes": rows * (2 * 2 * c["head_dim"] * 2 + (8 if c["state"] else 0)) +
                12 * B + B * math.ceil(S / c["block_size"]) * 4, "flops": rows}
    # tokens past the budget and how many of them are kept, the recent ones at random slots
    lo, hi, budget = c["lo"] * c["slots"], c["slots"], c["budget"]
    n = (lo + hi) / 2
    moved = 0.0 if n <= budget else budget * (n - budget) / n
    if op == "select":
        return {"bytes": B * H * (n * 8 + moved * 8 + 4) + 12 * B, "flops": B * H * n}
    row = 2 * c["head_dim"] * 2 + (8 if c["state"] else 0)
    return {"bytes": B * H * (moved * (2 * row + 8) + 4) + 64, "flops": B * H * moved}


# ------------------------------------------------------------------------------ 64 bits

def _slots_of(cache, bt_row, n):
    """Rows [n, heads, channels] of one sequence in 64 bits."""
    bs = cache.shape[1]
    t = torch.arange(n, device=cache.device)
    return cache[bt_row.long()[t // bs], t % bs].double()


def _exact_attend(s, c):
    B, H, D = c["batch"], c["kv_heads"], c["head_dim"]
    maps = 2 if c["op"] == "diff" else 1
    heads = c["heads"] if c["op"] == "diff" else c["q_heads"]
    G = heads // H
    out = torch.zeros(B, heads, maps * D, dtype=torch.float64, device="cuda")
    scores = s["scores"].double() if "scores" in s else None
    for b in range(B):
        n = int(s["lens"][b])
        if n == 0:
            continue
        k, v = _slots_of(s["k"], s["bt"][b], n), _slots_of(s["v"], s["bt"][b], n)
        q = s["q"][b].double()
        for h in range(H):
            total = torch.zeros(n, dtype=torch.float64, device="cuda")
            for j in range(h * G, (h + 1) * G):
                a = torch.softmax(k[:, maps * h] @ q[maps * j] / D ** 0.5, dim=0)
                if maps == 2:
                    second = torch.softmax(k[:, 2 * h + 1] @ q[2 * j + 1] / D ** 0.5, dim=0)
                    a = a - s["lam"][j].double() * second
                total += a.abs()
                o = a @ v[:, h]
                if c.get("norm"):
                    o = o / torch.sqrt((o * o).mean() + 1e-5) * s["w"].double() * 0.2
                out[b, j] = o
            if scores is not None:
                old = scores[b, h, :n]
                scores[b, h, :n] = total + (c["decay"] * old if c["decay"] else 0.0)
    return {"out": out, "scores": scores} if scores is not None else {"out": out}


def _exact_append(s, c):
    r = {x: s[x].double() for x in ("k", "v")}
    if c["state"]:
        r.update(scores=s["scores"].double(), positions=s["positions"].clone())
    for b in range(c["batch"]):
        start, m = int(s["start"][b]), int(s["new"][b])
        t = torch.arange(start, start + m, device="cuda")
        page = s["bt"][b].long()[t // c["block_size"]]
        r["k"][page, t % c["block_size"]] = s["kn"][b, :m].double()
        r["v"][page, t % c["block_size"]] = s["vn"][b, :m].double()
        if c["state"]:
            first = int(s["next_pos"][b])
            r["scores"][b, :, start:start + m] = 0.0
            r["positions"][b, :, start:start + m] = torch.arange(first, first + m, device="cuda",
                                                                 dtype=torch.int32)
    return r


def _exact_select(s, c):
    scores, pos = s["scores"].double().cpu().numpy(), s["positions"].cpu().numpy()
    lens, nxt = s["lens"].cpu().numpy(), s["next_pos"].cpu().numpy()
    B, H, T = scores.shape
    budget = c["budget"]
    M = max(1, min(budget, T - budget))
    src = np.full((B, H, M), -1, np.int32)
    dst = np.full((B, H, M), -1, np.int32)
    counts = np.zeros((B, H), np.int32)
    for b in range(B):
        n = int(lens[b])
        if n <= budget:
            continue
        for h in range(H):
            p = pos[b, h, :n]
            safe = (p < c["sinks"]) | (p >= nxt[b] - c["recent"])
            order = np.lexsort((np.arange(n), -scores[b, h, :n], ~safe))
            # protected slots are taken by slot alone, the rest by score and then by slot
            first = np.flatnonzero(safe)[:budget]
            rest = order[int(safe.sum()):][:budget - len(first)]
            kept = np.zeros(n, bool)
            kept[first] = True
            kept[rest] = True
            holes = np.flatnonzero(~kept[:budget])
            movers = budget + np.flatnonzero(kept[budget:])
            counts[b, h] = len(movers)
            src[b, h, :len(movers)] = movers[::-1]
            dst[b, h, :len(movers)] = holes
    new = np.minimum(lens, budget).astype(np.int32)
    return {"src": torch.from_numpy(src), "dst": torch.from_numpy(dst),
            "counts": torch.from_numpy(counts), "new_lens": torch.from_numpy(new)}


def _exact_compact(s, c):
    bs = c["block_size"]
    m = s["moves"]
    r = {x: s[x].double() for x in ("k", "v")}
    if c["state"]:
        r.update(scores=s["scores"].double(), positions=s["positions"].clone())
    counts = m["counts"].cpu()
    for b in range(c["batch"]):
        row = s["bt"][b].long()
        for h in range(c["kv_heads"]):
            k = int(counts[b, h])
            f, t = m["src"][b, h, :k].long(), m["dst"][b, h, :k].long()
            for x in ("k", "v"):
                r[x][row[t // bs], t % bs, h] = s[x][row[f // bs], f % bs, h].double()
            if c["state"]:
                r["scores"][b, h, t] = s["scores"][b, h, f].double()
                r["positions"][b, h, t] = s["positions"][b, h, f]
    return r


def exact(case, seed):
    s = prepare(case, seed)
    return {"scored": _exact_attend, "diff": _exact_attend, "append": _exact_append,
            "select": _exact_select, "compact": _exact_compact}[case["op"]](s, case)


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(4)]:
        print(c, work(c))
