"""Scored decode, append, selection and compaction on the GPU against oracle.evict (float64),
with bounds derived there from the arithmetic; and a run of them as a serving loop uses them."""
import numpy as np
import pytest
import torch

from evict_cases import PAIR_BITS, attend_case, check_out, check_scores, f64

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


def run_scored(c, dtype, decay=1.0, num_splits=None, what="", **kw):
    from bpt import evict
    from oracle import evict as ox
    old = c["scores"].clone()
    out = evict.paged_decode_attention_scored(c["q"], c["k"], c["v"], c["bt"], c["sl"],
                                              c["scores"], num_splits=num_splits, decay=decay, **kw)
    ref, tol, added = ox.decode(f64(c["q"]), f64(c["k"]), f64(c["v"]), c["bt"].cpu().numpy(),
                                c["sl"].tolist(), pair_bits=PAIR_BITS[dtype],
                                scale=kw.get("scale"))
    check_out(out, ref, tol, what)
    check_scores(c["scores"], old, added, c["sl"].tolist(), decay, what)
    return out


# ---------------------------------------------------------------------------- scored decode

@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (6, 2), (4, 1), (10, 2), (8, 1), (7, 1)])
def test_scored_head_layouts(dtype, D, Hq, Hkv):
    lens = [0, 1, 15, 16, 33, 200, 1100]
    for ns in (1, 3, None):
        c = attend_case(D + Hq, lens, Hq, Hkv, D, 16, dtype, garbage=float("nan"))
        run_scored(c, dtype, num_splits=ns, what=f"splits={ns}")


@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("decay", [1.0, 0.875, 0.0])
def test_scored_pages_and_decay(bs, decay):
    c = attend_case(bs, [1, bs - 1, bs, bs + 1, 5 * bs + 7], 8, 2, 128, bs, FP16)
    if decay == 0.0:
        c["scores"].fill_(float("nan"))   # decay 0 does not read them
    for ns in (None, 2):
        run_scored(c, FP16, decay=decay, num_splits=ns)


def test_scored_ragged_long_batch():
    c = attend_case(5, [9000, 1, 0, 8191, 33, 4096], 8, 2, 128, 32, BF16)
    run_scored(c, BF16)


def test_scored_scale_and_one_heavy_token():
    """A token that takes nearly all the weight next to ones whose weight underflows."""
    c = attend_case(6, [300, 70], 4, 1, 64, 16, FP16)
    row = c["bt"][0, 2].item()
    c["k"][row, 5, 0] = 8.0 * c["q"][0, 0].sign()
    run_scored(c, FP16, decay=0.0, scale=0.5)


def test_scored_strided_views():
    """Scores as rows of a wider, unaligned buffer; interleaved and head-major caches; q and out as
    slices of wider tensors."""
    from bpt import evict
    c = attend_case(7, [100, 37, 64], 6, 2, 64, 16, BF16)
    base = {x: c[x].clone() for x in ("k", "v", "q", "scores")}
    want_scores = base["scores"].clone()
    want = evict.paged_decode_attention_scored(c["q"], c["k"], c["v"], c["bt"], c["sl"],
                                               want_scores)
    wide = torch.full((3, 2, c["T"] + 5), -7.0, device="cuda")
    view = wide[:, :, 1:1 + c["T"]]
    kv = torch.stack([base["k"], base["v"]], dim=1)
    head_major = [base[x].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in "kv"]
    qkv = torch.randn(3, 6 + 4, 64, device="cuda").to(BF16)
    qkv[:, :6] = base["q"]
    outs = torch.zeros(3, 8, 64, dtype=BF16, device="cuda")
    for k, v in ((kv[:, 0], kv[:, 1]), head_major):
        view.copy_(base["scores"])
        out = evict.paged_decode_attention_scored(qkv[:, :6], k, v, c["bt"], c["sl"], view,
                                                  out=outs[:, 1:7])
        assert torch.equal(out, want) and torch.equal(view, want_scores)
        assert (wide[:, :, 0] == -7).all() and (wide[:, :, 1 + c["T"]:] == -7).all()
        assert (outs[:, 0] == 0).all() and (outs[:, 7] == 0).all()
    # scores by head first
    by_head = base["scores"].transpose(0, 1).contiguous().transpose(0, 1)
    evict.paged_decode_attention_scored(c["q"], c["k"], c["v"], c["bt"], c["sl"], by_head)
    assert torch.equal(by_head, want_scores)


def test_scored_shared_pages():
    """Two sequences read the same prefix pages: each keeps its own scores."""
    c = attend_case(8, [64, 64, 50], 4, 2, 64, 16, FP16)
    c["bt"][1, :4] = c["bt"][0, :4]
    c["bt"][2, :4] = c["bt"][0, :4]
    run_scored(c, FP16)


def test_scored_matches_the_fp16_decode():
    from bpt import evict, paged_decode_attention
    c = attend_case(9, [700, 1, 129], 32, 8, 128, 16, FP16)
    out = evict.paged_decode_attention_scored(c["q"], c["k"], c["v"], c["bt"], c["sl"],
                                              c["scores"])
    ref = paged_decode_attention(c["q"], c["k"], c["v"], c["bt"], c["sl"])
    # two fp32 computations, each rounded once: at most one step of fp16 apart, and the fp32 error
    assert ((out.float() - ref.float()).abs() <= ref.float().abs() * 2.0 ** -10 + 1e-5).all()


def test_scored_repeats_bitwise_and_by_graph():
    from bpt import evict
    c = attend_case(10, [900, 0, 333], 8, 2, 128, 16, FP16)
    start = c["scores"].clone()
    ws = torch.empty(evict.scored_workspace_bytes(c["q"], c["k"], c["bt"]), dtype=torch.uint8,
                     device="cuda")
    args = (c["q"], c["k"], c["v"], c["bt"], c["sl"], c["scores"])
    a = evict.paged_decode_attention_scored(*args, decay=0.5, workspace=ws).clone()
    sa = c["scores"].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c["scores"].copy_(start)
        b = evict.paged_decode_attention_scored(*args, decay=0.5, workspace=ws)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a, b) and torch.equal(sa, c["scores"])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = evict.paged_decode_attention_scored(*args, decay=0.5, workspace=ws)
    c["scores"].copy_(start)
    g.replay()
    assert torch.equal(a, out) and torch.equal(sa, c["scores"])
    g.replay()                                  # fades and adds again
    assert torch.allclose(c["scores"][0, :, :900], 0.5 * sa[0, :, :900] +
                          (sa - 0.5 * start)[0, :, :900], rtol=1e-5, atol=1e-7)


def test_scored_two_streams_and_two_graphs_at_once():
    """Calls that overlap on two streams, eager and captured, each with its own workspace, give what
    they give alone."""
    from bpt import evict
    cases = [attend_case(30 + i, lens, 8, 2, 128, 16, FP16)
             for i, lens in enumerate(([3000, 5], [2000, 1999, 64]))]
    run = lambda c, s: evict.paged_decode_attention_scored(  # noqa: E731
        c["q"], c["k"], c["v"], c["bt"], c["sl"], s, decay=0.0)
    alone = []
    for c in cases:
        s = c["scores"].clone()
        alone.append((run(c, s).clone(), s))
    streams = [torch.cuda.Stream() for _ in cases]
    graphs, held = [], []
    for c, st in zip(cases, streams):
        s = c["scores"].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = run(c, s)
        graphs.append(g)
        held.append((out, s))
    torch.cuda.synchronize()
    for turn in range(20):
        got = []
        for c, st, g, h in zip(cases, streams, graphs, held):
            with torch.cuda.stream(st):
                if turn % 2:
                    s = c["scores"].clone()
                    got.append((run(c, s), s))
                else:
                    h[1].copy_(c["scores"])
                    g.replay()
                    got.append(h)
        torch.cuda.synchronize()
        for a, b in zip(got, alone):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_scored_far_pages():
    """Pages past 2^31 elements of a cache (4.5 GB each)."""
    from bpt import evict
    bs, H, D = 256, 8, 128
    nb = (1 << 31) // (bs * H * D) + 16
    c = attend_case(11, [600], 8, 8, D, bs, FP16, spare=0)
    k = torch.empty(nb, bs, H, D, dtype=FP16, device="cuda")
    v = torch.empty_like(k)
    far = torch.tensor([[nb - 1, nb - 9, nb - 4, 0]], dtype=torch.int32, device="cuda")
    for i in range(3):
        k[far[0, i].long()] = c["k"][c["bt"][0, i].long()]
        v[far[0, i].long()] = c["v"][c["bt"][0, i].long()]
    s = c["scores"].clone()
    want = evict.paged_decode_attention_scored(c["q"], c["k"], c["v"], c["bt"], c["sl"], s)
    out = evict.paged_decode_attention_scored(c["q"], k, v, far, c["sl"], c["scores"])
    assert torch.equal(out, want) and torch.equal(s, c["scores"])


def test_scored_empty_batch_and_table():
    from bpt import evict
    c = attend_case(12, [5], 4, 2, 64, 16, FP16)
    out = evict.paged_decode_attention_scored(c["q"][:0], c["k"], c["v"], c["bt"][:0], c["sl"][:0],
                                              c["scores"][:0])
    assert out.shape == (0, 4, 64)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = evict.paged_decode_attention_scored(c["q"], c["k"], c["v"], c["bt"][:, :0], none,
                                              c["scores"][:, :, :0])
    assert (out == 0).all()


def test_scored_checked_mode(monkeypatch):
    from bpt import BptError, decode, evict
    monkeypatch.setattr(decode, "CHECKS", True)
    c = attend_case(13, [40], 4, 2, 64, 16, FP16)
    args = (c["q"], c["k"], c["v"], c["bt"], c["sl"], c["scores"])
    evict.paged_decode_attention_scored(*args)
    c["bt"][0, 1] = c["k"].shape[0]
    with pytest.raises(BptError, match="block_table"):
        evict.paged_decode_attention_scored(*args)


# ---------------------------------------------------------------------------- append

@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("D,S", [(64, 1), (128, 9), (256, 40), (40, 5)])
def test_append(dtype, D, S):
    from bpt import evict
    from oracle import evict as ox
    g = torch.Generator().manual_seed(D + S)
    B, H, bs, mb = 5, 3, 16, 6
    k, v = (torch.randn(B * mb + 2, bs, H, D, generator=g).to(dtype).cuda() for _ in "kv")
    kn, vn = (torch.randn(B, S, H, D, generator=g).to(dtype).cuda() for _ in "kv")
    bt = torch.randperm(B * mb + 2, generator=g)[:B * mb].reshape(B, mb).int()
    start = torch.tensor([0, 15, 16, 37, 90], dtype=torch.int32)
    new = torch.tensor([S, 0, S - S // 2, S + 3, S], dtype=torch.int32)   # the last runs past
    nxt = start + 1000
    T = mb * bs + 2
    scores = torch.rand(B, H, T, generator=g)
    pos = torch.randint(0, 9, (B, H, T), generator=g, dtype=torch.int32)
    want = [ox.append(f64(c), f64(n), new, start, bt.numpy()) for c, n in ((k, kn), (v, vn))]
    ws, wp = scores.clone(), pos.clone()
    for b in range(B):
        for t in range(min(int(new[b]), S)):
            s = int(start[b]) + t
            if s < mb * bs:
                ws[b, :, s] = 0
                wp[b, :, s] = int(nxt[b]) + t
    scores, pos = scores.cuda(), pos.cuda()
    evict.append_tokens(k, v, kn, vn, new.cuda(), start.cuda(), bt.cuda(), scores=scores,
                        positions=pos, next_pos=nxt.cuda())
    assert np.array_equal(f64(k), want[0]) and np.array_equal(f64(v), want[1])
    assert torch.equal(scores.cpu(), ws) and torch.equal(pos.cpu(), wp)


def test_append_views_and_differential_heads():
    """Rows out of a fused projection at an odd offset, a head-major cache, and a cache of 2 H key
    heads of D and H value heads of 2 D."""
    from bpt import evict
    from oracle import evict as ox
    g = torch.Generator().manual_seed(3)
    B, H, D, bs, mb, S = 2, 2, 64, 16, 3, 7
    k = torch.randn(B * mb, 2 * H, bs, D, generator=g).half().cuda().permute(0, 2, 1, 3)
    v = torch.randn(B * mb, bs, H, 2 * D, generator=g).half().cuda()
    fused = torch.randn(B, S, 4 * H * D + 3, generator=g).half().cuda()
    kn = fused[..., 1:1 + 2 * H * D].view(B, S, 2 * H, D)
    vn = fused[..., 2 + 2 * H * D:2 + 4 * H * D].view(B, S, H, 2 * D)
    bt = torch.randperm(B * mb, generator=g).reshape(B, mb).int()
    start, new = (torch.tensor(x, dtype=torch.int32).cuda() for x in ([3, 30], [S, 4]))
    want = [ox.append(f64(c), f64(n), new, start, bt.numpy()) for c, n in ((k, kn), (v, vn))]
    evict.append_tokens(k, v, kn, vn, new, start, bt.cuda())
    assert np.array_equal(f64(k), want[0]) and np.array_equal(f64(v), want[1])


def test_append_checked_mode(monkeypatch):
    from bpt import BptError, decode, evict
    monkeypatch.setattr(decode, "CHECKS", True)
    k, v = (torch.zeros(4, 16, 2, 64, device="cuda", dtype=FP16) for _ in "kv")
    new = torch.ones(1, 2, 2, 64, device="cuda", dtype=FP16)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    bt = i32(1, 2).view(1, 2)
    evict.append_tokens(k, v, new, new, i32(2), i32(30), bt)
    with pytest.raises(BptError, match="seq_len"):
        evict.append_tokens(k, v, new, new, i32(2), i32(31), bt)
    with pytest.raises(BptError, match="negative"):
        evict.append_tokens(k, v, new, new, i32(2), i32(-1), bt)
    before = k.clone()
    with pytest.raises(BptError, match="block_table"):
        evict.append_tokens(k, v, new, new, i32(2), i32(16), i32(1, 4).view(1, 2))
    assert torch.equal(k, before)


# ---------------------------------------------------------------------------- selection

def select_case(seed, B, H, T, lens, recent, kind):
    g = torch.Generator().manual_seed(seed)
    scores = torch.exp(2 * torch.randn(B, H, T, generator=g))
    if kind == "ties":
        scores = torch.randint(0, 4, (B, H, T), generator=g).float() / 4
    elif kind == "signs":
        scores = torch.randn(B, H, T, generator=g)
        scores[torch.rand(B, H, T, generator=g) < 0.1] = -0.0
        scores[torch.rand(B, H, T, generator=g) < 0.1] = 0.0
    elif kind == "odd":
        for x in (float("nan"), float("inf"), -float("inf"), -1.0, 1e-42):
            scores[torch.rand(B, H, T, generator=g) < 0.15] = x
    elif kind == "same":
        scores.fill_(0.25)
    pos = torch.argsort(torch.rand(B, H, T, generator=g), dim=-1).int()
    for b, n in enumerate(lens):           # positions 0 .. n - 1 of the valid slots, in disorder
        pos[b, :, :n] = torch.argsort(torch.rand(H, n, generator=g), dim=-1).int()
    return scores, pos, torch.tensor(lens, dtype=torch.int32)


@pytest.mark.parametrize("kind", ["weights", "ties", "signs", "odd", "same"])
@pytest.mark.parametrize("T,budget,recent,sinks", [(40, 1, 0, 0), (40, 39, 3, 2), (300, 128, 16, 4),
                                                   (1000, 257, 257, 0), (4500, 4096, 100, 4),
                                                   (64, 64, 1, 1), (16, 40, 2, 0)])
def test_select(kind, T, budget, recent, sinks):
    from bpt import evict
    from oracle import evict as ox
    lens = [T, 0, 1, max(T - 3, 0), min(budget, T), min(budget + 1, T)]
    scores, pos, sl = select_case(T + budget, len(lens), 2, T, lens, recent, kind)
    m = evict.select_evictions(scores.cuda(), pos.cuda(), sl.cuda(), sl.cuda(), budget,
                               recent=recent, sinks=sinks)
    want = ox.select(scores.numpy(), pos.numpy(), sl.numpy(), sl.numpy(), budget, recent, sinks)
    for got, w, name in zip(m, want, m._fields):
        assert np.array_equal(got.cpu().numpy(), w), name


def plain_select(scores, pos, n, nxt, budget, recent, sinks):
    """numpy's for one long row: kept slots."""
    s = np.where(np.isnan(scores[:n]), -np.inf, scores[:n].astype(np.float64))
    safe = (pos[:n] < sinks) | (pos[:n] >= nxt - recent)
    order = np.lexsort((np.arange(n), -s, ~safe))
    kept = np.zeros(n, bool)
    first = np.flatnonzero(safe)[:budget]
    kept[first] = True
    kept[order[int(safe.sum()):][:budget - len(first)]] = True
    return kept


@pytest.mark.parametrize("T,B,H", [(131072, 1, 2), (70001, 2, 1), (20000, 3, 5), (450000, 1, 1),
                                   (120000, 1, 80), (600001, 1, 1)])
@pytest.mark.parametrize("kind", ["weights", "same"])
def test_select_long_rows(T, B, H, kind):
    """Rows that a cluster shares: few and many of them, slices of 1 to 16 tiles a warp, and one
    longer than the registers of the largest cluster hold (read again in each pass)."""
    from bpt import evict
    lens = [T - 13 * b for b in range(B)]
    scores, pos, sl = select_case(T, B, H, T, lens, 1024, kind)
    for budget in (4096, T - 40):
        m = evict.select_evictions(scores.cuda(), pos.cuda(), sl.cuda(), sl.cuda(), budget,
                                   recent=1024, sinks=4)
        src, dst, counts = (x.cpu().numpy() for x in m[:3])
        for b in range(B):
            for h in range(0, H, 7):
                kept = plain_select(scores[b, h].numpy(), pos[b, h].numpy(), lens[b], lens[b],
                                    budget, 1024, 4)
                movers = budget + np.flatnonzero(kept[budget:])
                holes = np.flatnonzero(~kept[:budget])
                c = len(movers)
                assert counts[b, h] == c
                assert np.array_equal(src[b, h, :c], movers[::-1])
                assert np.array_equal(dst[b, h, :c], holes)
                assert (src[b, h, c:] == -1).all() and (dst[b, h, c:] == -1).all()


def test_views_of_short_rows():
    """A wide table and wide state rows, called through views of the slots in use: the same results
    as with the whole rows."""
    from bpt import evict
    c = attend_case(21, [300, 77], 4, 2, 64, 16, FP16)
    wide = torch.zeros(2, 4096 // 16, dtype=torch.int32, device="cuda")
    wide[:, :c["bt"].shape[1]] = c["bt"]
    scores = torch.zeros(2, 2, 4096, device="cuda")
    pos = torch.arange(4096, device="cuda").int().expand(2, 2, -1).contiguous()
    got = []
    for slots in (4096, 320):
        s = scores.clone()
        out = evict.paged_decode_attention_scored(c["q"], c["k"], c["v"], wide[:, :slots // 16],
                                                  c["sl"], s[:, :, :slots], num_splits=4)
        m = evict.select_evictions(s[:, :, :slots], pos[:, :, :slots], c["sl"], c["sl"], 100)
        got.append((out, s, m.src[:, :, :100], m.dst[:, :, :100], m.counts, m.new_lens))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_select_views_reuse_and_too_many_protected():
    """Unaligned rows of wider buffers; moves reused; positions that protect more than the budget
    (as a caller's mistake could) still keep exactly the budget."""
    from bpt import evict
    from oracle import evict as ox
    T, budget = 700, 200
    scores, pos, sl = select_case(1, 3, 2, T, [700, 300, 650], 10, "ties")
    pos[0] = 650
    ws = torch.zeros(3, 2, T + 9).cuda()
    wp = torch.zeros(2, 3, T + 6, dtype=torch.int32).cuda().transpose(0, 1)
    ws[:, :, 3:3 + T] = scores.cuda()
    wp[:, :, 1:1 + T] = pos.cuda()
    want = ox.select(scores.numpy(), pos.numpy(), sl.numpy(), sl.numpy(), budget, 100, 2)
    m = None
    for _ in range(2):
        m = evict.select_evictions(ws[:, :, 3:3 + T], wp[:, :, 1:1 + T], sl.cuda(), sl.cuda(),
                                   budget, recent=100, sinks=2, moves=m)
        for got, w in zip(m, want):
            assert np.array_equal(got.cpu().numpy(), w)
        m.src.fill_(5)
        m.dst.fill_(5)


def test_select_of_a_cluster_in_a_graph_and_on_two_streams():
    """Long rows (a cluster each): captured and replayed with new scores, and two calls at once."""
    from bpt import evict
    T, budget = 60000, 5000
    a = [x.cuda() for x in select_case(3, 1, 2, T, [T], 64, "weights")]
    b = [x.cuda() for x in select_case(4, 1, 2, T, [T - 7], 64, "weights")]
    want = [[t.clone() for t in evict.select_evictions(s, p, n, n, budget, recent=64)]
            for s, p, n in (a, b)]
    live = [x.clone() for x in a]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m = evict.select_evictions(*live, live[2], budget, recent=64)
    for case, w in ((a, want[0]), (b, want[1]), (a, want[0])):
        for x, y in zip(live, case):
            x.copy_(y)
        g.replay()
        assert all(torch.equal(x, y) for x, y in zip(m, w))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for st, (s, p, n) in zip(streams, (a, b)):
            with torch.cuda.stream(st):
                got.append(evict.select_evictions(s, p, n, n, budget, recent=64))
        torch.cuda.synchronize()
        for x, w in zip(got, want):
            assert all(torch.equal(i, j) for i, j in zip(x, w))


# ---------------------------------------------------------------------------- compaction

@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("H,DK,DV,bs", [(2, 64, 64, 16), (3, 128, 128, 32), (1, 256, 256, 64),
                                        (2, 256, 128, 256), (2, 40, 8, 16)])
def test_evict_and_compact(dtype, H, DK, DV, bs):
    from bpt import evict
    from oracle import evict as ox
    g = torch.Generator().manual_seed(DK + bs)
    lens, budget = [300, 0, 77, 101], 100
    mb = (max(lens) + bs - 1) // bs
    B, T = len(lens), mb * bs
    scores, pos, sl = select_case(DV, B, H, T, lens, 10, "weights")
    bt = torch.randperm(B * mb + 1, generator=g)[:B * mb].reshape(B, mb).int()
    k = torch.randn(B * mb + 1, bs, H, DK, generator=g).to(dtype)
    v = torch.randn(B * mb + 1, H, bs, DV, generator=g).to(dtype).permute(0, 2, 1, 3)  # head-major
    src, dst, counts, new = ox.select(scores.numpy(), pos.numpy(), sl.numpy(), sl.numpy(), budget,
                                      20, 3)
    want = [ox.compact(f64(x), bt.numpy(), src, dst, counts) for x in (k, v)]
    want += [ox.compact_rows(x.numpy(), src, dst, counts) for x in (scores, pos)]
    gk = k.cuda()
    gv = v.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3)
    gs, gp = scores.cuda(), pos.cuda()
    got_new = evict.evict_tokens(gk, gv, bt.cuda(), sl.cuda(), gs, gp, sl.cuda(), budget,
                                 recent=20, sinks=3)
    assert np.array_equal(got_new.cpu().numpy(), new)
    for got, w in zip((gk, gv), want[:2]):
        assert np.array_equal(f64(got), w)
    assert np.array_equal(gs.cpu().numpy(), want[2]) and np.array_equal(gp.cpu().numpy(), want[3])
    # the same moves again change nothing, and without state only the caches move
    m = evict.EvictionMoves(*(torch.from_numpy(x).cuda() for x in (src, dst, counts, new)))
    evict.compact_cache(gk, gv, bt.cuda(), m)
    assert np.array_equal(f64(gk), want[0]) and np.array_equal(f64(gv), want[1])


def test_append_and_compact_far_pages():
    """Pages past 2^31 elements of a cache (4.5 GB each) are written where the table says."""
    from bpt import evict
    bs, H, D = 256, 8, 128
    nb = (1 << 31) // (bs * H * D) + 16
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    k, v = (torch.empty(nb, bs, H, D, dtype=FP16, device="cuda") for _ in "kv")
    far = i32(nb - 1, nb - 5).view(1, 2)
    kn, vn = (torch.randn(1, 300, H, D, device="cuda").half() for _ in "kv")
    evict.append_tokens(k, v, kn, vn, i32(300), i32(0), far)
    src = torch.arange(299, 289, -1, device="cuda").int().expand(1, H, 10).contiguous()
    dst = torch.arange(10, device="cuda").int().expand(1, H, 10).contiguous()
    m = evict.EvictionMoves(src, dst, torch.full((1, H), 10, device="cuda").int(), i32(290))
    evict.compact_cache(k, v, far, m)
    for x, new in ((k, kn), (v, vn)):
        assert torch.equal(x[nb - 5, :44], new[0, 256:])
        assert torch.equal(x[nb - 1, 10:], new[0, 10:256])
        assert torch.equal(x[nb - 1, :10], new[0, 290:300].flip(0))


def test_compact_checked_mode(monkeypatch):
    from bpt import BptError, decode, evict
    monkeypatch.setattr(decode, "CHECKS", True)
    k, v = (torch.randn(4, 16, 1, 64, device="cuda").half() for _ in "kv")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    bt = i32(1, 2).view(1, 2)

    def moves(src, dst):
        return evict.EvictionMoves(i32(src, 20).view(1, 1, 2), i32(dst, 1).view(1, 1, 2),
                                   i32(2).view(1, 1), i32(16))
    before = k.clone()
    with pytest.raises(BptError, match="seq_len"):
        evict.compact_cache(k, v, bt, moves(32, 0))
    assert torch.equal(k[1, 1], before[2, 4])          # the valid move was made
    assert torch.equal(k[1, 0], before[1, 0])
    with pytest.raises(BptError, match="block_table"):
        evict.compact_cache(k, v, i32(1, 9).view(1, 2), moves(17, 0))


# ---------------------------------------------------------------------------- together

@pytest.mark.parametrize("maps", [1, 2])
def test_serving_loop(maps):
    """Prompt append, decode steps with scores, evictions whenever a sequence has grown by a page:
    after each step every kept token is the one that a list-based model of the cache keeps."""
    from bpt import diff, evict
    from oracle import evict as ox
    torch.manual_seed(maps)
    B, H, D, bs, budget, recent, sinks = 2, 2, 64, 16, 48, 12, 2
    mb = 8
    T = mb * bs
    heads = 4 * maps
    k = torch.zeros(B * mb, bs, maps * H, D, device="cuda", dtype=BF16)
    v = torch.zeros(B * mb, bs, H, maps * D, device="cuda", dtype=BF16)
    bt = torch.randperm(B * mb, device="cuda").reshape(B, mb).int()
    scores = torch.full((B, H, T), float("nan"), device="cuda")
    pos = torch.full((B, H, T), -1, device="cuda", dtype=torch.int32)
    sl, nxt = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2))
    lam = torch.tensor([0.3, 0.6, 0.2, 0.5], device="cuda")
    all_k = torch.zeros(B, 400, maps * H, D, device="cuda", dtype=BF16)
    all_v = torch.zeros(B, 400, H, maps * D, device="cuda", dtype=BF16)

    def append(S, lens):
        kn = torch.randn(B, S, maps * H, D, device="cuda").to(BF16)
        vn = torch.randn(B, S, H, maps * D, device="cuda").to(BF16)
        n = torch.tensor(lens, dtype=torch.int32, device="cuda")
        for b, m in enumerate(lens):
            all_k[b, int(nxt[b]):int(nxt[b]) + m] = kn[b, :m]
            all_v[b, int(nxt[b]):int(nxt[b]) + m] = vn[b, :m]
        evict.append_tokens(k, v, kn, vn, n, sl, bt, scores=scores, positions=pos, next_pos=nxt)
        sl.add_(n)
        nxt.add_(n)

    append(100, [100, 37])
    for step in range(40):
        append(1, [1, 1])
        q = torch.randn(B, heads, D, device="cuda").to(BF16)
        old = scores.clone()
        kw = dict(pair_bits=PAIR_BITS[BF16])
        if maps == 1:
            out = evict.paged_decode_attention_scored(q, k, v, bt, sl, scores)
        else:
            out = diff.paged_decode_attention_diff(q, k, v, bt, sl, lam, scores=scores)
            kw["lam"] = np.tile(f64(lam), (B, 1))
        ref, tol, added = ox.decode(f64(q), f64(k), f64(v), bt.cpu().numpy(), sl.tolist(), **kw)
        check_out(out, ref, tol, f"step {step}")
        check_scores(scores, old, added, sl.tolist(), 1.0, f"step {step}")
        if step % 16 == 0:
            want = ox.select(scores.cpu().numpy(), pos.cpu().numpy(), sl.cpu().numpy(),
                             nxt.cpu().numpy(), budget, recent, sinks)
            kk = k.view(B * mb, bs, H, maps * D)
            sl.copy_(evict.evict_tokens(kk, v, bt, sl, scores, pos, nxt, budget, recent=recent,
                                        sinks=sinks))
            assert np.array_equal(sl.cpu().numpy(), want[3])
        # what the cache says it holds at a slot is what was appended at that position
        for b in range(B):
            n = int(sl[b])
            t = torch.arange(n, device="cuda")
            page = bt[b].long()[t // bs]
            for h in range(H):
                at = pos[b, h, :n].long()
                assert len(set(at.tolist())) == n and int(at.max()) == int(nxt[b]) - 1
                assert set(range(int(nxt[b]) - min(recent, n), int(nxt[b]))) <= set(at.tolist())
                assert {0, 1} <= set(at.tolist())
                assert torch.equal(v[page, t % bs, h], all_v[b, at, h])
                kh = slice(maps * h, maps * h + maps)
                assert torch.equal(k[page, t % bs][:, kh], all_k[b, at][:, kh])


def test_step_captured_in_one_graph():
    """append, decode and eviction of a fixed batch captured once and replayed: lengths and
    positions advance on the device."""
    from bpt import evict
    torch.manual_seed(5)
    B, H, D, bs, mb, budget = 3, 2, 64, 16, 6, 64

    def fresh():
        g = torch.Generator(device="cuda").manual_seed(9)
        r = dict(k=torch.randn(B * mb, bs, H, D, generator=g, device="cuda").half(),
                 v=torch.randn(B * mb, bs, H, D, generator=g, device="cuda").half(),
                 scores=torch.rand(B, H, mb * bs, generator=g, device="cuda"),
                 sl=torch.tensor([64, 63, 10], dtype=torch.int32, device="cuda"))
        r["pos"] = torch.arange(mb * bs, device="cuda").int().expand(B, H, -1).contiguous()
        r["nxt"] = r["sl"].clone()
        return r
    bt = torch.randperm(B * mb, device="cuda").reshape(B, mb).int()
    one = torch.ones(B, dtype=torch.int32, device="cuda")
    q = torch.randn(B, 4, D, device="cuda").half()
    kn, vn = (torch.randn(B, 1, H, D, device="cuda").half() for _ in "kv")

    def step(s, out):
        evict.append_tokens(s["k"], s["v"], kn, vn, one, s["sl"], bt, scores=s["scores"],
                            positions=s["pos"], next_pos=s["nxt"])
        s["sl"] += one
        s["nxt"] += one
        evict.paged_decode_attention_scored(q, s["k"], s["v"], bt, s["sl"], s["scores"], out=out)
        s["sl"].copy_(evict.evict_tokens(s["k"], s["v"], bt, s["sl"], s["scores"], s["pos"],
                                         s["nxt"], budget, recent=8, sinks=2))

    eager, out_e = fresh(), torch.empty_like(q)
    warm = fresh()
    step(warm, torch.empty_like(q))
    captured, out_g = fresh(), torch.empty_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(captured, out_g)
    for t, x in fresh().items():
        captured[t].copy_(x)
    for _ in range(7):
        step(eager, out_e)
        g.replay()
        assert torch.equal(out_e, out_g)
    assert eager["sl"].tolist() == [64, 64, 17]
    for t in eager:
        assert torch.equal(eager[t], captured[t]), t
