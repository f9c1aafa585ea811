"""Host side of the scored decode, the append and the eviction: refusals of the Python entry points
(raised before anything is launched), the C ABI's own argument checks, workspace sizes, and the
float64 oracle against plain restatements."""
import ctypes

import numpy as np
import pytest
import torch

from bpt import BptArgumentError, _lib, diff, evict
from oracle import attention as oa
from oracle import evict as ox

c_i32, c_i64, c_f32, c_vp = ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p


class ScoredDecode(ctypes.Structure):
    """bpt_scored_decode (include/bpt.h)."""
    _fields_ = [(n, c_i32) for n in ("dtype", "maps", "batch", "q_heads", "kv_heads", "head_dim",
                                     "block_size", "max_blocks", "num_splits", "sm_count")] + \
               [(n, c_f32) for n in ("scale", "decay", "norm_eps", "out_scale")] + \
               [("num_blocks", c_i64), ("q", c_vp), ("q_stride", c_i64 * 2), ("k_cache", c_vp),
                ("k_stride", c_i64 * 3), ("v_cache", c_vp), ("v_stride", c_i64 * 3),
                ("block_table", c_vp), ("bt_stride", c_i64), ("seq_lens", c_vp), ("out", c_vp),
                ("out_stride", c_i64 * 2), ("scores", c_vp), ("scores_stride", c_i64 * 2),
                ("lam", c_vp), ("lam_stride", c_i64 * 2), ("norm_weight", c_vp)]


class PagedCache(ctypes.Structure):
    """bpt_paged_cache (include/bpt.h)."""
    _fields_ = [(n, c_i32) for n in ("block_size", "k_heads", "v_heads", "k_dim", "v_dim")] + \
               [("num_blocks", c_i64), ("k", c_vp), ("k_stride", c_i64 * 3), ("v", c_vp),
                ("v_stride", c_i64 * 3)]


def tensors(maps=1, dtype=torch.float16, B=2, Hq=4, H=2, D=64, bs=16, mb=2):
    """Valid arguments but for being on the CPU, which is the last thing to be refused."""
    return dict(q=torch.zeros(B, Hq, D, dtype=dtype),
                k=torch.zeros(4, bs, maps * H, D, dtype=dtype),
                v=torch.zeros(4, bs, H, maps * D, dtype=dtype),
                bt=torch.zeros(B, mb, dtype=torch.int32), sl=torch.zeros(B, dtype=torch.int32),
                scores=torch.zeros(B, H, mb * bs))


def scored(t, **kw):
    return evict.paged_decode_attention_scored(t["q"], t["k"], t["v"], t["bt"], t["sl"],
                                               t["scores"], **kw)


REFUSED = [
    ("no CPU", lambda t: None),
    ("dtype", lambda t: t.update(q=t["q"].bfloat16())),
    ("float16 or both", lambda t: t.update(k=t["k"].float(), v=t["v"].float(), q=t["q"].float())),
    ("head_dim", lambda t: t.update(q=torch.zeros(2, 4, 128, dtype=torch.float16))),
    ("multiple", lambda t: t.update(q=t["q"][:, :3])),
    ("power of two", lambda t: t.update(k=t["k"][:, :12], v=t["v"][:, :12])),
    ("same pages", lambda t: t.update(k=t["k"][:3])),
    ("heads for each head", lambda t: t.update(k=t["k"][:, :, :1])),
    ("block_table", lambda t: t.update(bt=t["bt"].long())),
    ("block_table", lambda t: t.update(bt=t["bt"][:1])),
    ("block_table", lambda t: t.update(bt=torch.zeros(2, 4, dtype=torch.int32)[:, ::2])),
    ("seq_lens", lambda t: t.update(sl=t["sl"].long())),
    ("seq_lens", lambda t: t.update(sl=torch.zeros(4, dtype=torch.int32)[::2])),
    ("scores must be float32", lambda t: t.update(scores=t["scores"].double())),
    ("scores must be float32", lambda t: t.update(scores=t["scores"][:, :, :31])),
    ("scores must be float32", lambda t: t.update(scores=torch.zeros(2, 2, 64)[:, :, ::2])),
    ("expanded", lambda t: t.update(scores=torch.zeros(2, 1, 32).expand(2, 2, 32))),
    ("unit inner", lambda t: t.update(q=torch.zeros(2, 4, 128, dtype=torch.float16)[:, :, ::2])),
    ("head_dim\\) stride", lambda t: t.update(k=torch.zeros(4, 16, 2, 128,
                                                           dtype=torch.float16)[..., ::2])),
]


@pytest.mark.parametrize("i", range(len(REFUSED)))
def test_scored_refusals(i):
    match, change = REFUSED[i]
    t = tensors()
    change(t)
    with pytest.raises(BptArgumentError, match=match):
        scored(t)


@pytest.mark.parametrize("decay", [-0.5, float("nan"), float("inf")])
def test_scored_refuses_decay(decay):
    with pytest.raises(BptArgumentError, match="decay"):
        scored(tensors(), decay=decay)


@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan"), float("inf")])
def test_refuses_scale(scale):
    """The C ABI takes a scale <= 0 for the default; Python has None for that."""
    with pytest.raises(BptArgumentError, match="scale"):
        scored(tensors(), scale=scale)
    t = tensors(maps=2)
    with pytest.raises(BptArgumentError, match="scale"):
        diff.paged_decode_attention_diff(t["q"], t["k"], t["v"], t["bt"], t["sl"],
                                         torch.zeros(2), scale=scale)


def test_scored_needs_scores():
    t = tensors()
    t["scores"] = None
    with pytest.raises(BptArgumentError, match="scores"):
        scored(t)


@pytest.mark.parametrize("match,kw", [
    ("no CPU", {}), ("lam", dict(lam=torch.zeros(3))), ("lam", dict(lam=torch.zeros(2).half())),
    ("lam", dict(lam=torch.zeros(3, 2))), ("lam", dict(lam=None)),
    ("norm_weight", dict(norm_weight=torch.ones(64))),
    ("norm_weight", dict(norm_weight=torch.ones(256)[::2])),
    ("norm_eps", dict(norm_weight=torch.ones(128), norm_eps=-1.0)),
    ("scores", dict(scores=torch.zeros(2, 4, 32)))])
def test_diff_refusals(match, kw):
    t = tensors(maps=2)
    args = dict(lam=torch.zeros(2), scores=t["scores"])
    args.update(kw)
    with pytest.raises(BptArgumentError, match=match):
        diff.paged_decode_attention_diff(t["q"], t["k"], t["v"], t["bt"], t["sl"], **args)
    with pytest.raises(BptArgumentError):     # an odd number of q heads
        diff.paged_decode_attention_diff(t["q"][:, :3], t["k"], t["v"], t["bt"], t["sl"],
                                         torch.zeros(1))


def test_binding_without_its_library():
    """The extension module alone, before bpt.evict gave it the library, refuses to work."""
    import subprocess
    import sys
    code = ("import sys, torch; sys.path.insert(0, %r); import bpt._bind as b\n"
            "t = torch.zeros(1, dtype=torch.int32)\n"
            "try: b.compact_cache(t, t, t, t, t, t, None, None, None)\n"
            "except RuntimeError as e: print('refused:', e)")
    import bpt
    import os
    r = subprocess.run([sys.executable, "-c",
                        code % os.path.dirname(os.path.dirname(bpt.__file__))],
                       capture_output=True, text=True, timeout=300)
    assert r.stdout.startswith("refused: bpt/_bind is used through"), r.stdout + r.stderr


def test_diff_lambda_refusals():
    v = torch.zeros(64)
    with pytest.raises(BptArgumentError):
        diff.diff_lambda(v, v, v, torch.zeros(32), 0.8, 4)
    with pytest.raises(BptArgumentError):
        diff.diff_lambda(*[torch.zeros(3, 64)] * 4, 0.8, 4)
    assert torch.equal(diff.diff_lambda(v, v, v, v, 0.5, 4), torch.full((4,), 0.5))


def test_append_refusals():
    t = tensors()
    new = torch.zeros(2, 3, 2, 64, dtype=torch.float16)
    pos = torch.zeros(2, 2, 32, dtype=torch.int32)

    def call(kn=new, vn=new, n=t["sl"], k=t["k"], **kw):
        evict.append_tokens(k, t["v"], kn, vn, n, t["sl"], t["bt"], **kw)
    for match, kw in (("no CPU", {}), ("k_new/v_new must be", dict(kn=new[:, :2])),
                      ("k_new/v_new must be", dict(vn=new[:, :, :1])),
                      ("cache's dtype", dict(kn=new.bfloat16())),
                      ("new_lens", dict(n=t["sl"].float())),
                      ("need next_pos", dict(positions=pos)),
                      ("positions must be", dict(positions=pos.float(), next_pos=t["sl"])),
                      ("positions must be", dict(positions=pos[..., :20], next_pos=t["sl"])),
                      ("expanded", dict(k=t["k"][:1].expand(4, 16, 2, 64)))):
        with pytest.raises(BptArgumentError, match=match):
            call(**kw)


def test_select_refusals():
    s, p, n = torch.zeros(2, 3, 40), torch.zeros(2, 3, 40, dtype=torch.int32), torch.zeros(
        2, dtype=torch.int32)

    def call(s=s, p=p, n=n, budget=8, **kw):
        return evict.select_evictions(s, p, n, n, budget, **kw)
    for match, kw in (("no CPU", {}), ("budget", dict(budget=0)), ("budget", dict(budget=-3)),
                      ("budget", dict(budget=1 << 31)), ("budget", dict(recent=-1)),
                      ("budget", dict(sinks=-1)), ("budget", dict(recent=5, sinks=4)),
                      ("budget", dict(recent=1 << 62, sinks=1 << 62)),
                      ("positions must be", dict(p=p.float())),
                      ("same slots", dict(p=p[..., :20])), ("seq_lens", dict(n=n[:1]))):
        with pytest.raises(BptArgumentError, match=match):
            call(**kw)


def test_compact_refusals():
    t = tensors()
    i32 = dict(dtype=torch.int32)
    m = evict.EvictionMoves(torch.zeros(2, 2, 5, **i32), torch.zeros(2, 2, 5, **i32),
                            torch.zeros(2, 2, **i32), torch.zeros(2, **i32))

    def call(k=t["k"], m=m, **kw):
        evict.compact_cache(k, t["v"], t["bt"], m, **kw)
    for match, kw in (("no CPU", {}), ("same heads", dict(k=t["k"][:, :, :1])),
                      ("moves", dict(m=m._replace(src=m.src[:, :, :4]))),
                      ("moves", dict(m=m._replace(counts=m.counts[:1]))),
                      ("moves must be contiguous", dict(m=m._replace(counts=m.counts.float()))),
                      ("scores", dict(scores=torch.zeros(2, 3, 32))),
                      ("unit inner", dict(scores=torch.zeros(2, 2, 1).expand(2, 2, 32))),
                      ("expanded", dict(scores=torch.zeros(2, 1, 32).expand(2, 2, 32)))):
        with pytest.raises(BptArgumentError, match=match):
            call(**kw)


# ------------------------------------------------------------------------------ the C ABI alone

def decode_args(**kw):
    a = ScoredDecode(dtype=1, maps=1, batch=1, q_heads=4, kv_heads=2, head_dim=64, block_size=16,
                     max_blocks=2, sm_count=148, decay=1.0, num_blocks=4)
    fake = 0x100000
    a.q = a.k_cache = a.v_cache = a.block_table = a.seq_lens = a.out = fake
    a.q_stride[:] = (256, 64)
    a.k_stride[:] = a.v_stride[:] = (2048, 128, 64)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("status,kw", [
    (_lib.ERR_INVALID_ARGUMENT, dict(maps=3)), (_lib.ERR_INVALID_ARGUMENT, dict(dtype=0)),
    (_lib.ERR_INVALID_ARGUMENT, dict(q_heads=5)), (_lib.ERR_INVALID_ARGUMENT, dict(batch=-1)),
    (_lib.ERR_INVALID_ARGUMENT, dict(q=None)), (_lib.ERR_INVALID_ARGUMENT, dict(block_table=None)),
    (_lib.ERR_INVALID_ARGUMENT, dict(maps=2)),                      # no lam
    (_lib.ERR_UNSUPPORTED_SHAPE, dict(q_heads=18)), (_lib.ERR_UNSUPPORTED_SHAPE, dict(head_dim=96)),
    (_lib.ERR_UNSUPPORTED_SHAPE, dict(head_dim=32)),
    (_lib.ERR_UNSUPPORTED_SHAPE, dict(maps=2, head_dim=256, lam=0x100000)),
    (_lib.ERR_UNSUPPORTED_SHAPE, dict(block_size=8)),
    (_lib.ERR_UNSUPPORTED_SHAPE, dict(block_size=512)),
    (_lib.ERR_UNSUPPORTED_SHAPE, dict(batch=65536)),
    (_lib.ERR_ALIGNMENT, dict(q=0x100002)), (0, dict(batch=0)),
])
def test_abi_decode_refusals(status, kw):
    a = decode_args(**kw)
    lib = _lib.lib()
    rc = lib.bpt_decode_scored(ctypes.byref(a), c_vp(0x200000), ctypes.c_size_t(1 << 30), None)
    assert rc == status


def test_abi_decode_workspace():
    lib = _lib.lib()
    lib.bpt_scored_workspace_bytes.restype = ctypes.c_size_t
    args = [c_i32(x) for x in (64, 1, 1, 4, 1)]
    with_scores = lib.bpt_scored_workspace_bytes(*args, c_i64(32))
    without = lib.bpt_scored_workspace_bytes(*args, c_i64(0))
    assert with_scores >= without + 4 * 32 * 4 and without >= 256 + 4 * 66 * 4
    # 64 sequences of 128k tokens, 32 rows: the logits alone pass 2^30 bytes
    big = lib.bpt_scored_workspace_bytes(*[c_i32(x) for x in (128, 1, 64, 32, 8)], c_i64(131072))
    assert big > 64 * 32 * 131072 * 4
    a = decode_args()
    for size, want in ((without - 1, _lib.ERR_WORKSPACE_TOO_SMALL),):
        assert lib.bpt_decode_scored(ctypes.byref(a), c_vp(0x200000), ctypes.c_size_t(size),
                                     None) == want
    assert lib.bpt_decode_scored(ctypes.byref(a), c_vp(0x200004), ctypes.c_size_t(1 << 30),
                                 None) == _lib.ERR_ALIGNMENT
    assert lib.bpt_decode_scored(None, None, ctypes.c_size_t(0), None) == _lib.ERR_INVALID_ARGUMENT


def test_abi_decode_splits():
    """One 32-token chunk a split while that is one wave of 4 (width 64: 5, 256: 2) CTAs an SM, else
    the decode planner's count; requests are clamped to the chunks."""
    f = _lib.lib().bpt_effective_splits_scored
    plan = _lib.lib().bpt_plan_splits

    def splits(*x):
        return f(*[c_i32(i) for i in x])
    assert splits(128, 1, 1, 8, 16, 64, 0, 148) == 32       # 1024 tokens, 256 CTAs
    assert splits(64, 2, 1, 8, 16, 64, 0, 148) == 32        # differential, the same width
    assert splits(128, 1, 1, 8, 16, 256, 0, 148) == plan(1, 8, 16, 256, 148) == 64
    assert splits(128, 1, 64, 8, 16, 4096, 0, 148) == plan(64, 8, 16, 4096, 148)
    assert splits(128, 2, 1, 8, 16, 128, 0, 148) == 32      # 512 CTAs of one chunk are 2 waves
    assert splits(128, 2, 8, 4, 32, 512, 0, 148) == 9       # 2 CTAs an SM: 296 / 32
    assert splits(64, 1, 1, 8, 16, 184, 0, 148) == 92       # 736 of 740 CTAs
    assert splits(128, 1, 2, 8, 16, 4, 7, 148) == 2
    assert splits(128, 1, 1, 8, 16, 0, 0, 148) == 1


def cache_args(**kw):
    c = PagedCache(block_size=16, k_heads=2, v_heads=2, k_dim=64, v_dim=64, num_blocks=4,
                   k=0x100000, v=0x200000)
    c.k_stride[:] = c.v_stride[:] = (2048, 128, 64)
    for n, v in kw.items():
        setattr(c, n, v)
    return c


@pytest.mark.parametrize("status,kw", [
    (_lib.ERR_INVALID_ARGUMENT, dict(k=None)), (_lib.ERR_INVALID_ARGUMENT, dict(k_heads=0)),
    (_lib.ERR_INVALID_ARGUMENT, dict(k_heads=4)), (_lib.ERR_UNSUPPORTED_SHAPE, dict(block_size=24)),
    (_lib.ERR_UNSUPPORTED_SHAPE, dict(block_size=512)), (_lib.ERR_ALIGNMENT, dict(k=0x100008)),
    (_lib.ERR_ALIGNMENT, dict(v_dim=60))])
def test_abi_compact_refusals(status, kw):
    c, p = cache_args(**kw), c_vp(0x300000)
    rc = _lib.lib().bpt_compact_cache(
        ctypes.byref(c), p, c_i64(2), c_i32(2), p, p, p, c_i32(4), c_i32(1), None, c_i64(0),
        c_i64(0), None, c_i64(0), c_i64(0), c_i32(32), None, None)
    assert rc == status


@pytest.mark.parametrize("status,kw", [
    (_lib.ERR_INVALID_ARGUMENT, dict(v=None)), (_lib.ERR_INVALID_ARGUMENT, dict(num_blocks=-1)),
    (_lib.ERR_UNSUPPORTED_SHAPE, dict(block_size=48))])
def test_abi_append_refusals(status, kw):
    c, p, st = cache_args(**kw), c_vp(0x300000), (c_i64 * 3)(128, 128, 64)
    rc = _lib.lib().bpt_append_tokens(
        ctypes.byref(c), p, st, p, st, p, p, p, c_i64(2), c_i32(2), c_i32(1), c_i32(1), None,
        c_i64(0), c_i64(0), None, c_i64(0), c_i64(0), None, None, None)
    assert rc == status


@pytest.mark.parametrize("budget,recent,sinks,alias", [(0, 0, 0, False), (8, 5, 4, False),
                                                       (8, -1, 0, False), (8, 0, 0, True)])
def test_abi_select_refusals(budget, recent, sinks, alias):
    p, other = c_vp(0x100000), c_vp(0x200000)
    rc = _lib.lib().bpt_select_evictions(
        p, c_i64(64), c_i64(32), p, c_i64(64), c_i64(32), p, p, c_i32(1), c_i32(2), c_i32(32),
        c_i32(budget), c_i32(recent), c_i32(sinks), other, other, other, p if alias else other,
        None)
    assert rc == _lib.ERR_INVALID_ARGUMENT


def test_abi_moves():
    f = _lib.lib().bpt_evict_moves
    assert [f(c_i32(b), c_i32(t)) for b, t in ((10, 12), (10, 100), (10, 10), (10, 4))] == \
        [2, 10, 1, 1]


# ------------------------------------------------------------------------------ the oracle

def test_oracle_decode_is_the_attention_oracle():
    """oracle.evict.decode against oracle.attention (fp32, pinned to the reference), and the weights
    against a direct softmax."""
    rng = np.random.default_rng(0)
    q = rng.standard_normal((2, 4, 16)).astype(np.float32)
    k, v = (rng.standard_normal((6, 8, 2, 16)).astype(np.float32) for _ in "kv")
    bt = np.array([[3, 1, 0], [5, 2, 4]], np.int32)
    out, tol, added = ox.decode(q, k, v, bt, [19, 8])
    ref = oa.paged_decode_attention_ref(q, k, v, bt, np.array([19, 8]))
    assert np.abs(out - ref).max() < 1e-5 and (tol > 0).all() and tol.max() < 1e-3
    for b, n in ((0, 19), (1, 8)):
        kk = ox.slots_of(k, bt[b], n)
        for h in range(2):
            x = q[b, 2 * h:2 * h + 2].astype(np.float64) @ kk[:, h].T / 4.0
            w = np.exp(x) / np.exp(x).sum(-1, keepdims=True)
            assert np.abs(added[b][0][h] - w.sum(0)).max() < 1e-12
        assert abs(added[b][0].sum() - 4.0) < 1e-12      # every q head hands out a weight of 1


def test_oracle_differential():
    """lam 0 is the first map alone; equal maps leave (1 - lam) of one."""
    rng = np.random.default_rng(1)
    q = rng.standard_normal((1, 4, 8))
    k, v = rng.standard_normal((2, 16, 2, 8)), rng.standard_normal((2, 16, 1, 16))
    bt, n = np.array([[1, 0]], np.int32), [23]
    one, _, _ = ox.decode(q[:, ::2], k[:, :, :1], v[..., :8], bt, n)
    zero, _, _ = ox.decode(q, k, v, bt, n, lam=np.zeros((1, 2)))
    assert np.abs(zero[..., :8] - one).max() < 1e-12
    q[:, 1::2], k[:, :, 1] = q[:, ::2], k[:, :, 0]
    third, _, added = ox.decode(q, k, v, bt, n, lam=np.full((1, 2), 1 / 3))
    zero, _, _ = ox.decode(q, k, v, bt, n, lam=np.zeros((1, 2)))
    assert np.abs(third - zero * 2 / 3).max() < 1e-12
    assert abs(added[0][0].sum() - 2 * 2 / 3) < 1e-12


def test_oracle_select_and_compact_keep_the_best():
    rng = np.random.default_rng(2)
    B, H, T, budget = 2, 2, 50, 20
    scores = rng.random((B, H, T)).astype(np.float32)
    pos = np.stack([rng.permutation(T) for _ in range(B * H)]).reshape(B, H, T).astype(np.int32)
    lens = np.array([50, 12])
    src, dst, counts, new = ox.select(scores, pos, lens, np.array([50, 50]), budget, 5, 2)
    assert new.tolist() == [20, 12] and (counts[1] == 0).all()
    s, p = (ox.compact_rows(x, src, dst, counts) for x in (scores, pos))
    for h in range(H):
        held = set(p[0, h, :budget].tolist())
        assert len(held) == budget and {0, 1} <= held and set(range(45, 50)) <= held
        rest = [float(x) for x, t in zip(scores[0, h], pos[0, h]) if t not in held]
        free = [float(x) for x, t in zip(s[0, h, :budget], p[0, h, :budget])
                if 2 <= t < 45]
        assert min(free) >= max(rest)
        assert np.array_equal(s[1], scores[1]) and np.array_equal(p[1], pos[1])
