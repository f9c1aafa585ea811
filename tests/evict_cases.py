"""Inputs and checks shared by the tests of the scored and differential decode and of eviction."""
import numpy as np
import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}   # half a subnormal step
PAIR_BITS = {torch.float16: 21, torch.bfloat16: 16}


def f64(t):
    return t.detach().double().cpu().numpy()


def attend_case(seed, lens, q_heads, kv_heads, D, bs, dtype, maps=1, spare=3, garbage=None,
                device="cuda"):
    """q, caches of random pages and a table that is wider than needed. ``garbage`` fills
    every slot that no sequence owns."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    pages = [(n + bs - 1) // bs for n in lens]
    mb = max(pages + [0]) + 1
    nb = sum(pages) + spare
    perm = torch.randperm(nb, generator=g)
    bt = torch.zeros(B, mb, dtype=torch.int32)
    used = torch.zeros(nb, bs, dtype=torch.bool)
    at = 0
    for b, p in enumerate(pages):
        bt[b, :p] = perm[at:at + p].int()
        at += p
        for i in range(p):
            used[bt[b, i], :min(bs, lens[b] - i * bs)] = True
    c = dict(q=torch.randn(B, q_heads, D, generator=g),
             k=torch.randn(nb, bs, maps * kv_heads, D, generator=g),
             v=torch.randn(nb, bs, kv_heads, maps * D, generator=g))
    if garbage is not None:
        c["k"][~used] = garbage
        c["v"][~used] = garbage
    c = {x: t.to(dtype).to(device) for x, t in c.items()}
    c.update(bt=bt.to(device), sl=torch.tensor(lens, dtype=torch.int32, device=device),
             T=mb * bs, scores=torch.rand(B, kv_heads, mb * bs, generator=g).to(device))
    return c


def check_out(out, ref, tol, what):
    got = f64(out)
    assert np.isfinite(got).all(), f"{what}: not finite"
    allow = tol + (np.abs(ref) + tol) * HALF_STEP[out.dtype] + SMALLEST[out.dtype]
    worst = np.max(np.abs(got - ref) / np.maximum(allow, 1e-300)) if ref.size else 0.0
    assert (np.abs(got - ref) <= allow).all(), f"{what}: {worst:.3g} of what fp32 may be off"


def check_scores(new, old, added, lens, decay, what):
    new, old = f64(new), f64(old)
    for b, (add, tol) in enumerate(added):
        n = int(lens[b])
        want = add + (decay * old[b, :, :n] if decay else 0.0)
        # the product with the decay and its sum are one or two fp32 roundings
        allow = tol + 2 * 2.0 ** -24 * (np.abs(want) + 2 * np.abs(add)) + 2.0 ** -149
        d = np.abs(new[b, :, :n] - want)
        assert (d <= allow).all(), f"{what}: sequence {b}, {np.max(d / allow):.3g} of the bound"
        assert np.array_equal(new[b, :, n:], old[b, :, n:], equal_nan=True), f"{what}: past {b}"
