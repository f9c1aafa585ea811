"""Differential decode on the GPU against oracle.evict (float64)."""
import numpy as np
import pytest
import torch

from evict_cases import PAIR_BITS, attend_case, check_out, check_scores, f64

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


def run_diff(c, lam, dtype, scored=True, norm=None, decay=1.0, out_scale=1.0, what="", **kw):
    from bpt import diff
    from oracle import evict as ox
    B, H = c["q"].shape[0], c["q"].shape[1] // 2
    old = c["scores"].clone()
    out = diff.paged_decode_attention_diff(
        c["q"], c["k"], c["v"], c["bt"], c["sl"], lam, norm_weight=norm, out_scale=out_scale,
        scores=c["scores"] if scored else None, decay=decay, **kw)
    ref, tol, added = ox.decode(
        f64(c["q"]), f64(c["k"]), f64(c["v"]), c["bt"].cpu().numpy(), c["sl"].tolist(),
        lam=np.broadcast_to(f64(lam), (B, H)), norm_weight=None if norm is None else f64(norm),
        out_scale=out_scale, pair_bits=PAIR_BITS[dtype])
    check_out(out, ref, tol, what)
    if scored:
        check_scores(c["scores"], old, added, c["sl"].tolist(), decay, what)
    else:
        assert torch.equal(c["scores"], old)
    return out


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 2), (3, 1), (8, 2)])
@pytest.mark.parametrize("norm", [False, True])
def test_diff_head_layouts(dtype, D, H, Hkv, norm):
    lens = [0, 1, 15, 16, 33, 200, 1100]
    lam = torch.linspace(-0.3, 0.9, H, device="cuda")
    w = torch.linspace(0.5, 1.5, 2 * D, device="cuda") if norm else None
    for ns, scored in ((1, True), (3, False), (None, True)):
        c = attend_case(D + H, lens, 2 * H, Hkv, D, 16, dtype, maps=2, garbage=float("nan"))
        run_diff(c, lam, dtype, scored=scored, norm=w, out_scale=0.2 if norm else 1.0,
                 num_splits=ns, what=f"splits={ns}")


@pytest.mark.parametrize("bs", [16, 64, 256])
@pytest.mark.parametrize("decay", [1.0, 0.5, 0.0])
def test_diff_pages_decay_and_lam_by_token(bs, decay):
    c = attend_case(bs, [1, bs - 1, bs, 5 * bs + 7], 8, 2, 64, bs, BF16, maps=2)
    if decay == 0.0:
        c["scores"].fill_(float("nan"))
    lam = torch.rand(4, 8, device="cuda")[:, ::2]                 # [B, H], strided
    run_diff(c, lam, BF16, decay=decay)


def test_diff_lam_zero_is_the_first_map():
    """lam 0 leaves plain attention of the even q heads over the even key heads."""
    from bpt import diff, evict
    c = attend_case(3, [500, 40], 8, 2, 64, 16, FP16, maps=2)
    s1, s2 = c["scores"].clone(), c["scores"].clone()
    out = diff.paged_decode_attention_diff(c["q"], c["k"], c["v"], c["bt"], c["sl"],
                                           torch.zeros(4, device="cuda"), scores=s1)
    for half in range(2):
        want = evict.paged_decode_attention_scored(
            c["q"][:, ::2].contiguous(), c["k"][:, :, ::2].contiguous(),
            c["v"][..., 64 * half:64 * half + 64].contiguous(), c["bt"], c["sl"],
            s2 if half == 0 else c["scores"])
        got = out[..., 64 * half:64 * half + 64]
        assert ((got.float() - want.float()).abs() <= want.float().abs() * 2.0 ** -10 + 1e-5).all()
    assert torch.allclose(s1, s2, rtol=1e-5, atol=1e-7)


def test_diff_equal_maps_cancel():
    """lam 1 and two equal maps: every weight is 0, so out is 0 and the norm divides by no 0."""
    c = attend_case(4, [70, 3], 4, 2, 64, 16, FP16, maps=2)
    c["q"][:, 1::2] = c["q"][:, ::2]
    c["k"][:, :, 1::2] = c["k"][:, :, ::2]
    from bpt import diff
    out = diff.paged_decode_attention_diff(c["q"], c["k"], c["v"], c["bt"], c["sl"],
                                           torch.ones(2, device="cuda"),
                                           norm_weight=torch.ones(128, device="cuda"))
    assert torch.isfinite(out).all()
    # both maps' fp32 weights differ by rounding at most: |o| <= 2 * 2^-18 * max|v|, over sqrt(eps)
    assert out.abs().max().item() <= 2.0 ** -17 * 6.0 / 1e-5 ** 0.5


def test_diff_views_and_graph():
    from bpt import diff
    c = attend_case(5, [300, 41], 12, 2, 128, 32, FP16, maps=2)
    lam = torch.rand(6, device="cuda")
    w = torch.rand(256, device="cuda")
    kw = dict(norm_weight=w, out_scale=0.5)
    want = diff.paged_decode_attention_diff(c["q"], c["k"], c["v"], c["bt"], c["sl"], lam, **kw)
    k, v = (c[x].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in "kv")
    out = diff.paged_decode_attention_diff(c["q"], k, v, c["bt"], c["sl"], lam, **kw)
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = diff.paged_decode_attention_diff(c["q"], c["k"], c["v"], c["bt"], c["sl"], lam, **kw)
    got.zero_()
    g.replay()
    assert torch.equal(got, want)


def test_diff_lambda():
    from bpt import diff
    v = [torch.randn(64, dtype=torch.bfloat16) * 0.1 for _ in range(4)]
    lam = diff.diff_lambda(*v, 0.8, 5)
    a, b, c, d = (x.double() for x in v)
    want = torch.exp(a @ b) - torch.exp(c @ d) + 0.8
    assert lam.shape == (5,) and (lam.double() - want).abs().max() < 1e-6
