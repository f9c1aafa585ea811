"""How exactly the scored and the differential decode carry the softmax weights into the product with
the values. The values cancel or leave out what is large, so that the 16-bit rounding of the output
does not hide the weights' own error."""
import numpy as np
import pytest
import torch

from evict_cases import attend_case, f64

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


def bf16(x):
    """float64 values rounded to bf16, as float64."""
    return torch.tensor(x, dtype=torch.float64).bfloat16().double().numpy()


@pytest.mark.parametrize("G", [1, 4, 5, 8])
@pytest.mark.parametrize("maps", [1, 2])
def test_bf16_weights_keep_fp32_precision(G, maps):
    """Two tokens of weight 1 take away the first two bf16 limbs of the weight w of a third: what is
    left is the part of w that a pair of bf16 numbers cannot hold.

    q row g is 1 in its own channel only, so a logit is one exact product and x = k / 8 (log2: one
    rounding of the scale and one of the product, 2^-23 |x| with |x| <= 1, ln 2 of it in the weight);
    the exponential is off by 2^-22. At most 4 products of a 16-token tile are not 0, none above 1:
    2 tensor-core steps that truncate them at 2^-23 stay below 2^-20. So o L is off by at most
    2^-21.3 + 2^-20 < 2^-19.4, and a pair of limbs by up to 2^-18, as the test makes sure. The
    output's rounding, 2^-9 of something below 2^-17, and the quotient are covered by 2^-19.2."""
    if maps == 2 and G % 2:
        G += 1
    from bpt import diff, evict
    B, D, n = 24, 64, 3
    width = maps * D
    c = attend_case(G, [n] * B, G, 1, D, 16, BF16, maps=maps)
    g = torch.Generator().manual_seed(G)
    q = torch.zeros(B, G, D)
    for r in range(G):
        q[:, r, r] = 1.0
    kx = -(torch.rand(B, G, generator=g) * 4 + 1).bfloat16().double()       # logits -5/8 .. -1/8
    w = np.exp(kx.numpy() / 8)
    hi = bf16(w)
    mid = bf16(w - hi)
    rest = w - hi - mid
    assert np.abs(rest).max() > 2.0 ** -18.5 and (w > 0.5).all()   # a pair of limbs is off by this
    c["q"].copy_(q)
    c["k"].zero_()
    c["v"].zero_()
    rows = c["bt"][:, 0].long()
    for b in range(B):
        for r in range(G):
            # differential: row r meets key head r % 2
            c["k"][rows[b], 2, r % maps, r] = float(kx[b, r])
        for d in range(width):
            c["v"][rows[b], :3, 0, d] = torch.tensor([-hi[b, d % G], -mid[b, d % G], 1.0])
    L = 2 + w
    if maps == 1:
        out = evict.paged_decode_attention_scored(c["q"], c["k"], c["v"], c["bt"], c["sl"],
                                                  c["scores"])
        rows_of = [(r, r) for r in range(G)]
    else:
        # lam 0: the first map (even rows) alone
        out = diff.paged_decode_attention_diff(c["q"], c["k"], c["v"], c["bt"], c["sl"],
                                               torch.zeros(G // 2, device="cuda"))
        rows_of = [(r // 2, r) for r in range(0, G, 2)]
    got = f64(out)
    for j, r in rows_of:
        d = np.arange(r, width, G)
        want = (rest[:, r] / L[:, r])[:, None]
        assert (np.abs(got[:, j, d] - want) * L[:, r][:, None] <= 2.0 ** -19.2).all()


@pytest.mark.parametrize("G", [1, 4, 8])
@pytest.mark.parametrize("maps", [1, 2])
def test_fp16_tail_beside_a_sink(G, maps):
    """One token far above all the others, whose value is 0: the output is what the others, each of
    a tiny weight, leave. All in one split, so that the sink's warp holds half of them.

    The logits are single exact products as above, |x| <= 32 in log2: 2^-23 * 32 ln 2 of error in a
    weight, and 2^-22 of the exponential: below 2^-18.4. A weight is carried with 2^-22 of itself or
    2^-40 of the sink's. The sum of n equal terms adds sqrt(n) 2^-23, the joins 2^-20, the output's
    rounding 2^-11 of itself (nothing is below fp16's normal range)."""
    if maps == 2 and G % 2:
        G += 1
    from bpt import diff, evict
    n, D = 2000, 64
    nats = [4, 8, 12, 14, 17, 20]
    B, width = len(nats), maps * D
    c = attend_case(G, [n] * B, G, 1, D, 16, FP16, maps=maps)
    c["q"].zero_()
    c["q"][:, :, 0] = 1.0
    c["k"].zero_()
    c["v"].fill_(200.0)
    for b, x in enumerate(nats):
        pages = c["bt"][b, :n // 16].long()
        c["k"][pages, :, :, 0] = -8.0 * x
        c["k"][pages[0], 0] = 0.0
        c["v"][pages[0], 0] = 0.0
    if maps == 1:
        out = evict.paged_decode_attention_scored(c["q"], c["k"], c["v"], c["bt"], c["sl"],
                                                  c["scores"], num_splits=1)
    else:
        out = diff.paged_decode_attention_diff(c["q"], c["k"], c["v"], c["bt"], c["sl"],
                                               torch.zeros(G // 2, device="cuda"), num_splits=1)
    e = np.exp(-np.array(nats, np.float64))
    L = 1.0 + (n - 1) * e
    want = (n - 1) * e * 200.0 / L
    tol = want * (2.0 ** -18.4 + 2.0 ** -22 + np.sqrt(n) * 2.0 ** -23 + 2.0 ** -20) + \
        (n - 1) * 2.0 ** -40 * 200.0 / L
    got = f64(out).reshape(B, -1)
    assert want.min() > 2.0 ** -13
    worst = np.abs(got - want[:, None]).max(axis=1)
    assert (worst <= tol + (want + tol) * 2.0 ** -11).all(), worst / want
