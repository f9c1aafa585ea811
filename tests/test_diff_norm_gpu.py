"""The differential decode's norm at its border: norm_eps 0 and rows of zeros."""
import numpy as np
import pytest
import torch

from evict_cases import PAIR_BITS, attend_case, check_out, f64

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("eps", [0.0, 1e-50, 1e-5])
def test_empty_sequence_with_a_norm(dtype, D, eps):
    """norm_eps 0 (and one that is 0 in fp32): an empty sequence gives zeros, the others are
    normalised by their mean square alone."""
    from bpt import diff
    from oracle import evict as ox
    lens = [0, 1, 40, 0, 700]
    c = attend_case(D, lens, 8, 2, D, 16, dtype, maps=2, garbage=float("nan"))
    lam = torch.linspace(0.1, 0.7, 4, device="cuda")
    w = torch.linspace(0.5, 1.5, 2 * D, device="cuda")
    for ns in (1, None):
        out = diff.paged_decode_attention_diff(c["q"], c["k"], c["v"], c["bt"], c["sl"], lam,
                                               norm_weight=w, norm_eps=eps, out_scale=0.2,
                                               num_splits=ns)
        assert (out[0] == 0).all() and (out[3] == 0).all()
        live = [1, 2, 4]
        ref, tol, _ = ox.decode(f64(c["q"])[live], f64(c["k"]), f64(c["v"]),
                                c["bt"].cpu().numpy()[live], [lens[b] for b in live],
                                lam=np.tile(f64(lam), (3, 1)), norm_weight=f64(w),
                                norm_eps=np.float32(eps).astype(np.float64), out_scale=0.2,
                                pair_bits=PAIR_BITS[dtype])
        check_out(out[live], ref, tol, f"eps {eps}, splits {ns}")


def test_values_of_zero_with_a_norm():
    """Values of 0 leave a row of zeros; NaN values leave NaN."""
    from bpt import diff
    c = attend_case(1, [30, 20], 2, 1, 64, 16, FP16, maps=2)
    lam = torch.full((1,), 0.5, device="cuda")
    w = torch.ones(128, device="cuda")

    def run():
        return diff.paged_decode_attention_diff(c["q"], c["k"], c["v"], c["bt"], c["sl"], lam,
                                                norm_weight=w, norm_eps=0.0)
    c["v"].zero_()
    assert (run() == 0).all()
    c["v"][c["bt"][1, 0].long()] = float("nan")
    out = run()
    assert (out[0] == 0).all() and torch.isnan(out[1]).all()
