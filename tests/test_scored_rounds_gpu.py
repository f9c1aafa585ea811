"""The scoring kernel as large batches run it: CTAs of several rounds, and logits that are dropped
from L2 once read. Wide tables around short sequences reach both with little data."""
import numpy as np
import pytest
import torch

from evict_cases import PAIR_BITS, attend_case, check_out, check_scores, f64

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16
B, HKV, D, BS = 4, 4, 64, 64
LENS = ([20011, 0, 3071, 5], [9000, 14001, 1, 2048])
TOKENS = 1024                 # of a round of a scoring CTA
CTAS = 3                      # scoring CTAs an SM past which a CTA takes a second round
DROP_BYTES = 32 << 20


def widen(c, T, offset):
    """The case in a table of T slots; score rows that start ``offset`` floats into a wider buffer."""
    bt = torch.zeros(B, T // BS, dtype=torch.int32, device="cuda")
    bt[:, :c["bt"].shape[1]] = c["bt"]
    g = torch.Generator(device="cuda").manual_seed(T)
    wide = torch.rand(B, HKV, T + 2 * offset, generator=g, device="cuda")
    c.update(bt=bt, wide=wide, scores=wide[:, :, offset:offset + T], T=T)
    return c


@pytest.mark.parametrize("decay,offset", [(0.0, 0), (0.5, 0), (0.5, 3)])
@pytest.mark.parametrize("drop", [False, True])
@pytest.mark.parametrize("maps,rows,dtype", [(1, 4, FP16), (1, 6, BF16), (2, 4, BF16),
                                             (2, 8, FP16), (1, 8, FP16), (1, 1, FP16)])
def test_rounds_and_dropped_logits(maps, rows, dtype, drop, decay, offset):
    """Two batches in turn through one workspace: every call rewrites lines that the last one
    dropped. The first batch again gives the same bits, and so does a workspace whose logits do
    not start at a line, which are never dropped."""
    from bpt import diff, evict
    from oracle import evict as ox
    q_heads = HKV * rows
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    T = 60 * TOKENS if not drop else max(60 * TOKENS, -(-DROP_BYTES // (B * q_heads * 4 * TOKENS)) *
                                         TOKENS)
    assert T // TOKENS * B * HKV >= 2 * CTAS * sms                     # two rounds at least
    assert (B * q_heads * T * 4 >= DROP_BYTES) == drop
    cases = [widen(attend_case(i + rows, lens, q_heads, HKV, D, BS, dtype, maps=maps), T, offset)
             for i, lens in enumerate(LENS)]
    lam = torch.linspace(-0.2, 0.8, q_heads // 2, device="cuda") if maps == 2 else None
    need = evict.scored_workspace_bytes(cases[0]["q"], cases[0]["k"], cases[0]["bt"], maps=maps)
    room = torch.empty(need + 256, dtype=torch.uint8, device="cuda")

    def run(c, ws):
        args = (c["q"], c["k"], c["v"], c["bt"], c["sl"])
        kw = dict(decay=decay, workspace=ws)
        if maps == 1:
            return evict.paged_decode_attention_scored(*args, c["scores"], **kw)
        return diff.paged_decode_attention_diff(*args, lam, scores=c["scores"], **kw)

    first = None
    for turn, (i, ws) in enumerate(((0, room[:need]), (1, room[:need]), (0, room[:need]),
                                    (0, room[16:16 + need]), (0, None))):
        c = cases[i]
        start = c["wide"].clone()
        out = run(c, ws)
        what = f"turn {turn}"
        if i == 0 and first is not None:
            assert torch.equal(out, first[0]) and torch.equal(c["wide"], first[1]), what
        else:
            ref, tol, added = ox.decode(
                f64(c["q"]), f64(c["k"]), f64(c["v"]), c["bt"].cpu().numpy(), LENS[i],
                lam=None if lam is None else np.tile(f64(lam), (B, 1)),
                pair_bits=PAIR_BITS[dtype])
            check_out(out, ref, tol, what)
            check_scores(c["scores"], start[:, :, offset:offset + T], added, LENS[i], decay, what)
            assert torch.equal(c["wide"][:, :, :offset], start[:, :, :offset])
            assert torch.equal(c["wide"][:, :, offset + T:], start[:, :, offset + T:])
            if i == 0:
                first = (out.clone(), c["wide"].clone())
        c["wide"].copy_(start)


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("D,Hq,Hkv", [(64, 3, 1), (128, 8, 2), (256, 10, 2)])
def test_one_map_without_scores(dtype, D, Hq, Hkv):
    """maps 1 with no scores (`scores` NULL in the C ABI): the output of the scored call, bit for bit,
    from a workspace without logits."""
    from bpt import evict
    c = attend_case(D, [0, 1, 33, 500, 2100], Hq, Hkv, D, 32, dtype, garbage=float("nan"))
    want = evict.paged_decode_attention_scored(c["q"], c["k"], c["v"], c["bt"], c["sl"],
                                               c["scores"])
    need = evict.scored_workspace_bytes(c["q"], c["k"], c["bt"], scored=False)
    assert need < evict.scored_workspace_bytes(c["q"], c["k"], c["bt"])
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    for w in (ws, None):
        out = evict._bind().decode_scored(1, c["q"], c["k"], c["v"], c["bt"], c["sl"], None, None,
                                          None, 1.0, None, w, None, None, 0.0, 1.0)
        assert torch.equal(out, want)
