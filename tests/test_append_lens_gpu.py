"""Lengths that an append cannot serve: flagged in checked mode, clamped without it."""
import pytest
import torch

pytestmark = pytest.mark.gpu

FP16 = torch.float16


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("S", [0, 1, 3])
@pytest.mark.parametrize("where", [0, 2])
def test_append_new_lens_outside_the_rows(monkeypatch, S, where):
    """More tokens than rows were given, or fewer than none, in the first or a later sequence. The
    caller's seq_lens + new_lens would cover slots that nobody wrote."""
    from bpt import BptError, decode, evict
    monkeypatch.setattr(decode, "CHECKS", True)
    k, v = (torch.zeros(6, 16, 2, 64, device="cuda", dtype=FP16) for _ in "kv")
    new = torch.ones(3, S, 2, 64, device="cuda", dtype=FP16)
    bt = i32(0, 1, 2, 3, 4, 5).view(3, 2)
    start = i32(4, 4, 4)

    def run(n, **kw):
        lens = [0, 0, 0]
        lens[where] = n
        evict.append_tokens(k, v, new, new, i32(*lens), start, bt, **kw)
    run(S)
    run(0)
    written = k.clone()
    assert int((written != 0).any(-1).any(-1).sum()) == S
    for bad in (S + 1, 1 << 30, -1):
        with pytest.raises(BptError, match="new_lens"):
            run(bad)
        # rows in hand are written all the same, and nothing else
        assert torch.equal(k, written) and torch.equal(v, written)
    monkeypatch.setattr(decode, "CHECKS", False)
    scores = torch.ones(3, 2, 32, device="cuda")
    run(S + 7, scores=scores)
    assert torch.equal(k, written)
    assert int((scores == 0).sum()) == 2 * S
