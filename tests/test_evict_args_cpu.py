"""Arguments at the border of what the scored decode and the eviction accept: refused with an error
before anything is launched."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from bpt import BptArgumentError, _lib, diff
from test_evict_cpu import cache_args, decode_args, scored, tensors

c_i32, c_i64, c_vp = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p
FLOAT_MAX = torch.finfo(torch.float32).max


def test_workspace_of_an_operator_that_does_not_exist():
    """maps 0 divided by zero, which ends the process: asked in one of its own."""
    import bpt
    code = ("import sys, torch; sys.path.insert(0, %r); from bpt import evict\n"
            "q = torch.zeros(2, 4, 64, dtype=torch.float16)\n"
            "k = torch.zeros(4, 16, 2, 64, dtype=torch.float16)\n"
            "bt = torch.zeros(2, 2, dtype=torch.int32)\n"
            "for maps in (0, 3, -1):\n"
            "    try: evict.scored_workspace_bytes(q, k, bt, 1, maps=maps)\n"
            "    except ValueError as e: print('refused:', e)\n"
            "for x in (q[:, :0], q[..., :0]):\n"
            "    try: evict.scored_workspace_bytes(x, k, bt, 1)\n"
            "    except ValueError as e: print('refused:', e)\n"
            "for x, maps in ((k[:, :, :0], 1), (k[:, :, :1], 2)):\n"
            "    try: evict.scored_workspace_bytes(q, x, bt, 1, maps=maps)\n"
            "    except ValueError as e: print('refused:', e)\n")
    r = subprocess.run([sys.executable, "-c",
                        code % os.path.dirname(os.path.dirname(bpt.__file__))],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr)
    assert r.stdout.count("refused:") == 7, r.stdout


@pytest.mark.parametrize("scale", [1e-50, 1e39, FLOAT_MAX])
def test_scale_that_fp32_cannot_hold(scale):
    """1e-50 is 0 in fp32, which the C ABI takes for the default; log2(e) of the largest is infinite."""
    with pytest.raises(BptArgumentError, match="scale"):
        scored(tensors(), scale=scale)
    t = tensors(maps=2)
    with pytest.raises(BptArgumentError, match="scale"):
        diff.paged_decode_attention_diff(t["q"], t["k"], t["v"], t["bt"], t["sl"],
                                         torch.zeros(2), scale=scale)


def test_small_scale_is_no_error():
    with pytest.raises(BptArgumentError, match="no CPU"):
        scored(tensors(), scale=1e-40)


@pytest.mark.parametrize("decay", [1e39, 1e300])
def test_decay_that_fp32_cannot_hold(decay):
    with pytest.raises(BptArgumentError, match="decay"):
        scored(tensors(), decay=decay)


@pytest.mark.parametrize("eps", [1e39, float("inf"), float("nan")])
def test_norm_eps_that_fp32_cannot_hold(eps):
    t = tensors(maps=2)
    with pytest.raises(BptArgumentError, match="norm_eps"):
        diff.paged_decode_attention_diff(t["q"], t["k"], t["v"], t["bt"], t["sl"], torch.zeros(2),
                                         norm_weight=torch.ones(128), norm_eps=eps)


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("status,kw", [
    (_lib.ERR_INVALID_ARGUMENT, dict(scale=NAN)), (_lib.ERR_INVALID_ARGUMENT, dict(scale=INF)),
    (_lib.ERR_INVALID_ARGUMENT, dict(scale=FLOAT_MAX)),
    (_lib.ERR_INVALID_ARGUMENT, dict(scores=0x300000, decay=NAN)),
    (_lib.ERR_INVALID_ARGUMENT, dict(scores=0x300000, decay=INF)),
    (_lib.ERR_INVALID_ARGUMENT, dict(maps=2, lam=0x300000, norm_weight=0x310000, norm_eps=NAN)),
    (_lib.ERR_INVALID_ARGUMENT, dict(maps=2, lam=0x300000, norm_weight=0x310000, norm_eps=-1.0)),
    # what is not used is not looked at: these get as far as the workspace
    (_lib.ERR_WORKSPACE_TOO_SMALL, dict(scale=-1.0)), (_lib.ERR_WORKSPACE_TOO_SMALL,
                                                       dict(decay=NAN)),
    (_lib.ERR_WORKSPACE_TOO_SMALL, dict(maps=2, lam=0x300000, norm_eps=NAN)),
])
def test_abi_numbers(status, kw):
    rc = _lib.lib().bpt_decode_scored(ctypes.byref(decode_args(**kw)), c_vp(0x200000),
                                      ctypes.c_size_t(16), None)
    assert rc == status


# B=3, 2 kv heads, 32 slots, budget 8: 6 rows of 8 moves. Addresses of non-overlapping arrays.
SELECT = dict(scores=0x100000, positions=0x110000, seq_lens=0x120000, next_pos=0x121000,
              src=0x130000, dst=0x131000, counts=0x132000, new_lens=0x133000)


def select_rc(batch=3, slots=32, pos_sb=64, pos_sh=32, **kw):
    """bpt_select_evictions at these addresses, refused before a launch in every case used here."""
    a = {k: c_vp(v) for k, v in {**SELECT, **kw}.items()}
    return _lib.lib().bpt_select_evictions(
        a["scores"], c_i64(64), c_i64(32), a["positions"], c_i64(pos_sb), c_i64(pos_sh),
        a["seq_lens"], a["next_pos"], c_i32(batch), c_i32(2), c_i32(slots), c_i32(8), c_i32(0),
        c_i32(0), a["src"], a["dst"], a["counts"], a["new_lens"], None)


@pytest.mark.parametrize("kw", [
    dict(new_lens=SELECT["next_pos"]), dict(new_lens=SELECT["next_pos"] + 8),
    dict(new_lens=SELECT["seq_lens"] - 8), dict(new_lens=SELECT["seq_lens"]),
    dict(counts=SELECT["seq_lens"] - 20), dict(src=SELECT["next_pos"] - 4 * 47),
    dict(dst=SELECT["seq_lens"]), dict(dst=SELECT["src"] + 4 * 47),
    dict(counts=SELECT["new_lens"] - 20), dict(src=SELECT["scores"] + 4 * 191),
    dict(src=SELECT["positions"] - 4 * 47),
    dict(dst=SELECT["positions"] - 4 * 128, pos_sb=-64)])
def test_abi_select_results_on_inputs(kw):
    """One CTA writes new_lens and the moves that others of the row have still to read the inputs
    of: overlapping arrays are refused, shifted ones too."""
    assert select_rc(**kw) == _lib.ERR_INVALID_ARGUMENT


def test_abi_select_neighbours_are_no_overlap():
    """Arrays that touch pass the check: with 2^26 sequences the next refusal is the grid's size."""
    far = {k: i << 40 for i, k in enumerate(SELECT, 1)}
    end = far["src"] + 4 * (1 << 27) * 8
    assert select_rc(batch=1 << 26, **{**far, "dst": end}) == _lib.ERR_UNSUPPORTED_SHAPE
    assert select_rc(batch=1 << 26, **{**far, "dst": end - 4}) == _lib.ERR_INVALID_ARGUMENT


INT32_MAX = 2 ** 31 - 1


@pytest.mark.parametrize("word,status", [
    (INT32_MAX, _lib.ERR_UNSUPPORTED_SHAPE), (INT32_MAX - 1, _lib.ERR_INVALID_ARGUMENT),
    ((1 << 34) - 3, _lib.ERR_UNSUPPORTED_SHAPE), ((1 << 34) - 2, _lib.ERR_INVALID_ARGUMENT),
    (5 << 33, _lib.ERR_UNSUPPORTED_SHAPE), ((1 << 37) + (1 << 34) + 5, _lib.ERR_INVALID_ARGUMENT)])
def test_abi_select_results_between_rows(word, status):
    """new_lens (3 words) in the room between two rows of positions is no overlap, and on a row it is.
    Rows of 2^31 - 1 slots, 2^34 words apart: what passes is refused for that length afterwards."""
    far = {k: i << 50 for i, k in enumerate(SELECT, 1)}
    far["new_lens"] = far["positions"] + 4 * word
    assert select_rc(slots=INT32_MAX, pos_sb=1 << 36, pos_sh=1 << 34, **far) == status


@pytest.mark.parametrize("bs,max_blocks,status", [
    (16, INT32_MAX // 16, _lib.ERR_UNSUPPORTED_SHAPE),          # 2^31 - 16 slots
    (32, INT32_MAX // 32, _lib.ERR_UNSUPPORTED_SHAPE),
    (16, INT32_MAX // 16 - 2, _lib.ERR_WORKSPACE_TOO_SMALL)])
def test_abi_decode_next_to_2_31_slots(bs, max_blocks, status):
    """The last chunk's end has to be an int too."""
    a = decode_args(block_size=bs, max_blocks=max_blocks)
    assert _lib.lib().bpt_decode_scored(ctypes.byref(a), c_vp(0x200000), ctypes.c_size_t(16),
                                        None) == status


@pytest.mark.parametrize("slots", [INT32_MAX, INT32_MAX - 2000])
def test_abi_select_next_to_2_31_slots(slots):
    """A cluster's last slice ends up to 16 tiles past the row: refused where that passes an int."""
    far = {k: i << 40 for i, k in enumerate(SELECT, 1)}
    assert select_rc(slots=slots, **far) == _lib.ERR_UNSUPPORTED_SHAPE


@pytest.mark.parametrize("moves", [INT32_MAX, INT32_MAX - 100])
def test_abi_compact_next_to_2_31_moves(moves):
    c, p = cache_args(), c_vp(0x300000)
    rc = _lib.lib().bpt_compact_cache(
        ctypes.byref(c), p, c_i64(2), c_i32(2), p, p, p, c_i32(moves), c_i32(1), None, c_i64(0),
        c_i64(0), None, c_i64(0), c_i64(0), c_i32(32), None, None)
    assert rc == _lib.ERR_UNSUPPORTED_SHAPE
