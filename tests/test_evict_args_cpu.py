"""Arguments at the border of what the scored decode and the eviction accept: refused with an error
before anything is launched."""
import os
import subprocess
import sys


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
