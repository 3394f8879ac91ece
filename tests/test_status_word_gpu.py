"""The status word when the first call of a process is being captured."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

SCRIPT = """
import torch
from avelang_b200 import _lib, gdn, linear_attention as L
bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
idx = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
pool, inside, beyond = torch.zeros(3, 2, 64, 64, device="cuda"), idx(0, 2), idx(0, 3)
args = bf(2, 1, 1, 64), bf(2, 1, 1, 64), bf(2, 1, 2, 64)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    L.fused_recurrent_linear_attention(*args, initial_state=pool, state_indices=inside)
assert gdn.read_status() == 0
L.fused_recurrent_linear_attention(*args, initial_state=pool, state_indices=beyond)
graph.replay()
assert gdn.read_status() == _lib.DEV_BAD_SLOT
graph.replay()
assert gdn.read_status() == 0
"""


def test_a_replay_leaves_what_other_calls_have_flagged(built_lib):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", SCRIPT], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
