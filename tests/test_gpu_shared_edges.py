"""Decode plans and their attention where they can go wrong: caches of several head dims in one
process, reorders that cross a plan's groups, replays after other sets, values that are not
finite."""
import os
import subprocess
import sys

import pytest
import torch

from test_gpu_shared_attention import Batch, _rand, _turn, layout  # noqa: F401 (layout: autouse)

pytestmark = pytest.mark.gpu

sb = pytest.importorskip("synapse_b200")

U = 2.0 ** -24


def _attend(b, plan=None, rows=None, layer=0, window=0):
    """One call for the rows (sequences) of a plan; output rows in the order of `rows`."""
    qkv = b.qkv if rows is None else b.qkv[rows].contiguous()
    return sb.attention_decode_shared(plan or b.plan, layer, qkv, None, None, 1e-6, b.cos, b.sin, window=window)


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


ASCENDING = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import synapse_b200 as sb
from test_gpu_shared_attention import Batch
ctx = sb.Context(0)
for hd in (20, 32, 36, 60, 72, 80, 96, 112, 124):
    Batch(ctx, 1, 2, hd, 16, [70], [[1, 2]], seed=hd).check()
print("ascending ok")
"""


def test_head_dims_in_ascending_order():
    """A process whose caches get wider heads one after another (a kernel's shared memory grows
    with the head dim): in a process of its own, since others may have come in another order."""
    tests = os.path.dirname(os.path.abspath(__file__))
    code = ASCENDING.format(root=os.path.dirname(tests), tests=tests)
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=600)
    assert out.returncode == 0 and "ascending ok" in out.stdout, out.stdout + out.stderr
