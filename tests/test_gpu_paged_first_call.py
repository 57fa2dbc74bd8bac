"""The first paged call of a process on a device makes the word that all later ones report in. It is not made inside a capture, where it
would belong to the graph and be zeroed by every replay, so that what an eager call reports would be lost."""
import os
import subprocess
import sys
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
gpu = pytest.mark.gpu

PROGRAM = """
import torch
from thunderworld_b200 import ops
z = lambda *s, dtype=torch.int32: torch.zeros(s, dtype=dtype, device='cuda')
q, pool, table, lengths = z(2, 4, 64, dtype=torch.bfloat16), z(3, 2, 16, 64, dtype=torch.bfloat16), z(2, 5), z(2)
calls = [lambda: ops.paged_attention(q, pool, pool, table, lengths), lambda: ops.cache_free_(table, lengths, z(3) if not capturing else refs, slots, 16)]
refs, slots, capturing = z(3), z(1) + 7, True
torch.cuda.synchronize()
for call in calls:
    refused = False
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            call()
    except RuntimeError as e:
        refused = 'cannot be captured' in str(e)
    assert refused
assert ops.device_status() == 0
capturing = False
calls[0]()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    calls[0]()
calls[1]()                               # a slot outside: reported, and not taken back by a replay
graph.replay()
assert ops.device_status() == 11
print('done')
"""


@gpu
def test_the_first_paged_call_is_not_captured():
    run = subprocess.run([sys.executable, '-c', PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip().endswith('done'), run.stderr[-2000:]
