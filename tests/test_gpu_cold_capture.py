"""The first calls of a process inside a capture: nothing they set up on first use may need an uncaptured call before."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import torch
from orca_amd import ops
w, vocab = 32, 500
g = torch.Generator().manual_seed(1)
lists = [torch.randint(0, vocab, (n,), generator=g).cuda() for n in (600, 8000, 9000)]
grads = [torch.randint(-8, 9, (i.numel(), w), generator=g).float().cuda() for i in lists]          # whole numbers: the sums are exact
table = torch.randn(vocab, w, generator=g).cuda()
many = [torch.randn(64, 33, generator=g).cuda() for _ in range(250)]
flat = [torch.empty(250 * 64 * 33, device="cuda")]
def calls():
  out = []
  for ids, grad in zip(lists, grads):
    r = ops.embedding_backward_rows(grad, ids, vocab)
    out += [ops.embedding(table, ids, 0.5), ops.embedding_backward(grad, ids, vocab), r.ids, r.rows, r.count]
  return out + [ops.clip_grad_norm(many, 1.0, flat=flat), flat[0]]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
  got = calls()
for k in range(3):
  for grad in grads:
    grad.add_(k)
  graph.replay()
  torch.cuda.synchronize()
  first = [x.clone() for x in got]
  want = calls()
  for i in range(3):
    n = int(want[5 * i + 4])
    assert int(first[5 * i + 4]) == n and torch.equal(first[5 * i + 2][:n], want[5 * i + 2][:n]) and torch.equal(first[5 * i + 3][:n], want[5 * i + 3][:n]), (k, i)
    assert torch.equal(first[5 * i], want[5 * i]) and torch.equal(first[5 * i + 1], want[5 * i + 1]), (k, i)
    ref = torch.zeros(vocab, w, device="cuda").index_add_(0, lists[i], grads[i])
    assert torch.equal(want[5 * i + 1], ref)
  assert torch.equal(first[-2], want[-2]) and torch.equal(first[-1], want[-1]), k
print("replays agree")
"""


def test_first_calls_in_a_capture():
  r = subprocess.run([sys.executable, "-c", PROGRAM], capture_output=True, text=True, timeout=100, cwd=ROOT)
  assert r.returncode == 0 and "replays agree" in r.stdout, r.stderr[-2000:]
