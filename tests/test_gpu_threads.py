"""Calls from several threads at once, in a process whose first calls these are (a kernel's LDS is allowed on its first use)."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu

PROGRAM = """
import threading
import torch
from orca_amd import ops
ops._load_host()
n, w, vocab, threads = 8000, 32, 500, 6
g = torch.Generator().manual_seed(1)
ids = torch.randint(0, vocab, (n,), generator=g).cuda()
grad = torch.randint(-8, 9, (n, w), generator=g).float().cuda()          # whole numbers: the sums are exact
want = torch.zeros(vocab, w, device="cuda").index_add_(0, ids, grad)
torch.cuda.synchronize()
start, bad = threading.Barrier(threads), []
def call(k):
  with torch.cuda.stream(torch.cuda.Stream()):
    start.wait()
    try:
      for _ in range(3):
        if k % 2:
          got = ops.embedding_backward(grad, ids, vocab)
        else:
          r = ops.embedding_backward_rows(grad, ids, vocab)
          got = torch.zeros(vocab, w, device="cuda")
          got[r.ids[:int(r.count)]] = r.rows[:int(r.count)]
        torch.cuda.current_stream().synchronize()
        if not torch.equal(got, want):
          bad.append((k, "differs"))
    except Exception as e:
      bad.append((k, repr(e)))
ts = [threading.Thread(target=call, args=(k,)) for k in range(threads)]
[t.start() for t in ts]
[t.join() for t in ts]
assert not bad, bad
print("threads agree")
"""


def test_first_calls_of_several_threads():
  r = subprocess.run([sys.executable, "-c", PROGRAM], capture_output=True, text=True, timeout=100, cwd=ROOT)
  assert r.returncode == 0 and "threads agree" in r.stdout, r.stderr[-2000:]
