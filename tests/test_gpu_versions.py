"""The calls that write into their caller's tensors count as in-place changes: autograd refuses a backward pass through a value that was
saved and then changed."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
  from orca_amd import ops as o
  return o


def writes(ops):
  """(what is written, the call)"""
  ids, grad, table = torch.tensor([1, 0, 2], device=DEV), torch.randn(3, 4, device=DEV), torch.randn(5, 4, device=DEV)
  f = lambda *s: torch.randn(*s, device=DEV)
  out, dense, g, h, flat, rows = f(3, 4), f(5, 4), f(6), f(4, 6), [f(30)], (ids.clone(), f(3, 4), torch.zeros(1, dtype=torch.int32, device=DEV))
  rg = ops.embedding_backward_rows(grad, ids, 5)
  return [([out], lambda: ops.embedding(table, ids, out=out)), ([dense], lambda: ops.embedding_backward(grad, ids, 5, out=dense)),
          ([dense], lambda: ops.embedding_backward(grad, ids, 5, out=dense, accumulate=True)),
          (list(rows), lambda: ops.embedding_backward_rows(grad, ids, 5, out=rows)),
          ([g, h[1:3], h[:1].t(), rg.rows], lambda: ops.clip_grad_norm([g, h[1:3], h[:1].t(), rg], 0.1)),
          (flat, lambda: ops.clip_grad_norm([g, h], 0.1, flat=flat))]


def test_versions_move(ops):
  for i, (tensors, call) in enumerate(writes(ops)):
    before = [t._version for t in tensors]
    call()
    assert all(t._version > v for t, v in zip(tensors, before)), i


def test_what_is_only_read_keeps_its_version(ops):
  ids, grad, table, g = torch.tensor([1, 0, 2], device=DEV), torch.randn(3, 4, device=DEV), torch.randn(5, 4, device=DEV), torch.randn(9, device=DEV)
  before = [t._version for t in (ids, grad, table, g)]
  ops.embedding(table, ids), ops.embedding_backward(grad, ids, 5), ops.embedding_backward_rows(grad, ids, 5)
  ops.grad_norm([g, table]), ops.clip_grad_norm([g], 0.1, flat=[torch.empty(9, device=DEV)])
  assert [t._version for t in (ids, grad, table, g)] == before


def test_a_saved_gradient_that_is_clipped(ops):
  """a gradient kept in a graph (create_graph=True), clipped in place, then differentiated"""
  x = torch.randn(8, device=DEV, requires_grad=True)
  grad, = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
  loss = grad.square().sum()
  ops.clip_grad_norm([grad], 1e-3)
  with pytest.raises(RuntimeError, match="inplace"):
    loss.backward()


def test_inference_tensors(ops):
  """they have no version: written as before"""
  with torch.inference_mode():
    g, out = torch.ones(16, device=DEV), torch.empty(2, 4, device=DEV)
  assert float(ops.clip_grad_norm([g], 1.0)) == 4.0 and bool((g < 1).all())
  ops.embedding(torch.ones(3, 4, device=DEV), torch.tensor([0, 2], device=DEV), out=out)
  assert bool((out == 1).all())
