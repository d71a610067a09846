"""The imaginary part of a conjugated tensor is a float view whose memory holds the values with the other sign."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
  from orca_amd import ops as o
  return o


def negated(*shape):
  z = torch.randn(*shape, dtype=torch.complex64, device=DEV)
  v = z.conj().imag
  assert v.is_neg()
  return z, v


def test_gradients_of_a_lookup(ops):
  ids = torch.tensor([1, 0, 1], device=DEV)
  for w in (1, 4):
    z, g = negated(3, w)
    assert torch.equal(ops.embedding_backward(g, ids, 2), ops.embedding_backward(-z.imag.contiguous(), ids, 2))
  z, g = negated(1, 1)
  assert torch.equal(ops.embedding_backward_rows(g, ids[:1], 2).rows, -z.imag)


def test_clipping(ops):
  for shape in ((1,), (5, 7)):
    z, g = negated(*shape)
    keep = z.clone()
    norm = ops.clip_grad_norm([g], 0.0)
    assert float(norm) > 0 and bool((g == 0).all()) and torch.equal(z.real, keep.real) and bool((z.imag == 0).all())
    z, g = negated(*shape)
    flat = torch.empty(g.numel(), device=DEV)
    ops.clip_grad_norm([g], 1e9, flat=[flat])
    assert torch.equal(flat.view(shape), -z.imag)


def test_what_cannot_be_read_as_it_lies(ops):
  _, v = negated(1, 1)
  ids = torch.zeros(1, dtype=torch.int64, device=DEV)
  plain, count = torch.ones(1, 1, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
  for call in (lambda: ops.embedding(v, ids), lambda: ops.embedding(plain, ids, out=v), lambda: ops.embedding_backward(plain, ids, 1, out=v),
               lambda: ops.embedding_backward_rows(plain, ids, 1, out=(ids.clone(), v, count)), lambda: ops.clip_grad_norm([plain], 1.0, flat=[v.view(1)]),
               lambda: ops.grad_norm([ops.RowGrad(ids, v, count, 1)])):
    with pytest.raises(ValueError):
      call()
