"""Derivatives of torch.ops.orca.embedding beyond the first: against plain indexing, on the CPU with stand-ins for the two kernels (the
registration is what is tested) and on the GPU with the kernels."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from orca_amd import ops, torch_ops  # noqa: F401

V, W = 9, 5
IDS = torch.tensor([[3, 0, 3], [8, 2, 3]])


def plain(table, ids, scale, padding_idx):
  """the same lookup by indexing: the padding id's row enters as a constant"""
  rows = table[ids]
  if padding_idx >= 0:
    rows = torch.where((ids == padding_idx).unsqueeze(-1), rows.detach(), rows)
  return rows * scale


@pytest.fixture
def stand_ins(monkeypatch):
  def embedding(table, ids, scale=1.0, out=None):
    return table.detach()[ids.clamp(min=0)] * scale * (ids >= 0).unsqueeze(-1)

  def embedding_backward(g, ids, num_rows, scale=1.0, padding_idx=None):
    ids, g = ids.reshape(-1), g.detach().reshape(-1, g.shape[-1])
    keep = (ids >= 0) & (ids != padding_idx)
    return torch.zeros(num_rows, g.shape[1], dtype=g.dtype).index_add_(0, ids[keep], g[keep]) * scale
  monkeypatch.setattr(ops, "embedding", embedding)
  monkeypatch.setattr(ops, "embedding_backward", embedding_backward)


def penalty(look, table, weight, ids, scale, padding):
  """a loss with a gradient penalty beside another term: its gradient, and the penalty's part of it"""
  out = look(table, ids, scale, padding)
  grad, = torch.autograd.grad((out ** 3 * weight).sum(), table, create_graph=True)
  pen, = torch.autograd.grad(grad.square().sum(), table, retain_graph=True)
  both, = torch.autograd.grad(out.sum() + grad.square().sum(), table)
  return grad.detach(), pen, both


@pytest.mark.parametrize("padding", [-1, 3])
def test_second_derivative(stand_ins, padding):
  g = torch.Generator().manual_seed(1)
  table = torch.randn(V, W, generator=g, dtype=torch.float64, requires_grad=True)
  weight = torch.randn(2, 3, W, generator=g, dtype=torch.float64)
  got = penalty(torch.ops.orca.embedding, table, weight, IDS, 0.5, padding)
  want = penalty(plain, table, weight, IDS, 0.5, padding)
  for a, b in zip(got, want):
    assert torch.allclose(a, b, rtol=1e-12, atol=1e-12) and bool((b != 0).any())
  look = lambda t: torch.ops.orca.embedding(t, IDS, 0.5, -1) ** 3 * weight
  assert torch.autograd.gradcheck(look, (table,)) and torch.autograd.gradgradcheck(look, (table,))


def test_gradient_of_the_gradient_alone(stand_ins):
  """the gradient is linear in what came in: its own derivative is the lookup"""
  grad_out = torch.randn(2, 3, W, dtype=torch.float64, requires_grad=True)
  other = torch.randn(V, W, dtype=torch.float64)
  d, = torch.autograd.grad((torch.ops.orca.embedding_backward(grad_out, IDS, V, 2.0, 3) * other).sum(), grad_out)
  assert torch.equal(d, other[IDS] * 2.0 * (IDS != 3).unsqueeze(-1))


def test_forward_mode_raises(stand_ins):
  """a tangent is not dropped, whether the table requires a gradient or not"""
  table = torch.randn(V, W)
  look = lambda t: torch.ops.orca.embedding(t, IDS, 1.0, -1)
  with fwd.dual_level():
    for t in (table, table.clone().requires_grad_()):
      with pytest.raises(NotImplementedError):
        look(fwd.make_dual(t, torch.ones_like(table)))
    assert torch.equal(look(table), table[IDS])                       # a table without a tangent
    with pytest.raises(NotImplementedError):
      torch.ops.orca.embedding_backward(fwd.make_dual(torch.randn(2, 3, W), torch.randn(2, 3, W)), IDS, V, 1.0, -1)
  with pytest.raises(NotImplementedError):
    torch.func.jvp(look, (table,), (table,))
  out, tangent = torch.func.jvp(lambda y: look(table) * y, (torch.tensor(2.0),), (torch.tensor(1.0),))
  assert torch.equal(out, table[IDS] * 2) and torch.equal(tangent, table[IDS])


def test_without_a_graph(stand_ins):
  table = torch.randn(V, W, requires_grad=True)
  with torch.no_grad():
    assert not torch.ops.orca.embedding(table, IDS, 1.0, -1).requires_grad
  with torch.inference_mode():
    assert torch.equal(torch.ops.orca.embedding(table, IDS, 1.0, -1), table[IDS])
  assert not torch.ops.orca.embedding(table.detach(), IDS, 1.0, -1).requires_grad
  grad, = torch.autograd.grad(torch.ops.orca.embedding(table, IDS, 1.0, -1).sum(), table)
  assert not grad.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("padding", [-1, 3])
@pytest.mark.parametrize("wide", [False, True])
def test_second_derivative_of_the_kernels(padding, wide):
  """against plain indexing in fp64.  With x = scale * table, a row's gradient is the sum of 3 scale w x^2 over its occurrences, the
  penalty's of 2 grad * 6 scale^2 w x: products and sums of at most 6 occurrences, under 24 roundings of u = 2^-24 relative to the sums of
  the absolute values"""
  g = torch.Generator().manual_seed(2)
  dev, u = "cuda:0", 2.0 ** -24
  table = torch.randn(V, W, generator=g).to(dev).requires_grad_()
  weight = torch.randn(2, 3, W, generator=g).to(dev)
  ids = IDS.to(dev) if wide else IDS.to(dev).int()
  got = penalty(torch.ops.orca.embedding, table, weight, ids, 0.5, padding)
  want = penalty(plain, table.detach().cpu().double().requires_grad_(), weight.cpu().double(), IDS, 0.5, padding)
  size = penalty(plain, table.detach().cpu().double().abs().requires_grad_(), weight.cpu().double().abs(), IDS, 0.5, padding)
  for a, b, s in zip(got, want, size):
    assert bool(((a.cpu().double() - b).abs() <= 24 * u * s).all())


def test_the_module_offers_the_ops(stand_ins):
  """as torch_ops.tgat_gather and the others; symbolic sizes pass through the schema"""
  table = torch.randn(V, W, requires_grad=True)
  out = torch_ops.embedding(table, IDS, 2.0, -1)
  grad, = torch.autograd.grad(out.sum(), table, retain_graph=True)
  assert torch.equal(out, table[IDS] * 2) and torch.equal(grad, torch_ops.embedding_backward(torch.ones(2, 3, W), IDS, V, 2.0, -1))
  assert str(torch.ops.orca.embedding.default._schema) == "orca::embedding(Tensor table, Tensor ids, float scale, SymInt padding_idx) -> Tensor"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tracing(dtype):
  """shapes and types without data, through the derivative too; no kernel and no stand-in is called"""
  from torch._subclasses.fake_tensor import FakeTensorMode
  with FakeTensorMode():
    table = torch.empty(V, W, dtype=dtype, requires_grad=True)
    out = torch.ops.orca.embedding(table, torch.zeros(2, 3, dtype=torch.int32), 0.5, 0)
    assert out.shape == (2, 3, W) and out.dtype == dtype
    grad, = torch.autograd.grad(out.sum(), table, retain_graph=True)
    assert grad.shape == (V, W) and grad.dtype == dtype
    again, = torch.autograd.grad((out.square().sum()), table, create_graph=True)
    assert torch.autograd.grad(again.sum(), table)[0].shape == (V, W)


@pytest.mark.parametrize("padding", [-1, 3])
def test_registrations(stand_ins, padding):
  """torch's own check of an op's schema, derivative, tracing and compiled backward"""
  table = torch.randn(V, W, requires_grad=True)
  torch.library.opcheck(torch.ops.orca.embedding.default, (table, IDS, 0.5, padding))
  torch.library.opcheck(torch.ops.orca.embedding_backward.default, (torch.randn(2, 3, W, requires_grad=True), IDS, V, 0.5, padding))
