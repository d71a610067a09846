"""A learned table in front of the framework's attention layer, trained with the fused optimizer: lookup -> orca::tgat_dense -> loss ->
gradients -> clipped Adam step, and what the layer keeps from its parameters follows the step."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
B, K, DE, V, W = 40, 10, 172, 300, 100


def make_layer(seed):
  from orca_amd.api.temporal_attention import TemporalAttentionLayer
  torch.manual_seed(seed)
  return TemporalAttentionLayer(W, W, DE, W, W, n_head=2, dropout=0.0).to(DEV)


def batch(seed):
  g = torch.Generator().manual_seed(seed)
  ids = (torch.rand(B, K + 1, generator=g) ** 3 * V).long()
  ids[:, 1:][torch.rand(B, K, generator=g) < 0.3] = 0                    # short neighbour lists end in the padding id
  mask = ids[:, 1:] == 0
  times = lambda *s: torch.cos(torch.rand(*s, generator=g) * 6)
  return (ids.to(DEV), mask.to(DEV), times(B, 1, W).to(DEV), times(B, K, W).to(DEV), torch.randn(B, K, DE, generator=g).to(DEV),
          torch.randn(B, W, generator=g).to(DEV))


def forward(layer, rows, mask, st, nt, edge):
  return layer(rows[:, 0].contiguous(), st, rows[:, 1:].contiguous(), nt, edge, mask.clone())[0]


def test_the_table_gets_the_gradient_of_its_rows():
  """the table's gradient is the fp64 sum, by id, of what the layer returns for the rows; the padding id's row gets none"""
  from orca_amd import torch_ops  # noqa: F401
  layer = make_layer(1)
  table = (torch.randn(V, W, generator=torch.Generator().manual_seed(2)) * 0.5).to(DEV).requires_grad_()
  ids, mask, st, nt, edge, target = batch(3)
  scale = 1.5
  (forward(layer, torch.ops.orca.embedding(table, ids, scale, 0), mask, st, nt, edge) - target).square().sum().backward()
  rows = (table.detach()[ids] * scale).requires_grad_()
  grad, = torch.autograd.grad((forward(layer, rows, mask, st, nt, edge) - target).square().sum(), rows)
  keep = ids != 0
  z = torch.zeros(V, W, dtype=torch.float64, device=DEV)
  G, S = z.clone().index_add_(0, ids[keep], grad[keep].double()) * scale, z.index_add_(0, ids[keep], grad[keep].double().abs()) * scale
  m = torch.bincount(ids[keep], minlength=V)[:, None]
  assert bool(((table.grad.double() - G).abs() <= 1.01 * ((m + 3) * U * S) + 1e-38).all()) and not bool(table.grad[0].any())
  assert bool((table.grad[m[:, 0] > 0] != 0).any(1).all())


@pytest.mark.parametrize("detach", [True, False])
@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_the_layer_follows_the_fused_step(detach, max_norm):
  """the layer's packed weights after a step are those of a layer that is made with the stepped parameters"""
  from orca_amd import ops, torch_ops  # noqa: F401
  layer, table = make_layer(4), torch.nn.Parameter(torch.randn(V, W, generator=torch.Generator().manual_seed(5)).to(DEV))
  ids, mask, st, nt, edge, target = batch(6)
  params = {"table": table, **dict(layer.named_parameters())}
  opt = ops.FusedAdam({k: p.detach() if detach else p for k, p in params.items()}, lr=1e-2)
  last = None
  for _ in range(3):
    out = forward(layer, torch.ops.orca.embedding(table, ids, 1.0, 0), mask, st, nt, edge)
    assert last is None or not torch.equal(out, last)
    last = out.detach()
    grads = dict(zip(params, torch.autograd.grad((out - target).square().sum(), list(params.values()), allow_unused=True)))
    before = {k: p._version for k, p in params.items()}
    opt.step(grads, max_norm=max_norm)
    assert all(params[k]._version > before[k] for k, g in grads.items() if g is not None)
    fresh = make_layer(7)
    fresh.load_state_dict(layer.state_dict())
    with torch.no_grad():
      rows = torch.ops.orca.embedding(table, ids, 1.0, 0)
      assert torch.equal(forward(layer, rows, mask, st, nt, edge), forward(fresh, rows, mask, st, nt, edge))


def test_a_stale_graph_is_refused():
  """as with torch's optimizers: no backward pass through values that the step has replaced"""
  from orca_amd import ops
  p = torch.nn.Parameter(torch.ones(8, device=DEV))
  loss = (p * p).sum()
  ops.FusedAdam({"p": p}).step({"p": torch.ones(8, device=DEV)})
  with pytest.raises(RuntimeError, match="inplace"):
    loss.backward()
