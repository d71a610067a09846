"""Clipping inside the optimizer step (FusedAdam.step(max_norm=), OrcaEngine.step_optimizer(max_norm=)), row-sparse gradients in it
(orca_adam_rows), and a learned table trained end to end with them, against fp64.

Tolerance of an Adam update from an fp32 state (u = 2^-24): the gradient carries the rounding of the coefficient and of the product
(2u |g|), m three roundings of its own, v three and twice the gradient's, the quotient five; the sum with p one:
  |p - p64| <= 1.1 (u |p| + step (5u (|m0| + |g|)) / d + 14u |update|),   d = sqrt(v) / sqrt(1 - b2^t) + eps,   step = lr / (1 - b1^t)"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
B1, B2, EPS = 0.9, 0.999, 1e-8


@pytest.fixture(scope="module")
def ops():
  from orca_amd import ops as o
  return o


def adam64(p, m, v, g, lr, t):
  """one step in fp64 from fp32 tensors: (p, m, v, bound of p's error)"""
  p, m0, v, g = (x.detach().cpu().double() for x in (p, m, v, g))
  m = m0 + (1 - B1) * (g - m0)
  v = B2 * v + (1 - B2) * g * g
  step, d = lr / (1 - B1 ** t), v.sqrt() / math.sqrt(1 - B2 ** t) + EPS
  up = step * m / d
  lim = 1.1 * (U * (p - up).abs() + step * 5 * U * (m0.abs() + g.abs()) / d + 14 * U * up.abs()) + 1e-38
  return p - up, m, v, lim


def check_step(before, after, g, lr, t, what):
  (p0, m0, v0), (p1, m1, v1) = before, after
  p, m, v, lim = adam64(p0, m0, v0, g, lr, t)
  gm = g.detach().cpu().double().abs()
  assert bool(((p1.cpu().double() - p).abs() <= lim).all()), what
  assert bool(((m1.cpu().double() - m).abs() <= 5.5 * U * (m0.cpu().double().abs() + gm) + 1e-38).all()), what
  assert bool(((v1.cpu().double() - v).abs() <= 8 * U * v + 1e-38).all()), what


def snapshot(opt, k):
  n = opt.params[k].numel()
  return tuple(x.clone().reshape(opt.params[k].shape) for x in (opt.params[k], opt.exp_avg[k][:n], opt.exp_avg_sq[k][:n]))


@pytest.mark.parametrize("max_norm", [0.3, 1e6])
def test_adam_with_clipping(ops, max_norm):
  g = torch.Generator().manual_seed(3)
  shapes = [(200, 200), (300,), (1,), (7, 13), (100, 372)] + [(33,)] * 60
  opt = ops.FusedAdam({f"p{i}": torch.randn(*s, generator=g).to(DEV) for i, s in enumerate(shapes)}, lr=1e-3)
  for t in range(1, 4):
    grads = {k: (torch.randn(*p.shape, generator=g) * 0.1).to(DEV) for k, p in opt.params.items()}
    keep = {k: x.clone() for k, x in grads.items()}
    before = {k: snapshot(opt, k) for k in opt.params}
    norm = opt.step(grads, max_norm=max_norm)
    want = math.sqrt(sum(float((x.double() ** 2).sum()) for x in grads.values()))
    assert abs(float(norm) - want) <= want * 1.01 * U
    c = min(1.0, max_norm / (want + 1e-6))
    for k in opt.params:
      assert torch.equal(grads[k], keep[k]), "the gradients stay"
      check_step(before[k], snapshot(opt, k), keep[k].double() * c, 1e-3, t, f"{k} step {t}")
  assert opt.step({}, max_norm=1.0) == 0.0           # nothing to do: norm 0


def test_without_clipping_nothing_changes(ops):
  """max_norm that does not bind gives the bits of a step without it (the coefficient is exactly 1)"""
  g = torch.Generator().manual_seed(5)
  P = {f"p{i}": torch.randn(1000 + i, generator=g) for i in range(5)}
  a, b = (ops.FusedAdam({k: v.clone().to(DEV) for k, v in P.items()}, lr=1e-2) for _ in range(2))
  for _ in range(3):
    grads = {k: torch.randn(v.shape, generator=g).to(DEV) for k, v in P.items()}
    assert a.step(grads) is None
    b.step(grads, max_norm=1e9)
    assert all(torch.equal(a.params[k], b.params[k]) for k in P)


@pytest.mark.parametrize("width", [1, 7, 64, 100, 257])
@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_rows_update_alone(ops, width, max_norm):
  """only the rows of a RowGrad move, with the arithmetic of the dense step; the others and their moments keep their bits"""
  V, n = 500, 700
  g = torch.Generator().manual_seed(width)
  opt = ops.FusedAdam({"t": torch.randn(V, width, generator=g).to(DEV), "w": torch.randn(31, generator=g).to(DEV)}, lr=1e-2)
  for t in range(1, 4):
    ids = (torch.rand(n, generator=g) ** 3 * V).long().to(DEV)
    rg = ops.embedding_backward_rows(torch.randn(n, width, generator=g).to(DEV), ids, V, padding_idx=0)
    w = torch.randn(31, generator=g).to(DEV)
    before = {k: snapshot(opt, k) for k in ("t", "w")}
    norm = opt.step({"t": rg, "w": w}, max_norm=max_norm)
    k = int(rg.count)
    live = rg.ids[:k]
    c = 1.0
    if max_norm is not None:
      want = math.sqrt(float((rg.rows[:k].double() ** 2).sum() + (w.double() ** 2).sum()))
      assert abs(float(norm) - want) <= want * 1.01 * U
      c = min(1.0, max_norm / (want + 1e-6))
    after = {k: snapshot(opt, k) for k in ("t", "w")}
    check_step(before["w"], after["w"], w.double() * c, 1e-2, t, "dense beside it")
    check_step([x[live] for x in before["t"]], [x[live] for x in after["t"]], rg.rows[:k].double() * c, 1e-2, t, f"rows, step {t}")
    rest = torch.ones(V, dtype=torch.bool, device=DEV)
    rest[live] = False
    assert rest[0] and all(torch.equal(x[rest], y[rest]) for x, y in zip(before["t"], after["t"]))


def test_rows_and_dense_agree(ops):
  """where every row has an occurrence, the row-sparse and the dense gradient make the same step, bit for bit"""
  V, n, w = 40, 3000, 20
  g = torch.Generator().manual_seed(2)
  table = torch.randn(V, w, generator=g)
  ids = torch.cat([torch.arange(V), torch.randint(0, V, (n - V,), generator=g)]).to(DEV)
  grad = torch.randn(n, w, generator=g).to(DEV)
  a, b = (ops.FusedAdam({"t": table.clone().to(DEV)}, lr=1e-2) for _ in range(2))
  for _ in range(3):
    na = a.step({"t": ops.embedding_backward(grad, ids, V)}, max_norm=1.0)
    nb = b.step({"t": ops.embedding_backward_rows(grad, ids, V)}, max_norm=1.0)
    assert abs(float(na) - float(nb)) <= 2 * U * float(na)
    assert torch.allclose(a.params["t"], b.params["t"], rtol=0, atol=64 * U * 3)      # the norms may round apart: c, then g, m, v, p


def test_a_learned_table_end_to_end(ops):
  """lookup -> squared distance to targets -> gradient -> clip -> Adam, dense through autograd and row-sparse by hand, against the
  same steps in fp64 on the CPU.  Each step starts the fp64 side from the GPU's fp32 state, so that the bounds are one step's."""
  from orca_amd import torch_ops  # noqa: F401
  V, w, n, scale = 300, 24, 900, 0.5
  g = torch.Generator().manual_seed(8)
  table = (torch.randn(V, w, generator=g) * 0.1).to(DEV)
  opt = ops.FusedAdam({"table": table}, lr=1e-2)
  for t in range(1, 5):
    ids = (torch.rand(n, generator=g) ** 2 * V).long()
    target = torch.randn(n, w, generator=g)
    before = snapshot(opt, "table")
    leaf = table.detach().clone().requires_grad_()
    out = torch.ops.orca.embedding(leaf, ids.to(DEV), scale, 0)
    (0.5 * (out - target.to(DEV)) ** 2).sum().backward()
    d_out = out.detach() - target.to(DEV)
    rg = ops.embedding_backward_rows(d_out, ids.to(DEV), V, scale=scale, padding_idx=0)
    k = int(rg.count)
    dense = leaf.grad
    assert torch.equal(dense[rg.ids[:k]], rg.rows[:k])
    norm = opt.step({"table": rg}, max_norm=2.0)
    # fp64: the formula's gradient, rows of the padding id left out
    p64 = before[0].cpu().double()
    r = scale * p64[ids] - target.double()
    keep = ids != 0
    G = torch.zeros(V, w, dtype=torch.float64).index_add_(0, ids[keep], r[keep]) * scale
    S = torch.zeros(V, w, dtype=torch.float64).index_add_(0, ids[keep], (r.abs() + (scale * p64[ids]).abs())[keep]) * scale
    m = torch.bincount(ids[keep], minlength=V)[:, None]
    slack = 1.01 * (m + 4) * U * S + 1e-38                  # each r carries two roundings, the sum m, the product one
    assert bool(((dense.cpu().double() - G).abs() <= slack).all())
    want = float((G ** 2).sum().sqrt())
    assert abs(float(norm) - want) <= float((slack ** 2).sum().sqrt()) + 1.01 * U * want
    c = min(1.0, 2.0 / (want + 1e-6))
    live = rg.ids[:k].cpu()
    check_step([x.cpu()[live] for x in before], [x.cpu()[live] for x in snapshot(opt, "table")], rg.rows[:k].cpu().double() * c, 1e-2, t,
               f"step {t}")


@pytest.mark.parametrize("fused", [True, False])
def test_engine_step_with_max_norm(ops, fused):
  """OrcaEngine.step_optimizer(grads, max_norm): the norm over the trained parameters' gradients, and parameters as a step with
  gradients clipped beforehand in fp64 and rounded gives them (the clipped gradients differ by 3u, see the bound above)"""
  from orca_amd import synth
  from orca_amd.engine import OrcaEngine
  N, E, bs, K, d_e = 600, 8000, 60, 10, 172
  src, dst, eidx, ts = synth.powerlaw_graph(N, E, DEV, seed=6)
  ef = synth.edge_features(E, d_e, DEV)
  eng = OrcaEngine(synth.tgn_state_dict(d_e, 2, seed=3), ef, N + 1, 2, K, reuse=True, budget=0, device=DEV)
  eng.set_neighbor_finder(ops.CSR.from_edges_device(src, dst, eidx, ts, N + 1))
  s = 5000
  neg = torch.randint(1, N + 1, (bs,), generator=torch.Generator().manual_seed(1)).to(DEV)
  eng.optimizer(lr=1e-3, fused=fused)
  assert eng.step_optimizer({}) is None
  _, grads = eng.train_step(src[s:s + bs], dst[s:s + bs], neg, ts[s:s + bs], eidx[s:s + bs])
  grads = {k: v.clone() for k, v in grads.items()}
  trained = eng._opt.params if fused else eng._opt_params
  mine = {k: g for k, g in grads.items() if k in trained}
  want = math.sqrt(sum(float((g.double() ** 2).sum()) for g in mine.values()))
  c = min(1.0, 0.25 * want / (want + 1e-6))
  before = {k: v.clone() for k, v in eng.params.items()}
  exact = {k: g.double() * c for k, g in mine.items()}
  norm = eng.step_optimizer(grads, max_norm=0.25 * want)
  assert abs(float(norm) - want) <= 1.01 * U * want
  moved = 0
  for k, g in exact.items():
    p0 = before[k]
    z = torch.zeros_like(p0)
    p, _, _, lim = adam64(p0, z, z, g.reshape(p0.shape), 1e-3, 1)
    # torch.optim.Adam's own order of operations costs a few roundings more of the update
    lim = lim + 8 * U * (p - p0.cpu().double()).abs()
    assert bool(((eng.params[k].cpu().double() - p).abs() <= lim).all()), k
    moved += int((eng.params[k] != p0).any())
  assert moved >= 20


def test_refusals(ops):
  from orca_amd._lib import OrcaError
  opt = ops.FusedAdam({"t": torch.zeros(10, 4, device=DEV)}, lr=1e-2)
  ids, cnt = torch.zeros(3, dtype=torch.int64, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
  for rows, n_rows in ((torch.zeros(3, 5, device=DEV), 10), (torch.zeros(3, 4, device=DEV), 11), (torch.zeros(3, 4, device=DEV).bfloat16(), 10)):
    with pytest.raises(OrcaError):
      opt.step({"t": ops.RowGrad(ids, rows, cnt, n_rows)})
  with pytest.raises(ValueError):
    opt.step({"t": torch.zeros(10, 4, device=DEV)}, max_norm=-1.0)
  assert opt.steps["t"] == 0


def test_row_gradients_that_do_not_fit(ops):
  """a RowGrad made by hand: fewer rows than ids, other types, gaps, another device"""
  from orca_amd._lib import OrcaError
  opt = ops.FusedAdam({"t": torch.zeros(10, 4, device=DEV)}, lr=1e-2)
  ids, rows, cnt = torch.arange(3, device=DEV), torch.ones(3, 4, device=DEV), torch.full((1,), 3, dtype=torch.int32, device=DEV)
  for bad in (ops.RowGrad(ids, rows[:2], cnt, 10), ops.RowGrad(ids.int(), rows, cnt, 10), ops.RowGrad(ids, rows, cnt.long(), 10),
              ops.RowGrad(ids, torch.ones(3, 8, device=DEV)[:, ::2], cnt, 10), ops.RowGrad(torch.arange(6, device=DEV)[::2], rows, cnt, 10),
              ops.RowGrad(ids.cpu(), rows, cnt, 10), ops.RowGrad(ids, rows, cnt.cpu(), 10), ops.RowGrad(ids, rows, cnt.repeat(2), 10),
              ops.RowGrad(ids, rows.reshape(12), cnt, 10)):
    for max_norm in (None, 1.0):
      with pytest.raises(OrcaError):
        opt.step({"t": bad}, max_norm=max_norm)
  assert opt.steps["t"] == 0 and bool((opt.params["t"] == 0).all())
  opt.step({"t": ops.RowGrad(ids, rows, cnt, 10)})
  assert bool((opt.params["t"][:3] != 0).all()) and bool((opt.params["t"][3:] == 0).all())
