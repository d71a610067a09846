"""orca_embedding_forward / _backward / _backward_rows (ops.embedding, ops.embedding_backward, ops.embedding_backward_rows) against
plain fp64 sums, at the sizes where tiles, windows and chunks end, with ids that are absent, padded, out of range or all the same.

Tolerances, element by element (u = half a step of fp32 = 2^-24, h = half a step of the output's type, relative; t = half the
output's smallest step, absolute):
  lookup    one fp32 product, one rounding:                         (u + h) |x| + t
  gradient  m additions in fp32, one product, one rounding:         (m + 2) u |scale| sum|g| + h |G| + t
(second-order terms are under the 1 % by which each bound is widened)"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops():
  from orca_amd import ops as o
  return o


def half(t):
  return torch.finfo(t).eps / 2 if t != torch.float32 else U


def tiny(t):
  return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def make_ids(kind, n, vocab, seed, dtype=torch.int64):
  g = torch.Generator().manual_seed(seed)
  if kind == "same":
    ids = torch.full((n,), vocab // 2)
  elif kind == "distinct":
    ids = torch.randperm(max(n, vocab), generator=g)[:n]
  elif kind == "hubs":
    ids = ((torch.rand(n, generator=g) ** 6) * vocab).long()
  elif kind == "bad":       # a third outside the table, among them the types' extremes
    ids = torch.randint(0, vocab, (n,), generator=g)
    ids[::3] = torch.randint(vocab, vocab + 3, (ids[::3].numel(),), generator=g)
    ids[1::9] = -1
    ids[::17] = torch.iinfo(dtype).min
    ids[5::19] = torch.iinfo(dtype).max
  else:
    ids = torch.randint(0, vocab, (n,), generator=g)
  return ids.to(dtype)


def reference(grad, ids, vocab, scale, padding):
  """(G, the tolerance's sum of |g|, occurrences) in fp64 on the CPU"""
  ids, grad = ids.cpu().long().reshape(-1), grad.detach().cpu().double().reshape(ids.numel(), -1)
  keep = (ids >= 0) & (ids < vocab)
  if padding is not None:
    keep &= ids != padding
  ids, grad = ids[keep], grad[keep]
  z = torch.zeros(vocab, grad.shape[1], dtype=torch.float64)
  return (z.clone().index_add_(0, ids, grad) * scale, z.index_add_(0, ids, grad.abs()) * abs(scale),
          torch.bincount(ids, minlength=vocab))


def bound(G, S, m, t):
  return 1.01 * ((m[:, None] + 2) * U * S + half(t) * G.abs()) + tiny(t)


def check_grad(got, grad, ids, vocab, scale, padding):
  G, S, m = reference(grad, ids, vocab, scale, padding)
  off = (got.cpu().double() - G).abs()
  lim = bound(G, S, m, got.dtype)
  assert bool((off <= lim).all()), f"off {float((off - lim).max()):.3e} over the bound"
  assert bool((got.cpu()[m == 0] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 3, 4, 7, 8, 9, 100, 173, 257, 1000])
@pytest.mark.parametrize("n", [1, 2, 255, 1031])
def test_lookup(ops, dtype, width, n):
  table = torch.randn(77, width, generator=torch.Generator().manual_seed(n)).to(dtype).to(DEV)
  for id_type in (torch.int64, torch.int32):
    ids = make_ids("bad", n, 77, n + width, id_type).to(DEV)
    out = ops.embedding(table, ids, scale=1.7)
    c = ids.cpu().long()
    ok = (c >= 0) & (c < 77)
    exp = table.cpu().double()[torch.where(ok, c, 0)] * ok[:, None] * float(np.float32(1.7))
    off = (out.cpu().double() - exp).abs()
    assert out.shape == (n, width) and out.dtype == dtype
    assert bool((off <= 1.01 * (U + half(dtype)) * exp.abs() + tiny(dtype)).all())
    assert torch.equal(ops.embedding(table, ids)[ok.to(DEV)], table[ids[ok.to(DEV)].long()])      # scale 1: the rows themselves


def test_lookup_shapes_strides_and_guards(ops):
  base = torch.randn(50, 64, device=DEV)
  table = base[:, 5:42]                                   # rows strided, not 16-byte aligned
  ids = torch.randint(0, 50, (4, 6, 5), device=DEV)
  out = ops.embedding(table, ids, scale=2.0)
  assert out.shape == (4, 6, 5, 37) and torch.equal(out, table[ids] * 2)
  assert torch.equal(ops.embedding(table, ids.transpose(0, 2), scale=2.0), table[ids.transpose(0, 2)] * 2)
  assert torch.equal(ops.embedding(base[:1].expand(9, 64), ids % 9), base[:1].expand(9, 64)[ids % 9])
  assert ops.embedding(table, ids[:0]).shape == (0, 6, 5, 37)
  assert bool((ops.embedding(table[:0], ids) == 0).all())                       # an empty table: every id lies outside
  room = torch.full((3 + 120 * 37 + 3,), 7.0, device=DEV)                       # the output inside a larger buffer
  got = ops.embedding(table, ids.reshape(-1), out=room[3:3 + 120 * 37].view(120, 37))
  assert torch.equal(got, table[ids.reshape(-1)]) and bool((room[:3] == 7).all()) and bool((room[-3:] == 7).all())
  nan = base.clone()
  nan[3] = float("nan")
  nan[4] = float("inf")
  got = ops.embedding(nan, torch.tensor([3, 4, 5], device=DEV), scale=0.5)
  assert bool(got[0].isnan().all()) and bool(got[1].isinf().all()) and torch.equal(got[2], base[5] * 0.5)


def test_lookup_offsets_past_32_bits(ops):
  """rows behind 2^32 bytes and 2^31 elements of a table, and an output of that size"""
  table = torch.empty(2_200_000, 1024, dtype=torch.bfloat16, device=DEV)      # 2.25e9 elements
  table[0], table[2_199_999], table[2_097_153] = 1.0, 2.0, 3.0
  ids = torch.tensor([2_199_999, 0, 2_097_153], device=DEV)
  assert ops.embedding(table, ids)[:, 1000].tolist() == [2.0, 1.0, 3.0]
  big = ops.embedding(table[2_199_999:], torch.zeros(2_200_000, dtype=torch.int32, device=DEV), out=table.clone())
  assert bool((big[-1] == 2).all()) and bool((big[2_097_150] == 2).all())


SIZES = [1, 2, 31, 32, 33, 64, 65, 1024, 1025, 2047, 2048, 2049, 5000, 20000]


@pytest.mark.parametrize("kind", ["uniform", "hubs", "same", "distinct", "bad"])
@pytest.mark.parametrize("n", SIZES)
def test_gradient_sizes(ops, kind, n):
  vocab = 31 if kind == "same" else max(n, 300)
  ids = make_ids(kind, n, vocab, n).to(DEV)
  grad = torch.randn(n, 20, generator=torch.Generator().manual_seed(1)).to(DEV)
  got = ops.embedding_backward(grad, ids, vocab, scale=0.75)
  check_grad(got, grad, ids, vocab, 0.75, None)
  assert torch.equal(got, ops.embedding_backward(grad, ids, vocab, scale=0.75)), "the same call gives the same bits"
  rg = ops.embedding_backward_rows(grad, ids, vocab, scale=0.75)
  u = torch.unique(ids[(ids >= 0) & (ids < vocab)])
  k = int(rg.count)
  assert k == u.numel() and torch.equal(rg.ids[:k], u)
  assert torch.equal(rg.rows[:k], got[u]), "both forms add in the same order"


@pytest.mark.parametrize("width", [1, 2, 3, 5, 8, 15, 16, 17, 100, 172, 255, 256, 257, 520, 2049])
@pytest.mark.parametrize("g_type,o_type", [(torch.float32, None), (torch.bfloat16, None), (torch.float16, None),
                                           (torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
def test_gradient_widths_and_types(ops, width, g_type, o_type):
  n, vocab = 700, 129
  ids = make_ids("hubs", n, vocab, width, torch.int32).to(DEV)
  grad = torch.randn(n, width, generator=torch.Generator().manual_seed(width)).to(g_type).to(DEV)
  got = ops.embedding_backward(grad, ids, vocab, scale=1.3, padding_idx=0, dtype=o_type)
  assert got.dtype == (o_type or g_type)
  check_grad(got, grad, ids, vocab, float(np.float32(1.3)), 0)
  rg = ops.embedding_backward_rows(grad, ids, vocab, scale=1.3, padding_idx=0, dtype=o_type)
  k = int(rg.count)
  assert torch.equal(rg.rows[:k], got[rg.ids[:k]]) and bool((rg.ids[:k] != 0).all())


@pytest.mark.parametrize("vocab", [1, 2, 3, 127, 128, 1023, 1024, 2047, 2048, 65535, 65536, (1 << 22) - 1, 1 << 22, (1 << 24) + 5, (1 << 31) - 2])
def test_row_numbers_up_to_31_bits(ops, vocab):
  """every number of radix passes and digit widths; the row-sparse form has no table of that many rows"""
  n = 3000
  g = torch.Generator().manual_seed(3)
  ids = torch.randint(0, vocab, (n,), generator=g)
  ids[:4] = torch.tensor([0, vocab - 1, vocab // 2, vocab - 1])
  grad = torch.randn(n, 4, generator=g)
  rg = ops.embedding_backward_rows(grad.to(DEV), ids.to(DEV), vocab)
  u, inv = torch.unique(ids, return_inverse=True)
  k = int(rg.count)
  assert k == u.numel() and torch.equal(rg.ids[:k].cpu(), u)
  z = torch.zeros(k, 4, dtype=torch.float64)
  G, S = z.clone().index_add_(0, inv, grad.double()), z.index_add_(0, inv, grad.double().abs())
  assert bool(((rg.rows[:k].cpu().double() - G).abs() <= bound(G, S, torch.bincount(inv), torch.float32)).all())


def test_long_run_over_many_tiles(ops):
  """300,000 positions: 40 % of them one id, a second hub, the rest spread; and everything one id"""
  n, vocab = 300_000, 50_000
  g = torch.Generator().manual_seed(9)
  ids = torch.randint(0, vocab, (n,), generator=g)
  r = torch.rand(n, generator=g)
  ids[r < 0.4], ids[r > 0.9] = 777, 778
  grad = torch.randn(n, 12, generator=g)
  for i in (ids, torch.full((n,), 49_999)):
    got = ops.embedding_backward(grad.to(DEV), i.to(DEV), vocab)
    check_grad(got, grad, i, vocab, 1.0, None)


@pytest.mark.parametrize("width", [1, 3, 4, 7, 8, 17, 100, 129, 257, 1030])
@pytest.mark.parametrize("g_type,o_type", [(torch.float32, None), (torch.bfloat16, None), (torch.float16, None), (torch.bfloat16, torch.float32)])
def test_long_lists_widths_and_types(ops, width, g_type, o_type):
  """more ids than a short list has: the windows' sums and their joins, accumulated into a strided table, and the row-sparse form"""
  n, vocab = 8193 + width % 5, 700
  ids = make_ids("hubs", n, vocab, width, torch.int32).to(DEV)
  grad = torch.randn(n, width, generator=torch.Generator().manual_seed(width)).to(g_type).to(DEV)
  got = ops.embedding_backward(grad, ids, vocab, scale=0.5, padding_idx=3, dtype=o_type)
  check_grad(got, grad, ids, vocab, 0.5, 3)
  rg = ops.embedding_backward_rows(grad, ids, vocab, scale=0.5, padding_idx=3, dtype=o_type)
  k = int(rg.count)
  assert torch.equal(rg.rows[:k], got[rg.ids[:k]]) and bool((rg.ids[:k] != 3).all())
  base = torch.full((vocab, width + 3), 2.0, dtype=got.dtype, device=DEV)
  out = base[:, 1:1 + width]
  start = torch.randn(vocab, width, generator=torch.Generator().manual_seed(4)).to(got.dtype).to(DEV)
  out.copy_(start)
  ops.embedding_backward(grad, ids, vocab, scale=0.5, padding_idx=3, out=out, accumulate=True)
  G, S, m = reference(grad, ids, vocab, 0.5, 3)
  exp = start.cpu().double() + G
  lim = 1.01 * ((m[:, None] + 2) * U * S + (half(out.dtype) + U) * exp.abs()) + tiny(out.dtype)
  assert bool(((out.cpu().double() - exp).abs() <= lim).all())
  assert bool((base[:, 0] == 2).all()) and bool((base[:, 1 + width:] == 2).all()), "what lies between the rows"
  out.fill_(9)
  assert torch.equal(ops.embedding_backward(grad, ids, vocab, scale=0.5, padding_idx=3, out=out), got)
  assert bool((base[:, 0] == 2).all()) and bool((base[:, 1 + width:] == 2).all())


def test_few_ids_in_a_tall_table(ops):
  """more rows than the short list's workgroups can mark: the zeros come from the sort's launches"""
  V = 17_000_003
  ids = torch.tensor([0, V - 1, 5, V - 1, 16_777_216, -7, V], device=DEV)
  got = ops.embedding_backward(torch.arange(1.0, 8.0, device=DEV)[:, None], ids, V)
  assert got[[0, 5, 16_777_216, V - 1], 0].tolist() == [1.0, 3.0, 5.0, 6.0] and int((got != 0).sum()) == 4
  got.fill_(1.0)
  ops.embedding_backward(torch.ones(7, 1, device=DEV), ids, V, out=got, accumulate=True)
  assert got[[0, 5, 16_777_216, V - 1, 1], 0].tolist() == [2.0, 2.0, 2.0, 3.0, 1.0]


def test_large_gradients_and_tables(ops):
  """the accesses past the caches: 150 MB of gradient rows, a table of 420 MB"""
  n, w, vocab = 73_000, 1024, 205_000
  g = torch.Generator(device=DEV).manual_seed(1)
  grad = torch.empty(n, w, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
  ids = (torch.rand(n, generator=g, device=DEV) ** 3 * vocab).long()
  got = ops.embedding_backward(grad, ids, vocab, scale=2.0)
  G = torch.zeros(vocab, w, device=DEV, dtype=torch.float64).index_add_(0, ids, grad.double()).mul_(2.0)
  S = torch.zeros(vocab, w, device=DEV, dtype=torch.float64).index_add_(0, ids, grad.double().abs()).mul_(2.0)
  m = torch.bincount(ids, minlength=vocab)[:, None]
  assert bool(((got.double() - G).abs() <= 1.01 * ((m + 2) * U * S + half(torch.bfloat16) * G.abs()) + tiny(torch.bfloat16)).all())
  rg = ops.embedding_backward_rows(grad, ids, vocab, scale=2.0)
  k = int(rg.count)
  assert torch.equal(rg.rows[:k], got[rg.ids[:k]])


def test_empty_and_all_padding(ops):
  e = torch.empty(0, 8, device=DEV)
  none = torch.empty(0, dtype=torch.int64, device=DEV)
  assert bool((ops.embedding_backward(e, none, 5) == 0).all())
  assert int(ops.embedding_backward_rows(e, none, 5).count) == 0
  grad = torch.full((40, 8), float("nan"), device=DEV)           # padded rows are not used, whatever they hold
  ids = torch.full((40,), 3, device=DEV)
  assert bool((ops.embedding_backward(grad, ids, 5, padding_idx=3) == 0).all())
  assert int(ops.embedding_backward_rows(grad, ids, 5, padding_idx=3).count) == 0
  assert ops.embedding_backward(grad, ids, 0).shape == (0, 8)
  assert int(ops.embedding_backward_rows(grad, ids, 0).count) == 0
  ids[7] = 4
  grad[7] = 2.0
  got = ops.embedding_backward(grad, ids, 5, padding_idx=3)
  assert bool((got[4] == 2).all()) and bool((got[:4] == 0).all())
  ids[8] = 1
  got = ops.embedding_backward(grad, ids, 5, padding_idx=3)
  assert bool(got[1].isnan().all()) and bool((got[4] == 2).all()) and bool((got[[0, 2, 3]] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [3, 37, 100, 130])
def test_accumulate_and_strided_tables(ops, dtype, width):
  n, vocab = 900, 61
  ids = make_ids("hubs", n, vocab, 5).to(DEV)
  grad = torch.randn(n, width, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
  base = torch.full((vocab, width + 5), 3.0, dtype=dtype, device=DEV)
  out = base[:, 2:2 + width]
  assert ops.embedding_backward(grad, ids, vocab, out=out) is out
  assert torch.equal(out, ops.embedding_backward(grad, ids, vocab))
  assert bool((base[:, :2] == 3).all()) and bool((base[:, 2 + width:] == 3).all()), "what lies between the rows"
  start = torch.randn(vocab, width, generator=torch.Generator().manual_seed(4)).to(dtype).to(DEV)
  out.copy_(start)
  ops.embedding_backward(grad, ids, vocab, out=out, accumulate=True)
  G, S, m = reference(grad, ids, vocab, 1.0, None)
  exp = start.cpu().double() + G
  lim = 1.01 * ((m[:, None] + 2) * U * S + (half(dtype) + U) * exp.abs()) + tiny(dtype)
  assert bool(((out.cpu().double() - exp).abs() <= lim).all())
  assert torch.equal(out[(m == 0).to(DEV)], start[(m == 0).to(DEV)]), "rows without an occurrence stay"
  assert bool((base[:, :2] == 3).all()) and bool((base[:, 2 + width:] == 3).all())


def test_gradients_that_are_views(ops):
  """row stride 0 (the gradient of a sum over rows), a slice of wider rows, a transposed matrix, ids of two axes"""
  ids = make_ids("hubs", 600, 50, 1).to(DEV)
  one = torch.randn(24, device=DEV)
  wide = torch.randn(600, 40, device=DEV)
  for grad in (one.expand(600, 24), wide[:, 7:31], torch.randn(24, 600, device=DEV).t(), torch.ones((), device=DEV).expand(600, 24)):
    check_grad(ops.embedding_backward(grad, ids, 50), grad, ids, 50, 1.0, None)
  g3 = torch.randn(20, 30, 24, device=DEV)
  i3 = ids.view(20, 30)
  assert torch.equal(ops.embedding_backward(g3, i3, 50), ops.embedding_backward(g3.reshape(600, 24), ids, 50))
  assert torch.equal(ops.embedding_backward(g3.transpose(0, 1), i3.t(), 50), ops.embedding_backward(g3.transpose(0, 1).contiguous(), i3.t().contiguous(), 50))


def test_row_buffers_stay_behind_the_count(ops):
  n, vocab = 3000, 40
  ids = make_ids("hubs", n, vocab, 3).to(DEV)
  grad = torch.randn(n, 10, device=DEV)
  out = (torch.full((n,), -5, dtype=torch.int64, device=DEV), torch.full((n, 10), 9.0, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV))
  rg = ops.embedding_backward_rows(grad, ids, vocab, out=out)
  k = int(rg.count)
  assert rg.ids is out[0] and rg.rows is out[1] and 0 < k <= 40
  assert bool((rg.ids[k:] == -5).all()) and bool((rg.rows[k:] == 9).all())
  check_grad(torch.zeros(vocab, 10, device=DEV).index_copy_(0, rg.ids[:k], rg.rows[:k]), grad, ids, vocab, 1.0, None)


def test_autograd_op(ops):
  """orca::embedding: gradient against the formula, against differences of the loss, and with a broadcast gradient"""
  from orca_amd import torch_ops  # noqa: F401
  g = torch.Generator().manual_seed(6)
  table = torch.randn(23, 12, generator=g).to(DEV).requires_grad_()
  ids = torch.randint(0, 23, (5, 31), generator=g).to(DEV)
  w = torch.randn(5, 31, 12, generator=g).to(DEV)
  out = torch.ops.orca.embedding(table, ids, 0.5, 0)
  (out * w).sum().backward()
  check_grad(table.grad, w, ids, 23, 0.5, 0)
  # differences: the loss is linear in the table, so a step of 1 along a direction changes it by the gradient's product
  d = torch.randn(23, 12, generator=g).to(DEV)
  d[0] = 0                                                    # (the padding row has no gradient, by its definition)
  with torch.no_grad():
    diff = ((torch.ops.orca.embedding(table + d, ids, 0.5, 0).double() - torch.ops.orca.embedding(table - d, ids, 0.5, 0).double()) * w.double()).sum() / 2
  want = (table.grad.double() * d.double()).sum()
  # each of the 1860 products carries two lookups of 2u and the rounding of table +- d: 4u (|table| + |d|) |w| / 2 each
  lim = float((4 * U * 0.5 * (table.detach().abs() + d.abs()).double()[ids] * w.double().abs()).sum()) + 155 * U * float((w.abs().double().sum() * d.abs().max()))
  assert abs(float(diff - want)) <= lim
  table.grad = None
  torch.ops.orca.embedding(table, ids, 1.0, -1).sum().backward()
  assert torch.equal(table.grad, torch.bincount(ids.reshape(-1), minlength=23).float()[:, None].expand(23, 12))


def test_captured_and_replayed(ops):
  """lookup, dense and row-sparse gradient in one HIP graph; other eager work and other contents between the replays"""
  n, vocab, w = 5000, 3000, 36
  table = torch.randn(vocab, w, device=DEV)
  ids, grad = torch.zeros(n, dtype=torch.int64, device=DEV), torch.zeros(n, w, device=DEV)

  def step():
    return (ops.embedding(table, ids, 0.5), ops.embedding_backward(grad, ids, vocab, 0.5, padding_idx=0), ops.embedding_backward_rows(grad, ids, vocab))

  s = torch.cuda.Stream()
  s.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(s):
    step()
  torch.cuda.current_stream().wait_stream(s)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out, dense, rg = step()
  for r in range(4):
    ids.copy_(make_ids(["uniform", "hubs", "same", "distinct"][r], n, vocab if r != 3 else n, r).clamp_(max=vocab - 1))
    grad.copy_(torch.randn(n, w, generator=torch.Generator().manual_seed(r)))
    graph.replay()
    torch.cuda.synchronize()
    e_out, e_dense, e_rg = step()
    k = int(e_rg.count)
    assert torch.equal(out, e_out) and torch.equal(dense, e_dense), f"replay {r}"
    assert int(rg.count) == k and torch.equal(rg.ids[:k], e_rg.ids[:k]) and torch.equal(rg.rows[:k], e_rg.rows[:k]), f"replay {r}"


def test_two_streams_at_once(ops):
  """calls on two streams share nothing"""
  vocab, w = 4000, 50
  data = [(torch.randn(9000, w, device=DEV), make_ids("hubs", 9000, vocab, k).to(DEV)) for k in range(2)]
  want = [ops.embedding_backward(g, i, vocab) for g, i in data]
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream(), torch.cuda.Stream()]
  got = [[], []]
  for _ in range(5):
    for k, s in enumerate(streams):
      with torch.cuda.stream(s):
        got[k].append(ops.embedding_backward(*data[k], vocab))
  torch.cuda.synchronize()
  for k in range(2):
    assert all(torch.equal(x, want[k]) for x in got[k])


def test_refusals_on_the_device(ops):
  t, ids = torch.zeros(5, 8, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
  g = torch.zeros(3, 8, device=DEV)
  with pytest.raises(TypeError):
    ops.embedding(t.double(), ids)
  with pytest.raises(TypeError):
    ops.embedding(t, ids.float())
  with pytest.raises(ValueError):
    ops.embedding(t.t(), ids)
  with pytest.raises(ValueError):
    ops.embedding(t, ids, out=torch.zeros(3, 7, device=DEV))
  with pytest.raises(ValueError):
    ops.embedding(torch.zeros(1, 65537, device=DEV), ids)
  with pytest.raises(ValueError):
    ops.embedding_backward(g[:2], ids, 5)
  with pytest.raises(TypeError):
    ops.embedding_backward(g, ids, 5, dtype=torch.bfloat16)
  with pytest.raises(ValueError):
    ops.embedding_backward(g, ids, 5, accumulate=True)
  with pytest.raises(ValueError):
    ops.embedding_backward(g, ids, 5, out=torch.zeros(8, device=DEV).expand(5, 8))
  with pytest.raises(ValueError):
    ops.embedding_backward(g, ids, -1)
  with pytest.raises(ValueError):
    ops.embedding_backward_rows(g, ids, 1 << 31)
  with pytest.raises(ValueError):
    ops.embedding_backward_rows(g, ids, 5, out=(ids, g, torch.zeros(1, device=DEV)))


def test_outputs_apart_from_inputs(ops):
  """an output that shares memory with what the call reads is refused; neighbours in one buffer are not"""
  buf = torch.randn(20, 8, device=DEV)
  ids = torch.tensor([1, 0, 3], device=DEV)
  for out in (buf[:3], buf[2:5]):
    with pytest.raises(ValueError, match="overlaps"):
      ops.embedding(buf[:4], ids, out=out)
  with pytest.raises(ValueError, match="overlaps"):
    ops.embedding_backward(buf[:3], ids, 5, out=buf[2:7])
  with pytest.raises(ValueError, match="overlaps"):
    ops.embedding_backward_rows(buf[:3], ids, 5, out=(torch.zeros(3, dtype=torch.int64, device=DEV), buf[1:4], torch.zeros(1, dtype=torch.int32, device=DEV)))
  with pytest.raises(ValueError, match="overlaps"):
    ops.embedding_backward_rows(buf[:3], ids, 5, out=(ids, torch.zeros(3, 8, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)))
  want = buf[:4][ids].clone()
  assert torch.equal(ops.embedding(buf[:4], ids, out=buf[4:7]), want)
  before = buf[:4].clone()
  got = ops.embedding_backward(buf[:3], ids, 5, out=buf[10:15])
  check_grad(got, before[:3], ids, 5, 1.0, None)
  assert torch.equal(buf[:4], before)


def test_long_lists_captured_and_replayed(ops):
  """the sort's launches in a graph, other contents and eager work between the replays"""
  n, vocab, w = 12000, 5000, 20
  ids, grad = torch.zeros(n, dtype=torch.int32, device=DEV), torch.zeros(n, w, device=DEV, dtype=torch.bfloat16)

  def step():
    return ops.embedding_backward(grad, ids, vocab, 2.0, dtype=torch.float32), ops.embedding_backward_rows(grad, ids, vocab)

  step()
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    dense, rg = step()
  for r, kind in enumerate(["uniform", "same", "hubs"]):
    ids.copy_(make_ids(kind, n, vocab, r).clamp_(max=vocab - 1))
    grad.copy_(torch.randn(n, w, generator=torch.Generator().manual_seed(r)))
    graph.replay()
    torch.cuda.synchronize()
    e_dense, e_rg = step()
    k = int(e_rg.count)
    assert torch.equal(dense, e_dense), f"replay {r}"
    assert int(rg.count) == k and torch.equal(rg.ids[:k], e_rg.ids[:k]) and torch.equal(rg.rows[:k], e_rg.rows[:k]), f"replay {r}"


def test_autograd_on_another_stream(ops):
  """forward under a stream: the backward pass runs on it, behind what the gradient's producer left there"""
  from orca_amd import torch_ops  # noqa: F401
  vocab, w, n = 3000, 64, 20000
  g = torch.Generator().manual_seed(8)
  table = torch.randn(vocab, w, generator=g).to(DEV).requires_grad_()
  ids, wgt = torch.randint(0, vocab, (n,), generator=g).to(DEV), torch.randn(n, w, generator=g).to(DEV)
  torch.cuda.synchronize()
  s = torch.cuda.Stream()
  with torch.cuda.stream(s):
    grad, = torch.autograd.grad((torch.ops.orca.embedding(table, ids, 1.0, -1) * wgt).sum(), table)
  s.synchronize()
  check_grad(grad, wgt, ids, vocab, 1.0, None)


def test_neighbouring_hubs_row_sparse(ops):
  """frequent ids side by side (each longer than a team adds alone), among rare ones, over widths with few and many teams"""
  for n, w, seed in ((700, 2, 0), (2048, 40, 1), (2049, 3, 2), (6000, 100, 3), (8192, 16, 4), (8192, 128, 5), (1024, 1024, 6)):
    g = torch.Generator().manual_seed(seed)
    ids = torch.where(torch.rand(n, generator=g) < 0.8, torch.randint(500, 508, (n,), generator=g), torch.randint(0, 4000, (n,), generator=g)).to(DEV)
    grad = torch.randn(n, w, generator=g).to(DEV)
    rg = ops.embedding_backward_rows(grad, ids, 4000)
    k = int(rg.count)
    assert torch.equal(rg.ids[:k], torch.unique(ids))
    check_grad(torch.zeros(4000, w, device=DEV).index_copy_(0, rg.ids[:k], rg.rows[:k]), grad, ids, 4000, 1.0, None)


def test_tables_of_all_heights_behind_short_lists(ops):
  """both ways to the zeros: marked rows in the sum's launch, and a fill ahead of it (from 128 MB on, or 16.8 million rows)"""
  for vocab, w, t in ((250000, 128, torch.bfloat16), (250001, 160, torch.float32), (16777217, 2, torch.bfloat16), (16777216, 1, torch.float32)):
    ids = torch.tensor([0, vocab - 1, 7, 7, vocab, -1, vocab // 2], device=DEV)
    grad = torch.randn(7, w, device=DEV).to(t)
    out = torch.full((vocab, w), 3.0, dtype=t, device=DEV)
    got = ops.embedding_backward(grad, ids, vocab, out=out)
    rows = torch.tensor([0, 7, vocab // 2, vocab - 1], device=DEV)
    assert int((got != 0).any(1).sum()) == 4
    exp = torch.stack([grad[0].double(), grad[2].double() + grad[3].double(), grad[6].double(), grad[1].double()])
    # one fp32 sum of two (half a step of 2^-24) and one rounding to the type
    lim = exp.abs() * (2.0 ** -24 + torch.finfo(t).eps / 2) * 1.01 + 1e-30
    assert bool(((got[rows].double() - exp).abs() <= lim).all())


def test_zeros_of_strided_tables(ops):
  """a fill that leaves the gaps alone: rows of one piece and of several, by the sort's launches, ahead of a short list and alone"""
  for n, vocab, w, ld, t in ((0, 300, 1500, 1501, torch.float32), (0, 5000, 3, 7, torch.bfloat16), (9000, 300, 2049, 2056, torch.float32),
                             (9000, 4000, 5, 6, torch.float16), (3, 6000, 1100, 1111, torch.float32), (3, 1 << 20, 3, 16, torch.float32)):
    g = torch.Generator().manual_seed(n + w)
    ids = torch.randint(0, vocab, (n,), generator=g).to(DEV)
    grad = torch.randn(n, w, generator=g).to(t).to(DEV)
    buf = torch.full((vocab, ld), 5.0, dtype=t, device=DEV)
    ops.embedding_backward(grad, ids, vocab, out=buf[:, :w])
    assert bool((buf[:, w:] == 5).all())
    if n > 100:
      check_grad(buf[:, :w], grad, ids, vocab, 1.0, None)
    else:
      assert int((buf[:, :w] != 0).any(1).sum()) == torch.unique(ids).numel()


@pytest.mark.parametrize("n,width,t", [(8192, 2048, torch.float32), (2000, 8001, torch.bfloat16), (250, 65536, torch.float32), (2049, 513, torch.float16),
                                       (2048, 512, torch.float32), (2048, 513, torch.float32), (1500, 4099, torch.bfloat16), (64, 8192, torch.float16)])
@pytest.mark.parametrize("kind", ["hubs", "same"])
def test_short_lists_of_wide_rows(ops, n, width, t, kind):
  """rows over many column blocks, up to the most values that a short list has, and their sums again"""
  vocab = 300
  g = torch.Generator(device=DEV).manual_seed(n + width)
  ids = make_ids(kind, n, vocab, n).clamp_(max=vocab - 1).to(DEV)
  grad = torch.empty(n, width, device=DEV).normal_(generator=g).to(t)
  got = ops.embedding_backward(grad, ids, vocab, scale=0.5)
  G = torch.zeros(vocab, width, device=DEV, dtype=torch.float64).index_add_(0, ids, grad.double()).mul_(0.5)
  S = torch.zeros(vocab, width, device=DEV, dtype=torch.float64).index_add_(0, ids, grad.double().abs()).mul_(0.5)
  m = torch.bincount(ids, minlength=vocab)[:, None]
  assert bool(((got.double() - G).abs() <= 1.01 * ((m + 2) * U * S + half(t) * G.abs()) + tiny(t)).all())
  rg = ops.embedding_backward_rows(grad, ids, vocab, scale=0.5)
  k = int(rg.count)
  assert torch.equal(rg.ids[:k], torch.unique(ids)) and torch.equal(rg.rows[:k], got[rg.ids[:k]])
  assert torch.equal(ops.embedding_backward(grad, ids, vocab, scale=0.5), got)


def test_autograd_captured(ops):
  """forward and backward in one graph (no eager graph of the leaf is alive), replayed with other contents beside eager work"""
  from orca_amd import torch_ops  # noqa: F401
  vocab, w, n = 900, 24, 1500
  table = torch.randn(vocab, w, device=DEV).requires_grad_()
  ids, wgt = torch.zeros(n, dtype=torch.int64, device=DEV), torch.zeros(n, w, device=DEV)

  def step():
    out = torch.ops.orca.embedding(table, ids, 0.5, 0)
    return torch.autograd.grad(out, table, wgt)[0]

  s = torch.cuda.Stream()
  s.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(s):
    for _ in range(2):
      step()
  torch.cuda.current_stream().wait_stream(s)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    grad = step()
  for r in range(3):
    g = torch.Generator().manual_seed(r)
    ids.copy_(torch.randint(0, vocab, (n,), generator=g))
    wgt.copy_(torch.randn(n, w, generator=g))
    graph.replay()
    torch.cuda.synchronize()
    check_grad(grad, wgt, ids, vocab, 0.5, 0)
    assert torch.equal(grad, ops.embedding_backward(wgt, ids, vocab, 0.5, 0)), f"replay {r}"


@pytest.mark.parametrize("n", [8193, 20001, 70000, 131072, 131073])
@pytest.mark.parametrize("vocab", [1, 100, 1 << 14, 400_000, 4_000_003, 10_000_001, (1 << 31) - 2])
def test_long_lists_and_row_numbers(ops, n, vocab):
  """every number of passes, digit widths, and one to four pairs per thread: half the ids are hubs"""
  g = torch.Generator().manual_seed(n + vocab % 1000)
  ids = torch.where(torch.rand(n, generator=g) < 0.5, torch.randint(0, vocab, (n,), generator=g), torch.randint(0, 9, (n,), generator=g) * 7919 % vocab)
  ids[0], ids[1], ids[2] = vocab - 1, -1, vocab
  grad = torch.randn(n, 3, generator=g)
  rg = ops.embedding_backward_rows(grad.to(DEV), ids.to(DEV), vocab, padding_idx=7919 % vocab if vocab > 1 else None)
  ok = (ids >= 0) & (ids < vocab) & ((ids != 7919 % vocab) | (vocab == 1))
  u, inv = torch.unique(ids[ok], return_inverse=True)
  k = int(rg.count)
  assert k == u.numel() and torch.equal(rg.ids[:k].cpu(), u)
  z = torch.zeros(k, 3, dtype=torch.float64)
  G, S = z.clone().index_add_(0, inv, grad[ok].double()), z.index_add_(0, inv, grad[ok].double().abs())
  assert bool(((rg.rows[:k].cpu().double() - G).abs() <= bound(G, S, torch.bincount(inv), torch.float32)).all())
