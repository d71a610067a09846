"""orca_grad_norm / orca_clip_grads (ops.grad_norm, ops.clip_grad_norm) against fp64.

Tolerances (u = 2^-24, h = half a step of a gradient's type, t = half its smallest step): squares and sums are fp64, so the norm is
off by its rounding to fp32, u (and 2^-40 for everything in 64 bits); a clipped value by the rounding of the coefficient, of the
product and to its type: (2u + h) |x| + t, widened by 1 % for second-order terms."""
import math

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


def make(sizes, types, seed=0, std=0.1):
  g = torch.Generator().manual_seed(seed)
  return [(torch.randn(s, generator=g) * std).to(types[i % len(types)]).to(DEV) for i, s in enumerate(sizes)]


def norm64(grads):
  return math.sqrt(sum(float((x.double() ** 2).sum()) for x in grads))


def check_norm(got, want):
  assert got.dtype == torch.float32 and got.shape == ()
  assert abs(float(got) - want) <= want * (U + 2.0 ** -40) * 1.01


def check_scaled(got, x, c):
  exp = x.cpu().double() * c
  t = x.dtype
  lim = 1.01 * (2 * U + half(t)) * exp.abs() + torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
  assert got.dtype == t and bool(((got.cpu().double().reshape(exp.shape) - exp).abs() <= lim).all())


LISTS = {
    "one value": [1],
    "empty among them": [0, 5, 0, 0, 77, 0],
    "tile edges": [8191, 8192, 8193, 16384, 1, 16385],
    "97 tensors": [3 + 37 * i for i in range(97)],
    "300 tensors": [1 + (i * 7919) % 2500 for i in range(300)],
    "one large": [3_000_001],
    "large and small": [5_000_000, 1, 100, 141600, 3],
}


@pytest.mark.parametrize("types", [TYPES[:1], TYPES[1:2], TYPES[2:], TYPES], ids=["f32", "bf16", "f16", "mixed"])
@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("max_norm", [0.5, 1e6])
def test_norm_and_clip(ops, types, name, max_norm):
  grads = make(LISTS[name], types)
  keep = [x.clone() for x in grads]
  want = norm64(grads)
  c = min(1.0, max_norm / (want + 1e-6))
  check_norm(ops.grad_norm(grads), want)
  norm, coef = ops.grad_norm({str(i): x for i, x in enumerate(grads)}, max_norm)
  check_norm(norm, want)
  assert abs(float(coef) - c) <= U * c * 1.01
  order = list(dict.fromkeys(x.dtype for x in grads))
  flat = [torch.full((sum(x.numel() for x in grads if x.dtype is t) + 4,), 5.0, dtype=t, device=DEV) for t in order]
  check_norm(ops.clip_grad_norm(grads, max_norm, flat=[f[1:-3] for f in flat]), want)
  assert all(torch.equal(a, b) for a, b in zip(grads, keep)), "with flat buffers the gradients stay"
  for t, f in zip(order, flat):
    assert bool((f[:1] == 5).all()) and bool((f[-3:] == 5).all())
    check_scaled(f[1:-3], torch.cat([x for x in keep if x.dtype is t]), c)
  check_norm(ops.clip_grad_norm(grads, max_norm), want)
  at = {t: 1 for t in order}
  for a, b in zip(grads, keep):
    n = a.numel()
    f = flat[order.index(a.dtype)][at[a.dtype]:at[a.dtype] + n]
    at[a.dtype] += n
    assert torch.equal(a, f), "in place and flat: the same bits"
    if c == 1.0:
      assert torch.equal(a, b)


def test_same_bits_and_torch(ops):
  grads = make([100, 40000, 74400, 31, 141600, 1], TYPES[:1], seed=3)
  a, b = ops.grad_norm(grads), ops.grad_norm(grads)
  assert torch.equal(a, b)
  ps = [torch.nn.Parameter(x.clone()) for x in grads]
  for p, x in zip(ps, grads):
    p.grad = x.clone()
  t = torch.nn.utils.clip_grad_norm_(ps, 2.0)
  ops.clip_grad_norm(grads, 2.0)
  assert abs(float(t) - float(a)) <= 1e-5 * float(a)           # torch adds in fp32
  for p, x in zip(ps, grads):
    assert float((p.grad - x).abs().max()) <= 1e-5 * float(x.abs().max())


def test_no_overflow_no_underflow(ops):
  big = [torch.full((1000,), 1e30, device=DEV), torch.full((3,), 2e38, device=DEV)]
  check_norm(ops.grad_norm(big[:1]), norm64(big[:1]))
  assert math.isinf(float(ops.grad_norm([torch.full((100,), 3e38, device=DEV)])))       # the norm itself is past fp32
  small = [torch.full((5000,), 1e-30, device=DEV)]
  check_norm(ops.grad_norm(small), norm64(small))


def test_not_finite(ops):
  """as torch: a NaN norm makes everything NaN, an infinite one makes finite values 0 and the infinite ones NaN"""
  for bad, other in ((float("nan"), None), (float("inf"), 0.0), (float("-inf"), 0.0)):
    grads = make([100, 9000], TYPES[:2])
    grads[1][8999] = bad
    norm = ops.clip_grad_norm(grads, 1.0)
    assert (math.isnan(float(norm)) if other is None else math.isinf(float(norm)))
    assert bool(grads[1][8999].isnan())
    assert bool(grads[0].isnan().all() if other is None else (grads[0] == 0).all())


def test_zero_gradients_and_empty_lists(ops):
  z = [torch.zeros(50, device=DEV)]
  assert float(ops.clip_grad_norm(z, 1.0)) == 0.0 and bool((z[0] == 0).all())
  assert float(ops.grad_norm([])) == 0.0 and float(ops.clip_grad_norm([], 1.0)) == 0.0
  assert float(ops.grad_norm([None, torch.ones(4, device=DEV), None])) == 2.0
  assert float(ops.clip_grad_norm([torch.empty(0, device=DEV)], 1.0)) == 0.0
  g = [torch.ones(4, device=DEV)]
  assert float(ops.clip_grad_norm(g, 0.0)) == 2.0 and bool((g[0] == 0).all())


def test_views(ops):
  """transposed, strided and offset tensors; a base whose other elements stay"""
  base = torch.randn(60, 70, generator=torch.Generator().manual_seed(1)).to(DEV)
  keep = base.clone()
  flat = torch.randn(1001, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
  fk = flat.clone()
  grads = [base[:30, :20].t(), base[30:, 40:], flat[1:998]]
  want = norm64(grads)
  c = 0.25 / (want + 1e-6)
  check_norm(ops.clip_grad_norm(grads, 0.25), want)
  check_scaled(grads[0], keep[:30, :20].t(), c)
  check_scaled(grads[1], keep[30:, 40:], c)
  check_scaled(flat[1:998], fk[1:998], c)
  assert torch.equal(flat[:1], fk[:1]) and torch.equal(flat[998:], fk[998:])
  assert torch.equal(base[:30, 20:], keep[:30, 20:]) and torch.equal(base[30:, :40], keep[30:, :40])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count", [0, 1, 17, 600])
def test_row_sparse_gradients(ops, dtype, count):
  """only the first *count rows are there; the others (NaN here) are not read and not written"""
  rows = torch.randn(600, 37, generator=torch.Generator().manual_seed(count)).to(dtype).to(DEV)
  rows[count:] = float("nan")
  keep = rows.clone()
  rg = ops.RowGrad(torch.arange(600, device=DEV), rows, torch.tensor([count], dtype=torch.int32, device=DEV), 1000)
  dense = make([501], [dtype])[0]
  want = norm64([rows[:count], dense])
  check_norm(ops.grad_norm([rg, dense]), want)
  c = min(1.0, 0.5 / (want + 1e-6))
  flat = torch.full((600 * 37 + 501,), 4.0, dtype=dtype, device=DEV)
  check_norm(ops.clip_grad_norm([rg, dense], 0.5, flat=[flat]), want)
  check_scaled(flat[:count * 37].view(count, 37), keep[:count], c)
  assert bool((flat[count * 37:600 * 37] == 4).all())
  check_norm(ops.clip_grad_norm([rg, dense], 0.5), want)
  check_scaled(rows[:count], keep[:count], c)
  assert bool(rows[count:].isnan().all())


def test_many_row_sparse_gradients(ops):
  """more of them than one launch takes, between dense ones"""
  g = torch.Generator().manual_seed(7)
  rgs = [ops.RowGrad(torch.arange(50, device=DEV), torch.randn(50, 9 + i, generator=g).to(DEV),
                     torch.tensor([3 * i], dtype=torch.int32, device=DEV), 100) for i in range(11)]
  dense = make([4097, 3, 20000], TYPES[:1])
  lst = [dense[0]] + rgs[:6] + [dense[1]] + rgs[6:] + [dense[2]]
  keep = [r.rows.clone() for r in rgs]
  want = norm64([r.rows[:3 * i] for i, r in enumerate(rgs)] + dense)
  check_norm(ops.grad_norm(lst), want)
  flat = torch.full((sum(r.rows.numel() for r in rgs) + sum(d.numel() for d in dense),), 6.0, device=DEV)
  check_norm(ops.clip_grad_norm(lst, 0.5, flat=[flat]), want)
  c, at = 0.5 / (want + 1e-6), dense[0].numel()
  for i, r in enumerate(rgs):
    n, live = r.rows.numel(), 3 * i * r.rows.shape[1]
    check_scaled(flat[at:at + live].view(3 * i, -1) if i else flat[:0].view(0, 9), keep[i][:3 * i], c)
    assert bool((flat[at + live:at + n] == 6).all())
    at += n + (dense[1].numel() if i == 5 else 0)
  check_norm(ops.clip_grad_norm(lst, 0.5), want)
  for i, r in enumerate(rgs):
    check_scaled(r.rows[:3 * i], keep[i][:3 * i], c)
    assert torch.equal(r.rows[3 * i:], keep[i][3 * i:])


def test_large_flat_copy(ops):
  """a list of 120 MB: read and written past the caches"""
  grads = [torch.randn(s, generator=torch.Generator(device=DEV).manual_seed(s), device=DEV) * 0.01 for s in (20_000_001, 9_999_999, 5)]
  flat = torch.empty(sum(x.numel() for x in grads), device=DEV)
  want = norm64(grads)
  check_norm(ops.clip_grad_norm(grads, 1.0, flat=[flat]), want)
  exp = torch.cat(grads).double() * (1.0 / (want + 1e-6))
  assert bool(((flat.double() - exp).abs() <= 1.01 * 3 * U * exp.abs() + 1e-45).all())


def test_captured_and_replayed(ops):
  grads = make([100, 40000, 3, 9001], TYPES)
  flat = [torch.empty(sum(x.numel() for x in grads if x.dtype is t), dtype=t, device=DEV) for t in dict.fromkeys(x.dtype for x in grads)]
  ops.clip_grad_norm(grads, 1.0, flat=flat)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    norm = ops.clip_grad_norm(grads, 1.0, flat=flat)
  for r in range(4):
    for x, y in zip(grads, make([100, 40000, 3, 9001], TYPES, seed=10 + r, std=0.3)):
      x.copy_(y)
    graph.replay()
    torch.cuda.synchronize()
    got = [f.clone() for f in flat]
    e = ops.clip_grad_norm(grads, 1.0, flat=flat)
    assert torch.equal(norm, e) and all(torch.equal(a, b) for a, b in zip(got, flat)), f"replay {r}"


def test_refusals(ops):
  g = torch.ones(4, device=DEV)
  with pytest.raises(TypeError):
    ops.grad_norm([g.double()])
  with pytest.raises(TypeError):
    ops.grad_norm([3.0])
  from orca_amd._lib import OrcaError
  with pytest.raises(OrcaError):
    ops.grad_norm([g, g.cpu()])
  with pytest.raises(ValueError):
    ops.clip_grad_norm([g, g], 1.0)
  with pytest.raises(ValueError):
    ops.clip_grad_norm([g], -1.0)
  with pytest.raises(ValueError):
    ops.clip_grad_norm([g], float("nan"))
  with pytest.raises(ValueError):
    ops.clip_grad_norm([g[:1].expand(9)], 1.0)
  with pytest.raises(ValueError):
    ops.clip_grad_norm([g], 1.0, flat=[torch.empty(5, device=DEV)])
  with pytest.raises(ValueError):
    ops.clip_grad_norm([g], 1.0, flat=[])
  assert bool((g == 1).all())


def test_overlaps_are_refused(ops):
  buf = torch.ones(100, device=DEV)
  with pytest.raises(ValueError, match="overlap"):
    ops.clip_grad_norm([buf[:50], buf[49:]], 1.0)
  with pytest.raises(ValueError, match="overlap"):
    ops.clip_grad_norm([buf[:50]], 1.0, flat=[buf[40:90]])
  with pytest.raises(ValueError, match="overlap"):
    ops.clip_grad_norm([buf[:10], torch.ones(4, device=DEV, dtype=torch.float16)], 1.0, flat=[buf[20:30], buf.view(torch.float16)[58:62]])
  assert bool((buf == 1).all())
  # neighbours: 20 squares of 1
  norm = ops.clip_grad_norm([buf[:10], buf[10:20]], 1e-3, flat=[buf[20:40]])
  assert abs(float(norm) - 20 ** 0.5) <= 20 ** 0.5 * 2 * U and bool((buf[:20] == 1).all()) and bool((buf[20:40] < 1).all()) and bool((buf[40:] == 1).all())


def test_on_another_stream(ops):
  s = torch.cuda.Stream()
  grads = make([100, 300000], TYPES[:1], seed=4)
  want = [x.clone() for x in grads]
  n0 = ops.clip_grad_norm(want, 0.5)
  torch.cuda.synchronize()
  with torch.cuda.stream(s):
    got = [x * 1.0 for x in grads]
    n1 = ops.clip_grad_norm(got, 0.5)
  s.synchronize()
  assert torch.equal(n0, n1) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("flat", [True, False])
@pytest.mark.parametrize("parts", [1, 700])
def test_long_lists(ops, flat, parts):
  """170 MB (three launches, a piece or four per workgroup) as one tensor and as hundreds, odd sizes, with a row-sparse one in front"""
  sizes = [85000001 // parts + (i % 3) for i in range(parts)]
  base = torch.randn(sum(sizes), device=DEV, generator=torch.Generator(DEV).manual_seed(parts)).bfloat16()
  grads, at = [], 0
  for k in sizes:
    grads.append(base[at:at + k])
    at += k
  rows = ops.RowGrad(torch.arange(50, device=DEV), torch.full((50, 7), 3.0, device=DEV), torch.full((1,), 20, dtype=torch.int32, device=DEV), 50)
  want = float((base.double().square().sum() + 140 * 9.0).sqrt())
  before, out = base.clone(), [torch.full((350,), 8.0, device=DEV), torch.empty_like(base)]
  max_norm = want / 3
  norm = ops.clip_grad_norm([rows] + grads, max_norm, flat=out if flat else None)
  # the norm: fp64 sums, one rounding to fp32.  The products: a coefficient rounded to fp32, one product, one rounding to bf16
  assert abs(float(norm) - want) <= want * 2 * U
  exp = before.double() * (max_norm / (want + 1e-6))
  got = (out[1] if flat else base).double()
  assert bool(((got - exp).abs() <= exp.abs() * (2.0 ** -8 + 4 * U)).all())
  r = out[0] if flat else rows.rows.reshape(-1)
  assert bool(((r[:140] - 1.0).abs() <= 4 * U + 1e-6 / want * 2).all()) and bool((r[140:] == (8.0 if flat else 3.0)).all())
  if flat:
    assert torch.equal(base, before)
  else:
    again = base.clone()
    ops.clip_grad_norm(grads, 1e9)
    assert torch.equal(base, again)
  n1, c = ops.grad_norm([before] if parts == 1 else [g.clone() for g in grads], max_norm)
  assert bool(torch.isfinite(n1)) and 0 < float(c) < 1
