"""The longest lists (whose norm is read past the caches) and lists over several launches with more pieces than each launch's share of the
partial sums, against fp64 on the GPU.

Tolerances: the norm carries its rounding to fp32 (2^-24; 2^-40 for everything in 64 bits); a product the coefficient's rounding, its own and
the one to its type: (2 2^-24 + half a step) |x|, and half the type's smallest step; all widened by 1 %."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
  from orca_amd import ops as o
  return o


def norm64(grads):
  return float(torch.stack([sum(p.double().square().sum() for p in g.split(1 << 27)) for g in grads]).sum().sqrt())


def scaled(got, x, c):
  """got == c * x, in pieces (fp64 copies of a list of 800 MB would be 3.2 GB each)"""
  t = x.dtype
  rel, least = 1.01 * (2 * U + torch.finfo(t).eps / 2), torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
  return all(bool(((a.double() - b.double() * c).abs() <= rel * (b.double() * c).abs() + least).all()) for a, b in zip(got.split(1 << 26), x.split(1 << 26)))


@pytest.mark.parametrize("flat", [True, False])
@pytest.mark.parametrize("mb", [640, 660, 800])
def test_past_the_caches(ops, flat, mb):
  """one long 16-bit tensor, others with odd tails, 32-bit ones beside them"""
  g = torch.Generator(device=DEV).manual_seed(mb)
  sizes = [(mb * 1_000_000 - 40_000_000) // 2 + 1, 7, 4_999_999, 1, 5_000_003]
  types = [torch.bfloat16, torch.bfloat16, torch.float32, torch.float32, torch.float32]
  grads = [torch.empty(s, dtype=t, device=DEV).normal_(generator=g) for s, t in zip(sizes, types)]
  keep = [x.clone() for x in grads]
  want = norm64(grads)
  max_norm = want / 7
  c = max_norm / (want + 1e-6)
  out = [torch.full((sum(sizes[:2]) + 8,), 3.0, dtype=torch.bfloat16, device=DEV), torch.full((sum(sizes[2:]) + 8,), 3.0, device=DEV)]
  norm, coef = ops.grad_norm(grads, max_norm)
  assert abs(float(norm) - want) <= 1.01 * want * (U + 2.0 ** -40) and abs(float(coef) - c) <= 1.01 * U * c
  assert torch.equal(norm, ops.clip_grad_norm(grads, max_norm, flat=[f[4:-4] for f in out] if flat else None))
  if flat:
    assert all(torch.equal(a, b) for a, b in zip(grads, keep))
    assert all(bool((f[:4] == 3).all()) and bool((f[-4:] == 3).all()) for f in out)
    got = list(out[0][4:-4].split(sizes[:2])) + list(out[1][4:-4].split(sizes[2:]))
  else:
    got = grads
  assert all(scaled(a, x, c) for a, x in zip(got, keep))


@pytest.mark.parametrize("count,size,dtype", [(700, 50_001, torch.bfloat16), (1300, 40_003, torch.float16), (2500, 6_001, torch.float32), (3100, 20_001, torch.bfloat16),
                                              (3000, 300_001, torch.bfloat16)])
def test_many_launches(ops, count, size, dtype):
  """each launch's workgroups are its share of the partial sums that a call has (2048; of long lists 8192): the sums beyond would lie outside
  the workspace.  A tensor in sixteen differs, so that a workgroup's share that is left out shows in the norm"""
  g = torch.Generator(device=DEV).manual_seed(count)
  base = torch.empty(count * size, device=DEV).normal_(generator=g).to(dtype)
  grads = list(base.split(size))
  for i in range(0, count, 16):
    grads[i].mul_(3)
  keep, want = base.clone(), norm64([base])
  norm, coef = ops.grad_norm(grads, want / 2)
  assert abs(float(norm) - want) <= 1.01 * want * (U + 2.0 ** -40)
  flat = torch.empty_like(base)
  c = want / 2 / (want + 1e-6)
  assert torch.equal(ops.clip_grad_norm(grads, want / 2, flat=[flat]), norm) and scaled(flat, keep, c)
  assert torch.equal(ops.clip_grad_norm(grads, want / 2), norm) and torch.equal(base, flat)


@pytest.mark.parametrize("count", [5, 4096, 4097, 8200])
def test_row_sparse_gradients_by_the_thousand(ops, count):
  """four of them in a launch: up to half of the partial sums are launches, more are refused"""
  rows, n = torch.ones(count, 4, device=DEV), torch.ones(count, dtype=torch.int32, device=DEV)
  lst = [ops.RowGrad(torch.zeros(1, dtype=torch.int64, device=DEV), rows[i:i + 1], n[i:i + 1], 9) for i in range(count)]
  if count > 4096:
    with pytest.raises(ValueError, match="too many"):
      ops.clip_grad_norm(lst, 1.0)
    assert bool((rows == 1).all())
    return
  want = (4.0 * count) ** 0.5
  assert abs(float(ops.clip_grad_norm(lst, want / 2)) - want) <= 1.01 * want * (U + 2.0 ** -40)
  assert bool(((rows - 0.5).abs() <= 4 * U + 1e-6).all())
