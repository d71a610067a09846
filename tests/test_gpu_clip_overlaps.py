"""Lists of gradients whose tensors share memory, by the tensors themselves and not by the copies that the call makes of strided ones."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
  from orca_amd import ops as o
  return o


def test_strided_tensors_twice(ops):
  base = torch.randn(30, 40, device=DEV)
  cube = torch.randn(6, 7, 8, device=DEV)
  keep, keep3 = base.clone(), cube.clone()
  for bad in ([base, base.t()], [base.t(), base.t()], [base[:, :20], base[:, :20]], [base[:, :21], base[:, 20:]], [base[:, ::2], base[5:6]],
              [base[:, :5], base[3:].t()], [cube[:, 1:3], cube[:, :, 2:4]], [cube[::2, 1:3, ::3], cube[4, 2]], [cube[:4], cube[3:, :, 1:]],
              [base[:3], cube, base[2:, :7]]):
    with pytest.raises(ValueError, match="overlap"):
      ops.clip_grad_norm(bad, 1.0)
  assert torch.equal(base, keep) and torch.equal(cube, keep3)


def test_views_that_interleave(ops):
  """column blocks, even and odd columns, planes of one cube: every element once"""
  base, cube = torch.randn(30, 40, device=DEV), torch.randn(6, 7, 8, device=DEV)
  keep = torch.cat([base.reshape(-1), cube.reshape(-1)]).double().cpu()
  parts = [base[:, :11].t(), base[:, 11:20], base[:, 20::2], base[:, 21::2], cube[:, :3, :4], cube[:, 3:, :4], cube[:, :, 4:6].permute(2, 0, 1), cube[:, :, 6:]]
  want = float(keep.square().sum().sqrt())
  norm = ops.clip_grad_norm(parts, 0.5)
  assert abs(float(norm) - want) <= 1.01 * U * want
  exp = keep * (0.5 / (want + 1e-6))
  got = torch.cat([base.reshape(-1), cube.reshape(-1)]).double().cpu()
  assert bool(((got - exp).abs() <= 1.01 * 3 * U * exp.abs()).all())        # coefficient, product, one more for the second order


def test_flat_buffers_and_strided_gradients(ops):
  """a flat buffer inside the storage of a gradient that is copied"""
  buf = torch.randn(20, 16, device=DEV)
  keep = buf.clone()
  g = buf[:, :4]
  with pytest.raises(ValueError, match="overlaps a gradient"):
    ops.clip_grad_norm([g], 1.0, flat=[buf.view(-1)[:80]])
  with pytest.raises(ValueError, match="overlaps a gradient"):
    ops.clip_grad_norm([buf.t()[:4]], 1.0, flat=[buf.view(-1)[240:]])
  assert torch.equal(buf, keep)
  small = torch.randn(2, 3, device=DEV)
  ops.clip_grad_norm([buf[:3, :2]], 1.0, flat=[buf.view(-1)[34:40]])          # behind the last row
  assert torch.equal(buf[:3, :2], keep[:3, :2]) and not torch.equal(buf[2, 2:8], keep[2, 2:8])
  assert math.isfinite(float(ops.clip_grad_norm([small.t()], 1.0)))


def test_an_empty_gradient_inside_a_flat_buffer(ops):
  """it has no byte to share, whatever its address"""
  buf, g = torch.ones(10, device=DEV), torch.full((4,), 2.0, device=DEV)
  norm = ops.clip_grad_norm([buf[2:2], g], 1.0, flat=[buf[:4]])
  assert abs(float(norm) - 4.0) <= 8 * U and bool((buf[4:] == 1).all()) and bool((buf[:4] < 1).all())
