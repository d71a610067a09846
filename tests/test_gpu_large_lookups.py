"""Lookups whose output goes past the caches (256 MB and more) and those just under it: the rows themselves at scale 1, one rounded product
otherwise, nothing outside the output."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width", [3, 37, 100, 2048])
@pytest.mark.parametrize("mb", [255, 261])
def test_both_sides_of_the_rule(dtype, width, mb):
  from orca_amd import ops
  n = mb * 1_000_000 // (width * torch.finfo(dtype).bits // 8) + 1
  g = torch.Generator(device=DEV).manual_seed(width)
  table = torch.randn(5000, width, device=DEV, generator=g).to(dtype)
  ids = torch.randint(-1, 5001, (n,), device=DEV, generator=g)
  room = torch.full((n * width + 16,), 7.0, dtype=dtype, device=DEV)
  out = ops.embedding(table, ids, out=room[8:-8].view(n, width))
  ok = (ids >= 0) & (ids < 5000)
  want = table[torch.where(ok, ids, 0)] * ok[:, None]
  assert torch.equal(out, want) and bool((room[:8] == 7).all()) and bool((room[-8:] == 7).all())
  assert torch.equal(ops.embedding(table, ids, scale=0.37, out=out), (want.float() * 0.37).to(dtype))      # fp32 product, one rounding
