"""Short lists over tables whose rows the sums' workgroups mark and zero themselves, up to the most that they can mark (65,536 rows for each of
256 workgroups), and the first tables that are filled ahead instead; the other tests' tall tables are all filled ahead.

Tolerance: sums of m fp32 values, one product: (m + 2) 2^-24 sum|g| and half a step of the output's type, widened by 1 %; and half the type's
smallest step: below the smallest normal value v the steps are v * eps apart for all values (fp16: 2^-14 and 2^-24, so that a value under 2^-14 is
off by up to 2^-25 however small it is)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
MOST = 256 * 65536


@pytest.fixture(scope="module")
def ops():
  from orca_amd import ops as o
  return o


def check(ops, ids, vocab, width, dtype, seed, out=None):
  n = ids.numel()
  grad = torch.randn(n, width, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)
  got = ops.embedding_backward(grad, ids, vocab, scale=0.5, out=out)
  keep = (ids >= 0) & (ids < vocab)
  u, inv = torch.unique(ids[keep].long(), return_inverse=True)
  z = torch.zeros(u.numel(), width, dtype=torch.float64, device=DEV)
  G, S = z.clone().index_add_(0, inv, grad[keep].double()) * 0.5, z.index_add_(0, inv, grad[keep].double().abs()) * 0.5
  m = torch.bincount(inv)[:, None]
  half, least = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
  assert bool(((got[u].double() - G).abs() <= 1.01 * ((m + 2) * U * S + half * G.abs()) + least).all())
  touched = torch.zeros(vocab, dtype=torch.bool, device=DEV)
  touched[u] = True
  assert not bool((got.ne(0).any(1) & ~touched).any()), "rows without an occurrence are zero"
  return u


def edges(vocab, n, seed):
  """ids at both ends of every workgroup's share, among random ones and ids outside the table"""
  g = torch.Generator().manual_seed(seed)
  ids = torch.randint(0, vocab, (n,), generator=g)
  share = vocab * torch.arange(257) // 256
  at = torch.cat([share[:-1], share[1:] - 1])
  k = min(n // 2, at.numel())
  ids[:k] = at[torch.linspace(0, at.numel() - 1, k).long()]
  ids[-3:] = torch.tensor([-1, vocab, vocab + 63])
  return ids.to(DEV)


@pytest.mark.parametrize("vocab,width,dtype", [(MOST, 1, torch.float32), (MOST - 1, 1, torch.float32), (MOST, 4, torch.bfloat16), (MOST - 65537, 2, torch.float16),
                                               (MOST + 1, 1, torch.float32), (400_000, 100, torch.float32), (400_001, 100, torch.float32)])
@pytest.mark.parametrize("n", [2500, 8192])
def test_tall_tables_of_mid_sized_lists(ops, vocab, width, dtype, n):
  """up to 160 MB (the last ones are at and past it), into memory that holds something else"""
  out = torch.full((vocab, width), 3.0, dtype=dtype, device=DEV)
  check(ops, edges(vocab, n, vocab % 1000 + n), vocab, width, dtype, n, out)


@pytest.mark.parametrize("vocab,width,dtype", [(9_999_999, 1, torch.bfloat16), (10_000_000, 1, torch.float16), (5_000_000, 1, torch.float32), (49_999, 100, torch.float32),
                                               (50_001, 100, torch.float32), (2_500_000, 4, torch.bfloat16)])
@pytest.mark.parametrize("n", [1, 64, 600, 2048])
def test_tables_of_tiny_lists(ops, vocab, width, dtype, n):
  """up to 20 MB (and one past it)"""
  out = torch.full((vocab, width), 3.0, dtype=dtype, device=DEV)
  ids = edges(vocab, n, n) if n >= 64 else torch.tensor([vocab - 1], device=DEV)
  check(ops, ids, vocab, width, dtype, n, out)


def test_ids_packed_into_one_share(ops):
  """all occurrences in one workgroup's rows, the last bit of its map among them"""
  vocab = MOST
  ids = torch.cat([torch.arange(vocab - 3000, vocab), torch.arange(65536 - 500, 65536 + 500)]).to(DEV)
  u = check(ops, ids, vocab, 1, torch.float32, 5, torch.full((vocab, 1), 3.0, device=DEV))
  assert u.numel() == 4000
