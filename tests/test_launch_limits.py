"""A launch has under 2^32 threads: lists that would need more are refused before anything is launched, and the zero fill of a table with
gaps (a piece per row) goes round instead."""
import pytest
import torch

from orca_amd import _lib

P = 0x1000      # an address that nothing reads
DEV = "cuda:0"


def refused(rc, text):
  assert rc == -1, rc
  assert text in _lib.load().orca_last_error().decode()


@pytest.mark.parametrize("dtype,width,chunks", [(0, 1, 1), (0, 4, 1), (1, 7, 7), (0, 100, 25), (2, 65536, 8192)])
def test_lookups_past_a_launch(dtype, width, chunks):
  n = -(-(1 << 34) // chunks)                       # 2^24 workgroups of 256 threads with four chunks each
  refused(_lib.load().orca_embedding_forward(P, dtype, 4, width, width, P, None, n, 1.0, P, None), "too many")


@pytest.mark.parametrize("rows", [False, True])
def test_gradients_past_a_launch(rows):
  L, n, width, ws = _lib.load(), (1 << 31) - 1, 65536, 1 << 60
  if rows:
    rc = L.orca_embedding_backward_rows(P, 0, 0, P, None, n, width, 4, -1, 1.0, P, P, 0, P, P, ws, None)
  else:
    rc = L.orca_embedding_backward(P, 0, 0, P, None, n, width, 4, -1, 1.0, 0, P, 0, width, P, ws, None)
  refused(rc, "too many")


def test_adam_past_a_launch():
  import ctypes
  a = (ctypes.c_void_p * 1)(P)
  size = (ctypes.c_int64 * 1)(1 << 34)
  refused(_lib.load().orca_adam_step(1, a, a, a, a, size, 1e-3, 0.9, 0.999, 1e-8, 1, None), "too many")
  refused(_lib.load().orca_adam_step_scaled(1, a, a, a, a, size, 1e-3, 0.9, 0.999, 1e-8, 1, P, None), "too many")


@pytest.mark.gpu
@pytest.mark.parametrize("n", [0, 3, 9000])
@pytest.mark.parametrize("rows", [(1 << 22) + 5, (1 << 24) + 3, 100_000_001])
def test_fill_of_many_rows_with_gaps(n, rows):
  """more rows than a launch may have workgroups: alone, ahead of a short list, and in the launches of a long list's sort"""
  from orca_amd import ops
  buf = torch.full((rows, 2), 5.0, dtype=torch.bfloat16, device=DEV)
  ids = torch.arange(n, device=DEV) * (rows // max(n, 1)) + (rows - 1) % max(rows // max(n, 1), 1)
  grad = torch.ones(n, 1, dtype=torch.bfloat16, device=DEV)
  ops.embedding_backward(grad, ids, rows, out=buf[:, :1])
  assert bool((buf[:, 1] == 5).all())
  assert int((buf[:, 0] != 0).sum()) == n and bool((buf[ids, 0] == 1).all())
