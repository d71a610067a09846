"""Outputs that share memory with what a call reads are refused, whatever the strides; views of one buffer that do not meet are not."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
  from orca_amd import ops as o
  return o


def test_strided_tables(ops):
  buf = torch.randn(20, 16, device=DEV)
  keep = buf.clone()
  ids = torch.tensor([1, 0, 19], device=DEV)
  table = buf[:, :8]
  for out in (buf[2:3, :8], buf.view(-1)[:24].view(3, 8), buf.view(-1)[296:].view(3, 8), buf[:, 4:12][:1]):
    with pytest.raises(ValueError, match="overlaps"):
      ops.embedding(table, ids[:out.shape[0]], out=out)
  assert torch.equal(buf, keep)
  got = ops.embedding(table, ids[:1], out=buf[5:6, 8:])                    # the gap behind a row
  assert torch.equal(got, keep[1:2, :8]) and torch.equal(buf[:, :8], keep[:, :8])
  tail = torch.randn(40, 16, device=DEV)
  assert torch.equal(ops.embedding(tail[:20, :8], ids, out=tail.view(-1)[312:336].view(3, 8)), tail[ids, :8])      # behind the last row


def test_strided_gradients(ops):
  buf = torch.randn(12, 24, device=DEV)
  keep = buf.clone()
  ids = torch.tensor([1, 0, 3, 1], device=DEV)
  for out in (buf[3:8, :8], buf[3:8, 4:12], buf[:5, 7:15], buf[3:4, :8]):
    with pytest.raises(ValueError, match="overlaps"):
      ops.embedding_backward(buf[:4, :8], ids, out.shape[0], out=out)
  with pytest.raises(ValueError, match="overlaps"):
    ops.embedding_backward(buf[:1, :8].expand(4, 8), ids, 5, out=buf[:5, 4:12])
  assert torch.equal(buf, keep)
  want = ops.embedding_backward(keep[:4, :8], ids, 5)
  for out in (buf[:5, 8:16], buf[4:9, :8], buf[7:, 16:]):                  # other columns, other rows
    assert torch.equal(ops.embedding_backward(buf[:4, :8], ids, 5, out=out), want)
  assert torch.equal(buf[:4, :8], keep[:4, :8])
