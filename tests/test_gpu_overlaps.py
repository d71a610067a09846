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


def test_ids_in_the_output(ops):
  """the ids and the output in one storage, seen as different types"""
  buf = torch.zeros(64, dtype=torch.int64, device=DEV)
  buf[:4] = torch.tensor([1, 0, 3, 1], device=DEV)
  f = buf.view(torch.float32)                                    # 128 values: the ids are the first 8
  table, grad = torch.randn(5, 8, device=DEV), torch.randn(4, 8, device=DEV)
  for ids, n in ((buf[:4], 8), (buf.view(torch.int32)[:8:2], 8)):          # (the second is copied: its copy shares nothing)
    if ids.dtype == torch.int64:
      with pytest.raises(ValueError, match="overlaps the ids"):
        ops.embedding(table, ids, out=f[n - 1:n + 31].view(4, 8))
      with pytest.raises(ValueError, match="overlaps the ids"):
        ops.embedding_backward(grad, ids, 5, out=f[n - 2:n + 38].view(5, 8))
    assert torch.equal(ops.embedding(table, ids, out=f[n:n + 32].view(4, 8)), table[ids.long()])
    assert torch.equal(ops.embedding_backward(grad, ids, 5, out=f[n:n + 40].view(5, 8)), ops.embedding_backward(grad, ids.clone(), 5))
  assert buf[:4].tolist() == [1, 0, 3, 1]


def test_row_outputs_in_one_storage(ops):
  ids, grad = torch.tensor([1, 0, 3, 1], device=DEV), torch.randn(4, 8, device=DEV)
  buf = torch.zeros(64, dtype=torch.int64, device=DEV)
  f, i = buf.view(torch.float32), buf.view(torch.int32)
  out = lambda a, r, c: (buf[a:a + 4], f[r:r + 32].view(4, 8), i[c:c + 1])
  for bad in (out(0, 7, 50), out(0, 8, 7), out(0, 8, 39), out(3, 0, 50)):
    with pytest.raises(ValueError, match="overlaps"):
      ops.embedding_backward_rows(grad, ids, 5, out=bad)
  for bad in ((buf[:4], f[8:40].view(4, 8), grad.view(torch.int32)[3, 7:]), (buf[:4], f[8:40].view(4, 8), ids.view(torch.int32)[1:2]),
              (grad.view(torch.int64).view(-1)[12:], f[8:40].view(4, 8), i[60:61]), (buf[:4], ids.view(torch.float32)[:0].expand(0), i[60:61])):
    with pytest.raises(ValueError):
      ops.embedding_backward_rows(grad, ids, 5, out=bad)
  assert not bool(buf.any()) and ids.tolist() == [1, 0, 3, 1]
  got, want = ops.embedding_backward_rows(grad, ids, 5, out=out(0, 8, 40)), ops.embedding_backward_rows(grad, ids, 5)
  assert int(got.count) == int(want.count) == 3 and torch.equal(got.ids[:3], want.ids[:3]) and torch.equal(got.rows[:3], want.rows[:3])


def test_a_flag_without_a_truth_value(ops):
  """what raises when it is asked for its truth value raises out of the call, and nothing is written"""
  class Odd:
    def __bool__(self):
      raise KeyError("no truth value")
  ids, grad, out = torch.tensor([1, 0], device=DEV), torch.ones(2, 4, device=DEV), torch.full((3, 4), 7.0, device=DEV)
  with pytest.raises(KeyError, match="no truth value"):
    ops.embedding_backward(grad, ids, 3, out=out, accumulate=Odd())
  with pytest.raises(RuntimeError):
    ops.embedding_backward(grad, ids, 3, out=out, accumulate=torch.zeros(2))
  assert bool((out == 7).all())
