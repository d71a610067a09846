"""What the embedding and clipping entry points refuse, checked without a GPU: CPU tensors at the Python boundary, and arguments at
the C boundary (every refusal comes before the first launch, so the made-up addresses are never used)."""
import ctypes

import pytest
import torch

from orca_amd import _lib, ops

P = 0x1000      # an address that nothing reads


def refused(rc, text):
  assert rc == -1, rc
  assert text in _lib.load().orca_last_error().decode(), _lib.load().orca_last_error()


def test_no_cpu_tensors():
  t, ids, g = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64), torch.zeros(3, 8)
  for call in (lambda: ops.embedding(t, ids), lambda: ops.embedding_backward(g, ids, 4), lambda: ops.embedding_backward_rows(g, ids, 4),
               lambda: ops.grad_norm([g]), lambda: ops.clip_grad_norm([g], 1.0)):
    with pytest.raises(_lib.OrcaError):
      call()
  for call in (lambda: ops.embedding(t.double(), ids), lambda: ops.embedding_backward(g.int(), ids, 4), lambda: ops.grad_norm([g.double()]),
               lambda: ops.grad_norm(["x"])):
    with pytest.raises(TypeError):
      call()


def forward(dtype=0, n_rows=4, width=8, ld=8, i64=P, i32=None, n=3, out=P, table=P):
  return _lib.load().orca_embedding_forward(table, dtype, n_rows, width, ld, i64, i32, n, 1.0, out, None)


def test_forward_refusals():
  refused(forward(dtype=3), "unknown type")
  refused(forward(dtype=-1), "unknown type")
  refused(forward(width=0), "width")
  refused(forward(width=65537), "width")
  refused(forward(n=-1), "negative size")
  refused(forward(n_rows=-1), "negative size")
  refused(forward(ld=-8), "negative size")
  refused(forward(table=None), "null")
  refused(forward(out=None), "null")
  refused(forward(i64=None), "list of ids")
  refused(forward(i32=P), "list of ids")
  refused(forward(n=1 << 39, width=65536), "too many")
  assert forward(n=0, table=None, i64=None, out=None) == 0


def backward(rows=False, g=P, dtype=0, ld=8, i64=P, i32=None, n=3, width=8, num_rows=4, out=P, out_dtype=0, ld_out=8, ws=P, ws_bytes=1 << 40, ids=P, count=P):
  L = _lib.load()
  if rows:
    return L.orca_embedding_backward_rows(g, dtype, ld, i64, i32, n, width, num_rows, -1, 1.0, ids, out, out_dtype, count, ws, ws_bytes, None)
  return L.orca_embedding_backward(g, dtype, ld, i64, i32, n, width, num_rows, -1, 1.0, 0, out, out_dtype, ld_out, ws, ws_bytes, None)


@pytest.mark.parametrize("rows", [False, True])
def test_backward_refusals(rows):
  refused(backward(rows, n=-1), "ids")
  refused(backward(rows, n=1 << 31), "ids")
  refused(backward(rows, num_rows=(1 << 31) - 1), "rows")
  refused(backward(rows, num_rows=-1), "rows")
  refused(backward(rows, width=0), "width")
  refused(backward(rows, width=65537), "width")
  refused(backward(rows, dtype=1, out_dtype=2), "type")
  refused(backward(rows, dtype=0, out_dtype=1), "type")
  refused(backward(rows, dtype=5, out_dtype=5), "type")
  refused(backward(rows, g=None), "null gradient")
  refused(backward(rows, i64=None), "list of ids")
  refused(backward(rows, i32=P), "list of ids")
  refused(backward(rows, ld=-1), "stride")
  refused(backward(rows, ws=None), "workspace")
  need = _lib.load().orca_embedding_backward_workspace_bytes(3, 8, 4)
  refused(backward(rows, ws_bytes=need - 1), "workspace")
  if rows:
    refused(backward(True, count=None), "null output")
    refused(backward(True, ids=None), "null output")
    refused(backward(True, out=None), "null output")
  else:
    refused(backward(out=None), "null table")
    refused(backward(ld_out=7), "overlap")
    assert backward(num_rows=0, out=None) == 0


def test_workspace_sizes():
  f = _lib.load().orca_embedding_backward_workspace_bytes
  assert f(0, 1, 0) >= 0 and f((1 << 31) - 1, 1, (1 << 31) - 2) > 0
  for bad in ((-1, 8, 4), (1 << 31, 8, 4), (3, 0, 4), (3, 65537, 4), (3, 8, -1), (3, 8, (1 << 31) - 1)):
    assert f(*bad) == -1
  assert _lib.load().orca_grad_norm_workspace_bytes() > 0


def clip(n=1, grads=(P,), sizes=(4,), dtypes=b"\0", rows=None, widths=None, max_norm=1.0, flat=None, norm=P, ws=P, norm_only=False):
  a = lambda t, v: None if v is None else (t * max(len(v), 1))(*v)
  args = [n, a(ctypes.c_void_p, grads), a(ctypes.c_int64, sizes), dtypes, a(ctypes.c_void_p, rows), a(ctypes.c_int32, widths), max_norm]
  if norm_only:
    return _lib.load().orca_grad_norm(*args, norm, None, ws, None)
  return _lib.load().orca_clip_grads(*args, a(ctypes.c_void_p, flat), norm, ws, None)


@pytest.mark.parametrize("norm_only", [False, True])
def test_clip_refusals(norm_only):
  bad = lambda text, **kw: refused(clip(norm_only=norm_only, **kw), text)
  bad("tensors", n=-1)
  bad("tensors", n=65537)
  bad("null", norm=None)
  bad("null", ws=None)
  bad("null", grads=None)
  bad("max_norm", max_norm=-0.5)
  bad("max_norm", max_norm=float("nan"))
  bad("null, or a bad size", grads=(0,))
  bad("null, or a bad size", sizes=(-1,))
  bad("null, or a bad size", sizes=(1 << 40,))
  bad("unknown type", dtypes=b"\3")
  bad("null", rows=(P,))
  bad("width", rows=(P,), widths=(0,))
  if not norm_only:
    bad("no flat buffer", flat=(0, P, P))


def test_adam_rows_refusals():
  def rows(ids=P, g=P, count=P, room=3, num_rows=4, width=8, p=P, m=P, v=P, step=1):
    return _lib.load().orca_adam_rows(ids, g, count, room, num_rows, width, p, m, v, 1e-3, 0.9, 0.999, 1e-8, step, None, None)
  for bad in (dict(room=-1), dict(room=1 << 31), dict(num_rows=-1), dict(width=0), dict(step=0)):
    refused(rows(**bad), "bad sizes")
  for bad in ("ids", "g", "count", "p", "m", "v"):
    refused(rows(**{bad: None}), "null argument")
  assert rows(room=0, ids=None) == 0
  refused(_lib.load().orca_adam_step_scaled(1, None, None, None, None, None, 1e-3, 0.9, 0.999, 1e-8, 1, None, None), "bad arguments")


def test_unaligned_workspaces():
  for rows in (False, True):
    refused(backward(rows, ws=P + 8), "aligned")
  for norm_only in (False, True):
    refused(clip(ws=P + 4, norm_only=norm_only), "aligned")
