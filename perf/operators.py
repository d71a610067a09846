"""The cases on which the embedding and gradient-clipping operators are timed and checked.

lookup   out[p] = scale * table[ids[p]]
grad     the gradient of lookup for the table, as a dense table
rows     the same gradient as (ascending distinct ids, their rows, their number on the device)
clip     the 2-norm over a list of gradient tensors, and the tensors scaled to at most max_norm

Ids are "power" (density 1 / rank: tokens by frequency, or hub nodes), "hashed" (the same, spread over the table: node ids carry
no order) or "uniform".  pad >= 0 is the id whose row gets no gradient; an eighth of the ids are it (the samplers fill short
neighbour lists with id 0)."""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
  return [
      # the roots of a batch of 200 interactions ([src; dst; neg]) in a table of the Wikipedia graph's 9,227 nodes: latency
      dict(name="lookup roots", op="lookup", n=600, vocab=9228, width=100, dtype="f32", ids="hashed", wide_ids=True, pad=-1, scale=1.0),
      # an odd width and an odd count in half precision: feature rows of 172 values and one more
      dict(name="lookup odd", op="lookup", n=10007, vocab=54321, width=173, dtype="f16", ids="uniform", wide_ids=False, pad=-1, scale=0.5),
      # the roots and sampled neighbours of 1,365 interactions, K = 10, in a graph of a million nodes
      dict(name="lookup batch", op="lookup", n=45045, vocab=1000001, width=100, dtype="f32", ids="hashed", wide_ids=False, pad=0, scale=1.0),
      # 64 k tokens of a wide 16-bit table, scaled by sqrt(width)
      dict(name="lookup tokens", op="lookup", n=65536, vocab=100000, width=2048, dtype="bf16", ids="power", wide_ids=True, pad=-1, scale=math.sqrt(2048)),
      # the gradients of the same four
      dict(name="grad roots", op="grad", n=600, vocab=9228, width=100, dtype="f32", ids="hashed", wide_ids=True, pad=-1, scale=1.0),
      dict(name="grad batch", op="grad", n=45045, vocab=1000001, width=100, dtype="f32", ids="hashed", wide_ids=False, pad=0, scale=1.0),
      dict(name="grad tokens", op="grad", n=65536, vocab=100000, width=2048, dtype="bf16", ids="power", wide_ids=True, pad=-1, scale=math.sqrt(2048)),
      # row-sparse: 200 interactions with their K = 10 neighbours in the Wiki-Talk graph's 1,140,149 nodes
      dict(name="rows 200", op="rows", n=6600, vocab=1140150, width=100, dtype="f32", ids="hashed", wide_ids=False, pad=0, scale=1.0),
      # row-sparse: 1,365 interactions with K = 20 neighbours in a graph of ten million nodes
      dict(name="rows k20", op="rows", n=85995, vocab=10000001, width=100, dtype="f32", ids="hashed", wide_ids=False, pad=0, scale=1.0),
      # the parameter gradients of a two-layer TGN with 172-d edge features
      dict(name="clip tgn", op="clip", tensors=0, total=0, dtype="f32", second="f32", max_norm=1.0),
      # many small tensors of odd sizes, half of them 16-bit
      dict(name="clip odd", op="clip", tensors=211, total=3000000, dtype="bf16", second="f32", max_norm=1.0),
      # a large model's gradients: matrices in 16 bits, their small vectors in 32
      dict(name="clip large", op="clip", tensors=300, total=400000000, dtype="bf16", second="f32", max_norm=1.0),
  ]


def _log(rng, low, high):
  return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
  """A case of the listed ones' ranges: 1 to 131,072 ids of 1 to 4096 values in tables of 2 to 10 million rows; 1 to 400
  tensors of 1 to 2e8 values in all."""
  op = rng.choice(["lookup", "grad", "rows", "clip"])
  if op == "clip":
    tensors = _log(rng, 1, 400)
    return dict(op=op, tensors=tensors, total=_log(rng, max(tensors, 100), 200000000), dtype=rng.choice(["f32", "bf16", "f16"]),
                second=rng.choice(["f32", "bf16"]), max_norm=rng.choice([0.5, 1.0, 1e6]))
  width = _log(rng, 1, 4096)
  n = min(_log(rng, 1, 131072), 120000000 // width)
  vocab = min(_log(rng, 2, 10000000), 160000000 // width)
  return dict(op=op, n=n, vocab=vocab, width=width, dtype=rng.choice(["f32", "bf16", "f16"]),
              ids=rng.choice(["power", "hashed", "uniform"]), wide_ids=rng.random() < 0.5, pad=rng.choice([-1, 0]),
              scale=rng.choice([1.0, 0.125, math.sqrt(width)]))


def _sizes(case):
  """The sizes of a clip case's tensors, from the case alone; the first of the two types takes the even places."""
  if case["tensors"] == 0:
    layer = [40000, 74400, 74400, 600, 40000, 200, 30000, 100, 10000, 100, 100, 100]
    return layer + layer + [141600, 30000, 300, 300, 20000, 100, 100, 1]
  rng = random.Random(case["tensors"] * 1000003 + case["total"])
  weight = [10.0 ** rng.uniform(-3, 0) if i % 2 else 1.0 + rng.random() for i in range(case["tensors"])]
  left = case["total"] / sum(weight)
  return [max(1, int(w * left)) for w in weight]


def _ids(case, g):
  n, vocab = case["n"], case["vocab"]
  u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
  if case["ids"] == "uniform":
    ids = (u * vocab).long()
  else:
    ids = torch.exp(u * math.log(vocab + 1.0)).long() - 1
    if case["ids"] == "hashed":
      ids = ids * 2654435761 % vocab
  ids.clamp_(0, vocab - 1)
  if case["pad"] >= 0:
    ids = torch.where(torch.rand(n, generator=g, device="cuda") < 0.125, case["pad"], ids)
  return ids if case["wide_ids"] else ids.int()


def prepare(case, seed):
  g = torch.Generator(device="cuda")
  g.manual_seed(int(seed))
  state = dict(case)
  if case["op"] == "clip":
    grads, flat = [], {}
    for i, size in enumerate(_sizes(case)):
      x = torch.empty(size, dtype=DTYPES[case["dtype"] if i % 2 == 0 else case["second"]], device="cuda").normal_(generator=g)
      grads.append(x.mul_(0.002 * (1 + i % 5)))
      flat[x.dtype] = flat.get(x.dtype, 0) + size
    # clipped gradients go to one flat buffer for each type, without gaps
    state.update(grads=grads, flat=[torch.empty(size, dtype=t, device="cuda") for t, size in flat.items()],
                 groups=[[x for x in grads if x.dtype is t] for t in flat])
    return state
  state["ids"] = _ids(case, g)
  t = DTYPES[case["dtype"]]
  if case["op"] == "lookup":
    state["table"] = torch.empty(case["vocab"], case["width"], dtype=t, device="cuda").normal_(generator=g)
    return state
  state["grad"] = torch.empty(case["n"], case["width"], dtype=t, device="cuda").normal_(generator=g)
  if case["op"] == "rows":   # the buffers that a training loop keeps: what lies behind the last row stays as it is
    state["out"] = (torch.zeros(case["n"], dtype=torch.int64, device="cuda"),
                    torch.zeros(case["n"], case["width"], dtype=t, device="cuda"),
                    torch.zeros(1, dtype=torch.int32, device="cuda"))
  return state


def run(state):
  return {"lookup": _lookup, "grad": _grad, "rows": _rows, "clip": _clip}[state["op"]](state)


def _lookup(s):
  if own:
    from orca_amd import ops
    return ops.embedding(s["table"], s["ids"], scale=s["scale"])
  return (s["table"][s["ids"]].float() * s["scale"]).to(s["table"].dtype)


def _grad(s):
  if own:
    from orca_amd import ops
    return ops.embedding_backward(s["grad"], s["ids"], s["vocab"], scale=s["scale"], padding_idx=s["pad"])
  g = s["grad"].float() * s["scale"]
  if s["pad"] >= 0:
    g = g * (s["ids"] != s["pad"]).unsqueeze(1)
  return torch.zeros(s["vocab"], s["width"], device=g.device).index_add_(0, s["ids"], g).to(s["grad"].dtype)


def _rows(s):
  if own:
    from orca_amd import ops
    r = ops.embedding_backward_rows(s["grad"], s["ids"], s["vocab"], scale=s["scale"], padding_idx=s["pad"], out=s["out"])
    return r.ids, r.rows, r.count
  n, vocab = s["n"], s["vocab"]
  key, order = torch.sort(torch.where(s["ids"] == s["pad"], vocab, s["ids"]).long(), stable=True)
  rank = torch.cumsum(torch.cat([key[:1] * 0, (key[1:] != key[:-1]).long()]), 0)
  count = torch.where(key < vocab, rank + 1, 0).amax().int().reshape(1)
  rank = torch.where(key < vocab, rank, n)                      # what is padded goes to a row behind the last
  ids = torch.zeros(n + 1, dtype=torch.int64, device=key.device).index_copy_(0, rank, key)
  rows = torch.zeros(n + 1, s["width"], device=key.device).index_add_(0, rank, s["grad"][order].float() * s["scale"])
  return ids[:n], rows[:n].to(s["grad"].dtype), count


def _clip(s):
  if own:
    from orca_amd import ops
    return ops.clip_grad_norm(s["grads"], s["max_norm"], flat=s["flat"]), s["flat"]
  flat = [torch.cat(x) for x in s["groups"]]
  norm = torch.stack([x.float().square().sum() for x in flat]).sum().sqrt()
  c = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
  return norm, [(x.float() * c).to(x.dtype) for x in flat]


def _distinct(case, n):
  """Expected number of distinct ids among n (densities as in _ids; collisions of the hash left aside)."""
  vocab = case["vocab"]
  if case["ids"] == "uniform":
    return max(1.0, -vocab * math.expm1(-n / vocab))
  edge = np.exp(np.linspace(0.0, math.log(vocab + 1.0), 4097))
  v = np.sqrt(edge[1:] * edge[:-1])
  return float(max(1.0, min(n, np.sum((edge[1:] - edge[:-1]) * -np.expm1(-n / (v * math.log(vocab + 1.0)))))))


def work(case):
  if case["op"] == "clip":
    sizes = _sizes(case)
    total = sum(s * BYTES[case["dtype"] if i % 2 == 0 else case["second"]] for i, s in enumerate(sizes))
    return {"bytes": 2 * total + 4, "flops": 3 * sum(sizes)}
  n, row = case["n"], case["width"] * BYTES[case["dtype"]]
  real = n if case["pad"] < 0 else n * 0.875
  distinct, ids = _distinct(case, real), n * (8 if case["wide_ids"] else 4)
  if case["op"] == "lookup":
    return {"bytes": ids + (distinct + n) * row, "flops": n * case["width"]}
  flops = (real + distinct) * case["width"]
  if case["op"] == "grad":
    return {"bytes": ids + real * row + case["vocab"] * row, "flops": flops}
  return {"bytes": ids + real * row + distinct * (row + 8) + 4, "flops": flops}


def exact(case, seed):
  """The definitions in 64 bits: sums over the occurrences of each id, taken by index_put_ in the ids' own order."""
  s = prepare(case, seed)
  if case["op"] == "clip":
    square = 0.0
    for x in s["grads"]:
      square += float((x.double() ** 2).sum())
    norm = math.sqrt(square)
    c = min(1.0, case["max_norm"] / (norm + 1e-6))
    return (torch.tensor(norm, dtype=torch.float64), [torch.cat([x.double() for x in grads]).mul_(c) for grads in s["groups"]])
  ids = s["ids"].long()
  if case["op"] == "lookup":
    return torch.index_select(s["table"], 0, ids).double().mul_(case["scale"])
  keep = (ids != case["pad"]).nonzero().reshape(-1)
  ids, grad = ids[keep], s["grad"][keep].double()
  if case["op"] == "grad":
    table = torch.zeros(case["vocab"], case["width"], dtype=torch.float64, device=ids.device)
    return table.index_put_((ids,), grad, accumulate=True).mul_(case["scale"])
  unique, inverse = torch.unique(ids, return_inverse=True)
  rows = torch.zeros(case["n"], case["width"], dtype=torch.float64, device=ids.device)
  rows.index_put_((inverse,), grad, accumulate=True).mul_(case["scale"])
  out = torch.zeros(case["n"], dtype=torch.int64, device=ids.device)
  out[:unique.numel()] = unique
  return out, rows, torch.tensor([unique.numel()], dtype=torch.int32)
