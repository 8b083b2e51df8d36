"""Timed cases of the microscaled 4-bit and expert operators.

Six operators, each in its plain form (elementary torch operations in 32 bits)
and, where `own` is true, through the framework's entry points:

  quantize          rows -> E2M1 values with one power-of-two scale per 32, and
                    back (mx.quantize, mx.dequantize)
  linear            y = act(Q(x) Q(W)^T + b), Q the quantisation above
                    (mx.linear)
  dispatch          (token, choice) pairs sorted by expert and the tokens' rows
                    in that order (experts.sort, experts.gather)
  experts           the product above with each sorted row's expert's weights
                    (experts.linear)
  combine           the rows back in token order, weighted and summed over a
                    token's choices (experts.combine)
  combine_backward  its gradients (experts.combine_backward)
"""

import importlib.util
import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}
BLOCK = 32


def _package():
  """The engine package (its folder's name has a hyphen)."""
  name = "xla_serving_b200"
  if name not in sys.modules:
    folder = os.path.join(os.path.dirname(os.path.dirname(
        os.path.abspath(__file__))), "xla-serving_b200")
    spec = importlib.util.spec_from_file_location(
        name, os.path.join(folder, "__init__.py"),
        submodule_search_locations=[folder])
    module = importlib.util.module_from_spec(spec)
    sys.modules[name] = module
    spec.loader.exec_module(module)
  return sys.modules[name]


# ---------------------------------------------------------------- the cases


def listed():
  return [
      # One decoding step's hidden rows before a 4-bit layer: latency.
      dict(name="quantize_step", op="quantize", rows=8, cols=4096,
           dtype="bf16"),
      # The interaction rows of a large ranking batch (479 wide: a block is
      # cut short and rows start off the 16-byte grid).
      dict(name="quantize_tower", op="quantize", rows=65536, cols=479,
           dtype="f32"),
      # A layer for a handful of tokens: the weights are all the traffic.
      dict(name="linear_step", op="linear", rows=4, cols=4096, out=4096,
           dtype="bf16", bias=False, relu=False),
      # The same kind of layer for a long prompt or a training batch.
      dict(name="linear_prompt", op="linear", rows=8192, cols=4096, out=8192,
           dtype="bf16", bias=True, relu=True),
      # A decoding step's tokens to 64 experts: latency.
      dict(name="dispatch_step", op="dispatch", tokens=64, topk=4, experts=64,
           cols=2048, dtype="bf16", padded=0.0),
      # A prompt's tokens, a twentieth of them padding, to 128 experts.
      dict(name="dispatch_prompt", op="dispatch", tokens=16384, topk=8,
           experts=128, cols=2048, dtype="bf16", padded=0.05),
      # Experts of a decoding step: a few rows each, all weights read.
      dict(name="experts_step", op="experts", tokens=64, topk=4, experts=64,
           cols=2048, out=1024, dtype="bf16", bias=False, relu=True,
           padded=0.0),
      # Experts of a prompt: uneven groups of hundreds of rows.
      dict(name="experts_prompt", op="experts", tokens=8192, topk=4,
           experts=64, cols=2048, out=2048, dtype="bf16", bias=False,
           relu=True, padded=0.05),
      # The way back for the two dispatch cases.
      dict(name="combine_step", op="combine", tokens=64, topk=4, experts=64,
           cols=2048, dtype="bf16", padded=0.0),
      dict(name="combine_prompt", op="combine", tokens=16384, topk=8,
           experts=128, cols=2048, dtype="bf16", padded=0.05),
      # Training: a small batch in 32 bits with an odd width, and a full one.
      dict(name="combine_backward_odd", op="combine_backward", tokens=1000,
           topk=2, experts=8, cols=479, dtype="f32", padded=0.02),
      dict(name="combine_backward_batch", op="combine_backward",
           tokens=16384, topk=8, experts=128, cols=2048, dtype="bf16",
           padded=0.05),
  ]


def _log_int(rng, low, high):
  return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
  op = rng.choice(["quantize", "linear", "dispatch", "experts", "combine",
                   "combine_backward"])
  dtype = rng.choice(["bf16", "f32"])
  if op == "quantize":
    cols = _log_int(rng, 32, 8192)
    rows = _log_int(rng, 1, min(65536, (1 << 25) // cols))
    return dict(op=op, rows=rows, cols=cols, dtype=dtype)
  if op == "linear":
    cols, out = _log_int(rng, 64, 8192), _log_int(rng, 64, 8192)
    rows = _log_int(rng, 1, min(8192, (1 << 38) // (cols * out)))
    return dict(op=op, rows=rows, cols=cols, out=out, dtype=dtype,
                bias=rng.random() < 0.5, relu=rng.random() < 0.5)
  experts = _log_int(rng, 4, 128)
  topk = rng.randint(1, min(8, experts))
  case = dict(op=op, topk=topk, experts=experts, dtype=dtype,
              padded=rng.choice([0.0, 0.02, 0.1]))
  if op == "experts":
    cols, out = _log_int(rng, 64, 2048), _log_int(rng, 64, 2048)
    tokens = _log_int(rng, 1, 32768 // topk)
    return dict(case, tokens=tokens, cols=cols, out=out,
                bias=rng.random() < 0.5, relu=rng.random() < 0.5)
  cols = _log_int(rng, 64, 4096)
  most = (1 << 27) // (topk * cols)
  return dict(case, tokens=_log_int(rng, 1, min(16384, most)), cols=cols)


# ------------------------------------------------------------------- inputs


def _activations(gen, rows, cols, dtype):
  """Rows of differing size with a few large columns, as hidden states have."""
  x = torch.randn((rows, cols), generator=gen, device="cuda")
  x *= torch.exp(0.5 * torch.randn((rows, 1), generator=gen, device="cuda"))
  x *= 1 + 9 * (torch.rand((cols,), generator=gen, device="cuda") < 0.01)
  return x.to(dtype)


def _choices(gen, case):
  """A token's distinct experts, popular ones more often; the last tokens of
  a padded batch choose none (-1)."""
  tokens, experts = case["tokens"], case["experts"]
  skew = 0.3 * torch.randn((experts,), generator=gen, device="cuda")
  score = skew + torch.randn((tokens, experts), generator=gen, device="cuda")
  top = torch.topk(score, case["topk"], dim=1)
  ids = top.indices.to(torch.int32)
  weights = torch.softmax(top.values, dim=1)
  real = tokens - int(tokens * case["padded"])
  ids[real:] = -1
  return ids, weights


def _sorted_pairs(ids, experts):
  """offsets [experts + 1], order [pairs] and slots like ids, as
  experts.sort gives them: kept pairs by expert, then by pair; -1 elsewhere."""
  flat = ids.reshape(-1).long()
  kept = (flat >= 0) & (flat < experts)
  key = torch.where(kept, flat, experts)
  by = torch.argsort(key, stable=True)
  counts = (key[:, None] == torch.arange(experts, device=ids.device)).sum(0)
  offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
  row = torch.arange(flat.numel(), device=ids.device)
  order = torch.where(row < offsets[-1], by, -1)
  slots = torch.empty_like(by).scatter_(0, by, row)
  slots = torch.where(kept, slots, -1).reshape(ids.shape)
  return offsets.int(), order.int(), slots.int()


def prepare(case, seed):
  gen = torch.Generator(device="cuda")
  gen.manual_seed(seed)
  op, dtype = case["op"], _DTYPES[case["dtype"]]
  s = dict(op=op)
  if op == "quantize":
    s["x"] = _activations(gen, case["rows"], case["cols"], dtype)
    return s
  if op in ("linear", "experts"):
    rows = case["rows"] if op == "linear" else case["tokens"]
    s["x"] = _activations(gen, rows, case["cols"], dtype)
    groups = case.get("experts", 1)
    shape = (groups, case["out"], case["cols"])
    w = torch.randn(shape, generator=gen, device="cuda")
    w *= case["cols"] ** -0.5
    s["bias"] = (torch.randn((groups, case["out"]), generator=gen,
                             device="cuda") if case["bias"] else None)
    if op == "linear":
      w, s["bias"] = w[0], s["bias"][0] if case["bias"] else None
    s["relu"] = case["relu"]
    if own:  # the weights in 4 bits, laid out once
      s["w"] = _package().mx.quantize(w)
    else:    # the same weights' values
      s["w"] = _fp4_values(w)
  if op == "linear":
    return s
  s["ids"], s["weights"] = _choices(gen, case)
  s["experts"] = case["experts"]
  if op == "dispatch":
    s["x"] = _activations(gen, case["tokens"], case["cols"], dtype)
    return s
  s["offsets"], s["order"], s["slots"] = _sorted_pairs(s["ids"],
                                                       case["experts"])
  s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
  if op in ("combine", "combine_backward"):
    pairs = case["tokens"] * case["topk"]
    s["y"] = _activations(gen, pairs, case["cols"], dtype)
    s["grad"] = _activations(gen, case["tokens"], case["cols"], dtype)
  if own:
    s["plan"] = _package().experts.ExpertPlan(s["offsets"], s["order"],
                                              s["slots"])
  return s


# --------------------------------------------------------------- plain forms


def _fp4_values(x):
  """The values x stands for after quantisation to E2M1 with one power of two
  per 32 along the last axis, in 32 bits: the scale is 2^(floor(log2 max|x|) -
  2), at least 2^-127; x / scale is rounded to the nearest of 0, .5, 1, 1.5,
  2, 3, 4, 6 (ties to the even code, larger ones to 6)."""
  cols = x.shape[-1]
  pad = -cols % BLOCK
  v = torch.nn.functional.pad(x.float(), (0, pad))
  v = v.reshape(*x.shape[:-1], -1, BLOCK)
  most = v.abs().amax(-1, keepdim=True)
  exponent = torch.frexp(most).exponent - 3
  exponent = torch.where(most > 0, exponent, -127).clamp(min=-127)
  up = ((127 - exponent).int() << 23).view(torch.float32)
  a = (v * up).abs().clamp(max=6.0)
  step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
  a = torch.round(a / step) * step
  down = ((exponent.clamp(min=-126) + 127).int() << 23).view(torch.float32)
  down = torch.where(exponent < -126, 0.5 * down, down)
  v = torch.copysign(a, v) * down
  return v.reshape(*x.shape[:-1], cols + pad)[..., :cols]


def _activated(y, bias, relu, dtype):
  if bias is not None:
    y = y + bias
  if relu:
    y = torch.relu(y)
  return y.to(dtype)


def _plain_linear(s):
  x = s["x"]
  return _activated(_fp4_values(x) @ s["w"].t(), s["bias"], s["relu"],
                    x.dtype)


def _plain_dispatch(s):
  x, ids = s["x"], s["ids"]
  offsets, order, slots = _sorted_pairs(ids, s["experts"])
  rows = x[order.clamp(min=0).long() // ids.shape[1]]
  rows = torch.where((order >= 0)[:, None], rows, torch.zeros_like(rows))
  return offsets, order, slots, rows


def _plain_experts(s):
  """Each expert's rows in a slab of their own, one batched product, and the
  rows back where they were; rows behind the last expert's are zero."""
  x, order, offsets = s["x"], s["order"].long(), s["offsets"].long()
  topk, experts = s["ids"].shape[1], s["experts"]
  row = torch.arange(order.numel(), device=x.device)
  expert = (row[:, None] >= offsets[None, 1:]).sum(1).clamp(max=experts - 1)
  kept = row < offsets[-1]
  at = torch.where(kept, expert * s["most"] + row - offsets[expert],
                   experts * s["most"])
  slab = x.new_zeros((experts * s["most"] + 1, x.shape[1]),
                     dtype=torch.float32)
  slab[at] = _fp4_values(x)[order.clamp(min=0) // topk]
  slab = slab[:-1].reshape(experts, s["most"], x.shape[1])
  y = torch.bmm(slab, s["w"].transpose(1, 2))
  bias = None if s["bias"] is None else s["bias"][:, None, :]
  y = _activated(y, bias, s["relu"], x.dtype).reshape(-1, s["w"].shape[1])
  y = y[at.clamp(max=y.shape[0] - 1)]
  return torch.where(kept[:, None], y, torch.zeros_like(y))


def _plain_combine(s):
  y, slots = s["y"], s["slots"]
  rows = y[slots.clamp(min=0).long()].float()
  w = torch.where(slots >= 0, s["weights"], 0.0)
  rows = torch.where((slots >= 0)[..., None], rows, 0.0)
  return (w[..., None] * rows).sum(1).to(y.dtype)


def _plain_combine_backward(s):
  y, order, slots = s["y"], s["order"], s["slots"]
  topk = slots.shape[1]
  grad = s["grad"].float()
  pair = order.clamp(min=0).long()
  gy = s["weights"].reshape(-1)[pair][:, None] * grad[pair // topk]
  gy = torch.where((order >= 0)[:, None], gy, 0.0).to(y.dtype)
  rows = y[slots.clamp(min=0).long()].float()
  gw = (rows * grad[:, None, :]).sum(2)
  return gy, torch.where(slots >= 0, gw, 0.0)


_PLAIN = {"linear": _plain_linear, "dispatch": _plain_dispatch,
          "experts": _plain_experts, "combine": _plain_combine,
          "combine_backward": _plain_combine_backward}


def _own_run(s):
  package = _package()
  mx, experts, op = package.mx, package.experts, s["op"]
  act = mx.ACT_RELU if s.get("relu") else mx.ACT_NONE
  if op == "quantize":
    return mx.dequantize(mx.quantize(s["x"]), dtype=s["x"].dtype)
  if op == "linear":
    return mx.linear(s["x"], s["w"], s["bias"], act)
  if op == "dispatch":
    plan = experts.sort(s["ids"], s["experts"])
    return (plan.offsets, plan.order, plan.slots,
            experts.gather(s["x"], plan))
  if op == "experts":
    return experts.linear(s["x"], s["plan"], s["w"], s["bias"], act)
  if op == "combine":
    return experts.combine(s["y"], s["plan"], s["weights"])
  return experts.combine_backward(s["grad"], s["y"], s["plan"], s["weights"])


def run(state):
  if own:
    return _own_run(state)
  if state["op"] == "quantize":
    return _fp4_values(state["x"]).to(state["x"].dtype)
  return _PLAIN[state["op"]](state)


# ------------------------------------------------------------ work and truth


def work(case):
  """Bytes: inputs once, outputs once (4-bit values with a scale byte per 32;
  the quantised rows themselves, written and read back, in "quantize"). Padding
  tokens' rows are not read. Flops: multiply and add of each product."""
  op, size = case["op"], _SIZE[case["dtype"]]
  packed = 0.5 + 1 / BLOCK
  if op == "quantize":
    n = case["rows"] * case["cols"]
    return {"bytes": n * (2 * size + 2 * packed), "flops": 0}
  if op == "linear":
    rows, cols, out = case["rows"], case["cols"], case["out"]
    return {"bytes": rows * cols * size + out * cols * packed +
                     rows * out * size + 4 * out * case["bias"],
            "flops": 2 * rows * cols * out}
  tokens, topk, experts = case["tokens"], case["topk"], case["experts"]
  real = tokens - int(tokens * case["padded"])
  pairs, cols = tokens * topk, case["cols"]
  plan = 4 * (2 * pairs + experts + 1)
  if op == "dispatch":
    return {"bytes": 4 * pairs + plan + (real + pairs) * cols * size,
            "flops": 0}
  if op == "experts":
    out = case["out"]
    used = min(experts, real * topk)
    return {"bytes": plan + real * cols * size + used * out * cols * packed +
                     pairs * out * size + 4 * experts * out * case["bias"],
            "flops": 2 * real * topk * cols * out}
  if op == "combine":
    return {"bytes": 8 * pairs + (real * topk + tokens) * cols * size,
            "flops": 2 * real * topk * cols}
  return {"bytes": 16 * pairs + (real * topk + pairs + real) * cols * size,
          "flops": 3 * real * topk * cols}


def _exact_fp4(x):
  """The quantised values in 64 bits, from the definition: a search over the
  eight magnitudes, the smaller or larger one at a tie by its code's parity."""
  cols = x.shape[-1]
  blocks = -(-cols // BLOCK)
  v = x.new_zeros((*x.shape[:-1], blocks * BLOCK), dtype=torch.float64)
  v[..., :cols] = x
  v = v.reshape(*x.shape[:-1], blocks, BLOCK)
  most = v.abs().amax(-1, keepdim=True)
  exponent = (most.view(torch.int64) >> 52) - 1023  # floor(log2), exactly
  scale = ((exponent.clamp(min=-125) - 2 + 1023) << 52).view(torch.float64)
  a = v.abs() / scale
  grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
  q = torch.zeros_like(a)
  for k in range(7):
    middle = (grid[k] + grid[k + 1]) / 2
    over = a > middle if k % 2 == 0 else a >= middle
    q += over * (grid[k + 1] - grid[k])
  v = torch.sign(v) * q * scale
  return v.reshape(*x.shape[:-1], blocks * BLOCK)[..., :cols]


def exact(case, seed):
  global own
  was, own = own, False
  s = prepare(case, seed)
  own = was
  op = case["op"]
  if op == "quantize":
    return _exact_fp4(s["x"])
  if op == "linear":
    y = _exact_fp4(s["x"]) @ s["w"].double().t()
    if s["bias"] is not None:
      y += s["bias"].double()
    return y.clamp(min=0) if s["relu"] else y
  ids, experts = s["ids"], case["experts"]
  tokens, topk = ids.shape
  flat = ids.reshape(-1).long()
  if op == "dispatch":
    by = torch.cat([(flat == e).nonzero()[:, 0] for e in range(experts)])
    rows = torch.zeros((tokens * topk, case["cols"]), dtype=torch.float64,
                       device="cuda")
    rows[:by.numel()] = s["x"].double()[by // topk]
    return None, None, None, rows
  by = [(flat == e).nonzero()[:, 0] for e in range(experts)]
  if op == "experts":
    x = _exact_fp4(s["x"])
    y = torch.zeros((tokens * topk, case["out"]), dtype=torch.float64,
                    device="cuda")
    at = 0
    for e in range(experts):
      rows = x[by[e] // topk] @ s["w"][e].double().t()
      if s["bias"] is not None:
        rows += s["bias"][e].double()
      y[at:at + by[e].numel()] = rows.clamp(min=0) if s["relu"] else rows
      at += by[e].numel()
    return y
  pair = torch.cat(by)
  weight = s["weights"].double().reshape(-1)
  if op == "combine":
    out = torch.zeros((tokens, case["cols"]), dtype=torch.float64,
                      device="cuda")
    for j in range(topk):
      at = (pair % topk == j).nonzero()[:, 0]
      out[pair[at] // topk] += (weight[pair[at], None] *
                                s["y"][at].double())
    return out
  grad = s["grad"].double()
  gy = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
  gw = torch.zeros((tokens * topk,), dtype=torch.float64, device="cuda")
  for e in range(experts):
    at = int(s["offsets"][e])
    mine = slice(at, at + by[e].numel())
    g = grad[by[e] // topk]
    gy[mine] = weight[by[e], None] * g
    gw[by[e]] = (g * s["y"][mine].double()).sum(1)
  return gy, gw.reshape(tokens, topk)
