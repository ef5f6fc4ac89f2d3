"""Timed cases of the operators that route tokens to experts: the choice of the experts, the sort of the chosen pairs by
expert, the rows' way there and back, and the experts' products.

listed()             the cases, by name;  draw(rng): one more case of the same ranges
prepare(case, seed)  what a program holds before the call, on the GPU
run(state)           one pass: elementary torch operations in 32 bits, or, where ``own`` is set, the package's operators
exact(case, seed)    the same outputs from the definitions, in 64 bits
work(case)           bytes and operations that one pass cannot do without
"""
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}


def listed():
  return [
    # The router of a served model at a single token: nothing but latency.
    dict(name="topk_one_token", op="topk", dtype="bfloat16", tokens=1, experts=64, k=6, normalize=True, padding=0.0,
         backward=False),
    # The router of a training step over a padded batch: probabilities over all experts, a tenth of the tokens is
    # padding, gradient of the logits.
    dict(name="topk_training", op="topk", dtype="float32", tokens=32_771, experts=128, k=8, normalize=False, padding=0.1,
         backward=True),
    # The pairs of a small batch that decodes a token a sequence.
    dict(name="sort_decode", op="sort", tokens=37, experts=8, k=2, padding=0.0),
    # The pairs of long packed prompts over many experts, some tokens padding.
    dict(name="sort_prompts", op="sort", tokens=65_537, experts=256, k=8, padding=0.05),
    # Rows of a short prompt in an odd width, in 32 bits.
    dict(name="dispatch_odd", op="dispatch", dtype="float32", tokens=129, experts=16, k=3, width=1_023, padding=0.1,
         backward=False),
    # A training step's rows to their experts, and their gradients back.
    dict(name="dispatch_training", op="dispatch", dtype="bfloat16", tokens=16_385, experts=64, k=8, width=2_048,
         padding=0.05, backward=True),
    # The experts' answers of a decoding batch put together.
    dict(name="combine_decode", op="combine", dtype="float16", tokens=16, experts=64, k=8, width=4_096, padding=0.0,
         backward=False),
    # A training step: the weighted sum, the gradients of the rows and of the weights.
    dict(name="combine_training", op="combine", dtype="bfloat16", tokens=16_385, experts=64, k=8, width=2_048,
         padding=0.05, backward=True),
    # Four decoded tokens on eight experts each: the time is that of reading the experts met.
    dict(name="matmul_decode", op="matmul", dtype="bfloat16", tokens=4, experts=64, k=8, width=2_048, out=1_536,
         layout="nk", padding=0.0, backward=False),
    # A packed prompt over many narrow experts, uneven counts, weights stored input-major.
    dict(name="matmul_prompt", op="matmul", dtype="float16", tokens=4_099, experts=64, k=8, width=2_048, out=1_024,
         layout="kn", padding=0.02, backward=False),
    # A training step of few wide experts: product, gradients of rows and weights.
    dict(name="matmul_training", op="matmul", dtype="bfloat16", tokens=16_384, experts=8, k=2, width=2_048, out=4_096,
         layout="nk", padding=0.0, backward=True),
    # The same in 32 bits, in odd sizes, with padding.
    dict(name="matmul_training_odd", op="matmul", dtype="float32", tokens=1_001, experts=7, k=3, width=515, out=771,
         layout="kn", padding=0.1, backward=True),
  ]


_MOST_FLOPS = 6.0 * 16_384 * 2 * 2_048 * 4_096  # of the largest listed case
_MOST_VALUES = 16_385 * 8 * 2_048  # of rows, in the largest listed cases of the two ways


def _log(rng, low, high):
  return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)) )))))


def draw(rng):
  op = rng.choice(["topk", "sort", "dispatch", "combine", "matmul", "matmul"])
  padding = rng.choice([0.0, 0.03, 0.3])
  dtype = rng.choice(["float32", "float16", "bfloat16", "bfloat16"])
  experts = _log(rng, 2, 256)
  k = rng.randint(1, min(8, experts))
  backward = rng.random() < 0.5
  if op == "topk":
    return dict(op=op, dtype=dtype, tokens=_log(rng, 1, 32_771), experts=experts, k=k, normalize=rng.random() < 0.5,
                padding=padding, backward=backward)
  if op == "sort":
    return dict(op=op, tokens=_log(rng, 1, 65_537), experts=experts, k=k, padding=padding)
  if op in ("dispatch", "combine"):
    tokens, width = _log(rng, 1, 16_385), _log(rng, 64, 4_096)
    if rng.random() < 0.6:
      width = max(64, width // 64 * 64)
    values = _MOST_VALUES // (2 if dtype == "float32" else 1)
    tokens = max(1, min(tokens, values // (k * width)))
    return dict(op=op, dtype=dtype, tokens=tokens, experts=experts, k=k, width=width, padding=padding, backward=backward)
  width, out = _log(rng, 64, 4_096), _log(rng, 64, 4_096)
  if rng.random() < 0.7:
    width, out = max(64, width // 64 * 64), max(64, out // 64 * 64)
  experts = max(1, min(experts, 2 ** 28 // (width * out)))
  k = min(k, experts)
  flops = _MOST_FLOPS / (16 if dtype == "float32" else 2) / (6 if backward else 2)
  tokens = max(1, min(_log(rng, 1, 16_384), int(flops / (k * width * out)), 2 ** 28 // (k * max(width, out))))
  return dict(op="matmul", dtype=dtype, tokens=tokens, experts=experts, k=k, width=width, out=out,
              layout=rng.choice(["nk", "kn"]), padding=padding, backward=backward)


def _chosen(case, generator, device):
  """k different experts a token, some experts more wanted than others; -1 for the tokens that are padding."""
  tokens, experts, k = case["tokens"], case["experts"], case["k"]
  wanted = torch.randn(tokens, experts, generator=generator, device=device)
  wanted += 0.5 * torch.randn(experts, generator=generator, device=device)
  chosen = torch.topk(wanted, k, dim=1).indices.to(torch.int32)
  padded = torch.rand(tokens, generator=generator, device=device) < case["padding"]
  return torch.where(padded[:, None], torch.full_like(chosen, -1), chosen).contiguous()


def _arrays(chosen, experts):
  """indptr, order, position of the chosen pairs."""
  flat = chosen.reshape(-1).to(torch.int64)
  key = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
  order = torch.argsort(key, stable=True)
  counts = (key[:, None] == torch.arange(experts, device=flat.device)).sum(0)
  indptr = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
  place = torch.empty_like(order)
  place[order] = torch.arange(order.shape[0], device=flat.device)
  none = torch.full_like(order, -1)
  position = torch.where(key < experts, place, none)
  order = torch.where(key[order] < experts, order, none)
  return indptr.to(torch.int32), order.to(torch.int32), position.to(torch.int32).reshape(chosen.shape)


def prepare(case, seed):
  device = torch.device("cuda")
  generator = torch.Generator(device=device)
  generator.manual_seed(seed)
  state = dict(case)
  op, tokens, k = case["op"], case["tokens"], case["k"]
  if op == "topk":
    dtype = _DTYPES[case["dtype"]]
    # (logits of an unsharp router; in 16 bits many of a row are equal)
    logits = 1.5 * torch.randn(tokens, case["experts"], generator=generator, device=device)
    logits += torch.randn(case["experts"], generator=generator, device=device)
    state["logits"] = logits.to(dtype).requires_grad_(case["backward"])
    state["mask"] = None
    if case["padding"]:
      state["mask"] = torch.rand(tokens, generator=generator, device=device) >= case["padding"]
    state["ct"] = torch.randn(tokens, k, generator=generator, device=device)
    return state
  chosen = _chosen(case, generator, device)
  if op == "sort":
    state["chosen"] = chosen
    return state
  dtype = _DTYPES[case["dtype"]]
  state["indptr"], state["order"], state["position"] = _arrays(chosen, case["experts"])
  pairs = tokens * k

  def normal(*shape, scale=1.0):
    return (scale * torch.randn(*shape, generator=generator, device=device)).to(dtype)

  if op == "dispatch":
    state["tokens_"] = normal(tokens, case["width"]).requires_grad_(case["backward"])
    if case["backward"]:
      state["ct"] = normal(pairs, case["width"])
  elif op == "combine":
    state["rows"] = normal(pairs, case["width"]).requires_grad_(case["backward"])
    weights = torch.softmax(torch.randn(tokens, k, generator=generator, device=device), dim=1)
    state["weights"] = weights.requires_grad_(case["backward"])
    if case["backward"]:
      state["ct"] = normal(tokens, case["width"])
  else:
    width, out, experts = case["width"], case["out"], case["experts"]
    state["rows"] = normal(pairs, width).requires_grad_(case["backward"])
    shape = (experts, out, width) if case["layout"] == "nk" else (experts, width, out)
    state["stored"] = normal(*shape, scale=width ** -0.5).requires_grad_(case["backward"])
    if case["backward"]:
      state["ct"] = normal(pairs, out)
    # (the longest expert's rows: what a padded batched product is sized for)
    state["longest"] = int((state["indptr"][1:] - state["indptr"][:-1]).max())
  return state


def _own(s):
  import brainpylib_amd as bpl
  op = s["op"]
  if op == "topk":
    weights, experts = bpl.expert_topk(s["logits"], k=s["k"], normalize=s["normalize"], mask=s["mask"])
    if not s["backward"]:
      return weights, experts
    return (weights.detach(), experts) + torch.autograd.grad(weights, s["logits"], s["ct"])
  if op == "sort":
    return bpl.expert_sort(s["chosen"], num_experts=s["experts"])
  if op == "dispatch":
    inputs = (s["tokens_"],)
    out = bpl.expert_dispatch(s["tokens_"], s["order"], s["position"])
  elif op == "combine":
    inputs = (s["rows"], s["weights"])
    out = bpl.expert_combine(s["rows"], s["weights"], s["order"], s["position"])
  else:
    inputs = (s["rows"], s["stored"])
    weight = s["stored"].transpose(1, 2) if s["layout"] == "nk" else s["stored"]
    out = bpl.expert_matmul(s["rows"], weight, s["indptr"])
  if not s["backward"]:
    return (out,)
  return (out.detach(),) + torch.autograd.grad(out, inputs, s["ct"])


def _plain_topk(s):
  logits, k = s["logits"].detach(), s["k"]
  x = logits.float()
  ranked, experts = torch.sort(x, dim=1, descending=True, stable=True)
  e = torch.exp(x - ranked[:, :1])
  total = e.sum(1, keepdim=True)
  weights = torch.exp(ranked[:, :k] - ranked[:, :1])
  weights = weights / (weights.sum(1, keepdim=True) if s["normalize"] else total)
  experts = experts[:, :k]
  live = torch.ones_like(x[:, :1], dtype=torch.bool) if s["mask"] is None else s["mask"][:, None]
  out = torch.where(live, weights, 0.0), torch.where(live, experts, -1).to(torch.int32)
  if not s["backward"]:
    return out
  inner = (weights * s["ct"]).sum(1, keepdim=True)
  grad = torch.zeros_like(x) if s["normalize"] else -(e / total) * inner
  grad = grad.scatter_add(1, experts, weights * (s["ct"] - inner) if s["normalize"] else weights * s["ct"])
  return out + (torch.where(live, grad, 0.0).to(logits.dtype),)


def _plain_sort(s):
  return _arrays(s["chosen"], s["experts"])


def _rows_of(values, position):
  """values[position] in 32 bits, zero where position is -1: (tokens, k, width)."""
  picked = values.float()[position.clamp(min=0).to(torch.int64)]
  return torch.where((position >= 0)[..., None], picked, 0.0)


def _plain_dispatch(s):
  tokens, order, k = s["tokens_"].detach(), s["order"], s["k"]
  rows = tokens.float()[(order.clamp(min=0) // k).to(torch.int64)]
  rows = torch.where((order >= 0)[:, None], rows, 0.0).to(tokens.dtype)
  if not s["backward"]:
    return (rows,)
  return rows, _rows_of(s["ct"], s["position"]).sum(1).to(tokens.dtype)


def _plain_combine(s):
  rows, weights, order, k = s["rows"].detach(), s["weights"].detach(), s["order"], s["k"]
  picked = _rows_of(rows, s["position"])
  out = (picked * weights[..., None]).sum(1).to(rows.dtype)
  if not s["backward"]:
    return (out,)
  ct = s["ct"].float()
  at = order.clamp(min=0).to(torch.int64)
  d_rows = torch.where((order >= 0)[:, None], ct[at // k] * weights.reshape(-1)[at][:, None], 0.0).to(rows.dtype)
  return out, d_rows, (picked * ct[:, None]).sum(2)


def _plain_matmul(s):
  rows, stored, indptr, longest = s["rows"].detach(), s["stored"].detach(), s["indptr"].to(torch.int64), s["longest"]
  dtype, n = rows.dtype, rows.shape[0]
  if longest == 0:
    out = rows.new_zeros(n, s["out"])
    return (out, torch.zeros_like(rows), torch.zeros_like(stored)) if s["backward"] else (out,)
  # one batched product over the experts, each padded to the longest's rows
  at = indptr[:-1, None] + torch.arange(longest, device=rows.device)
  inside = at < indptr[1:, None]
  at = torch.where(inside, at, 0)

  def padded(values):
    return torch.where(inside[..., None], values.float()[at], 0.0)

  def unpadded(values):
    back = values.new_zeros(n, values.shape[2])
    back[at[inside]] = values[inside]
    return back.to(dtype)

  weight = stored.float()
  other = weight.transpose(1, 2).contiguous()
  by_k, by_n = (other, weight) if s["layout"] == "nk" else (weight, other)  # (experts, width, out), (experts, out, width)
  a = padded(rows)
  out = unpadded(torch.bmm(a, by_k))
  if not s["backward"]:
    return (out,)
  ct = padded(s["ct"])
  left, right = (ct, a) if s["layout"] == "nk" else (a, ct)
  return out, unpadded(torch.bmm(ct, by_n)), torch.bmm(left.transpose(1, 2).contiguous(), right).to(dtype)


def run(state):
  if own:
    return _own(state)
  return {"topk": _plain_topk, "sort": _plain_sort, "dispatch": _plain_dispatch, "combine": _plain_combine,
          "matmul": _plain_matmul}[state["op"]](state)


def exact(case, seed):
  s = prepare(case, seed)
  op, k = case["op"], case["k"]
  if op == "sort":
    return None  # (whole numbers)
  if op == "topk":
    x = s["logits"].detach().double()
    live = torch.ones_like(x[:, 0], dtype=torch.bool) if s["mask"] is None else s["mask"]
    left, experts = x.clone(), []
    for _ in range(k):  # the largest that is left, the first of equals
      is_most = left == left.max(1, keepdim=True).values
      first = torch.where(is_most, torch.arange(x.shape[1], device=x.device), x.shape[1]).min(1).values
      experts.append(first)
      left.scatter_(1, first[:, None], -math.inf)
    experts = torch.stack(experts, 1)
    taken = torch.zeros_like(x).scatter_(1, experts, 1.0)
    scaled = torch.exp(x - x.max(1, keepdim=True).values)
    p = scaled / (scaled * (taken if case["normalize"] else 1.0)).sum(1, keepdim=True)
    weights = p.gather(1, experts) * live[:, None]
    out = (weights, None)
    if case["backward"]:
      g = torch.zeros_like(x).scatter_(1, experts, s["ct"].double())
      p_from = p * taken if case["normalize"] else p
      out += ((p_from * (g - (p * g).sum(1, keepdim=True))) * live[:, None],)
    return out
  position = s["position"].to(torch.int64)
  if op == "matmul":
    rows, stored = s["rows"].detach().double(), s["stored"].detach()
    indptr = s["indptr"].tolist()
    out = rows.new_zeros(rows.shape[0], case["out"])
    d_rows = torch.zeros_like(rows)
    d_stored = torch.zeros(stored.shape, dtype=torch.float64, device=rows.device) if case["backward"] else None
    for e, (a, b) in enumerate(zip(indptr[:-1], indptr[1:])):
      w = stored[e].double() if case["layout"] == "kn" else stored[e].double().t()
      out[a:b] = rows[a:b] @ w
      if case["backward"]:
        ct = s["ct"][a:b].double()
        d_rows[a:b] = ct @ w.t()
        d_stored[e] = rows[a:b].t() @ ct if case["layout"] == "kn" else ct.t() @ rows[a:b]
    return (out, d_rows, d_stored) if case["backward"] else (out,)
  # the two ways, one of a token's k places after the other
  if op == "dispatch":
    tokens = s["tokens_"].detach().double()
    rows = tokens.new_zeros(tokens.shape[0] * k, case["width"])
    back = torch.zeros_like(tokens)
    for i in range(k):
      t = (position[:, i] >= 0).nonzero()[:, 0]
      rows[position[t, i]] = tokens[t]
      if case["backward"]:
        back[t] += s["ct"][position[t, i]].double()
    return (rows, back) if case["backward"] else (rows,)
  rows, weights = s["rows"].detach(), s["weights"].detach().double()
  out = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device=rows.device)
  d_rows = torch.zeros(rows.shape, dtype=torch.float64, device=rows.device) if case["backward"] else None
  d_weights = torch.zeros_like(weights)
  for i in range(k):
    t = (position[:, i] >= 0).nonzero()[:, 0]
    row = rows[position[t, i]].double()
    out[t] += weights[t, i][:, None] * row
    if case["backward"]:
      ct = s["ct"][t].double()
      d_rows[position[t, i]] = weights[t, i][:, None] * ct
      d_weights[t, i] = (ct * row).sum(1)
  return (out, d_rows, d_weights) if case["backward"] else (out,)


def work(case):
  op, tokens, k, experts = case["op"], case["tokens"], case["k"], case["experts"]
  pairs = tokens * k
  if op == "sort":
    return {"bytes": 12.0 * pairs + 4.0 * (experts + 1), "flops": 0.0}
  size = _BYTES[case["dtype"]]
  if op == "topk":
    logits = float(tokens * experts * size)
    mask = tokens if case["padding"] else 0
    moved = logits + mask + 8.0 * pairs
    if case["backward"]:
      moved += logits + 4.0 * pairs
    return {"bytes": moved, "flops": 4.0 * tokens * experts * (2 if case["backward"] else 1)}
  width = case["width"]
  index = 8.0 * pairs
  if op == "dispatch":
    one_way = float(tokens * width * size + pairs * width * size)
    return {"bytes": index + one_way * (2 if case["backward"] else 1),
            "flops": float(pairs * width) if case["backward"] else 0.0}
  if op == "combine":
    values = float(tokens * width * size + pairs * width * size) + 4.0 * pairs
    if case["backward"]:
      values += float(tokens * width * size + pairs * width * size) + 4.0 * pairs
    return {"bytes": index + values, "flops": 2.0 * pairs * width * (2.5 if case["backward"] else 1)}
  out = case["out"]
  met = experts * (1.0 - (1.0 - 1.0 / experts) ** pairs) if experts > 1 else 1.0
  moved = pairs * (width + out) + met * width * out
  if case["backward"]:
    moved += pairs * (width + out) + experts * width * out
  return {"bytes": float(moved * size), "flops": 2.0 * pairs * width * out * (3 if case["backward"] else 1)}
