"""Plain implementations of the expert operators in 64 bits on the CPU, one token, pair or expert after the other, and how
far a result that is computed in 32 bits and rounded once may lie from them."""
import numpy as np
import torch

STEP = 2.0 ** -24  # half a step of float32, relative to the value


def half_step(dtype):
  return torch.finfo(dtype).eps / 2


def topk(logits, k, normalize, mask=None):
  """(weights, chosen) of float64 logits (numpy)."""
  n, experts = logits.shape
  weights, chosen = np.zeros((n, k)), np.full((n, k), -1, np.int32)
  for t in range(n):
    if mask is not None and not mask[t]:
      continue
    row = logits[t]
    # NaN before every number, then falling, the lowest index first among equals; -inf never
    ranked = sorted((e for e in range(experts) if not row[e] == -np.inf), key=lambda e: (not np.isnan(row[e]), -row[e], e))
    taken = ranked[:k]
    if not taken:
      continue
    with np.errstate(invalid="ignore"):
      scaled = np.exp(row - row[taken[0]])
      total = scaled[taken].sum() if normalize else scaled.sum()
      weights[t, :len(taken)] = scaled[taken] / total
    chosen[t, :len(taken)] = taken
  return weights, chosen


def topk_gradient(logits, weights, chosen, ct, normalize):
  """By the definition of the softmax's derivative, from 64-bit weights."""
  grad = np.zeros_like(logits)
  for t in range(logits.shape[0]):
    taken = [i for i in range(chosen.shape[1]) if chosen[t, i] >= 0]
    if not taken:
      continue
    inner = sum(weights[t, i] * ct[t, i] for i in taken)
    if not normalize:
      p = np.exp(logits[t] - logits[t].max())
      grad[t] = -p / p.sum() * inner
    for i in taken:
      grad[t, chosen[t, i]] += weights[t, i] * (ct[t, i] - (inner if normalize else 0.0))
  return grad


def sort(experts, num_experts):
  flat = experts.reshape(-1).astype(np.int64)
  order, indptr = [], [0]
  for e in range(num_experts):
    order += [p for p in range(flat.shape[0]) if flat[p] == e] if flat.shape[0] < 5000 else np.nonzero(flat == e)[0].tolist()
    indptr.append(len(order))
  position = np.full(flat.shape[0], -1, np.int32)
  position[order] = np.arange(len(order))
  order = np.array(order + [-1] * (flat.shape[0] - len(order)), np.int32)
  return np.array(indptr, np.int32), order, position.reshape(experts.shape)


def matmul(rows, weight, indptr):
  out = torch.zeros(rows.shape[0], weight.shape[2], dtype=torch.float64)
  for e in range(weight.shape[0]):
    a, b = int(indptr[e]), int(indptr[e + 1])
    out[a:b] = rows[a:b].double() @ weight[e].double()
  return out


def matmul_gradients(rows, weight, indptr, ct):
  d_rows, d_weight = torch.zeros(rows.shape, dtype=torch.float64), torch.zeros(weight.shape, dtype=torch.float64)
  for e in range(weight.shape[0]):
    a, b = int(indptr[e]), int(indptr[e + 1])
    d_rows[a:b] = ct[a:b].double() @ weight[e].double().t()
    d_weight[e] = rows[a:b].double().t() @ ct[a:b].double()
  return d_rows, d_weight


def check_sums(got, want, magnitude, terms, what):
  """A sum of ``terms`` products in 32 bits, in any order: each addition off by at most a whole step (2^-23; half of one where
  the unit rounds to nearest) of a partial sum, none of which is above ``magnitude``, the sum of the absolute addends; an
  addend of float32 factors is rounded as well.  Then one rounding to the type of ``got`` (for results below the type's
  normal numbers: to its smallest step)."""
  got_, want = got.detach().cpu().double(), want.double()
  bound = (terms + 1) * 2 * STEP * magnitude.double()
  bound += half_step(got.dtype) * (want.abs() + bound) + torch.finfo(got.dtype).smallest_normal * half_step(got.dtype)
  off = (got_ - want).abs()
  assert torch.isfinite(got_).all(), what
  assert (off <= bound).all(), "%s: %g off, %g allowed" % (what, float((off - bound).max()), float(bound.max()))
