"""The expert operators on the GPU against plain implementations in 64 bits."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import brainpylib_amd as bpl
import experts_plain as plain
from experts_plain import STEP, check_sums, half_step

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def normal(seed, *shape, dtype=torch.float32, scale=1.0):
  g = torch.Generator().manual_seed(seed)
  return (scale * torch.randn(*shape, generator=g)).to(dtype)


def choices(seed, tokens, k, experts, dropped=0.1, skew=1.0):
  """Different experts a token, uneven; some tokens and some single pairs without one."""
  rng = np.random.default_rng(seed)
  want = rng.standard_normal((tokens, experts)) + skew * rng.standard_normal(experts)
  chosen = np.argsort(-want, axis=1)[:, :k].astype(np.int32)
  chosen[rng.random(tokens) < dropped] = -1
  chosen[rng.random((tokens, k)) < dropped / 2] = experts + 3
  return chosen


def arrays(seed, tokens, k, experts, dropped=0.1):
  indptr, order, position = plain.sort(choices(seed, tokens, k, experts, dropped), experts)
  return [torch.from_numpy(a) for a in (indptr, order, position)]


def counts(seed, rows, experts, empty=0.2):
  """indptr of uneven experts, some of them without rows, and rows behind the last."""
  rng = np.random.default_rng(seed)
  share = rng.exponential(size=experts) * (rng.random(experts) >= empty)
  behind = rng.integers(0, rows // 8 + 1)
  each = np.floor(share / max(share.sum(), 1e-9) * (rows - behind)).astype(np.int64)
  return torch.from_numpy(np.concatenate([[0], np.cumsum(each)]).astype(np.int32))


# ---- expert_topk ------------------------------------------------------------------------------------------------------
def check_topk(logits, k, normalize, mask=None, ct=None):
  x = logits.double().numpy()
  want_w, want_e = plain.topk(x, k, normalize, None if mask is None else mask.numpy())
  given = logits.cuda().requires_grad_(ct is not None)
  w, e = bpl.expert_topk(given, k=k, normalize=normalize, mask=None if mask is None else mask.cuda())
  assert w.dtype == torch.float32 and e.dtype == torch.int32 and not e.requires_grad
  assert np.array_equal(e.cpu().numpy(), want_e)
  got = w.detach().double().cpu().numpy()
  assert np.array_equal(np.isnan(got), np.isnan(want_w))
  # exp: its argument is off by half a step of it, which is at most the spread of the row, its value by two steps; the sum
  # by half a step an addend, the quotient by two and a half steps; the smallest numbers by a step of theirs
  finite = np.isfinite(x)
  spread = np.where(finite, x, 0).max() - np.where(finite, x, 0).min()
  rel = (min(spread, 104.0) * 2 + x.shape[1] + 12) * STEP
  fine = ~np.isnan(want_w)
  assert (np.abs(got - want_w)[fine] <= rel * want_w[fine] + 2.0 ** -125).all()
  if ct is None:
    return
  want = plain.topk_gradient(x, want_w, want_e, ct.double().numpy(), normalize)
  (grad,) = torch.autograd.grad(w, given, ct.cuda())
  assert grad.dtype == logits.dtype and grad.shape == logits.shape
  # each of the factors by rel, their differences and sums of k products by half a step each; then the type's rounding
  size = np.abs(want_w * np.where(want_e >= 0, ct.double().numpy(), 0)).sum(1, keepdims=True)
  bound = (rel * 3 + (k + 4) * STEP) * 2 * size
  off = np.abs(grad.double().cpu().numpy() - want)
  tiny = torch.finfo(logits.dtype).smallest_normal * half_step(logits.dtype)
  assert (off <= bound + half_step(logits.dtype) * (np.abs(want) + bound) + tiny).all(), (off - bound).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens, experts, k", [
  (1, 1, 1), (1, 64, 6), (5, 8, 2), (3, 8, 8), (33, 65, 9), (7, 60, 9), (130, 128, 8), (31, 127, 17), (64, 256, 8), (9, 257, 33),
  (40, 512, 4), (6, 513, 64), (3, 1000, 16), (17, 1024, 64), (2, 100, 64)])
def test_topk(cuda, dtype, tokens, experts, k):
  logits = normal(tokens + experts, tokens, experts, dtype=dtype, scale=2.0)
  logits[:, experts // 2] = logits[:, 0]  # equal ones, beyond those that 16 bits make
  ct = normal(7, tokens, k)
  for normalize in (True, False):
    check_topk(logits, k, normalize, ct=ct)
  mask = torch.rand(tokens, generator=torch.Generator().manual_seed(3)) < 0.6
  ct[~mask] = float("nan")  # (a row of padding has no gradient, whatever the cotangent holds)
  for normalize in (True, False):
    check_topk(logits, k, normalize, mask=mask, ct=ct)


@pytest.mark.parametrize("dtype", DTYPES)
def test_topk_of_masked_infinite_and_lowest_logits(cuda, dtype):
  low = torch.finfo(dtype).min
  inf, nan = float("inf"), float("nan")
  rows = torch.tensor([
    [-inf] * 8,                                  # nothing left
    [-inf, 1.0, -inf, -inf, 0.5, -inf, -inf, -inf],  # fewer than k
    [low] * 8,                                   # the lowest value everywhere: even weights
    [low, low, 3.0, low, low, low, low, low],
    [0.0, -0.0, 0.0, -0.0, -1.0, -2.0, -3.0, -4.0],  # the two zeros are equal
    [-inf, low, -inf, -inf, -inf, -inf, -inf, -inf],
  ]).to(dtype)
  ct = normal(1, 6, 4)
  for normalize in (True, False):
    check_topk(rows, 4, normalize, ct=ct)
  check_topk(torch.tensor([[1.0, nan, 2.0, nan, 3.0], [nan] * 5]).to(dtype), 3, True)
  w, e = bpl.expert_topk(torch.tensor([[1.0, inf, 2.0, inf]], dtype=dtype).cuda(), k=3)
  assert e.tolist() == [[1, 3, 2]] and torch.isnan(w).all()  # (inf - inf)


def test_topk_gradient_against_differences(cuda):
  # Differences of step h in 32 bits: weights are off by r = (2 * 12 + 7 + 12) 2^-24 each (as in check_topk), so a
  # difference by 2 r sum|ct| / (2 h), and by the cubic term, h^2 / 6 times the third derivative, which is below 2 sum|ct|.
  x, ct, h = normal(5, 4, 7), normal(6, 4, 3), 2.0 ** -7
  bound = ((2 * 12 + 7 + 12) * STEP / h + h * h / 3) * ct.abs().sum(1, keepdim=True).double()
  for normalize in (True, False):
    given = x.cuda().requires_grad_()
    w, e = bpl.expert_topk(given, k=3, normalize=normalize)
    (grad,) = torch.autograd.grad(w, given, ct.cuda())
    for j in range(7):
      step = torch.zeros_like(x)
      step[:, j] = h
      up, e_up = bpl.expert_topk((x + step).cuda(), k=3, normalize=normalize)
      down, e_down = bpl.expert_topk((x - step).cuda(), k=3, normalize=normalize)
      same = ((e_up == e) & (e_down == e)).all(1).cpu()
      slope = ((up.double() - down.double()).cpu() * ct).sum(1) / (2 * h)
      off = (slope - grad[:, j].double().cpu()).abs()[:, None]
      assert same.any() and (off <= bound)[same].all()


# ---- expert_sort ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens, k, experts", [
  (0, 2, 5), (1, 1, 1), (1, 8, 64), (37, 2, 8), (63, 1, 3), (64, 1, 3), (65, 1, 1024), (511, 8, 7), (512, 8, 255), (4097, 1, 256),
  (4099, 3, 511), (30_001, 8, 64), (9_000, 7, 1023), (170_000, 8, 33)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.uint32])
def test_sort(cuda, tokens, k, experts, dtype):
  chosen = choices(tokens, tokens, min(k, experts), experts) if tokens < 50_000 else \
    np.random.default_rng(1).integers(-2, experts + 2, (tokens, k)).astype(np.int32)
  given = torch.from_numpy(chosen).cuda()
  got = bpl.expert_sort(given.view(dtype), num_experts=experts)
  for a, b in zip(got, plain.sort(chosen, experts)):
    assert a.dtype == torch.int32 and np.array_equal(a.cpu().numpy(), b)
  flat = bpl.expert_sort(given.reshape(-1), num_experts=experts)
  assert torch.equal(flat[2], got[2].reshape(-1)) and torch.equal(flat[1], got[1])


def test_sort_of_one_expert_of_none_and_of_strided_pairs(cuda):
  for value in (0, 5, -1):
    chosen = np.full((3000, 4), value, np.int32)
    for a, b in zip(bpl.expert_sort(torch.from_numpy(chosen).cuda(), num_experts=6), plain.sort(chosen, 6)):
      assert np.array_equal(a.cpu().numpy(), b)
  chosen = choices(4, 500, 6, 20)
  given = torch.from_numpy(np.ascontiguousarray(chosen.T)).cuda().t()
  for a, b in zip(bpl.expert_sort(given, num_experts=20), plain.sort(chosen, 20)):
    assert np.array_equal(a.cpu().numpy(), b)


# ---- expert_dispatch, expert_combine ----------------------------------------------------------------------------------
WAYS = [(1, 1, 1, 1), (1, 8, 16, 4096), (5, 2, 4, 7), (33, 3, 5, 1023), (64, 8, 16, 512), (9, 64, 70, 130), (17, 9, 12, 2049),
        (700, 4, 9, 264), (3, 2, 3, 9001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens, k, experts, width", WAYS)
def test_dispatch(cuda, dtype, tokens, k, experts, width):
  _, order, position = arrays(width, tokens, k, experts)
  x = normal(1, tokens, width, dtype=dtype)
  given = x.cuda().requires_grad_()
  rows = bpl.expert_dispatch(given, order.cuda(), position.cuda())
  live = order >= 0
  want = torch.where(live[:, None], x[order.clamp(min=0).long() // k], torch.zeros((), dtype=dtype))
  assert rows.dtype == dtype and torch.equal(rows.detach().cpu(), want)
  ct = normal(2, tokens * k, width, dtype=dtype)
  ct[~live] = float("nan")  # (rows that no pair leads to)
  (grad,) = torch.autograd.grad(rows, given, ct.cuda())
  picked = torch.where((position >= 0)[..., None], ct.double()[position.clamp(min=0).long()], 0.0)
  check_sums(grad, picked.sum(1), picked.abs().sum(1), k, "d_tokens")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens, k, experts, width", WAYS)
def test_combine(cuda, dtype, tokens, k, experts, width):
  _, order, position = arrays(width + 1, tokens, k, experts)
  rows, weights = normal(1, tokens * k, width, dtype=dtype), normal(2, tokens, k).abs()
  rows[order < 0] = float("nan")
  weights[position < 0] = float("inf")  # (what belongs to no pair is not looked at)
  given, by = rows.cuda().requires_grad_(), weights.cuda().requires_grad_()
  out = bpl.expert_combine(given, by, order.cuda(), position.cuda())
  live = position >= 0
  picked = torch.where(live[..., None], rows.double()[position.clamp(min=0).long()], 0.0)
  w = torch.where(live, weights.double(), 0.0)
  assert out.dtype == dtype
  check_sums(out, (picked * w[..., None]).sum(1), (picked * w[..., None]).abs().sum(1), k, "out")
  ct = normal(3, tokens, width, dtype=dtype)
  d_rows, d_weights = torch.autograd.grad(out, (given, by), ct.cuda())
  at = order.clamp(min=0).long()
  want = torch.where((order >= 0)[:, None], ct.double()[at // k] * weights.double().reshape(-1)[at][:, None], 0.0)
  check_sums(d_rows, want, want.abs(), 1, "d_rows")
  products = picked * ct.double()[:, None]
  assert d_weights.dtype == torch.float32
  check_sums(d_weights, products.sum(2), products.abs().sum(2), width, "d_weights")
  assert (d_weights.cpu()[~live] == 0).all()
  # one gradient at a time is the same
  for i, leaf in enumerate((given, by)):
    again = bpl.expert_combine(given if i == 0 else given.detach(), by if i == 1 else by.detach(), order.cuda(), position.cuda())
    (alone,) = torch.autograd.grad(again, leaf, ct.cuda())
    assert torch.equal(alone, (d_rows, d_weights)[i])


def test_index_arrays_that_do_not_answer_each_other(cuda):
  # out of range, the same row twice, a row that says another pair: such pairs and rows count as none, there and back
  position = torch.tensor([[0, 1], [1, 7], [-5, 3], [2 ** 30, 2]], dtype=torch.int32)
  order = torch.tensor([0, 2, 100, 5, -9, 1, 3, 6], dtype=torch.int32)
  flat = position.reshape(-1).long()
  pairs = [p for p in range(8) if 0 <= flat[p] < 8 and order[flat[p]] == p]  # 0 -> 0, 2 -> 1, 5 -> 3
  assert pairs == [0, 2, 5]
  x, rows, weights = normal(1, 4, 40), normal(2, 8, 40), normal(3, 4, 2)
  want_rows, want_out, want_d = torch.zeros(8, 40), torch.zeros(4, 40), torch.zeros(8, 40)
  want_dw = torch.zeros(4, 2)
  for p in pairs:
    want_rows[flat[p]] = x[p // 2]
    want_out[p // 2] += weights.reshape(-1)[p] * rows[flat[p]]
    want_d[flat[p]] = weights.reshape(-1)[p] * x[p // 2]
    want_dw.reshape(-1)[p] = (x[p // 2].double() * rows[flat[p]].double()).sum()
  o, q = order.cuda(), position.cuda()
  assert torch.equal(bpl.expert_dispatch(x.cuda(), o, q).cpu(), want_rows)
  given, by = rows.cuda().requires_grad_(), weights.cuda().requires_grad_()
  out = bpl.expert_combine(given, by, o, q)
  assert torch.equal(out.detach().cpu(), want_out)
  d_rows, d_weights = torch.autograd.grad(out, (given, by), x.cuda())
  assert torch.equal(d_rows.cpu(), want_d)
  check_sums(d_weights, want_dw.double(), torch.full((4, 2), 100.0), 40, "d_weights")


def test_rows_of_more_elements_than_32_bits_number(cuda):
  tokens, k, width = 35_000, 2, 65_600  # 4.6e9 elements of rows
  order = torch.arange(tokens * k, dtype=torch.int32).flip(0).cuda()
  position = order.reshape(tokens, k)  # (its own inverse)
  x = (torch.arange(tokens, device="cuda") % 251).to(torch.bfloat16)[:, None].expand(tokens, width).contiguous()
  rows = bpl.expert_dispatch(x, order, position)
  for r in (0, 1, 32_739, 32_740, 65_471, 65_472, tokens * k - 1):
    t = (tokens * k - 1 - r) // k
    assert (rows[r].float() == t % 251).all(), r
  out = bpl.expert_combine(rows, torch.full((tokens, k), 0.5, device="cuda"), order, position)
  assert torch.equal(out, x)


# ---- expert_matmul ----------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1, 1), (1, 4, 8, 8), (8, 8, 64, 32), (32, 5, 130, 70), (100, 3, 17, 65), (257, 4, 200, 129), (300, 2, 515, 257),
          (900, 7, 96, 384), (1500, 40, 264, 136), (2048, 2, 256, 512), (64, 1024, 40, 48), (700, 3, 1, 33), (700, 3, 33, 1),
          (1100, 1, 1030, 300), (2, 8, 4096, 264), (3, 5, 4100, 70), (40, 2, 6001, 33)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out_major", [False, True])
@pytest.mark.parametrize("n, experts, inner, out", SHAPES)
def test_matmul(cuda, dtype, out_major, n, experts, inner, out):
  indptr = counts(n + inner, n, experts)
  rows, ct = normal(1, n, inner, dtype=dtype), normal(2, n, out, dtype=dtype)
  weight = normal(3, experts, inner, out, dtype=dtype)
  behind = int(indptr[-1])
  rows[behind:], ct[behind:] = float("nan"), float("inf")  # (rows of no expert are not looked at)
  given = rows.cuda().requires_grad_()
  stored = (weight.transpose(1, 2).contiguous() if out_major else weight).cuda().requires_grad_()
  view = stored.transpose(1, 2) if out_major else stored
  got = bpl.expert_matmul(given, view, indptr.cuda())
  assert got.dtype == dtype and got.shape == (n, out)
  check_sums(got, plain.matmul(rows, weight, indptr), plain.matmul(rows.abs(), weight.abs(), indptr), inner, "out")
  assert (got[behind:] == 0).all()
  d_rows, d_stored = torch.autograd.grad(got, (given, stored), ct.cuda())
  want = plain.matmul_gradients(rows, weight, indptr, ct)
  size = plain.matmul_gradients(rows.abs(), weight.abs(), indptr, ct.abs())
  check_sums(d_rows, want[0], size[0], out, "d_rows")
  assert (d_rows[behind:] == 0).all() and d_stored.is_contiguous()
  d_weight = d_stored.transpose(1, 2) if out_major else d_stored
  check_sums(d_weight, want[1], size[1], int((indptr[1:] - indptr[:-1]).max()) + 1, "d_weight")


@pytest.mark.parametrize("dtype, out_major, n, experts, inner, out", [
  (torch.bfloat16, True, 20_000, 4, 520, 1024), (torch.float16, False, 20_100, 5, 512, 1000), (torch.bfloat16, False, 18_000, 3, 517, 1031),
  (torch.float32, True, 9000, 3, 130, 520), (torch.bfloat16, True, 9000, 30, 96, 520)])
def test_matmul_of_many_tiles(cuda, dtype, out_major, n, experts, inner, out):
  # more tiles than the card holds: the largest ones and what is left over of them, and the middle ones
  indptr = counts(n, n, experts)
  rows, ct, weight = normal(1, n, inner, dtype=dtype), normal(2, n, out, dtype=dtype), normal(3, experts, inner, out, dtype=dtype)
  behind = int(indptr[-1])
  rows[behind:], ct[behind:] = float("nan"), float("nan")
  given = rows.cuda().requires_grad_()
  stored = (weight.transpose(1, 2).contiguous() if out_major else weight).cuda().requires_grad_()
  got = bpl.expert_matmul(given, stored.transpose(1, 2) if out_major else stored, indptr.cuda())
  check_sums(got, plain.matmul(rows, weight, indptr), plain.matmul(rows.abs(), weight.abs(), indptr), inner, "out")
  assert (got[behind:] == 0).all()
  d_rows, d_stored = torch.autograd.grad(got, (given, stored), ct.cuda())
  want, size = plain.matmul_gradients(rows, weight, indptr, ct), plain.matmul_gradients(rows.abs(), weight.abs(), indptr, ct.abs())
  check_sums(d_rows, want[0], size[0], out, "d_rows")
  d_weight = d_stored.transpose(1, 2) if out_major else d_stored
  check_sums(d_weight, want[1], size[1], int((indptr[1:] - indptr[:-1]).max()) + 1, "d_weight")


@pytest.mark.parametrize("dtype, out_major, inner, out", [
  (torch.bfloat16, True, 4160, 1024), (torch.float16, False, 4160, 1024), (torch.bfloat16, False, 4100, 1000), (torch.float16, True, 4163, 1001)])
def test_matmul_of_many_large_tiles(cuda, dtype, out_major, inner, out):
  # a long inner dimension: the largest tiles, those left over in quarters, in whole pieces and not; one expert has no rows.
  # Whole numbers: every sum is exact in 32 bits in any order (below 2 * 7,800 < 2^24), one rounding is left, and it is to nearest
  # on both sides.
  indptr = torch.tensor([0, 5200, 5200, 13_000, 19_900], dtype=torch.int32)
  n, experts = 20_000, 4
  g = torch.Generator().manual_seed(inner)
  rows = torch.randint(-2, 3, (n, inner), generator=g).to(dtype).cuda()
  ct = torch.randint(-1, 2, (n, out), generator=g).to(dtype).cuda()
  weight = torch.randint(-1, 2, (experts, inner, out), generator=g).to(dtype).cuda()
  rows[19_900:], ct[19_900:] = float("nan"), float("nan")
  given = rows.clone().requires_grad_()
  stored = (weight.transpose(1, 2).contiguous() if out_major else weight).clone().requires_grad_()
  got = bpl.expert_matmul(given, stored.transpose(1, 2) if out_major else stored, indptr.cuda())
  d_rows, d_stored = torch.autograd.grad(got, (given, stored), ct)
  d_weight = d_stored.transpose(1, 2) if out_major else d_stored
  for e in range(experts):
    at = slice(int(indptr[e]), int(indptr[e + 1]))
    x, c, w = rows[at].float(), ct[at].float(), weight[e].float()
    assert torch.equal(got[at], (x @ w).to(dtype)), e
    assert torch.equal(d_rows[at], (c @ w.t().contiguous()).to(dtype)), e
    assert torch.equal(d_weight[e], (x.t().contiguous() @ c).to(dtype)), e
  assert (got[19_900:] == 0).all() and (d_rows[19_900:] == 0).all()


def test_results_that_are_stored_past_the_caches(cuda):
  # more than 64 MB in whole lines: products, rows to the experts and the gradients
  indptr = torch.tensor([0, 20_000, 20_000, 33_000], dtype=torch.int32)
  g = torch.Generator().manual_seed(0)
  rows = torch.randint(-2, 3, (34_000, 64), generator=g).to(torch.bfloat16)
  weight = torch.randint(-1, 2, (3, 64, 1024), generator=g).to(torch.bfloat16)
  got = bpl.expert_matmul(rows.cuda(), weight.cuda(), indptr.cuda())
  want = torch.cat([rows[:20_000].float().cuda() @ weight[0].float().cuda(), rows[20_000:33_000].float().cuda() @ weight[2].float().cuda(),
                    torch.zeros(1000, 1024, device="cuda")])
  assert torch.equal(got.float(), want)  # (whole numbers below 256)
  chosen = torch.from_numpy(choices(5, 4099, 8, 16)).cuda()
  _, order, position = bpl.expert_sort(chosen, num_experts=16)
  x = normal(1, 4099, 1088, dtype=torch.bfloat16).cuda()
  sent = bpl.expert_dispatch(x, order, position)
  live = order >= 0
  assert torch.equal(sent, torch.where(live[:, None], x[order.clamp(min=0).long() // 8], 0.0))
  by = normal(2, 4099, 8).cuda()
  given = sent.clone().requires_grad_()
  (d_rows,) = torch.autograd.grad(bpl.expert_combine(given, by, order, position), given, x)
  at = order.clamp(min=0).long()
  exact = torch.where(live[:, None], by.double().reshape(-1)[at][:, None] * x.double()[at // 8], 0.0)
  check_sums(d_rows, exact.cpu(), exact.abs().cpu(), 1, "d_rows")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, experts, inner, out", [(5000, 1, 64, 72), (9000, 3, 33, 50), (20_000, 2, 130, 64), (6000, 5, 8, 300)])
def test_matmul_gradient_of_few_results_over_many_rows(cuda, dtype, n, experts, inner, out):
  # an expert's rows are split into parts, and those added: the experts' numbers of rows are uneven, one has none
  indptr = counts(n + out, n, experts, empty=0.0)
  if experts > 2:
    indptr[2] = indptr[1]
  rows, ct = normal(1, n, inner, dtype=dtype), normal(2, n, out, dtype=dtype)
  behind = int(indptr[-1])
  rows[behind:], ct[behind:] = float("nan"), float("inf")
  weight = torch.zeros(experts, inner, out, dtype=dtype)
  want = plain.matmul_gradients(rows, weight, indptr, ct)[1]
  size = plain.matmul_gradients(rows.abs(), weight, indptr, ct.abs())[1]
  for out_major in (False, True):
    stored = (weight.transpose(1, 2).contiguous() if out_major else weight).cuda().requires_grad_()
    got = bpl.expert_matmul(rows.cuda(), stored.transpose(1, 2) if out_major else stored, indptr.cuda())
    (d_stored,) = torch.autograd.grad(got, stored, ct.cuda())
    check_sums(d_stored.transpose(1, 2) if out_major else d_stored, want, size, int((indptr[1:] - indptr[:-1]).max()) + 1, "d_weight")


@pytest.mark.parametrize("dtype", DTYPES)
def test_matmul_one_at_the_edges_of_the_tiles(cuda, dtype):
  # whole numbers, small enough that every product and sum is exact: equal, element for element
  for n in (15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257):
    for inner, out in ((31, 127), (32, 128), (33, 129), (64, 256), (65, 257), (128, 130), (200, 64)):
      g = torch.Generator().manual_seed(n)
      rows = torch.randint(-2, 3, (n + 40, inner), generator=g).to(dtype)
      weight = torch.randint(-1, 2, (3, inner, out), generator=g).to(dtype)
      indptr = torch.tensor([0, 5, 5, 5 + n], dtype=torch.int32)
      want = plain.matmul(rows, weight, indptr)
      assert want.abs().max() < 256  # (exact in bfloat16 too)
      for w in (weight.cuda(), weight.transpose(1, 2).contiguous().cuda().transpose(1, 2)):
        got = bpl.expert_matmul(rows.cuda(), w, indptr.cuda())
        assert torch.equal(got.double().cpu(), want), (n, inner, out)


@pytest.mark.parametrize("dtype", DTYPES)
def test_matmul_of_the_smallest_and_largest_numbers(cuda, dtype):
  # numbers below the type's normal ones count, and results beyond its largest are infinite
  info = torch.finfo(dtype)
  tiny = info.smallest_normal * info.eps if dtype != torch.float32 else info.smallest_normal / 4
  rows = torch.zeros(40, 64, dtype=dtype)
  rows[:, 0], rows[:, 1], rows[:, 2] = 3 * tiny, info.max, info.max
  weight = torch.zeros(1, 64, 72, dtype=dtype)
  weight[0, 0, :8] = 1.0 if dtype != torch.float16 else 1024.0
  weight[0, 1, 8:16], weight[0, 1, 16:24], weight[0, 2, 16:24] = 1.0, 1.0, 1.0
  weight[0, 1, 24:32], weight[0, 2, 24:32] = 1.0, -1.0
  indptr = torch.tensor([0, 40], dtype=torch.int32)
  want = plain.matmul(rows, weight, indptr)
  for w in (weight.cuda(), weight.transpose(1, 2).contiguous().cuda().transpose(1, 2)):
    got = bpl.expert_matmul(rows.cuda(), w, indptr.cuda()).cpu()
    assert torch.equal(got[:, :8].double(), want[:, :8]) and (got[:, :8] != 0).all()
    assert torch.equal(got[:, 8:16].double(), want[:, 8:16])
    assert torch.isinf(got[:, 16:24]).all() and (got[:, 24:] == 0).all()


def test_matmul_gradients_against_differences(cuda):
  # The product is linear in either operand, so differences of any step are exact but for rounding: 2 products of inner
  # terms, off by check_sums' bound each.
  n, inner, out = 50, 9, 11
  indptr = torch.tensor([0, 20, 20, 45], dtype=torch.int32)
  rows, weight, ct = normal(1, n, inner), normal(2, 3, inner, out), normal(3, n, out)
  d = normal(4, n, inner), normal(5, 3, inner, out)
  given, w = rows.cuda().requires_grad_(), weight.cuda().requires_grad_()
  grads = torch.autograd.grad(bpl.expert_matmul(given, w, indptr.cuda()), (given, w), ct.cuda())
  for i in range(2):
    up = bpl.expert_matmul((rows + d[0]).cuda() if i == 0 else given, (weight + d[1]).cuda() if i == 1 else w, indptr.cuda())
    down = bpl.expert_matmul((rows - d[0]).cuda() if i == 0 else given, (weight - d[1]).cuda() if i == 1 else w, indptr.cuda())
    slope = (((up.double() - down.double()) / 2).cpu() * ct.double()).sum()
    along = (grads[i].double().cpu() * d[i].double()).sum()
    size = plain.matmul(rows.abs() + d[0].abs(), weight.abs() + d[1].abs(), indptr)
    # (the sums of x + d and x - d are rounded too, half a step of each operand)
    bound = (max(inner, n) + 4) * 8 * STEP * float((size * ct.abs().double()).sum())
    assert abs(float(slope - along)) <= bound


def test_matmul_of_an_indptr_that_is_none(cuda):
  # whatever it holds, nothing outside the arrays is touched and the call ends; a prefix that is in order is right
  rows, weight = normal(1, 64, 16).cuda(), normal(2, 4, 16, 24).cuda()
  guard = torch.full((64 * 24 + 4096,), 7.0, device="cuda")
  for values in ([0, 10, 5, 70, -3], [0, 2 ** 31 - 1, 3, 4, 5], [-1, -1, -1, -1, -1], [9, 9, 9, 9, 9], [0, 64, 64, 64, 64]):
    out = bpl.expert_matmul(rows, weight, torch.tensor(values, dtype=torch.int32).cuda())
    torch.cuda.synchronize()
    assert out.shape == (64, 24)
  assert (guard == 7).all()
  assert torch.isfinite(out).all()


def test_matmul_weights_of_more_elements_than_32_bits_number(cuda):
  experts, inner, out = 520, 2048, 4160  # 4.4e9 elements
  weight = torch.empty(experts, inner, out, dtype=torch.bfloat16, device="cuda")
  weight.copy_((torch.arange(experts, device="cuda") % 64).to(torch.bfloat16)[:, None, None].expand_as(weight))
  rows = torch.zeros(520, inner, dtype=torch.bfloat16, device="cuda")
  rows[:, 5] = 1.0
  rows[:, inner - 1] = 2.0
  indptr = torch.arange(521, dtype=torch.int32, device="cuda")
  got = bpl.expert_matmul(rows, weight, indptr)
  want = 3.0 * (torch.arange(experts, device="cuda") % 64)
  assert torch.equal(got.float(), want[:, None].expand(520, out))
  got = bpl.expert_matmul(rows, weight.view(experts, out, inner).transpose(1, 2), indptr)
  assert torch.equal(got.float(), want[:, None].expand(520, out))


# ---- all of them, as they are used ------------------------------------------------------------------------------------
def block(x, gate, up, down, k, mask=None):
  """Two products with an activation between, of the k experts of every token."""
  weights, experts = bpl.expert_topk(x @ gate, k=k, mask=mask)
  indptr, order, position = bpl.expert_sort(experts, num_experts=gate.shape[1])
  rows = bpl.expert_matmul(bpl.expert_dispatch(x, order, position), up, indptr)
  rows = bpl.expert_matmul(torch.nn.functional.silu(rows), down, indptr)
  return bpl.expert_combine(rows, weights, order, position)


def plain_block(x, gate, up, down, k, mask, chosen):
  """The same token by token in 64 bits, with torch's own gradients; the choice is given (ties of rounded logits)."""
  logits = x @ gate
  out = torch.zeros_like(x)
  for t in range(x.shape[0]):
    taken = [int(e) for e in chosen[t] if e >= 0]
    if taken:
      w = torch.softmax(logits[t, taken], dim=0)
      out[t] = sum(w[i] * (torch.nn.functional.silu(x[t] @ up[e]) @ down[e]) for i, e in enumerate(taken))
  return out


@pytest.mark.parametrize("tokens, padded", [(1, False), (50, True)])
def test_a_block_of_experts_and_its_gradients(cuda, tokens, padded):
  width, hidden, experts, k = 40, 56, 6, 2
  leaves = [normal(i, *s, scale=c) for i, (s, c) in enumerate((((tokens, width), 1.0), ((width, experts), 0.3),
            ((experts, width, hidden), 0.2), ((experts, hidden, width), 0.2)))]
  mask = torch.arange(tokens) % 7 != 3 if padded else None
  mine = [t.cuda().requires_grad_() for t in leaves]
  out = block(*mine, k, None if mask is None else mask.cuda())
  _, chosen = bpl.expert_topk(mine[0].detach() @ mine[1].detach(), k=k, mask=None if mask is None else mask.cuda())
  theirs = [t.double().requires_grad_() for t in leaves]
  want = plain_block(*theirs, k, mask, chosen.cpu())
  ct = normal(9, tokens, width)
  got = torch.autograd.grad(out, mine, ct.cuda())
  wanted = torch.autograd.grad(want, theirs, ct.double(), allow_unused=True)
  # a chain of five operators, each of whose sums of at most 56 (tokens * k: 100) terms is off by a step a term of the sum
  # of its absolute addends; those exceed the result by less than 100 for these inputs: compared to the largest entry
  for a, b in zip((out,) + got, (want,) + wanted):
    assert (a.double().cpu() - b).abs().max() <= 5 * 100 * 2 * STEP * 100 * max(1.0, float(b.abs().max()))
  if padded:
    assert (out[~mask] == 0).all() and (got[0][~mask] == 0).all()


def test_strided_operands_and_broadcast_gradients(cuda):
  _, order, position = arrays(1, 30, 2, 5)
  o, p = order.cuda(), position.cuda()
  wide = normal(1, 30, 100).cuda().requires_grad_()
  part = wide[:, 10:60]  # rows that do not lie together
  rows = bpl.expert_dispatch(part, o, p)
  assert torch.equal(rows, bpl.expert_dispatch(part.detach().contiguous(), o, p))
  rows.sum().backward()  # (a cotangent of stride 0)
  assert (wide.grad[:, 60:] == 0).all()
  assert torch.equal(wide.grad[:, 10], (position >= 0).sum(1).float().cuda())
  # one matrix for all experts: its gradient is the sum of theirs
  indptr = torch.tensor([0, 10, 25, 40], dtype=torch.int32).cuda()
  shared = normal(2, 50, 9).cuda().requires_grad_()
  x = normal(3, 40, 50).cuda()
  out = bpl.expert_matmul(x, shared.expand(3, 50, 9), indptr)
  ct = normal(4, 40, 9).cuda()
  out.backward(ct)
  check_sums(shared.grad, x.double().cpu().t() @ ct.double().cpu(), x.double().cpu().abs().t() @ ct.double().cpu().abs(), 45, "shared")
  # a weight of some other storage, operands from the host
  other = normal(5, 50, 3, 9).cuda().permute(1, 0, 2)
  assert torch.equal(bpl.expert_matmul(x, other, indptr), bpl.expert_matmul(x, other.contiguous(), indptr))
  assert torch.equal(bpl.expert_matmul(x.cpu(), other, indptr.cpu()), bpl.expert_matmul(x, other, indptr))
  # an offset that leaves 16-byte loads unaligned
  base = normal(6, 40 * 64 + 1, dtype=torch.bfloat16).cuda()
  w = normal(7, 3 * 64 * 32 + 3, dtype=torch.bfloat16).cuda()
  a = bpl.expert_matmul(base[1:].view(40, 64), w[3:].view(3, 64, 32), indptr)
  assert torch.equal(a, bpl.expert_matmul(base[1:].clone().view(40, 64), w[3:].clone().view(3, 64, 32), indptr))


def test_empty_operands(cuda):
  for tokens, k, width in ((0, 2, 8), (4, 0, 8), (4, 2, 0)):
    order, position = (torch.arange(tokens * k, dtype=torch.int32).cuda() for _ in range(2))
    position = position.reshape(tokens, k)
    x = torch.ones(tokens, width, device="cuda", requires_grad=True)
    rows = bpl.expert_dispatch(x, order, position)
    weights = torch.ones(tokens, k, device="cuda", requires_grad=True)
    out = bpl.expert_combine(rows, weights, order, position)
    assert out.shape == (tokens, width) and (out == (k > 0) * k).all()
    out.sum().backward()
    assert weights.grad.shape == (tokens, k) and (weights.grad == width).all() and (x.grad == k).all()
  w, e = bpl.expert_topk(torch.zeros(0, 4, device="cuda", requires_grad=True), k=2)
  assert w.shape == (0, 2) and e.shape == (0, 2)
  w.sum().backward()
  for n, inner, out in ((0, 4, 5), (6, 0, 5), (6, 4, 0)):
    x = torch.ones(n, inner, device="cuda", requires_grad=True)
    weight = torch.ones(2, inner, out, device="cuda", requires_grad=True)
    got = bpl.expert_matmul(x, weight, torch.tensor([0, n // 2, n], dtype=torch.int32).cuda())
    assert got.shape == (n, out) and (got == inner).all()
    got.sum().backward()
    assert (x.grad == out).all() and (weight.grad == n // 2).all()


def test_another_stream(cuda):
  _, order, position = arrays(2, 64, 4, 8)
  o, p, x = order.cuda(), position.cuda(), normal(1, 64, 300).cuda()
  want = bpl.expert_dispatch(x, o, p)
  torch.cuda.synchronize()
  s = torch.cuda.Stream()
  with torch.cuda.stream(s):
    got = bpl.expert_dispatch(x, o, p)
    experts = torch.from_numpy(choices(3, 9000, 4, 16)).cuda()
    arrays_ = bpl.expert_sort(experts, num_experts=16)
  s.synchronize()
  assert torch.equal(got, want)
  for a, b in zip(arrays_, plain.sort(experts.cpu().numpy(), 16)):
    assert np.array_equal(a.cpu().numpy(), b)


def test_second_order_and_forward_mode_are_refused(cuda):
  x = normal(1, 6, 8).cuda().requires_grad_()
  w, _ = bpl.expert_topk(x, k=2)
  (g,) = torch.autograd.grad(w.square().sum(), x, create_graph=True)
  with pytest.raises(NotImplementedError):
    torch.autograd.grad(g.sum(), x)
  indptr = torch.tensor([0, 3, 6], dtype=torch.int32).cuda()
  weight = normal(2, 2, 8, 5).cuda().requires_grad_()
  g = torch.autograd.grad(bpl.expert_matmul(x, weight, indptr).sum(), x, create_graph=True)[0]
  with pytest.raises(NotImplementedError):
    torch.autograd.grad(g.sum(), weight)
  from torch.autograd import forward_ad
  with forward_ad.dual_level():
    dual = forward_ad.make_dual(x.detach(), torch.ones_like(x))
    with pytest.raises(NotImplementedError):
      bpl.expert_matmul(dual, weight.detach(), indptr)


def test_captured_training_step_replays(cuda):
  tokens, width, hidden, experts, k = 300, 64, 96, 8, 2
  leaves = [normal(i, *s, scale=c).to(torch.bfloat16).cuda().requires_grad_() for i, (s, c) in enumerate((
    ((tokens, width), 1.0), ((width, experts), 0.3), ((experts, width, hidden), 0.2), ((experts, hidden, width), 0.2)))]
  ct = normal(9, tokens, width, dtype=torch.bfloat16).cuda()

  def step():
    out = block(*leaves, k)
    return (out.detach(),) + torch.autograd.grad(out, leaves, ct)

  s = torch.cuda.Stream()
  s.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(s):
    step()
  torch.cuda.synchronize()
  graphs = []
  for _ in range(2):  # two graphs of one stream, whose replays alternate
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
      captured = step()
    graphs.append((g, captured))
  for i in range(6):
    with torch.no_grad():
      leaves[0].copy_(normal(100 + i, tokens, width, dtype=torch.bfloat16).cuda())
    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    g, captured = graphs[i % 2]
    for t in captured:
      t.detach().zero_()
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(captured, want):
      assert torch.equal(a, b), i


def test_captured_cold(cuda):
  child = os.path.join(os.path.dirname(os.path.abspath(__file__)), "expert_capture_child.py")
  r = subprocess.run([sys.executable, "-u", child], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
  assert r.returncode == 0 and "captured cold: ok" in r.stdout, r.stdout[-2000:]


def test_two_streams_at_once(cuda):
  # products whose workgroups fill the card, sorts with room of their own: each as if it were alone
  indptr = torch.tensor([0, 1500, 1500, 4000], dtype=torch.int32).cuda()
  operands = [(normal(i, 4000, 512, dtype=torch.bfloat16).cuda(), normal(10 + i, 3, 512, 640, dtype=torch.bfloat16).cuda(),
               torch.from_numpy(choices(i, 20_000, 4, 40)).cuda()) for i in range(2)]

  def work(x, w, chosen):
    return (bpl.expert_matmul(x, w, indptr),) + bpl.expert_sort(chosen, num_experts=40)

  want = [work(*o) for o in operands]
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream() for _ in operands]
  got = [[], []]
  for _ in range(8):
    for s, o, g in zip(streams, operands, got):
      with torch.cuda.stream(s):
        g.append(work(*o))
  torch.cuda.synchronize()
  for g, w in zip(got, want):
    for result in g:
      for a, b in zip(result, w):
        assert torch.equal(a, b)


def test_captured_sort_of_many_pairs_replays(cuda):
  given = torch.zeros(40_000, 2, dtype=torch.int32, device="cuda")
  s = torch.cuda.Stream()
  g = torch.cuda.CUDAGraph()
  with torch.cuda.stream(s):
    bpl.expert_sort(given, num_experts=50)
  torch.cuda.synchronize()
  with torch.cuda.graph(g, stream=s):
    got = bpl.expert_sort(given, num_experts=50)
  for i in range(4):
    chosen = np.random.default_rng(i).integers(-1, 51, given.shape).astype(np.int32)
    given.copy_(torch.from_numpy(chosen))
    bpl.expert_sort(given, num_experts=7)  # eager work between
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, plain.sort(chosen, 50)):
      assert np.array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_operands_of_one_element_from_the_host(cuda, dtype):
  def one(*shape, value=1.5):
    return torch.full(shape, value, dtype=dtype)
  weights, chosen = bpl.expert_topk(one(1, 1), k=1)
  assert weights.tolist() == [[1.0]] and chosen.tolist() == [[0]]
  indptr, order, position = bpl.expert_sort(chosen.cpu(), num_experts=1)
  assert (indptr.tolist(), order.tolist(), position.tolist()) == ([0, 1], [0], [[0]])
  rows = bpl.expert_dispatch(one(1, 1), order.cpu(), position.cpu())
  out = bpl.expert_matmul(one(1, 1), one(1, 1, 1, value=-2.0), indptr.cpu())
  back = bpl.expert_combine(one(1, 1, value=-3.0), weights.cpu(), order.cpu(), position.cpu())
  assert (rows.tolist(), out.tolist(), back.tolist()) == ([[1.5]], [[-3.0]], [[-3.0]])
  assert rows.dtype == out.dtype == back.dtype == dtype
  given = one(1, 1).requires_grad_()  # (a gradient goes back to the host)
  bpl.expert_matmul(given, one(1, 1, 1, value=-2.0), indptr).sum().backward()
  assert given.grad.device.type == "cpu" and given.grad.tolist() == [[-2.0]]
