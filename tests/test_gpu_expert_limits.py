"""The expert operators at the ends of their ranges: as many pairs as there may be, arrays of more elements than 32 bits number,
lines longer than those that go straight to LDS.  Whole numbers everywhere, small enough that sums are exact in 32 bits."""
import pytest
import torch

import brainpylib_amd as bpl

pytestmark = pytest.mark.gpu


def whole(seed, most, *shape, dtype=torch.float32):
  g = torch.Generator(device="cuda").manual_seed(seed)
  return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(dtype)


def test_sort_of_as_many_pairs_as_there_may_be(cuda):
  pairs, experts, part = 2 ** 31 - 1, 37, 2 ** 27
  chosen = torch.empty(pairs, dtype=torch.int32, device="cuda")
  counts = torch.zeros(experts + 3, dtype=torch.int64, device="cuda")
  g = torch.Generator(device="cuda").manual_seed(0)
  for a in range(0, pairs, part):
    some = torch.randint(-1, experts + 2, (min(part, pairs - a),), generator=g, device="cuda", dtype=torch.int32)
    chosen[a:a + part] = some
    counts += torch.bincount(some.long() + 1, minlength=experts + 3)
  indptr, order, position = bpl.expert_sort(chosen, num_experts=experts)
  want = torch.cat([counts[:1] * 0, counts[1:experts + 1].cumsum(0)])
  assert torch.equal(indptr.long(), want)
  end = int(want[-1])
  for a in range(0, pairs, part):
    b = min(a + part, pairs)
    # every pair's row lies among its expert's and names the pair; a dropped one has none
    at, of = position[a:b].long(), chosen[a:b].long()
    there = (of >= 0) & (of < experts)
    assert torch.equal(at < 0, ~there) and (at[~there] == -1).all()
    at, of = at[there], of[there]
    assert ((at >= want[of]) & (at < want[of + 1])).all()
    assert torch.equal(order[at].long(), (torch.arange(a, b, device="cuda"))[there])
    # within an expert the pairs keep their order
    rows = order[a:min(b + 1, pairs)].long()
    inside = torch.arange(a, a + rows.shape[0] - 1, device="cuda")
    first = torch.isin(inside + 1, want)
    assert ((rows[1:] > rows[:-1]) | first | (inside + 1 >= end)).all()
    assert (order[max(a, end):max(b, end)] == -1).all()


def test_choice_of_more_logits_than_32_bits_number(cuda):
  tokens, experts, k = 4_300_000, 1024, 3
  logits = torch.zeros(tokens, experts, dtype=torch.bfloat16, device="cuda")
  t = torch.arange(tokens, device="cuda")
  best = (t * 7919) % experts
  logits[t, best] = 2.0
  logits[t, (best + 5) % experts] = 1.0
  given = logits.requires_grad_()
  weights, chosen = bpl.expert_topk(given, k=k)
  assert torch.equal(chosen[:, 0].long(), best) and torch.equal(chosen[:, 1].long(), (best + 5) % experts)
  w = torch.softmax(torch.tensor([2.0, 1.0, 0.0], dtype=torch.float64), 0).cuda()
  assert ((weights.double() - w).abs() <= 16 * 2.0 ** -24).all()  # (exp, a sum of three and a quotient, below 1)
  ct = torch.zeros(tokens, k, device="cuda")
  ct[:, 0] = 1.0
  (grad,) = torch.autograd.grad(weights, given, ct)
  for a in (0, 4_194_300, tokens - 8):  # (the first rows, those around element 2^32 and the last)
    rows, b = grad[a:a + 8].double(), best[a:a + 8]
    assert (rows[torch.arange(8), b] - w[0] * (1 - w[0])).abs().max() <= 2.0 ** -9  # (below 1/4, rounded to 8 bits)
    assert (rows[torch.arange(8), (b + 5) % experts] + w[0] * w[1]).abs().max() <= 2.0 ** -9
    assert ((rows != 0).sum(1) == 3).all()


def test_gradients_of_combine_of_more_elements_than_32_bits_number(cuda):
  tokens, k, width = 35_000, 2, 65_600  # 4.6e9 elements of rows
  order = torch.arange(tokens * k, dtype=torch.int32).flip(0).cuda()
  position = order.reshape(tokens, k)  # (its own inverse)
  rows = (torch.arange(tokens * k, device="cuda") % 7 - 3).to(torch.bfloat16)[:, None].expand(-1, width).contiguous().requires_grad_()
  weights = whole(1, 3, tokens, k).requires_grad_()
  ct = (torch.arange(tokens, device="cuda") % 5 - 2).to(torch.bfloat16)[:, None].expand(-1, width).contiguous()
  out = bpl.expert_combine(rows, weights, order, position)
  d_rows, d_weights = torch.autograd.grad(out, (rows, weights), ct)
  at = position.long()
  assert torch.equal(d_weights, rows.detach()[:, 0][at].float() * ct[:, :1].float() * width)
  for r in (0, 1, 32_739, 32_740, 65_471, 65_472, tokens * k - 1):
    p = tokens * k - 1 - r
    assert (d_rows[r].float() == weights.detach().reshape(-1)[p] * ct[p // k, 0].float()).all(), r


@pytest.mark.parametrize("out_major", [False, True])
def test_products_of_rows_of_more_elements_than_32_bits_number(cuda, out_major):
  n, inner, out = 70_000, 65_600, 8
  indptr = torch.tensor([0, 30_001, 69_990], dtype=torch.int32).cuda()
  a = whole(1, 1, n)
  rows = a.to(torch.bfloat16)[:, None].expand(n, inner).contiguous().requires_grad_()
  weight = whole(2, 1, 2, inner, out, dtype=torch.bfloat16)
  ct = whole(3, 1, n, out, dtype=torch.bfloat16)
  stored = (weight.transpose(1, 2).contiguous() if out_major else weight.clone()).requires_grad_()
  got = bpl.expert_matmul(rows, stored.transpose(1, 2) if out_major else stored, indptr)
  d_rows, d_stored = torch.autograd.grad(got, (rows, stored), ct)
  d_weight = d_stored.transpose(1, 2) if out_major else d_stored
  for e, (i, j) in enumerate(((0, 30_001), (30_001, 69_990))):
    assert torch.equal(got[i:j], (a[i:j, None] * weight[e].float().sum(0)).to(torch.bfloat16))
    per_column = (a[i:j, None].double() * ct[i:j].double()).sum(0).to(torch.bfloat16)
    assert torch.equal(d_weight[e], per_column.expand(inner, out))
    for r in (i, j - 1, min(j - 1, 65_472)):
      assert torch.equal(d_rows[r], (weight[e].double() @ ct[r].double()).to(torch.bfloat16)), r
  assert (got[69_990:] == 0).all() and (d_rows[69_990:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("inner, out", [(2 ** 20 + 8, 8), (8, 2 ** 20 + 8), (2 ** 20 + 3, 2)])
@pytest.mark.parametrize("out_major", [False, True])
def test_lines_longer_than_those_that_go_straight_to_lds(cuda, dtype, inner, out, out_major):
  n = 70
  indptr = torch.tensor([0, 3, 3, 67], dtype=torch.int32).cuda()
  # (a sum over 2^20 of -1, 0 and 1 is some thousands: within half precision's range)
  rows, ct, weight = whole(1, 1, n, inner, dtype=dtype), whole(2, 1, n, out, dtype=dtype), whole(3, 1, 3, inner, out, dtype=dtype)
  rows[67:], ct[67:] = float("nan"), float("nan")
  given = rows.clone().requires_grad_()
  stored = (weight.transpose(1, 2).contiguous() if out_major else weight.clone()).requires_grad_()
  got = bpl.expert_matmul(given, stored.transpose(1, 2) if out_major else stored, indptr)
  d_rows, d_stored = torch.autograd.grad(got, (given, stored), ct)
  d_weight = d_stored.transpose(1, 2) if out_major else d_stored
  for e, (i, j) in enumerate(((0, 3), (3, 3), (3, 67))):
    x, c, w = rows[i:j].double(), ct[i:j].double(), weight[e].double()
    assert torch.equal(got[i:j], (x @ w).to(dtype)), e
    assert torch.equal(d_rows[i:j], (c @ w.t().contiguous()).to(dtype)), e
    assert torch.equal(d_weight[e], (x.t().contiguous() @ c).to(dtype)), e
  assert (got[67:] == 0).all() and (d_rows[67:] == 0).all()
