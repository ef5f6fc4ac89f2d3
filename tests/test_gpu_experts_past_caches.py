"""expert_matmul with the largest tiles and results of 64 MB and more, which are stored past the caches: how training steps
run in 16 bits."""
import pytest
import torch

import brainpylib_amd as bpl

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("out_major", [False, True])
def test_largest_tiles_stored_past_the_caches(cuda, dtype, out_major):
  # The product (159 MB), the gradient of the rows (88 MB, the product with the other storage) and that of the weights (73 MB)
  # in tiles of 256 x 256, those at the edges among them; one expert has no rows, and there are rows behind the last.
  # Whole numbers: every sum is exact in 32 bits in any order (below 2 * 7,798 < 2^24), one rounding is left, and it is to nearest
  # on both sides.  A store whose data is changed while it is read goes by the moment: three passes.
  inner, out, n, experts = 2304, 4160, 20_000, 4
  indptr = [0, 5203, 5203, 13_001, 19_900]
  ends = torch.tensor(indptr, dtype=torch.int32).cuda()
  for seed in range(3):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def whole(most, *shape):
      return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(dtype)
    rows, ct, weight = whole(2, n, inner), whole(1, n, out), whole(1, experts, inner, out)
    rows[indptr[-1]:], ct[indptr[-1]:] = float("nan"), float("nan")
    given = rows.clone().requires_grad_()
    stored = (weight.transpose(1, 2).contiguous() if out_major else weight.clone()).requires_grad_()
    got = bpl.expert_matmul(given, stored.transpose(1, 2) if out_major else stored, ends)
    d_rows, d_stored = torch.autograd.grad(got, (given, stored), ct)
    d_weight = d_stored.transpose(1, 2) if out_major else d_stored
    for e in range(experts):
      at = slice(indptr[e], indptr[e + 1])
      x, c, w = rows[at].float(), ct[at].float(), weight[e].float()
      assert torch.equal(got[at], (x @ w).to(dtype)), (seed, e)
      assert torch.equal(d_rows[at], (c @ w.t().contiguous()).to(dtype)), (seed, e)
      assert torch.equal(d_weight[e], (x.t().contiguous() @ c).to(dtype)), (seed, e)
    assert (got[indptr[-1]:] == 0).all() and (d_rows[indptr[-1]:] == 0).all()


@pytest.mark.parametrize("dtype, width, megabytes", [(torch.bfloat16, 1000, 70), (torch.bfloat16, 1000, 300), (torch.float32, 516, 140),
                                                     (torch.float32, 516, 270), (torch.float16, 1024, 70)])
def test_gradients_of_combine_of_rows_that_share_lines(cuda, dtype, width, megabytes):
  # rows that end within a line of 128 bytes, below and above what the last cache holds, and rows that do not
  k = 4
  tokens = (megabytes << 20) // (k * width * dtype.itemsize) + 1
  pairs = tokens * k
  g = torch.Generator(device="cuda").manual_seed(width)
  order = torch.randperm(pairs, generator=g, device="cuda").to(torch.int32)
  position = torch.empty_like(order)
  position[order.long()] = torch.arange(pairs, dtype=torch.int32, device="cuda")
  # whole numbers: every product and sum is exact
  rows = torch.randint(-2, 3, (pairs, width), generator=g, device="cuda").to(dtype).requires_grad_()
  weights = torch.randint(-3, 4, (tokens, k), generator=g, device="cuda").float().requires_grad_()
  ct = torch.randint(-2, 3, (tokens, width), generator=g, device="cuda").to(dtype)
  out = bpl.expert_combine(rows, weights, order, position.reshape(tokens, k))
  d_rows, d_weights = torch.autograd.grad(out, (rows, weights), ct)
  at = order.long()
  assert torch.equal(d_rows, (ct[at // k].float() * weights.detach().reshape(-1)[at][:, None]).to(dtype))
  picked = rows.detach()[position.long()].reshape(tokens, k, width).float()
  assert torch.equal(d_weights, (picked * ct[:, None].float()).sum(2))
