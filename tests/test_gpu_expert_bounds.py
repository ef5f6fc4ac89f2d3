"""The expert products on index arrays that are none: nothing outside the arrays is read or written, and the work is bounded.
Operands and results lie within one allocation each, between parts that are watched."""
import pytest
import torch

from brainpylib_amd import _lib

pytestmark = pytest.mark.gpu

GUARD = 4096  # elements on either side
BROKEN = [[0, 10, 5, 70, -3], [0, 2 ** 31 - 1, 3, 4, 5], [-1, -1, -1, -1, -1], [9, 9, 9, 9, 9], [64, 0, 64, 0, 64], [0, 64, 64, 64, 64]]
SUFFIX = {torch.float32: "_float", torch.float16: "_half", torch.bfloat16: "_bfloat16"}


def guarded(values, guard):
  """(allocation, the tensor in its middle) with ``guard`` on both sides."""
  base = torch.full((2 * GUARD + values.numel(),), guard, dtype=values.dtype, device="cuda")
  inner = base[GUARD:GUARD + values.numel()].view(values.shape)
  inner.copy_(values)
  return base, inner


def untouched(base, guard):
  return bool((base[:GUARD] == guard).all() and (base[-GUARD:] == guard).all())


def ranges(indptr, rows):
  """The rows of every expert as the kernels read indptr: unsigned, within the rows, from 0."""
  ends = [0] + [min(v % 2 ** 32, rows) for v in indptr[1:]]
  return [(a, max(a, b)) for a, b in zip(ends[:-1], ends[1:])]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("inner, out", [(16, 24), (33, 50), (64, 130)])
@pytest.mark.parametrize("out_major", [False, True])
@pytest.mark.parametrize("parts", [1, 3])
def test_products_stay_within_their_arrays(cuda, dtype, inner, out, out_major, parts):
  n, experts = 64, 4
  g = torch.Generator().manual_seed(inner)

  def whole(*shape):  # (small whole numbers: every sum is exact in 32 bits, and below 256: in 16 too)
    return torch.randint(-1, 2, shape, generator=g).to(dtype)
  x, weight, ct = whole(n, inner), whole(experts, inner, out), whole(n, out)
  nan = float("nan")
  (_, rows), (_, cts) = guarded(x, nan), guarded(ct, nan)
  stored = weight.transpose(1, 2).contiguous() if out_major else weight
  _, w = guarded(stored, nan)
  opaque = _lib.build_expert_descriptor(0, parts, experts, n, inner, out, 4 if out_major else 0)
  for values in BROKEN:
    _, indptr = guarded(torch.tensor(values, dtype=torch.int32), 1 << 20)
    of = ranges(values, n)
    y_base, y = guarded(torch.full((n, out), 7.0, dtype=dtype), 5.0)
    s_base, scratch = guarded(torch.zeros(parts, n, out), 5.0)
    _lib.custom_call("expert_matmul" + SUFFIX[dtype], [rows, w, indptr, y, scratch], opaque)
    torch.cuda.synchronize()
    assert untouched(y_base, 5.0) and untouched(s_base, 5.0), values
    got, behind = y.float().cpu(), min(values[-1] % 2 ** 32, n)
    assert torch.isfinite(got).all(), values
    for r in range(n):  # rows that one expert claims and no zero
      claim = [e for e, (a, b) in enumerate(of) if a <= r < b]
      if len(claim) == 1 and r < behind:
        assert torch.equal(got[r], x[r].float() @ weight[claim[0]].float()), (values, r)
      elif not claim and r >= behind:
        assert (got[r] == 0).all(), (values, r)
    d_base, d = guarded(torch.full(stored.shape, 7.0, dtype=dtype), 5.0)
    s_base, scratch = guarded(torch.zeros((parts,) + tuple(stored.shape)), 5.0)
    _lib.custom_call("expert_matmul_gradient" + SUFFIX[dtype], [rows, cts, indptr, d, scratch], opaque)
    torch.cuda.synchronize()
    assert untouched(d_base, 5.0) and untouched(s_base, 5.0), values
    for e, (a, b) in enumerate(of):  # (also where several experts claim a row)
      want = x[a:b].float().t() @ ct[a:b].float()
      assert torch.equal(d[e].float().cpu(), want.t() if out_major else want), (values, e)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_that_many_experts_claim_are_not_worked_on_by_all_of_them(cuda, dtype):
  # 40 experts claim the first 16,320 rows, the last one the 64 behind them: more tiles of any height (16 to 256) than an indptr in
  # order can have (16,384 / height + 80), and what is beyond those is left out, the last expert's rows among it
  n, claimed, experts, inner, out = 16_384, 16_320, 80, 8, 8
  for height in (16, 64, 128, 256):
    assert 40 * -(-claimed // height) > n // height + experts
  indptr = torch.tensor([0, claimed] * 40 + [n], dtype=torch.int32).cuda()
  x = torch.randint(-2, 3, (n, inner), generator=torch.Generator().manual_seed(0)).to(dtype).cuda()
  w = torch.ones(experts, inner, out, dtype=dtype, device="cuda")  # (the same for all: whoever comes last)
  y = torch.full((n, out), 7.5, dtype=dtype, device="cuda")
  _lib.custom_call("expert_matmul" + SUFFIX[dtype], [x, w, indptr, y, y], _lib.build_expert_descriptor(0, 1, experts, n, inner, out, 0))
  torch.cuda.synchronize()
  assert torch.equal(y[:claimed], (x[:claimed].float() @ w[0].float()).to(dtype))
  assert (y[claimed:] == 7.5).all()
