"""The expert operators inside the transforms of torch.func, and where autograd differentiates or batches their gradients.  The
targets are replaced by sums on the CPU that look at the buffers' memory, which a transform's wrapper does not have: the
rules themselves are what is tested."""
import struct

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import brainpylib_amd as bpl
from brainpylib_amd import expert_ops

T, E, K, D, H = 7, 4, 2, 3, 5


def _targets(name, buffers, opaque):
  for t in buffers:
    assert type(t) is torch.Tensor and t.is_contiguous()
    t.data_ptr()  # (raises for a transform's wrapper)
  tokens, k, experts, rows, width, out, flags = struct.unpack("<7I", opaque)
  name = name.rsplit("_", 1)[0] if name != "expert_sort" else name
  if name == "expert_topk":
    logits, _, weights, chosen = buffers
    top = torch.topk(logits, k, dim=1)
    chosen.copy_(top.indices)
    weights.copy_(torch.softmax(top.values, 1) if flags & 1 else torch.softmax(logits, 1).gather(1, top.indices))
  elif name == "expert_topk_gradient":
    logits, chosen, weights, ct, grad = buffers
    inner = (weights * ct).sum(1, keepdim=True)
    at = chosen.long()
    if flags & 1:
      grad.zero_().scatter_(1, at, weights * (ct - inner))
    else:
      grad.copy_(-torch.softmax(logits, 1) * inner).scatter_add_(1, at, weights * ct)
  elif name == "expert_sort":
    chosen, indptr, order, position, _ = buffers
    flat = chosen.reshape(-1)
    order.copy_(torch.argsort(flat, stable=True))
    position.view(-1)[order.long()] = torch.arange(len(flat), dtype=torch.int32)
    indptr.copy_(torch.searchsorted(flat.sort().values, torch.arange(experts + 1, dtype=torch.int32)))
  elif name == "expert_dispatch":
    x, order, _, rows_ = buffers
    rows_.copy_(x[order.long() // k])
  elif name == "expert_dispatch_gradient":
    d_rows, _, position, d_x = buffers
    d_x.copy_(d_rows[position.long()].sum(1))
  elif name == "expert_combine":
    rows_, weights, _, position, y = buffers
    y.copy_((rows_[position.long()] * weights[..., None]).sum(1))
  elif name == "expert_combine_gradient":
    rows_, weights, order, position, ct, d_rows, d_weights = buffers
    if flags & 8:
      d_rows.copy_(ct[order.long() // k] * weights.reshape(-1)[order.long()][:, None])
    if flags & 16:
      d_weights.copy_((rows_[position.long()] * ct[:, None]).sum(2))
  elif name == "expert_matmul":
    a, stored, indptr, y, _ = buffers
    for e in range(experts):
      at = slice(int(indptr[e]), int(indptr[e + 1]))
      y[at] = a[at] @ (stored[e].t() if flags & 4 else stored[e])
  else:
    assert name == "expert_matmul_gradient"
    a, ct, indptr, d, _ = buffers
    for e in range(experts):
      at = slice(int(indptr[e]), int(indptr[e + 1]))
      d[e] = ct[at].t() @ a[at] if flags & 4 else a[at].t() @ ct[at]


@pytest.fixture
def on_cpu(monkeypatch):
  monkeypatch.setattr(expert_ops, "_call", _targets)
  monkeypatch.setattr(expert_ops, "device_of", lambda *tensors: torch.device("cpu"))


def leaves():
  g = torch.Generator().manual_seed(2)
  return [torch.randn(*shape, generator=g) for shape in ((T, D), (D, E), (E, D, H), (E, D, H))]


def block(x, gate, up, down, normalize=True):
  weights, experts = bpl.expert_topk(x @ gate, k=K, normalize=normalize)
  indptr, order, position = bpl.expert_sort(experts, num_experts=E)
  rows = bpl.expert_matmul(bpl.expert_dispatch(x, order, position), up, indptr)
  return bpl.expert_combine(bpl.expert_matmul(torch.tanh(rows), down.transpose(1, 2), indptr), weights, order, position)


def loss(*operands, **kw):
  return block(*operands, **kw).square().sum()


def gradients(*operands, **kw):
  mine = [t.clone().requires_grad_() for t in operands]
  return torch.autograd.grad(loss(*mine, **kw), mine)


def plain_block(x, gate, up, down, normalize=True):
  """The same with torch's own operators, every expert for every token."""
  p = torch.softmax(x @ gate, 1)
  taken = torch.zeros_like(p).scatter(1, torch.topk(p, K, dim=1).indices, 1.0)
  w = p * taken
  if normalize:
    w = w / w.sum(1, keepdim=True)
  y = torch.stack([torch.tanh(x @ up[e]) @ down[e].t() for e in range(E)], 1)
  return (w[..., None] * y).sum(1)


def close(got, want):
  # (sums of a few products in 32 bits in another order, numbers of about 1)
  assert len(got) == len(want)
  for a, b in zip(got, want):
    torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("normalize", [True, False])
def test_the_replaced_targets_and_the_rules(on_cpu, normalize):
  mine, theirs = ([t.clone().requires_grad_() for t in leaves()] for _ in range(2))
  out, want = block(*mine, normalize=normalize), plain_block(*theirs, normalize=normalize)
  close([out], [want])
  close(torch.autograd.grad(out.square().sum(), mine), torch.autograd.grad(want.square().sum(), theirs))


@pytest.mark.parametrize("normalize", [True, False])
def test_grad(on_cpu, normalize):
  operands = leaves()
  want = gradients(*operands, normalize=normalize)
  got = torch.func.grad(lambda *o: loss(*o, normalize=normalize), argnums=(0, 1, 2, 3))(*operands)
  assert all(torch.equal(a, b) for a, b in zip(got, want))
  # with respect to some: the others are no part of the transform
  for i in range(4):
    alone = torch.func.grad(lambda t: loss(*operands[:i], t, *operands[i + 1:], normalize=normalize))(operands[i])
    assert torch.equal(alone, want[i])
  value, grads = torch.func.grad_and_value(lambda x: loss(x, *operands[1:], normalize=normalize))(operands[0])[::-1]
  assert torch.equal(value, loss(*operands, normalize=normalize)) and torch.equal(grads, want[0])


def test_vjp(on_cpu):
  operands = leaves()
  ct = torch.linspace(-1, 1, T * D).reshape(T, D)
  out, pull = torch.func.vjp(block, *operands)
  mine = [t.clone().requires_grad_() for t in operands]
  assert torch.equal(out, block(*operands))
  for a, b in zip(pull(ct), torch.autograd.grad(block(*mine), mine, ct)):
    assert torch.equal(a, b)


def test_operators_on_what_is_no_part_of_the_transform(on_cpu):
  operands = leaves()

  def scaled(s):
    assert not block(*operands).requires_grad
    return s * loss(*operands)
  assert torch.equal(torch.func.grad(scaled)(torch.tensor(2.0)), loss(*operands))


def one_by_one():
  """(operator, its differentiable operands, the call) for each of them"""
  x, gate, up, _ = leaves()
  order = torch.arange(T * K, dtype=torch.int32)
  position = order.reshape(T, K)
  indptr = torch.tensor([0, 2, 5, 9, T * K], dtype=torch.int32)
  rows = torch.cat([x, x + 1])
  return [("expert_topk", (x @ gate,), lambda t: bpl.expert_topk(t, k=K)[0]),
          ("expert_dispatch", (x,), lambda t: bpl.expert_dispatch(t, order, position)),
          ("expert_combine", (rows, torch.rand(T, K)), lambda t, w: bpl.expert_combine(t, w, order, position)),
          ("expert_matmul", (rows, up), lambda t, w: bpl.expert_matmul(t, w, indptr))]


@pytest.mark.parametrize("at", range(4))
def test_batches_are_refused(on_cpu, at):
  name, operands, call = one_by_one()[at]
  batch = [torch.stack([t, t]) for t in operands]
  with pytest.raises(NotImplementedError, match=name + ".*vmap"):
    torch.func.vmap(call)(*batch)
  with pytest.raises(NotImplementedError, match=name + ".*vmap"):
    torch.func.vmap(torch.func.grad(lambda *o: call(*o).sum()))(*batch)
  with pytest.raises(NotImplementedError, match=name + ".*vmap"):
    torch.func.jacrev(call)(*operands)
  mine = [t.clone().requires_grad_() for t in operands]
  out = call(*mine)
  with pytest.raises(NotImplementedError, match=name + ".*vmap"):
    torch.autograd.grad(out, mine, torch.ones(2, *out.shape), is_grads_batched=True)


def test_sorting_a_batch_is_refused(on_cpu):
  with pytest.raises(NotImplementedError, match="expert_sort.*vmap"):
    torch.func.vmap(lambda e: bpl.expert_sort(e, num_experts=E))(torch.zeros(2, T, K, dtype=torch.int32))


def test_operators_inside_vmap_on_what_is_not_batched(on_cpu):
  operands = leaves()
  got = torch.func.vmap(lambda s: s * block(*operands))(torch.tensor([1.0, 2.0]))
  assert torch.equal(got[1], 2 * block(*operands))


@pytest.mark.parametrize("at", range(4))
def test_forward_mode_is_refused(on_cpu, at):
  name, operands, call = one_by_one()[at]
  ones = tuple(torch.ones_like(t) for t in operands)
  with pytest.raises(NotImplementedError, match=name + ".*forward-mode"):
    torch.func.jvp(call, operands, ones)
  out = call(operands[0].clone().requires_grad_(), *operands[1:])
  with fwAD.dual_level(), pytest.raises(NotImplementedError, match=name + ".*forward-mode"):
    out.backward(fwAD.make_dual(torch.ones_like(out), torch.ones_like(out)))


@pytest.mark.parametrize("at", range(4))
def test_second_order_is_refused(on_cpu, at):
  name, operands, call = one_by_one()[at]
  mine = [t.clone().requires_grad_() for t in operands]
  first = torch.autograd.grad(call(*mine).square().sum(), mine, create_graph=True)
  for g in first:
    assert g.requires_grad
    with pytest.raises(NotImplementedError, match=name + " has gradients of first order only"):
      torch.autograd.grad(g.sum(), mine, retain_graph=True, allow_unused=True)
  with pytest.raises(NotImplementedError, match=name + " has gradients of first order only"):
    torch.func.grad(lambda *o: torch.func.grad(lambda *i: call(*i).square().sum())(*o).sum())(*operands)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_grad_and_vjp_on_the_gpu(cuda, dtype):
  operands = [t.to(dtype).cuda() for t in leaves()]
  want = gradients(*operands)
  for a, b in zip(torch.func.grad(loss, argnums=(0, 1, 2, 3))(*operands), want):
    assert torch.equal(a, b)
  out, pull = torch.func.vjp(block, *operands)
  mine = [t.clone().requires_grad_() for t in operands]
  again = block(*mine)
  ct = torch.ones_like(out)
  assert torch.equal(out, again.detach())
  for a, b in zip(pull(ct), torch.autograd.grad(again, mine, ct)):
    assert torch.equal(a, b)
  rows = [t.clone().requires_grad_() for t in operands]
  with pytest.raises(NotImplementedError, match="vmap"):
    y = block(*rows)
    torch.autograd.grad(y, rows, torch.ones(2, *y.shape, device="cuda", dtype=dtype), is_grads_batched=True)
