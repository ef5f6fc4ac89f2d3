"""Routing of tokens to experts, and the experts' products (host side).

A mixture of experts is a network of which every token meets only a few parts: the routing is a sparse tokens x experts
matrix with ``k`` nonzeros a row, its index arrays are built on the GPU as ``coo_to_csr`` builds those of synapses, and
only the products that it names are computed.  The reference has no such operators.

    weights, experts = expert_topk(logits, k=k)                       # the nonzeros of every row
    indptr, order, position = expert_sort(experts, num_experts=n)     # the same by expert
    rows = expert_dispatch(tokens, order, position)                   # a row for every nonzero, sorted by expert
    rows = expert_matmul(rows, weight, indptr)                        # every expert's rows times its matrix
    out = expert_combine(rows, weights, order, position)              # the weighted sum of every token's rows

Values are float32, float16 or bfloat16; sums, softmax and routing weights are held in 32 bits.  Gradients are of first
order, in backward mode: of ``autograd`` or of ``torch.func.grad`` and ``vjp``.  Forward mode and batches (``jvp``, ``vmap`` and what
uses it, as ``jacrev`` and ``is_grads_batched`` do) are refused with NotImplementedError.  No call waits for the GPU or reads a count back, so all of them can be captured into a HIP graph;
none uses scratch memory that outlives it, so graphs share none.  Results do not depend on the order of atomics.
"""
import torch

from . import _lib
from ._tensors import as_tensor, device_of, has_tangent, is_index_dtype, to_device

__all__ = ["expert_topk", "expert_sort", "expert_dispatch", "expert_combine", "expert_matmul"]

_TYPE_NAME = {torch.float32: '_float', torch.float16: '_half', torch.bfloat16: '_bfloat16'}
_NORMALIZE, _MASKED, _OUT_MAJOR, _D_ROWS, _D_WEIGHTS = 1, 2, 4, 8, 16  # BPL_EXPERT_* of the descriptor
_MOST_EXPERTS, _MOST_PER_TOKEN, _MOST = 1024, 64, 2 ** 31 - 1


def _current_device():
  """The current device's index, replaced by torch's own function at its first call (``torch.cuda.current_device`` looks
  first whether the device has been set up, which the tensors at hand say)."""
  global _current_device
  _current_device = getattr(torch._C, '_cuda_getDevice', torch.cuda.current_device)
  return _current_device()


def _call(name, buffers, opaque):
  device = buffers[0].device
  if device.index == _current_device():
    _lib.custom_call(name, buffers, opaque)
  else:  # (a kernel is launched on the current device, whatever the stream's)
    with torch.cuda.device(device):
      _lib.custom_call(name, buffers, opaque)


def _move(*tensors):
  device = device_of(*tensors)
  return [to_device(t, device) for t in tensors]


def _check_values(name, t, ndim):
  if t.dtype not in _TYPE_NAME:
    raise TypeError(f'Only support float32, float16 and bfloat16. But we got {t.dtype} for {name}.')
  if t.ndim != ndim:
    raise ValueError(f'{name} should be a {ndim}D array. But we got {t.ndim}-D array.')
  if max(t.shape, default=0) > _MOST:
    raise ValueError(f'{name} should have at most 2^31 - 1 entries in each dimension, got {tuple(t.shape)}.')


def _check_index(name, t, ndim):
  if not is_index_dtype(t.dtype):
    raise ValueError(f'{name} should have int32 or uint32 type, got {t.dtype}.')
  if t.ndim != ndim:
    raise ValueError(f'{name} should be a {ndim}D array. But we got {t.ndim}-D array.')


def _check_pairs(order, position, tokens):
  _check_index('order', order, 1)
  _check_index('position', position, 2)
  if position.shape[0] != tokens:
    raise ValueError(f'position should have a row for each of the {tokens} tokens, got {tuple(position.shape)}.')
  if position.shape[1] > _MOST_PER_TOKEN:
    raise ValueError(f'Only support up to {_MOST_PER_TOKEN} experts a token, got {position.shape[1]}.')
  if order.shape[0] != position.numel():
    raise ValueError(f'order should have an entry for each entry of position, got {order.shape[0]} != {position.numel()}.')
  if position.numel() > _MOST:
    raise ValueError('Only support up to 2^31 - 1 pairs of a token and an expert.')


def _check_experts(n):
  if not 1 <= n <= _MOST_EXPERTS:
    raise ValueError(f'Only support 1 to {_MOST_EXPERTS} experts, got {n}.')


def _differentiable(name, *tensors):
  """Whether a gradient is asked for; tangents are refused."""
  wanted = False
  for t in tensors:
    if has_tangent(t):
      raise NotImplementedError(f'{name} has no forward-mode differentiation.')
    wanted = wanted or t.requires_grad
  return wanted and torch.is_grad_enabled()


# ---- transforms of torch.func -----------------------------------------------------------------------------------------
# Inside one tensors are wrappers without memory of their own, those that are made there too.  torch looks under them for
# an autograd function whose context is set up by a step of its own; that step costs 5 us of host time a call, so that
# functions have it only where a transform is active.
_transforms_active = torch._C._are_functorch_transforms_active


class _Launch(torch.autograd.Function):
  """launch(*args), on the tensors underneath where a transform is active.  No gradient can be had of it: it takes part in the
  graph of what it is computed from."""

  @staticmethod
  def forward(name, launch, *args):
    return launch(*args)

  @staticmethod
  def setup_context(ctx, inputs, output):
    ctx.name, ctx.inputs = inputs[0], len(inputs)
    outputs = output if isinstance(output, tuple) else (output,)
    ctx.mark_non_differentiable(*[t for t in outputs if t is not None and not t.is_floating_point()])
    ctx.set_materialize_grads(False)

  @staticmethod
  def backward(ctx, *cts):
    if all(ct is None for ct in cts):
      return (None,) * ctx.inputs
    raise NotImplementedError(f'{ctx.name} has gradients of first order only.')

  @staticmethod
  def vmap(info, in_dims, name, *args):
    raise NotImplementedError(f'{name} has no rule for batches (vmap).')


def _gradient(name, launch, ct, *args):
  """launch(ct, *args): gradients, of which none can be had."""
  if has_tangent(ct):
    raise NotImplementedError(f'{name} has no forward-mode differentiation.')
  if _transforms_active():
    return _Launch.apply(name, launch, ct, *args)
  try:
    ct.data_ptr()
  except RuntimeError:  # (a batch of cotangents, which is no active transform for the backward pass)
    raise NotImplementedError(f'{name} has no rule for batches (vmap).') from None
  return _Launch.apply(name, launch, ct, *args) if torch.is_grad_enabled() else launch(ct, *args)  # (create_graph)


class _Operator(torch.autograd.Function):
  """What the operators' differentiation rules share: the operator's ``name``, its ``launch`` and ``keep``, which sets up the context.
  Each is made into a second one for transforms, ``inside``."""

  @classmethod
  def forward(cls, ctx, *inputs):
    output = cls.launch(*inputs)
    cls.keep(ctx, inputs, output)
    return output

  @classmethod
  def run(cls, *inputs):
    return (cls.inside if _transforms_active() else cls).apply(*inputs)


def _inside_transforms(operator):
  """Class decorator: adds ``inside``."""
  def vmap(info, in_dims, *inputs):
    raise NotImplementedError(f'{operator.name} has no rule for batches (vmap).')

  operator.inside = type(operator.__name__ + 'Inside', (operator,), {
    'forward': staticmethod(operator.launch), 'setup_context': staticmethod(operator.keep), 'vmap': staticmethod(vmap)})
  return operator


# ---- expert_topk ------------------------------------------------------------------------------------------------------
def _topk(logits, mask, k, normalize):
  n, experts = logits.shape
  weights = torch.empty((n, k), dtype=torch.float32, device=logits.device)
  chosen = torch.empty((n, k), dtype=torch.int32, device=logits.device)
  flags = (_NORMALIZE if normalize else 0) | (0 if mask is None else _MASKED)
  opaque = _lib.build_expert_descriptor(n, k, experts, 0, 0, 0, flags)
  _call('expert_topk' + _TYPE_NAME[logits.dtype], [logits, logits if mask is None else mask, weights, chosen], opaque)
  return weights, chosen


def _topk_gradient(ct, logits, chosen, weights, normalize):
  grad = torch.empty_like(logits)
  opaque = _lib.build_expert_descriptor(logits.shape[0], chosen.shape[1], logits.shape[1], 0, 0, 0, _NORMALIZE if normalize else 0)
  _call('expert_topk_gradient' + _TYPE_NAME[logits.dtype], [logits, chosen, weights, ct.contiguous(), grad], opaque)
  return grad


@_inside_transforms
class _ExpertTopk(_Operator):
  """With w the weights, g their cotangent: normalized, the chosen logits' cotangents are w (g - sum w g) and the others'
  0; else, with p the softmax over all experts, p ([chosen] g - sum w g)."""
  name = 'expert_topk'
  launch = staticmethod(_topk)

  @staticmethod
  def keep(ctx, inputs, output):
    logits, _, _, ctx.normalize = inputs
    weights, chosen = output
    ctx.mark_non_differentiable(chosen)
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(logits, chosen, weights)

  @staticmethod
  def backward(ctx, ct, _):
    if ct is None:
      return None, None, None, None
    return _gradient('expert_topk', _topk_gradient, ct, *ctx.saved_tensors, ctx.normalize), None, None, None


def expert_topk(logits, *, k: int, normalize: bool = True, mask=None):
  """Chooses ``k`` experts for every token.

  logits  (tokens, experts) float32 | float16 | bfloat16, up to 1,024 experts
  k       experts a token, 1 to min(experts, 64)
  mask    (tokens,) bool, False for rows of padding; None: there are none
  returns ``(weights, experts)``: float32 and int32 of shape (tokens, k), the largest logit first and the lowest index
          first among equal ones.  The weights are the softmax over the chosen experts (``normalize``), or theirs of the
          softmax over all.

  A logit of -inf is never chosen; places that are left over, and all those of a row of padding, hold expert -1 and weight 0,
  and have no gradient.  The lowest finite value is a logit like any other.  NaN counts as larger than every number and
  makes its row's weights NaN."""
  logits = as_tensor(logits)
  _check_values('logits', logits, 2)
  _check_experts(logits.shape[1])
  if not 1 <= k <= min(logits.shape[1], _MOST_PER_TOKEN):
    raise ValueError(f'k should be 1 to {min(logits.shape[1], _MOST_PER_TOKEN)}, got {k}.')
  if logits.shape[0] * k > _MOST:
    raise ValueError('Only support up to 2^31 - 1 pairs of a token and an expert.')
  if mask is None:
    logits, = _move(logits)
  else:
    mask = as_tensor(mask)
    if mask.dtype != torch.bool or tuple(mask.shape) != (logits.shape[0],):
      raise ValueError(f'mask should be a bool for each of the {logits.shape[0]} tokens, got {mask.dtype} {tuple(mask.shape)}.')
    logits, mask = _move(logits, mask)
  if _differentiable('expert_topk', logits):
    return _ExpertTopk.run(logits, mask, int(k), bool(normalize))
  if _transforms_active():
    return _Launch.apply('expert_topk', _topk, logits, mask, int(k), bool(normalize))
  return _topk(logits, mask, int(k), bool(normalize))


# ---- expert_sort ------------------------------------------------------------------------------------------------------
def _sort(experts, num_experts):
  pairs, device = experts.numel(), experts.device
  indptr = torch.empty(num_experts + 1, dtype=torch.int32, device=device)
  order = torch.empty(pairs, dtype=torch.int32, device=device)
  position = torch.empty(experts.shape, dtype=torch.int32, device=device)
  room = _lib.expert_sort_scratch_bytes(pairs, num_experts)
  scratch = torch.empty(room // 4, dtype=torch.int32, device=device) if room else indptr  # (not used)
  opaque = _lib.build_expert_descriptor(pairs, 1, num_experts, 0, 0, 0, 0)
  _call('expert_sort', [experts, indptr, order, position, scratch], opaque)
  return indptr, order, position


def expert_sort(experts, *, num_experts: int):
  """Sorts pairs of a token and an expert by expert, in the pairs' order within one.

  experts  (tokens, k) or (pairs,) int32 | uint32; what is outside [0, num_experts) is dropped
  returns  ``(indptr, order, position)``, int32: expert ``e`` has the rows ``indptr[e]`` to ``indptr[e + 1] - 1``; row ``r``
           holds pair ``order[r]`` (pairs are numbered row by row), -1 from row ``indptr[num_experts]`` on; pair ``p`` has row
           ``position.reshape(-1)[p]``, -1 where it was dropped.  ``position`` has the shape of ``experts``."""
  experts = as_tensor(experts)
  _check_index('experts', experts, 1 if experts.ndim == 1 else 2)
  _check_experts(num_experts)
  if experts.numel() > _MOST:
    raise ValueError('Only support up to 2^31 - 1 pairs of a token and an expert.')
  experts, = _move(experts)
  if _transforms_active():
    return _Launch.apply('expert_sort', _sort, experts, num_experts)
  return _sort(experts, num_experts)


# ---- expert_dispatch, expert_combine ----------------------------------------------------------------------------------
def _pairs_opaque(position, width, flags=0):
  return _lib.build_expert_descriptor(position.shape[0], position.shape[1], 1, 0, width, 0, flags)


def _dispatch(tokens, order, position):
  rows = torch.empty((order.shape[0], tokens.shape[1]), dtype=tokens.dtype, device=tokens.device)
  _call('expert_dispatch' + _TYPE_NAME[tokens.dtype], [tokens, order, position, rows],
        _pairs_opaque(position, tokens.shape[1]))
  return rows


def _dispatch_gradient(ct, order, position):
  grad = torch.empty((position.shape[0], ct.shape[1]), dtype=ct.dtype, device=ct.device)
  _call('expert_dispatch_gradient' + _TYPE_NAME[ct.dtype], [ct.contiguous(), order, position, grad],
        _pairs_opaque(position, ct.shape[1]))
  return grad


@_inside_transforms
class _ExpertDispatch(_Operator):
  """The cotangent of a token is the sum of its rows' cotangents."""
  name = 'expert_dispatch'
  launch = staticmethod(_dispatch)

  @staticmethod
  def keep(ctx, inputs, output):
    ctx.save_for_backward(*inputs[1:])
    ctx.set_materialize_grads(False)

  @staticmethod
  def backward(ctx, ct):
    if ct is None:
      return None, None, None
    return _gradient('expert_dispatch', _dispatch_gradient, ct, *ctx.saved_tensors), None, None


def expert_dispatch(tokens, order, position):
  """The tokens' rows in the order of the experts: ``rows[position[t, i]] = tokens[t]``.

  tokens    (tokens, width) float32 | float16 | bfloat16
  order     (tokens * k,) and  position (tokens, k), as ``expert_sort`` gives them (k up to 64)
  returns   (tokens * k, width): rows that no pair leads to (those behind the last expert's) are zero.

  A pair counts only where the two arrays answer each other, ``order[position[t, i]] == t * k + i``."""
  tokens, order, position = as_tensor(tokens), as_tensor(order), as_tensor(position)
  _check_values('tokens', tokens, 2)
  _check_pairs(order, position, tokens.shape[0])
  tokens, order, position = _move(tokens, order, position)
  if _differentiable('expert_dispatch', tokens):
    return _ExpertDispatch.run(tokens, order, position)
  if _transforms_active():
    return _Launch.apply('expert_dispatch', _dispatch, tokens, order, position)
  return _dispatch(tokens, order, position)


def _combine(rows, weights, order, position):
  out = torch.empty((position.shape[0], rows.shape[1]), dtype=rows.dtype, device=rows.device)
  _call('expert_combine' + _TYPE_NAME[rows.dtype], [rows, weights, order, position, out],
        _pairs_opaque(position, rows.shape[1]))
  return out


def _combine_gradient(ct, rows, weights, order, position, want_rows, want_weights):
  d_rows = torch.empty_like(rows) if want_rows else None
  d_weights = torch.empty_like(weights) if want_weights else None
  opaque = _pairs_opaque(position, rows.shape[1], (_D_ROWS if want_rows else 0) | (_D_WEIGHTS if want_weights else 0))
  _call('expert_combine_gradient' + _TYPE_NAME[rows.dtype],
        [rows, weights, order, position, ct.contiguous(), d_rows if want_rows else rows, d_weights if want_weights else weights],
        opaque)
  return d_rows, d_weights


@_inside_transforms
class _ExpertCombine(_Operator):
  """The cotangent of a row is its token's times the pair's weight, that of the weight their inner product with the row."""
  name = 'expert_combine'
  launch = staticmethod(_combine)

  @staticmethod
  def keep(ctx, inputs, output):
    ctx.save_for_backward(*inputs)
    ctx.set_materialize_grads(False)

  @staticmethod
  def backward(ctx, ct):
    wanted = ctx.needs_input_grad[:2]
    if ct is None or not any(wanted):
      return None, None, None, None
    return _gradient('expert_combine', _combine_gradient, ct, *ctx.saved_tensors, *wanted) + (None, None)


def expert_combine(rows, weights, order, position):
  """The experts' rows put together for every token: ``out[t] = sum over i of weights[t, i] * rows[position[t, i]]``.

  rows      (tokens * k, width) float32 | float16 | bfloat16, sorted by expert
  weights   (tokens, k) float32, as ``expert_topk`` gives them
  order, position   as ``expert_sort`` gives them
  returns   (tokens, width) of the rows' type; the sum is held in 32 bits.

  Pairs that were dropped contribute nothing, whatever stands in their weight, and have gradient 0; a token without any is
  zero."""
  rows, weights, order, position = as_tensor(rows), as_tensor(weights), as_tensor(order), as_tensor(position)
  _check_values('rows', rows, 2)
  _check_pairs(order, position, position.shape[0] if position.ndim == 2 else 0)
  if weights.dtype != torch.float32:
    raise TypeError(f'weights should be float32, got {weights.dtype}.')
  if weights.shape != position.shape:
    raise ValueError(f'weights should have the shape of position, got {tuple(weights.shape)} != {tuple(position.shape)}.')
  if rows.shape[0] != order.shape[0]:
    raise ValueError(f'rows should have a row for each entry of order, got {rows.shape[0]} != {order.shape[0]}.')
  rows, weights, order, position = _move(rows, weights, order, position)
  if _differentiable('expert_combine', rows, weights):
    return _ExpertCombine.run(rows, weights, order, position)
  if _transforms_active():
    return _Launch.apply('expert_combine', _combine, rows, weights, order, position)
  return _combine(rows, weights, order, position)


# ---- expert_matmul ----------------------------------------------------------------------------------------------------
def _matmul(rows, stored, indptr, out_major):
  """rows @ weight by expert; ``stored`` is the weight as it lies in memory, (experts, out, inner) where ``out_major``."""
  n, inner = rows.shape
  experts, out_width = stored.shape[0], stored.shape[1] if out_major else stored.shape[2]
  out = torch.empty((n, out_width), dtype=rows.dtype, device=rows.device)
  parts = _lib.expert_matmul_parts(n, experts, inner, out_width, rows.element_size())
  scratch = out if parts == 1 else torch.empty((parts, n, out_width), dtype=torch.float32, device=rows.device)
  opaque = _lib.build_expert_descriptor(0, parts, experts, n, inner, out_width, _OUT_MAJOR if out_major else 0)
  _call('expert_matmul' + _TYPE_NAME[rows.dtype], [rows, stored, indptr, out, scratch], opaque)
  return out


def _matmul_gradient(ct, rows, indptr, shape, out_major):
  """The cotangent of the weight as it lies in memory, ``shape``."""
  d_stored = torch.empty(shape, dtype=rows.dtype, device=rows.device)
  parts = _lib.expert_matmul_gradient_parts(rows.shape[0], shape[0], rows.shape[1], ct.shape[1], rows.element_size())
  scratch = d_stored if parts == 1 else torch.empty((parts,) + shape, dtype=torch.float32, device=rows.device)
  opaque = _lib.build_expert_descriptor(0, parts, shape[0], rows.shape[0], rows.shape[1], ct.shape[1],
                                        _OUT_MAJOR if out_major else 0)
  _call('expert_matmul_gradient' + _TYPE_NAME[rows.dtype], [rows, ct.contiguous(), indptr, d_stored, scratch], opaque)
  return d_stored


@_inside_transforms
class _ExpertMatmul(_Operator):
  """The rows' cotangent is the product with the transposed weights, the weights' is rows_e^T @ ct_e for every expert."""
  name = 'expert_matmul'
  launch = staticmethod(_matmul)

  @staticmethod
  def keep(ctx, inputs, output):
    ctx.out_major = inputs[3]
    ctx.save_for_backward(*inputs[:3])
    ctx.set_materialize_grads(False)

  @staticmethod
  def backward(ctx, ct):
    if ct is None:
      return None, None, None, None
    rows, stored, indptr = ctx.saved_tensors
    ct = ct.contiguous()
    d_rows = d_stored = None
    if ctx.needs_input_grad[0]:
      d_rows = _gradient('expert_matmul', _matmul, ct, stored, indptr, not ctx.out_major)
    if ctx.needs_input_grad[1]:
      d_stored = _gradient('expert_matmul', _matmul_gradient, ct, rows, indptr, tuple(stored.shape), ctx.out_major)
    return d_rows, d_stored, None, None


def expert_matmul(rows, weight, indptr):
  """Every expert's rows times its matrix: ``out[r] = rows[r] @ weight[e]`` for ``indptr[e] <= r < indptr[e + 1]``.

  rows      (rows, inner) float32 | float16 | bfloat16, sorted by expert
  weight    (experts, inner, out) of the rows' type, up to 1,024 experts.  Both storages are taken as they are: contiguous,
            or the transposed view of a contiguous (experts, out, inner); its gradient is stored the same way.
  indptr    (experts + 1,) int32 | uint32, not decreasing from 0, as ``expert_sort`` gives it
  returns   (rows, out); rows from ``indptr[experts]`` on are zero.  Sums are held in 32 bits.

  indptr is trusted to split the rows as said, as index arrays are elsewhere in the package; whatever it holds, nothing
  outside the arrays is touched."""
  rows, weight, indptr = as_tensor(rows), as_tensor(weight), as_tensor(indptr)
  _check_values('rows', rows, 2)
  _check_values('weight', weight, 3)
  _check_index('indptr', indptr, 1)
  if weight.dtype != rows.dtype:
    raise TypeError(f'The types of rows and weight should be the same. But we got {rows.dtype} != {weight.dtype}.')
  _check_experts(weight.shape[0])
  if weight.shape[1] != rows.shape[1]:
    raise ValueError(f'Shape mismatch, rows {tuple(rows.shape)} @ weight {tuple(weight.shape)}.')
  if indptr.shape[0] != weight.shape[0] + 1:
    raise ValueError(f'indptr should have experts + 1 = {weight.shape[0] + 1} entries, got {indptr.shape[0]}.')
  out_major = not weight.is_contiguous() and weight.transpose(1, 2).is_contiguous()
  rows, stored, indptr = _move(rows, weight.transpose(1, 2) if out_major else weight, indptr)
  if _differentiable('expert_matmul', rows, stored):
    return _ExpertMatmul.run(rows, stored, indptr, out_major)
  if _transforms_active():
    return _Launch.apply('expert_matmul', _matmul, rows, stored, indptr, out_major)
  return _matmul(rows, stored, indptr, out_major)
