"""What the expert operators refuse, on the CPU: the wrappers before any device is needed, the targets before any launch;
and the plain implementations that the GPU tests compare with, against each other."""
import ctypes
import struct

import numpy as np
import pytest
import torch

import brainpylib_amd as bpl
import experts_plain as plain
from brainpylib_amd import _lib

TYPES = ("float", "half", "bfloat16")


def ints(*shape):
  return torch.zeros(shape, dtype=torch.int32)


def test_the_operators_are_exported():
  for name in ("expert_topk", "expert_sort", "expert_dispatch", "expert_combine", "expert_matmul"):
    assert name in bpl.__all__ and callable(getattr(bpl, name))
  names = set(_lib.target_names())
  assert "expert_sort" in names
  for name in ("topk", "topk_gradient", "dispatch", "dispatch_gradient", "combine", "combine_gradient", "matmul",
               "matmul_gradient"):
    for t in TYPES:
      assert "expert_%s_%s" % (name, t) in names


def test_descriptor():
  from brainpylib_amd import gpu_ops
  want = struct.pack("<7I", 1, 2, 3, 4, 5, 6, 7)
  assert _lib.build_expert_descriptor(1, 2, 3, 4, 5, 6, 7) == want
  assert gpu_ops.build_expert_descriptor(1, 2, 3, 4, 5, 6, 7) == want


def test_sort_scratch_is_for_long_lists_only():
  assert _lib.expert_sort_scratch_bytes(0, 8) == 0
  assert _lib.expert_sort_scratch_bytes(64, 1024) == 0
  assert _lib.expert_sort_scratch_bytes(1 << 20, 64) >= 4 * 65 * 2
  assert _lib.expert_sort_scratch_bytes(2 ** 31 - 1, 1024) < 1 << 26


def test_gradient_is_split_where_results_are_few():
  parts = _lib.expert_matmul_gradient_parts
  assert parts(100, 8, 2048, 2048, 2) == 1 and parts(0, 8, 64, 64, 4) == 1 and parts(100_000, 4, 0, 64, 4) == 1
  assert parts(1 << 20, 64, 4096, 4096, 2) == 1
  for width, out in ((64, 64), (30, 700), (700, 30), (1, 5), (5, 1)):
    for element in (2, 4):
      assert 1 < parts(100_000, 2, width, out, element) <= 64


def test_product_is_split_where_results_are_few_and_the_inner_dimension_is_long():
  parts = _lib.expert_matmul_parts
  assert parts(0, 8, 4096, 64, 2) == 1 and parts(2, 8, 0, 64, 2) == 1 and parts(2, 8, 1024, 64, 2) == 1
  assert parts(4096, 8, 4096, 4096, 2) == 1 and parts(512, 64, 4096, 4096, 4) == 1
  for rows, experts, width, out in ((2, 8, 4096, 264), (3, 5, 4100, 70), (40, 2, 6001, 33), (1, 1024, 2 ** 20, 1)):
    for element in (2, 4):
      assert 1 < parts(rows, experts, width, out, element) <= 16


@pytest.mark.parametrize("call, error", [
  (lambda: bpl.expert_topk(torch.zeros(2, 4, dtype=torch.float64), k=1), TypeError),
  (lambda: bpl.expert_topk(torch.zeros(2, 4, dtype=torch.int32), k=1), TypeError),
  (lambda: bpl.expert_topk(torch.zeros(4), k=1), ValueError),
  (lambda: bpl.expert_topk(torch.zeros(2, 4), k=0), ValueError),
  (lambda: bpl.expert_topk(torch.zeros(2, 4), k=5), ValueError),
  (lambda: bpl.expert_topk(torch.zeros(2, 128), k=65), ValueError),
  (lambda: bpl.expert_topk(torch.zeros(2, 1025), k=2), ValueError),
  (lambda: bpl.expert_topk(torch.zeros(2, 0), k=1), ValueError),
  (lambda: bpl.expert_topk(torch.zeros(2, 4), k=1, mask=torch.ones(3, dtype=torch.bool)), ValueError),
  (lambda: bpl.expert_topk(torch.zeros(2, 4), k=1, mask=torch.ones(2)), ValueError),
  (lambda: bpl.expert_sort(torch.zeros(4, 2, dtype=torch.int64), num_experts=4), ValueError),
  (lambda: bpl.expert_sort(ints(2, 2, 2), num_experts=4), ValueError),
  (lambda: bpl.expert_sort(ints(4, 2), num_experts=0), ValueError),
  (lambda: bpl.expert_sort(ints(4, 2), num_experts=1025), ValueError),
  (lambda: bpl.expert_dispatch(torch.zeros(4, 8, dtype=torch.float64), ints(8), ints(4, 2)), TypeError),
  (lambda: bpl.expert_dispatch(torch.zeros(4), ints(8), ints(4, 2)), ValueError),
  (lambda: bpl.expert_dispatch(torch.zeros(5, 8), ints(8), ints(4, 2)), ValueError),
  (lambda: bpl.expert_dispatch(torch.zeros(4, 8), ints(7), ints(4, 2)), ValueError),
  (lambda: bpl.expert_dispatch(torch.zeros(4, 8), ints(8), ints(8)), ValueError),
  (lambda: bpl.expert_dispatch(torch.zeros(4, 8), ints(8).long(), ints(4, 2)), ValueError),
  (lambda: bpl.expert_dispatch(torch.zeros(1, 8), ints(65), ints(1, 65)), ValueError),
  (lambda: bpl.expert_combine(torch.zeros(8, 8), torch.zeros(4, 2, dtype=torch.bfloat16), ints(8), ints(4, 2)), TypeError),
  (lambda: bpl.expert_combine(torch.zeros(8, 8), torch.zeros(4, 3), ints(8), ints(4, 2)), ValueError),
  (lambda: bpl.expert_combine(torch.zeros(7, 8), torch.zeros(4, 2), ints(8), ints(4, 2)), ValueError),
  (lambda: bpl.expert_combine(torch.zeros(8, 8), torch.zeros(4, 2), ints(8), ints(8)), ValueError),
  (lambda: bpl.expert_matmul(torch.zeros(8, 4), torch.zeros(2, 4, 3, dtype=torch.bfloat16), ints(3)), TypeError),
  (lambda: bpl.expert_matmul(torch.zeros(8, 4, dtype=torch.float64), torch.zeros(2, 4, 3, dtype=torch.float64), ints(3)), TypeError),
  (lambda: bpl.expert_matmul(torch.zeros(8, 4), torch.zeros(2, 5, 3), ints(3)), ValueError),
  (lambda: bpl.expert_matmul(torch.zeros(8, 4), torch.zeros(4, 3), ints(3)), ValueError),
  (lambda: bpl.expert_matmul(torch.zeros(8, 4), torch.zeros(2, 4, 3), ints(2)), ValueError),
  (lambda: bpl.expert_matmul(torch.zeros(8, 4), torch.zeros(2, 4, 3), ints(3).long()), ValueError),
  (lambda: bpl.expert_matmul(torch.zeros(8, 4), torch.zeros(0, 4, 3), ints(1)), ValueError),
])
def test_refused_arguments(call, error):
  with pytest.raises(error):
    call()


@pytest.mark.parametrize("name", ["expert_topk_half", "expert_topk_gradient_float", "expert_sort", "expert_dispatch_bfloat16",
                                  "expert_combine_float", "expert_combine_gradient_half", "expert_matmul_bfloat16",
                                  "expert_matmul_gradient_float"])
@pytest.mark.parametrize("fields, why", [
  ((4, 2, 0, 8, 8, 8, 0), "experts"), ((4, 2, 1025, 8, 8, 8, 0), "experts"), ((4, 65, 100, 8, 8, 8, 0), "experts a token"),
  ((2 ** 31 - 1, 2, 4, 8, 8, 8, 0), "2^31"), ((4, 2, 4, 2 ** 31, 8, 8, 0), "2^31"), ((4, 2, 4, 8, 2 ** 32 - 1, 8, 0), "2^31"),
  ((4, 2, 4, 8, 8, 2 ** 31, 0), "2^31"),
])
def test_targets_refuse_sizes_beyond_their_limits(name, fields, why, capfd):
  _lib.lib().bpl_clear_error()
  opaque = struct.pack("<7I", *fields)
  _lib.target(name)(None, (ctypes.c_void_p * 8)(), opaque, len(opaque))
  assert name in _lib.last_error() and why in _lib.last_error()
  _lib.lib().bpl_clear_error()


def test_topk_target_refuses_more_places_than_experts(capfd):
  opaque = struct.pack("<7I", 4, 5, 4, 0, 0, 0, 0)
  for name in ("expert_topk_float", "expert_topk_gradient_float"):
    _lib.target(name)(None, (ctypes.c_void_p * 8)(), opaque, len(opaque))
    assert "experts a token" in _lib.last_error()
    _lib.lib().bpl_clear_error()


def test_operators_need_a_device():
  if torch.cuda.is_available():
    pytest.skip("there is a device")
  with pytest.raises(RuntimeError):
    bpl.expert_topk(torch.zeros(2, 4), k=1)


def test_the_plain_choice_and_sort():
  x = np.array([[0.0, 2.0, 2.0, -np.inf], [-np.inf] * 4, [np.nan, 3.0, np.inf, 1.0], [-1.0, -0.0, 0.0, -2.0]])
  w, e = plain.topk(x, 3, True)
  assert e.tolist() == [[1, 2, 0], [-1, -1, -1], [0, 2, 1], [1, 2, 0]]
  assert np.isnan(w[2]).all() and w[1].tolist() == [0, 0, 0] and abs(w[0].sum() - 1) < 1e-15
  indptr, order, position = plain.sort(np.array([[2, 0], [-1, 2], [0, 7]]), 3)
  assert indptr.tolist() == [0, 2, 2, 4] and order.tolist() == [1, 4, 0, 3, -1, -1]
  assert position.tolist() == [[2, 0], [-1, 3], [1, -1]]


@pytest.mark.parametrize("normalize", [True, False])
def test_the_plain_gradient_of_the_choice_against_differences(normalize):
  rng = np.random.default_rng(0)
  x, ct = rng.standard_normal((3, 7)), rng.standard_normal((3, 4))
  w, e = plain.topk(x, 4, normalize)
  grad = plain.topk_gradient(x, w, e, ct, normalize)
  h = 1e-5  # (differences of a smooth function in 64 bits: off by h^2 and 1e-16 / h)
  for t in range(3):
    for j in range(7):
      up, down = x.copy(), x.copy()
      up[t, j] += h
      down[t, j] -= h
      slope = ((plain.topk(up, 4, normalize)[0] - plain.topk(down, 4, normalize)[0]) * ct).sum() / (2 * h)
      assert abs(slope - grad[t, j]) < 1e-8


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["plain", "inference", "parameter", "transform"])
def test_one_element_on_the_host_goes_to_the_device_in_every_type(dtype, kind, monkeypatch):
  # (the meta device stands for a GPU; the copies are told apart by their values' bits)
  from brainpylib_amd import _tensors
  monkeypatch.setattr(_tensors, "_HOST_SCALARS", {})
  device = torch.device("meta")
  with torch.inference_mode(kind == "inference"):
    operands = [torch.full((1, 1), v, dtype=dtype) for v in (1.5, -1.5, 0.0, -0.0, float("nan"))]
  if kind == "parameter":
    operands = [torch.nn.Parameter(t, requires_grad=False) for t in operands]

  def move(x):
    for t in operands:
      moved = _tensors.to_device(t, device)
      assert moved.dtype == dtype and moved.shape == (1, 1) and moved.device == device
      assert _tensors.to_device(t.clone() if kind == "plain" else t, device) is moved
    return x.sum()
  if kind == "transform":
    torch.func.grad(move)(torch.ones(2))
  else:
    move(torch.ones(2))
  assert len(_tensors._HOST_SCALARS) == len(operands)
