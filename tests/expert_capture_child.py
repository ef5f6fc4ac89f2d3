"""Run as a process of its own by tests/test_gpu_experts.py: the expert operators captured into a HIP graph COLD, their first
calls in the process being the captured ones (library, modules and kernel attributes are looked up under the capture), on a
stream that nothing has used.  Every replay is compared with the eager result.  Exit code 0 = every check passed."""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

import brainpylib_amd as bpl  # noqa: E402


def main():
  torch.manual_seed(0)
  tokens, experts, width, hidden, k = 3000, 16, 264, 520, 4
  x = torch.randn(tokens, width, device="cuda").to(torch.bfloat16)
  logits = torch.randn(tokens, experts, device="cuda")
  up = torch.randn(experts, width, hidden, device="cuda").to(torch.bfloat16)
  down = torch.randn(experts, width, hidden, device="cuda").to(torch.bfloat16).transpose(1, 2)  # stored out-major
  few = torch.randn(2, 4096, device="cuda")
  long = torch.randn(experts, 4096, 96, device="cuda")
  ends = torch.tensor([0] + [1] * 5 + [2] * 11, dtype=torch.int32, device="cuda")

  def step():
    weights, chosen = bpl.expert_topk(logits, k=k)
    indptr, order, position = bpl.expert_sort(chosen, num_experts=experts)
    rows = bpl.expert_matmul(bpl.expert_dispatch(x, order, position), up, indptr)
    out = bpl.expert_combine(bpl.expert_matmul(rows, down, indptr), weights, order, position)
    return out, order, bpl.expert_matmul(few, long, ends)  # (the last is split over its inner dimension)

  torch.cuda.synchronize()
  g = torch.cuda.CUDAGraph()
  with torch.cuda.graph(g, stream=torch.cuda.Stream()):
    captured = step()
  for i in range(3):
    logits.copy_(torch.randn(tokens, experts, device="cuda"))
    few.copy_(torch.randn(2, 4096, device="cuda"))
    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    for t in captured:
      t.zero_()
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(captured, want):
      assert torch.equal(a, b), i
  print("captured cold: ok", flush=True)


if __name__ == "__main__":
  main()
