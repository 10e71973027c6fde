"""The device memory that a call of linear attention takes, as the caching allocator counts it: whole blocks, whatever
blocks the program has left it with before."""

import pytest
import torch

from test_state_operators_gpu import DEV, _Call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rest", [0, 512, 300 << 10, (1 << 20) - 512, 1 << 20])
@pytest.mark.parametrize("nq,nkv,d,lens", [(2, 1, 128, [2500]), (8, 8, 64, [900, 300])])
def test_a_call_takes_no_more_than_is_stated_whatever_lies_in_the_cache(dtype, rest, nq, nkv, d, lens):
  from miniinfer_amd.kernels import ops
  c = _Call(dtype, nq, nkv, d, lens, seed=9)
  qkv, state, rows, cu, g = c.device()
  out = torch.empty(c.T, nq * d, dtype=dtype, device=DEV)
  call = lambda: ops.linear_attention(*c.parts(qkv), nq, nkv, d, out, state, rows, cu, g, c.scale)
  stats = torch.cuda.memory_stats
  call()
  torch.cuda.synchronize()
  torch.cuda.reset_peak_memory_stats()
  before = stats()["requested_bytes.all.current"]
  call()
  asked = stats()["requested_bytes.all.peak"] - before
  stated = ops.linear_attention_workspace(c.T, len(lens), nkv, d, out.element_size(), ops.compute_units())
  assert 1 << 20 < asked <= stated
  # a free block that is larger by `rest`, between two that are held
  torch.cuda.empty_cache()
  held = [torch.empty(asked, dtype=torch.uint8, device=DEV)]
  block = torch.empty(asked + rest, dtype=torch.uint8, device=DEV)
  held.append(torch.empty(asked, dtype=torch.uint8, device=DEV))
  del block
  torch.cuda.synchronize()
  torch.cuda.reset_peak_memory_stats()
  before = torch.cuda.memory_allocated()
  call()
  assert asked <= torch.cuda.max_memory_allocated() - before <= stated
