"""Linear attention of requests that are walked over whole, chunk by chunk in one workgroup for each head: every number of
query heads to a kv head (the order in which tiles are asked for and waited for follows from it), every kind of tile, rows
that are aligned and rows that are not.  (A longest request stated as one token, which only chooses how the work is cut,
makes any call such a walk.)  References and tolerances: those of `test_state_operators_gpu`."""

import pytest
import torch

from test_state_operators_gpu import DEV, _Call

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1, 64), (4, 2, 64), (3, 1, 16), (1, 1, 80), (4, 2, 96), (1, 1, 128), (2, 1, 128), (3, 1, 128), (5, 1, 128),
          (2, 1, 200), (1, 1, 256), (4, 1, 256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", SHAPES)
def test_whole_walks(dtype, nq, nkv, d):
  for lens in ([330, 1, 197], [128], [64, 192]):
    c = _Call(dtype, nq, nkv, d, lens, seed=len(lens), behind=1)
    out, state = c.run(max_len=1)
    c.check(out, state)
    for _ in range(2):                                  # the same bits again
      again = c.run(max_len=1)
      assert torch.equal(out, again[0]) and torch.equal(state, again[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", [(2, 1, 64), (3, 1, 128), (1, 1, 256)])
def test_whole_walks_over_unaligned_rows(dtype, nq, nkv, d):
  from miniinfer_amd.kernels import ops
  c = _Call(dtype, nq, nkv, d, [150, 70], seed=5)
  qkv, state, rows, cu, g = c.device()
  wide = torch.zeros(c.T, qkv.shape[1] + 3, dtype=dtype, device=DEV)
  wide[:, 1:1 + qkv.shape[1]] = qkv
  out = torch.full((c.T, nq * d), 7.0, dtype=dtype, device=DEV)
  ops.linear_attention(*c.parts(wide[:, 1:1 + qkv.shape[1]]), nq, nkv, d, out, state, rows, cu, g, c.scale, 1)
  c.check(out.cpu(), state.cpu())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", [(1, 1, 64), (4, 2, 128), (2, 1, 256)])
@pytest.mark.parametrize("at", [5, 64, 149])
def test_values_that_are_not_finite_in_whole_walks(dtype, nq, nkv, d, at):
  """They reach their own column of later tokens' outputs and nothing else."""
  c = _Call(dtype, nq, nkv, d, [40, 150, 90], seed=6)
  c.parts(c.qkv)[2][c.cu[1] + at, 3] = float("inf")
  c.parts(c.qkv)[2][c.cu[2] + 7, (nkv - 1) * d + d - 1] = float("nan")
  want, want_state = c.want()
  out, state = c.run(max_len=1)
  ok = want.isfinite()
  assert torch.equal(out.isfinite(), ok) and torch.equal(state.isfinite(), want_state.isfinite())
  # (as a whole: half a step of the output's type, or of a 32-bit sum's some hundred roundings, which mostly cancel)
  assert float((out.double() - want)[ok].norm() / want[ok].norm()) <= max(torch.finfo(dtype).eps / 2, 2e-6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", [(1, 1, 64), (2, 1, 80), (2, 1, 128), (1, 1, 256)])
@pytest.mark.parametrize("segment", [128, 320])
def test_segments_of_several_chunks(dtype, nq, nkv, d, segment, monkeypatch):
  """(Few tokens are cut into single chunks; the length of a segment is the rule's to choose.)"""
  from miniinfer_amd.kernels import ops
  monkeypatch.setattr(ops, "linear_attention_segment", lambda *a, **k: segment)
  c = _Call(dtype, nq, nkv, d, [1000, 2, 0, 641, 320], seed=8, before=2)
  out, state = c.run()
  c.check(out, state)
  again = c.run()
  assert torch.equal(out, again[0]) and torch.equal(state, again[1])
