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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_call_allocates_no_more_than_is_stated(dtype):
  from miniinfer_amd.kernels import ops
  for nq, nkv, d, lens in ((2, 1, 128, [2500]), (8, 8, 64, [900, 300]), (2, 2, 256, [700, 700, 5])):
    c = _Call(dtype, nq, nkv, d, lens, seed=9)
    qkv, state, rows, cu, g = c.device()
    out = torch.empty(c.T, nq * d, dtype=dtype, device=DEV)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.linear_attention(*c.parts(qkv), nq, nkv, d, out, state, rows, cu, g, c.scale)
    room = ops.linear_attention_workspace(c.T, len(lens), nkv, d, out.element_size(), ops.compute_units())
    assert 0 < torch.cuda.max_memory_allocated() - before <= room + 512          # (the allocator's grain)


def test_the_engine_leaves_room_for_it(tmp_path):
  from miniinfer_amd import LLMEngine
  from miniinfer_amd.kernels import ops
  from test_linear_attention_model_gpu import _write
  _write(str(tmp_path / "m"), "bfloat16")
  with LLMEngine(model=str(tmp_path / "m"), dtype="bfloat16", page_size=16, num_pages=40, max_num_seqs=8,
                 tune_products=False) as eng:
    counted = eng.activation_bytes()
    stated = eng.model.largest_workspace_bytes(eng.config.max_num_batched_tokens, 8)
    eng.model.largest_workspace_bytes = lambda *a: 0
    assert stated > 0 and counted - eng.activation_bytes() == stated
