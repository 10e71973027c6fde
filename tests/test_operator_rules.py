"""How linear attention cuts its work, and calls that beam search and the operators behind it turn down on the host (no
GPU)."""

from types import SimpleNamespace

import pytest
import torch

from miniinfer_amd.cache.manager import CacheManager
from miniinfer_amd.engine.beam_search import BeamSearcher, Search
from miniinfer_amd.kernels import ops
from miniinfer_amd.kernels.ops import KernelError
from miniinfer_amd.parts import FixedState
from miniinfer_amd.sampling import BeamSearchParams


@pytest.mark.parametrize("nkv,d,itemsize,columns,each", [(1, 8, 2, 64, 2), (12, 64, 4, 64, 2), (8, 128, 2, 128, 1),
                                                         (8, 128, 4, 128, 1), (4, 256, 2, 128, 1), (4, 256, 4, 64, 1),
                                                         (700, 128, 2, 128, 1)])
def test_segments_are_whole_chunks_and_fill_the_chip_once(nkv, d, itemsize, columns, each):
  for tokens in (0, 1, 63, 64, 65, 129, 1000, 2048, 9001, 32768, 1 << 20):
    for requests in (1, 2, 7, 24, 300):
      for longest in {min(tokens, x) for x in (1, 64, 300, 5000, 1 << 20)}:
        s = ops.linear_attention_segment(tokens, requests, longest, nkv, d, itemsize)
        assert s % 64 == 0 and s >= 0
        if s == 0:
          continue
        assert longest > 2 * s                      # a cut request has three segments and more
        # at most one workgroup for each place on the chip, short last segments counted, unless segments are as short
        # or as long as they may be
        places = 256 * each // (nkv * -(-d // columns))
        units = tokens // s + requests
        assert s == 64 or units <= places + 1 or s == -(-tokens // (64 * max(1, places // 2))) * 64
  places = 256 * each // (nkv * -(-d // columns))           # (where the heads alone fill the chip nothing is cut)
  assert (ops.linear_attention_segment(1 << 20, 1, 1 << 20, nkv, d, itemsize) > 0) == (places > 2)


def test_segments_at_the_measured_sizes():
  rule = ops.linear_attention_segment
  assert rule(2048, 1, 2048, 8, 128) == 64 and rule(32768, 1, 32768, 8, 128) == 1024
  assert rule(8192, 1, 8192, 32, 64) == 512 and rule(8192, 8, 2500, 8, 128) == 384
  assert rule(9001, 24, 950, 12, 80) == 0 and rule(100, 1, 100, 8, 128) == 0 and rule(130, 1, 130, 8, 128) == 64


@pytest.mark.parametrize("alias", ["q", "k", "v"])
def test_linear_attention_refuses_to_write_over_its_inputs(alias):
  a = {n: torch.zeros(3, 16) for n in ("q", "k", "v", "out")}
  a["out"] = a[alias]
  common = (1, 1, 16, a["out"], torch.zeros(2, 1, 16, 16))
  with pytest.raises(KernelError, match="shares memory"):
    ops.linear_attention(a["q"], a["k"], a["v"], *common, torch.zeros(1, dtype=torch.int32),
                         torch.zeros(2, dtype=torch.int32), torch.zeros(1), 1.0)
  with pytest.raises(KernelError, match="shares memory"):
    ops.linear_attention_step(a["q"], a["k"], a["v"], *common, torch.zeros(3, dtype=torch.int32), torch.zeros(1), 1.0)


def test_move_rows_refuses_a_buffer_twice():
  t, i = torch.zeros(2, 5, 4), torch.zeros(1, dtype=torch.int32)
  with pytest.raises(KernelError, match="twice"):
    ops.move_rows([t, torch.zeros(2, 5), t], i, i)


@pytest.mark.parametrize("tokens,slots,fits", [(64, 8, True), (4, 8, True), (3, 8, False), (64, 3, False)])
def test_a_search_needs_a_slot_and_a_token_of_a_step_for_each_beam(tokens, slots, fits):
  need = FixedState(shape=(1, 2, 2), dtype=torch.float32)
  cache = CacheManager([need], page_size=4, num_pages=8, max_requests=slots, max_model_len=16,
                       dtype=torch.float32, device="cpu")
  engine = SimpleNamespace(cache=cache, runner=None, scheduler=SimpleNamespace(eos_token_ids=[]),
                           config=SimpleNamespace(max_num_batched_tokens=tokens))
  searcher = BeamSearcher(engine, BeamSearchParams(num_beams=4, max_tokens=2))
  search = Search(0, [1, 2, 3], 2)
  assert searcher._fits([search]) is fits
  if not fits:
    with pytest.raises(ValueError, match="does not fit"):
      searcher.run([[1, 2, 3]])


@pytest.mark.parametrize("eos,stop,ignore,most", [([], [], False, 64), ([7], [], False, 32), ([7, 9], [], False, 21),
                                                  ([7, 9], [9, 11, 12], False, 12), ([7, 9], [], True, 64)])
def test_a_search_has_candidates_for_every_beam_whatever_ends(eos, stop, ignore, most):
  """Of the candidates, every beam may bring every token that ends it; num_beams others have to be left."""
  engine = SimpleNamespace(cache=None, runner=None, config=None, scheduler=SimpleNamespace(eos_token_ids=eos))
  new = lambda n: BeamSearcher(engine, BeamSearchParams(num_beams=n, stop_token_ids=stop, ignore_eos=ignore))
  assert new(most).count <= ops.BEAM_MAX_COUNT
  assert new(most).count >= most * (1 + len(set(stop) | (set() if ignore else set(eos))))
  with pytest.raises(ValueError, match="at most"):
    new(most + 1)


@pytest.mark.parametrize("nkv,d,itemsize", [(1, 8, 2), (12, 64, 4), (32, 64, 2), (8, 128, 2), (12, 80, 2), (4, 256, 4), (700, 128, 2)])
def test_the_stated_workspace_holds_every_call(nkv, d, itemsize):
  """For all token and request counts up to those it is stated for."""
  for most_tokens in (1, 128, 129, 1000, 8192, 40000):
    for most_requests in (1, 5, 64, 256):
      room = ops.linear_attention_workspace(most_tokens, most_requests, nkv, d, itemsize)
      for tokens in {most_tokens, most_tokens // 2, most_tokens // 3, min(most_tokens, 200)}:
        for requests in {1, most_requests, max(1, most_requests // 2)}:
          segment = ops.linear_attention_segment(tokens, requests, tokens, nkv, d, itemsize)
          if segment:
            assert 4 * (tokens // segment + requests) * nkv * d * d <= room


def test_parts_state_their_workspaces():
  from miniinfer_amd.parts import Part

  class Child(Part):
    def __init__(self, each):
      self.each = each

    def workspace_bytes(self, tokens, requests):
      return self.each * tokens + requests

  class Parent(Part):
    def children(self):
      return [("a", Child(3)), ("b", Child(5))]

  assert Parent().largest_workspace_bytes(7, 2) == 37 and Part().largest_workspace_bytes(7, 2) == 0
