"""The fixed-size states count when the cache is sized: `storage_bytes` is what the manager allocates, and the pages get
what the states leave (on the CPU)."""

from types import SimpleNamespace

import pytest
import torch

from miniinfer_amd.cache import CacheManager
from miniinfer_amd.engine.llm_engine import LLMEngine
from miniinfer_amd.parts import FixedState, PagedKV

GB = 1 << 30


@pytest.mark.parametrize("needs", [
  [FixedState((3,), torch.float32)],
  [PagedKV(2, 8), FixedState((2, 4, 4), torch.float32), PagedKV(2, 8), FixedState((2, 4, 4), torch.float32)],
  [FixedState((5, 7)), PagedKV(1, 16, page_size=32, dtype=torch.float32), None, PagedKV(2, 8, window=20, page_size=4),
   FixedState((3,), torch.float64)],
  [PagedKV(2, 8)],
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("requests", [1, 6])
def test_storage_bytes_are_what_is_allocated(needs, dtype, requests):
  m = CacheManager(needs, page_size=8, num_pages=20, max_requests=requests, max_model_len=64, dtype=dtype, device="cpu",
                   max_step_tokens=40)
  held = [t for g in m.paged for t in (g.k, g.v)] + [s.state for s in m.states]
  assert CacheManager.storage_bytes(needs, 8, 20, requests, 40, dtype) == sum(t.numel() * t.element_size() for t in held)
  assert CacheManager.state_bytes(needs, requests, dtype) == sum(s.state.numel() * s.state.element_size() for s in m.states)


def _pages(monkeypatch, needs, free, activations=GB, requests=256, max_model_len=32768):
  monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (free, 288 * GB))
  engine = SimpleNamespace(config=SimpleNamespace(max_num_seqs=requests, page_size=16, max_num_batched_tokens=8192,
                                                  gpu_memory_utilization=1.0),
                           max_model_len=max_model_len, dtype=torch.bfloat16, device="cuda", activation_bytes=lambda: activations)
  return LLMEngine._pages_from_memory(engine, needs)


def test_the_pages_get_what_the_states_leave(monkeypatch):
  """24 layers of 8 heads of 128 for 256 requests: 3 GiB of states."""
  linear, paged = FixedState((8, 128, 128), torch.float32), PagedKV(8, 128)
  needs = [linear] * 24 + [paged] * 4
  states = CacheManager.state_bytes(needs, 256, torch.bfloat16)
  assert states == 24 * 257 * 8 * 128 * 128 * 4 and states > 3 * GB
  free = 20 * GB
  pages = _pages(monkeypatch, needs, free)
  assert 1 < pages < 256 * 2048                      # bound by memory
  size = lambda n: CacheManager.storage_bytes(needs, 16, n, 256, 8192, torch.bfloat16)
  assert size(pages) <= free - GB < size(pages + 1)
  alone = _pages(monkeypatch, [paged] * 4, free)
  assert (alone - pages) * CacheManager.bytes_per_page(needs, 16, torch.bfloat16) == pytest.approx(states, rel=1e-3)


def test_states_that_do_not_fit_are_an_error(monkeypatch):
  linear, paged = FixedState((8, 128, 128), torch.float32), PagedKV(8, 128)
  for needs in ([linear] * 24 + [paged], [linear] * 24):
    with pytest.raises(RuntimeError, match="not enough device memory.*states of 256 requests 3084 MiB"):
      _pages(monkeypatch, needs, 4 * GB)
  assert _pages(monkeypatch, [linear] * 24, 5 * GB) == 256 * 2048          # (no layer is paged: the pages are only counted)
  assert _pages(monkeypatch, [linear] * 24, 5 * GB, requests=1, max_model_len=16) == 1
  assert _pages(monkeypatch, [], 2 * GB) == 256 * 2048
