"""Beam search over a cache with window groups: what it asks the pools for is what its requests come to hold, and prompts
that the cache holds are searched (on the CPU: the steps' page accounting is real, the logits are random)."""

import random
from types import SimpleNamespace

import pytest
import torch

from miniinfer_amd.cache import CacheManager
from miniinfer_amd.engine import beam_search as module
from miniinfer_amd.engine.beam_search import BeamSearcher, Search
from miniinfer_amd.parts import PagedKV
from miniinfer_amd.sampling import BeamSearchParams

VOCAB = 11


class _Runner:
  """Steps that only grow and commit requests, and note the most pages of each group that were held at once."""

  def __init__(self, cache, budget, seed):
    self.cache, self.budget = cache, budget
    self.generator = torch.Generator().manual_seed(seed)
    self.peak = [0] * len(cache.paged)

  def note(self):
    self.peak = [max(p, g.pool.num_held) for p, g in zip(self.peak, self.cache.paged)]

  def step(self, entries):
    assert sum(len(e.tokens) for e in entries) <= self.budget
    for e in entries:
      self.cache.grow(e.req, self.cache.length(e.req) + len(e.tokens))
    self.note()
    for e in entries:
      self.cache.commit(e.req, self.cache.length(e.req) + len(e.tokens))
    return torch.randn(sum(len(e.want) for e in entries), VOCAB, generator=self.generator)


def _beam_select(logits, scores, num_beams, count, **_):
  p = torch.log_softmax(logits.double(), -1) + scores.double()[:, None]
  value, index = p.view(-1, num_beams * VOCAB).sort(dim=-1, descending=True, stable=True)
  value, index = value[:, :count], index[:, :count]
  return value, index // VOCAB, index % VOCAB


def _searcher(monkeypatch, needs, params, seed=0, page_size=4, num_pages=1 << 12, requests=4, budget=32, max_model_len=1 << 16):
  monkeypatch.setattr(module.ops, "beam_select", _beam_select)
  cache = CacheManager(needs, page_size=page_size, num_pages=num_pages, max_requests=requests, max_model_len=max_model_len,
                       dtype=torch.float32, device="cpu", allocate=False, max_step_tokens=budget)
  engine = SimpleNamespace(cache=cache, runner=_Runner(cache, budget, seed), scheduler=SimpleNamespace(eos_token_ids=[3]),
                           config=SimpleNamespace(max_num_batched_tokens=budget))
  return BeamSearcher(engine, params)


def test_a_prompt_longer_than_the_pool_of_a_window_group_is_searched(monkeypatch):
  needs = [PagedKV(8, 128), PagedKV(8, 128, window=1024)]
  s = _searcher(monkeypatch, needs, BeamSearchParams(num_beams=4, max_tokens=6), page_size=16, num_pages=20000, requests=8,
                budget=8192)
  prompt = [1] * 32768
  assert s.cache.never_fits(len(prompt) + 6) is None
  assert s.cache.paged[1].pool.num_pages < 32768 // 16
  assert s._fits([Search(0, prompt, 6)])
  found = s.run([prompt, prompt])
  assert [len(f.finished) for f in found] == [4, 4] and s.cache.all_pages_free()


@pytest.mark.parametrize("window,page_size,budget,beams", [(1, 4, 4, 4), (5, 4, 8, 4), (16, 4, 32, 2), (24, 8, 16, 3), (64, 4, 512, 4), (7, 1, 9, 4)])
def test_searches_hold_no_more_than_they_ask_for(monkeypatch, window, page_size, budget, beams):
  """Beams for every slot: a pool made for so many requests holds them all."""
  rng = random.Random(window)
  for seed in range(6):
    tokens = rng.choice([1, 2, 9, 40])
    params = BeamSearchParams(num_beams=beams, max_tokens=tokens, ignore_eos=seed % 2 == 0, stop_token_ids=[5])
    needs = [PagedKV(1, 8), PagedKV(1, 8, window=window), PagedKV(2, 8, window=3 * window, page_size=2 * page_size)]
    s = _searcher(monkeypatch, needs, params, seed=seed, page_size=page_size, requests=beams * rng.choice([1, 2, 3]), budget=budget)
    prompts = [[1] * rng.choice([1, 3, 17, 150, 700]) for _ in range(5)]
    asked = []
    fits = s._fits
    s._fits = lambda live: fits(live) and (asked.append(s._pages(live)) or True)
    advance = s._advance

    def watched(*a):
      advance(*a)
      s.runner.note()
    s._advance = watched
    found = s.run(prompts)
    assert all(f.finished for f in found)
    assert all(p <= max(a[g] for a in asked) for g, p in enumerate(s.runner.peak)), (s.runner.peak, asked)
    s.cache.check()
    assert s.cache.all_pages_free() and not s.cache.live_requests()
