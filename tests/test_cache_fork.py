"""Forked requests in the cache manager: shared and copied pages, states, and the books (on the CPU)."""

import pytest
import torch

from miniinfer_amd.cache import CacheError, CacheManager, OutOfPages, OutOfSlots, PagePool
from miniinfer_amd.parts import FixedState, PagedKV


def _manager(num_pages=20, max_requests=6, window=None, allocate=True):
  needs = [PagedKV(2, 8), FixedState((2, 4, 4), torch.float32), PagedKV(2, 8), PagedKV(1, 8, window=window or 6, page_size=2),
           FixedState((3,), torch.float32)]
  return CacheManager(needs, page_size=4, num_pages=num_pages, max_requests=max_requests, max_model_len=64,
                      dtype=torch.float32, device="cpu", allocate=allocate)


def _write(m, req, lo, hi, seed):
  """Stands for a step: random keys and values of tokens lo .. hi - 1 and new states."""
  g = torch.Generator().manual_seed(seed)
  m.grow(req, hi)
  for gi, grp in enumerate(m.paged):
    for t in range(lo, hi):
      page, off = m.table(gi, req)[t // grp.page_size], t % grp.page_size
      grp.k[:, page, :, off] = torch.randn(grp.k[:, page, :, off].shape, generator=g)
      grp.v[:, page, :, :, off] = torch.randn(grp.v[:, page, :, :, off].shape, generator=g)
  for s in m.states:
    s.state[:, m.slot(req)] = torch.randn(s.state[:, 0].shape, generator=g)
  m.commit(req, hi)


def _contents(m, req):
  out = []
  for gi, grp in enumerate(m.paged):
    for t in range(m.length(req)):
      page, off = m.table(gi, req)[t // grp.page_size], t % grp.page_size
      if page:
        out += [grp.k[:, page, :, off].clone(), grp.v[:, page, :, :, off].clone()]
  return out + [s.state[:, m.slot(req)].clone() for s in m.states]


def _same(a, b):
  return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_pool_counts_the_holders_of_a_page():
  pool = PagePool(5)
  a, b = pool.alloc(2)
  pool.share([a, a])
  assert pool.held() == sorted([a, a, a, b]) and pool.num_held == 2 and pool.num_free == 3
  pool.free([a])
  pool.free([a, b])
  assert pool.num_free == 4 and pool.held() == [a]
  pool.free([a])
  assert pool.num_free == 5
  with pytest.raises(CacheError):
    pool.free([a])
  with pytest.raises(CacheError):
    pool.share([a])
  with pytest.raises(CacheError):
    pool.share([0])


@pytest.mark.parametrize("length", [0, 1, 4, 5, 8, 11])
def test_a_fork_holds_what_its_parent_holds_and_goes_its_own_way(length):
  m = _manager()
  m.admit("p")
  if length:
    _write(m, "p", 0, length, 1)
  before = _contents(m, "p")
  m.fork([("p", "a"), ("p", "b")])
  m.check()
  for r in ("p", "a", "b"):
    assert m.length(r) == length and _same(_contents(m, r), before)
  for gi, g in enumerate(m.paged):
    full = length // g.page_size
    for r in ("a", "b"):
      assert m.table(gi, r)[:full] == m.table(gi, "p")[:full]          # full pages are shared
      assert len(m.table(gi, r)) == -(-length // g.page_size)
    if length % g.page_size:
      assert len({m.table(gi, r)[full] for r in ("p", "a", "b")}) == 3   # the page that is written next is not
  # each goes on by itself
  for i, r in enumerate(("p", "a", "b")):
    _write(m, r, length, length + 5, 10 + i)
    m.check()
  first = len(before) - len(m.states)
  kept = {r: _contents(m, r) for r in ("p", "a", "b")}
  assert not _same(kept["p"], kept["a"])
  m.release("p")
  m.check()
  assert _same(_contents(m, "a"), kept["a"]) and _same(_contents(m, "b"), kept["b"])
  m.release("a")
  m.release("b")
  m.check()
  assert m.all_pages_free() and m.num_free_slots() == 6 and first >= 0


def test_pages_of_a_window_come_back_with_their_last_holder():
  m = _manager(window=6)
  m.admit("p")
  _write(m, "p", 0, 9, 1)
  m.fork([("p", "a")])
  free = m.paged[1].pool.num_free
  _write(m, "p", 9, 15, 2)                 # the parent's window has passed pages that the child still sees
  m.check()
  assert all(p for p in m.table(1, "a")[2:])
  _write(m, "a", 9, 15, 3)
  m.check()
  m.release("p")
  m.release("a")
  m.check()
  assert m.all_pages_free() and free >= 0


def test_forks_of_forks_and_many_at_once():
  m = _manager(num_pages=60, max_requests=12)
  m.admit(0)
  _write(m, 0, 0, 7, 1)
  live, nxt = [0], 1
  for step in range(6):
    pairs = [(r, nxt + i) for i, r in enumerate(live[:5])]
    nxt += len(pairs)
    want = {c: _contents(m, p) for p, c in pairs}
    m.fork(pairs)
    m.check()
    assert all(_same(_contents(m, c), w) for c, w in want.items())
    live += [c for _, c in pairs]
    while len(live) > 6:
      m.release(live.pop(0))
      m.check()
    for i, r in enumerate(live):
      _write(m, r, m.length(r), m.length(r) + 1 + i % 3, 100 * step + i)
    m.check()
  for r in live:
    m.release(r)
  assert m.all_pages_free()


def test_refused_forks_change_nothing():
  m = _manager(num_pages=3, max_requests=3)
  m.admit("p")
  _write(m, "p", 0, 6, 1)
  state = (m.room(), m.num_free_slots(), _contents(m, "p"))
  with pytest.raises(CacheError, match="not admitted"):
    m.fork([("x", "a")])
  with pytest.raises(CacheError, match="admitted already"):
    m.fork([("p", "p")])
  with pytest.raises(CacheError, match="admitted already"):
    m.fork([("p", "a"), ("p", "a")])
  with pytest.raises(OutOfSlots):
    m.fork([("p", c) for c in "abc"])
  with pytest.raises(OutOfPages):
    m.fork([("p", "a"), ("p", "b")])
  m.check()
  assert (m.room(), m.num_free_slots()) == state[:2] and _same(_contents(m, "p"), state[2])
  m.fork([])
  m.fork([("p", "a")])
  m.check()


def test_forks_without_storage():
  m = _manager(allocate=False)
  m.admit("p")
  m.grow("p", 6)
  m.commit("p", 6)
  m.fork([("p", "a")])
  m.check()
  m.release("p")
  m.release("a")
  assert m.all_pages_free()
