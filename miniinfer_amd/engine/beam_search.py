"""Beam search over the engine's step function: `LLMEngine.beam_search`.

The beams of a search are requests of the cache.  Every step runs the live beams of all prompts as one batch of single
tokens, `ops.beam_select` picks the best continuations of each prompt's beams, and the cache is brought in line with
them on the host where that is enough: a beam with one continuation goes on as the request it is, one with several is
forked (`CacheManager.fork`: full pages are shared, the last page and the fixed-size states copied), one without gives
its pages and slot back."""

from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, List, Sequence, Tuple

import torch

from ..kernels import ops
from ..sampling import BeamSearchParams
from .runner import StepEntry


@dataclass
class Beam:
  req: Tuple                    # its request in the cache
  tokens: List[int]             # generated so far
  score: float                  # sum of their log-probabilities, in 64 bits as they are compared


@dataclass
class Hypothesis:
  tokens: List[int]
  score: float
  reason: str
  penalised: float


@dataclass
class Search:
  """One prompt's search."""
  index: int
  prompt: List[int]
  max_tokens: int
  beams: List[Beam] = field(default_factory=list)
  finished: List[Hypothesis] = field(default_factory=list)      # best first, at most num_beams
  done: bool = False

  def finish(self, params: BeamSearchParams, tokens: List[int], score: float, reason: str) -> None:
    self.finished.append(Hypothesis(tokens, score, reason, score / len(tokens) ** params.length_penalty))
    self.finished.sort(key=lambda h: -h.penalised)
    del self.finished[params.num_beams:]

  def settled(self, params: BeamSearchParams) -> bool:
    """Whether no running beam can push out one of num_beams finished hypotheses."""
    if not self.beams:
      return True
    if len(self.finished) < params.num_beams:
      return False
    if params.early_stopping:
      return True
    best = max(b.score for b in self.beams)
    # the length at which the best running beam's score would count most
    length = len(self.beams[0].tokens) if params.length_penalty <= 0 else self.max_tokens
    return best / length ** params.length_penalty <= self.finished[-1].penalised


class BeamSearcher:
  def __init__(self, engine, params: BeamSearchParams):
    self.engine, self.params = engine, params
    self.cache, self.runner = engine.cache, engine.runner
    self.next_request = 0
    stop = set(params.stop_token_ids)
    if not params.ignore_eos:
      stop |= set(engine.scheduler.eos_token_ids)
    self.stop = stop
    # enough candidates that num_beams of them go on whatever the others end with
    self.count = (1 + len(stop)) * params.num_beams
    if self.count > ops.BEAM_MAX_COUNT:
      raise ValueError(f"num_beams={params.num_beams} with {len(stop)} tokens that end a hypothesis: at most "
                       f"{ops.BEAM_MAX_COUNT // (1 + len(stop))} are supported")

  # ------------------------------------------------------------------ requests
  def _new_request(self) -> Tuple:
    self.next_request += 1
    return ("beam", self.next_request)

  def _pages(self, searches: Sequence[Search]) -> List[int]:
    """The most pages that searches side by side hold at once, per cache group: their prompts', shared, and for each beam
    those of its own tokens, with the page that the prompt ends in and the one that a fork starts on.  Of a group with a
    window a request keeps what its next token can see, at most ceil(window / page) + 1 pages, and in a step the new
    tokens' beside them: one page of a beam, while the prompts are read those of a step's tokens."""
    out = []
    for g in self.cache.paged:
      pages = lambda n: -(-n // g.page_size)
      prompts = [pages(len(s.prompt)) for s in searches]
      own = [self.params.num_beams * (pages(s.max_tokens) + 2) for s in searches]
      if g.need.window is None:
        out.append(sum(prompts) + sum(own))
        continue
      keeps = pages(g.need.window) + 1
      reading = min(sum(prompts), sum(min(p, keeps + 1) for p in prompts) + pages(self.engine.config.max_num_batched_tokens))
      searching = sum(min(min(p, keeps) + o, self.params.num_beams * (keeps + 1)) for p, o in zip(prompts, own))
      out.append(max(reading, searching))
    return out

  def _fits(self, searches: Sequence[Search]) -> bool:
    beams = len(searches) * self.params.num_beams          # the tokens of a step
    if beams > self.cache.num_free_slots() or beams > self.engine.config.max_num_batched_tokens:
      return False
    return all(need <= room for need, room in zip(self._pages(searches), self.cache.room()))

  # ------------------------------------------------------------------ steps
  def _prefill(self, searches: Sequence[Search]) -> torch.Tensor:
    """Every prompt through the model, in portions of the token budget; logits [prompts, vocab] of their last tokens."""
    budget = self.engine.config.max_num_batched_tokens
    at: Dict[int, int] = {}
    rows: Dict[int, torch.Tensor] = {}
    for s in searches:
      s.beams = [Beam(self._new_request(), [], 0.0)]
      self.cache.admit(s.beams[0].req)
      at[s.index] = 0
    while any(at[s.index] < len(s.prompt) for s in searches):
      entries, ends, left = [], [], budget
      for s in searches:
        first = at[s.index]
        n = min(left, len(s.prompt) - first)
        if n > 0:
          last = first + n == len(s.prompt)
          entries.append(StepEntry(s.beams[0].req, s.prompt[first:first + n], [n - 1] if last else []))
          at[s.index] += n
          left -= n
          if last:
            ends.append(s.index)
      logits = self.runner.step(entries)
      for i, index in enumerate(ends):
        rows[index] = logits[i:i + 1].clone()      # (a captured step's logits are overwritten by the next)
    return torch.cat([rows[s.index] for s in searches])

  def _advance(self, searches: Sequence[Search], logits: torch.Tensor, width: int) -> None:
    """Picks every search's next beams from `logits` [searches * width, vocab] and brings the cache in line."""
    V = logits.shape[1]
    scores: List[float] = []
    for s in searches:
      scores += [b.score for b in s.beams] + [float("-inf")] * (width - len(s.beams))
    count = min(self.count, width * V)
    got = ops.beam_select(logits, torch.tensor(scores, dtype=torch.float64).to(logits.device), width, count,
                          score_dtype=torch.float64)
    values, beams, tokens = (t.tolist() for t in got)
    forks: List[Tuple] = []
    for s, vs, bs, ts in zip(searches, values, beams, tokens):
      chosen: List[Tuple[int, Beam]] = []
      for rank, (v, b, t) in enumerate(zip(vs, bs, ts)):
        if len(chosen) == self.params.num_beams or v == float("-inf"):
          break
        hyp = s.beams[b].tokens + [t]
        if t in self.stop:
          if rank < self.params.num_beams:         # (a worse one would not have been among the beams)
            s.finish(self.params, hyp, v, "stop" if t in self.params.stop_token_ids else "eos")
        elif len(hyp) == s.max_tokens:
          s.finish(self.params, hyp, v, "length")
          chosen.append((b, None))
        else:
          chosen.append((b, Beam(s.beams[b].req, hyp, v)))
      went_on = set()
      old = s.beams
      s.beams = []
      for b, beam in chosen:
        if beam is None:
          continue
        if b in went_on:
          beam.req = self._new_request()
          forks.append((old[b].req, beam.req))
        went_on.add(b)
        s.beams.append(beam)
      s.done = s.settled(self.params)
      if s.done:                                   # nothing of it goes on
        forks = [f for f in forks if f[1] not in {x.req for x in s.beams}]
        s.beams, went_on = [], set()
      for b, beam in enumerate(old):
        if b not in went_on:
          self.cache.release(beam.req)
    if forks:
      self.cache.fork(forks)

  def run(self, prompts: Sequence[List[int]]) -> List[Search]:
    """All prompts, as many at a time as the slots and pages hold."""
    searches = [Search(i, p, self.params.max_tokens) for i, p in enumerate(prompts)]
    waiting = list(searches)
    for s in searches:
      if not self._fits([s]):
        raise ValueError(f"a beam search of {self.params.num_beams} beams over a prompt of {len(s.prompt)} tokens plus "
                         f"max_tokens={s.max_tokens} does not fit the cache ({self._pages([s])} pages per group, "
                         f"{self.cache.room()} free; {self.cache.num_free_slots()} request slots; steps of "
                         f"{self.engine.config.max_num_batched_tokens} tokens)")
    try:
      while waiting:
        live = [waiting.pop(0)]
        while waiting and self._fits(live + waiting[:1]):
          live.append(waiting.pop(0))
        self._advance(live, self._prefill(live), 1)
        live = [s for s in live if not s.done]
        while live:
          width = max(len(s.beams) for s in live)
          logits = self.runner.step([StepEntry(b.req, [b.tokens[-1]], [0]) for s in live for b in s.beams])
          if any(len(s.beams) < width for s in live):      # beams that do not take part stand in for the missing ones
            rows, at = [], 0
            for s in live:
              rows += list(range(at, at + len(s.beams))) + [at] * (width - len(s.beams))
              at += len(s.beams)
            logits = logits.index_select(0, torch.tensor(rows, device=logits.device))
          self._advance(live, logits, width)
          live = [s for s in live if not s.done]
    finally:                           # (nothing is left but after an error)
      for req in self.cache.live_requests():
        if isinstance(req, tuple) and req[0] == "beam":
          self.cache.release(req)
    return searches
