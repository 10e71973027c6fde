"""Beam search as it is defined, over a function that gives a whole sequence's logits: every hypothesis is recomputed from
its first token at every step."""

import torch


def beam_search(logits_of, prompt, num_beams, max_tokens, stop=(), length_penalty=1.0, early_stopping=False):
  """logits_of(tokens) -> [len, vocab] float64.  Returns (hypotheses best first: (tokens, log-probability, penalised),
  the smallest difference that decided anything)."""
  beams = [([], 0.0)]
  finished, gap = [], float("inf")
  while beams:
    cand = []
    for b, (toks, score) in enumerate(beams):
      logp = torch.log_softmax(logits_of(list(prompt) + toks)[-1].double(), -1)
      cand += [(score + float(p), b, t) for t, p in enumerate(logp)]
    cand.sort(key=lambda c: (-c[0], c[1], c[2]))
    nxt = []
    looked = 0
    for rank, (score, b, t) in enumerate(cand):
      if len(nxt) == num_beams:
        break
      looked = rank + 1
      toks = beams[b][0] + [t]
      if t in stop:
        if rank < num_beams:
          finished.append((toks, score, score / len(toks) ** length_penalty))
      elif len(toks) == max_tokens:
        finished.append((toks, score, score / len(toks) ** length_penalty))
        nxt.append(None)
      else:
        nxt.append((toks, score))
    for x, y in zip(cand[:looked], cand[1:looked + 1]):
      gap = min(gap, x[0] - y[0])
    finished.sort(key=lambda h: -h[2])
    for x, y in zip(finished[:num_beams], finished[1:num_beams + 1]):
      gap = min(gap, x[2] - y[2])
    del finished[num_beams:]
    beams = [b for b in nxt if b is not None]
    if beams and len(finished) == num_beams:
      length = len(beams[0][0]) if length_penalty <= 0 else max_tokens
      bound = max(s for _, s in beams) / length ** length_penalty
      gap = min(gap, abs(bound - finished[-1][2]))
      if early_stopping or bound <= finished[-1][2]:
        break
  return finished, gap
