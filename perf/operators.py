"""What the operators for fixed-state layers and beam search are measured on: linear attention with a decay for each head
(prompts and single tokens), beam search's selection over beams and vocabulary, and moves of cache pages and state rows.

`run` computes the plain form (elementary torch operations, 32-bit; 64-bit where 32 lose what matters) or, with `own`
set, calls this package's kernels."""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------------------- cases

def listed():
  return [
    # one short prompt into a fresh request: a launch's latency
    dict(name="prompt_33", op="prompt", dtype="bf16", seqs=1, tokens=33, nq=16, nkv=8, d=128),
    # one prompt of the benchmark's length, the 0.6B shape's heads
    dict(name="prompt_2048", op="prompt", dtype="bf16", seqs=1, tokens=2048, nq=16, nkv=8, d=128),
    # a step of prompt portions of many lengths, a head size that is no power of two
    dict(name="prompt_ragged", op="prompt", dtype="bf16", seqs=24, tokens=9001, nq=12, nkv=12, d=80),
    # one long prompt, the 8B shape's heads
    dict(name="prompt_32768", op="prompt", dtype="bf16", seqs=1, tokens=32768, nq=32, nkv=8, d=128),
    # the 32-bit path: a few prompts
    dict(name="prompt_f32", op="prompt", dtype="f32", seqs=3, tokens=1500, nq=16, nkv=8, d=64),
    # decode of one request
    dict(name="step_1", op="step", dtype="bf16", seqs=1, nq=16, nkv=8, d=128),
    # decode of a full batch
    dict(name="step_64", op="step", dtype="bf16", seqs=64, nq=32, nkv=8, d=128),
    # 32-bit decode of many requests, a head size that is no power of two
    dict(name="step_f32_200", op="step", dtype="f32", seqs=200, nq=6, nkv=6, d=80),
    # a few short searches over a small vocabulary of odd size
    dict(name="beam_3x5", op="beam", groups=3, beams=5, vocab=32003, count=10, first=False),
    # a batch of searches over the presets' vocabulary
    dict(name="beam_32x8", op="beam", groups=32, beams=8, vocab=151936, count=16, first=False),
    # a fork in a search: the last, partly filled pages of twelve requests in all layers, keys and values
    dict(name="move_pages", op="pages", dtype="bf16", layers=28, pages=256, nkv=8, d=128, page=16, moves=12),
    # the states of 64 beams change places in the fixed-state layers
    dict(name="move_states", op="states", dtype="f32", layers=12, rows=65, nkv=8, d=128, moves=64),
  ]


def _log_int(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  op = rng.choice(["prompt", "prompt", "step", "step", "beam", "beam", "pages", "states"])
  if op in ("prompt", "step"):
    nkv = rng.choice([1, 2, 4, 8, 12, 16])
    nq = nkv * rng.choice([1, 1, 2, 4])
    d = rng.choice([16, 32, 64, 80, 96, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "step":
      return dict(op=op, dtype=dtype, seqs=_log_int(rng, 1, 256), nq=nq, nkv=nkv, d=d)
    tokens = _log_int(rng, 1, max(2, min(32768, 32768 * 32 * 128 // (nq * d * (4 if dtype == "f32" else 1)))))
    return dict(op=op, dtype=dtype, seqs=min(tokens, _log_int(rng, 1, 48)), tokens=tokens, nq=nq, nkv=nkv, d=d)
  if op == "beam":
    beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
    vocab = _log_int(rng, 256, 151936)
    return dict(op=op, groups=_log_int(rng, 1, max(1, 256 // beams)), beams=beams, vocab=vocab, count=2 * beams,
                first=rng.random() < 0.3)
  if op == "pages":
    page = rng.choice([8, 16, 32])
    return dict(op=op, dtype=rng.choice(["bf16", "f32"]), layers=rng.choice([1, 2, 3, 12, 28]), pages=rng.randint(40, 250),
                nkv=rng.choice([1, 2, 4, 8]), d=rng.choice([32, 64, 80, 128]), page=page, moves=_log_int(rng, 1, 20))
  rows = rng.randint(2, 65)
  return dict(op=op, dtype="f32", layers=rng.randint(1, 12), rows=rows, nkv=rng.choice([1, 3, 8]),
              d=rng.choice([16, 64, 80, 128]), moves=rng.randint(1, rows - 1))


# ------------------------------------------------------------------------------------------------------------ inputs

def _log_decay(nkv):
  """Decays from exp(-1/256) to exp(-0.7): heads that forget after a few tokens and heads that hardly do."""
  return torch.tensor([-0.7 * 2.0 ** (-7.5 * h / max(1, nkv - 1)) for h in range(nkv)], dtype=torch.float32)


def _lengths(tokens, seqs, gen):
  """`seqs` lengths of at least one token, as different as prompts are, that add up to `tokens`."""
  w = torch.rand(seqs, generator=gen, dtype=torch.float64) ** 2 + 0.02
  n = 1 + torch.floor(w / w.sum() * (tokens - seqs)).long()
  n[0] += tokens - int(n.sum())
  return n


def prepare(case, seed):
  """Every tensor that a program has in hand before the call; integer tensors are int32 as the step function lays them
  out, the fused projection q | k | v is one buffer of rows."""
  gen = torch.Generator().manual_seed(seed)
  dgen = torch.Generator(DEV).manual_seed(seed)
  op = case["op"]
  st = dict(case)
  if op in ("prompt", "step"):
    nq, nkv, d, B = case["nq"], case["nkv"], case["d"], case["seqs"]
    T = case["tokens"] if op == "prompt" else B
    lens = _lengths(T, B, gen) if op == "prompt" else torch.ones(B, dtype=torch.long)
    qkv = torch.randn(T, (nq + 2 * nkv) * d, generator=dgen, device=DEV).to(DTYPES[case["dtype"]])
    st.update(qkv=qkv, scale=d ** -0.5, log_decay=_log_decay(nkv).to(DEV),
              state=torch.randn(B + 1, nkv, d, d, generator=dgen, device=DEV),        # the last row is no request's
              rows=torch.randperm(B, generator=gen).to(torch.int32).to(DEV),
              cu=torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)]).to(torch.int32).to(DEV),
              longest=int(lens.max()))
  elif op == "beam":
    G, W, V = case["groups"], case["beams"], case["vocab"]
    # logits of a model's spread; running scores are sums of log-probabilities, near one another within a group
    base = -40.0 * torch.rand(G, 1, generator=dgen, device=DEV)
    st.update(logits=torch.randn(G * W, V, generator=dgen, device=DEV) * 2.5,
              scores=(base - 3.0 * torch.rand(G, W, generator=dgen, device=DEV)).view(-1))
    if case["first"]:      # the first step of a search: one beam lives in each group
      st["scores"].view(G, W)[:, 1:] = -math.inf
  elif op == "pages":
    L, N, h, d, P, n = (case[x] for x in ("layers", "pages", "nkv", "d", "page", "moves"))
    dt = DTYPES[case["dtype"]]
    order = torch.randperm(N, generator=gen) + 1                                       # page 0 is never handed out
    st.update(buffers=[torch.randn(L, N + 1, h, P, d, generator=dgen, device=DEV, dtype=dt),
                       torch.randn(L, N + 1, h, d, P, generator=dgen, device=DEV, dtype=dt)],
              dst=order[:n].to(torch.int32).to(DEV),
              # a page is forked more than once; no page is both read and written
              src=order[n:][torch.randint(0, n, (n,), generator=gen)].to(torch.int32).to(DEV))
  else:
    L, N, h, d, n = (case[x] for x in ("layers", "rows", "nkv", "d", "moves"))
    order = torch.randperm(N - 1, generator=gen)[:n]                                   # the last row is scratch
    # each beam's parent: rows are read and written, some by several, some by themselves
    st.update(buffers=[torch.randn(L, N, h, d, d, generator=dgen, device=DEV)], dst=order.to(torch.int32).to(DEV),
              src=order[torch.randint(0, n, (n,), generator=gen)].to(torch.int32).to(DEV))
  return st


# --------------------------------------------------------------------------------------------------------- plain forms

CHUNK = 128


def _plain_prompt(st):
  """S_t = a S_{t-1} + k_t v_t^T, o_t = scale q_t S_t, chunk by chunk: within a chunk the masked products of queries and
  keys, across chunks the states at the chunks' starts."""
  nq, nkv, d, B, C = st["nq"], st["nkv"], st["d"], st["seqs"], CHUNK
  cu, rows, rep = st["cu"].long(), st["rows"].long(), st["nq"] // st["nkv"]
  n = -(-st["longest"] // C)
  at = cu[:-1, None] + torch.arange(n * C, device=DEV)
  live = at < cu[1:, None]
  x = torch.where(live[..., None], st["qkv"][at.clamp(max=st["qkv"].shape[0] - 1)].float(), 0.0)
  q = x[..., :nq * d].reshape(B, n, C, nkv, rep, d).permute(0, 3, 4, 1, 2, 5)              # [B, h, r, n, C, d]
  k = x[..., nq * d:(nq + nkv) * d].reshape(B, n, C, nkv, d).permute(0, 3, 1, 2, 4)        # [B, h, n, C, d]
  v = x[..., (nq + nkv) * d:].reshape(B, n, C, nkv, d).permute(0, 3, 1, 2, 4)
  g = st["log_decay"].double()

  def power(e):      # a^e for each head, [h, *e.shape]; zero where e is negative
    return torch.where(e >= 0, torch.exp(g.view(-1, *[1] * e.dim()) * e.clamp(min=0)), 0.0).float()

  i, c = torch.arange(C, device=DEV), torch.arange(n, device=DEV)
  added = (k * power(C - 1 - i)[:, None, :, None]).transpose(-1, -2) @ v                   # [B, h, n, d, d]
  state = st["state"][rows]                                                                # [B, h, d, d]
  before = (power((c[:, None] - 1 - c) * C).expand(B, -1, -1, -1) @ added.reshape(B, nkv, n, d * d)).view(B, nkv, n, d, d) \
      + power(c * C)[:, :, None, None] * state[:, :, None]
  scores = (q @ k[:, :, None].transpose(-1, -2)) * power(i[:, None] - i)[:, None, None]
  o = scores @ v[:, :, None] + (q * power(i + 1)[:, None, None, :, None]) @ before[:, :, None]
  o = (o * st["scale"]).permute(0, 3, 4, 1, 2, 5).reshape(B, n * C, nq * d)
  out = o[live].to(st["qkv"].dtype)
  # the states after the last tokens
  length = (cu[1:] - cu[:-1])
  left = (length[:, None] - 1 - torch.arange(n * C, device=DEV))
  kt = k.reshape(B, nkv, n * C, d) * power(left).transpose(0, 1)[..., None]
  st["state"][rows] = power(length).t()[:, :, None, None] * state + kt.transpose(-1, -2) @ v.reshape(B, nkv, n * C, d)
  return dict(out=out, state=st["state"])


def _plain_step(st):
  nq, nkv, d, B = st["nq"], st["nkv"], st["d"], st["seqs"]
  rows = st["rows"].long()
  x = st["qkv"].float()
  q = x[:, :nq * d].view(B, nkv, nq // nkv, d)
  k = x[:, nq * d:(nq + nkv) * d].view(B, nkv, d, 1)
  v = x[:, (nq + nkv) * d:].view(B, nkv, 1, d)
  state = st["state"][rows] * torch.exp(st["log_decay"])[:, None, None] + k * v
  st["state"][rows] = state
  return dict(out=((q @ state) * st["scale"]).reshape(B, nq * d).to(st["qkv"].dtype), state=st["state"])


def _plain_beam(st):
  """In 64 bits: candidates of different beams lie closer to one another than 32 bits of a score tell apart."""
  G, W, V, K = st["groups"], st["beams"], st["vocab"], st["count"]
  x = st["logits"].double()
  x = x - x.amax(-1, keepdim=True)
  score = (x - x.exp().sum(-1, keepdim=True).log() + st["scores"].double()[:, None]).view(G, W * V)
  value, index = score.topk(min(K + 8, W * V), dim=-1)      # a few more than asked for, so that equals can be put in order
  index, order = index.sort(dim=-1)
  value, order = value.gather(1, order).sort(dim=-1, descending=True, stable=True)
  index = index.gather(1, order)[:, :K]
  return dict(scores=value[:, :K].float(), beams=(index // V).int(), tokens=(index % V).int())


def _plain_move(st):
  src, dst = st["src"].long(), st["dst"].long()
  first, last = st["buffers"][0], st["buffers"][-1]
  first[:, dst] = first[:, src]
  if last is not first:
    last[:, dst] = last[:, src]
  return list(st["buffers"])


def _own(st):
  from miniinfer_amd.kernels import ops
  op = st["op"]
  if op in ("prompt", "step"):
    nq, nkv, d, qkv = st["nq"], st["nkv"], st["d"], st["qkv"]
    q, k, v = qkv[:, :nq * d], qkv[:, nq * d:(nq + nkv) * d], qkv[:, (nq + nkv) * d:]
    out = torch.empty((qkv.shape[0], nq * d), dtype=qkv.dtype, device=qkv.device)
    if op == "prompt":
      ops.linear_attention(q, k, v, nq, nkv, d, out, st["state"], st["rows"], st["cu"], st["log_decay"], st["scale"],
                           max_len=st["longest"])
    else:
      ops.linear_attention_step(q, k, v, nq, nkv, d, out, st["state"], st["rows"], st["log_decay"], st["scale"])
    return dict(out=out, state=st["state"])
  if op == "beam":
    scores, beams, tokens = ops.beam_select(st["logits"], st["scores"], st["beams"], st["count"])
    return dict(scores=scores, beams=beams, tokens=tokens)
  ops.move_rows(st["buffers"], st["src"], st["dst"])
  return list(st["buffers"])


def run(state):
  if own:
    return _own(state)
  op = state["op"]
  return {"prompt": _plain_prompt, "step": _plain_step, "beam": _plain_beam, "pages": _plain_move,
          "states": _plain_move}[op](state)


# -------------------------------------------------------------------------------------------------------- what it costs

def work(case):
  op = case["op"]
  if op in ("prompt", "step"):
    nq, nkv, d, B = case["nq"], case["nkv"], case["d"], case["seqs"]
    T = case["tokens"] if op == "prompt" else B
    size = 2 if case["dtype"] == "bf16" else 4
    # q, k, v and the output once, each request's state read and written; a multiply and an add for every element of a
    # state and token (k v^T), and for every query head's product with it
    return dict(bytes=T * (2 * nq + 2 * nkv) * d * size + 2 * B * nkv * d * d * 4, flops=2 * T * (nq + nkv) * d * d)
  if op == "beam":
    n = case["groups"] * case["beams"] * case["vocab"]
    # every logit once; a subtraction, an exponential and an addition each
    return dict(bytes=4 * n + 12 * case["groups"] * case["count"], flops=3 * n)
  # every destination written, every row that is a source (some are one twice) read once
  n, size = case["moves"], 2 if case["dtype"] == "bf16" else 4
  rows = n + n * (1 - (1 - 1 / n) ** n)
  row = 2 * case["nkv"] * case["d"] * case["page"] if op == "pages" else case["nkv"] * case["d"] * case["d"]
  return dict(bytes=rows * case["layers"] * row * size, flops=0)


# --------------------------------------------------------------------------------------------------- 64-bit definitions

def exact(case, seed):
  """From the definitions: the recurrence token by token; the log-probabilities of each row one after the other.  Moved
  rows are no computed numbers."""
  op = case["op"]
  if op in ("pages", "states"):
    return None
  st = prepare(case, seed)
  if op == "beam":
    G, W, V, K = case["groups"], case["beams"], case["vocab"], case["count"]
    scores, beams, tokens = [], [], []
    for g in range(G):
      rows = [float(st["scores"][r]) + torch.log_softmax(st["logits"][r].double(), 0) for r in range(g * W, g * W + W)]
      value, index = torch.sort(torch.cat(rows), descending=True, stable=True)
      scores.append(value[:K])
      beams.append(torch.div(index[:K], V, rounding_mode="floor"))
      tokens.append(torch.remainder(index[:K], V))
    return dict(scores=torch.stack(scores), beams=torch.stack(beams).int(), tokens=torch.stack(tokens).int())
  nq, nkv, d, B = case["nq"], case["nkv"], case["d"], case["seqs"]
  x = st["qkv"].double()
  start = st["cu"][:-1].long()
  length = st["cu"][1:].long() - start
  longest = int(length.max())
  if longest * max(1.0, B * nq * d * d / 2.5e6) > 120000:
    return None
  rows = st["rows"].long()
  state = st["state"].double()
  S = state[rows]
  a = torch.exp(st["log_decay"].double()).view(1, nkv, 1, 1)
  out = torch.zeros(x.shape[0] + 1, nq * d, dtype=torch.float64, device=DEV)      # a last row for ended sequences
  for t in range(longest):
    live = t < length
    tok = torch.where(live, start + t, 0)
    y = x[tok]
    k = y[:, nq * d:(nq + nkv) * d].reshape(B, nkv, d, 1)
    v = y[:, (nq + nkv) * d:].reshape(B, nkv, 1, d)
    S = torch.where(live.view(B, 1, 1, 1), a * S + k * v, S)
    q = y[:, :nq * d].reshape(B, nkv, nq // nkv, d)
    o = (q[..., None] * S[:, :, None]).sum(-2).reshape(B, nq * d) * st["scale"]
    out[torch.where(live, tok, x.shape[0])] = o
  state[rows] = S
  return dict(out=out[:-1], state=state)
