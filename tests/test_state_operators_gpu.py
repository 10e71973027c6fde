"""Linear attention, beam selection and row moves, each against a plain statement in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of 32 bits, and every sum of n terms in 32 bits, in any order, is
within n u of the sum of the terms' magnitudes.  For linear attention that sum is what the same recurrence gives for the
magnitudes of its inputs (`_recurrence` of |q|, |k|, |v|, |S|): a state's element passes at most two roundings a token
(decay and addition) and two for each power of the decay it is scaled with, an output d additions more.  Where the kernel multiplies on
the matrix cores with bfloat16 operands, a 32-bit factor is split into two or more bfloat16 parts, so a term is off by
at most 2^-16 of its magnitude.  A bfloat16 output is rounded once: half a step, 2^-8 of the value."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24


# ------------------------------------------------------------------------------------------------- linear attention

def _recurrence(q, k, v, state, rows, cu, log_decay, scale, nq, nkv, d):
  """out [T, nq * d] (NaN where no request is), states; float64 on the CPU, token by token."""
  T = q.shape[0]
  rep = nq // nkv
  q, k, v = q.double().view(T, nkv, rep, d), k.double().view(T, nkv, d, 1), v.double().view(T, nkv, 1, d)
  a = torch.exp(log_decay.double()).view(nkv, 1, 1)
  out = torch.full((T, nkv, rep, d), float("nan"), dtype=torch.float64)
  state = state.double().clone()
  for b in range(len(rows)):
    S = state[rows[b]]
    for t in range(cu[b], cu[b + 1]):
      S = a * S + k[t] * v[t]
      out[t] = (q[t].unsqueeze(-1) * S.unsqueeze(1)).sum(2) * scale
    state[rows[b]] = S
  return out.view(T, nq * d), state


class _Call:
  """Inputs of a call, on the CPU and on the device; the device's q, k and v are parts of one fused buffer."""

  def __init__(self, dtype, nq, nkv, d, lens, seed=0, spare_rows=2, before=0, behind=0, log_decay=None, scale=None):
    g = torch.Generator().manual_seed(seed)
    self.nq, self.nkv, self.d, self.lens = nq, nkv, d, list(lens)
    self.T = before + sum(lens) + behind
    self.cu = [before]
    for n in lens:
      self.cu.append(self.cu[-1] + n)
    self.qkv = torch.randn(self.T, (nq + 2 * nkv) * d, generator=g).to(dtype)
    self.state = torch.randn(len(lens) + spare_rows, nkv, d, d, generator=g)
    self.rows = torch.randperm(len(lens) + spare_rows, generator=g)[:len(lens)].tolist()
    self.log_decay = torch.tensor([-0.7 * 2.0 ** (-7.5 * h / max(1, nkv - 1)) for h in range(nkv)]) if log_decay is None \
        else torch.tensor(log_decay, dtype=torch.float32)
    self.scale = d ** -0.5 if scale is None else scale
    self.dtype = dtype

  def parts(self, qkv):
    n = self.nq * self.d
    m = self.nkv * self.d
    return qkv[:, :n], qkv[:, n:n + m], qkv[:, n + m:]

  def want(self):
    return _recurrence(*self.parts(self.qkv), self.state, self.rows, self.cu, self.log_decay, self.scale, self.nq, self.nkv, self.d)

  def magnitudes(self):
    return _recurrence(*self.parts(self.qkv.abs()), self.state.abs(), self.rows, self.cu, self.log_decay, self.scale, self.nq,
                       self.nkv, self.d)

  def device(self):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    return self.qkv.to(DEV), self.state.to(DEV), i32(self.rows), i32(self.cu), self.log_decay.to(DEV)

  def run(self, max_len=None, step=False):
    from miniinfer_amd.kernels import ops
    qkv, state, rows, cu, g = self.device()
    out = torch.full((self.T, self.nq * self.d), 7.0, dtype=self.dtype, device=DEV)
    if step:
      ops.linear_attention_step(*self.parts(qkv), self.nq, self.nkv, self.d, out, state, rows, g, self.scale)
    else:
      ops.linear_attention(*self.parts(qkv), self.nq, self.nkv, self.d, out, state, rows, cu, g, self.scale, max_len)
    return out.cpu(), state.cpu()

  def check(self, out, state, steps=None):
    """steps: tokens of a request so far (default: this call's longest)."""
    want, want_state = self.want()
    mag, mag_state = self.magnitudes()
    n = max(self.lens + [1]) if steps is None else steps
    split = 0.0 if self.dtype == torch.float32 else 2.0 ** -16
    live = slice(self.cu[0], self.cu[-1])
    half = torch.finfo(self.dtype).eps / 2
    bound = half * want.abs() + (split + (4 * n + self.d + 8) * U) * mag * (1 + half)
    assert bool(((out.double() - want).abs() <= bound)[live].all()), _worst(out.double()[live], want[live], bound[live])
    touched = torch.zeros(self.state.shape[0], dtype=torch.bool)
    touched[[r for r, m in zip(self.rows, self.lens) if m]] = True
    assert torch.equal(state[~touched], self.state[~touched])           # nobody else's state
    # (a state is 32 bits whatever the inputs are: its products are split finely enough that 2^-22 is left of a term)
    bound = ((2.0 ** -22 if split else 0.0) + (4 * n + 8) * U) * mag_state
    assert bool(((state.double() - want_state).abs() <= bound)[touched].all()), \
        _worst(state.double()[touched], want_state[touched], bound[touched])
    outside = torch.ones(self.T, dtype=torch.bool)
    outside[live] = False
    assert bool((out[outside] == 7.0).all())                            # rows of no request
    # as a whole the error is a rounding's, far below the bound of each element
    if self.cu[-1] > self.cu[0]:
      assert float((out.double() - want)[live].norm() / want[live].norm()) <= (half if split else 2e-6)
      assert float((state.double() - want_state)[touched].norm() / want_state[touched].norm()) <= 2e-6


def _worst(got, want, bound):
  r = ((got - want).abs() / bound.clamp_min(1e-300)).flatten()
  i = int(r.nan_to_num(float("inf")).argmax())
  return f"worst: {got.flatten()[i]} for {want.flatten()[i]}, bound {bound.flatten()[i]}"


SHAPES = [(1, 1, 8), (4, 2, 16), (3, 3, 40), (5, 1, 64), (12, 12, 80), (8, 4, 128), (2, 1, 200), (2, 2, 256)]
LENS = [[1], [2], [17], [63, 1], [64], [65], [0, 5, 0, 130, 1], [257, 0, 77, 3]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", SHAPES)
def test_linear_attention(dtype, nq, nkv, d):
  for i, lens in enumerate(LENS):
    c = _Call(dtype, nq, nkv, d, lens, seed=i, before=i % 3, behind=(i + 1) % 3)
    c.check(*c.run(max_len=max(lens) if i % 2 else None))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d,lens", [(2, 1, 128, [2500]), (2, 2, 64, [1200, 3, 700, 0, 129]), (1, 1, 80, [1, 1999]),
                                           (2, 1, 256, [640])])
def test_linear_attention_of_long_prompts(dtype, nq, nkv, d, lens):
  c = _Call(dtype, nq, nkv, d, lens, seed=3, behind=2)
  c.check(*c.run())


def test_linear_attention_of_many_requests():
  g = torch.Generator().manual_seed(5)
  lens = torch.randint(0, 40, (150,), generator=g).tolist()
  c = _Call(torch.bfloat16, 4, 2, 32, lens, seed=4)
  c.check(*c.run(max_len=40))
  c.check(*c.run())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", SHAPES)
def test_linear_attention_step(dtype, nq, nkv, d):
  for B in (1, 3, 70):
    c = _Call(dtype, nq, nkv, d, [1] * B, seed=B)
    c.check(*c.run(step=True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_attention_step_of_many_requests(dtype):
  """So many states that they are read past the caches."""
  c = _Call(dtype, 4, 2, 128, [1] * 530, seed=6)
  c.check(*c.run(step=True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("log_decay", [[float("-inf"), 0.0], [-30.0, -1e-6], [-200.0, 0.01]])
def test_linear_attention_at_the_ends_of_the_decay(dtype, log_decay):
  """No memory at all, no forgetting, powers that leave the range of 32 bits, a state that grows."""
  c = _Call(dtype, 4, 2, 64, [150, 1, 64], seed=7, log_decay=log_decay)
  c.check(*c.run())
  c = _Call(dtype, 4, 2, 64, [1] * 5, seed=8, log_decay=log_decay)
  c.check(*c.run(step=True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("part,value", [("v", float("inf")), ("v", float("nan")), ("k", float("-inf")), ("k", float("nan")),
                                        ("q", float("nan")), ("q", float("inf"))])
@pytest.mark.parametrize("d", [64, 80])
def test_linear_attention_keeps_what_is_not_finite_to_where_it_belongs(dtype, part, value, d):
  """A value that is not finite makes what depends on it not finite (later tokens of its request in its head, or the
  query's own output), and nothing else: no earlier token, no other head or request."""
  for at in (0, 70, 129):
    c = _Call(dtype, 4, 2, d, [40, 130, 20], seed=9)
    t = c.cu[1] + at
    c.parts(c.qkv)["qkv".index(part)][t, d + 3 if part == "q" else 3] = value
    want, want_state = c.want()
    out, state = c.run()
    ok = want.isfinite()
    assert torch.equal(out.isfinite(), ok) and torch.equal(state.isfinite(), want_state.isfinite())
    assert float((out.double() - want)[ok].norm() / want[ok].norm()) <= max(torch.finfo(dtype).eps / 2, 2e-6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_attention_with_a_state_row_that_does_not_exist(dtype):
  from miniinfer_amd.kernels import ops
  c = _Call(dtype, 4, 2, 64, [100, 3, 40], seed=11)
  qkv, state, rows, cu, g = c.device()
  rows[1] = 99
  out = torch.zeros(c.T, 4 * 64, dtype=dtype, device=DEV)
  ops.linear_attention(*c.parts(qkv), 4, 2, 64, out, state, rows, cu, g, c.scale)
  assert bool(out[100:103].isnan().all()) and bool(out[:100].isfinite().all()) and bool(out[103:].isfinite().all())
  assert torch.equal(state[c.rows[1]].cpu(), c.state[c.rows[1]])
  rows[:] = -1
  out.zero_()
  ops.linear_attention_step(*c.parts(qkv[:3]), 4, 2, 64, out[:3], state, rows, g, c.scale)
  assert bool(out[:3].isnan().all()) and not bool(out[3:].any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens", [[100, 3, 40, 70], [1, 600, 3, 400]])
def test_requests_on_the_idle_row_start_from_nothing_and_leave_nothing(dtype, lens):
  """Any number of them in a call, beside requests with states of their own, whole and in segments."""
  from miniinfer_amd.kernels import ops
  c = _Call(dtype, 4, 2, 64, lens, seed=31)
  idle = c.state.shape[0] - 1
  c.rows = [0, idle, 1, idle]
  c.state[idle] = float("nan")                      # nobody reads it
  qkv, state, rows, cu, g = c.device()
  out = torch.full((c.T, 4 * 64), 7.0, dtype=dtype, device=DEV)
  ops.linear_attention(*c.parts(qkv), 4, 2, 64, out, state, rows, cu, g, c.scale, idle_row=idle)
  assert bool(state[idle].isnan().all())
  # the same with a row of zeros for each
  alone = _Call(dtype, 4, 2, 64, lens, seed=31)
  alone.rows = [0, 2, 1, 3]
  alone.state = c.state.clone()
  alone.state[2:4] = 0.0
  alone.state = alone.state[:4]
  got = torch.cat([state[:2].cpu(), alone.run()[1][2:4]])
  alone.check(out.cpu(), got)
  step = torch.full((4, 4 * 64), 7.0, dtype=dtype, device=DEV)
  ops.linear_attention_step(*c.parts(qkv[:4]), 4, 2, 64, step, state, rows, g, c.scale, idle_row=idle)
  assert bool(step.isfinite().all()) and bool(state[idle].isnan().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_attention_with_strides(dtype):
  """Rows of q, k, v and out in wider buffers at odd offsets, states in every second row of a larger buffer."""
  from miniinfer_amd.kernels import ops
  nq, nkv, d = 4, 2, 40
  c = _Call(dtype, nq, nkv, d, [70, 2], seed=12)
  qkv, state, rows, cu, g = c.device()
  wide = [torch.zeros(c.T, p.shape[1] + 7, dtype=dtype, device=DEV) for p in c.parts(qkv)]
  parts = [w[:, 3:3 + p.shape[1]] for w, p in zip(wide, c.parts(qkv))]
  for p, x in zip(parts, c.parts(qkv)):
    p.copy_(x)
  big = torch.zeros(2 * state.shape[0], nkv, d, d, device=DEV)
  big[::2] = state
  room = torch.full((c.T, nq * d + 5), 7.0, dtype=dtype, device=DEV)
  out = room[:, 1:1 + nq * d]
  ops.linear_attention(*parts, nq, nkv, d, out, big[::2], rows, cu, g, c.scale)
  c.check(out.cpu(), big[::2].cpu())
  assert not bool(big[1::2].any()) and bool((room[:, 0] == 7.0).all()) and bool((room[:, 1 + nq * d:] == 7.0).all())
  first = [p[:2] for p in parts]
  s2 = torch.zeros_like(big)
  s2[::2] = state
  step = _Call(dtype, nq, nkv, d, [1, 1], seed=12)
  step.qkv, step.state, step.rows = c.qkv[:2], c.state, c.rows
  ops.linear_attention_step(*first, nq, nkv, d, out[:2], s2[::2], rows, g, c.scale)
  step.T = 2
  step.check(out[:2].cpu(), s2[::2].cpu())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_prompt_in_portions_and_single_tokens(dtype):
  """The state that one call leaves is what the next goes on from, whichever form the tokens went through."""
  from miniinfer_amd.kernels import ops
  c = _Call(dtype, 4, 2, 64, [300], seed=13)
  qkv, state, rows, cu, g = c.device()
  out = torch.full((300, 4 * 64), 7.0, dtype=dtype, device=DEV)
  at = 0
  for n in (1, 130, 1, 1, 64, 3, 90, 10):
    part = [p[at:at + n] for p in c.parts(qkv)]
    if n == 1:
      ops.linear_attention_step(*part, 4, 2, 64, out[at:at + 1], state, rows, g, c.scale)
    else:
      ops.linear_attention(*part, 4, 2, 64, out[at:at + n], state, rows, torch.tensor([0, n], dtype=torch.int32, device=DEV),
                           g, c.scale)
    at += n
  assert at == 300
  c.check(out.cpu(), state.cpu())


def test_linear_attention_gives_the_same_bits_again():
  c = _Call(torch.bfloat16, 4, 2, 128, [2000, 5], seed=14)
  a, b = c.run(), c.run()
  assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_linear_attention_on_another_stream_and_in_graphs():
  """Two captured calls that live side by side, replayed in turn with eager work between."""
  from miniinfer_amd.kernels import ops
  cs = [_Call(torch.bfloat16, 4, 2, 64, lens, seed=20 + i) for i, lens in enumerate(([700, 9], [260]))]
  want = [c.run() for c in cs]
  held = []
  side = torch.cuda.Stream()
  for c in cs:
    qkv, state, rows, cu, g = c.device()
    start = state.clone()
    out = torch.empty(c.T, 4 * 64, dtype=c.dtype, device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      ops.linear_attention(*c.parts(qkv), 4, 2, 64, out, state, rows, cu, g, c.scale)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), want[len(held)][0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      state.copy_(start)
      ops.linear_attention(*c.parts(qkv), 4, 2, 64, out, state, rows, cu, g, c.scale)
    held.append((graph, out, state, qkv, rows, cu, g, start))
  for turn in range(3):
    for (graph, out, state, *_), w in zip(held, want):
      out.zero_()
      graph.replay()
      torch.cuda.synchronize()
      assert torch.equal(out.cpu(), w[0]) and torch.equal(state.cpu(), w[1])
      cs[turn % 2].run()


def test_linear_attention_of_a_state_beyond_32_bit_offsets():
  """A buffer of more than 2^31 elements: the last row is read and written where it is."""
  from miniinfer_amd.kernels import ops
  nq, nkv, d = 2, 2, 256
  rows_n = (2 ** 31) // (nkv * d * d) + 3
  state = torch.zeros(rows_n, nkv, d, d, device=DEV)
  c = _Call(torch.bfloat16, nq, nkv, d, [5, 1], seed=15, spare_rows=0)
  qkv, small, _, cu, g = c.device()
  at = [rows_n - 1, rows_n - 2]
  for i, r in enumerate(at):
    state[r] = small[c.rows[i]]
  out = torch.full((c.T, nq * d), 7.0, dtype=torch.bfloat16, device=DEV)
  ops.linear_attention(*c.parts(qkv), nq, nkv, d, out, state, torch.tensor(at, dtype=torch.int32, device=DEV), cu, g, c.scale)
  back = torch.empty_like(small)
  for i, r in enumerate(at):
    back[c.rows[i]] = state[r]
  c.check(out.cpu(), back.cpu())
  assert float(state[:rows_n - 2].abs().max()) == 0.0


# --------------------------------------------------------------------------------------------------- beam selection

def _beam_reference(logits, scores, W, count):
  """Every candidate's score in 64 bits, sorted (stable, so equal ones by beam and token)."""
  x = logits.double().cpu()
  x = torch.where(x.isnan(), float("-inf"), x)
  m = x.amax(-1, keepdim=True)
  y = torch.where(x == m, 0.0, x - m)
  s = scores.double().cpu()
  p = y - y.exp().sum(-1, keepdim=True).log() + s[:, None]
  p = torch.where((m == float("-inf")) | ~(s[:, None] > float("-inf")), float("-inf"), p)
  V = x.shape[1]
  value, index = p.view(-1, W * V).sort(dim=-1, descending=True, stable=True)
  return value[:, :count], (index[:, :count] // V).int(), (index[:, :count] % V).int()


def _check_beam(logits, scores, W, count):
  from miniinfer_amd.kernels import ops
  got = ops.beam_select(logits, scores, W, count)
  want = _beam_reference(logits, scores, W, count)
  assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
  g, w = got[0].cpu().double(), want[0]
  inf = w.isinf()
  assert torch.equal(g.isinf(), inf) and torch.equal(g[inf], w[inf])
  # 64-bit sums, rounded once to 32 bits
  assert bool(((g - w).abs() <= (U + 1e-9) * w.abs() + 1e-12)[~inf].all())


@pytest.mark.parametrize("G,W,V,count", [(1, 1, 1, 1), (1, 1, 64, 64), (2, 3, 7, 21), (3, 5, 32003, 10), (1, 4, 151936, 8), (5, 2, 1000, 4),
                                         (2, 64, 515, 64), (1, 32, 4097, 64), (40, 1, 50000, 2), (3, 16, 8192, 32),
                                         (70, 4, 129, 8)])
def test_beam_select(G, W, V, count):
  g = torch.Generator().manual_seed(G + W)
  logits = (torch.randn(G * W, V, generator=g) * 2.5).to(DEV)
  scores = (-5 * torch.rand(G * W, generator=g)).to(DEV)
  _check_beam(logits, scores, W, count)
  scores.view(G, W)[:, 1:] = float("-inf")        # the first step of a search
  _check_beam(logits, scores, W, min(count, V))
  _check_beam(logits, scores, W, count)           # (more than the live beam has, where the vocabulary is small)


@pytest.mark.parametrize("V", [5, 300, 20011])
def test_beam_select_orders_equal_scores(V):
  """Few distinct logits, the same in several beams: the lowest beam and token first."""
  g = torch.Generator().manual_seed(2)
  row = torch.randint(0, 3, (1, V), generator=g).float()
  logits = row.expand(8, V).contiguous().to(DEV)
  for scores in (torch.zeros(8), torch.tensor([0.0, -1.0] * 4)):
    for W in (1, 2, 4, 8):
      _check_beam(logits, scores.to(DEV), W, min(64, W * V))
  _check_beam(torch.zeros(4, V, device=DEV), torch.zeros(4, device=DEV), 4, 4)


@pytest.mark.parametrize("V", [9, 5000])
def test_beam_select_with_masked_tokens(V):
  """Masks of -inf, of the type's lowest value, whole rows of either, infinities and NaN."""
  g = torch.Generator().manual_seed(3)
  base = torch.randn(4, V, generator=g)
  scores = torch.tensor([-1.0, -2.0, -1.5, -0.5])
  inf, low = float("inf"), torch.finfo(torch.float32).min
  cases = []
  for fill in (-inf, low):
    x = base.clone()
    x[:, 3:] = fill                      # few tokens are left
    cases.append(x)
    x = base.clone()
    x[1] = fill                          # nothing is left of a row
    cases.append(x)
    cases.append(torch.full_like(base, fill))
  x = base.clone()
  x[2, 4] = x[2, 7] = inf                # two tokens share a row's mass
  x[0, 1] = float("nan")
  x[3] = float("nan")
  cases.append(x)
  for x in cases:
    for count in (1, 5, 16):
      _check_beam(x.to(DEV), scores.to(DEV), 4, count)
      _check_beam(x.to(DEV), scores.to(DEV), 2, min(count, 2 * V))
  s = scores.clone()
  s[:] = -inf
  _check_beam(base.to(DEV), s.to(DEV), 4, 8)
  s[1] = float("nan")
  _check_beam(base.to(DEV), s.to(DEV), 4, 8)


def test_beam_select_finds_the_best_wherever_they_lie():
  """All the best of a row side by side, one to every part of it, in its last tokens; and a row in falling order."""
  V, count = 30011, 32
  rows = []
  for place in (torch.arange(count) + 777, torch.arange(count) * (V // count), V - 1 - torch.arange(count), torch.arange(count) * 64):
    x = torch.randn(V, generator=torch.Generator().manual_seed(6))
    x[place] = 20 + torch.arange(count) * 0.01
    rows.append(x)
  rows.append(torch.linspace(3, -3, V))
  rows.append(torch.linspace(-3, 3, V))
  logits = torch.stack(rows).to(DEV)
  for W in (1, 2, 3, 6):
    _check_beam(logits, torch.zeros(6, device=DEV), W, count)


def test_beam_select_of_strided_rows():
  g = torch.Generator().manual_seed(4)
  for shift, V in ((1, 1001), (3, 4096), (2, 151)):
    wide = torch.randn(6, V + 9, generator=g).to(DEV)
    _check_beam(wide[:, shift:shift + V], torch.zeros(6, device=DEV), 3, 7)
    _check_beam(wide[::2, shift:shift + V], torch.zeros(3, device=DEV), 3, 7)


def test_beam_select_of_no_group_and_in_a_graph():
  from miniinfer_amd.kernels import ops
  s, b, t = ops.beam_select(torch.zeros(0, 50, device=DEV), torch.zeros(0, device=DEV), 4, 8)
  assert s.shape == b.shape == t.shape == (0, 8)
  g = torch.Generator().manual_seed(8)
  logits, scores = torch.randn(8, 20000, generator=g).to(DEV), torch.zeros(8, device=DEV)
  ops.beam_select(logits, scores, 4, 8)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    got = ops.beam_select(logits, scores, 4, 8)
  for turn in range(3):
    logits.copy_(torch.randn(8, 20000, generator=g))
    graph.replay()
    torch.cuda.synchronize()
    want = _beam_reference(logits, scores, 4, 8)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
    _check_beam(logits, scores, 2, 8)


# -------------------------------------------------------------------------------------------------------- row moves

def _check_move(buffers, src, dst):
  from miniinfer_amd.kernels import ops
  want = []
  for t in buffers:
    w = t.clone()
    for s, d in zip(src, dst):
      if 0 <= s < t.shape[1] and 0 <= d < t.shape[1]:
        w[:, d] = t[:, s]
    want.append(w)
  i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
  ops.move_rows(buffers, i32(src), i32(dst))
  for t, w in zip(buffers, want):
    assert torch.equal(t, w)


@pytest.mark.parametrize("dtype,row", [(torch.float32, (4, 16, 16)), (torch.bfloat16, (2, 16, 128)), (torch.uint8, (3,)), (torch.int16, (5, 7)),
                                       (torch.float64, (1,)), (torch.bfloat16, (2, 33)), (torch.uint8, (4099,))])
@pytest.mark.parametrize("L", [1, 3])
def test_move_rows(dtype, row, L):
  g = torch.Generator().manual_seed(1)
  N = 40
  make = lambda: torch.randint(0, 200, (L, N) + row, generator=g).to(dtype).to(DEV)
  perm = torch.randperm(N, generator=g).tolist()
  _check_move([make()], perm, list(range(N)))                       # every row changes its place
  _check_move([make()], [1, 0], [0, 1])
  _check_move([make()], [7] * 11, list(range(11)))                  # forks of one row, itself among them
  _check_move([make()], [5, 6, 7, 39], [6, 7, 5, 0])                # a cycle
  _check_move([make()], [-1, 3, 40, 4, 8], [2, -1, 9, 4, 1000])     # padding and rows that do not exist
  _check_move([make()], [], [])
  _check_move([make(), make()], [3, 9], [9, 10])


def test_move_rows_of_several_buffers_of_their_own_shapes():
  g = torch.Generator().manual_seed(2)
  bufs = [torch.randn(L, N, *row, generator=g).to(DEV) for L, N, row in ((2, 9, (3, 8)), (1, 20, (5,)), (4, 9, (64, 64)), (1, 9, (1,)))]
  _check_move(bufs, [0, 8, 3, 15], [8, 0, 1, 19])                   # (rows 15 and 19 are in the second buffer only)
  _check_move([torch.zeros(0, 5, 8, device=DEV), torch.randn(2, 5, 8, device=DEV), torch.zeros(2, 5, 0, device=DEV)], [1], [2])


@pytest.mark.parametrize("n", [300, 513, 2049, 5000, 16384])
def test_move_rows_of_long_lists(n):
  g = torch.Generator().manual_seed(n)
  buf = torch.randn(2, n + 100, 36, generator=g).to(DEV)
  _check_move_fast(buf, torch.randperm(n + 100, generator=g)[:n], torch.randperm(n + 100, generator=g)[:n])


def _check_move_fast(buf, src, dst):
  from miniinfer_amd.kernels import ops
  want = buf.clone()
  want[:, dst.to(DEV)] = buf[:, src.to(DEV)]
  ops.move_rows(buf, src.to(torch.int32).to(DEV), dst.to(torch.int32).to(DEV))
  assert torch.equal(buf, want)


def test_move_rows_with_strides():
  g = torch.Generator().manual_seed(3)
  big = torch.randn(6, 10, 12, generator=g).to(DEV)
  keep = big.clone()
  view = big[::2, 1::3, 2:9]
  _check_move([view], [0, 1, 2], [1, 2, 0])
  mask = torch.ones_like(big, dtype=torch.bool)
  mask[::2, 1::3, 2:9] = False
  assert torch.equal(big[mask], keep[mask])
  rows_first = torch.randn(7, 3, 16, generator=g).to(DEV)
  _check_move([rows_first.transpose(0, 1)], [0, 6], [6, 0])


def test_move_rows_beyond_32_bit_offsets_and_in_a_graph():
  from miniinfer_amd.kernels import ops
  buf = torch.zeros(2, 70000, 20000, dtype=torch.uint8, device=DEV)     # 2.8 GB
  buf[:, 69999] = 3
  buf[:, 1] = 5
  i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
  ops.move_rows(buf, i32([69999, 1]), i32([1, 69998]))
  assert bool((buf[:, 1] == 3).all()) and bool((buf[:, 69998] == 5).all()) and int(buf[:, 2:69998].max()) == 0
  small = torch.randn(3, 8, 64, device=DEV)
  src, dst = i32([1, 0, 3]), i32([0, 1, 7])
  want = small.clone()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    ops.move_rows(small, src, dst)
  for _ in range(3):
    want[:, dst.long()] = want[:, src.long()]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(small, want)
