"""Linear attention of inputs whose every product and sum is a 32-bit number: nothing is left to round but the output.

Large terms that cancel leave what their last bits say, so a form that gives its products fewer bits of a state or of a
weighted product of query and key than 32-bit numbers have (24) answers with zeros or with noise here.  The decay is 1,
whose powers are exact; results are therefore held to the 64-bit recurrence's, rounded once, bit by bit."""

import pytest
import torch

from test_state_operators_gpu import DEV, _recurrence

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -20


def _check(dtype, nq, nkv, d, lens, q, k, v, state, forms=("prompt",)):
  from miniinfer_amd.kernels import ops
  T, B = sum(lens), len(lens)
  cu = [sum(lens[:i]) for i in range(B + 1)]
  qkv = torch.cat([x.reshape(T, -1) for x in (q, k, v)], 1)
  assert torch.equal(qkv.to(dtype).double(), qkv.double())              # the inputs are numbers of this type
  g = torch.zeros(nkv)
  split = lambda x: (x[:, :nq * d], x[:, nq * d:(nq + nkv) * d], x[:, (nq + nkv) * d:])
  want, want_state = _recurrence(*split(qkv), state, list(range(B)), cu, g, 1.0, nq, nkv, d)
  assert torch.equal(want_state.float().double(), want_state)
  for form in forms:
    dev = qkv.to(dtype).to(DEV)
    s = state.to(DEV)
    out = torch.full((T, nq * d), 7.0, dtype=dtype, device=DEV)
    rows = torch.arange(B, dtype=torch.int32, device=DEV)
    if form == "prompt":
      ops.linear_attention(*split(dev), nq, nkv, d, out, s, rows, torch.tensor(cu, dtype=torch.int32, device=DEV), g.to(DEV), 1.0)
    else:
      for t in range(max(lens)):
        at = [b for b in range(B) if t < lens[b]]
        tok = torch.tensor([cu[b] + t for b in at], device=DEV)
        step = torch.empty((len(at), nq * d), dtype=dtype, device=DEV)
        ops.linear_attention_step(*split(dev[tok]), nq, nkv, d, step, s, rows[at], g.to(DEV), 1.0)
        out[tok] = step
    # (twice: to float32 and to the type, as the kernels do; both exact or the last one a rounding of an exact number)
    assert torch.equal(want.float().double(), want)
    assert torch.equal(out.cpu(), want.to(dtype)), form
    assert torch.equal(s.cpu().double(), want_state), form


SHAPES = [(2, 1, 16), (4, 2, 64), (2, 2, 80), (4, 2, 128), (1, 1, 200), (2, 1, 256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", SHAPES)
@pytest.mark.parametrize("lens", [[1], [33, 1, 70], [900]])
def test_what_a_state_gives_when_its_rows_cancel(dtype, nq, nkv, d, lens):
  """q S = (1 + 2^-9 + m 2^-20) - (1 + 2^-9)."""
  T, B = sum(lens), len(lens)
  m = 1 + torch.arange(d) % 15
  state = torch.zeros(B, nkv, d, d)
  state[:, :, 3] = 1 + 2.0 ** -9 + m * UNIT
  state[:, :, d - 2] = 1 + 2.0 ** -9
  q = torch.zeros(T, nq, d)
  q[:, :, 3] = 1.0
  q[:, :, d - 2] = -1.0
  none = torch.zeros(T, nkv, d)
  _check(dtype, nq, nkv, d, lens, q, none, none, state, ("prompt", "step") if max(lens) < 100 else ("prompt",))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", SHAPES)
@pytest.mark.parametrize("lens", [[2], [33, 1, 70], [900]])
def test_what_tokens_give_when_their_values_cancel(dtype, nq, nkv, d, lens):
  """(q k0) v - (q k1) v with q k0 = 1 + 2^-9 + m 2^-20, q k1 = 1 + 2^-9, for pairs of tokens in several chunks."""
  T, B = sum(lens), len(lens)
  q = torch.zeros(T, nq, d)
  q[:, :, 0] = 1.0
  q[:, :, 5] = 2.0 ** -9
  q[:, :, d - 1] = ((1 + torch.arange(T) % 15) * 2.0 ** -11)[:, None]
  k, v = torch.zeros(T, nkv, d), torch.zeros(T, nkv, d)
  first = 0
  for n in lens:
    for at in (0, 40, 70):                # (three pairs: sums of 23 bits and fewer)
      if at + 1 < n:
        k[first + at, :, [0, 5]] = 1.0
        k[first + at, :, d - 1] = 2.0 ** -9
        k[first + at + 1, :, [0, 5]] = 1.0
        v[first + at] = 1.0 + torch.arange(d) % 3
        v[first + at + 1] = -v[first + at]
    first += n
  _check(dtype, nq, nkv, d, lens, q, k, v, torch.zeros(B, nkv, d, d), ("prompt", "step") if max(lens) < 100 else ("prompt",))
