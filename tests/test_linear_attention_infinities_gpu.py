"""Infinities in linear attention: an infinite element of a state or of a value stays what it is in the state, as in the
recurrence, whichever form the tokens go through, also where a decay's power has left the range of 32 bits."""

import pytest
import torch

from test_state_operators_gpu import _Call

pytestmark = pytest.mark.gpu

INF = float("inf")
SHAPES = [(2, 2, 16), (4, 2, 64), (2, 2, 80), (4, 2, 128), (2, 2, 256)]
DECAYS = [None, [-30.0, -2.5], [-0.3, 0.0]]


def _same_kinds(got, want):
  """NaN, infinities of either sign and finite numbers in the same places."""
  return torch.equal(got.isnan(), want.isnan()) and torch.equal(got == INF, want == INF) and torch.equal(got == -INF, want == -INF)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", SHAPES)
@pytest.mark.parametrize("lens,max_len", [([1, 33, 150], 1), ([700, 3], None)])
@pytest.mark.parametrize("log_decay", DECAYS)
def test_infinite_states_stay_infinite(dtype, nq, nkv, d, lens, max_len, log_decay):
  c = _Call(dtype, nq, nkv, d, lens, seed=d, log_decay=log_decay)
  for b, row in enumerate(c.rows):
    c.state[row, 0, 5 + b, 3] = INF
    c.state[row, nkv - 1, d - 1, d - 2] = -INF
  want, want_state = c.want()
  assert int(want_state.isinf().sum()) == 2 * len(lens) and not bool(want_state.isnan().any())
  out, state = c.run(max_len=max_len)
  assert _same_kinds(state, want_state) and _same_kinds(out, want)
  ok = want.isfinite()
  # (as a whole: half a step of the output's type, or of a 32-bit sum's some hundred roundings, which mostly cancel)
  assert float((out.double() - want)[ok].norm() / want[ok].norm()) <= max(torch.finfo(dtype).eps / 2, 2e-6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", SHAPES)
@pytest.mark.parametrize("lens,max_len,at", [([40, 150], 1, 0), ([40, 150], 1, 149), ([9, 700], None, 100), ([9, 700], None, 699)])
@pytest.mark.parametrize("log_decay", DECAYS)
def test_infinite_values_leave_infinite_states(dtype, nq, nkv, d, lens, max_len, at, log_decay):
  """k is nowhere zero, so the state's column is infinite with the sign of k."""
  c = _Call(dtype, nq, nkv, d, lens, seed=d + 1, log_decay=log_decay)
  k, v = c.parts(c.qkv)[1:]
  k[k == 0] = 1.0
  v[c.cu[1] + at, 3] = INF
  v[c.cu[1] + at, nkv * d - 1] = -INF
  want, want_state = c.want()
  assert int(want_state.isinf().sum()) == 2 * d and not bool(want_state.isnan().any())
  out, state = c.run(max_len=max_len)
  assert _same_kinds(state, want_state) and torch.equal(out.isfinite(), want.isfinite())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("log_decay", DECAYS)
def test_single_tokens_keep_infinities(dtype, log_decay):
  c = _Call(dtype, 4, 2, 64, [1] * 3, seed=3, log_decay=log_decay)
  c.state[c.rows[0], 0, 5, 3] = INF
  c.state[c.rows[2], 1, 63, 62] = -INF
  k, v = c.parts(c.qkv)[1:]
  k[k == 0] = 1.0
  v[1, 64 + 7] = INF
  want, want_state = c.want()
  out, state = c.run(step=True)
  assert _same_kinds(state, want_state) and _same_kinds(out, want)
