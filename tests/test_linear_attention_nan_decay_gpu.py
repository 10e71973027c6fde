"""A decay that is NaN makes its head's outputs and states NaN, as in the recurrence, and no other head's."""

import pytest
import torch

from test_state_operators_gpu import _Call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,step", [([1, 33], False), ([700, 3], False), ([1, 1], True)])
def test_a_decay_that_is_nan(dtype, d, lens, step):
  c = _Call(dtype, 4, 2, d, lens, seed=2, log_decay=[float("nan"), -0.1])
  want, want_state = c.want()
  assert bool(want[:, :2 * d].isnan().all()) and bool(want[:, 2 * d:].isfinite().all())
  out, state = c.run(step=step)
  assert torch.equal(out.isnan(), want.isnan()) and torch.equal(state.isnan(), want_state.isnan())
