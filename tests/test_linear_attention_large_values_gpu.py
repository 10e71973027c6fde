"""Values near the end of the 32-bit range that a head has long forgotten: a power of its decay that has left the range must
not bring them back.  References and tolerances: those of `test_state_operators_gpu`."""

import pytest
import torch

from test_state_operators_gpu import _Call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", [(4, 2, 64), (2, 2, 80), (4, 2, 128), (2, 2, 256)])
@pytest.mark.parametrize("lens,max_len", [([150, 3, 40], 1), ([700, 5], None)])
@pytest.mark.parametrize("where", ["v", "state"])
def test_forgotten_values(dtype, nq, nkv, d, lens, max_len, where):
  c = _Call(dtype, nq, nkv, d, lens, seed=d, log_decay=[-30.0, -2.5])
  if where == "v":
    large = 1e38
    c.parts(c.qkv)[2][:1, :3] = large
  else:
    large = 1e35                        # (q S comes before its decay: d such terms have to stay in the range)
    c.state[c.rows[0], :, :, 2] = large
  out, state = c.run(max_len=max_len)
  want, want_state = c.want()
  mag, mag_state = c.magnitudes()
  n, u = max(lens), 2.0 ** -24
  half = torch.finfo(dtype).eps / 2
  # (a power is right to 2^-22 of itself down to the 32-bit range's last numbers, 2^-149 apart: `large` of those)
  last = 2.0 ** -149 * large * d
  bound = half * want.abs() + (2.0 ** -22 + (4 * n + d + 8) * u) * mag * (1 + half) + last * 4
  if dtype is torch.bfloat16 and where == "v":
    # (bfloat16's last numbers are 2^-133 apart, which is what a weighted product of query and key can lose, times one value)
    bound = bound + 2.0 ** -133 * large
  assert bool(((out.double() - want).abs() <= bound).all())
  assert bool(((state.double() - want_state).abs() <= (2.0 ** -22 + (4 * n + 8) * u) * mag_state + last).all())
