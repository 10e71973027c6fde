"""Outputs and buffers that share memory with others, wherever they begin, are turned down on the host; parts of one buffer
that lie between one another are not (a call that is taken ends at "run on the GPU only" here)."""

import itertools

import pytest
import torch

from miniinfer_amd.kernels import ops
from miniinfer_amd.kernels.ops import KernelError

NQ, NKV, D = 2, 1, 16


def _calls(q, k, v, out):
  T = q.shape[0]
  state, rows, g = torch.zeros(T + 1, NKV, D, D), torch.zeros(T, dtype=torch.int32), torch.zeros(NKV)
  yield lambda: ops.linear_attention(q, k, v, NQ, NKV, D, out, state, rows[:1], torch.zeros(2, dtype=torch.int32), g, 1.0)
  yield lambda: ops.linear_attention_step(q, k, v, NQ, NKV, D, out, state, rows, g, 1.0)


def _shares(out, *others):
  """By the places of all elements."""
  places = lambda t: set((t.data_ptr() + t.element_size() * sum(i * s for i, s in zip(at, t.stride())))
                         for at in itertools.product(*map(range, t.shape)))
  mine = places(out)
  return any(mine & places(t) for t in others)


@pytest.mark.parametrize("T", [1, 2, 5])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_attention_refuses_an_out_inside_its_inputs(T, dtype):
  n, m = NQ * D, NKV * D
  wide = torch.zeros(T + 2, 2 * n + 2 * m, dtype=dtype)
  flat = torch.zeros(4 * (T + 1) * (n + m), dtype=dtype)
  seen = set()
  for first in range(0, n + 2 * m + 1, 8):               # out in columns from `first` on of the buffer that q | k | v are parts of
    for down in (0, 1):
      q, k, v = wide[:T, :n], wide[:T, n:n + m], wide[:T, n + m:n + 2 * m]
      out = wide[down:down + T, first:first + n]
      shares = _shares(out, q, k, v)
      seen.add(shares)
      for call in _calls(q, k, v, out):
        with pytest.raises(KernelError, match="shares memory" if shares else "GPU only"):
          call()
  assert seen == {True, False}
  for at in (0, 8, T * n - 8, T * n, T * (n + m) - 8, T * (n + 2 * m) - 8, T * (n + 2 * m)):    # dense tensors of one buffer
    q, k, v = flat[:T * n].view(T, n), flat[T * n:T * (n + m)].view(T, m), flat[T * (n + m):T * (n + 2 * m)].view(T, m)
    out = flat[at:at + T * n].view(T, n)
    for call in _calls(q, k, v, out):
      with pytest.raises(KernelError, match="shares memory" if _shares(out, q, k, v) else "GPU only"):
        call()


def test_an_out_after_the_parts_of_a_wider_buffer_is_taken():
  T, n, m = 4, NQ * D, NKV * D
  wide = torch.zeros(T, 2 * n + 2 * m)
  q, k, v, out = wide[:, :n], wide[:, n:n + m], wide[:, n + m:n + 2 * m], wide[:, n + 2 * m:]
  for call in _calls(q, k, v, out):
    with pytest.raises(KernelError, match="GPU only"):
      call()
