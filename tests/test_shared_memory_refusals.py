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


def _move(*buffers):
  i = torch.zeros(1, dtype=torch.int32)
  ops.move_rows(list(buffers), i, i)


def _pairs():
  t = torch.zeros(3, 8, 4, 6)
  kv = torch.zeros(3, 2, 8, 4)                                   # [layers, keys and values, rows, ...]
  by_row = torch.zeros(3, 8, 2, 4)                               # a row's keys, then its values
  flat = torch.zeros(400)
  for a, b in ((t, t[:, 1:]), (t, t[1:]), (t[:2], t[1:]), (t[:, :5], t[:, 4:]), (t[:, ::2], t[:, 2::2]), (t[:, ::3], t[:, 1::2]),
               (flat[:80].view(2, 5, 8), flat[79:159].view(2, 5, 8)), (t[0:1], t[:, 3:4]), (by_row[:, :, 0, :3], by_row[:, :, 0, 2:]),
               (kv[:, 0], kv[:, :, 1])):
    yield a, b, True
  for a, b in ((t[:1], t[1:]), (t[:, :5], t[:, 5:]), (t[:, ::2], t[:, 1::2]), (t[::2], t[1::2]), (kv[:, 0], kv[:, 1]),
               (by_row[:, :, 0], by_row[:, :, 1]), (by_row[:, :, 0, :2], by_row[:, :, 0, 2:]),
               (flat[:80].view(2, 5, 8), flat[80:160].view(2, 5, 8)), (t[:1, :1], t[1:2, 1:2]), (t[:, 0:1], t[:, 7:]),
               (kv[:, 0].transpose(0, 1), kv[:, 1].transpose(0, 1))):
    yield a, b, False


@pytest.mark.parametrize("case", range(21))
@pytest.mark.parametrize("turned", [False, True])
def test_move_rows_refuses_buffers_that_share_memory(case, turned):
  a, b, shares = list(_pairs())[case]
  assert _shares(a, b) == shares
  with pytest.raises(KernelError, match="share memory|twice" if shares else "GPU only"):
    _move(*((b, a) if turned else (a, b)))
  with pytest.raises(KernelError, match="share memory|twice" if shares else "GPU only"):
    _move(torch.zeros(2, 3), a, torch.zeros(1, 4), b)


def test_move_rows_takes_no_buffers_that_share_memory():
  """Any two views of one buffer."""
  import random
  rng = random.Random(3)
  flat = torch.zeros(600)
  taken = refused = 0
  for _ in range(4000):
    views = []
    for _ in range(2):
      row, layers, rows = rng.randint(1, 5), rng.randint(1, 4), rng.randint(1, 5)
      per_row = row + rng.choice([0, 0, 1, 3, 7])
      per_layer = per_row * rows + rng.choice([0, 0, 1, 4, per_row])
      if rng.random() < 0.3:
        per_layer = row + rng.choice([0, 1, 3])
        per_row = per_layer * layers + rng.choice([0, 2])
      views.append(flat.as_strided((layers, rows, row), (per_layer, per_row, 1), rng.randint(0, 200)))
    shares = _shares(*views)
    with pytest.raises(KernelError) as e:
      _move(*views)
    if shares:
      assert "share memory" in str(e.value) or "twice" in str(e.value)
    taken, refused = taken + ("GPU only" in str(e.value)), refused + ("GPU only" not in str(e.value))
  assert taken > 500 and refused > 500
