"""What linear attention, beam selection and row moves refuse: every refusal is an error on the host, before a kernel is
launched, so these run without a GPU (a call with fitting arguments ends at "run on the GPU only")."""

import pytest
import torch

from miniinfer_amd.kernels import ops
from miniinfer_amd.kernels.ops import KernelError

NQ, NKV, D, T, B = 4, 2, 16, 6, 2


def _prompt(**change):
  a = dict(q=torch.zeros(T, NQ * D), k=torch.zeros(T, NKV * D), v=torch.zeros(T, NKV * D), nq=NQ, nkv=NKV, d=D,
           out=torch.zeros(T, NQ * D), state=torch.zeros(3, NKV, D, D), state_rows=torch.zeros(B, dtype=torch.int32),
           cu_q=torch.zeros(B + 1, dtype=torch.int32), log_decay=torch.zeros(NKV), scale=1.0)
  a.update(change)
  return ops.linear_attention(**a)


def _step(**change):
  a = dict(q=torch.zeros(T, NQ * D), k=torch.zeros(T, NKV * D), v=torch.zeros(T, NKV * D), nq=NQ, nkv=NKV, d=D,
           out=torch.zeros(T, NQ * D), state=torch.zeros(3, NKV, D, D), state_rows=torch.zeros(T, dtype=torch.int32),
           log_decay=torch.zeros(NKV), scale=1.0)
  a.update(change)
  return ops.linear_attention_step(**a)


@pytest.mark.parametrize("call", [_prompt, _step])
@pytest.mark.parametrize("change,message", [
  ({}, "GPU only"),
  (dict(nq=3), "multiple"),
  (dict(nkv=0), "multiple"),
  (dict(d=12), "head size"),
  (dict(d=264), "head size"),
  (dict(q=torch.zeros(T, NQ * D - 1)), "q "),
  (dict(k=torch.zeros(T - 1, NKV * D)), "k "),
  (dict(v=torch.zeros(T, NKV * D, dtype=torch.bfloat16)), "v "),
  (dict(q=torch.zeros(T, NQ * D, dtype=torch.float16)), "not supported"),
  (dict(q=torch.zeros(NQ * D, T).t()), "q "),
  (dict(out=torch.zeros(T, NQ * D + 1)), "out "),
  (dict(out=torch.zeros(1, NQ * D).expand(T, NQ * D)), "overlap"),
  (dict(state=torch.zeros(3, NKV, D, D, dtype=torch.bfloat16)), "states"),
  (dict(state=torch.zeros(3, NKV, D, D + 4)), "states"),
  (dict(state=torch.zeros(3, NKV, D, D).transpose(2, 3)), "states"),
  (dict(state=torch.zeros(1, NKV, D, D).expand(3, NKV, D, D)), "states"),
  (dict(state=torch.zeros(4 + 3 * NKV * D * D)[1:1 + 3 * NKV * D * D].view(3, NKV, D, D)), "16 bytes"),
  (dict(state_rows=torch.zeros(B, dtype=torch.int64)), "int32"),
  (dict(state_rows=torch.zeros(B + 1, dtype=torch.int32)), "requests|state rows"),
  (dict(log_decay=torch.zeros(NKV + 1)), "log_decay"),
  (dict(log_decay=torch.zeros(NKV, dtype=torch.float64)), "log_decay"),
])
def test_linear_attention_refuses(call, change, message):
  with pytest.raises(KernelError, match=message):
    call(**change)


def test_linear_attention_refuses_other_integers():
  with pytest.raises(KernelError, match="int32"):
    _prompt(cu_q=torch.zeros(B + 1, dtype=torch.int64))
  with pytest.raises(KernelError, match="entries"):
    _prompt(cu_q=torch.zeros(B, dtype=torch.int32))


@pytest.mark.parametrize("args,message", [
  ((torch.zeros(4, 10), torch.zeros(4), 2, 3), "GPU only"),
  ((torch.zeros(4, 10).double(), torch.zeros(4), 2, 3), "float32"),
  ((torch.zeros(4, 10, dtype=torch.bfloat16), torch.zeros(4), 2, 3), "float32"),
  ((torch.zeros(10, 4).t(), torch.zeros(4), 2, 3), "dense"),
  ((torch.zeros(1, 10).expand(4, 10), torch.zeros(4), 2, 3), "overlap"),
  ((torch.zeros(4, 10), torch.zeros(4), 3, 3), "groups"),
  ((torch.zeros(4, 10), torch.zeros(4), 0, 3), "groups"),
  ((torch.zeros(4, 0), torch.zeros(4), 2, 3), "groups"),
  ((torch.zeros(4, 10), torch.zeros(5), 2, 3), "scores"),
  ((torch.zeros(4, 10), torch.zeros(4).double(), 2, 3), "scores"),
  ((torch.zeros(4, 10), torch.zeros(4), 2, 0), "candidates"),
  ((torch.zeros(4, 10), torch.zeros(4), 2, 21), "candidates"),
  ((torch.zeros(4, 100), torch.zeros(4), 2, 65), "candidates"),
  ((torch.zeros(65, 100), torch.zeros(65), 65, 4), "beams"),
])
def test_beam_select_refuses(args, message):
  with pytest.raises(KernelError, match=message):
    ops.beam_select(*args)


def _i32(*x):
  return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("buffers,src,dst,message", [
  (torch.zeros(2, 5, 4), _i32(0), _i32(1), "GPU only"),
  ([], _i32(0), _i32(1), "buffers"),
  ([torch.zeros(2, 5, 4)] * 9, _i32(0), _i32(1), "buffers"),
  (torch.zeros(5), _i32(0), _i32(1), "layers"),
  (torch.zeros(2, 5, 4, 6).transpose(2, 3), _i32(0), _i32(1), "dense"),
  (torch.zeros(2, 1, 4).expand(2, 5, 4), _i32(0), _i32(1), "overlap"),
  (torch.zeros(1, 5, 4).expand(2, 5, 4), _i32(0), _i32(1), "overlap"),
  (torch.zeros(2, 5, 4), _i32(0, 1), _i32(1), "sources"),
  (torch.zeros(2, 5, 4), torch.zeros(1, dtype=torch.int64), _i32(1), "int32"),
  (torch.zeros(2, 5, 4), _i32(0), torch.zeros(1, dtype=torch.int64), "int32"),
  (torch.zeros(2, 5, 4), torch.zeros(16385, dtype=torch.int32), torch.zeros(16385, dtype=torch.int32), "at most"),
])
def test_move_rows_refuses(buffers, src, dst, message):
  with pytest.raises(KernelError, match=message):
    ops.move_rows(buffers, src, dst)
