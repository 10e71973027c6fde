"""Linear attention with a decay for each head: a mixer whose memory of a request is a state of fixed size, one matrix
[head_dim, head_dim] in 32-bit for each kv head, in the request's state slot.

The order of operations is that of the paged attention: one fused projection (rows q | k | v), per-head RMS norm of q and k
and their rotation where the spec asks for them, then S_t = a S_{t-1} + k_t v_t^T, o_t = scale q_t S_t, then the output
projection.  Prompt portions go through the chunked kernel, single tokens through the recurrent one."""

from __future__ import annotations

import torch

from ..kernels import ops
from .attention import PagedAttention
from .base import BuildContext, FixedState, register_mixer
from .linear import PendingLinear, linear


class LinearAttention(PagedAttention):
  kernel_modules = ("linear_attention",)

  def __init__(self, spec, ctx: BuildContext):
    super().__init__(spec, ctx)       # sizes, projections, head norms and the position encoding
    if len(spec.log_decay) != spec.num_kv_heads:
      raise ValueError(f"log_decay has {len(spec.log_decay)} entries for {spec.num_kv_heads} kv heads")
    self.log_decay = torch.tensor(spec.log_decay, dtype=torch.float32, device=ctx.device)

  def cache_requirement(self):
    return FixedState(shape=(self.nkv, self.d, self.d), dtype=torch.float32)

  def workspace_bytes(self, tokens: int, requests: int) -> int:
    itemsize = 2 if self.ctx.dtype == torch.bfloat16 else 4
    return ops.linear_attention_workspace(tokens, requests, self.nkv, self.d, itemsize, ops.compute_units())

  def _rotate(self, qkv: torch.Tensor, ctx) -> None:
    """Head norms and rotation of q and k, in place."""
    nq, nkv, d = self.nq, self.nkv, self.d
    table = self.position.rotary_table()
    q_weight = k_weight = None
    eps = 0.0
    if self.q_norm is not None and self.heads_norm_fused:
      q_weight, k_weight, eps = self.q_norm.weight, self.k_norm.weight, self.q_norm.eps
    elif self.q_norm is not None:
      self._norm_heads(qkv)
    if table is None and q_weight is None:
      return
    if qkv.shape[0] < 32:
      ops.qk_norm_rope_cache(qkv, nq, nkv, d, q_weight, k_weight, eps, table, ctx.positions, None, None, None, 1)
      return
    # many tokens: q and k one after the other as heads without values, which the quicker kernel takes
    ops.qk_norm_rope_cache(qkv[:, :nq * d], nq, 0, d, q_weight, None, eps, table, ctx.positions, None, None, None, 1)
    ops.qk_norm_rope_cache(qkv[:, nq * d:(nq + nkv) * d], nkv, 0, d, k_weight, None, eps, table, ctx.positions, None, None,
                           None, 1)

  def forward_lazy(self, x, ctx, cache) -> PendingLinear:
    nq, nkv, d = self.nq, self.nkv, self.d
    qkv = linear(x, self.qkv_weight, bias=self.qkv_bias)
    self._rotate(qkv, ctx)
    q, k, v = qkv[:, :nq * d], qkv[:, nq * d:(nq + nkv) * d], qkv[:, (nq + nkv) * d:]
    out = torch.empty((qkv.shape[0], nq * d), dtype=qkv.dtype, device=qkv.device)
    # entries with several tokens come first, single tokens last
    multi = ctx.num_multi
    idle = cache.state.shape[0] - 1     # the scratch row, which padding entries of captured steps share
    tokens = sum(ctx.q_lens[:multi])
    if multi:
      ops.linear_attention(q[:tokens], k[:tokens], v[:tokens], nq, nkv, d, out[:tokens], cache.state, ctx.req_slots[:multi],
                           ctx.cu_q[:multi + 1], self.log_decay, self.scale, max_len=ctx.max_q_len, idle_row=idle)
    if ctx.num_requests > multi:
      ops.linear_attention_step(q[tokens:], k[tokens:], v[tokens:], nq, nkv, d, out[tokens:], cache.state,
                                ctx.req_slots[multi:], self.log_decay, self.scale, idle_row=idle)
    return PendingLinear(out, self.o_weight, self.o_bias)


register_mixer("linear_attention", LinearAttention)
