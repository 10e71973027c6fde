"""Linear attention, fixed-size states, forks and beam search together: an architecture of linear attention layers (with
and without head norms, rotation and biases) beside paged attention, one of it with a window, is stepped whole, in
portions, in mixed batches and from captured steps, generates, and is searched by beams, against a plain
whole-sequence statement in 64 bits."""

import json
import math
import os
from dataclasses import dataclass

import numpy as np
import pytest
import torch

import plain_beam
import plain_qwen3 as plain
import trace_tools as tt

pytestmark = pytest.mark.gpu

HYBRID = dict(architectures=["ToyHybridForCausalLM"], vocab_size=210, hidden_size=48, num_heads=4, num_kv_heads=2, head_dim=16,
              intermediate_size=56, eps=2e-6, theta=2000.0, window=24, max_positions=400)
DECAY = ((-0.05, -0.4), (-0.002, -1.5))


def _register():
  from miniinfer_amd.config import (AttentionSpec, GatedMLPSpec, LayerSpec, LinearAttentionSpec, ModelSpec, NormSpec,
                                    RotarySpec, register_architecture)

  @dataclass(frozen=True)
  class HybridConfig:
    vocab_size: int
    hidden_size: int
    num_heads: int
    num_kv_heads: int
    head_dim: int
    intermediate_size: int
    eps: float
    theta: float
    window: int
    max_positions: int

    @classmethod
    def from_dict(cls, raw):
      return cls(**{k: raw[k] for k in cls.__dataclass_fields__})

    def build_spec(self):
      H, d = self.hidden_size, self.head_dim
      norm = NormSpec(size=H, eps=self.eps)
      rotary = RotarySpec(rotary_dim=d, theta=self.theta, max_positions=self.max_positions)
      sizes = dict(hidden_size=H, num_heads=self.num_heads, num_kv_heads=self.num_kv_heads, head_dim=d, scale=d ** -0.5)
      mixers = (
        LinearAttentionSpec(**sizes, log_decay=DECAY[0], position=rotary, qk_norm=NormSpec(d, self.eps)),
        AttentionSpec(**sizes, position=rotary, qk_norm=NormSpec(d, self.eps)),
        LinearAttentionSpec(**sizes, log_decay=DECAY[1], qkv_bias=True, o_bias=True),
        AttentionSpec(**sizes, position=rotary, window=self.window),
      )
      layers = tuple(LayerSpec(prefix=f"toy.layers.{i}.", mixer=m, mixer_norm=norm, feed_forward_norm=norm,
                               feed_forward=GatedMLPSpec(hidden_size=H, intermediate_size=self.intermediate_size))
                     for i, m in enumerate(mixers))
      return ModelSpec(architecture="ToyHybridForCausalLM", vocab_size=self.vocab_size, hidden_size=H, layers=layers,
                       run_order=(0, 1, 2, 3), final_norm=norm, embedding_name="toy.embed.weight", final_norm_prefix="toy.norm.",
                       head_name="toy.head.weight", optional_name_prefix="", max_positions=self.max_positions)

  register_architecture("ToyHybridForCausalLM", HybridConfig)


def _weights(seed=0, std=0.1):
  g = torch.Generator().manual_seed(seed)
  c = HYBRID
  H, V, nq, nkv, d, I = (c[k] for k in ("hidden_size", "vocab_size", "num_heads", "num_kv_heads", "head_dim", "intermediate_size"))
  mat = lambda *s: torch.randn(*s, generator=g) * std
  norm = lambda n: 1 + 0.1 * torch.randn(n, generator=g)
  w = {"toy.embed.weight": mat(V, H), "toy.norm.weight": norm(H), "toy.head.weight": mat(V, H) * 3}
  for i in range(4):
    p = f"toy.layers.{i}."
    w[p + "input_layernorm.weight"], w[p + "post_attention_layernorm.weight"] = norm(H), norm(H)
    for n, shape in (("q_proj", (nq * d, H)), ("k_proj", (nkv * d, H)), ("v_proj", (nkv * d, H)), ("o_proj", (H, nq * d))):
      w[p + f"self_attn.{n}.weight"] = mat(*shape)
      if i == 2:
        w[p + f"self_attn.{n}.bias"] = mat(shape[0])
    if i < 2:
      w[p + "self_attn.q_norm.weight"], w[p + "self_attn.k_norm.weight"] = norm(d), norm(d)
    for n, shape in (("gate_proj", (I, H)), ("up_proj", (I, H)), ("down_proj", (H, I))):
      w[p + f"mlp.{n}.weight"] = mat(*shape)
  return w


def _plain_logits(tokens, w):
  """Whole sequence, float64."""
  c = HYBRID
  T, nq, nkv, d = len(tokens), c["num_heads"], c["num_kv_heads"], c["head_dim"]
  ang = plain.rope_angles(torch.arange(T), d, c["theta"], torch.float64)
  h = w["toy.embed.weight"][torch.tensor(tokens)]
  for i in range(4):
    p = f"toy.layers.{i}."
    x = plain.rms_norm(h, w[p + "input_layernorm.weight"], c["eps"])
    proj = lambda n, heads: (x @ w[p + f"self_attn.{n}.weight"].T + w.get(p + f"self_attn.{n}.bias", 0.0)).reshape(T, heads, d)
    q, k, v = proj("q_proj", nq), proj("k_proj", nkv), proj("v_proj", nkv)
    if i < 2:
      q = plain.rms_norm(q, w[p + "self_attn.q_norm.weight"], c["eps"])
      k = plain.rms_norm(k, w[p + "self_attn.k_norm.weight"], c["eps"])
    if i != 2:
      q, k = plain.apply_rope_neox(q, ang), plain.apply_rope_neox(k, ang)
    if i in (0, 2):
      a = torch.exp(torch.tensor(DECAY[i // 2], dtype=torch.float64)).view(nkv, 1, 1)
      S = torch.zeros(nkv, d, d, dtype=torch.float64)
      o = []
      for t in range(T):
        S = a * S + k[t].unsqueeze(2) * v[t].unsqueeze(1)
        o.append((q[t].view(nkv, nq // nkv, d) @ S).reshape(nq, d) * d ** -0.5)
      o = torch.stack(o)
    else:
      mask = plain.causal_mask(T, T, torch.float64, window=c["window"] if i == 3 else None)
      o = plain.grouped_attention(q, k, v, d ** -0.5, mask)
    h = h + o.reshape(T, nq * d) @ w[p + "self_attn.o_proj.weight"].T + w.get(p + "self_attn.o_proj.bias", 0.0)
    x = plain.rms_norm(h, w[p + "post_attention_layernorm.weight"], c["eps"])
    h = h + plain.swiglu(x, w[p + "mlp.gate_proj.weight"], w[p + "mlp.up_proj.weight"], w[p + "mlp.down_proj.weight"])
  return plain.rms_norm(h, w["toy.norm.weight"], c["eps"]) @ w["toy.head.weight"].T


def _write(folder, dtype, seed=0):
  from safetensors.torch import save_file
  _register()
  file_dtype = torch.float32 if dtype == "float32" else torch.bfloat16
  w = {k: v.to(file_dtype) for k, v in _weights(seed).items()}
  os.makedirs(folder)
  with open(os.path.join(folder, "config.json"), "w") as f:
    json.dump(HYBRID, f)
  save_file({k: v.contiguous() for k, v in w.items()}, os.path.join(folder, "model.safetensors"))
  return {k: v.double() for k, v in w.items()}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_linear_attention_layers_are_built_and_stepped(tmp_path, dtype):
  from miniinfer_amd.engine.replay import Replayer
  w = _write(str(tmp_path / "m"), dtype)
  g = torch.Generator().manual_seed(1)
  requests = {f"r{i}": torch.randint(0, 210, (n,), generator=g).tolist() for i, n in enumerate((70, 33, 5, 150, 48))}
  want = {r: _plain_logits(t, w).float().numpy() for r, t in requests.items()}
  for steps in (tt.whole(requests), tt.tail_decoded(requests, 9), tt.portions(requests), tt.mixed(requests, max_live=3, seed=5)):
    rp = Replayer(str(tmp_path / "m"), dtype, tt.peak_tokens(steps, requests), page_size=8)
    assert len(rp.cache.paged) == 2 and rp.cache.states[0].layers == [0, 2] and rp.cache.states[0].state.shape[2:] == (2, 16, 16)
    outs = []
    for st in steps:
      outs.append(rp.step(st))
      rp.cache.check()
    assert rp.cache.all_pages_free()
    got = tt.gather(steps, outs, requests, 210)
    for r in requests:
      err = np.abs(got[r] - want[r]).max()
      scale = np.abs(want[r]).max()
      assert err <= (2e-4 if dtype == "float32" else 4e-2 * scale), f"request {r}: max err {err:.3g} (scale {scale:.3g})"


def _greedy(prompt, n, w):
  ids, out = list(prompt), []
  for _ in range(n):
    out.append(int(torch.argmax(_plain_logits(ids, w)[-1])))
    ids.append(out[-1])
  return out


@pytest.mark.parametrize("eager", [False, True])
def test_linear_attention_layers_generate(tmp_path, eager):
  """Decode steps from graphs (padded batches among them) and eagerly, requests preempted and recomputed."""
  from miniinfer_amd import LLMEngine, SamplingParams
  w = _write(str(tmp_path / "m"), "float32")
  g = torch.Generator().manual_seed(4)
  prompts = [torch.randint(0, 210, (n,), generator=g).tolist() for n in (30, 41, 25, 37)]
  want = [_greedy(p, 20, w) for p in prompts]
  with LLMEngine(model=str(tmp_path / "m"), dtype="float32", page_size=8, num_pages=20, max_num_seqs=3, max_num_batched_tokens=48,
                 enforce_eager=eager) as eng:
    assert eng.runner.use_graphs is (not eager)
    outs = eng.generate(prompts, SamplingParams(temperature=0.0, max_tokens=20, ignore_eos=True), use_tqdm=False)
    assert eng.scheduler.num_preemptions > 0 and eng.cache.all_pages_free()
  assert [o["token_ids"] for o in outs] == want


def _searches(logits_of, vocab, cases, margin=2e-3):
  """For each case (prompt length, beams, tokens, stop ids, length penalty, early stopping) the first prompt whose search no
  decision of which is closer than `margin`, the engine's 32-bit error many times over, and what it finds."""
  out = []
  for n, beams, tokens, stop, penalty, early in cases:
    for seed in range(200):
      prompt = torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(1000 * n + seed)).tolist()
      found, gap = plain_beam.beam_search(logits_of, prompt, beams, tokens, stop, penalty, early)
      if gap > margin:
        out.append((prompt, found))
        break
    else:
      raise AssertionError("no prompt without a close decision")
  return out


def _check_hypotheses(got, want):
  assert [h["token_ids"] for h in got] == [toks for toks, _, _ in want[:len(got)]]
  for h, (_, score, penalised) in zip(got, want):
    assert abs(h["cumulative_logprob"] - score) <= 1e-3 and abs(h["score"] - penalised) <= 1e-3


@pytest.mark.parametrize("eager", [False, True])
def test_beam_search_of_a_model_with_pages_and_states(tmp_path, eager):
  """Prompts of different lengths searched together: full pages shared, last pages and states forked, windows that
  pass, searches that end at different steps."""
  from miniinfer_amd import BeamSearchParams, LLMEngine
  w = _write(str(tmp_path / "m"), "float32", seed=2)
  logits_of = lambda t: _plain_logits(t, w)
  groups = (((3, 3, 6, (), 1.0, False), (8, 3, 6, (), 1.0, False), (29, 3, 6, (), 1.0, False), (1, 3, 6, (), 1.0, False)),
            ((7, 1, 5, (), 1.0, False),),
            ((12, 2, 7, (), 0.0, False), (20, 2, 7, (), 0.0, False)))
  with LLMEngine(model=str(tmp_path / "m"), dtype="float32", page_size=8, num_pages=80, max_num_seqs=9, max_num_batched_tokens=16,
                 enforce_eager=eager) as eng:
    for cases in groups:
      searches = _searches(logits_of, 210, cases)
      _, beams, tokens, _, penalty, early = cases[0]
      params = BeamSearchParams(num_beams=beams, max_tokens=tokens, length_penalty=penalty, early_stopping=early,
                                num_return=beams, ignore_eos=True)
      found = eng.beam_search([p for p, _ in searches], params)
      for got, (_, want) in zip(found, searches):
        _check_hypotheses(got, want)
        assert all(h["finish_reason"] == "length" for h in got)
      eng.cache.check()
      assert eng.cache.all_pages_free() and eng.cache.num_free_slots() == 9


def test_beam_search_with_stop_tokens_of_the_tiny_model(tmp_path):
  """Hypotheses that end early, by either stopping rule; one beam is greedy decoding; generation goes on as before."""
  import tiny_models as tm
  from miniinfer_amd import BeamSearchParams, LLMEngine, SamplingParams
  cfg, w = tm.make_model(str(tmp_path), "B", seed=0, dtype=torch.float32, std=0.05)
  w = {k: v.double() for k, v in w.items()}
  logits_of = lambda t: plain.qwen3_logits(t, w, dict(cfg))
  V = cfg["vocab_size"]
  with LLMEngine(model=str(tmp_path), dtype="float32", page_size=8, num_pages=100, max_num_seqs=8) as eng:
    prompt = tm.random_tokens(cfg, 21, seed=3)
    greedy = eng.generate([prompt], SamplingParams(temperature=0.0, max_tokens=9, ignore_eos=True), use_tqdm=False)[0]["token_ids"]
    one = eng.beam_search([prompt], BeamSearchParams(num_beams=1, max_tokens=9, ignore_eos=True))[0][0]
    assert one["token_ids"] == greedy
    # stop at tokens that the search would like to go on with
    stop = tuple(sorted({t for h in eng.beam_search([prompt], BeamSearchParams(num_beams=4, max_tokens=5, num_return=4,
                                                                              ignore_eos=True))[0] for t in h["token_ids"][1:3]}))[:2]
    for early in (False, True):
      cases = ((21, 4, 7, stop, 1.0, early), (5, 4, 7, stop, 1.0, early))
      searches = _searches(logits_of, V, cases)
      params = BeamSearchParams(num_beams=4, max_tokens=7, num_return=4, ignore_eos=True, stop_token_ids=list(stop),
                                early_stopping=early)
      for got, (_, want) in zip(eng.beam_search([p for p, _ in searches], params), searches):
        _check_hypotheses(got, want)
        assert all((h["finish_reason"] == "stop") == (h["token_ids"][-1] in stop) for h in got)
    again = eng.generate([prompt], SamplingParams(temperature=0.0, max_tokens=9, ignore_eos=True), use_tqdm=False)[0]["token_ids"]
    assert again == greedy and eng.cache.all_pages_free()


@pytest.mark.filterwarnings("error::UserWarning")      # (a captured step that does not reproduce the eager one warns)
def test_beam_search_in_bfloat16_and_more_beams_than_tokens(tmp_path):
  from miniinfer_amd import BeamSearchParams, LLMEngine
  _write(str(tmp_path / "m"), "bfloat16")
  with LLMEngine(model=str(tmp_path / "m"), dtype="bfloat16", page_size=16, num_pages=200, max_num_seqs=32,
                 tune_products=False) as eng:
    out = eng.beam_search([[1, 2, 3], [4] * 40], BeamSearchParams(num_beams=32, max_tokens=9, num_return=32, ignore_eos=True))
    for hyps in out:
      assert len(hyps) == 32 and len({tuple(h["token_ids"]) for h in hyps}) == 32
      assert all(len(h["token_ids"]) == 9 and math.isfinite(h["score"]) for h in hyps)
      assert [h["score"] for h in hyps] == sorted((h["score"] for h in hyps), reverse=True)
    assert eng.cache.all_pages_free() and eng.cache.num_free_slots() == 32


def test_what_beam_search_refuses(tmp_path):
  from miniinfer_amd import BeamSearchParams, LLMEngine, SamplingParams
  _write(str(tmp_path / "m"), "float32")
  for bad in (dict(num_beams=0), dict(max_tokens=0), dict(num_return=5, num_beams=4), dict(num_return=0), dict(stop_token_ids=[-1])):
    with pytest.raises(ValueError):
      BeamSearchParams(**bad)
  with LLMEngine(model=str(tmp_path / "m"), dtype="float32", page_size=8, num_pages=12, max_num_seqs=4) as eng:
    p = BeamSearchParams(num_beams=4, max_tokens=4)
    for prompts, params, message in (([[]], p, "at least one"), ([[300]], p, "outside"), ([[1] * 399], p, "exceeds"),
                                     ([[1, 2]], BeamSearchParams(num_beams=5), "does not fit"),
                                     ([[1] * 60], p, "does not fit"),
                                     ([[1, 2]], BeamSearchParams(num_beams=33), "at most"), (["text"], p, "tokenizer")):
      with pytest.raises(ValueError, match=message):
        eng.beam_search(prompts, params)
    eng.add_request([1, 2, 3], SamplingParams(max_tokens=2, temperature=0.0))
    with pytest.raises(RuntimeError, match="unfinished"):
      eng.beam_search([[1, 2]], p)
    while not eng.is_finished():
      eng.step()
    assert len(eng.beam_search([[1, 2]], BeamSearchParams(num_beams=2, max_tokens=3))[0]) == 1
    assert eng.cache.all_pages_free()
