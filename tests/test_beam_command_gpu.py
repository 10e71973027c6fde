"""Beam search from the command line."""

import json
import os
import subprocess
import sys

import pytest
import torch

import plain_beam
import plain_qwen3 as plain
import tiny_models as tm

pytestmark = pytest.mark.gpu


def _generate(folder, *options):
  root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
  return subprocess.run([sys.executable, "-m", "miniinfer_amd", "generate", "--model", folder, "--dtype", "float32", "--ignore-eos",
                         "--max-model-len", "64", "--num-pages", "40", "--quiet", *options],
                        capture_output=True, text=True, cwd=root, timeout=100)


def test_command_line_beams(tmp_path):
  cfg, w = tm.make_model(str(tmp_path / "m"), "A", seed=0, dtype=torch.float32, std=0.05)
  w = {k: v.double() for k, v in w.items()}
  # a prompt whose search no rounding decides (log-probabilities here are good to 1e-4)
  for seed in range(20):
    prompt = tm.random_tokens(cfg, 6, seed=seed)
    want, gap = plain_beam.beam_search(lambda t: plain.qwen3_logits(t, w, dict(cfg)), prompt, 3, 4)
    if gap > 1e-3:
      break
  assert gap > 1e-3
  ids = ",".join(map(str, prompt))
  proc = _generate(str(tmp_path / "m"), "--max-tokens", "4", "--beams", "3", "--prompt-ids", ids)
  assert proc.returncode == 0, proc.stderr[-2000:]
  got = json.loads(proc.stdout.strip().splitlines()[-1])
  assert got["token_ids"] == want[0][0] and abs(got["cumulative_logprob"] - want[0][1]) < 1e-3
  assert got["finish_reason"] == "length" and got["prompt"] == prompt
  proc = _generate(str(tmp_path / "m"), "--max-tokens", "4", "--beams", "3", "--temperature", "0.5", "--prompt-ids", ids)
  assert proc.returncode == 2 and "temperature" in proc.stderr
