"""What `generate --beams` prints for what a search found (no GPU)."""

import json
from contextlib import nullcontext
from types import SimpleNamespace

from miniinfer_amd import __main__ as command


def _run(monkeypatch, found):
  engine = SimpleNamespace(beam_search=lambda prompts, params: found)
  monkeypatch.setattr(command, "_engine", lambda args: nullcontext(engine))
  return command.main(["generate", "--model", "m", "--prompt-ids", "1,2", "--prompt-ids", "3", "--beams", "2"])


def test_the_best_hypothesis_of_every_prompt(monkeypatch, capsys):
  hyp = lambda n: {"text": "", "token_ids": [n], "cumulative_logprob": -1.0, "score": -1.0, "finish_reason": "length"}
  assert _run(monkeypatch, [[hyp(7), hyp(8)], [hyp(9)]]) == 0
  lines = [json.loads(x) for x in capsys.readouterr().out.splitlines()]
  assert lines == [{"prompt": [1, 2], **hyp(7)}, {"prompt": [3], **hyp(9)}]


def test_a_prompt_without_a_continuation_is_said_so(monkeypatch, capsys):
  """(A model whose logits are NaN.)"""
  hyp = {"text": "", "token_ids": [9], "cumulative_logprob": -1.0, "score": -1.0, "finish_reason": "length"}
  assert _run(monkeypatch, [[], [hyp]]) == 1
  got = capsys.readouterr()
  assert json.loads(got.out) == {"prompt": [3], **hyp} and "[1, 2]" in got.err and "no continuation" in got.err
