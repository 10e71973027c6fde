"""`generate --beams`: what the command turns down before it loads a model (no GPU)."""

import pytest

from miniinfer_amd import __main__ as command


@pytest.fixture
def engines(monkeypatch):
  """Counts the engines that a command makes; none can be made."""
  made = []

  def engine(args):
    made.append(args)
    raise RuntimeError("an engine")
  monkeypatch.setattr(command, "_engine", engine)
  return made


@pytest.mark.parametrize("options,message", [
  (["--beams", "-1"], "beams"),
  (["--beams", "33"], "32"),
  (["--beams", "4", "--top-k", "5"], "--top-k"),
  (["--beams", "4", "--top-p", "0.9"], "--top-p"),
  (["--beams", "4", "--temperature", "0.5"], "--temperature"),
  (["--beams", "4", "--temperature", "0"], "--temperature"),
])
def test_beams_refused(engines, capsys, options, message):
  assert command.main(["generate", "--model", "m", "--prompt-ids", "1,2", *options]) == 2
  assert message in capsys.readouterr().err and not engines


@pytest.mark.parametrize("options", [["--beams", "4"], ["--beams", "32"], ["--beams", "0", "--top-k", "5"], ["--top-p", "0.9"], []])
def test_beams_taken(engines, options):
  with pytest.raises(RuntimeError, match="an engine"):
    command.main(["generate", "--model", "m", "--prompt-ids", "1,2", *options])
  assert len(engines) == 1
