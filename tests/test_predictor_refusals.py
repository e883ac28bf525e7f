"""Configurations that the example predictor refuses instead of leaving a part of them out."""
import importlib.util
import sys
from pathlib import Path

import pytest


@pytest.fixture(scope="module")
def E():
    path = Path(__file__).resolve().parent.parent / "3dgs-project_amd" / "examples" / "predict_splats.py"
    spec = importlib.util.spec_from_file_location("predict_splats_refusals", path)
    module = importlib.util.module_from_spec(spec)
    sys.modules[spec.name] = module
    spec.loader.exec_module(module)
    return module


def test_a_recurrence_in_blocks_that_are_not_fused(E, monkeypatch, capsys):
    monkeypatch.setattr(E, "SplatPredictor", None)  # (nothing is built)
    monkeypatch.setattr(sys, "argv", ["predict_splats.py", "--scan", "1"])
    with pytest.raises(SystemExit) as end:
        E.main()
    assert end.value.code == 2 and "--scan needs --fused" in capsys.readouterr().err


@pytest.mark.parametrize("scan", [(-1,), (0, 9), (4,)])
def test_layers_that_are_not_there(E, scan):
    with pytest.raises(ValueError, match="layers 0 to 3"):
        E.SplatPredictor(E.Config(depth=4, fused=True, scan=scan), device="cpu")
    assert len(E.SplatPredictor(E.Config(depth=2, fused=True, scan=(0, 1)), device="cpu").layers) == 2
