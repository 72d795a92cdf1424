"""The decoding example's own check fails on logits that are not numbers."""
import importlib.util
import math
import os

import pytest

from .test_gpu_serving import _reference_core_for_gpu_tests  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("slot", [0, 2])
def test_logits_that_are_not_numbers_fail(cuda, monkeypatch, bad, slot):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode_layers.py")
    spec = importlib.util.spec_from_file_location("decode_layers", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    step, calls = mod.Decoder.step, []

    def poisoned(self):
        logits = step(self)
        calls.append(0)
        if len(calls) == 1:                               # the first step's logits are among those compared
            logits = logits.clone()
            logits[slot, 17] = bad
        return logits

    monkeypatch.setattr(mod.Decoder, "step", poisoned)
    assert not mod.main(steps=4, out=lambda *_: None) < 0.05
