"""The operators around the cache run together, as a serving loop uses them: packed prompts, then replayed steps."""
import importlib.util
import os

import pytest

from .test_gpu_step import _reference_core_for_gpu_tests  # noqa: F401

pytestmark = pytest.mark.gpu


def test_prompts_and_drawn_answers(cuda):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve_prompts.py")
    spec = importlib.util.spec_from_file_location("serve_prompts", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    off, wrong = mod.main(steps=6, out=lambda *_: None)
    assert off < 0.05 and wrong == 0, (off, wrong)
