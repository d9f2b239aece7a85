"""The synthetic decoder of the invariance harness, on the CPU in plain operations."""

from __future__ import annotations

import pytest
import torch

from model_invariance import run_investigation
from model_invariance.adapters import ADAPTERS, SyntheticDecoderAdapter
from model_invariance.harness import stack_samples

SMALL = dict(tokens=21, d=32, hidden=48, heads=4, kv_heads=2, layers=2, window=6, sinks=2, page=4, steps=3, device="cpu",
             dtype=torch.float32)


def run(adapter, samples):
    with torch.inference_mode():
        return adapter.run_model(adapter.load_model(), stack_samples(samples))["actions"]


def test_registered():
    assert ADAPTERS["synthetic_decoder"] is SyntheticDecoderAdapter
    assert SyntheticDecoderAdapter.preset("small", device="cpu").tokens == 77


def test_report():
    report = run_investigation(SyntheticDecoderAdapter(**SMALL), batch_sizes=(1, 2, 3))
    assert report["model"] == "synthetic_decoder" and report["repeatability"]["exact"]
    assert report["maximum_tested_batch"] == 3


def test_padding_does_not_reach_the_answer():
    adapter = SyntheticDecoderAdapter(**SMALL)
    samples = adapter.load_example_inputs(4)
    assert len({int(s["length"]) for s in samples}) > 1
    want = run(adapter, samples)
    for s in samples:
        s["x"][int(s["length"]):] = 1e4
    assert torch.equal(run(adapter, samples), want)


def test_a_token_behind_the_prompt_is_a_longer_prompt():
    """The first step's actions are those of a prompt that ends with the step's token.  In 64 bits but for the
    attention's 32: two layers' sums of at most 24 terms and the roundings around them leave far less than 1e-4."""
    adapter = SyntheticDecoderAdapter(**{**SMALL, "dtype": torch.float64})
    model = adapter.load_model()
    [s] = adapter.load_example_inputs(1)
    n = 13
    s["length"] = torch.tensor(n, dtype=torch.int32)
    with torch.inference_mode():
        first = adapter.run_model(model, stack_samples([s]))["actions"][0]
        s["x"][n] = model.embed @ torch.tanh(first[0])
        s["length"] = torch.tensor(n + 1, dtype=torch.int32)
        longer = adapter.run_model(model, stack_samples([s]))["actions"][0]
    assert float((first[1] - longer[0]).abs().max()) < 1e-4
    assert float((first[2] - longer[1]).abs().max()) < 1e-4


@pytest.mark.parametrize("name", ["small", "vla"])
def test_presets_are_whole(name):
    assert SyntheticDecoderAdapter.preset(name, device="cpu").cfg[0] % 64 == 0
