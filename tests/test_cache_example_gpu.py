"""The four paged-cache operators together, as examples/draft_and_verify.py uses them."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


def test_drafts_do_not_change_what_is_said(cuda):
    """Greedy generation says the same tokens with drafted trees as a token at a time, in fewer steps."""
    import draft_and_verify as example
    target = example.Target()
    prompt = torch.randint(0, target.vocab, (3, 50), generator=torch.Generator(device="cuda").manual_seed(7),
                           device="cuda")
    plain, plain_steps = example.generate(target, prompt, 24, depth=0)
    drafted, steps = example.generate(target, prompt, 24, depth=3)
    assert plain_steps == 24 and steps < plain_steps
    for a, b in zip(plain, drafted):
        assert a[:24] == b[:24]


def test_sampled_generation_runs(cuda):
    import draft_and_verify as example
    target = example.Target(seed=3)
    prompt = torch.randint(0, target.vocab, (2, 30), device="cuda")
    out, steps = example.generate(target, prompt, 10, depth=2, temperature=0.8)
    assert steps <= 10 and all(len(o) >= 10 and all(0 <= t < target.vocab for t in o) for o in out)
