"""Generation where the sequences of a batch take drafts at very different rates."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("depth", [1, 4])
def test_every_sequence_gets_its_tokens(cuda, depth):
    """The first sequence takes whole branches and the second one nothing; both say what they say alone."""
    import draft_and_verify as example

    class Uneven(example.Target):
        def logits(self, x, attended):
            return super().logits(x, torch.zeros_like(attended))  # as the drafter guesses

        def guesses(self, tokens, count):
            good = super().guesses(tokens, count + 2)
            return torch.cat([good[:1, :count], good[1:, 2:]])  # of the second sequence never the likeliest

    target = Uneven()
    prompt = torch.randint(0, target.vocab, (2, 20), generator=torch.Generator(device="cuda").manual_seed(5),
                           device="cuda")
    plain, _ = example.generate(target, prompt, 40, depth=0)
    out, steps = example.generate(target, prompt, 40, depth=depth)
    assert steps == 40 and len(out[0]) >= 40 and len(out[1]) == 40
    assert [o[:40] for o in out] == plain
