"""verify_drafts at the edges of its numbers, against the plain walk in 64 bits."""
import math

import pytest
import torch

from test_cache_gpu import BF16, F16, F32, check_walk, generator

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab,low,high", [(40, 3, 20), (3000, 17, 2999), (20011, 5, 17000), (128256, 100000, 100001)])
def test_zeros_of_either_sign_are_a_tie(cuda, dtype, vocab, low, high):
    """The greedy token is the lowest-index maximum, and -0 equals 0."""
    gen = generator(vocab)
    logits = (-1 - torch.randn(2, 3, vocab, generator=gen, device="cuda").abs()).to(dtype)
    logits[0, :, low], logits[0, :, high] = -0.0, 0.0
    logits[1, :, low], logits[1, :, high] = 0.0, -0.0
    tokens = torch.tensor([[0, high, low]] * 2, dtype=torch.int32, device="cuda")
    parents = torch.tensor([[-1, 0, 0]] * 2, dtype=torch.int32, device="cuda")
    assert check_walk(logits, tokens, parents, None, None, None, 0.0).tolist() == [1, 1]
