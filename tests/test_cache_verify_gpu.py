"""verify_drafts at the edges of its numbers, against the plain walk in 64 bits."""

import pytest
import torch

import t4a_b200 as t4
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


def test_tokens_follow_the_target_after_distinct_siblings(cuda):
    """Children drawn without replacement and children picked as the likeliest, without a draft: a chi-square
    statistic of 11 degrees of freedom, below 40 with probability 1 - 4e-5 for each."""
    gen, vocab, nodes, draws = generator(31), 12, 4, 20000
    logits = torch.randn(1, 1, vocab, generator=gen, device="cuda").expand(draws, nodes, vocab)
    guess = torch.softmax(torch.randn(vocab, generator=gen, device="cuda"), dim=0)
    parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device="cuda").expand(draws, nodes).contiguous()
    p = torch.softmax(logits[0, 0].double(), dim=0)
    drawn = torch.multinomial(guess.expand(draws, vocab), nodes, generator=gen).int()
    likeliest = guess.topk(nodes).indices.int().expand(draws, nodes).contiguous()
    for tokens in (drawn, likeliest):
        uniforms = torch.rand(draws, nodes, generator=gen, device="cuda")
        race = torch.empty(draws, vocab, device="cuda").exponential_(generator=gen).reciprocal_()
        said = t4.verify_drafts(logits, tokens, parents, uniforms=uniforms, race=race)[2][:, 0]
        seen = torch.bincount(said.long(), minlength=vocab).double()
        assert float(((seen - draws * p) ** 2 / (draws * p)).sum()) < 40
