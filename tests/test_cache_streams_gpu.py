"""How the paged-cache operators treat tensors that torch does more with: other streams, gradients."""
import pytest
import torch

import t4a_b200 as t4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("operator", ["write", "read", "attention", "verify"])
def test_inputs_outlive_a_call_on_another_stream(cuda, operator):
    """The other stream is still busy when the call returns; memory of the inputs, freed here, is filled anew on the
    current stream before the call's kernels run."""
    gen = torch.Generator(device="cuda").manual_seed(9)

    def inputs():
        normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")
        if operator in ("write", "read"):
            return dict(key=normal(256, 2, 64), slots=torch.arange(256, device="cuda"))
        if operator == "attention":
            return dict(q=normal(4, 3, 4, 64).half(), context=torch.full((4,), 40, dtype=torch.int32, device="cuda"))
        return dict(logits=normal(4, 3, 5000), tokens=torch.arange(12, dtype=torch.int32, device="cuda").view(4, 3),
                    parents=torch.tensor([[-1, 0, 0]] * 4, dtype=torch.int32, device="cuda"))

    k, v = (torch.randn(16, 16, 2, 64, generator=gen, device="cuda").half() for _ in range(2))
    table = torch.arange(16, dtype=torch.int32, device="cuda").view(4, 4)

    def call(x, stream):
        if operator == "write":
            t4.cache_write(x["key"], x["key"], k, v, x["slots"], stream=stream)
            return ()
        if operator == "read":
            return t4.cache_read(k, v, x["slots"], torch.float32, stream=stream)
        if operator == "attention":
            return t4.tree_attention(x["q"], k, v, table, x["context"], stream=stream)
        return t4.verify_drafts(x["logits"], x["tokens"], x["parents"], temperature=0.0, stream=stream)

    state = gen.get_state()
    want = [t.clone() for t in call(inputs(), None)] + [k.clone(), v.clone()]
    gen.set_state(state)
    x = inputs()
    shapes = [(t.shape, t.dtype) for t in x.values()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    k.zero_() if operator == "write" else None
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # some tenth of a second
    got = call(x, side)
    x.clear()
    others = [torch.full(shape, 1, dtype=dtype, device="cuda") for shape, dtype in shapes * 2]
    side.synchronize()
    torch.cuda.synchronize()
    assert others and all(torch.equal(a, b) for a, b in zip([*got, k, v], want))


def test_results_never_require_a_gradient(cuda):
    """Inputs that require one are taken, as the docstring says, and nothing is recorded."""
    k, v = (torch.zeros(4, 16, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    key = torch.randn(20, 2, 64, device="cuda", requires_grad=True)
    slots = torch.arange(20, device="cuda")
    t4.cache_write(key, key, k, v, slots)
    q = torch.randn(1, 2, 4, 64, device="cuda").half().requires_grad_()
    out, lse = t4.tree_attention(q, k, v, torch.arange(4, dtype=torch.int32, device="cuda")[None],
                                 torch.full((1,), 18, dtype=torch.int32, device="cuda"))
    assert not any(t.requires_grad for t in (k, v, out, lse, *t4.cache_read(k, v, slots, torch.float32)))


@pytest.mark.parametrize("batch,nodes,group", [(1, 1, 4), (5, 20, 2), (40, 2, 4)])
def test_lengths_written_right_before_a_call(cuda, batch, nodes, group):
    """The attention's kernels are set up while the one that writes the contexts still runs."""
    gen = torch.Generator(device="cuda").manual_seed(batch)
    k, v = (torch.randn(batch * 40, 16, 2, 64, generator=gen, device="cuda").half() for _ in range(2))
    table = torch.randperm(batch * 40, generator=gen, device="cuda").view(batch, 40).int()
    q = torch.randn(batch, nodes, 2 * group, 64, generator=gen, device="cuda").half()
    steps = torch.randint(0, 600, (50, batch), generator=gen, device="cuda", dtype=torch.int32)
    live = torch.randint(0, nodes + 1, (50, batch), generator=gen, device="cuda", dtype=torch.int32)
    want = []
    for i in range(50):
        torch.cuda.synchronize()
        want.append(t4.tree_attention(q, k, v, table, steps[i], nodes=live[i]))
        torch.cuda.synchronize()
    context, now = torch.zeros(batch, dtype=torch.int32, device="cuda"), torch.zeros_like(live[0])
    got = []
    for i in range(50):
        context.copy_(steps[i])
        now.copy_(live[i])
        got.append(t4.tree_attention(q, k, v, table, context, nodes=now))
    assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
