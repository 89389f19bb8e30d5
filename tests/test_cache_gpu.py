"""The paged-cache operators on the GPU against plain 64-bit implementations.

Tolerances follow from the roundings.  Codes and scales are F32 arithmetic without
freedom, so they are equal.  Attention: a weight is rounded once to F16 (BF16 for a BF16
cache), the output once to its type, so an output is off by at most (u_weight + u_out) *
sum w|v|, u = 2^-11 for F16 and 2^-8 for BF16; products, exponentials and sums in F32 add
less than 2^-13 of it.  The log-sum-exp is off by F32 roundings of scores whose terms add up
to `size`: 2^-18 of size + |lse| + 1 covers 256-term sums.  Counts, paths and tokens are equal;
log-probabilities are F32 sums of terms up to |log p|: 2^-18 of 1 + |log p|.
"""
import math
import random

import pytest
import torch

import cache_reference as ref
import t4a_b200 as t4

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
I8, E4M3, F16, BF16, F32 = torch.int8, torch.float8_e4m3fn, torch.float16, torch.bfloat16, torch.float32


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def codes_of(x, dtype):
    """(codes, scales) by the definition, in F32."""
    top = ref.CODE_MAX[dtype]
    most = x.float().abs().amax(dim=-1)
    fine = torch.isfinite(most)
    live = fine & (most >= 2.0 ** -100)
    inverse = torch.full_like(most, top) / torch.where(live, most, 1.0)
    y = torch.where(live.unsqueeze(-1), x.float() * inverse.unsqueeze(-1), 0.0)
    code = y.round().to(dtype) if dtype == I8 else y.clamp(-top, top).to(dtype)
    return code, torch.where(live, most * (1.0 / top), torch.where(fine, 0.0, math.nan))


def same(a, b):
    return torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a,
                       b.view(torch.uint8) if b.element_size() == 1 else b)


@pytest.mark.parametrize("rows,heads,dim,page", [(0, 4, 64, 16), (1, 1, 16, 1), (1, 8, 128, 16), (7, 3, 80, 5),
                                                 (33, 5, 96, 24), (130, 2, 256, 64), (1000, 8, 128, 16),
                                                 (257, 1, 48, 128)])
@pytest.mark.parametrize("source", [F32, F16, BF16])
@pytest.mark.parametrize("kind", [I8, E4M3, F16, BF16])
def test_write_then_read(cuda, rows, heads, dim, page, source, kind):
    gen = generator(rows * 31 + dim)
    pages = rows // page + 3
    k, v, ks, vs = ref.random_cache(gen, pages, page, heads, dim, kind)
    before = [t.clone() if t is not None else None for t in (k, v, ks, vs)]
    key, value = (torch.randn(rows, heads, dim, generator=gen, device="cuda").to(source) for _ in range(2))
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:rows].to(
        torch.int32 if rows % 2 else torch.int64)
    if rows > 4:
        slots[rows // 3], slots[rows // 2] = -1, pages * page
        key[2] = 0
        key[3, 0, dim - 1] = math.inf
        value[1, heads - 1, 0] = math.nan
        value[3] = 1e-37 if source != F16 else 0
    t4.cache_write(key, value, k, v, slots, k_scale=ks, v_scale=vs)
    inside = (slots >= 0) & (slots < pages * page)
    at = slots[inside].long()
    for cache, scale, old, old_scale, x in ((k, ks, before[0], before[2], key), (v, vs, before[1], before[3], value)):
        want = old.clone()
        flat = want.view(-1, heads, dim)
        if scale is None:
            flat[at] = x[inside].to(kind)
            assert torch.equal(cache.view(torch.int16), want.view(torch.int16)) or same(
                torch.nan_to_num(cache.float()), torch.nan_to_num(want.float()))
        else:
            code, s = codes_of(x[inside], kind)
            flat.view(torch.int8)[at] = code.view(torch.int8)
            assert torch.equal(cache.view(torch.int8), want.view(torch.int8))
            want_scale = old_scale.clone()
            want_scale.view(-1, heads)[at] = s
            assert torch.equal(torch.nan_to_num(scale, nan=-1.0), torch.nan_to_num(want_scale, nan=-1.0))
    got = t4.cache_read(k, v, slots, source, k_scale=ks, v_scale=vs)
    for cache, scale, y in ((k, ks, got[0]), (v, vs, got[1])):
        want = torch.zeros(rows, heads, dim, device="cuda")
        x = cache.view(-1, heads, dim)[at].float()
        want[inside] = x if scale is None else x * scale.view(-1, heads)[at].unsqueeze(-1)
        assert y.dtype == source
        assert torch.equal(torch.nan_to_num(y, nan=7.0), torch.nan_to_num(want.to(source), nan=7.0))


def test_rows_of_strided_and_unaligned_tensors(cuda):
    gen = generator(5)
    heads, dim, page, pages, rows = 3, 64, 8, 6, 20
    # A cache of [pages, heads, page, dim], scales of [heads, pages, page], K and V in one buffer.
    both = torch.zeros(pages, 2, heads, page, dim, dtype=I8, device="cuda")
    k, v = (both[:, i].transpose(1, 2) for i in range(2))
    ks, vs = (torch.zeros(heads, pages, page, device="cuda").permute(1, 2, 0) for _ in range(2))
    wide = torch.randn(rows, 2 * heads * dim + 3, generator=gen, device="cuda").to(BF16)
    key = wide[:, 1:1 + heads * dim].unflatten(1, (heads, dim))  # odd row starts
    value = wide[:, 2 + heads * dim:2 + 2 * heads * dim].unflatten(1, (heads, dim))
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:2 * rows][::2]
    t4.cache_write(key, value, k, v, slots, k_scale=ks, v_scale=vs)
    for cache, scale, x in ((k, ks, key), (v, vs, value)):
        code, s = codes_of(x, I8)
        assert torch.equal(cache[slots // page, slots % page], code)
        assert torch.equal(scale[slots // page, slots % page], s)
    out = tuple(torch.zeros(heads, rows, dim + 1, device="cuda").transpose(0, 1)[:, :, 1:] for _ in range(2))
    t4.cache_read(k, v, slots, F32, k_scale=ks, v_scale=vs, out=out)
    for cache, scale, y in ((k, ks, out[0]), (v, vs, out[1])):
        at = (slots // page, slots % page)
        assert torch.equal(y, cache[at].float() * scale[at].unsqueeze(-1))


def attention_case(seed, batch, nodes, kv, group, dim, page, contexts, kind, dtype, live=None, tree=True):
    gen, rng = generator(seed), random.Random(seed)
    contexts = (contexts * batch)[:batch]
    width = -(-(max(contexts) + nodes) // page)
    k, v, ks, vs = ref.random_cache(gen, batch * width + 1, page, kv, dim, kind)
    table = torch.randperm(batch * width + 1, generator=gen, device="cuda")[:batch * width].view(batch, width)
    q = (1.5 * torch.randn(batch, nodes, kv * group, dim, generator=gen, device="cuda")).to(dtype)
    sees = torch.stack([random_sees(rng, nodes, tree) for _ in range(batch)]).cuda()
    return dict(q=q, k=k, v=v, ks=ks, vs=vs, table=table.int(), sees=sees,
                context=torch.tensor(contexts, dtype=torch.int32, device="cuda"),
                live=torch.tensor(live or [nodes] * batch, dtype=torch.int32, device="cuda"))


def random_sees(rng, nodes, tree):
    return ref.random_tree(rng, nodes)[1] if tree else torch.tril(torch.ones(nodes, nodes, dtype=torch.bool))


def poison_unused(c):
    """Rows that no sequence sees hold the worst that they could."""
    page = c["k"].shape[1]
    used = torch.zeros(c["k"].shape[0] * page, dtype=torch.bool, device="cuda")
    for b in range(c["table"].shape[0]):
        place = torch.arange(min(int(c["context"][b]) + int(c["live"][b]), c["table"].shape[1] * page), device="cuda")
        used[c["table"][b, place // page].long() * page + place % page] = True
    for name in ("k", "v"):
        if c[name].dtype in (F16, BF16):
            c[name].view(-1, *c[name].shape[2:])[~used] = math.nan
        else:
            c[name + "s"].view(-1, c[name].shape[2])[~used] = math.nan
            if c[name].dtype == E4M3:
                c[name].view(torch.uint8).view(-1, *c[name].shape[2:])[~used] = 0x7f


def check_attention(c, mask="given", scale=None, **more):
    dim = c["q"].shape[3]
    s = dim ** -0.5 if scale is None else scale
    out, lse = t4.tree_attention(c["q"], c["k"], c["v"], c["table"], c["context"],
                                 mask=c["sees"] if mask == "given" else mask, nodes=c["live"], k_scale=c["ks"],
                                 v_scale=c["vs"], scale=scale, **more)
    want, want_lse, spread, size = ref.attention(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], c["context"],
                                                 c["sees"], c["live"], s)
    u_weight = UNIT[BF16] if c["k"].dtype == BF16 else UNIT[F16]
    bound = (u_weight + UNIT[c["q"].dtype] + 2.0 ** -13) * spread + 2.0 ** -24
    worst = float(((out.double() - want).abs() / bound).max()) if out.numel() else 0.0
    assert torch.isfinite(out).all() and worst <= 1.0, worst
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    off = ((lse.double() - want_lse).abs() / (2.0 ** -18 * (size + want_lse.abs() + 1)))[~empty]
    assert off.numel() == 0 or float(off.max()) <= 1.0, float(off.max())
    return out, lse


KINDS = [(BF16, BF16), (F16, F16), (I8, BF16), (I8, F16), (E4M3, BF16), (E4M3, F16)]


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("batch,nodes,kv,group,dim,page,contexts", [
    (1, 1, 1, 1, 64, 16, [0]),
    (1, 1, 2, 4, 128, 16, [1]),
    (3, 1, 2, 8, 128, 16, [63, 64, 65]),
    (2, 5, 1, 3, 96, 24, [100, 7]),
    (4, 13, 3, 2, 80, 1, [0, 30, 200, 511]),
    (1, 16, 2, 1, 16, 7, [1000]),
    (2, 33, 1, 1, 256, 64, [129, 700]),
    (5, 7, 2, 5, 112, 32, [3, 900, 17, 0, 64]),
    (2, 64, 1, 8, 128, 64, [1000, 333]),
    (1, 9, 1, 16, 64, 128, [5000]),
    (1, 3, 2, 40, 32, 16, [77]),
    (2, 200, 1, 4, 128, 16, [300, 40]),
    (1, 150, 1, 2, 256, 16, [200]),
])
def test_attention(cuda, kind, dtype, batch, nodes, kv, group, dim, page, contexts):
    c = attention_case(batch * 100 + nodes, batch, nodes, kv, group, dim, page, contexts, kind, dtype)
    poison_unused(c)
    check_attention(c)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("batch,nodes,kv,group,dim,page,contexts", [
    (48, 1, 8, 4, 128, 16, [700, 3, 1100, 64]),
    (40, 3, 8, 4, 64, 64, [500, 900, 20]),
    (37, 5, 6, 5, 96, 24, [800, 100, 1203]),
    (33, 9, 8, 5, 128, 16, [600, 1200, 3, 128]),
    (30, 40, 4, 4, 96, 24, [900, 77, 2000]),
    (24, 64, 5, 8, 64, 32, [1500, 100]),
    (24, 7, 6, 6, 256, 16, [700, 1000]),
    (64, 1, 8, 4, 80, 16, [700, 3, 1100, 64]),
    (64, 2, 8, 6, 112, 32, [500, 300, 9]),
    (64, 4, 8, 6, 48, 16, [400, 130]),
    (48, 9, 6, 6, 80, 16, [400, 630]),
    (32, 2, 8, 6, 208, 16, [400, 630]),
])
def test_blocks_that_take_several_tiles_and_units(cuda, kind, dtype, batch, nodes, kv, group, dim, page, contexts):
    c = attention_case(batch, batch, nodes, kv, group, dim, page, contexts, kind, dtype)
    poison_unused(c)
    check_attention(c)


@pytest.mark.parametrize("kind,dtype", [(I8, BF16), (I8, F16), (E4M3, BF16), (E4M3, F16)])
@pytest.mark.parametrize("batch,nodes,kv,group,dim,page,contexts", [
    (2, 3, 1, 8, 128, 16, [0, 40]),
    (3, 5, 2, 6, 112, 24, [300, 0, 65]),
    (24, 8, 8, 4, 128, 16, [600, 1200, 3, 128]),
    (16, 7, 6, 3, 112, 32, [700, 64]),
    (2, 4, 2, 8, 128, 64, [9000, 1]),
])
def test_attention_through_a_long_table(cuda, kind, dtype, batch, nodes, kv, group, dim, page, contexts):
    """A table with room for some 200000 places, most of it beyond the sequences."""
    c = attention_case(batch + 7, batch, nodes, kv, group, dim, page, contexts, kind, dtype)
    poison_unused(c)
    wide = torch.full((batch, 200000 // page + 1), -1, dtype=torch.int32, device="cuda")
    if wide.shape[1] > c["table"].shape[1]:
        wide[:, :c["table"].shape[1]] = c["table"]
        c["table"] = wide
    check_attention(c)


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_attention_without_a_mask_is_a_chain(cuda, kind, dtype):
    check_attention(attention_case(3, 2, 6, 2, 4, 128, 16, [50, 300], kind, dtype, tree=False), mask=None)


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_nodes_that_see_nothing(cuda, kind, dtype):
    c = attention_case(4, 4, 6, 2, 3, 64, 16, [0, 20, 0, 130], kind, dtype, live=[6, 0, 3, 4])
    c["sees"][0, 2] = False
    c["sees"][2] = False
    poison_unused(c)
    out, lse = check_attention(c)
    for b, i in ((0, 2), (1, 0), (2, 1), (3, 5)):
        assert (out[b, i] == 0).all() and (lse[b, i] == -math.inf).all()


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("nodes,group", [(5, 2), (20, 3), (40, 4)])
def test_unseen_rows_may_hold_anything(cuda, kind, dtype, nodes, group):
    """A drafted row with a NaN or an infinity reaches the nodes that see it, and no others."""
    c = attention_case(6, 2, nodes, 1, group, 128, 16, [40, 117], kind, dtype)
    page, bad = 16, 3
    for b in range(2):
        place = int(c["context"][b]) + bad
        at = (int(c["table"][b, place // page]), place % page)
        for name, odd in (("k", math.nan), ("v", math.inf if b else math.nan)):
            if kind in (F16, BF16):
                c[name][at] = odd
            else:
                c[name + "s"][at] = math.nan
    out, lse = t4.tree_attention(c["q"], c["k"], c["v"], c["table"], c["context"], mask=c["sees"], k_scale=c["ks"],
                                 v_scale=c["vs"])
    reached = c["sees"][:, :, bad][:, :, None].expand(lse.shape)
    assert torch.isnan(lse[reached]).all() and torch.isfinite(lse[~reached]).all()
    assert torch.isnan(out[reached]).all() and torch.isfinite(out[~reached]).all()
    clean = {k: t.clone() if torch.is_tensor(t) else t for k, t in c.items()}
    for b in range(2):
        place = int(c["context"][b]) + bad
        at = (int(c["table"][b, place // page]), place % page)
        for name in ("k", "v"):
            if kind in (F16, BF16):
                clean[name][at] = 0
            else:
                clean[name + "s"][at] = 1
    want, _, spread, _ = ref.attention(clean["q"], clean["k"], clean["v"], clean["ks"], clean["vs"], clean["table"],
                                       clean["context"], clean["sees"], clean["live"], 128 ** -0.5)
    u = UNIT[BF16] if kind == BF16 else UNIT[F16]
    off = (out.double() - want).abs() - (u + UNIT[dtype] + 2.0 ** -13) * spread - 2.0 ** -24
    assert float(off[~reached].max()) <= 0


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_attention_over_strided_tensors(cuda, kind, dtype):
    """Caches with heads outside the pages' places, rows of q at odd addresses, one mask for all sequences."""
    c = attention_case(8, 3, 6, 2, 3, 64, 8, [30, 9, 100], kind, dtype)
    for name in ("k", "v"):
        c[name] = c[name].transpose(1, 2).contiguous().transpose(1, 2)
        if c[name + "s"] is not None:
            c[name + "s"] = c[name + "s"].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    wide = torch.zeros(3, 6, 6 * 64 + 1, dtype=dtype, device="cuda")
    q = wide[:, :, 1:].unflatten(2, (6, 64))
    q.copy_(c["q"])
    c["q"] = q
    c["sees"] = c["sees"][:1].expand(3, 6, 6)
    c["table"] = torch.cat([c["table"], c["table"]], dim=1).t().contiguous().t()[:, :c["table"].shape[1]]
    out = torch.zeros(6, 3, 6, 65, dtype=dtype, device="cuda").permute(1, 0, 2, 3)[..., 1:]
    lse = torch.zeros(6, 6, 3, device="cuda").permute(2, 1, 0)
    got = check_attention(c, out=out, lse=lse)
    assert got[0] is out and got[1] is lse


def test_more_row_tiles_than_blocks(cuda):
    """300 tiles of query rows: every one passes over the whole cache by itself."""
    check_attention(attention_case(16, 1, 300, 1, 128, 64, 64, [90], I8, BF16))


def test_an_empty_cache(cuda):
    k, v = (torch.zeros(0, 16, 2, 64, dtype=F16, device="cuda") for _ in range(2))
    table = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    out, lse = t4.tree_attention(torch.ones(2, 3, 4, 64, dtype=F16, device="cuda"), k, v, table,
                                 torch.full((2,), 20, dtype=torch.int32, device="cuda"))
    assert (out == 0).all() and (lse == -math.inf).all()
    slots = torch.tensor([0, -1, 5], device="cuda")
    rows = torch.ones(3, 2, 64, dtype=F16, device="cuda")
    t4.cache_write(rows, rows, k, v, slots)
    assert all((x == 0).all() for x in t4.cache_read(k, v, slots, F32))


def test_calls_in_a_graph(cuda):
    """A captured step gives what the calls give, on new contents of the same tensors too."""
    gen = generator(17)
    c = attention_case(18, 3, 5, 2, 4, 64, 16, [90, 40, 200], E4M3, F16)
    key, value = (torch.randn(15, 2, 64, generator=gen, device="cuda").to(F16) for _ in range(2))
    places = c["context"][:, None].long() + torch.arange(5, device="cuda")
    slots = (c["table"].long().gather(1, places // 16) * 16 + places % 16).flatten()
    logits = torch.randn(3, 5, 3000, generator=gen, device="cuda")
    tokens = torch.randint(0, 3000, (3, 5), generator=gen, device="cuda", dtype=torch.int32)
    parents = torch.tensor([[-1, 0, 0, 1, 2]] * 3, dtype=torch.int32, device="cuda")
    uniforms = torch.rand(3, 5, generator=gen, device="cuda")
    race = torch.empty(3, 3000, device="cuda").exponential_(generator=gen).reciprocal_()

    def step():
        t4.cache_write(key, value, c["k"], c["v"], slots, k_scale=c["ks"], v_scale=c["vs"])
        got = t4.tree_attention(c["q"], c["k"], c["v"], c["table"], c["context"], mask=c["sees"], k_scale=c["ks"],
                                v_scale=c["vs"])
        return got + t4.verify_drafts(logits, tokens, parents, uniforms=uniforms, race=race)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(2):
        key.normal_(generator=gen)
        c["q"].normal_(generator=gen)
        logits.normal_(generator=gen)
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_refusals_from_python(cuda):
    c = attention_case(19, 2, 3, 2, 2, 64, 16, [30, 7], I8, F16)
    scales = dict(k_scale=c["ks"], v_scale=c["vs"])
    rows = torch.zeros(4, 2, 64, dtype=F16, device="cuda")
    slots = torch.arange(4, device="cuda")

    def attend(q=c["q"], k=c["k"], table=c["table"], context=c["context"], **more):
        return t4.tree_attention(q, k, c["v"], table, context, **{**scales, **more})

    with pytest.raises(TypeError):
        t4.cache_write(rows.double(), rows.double(), c["k"], c["v"], slots, **scales)
    with pytest.raises(TypeError):
        t4.cache_write(rows, rows.float(), c["k"], c["v"], slots, **scales)
    with pytest.raises(TypeError):
        t4.cache_write(rows, rows, c["k"], c["v"], slots.float(), **scales)
    with pytest.raises(TypeError):
        t4.cache_read(c["k"], c["v"], slots, torch.float64, **scales)
    with pytest.raises(ValueError):
        t4.cache_write(rows, rows, c["k"], c["v"], slots)  # no scales
    with pytest.raises(ValueError):
        t4.cache_write(rows, rows, c["k"], c["v"], slots.cpu(), **scales)
    with pytest.raises(ValueError):
        t4.cache_write(rows.cpu(), rows.cpu(), c["k"], c["v"], slots, **scales)
    with pytest.raises(t4.T4AError) as refused:
        t4.cache_write(rows[:, :1], rows[:, :1], c["k"], c["v"], slots, **scales)
    assert refused.value.status == 16
    with pytest.raises(TypeError):
        attend(q=c["q"].float())
    with pytest.raises(ValueError):
        attend(q=c["q"][0])
    with pytest.raises(TypeError):
        attend(table=c["table"].long())
    with pytest.raises(ValueError):
        attend(context=c["context"][:1])
    with pytest.raises(TypeError):
        attend(k=c["k"].view(torch.uint8))
    with pytest.raises(t4.T4AError):
        attend(workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    need = t4.tree_attention_workspace_bytes(c["q"], c["k"], c["v"], c["table"], **scales)
    first, second = attend(), attend(workspace=torch.empty(need, dtype=torch.uint8, device="cuda"))
    assert torch.equal(first[0], second[0])
    with pytest.raises(ValueError):
        t4.verify_drafts(torch.zeros(2, 3, 9, device="cuda"), torch.zeros(2, 4, dtype=torch.int32, device="cuda"),
                         torch.zeros(2, 3, dtype=torch.int32, device="cuda"), temperature=0.0)
    with pytest.raises(t4.T4AError):
        t4.verify_drafts(torch.zeros(2, 3, 9, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda"),
                         torch.zeros(2, 3, dtype=torch.int32, device="cuda"))  # no uniforms


def test_pages_outside_the_cache_are_not_seen(cuda):
    c = attention_case(9, 2, 3, 2, 2, 64, 16, [100, 40], I8, F16)
    c["table"][0, 2], c["table"][0, 4], c["table"][1, 0] = -1, c["k"].shape[0], 1 << 30
    check_attention(c)


def test_context_past_the_table_and_below_zero(cuda):
    c = attention_case(10, 3, 4, 1, 2, 64, 16, [60, 60, 60], BF16, BF16)
    c["context"] = torch.tensor([62, 1 << 30, -5], dtype=torch.int32, device="cuda")
    check_attention(c)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7])
def test_scales_of_the_scores(cuda, scale):
    check_attention(attention_case(11, 2, 3, 2, 2, 64, 16, [70, 5], E4M3, BF16), scale=scale)


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e6, 1e25])
def test_rows_of_very_different_sizes(cuda, kind, size):
    """Scales of V far apart, and zero rows among them, keep each weight's precision."""
    c = attention_case(12, 2, 4, 2, 4, 128, 16, [200, 90], kind, BF16)
    c["vs"][::2] *= size
    c["vs"][1] = 0
    c["k"].view(torch.int8)[2] = 0
    check_attention(c)


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_long_context_in_parts(cuda, kind, dtype):
    """One sequence over all SMs, with a maximum that comes late and then early."""
    c = attention_case(13, 1, 2, 1, 2, 64, 16, [30000], kind, dtype)
    rows = c["k"].view(-1, 64)
    at = (c["table"][0, :].long() * 16)[[3, 1800]]
    c["q"][0, 0], c["q"][0, 1] = rows[at[1]].to(dtype).float().sign() * 2, rows[at[0]].float().sign() * 2
    check_attention(c)


def test_attention_is_deterministic_and_runs_on_other_streams(cuda):
    c = attention_case(14, 9, 5, 2, 4, 128, 16, [700, 20, 1500], I8, BF16)
    first = check_attention(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        again = t4.tree_attention(c["q"], c["k"], c["v"], c["table"], c["context"], mask=c["sees"], nodes=c["live"],
                                  k_scale=c["ks"], v_scale=c["vs"], stream=side)
        side.synchronize()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_offsets_past_32_bits(cuda):
    """Pages whose bytes start past 2^32."""
    pages, page, heads, dim = 2, 16, 1, 64
    span = (1 << 32) + (1 << 20)
    pool = torch.zeros(2 * span + page * heads * dim, dtype=I8, device="cuda")
    k = torch.as_strided(pool, (pages, page, heads, dim), (2 * span - 4096, dim, dim, 1))
    v = torch.as_strided(pool, (pages, page, heads, dim), (span, dim, dim, 1), 8192)
    ks, vs = (torch.zeros(pages, page, heads, device="cuda") for _ in range(2))
    gen = generator(15)
    key, value = (torch.randn(20, heads, dim, generator=gen, device="cuda").to(F16) for _ in range(2))
    slots = torch.arange(20, device="cuda")
    t4.cache_write(key, value, k, v, slots, k_scale=ks, v_scale=vs)
    code, scale = codes_of(value, I8)
    assert torch.equal(v[1, :4], code[16:]) and torch.equal(vs[1, :4], scale[16:])
    c = dict(q=torch.randn(1, 1, 2, dim, generator=gen, device="cuda").to(F16), k=k, v=v, ks=ks, vs=vs,
             table=torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"),
             context=torch.tensor([19], dtype=torch.int32, device="cuda"),
             sees=torch.ones(1, 1, 1, dtype=torch.bool, device="cuda"),
             live=torch.ones(1, dtype=torch.int32, device="cuda"))
    check_attention(c)


# ---- verification ------------------------------------------------------------------------------------------

def check_walk(logits, tokens, parents, uniforms, draft, race, temperature):
    got = t4.verify_drafts(logits, tokens, parents, uniforms=uniforms, draft=draft, race=race, temperature=temperature)
    count, path, said, logs = (t.cpu() for t in got)
    for b in range(logits.shape[0]):
        n, p, s, g = ref.walk(logits[b].cpu(), tokens[b].cpu(), parents[b].cpu(),
                              None if uniforms is None else uniforms[b].cpu(), None if draft is None else draft[b].cpu(),
                              None if race is None else race[b].cpu(), temperature)
        rest = logits.shape[1] - n
        assert int(count[b]) == n
        assert path[b].tolist() == p + [-1] * rest
        assert said[b].tolist() == s + [-1] * (rest - 1)
        for x, y in zip(logs[b].tolist(), g + [0.0] * (rest - 1)):
            assert abs(x - y) <= 2.0 ** -18 * (1 + abs(y))
    return count


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0])
@pytest.mark.parametrize("batch,nodes,vocab", [(1, 1, 1), (3, 2, 37), (2, 5, 1000), (4, 9, 8191), (3, 6, 8195),
                                               (2, 12, 32003), (2, 4, 128256), (1, 3, 262144)])
def test_verify(cuda, dtype, with_draft, temperature, batch, nodes, vocab):
    seed = vocab + nodes
    gen, rng = generator(seed), random.Random(seed)
    logits = (2 * torch.randn(batch, nodes, vocab, generator=gen, device="cuda")).to(dtype)
    parents = torch.tensor([ref.random_tree(rng, nodes)[0] for _ in range(batch)], dtype=torch.int32, device="cuda")
    tokens = torch.randint(0, vocab, (batch, nodes), generator=gen, device="cuda", dtype=torch.int32)
    noise = torch.randn(batch, nodes, vocab, generator=gen, device="cuda")
    for b in range(batch):
        for i in range(1, nodes):
            above = int(parents[b, i])
            noise[b, above, int(tokens[b, i])] += 8
            if rng.random() < 0.7:
                logits[b, above, int(tokens[b, i])] = math.log(vocab) + rng.uniform(0, 4)
    draft = torch.softmax(noise, dim=2) if with_draft else None
    uniforms = torch.rand(batch, nodes, generator=gen, device="cuda")
    race = torch.empty(batch, vocab, device="cuda").exponential_(generator=gen).clamp_min_(1e-30).reciprocal_()
    check_walk(logits, tokens, parents, uniforms, draft, race, temperature)


def test_verify_walks_to_a_leaf(cuda):
    vocab, nodes = 500, 7
    logits = torch.zeros(2, nodes, vocab, device="cuda")
    tokens = torch.arange(2 * nodes, dtype=torch.int32, device="cuda").view(2, nodes)
    parents = torch.tensor([list(range(-1, nodes - 1))] * 2, dtype=torch.int32, device="cuda")
    for i in range(nodes - 1):
        logits[torch.arange(2), i, tokens[:, i + 1].long()] = 60.0
    uniforms = torch.full((2, nodes), 0.999, device="cuda")
    race = torch.ones(2, vocab, device="cuda")
    for temperature in (0.0, 1.0):
        assert check_walk(logits, tokens, parents, uniforms, None, race, temperature).tolist() == [6, 6]


def test_verify_of_odd_rows_and_tokens(cuda):
    """Logits of -infinity, NaN and the type's lowest value, siblings alike, tokens outside the vocabulary."""
    vocab, nodes = 4099, 8
    gen = generator(21)
    logits = torch.randn(2, nodes, vocab, generator=gen, device="cuda").to(BF16)
    logits[:, :, ::3] = -math.inf
    logits[:, :, 1::7] = torch.finfo(BF16).min
    logits[:, 0, 5:50] = math.nan
    parents = torch.tensor([[-1, 0, 0, 0, 0, 0, 2, 2], [-1, 0, 0, 0, 1, 1, 1, 3]], dtype=torch.int32, device="cuda")
    tokens = torch.tensor([[0, 2, 2, -1, vocab, 2, 8, 8], [0, 3, 5, 1 << 30, 11, 11, -7, 20]], dtype=torch.int32,
                          device="cuda")
    uniforms = torch.tensor([[0, .9, .99, 0, 0, 0, .5, .5], [0, 0, 0, .9, .9, .9, 0, 0]], device="cuda")
    race = torch.empty(2, vocab, device="cuda").exponential_(generator=gen).reciprocal_()
    draft = torch.softmax(torch.randn(2, nodes, vocab, generator=gen, device="cuda"), dim=2)
    for temperature in (0.0, 1.0):
        check_walk(logits, tokens, parents, uniforms, None, race, temperature)
        check_walk(logits, tokens, parents, uniforms, draft, race, temperature)


def test_verify_of_a_row_with_no_probability(cuda):
    logits = torch.full((1, 3, 70), -math.inf, device="cuda")
    tokens = torch.tensor([[0, 4, 5]], dtype=torch.int32, device="cuda")
    parents = torch.tensor([[-1, 0, 0]], dtype=torch.int32, device="cuda")
    ones = torch.ones(1, 70, device="cuda")
    for draft in (None, torch.full((1, 3, 70), 1 / 70, device="cuda")):
        count, path, said, logs = t4.verify_drafts(logits, tokens, parents, draft=draft,
                                                   uniforms=torch.zeros(1, 3, device="cuda"), race=ones)
        assert count.tolist() == [0] and path.tolist() == [[-1] * 3] and said.tolist() == [[0, -1, -1]]
        assert logs.tolist() == [[-math.inf, 0.0, 0.0]]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_verify_of_a_residual_with_nothing_left(cuda, dtype):
    """The draft takes all that the target has: after each child turned down the node's softmax again."""
    vocab = 20011
    logits = torch.full((2, 4, vocab), -math.inf, device="cuda").to(dtype)
    logits[0, :, 17001] = 3.0
    logits[1, :, 5] = -2.0
    logits[1, :, 19999] = -2.0
    draft = torch.full((2, 4, vocab), 1 / 2, device="cuda")
    draft[0, :, 17001] = 1.0
    tokens = torch.tensor([[0, 4, 9, 17000], [0, 4, 5, 7]], dtype=torch.int32, device="cuda")
    parents = torch.tensor([[-1, 0, 0, 0], [-1, 0, 0, 2]], dtype=torch.int32, device="cuda")
    uniforms = torch.full((2, 4), 0.25, device="cuda")
    race = torch.ones(2, vocab, device="cuda")
    assert check_walk(logits, tokens, parents, uniforms, draft, race, 1.0).tolist() == [0, 1]


def test_verify_of_strided_tensors(cuda):
    gen = generator(23)
    batch, nodes, vocab = 3, 5, 1003
    logits = torch.randn(nodes, batch, vocab + 5, generator=gen, device="cuda").to(F16).transpose(0, 1)[..., 3:-2]
    logits[:, :, 7] = 9.0
    draft = torch.softmax(torch.randn(nodes, batch, vocab, generator=gen, device="cuda"), dim=2).transpose(0, 1)
    race = torch.empty(vocab, batch, device="cuda").exponential_(generator=gen).reciprocal_().t()
    tokens = torch.tensor([[0, 7, 7, 9, 7]] * batch, dtype=torch.int32, device="cuda")
    parents = torch.tensor([[-1, 0, 1, 2, 2]] * batch, dtype=torch.int32, device="cuda")
    uniforms = torch.rand(batch, nodes, generator=gen, device="cuda")
    check_walk(logits, tokens, parents, uniforms, draft, race, 1.0)
    check_walk(logits, tokens, parents, uniforms, draft[:, :1].expand(batch, nodes, vocab), race, 1.0)


def test_verify_of_many_children(cuda):
    """A root with hundreds of children, few of them likely."""
    gen = generator(24)
    nodes, vocab = 600, 2000
    logits = (3 * torch.randn(1, nodes, vocab, generator=gen, device="cuda")).to(BF16)
    tokens = torch.randint(0, vocab, (1, nodes), generator=gen, device="cuda", dtype=torch.int32)
    parents = torch.zeros(1, nodes, dtype=torch.int32, device="cuda")
    uniforms = torch.rand(1, nodes, generator=gen, device="cuda")
    race = torch.empty(1, vocab, device="cuda").exponential_(generator=gen).reciprocal_()
    check_walk(logits, tokens, parents, uniforms, None, race, 1.0)


@pytest.mark.parametrize("draws", [20000])
def test_tokens_follow_the_target(cuda, draws):
    """Whatever the drafts, the first token said follows softmax(logits): a chi-square statistic of 11
    degrees of freedom, below 40 with probability 1 - 4e-5 for each of the two forms."""
    gen = generator(25)
    vocab, nodes = 12, 4
    logits = torch.randn(1, 1, vocab, generator=gen, device="cuda").expand(draws, nodes, vocab)
    draft_row = torch.softmax(torch.randn(vocab, generator=gen, device="cuda"), dim=0)
    parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device="cuda").expand(draws, nodes).contiguous()
    uniforms = torch.rand(draws, nodes, generator=gen, device="cuda")
    race = torch.empty(draws, vocab, device="cuda").exponential_(generator=gen).reciprocal_()
    sampled = torch.multinomial(draft_row, draws * nodes, replacement=True, generator=gen).view(draws, nodes).int()
    fixed = torch.tensor([0, 3, 5, 1], dtype=torch.int32, device="cuda").expand(draws, nodes).contiguous()
    p = torch.softmax(logits[0, 0].double(), dim=0)
    for tokens, draft in ((fixed, None), (sampled, draft_row.expand(draws, nodes, vocab))):
        said = t4.verify_drafts(logits, tokens, parents, uniforms=uniforms, draft=draft, race=race)[2][:, 0]
        seen = torch.bincount(said.long(), minlength=vocab).double()
        assert float(((seen - draws * p) ** 2 / (draws * p)).sum()) < 40
