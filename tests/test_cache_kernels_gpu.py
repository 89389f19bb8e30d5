"""tree_attention at row counts that reach each of its kernels, in forms where they differ.

With 2 cache heads: 6 query rows a cache head take the warp-level kernel for every cache, 24 the warp-level
one or tensor memory by the cache's kind and dim, 40 and 136 tensor memory (one tile of rows, and two).  Bounds
are those of check_attention.
"""
import math

import pytest
import torch

import cache_reference as ref
import t4a_b200 as t4
from test_cache_gpu import (BF16, E4M3, F16, I8, KINDS, UNIT, attention_case, check_attention, generator,
                            poison_unused)

pytestmark = pytest.mark.gpu

ROWS = [(3, 2), (12, 2), (20, 2), (34, 4)]  # nodes, query heads to a cache head


def poison_pages(c, pages):
    """Rows of these pages hold the worst that they could."""
    for name in ("k", "v"):
        if c[name].dtype in (F16, BF16):
            c[name][pages] = math.nan
        else:
            c[name + "s"][pages] = math.nan
            if c[name].dtype == E4M3:
                c[name].view(torch.uint8)[pages] = 0x7f


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("nodes,group", ROWS)
@pytest.mark.parametrize("dim", [64, 128])
def test_pages_outside_the_cache(cuda, kind, dtype, nodes, group, dim):
    """Whole tiles of 64 places and parts of tiles, in the context, among the drafted rows and first of all."""
    c = attention_case(nodes + dim, 3, nodes, 2, group, dim, 16, [700, 333, 90], kind, dtype)
    poison_unused(c)
    outside = {0: [4, 5, 6, 7, 9, 20, 41], 1: [0, 15, 16, 333 // 16], 2: [90 // 16]}
    for b, pages in outside.items():
        poison_pages(c, c["table"][b, pages].long())
        for i, page in enumerate(pages):
            c["table"][b, page] = [-1, c["k"].shape[0], 1 << 30, -(1 << 31)][i % 4]
    check_attention(c)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("nodes,group", ROWS)
def test_a_cache_that_no_table_reaches(cuda, kind, dtype, nodes, group):
    c = attention_case(nodes, 2, nodes, 2, group, 64, 16, [300, 17], kind, dtype)
    poison_pages(c, slice(None))
    c["table"][:] = -1
    out, lse = check_attention(c)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("nodes,group", [(2, 3), (4, 4), *ROWS])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("worst", [math.nan, math.inf, 1e20, 3e38])
def test_queries_of_dead_nodes_may_hold_anything(cuda, kind, dtype, nodes, group, dim, worst):
    c = attention_case(nodes * 7 + dim, 3, nodes, 2, group, dim, 16, [70, 33, 200], kind, dtype,
                       live=[nodes - 1, 1, (nodes + 1) // 2])
    for b in range(3):
        c["q"][b, int(c["live"][b]):] = min(worst, torch.finfo(dtype).max) if math.isfinite(worst) else worst
    out, lse = check_attention(c)
    for b in range(3):
        assert (out[b, int(c["live"][b]):] == 0).all() and (lse[b, int(c["live"][b]):] == -math.inf).all()


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("nodes,group", [(2, 3), (4, 4), *ROWS])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_query_rows_of_very_different_sizes(cuda, kind, nodes, group, dim):
    """Every row has the precision of its own magnitude, whatever the rows beside it hold."""
    c = attention_case(nodes * 5 + dim, 2, nodes, 2, group, dim, 16, [90, 33], kind, BF16)
    heads = torch.arange(2 * group, device="cuda")
    for i in range(nodes):
        size = torch.tensor([1.0, 1e-30, 1e12, 1e-3, 3e4, 1e20, 1.0], device="cuda")[(heads + i) % 7]
        c["q"][:, i] = (c["q"][:, i].float() * size[:, None]).to(BF16)
    check_attention(c)


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("nodes,group", ROWS)
def test_queries_near_the_largest_float(cuda, kind, nodes, group):
    """Scores of some 1e36 are finite, and so is what leads to them."""
    c = attention_case(nodes * 3, 2, nodes, 2, group, 128, 16, [90, 33], kind, BF16)
    c["q"] = (c["q"].float() * 1e36).to(BF16)
    check_attention(c)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("nodes,group", ROWS)
@pytest.mark.parametrize("scale", [3e5, -1e8, 1e10, 1e22])
def test_large_scores(cuda, kind, dtype, nodes, group, scale):
    """Scores whose last place is larger than the exponentials' range."""
    c = attention_case(nodes * 3, 2, nodes, 2, group, 64, 16, [90, 333], kind, dtype)
    check_attention(c, scale=scale)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("nodes,group", ROWS)
def test_scores_far_below_zero(cuda, kind, dtype, nodes, group):
    """All of a row's scores below -1e30: the row sees its tokens all the same."""
    c = attention_case(nodes * 3, 2, nodes, 2, group, 64, 16, [90, 333], kind, dtype)
    c["q"] = c["q"].abs()
    c["k"] = -c["k"].abs() if kind != E4M3 else (-c["k"].float().abs()).to(kind)
    out, lse = check_attention(c, scale=1e32)
    assert float(lse.max()) < -1e30


def check_relative(c):
    """As check_attention, for outputs far from 1: errors go by the outputs' own magnitudes alone."""
    scale = c["q"].shape[3] ** -0.5
    out, lse = t4.tree_attention(c["q"], c["k"], c["v"], c["table"], c["context"], mask=c["sees"], k_scale=c["ks"],
                                 v_scale=c["vs"])
    want, want_lse, spread, size = ref.attention(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], c["context"],
                                                 c["sees"], c["live"], scale)
    u = (UNIT[BF16] if c["k"].dtype == BF16 else UNIT[F16]) + UNIT[c["q"].dtype] + 2.0 ** -13
    assert float(((out.double() - want).abs() / spread).max()) <= u
    assert float(((lse.double() - want_lse).abs() / (size + want_lse.abs() + 1)).max()) <= 2.0 ** -18


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("nodes,group", ROWS)
@pytest.mark.parametrize("least", [2.0 ** -100, 1.5 * 2.0 ** -99])
def test_the_smallest_rows_that_are_kept(cuda, kind, nodes, group, least):
    """V rows whose largest magnitude is the least that the writer does not store as zeros."""
    c = attention_case(nodes, 2, nodes, 2, group, 64, 16, [90, 33], kind, BF16)
    rows = c["v"].shape[0] * 16
    gen = generator(nodes)
    value = torch.rand(rows, 2, 64, generator=gen, device="cuda") * 2 - 1
    value = (value / value.abs().amax(dim=2, keepdim=True)).clamp(-1, 1) * least
    key = torch.randn(rows, 2, 64, generator=gen, device="cuda")
    t4.cache_write(key, value, c["k"], c["v"], torch.arange(rows, device="cuda"), k_scale=c["ks"], v_scale=c["vs"])
    assert (c["vs"] > 0).all()
    check_relative(c)


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("nodes,group", ROWS)
def test_scales_below_zero_show(cuda, kind, nodes, group):
    """No writer makes a V scale below zero: who sees its row gets NaN, who does not its usual result."""
    c = attention_case(nodes, 2, nodes, 2, group, 64, 16, [40, 117], kind, BF16)
    want, want_lse = check_attention(c)
    for b, place in ((0, 40 + 1), (1, 117 + 1)):
        c["vs"][int(c["table"][b, place // 16]), place % 16] = -0.01
    out, lse = t4.tree_attention(c["q"], c["k"], c["v"], c["table"], c["context"], mask=c["sees"], k_scale=c["ks"],
                                 v_scale=c["vs"])
    reached = c["sees"][:, :, 1][:, :, None].expand(lse.shape)
    assert reached.any() and not reached.all()
    assert torch.isnan(lse[reached]).all() and torch.isnan(out[reached]).all()
    assert torch.equal(out[~reached], want[~reached]) and torch.equal(lse[~reached], want_lse[~reached])


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("nodes,group", ROWS)
def test_value_scales_as_far_apart_as_they_may_be(cuda, kind, nodes, group):
    """Scales of V from 2^-45 to 2^45: rows that hardly matter to the output count in the softmax all the same."""
    c = attention_case(nodes, 2, nodes, 2, group, 64, 16, [150, 700], kind, BF16)
    gen = generator(nodes)
    ends = torch.where(torch.rand(c["vs"].shape, generator=gen, device="cuda") < 0.1, 45.0, -45.0)
    c["vs"] = torch.exp2(ends)
    check_relative(c)


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("nodes,group", ROWS)
def test_a_weight_is_rounded_once(cuda, kind, nodes, group):
    """A maximum that rises within a tile by a factor that would round the weights before it once more, in the
    same direction for all of them, as the output's own rounding."""
    c = attention_case(nodes, 1, nodes, 2, group, 64, 16, [64], kind, F16)
    near = 1 + 0.98 * 2.0 ** -11  # F16 rounds it down to 1
    score = torch.full((64,), -200.0, dtype=torch.float64)  # in powers of two
    score[0], score[1:32], score[32] = 0.0, math.log2(near) - 1, 9 - math.log2(near)
    weight = torch.exp2(score)
    value = torch.where((score < 0) & (score > -2), 96.0, 0.0)
    c["q"][:] = 0
    c["q"][..., 0] = 1
    c["sees"][:] = False
    slot = (c["table"][0].long()[:, None] * 16 + torch.arange(16, device="cuda")).flatten()[:64]
    out = float((weight * value).sum() / weight.sum())
    three = near / (1 - 2 * 0.98 * 2.0 ** -11)  # what is left after two roundings down is `near` again
    size = three * 2.0 ** math.floor(math.log2(out)) / out
    for name, codes in (("k", torch.eye(1, 64).expand(64, 64)), ("v", value[:, None].expand(64, 64))):
        c[name].view(-1, 2, 64)[slot] = codes.to("cuda")[:, None].expand(64, 2, 64).to(kind)
    c["ks"].view(-1, 2)[slot] = (score / math.log2(math.e)).float().to("cuda")[:, None]
    c["vs"][:] = size
    check_attention(c, scale=1.0)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("nodes,group", ROWS)
def test_contexts_past_the_table_and_below_zero(cuda, kind, dtype, nodes, group):
    c = attention_case(nodes + 1, 4, nodes, 2, group, 64, 16, [200] * 4, kind, dtype)
    places = c["table"].shape[1] * 16
    c["context"] = torch.tensor([places - nodes // 2, places + 5, 1 << 30, -7], dtype=torch.int32, device="cuda")
    check_attention(c)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("nodes,group", ROWS)
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.3, 1.7])
def test_score_scales(cuda, kind, dtype, nodes, group, scale):
    check_attention(attention_case(nodes + 2, 2, nodes, 2, group, 64, 16, [170, 5], kind, dtype), scale=scale)


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("nodes,group", ROWS)
@pytest.mark.parametrize("size", [0.0, 1e-30, 1e-6, 1e6])
def test_value_rows_of_zero_and_of_very_different_sizes(cuda, kind, dtype, nodes, group, size):
    """Zero rows of V in the context, among the drafted rows, as a whole tile and as all that a node sees."""
    c = attention_case(nodes + 3, 3, nodes, 2, group, 128, 16, [400, 90, 0], kind, dtype)
    c["vs"][::2] *= size if dtype == BF16 or size < 1 else 1e2
    c["vs"][1] = 0
    c["vs"][c["table"][0, 8:12].long()] = 0
    c["vs"][c["table"][2].long()] = 0
    c["k"].view(torch.int8)[2] = 0
    check_attention(c)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("nodes,group", ROWS)
@pytest.mark.parametrize("dim", [64, 128])
def test_maxima_that_rise_late_and_early(cuda, kind, dtype, nodes, group, dim):
    """One sequence over many blocks, and short ones in one; rows whose best token comes first, last and between,
    in either half of a tile, each some hundreds of powers of two above the rest."""
    c = attention_case(nodes + 4, 3, nodes, 2, group, dim, 16, [9000, 300, 64], kind, dtype)
    for b, length in enumerate((9000, 300, 64)):
        for i in range(nodes):
            place = [0, length - 1, length // 2, 31, 33, 63, length - 33][i % 7]
            row = c["k"][int(c["table"][b, place // 16]), place % 16].float()
            c["q"][b, i] = (row.sign() * 3).repeat_interleave(group, dim=0).to(dtype)
    check_attention(c)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("nodes,group", ROWS)
@pytest.mark.parametrize("gap", [1, 2, 4])
def test_rows_off_16_bytes(cuda, kind, dtype, nodes, group, gap):
    """Queries and outputs at 2-, 4- and 8-byte boundaries, heads and batch in other orders, caches by heads."""
    c = attention_case(nodes + 5, 3, nodes, 2, group, 80, 8, [130, 9, 700], kind, dtype)
    for name in ("k", "v"):
        c[name] = c[name].transpose(1, 2).contiguous().transpose(1, 2)
        if c[name + "s"] is not None:
            c[name + "s"] = c[name + "s"].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    wide = torch.zeros(3, nodes, 2 * group * 80 + gap, dtype=dtype, device="cuda")
    q = wide[:, :, gap:].unflatten(2, (2 * group, 80))
    q.copy_(c["q"])
    c["q"] = q
    out = torch.zeros(2 * group, 3, nodes, 80 + gap, dtype=dtype, device="cuda").permute(1, 2, 0, 3)[..., gap:]
    check_attention(c, out=out)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("nodes,group", ROWS)
@pytest.mark.parametrize("dim", [64, 128])
def test_values_that_are_no_numbers(cuda, kind, dtype, nodes, group, dim):
    """NaN and infinite V values in several drafted rows reach the nodes that see them, also where a page of the
    context lies outside the cache, and in the tile that context and drafts share."""
    c = attention_case(nodes + 6, 3, nodes, 2, group, dim, 16, [700, 333, 90], kind, dtype)
    clean = {k: t.clone() if torch.is_tensor(t) else t for k, t in c.items()}
    reached = torch.zeros(3, nodes, dtype=torch.bool, device="cuda")
    for b in range(3):
        for x in (c, clean):
            x["table"][b, [1, 3]] = torch.tensor([-1, 1 << 30], dtype=torch.int32, device="cuda")
        for bad in (nodes - 1, nodes // 2):
            place = int(c["context"][b]) + bad
            at = (int(c["table"][b, place // 16]), place % 16)
            if kind == I8:
                c["vs"][at] = math.nan
            elif kind == E4M3:
                c["v"].view(torch.uint8)[at] = 0x7f
            else:
                c["v"][at] = math.nan if b else math.inf
            reached[b] |= c["sees"][b, :, bad]
    out, lse = t4.tree_attention(c["q"], c["k"], c["v"], c["table"], c["context"], mask=c["sees"], k_scale=c["ks"],
                                 v_scale=c["vs"])
    want, want_lse, spread, size = ref.attention(clean["q"], clean["k"], clean["v"], clean["ks"], clean["vs"],
                                                 clean["table"], clean["context"], clean["sees"], clean["live"],
                                                 dim ** -0.5)
    assert reached.any() and not torch.isfinite(out[reached]).any() and torch.isfinite(out[~reached]).all()
    u = (UNIT[BF16] if kind == BF16 else UNIT[F16]) + UNIT[dtype] + 2.0 ** -13
    assert float(((out.double() - want).abs() - u * spread - 2.0 ** -24)[~reached].max()) <= 0
    assert float(((lse.double() - want_lse).abs() / (size + want_lse.abs() + 1))[~reached].max()) <= 2.0 ** -18
