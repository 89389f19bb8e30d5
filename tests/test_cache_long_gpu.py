"""Attention where a block has thousands of tiles: products truncate as they add, so long sums are taken in passes.

Bounds are those of the other attention tests: (u_weight + u_out + 2^-13) * sum w|v|, the last term for what F32
products, exponentials and sums lose.
"""
import math

import pytest
import torch

import cache_reference as ref
import t4a_b200 as t4
from test_cache_gpu import BF16, E4M3, F16, I8, KINDS, UNIT, attention_case, check_attention, generator

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("nodes,group", [(1, 4), (2, 8), (20, 2)])
@pytest.mark.parametrize("context", [131072, 1 << 20])
def test_long_sums_of_one_sign(cuda, kind, dtype, nodes, group, context):
    """A sequence a block, over positive values: what one addition loses, all lose."""
    batch, page, dim = 592, 1024, 64
    gen = generator(nodes)
    k, v, ks, vs = ref.random_cache(gen, 1, page, 1, dim, kind)  # a page that all places lead to
    v = (v.float().abs() / v.float().abs().max() / 4 + 0.75).to(kind) if ks is None else (64 + v.float().abs() / 8).to(kind)
    q = (0.5 * torch.randn(1, nodes, group, dim, generator=gen, device="cuda")).to(dtype)
    table = torch.zeros(batch, context // page + 1, dtype=torch.int32, device="cuda")
    nothing = torch.zeros(1, nodes, nodes, dtype=torch.bool, device="cuda")
    out, lse = t4.tree_attention(q.expand(batch, nodes, group, dim), k, v, table,
                                 torch.full((batch,), context, dtype=torch.int32, device="cuda"),
                                 mask=nothing.expand(batch, nodes, nodes), k_scale=ks, v_scale=vs)
    live = torch.full((1,), nodes, device="cuda")
    want, want_lse, spread, size = ref.attention(q, k, v, ks, vs, table[:1, :2], torch.full((1,), page), nothing, live,
                                                 dim ** -0.5)
    u = (UNIT[BF16] if kind == BF16 else UNIT[F16]) + UNIT[dtype] + 2.0 ** -13
    assert float(((out.double() - want).abs() / spread).max()) <= u
    off = (lse.double() - want_lse - math.log(context // page)).abs()
    assert float((off / (size + want_lse.abs() + 1)).max()) <= 2.0 ** -18


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("nodes,group,dim", [(1, 4, 64), (2, 8, 64), (8, 4, 64), (20, 2, 64), (2, 4, 112), (20, 2, 112),
                                             (2, 8, 256)])
def test_units_of_several_passes(cuda, kind, dtype, nodes, group, dim):
    """Blocks with whole units and parts of units, of several passes and of one."""
    contexts, repeat = [70000, 45000, 33000, 64 * 512 + 5, 9000, 64 * 128 - 20, 0], 200
    c = attention_case(nodes + dim, len(contexts), nodes, 1, group, dim, 64, contexts, kind, dtype,
                       live=[nodes] * 6 + [nodes - 1])
    c["table"][0, 20:40] = -1  # more than a pass's first 10 tiles, and none of another's
    c["table"][1, 128:256] = -1
    if c["vs"] is not None:
        c["vs"][c["table"][2, :200].long()] = 0
    some = torch.arange(len(contexts), device="cuda").repeat(repeat)
    out, lse = t4.tree_attention(c["q"][some], c["k"], c["v"], c["table"][some], c["context"][some],
                                 mask=c["sees"][some], nodes=c["live"][some], k_scale=c["ks"], v_scale=c["vs"])
    want, want_lse, spread, size = ref.attention(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], c["context"],
                                                 c["sees"], c["live"], dim ** -0.5)
    u = (UNIT[BF16] if kind == BF16 else UNIT[F16]) + UNIT[dtype] + 2.0 ** -13
    off = (out.double() - want[some]).abs() / (u * spread + 2.0 ** -24)[some]
    assert torch.isfinite(out).all() and float(off.max()) <= 1
    empty = want_lse[some] == -torch.inf
    assert torch.equal(lse == -torch.inf, empty)
    off = (lse.double() - want_lse[some]).abs() / (2.0 ** -18 * (size + want_lse.abs() + 1))[some]
    assert float(off[~empty].max()) <= 1


@pytest.mark.parametrize("nodes,group", [(1, 4), (20, 2)])
def test_places_near_the_most(cuda, nodes, group):
    """2047 entries of a table that lead to one page of 2^20 places: sequences whose places almost fill 31 bits."""
    page, dim = 1 << 20, 64
    gen = generator(nodes)
    k, v, ks, vs = ref.random_cache(gen, 1, page, 1, dim, torch.int8)
    q = torch.randn(1, nodes, group, dim, generator=gen, device="cuda").half()
    table = torch.zeros(1, 2047, dtype=torch.int32, device="cuda")
    context = torch.full((1,), 2047 * page - nodes, dtype=torch.int32, device="cuda")
    sees = torch.ones(1, nodes, nodes, dtype=torch.bool, device="cuda")
    out, lse = t4.tree_attention(q, k, v, table, context, mask=sees, k_scale=ks, v_scale=vs)
    want, want_lse, spread, size = ref.attention(q, k, v, ks, vs, table[:, :1], torch.full((1,), page - nodes), sees,
                                                 torch.full((1,), nodes), dim ** -0.5)
    assert float(((out.double() - want).abs() / spread).max()) <= 2 * UNIT[F16] + 2.0 ** -13
    off = (lse.double() - want_lse - math.log(2047)).abs()
    assert float((off / (size + want_lse.abs() + 1)).max()) <= 2.0 ** -18


@pytest.mark.parametrize("kind,dtype,nodes,group,dim,context", [(I8, BF16, 300, 128, 64, 9000), (F16, F16, 300, 128, 64, 9000),
                                                                (E4M3, F16, 40, 120, 256, 33000), (BF16, BF16, 40, 120, 256, 33000)])
def test_several_passes_of_more_row_tiles_than_blocks(cuda, kind, dtype, nodes, group, dim, context):
    """Every tile of query rows has a block of its own, which goes over the whole cache in passes."""
    check_attention(attention_case(dim, 1, nodes, 1, group, dim, 64, [context], kind, dtype))
