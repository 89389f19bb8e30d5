"""Refusals of the paged-cache entries, without a device: every check comes before the launch, so the
buffers are addresses that nothing reads."""
import ctypes

import pytest

import t4a_b200 as t4
from t4a_b200 import abi

RANK_LENGTH, NEGATIVE, SPAN, BROADCAST, DTYPE = 2, 3, 7, 8, 9
SHAPE, TOO_LARGE, STRIDE, OP, WORKSPACE, NULL = 16, 19, 20, 25, 65, 66
SOMEWHERE = 1 << 20


def described(shape, strides=None, offset=0):
    layout = abi.numpy_layout(shape, strides, offset)
    length = 0 if 0 in shape else 1 + offset + sum((e - 1) * s for e, s in zip(layout.extents_list(),
                                                                              layout.strides_list()) if s > 0)
    return layout, length


def cache_of(kind=abi.I8, pages=4, page=16, heads=2, dim=64, scale_shape=None, k=None, v=None, **fields):
    c = abi.KVCache()
    c.kind = kind
    for name, given in (("k", k), ("v", v)):
        layout, length = given or described([pages, page, heads, dim])
        setattr(c, name + "_layout", layout)
        setattr(c, name + "_len", length)
        setattr(c, name, SOMEWHERE)
        layout, length = described(scale_shape or [pages, page, heads])
        setattr(c, name + "_scale_layout", layout)
        setattr(c, name + "_scale_len", length)
        setattr(c, name + "_scale", SOMEWHERE)
    for name, value in fields.items():
        setattr(c, name, value)
    return c


def rows_call(cache, entry="t4a_cache_write", dtype=abi.BF16, index=abi.I64, key=None, value=None, slots=None,
              key_at=SOMEWHERE, slots_at=SOMEWHERE, n=8):
    key, value = key or described([n, 2, 64]), value or described([n, 2, 64])
    slots = slots or described([n])
    r = ctypes.byref
    return getattr(t4.lib(), entry)(None, dtype, index, r(cache) if cache is not None else None, key_at, r(key[0]),
                                    key[1], SOMEWHERE, r(value[0]), value[1], slots_at, r(slots[0]), slots[1])


@pytest.mark.parametrize("entry", ["t4a_cache_write", "t4a_cache_read"])
def test_rows(entry):
    def status(cache=None, **more):
        return rows_call(cache or cache_of(), entry=entry, **more)

    assert rows_call(None, entry=entry) == NULL
    assert status(cache_of(kind=abi.F32)) == DTYPE and status(cache_of(kind=77)) == DTYPE
    assert status(dtype=abi.F64) == DTYPE and status(dtype=abi.I8) == DTYPE
    assert status(index=abi.F32) == DTYPE
    for dim in (0, 8, 24, 272):
        assert status(cache_of(dim=dim), key=described([8, 2, dim]), value=described([8, 2, dim])) == SHAPE
    assert status(key=described([8, 3, 64])) == SHAPE and status(value=described([7, 2, 64])) == SHAPE
    assert status(key=described([8, 128])) == RANK_LENGTH and status(slots=described([8, 1])) == RANK_LENGTH
    assert status(key=(described([8, 2, 64])[0], 1023)) == SPAN
    assert status(slots=(described([8])[0], 7)) == SPAN
    assert status(key=described([8, 2, 64], [256, 128, 2])) == STRIDE  # rows without unit stride
    assert status(cache_of(k=described([4, 16, 2, 64], [2048 + 8, 128, 64, 1]))) == STRIDE  # rows off 16 bytes
    assert status(cache_of(k_scale=None)) == NULL and status(cache_of(v_scale=None)) == NULL
    assert status(cache_of(scale_shape=[4, 16, 3])) == SHAPE
    assert status(key_at=None) == NULL and status(slots_at=None) == NULL
    assert status(key_at=SOMEWHERE + 1) == STRIDE
    bad = cache_of()
    bad.k = None
    assert status(bad) == NULL
    bad = cache_of()
    bad.v = SOMEWHERE + 8
    assert status(bad) == STRIDE
    # Nothing to do is no error, whatever the buffers are.
    assert status(n=0, key_at=None, slots_at=None) == 0


def test_destinations_do_not_broadcast():
    c = cache_of(k=described([4, 16, 2, 64], [0, 128, 64, 1]))
    assert rows_call(c) == BROADCAST
    assert rows_call(cache_of(), entry="t4a_cache_read", key=described([8, 2, 64], [0, 64, 1])) == BROADCAST
    assert rows_call(cache_of(), key=described([8, 2, 64], [0, 64, 1]), n=0, slots=described([0])) == SHAPE


def attention_call(cache, dtype=abi.BF16, q=None, out=None, lse=None, table=None, mask=None, context=SOMEWHERE,
                   workspace=SOMEWHERE, bytes_=1 << 30, q_at=SOMEWHERE, mask_at=None, lse_at=SOMEWHERE):
    q, out = q or described([3, 5, 4, 64]), out or described([3, 5, 4, 64])
    lse, table = lse or described([3, 5, 4]), table or described([3, 7])
    mask = mask or described([3, 5, 5])
    r = ctypes.byref
    return t4.lib().t4a_tree_attention(None, dtype, r(cache), SOMEWHERE, r(out[0]), out[1], lse_at, r(lse[0]), lse[1],
                                       q_at, r(q[0]), q[1], SOMEWHERE, r(table[0]), table[1], context, None, mask_at,
                                       r(mask[0]), mask[1], 0.125, workspace, bytes_)


def test_attention():
    assert attention_call(cache_of(), dtype=abi.F32) == DTYPE
    assert attention_call(cache_of(kind=abi.F16)) == DTYPE  # a 16-bit cache has the queries' type
    assert attention_call(cache_of(heads=3)) == SHAPE  # query heads are a multiple
    assert attention_call(cache_of(), q=described([3, 5, 4, 32])) == SHAPE
    assert attention_call(cache_of(), q=described([3, 20, 64])) == RANK_LENGTH
    assert attention_call(cache_of(), out=described([3, 5, 4, 48])) == SHAPE
    assert attention_call(cache_of(), out=described([3, 5, 4, 64], [0, 256, 64, 1])) == BROADCAST
    assert attention_call(cache_of(), q=described([3, 5, 4, 64], [2560, 512, 128, 2])) == STRIDE
    assert attention_call(cache_of(), table=described([2, 7])) == SHAPE
    assert attention_call(cache_of(), table=(described([3, 7])[0], 20)) == SPAN
    assert attention_call(cache_of(), lse=described([3, 5, 2])) == SHAPE
    assert attention_call(cache_of(), mask=described([3, 5, 4]), mask_at=SOMEWHERE) == SHAPE
    assert attention_call(cache_of(), q_at=None) == NULL and attention_call(cache_of(), context=None) == NULL
    assert attention_call(cache_of(), q_at=SOMEWHERE + 1) == STRIDE
    assert attention_call(cache_of(), workspace=None) == WORKSPACE
    assert attention_call(cache_of(), bytes_=16) == WORKSPACE
    assert attention_call(cache_of(), workspace=SOMEWHERE + 4) == WORKSPACE
    assert attention_call(cache_of(), q=described([3, 1 << 25, 4, 64]), out=described([3, 1 << 25, 4, 64])) == TOO_LARGE
    for shape in ([0, 5, 4, 64], [3, 0, 4, 64], [3, 5, 0, 64]):
        assert attention_call(cache_of(), q=described(shape), out=described(shape), lse=described(shape[:3]),
                              table=described([shape[0], 7]), q_at=None, workspace=None) == 0


def test_workspace_needs_no_buffers_and_bounds_what_is_used():
    n = ctypes.c_size_t()
    sizes = {}
    for rows, (nodes, heads) in {"few": (1, 4), "many": (64, 8)}.items():
        c = cache_of(k_scale=None, v_scale=None)
        c.k = c.v = None
        q, table = described([3, nodes, heads, 64])[0], described([3, 7])[0]
        assert t4.lib().t4a_tree_attention_workspace_bytes(abi.F16, ctypes.byref(c), ctypes.byref(q),
                                                           ctypes.byref(table), ctypes.byref(n)) == 0
        sizes[rows] = n.value
    assert 0 < sizes["few"] < sizes["many"] < 64 << 20
    assert t4.lib().t4a_tree_attention_workspace_bytes(abi.F16, ctypes.byref(cache_of()), None, None,
                                                       ctypes.byref(n)) == NULL


def verify_call(dtype=abi.BF16, logits=None, draft=None, race=None, temperature=1.0, logits_at=SOMEWHERE,
                uniforms=SOMEWHERE, draft_at=None, race_at=SOMEWHERE, count=SOMEWHERE):
    logits, draft = logits or described([3, 5, 100]), draft or described([3, 5, 100])
    race = race or described([3, 100])
    r = ctypes.byref
    return t4.lib().t4a_verify_drafts(None, dtype, logits_at, r(logits[0]), logits[1], SOMEWHERE, SOMEWHERE, uniforms,
                                      draft_at, r(draft[0]), draft[1], race_at, r(race[0]), race[1], temperature, count,
                                      SOMEWHERE, SOMEWHERE, None)


def test_verify():
    assert verify_call(dtype=abi.F64) == DTYPE and verify_call(dtype=abi.I8) == DTYPE
    assert verify_call(logits=described([3, 500])) == RANK_LENGTH
    assert verify_call(logits=described([3, 5, 100], [1000, 200, 2])) == STRIDE
    assert verify_call(logits=(described([3, 5, 100])[0], 1499)) == SPAN
    for shape in ([3, 0, 100], [3, 5, 0]):
        assert verify_call(logits=described(shape)) == SHAPE
    assert verify_call(logits=described([0, 5, 100]), logits_at=None) == 0
    assert verify_call(temperature=-1.0) == OP and verify_call(temperature=float("nan")) == OP
    assert verify_call(temperature=float("inf")) == OP
    assert verify_call(logits_at=None) == NULL and verify_call(count=None) == NULL
    assert verify_call(uniforms=None) == NULL and verify_call(race_at=None) == NULL
    assert verify_call(race=described([3, 99])) == SHAPE
    assert verify_call(draft=described([3, 4, 100]), draft_at=SOMEWHERE) == SHAPE
    assert verify_call(logits_at=SOMEWHERE + 1) == STRIDE
    assert verify_call(logits=described([1, 2000, 100]), race=described([1, 100])) == TOO_LARGE  # nodes
    assert verify_call(dtype=abi.F32, logits=described([1, 1, 1 << 20]), race=described([1, 1 << 20])) == TOO_LARGE
