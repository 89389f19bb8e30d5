"""Paged-cache operators over torch tensors (include/t4a_b200/cache.h): rows written into
a cache of pages (quantised where it holds 8-bit codes) and read back, attention of a
tree of drafted tokens over it, and the verification of the drafts.

Tensors are row-major views of the C layouts: a cache side is [pages, page_size, heads,
dim] (float16, bfloat16, int8 or float8_e4m3fn; any strides but 1 along dim), its scales
[pages, page_size, heads] float32.  Metadata is checked by the library, which refuses
with a T4AError; what ctypes could not pass on safely (a wrong dtype or device) is a
TypeError or ValueError here.  Layouts are kept by shape and strides, so that a call on
shapes seen before costs a few microseconds on the host.
"""
import ctypes
import functools

from . import abi
from .abi import F32, I32, I64, F16, BF16, I8, E4M3, KVCache, Layout

_ROW_TAGS = {}
_CACHE_TAGS = {}


def _tags():
    import torch
    _ROW_TAGS.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
    _CACHE_TAGS.update({torch.float16: F16, torch.bfloat16: BF16, torch.int8: I8, torch.float8_e4m3fn: E4M3})


def declare(l):
    """Signatures of the entries (called when the library is loaded)."""
    P, I, LL, SZ, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t, ctypes.c_float
    rows = [P, I, I, P, P, P, LL, P, P, LL, P, P, LL]
    for name, args in {
        "t4a_cache_write": rows,
        "t4a_cache_read": rows,
        "t4a_tree_attention_workspace_bytes": [I, P, P, P, ctypes.POINTER(SZ)],
        "t4a_tree_attention": [P, I, P, P, P, LL, P, P, LL, P, P, LL, P, P, LL, P, P, P, P, LL, F, P, SZ],
        "t4a_verify_drafts": [P, I, P, P, LL, P, P, P, P, P, LL, P, P, LL, F, P, P, P, P],
    }.items():
        fn = getattr(l, name)
        fn.restype, fn.argtypes = I, args


@functools.lru_cache(maxsize=4096)
def _described(shape, strides):
    """(address of a t4a_cuda_layout, reachable elements, the layout itself to keep it alive)."""
    layout = abi.numpy_layout(shape, strides)
    count = 0 if 0 in shape else 1 + sum((e - 1) * s for e, s in zip(shape, strides))
    return ctypes.addressof(layout), count, layout


@functools.lru_cache(maxsize=1024)
def _cache_template(kind, k, v, k_scale, v_scale):
    """The bytes of a t4a_kv_cache but for its pointers; each side is (shape, strides)."""
    c = KVCache()
    c.kind = kind
    for name, side in (("k", k), ("v", v), ("k_scale", k_scale), ("v_scale", v_scale)):
        if side is not None:
            _, count, layout = _described(*side)
            setattr(c, name + "_layout", layout)
            setattr(c, name + "_len", count)
    return bytes(c)


def _form(t):
    return tuple(t.shape), t.stride()


def _need(t, name, dtypes, device):
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: {t.dtype} is not supported")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")


def _device(t, name):
    import torch
    if not t.is_cuda:
        raise ValueError(f"{name} is not a CUDA tensor")
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"{name} is on {t.device}, which is not the current device")
    if not _ROW_TAGS:
        _tags()
    return t.device


def _cache(k_cache, v_cache, k_scale, v_scale, device):
    """The t4a_kv_cache of these tensors."""
    import torch
    _need(k_cache, "k_cache", _CACHE_TAGS, device)
    _need(v_cache, "v_cache", (k_cache.dtype,), device)
    kind = _CACHE_TAGS[k_cache.dtype]
    scaled = kind in (I8, E4M3)
    if scaled != (k_scale is not None) or scaled != (v_scale is not None):
        raise ValueError("k_scale and v_scale go with an 8-bit cache, and only with one")
    if scaled:
        _need(k_scale, "k_scale", (torch.float32,), device)
        _need(v_scale, "v_scale", (torch.float32,), device)
    c = KVCache.from_buffer_copy(_cache_template(kind, _form(k_cache), _form(v_cache),
                                                 _form(k_scale) if scaled else None,
                                                 _form(v_scale) if scaled else None))
    c.k, c.v = k_cache.data_ptr(), v_cache.data_ptr()
    if scaled:
        c.k_scale, c.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
    return c


def _check(status, where):
    if status != 0:
        from . import T4AError
        raise T4AError(status, where)


def _lib():
    from . import lib
    return lib()


def _stream(stream):
    import torch
    return (stream if stream is not None else torch.cuda.current_stream()).cuda_stream


def _used_on(stream, *tensors):
    """Tells the allocator that tensors made here are used on a stream that is not the current one."""
    import torch
    if stream is not None and stream != torch.cuda.current_stream():
        for t in tensors:
            t.record_stream(stream)


def _rows_call(entry, where, dtype, cache, key, value, slots, stream):
    import torch
    if slots.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"slots: {slots.dtype} is not supported")
    kl, kn, _ = _described(*_form(key))
    vl, vn, _ = _described(*_form(value))
    sl, sn, _ = _described(*_form(slots))
    _check(entry(_stream(stream), dtype, I64 if slots.dtype == torch.int64 else I32, ctypes.addressof(cache),
                 key.data_ptr(), kl, kn, value.data_ptr(), vl, vn, slots.data_ptr(), sl, sn), where)


def cache_write(key, value, k_cache, v_cache, slots, k_scale=None, v_scale=None, stream=None):
    """Rows key[n], value[n] ([n, heads, dim]; float32, float16 or bfloat16) into the cache at
    slots[n] = page * page_size + place (int32 or int64; outside the cache: dropped).  An 8-bit
    cache takes codes and one scale a row: scale = max|x| / 127 (int8) or / 448 (float8_e4m3fn)."""
    device = _device(key, "key")
    _need(key, "key", _ROW_TAGS, device)
    _need(value, "value", (key.dtype,), device)
    _need(slots, "slots", (slots.dtype,), device)
    _rows_call(_lib().t4a_cache_write, "cache_write", _ROW_TAGS[key.dtype],
               _cache(k_cache, v_cache, k_scale, v_scale, device), key, value, slots, stream)


def cache_read(k_cache, v_cache, slots, dtype, k_scale=None, v_scale=None, out=None, stream=None):
    """(key, value) [n, heads, dim] in `dtype` (float32, float16 or bfloat16): the rows at slots[n]
    as the values they stand for; zeros for a slot outside the cache.  `out`: a pair to write to."""
    import torch
    device = _device(k_cache, "k_cache")
    if dtype not in _ROW_TAGS:
        raise TypeError(f"cache_read: {dtype} is not supported")
    _need(slots, "slots", (slots.dtype,), device)
    if out is None:
        shape = (slots.shape[0], k_cache.shape[2], k_cache.shape[3])
        key, value = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        _used_on(stream, key, value)
    else:
        key, value = out
        _need(key, "out[0]", (dtype,), device)
        _need(value, "out[1]", (dtype,), device)
    _rows_call(_lib().t4a_cache_read, "cache_read", _ROW_TAGS[dtype],
               _cache(k_cache, v_cache, k_scale, v_scale, device), key, value, slots, stream)
    return key, value


@functools.lru_cache(maxsize=1024)
def _attention_bytes(dtype, template, q_form, table_form):
    n = ctypes.c_size_t()
    c = KVCache.from_buffer_copy(template)
    _check(_lib().t4a_tree_attention_workspace_bytes(dtype, ctypes.addressof(c), _described(*q_form)[0],
                                                     _described(*table_form)[0], ctypes.byref(n)),
           "tree_attention_workspace_bytes")
    return n.value


def tree_attention_workspace_bytes(q, k_cache, v_cache, page_table, k_scale=None, v_scale=None):
    """Bytes of workspace that tree_attention needs for these tensors' shapes."""
    device = _device(q, "q")
    _need(q, "q", _ROW_TAGS, device)
    c = _cache(k_cache, v_cache, k_scale, v_scale, device)
    return _attention_bytes(_ROW_TAGS[q.dtype], bytes(c), _form(q), _form(page_table))


def tree_attention(q, k_cache, v_cache, page_table, context, mask=None, nodes=None, k_scale=None, v_scale=None,
                   scale=None, out=None, lse=None, workspace=None, stream=None):
    """Attention of drafted nodes q ([batch, nodes, query heads, dim], float16 or bfloat16) to each
    sequence's context[b] committed tokens and to the nodes that they see; node j lies at place
    context[b] + j of the pages page_table[b] (int32).  mask [batch, nodes, nodes] (bool or uint8):
    whether node i sees node j; None: a chain, j <= i.  nodes [batch] (int32): live nodes.
    scale: dim ** -0.5 unless given.  One node is the decoding step of a single token.
    Returns (out like q, lse [batch, nodes, query heads] float32); a node that sees nothing gets
    zeros and -infinity."""
    import torch
    device = _device(q, "q")
    _need(q, "q", (torch.float16, torch.bfloat16), device)
    _need(page_table, "page_table", (torch.int32,), device)
    _need(context, "context", (torch.int32,), device)
    if q.dim() != 4:
        raise ValueError("q is [batch, nodes, query heads, dim]")
    batch, count, heads, dim = q.shape
    for name, t in (("context", context), ("nodes", nodes)):
        if t is None:
            continue
        _need(t, name, (torch.int32,), device)
        if t.shape != (batch,) or not t.is_contiguous():
            raise ValueError(f"{name} is a contiguous [batch]")
    c = _cache(k_cache, v_cache, k_scale, v_scale, device)
    tag = _ROW_TAGS[q.dtype]
    q_form, table_form = _form(q), _form(page_table)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
        _used_on(stream, out)
    else:
        _need(out, "out", (q.dtype,), device)
    if lse is None:
        lse = torch.empty((batch, count, heads), dtype=torch.float32, device=device)
        _used_on(stream, lse)
    else:
        _need(lse, "lse", (torch.float32,), device)
    template = _cache_template(c.kind, _form(k_cache), _form(v_cache), _form(k_scale) if k_scale is not None else None,
                               _form(v_scale) if v_scale is not None else None)
    if workspace is None:
        workspace = torch.empty(_attention_bytes(tag, template, q_form, table_form), dtype=torch.uint8, device=device)
        _used_on(stream, workspace)
    else:
        _need(workspace, "workspace", (torch.uint8,), device)
    if mask is not None:
        _need(mask, "mask", (torch.bool, torch.uint8), device)
        ml, mn, _ = _described(*_form(mask))
    ql, qn, _ = _described(*q_form)
    ol, on, _ = _described(*_form(out))
    ll, ln, _ = _described(*_form(lse))
    tl, tn, _ = _described(*table_form)
    _check(_lib().t4a_tree_attention(
        _stream(stream), tag, ctypes.addressof(c), out.data_ptr(), ol, on, lse.data_ptr(), ll, ln, q.data_ptr(), ql, qn,
        page_table.data_ptr(), tl, tn, context.data_ptr(), None if nodes is None else nodes.data_ptr(),
        None if mask is None else mask.data_ptr(), None if mask is None else ml, 0 if mask is None else mn,
        dim ** -0.5 if scale is None else scale, workspace.data_ptr(), workspace.numel()), "tree_attention")
    return out, lse


def verify_drafts(logits, tokens, parents, uniforms=None, draft=None, race=None, temperature=1.0, stream=None):
    """Walks each sequence's tree of drafted tokens: logits [batch, nodes, vocab] after each node,
    tokens and parents [batch, nodes] int32 (node 0: the last committed token; parents before their
    children).  Child x of a node is taken when uniforms[b, child] * draft[b, node, x] < r[x] (draft
    None: deterministic drafts, 1), r being softmax(logits / temperature) less what the children
    turned down before it took; the last token is argmax r * race.  temperature 0: argmaxes.
    Returns (count [batch], path [batch, nodes], said [batch, nodes], logs [batch, nodes]): nodes
    taken, which, the tokens with the last one behind them (-1 elsewhere), their log-probabilities."""
    import torch
    device = _device(logits, "logits")
    _need(logits, "logits", _ROW_TAGS, device)
    if logits.dim() != 3:
        raise ValueError("logits is [batch, nodes, vocab]")
    batch, nodes, vocab = logits.shape
    for name, t, dtype in (("tokens", tokens, torch.int32), ("parents", parents, torch.int32),
                           ("uniforms", uniforms, torch.float32)):
        if t is None:
            continue
        _need(t, name, (dtype,), device)
        if t.shape != (batch, nodes) or not t.is_contiguous():
            raise ValueError(f"{name} is a contiguous [batch, nodes]")
    dl = dn = rl = rn = None
    if draft is not None:
        _need(draft, "draft", (torch.float32,), device)
        dl, dn, _ = _described(*_form(draft))
    if race is not None:
        _need(race, "race", (torch.float32,), device)
        rl, rn, _ = _described(*_form(race))
    ints = torch.empty(batch * (2 * nodes + 1), dtype=torch.int32, device=device)
    count, path, said = ints[:batch], ints[batch:batch + batch * nodes], ints[batch + batch * nodes:]
    logs = torch.empty((batch, nodes), dtype=torch.float32, device=device)
    _used_on(stream, ints, logs)
    ll, ln, _ = _described(*_form(logits))
    _check(_lib().t4a_verify_drafts(
        _stream(stream), _ROW_TAGS[logits.dtype], logits.data_ptr(), ll, ln, tokens.data_ptr(), parents.data_ptr(),
        None if uniforms is None else uniforms.data_ptr(), None if draft is None else draft.data_ptr(), dl, dn or 0,
        None if race is None else race.data_ptr(), rl, rn or 0, temperature, count.data_ptr(), path.data_ptr(),
        said.data_ptr(), logs.data_ptr()), "verify_drafts")
    return count, path.view(batch, nodes), said.view(batch, nodes), logs
