"""Paged-cache operators over torch tensors (include/t4a_b200/cache.h): rows written into
a cache of pages (quantised where it holds 8-bit codes) and read back, attention of a
tree of drafted tokens over it, and the verification of the drafts.

Tensors are row-major views of the C layouts: a cache side is [pages, page_size, heads,
dim] (float16, bfloat16, int8 or float8_e4m3fn; any strides but 1 along dim), its scales
[pages, page_size, heads] float32.  The library checks layouts and refuses with a
T4AError; a wrong dtype is a TypeError, a tensor on another device or of another rank a
ValueError.  Calls run on the current stream, or on `stream`, whose allocations results
and workspace then are; inputs may be freed while that stream still reads them, but what
wrote them has to be waited for (stream.wait_stream).  The functions are native
(binding/cache_torch.cpp): a small call is a few microseconds on the host.  They serve
decoding and have no backward pass: results never require a gradient, whatever the inputs do.
"""
import ctypes
import importlib.machinery
import importlib.util
import os

from .abi import F32, F16, BF16

_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "_cache_torch.so")
_native = None
_ROW_TAGS = {}


def declare(l):
    """Signatures of the C entries (called when the library is loaded)."""
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


def native():
    """The loaded lib/_cache_torch.so.  Raises when it has not been built."""
    global _native
    if _native is None:
        import torch
        from . import lib
        lib()
        if not os.path.exists(_PATH):
            raise RuntimeError(f"_cache_torch.so is not built ({_PATH}); run t4a-cuda-kernels_b200/build.py")
        loader = importlib.machinery.ExtensionFileLoader("_cache_torch", _PATH)
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_cache_torch", loader))
        loader.exec_module(module)
        _ROW_TAGS.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
        _native = module
    return _native


def _call(name, stream, *args):
    if stream is None:
        return getattr(_native or native(), name)(*args)
    function = getattr(native(), name)
    import torch
    with torch.cuda.stream(stream):
        got = function(*args)
    for t in args:  # their memory is not given out again before the stream is through with it
        if torch.is_tensor(t):
            t.record_stream(stream)
    return got


def cache_write(key, value, k_cache, v_cache, slots, k_scale=None, v_scale=None, stream=None):
    """Rows key[n], value[n] ([n, heads, dim]; float32, float16 or bfloat16) into the cache at
    slots[n] = page * page_size + place (int32 or int64; outside the cache: dropped).  An 8-bit
    cache takes codes and one scale a row: scale = max|x| / 127 (int8) or / 448 (float8_e4m3fn)."""
    _call("write", stream, key, value, k_cache, v_cache, slots, k_scale, v_scale)


def cache_read(k_cache, v_cache, slots, dtype, k_scale=None, v_scale=None, out=None, stream=None):
    """(key, value) [n, heads, dim] in `dtype` (float32, float16 or bfloat16): the rows at slots[n]
    as the values they stand for; zeros for a slot outside the cache.  `out`: a pair to write to."""
    if _native is None:
        native()
    tag = _ROW_TAGS.get(dtype)
    if tag is None:
        raise TypeError(f"cache_read: {dtype} is not supported")
    key, value = (None, None) if out is None else out
    got = _call("read", stream, k_cache, v_cache, slots, tag, k_scale, v_scale, key, value)
    return got if out is None else tuple(out)


def tree_attention_workspace_bytes(q, k_cache, v_cache, page_table, k_scale=None, v_scale=None):
    """Bytes of workspace that tree_attention needs for these tensors' shapes."""
    return native().attention_bytes(q, k_cache, v_cache, page_table, k_scale, v_scale)


def tree_attention(q, k_cache, v_cache, page_table, context, mask=None, nodes=None, k_scale=None, v_scale=None,
                   scale=None, out=None, lse=None, workspace=None, stream=None):
    """Attention of drafted nodes q ([batch, nodes, query heads, dim], float16 or bfloat16) to each
    sequence's context[b] committed tokens and to the nodes that they see; node j lies at place
    context[b] + j of the pages page_table[b] (int32).  mask [batch, nodes, nodes] (bool or uint8):
    whether node i sees node j; None: a chain, j <= i.  nodes [batch] (int32): live nodes.
    scale: dim ** -0.5 unless given.  One node is the decoding step of a single token.
    Returns (out like q, lse [batch, nodes, query heads] float32); a node that sees nothing gets
    zeros and -infinity."""
    got = _call("attention", stream, q, k_cache, v_cache, page_table, context, mask, nodes, k_scale, v_scale, scale, out,
                lse, workspace)
    return (got[0] if out is None else out), (got[1] if lse is None else lse)


def verify_drafts(logits, tokens, parents, uniforms=None, draft=None, race=None, temperature=1.0, stream=None):
    """Walks each sequence's tree of drafted tokens: logits [batch, nodes, vocab] after each node,
    tokens and parents [batch, nodes] int32 (node 0: the last committed token; parents before their
    children).  Child x of a node is taken when uniforms[b, child] * draft[b, node, x] < r[x] (draft
    None: deterministic drafts, 1), r being softmax(logits / temperature) less what the children
    turned down before it took; the last token is argmax r * race.  temperature 0: argmaxes.
    With `draft` a node's children are independent draws from it, so siblings may be alike; children
    drawn without replacement, or picked as the likeliest, need draft=None for what is said to follow
    the target.
    Returns (count [batch], path [batch, nodes], said [batch, nodes], logs [batch, nodes]): nodes
    taken, which, the tokens with the last one behind them (-1 elsewhere), their log-probabilities."""
    return _call("verify", stream, logits, tokens, parents, uniforms, draft, race, temperature)
