"""ctypes binding of include/amem_kv.h: append to a paged key/value cache, and attention over it.

Tensors are whatever has `data_ptr()`, `shape`, `stride()`, `dtype` and `device` (torch's do); nothing here
imports their library. A program that uses torch imports it before this package loads its own library: the
process then has one HIP runtime, torch's.

    cache = kv.Cache(k, v)                      # [pages, heads, slots, dim]; 8 bits: also the two tensors of scales
    batch = kv.Batch(page_table, context, tokens=n, max_tokens=1, max_context=limit)
    kv.append(cache, batch, new_k, new_v, q, q, rotation=kv.Rotation(cos, sin), stream=stream)
    kv.attention(cache, batch, q, out, workspace=workspace, stream=stream)

A `Cache`, `Batch` or `Rotation` describes tensors (addresses, sizes, strides) and keeps them alive; what the tensors
hold may change between calls. `stream` is a hipStream_t as a number, `torch.cuda.current_stream().cuda_stream`
for instance. Arguments that do not fit raise ValueError before anything is enqueued; what the library refuses
raises KvError.
"""
import ctypes as C
import operator
import struct

from . import binding

BF16, F16, E4M3 = range(3)
MAX_AXES = 4
_TYPES = {"torch.bfloat16": BF16, "torch.float16": F16, "torch.float8_e4m3fn": E4M3, "torch.float32": -2, "torch.int32": -3}
_kinds = {}     # by the dtypes themselves, as they are met


def _kind(t):
    kind = _kinds.get(t.dtype)
    if kind is None:
        kind = _kinds[t.dtype] = _TYPES.get(str(t.dtype), -1)
    return kind



class KvError(RuntimeError):
    def __init__(self, what, code):
        super().__init__("%s failed: %d (refused arguments, or tracked memory while paused, if 1; the library's log says why)" % (what, code))
        self.code = code


class CacheInfo(C.Structure):
    _fields_ = [(n, C.c_uint64) for n in ("k", "v", "k_scale", "v_scale")] + [
        (n, C.c_int64) for n in ("page_stride", "head_stride", "slot_stride", "scale_page_stride", "scale_head_stride")] + [
        (n, C.c_int32) for n in ("type", "device", "pages", "kv_heads", "page_slots", "block_slots", "head_dim", "reserved")]


class BatchInfo(C.Structure):
    _fields_ = [(n, C.c_uint64) for n in ("page_table", "context", "cu_tokens")] + [("table_stride", C.c_int64)] + [
        (n, C.c_int32) for n in ("sequences", "table_pages", "tokens", "max_tokens", "max_context", "reserved")]


class AppendArgs(C.Structure):
    _fields_ = [(n, C.c_uint64) for n in ("k", "v", "q", "q_out", "cos", "sin", "positions")] + [
        (n, C.c_int64) for n in ("k_token_stride", "k_head_stride", "v_token_stride", "v_head_stride", "q_token_stride",
                                 "q_head_stride", "q_out_token_stride", "q_out_head_stride", "positions_stride")] + [
        (n, C.c_int32) for n in ("type", "q_heads", "rotary_dim", "interleaved", "table_rows", "axes")] + [
        ("sections", C.c_int32 * MAX_AXES)]


class AttentionArgs(C.Structure):
    _fields_ = [(n, C.c_uint64) for n in ("q", "out", "lse", "workspace", "workspace_bytes")] + [
        (n, C.c_int64) for n in ("q_token_stride", "q_head_stride", "out_token_stride", "out_head_stride")] + [
        ("scale", C.c_float)] + [(n, C.c_int32) for n in ("type", "q_heads", "causal", "window", "reserved")]


# The two records of a call's arguments as bytes: a quarter of what filling the structures takes.
_append_args = struct.Struct("=7Q9q10i").pack
_attention_args = struct.Struct("=5Q4qf5i").pack

# the records by address: a structure's byref, or bytes
_SIGNATURES = {
    "amem_kv_append": (C.c_int, [C.c_void_p] * 4),
    "amem_kv_attention": (C.c_int, [C.c_void_p] * 4),
    "amem_kv_attention_workspace": (C.c_int, [C.POINTER(CacheInfo), C.POINTER(BatchInfo), C.c_int, C.POINTER(C.c_uint64)]),
}
_entry = {}


def kv_abi_names():
    return sorted(_SIGNATURES)


def load():
    """The library, with the entry points of include/amem_kv.h declared."""
    lib = binding.load()
    if not _entry:
        found = {}
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
            found[name] = fn
        _entry.update(found)     # all at once: another thread may be about to call
    return lib


def _call(name, *args):
    if not _entry:
        load()
    code = _entry[name](*args)
    if code:
        raise KvError(name, code)


def _unfit(e):
    return ValueError("an argument is no number of its type: %s" % e)


def _need(ok, why):
    if not ok:
        raise ValueError(why)


def _device(t):
    _need(t.device.type == "cuda", "a tensor is not on a GPU")
    return t.device


def _is(t, dtype, device, what):
    if _kind(t) != _TYPES["torch." + dtype]:
        raise ValueError("%s is not %s" % (what, dtype))
    if t.device != device:
        raise ValueError("%s is on another device than the cache" % what)


def _int32(**numbers):
    """The numbers as they are, which ctypes would cut to 32 bits without a word."""
    out = []
    for what, x in numbers.items():
        try:
            x = operator.index(x)
        except TypeError:
            raise ValueError("%s is no whole number" % what) from None
        _need(-1 << 31 <= x < 1 << 31, "%s does not fit 32 bits" % what)
        out.append(x)
    return out


class Cache:
    """Keys and values [pages, heads, slots, dim], with equal strides and contiguous dims; e4m3 with their scales, float32
    [pages, heads, blocks], blocks contiguous."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        _need(len(k.shape) == 4 and tuple(k.shape) == tuple(v.shape) and k.stride() == v.stride() and k.dtype == v.dtype,
              "k and v differ, or are not [pages, heads, slots, dim]")
        kind, block = _kind(k), 0
        _need(kind >= 0, "k is not bfloat16, float16 or float8_e4m3fn")
        pages, heads, slots, dim = k.shape
        _int32(pages=pages, heads=heads, slots=slots, dim=dim)
        at = k.stride()
        _need(at[3] == 1 or dim == 1, "the dims of k are not contiguous")
        device = _device(k)
        _need(_device(v) == device, "k and v are on different devices")
        _need((kind == E4M3) == (k_scale is not None) == (v_scale is not None), "8 bits have scales, 16 have none")
        info = CacheInfo(k.data_ptr(), v.data_ptr(), 0, 0, at[0], at[1], at[2], 0, 0, kind, device.index or 0, pages, heads, slots, 0, dim, 0)
        if kind == E4M3:
            for t in (k_scale, v_scale):
                _is(t, "float32", device, "a tensor of scales")
            shape = tuple(k_scale.shape)
            _need(shape == tuple(v_scale.shape) and k_scale.stride() == v_scale.stride() and len(shape) == 3 and shape[:2] == (pages, heads)
                  and shape[2] > 0 and slots % shape[2] == 0 and (k_scale.stride()[2] == 1 or shape[2] == 1),
                  "the scales are not [pages, heads, blocks] with contiguous blocks")
            block = slots // shape[2]
            info.k_scale, info.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
            info.scale_page_stride, info.scale_head_stride = k_scale.stride()[:2]
            info.block_slots = block
        self.info, self.device, self.dim, self.heads, self.kind = info, device, dim, heads, kind
        self._keep = (k, v, k_scale, v_scale)
        self._ref = C.byref(info)


class Batch:
    """The sequences of a call: page_table int32 [sequences, pages] (rows may be strided), context int32 [sequences] (tokens
    in the cache, the new ones included), cu_tokens int32 [sequences + 1] or None where all have max_tokens rows,
    tokens: rows of the token tensors; max_context: no context is above it (None: what the table's pages hold, for which
    give page_slots)."""

    def __init__(self, page_table, context, tokens, cu_tokens=None, max_tokens=None, max_context=None, page_slots=None):
        device = _device(context)
        _need(len(context.shape) == 1, "context is not [sequences]")
        n = context.shape[0]
        for t, what in ((page_table, "page_table"), (context, "context"), (cu_tokens, "cu_tokens")):
            if t is not None:
                _is(t, "int32", device, what)
        _need(len(page_table.shape) == 2 and page_table.shape[0] == n and (page_table.stride()[1] == 1 or page_table.shape[1] < 2),
              "page_table is not [sequences, pages] with contiguous pages")
        _need(n < 2 or context.stride()[0] == 1, "context is not contiguous")
        if cu_tokens is not None:
            _need(tuple(cu_tokens.shape) == (n + 1,) and cu_tokens.stride()[0] == 1, "cu_tokens is not [sequences + 1]")
            max_tokens = tokens if max_tokens is None else max_tokens
        else:
            max_tokens = (tokens // n if n else 0) if max_tokens is None else max_tokens
        if max_context is None:
            _need(page_slots, "max_context or page_slots is needed")
            max_context = page_table.shape[1] * page_slots
        pages = page_table.shape[1]
        n, pages, tokens, max_tokens, max_context = _int32(sequences=n, pages=pages, tokens=tokens, max_tokens=max_tokens, max_context=max_context)
        stride = page_table.stride()[0] if n > 1 else pages
        _need(stride >= pages, "the rows of page_table overlap")
        self.info = BatchInfo(page_table.data_ptr(), context.data_ptr(), cu_tokens.data_ptr() if cu_tokens is not None else 0,
                              stride, n, pages, tokens, max_tokens, max_context, 0)
        self.device, self.tokens = device, tokens
        self._keep = (page_table, context, cu_tokens)
        self._ref = C.byref(self.info)


class Rotation:
    """Tables float32 [rows, pairs]; sections: how many pairs each axis has (None: one axis); interleaved: pairs are
    (2i, 2i + 1) and not (i, i + pairs)."""

    def __init__(self, cos, sin, sections=None, interleaved=False):
        self.device = _device(cos)
        for t in (cos, sin):
            _is(t, "float32", self.device, "a table of the rotation")
            _need(len(t.shape) == 2 and tuple(t.shape) == tuple(cos.shape) and t.stride() == (t.shape[1], 1), "the tables are not [rows, pairs] and contiguous")
        sections = tuple(sections) if sections else (cos.shape[1],)
        _need(len(sections) <= MAX_AXES and sum(sections) == cos.shape[1] and min(sections) >= 0, "sections are not the pairs of the axes")
        # as append() hands them over: addresses, rotary_dim, interleaved, rows, axes, sections
        self.packed = (cos.data_ptr(), sin.data_ptr(), 2 * cos.shape[1], int(interleaved), cos.shape[0], len(sections),
                       sections + (0,) * (MAX_AXES - len(sections)))
        self._keep = (cos, sin)


def _refuse_rows(shape, dtype, device, **tensors):
    """Says what is wrong with one of the tensors, which are to be `shape` with contiguous dims."""
    for what, t in tensors.items():
        _need(t.shape == shape and t.stride()[2] == 1, "%s is not [%d, %d, %d] with contiguous dims" % ((what,) + shape))
        _need(t.dtype == dtype, "%s has another type than the other rows" % what)
        _need(t.device == device, "%s is on another device than the cache" % what)


def _heads(q):
    shape = q.shape
    if len(shape) != 3:
        raise ValueError("q is not [tokens, heads, dim]")
    return shape[1]


def append(cache, batch, k, v, q=None, q_out=None, rotation=None, positions=None, stream=0):
    """Rows k and v [tokens, heads, dim] into the cache, k rotated; q rotated into q_out."""
    n, device, dtype = batch.tokens, cache.device, k.dtype
    kind = _kinds.get(dtype)
    if kind is None:
        kind = _kind(k)
    if kind != BF16 and kind != F16:
        raise ValueError("k is not bfloat16 or float16")
    if batch.device != device:
        raise ValueError("the batch is on another device than the cache")
    shape, k_at, v_at = (n, cache.heads, cache.dim), k.stride(), v.stride()
    if (k.shape != shape or v.shape != shape or k_at[2] != 1 or v_at[2] != 1 or v.dtype != dtype or k.device != device
            or v.device != device):
        _refuse_rows(shape, dtype, device, k=k, v=v)
    q_ptr = out_ptr = q_heads = 0
    q_at = out_at = (0, 0)
    if q is not None:
        if q_out is None:
            raise ValueError("q without q_out")
        q_heads = _heads(q)
        shape, q_at, out_at = (n, q_heads, cache.dim), q.stride(), q_out.stride()
        if (q.shape != shape or q_out.shape != shape or q_at[2] != 1 or out_at[2] != 1 or q.dtype != dtype or q_out.dtype != dtype
                or q.device != device or q_out.device != device):
            _refuse_rows(shape, dtype, device, q=q, q_out=q_out)
        q_ptr, out_ptr = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    cos = sin = where = apart = dim = interleaved = rows = axes = 0
    sections = (0, 0, 0, 0)
    if rotation is not None:
        if rotation.device != device:
            raise ValueError("the rotation is on another device than the cache")
        cos, sin, dim, interleaved, rows, axes, sections = rotation.packed
        if positions is not None:
            _is(positions, "int32", device, "positions")
            shape, at = tuple(positions.shape), positions.stride()
            _need(shape == (axes, n) or (axes == 1 and shape == (n,)), "positions are not [axes, tokens]")
            _need(n < 2 or at[-1] == 1, "positions are not contiguous")
            where, apart = positions.data_ptr(), at[0] if axes > 1 else n
        elif axes > 1:
            raise ValueError("several axes need positions")
    elif positions is not None:
        raise ValueError("positions without rotation")
    try:
        a = _append_args(k.data_ptr(), v.data_ptr(), q_ptr, out_ptr, cos, sin, where, k_at[0], k_at[1], v_at[0], v_at[1], q_at[0], q_at[1],
                         out_at[0], out_at[1], apart, kind, q_heads, dim, interleaved, rows, axes, *sections)
    except (struct.error, OverflowError) as e:
        raise _unfit(e) from None
    _call("amem_kv_append", cache._ref, batch._ref, a, stream)


def attention_workspace(cache, batch, q_heads):
    """Bytes of workspace that `attention` needs for these sizes."""
    n = C.c_uint64()
    _call("amem_kv_attention_workspace", cache._ref, batch._ref, *_int32(q_heads=q_heads), C.byref(n))
    return n.value


def attention(cache, batch, q, out, lse=None, scale=None, causal=True, window=0, workspace=None, stream=0):
    """out [tokens, heads, dim] = attention of q over the cache; lse float32 [tokens, heads]; scale: dim ** -0.5 if None;
    workspace: a contiguous tensor of at least attention_workspace() bytes."""
    n, dim, device, dtype, heads = batch.tokens, cache.dim, cache.device, q.dtype, _heads(q)
    kind = _kinds.get(dtype)
    if kind is None:
        kind = _kind(q)
    if kind != BF16 and kind != F16:
        raise ValueError("q is not bfloat16 or float16")
    if batch.device != device:
        raise ValueError("the batch is on another device than the cache")
    shape, q_at, out_at = (n, heads, dim), q.stride(), out.stride()
    if (q.shape != shape or out.shape != shape or q_at[2] != 1 or out_at[2] != 1 or out.dtype != dtype or q.device != device
            or out.device != device):
        _refuse_rows(shape, dtype, device, q=q, out=out)
    lse_ptr = at = size = 0
    if lse is not None:
        _is(lse, "float32", device, "lse")
        if lse.shape != (n, heads) or not lse.is_contiguous():
            raise ValueError("lse is not [tokens, heads] and contiguous")
        lse_ptr = lse.data_ptr()
    if workspace is not None:
        if workspace.device != device or not workspace.is_contiguous():
            raise ValueError("workspace is on another device, or strided")
        at, size = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    try:
        a = _attention_args(q.data_ptr(), out.data_ptr(), lse_ptr, at, size, q_at[0], q_at[1], out_at[0], out_at[1],
                            dim ** -0.5 if scale is None else scale, kind, heads, 1 if causal else 0, window, 0)
    except (struct.error, OverflowError) as e:
        raise _unfit(e) from None
    _call("amem_kv_attention", cache._ref, batch._ref, a, stream)
