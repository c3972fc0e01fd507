"""Paged serving operators on torch CUDA tensors: rotary positions, attention over
packed prompts, attention of drafted token trees over a paged cache, the cache's
page operations, and the host's book of pages.

Each call checks its tensors, passes their addresses to the C ABI
(include/promptboot_b200.h has the definitions) on the tensors' device and its
current torch stream, and returns at once.  Index tensors are contiguous int32
(or uint32); -1 stands for no position, slot, page or kept node, and is not an offset
or a context length.  Head tensors are [rows, heads, head_dim] of
float32, float16 or bfloat16 with a contiguous last dimension, any other strides a
multiple of 16 bytes, so that views of a stacked q/k/v projection serve as they
are.  An output shares no memory with an input unless its call says that it may.  Refused arguments raise OperatorError.  There are no gradients: a tensor that
asks for one, one of a cache too, is refused unless grad mode is off, and one that
carries a forward-mode tangent always.
"""
from __future__ import annotations

import ctypes
import functools

import torch
import torch.autograd.forward_ad as _forward

from . import _lib
from .api import DeviceError

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_I32, _U32, _I64, _U64 = torch.int32, torch.uint32, torch.int64, torch.uint64
_LAYOUTS = {False: 0, True: 1}
_SCALINGS = {"none": 0, "linear": 1, "bands": 2, "yarn": 3}
_ref = ctypes.byref
_Rows = _lib.PbRows
_empty_like = torch.empty_like
# Tells autograd of tensors that a kernel has written: a backward pass that saved one
# then raises an error instead of reading what is no longer there.
_written = torch.autograd.graph.increment_version


class OperatorError(ValueError):
    """Arguments that an operator refuses; `status` is the C ABI's."""

    def __init__(self, text: str, status: int = 4):
        self.status = status
        super().__init__(text)


def _u32(x, name):
    """x as the C ABI takes it, which would cut a larger number to 32 bits."""
    if not 0 <= x < 1 << 32:
        raise OperatorError(f"{name} is out of range")
    return x


class _Handle(ctypes.c_void_p):
    """A handle of the C ABI, destroyed with its last holder: copies of an object share it.
    It is not copied itself, so its object cannot be pickled or copied deeply."""

    def __init__(self, destroy):
        super().__init__()
        self._destroy = destroy

    def __reduce_ex__(self, protocol):
        raise TypeError("handles of the C ABI cannot be pickled or copied")

    def __del__(self):
        try:
            if self.value:
                getattr(_lib.load(), self._destroy)(self)
                self.value = None
        except Exception:
            pass


def _check(status: int):
    if status == 0:
        return
    text = _lib.last_error()
    if status == 100:
        raise DeviceError(text)
    raise OperatorError(text, status)


# A decode step makes these calls once per layer, so what they do per tensor is kept
# to a handful of attribute reads: a device is compared by its number, a stream is
# taken as its handle.
if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    def _stream(device: int) -> int:
        return torch._C._cuda_getCurrentRawStream(device)
else:
    def _stream(device: int) -> int:
        return torch.cuda.current_stream(device).cuda_stream


def _call(device: int, fn, *args):
    """fn(*args, the device's current stream) with the device current."""
    if device == torch.cuda.current_device():
        status = fn(*args, _stream(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _stream(device))
    if status:
        _check(status)


def _heads(t, dtype, device, name):
    """[rows, heads, head_dim] of a type and device, as the C ABI takes it."""
    s = t.stride()
    if len(s) != 3 or s[2] != 1:
        raise OperatorError(f"{name} must be [rows, heads, head_dim] with a contiguous last dimension")
    if t.dtype is not dtype or t.get_device() != device:
        raise OperatorError(f"{name} has another type or device")
    if t.requires_grad and torch.is_grad_enabled() or _forward._current_level >= 0 and _tangent(t):
        raise OperatorError(f"{name} asks for a gradient, which the serving operators do not have")
    return _Rows(t.data_ptr(), s[0], s[1])


def _tangent(t):
    """Whether t carries a tangent of the forward mode.  Callers look first whether a
    level of it is open (_current_level), without which there are none."""
    return _forward.unpack_dual(t).tangent is not None


def _no_gradient(cache):
    """Refuses a cache whose tensors ask for a gradient (they may since it was made)."""
    if (cache.k.requires_grad or cache.v.requires_grad) and torch.is_grad_enabled() \
            or _forward._current_level >= 0 and (_tangent(cache.k) or _tangent(cache.v)):
        raise OperatorError("the cache asks for a gradient, which the serving operators do not have")


def _first(t, name):
    """(type, device) of the tensor that sets them for the others."""
    dtype, device = t.dtype, t.get_device()
    if dtype not in _TYPES or device < 0:
        raise OperatorError(f"{name} must be a float32, float16 or bfloat16 CUDA tensor")
    return dtype, device


def _index(t, shape, device, name, signed=_I32, unsigned=_U32):
    if (t.dtype is not signed and t.dtype is not unsigned) or t.get_device() != device or t.shape != shape \
            or not t.is_contiguous():
        raise OperatorError(f"{name} must be a contiguous {signed} tensor {list(shape)} on cuda:{device}")
    return t.data_ptr()


class PageCache:
    """A paged cache over two tensors [layers, pages, kv_heads, page_size, head_dim]
    whose layers are contiguous; it holds the tensors, not a copy."""

    def __init__(self, k, v):
        shape, strides = k.shape, k.stride()
        if len(shape) != 5 or v.shape != shape or v.stride() != strides or v.dtype is not k.dtype \
                or v.get_device() != k.get_device():
            raise OperatorError("k and v must be alike: [layers, pages, kv_heads, page_size, head_dim]")
        self.dtype, self.device = _first(k, "a cache")
        layers, pages, heads, size, dim = shape
        if strides[4] != 1 or strides[3] != dim or strides[2] != size * dim or strides[1] != heads * size * dim:
            raise OperatorError("each layer of a cache must be contiguous")
        self.k, self.v = k, v
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, size, dim
        self._c = _lib.PbCache(k.data_ptr(), v.data_ptr(), strides[0], _TYPES[self.dtype], layers,
                               pages, size, heads, dim)

    @classmethod
    def empty(cls, layers, pages, kv_heads, page_size, head_dim, dtype=torch.bfloat16, device="cuda"):
        """A cache of new, unset memory."""
        shape = (layers, pages, kv_heads, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device),
                   torch.empty(shape, dtype=dtype, device=device))

    def copy_pages(self, pairs):
        """Copies page pairs[i, 0] to page pairs[i, 1] in every layer.  A page may be the
        source of several pairs, but the target of one only, and not a source then."""
        _no_gradient(self)
        n = pairs.shape[0]
        at = _index(pairs, (n, 2), self.device, "pairs")
        _call(self.device, _lib.load().pb_cache_copy_pages_device, _ref(self._c), n, at)
        _written((self.k, self.v))

    def keep(self, tables, contexts, counts, nodes):
        """Moves the accepted nodes of each sequence's draft tree behind its
        context, in every layer: position contexts[s] + nodes[s, i] to contexts[s]
        + i for i < counts[s] (-1: none).  The nodes ascend; an entry that does not is
        left out.  tables [seqs, width] as in tree_attention; pages that are written
        must belong to one sequence each."""
        _no_gradient(self)
        device, seqs = self.device, contexts.shape[0]
        width, most = tables.shape[-1], nodes.shape[-1]
        a = _index(tables, (seqs, width), device, "tables")
        b = _index(contexts, (seqs,), device, "contexts")
        c = _index(counts, (seqs,), device, "counts")
        d = _index(nodes, (seqs, most), device, "nodes")
        _call(device, _lib.load().pb_cache_keep_device, _ref(self._c), seqs, a, width, b, c, d, most)
        _written((self.k, self.v))


class Rotary:
    """Rotary positions of one model: which elements pair up and how far each pair
    turns per position.  scaling "none", "linear", "bands" or "yarn"; see
    pb_rotary_config for the formulas and the meaning of 0."""

    def __init__(self, head_dim, rotary_dim=None, theta=1e6, interleaved=False, scaling="none", factor=1.0,
                 original_context=0, low=0.0, high=0.0, magnitude=0.0):
        if scaling not in _SCALINGS:
            raise OperatorError(f"scaling must be one of {', '.join(_SCALINGS)}")
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        config = _lib.PbRotaryConfig(_u32(head_dim, "head_dim"), _u32(rotary_dim, "rotary_dim"),
                                     _LAYOUTS[bool(interleaved)], _SCALINGS[scaling], theta, factor,
                                     original_context, low, high, magnitude)
        self.head_dim = head_dim
        self._h = _Handle("pb_rotary_destroy")
        _check(_lib.load().pb_rotary_create(_ref(config), _ref(self._h)))

    def apply(self, q, k, positions, q_out=None, k_out=None):
        """(q, k) turned, in new tensors or in q_out and k_out, which may be q and k.  Rows
        at position -1 stay as they were, unset in a new tensor."""
        dtype, device = _first(q, "q")
        q_in, k_in = _heads(q, dtype, device, "q"), _heads(k, dtype, device, "k")
        rows, heads, dim = q.shape
        k_rows, k_heads, k_dim = k.shape
        if dim != self.head_dim or k_dim != dim or k_rows != rows:
            raise OperatorError("q and k must have the same rows and the plan's head_dim")
        at = _index(positions, (rows,), device, "positions")
        q_out = _empty_like(q) if q_out is None else q_out
        k_out = _empty_like(k) if k_out is None else k_out
        q_to, k_to = _heads(q_out, dtype, device, "q_out"), _heads(k_out, dtype, device, "k_out")
        if q_out.shape != q.shape or k_out.shape != k.shape:
            raise OperatorError("q_out and k_out must have the shapes of q and k")
        if rows:
            _call(device, _lib.load().pb_rotary_device, self._h, _TYPES[dtype], rows, at, heads, _ref(q_in), _ref(q_to),
                  k_heads, _ref(k_in), _ref(k_to))
            _written((q_out, k_out))
        return q_out, k_out

    def apply_to_cache(self, q, k, v, positions, cache, slots, layer=0, q_out=None):
        """q turned, as apply; k turned and v go to `layer` of the cache at
        slots[row] = page * page_size + slot in the page (-1: nowhere).  Of rows with
        the same slot it holds a mix."""
        _no_gradient(cache)
        dtype, device = cache.dtype, cache.device
        q_in, k_in, v_in = (_heads(q, dtype, device, "q"), _heads(k, dtype, device, "k"),
                            _heads(v, dtype, device, "v"))
        rows, heads, dim = q.shape
        if dim != self.head_dim:
            raise OperatorError("q must have the plan's head_dim")
        if k.shape != (rows, cache.kv_heads, dim) or v.shape != k.shape:
            raise OperatorError("k and v must be [rows, the cache's heads, head_dim]")
        a = _index(positions, (rows,), device, "positions")
        b = _index(slots, (rows,), device, "slots")
        q_out = _empty_like(q) if q_out is None else q_out
        q_to = _heads(q_out, dtype, device, "q_out")
        if q_out.shape != q.shape:
            raise OperatorError("q_out must have the shape of q")
        if rows:
            _call(device, _lib.load().pb_rotary_cache_device, self._h, rows, a, heads, _ref(q_in), _ref(q_to),
                  _ref(k_in), _ref(v_in), _ref(cache._c), _u32(layer, "layer"), b)
            _written((q_out, cache.k, cache.v))
        return q_out


def prompt_attention(q, k, v, offsets, kv_offsets=None, scale=None, out=None):
    """Causal attention of packed prompts: sequence s has the rows offsets[s] to
    offsets[s + 1] of q and kv_offsets[s] to kv_offsets[s + 1] (default: the same)
    of k and v, aligned at their ends.  scale defaults to head_dim ** -0.5.  Rows
    behind offsets[-1] are left as they were (unset in a new tensor)."""
    dtype, device = _first(q, "q")
    q_in, k_in, v_in = _heads(q, dtype, device, "q"), _heads(k, dtype, device, "k"), _heads(v, dtype, device, "v")
    rows, heads, dim = q.shape
    k_rows, k_heads, k_dim = k.shape
    if k_dim != dim or v.shape != k.shape:
        raise OperatorError("k and v must have one shape and q's head_dim")
    n = offsets.shape[0]
    a = _index(offsets, (n,), device, "offsets")
    b = None if kv_offsets is None else _index(kv_offsets, (n,), device, "kv_offsets")
    out = _empty_like(q) if out is None else out
    to = _heads(out, dtype, device, "out")
    if out.shape != q.shape:
        raise OperatorError("out must have the shape of q")
    _call(device, _lib.load().pb_prompt_attention_device, _TYPES[dtype], dim, heads, k_heads, n - 1, rows, k_rows,
          _ref(q_in), _ref(k_in), _ref(v_in), _ref(to), a, b, dim ** -0.5 if scale is None else scale)
    _written(out)
    return out


@functools.lru_cache(maxsize=256)
def _workspace_bytes(device, type_, dim, heads, kv_heads, seqs, rows):
    with torch.cuda.device(device):
        got = int(_lib.load().pb_tree_attention_workspace(type_, dim, heads, kv_heads, seqs, rows))
    if not got:
        raise OperatorError(_lib.last_error())  # (which is not cached)
    return got


def tree_workspace_bytes(cache, heads, seqs, rows):
    """Bytes of workspace that tree_attention needs for these sizes."""
    return _workspace_bytes(cache.device, _TYPES[cache.dtype], cache.head_dim, _u32(heads, "heads"), cache.kv_heads,
                            _u32(seqs, "seqs"), _u32(rows, "rows"))


def tree_attention(q, cache, tables, contexts, offsets, visible, layer=0, scale=None, out=None, workspace=None):
    """Attention of drafted nodes over a paged cache: the rows offsets[s] to
    offsets[s + 1] of q are sequence s's nodes, whose keys and values stand at
    position contexts[s] + node; a row sees the contexts[s] positions before them
    and node j where bit j of visible[row] (int64) is set.  Position p is in page
    tables[s, p // page_size].  One node with visible 1 is plain decode.
    `workspace`: a uint8 tensor of tree_workspace_bytes, for calls that never
    overlap; by default one from torch's allocator."""
    _no_gradient(cache)
    dtype, device = cache.dtype, cache.device
    q_in = _heads(q, dtype, device, "q")
    rows, heads, dim = q.shape
    if dim != cache.head_dim:
        raise OperatorError("q must have the cache's head_dim")
    seqs, width = contexts.shape[0], tables.shape[-1]
    a = _index(tables, (seqs, width), device, "tables")
    b = _index(contexts, (seqs,), device, "contexts")
    c = _index(offsets, (seqs + 1,), device, "offsets")
    d = _index(visible, (rows,), device, "visible", _I64, _U64)
    out = _empty_like(q) if out is None else out
    to = _heads(out, dtype, device, "out")
    if out.shape != q.shape:
        raise OperatorError("out must have the shape of q")
    if not rows:
        return out
    if workspace is None:
        need = _workspace_bytes(device, _TYPES[dtype], dim, heads, cache.kv_heads, seqs, rows)
        workspace = torch.empty(need, dtype=torch.uint8, device=cache.k.device)
    elif workspace.dtype is not torch.uint8 or workspace.get_device() != device or not workspace.is_contiguous():
        raise OperatorError("workspace must be a contiguous uint8 tensor on q's device")
    _call(device, _lib.load().pb_tree_attention_device, _ref(cache._c), _u32(layer, "layer"), heads, seqs, rows,
          _ref(q_in), _ref(to), a, width, b, c, d, dim ** -0.5 if scale is None else scale,
          workspace.data_ptr(), workspace.numel())
    _written(out)
    return out


def attention_status(device=None):
    """Waits for the device's current stream and raises DeviceError where an attention on
    that device, on any stream, gave up waiting since this thread last asked (the outputs
    of that attention are not complete)."""
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise OperatorError(f"attention_status: {device} is not a CUDA device")
    _call(torch.cuda.current_device() if device.index is None else device.index, _lib.load().pb_attention_status)


class PagePool:
    """The host's book of a cache's pages: which pages each sequence holds, shared
    between forks until one of them writes.  One thread at a time."""

    def __init__(self, pages, page_size, max_seqs):
        self._h = _Handle("pb_pool_destroy")
        _check(_lib.load().pb_pool_create(_u32(pages, "pages"), _u32(page_size, "page_size"),
                                          _u32(max_seqs, "max_seqs"), _ref(self._h)))
        self.pages, self.page_size = pages, page_size

    def open(self):
        """A new sequence without tokens."""
        seq = ctypes.c_uint32()
        _check(_lib.load().pb_pool_open(self._h, _ref(seq)))
        return seq.value

    def fork(self, seq):
        """A new sequence that shares every page of `seq`."""
        child = ctypes.c_uint32()
        _check(_lib.load().pb_pool_fork(self._h, _u32(seq, "seq"), _ref(child)))
        return child.value

    def extend(self, seq, tokens):
        """Room for `tokens` more; None, or the (from, to) pair of pages that
        PageCache.copy_pages has to copy before anything is written."""
        pair, needed = (ctypes.c_uint32 * 2)(), ctypes.c_uint32()
        _check(_lib.load().pb_pool_extend(self._h, _u32(seq, "seq"), _u32(tokens, "tokens"), pair, _ref(needed)))
        return None if pair[0] == 0xFFFFFFFF else (pair[0], pair[1])

    def truncate(self, seq, length):
        """Cuts a sequence to `length` tokens and frees the pages behind them."""
        _check(_lib.load().pb_pool_truncate(self._h, _u32(seq, "seq"), _u32(length, "length")))

    def free(self, seq):
        _check(_lib.load().pb_pool_free(self._h, _u32(seq, "seq")))

    def compact(self):
        """Moves the pages in use to the lowest ids: ([(from, to), ...] for
        PageCache.copy_pages, pages in use)."""
        pairs = (ctypes.c_uint32 * (2 * self.pages))()
        n, used, needed = ctypes.c_uint32(), ctypes.c_uint32(), ctypes.c_uint32()
        _check(_lib.load().pb_pool_compact(self._h, pairs, self.pages, _ref(n), _ref(used), _ref(needed)))
        return [(pairs[2 * i], pairs[2 * i + 1]) for i in range(n.value)], used.value

    def pages_of(self, seq):
        """The page ids of a sequence, in order."""
        return self._table(seq)[0]

    def length(self, seq):
        return self._table(seq)[1]

    def free_pages(self):
        return int(_lib.load().pb_pool_free_pages(self._h))

    def tables(self, seqs, device="cuda"):
        """int32 [len(seqs), width] page ids for tree_attention and keep, -1 behind a
        sequence's last page."""
        rows = [self.pages_of(s) for s in seqs]
        width = max([len(r) for r in rows] + [1])
        rows = [r + [-1] * (width - len(r)) for r in rows]
        return torch.tensor(rows, dtype=torch.int32, device=device).view(len(rows), width)

    def slots(self, seq, start, count, device="cuda"):
        """int32 cache slots of `count` positions from `start` on, for Rotary.apply_to_cache."""
        ids, length = self._table(seq)
        if start < 0 or count < 0 or start + count > length:
            raise OperatorError(f"sequence {seq} has {length} tokens")
        size = self.page_size
        return torch.tensor([ids[p // size] * size + p % size for p in range(start, start + count)],
                            dtype=torch.int32, device=device)

    def _table(self, seq):
        length, needed = ctypes.c_uint32(), ctypes.c_uint32()
        lib = _lib.load()
        table = (ctypes.c_uint32 * self.pages)()
        _check(lib.pb_pool_table(self._h, _u32(seq, "seq"), table, self.pages, _ref(length), _ref(needed)))
        return list(table[:needed.value]), length.value
