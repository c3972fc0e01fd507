"""Paged serving operators on torch CUDA tensors: rotary positions, attention over
packed prompts, attention of drafted token trees over a paged cache, the cache's
page operations, and the host's book of pages.

Each call checks its tensors, passes their addresses to the C ABI
(include/promptboot_b200.h has the definitions) on the tensors' device and its
current torch stream, and returns at once.  Index tensors are contiguous int32
(or uint32), -1 standing for none; head tensors are [rows, heads, head_dim] of
float32, float16 or bfloat16 with a contiguous last dimension, any other strides a
multiple of 16 bytes, so that views of a stacked q/k/v projection serve as they
are.  Refused arguments raise OperatorError.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from .api import DeviceError

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_INDEX = (torch.int32, torch.uint32)
_LAYOUTS = {False: 0, True: 1}
_SCALINGS = {"none": 0, "linear": 1, "bands": 2, "yarn": 3}
_ref = ctypes.byref


class OperatorError(ValueError):
    """Arguments that an operator refuses; `status` is the C ABI's."""

    def __init__(self, text: str, status: int = 4):
        self.status = status
        super().__init__(text)


def _check(status: int):
    if status == 0:
        return
    text = _lib.last_error()
    if status == 100:
        raise DeviceError(text)
    raise OperatorError(text, status)


def _heads(t, like, name):
    """[rows, heads, head_dim] of like's type and device, as the C ABI takes it."""
    if t.dim() != 3 or t.stride(2) != 1:
        raise OperatorError(f"{name} must be [rows, heads, head_dim] with a contiguous last dimension")
    if t.dtype != like.dtype or t.device != like.device:
        raise OperatorError(f"{name} has another type or device")
    return _lib.PbRows(t.data_ptr(), t.stride(0), t.stride(1))


def _first(t, name):
    """_heads of the tensor that sets type and device."""
    if t.dtype not in _TYPES or not t.is_cuda:
        raise OperatorError(f"{name} must be a float32, float16 or bfloat16 CUDA tensor")
    return _heads(t, t, name)


def _index(t, shape, device, name, types=_INDEX):
    if t.dtype not in types or t.device != device or not t.is_contiguous() or t.shape != shape:
        raise OperatorError(f"{name} must be a contiguous {types[0]} tensor {list(shape)} on {device}")
    return t.data_ptr()


class _on:
    """The device of a call, made current where it is not, and its current stream."""

    def __init__(self, device):
        self._guard = torch.cuda.device(device) if device.index != torch.cuda.current_device() else None
        self.stream = torch.cuda.current_stream(device).cuda_stream

    def __enter__(self):
        if self._guard is not None:
            self._guard.__enter__()
        return self.stream

    def __exit__(self, *what):
        if self._guard is not None:
            self._guard.__exit__(*what)


class PageCache:
    """A paged cache over two tensors [layers, pages, kv_heads, page_size, head_dim]
    whose layers are contiguous; it holds the tensors, not a copy."""

    def __init__(self, k, v):
        if k.dim() != 5 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.device != v.device:
            raise OperatorError("k and v must be alike: [layers, pages, kv_heads, page_size, head_dim]")
        if k.dtype not in _TYPES or not k.is_cuda:
            raise OperatorError("a cache holds float32, float16 or bfloat16 CUDA tensors")
        layers, pages, heads, size, dim = k.shape
        if k.stride()[1:] != (heads * size * dim, size * dim, dim, 1):
            raise OperatorError("each layer of a cache must be contiguous")
        self.k, self.v = k, v
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, size, dim
        self._c = _lib.PbCache(k.data_ptr(), v.data_ptr(), k.stride(0), _TYPES[k.dtype], layers,
                               pages, size, heads, dim)

    @classmethod
    def empty(cls, layers, pages, kv_heads, page_size, head_dim, dtype=torch.bfloat16, device="cuda"):
        """A cache of new, unset memory."""
        shape = (layers, pages, kv_heads, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device),
                   torch.empty(shape, dtype=dtype, device=device))

    def copy_pages(self, pairs):
        """Copies page pairs[i, 0] to page pairs[i, 1] in every layer."""
        at = _index(pairs, (pairs.shape[0], 2), self.k.device, "pairs")
        with _on(self.k.device) as stream:
            _check(_lib.load().pb_cache_copy_pages_device(_ref(self._c), pairs.shape[0], at, stream))

    def keep(self, tables, contexts, counts, nodes):
        """Moves the accepted nodes of each sequence's draft tree behind its
        context, in every layer: position contexts[s] + nodes[s, i] to contexts[s]
        + i for i < counts[s].  tables [seqs, width] as in tree_attention."""
        device, seqs = self.k.device, contexts.shape[0]
        a = _index(tables, (seqs, tables.shape[-1]), device, "tables")
        b = _index(contexts, (seqs,), device, "contexts")
        c = _index(counts, (seqs,), device, "counts")
        d = _index(nodes, (seqs, nodes.shape[-1]), device, "nodes")
        with _on(device) as stream:
            _check(_lib.load().pb_cache_keep_device(_ref(self._c), seqs, a, tables.shape[1], b, c, d,
                                                    nodes.shape[1], stream))


class Rotary:
    """Rotary positions of one model: which elements pair up and how far each pair
    turns per position.  scaling "none", "linear", "bands" or "yarn"; see
    pb_rotary_config for the formulas and the meaning of 0."""

    def __init__(self, head_dim, rotary_dim=None, theta=1e6, interleaved=False, scaling="none", factor=1.0,
                 original_context=0, low=0.0, high=0.0, magnitude=0.0):
        if scaling not in _SCALINGS:
            raise OperatorError(f"scaling must be one of {', '.join(_SCALINGS)}")
        config = _lib.PbRotaryConfig(head_dim, rotary_dim or head_dim, _LAYOUTS[bool(interleaved)],
                                     _SCALINGS[scaling], theta, factor, original_context, low, high, magnitude)
        self.head_dim = head_dim
        self._h = ctypes.c_void_p()
        _check(_lib.load().pb_rotary_create(_ref(config), _ref(self._h)))

    def __del__(self):
        try:
            if self._h:
                _lib.load().pb_rotary_destroy(self._h)
                self._h = None
        except Exception:
            pass

    def apply(self, q, k, positions, q_out=None, k_out=None):
        """(q, k) turned, in new tensors or in q_out and k_out, which may be q and k."""
        q_in = _first(q, "q")
        k_in = _heads(k, q, "k")
        rows = q.shape[0]
        if q.shape[2] != self.head_dim or k.shape[2] != self.head_dim or k.shape[0] != rows:
            raise OperatorError("q and k must have the same rows and the plan's head_dim")
        at = _index(positions, (rows,), q.device, "positions")
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if q_out is None else q_out
        k_out = torch.empty(k.shape, dtype=q.dtype, device=q.device) if k_out is None else k_out
        q_to, k_to = _heads(q_out, q, "q_out"), _heads(k_out, q, "k_out")
        if q_out.shape != q.shape or k_out.shape != k.shape:
            raise OperatorError("q_out and k_out must have the shapes of q and k")
        if rows:
            with _on(q.device) as stream:
                _check(_lib.load().pb_rotary_device(
                    self._h, _TYPES[q.dtype], rows, at, q.shape[1], _ref(q_in), _ref(q_to), k.shape[1],
                    _ref(k_in), _ref(k_to), stream))
        return q_out, k_out

    def apply_to_cache(self, q, k, v, positions, cache, slots, layer=0, q_out=None):
        """q turned, as apply; k turned and v go to `layer` of the cache at
        slots[row] = page * page_size + slot in the page (-1: nowhere)."""
        q_in = _first(q, "q")
        k_in, v_in = _heads(k, cache.k, "k"), _heads(v, cache.k, "v")
        rows = q.shape[0]
        if q.dtype != cache.k.dtype or q.device != cache.k.device or q.shape[2] != self.head_dim:
            raise OperatorError("q must have the cache's type and device and the plan's head_dim")
        if k.shape != (rows, cache.kv_heads, self.head_dim) or v.shape != k.shape:
            raise OperatorError("k and v must be [rows, the cache's heads, head_dim]")
        a = _index(positions, (rows,), q.device, "positions")
        b = _index(slots, (rows,), q.device, "slots")
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if q_out is None else q_out
        q_to = _heads(q_out, q, "q_out")
        if q_out.shape != q.shape:
            raise OperatorError("q_out must have the shape of q")
        if rows:
            with _on(q.device) as stream:
                _check(_lib.load().pb_rotary_cache_device(
                    self._h, rows, a, q.shape[1], _ref(q_in), _ref(q_to), _ref(k_in), _ref(v_in),
                    _ref(cache._c), layer, b, stream))
        return q_out


def prompt_attention(q, k, v, offsets, kv_offsets=None, scale=None, out=None):
    """Causal attention of packed prompts: sequence s has the rows offsets[s] to
    offsets[s + 1] of q and kv_offsets[s] to kv_offsets[s + 1] (default: the same)
    of k and v, aligned at their ends.  scale defaults to head_dim ** -0.5.  Rows
    behind offsets[-1] are left as they were (unset in a new tensor)."""
    q_in = _first(q, "q")
    k_in, v_in = _heads(k, q, "k"), _heads(v, q, "v")
    rows, heads, dim = q.shape
    if k.shape != v.shape or k.shape[2] != dim:
        raise OperatorError("k and v must have one shape and q's head_dim")
    seqs = offsets.shape[0] - 1
    a = _index(offsets, (seqs + 1,), q.device, "offsets")
    b = None if kv_offsets is None else _index(kv_offsets, (seqs + 1,), q.device, "kv_offsets")
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else out
    to = _heads(out, q, "out")
    if out.shape != q.shape:
        raise OperatorError("out must have the shape of q")
    with _on(q.device) as stream:
        _check(_lib.load().pb_prompt_attention_device(
            _TYPES[q.dtype], dim, heads, k.shape[1], seqs, rows, k.shape[0], _ref(q_in), _ref(k_in),
            _ref(v_in), _ref(to), a, b, dim ** -0.5 if scale is None else scale, stream))
    return out


@functools.lru_cache(maxsize=256)
def _workspace_bytes(device, type_, dim, heads, kv_heads, seqs, rows):
    return int(_lib.load().pb_tree_attention_workspace(type_, dim, heads, kv_heads, seqs, rows))


def tree_workspace_bytes(cache, heads, seqs, rows):
    """Bytes of workspace that tree_attention needs for these sizes."""
    with _on(cache.k.device):
        got = _workspace_bytes(cache.k.device.index, cache._c.type, cache.head_dim, heads, cache.kv_heads, seqs, rows)
    if not got:
        raise OperatorError(_lib.last_error())
    return got


def tree_attention(q, cache, tables, contexts, offsets, visible, layer=0, scale=None, out=None, workspace=None):
    """Attention of drafted nodes over a paged cache: the rows offsets[s] to
    offsets[s + 1] of q are sequence s's nodes, whose keys and values stand at
    position contexts[s] + node; a row sees the contexts[s] positions before them
    and node j where bit j of visible[row] (int64) is set.  Position p is in page
    tables[s, p // page_size].  One node with visible 1 is plain decode.
    `workspace`: a uint8 tensor of tree_workspace_bytes, for calls that never
    overlap; by default one from torch's allocator."""
    q_in = _first(q, "q")
    rows, heads, dim = q.shape
    seqs = contexts.shape[0]
    if q.dtype != cache.k.dtype or q.device != cache.k.device or dim != cache.head_dim:
        raise OperatorError("q must have the cache's type, device and head_dim")
    a = _index(tables, (seqs, tables.shape[-1]), q.device, "tables")
    b = _index(contexts, (seqs,), q.device, "contexts")
    c = _index(offsets, (seqs + 1,), q.device, "offsets")
    d = _index(visible, (rows,), q.device, "visible", (torch.int64, torch.uint64))
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else out
    to = _heads(out, q, "out")
    if out.shape != q.shape:
        raise OperatorError("out must have the shape of q")
    if not rows:
        return out
    with _on(q.device) as stream:
        if workspace is None:
            need = _workspace_bytes(q.device.index, cache._c.type, dim, heads, cache.kv_heads, seqs, rows)
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        elif workspace.dtype != torch.uint8 or workspace.device != q.device or not workspace.is_contiguous():
            raise OperatorError("workspace must be a contiguous uint8 tensor on q's device")
        _check(_lib.load().pb_tree_attention_device(
            _ref(cache._c), layer, heads, seqs, rows, _ref(q_in), _ref(to), a, tables.shape[1], b, c, d,
            dim ** -0.5 if scale is None else scale, workspace.data_ptr(), workspace.numel(), stream))
    return out


class PagePool:
    """The host's book of a cache's pages: which pages each sequence holds, shared
    between forks until one of them writes."""

    def __init__(self, pages, page_size, max_seqs):
        self._h = ctypes.c_void_p()
        _check(_lib.load().pb_pool_create(pages, page_size, max_seqs, _ref(self._h)))
        self.pages, self.page_size = pages, page_size

    def __del__(self):
        try:
            if self._h:
                _lib.load().pb_pool_destroy(self._h)
                self._h = None
        except Exception:
            pass

    def open(self):
        """A new sequence without tokens."""
        seq = ctypes.c_uint32()
        _check(_lib.load().pb_pool_open(self._h, _ref(seq)))
        return seq.value

    def fork(self, seq):
        """A new sequence that shares every page of `seq`."""
        child = ctypes.c_uint32()
        _check(_lib.load().pb_pool_fork(self._h, seq, _ref(child)))
        return child.value

    def extend(self, seq, tokens):
        """Room for `tokens` more; None, or the (from, to) pair of pages that
        PageCache.copy_pages has to copy before anything is written."""
        pair, needed = (ctypes.c_uint32 * 2)(), ctypes.c_uint32()
        _check(_lib.load().pb_pool_extend(self._h, seq, tokens, pair, _ref(needed)))
        return None if pair[0] == 0xFFFFFFFF else (pair[0], pair[1])

    def truncate(self, seq, length):
        """Cuts a sequence to `length` tokens and frees the pages behind them."""
        _check(_lib.load().pb_pool_truncate(self._h, seq, length))

    def free(self, seq):
        _check(_lib.load().pb_pool_free(self._h, seq))

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
        return torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32, device=device)

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
        _check(lib.pb_pool_table(self._h, seq, table, self.pages, _ref(length), _ref(needed)))
        return list(table[:needed.value]), length.value
