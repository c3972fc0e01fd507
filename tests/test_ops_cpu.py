"""Host side of the paged serving operators: the C ABI's refusals, which come before
anything touches a device, and the book of a cache's pages."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from promptboot_b200 import _lib

torch = pytest.importorskip("torch")
from promptboot_b200 import ops  # noqa: E402

CAPACITY, ALIGNMENT, STATE = 4, 5, 1
FAKE = 1 << 20  # an address that is only looked at


def ref(x):
    return ctypes.byref(x)


def rows(data=FAKE, row=128, head=64):
    return _lib.PbRows(data, row, head)


def cache(**changes):
    c = _lib.PbCache(FAKE, 2 * FAKE, 1 << 20, 2, 2, 8, 16, 2, 64)
    for name, value in changes.items():
        setattr(c, name, value)
    return c


def refused(status, want, text):
    assert status == want and text in _lib.last_error(), (status, _lib.last_error())


@pytest.mark.parametrize("changes,text", [
    (dict(head_dim=60), "multiples of 16"), (dict(rotary_dim=72), "multiples of 16"),
    (dict(rotary_dim=80), "rotary_dim <= head_dim"), (dict(head_dim=272, rotary_dim=16), "256"),
    (dict(layout=2), "unknown"), (dict(scaling=4), "unknown"), (dict(theta=1.0), "theta"),
    (dict(theta=float("nan")), "theta"), (dict(magnitude=-1.0), "magnitude"),
    (dict(scaling=1, factor=0.5), "factor"), (dict(scaling=1, factor=float("inf")), "factor"),
    (dict(scaling=2, original=0.0), "original"), (dict(scaling=3, low=8.0, high=4.0), "low < high"),
    (dict(scaling=3, original=float("nan")), "original"),
])
def test_rotary_configurations_refused(changes, text):
    c = _lib.PbRotaryConfig(64, 64, 0, 0, 1e4, 2.0, 4096.0, 0.0, 0.0, 0.0)
    for name, value in changes.items():
        setattr(c, name, value)
    h = ctypes.c_void_p(1)
    refused(_lib.load().pb_rotary_create(ref(c), ref(h)), CAPACITY, text)
    assert not h.value


def test_rotary_refusals():
    lib, plan = _lib.load(), ops.Rotary(64)
    q, k = rows(), rows()

    def turn(type_=0, n=4, positions=FAKE, q=q, q_out=q, k_heads=2, k=k, k_out=k):
        return lib.pb_rotary_device(plan._h, type_, n, positions, 2, q and ref(q), q_out and ref(q_out), k_heads,
                                    k and ref(k), k_out and ref(k_out), None)
    refused(turn(type_=3), CAPACITY, "type")
    refused(turn(n=0), CAPACITY, "rows")
    refused(turn(positions=None), CAPACITY, "NULL")
    refused(turn(q=None), CAPACITY, "q is NULL")
    refused(turn(k_out=None), CAPACITY, "k_out is NULL")
    refused(turn(q=rows(FAKE + 4)), ALIGNMENT, "16-byte")
    refused(turn(k=rows(row=130)), ALIGNMENT, "16-byte")
    refused(turn(q_out=rows(row=256)), CAPACITY, "strides")

    def store(c, layer=0, slots=FAKE, v=rows()):
        return lib.pb_rotary_cache_device(plan._h, 4, FAKE, 2, ref(q), ref(q), ref(k), v and ref(v), ref(c), layer,
                                          slots, None)
    refused(store(cache(), layer=2), CAPACITY, "layer")
    refused(store(cache(), slots=None), CAPACITY, "NULL")
    refused(store(cache(), v=None), CAPACITY, "v is NULL")
    refused(store(cache(head_dim=128, layer_stride=1 << 21)), CAPACITY, "head_dim")


@pytest.mark.parametrize("changes,status,text", [
    (dict(k=None), CAPACITY, "NULL"), (dict(type=7), CAPACITY, "type"), (dict(page_size=24), CAPACITY, "page_size"),
    (dict(page_size=8), CAPACITY, "page_size"), (dict(page_size=512), CAPACITY, "page_size"),
    (dict(pages=0), CAPACITY, "pages"), (dict(layers=0), CAPACITY, "layers"), (dict(kv_heads=0), CAPACITY, "heads"),
    (dict(pages=1 << 27), CAPACITY, "2^31"), (dict(head_dim=72), CAPACITY, "head_dim"),
    (dict(v=FAKE + 8), ALIGNMENT, "16-byte"), (dict(layer_stride=(1 << 20) + 4), ALIGNMENT, "16-byte"),
    (dict(layer_stride=128), CAPACITY, "smaller"),
])
def test_caches_refused_by_every_operator(changes, status, text):
    lib, c = _lib.load(), cache(**changes)
    refused(lib.pb_cache_copy_pages_device(ref(c), 1, FAKE, None), status, text)
    refused(lib.pb_cache_keep_device(ref(c), 1, FAKE, 1, FAKE, FAKE, FAKE, 1, None), status, text)
    refused(lib.pb_tree_attention_device(ref(c), 0, 2, 1, 1, ref(rows()), ref(rows()), FAKE, 1, FAKE, FAKE, FAKE, 1.0,
                                         FAKE, 1 << 40, None), status, text)


def test_page_operations_without_work_or_arguments():
    lib, c = _lib.load(), cache()
    assert lib.pb_cache_copy_pages_device(ref(c), 0, None, None) == 0
    assert lib.pb_cache_keep_device(ref(c), 0, None, 0, None, None, None, 0, None) == 0
    refused(lib.pb_cache_copy_pages_device(ref(c), 1, None, None), CAPACITY, "NULL")
    refused(lib.pb_cache_keep_device(ref(c), 1, FAKE, 0, FAKE, FAKE, FAKE, 1, None), CAPACITY, "empty table")
    refused(lib.pb_cache_keep_device(ref(c), 1, FAKE, 1, FAKE, None, FAKE, 1, None), CAPACITY, "NULL")


def test_prompt_attention_refusals():
    lib = _lib.load()

    def prompt(type_=2, dim=64, heads=4, kv_heads=2, seqs=1, n=8, kv_n=8, q=rows(), k=rows(), out=rows(), offsets=FAKE,
               kv_offsets=FAKE, scale=1.0):
        return lib.pb_prompt_attention_device(type_, dim, heads, kv_heads, seqs, n, kv_n, q and ref(q), ref(k), ref(k),
                                              ref(out), offsets, kv_offsets, scale, None)
    refused(prompt(type_=9), CAPACITY, "type")
    for dim in (0, 32, 96, 256):
        refused(prompt(dim=dim), CAPACITY, "head_dim")
    refused(prompt(heads=3), CAPACITY, "multiple of kv_heads")
    refused(prompt(kv_heads=0), CAPACITY, "multiple of kv_heads")
    refused(prompt(seqs=0), CAPACITY, "sequences")
    refused(prompt(seqs=2049), CAPACITY, "sequences")
    refused(prompt(n=1 << 29), CAPACITY, "2^30")
    refused(prompt(kv_n=1 << 30), CAPACITY, "2^30")
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        refused(prompt(scale=scale), CAPACITY, "scale")
    refused(prompt(kv_offsets=None, kv_n=9), CAPACITY, "kv_offsets")
    refused(prompt(offsets=None), CAPACITY, "q_offsets")
    refused(prompt(q=None), CAPACITY, "q is NULL")
    refused(prompt(out=rows(head=68)), ALIGNMENT, "out")
    assert prompt(n=0) == 0


def test_attention_scales_whose_power_of_two_is_not_finite_are_refused():
    """Weights are powers of two: scale log2(e) has to be finite too."""
    lib, r = _lib.load(), rows()
    for scale in (2.4e38, 3e38):
        refused(lib.pb_prompt_attention_device(2, 64, 4, 2, 1, 8, 8, ref(r), ref(r), ref(r), ref(r), FAKE, FAKE, scale,
                                               None), CAPACITY, "scale")
        refused(lib.pb_tree_attention_device(ref(cache()), 0, 4, 1, 8, ref(r), ref(r), FAKE, 4, FAKE, FAKE, FAKE, scale,
                                             FAKE, 1 << 40, None), CAPACITY, "scale")
    # the next check speaks where the scale will do
    refused(lib.pb_prompt_attention_device(2, 64, 4, 2, 1, 8, 1 << 30, ref(r), ref(r), ref(r), ref(r), FAKE, FAKE,
                                           2.3e38, None), CAPACITY, "kv_rows")


def test_outputs_whose_rows_or_heads_lie_on_one_another_are_refused():
    lib, plan, r = _lib.load(), ops.Rotary(64), rows()
    for bad in (rows(row=0), rows(head=0)):
        refused(lib.pb_prompt_attention_device(2, 64, 4, 2, 1, 8, 8, ref(r), ref(r), ref(r), ref(bad), FAKE, FAKE, 1.0,
                                               None), CAPACITY, "out needs a row stride")
        refused(lib.pb_tree_attention_device(ref(cache()), 0, 4, 1, 8, ref(r), ref(bad), FAKE, 4, FAKE, FAKE, FAKE, 1.0,
                                             FAKE, 1 << 40, None), CAPACITY, "out needs a row stride")
        refused(lib.pb_rotary_device(plan._h, 0, 4, FAKE, 2, ref(bad), ref(bad), 0, None, None, None), CAPACITY,
                "q_out needs a row stride")
        refused(lib.pb_rotary_device(plan._h, 0, 4, FAKE, 2, ref(r), ref(r), 2, ref(r), ref(bad), None), CAPACITY,
                "k_out needs a row stride")
        refused(lib.pb_rotary_cache_device(plan._h, 4, FAKE, 2, ref(r), ref(bad), ref(r), ref(r), ref(cache()), 0, FAKE,
                                           None), CAPACITY, "q_out needs a row stride")
    # one row of one head has no strides to speak of: the next check speaks
    refused(lib.pb_rotary_device(plan._h, 0, 1, FAKE, 1, ref(r), ref(rows(row=0, head=0)), 1, ref(r), None, None),
            CAPACITY, "k_out is NULL")


def test_workspaces_refused_twice_say_why_twice(monkeypatch):
    import contextlib
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    cache = ops.PageCache.__new__(ops.PageCache)
    cache.device, cache.dtype, cache.head_dim, cache.kv_heads = 0, torch.bfloat16, 64, 2
    for _ in range(2):
        with pytest.raises(ops.OperatorError, match="multiple of kv_heads"):
            ops.tree_workspace_bytes(cache, 3, 1, 8)
        with pytest.raises(ops.OperatorError, match="sequences"):
            ops.tree_workspace_bytes(cache, 4, 4096, 8)
    assert ops.tree_workspace_bytes(cache, 4, 1, 8) == ops.tree_workspace_bytes(cache, 4, 1, 8) > 0
    with pytest.raises(ops.OperatorError, match="out of range"):
        ops.tree_workspace_bytes(cache, 4, 1, (1 << 32) + 8)


def test_tree_attention_refusals():
    lib = _lib.load()

    def tree(c=cache(), layer=0, heads=4, seqs=1, n=8, q=rows(), tables=FAKE, width=4, visible=FAKE, work=FAKE,
             size=1 << 40):
        return lib.pb_tree_attention_device(ref(c), layer, heads, seqs, n, q and ref(q), ref(rows()), tables, width,
                                            FAKE, FAKE, visible, 1.0, work, size, None)
    refused(tree(layer=2), CAPACITY, "layer")
    refused(tree(c=cache(head_dim=32)), CAPACITY, "head_dim must be 64 or 128")
    refused(tree(heads=5), CAPACITY, "multiple of kv_heads")
    refused(tree(q=None), CAPACITY, "q is NULL")
    refused(tree(tables=None), CAPACITY, "NULL")
    refused(tree(width=0), CAPACITY, "empty table")
    refused(tree(visible=None), CAPACITY, "NULL")
    refused(tree(width=1 << 28), CAPACITY, "reach too far")
    refused(tree(width=1 << 25, seqs=2048), CAPACITY, "reach too far")
    refused(tree(work=None), CAPACITY, "workspace")
    refused(tree(size=64), CAPACITY, "workspace")
    refused(tree(work=FAKE + 8), ALIGNMENT, "workspace")
    assert tree(n=0) == 0
    assert lib.pb_tree_attention_workspace(2, 96, 4, 2, 1, 8) == 0


def test_wrappers_refuse_tensors_off_the_gpu():
    x = torch.zeros(4, 2, 64)
    with pytest.raises(ops.OperatorError, match="CUDA"):
        ops.prompt_attention(x, x, x, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ops.OperatorError, match="CUDA"):
        ops.PageCache(torch.zeros(1, 2, 1, 16, 64), torch.zeros(1, 2, 1, 16, 64))
    with pytest.raises(ops.OperatorError, match="scaling"):
        ops.Rotary(64, scaling="ntk")


def test_a_cache_that_asks_for_gradients_is_refused_before_its_call():
    cache = ops.PageCache.__new__(ops.PageCache)  # its calls look at the tensors before anything else
    cache.k, cache.v = torch.zeros(1, 2, 1, 16, 64), torch.zeros(1, 2, 1, 16, 64, requires_grad=True)
    for call in (lambda: cache.copy_pages(None), lambda: cache.keep(None, None, None, None),
                 lambda: ops.tree_attention(None, cache, None, None, None, None),
                 lambda: ops.Rotary(64).apply_to_cache(None, None, None, None, cache, None)):
        with pytest.raises(ops.OperatorError, match="the cache asks for a gradient"):
            call()


def test_tensors_with_a_tangent_are_refused():
    import torch.autograd.forward_ad as forward
    x = torch.zeros(4, 2, 64)
    cache = ops.PageCache.__new__(ops.PageCache)
    cache.k, cache.v = torch.zeros(1, 2, 1, 16, 64), torch.zeros(1, 2, 1, 16, 64)
    with forward.dual_level():
        dual = forward.make_dual(x, x + 1)
        with torch.no_grad(), pytest.raises(ops.OperatorError, match="q asks for a gradient"):
            ops._heads(dual, torch.float32, -1, "q")
        ops._heads(x, torch.float32, -1, "q")
        ops._no_gradient(cache)
        cache.v = forward.make_dual(cache.v, cache.k)
        with pytest.raises(ops.OperatorError, match="the cache asks for a gradient"):
            ops._no_gradient(cache)

    def use(t):
        ops._heads(t, torch.float32, -1, "k")
        return t
    with pytest.raises(ops.OperatorError, match="k asks for a gradient"):
        torch.func.jvp(use, (x,), (x,))
    with pytest.raises(ops.OperatorError, match="k asks for a gradient"):
        torch.func.grad(lambda t: use(t).sum())(x)


def test_attention_status_asks_the_device_that_is_meant(monkeypatch):
    asked = []
    monkeypatch.setattr(ops, "_call", lambda device, fn: asked.append(device))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    for device in (None, "cuda", torch.device("cuda"), "cuda:0", torch.device("cuda", 2), 1):
        ops.attention_status(device)
    assert asked == [3, 3, 3, 0, 2, 1]
    with pytest.raises(ops.OperatorError, match="CUDA"):
        ops.attention_status("cpu")


def test_every_thread_is_told_of_each_failure_once(tmp_path):
    """What pb_attention_status says of a device's count, by host thread."""
    import pathlib
    import subprocess
    import threading
    csrc = pathlib.Path(_lib.__file__).parent / "csrc"
    source, built = tmp_path / "told.cpp", tmp_path / "told.so"
    source.write_text('#include "pb_told.h"\nextern "C" int news(int device, unsigned count) '
                      '{ static thread_local pb::Told told; return told.news(device, count); }\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", str(csrc), str(source), "-o", str(built)], check=True)
    news = ctypes.CDLL(str(built)).news
    assert [news(0, n) for n in (0, 0, 2, 2, 3, 3)] == [0, 0, 1, 0, 1, 0]
    assert [news(1, n) for n in (0, 1, 1)] == [0, 1, 0] and news(0, 3) == 0  # by device
    other = []
    thread = threading.Thread(target=lambda: other.extend(news(0, 3) for _ in range(2)))
    thread.start()
    thread.join()
    assert other == [1, 0]  # what one thread asked takes nothing from another
    assert news(0, 3) == 0 and news(0, 4) == 1
    assert [news(64, 0), news(64, 2), news(64, 2), news(-1, 0)] == [0, 1, 1, 0]


# ---------------------------------------------------------------- the book of pages

def test_pool_shares_pages_until_one_sequence_writes():
    pool = ops.PagePool(8, 16, 3)
    a = pool.open()
    assert pool.extend(a, 20) is None and pool.pages_of(a) == [0, 1] and pool.length(a) == 20
    b = pool.fork(a)
    assert pool.pages_of(b) == [0, 1] and pool.free_pages() == 6
    assert pool.extend(b, 0) is None and pool.pages_of(b) == [0, 1]  # nothing will be written
    pair = pool.extend(b, 1)
    assert pair == (1, 2) and pool.pages_of(b) == [0, 2] and pool.pages_of(a) == [0, 1]
    assert pool.extend(a, 1) is None  # its last page is its own again
    pool.truncate(b, 16)
    assert pool.pages_of(b) == [0] and pool.free_pages() == 6
    assert pool.extend(b, 1) is None  # a full shared page needs no copy
    pool.free(a)
    assert pool.free_pages() == 6 and pool.pages_of(b)[0] == 0
    pool.free(b)
    assert pool.free_pages() == 8


def test_pool_refusals_change_nothing():
    pool = ops.PagePool(4, 16, 2)
    a = pool.open()
    pool.extend(a, 40)
    for _ in range(2):
        with pytest.raises(ops.OperatorError, match="too few free pages"):
            pool.extend(a, 25)
        assert pool.pages_of(a) == [0, 1, 2] and pool.length(a) == 40 and pool.free_pages() == 1
    b = pool.fork(a)
    with pytest.raises(ops.OperatorError, match="too few free pages"):
        pool.extend(b, 10)  # one new page and the copy of the shared last one
    assert pool.pages_of(b) == [0, 1, 2] and pool.length(b) == 40
    with pytest.raises(ops.OperatorError, match="every sequence is open"):
        pool.fork(a)
    with pytest.raises(ops.OperatorError, match="shorter"):
        pool.truncate(a, 41)
    with pytest.raises(ops.OperatorError, match="has 40 tokens"):
        pool.slots(a, 30, 11, device="cpu")
    with pytest.raises(ops.OperatorError) as e:
        pool.free(7)
    assert e.value.status == STATE
    pool.free(b)
    with pytest.raises(ops.OperatorError, match="not open"):
        pool.free(b)
    with pytest.raises(ops.OperatorError, match="too few"):
        pool.extend(a, 2**32 - 1)
    for bad in ((0, 16, 1), (4, 0, 1), (4, 16, 0), (1 << 27, 16, 1)):
        with pytest.raises(ops.OperatorError):
            ops.PagePool(*bad)


def test_numbers_past_32_bits_are_refused_not_cut():
    pool, big = ops.PagePool(8, 16, 2), 1 << 32
    a = pool.open()
    pool.extend(a, 40)
    for bad in (lambda: pool.extend(a, big + 5), lambda: pool.extend(a, -1), lambda: pool.truncate(a, big),
                lambda: pool.truncate(a, big + 20), lambda: pool.fork(a + big), lambda: pool.free(a + big),
                lambda: pool.pages_of(a + big), lambda: pool.length(a - big), lambda: ops.PagePool(big + 4, 16, 2),
                lambda: ops.PagePool(4, big + 16, 2), lambda: ops.PagePool(4, 16, big + 2),
                lambda: ops.Rotary(big + 64), lambda: ops.Rotary(64, big + 32), lambda: ops.Rotary(64, -big + 32)):
        with pytest.raises(ops.OperatorError, match="out of range"):
            bad()
        assert pool.pages_of(a) == [0, 1, 2] and pool.length(a) == 40 and pool.free_pages() == 5
    with pytest.raises(ops.OperatorError, match="rotary_dim"):
        ops.Rotary(64, 0)  # no rotation is not the whole head


def test_copies_of_a_plan_or_a_pool_share_what_is_destroyed_once(monkeypatch):
    import copy
    import pickle
    lib, gone = _lib.load(), []

    class Spy:
        def __getattr__(self, name):
            if name.endswith("_destroy"):
                return lambda h: (gone.append(name), getattr(lib, name)(h))
            return getattr(lib, name)
    monkeypatch.setattr(ops._lib, "load", Spy)
    pool, plan = ops.PagePool(8, 16, 2), ops.Rotary(64)
    for whole in (copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError, match="copied"):
            whole(pool)
        with pytest.raises(TypeError, match="copied"):
            whole(plan)
    others = copy.copy(pool), copy.copy(plan)
    del pool, plan
    assert gone == []
    assert others[0].extend(others[0].open(), 40) is None and others[0].free_pages() == 5
    del others
    assert sorted(gone) == ["pb_pool_destroy", "pb_rotary_destroy"]
    with pytest.raises(ops.OperatorError):
        ops.PagePool(0, 16, 2)  # nothing was made, nothing is destroyed
    assert len(gone) == 2


def test_pool_tables_and_slots_of_nothing_keep_their_shapes():
    pool = ops.PagePool(8, 16, 2)
    assert pool.tables([], device="cpu").shape == (0, 1)
    a = pool.open()
    assert pool.tables([a], device="cpu").tolist() == [[-1]] and pool.slots(a, 0, 0, device="cpu").shape == (0,)
    pool.extend(a, 17)
    assert pool.tables([a, a], device="cpu").tolist() == [[0, 1], [0, 1]]


def test_a_pool_takes_memory_for_the_sequences_that_are_open_not_for_all_it_may_open():
    import subprocess
    import sys
    code = """
import ctypes, resource
from promptboot_b200 import _lib
lib, pool, seq, child = _lib.load(), ctypes.c_void_p(), ctypes.c_uint32(), ctypes.c_uint32()
pair, needed = (ctypes.c_uint32 * 2)(), ctypes.c_uint32()
size = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (size + (1 << 30),) * 2)
assert lib.pb_pool_create(64, 16, 2**32 - 1, ctypes.byref(pool)) == 0, _lib.last_error()
for want in range(1000):
    assert lib.pb_pool_open(pool, ctypes.byref(seq)) == 0 and seq.value == want
assert lib.pb_pool_extend(pool, 999, 40, pair, ctypes.byref(needed)) == 0
assert lib.pb_pool_fork(pool, 999, ctypes.byref(child)) == 0 and child.value == 1000
assert lib.pb_pool_free(pool, 7) == 0 and lib.pb_pool_open(pool, ctypes.byref(seq)) == 0 and seq.value == 7
"""
    assert subprocess.run([sys.executable, "-c", code], timeout=120).returncode == 0


def test_pool_short_arrays_are_refused_with_the_number_needed():
    lib, pool = _lib.load(), ops.PagePool(8, 16, 2)
    a, b = pool.open(), pool.open()
    pool.extend(a, 40)
    pool.extend(b, 40)
    table, length, needed = (ctypes.c_uint32 * 4)(), ctypes.c_uint32(), ctypes.c_uint32()
    refused(lib.pb_pool_table(pool._h, a, table, 2, ref(length), ref(needed)), CAPACITY, "too short")
    assert needed.value == 3
    assert lib.pb_pool_table(pool._h, a, table, 4, ref(length), ref(needed)) == 0
    assert list(table) == [0, 1, 2, 0xFFFFFFFF] and length.value == 40
    pool.free(a)
    n, used = ctypes.c_uint32(), ctypes.c_uint32()
    refused(lib.pb_pool_compact(pool._h, table, 2, ref(n), ref(used), ref(needed)), CAPACITY, "too short")
    assert needed.value == 3 and pool.pages_of(b) == [3, 4, 5]


def test_pool_against_a_plain_book():
    """Random opens, forks, writes, cuts and compactions, with the tokens of every
    sequence held in a plain list beside the pages."""
    rng = np.random.default_rng(0)
    page, pages = 4, 24
    pool, memory, books, fresh = ops.PagePool(pages, page, 6), np.zeros((pages, page), int), {}, iter(range(1, 10**6))
    for _ in range(4000):
        what = rng.integers(0, 6)
        seq = int(rng.choice(list(books))) if books else None
        try:
            if what == 0 or seq is None:
                books[pool.open()] = []
            elif what == 1:
                child = pool.fork(seq)
                books[child] = list(books[seq])
            elif what == 2 and rng.random() < 0.5:
                pool.free(seq)
                del books[seq]
            elif what == 3:
                cut = int(rng.integers(0, len(books[seq]) + 1))
                pool.truncate(seq, cut)
                del books[seq][cut:]
            elif what == 4 and rng.random() < 0.2:
                moves, used = pool.compact()
                assert len({t for _, t in moves} | {f for f, _ in moves}) == 2 * len(moves)
                for a, b in moves:
                    memory[b] = memory[a]
                assert all(p < used for s in books for p in pool.pages_of(s)) and used == pages - pool.free_pages()
            else:
                tokens = [next(fresh) for _ in range(int(rng.integers(0, 11)))]
                pair = pool.extend(seq, len(tokens))
                if pair:
                    memory[pair[1]] = memory[pair[0]]
                start = len(books[seq])
                books[seq] += tokens
                for slot, token in zip(pool.slots(seq, start, len(tokens), device="cpu").tolist(), tokens):
                    memory[slot // page, slot % page] = token
        except ops.OperatorError as e:
            assert e.status == CAPACITY
        for s, tokens in books.items():
            ids = pool.pages_of(s)
            assert pool.length(s) == len(tokens) and len(ids) == -(-len(tokens) // page)
            assert [memory[ids[i // page], i % page] for i in range(len(tokens))] == tokens
    used = {p for s in books for p in pool.pages_of(s)}
    assert pool.free_pages() == pages - len(used)
