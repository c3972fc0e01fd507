"""The paged serving operators (promptboot_b200.ops) on the GPU against their
definitions in binary64.

Tolerances are bounds, not fits.  A result rounded to its type is off by half a
step, eps / 2 of its value (and half the smallest subnormal); what comes before it
is bounded per element:
 * rotary: the angle in turns is rounded to binary32 after its whole part is taken
   off (2^-25 of half a turn), sincospi is within 2 ulp, and the two products, the
   sum and the magnitude round once each: at most 7e-7 m (|a| + |b|) in all;
 * attention: a score of d products summed in binary32 is off by 2 d 2^-24 of the
   sum of their magnitudes (twice, for sums that truncate), which scales its weight
   by as much times the scale; weights round to the type of v where products run on
   the tensor cores (eps / 2), the exponential adds 2^-21, and n sums add n 2^-23.
   All of these are relative to weights, so the result is off by at most their sum
   (twice the score's part: it enters the sum of weights too) times the weighted
   mean of |v|.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from promptboot_b200 import ops  # noqa: E402

TYPES = [torch.float32, torch.float16, torch.bfloat16]
NAN = float("nan")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts(counts):
    return i32(np.concatenate([[0], np.cumsum(counts)]).tolist())


def half_step(dtype, y):
    """Half a step of the type at y, in binary64."""
    info = torch.finfo(dtype)
    return y.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def assert_within(got, want, bound):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (int(bad.sum()), off[bad].max().item(), (off / bound)[bad].max().item(),
                           bad.nonzero()[:3].tolist())


# ------------------------------------------------------------------------ rotary

def frequencies(rd, theta, scaling, factor, original, low, high):
    f = theta ** (-2.0 * np.arange(rd // 2) / rd)
    if scaling == "linear":
        return f / factor
    if scaling == "bands":
        keep = np.clip((original * f / (2 * math.pi) - low) / (high - low), 0, 1)
        return f / factor * (1 - keep) + f * keep
    if scaling == "yarn":
        def place(turns):
            return rd * math.log(original / (2 * math.pi * turns)) / (2 * math.log(theta))
        i0, i1 = max(math.floor(place(high)), 0), min(math.ceil(place(low)), rd - 1)
        i1 = i1 if i1 > i0 else i0 + 0.001
        keep = 1 - np.clip((np.arange(rd // 2) - i0) / (i1 - i0), 0, 1)
        return f / factor * (1 - keep) + f * keep
    return f


def turned(x, positions, f, interleaved, magnitude):
    """(turned rows, |a| + |b| of each element's pair) in binary64."""
    x = x.double()
    rd = 2 * len(f)
    angle = positions.double()[:, None] * torch.tensor(f, device="cuda")
    c, s = angle.cos()[:, None] * magnitude, angle.sin()[:, None] * magnitude
    y, size = x.clone(), torch.zeros_like(x)
    a_at = slice(0, rd, 2) if interleaved else slice(0, rd // 2)
    b_at = slice(1, rd, 2) if interleaved else slice(rd // 2, rd)
    a, b = x[..., a_at], x[..., b_at]
    y[..., a_at], y[..., b_at] = a * c - b * s, b * c + a * s
    size[..., a_at] = size[..., b_at] = a.abs() + b.abs()
    return y, size


ROTARY = [  # head_dim, rotary_dim, interleaved, scaling, theta, factor, original, low, high
    (64, 64, False, "none", 1e6, 1.0, 0, 0, 0),
    (64, 64, True, "linear", 1e4, 4.0, 0, 0, 0),
    (128, 64, False, "bands", 5e5, 8.0, 8192, 0, 0),
    (128, 32, True, "yarn", 1e6, 4.0, 32768, 0, 0),
    (64, 64, False, "yarn", 1e4, 2.5, 2048, 0.5, 16.0),
    (80, 16, True, "bands", 1e4, 2.0, 4096, 1.0, 2.0),
    (256, 256, False, "none", 1e4, 1.0, 0, 0, 0),
    (16, 16, True, "none", 1e4, 1.0, 0, 0, 0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", ROTARY, ids=lambda s: f"{s[0]}-{s[1]}-{'adjacent' if s[2] else 'halves'}-{s[3]}")
@pytest.mark.parametrize("rows,heads,kv_heads", [(1, 14, 2), (37, 3, 1), (2100, 5, 2)])
def test_rotary_matches_the_definition(dtype, shape, rows, heads, kv_heads):
    dim, rd, interleaved, scaling, theta, factor, original, low, high = shape
    g = gen(rows + dim)
    q, k = normal(g, rows, heads, dim, dtype=dtype, scale=3.0), normal(g, rows, kv_heads, dim, dtype=dtype)
    positions = torch.randint(0, 1 << 20, (rows,), generator=g, device="cuda", dtype=torch.int32)
    positions[0] = 0
    plan = ops.Rotary(dim, rd, theta, interleaved, scaling, factor, original, low, high)
    f = frequencies(rd, theta, scaling, factor, original, low or 1.0, high or (32.0 if scaling == "yarn" else 4.0))
    m = 0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0
    q1, k1 = plan.apply(q, k, positions)
    for got, x in ((q1, q), (k1, k)):
        want, size = turned(x, positions, f, interleaved, m)
        assert got.dtype == dtype
        assert_within(got, want, half_step(dtype, want) + 7e-7 * m * size)
        assert torch.equal(got[..., rd:], x[..., rd:])
    # in place gives the same bits
    plan.apply(q, k, positions, q_out=q, k_out=k)
    assert torch.equal(q, q1) and torch.equal(k, k1)


def test_rotary_far_positions_magnitude_and_rows_left_out():
    """Positions up to 2^32 - 2 keep their angle; 0xffffffff leaves a row alone."""
    g = gen(3)
    q, k = normal(g, 6, 2, 64), normal(g, 6, 1, 64)
    at = np.array([0, 1, 2**24 + 1, 2**31 + 5, 2**32 - 2, 2**32 - 1], dtype=np.uint32)
    positions = torch.from_numpy(at.view(np.int32)).cuda()
    plan = ops.Rotary(64, theta=1e4, magnitude=1.75)
    q_out, k_out = torch.full_like(q, NAN), torch.full_like(k, NAN)
    plan.apply(q, k, positions, q_out, k_out)
    f = frequencies(64, 1e4, "none", 1, 0, 0, 0)
    # an angle of 2^32 is off by 2^32 2^-53 of a turn before it is reduced: below 4e-6
    for got, x in ((q_out, q), (k_out, k)):
        want, size = turned(x, torch.from_numpy(at.astype(np.float64)).cuda(), f, False, 1.75)
        assert_within(got[:5], want[:5], half_step(torch.float32, want[:5]) + (1.75 * 7e-7 + 8e-6) * size[:5])
        assert got[5].isnan().all()


def test_rotary_of_stacked_projection_views():
    g = gen(4)
    stacked = normal(g, 50, 14 + 2 + 2, 64, dtype=torch.bfloat16)
    q, k = stacked[:, :14], stacked[:, 14:16]
    positions = torch.arange(50, dtype=torch.int32, device="cuda")
    plan = ops.Rotary(64)
    want = plan.apply(q.contiguous(), k.contiguous(), positions)
    v = stacked[:, 16:].clone()
    plan.apply(q, k, positions, q_out=q, k_out=k)  # in place in the stack
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(stacked[:, 16:], v)
    by_head = torch.empty(14, 50, 64, dtype=torch.bfloat16, device="cuda")
    plan.apply(normal(gen(4), 50, 18, 64, dtype=torch.bfloat16)[:, :14], k, positions, q_out=by_head.transpose(0, 1))
    assert torch.equal(by_head.transpose(0, 1), want[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,rows", [(16, 1), (64, 45), (256, 1200)])
def test_rotary_to_cache(dtype, page, rows):
    g = gen(rows)
    pages, layers, dim, kv_heads = rows // page + 4, 3, 64, 2
    q = normal(g, rows, 6, dim, dtype=dtype)
    k, v = normal(g, rows, kv_heads, dim, dtype=dtype), normal(g, rows, kv_heads, dim, dtype=dtype)
    cache = ops.PageCache(normal(g, layers, pages, kv_heads, page, dim, dtype=dtype),
                          normal(g, layers, pages, kv_heads, page, dim, dtype=dtype))
    positions = torch.randint(0, 40000, (rows,), generator=g, device="cuda", dtype=torch.int32)
    slots = torch.randperm(pages * page, generator=g, device="cuda", dtype=torch.int32)[:rows].contiguous()
    if rows > 10:
        slots[2], slots[3], slots[4] = -1, pages * page, 2**31 - 1  # none, just past the cache, far past it
        positions[5] = -1
    plan = ops.Rotary(dim)
    want_q, want_k = plan.apply(q, k, positions)
    want = [cache.k.clone(), cache.v.clone()]
    for r, (s, p) in enumerate(zip(slots.tolist(), positions.tolist())):
        if 0 <= s < pages * page and p >= 0:
            want[0][1, s // page, :, s % page] = want_k[r]
            want[1][1, s // page, :, s % page] = v[r]
    q_out = torch.zeros_like(q)
    plan.apply_to_cache(q, k, v, positions, cache, slots, layer=1, q_out=q_out)
    there = positions >= 0
    assert torch.equal(q_out[there], want_q[there]) and not q_out[~there].any()
    assert torch.equal(cache.k, want[0]) and torch.equal(cache.v, want[1])


# --------------------------------------------------------------------- attention

def attend(q, k, v, seen, scale, dtype):
    """(result, bound) of one head in binary64: q [t, d], k and v [n, d], seen [t, n].
    Keys and values that a row does not see are taken out of its sums."""
    q, k, v = q.double(), k.double(), v.double()
    hidden = ~seen.any(0)
    k, v = k.masked_fill(hidden[:, None], 0.0), v.masked_fill(hidden[:, None], 0.0)
    d, n = q.shape[1], k.shape[0]
    if n == 0:
        return torch.zeros_like(q), torch.full_like(q, 1e-300)
    s = (q @ k.t() * scale).masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    y, mean = p @ v, p @ v.abs()
    size = (q.abs() @ k.abs().t() * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    weights = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    part = 2 * (2 * d * 2.0**-24 * size + 2.0**-21) + weights + n * 2.0**-23
    return y, half_step(dtype, y) + part * mean


def check_heads(got, q, keys, values, seen, scale, dtype):
    """got, q [t, heads, d]; keys and values [n, kv_heads, d]."""
    group = q.shape[1] // keys.shape[1]
    for h in range(q.shape[1]):
        y, bound = attend(q[:, h], keys[:, h // group], values[:, h // group], seen, scale, dtype)
        assert_within(got[:, h], y, bound)


def causal(t, n):
    return torch.ones(t, n, dtype=torch.bool, device="cuda").tril(n - t)


PROMPTS = [  # tokens and keys of each sequence
    ([1], None), ([5, 0, 1, 130, 0], None), ([257], None), ([64, 128, 127, 129, 2], None),
    ([3, 40, 200], [700, 41, 200]), ([20, 9, 5], [4, 0, 9]), ([1, 1, 1], [1, 129, 1000]), ([1500, 33], None),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 14, 2), (128, 4, 4), (64, 3, 1), (128, 16, 2)])
@pytest.mark.parametrize("tokens,keys", PROMPTS, ids=[f"{a}-{b}" for a, b in PROMPTS])
def test_prompt_attention_matches_the_definition(dtype, dim, heads, kv_heads, tokens, keys):
    g = gen(sum(tokens) + dim)
    extra = 3  # rows behind the last sequence
    q = normal(g, sum(tokens) + extra, heads, dim, dtype=dtype, scale=2.0)
    counts = keys or tokens
    n = sum(counts) + (extra if keys is None else 0)
    k, v = normal(g, n, kv_heads, dim, dtype=dtype), normal(g, n, kv_heads, dim, dtype=dtype)
    out = torch.full_like(q, 7.0)
    got = ops.prompt_attention(q, k, v, starts(tokens), None if keys is None else starts(keys), out=out)
    assert got is out and (out[sum(tokens):] == 7.0).all()
    at = kv_at = 0
    for t, c in zip(tokens, counts):
        check_heads(out[at:at + t], q[at:at + t], k[kv_at:kv_at + c], v[kv_at:kv_at + c], causal(t, c),
                    dim ** -0.5, dtype)
        at, kv_at = at + t, kv_at + c


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_attention_keeps_out_what_a_row_does_not_see(dtype, dim):
    """A NaN or an infinity in a key or a value reaches the rows that see it and no
    other: not earlier rows, not the next sequence, not rows past the keys."""
    g = gen(8)
    tokens = [70, 133, 20]
    total = sum(tokens)
    q, k, v = (normal(g, total + 5, h, dim, dtype=dtype) for h in (4, 2, 2))
    want = ops.prompt_attention(q, k, v, starts(tokens))[:total].clone()
    k[total:], v[total:] = NAN, math.inf
    k[100, 0], v[100, 1, 3] = NAN, NAN   # sequence 1, token 30
    v[150, 0, 5], v[150, 0, 6] = math.inf, -math.inf   # its token 80
    v[69, 0], k[69, 1] = NAN, math.inf   # the last token of sequence 0
    got = ops.prompt_attention(q, k, v, starts(tokens))[:total]
    clean = torch.ones(total, dtype=torch.bool, device="cuda")
    clean[69] = False
    clean[100:203] = False
    assert torch.equal(got[clean], want[clean])
    assert got[100:203, :2].isnan().all()      # heads of key head 0 see a NaN score
    assert got[100:203, 2:, 3].isnan().all()   # a NaN value stays in its component
    assert torch.equal(got[100:203, 2:, 4], want[100:203, 2:, 4])
    assert got[69, :2].isnan().all()


def test_prompt_attention_infinite_value_reaches_its_component():
    for dtype in TYPES:
        g = gen(9)
        q, k, v = (normal(g, 40, 1, 64, dtype=dtype) for _ in range(3))
        want = ops.prompt_attention(q, k, v, starts([40])).clone()
        v[25, 0, 5], v[25, 0, 6] = math.inf, -math.inf
        got = ops.prompt_attention(q, k, v, starts([40]))
        assert (got[25:, 0, 5] == math.inf).all() and (got[25:, 0, 6] == -math.inf).all()
        got[25:, 0, 5:7] = want[25:, 0, 5:7]
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 14, 2), (128, 32, 8)])
def test_prompt_attention_of_many_short_prompts_with_infinite_values(dtype, dim, heads, kv_heads):
    """More units than the GPU holds, half of them with a value that is not finite: it
    reaches its component in the rows that see it and changes no other bit, whatever the
    units before and after are doing."""
    g, rng = gen(25), np.random.default_rng(25)
    lengths = [int(n) for n in rng.integers(1, 120, 200)]
    first = np.concatenate([[0], np.cumsum(lengths)])
    n = int(first[-1])
    q, k, v = (normal(g, n, h, dim, dtype=dtype) for h in (heads, kv_heads, kv_heads))
    want = ops.prompt_attention(q, k, v, starts(lengths))
    check_heads(want[:lengths[0]], q[:lengths[0]], k[:lengths[0]], v[:lengths[0]], causal(lengths[0], lengths[0]),
                dim ** -0.5, dtype)
    hit = torch.zeros_like(want, dtype=torch.bool)
    for s in range(0, 200, 2):
        at, c = int(first[s]) + int(rng.integers(lengths[s])), s % dim
        v[at, :, c] = math.inf
        hit[at:int(first[s + 1]), :, c] = True
    for _ in range(10):
        got = ops.prompt_attention(q, k, v, starts(lengths))
        assert torch.equal(got.isinf(), hit)
        assert torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_attention_of_prompts_without_keys_between_infinite_values(dtype, dim):
    """A unit without key tiles makes no warp wait for another: what the unit before it
    has still to write does not mix with the unit after it."""
    g, rng = gen(28), np.random.default_rng(28)
    tokens = [int(t) if s % 2 else 4 for s, t in enumerate(rng.integers(1, 33, 2000))]
    keys = [t if s % 2 else 0 for s, t in enumerate(tokens)]
    first, key = np.concatenate([[0], np.cumsum(tokens)]), np.concatenate([[0], np.cumsum(keys)])
    q = normal(g, sum(tokens), 4, dim, dtype=dtype)
    k, v = (normal(g, sum(keys), 1, dim, dtype=dtype) for _ in range(2))
    at = starts(tokens), starts(keys)
    want = ops.prompt_attention(q, k, v, *at)
    hit, none = torch.zeros_like(want, dtype=torch.bool), torch.zeros(sum(tokens), dtype=torch.bool, device="cuda")
    for s, t in enumerate(tokens):
        if keys[s]:
            i, c = int(rng.integers(t)), s % dim
            v[int(key[s]) + i, 0, c] = math.inf
            hit[int(first[s]) + i:int(first[s + 1]), :, c] = True
        else:
            none[int(first[s]):int(first[s + 1])] = True
    for _ in range(20):
        got = ops.prompt_attention(q, k, v, *at)
        assert torch.equal(got.isinf(), hit) and torch.equal(got[~hit], want[~hit])
        assert not got[none].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_attention_of_stacked_views_and_a_given_scale(dtype):
    g = gen(10)
    stacked = normal(g, 300, 18, 64, dtype=dtype)
    q, k, v = stacked[:, :14], stacked[:, 14:16], stacked[:, 16:]
    by_head = torch.zeros(14, 300, 64, dtype=dtype, device="cuda")
    tokens = [170, 130]
    ops.prompt_attention(q, k, v, starts(tokens), scale=0.3, out=by_head.transpose(0, 1))
    for at, t in ((0, 170), (170, 130)):
        rows = slice(at, at + t)
        check_heads(by_head.transpose(0, 1)[rows], q[rows], k[rows], v[rows], causal(t, t), 0.3, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_attention_of_keys_by_head_and_of_one_expanded_head(dtype):
    g = gen(13)
    q = normal(g, 200, 4, 64, dtype=dtype)
    k, v = (normal(g, 2, 200, 64, dtype=dtype).transpose(0, 1) for _ in range(2))  # stored [heads, rows, dim]
    got = ops.prompt_attention(q, k, v, starts([150, 50]))
    assert torch.equal(got, ops.prompt_attention(q, k.contiguous(), v.contiguous(), starts([150, 50])))
    one = k[:, :1].expand(200, 4, 64)  # a head stride of zero
    got = ops.prompt_attention(q, one, v[:, 1:].expand(200, 4, 64), starts([150, 50]))
    want = ops.prompt_attention(q, k[:, :1].contiguous(), v[:, 1:].contiguous(), starts([150, 50]))
    # four key heads or one with four query heads: the same sums over other row tiles
    at = 0
    for t in (150, 50):
        check_heads(got[at:at + t], q[at:at + t], one[at:at + t], v[at:at + t, 1:].expand(t, 4, 64), causal(t, t), 0.125, dtype)
        check_heads(want[at:at + t], q[at:at + t], k[at:at + t, :1], v[at:at + t, 1:], causal(t, t), 0.125, dtype)
        at += t


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_attention_without_keys_is_zero(dtype):
    g = gen(14)
    q, none = normal(g, 30, 4, 64, dtype=dtype), normal(g, 1, 2, 64, dtype=dtype)[:0]
    assert not ops.prompt_attention(q, none, none, starts([10, 20]), kv_offsets=starts([0, 0])).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_with_offsets_that_do_not_ascend_stays_in_its_buffers(dtype):
    """Results are those of the sequences that are there; the others have no rows."""
    g, rng = gen(15), np.random.default_rng(15)
    q, k, v = (normal(g, 64, h, 64, dtype=dtype) for h in (4, 2, 2))
    out = torch.full_like(q, 3.0)
    ops.prompt_attention(q, k, v, i32([60, 20, 20, 64, 10]), out=out)  # 60..20 and 64..10 are none
    assert torch.equal(out[20:], ops.prompt_attention(q[20:], k[20:], v[20:], i32([0, 44]))) and (out[:20] == 3.0).all()
    cache, tables, _, _ = paged(g, rng, [40, 40, 40], 16, 2, 64, dtype)
    visible = masks([1] * 64)
    out = torch.full_like(q, 3.0)
    ops.tree_attention(q, cache, tables, i32([39, 39, 39]), i32([5, 3, 4, 2]), visible, layer=1, out=out)
    assert (out[:3] == 3.0).all() and (out[4:] == 3.0).all() and not (out[3] == 3.0).any()


def test_prompt_attention_cuts_offsets_at_the_rows():
    g = gen(11)
    q, k, v = (normal(g, 40, 2, 64) for _ in range(3))
    want = ops.prompt_attention(q, k, v, i32([0, 25, 40]))
    got = ops.prompt_attention(q, k, v, i32([0, 25, 1000]))
    assert torch.equal(got, want)
    out = torch.full_like(q, 5.0)
    ops.prompt_attention(q, k, v, i32([30, 10, 10, 2**31 - 1]), out=out)  # the first descends: no rows
    assert (out[:10] == 5.0).all() and not (out[10:] == 5.0).any()


def test_prompt_attention_large_scores_and_growing_maxima():
    """Scores of some hundreds, growing along the keys, so that the running maximum
    moves at every tile; and a row of equal scores."""
    for dtype in TYPES:
        g = gen(12)
        n, dim = 700, 64
        q = torch.ones(n, 1, dim, device="cuda")
        k = torch.linspace(-6, 6, n, device="cuda")[:, None, None].expand(n, 1, dim).contiguous()
        k[::3] *= -1
        q, k = q.to(dtype), k.to(dtype)
        v = normal(g, n, 1, dim, dtype=dtype)
        got = ops.prompt_attention(q, k, v, starts([n]), scale=0.7)
        check_heads(got, q, k, v, causal(n, n), 0.7, dtype)
        got = ops.prompt_attention(q, k * 0, v, starts([n]))
        check_heads(got, q, k * 0, v, causal(n, n), 0.125, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_scores_that_are_all_minus_infinity_is_zero(dtype, dim):
    """As of a row that sees nothing, over tiles that every row sees whole too."""
    g, rng = gen(32), np.random.default_rng(32)
    q, k, v = (normal(g, 300, h, dim, dtype=dtype) for h in (4, 2, 2))
    q[..., 0], k[:, 1, 0] = 1.0, -math.inf
    got = ops.prompt_attention(q, k, v, starts([300]))
    assert not got[:, 2:].any() and got[:, :2].any(-1).all()
    for nodes in (1, 20, 60):
        cache, tables, _, _ = paged(g, rng, [400 + nodes], 16, 2, dim, dtype)
        cache.k[1][:, 1, :, 0] = -math.inf
        q = normal(g, nodes, 4, dim, dtype=dtype)
        q[..., 0] = 1.0
        got = ops.tree_attention(q, cache, tables, i32([400]), starts([nodes]),
                                 masks([1 << i for i in range(nodes)]), layer=1)
        assert not got[:, 2:].any() and got[:, :2].any(-1).all()


def masks(values):
    return torch.from_numpy(np.array(values, dtype=np.uint64).view(np.int64)).cuda()


def random_tree(rng, t):
    bits = []
    for i in range(t):
        parent = int(rng.integers(-1, i)) if i else -1
        bits.append((bits[parent] if 0 <= parent < 64 else 0) | (1 << i if i < 64 else 0))
    return bits


def paged(g, rng, lengths, page, kv_heads, dim, dtype, layers=2, junk=None):
    """A cache whose sequences lie on scattered pages, with `junk` in every slot that
    holds none of their positions; and the sequences' keys and values."""
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 3
    ids = rng.permutation(pages)
    cache = ops.PageCache.empty(layers, pages, kv_heads, page, dim, dtype)
    cache.k.fill_(1.0 if junk is None else junk)
    cache.v.fill_(1.0 if junk is None else junk)
    width = max(need + [1]) + 1
    table = np.full((len(lengths), width), -1, dtype=np.int32)
    keys, values, at = [], [], 0
    for s, n in enumerate(lengths):
        mine = ids[at:at + need[s]]
        at += need[s]
        table[s, :need[s]] = mine
        k, v = normal(g, n, kv_heads, dim, dtype=dtype), normal(g, n, kv_heads, dim, dtype=dtype)
        p = np.arange(n)
        where = torch.from_numpy(mine[p // page].astype(np.int64)).cuda(), slice(None), torch.from_numpy(p % page).cuda()
        cache.k[1][where], cache.v[1][where] = k, v
        keys.append(k)
        values.append(v)
    return cache, torch.from_numpy(table).cuda(), keys, values


def check_tree(got, q, contexts, nodes, visible, keys, values, scale, dtype):
    at = 0
    for s, (c, t) in enumerate(zip(contexts, nodes)):
        n = c + min(t, 64)
        seen = torch.zeros(t, n, dtype=torch.bool, device="cuda")
        seen[:, :c] = True
        for i in range(t):
            for j in range(n - c):
                seen[i, c + j] = (visible[at + i] >> j) & 1
        check_heads(got[at:at + t], q[at:at + t], keys[s][:n], values[s][:n], seen, scale, dtype)
        at += t


TREES = [  # contexts, nodes
    ([0], [1]), ([1], [1]), ([300, 17, 0, 128], [1, 1, 1, 1]), ([127, 129, 64], [1, 2, 5]),
    ([1000, 0, 5, 250], [17, 33, 0, 9]), ([90, 200], [64, 63]), ([40], [70]), ([4097, 3, 2000], [4, 4, 8]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,kv_heads,page", [(64, 14, 2, 16), (128, 4, 4, 64), (64, 8, 1, 256), (128, 16, 2, 32),
                                                     (64, 4, 2, 128)])
@pytest.mark.parametrize("contexts,nodes", TREES, ids=[f"{a}-{b}" for a, b in TREES])
def test_tree_attention_matches_the_definition(dtype, dim, heads, kv_heads, page, contexts, nodes):
    g, rng = gen(sum(contexts) + dim), np.random.default_rng(sum(contexts) + page)
    # slots behind the last position hold NaN: they are seen by none
    cache, tables, keys, values = paged(g, rng, [c + t for c, t in zip(contexts, nodes)], page, kv_heads, dim, dtype,
                                        junk=NAN)
    q = normal(g, sum(nodes) + 2, heads, dim, dtype=dtype, scale=2.0)
    visible = [b for t in nodes for b in random_tree(rng, t)]
    out = torch.full_like(q, 7.0)
    got = ops.tree_attention(q, cache, tables, i32(contexts), starts(nodes), masks(visible + [0, 0]), layer=1, out=out)
    assert got is out and (out[sum(nodes):] == 7.0).all()
    check_tree(out, q, contexts, nodes, visible, keys, values, dim ** -0.5, dtype)


def check_groups(got, q, keys, values, seen, dtype):
    """check_heads for many heads: the heads that share a key head as rows of one."""
    dim, group = q.shape[2], q.shape[1] // keys.shape[1]
    rows = seen.repeat_interleave(group, 0)
    for h in range(keys.shape[1]):
        mine = slice(h * group, (h + 1) * group)
        y, bound = attend(q[:, mine].reshape(-1, dim), keys[:, h], values[:, h], rows, dim ** -0.5, dtype)
        assert_within(got[:, mine].reshape(-1, dim), y, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 1024, 1), (128, 1024, 8), (64, 512, 512), (128, 129, 3)])
def test_attention_of_the_most_heads(dtype, dim, heads, kv_heads):
    g, rng = gen(34), np.random.default_rng(34)
    tokens, keys = [3, 0, 1, 70], [3, 5, 130, 69]
    q = normal(g, sum(tokens), heads, dim, dtype=dtype)
    k, v = (normal(g, sum(keys), kv_heads, dim, dtype=dtype) for _ in range(2))
    got = ops.prompt_attention(q, k, v, starts(tokens), kv_offsets=starts(keys))
    at = kv_at = 0
    for t, n in zip(tokens, keys):
        check_groups(got[at:at + t], q[at:at + t], k[kv_at:kv_at + n], v[kv_at:kv_at + n], causal(t, n), dtype)
        at, kv_at = at + t, kv_at + n
    contexts, nodes = [40, 500, 0], [1, 3, 2]
    cache, tables, keys, values = paged(g, rng, [c + t for c, t in zip(contexts, nodes)], 16, kv_heads, dim, dtype)
    q = normal(g, sum(nodes), heads, dim, dtype=dtype)
    got = ops.tree_attention(q, cache, tables, i32(contexts), starts(nodes), masks([1, 1, 2, 5, 1, 3]), layer=1)
    at = 0
    for s, (c, t, bits) in enumerate(zip(contexts, nodes, ([1], [1, 2, 5], [1, 3]))):
        seen = torch.tensor([[j < c or b >> (j - c) & 1 == 1 for j in range(c + t)] for b in bits], device="cuda")
        check_groups(got[at:at + t], q[at:at + t], keys[s], values[s], seen, dtype)
        at += t


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_the_most_sequences(dtype):
    """2048 of them, one with nearly all the rows; one more is refused."""
    g, rng = gen(35), np.random.default_rng(35)
    tokens = [1] * 2048
    tokens[1000], tokens[1001], tokens[7] = 300, 0, 64
    q, k, v = (normal(g, sum(tokens), h, 64, dtype=dtype) for h in (4, 1, 1))
    got = ops.prompt_attention(q, k, v, starts(tokens))
    first = np.concatenate([[0], np.cumsum(tokens)])
    for s in (0, 7, 999, 1000, 1002, 2047):
        rows = slice(int(first[s]), int(first[s + 1]))
        check_heads(got[rows], q[rows], k[rows], v[rows], causal(tokens[s], tokens[s]), 0.125, dtype)
    alone = torch.tensor([s not in (7, 1000) for s in np.repeat(np.arange(2048), tokens)], device="cuda")
    assert torch.equal(got[alone], v[alone].expand(-1, 4, -1))  # one key: its value
    contexts = [int(c) for c in rng.integers(0, 40, 2048)]
    contexts[1000] = 5000
    nodes = [min(t, 64) for t in tokens]
    cache, tables, keys, values = paged(g, rng, [c + t for c, t in zip(contexts, nodes)], 16, 1, 64, dtype)
    q = normal(g, sum(nodes), 4, 64, dtype=dtype)
    visible = [b for t in nodes for b in random_tree(rng, t)]
    got = ops.tree_attention(q, cache, tables, i32(contexts), starts(nodes), masks(visible), layer=1)
    first = np.concatenate([[0], np.cumsum(nodes)])
    for s in (0, 7, 999, 1000, 1002, 2047):
        rows = slice(int(first[s]), int(first[s + 1]))
        check_tree(got[rows], q[rows], contexts[s:s + 1], nodes[s:s + 1], visible[rows], keys[s:s + 1],
                   values[s:s + 1], 0.125, dtype)
    with pytest.raises(ops.OperatorError, match="sequences"):
        ops.prompt_attention(q, q[:, :1], q[:, :1], i32([0] * 2050))


@pytest.mark.parametrize("dtype", TYPES)
def test_tree_attention_rows_that_see_nothing_and_odd_masks(dtype):
    """Masks that leave a row empty without a context, that skip the row's own node,
    and whose bits past the last node mean nothing."""
    g, rng = gen(20), np.random.default_rng(20)
    contexts, nodes = [0, 30], [4, 4]
    cache, tables, keys, values = paged(g, rng, [4, 34], 16, 2, 64, dtype)
    q = normal(g, 8, 6, 64, dtype=dtype)
    visible = [0, 1, 0b1110, 2**64 - 1, 0, 0b0100, 2**63 + 1, 2**64 - 16]
    got = ops.tree_attention(q, cache, tables, i32(contexts), starts(nodes), masks(visible), layer=1)
    assert not got[0].any()
    check_tree(got, q, contexts, nodes, visible, keys, values, 0.125, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nodes", [1, 12])
def test_tree_attention_keeps_out_what_a_node_does_not_see(dtype, nodes):
    """NaN keys and values of a node that others do not see stay with it."""
    g, rng = gen(21), np.random.default_rng(21)
    contexts = [200, 75]
    cache, tables, keys, values = paged(g, rng, [c + nodes for c in contexts], 32, 2, 64, dtype)
    q = normal(g, 2 * nodes, 8, 64, dtype=dtype)
    visible = [1 << i for i in range(nodes)] * 2
    args = (tables, i32(contexts), starts([nodes] * 2), masks(visible))
    want = ops.tree_attention(q, cache, *args, layer=1).clone()
    bad = 200 + nodes - 1
    page, slot = int(tables[0, bad // 32]), bad % 32
    cache.v[1, page, 0, slot] = math.inf
    cache.v[1, page, 1, slot, 7] = NAN
    got = ops.tree_attention(q, cache, *args, layer=1)
    others = [r for r in range(2 * nodes) if r != nodes - 1]
    assert torch.equal(got[others], want[others])
    assert (got[nodes - 1, :4] == math.inf).all() and got[nodes - 1, 4:, 7].isnan().all()
    cache.k[1, page, :, slot] = NAN
    got = ops.tree_attention(q, cache, *args, layer=1)
    assert torch.equal(got[others], want[others]) and got[nodes - 1].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,nodes,context", [(64, 1, 900), (64, 12, 200), (64, 48, 3000), (128, 12, 700)])
def test_tree_attention_of_what_is_not_a_number_over_split_contexts(dtype, dim, nodes, context):
    """A NaN in a query makes its row NaN and no other, NaN keys all rows that see them,
    where whole runs of a split context have no score that is a number."""
    g, rng = gen(29), np.random.default_rng(29)
    cache, tables, keys, values = paged(g, rng, [context + nodes], 16, 2, dim, dtype)
    q = normal(g, nodes, 8, dim, dtype=dtype)
    visible = random_tree(rng, nodes)
    args = (tables, i32([context]), starts([nodes]), masks(visible))
    want = ops.tree_attention(q, cache, *args, layer=1)
    bad = q.clone()
    bad[nodes // 2, 3, 5] = NAN
    got = ops.tree_attention(bad, cache, *args, layer=1)
    assert got[nodes // 2, 3].isnan().all()
    got[nodes // 2, 3] = want[nodes // 2, 3]
    check_tree(got, q, [context], [nodes], visible, keys, values, dim ** -0.5, dtype)
    at = torch.arange(64, 64 + context // 2, device="cuda")
    cache.k[1][tables[0, at // 16].long(), 1, at % 16] = NAN
    got = ops.tree_attention(q, cache, *args, layer=1)
    assert torch.equal(got[:, :4], want[:, :4]) and got[:, 4:].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_tree_attention_tables_that_end_and_pages_outside_the_cache(dtype):
    """Positions past the table are not seen; a page id outside the cache is zeros."""
    g, rng = gen(22), np.random.default_rng(22)
    cache, tables, keys, values = paged(g, rng, [64], 16, 1, 64, dtype)
    q = normal(g, 1, 2, 64, dtype=dtype)
    short = tables[:, :2].contiguous()  # 32 positions
    got = ops.tree_attention(q, cache, short, i32([60]), i32([0, 1]), masks([1]), layer=1)
    seen = torch.ones(1, 32, dtype=torch.bool, device="cuda")
    check_heads(got, q, keys[0][:32], values[0][:32], seen, 0.125, dtype)
    lost = tables[:, :4].clone()
    lost[0, 1], lost[0, 2] = -1, cache.pages
    keys[0][16:48], values[0][16:48] = 0, 0
    got = ops.tree_attention(q, cache, lost, i32([63]), i32([0, 1]), masks([1]), layer=1)
    check_heads(got, q, keys[0], values[0], torch.ones(1, 64, dtype=torch.bool, device="cuda"), 0.125, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,nodes", [(64, 3, 1), (64, 3, 5), (128, 5, 1), (128, 5, 3), (64, 3, 40)])
def test_tree_attention_of_growing_and_of_falling_scores(dtype, dim, heads, nodes):
    """The maximum moves in every tile, or in the first alone, by far more than the
    sums could bear without being scaled; and all scores alike."""
    g, rng = gen(24), np.random.default_rng(24)
    n = 900
    cache, tables, keys, values = paged(g, rng, [n + nodes] * 3, 16, 1, dim, dtype)
    ramp = torch.linspace(-6, 6, n + nodes, device="cuda")[:, None, None].expand(-1, 1, dim).to(dtype)
    for s, rows in enumerate([ramp, ramp.flip(0), ramp * 0 + 1]):
        keys[s] = rows.contiguous()
        ids = tables[s, :-(-(n + nodes) // 16)].long()
        p = torch.arange(n + nodes, device="cuda")
        cache.k[1][ids[p // 16], :, p % 16] = keys[s]
    q = torch.ones(3 * nodes, heads, dim, device="cuda", dtype=dtype)
    visible = [b for _ in range(3) for b in random_tree(rng, nodes)]
    got = ops.tree_attention(q, cache, tables, i32([n] * 3), starts([nodes] * 3), masks(visible), layer=1, scale=0.7)
    check_tree(got, q, [n] * 3, [nodes] * 3, visible, keys, values, 0.7, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 14, 2), (64, 15, 1), (64, 24, 1), (128, 6, 2), (128, 11, 1)])
def test_tree_attention_of_few_rows_beside_slots_without_keys(dtype, dim, heads, kv_heads):
    """Keys that end at every place of a tile: what the slots behind them hold changes no
    bit, however often a tile's value rows are cleaned in shared memory by the lanes that
    have them and read by others."""
    got = {}
    for junk in (0.5, NAN, math.inf):
        g, rng = gen(27), np.random.default_rng(27)
        contexts = list(range(1, 68))
        cache, tables, keys, values = paged(g, rng, [c + 1 for c in contexts], 16, kv_heads, dim, dtype, junk=junk)
        q = normal(g, len(contexts), heads, dim, dtype=dtype, scale=2.0)
        args = (q, cache, tables, i32(contexts), starts([1] * len(contexts)), masks([1] * len(contexts)))
        got[junk] = ops.tree_attention(*args, layer=1)
        assert all(torch.equal(got[junk], ops.tree_attention(*args, layer=1)) for _ in range(50))
    check_tree(got[0.5], q, contexts, [1] * len(contexts), [1] * len(contexts), keys, values, dim ** -0.5, dtype)
    assert torch.equal(got[0.5], got[NAN]) and torch.equal(got[0.5], got[math.inf])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("seqs,nodes", [(1, 1), (2, 48), (300, 1), (40, 3)])
def test_tree_attention_of_long_and_of_many_contexts(dtype, seqs, nodes):
    """Contexts that are split over many CTAs, and more sequences than CTAs; the
    second call on the same workspace gives the same bits."""
    g, rng = gen(23), np.random.default_rng(seqs)
    contexts = [30011, 12345][:seqs] if seqs < 3 else [int(c) for c in rng.integers(0, 900, seqs)]
    cache, tables, keys, values = paged(g, rng, [c + nodes for c in contexts], 64, 2, 64, dtype)
    q = normal(g, seqs * nodes, 14, 64, dtype=dtype, scale=2.0)
    visible = [b for _ in range(seqs) for b in random_tree(rng, nodes)]
    work = torch.full((ops.tree_workspace_bytes(cache, 14, seqs, seqs * nodes),), 255, dtype=torch.uint8, device="cuda")
    args = (q, cache, tables, i32(contexts), starts([nodes] * seqs), masks(visible))
    got = ops.tree_attention(*args, layer=1, workspace=work)
    check_tree(got, q, contexts, [nodes] * seqs, visible, keys, values, 0.125, dtype)
    assert torch.equal(got, ops.tree_attention(*args, layer=1, workspace=work))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_gives_the_same_bits_every_time(dtype):
    """Many calls on the same inputs: split contexts with several pieces per CTA, and
    packed prompts with several units per CTA.  A lost wait shows here first."""
    for seqs, nodes, dim, kv_heads, heads in ((16, 12, 128, 8, 32), (2, 48, 64, 2, 14), (60, 1, 64, 2, 14), (20, 5, 64, 2, 8)):
        g, rng = gen(24), np.random.default_rng(seqs)
        contexts = [int(c) for c in rng.integers(200, 3000 if seqs > 2 else 30000, seqs)]
        cache, tables, _, _ = paged(g, rng, [c + nodes for c in contexts], 64, kv_heads, dim, dtype)
        q = normal(g, seqs * nodes, heads, dim, dtype=dtype, scale=2.0)
        visible = masks([b for _ in range(seqs) for b in random_tree(rng, nodes)])
        args = (q, cache, tables, i32(contexts), starts([nodes] * seqs), visible)
        want = ops.tree_attention(*args, layer=1)
        assert all(torch.equal(want, ops.tree_attention(*args, layer=1)) for _ in range(400))
    for tokens, dim in (([1200, 100, 1], 64), ([64] * 60, 128)):
        g, n = gen(25), sum(tokens)
        q, k, v = (normal(g, n, h, dim, dtype=dtype, scale=1.5) for h in (14, 2, 2))
        want = ops.prompt_attention(q, k, v, starts(tokens))
        assert all(torch.equal(want, ops.prompt_attention(q, k, v, starts(tokens))) for _ in range(400))


# ------------------------------------------------------------------------- pages

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layers,page,kv_heads,dim,n", [(1, 16, 1, 16, 1), (3, 32, 2, 64, 7), (2, 256, 1, 128, 40), (24, 16, 3, 48, 5)])
def test_copy_pages(dtype, layers, page, kv_heads, dim, n):
    g = gen(n)
    pages = 2 * n + 3
    big = normal(g, layers + 1, pages, kv_heads, page, dim, dtype=dtype)
    other = normal(g, layers + 1, pages, kv_heads, page, dim, dtype=dtype)
    cache = ops.PageCache(big[:layers], other[:layers])
    ids = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    pairs = ids[:2 * n].reshape(-1, 2).contiguous()
    lost = i32([[0, pages], [-1, 1], [pages, 2]])  # left out
    want = [big.clone(), other.clone()]
    for a, b in pairs.tolist():
        for w in want:
            w[:layers, b] = w[:layers, a]
    cache.copy_pages(torch.cat([pairs, lost]))
    assert torch.equal(big, want[0]) and torch.equal(other, want[1])
    cache.copy_pages(pairs[:0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,kv_heads,dim", [(16, 2, 64), (64, 1, 128), (32, 3, 16)])
def test_keep_moves_the_accepted_path(dtype, page, kv_heads, dim):
    g, rng = gen(page), np.random.default_rng(page)
    contexts = [0, 13, 16, 100, 255]
    paths = [[0, 1, 2], [2, 5, 9, 10, 11, 20, 21, 30, 33, 40], [], [63], [0, 2, 3]]
    counts = [len(p) for p in paths]
    counts[4] = 2  # the rest of the row is not kept
    cache, tables, _, _ = paged(g, rng, [c + 64 for c in contexts], page, kv_heads, dim, dtype)
    cache.k.copy_(normal(g, *cache.k.shape, dtype=dtype))
    cache.v.copy_(normal(g, *cache.v.shape, dtype=dtype))
    want, table = [cache.k.clone(), cache.v.clone()], tables.tolist()
    for s, (c, path) in enumerate(zip(contexts, paths)):
        for w, x in zip(want, (cache.k, cache.v)):
            for i, n in enumerate(path[:counts[s]]):
                a, b = c + n, c + i
                w[:, table[s][b // page], :, b % page] = x[:, table[s][a // page], :, a % page]
    nodes = i32([p + [0] * (10 - len(p)) for p in paths])
    cache.keep(tables, i32(contexts), i32(counts), nodes)
    assert torch.equal(cache.k, want[0]) and torch.equal(cache.v, want[1])


def test_keep_leaves_out_entries_that_are_no_path():
    """Below their own index, not ascending, past the table, on a page outside the
    cache; a count past the row is cut."""
    g, rng = gen(30), np.random.default_rng(30)
    cache, tables, _, _ = paged(g, rng, [64], 16, 1, 64, torch.float32, layers=2)
    cache.k.copy_(normal(g, *cache.k.shape))
    cache.v.copy_(cache.k + 1)
    tables = tables[:, :4].contiguous()
    tables[0, 3] = -1
    table = tables[0].tolist()
    before = cache.k.clone()
    # from position 10: 3 -> 0; 2 does not ascend; 5 -> 2; 5 again; 2^31 - 1 and 60 are past; 6 is below itself
    cache.keep(tables, i32([10]), i32([99]), i32([[3, 2, 5, 5, 40, 2**31 - 1, 6]]))
    want = before.clone()

    def move(w, x, a, b):
        w[:, table[b // 16], :, b % 16] = x[:, table[a // 16], :, a % 16]
    move(want, before, 13, 10)
    move(want, before, 15, 12)
    assert torch.equal(cache.k, want)
    assert torch.equal(cache.v, want + 1)


def test_keep_of_long_rows_with_entries_that_stand_for_none():
    """-1 is above every node: what stands behind it is left out, within 32 entries and
    beyond; a row of more than 128 entries goes on where it stopped."""
    g = gen(31)
    cache = ops.PageCache.empty(1, 40, 1, 16, 16, torch.float32)
    cache.k.copy_(normal(g, *cache.k.shape))
    cache.v.copy_(cache.k + 1)
    before = cache.k.clone()
    tables = torch.arange(40, dtype=torch.int32, device="cuda").view(2, 20)
    path = list(range(3, 203))
    rows = [path, path[:31] + [-1] + path[32:]]
    cache.keep(tables, i32([7, 7]), i32([200, 200]), i32(rows))
    want = before.clone()
    for s, count in enumerate([200, 31]):
        for i in range(count):
            a, b = 10 + i, 7 + i
            want[0, 20 * s + b // 16, :, b % 16] = before[0, 20 * s + a // 16, :, a % 16]
    assert torch.equal(cache.k, want) and torch.equal(cache.v, want + 1)


def test_keep_of_no_nodes_and_of_a_count_that_stands_for_none():
    g = gen(33)
    cache = ops.PageCache.empty(2, 12, 1, 16, 64, torch.float32)
    cache.k.copy_(normal(g, *cache.k.shape))
    cache.v.copy_(cache.k + 1)
    want = cache.k.clone()
    tables = torch.arange(12, dtype=torch.int32, device="cuda").view(3, 4)
    cache.keep(tables, i32([5, 5, 5]), i32([-1, 0, 1]), i32([[2, 4], [3, 6], [3, 6]]))
    want[:, 8, :, 5] = want[:, 8, :, 8]
    assert torch.equal(cache.k, want) and torch.equal(cache.v, want + 1)


@pytest.mark.parametrize("dtype,pages", [(torch.float32, 9000), (torch.bfloat16, 18000)])
def test_places_past_32_bits(dtype, pages):
    """A cache of more than 2^31 elements a side (2^32 in 16 bits), and packed rows as far
    apart: every operator on the last of them."""
    g, rng = gen(36), np.random.default_rng(36)
    cache = ops.PageCache.empty(1, pages, 8, 256, 128, dtype)
    assert cache.k.numel() * cache.k.itemsize > 1 << 33
    tables = i32([[pages - 1, 2, pages - 3], [pages - 4, pages - 5, 1]])
    contexts, nodes, lengths = [520, 300], [9, 2], [529, 302]
    keys, values = [], []
    for s, n in enumerate(lengths):
        k, v = (normal(g, n, 8, 128, dtype=dtype) for _ in range(2))
        at = torch.arange(n, device="cuda")
        slots = tables[s][at // 256] * 256 + at.to(torch.int32) % 256
        zero = torch.zeros(n, dtype=torch.int32, device="cuda")  # at position 0 nothing turns
        ops.Rotary(128).apply_to_cache(k, k, v, zero, cache, slots.to(torch.int32))
        keys.append(k)
        values.append(v)
    visible = [b for t in nodes for b in random_tree(rng, t)]
    for heads in (8, 32):
        q = normal(g, sum(nodes), heads, 128, dtype=dtype)
        got = ops.tree_attention(q, cache, tables, i32(contexts), starts(nodes), masks(visible))
        check_tree(got, q, contexts, nodes, visible, keys, values, 128 ** -0.5, dtype)
    cache.copy_pages(i32([[pages - 1, pages - 2]]))
    cache.keep(tables, i32(contexts), i32([2, 1]), i32([[3, 8], [1, 0]]))
    for x, y in ((cache.k, keys), (cache.v, values)):
        assert torch.equal(x[0, pages - 2].transpose(0, 1), y[0][:256])
        assert torch.equal(x[0, pages - 3, :, 8:10].transpose(0, 1), y[0][[523, 528]])
        assert torch.equal(x[0, pages - 5, :, 44], y[1][301])
    apart = cache.k.view(-1)
    far = apart.numel() // 3 // 64 * 64
    q, k, v, out = (apart[i * 4096:].as_strided((3, h, 64), (far, 64, 1), i * 4096) for i, h in enumerate((4, 2, 2, 4)))
    for x in (q, k, v):
        x.copy_(normal(g, *x.shape, dtype=dtype))
    want_q, want_k = ops.Rotary(64).apply(q.contiguous(), k.contiguous(), i32([7, 8, 9]))
    ops.Rotary(64).apply(q, k, i32([7, 8, 9]), q_out=q, k_out=k)
    assert torch.equal(q, want_q) and torch.equal(k, want_k)
    ops.prompt_attention(q, k, v, i32([0, 3]), out=out)
    assert torch.equal(out, ops.prompt_attention(want_q, want_k, v.contiguous(), i32([0, 3])))


# ------------------------------------------------------------- streams and graphs

def test_operators_on_a_side_stream_and_in_graphs():
    """Each operator captured into a graph and replayed on new inputs; two graphs of
    tree attention with workspaces of their own; a side stream while the default
    stream is busy."""
    g, rng = gen(40), np.random.default_rng(40)
    dtype = torch.bfloat16
    contexts, nodes = [500, 60], [6, 3]
    cache, tables, keys, values = paged(g, rng, [506, 63], 16, 2, 64, dtype)
    q, k, v = (normal(g, 9, h, 64, dtype=dtype) for h in (14, 2, 2))
    visible = [b for t in nodes for b in random_tree(rng, t)]
    plan, positions = ops.Rotary(64), i32(list(range(9)))
    slots = i32([-1] * 9)
    cs, offs, vis = i32(contexts), starts(nodes), masks(visible)
    pairs = i32([[0, 1]]) * 0 - 1

    def chain():
        turned_q = plan.apply_to_cache(q, k, v, positions, cache, slots, layer=1)
        tree = ops.tree_attention(turned_q, cache, tables, cs, offs, vis, layer=1)
        kept = ops.prompt_attention(tree, k, v, offs)
        cache.copy_pages(pairs)
        cache.keep(tables, cs, i32_zero, nodes_zero)
        return tree, kept

    i32_zero, nodes_zero = i32([0, 0]), i32([[0], [0]])
    want = [x.clone() for x in chain()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(chain())
        graphs.append(graph)
    fresh = normal(g, 9, 14, 64, dtype=dtype)
    q.copy_(fresh)
    graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    want = chain()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("dtype", TYPES)
def test_operators_that_write_the_cache_on_a_side_stream_and_in_graphs(dtype):
    """A drafting step with rows that go to their pages, a page that is copied and paths
    that are kept: on a side stream while the default stream is held up, and from two
    graphs on new inputs, it leaves the outputs and the cache that a plain call leaves."""
    g, rng = gen(41), np.random.default_rng(41)
    contexts, nodes, page = [500, 60], [6, 3], 16
    cache, tables, _, _ = paged(g, rng, [c + t for c, t in zip(contexts, nodes)], page, 2, 64, dtype)
    cache.k.copy_(normal(g, *cache.k.shape, dtype=dtype))
    cache.v.copy_(normal(g, *cache.v.shape, dtype=dtype))
    clean = cache.k.clone(), cache.v.clone()
    table = tables.tolist()
    spare = min(set(range(cache.pages)) - {p for row in table for p in row})
    pairs = i32([[table[1][0], spare]])
    at = [table[s][(c + j) // page] * page + (c + j) % page
          for s, (c, t) in enumerate(zip(contexts, nodes)) for j in range(t)]
    slots = i32(at)
    counts, accepted = i32([2, 1]), i32([[1, 5], [2, 0]])
    q, k, v = (normal(g, 9, h, 64, dtype=dtype) for h in (14, 2, 2))
    plan, positions = ops.Rotary(64), i32(list(range(9)))
    cs, offs, vis = i32(contexts), starts(nodes), masks([b for t in nodes for b in random_tree(rng, t)])

    def reset():
        cache.k.copy_(clean[0])
        cache.v.copy_(clean[1])

    def chain():
        turned_q = plan.apply_to_cache(q, k, v, positions, cache, slots, layer=1)
        tree = ops.tree_attention(turned_q, cache, tables, cs, offs, vis, layer=1)
        packed = ops.prompt_attention(tree, k, v, offs)
        cache.copy_pages(pairs)
        cache.keep(tables, cs, counts, accepted)
        return turned_q, tree, packed

    def plain():
        reset()
        want = [x.clone() for x in (*chain(), cache.k, cache.v)]
        for now, before in zip(want[3:], clean):  # each of the three has written
            def row(x, i):
                return x[1, at[i] // page, :, at[i] % page]
            assert not torch.equal(row(now, 3), row(before, 3)) and torch.equal(row(now, 1), row(now, 5))
            assert torch.equal(now[:, spare], now[:, table[1][0]]) and not torch.equal(now[:, spare], before[:, spare])
        return want

    def same(got, want):
        return all(torch.equal(a, b) for a, b in zip((*got, cache.k, cache.v), want))
    want = plain()
    reset()
    side, held = torch.cuda.Stream(), torch.cuda.Event()
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda._sleep(400_000_000)  # some 0.2 s
    held.record()
    with torch.cuda.stream(side):
        got = chain()
    side.synchronize()
    assert not held.query()  # the default stream was still at it
    assert same(got, want)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(chain())
        graphs.append(graph)
    for _ in range(2):
        for x in (q, k, v):
            x.copy_(normal(g, *x.shape, dtype=dtype))
        want = plain()
        for graph, out in zip(graphs, outs):
            reset()
            graph.replay()
            assert same(out, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_calls_on_two_streams_at_once_give_the_bits_of_calls_in_turn(dtype):
    g, rng = gen(26), np.random.default_rng(26)
    jobs = []
    for nodes, seqs, dim in ((1, 40, 64), (20, 6, 128)):
        contexts = [int(c) for c in rng.integers(100, 3000, seqs)]
        cache, tables, _, _ = paged(g, rng, [c + nodes for c in contexts], 32, 2, dim, dtype)
        q = normal(g, seqs * nodes, 8, dim, dtype=dtype)
        visible = [b for _ in range(seqs) for b in random_tree(rng, nodes)]
        jobs.append(lambda q=q, cache=cache, args=(tables, i32(contexts), starts([nodes] * seqs), masks(visible)):
                    ops.tree_attention(q, cache, *args, layer=1))
    lengths = [int(n) for n in rng.integers(1, 200, 60)]
    q, k, v = (normal(g, sum(lengths), h, 64, dtype=dtype) for h in (8, 2, 2))
    jobs.append(lambda at=starts(lengths): ops.prompt_attention(q, k, v, at))
    want = [job() for job in jobs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(60):
        with torch.cuda.stream(streams[i % 2]):
            got.append((i % 3, jobs[i % 3]()))
    torch.cuda.synchronize()
    for j, y in got:
        assert torch.equal(y, want[j])


def test_first_calls_of_a_process_may_be_captured():
    """Nothing has to be set up before a capture."""
    import subprocess
    import sys
    code = """
import torch
from promptboot_b200 import ops
i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
q, k = torch.randn(4, 2, 64, device="cuda").bfloat16(), torch.randn(4, 1, 64, device="cuda").bfloat16()
cache = ops.PageCache.empty(1, 4, 1, 16, 64)
cache.k.zero_(); cache.v.fill_(1.0)
offsets, tables, contexts, one, at = i([0, 4]), i([[0, 1]]), i([9]), torch.ones(4, dtype=torch.int64, device="cuda"), i([0, 1, 2, 3])
slots, pairs, counts, nodes = i([-1] * 4), i([[0, 2]]), i([1]), i([[0]])
plan = ops.Rotary(64)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    a = plan.apply_to_cache(q, k, k, at, cache, slots)
    b = ops.prompt_attention(a, k, k, offsets)
    c = ops.tree_attention(a, cache, tables, contexts, offsets, one)
    d = ops.prompt_attention(q.float(), k.float(), k.float(), offsets)
    cache.copy_pages(pairs)
    cache.keep(tables, contexts, counts, nodes)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(c, torch.ones_like(c)) and torch.equal(b, ops.prompt_attention(a, k, k, offsets))
from promptboot_b200 import _lib
assert _lib.load().pb_attention_status(None) == 0
"""
    assert subprocess.run([sys.executable, "-c", code], timeout=120).returncode == 0


# ---------------------------------------------------------------- the run of them

@pytest.mark.parametrize("dtype", TYPES)
def test_a_drafting_step_of_forked_sequences(dtype):
    """Prompt, fork, drafted trees, kept paths and one more token: what every layer
    attends to is what plain attention over the same tokens in a row gives."""
    g = gen(50)
    heads, kv_heads, dim, page, layers = 14, 2, 64, 16, 2
    pool = ops.PagePool(64, page, 8)
    cache = ops.PageCache.empty(layers, 64, kv_heads, page, dim, dtype)
    cache.k.fill_(NAN)
    cache.v.fill_(NAN)
    plan = ops.Rotary(dim, scaling="yarn", factor=4.0, original_context=32768)
    length = 57

    def rows(n):
        return tuple(normal(g, n, h, dim, dtype=dtype) for h in (heads, kv_heads, kv_heads))

    def position(first, n):
        return torch.arange(first, first + n, dtype=torch.int32, device="cuda")

    # the prompt: turned into the cache, and attended from the packed rows
    parent = pool.open()
    assert pool.extend(parent, length) is None
    q, k, v = rows(length)
    for layer in range(layers):
        tq = plan.apply_to_cache(q, k, v, position(0, length), cache, pool.slots(parent, 0, length), layer=layer)
    tk = plan.apply(q, k, position(0, length))[1]
    got = ops.prompt_attention(tq, tk, v, starts([length]))
    check_heads(got, tq, tk, v, causal(length, length), dim ** -0.5, dtype)
    # two forks of it draft: the shared last page is copied before it is written
    seqs, paths, nodes = [parent, pool.fork(parent)], [[0, 2, 5], [1, 3]], [7, 4]
    trees = [[1, 3, 5, 9, 17, 0b100101, 0b1000000], [1, 2, 5, 0b1010]]
    pairs = [pool.extend(s, t) for s, t in zip(seqs, nodes)]
    assert [p is None for p in pairs] == [False, True]
    cache.copy_pages(i32([list(pairs[0])]))
    drafts = [rows(t) for t in nodes]
    dq, dk, dv = (torch.cat([d[i] for d in drafts]) for i in range(3))
    depth = torch.cat([i32([bin(b).count("1") - 1 for b in tree]) for tree in trees])
    slots = torch.cat([pool.slots(s, length, t) for s, t in zip(seqs, nodes)])
    tables, contexts = pool.tables(seqs), i32([length, length])
    visible = masks([b for tree in trees for b in tree])
    for layer in range(layers):
        tq = plan.apply_to_cache(dq, dk, dv, length + depth, cache, slots, layer=layer)
    got = ops.tree_attention(tq, cache, tables, contexts, starts(nodes), visible, layer=1)
    at = 0
    for s, t in enumerate(nodes):
        for i in range(t):  # each node against its path laid out in a row
            path = [j for j in range(t) if trees[s][i] >> j & 1]
            row_k = torch.cat([k, drafts[s][1][path]])
            tk = plan.apply(torch.cat([q, drafts[s][0][path]]), row_k, position(0, length + len(path)))[1]
            row_v = torch.cat([v, drafts[s][2][path]])
            seen = torch.ones(1, length + len(path), dtype=torch.bool, device="cuda")
            check_heads(got[at + i:at + i + 1], tq[at + i:at + i + 1], tk, row_v, seen, dim ** -0.5, dtype)
        at += t
    # the accepted paths stay, the rest of the pages goes back
    width = max(len(p) for p in paths)
    cache.keep(tables, contexts, i32([len(p) for p in paths]), i32([p + [0] * (width - len(p)) for p in paths]))
    for s, path in zip(seqs, paths):
        pool.truncate(s, length + len(path))
    # compaction moves pages under the sequences
    extra = pool.open()
    pool.extend(extra, 5 * page)
    hold = pool.fork(extra)
    pool.free(extra)
    pool.free(hold)
    moves, used = pool.compact()
    assert used + pool.free_pages() == 64
    if moves:
        cache.copy_pages(i32([list(m) for m in moves]))
    assert all(p < used for s in seqs for p in pool.pages_of(s))
    # one more token each, by plain decode
    for s in seqs:
        pair = pool.extend(s, 1)
        assert pair is None
    nq, nk, nv = rows(2)
    ends = [length + len(p) for p in paths]
    slots = torch.cat([pool.slots(s, e, 1) for s, e in zip(seqs, ends)])
    for layer in range(layers):
        tq = plan.apply_to_cache(nq, nk, nv, i32(ends), cache, slots, layer=layer)
    for layer in range(layers):
        got = ops.tree_attention(tq, cache, pool.tables(seqs), i32(ends), i32([0, 1, 2]), masks([1, 1]), layer=layer)
        for s, path in enumerate(paths):
            row_k = torch.cat([k, drafts[s][1][path], nk[s:s + 1]])
            row_v = torch.cat([v, drafts[s][2][path], nv[s:s + 1]])
            tk = plan.apply(row_k, row_k, position(0, ends[s] + 1))[1]
            seen = torch.ones(1, ends[s] + 1, dtype=torch.bool, device="cuda")
            check_heads(got[s:s + 1], tq[s:s + 1], tk, row_v, seen, dim ** -0.5, dtype)


# ---------------------------------------------------------------------- refusals

def test_refusals_launch_nothing():
    q = torch.zeros(4, 2, 64, device="cuda")
    k = torch.zeros(4, 1, 64, device="cuda")
    with pytest.raises(ops.OperatorError, match="another type"):
        ops.prompt_attention(q, k.half(), k.half(), i32([0, 4]))
    with pytest.raises(ops.OperatorError, match="offsets"):
        ops.prompt_attention(q, k, k, torch.tensor([0, 4], device="cuda"))
    with pytest.raises(ops.OperatorError, match="head_dim must be"):
        ops.prompt_attention(q[..., :32], k[..., :32], k[..., :32], i32([0, 4]))
    with pytest.raises(ops.OperatorError, match="aligned") as e:
        wide = torch.zeros(4, 2, 66, device="cuda")
        ops.prompt_attention(wide[..., 1:65], k, k, i32([0, 4]))
    assert e.value.status == 5
    with pytest.raises(ops.OperatorError, match="multiple of kv_heads"):
        ops.prompt_attention(torch.zeros(4, 3, 64, device="cuda"), torch.zeros(4, 2, 64, device="cuda"),
                             torch.zeros(4, 2, 64, device="cuda"), i32([0, 4]))
    with pytest.raises(ops.OperatorError, match="scale"):
        ops.prompt_attention(q, k, k, i32([0, 4]), scale=NAN)
    with pytest.raises(ops.OperatorError, match="kv_offsets"):
        ops.prompt_attention(q, k[:3], k[:3], i32([0, 4]))
    cache = ops.PageCache.empty(1, 4, 1, 16, 64, torch.float32)
    args = (i32([[0, 1]]), i32([9]), i32([0, 1]), masks([1]))
    with pytest.raises(ops.OperatorError, match="workspace"):
        ops.tree_attention(q[:1], cache, *args, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ops.OperatorError, match="layer"):
        ops.tree_attention(q[:1], cache, *args, layer=1)
    with pytest.raises(ops.OperatorError, match="another type"):
        ops.tree_attention(q[:1].half(), cache, *args)
    with pytest.raises(ops.OperatorError, match="contiguous"):
        ops.PageCache(cache.k.transpose(2, 3), cache.v.transpose(2, 3))
    with pytest.raises(ops.OperatorError, match="strides"):
        stack = torch.zeros(4, 6, 64, device="cuda")
        ops.Rotary(64).apply(stack[:, :2], stack[:, 2:3], i32([0, 1, 2, 3]), q_out=stack.view(-1)[:512].view(4, 2, 64))
    assert ops.prompt_attention(q[:0], k[:0], k[:0], i32([0, 0])).shape == (0, 2, 64)


def test_tensors_that_ask_for_gradients_are_refused_and_the_status_is_clean():
    q = torch.zeros(4, 2, 64, device="cuda", requires_grad=True)
    k = torch.zeros(4, 2, 64, device="cuda")
    with pytest.raises(ops.OperatorError, match="gradient"):
        ops.prompt_attention(q, k, k, i32([0, 4]))
    with torch.no_grad():
        assert not ops.prompt_attention(q, k, k, i32([0, 4])).any()
    ops.attention_status()
    ops.attention_status("cuda:0")


def test_caches_that_ask_for_gradients_are_refused_by_every_call():
    cache = ops.PageCache.empty(1, 4, 1, 16, 64, torch.float32)
    cache.k.zero_()
    cache.v.zero_()
    q, k = torch.zeros(1, 2, 64, device="cuda"), torch.zeros(1, 1, 64, device="cuda")
    one, plan = i32([1]), ops.Rotary(64)
    calls = [lambda: ops.tree_attention(q, cache, i32([[0, 1]]), i32([9]), i32([0, 1]), masks([1])),
             lambda: plan.apply_to_cache(q, k, k, one, cache, one),
             lambda: cache.copy_pages(i32([[0, 1]])),
             lambda: cache.keep(i32([[0, 1]]), i32([9]), one, i32([[1]]))]
    for side in (cache.k, cache.v):
        side.requires_grad_()
        for call in calls:
            with pytest.raises(ops.OperatorError, match="the cache asks for a gradient"):
                call()
            with torch.no_grad():
                call()
        side.requires_grad_(False)
    for call in calls:
        call()


def test_a_backward_pass_learns_that_a_tensor_it_saved_was_written():
    g = gen(60)
    q, k, one = normal(g, 1, 2, 64), normal(g, 1, 2, 64), i32([1])
    cache = ops.PageCache(normal(g, 1, 4, 2, 16, 64), normal(g, 1, 4, 2, 16, 64))
    plan, tree = ops.Rotary(64), (i32([[0, 1]]), i32([9]), i32([0, 1]), masks([1]))
    calls = [(q, lambda: plan.apply(q, k, one, q_out=q)), (k, lambda: plan.apply(q, k, one, k_out=k)),
             (q, lambda: plan.apply_to_cache(q, k, k, one, cache, one, q_out=q)),
             (cache.k, lambda: plan.apply_to_cache(q, k, k, one, cache, one)),
             (cache.v, lambda: plan.apply_to_cache(q, k, k, one, cache, one)),
             (cache.k, lambda: cache.copy_pages(i32([[0, 1]]))), (cache.v, lambda: cache.copy_pages(i32([[0, 1]]))),
             (cache.k, lambda: cache.keep(tree[0], tree[1], one, i32([[1]]))),
             (cache.v, lambda: cache.keep(tree[0], tree[1], one, i32([[1]]))),
             (q, lambda: ops.prompt_attention(k, k, k, i32([0, 1]), out=q)),
             (q, lambda: ops.tree_attention(k, cache, *tree, out=q))]
    for saved, call in calls:
        w = torch.ones(64, device="cuda", requires_grad=True)
        y = (saved * w).sum()
        y.backward(retain_graph=True)
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    # what is only read keeps its version, and tensors of the inference mode have none
    before = [t._version for t in (q, k, cache.k, cache.v)]
    ops.prompt_attention(q, k, k, i32([0, 1]))
    ops.tree_attention(q, cache, *tree)
    plan.apply(q, k, one)
    assert before == [t._version for t in (q, k, cache.k, cache.v)]
    with torch.inference_mode():
        q, k = normal(g, 1, 2, 64), normal(g, 1, 2, 64)
        cache = ops.PageCache.empty(1, 4, 2, 16, 64, torch.float32)
        assert plan.apply_to_cache(q, k, k, one, cache, one, q_out=q) is q
        cache.copy_pages(i32([[0, 1]]))


def test_layers_past_32_bits_are_refused_not_cut():
    q, k, one = torch.zeros(1, 2, 64, device="cuda"), torch.zeros(1, 1, 64, device="cuda"), i32([1])
    cache = ops.PageCache.empty(1, 4, 1, 16, 64, torch.float32)
    for layer in (1 << 32, -1):
        with pytest.raises(ops.OperatorError, match="layer"):
            ops.tree_attention(q, cache, i32([[0, 1]]), i32([9]), i32([0, 1]), masks([1]), layer=layer)
        with pytest.raises(ops.OperatorError, match="layer"):
            ops.Rotary(64).apply_to_cache(q, k, k, one, cache, one, layer=layer)
