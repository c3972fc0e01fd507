"""Cases of the paged-serving operators: rotary positions, attention over packed
prompts, attention of drafted token trees over a paged cache, and the cache's page
copies and draft compaction.

`run` computes a case in plain torch operations (`own` false) or through
promptboot_b200.ops (`own` true); `exact` restates the definition in binary64.
Shapes follow the model the engine decodes (14 query heads and 2 key/value heads
of 64) and a generic wider one (32 and 8 heads of 128).
"""
import functools
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One decode step of 32 sequences: rotate q and k, write k and v to their pages.
        dict(name="rotary step of 32", op="rotary", type="bf16", rows=32, q_heads=14, kv_heads=2, dim=64,
             rotary=64, interleaved=False, scaling="yarn", reach=131072, pages=512, page=16, mix=1),
        # A packed batch of prompts of a wider model, half of each head rotated, adjacent pairs.
        dict(name="rotary prompts 16421", op="rotary", type="f16", rows=16421, q_heads=32, kv_heads=8, dim=128,
             rotary=64, interleaved=True, scaling="bands", reach=131072, pages=0, page=0, mix=2),
        # Three chat turns that arrive together, in the engine's own precision: latency of the smallest prefill.
        dict(name="prompts 3 short", op="prompt", type="f32", seqs=3, tokens=131, prefix=0, q_heads=14, kv_heads=2,
             dim=64, mix=3),
        # A prefill batch of ragged prompts, some with a cached prefix before them.
        dict(name="prompts 24 ragged", op="prompt", type="f16", seqs=24, tokens=12345, prefix=256, q_heads=32,
             kv_heads=8, dim=128, mix=5),
        # One long document.
        dict(name="prompt 16384", op="prompt", type="bf16", seqs=1, tokens=16384, prefix=0, q_heads=14, kv_heads=2,
             dim=64, mix=6),
        # Batched decode without drafts: 256 sequences half way through 512..1535 positions.
        dict(name="tree 256 single tokens", op="tree", type="bf16", seqs=256, least=512, most=1535, nodes=1,
             q_heads=14, kv_heads=2, dim=64, page=16, mix=7),
        # Long-context speculative decoding: 8 sequences near the end of 32768 positions, up to 48 drafts each.
        dict(name="tree 8 long contexts", op="tree", type="bf16", seqs=8, least=30000, most=32700, nodes=48,
             q_heads=14, kv_heads=2, dim=64, page=64, mix=8),
        # Small drafts over a wider model's cache.
        dict(name="tree 16 wide heads", op="tree", type="f16", seqs=16, least=700, most=9000, nodes=12, q_heads=32,
             kv_heads=8, dim=128, page=32, mix=9),
        # A beam step: eight sequences fork, each copies its partly filled last page in all 24 layers.
        dict(name="copy 8 pages", op="copy", type="bf16", layers=24, pages=64, copies=8, kv_heads=2, dim=64,
             page=16, mix=10),
        # Compaction of a busy pool: pages move to the front so that its tail can be given back.
        dict(name="copy 1000 pages", op="copy", type="bf16", layers=24, pages=2100, copies=1000, kv_heads=2, dim=64,
             page=32, mix=11),
        # One sequence keeps the accepted path of its draft tree.
        dict(name="keep 1 path", op="keep", type="bf16", layers=24, seqs=1, most=300, nodes=48, q_heads=14,
             kv_heads=2, dim=64, page=16, mix=12),
        # 128 sequences keep theirs in one call.
        dict(name="keep 128 paths", op="keep", type="f32", layers=24, seqs=128, most=500, nodes=40, q_heads=14,
             kv_heads=2, dim=64, page=32, mix=13),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotary", "prompt", "prompt", "tree", "tree", "copy", "keep"])
    case = dict(op=op, type=rng.choice(["f32", "f16", "bf16", "bf16"]), mix=rng.randrange(1 << 20))
    case["q_heads"], case["kv_heads"], case["dim"] = rng.choice(
        [(14, 2, 64), (14, 2, 64), (32, 8, 128), (8, 8, 64), (12, 4, 128), (16, 1, 64)])
    page = rng.choice([16, 32, 64, 128])
    if op == "rotary":
        dim = case["dim"]
        case.update(rows=_log(rng, 1, 12000), rotary=rng.choice([dim, dim, dim // 2, dim // 4]),
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "yarn", "bands"]),
                    reach=_log(rng, 2048, 1000000), pages=0, page=0)
        if rng.random() < 0.5:
            case.update(pages=(case["rows"] + 8 * page) // page + 3, page=page)
    elif op == "prompt":
        seqs = _log(rng, 1, 48)
        most = 2500 if case["type"] == "f32" else 9000
        case.update(seqs=seqs, tokens=max(seqs, _log(rng, 24, most)), prefix=rng.choice([0, 0, 100, 900]))
    elif op == "tree":
        seqs, least = _log(rng, 1, 256), _log(rng, 1, 8000)
        row = 2 * case["kv_heads"] * case["dim"] * DTYPES[case["type"]].itemsize
        most = max(least, min(32000, 2 * least, 200_000_000 // (row * seqs)))
        least = min(least, most)
        case.update(seqs=seqs, least=least, most=most, nodes=rng.choice([1, 1, _log(rng, 2, 64)]), page=page)
        if case["type"] == "f32":
            case["nodes"] = min(case["nodes"], 8)
    elif op == "copy":
        copies = _log(rng, 1, 500)
        case.update(layers=rng.choice([1, 12, 24]), pages=2 * copies + rng.randrange(40), copies=copies, page=16)
    else:
        case.update(layers=rng.choice([1, 12, 24]), seqs=_log(rng, 1, 64), most=_log(rng, 20, 400),
                    nodes=rng.randrange(2, 65), page=16)
    return case


# ---------------------------------------------------------------- what a case holds

def _split(case):
    """Tokens of each packed prompt: every sequence has one at least, the rest by random shares."""
    r = random.Random(case["mix"])
    n = case["seqs"]
    share = [r.random() + 0.05 for _ in range(n)]
    rest = case["tokens"] - n
    got = [1 + int(rest * s / sum(share)) for s in share]
    got[-1] += case["tokens"] - sum(got)
    before = [r.randrange(case["prefix"] + 1) if case["prefix"] else 0 for _ in range(n)]
    return got, before


def _contexts(case):
    """Context length and node count of each drafting sequence."""
    r = random.Random(case["mix"])
    least = case.get("least", 1)
    pairs = [(r.randrange(least, case["most"] + 1), case["nodes"] if k == 0 else r.randrange(1 + case["nodes"] // 2, case["nodes"] + 1))
             for k in range(case["seqs"])]
    return [c for c, _ in pairs], [t for _, t in pairs]


def _accepted(case):
    """The accepted node indices of each sequence's tree: an ascending path, seldom whole."""
    r = random.Random(case["mix"] + 1)
    _, nodes = _contexts(case)
    paths = []
    for t in nodes:
        path, at = [], 0
        while at < t and len(path) < 16:
            path.append(at)
            at += 1 + r.randrange(6)
        paths.append(path)
    return paths


def _yarn_span(case, theta):
    def place(turns):
        return case["rotary"] * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(theta))
    low, high = max(math.floor(place(32.0)), 0), min(math.ceil(place(1.0)), case["rotary"] - 1)
    return float(low), float(high) if high > low else low + 0.001


def _scaling(case):
    """(theta, factor, original context) of a rotary case."""
    return {"none": (1e6, 1.0, 32768), "linear": (1e4, 4.0, 32768), "yarn": (1e6, 4.0, 32768),
            "bands": (5e5, 8.0, 8192)}[case["scaling"]]


def _frequencies(case):
    """Angle per position of each rotated pair, and the factor on cosine and sine."""
    theta, factor, original = _scaling(case)
    half = case["rotary"] // 2
    freq = theta ** (-torch.arange(half, dtype=torch.float64) / half)
    if case["scaling"] == "linear":
        return freq / factor, 1.0
    if case["scaling"] == "yarn":
        low, high = _yarn_span(case, theta)
        ramp = ((torch.arange(half, dtype=torch.float64) - low) / (high - low)).clamp(0, 1)
        return freq / factor * ramp + freq * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if case["scaling"] == "bands":
        turns = original * freq / (2 * math.pi)
        smooth = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return freq / factor * (1 - smooth) + freq * smooth, 1.0
    return freq, 1.0


def _starts(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return at


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(case, tokens, gen):
    """Page ids of each sequence, scattered over the pool; a row's unused ids repeat its last."""
    page = case["page"]
    need = [-(-t // page) for t in tokens]
    pool = sum(need) + 5
    ids = torch.randperm(pool, generator=gen, device="cuda", dtype=torch.int32)
    start = torch.tensor(_starts(need), device="cuda")
    at = torch.arange(max(need), device="cuda")[None, :].minimum(torch.tensor(need, device="cuda")[:, None] - 1)
    return ids[start[:-1, None] + at].contiguous(), pool


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    def cache(layers, pages):
        shape = (layers, pages, case["kv_heads"], case["page"], case["dim"])
        return normal(*shape), normal(*shape)

    state = dict(case=case)
    if case["op"] == "rotary":
        rows, dim = case["rows"], case["dim"]
        state["q"] = normal(rows, case["q_heads"], dim)
        state["k"] = normal(rows, case["kv_heads"], dim)
        state["positions"] = torch.randint(0, case["reach"], (rows,), generator=gen, device="cuda", dtype=torch.int32)
        freq, state["magnitude"] = _frequencies(case)
        state["frequencies"] = freq.cuda()
        if case["pages"]:
            state["v"] = normal(rows, case["kv_heads"], dim)
            state["cache_k"], state["cache_v"] = cache(1, case["pages"])
            slots = torch.randperm(case["pages"] * case["page"], generator=gen, device="cuda", dtype=torch.int32)
            state["slots"] = slots[:rows].contiguous()
    elif case["op"] == "prompt":
        tokens, before = _split(case)
        keys = [t + b for t, b in zip(tokens, before)]
        state["q"] = normal(sum(tokens), case["q_heads"], case["dim"], scale=1.5)
        state["k"] = normal(sum(keys), case["kv_heads"], case["dim"])
        state["v"] = normal(sum(keys), case["kv_heads"], case["dim"])
        state["offsets"], state["kv_offsets"] = _i32(_starts(tokens)), _i32(_starts(keys))
        state["longest"], state["longest_kv"] = max(tokens), max(keys)
    elif case["op"] == "tree":
        contexts, nodes = _contexts(case)
        state["tables"], pool = _tables(case, [c + t for c, t in zip(contexts, nodes)], gen)
        state["cache_k"], state["cache_v"] = cache(1, pool)
        state["q"] = normal(sum(nodes), case["q_heads"], case["dim"], scale=1.5)
        state["contexts"], state["offsets"] = _i32(contexts), _i32(_starts(nodes))
        state["longest"], state["most_nodes"] = max(c + t for c, t in zip(contexts, nodes)), max(nodes)
        r, visible = random.Random(seed), []
        for t in nodes:
            own_bits = []
            for i in range(t):
                parent = r.randrange(max(0, i - 6), i) if i and r.random() < 0.9 else -1
                own_bits.append((own_bits[parent] if parent >= 0 else 0) | 1 << i)
            visible += own_bits
        state["visible"] = torch.tensor([b - (1 << 64) if b >> 63 else b for b in visible], device="cuda")
    elif case["op"] == "copy":
        state["cache_k"], state["cache_v"] = cache(case["layers"], case["pages"])
        ids = torch.randperm(case["pages"], generator=gen, device="cuda", dtype=torch.int32)
        state["pairs"] = ids[:2 * case["copies"]].reshape(2, -1).t().contiguous()
    else:
        contexts, nodes = _contexts(case)
        paths = _accepted(case)
        state["tables"], pool = _tables(case, [c + t for c, t in zip(contexts, nodes)], gen)
        state["cache_k"], state["cache_v"] = cache(case["layers"], pool)
        width = max(len(p) for p in paths)
        state["contexts"], state["counts"] = _i32(contexts), _i32([len(p) for p in paths])
        state["nodes"] = _i32([p + [0] * (width - len(p)) for p in paths])
    return state


# ---------------------------------------------------------------- the plain forms

def _plain_rotary(state):
    case, half = state["case"], state["case"]["rotary"] // 2
    angle = state["positions"].double()[:, None] * state["frequencies"]
    cos = (angle.cos() * state["magnitude"]).float()[:, None]
    sin = (angle.sin() * state["magnitude"]).float()[:, None]

    def turned(x):
        y = x.float().clone()
        part = x[..., :2 * half].float()
        if case["interleaved"]:
            a, b = part[..., 0::2], part[..., 1::2]
            y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * cos - b * sin, b * cos + a * sin
        else:
            a, b = part[..., :half], part[..., half:]
            y[..., :half], y[..., half:2 * half] = a * cos - b * sin, b * cos + a * sin
        return y.to(x.dtype)

    q, k = turned(state["q"]), turned(state["k"])
    if not case["pages"]:
        return q, k
    slot = state["slots"].long()
    at = (slot // case["page"], slice(None), slot % case["page"])
    state["cache_k"][0][at] = k
    state["cache_v"][0][at] = state["v"]
    return q, state["cache_k"], state["cache_v"]


def _attend(q, k, v, seen):
    """q [n, g*t, d], k and v [n, l, d], seen [n, g*t, l]: rows that see nothing are zero."""
    s = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(q.shape[-1]))
    s = s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top.isfinite(), top, 0.0)).exp_()
    return (p @ v) / p.sum(-1, keepdim=True).clamp_min(1e-37)


def _padded(starts, longest, rows):
    """Row index of each (sequence, place) and whether the place holds one."""
    at = torch.arange(longest, device="cuda")
    there = at[None, :] < (starts[1:] - starts[:-1])[:, None]
    return (starts[:-1, None] + at[None, :]).clamp_max(rows - 1).long(), there


def _packed(out, starts, rows):
    """The packed rows [rows, heads, dim] of out [n, kv_heads, group, t, dim]."""
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(starts[1:], row, right=True, out_int32=True)
    return out.permute(0, 3, 1, 2, 4)[seq, row - starts[seq]].reshape(rows, -1, out.shape[-1])


def _plain_prompt(state):
    q, k, v = state["q"], state["k"], state["v"]
    rows, heads, dim = q.shape
    kv_heads = k.shape[1]
    group = heads // kv_heads
    at, there = _padded(state["offsets"], state["longest"], rows)
    kv_at, kv_there = _padded(state["kv_offsets"], state["longest_kv"], k.shape[0])
    n, t, l = at.shape[0], at.shape[1], kv_at.shape[1]
    qs = q[at].float().view(n, t, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n * kv_heads, group * t, dim)
    ks = k[kv_at].float().transpose(1, 2).reshape(n * kv_heads, l, dim)
    vs = v[kv_at].float().transpose(1, 2).reshape(n * kv_heads, l, dim)
    behind = (kv_there.sum(1) - there.sum(1))[:, None, None]
    seen = torch.arange(l, device="cuda")[None, None, :] <= torch.arange(t, device="cuda")[None, :, None] + behind
    seen = seen & kv_there[:, None, :]
    seen = seen[:, None, None].expand(n, kv_heads, group, t, l).reshape(n * kv_heads, group * t, l)
    out = _attend(qs, ks, vs, seen).view(n, kv_heads, group, t, dim)
    return _packed(out, state["offsets"], rows).to(q.dtype)


def _plain_tree(state):
    q, tables = state["q"], state["tables"].long()
    rows, heads, dim = q.shape
    kv_heads = state["cache_k"].shape[2]
    group = heads // kv_heads
    at, there = _padded(state["offsets"], state["most_nodes"], rows)
    n, t = at.shape
    qs = q[at].float().view(n, t, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n * kv_heads, group * t, dim)
    ks = state["cache_k"][0][tables].float().transpose(1, 2).reshape(n * kv_heads, -1, dim)
    vs = state["cache_v"][0][tables].float().transpose(1, 2).reshape(n * kv_heads, -1, dim)
    node = torch.arange(ks.shape[1], device="cuda")[None, :] - state["contexts"][:, None]
    bit = (state["visible"][at][:, :, None] >> node.clamp(0, 63)[:, None, :]) & 1
    seen = (node < 0)[:, None, :] | ((node < 64)[:, None, :] & (bit == 1))
    seen = seen & (node < there.sum(1)[:, None])[:, None, :]
    seen = seen[:, None, None].expand(n, kv_heads, group, t, -1).reshape(n * kv_heads, group * t, -1)
    out = _attend(qs, ks, vs, seen).view(n, kv_heads, group, t, dim)
    return _packed(out, state["offsets"], rows).to(q.dtype)


def _plain_copy(state):
    source, target = state["pairs"].long().unbind(1)
    state["cache_k"][:, target] = state["cache_k"][:, source]
    state["cache_v"][:, target] = state["cache_v"][:, source]
    return state["cache_k"], state["cache_v"]


def _plain_keep(state):
    page = state["case"]["page"]
    place = torch.arange(state["nodes"].shape[1], device="cuda")[None, :]
    held = place < state["counts"][:, None]
    target = (state["contexts"][:, None] + place).clamp_max(state["tables"].shape[1] * page - 1)
    source = torch.where(held, state["contexts"][:, None] + state["nodes"], target)

    def spot(position):
        return state["tables"].gather(1, position // page).long(), slice(None), position % page

    for name in ("cache_k", "cache_v"):
        state[name][(slice(None),) + spot(target)] = state[name][(slice(None),) + spot(source)]
    return state["cache_k"], state["cache_v"]


# ---------------------------------------------------------------- one pass

@functools.lru_cache(maxsize=None)
def _rotary_plan(dim, rotary, interleaved, scaling, theta, factor, original):
    """The program's one rotary plan for its model."""
    from promptboot_b200 import ops
    return ops.Rotary(dim, rotary_dim=rotary, theta=theta, interleaved=interleaved, scaling=scaling, factor=factor,
                      original_context=original)


def run(state):
    case, op = state["case"], state["case"]["op"]
    if not own:
        return {"rotary": _plain_rotary, "prompt": _plain_prompt, "tree": _plain_tree, "copy": _plain_copy,
                "keep": _plain_keep}[op](state)
    from promptboot_b200 import ops
    if op == "prompt":
        return ops.prompt_attention(state["q"], state["k"], state["v"], state["offsets"],
                                    kv_offsets=state["kv_offsets"])
    if op == "rotary":
        plan = _rotary_plan(case["dim"], case["rotary"], case["interleaved"], case["scaling"], *_scaling(case))
        if not case["pages"]:
            return plan.apply(state["q"], state["k"], state["positions"])
        cache = ops.PageCache(state["cache_k"], state["cache_v"])
        q = plan.apply_to_cache(state["q"], state["k"], state["v"], state["positions"], cache, state["slots"])
        return q, state["cache_k"], state["cache_v"]
    cache = ops.PageCache(state["cache_k"], state["cache_v"])
    if op == "tree":
        return ops.tree_attention(state["q"], cache, state["tables"], state["contexts"], state["offsets"],
                                  state["visible"])
    if op == "copy":
        cache.copy_pages(state["pairs"])
    else:
        cache.keep(state["tables"], state["contexts"], state["counts"], state["nodes"])
    return state["cache_k"], state["cache_v"]


def work(case):
    size = DTYPES[case["type"]].itemsize
    row, kv_row = case["kv_heads"] * case["dim"] * size, 2 * case["kv_heads"] * case["dim"] * size
    q_row = case.get("q_heads", 0) * case["dim"] * size
    if case["op"] == "rotary":
        # q in and out, k in and out, and v in and out where it goes to the cache
        held = case["rows"] * (2 * q_row + 2 * row + (2 * row + 4 if case["pages"] else 0) + 4)
        return {"bytes": held, "flops": 3 * case["rows"] * (case["q_heads"] + case["kv_heads"]) * case["rotary"]}
    if case["op"] == "prompt":
        tokens, before = _split(case)
        pairs = sum(t * b + t * (t + 1) // 2 for t, b in zip(tokens, before))
        return {"bytes": 2 * sum(tokens) * q_row + sum(map(sum, zip(tokens, before))) * kv_row,
                "flops": 4 * case["dim"] * case["q_heads"] * pairs}
    if case["op"] == "tree":
        contexts, nodes = _contexts(case)
        pairs = sum(t * (c + (t + 1) / 2) for c, t in zip(contexts, nodes))
        return {"bytes": sum(map(sum, zip(contexts, nodes))) * kv_row + 2 * sum(nodes) * q_row,
                "flops": 4 * case["dim"] * case["q_heads"] * pairs}
    if case["op"] == "copy":
        return {"bytes": 2 * case["copies"] * case["layers"] * case["page"] * kv_row, "flops": 0}
    moved = sum(sum(n != i for i, n in enumerate(p)) for p in _accepted(case))
    return {"bytes": 2 * max(1, moved) * case["layers"] * kv_row, "flops": 0}


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_rotary(case, state):
    freq, magnitude = _frequencies(case)
    angle = torch.outer(state["positions"].double(), freq.cuda())
    turn = torch.polar(torch.full_like(angle, magnitude), angle)[:, None, :]
    half = case["rotary"] // 2

    def turned(x):
        x = x.double()
        head, rest = x[..., :2 * half], x[..., 2 * half:]
        shape = (half, 2) if case["interleaved"] else (2, half)
        pairs = head.unflatten(-1, shape)
        pairs = pairs if case["interleaved"] else pairs.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z if case["interleaved"] else z.transpose(-1, -2)
        return torch.cat([z.flatten(-2), rest], -1)

    q, k = turned(state["q"]), turned(state["k"])
    if not case["pages"]:
        return q, k
    ck, cv = state["cache_k"].double(), state["cache_v"].double()
    for into, rows in ((ck, k), (cv, state["v"].double())):
        flat = into[0].transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])
        flat = flat.index_copy(0, state["slots"].long(), rows)
        into[0] = flat.view(case["pages"], case["page"], case["kv_heads"], case["dim"]).transpose(1, 2)
    return q, ck, cv


def _exact_rows(q, k, v, seen):
    """q [t, d], k and v [l, d], seen [t, l] of one head."""
    s = (q.double() @ k.double().t()) / math.sqrt(q.shape[-1])
    return torch.softmax(s.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0) @ v.double()


def _exact_prompt(case, state):
    tokens, before = _split(case)
    q, k, v = state["q"], state["k"], state["v"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    group, at, kv_at = case["q_heads"] // case["kv_heads"], 0, 0
    for t, b in zip(tokens, before):
        seen = torch.ones(t, t + b, dtype=torch.bool, device="cuda").tril(b)
        for h in range(case["q_heads"]):
            keys = slice(kv_at, kv_at + t + b), h // group
            out[at:at + t, h] = _exact_rows(q[at:at + t, h], k[keys], v[keys], seen)
        at, kv_at = at + t, kv_at + t + b
    return out


def _exact_tree(case, state):
    contexts, nodes = _contexts(case)
    q, page, at = state["q"], case["page"], 0
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    group = case["q_heads"] // case["kv_heads"]
    for i, (c, t) in enumerate(zip(contexts, nodes)):
        ids = state["tables"][i, :-(-(c + t) // page)].long()
        seen = torch.ones(t, c + t, dtype=torch.bool, device="cuda")
        bits = state["visible"][at:at + t]
        seen[:, c:] = torch.stack([(bits >> j) & 1 for j in range(t)], 1) == 1
        for h in range(case["kv_heads"]):
            k = state["cache_k"][0, ids, h].reshape(-1, case["dim"])[:c + t]
            v = state["cache_v"][0, ids, h].reshape(-1, case["dim"])[:c + t]
            rows = q[at:at + t, h * group:(h + 1) * group].reshape(t * group, -1)
            got = _exact_rows(rows, k, v, seen.repeat_interleave(group, 0))
            out[at:at + t, h * group:(h + 1) * group] = got.view(t, group, -1)
        at += t
    return out


def _exact_moves(case, state):
    """(page, slot) pairs that a copy or a compaction moves, from a host's view of it."""
    if case["op"] == "copy":
        return None
    contexts, _ = _contexts(case)
    tables, page, moves = state["tables"].tolist(), case["page"], []
    for i, path in enumerate(_accepted(case)):
        for j, n in enumerate(path):
            a, b = contexts[i] + n, contexts[i] + j
            moves.append((tables[i][a // page], a % page, tables[i][b // page], b % page))
    return torch.tensor(moves).cuda().t()


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, state)
    if case["op"] == "prompt":
        return _exact_prompt(case, state)
    if case["op"] == "tree":
        return _exact_tree(case, state)
    moves, got = _exact_moves(case, state), []
    for x in (state["cache_k"], state["cache_v"]):
        y = x.double()
        if moves is None:
            pairs = state["pairs"].tolist()
            y[:, [b for _, b in pairs]] = x.double()[:, [a for a, _ in pairs]]
        else:
            y[:, moves[2], :, moves[3]] = x.double()[:, moves[0], :, moves[1]]
        got.append(y)
    return tuple(got)
