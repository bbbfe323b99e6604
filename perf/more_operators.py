"""A verify round of a model with sliding-window layers, as cases that can be timed and compared.

Three operators: the rotation of Q and K from positions and frequencies with the K/V scatter, the packed
tree attention that sees a window of its past and a few first tokens, and the log probabilities of given
tokens with the entropy and the top alternatives of their rows.  Each case is one call.  ``run`` computes
it either in elementary torch operations or, where ``own`` is set, by the package's public entry point;
both take the tensors that a serving program has in hand before the call.
"""
import math
import os
import random
import sys
from types import SimpleNamespace

import numpy as np
import torch

own = False

_DEVICE = "cuda"
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _package():
    where = os.path.join(os.getcwd(), "nano-vllm-jetspec_amd")
    if where not in sys.path:
        sys.path.insert(0, where)
    import jetspec_amd

    return jetspec_amd


# --------------------------------------------------------------------------- cases
def _window(**kw):
    case = {"kind": "window", "dtype": "bf16", "out32": False, "kv_heads": 8, "groups": 4, "head_dim": 128, "page": 256,
            "requests": 1, "prefix_lo": 0, "prefix_hi": 0, "tree_lo": 1, "tree_hi": 1, "chain": False, "window": 1024,
            "sinks": 4, "evicted": True, "gain": 1.0, "layout": 0}
    case.update(kw)
    return case


def _rotary(**kw):
    case = {"kind": "rotary", "dtype": "bf16", "rows": 16, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "turned": 128,
            "interleaved": False, "factor": 1.0, "page": 256, "length": 32768, "layout": 0}
    case.update(kw)
    return case


def _logprobs(**kw):
    case = {"kind": "logprobs", "dtype": "bf16", "held": 0, "rows": 8, "vocab": 151936, "tokens": 1, "top": 5, "masked": 0.0,
            "gain": 2.5, "layout": 0}
    case.update(kw)
    return case


def listed():
    return [
        # One interactive request decoding a single token far past its window: latency.
        _window(name="window_one_token", prefix_lo=9001, prefix_hi=9001, layout=1),
        # A small serving batch: ragged contexts on both sides of the window, trees of 16 to 64 drafted tokens.
        _window(name="window_trees_c8", requests=8, prefix_lo=256, prefix_hi=16384, tree_lo=16, tree_hi=64, window=4096,
                layout=2),
        # A full batch of trees at long contexts, the largest attention.
        _window(name="window_trees_c64_long", requests=64, prefix_lo=8192, prefix_hi=32768, tree_lo=64, tree_hi=64,
                window=8192, sinks=16, layout=3),
        # A full batch of single tokens: the cache's bytes are what counts.
        _window(name="window_decode_c128", requests=128, prefix_lo=2048, prefix_hi=32768, window=4096, layout=4),
        # Prefill chunks longer than the window, over what came before.
        _window(name="window_chunks", requests=8, prefix_lo=0, prefix_hi=8192, tree_lo=1024, tree_hi=1024, chain=True,
                window=512, sinks=0, gain=2.0, layout=5),
        # A tensor-parallel shard with one KV head in f16, FP32 results, head size 64, small pages, nothing evicted.
        _window(name="window_shard_f16", dtype="f16", out32=True, requests=32, kv_heads=1, groups=8, head_dim=64, page=16,
                prefix_lo=500, prefix_hi=8192, tree_lo=5, tree_hi=33, window=777, sinks=1, evicted=False, gain=3.0,
                layout=6),
        # One request's tree, one layer: a launch among thousands.
        _rotary(name="rotary_one_tree", rows=16, layout=7),
        # A full batch of trees, interleaved pairs on half of the head, at positions past the trained length.
        _rotary(name="rotary_c64_part", rows=4096, turned=64, interleaved=True, factor=8.0, length=262144, layout=8),
        # A prefill batch in fp32, a head size and a part that are no powers of two.
        _rotary(name="rotary_prefill_f32", dtype="f32", rows=6001, q_heads=10, kv_heads=5, head_dim=80, turned=40, page=48,
                layout=9),
        # The answers of a decode batch: one emitted token a request and its alternatives.
        _logprobs(name="logprobs_decode", rows=8, top=5, layout=10),
        # Every node of a full batch of trees: the largest.
        _logprobs(name="logprobs_trees_c64", rows=4096, top=20, layout=11),
        # The accepted rows of a smaller model's batch in fp32, a vocabulary of no round size with forbidden words, the
        # children of each node as its given tokens.
        _logprobs(name="logprobs_accepted_f32", dtype="f32", held=1024, rows=333, vocab=50257, tokens=4, top=0, masked=0.3,
                  layout=12),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    layout = rng.randrange(1, 1 << 30)
    kind = rng.choice(["decode", "decode", "trees", "trees", "long", "chunks", "chunks", "rotary", "rotary", "rotary",
                       "logprobs", "logprobs", "logprobs"])
    if kind in ("decode", "trees", "long", "chunks"):
        types = {"dtype": rng.choice(["bf16", "bf16", "f16"]), "gain": rng.choice([1.0, 2.0, 3.0]),
                 "head_dim": rng.choice([64, 80, 96, 128, 128, 128, 256]), "page": rng.choice([16, 48, 128, 256]),
                 "window": _log(rng, 1, 8192), "sinks": rng.choice([0, 1, 4, 4, 16, 100]), "layout": layout,
                 "evicted": rng.random() < 0.6, "out32": rng.random() < 0.25}
        heads = rng.choice([{"kv_heads": 8, "groups": 4}, {"kv_heads": 8, "groups": 5}, {"kv_heads": 1, "groups": 16},
                            {"kv_heads": 2, "groups": 8}, {"kv_heads": 4, "groups": 1}, {"kv_heads": 3, "groups": 7}])
        if kind == "decode":
            top = _log(rng, 2, 32768)
            return _window(requests=_log(rng, 1, 64 if types["head_dim"] <= 128 else 32), prefix_lo=rng.choice([0, top // 3]), prefix_hi=top, **heads, **types)
        if kind == "trees":
            top, tree = _log(rng, 33, 16384), _log(rng, 2, 200)
            return _window(requests=_log(rng, 1, 12), prefix_lo=top // 8, prefix_hi=top, tree_lo=max(1, tree // 4),
                           tree_hi=tree, **heads, **types)
        if kind == "long":
            top = _log(rng, 8192, 32768)
            types.update(head_dim=min(types["head_dim"], 128), out32=False)
            return _window(requests=_log(rng, 2, 48), prefix_lo=top // 4, prefix_hi=top, tree_lo=rng.randint(1, 16),
                           tree_hi=_log(rng, 16, 64), **types)
        types.update(head_dim=min(types["head_dim"], 128), window=min(types["window"], 2048))
        return _window(requests=_log(rng, 1, 6), prefix_lo=0, prefix_hi=_log(rng, 1, 8192), tree_lo=rng.randint(65, 500),
                       tree_hi=_log(rng, 500, 1500), chain=True, **heads, **types)
    if kind == "rotary":
        kv, dim = rng.choice([1, 2, 8, 5]), rng.choice([64, 80, 96, 128, 128, 256])
        return _rotary(dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), rows=_log(rng, 1, 9000), kv_heads=kv,
                       q_heads=kv * rng.choice([1, 4, 5, 8]), head_dim=dim,
                       turned=rng.choice([dim, dim, dim // 2, dim // 4, 6]), interleaved=rng.random() < 0.5,
                       factor=rng.choice([1.0, 4.0, 32.0]), page=rng.choice([16, 48, 256]), length=_log(rng, 512, 1 << 20),
                       layout=layout)
    vocab = rng.choice([151936, 50257, _log(rng, 2, 262144), _log(rng, 1000, 262144)])
    rows = _log(rng, 1, min(4096, 250000000 // vocab))
    return _logprobs(dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), rows=rows, held=rng.choice([0, 0, rows + rows // 2 + 1]),
                     vocab=vocab, tokens=rng.choice([1, 1, 3, 8]), top=min(vocab, rng.choice([0, 1, 5, 20, 64])),
                     masked=rng.choice([0.0, 0.0, 0.5]), gain=rng.choice([0.1, 1.0, 2.5, 6.0]), layout=layout)


# --------------------------------------------------------------------------- layouts (from the case alone)
def _between(rng, lo, hi, n):
    return rng.integers(lo, hi + 1, size=n)


def _trees(case):
    """Prefix lengths, tree sizes, parent arrays and depths of an attention case."""
    rng = np.random.default_rng(case["layout"])
    n = case["requests"]
    prefixes, sizes = _between(rng, case["prefix_lo"], case["prefix_hi"], n), _between(rng, case["tree_lo"], case["tree_hi"], n)
    parents, depths = [], []
    for size in sizes:
        if case["chain"]:
            parents.append(np.arange(-1, size - 1))
            depths.append(np.arange(size))
            continue
        depth, of = [0], [-1]
        for node in range(1, int(size)):
            fits = [j for j in range(node) if depth[j] < 8]
            up = fits[int(rng.integers(len(fits)))]
            of.append(up)
            depth.append(depth[up] + 1)
        parents.append(np.asarray(of))
        depths.append(np.asarray(depth))
    return prefixes, sizes, parents, depths


def _ancestors(parents):
    n = len(parents)
    if np.array_equal(parents, np.arange(-1, n - 1)):
        return np.tril(np.ones((n, n), dtype=bool))
    seen = np.zeros((n, n), dtype=bool)
    for node, up in enumerate(parents):
        if up >= 0:
            seen[node] = seen[up]
        seen[node, node] = True
    return seen


def _reach(prefix, depth, case):
    """Prefix keys below `sinks`, and from where on the rows at these depths see the others."""
    sinks = min(case["sinks"], prefix)
    return sinks, np.clip(prefix + depth - case["window"] + 1, sinks, prefix)


def _seen(prefix, parents, depth, case):
    """How many pairs of a row and a key there are, and the keys that some row sees: prefix keys, nodes."""
    sinks, start = _reach(prefix, depth, case)
    near = (depth[:, None] - depth[None, :] < case["window"]) | (prefix + depth[None, :] < case["sinks"])
    nodes = _ancestors(parents) & near
    return int((sinks + prefix - start).sum() + nodes.sum()), int(sinks + prefix - start.min()), int(nodes.any(0).sum())


# --------------------------------------------------------------------------- inputs
def _ints(values, kind=torch.int32):
    return torch.as_tensor(np.ascontiguousarray(values), dtype=kind, device=_DEVICE)


def _normal(gen, shape, dtype, gain=1.0):
    out = torch.empty(shape, dtype=dtype, device=_DEVICE)
    flat, step = out.view(-1), 1 << 28
    for at in range(0, flat.numel(), step):
        n = min(step, flat.numel() - at)
        flat[at:at + n] = torch.randn(n, generator=gen, device=_DEVICE) * gain
    return out


def _prepare_window(case, seed):
    gen = torch.Generator(device=_DEVICE).manual_seed(seed)
    rng = np.random.default_rng(seed)
    prefixes, sizes, parents, depths = _trees(case)
    page, heads, dim = case["page"], case["kv_heads"], case["head_dim"]
    counts = -(-prefixes // page)
    held = []   # pages of a request that are still in the pool: the window and the first tokens reach them
    for prefix, n in zip(prefixes, counts):
        at = np.arange(n)
        sinks, start = _reach(int(prefix), np.zeros(1, dtype=np.int64), case)
        held.append(at if not case["evicted"] else at[(at * page < sinks) | ((at + 1) * page > start[0])])
    scratch = -(-int(sizes.sum()) // page) + 1
    order = rng.permutation(sum(len(h) for h in held) + scratch + 1)
    tables = np.full((len(prefixes), max(1, int(counts.max()))), -1)
    at = 0
    for r, h in enumerate(held):
        tables[r, h] = order[at:at + len(h)]
        at += len(h)
    slots = (order[at:at + scratch, None] * page + np.arange(page)).reshape(-1)
    slots = slots[rng.permutation(slots.size)[:int(sizes.sum())]]
    cu = np.concatenate([[0], np.cumsum(sizes)])
    request = np.repeat(np.arange(len(sizes)), sizes)
    squares = np.concatenate([[0], np.cumsum(sizes * sizes)])
    bias = np.concatenate([np.where(_ancestors(of), 0.0, -np.inf).reshape(-1) for of in parents]).astype(np.float32)
    metadata = SimpleNamespace(
        cu_seqlens_q=_ints(cu), query_to_request=_ints(request), query_local_row=_ints(np.arange(cu[-1]) - cu[request]),
        prefix_lens=_ints(prefixes), block_tables=_ints(tables), tree_slots=_ints(slots, torch.int64),
        qq_bias=torch.as_tensor(bias, device=_DEVICE), qq_bias_offsets=_ints(squares, torch.int64),
        node_counts=_ints(sizes), block_size=page, prefix_lengths=tuple(map(int, prefixes)),
        query_offsets=tuple(map(int, cu)), node_counts_host=tuple(map(int, sizes)),
        block_tables_host=tuple(tuple(map(int, row[:n])) for row, n in zip(tables, counts)),
        tree_slot_ids=tuple(map(int, slots)), request_ids=tuple(range(len(sizes))), ancestor_words=None,
        num_requests=len(sizes), total_queries=int(cu[-1]))
    shape = (order.size, page, heads, dim)
    k, v = _normal(gen, shape, _TYPES[case["dtype"]]), _normal(gen, shape, _TYPES[case["dtype"]], 0.7)
    q = _normal(gen, (int(cu[-1]), heads * case["groups"], dim), _TYPES[case["dtype"]], case["gain"])
    return SimpleNamespace(kind="window", q=q, k=k, v=v, metadata=metadata, positions=_ints(
        np.repeat(prefixes, sizes) + np.concatenate(depths), torch.int64), scale=dim ** -0.5, groups=case["groups"],
        window=case["window"], sinks=case["sinks"], out=torch.float32 if case["out32"] else q.dtype)


def _frequencies(case):
    """Angles a token: powers of 1e-6 over the turned part, slow ones divided by the factor, blended between
    1 and 32 turns over the length that the unscaled ones were made for."""
    n = case["turned"] // 2
    plain = 1e6 ** (-np.arange(n, dtype=np.float64) / n)
    turns = plain * (case["length"] / case["factor"]) / (2 * math.pi)
    keep = np.clip((turns - 1) / 31, 0, 1)
    return plain * (keep + (1 - keep) / case["factor"])


def _prepare_rotary(case, seed):
    gen = torch.Generator(device=_DEVICE).manual_seed(seed)
    rng = np.random.default_rng(seed)
    rows, hq, hk, dim = case["rows"], case["q_heads"], case["kv_heads"], case["head_dim"]
    dtype = _TYPES[case["dtype"]]
    # Q, K and V as a fused projection leaves them: columns of one matrix.
    qkv = _normal(gen, (rows, hq + 2 * hk, dim), dtype, 2.0)
    pages = -(-rows // case["page"]) + 2
    pool = (pages, case["page"], hk, dim)
    return SimpleNamespace(
        kind="rotary", q=qkv[:, :hq], k=qkv[:, hq:hq + hk], v=qkv[:, hq + hk:],
        positions=_ints(rng.integers(0, case["length"], size=rows), torch.int64),
        frequencies=torch.as_tensor(_frequencies(case), device=_DEVICE), k_pool=_normal(gen, pool, dtype),
        v_pool=_normal(gen, pool, dtype), slots=_ints(rng.permutation(pages * case["page"])[:rows], torch.int64),
        out=torch.empty((rows, hq, dim), dtype=dtype, device=_DEVICE), interleaved=case["interleaved"],
        gain=1.0 if case["factor"] == 1.0 else 0.1 * math.log(case["factor"]) + 1.0)


def _prepare_logprobs(case, seed):
    gen = torch.Generator(device=_DEVICE).manual_seed(seed)
    rng = np.random.default_rng(seed)
    rows, vocab = case["rows"], case["vocab"]
    held = max(case["held"], rows)
    # Rows from nearly certain to nearly flat, as a model's are.
    logits = _normal(gen, (held, vocab), _TYPES[case["dtype"]], case["gain"])
    peaks = torch.rand((held, min(vocab, 8)), generator=gen, device=_DEVICE) * (5 * case["gain"])
    where = torch.randint(0, vocab, peaks.shape, generator=gen, device=_DEVICE)
    logits.scatter_(1, where, peaks.to(logits.dtype))
    if case["masked"]:
        # Words that a grammar forbids; the first peak stays.
        keep = logits.gather(1, where[:, :1])
        logits[:, torch.rand(vocab, generator=gen, device=_DEVICE) < case["masked"]] = -torch.inf
        logits.scatter_(1, where[:, :1], keep)
    picked = np.sort(rng.permutation(held)[:rows]) if case["held"] else None
    tokens = rng.integers(0, vocab, size=(rows, case["tokens"]))
    likely = where.cpu().numpy()[picked if picked is not None else slice(None)]
    tokens = np.where(rng.random(tokens.shape) < 0.5, likely[:, :1], tokens)
    if case["tokens"] > 1:
        tokens[:, 1:][rng.random((rows, case["tokens"] - 1)) < 0.2] = -1   # nodes with fewer children
    else:
        tokens = tokens[:, 0]
    return SimpleNamespace(kind="logprobs", logits=logits, tokens=_ints(tokens, torch.int64), top=case["top"],
                           rows=None if picked is None else _ints(picked, torch.int64))


def prepare(case, seed):
    return {"window": _prepare_window, "rotary": _prepare_rotary, "logprobs": _prepare_logprobs}[case["kind"]](case, seed)


# --------------------------------------------------------------------------- plain forms
def _plain_window(s):
    m = s.metadata
    n, most_t = m.num_requests, max(m.node_counts_host)
    heads, dim = s.k.shape[2], s.k.shape[3]
    prefix, nodes, start = m.prefix_lens.long()[:, None], m.node_counts.long()[:, None], m.cu_seqlens_q.long()[:-1, None]
    # The keys a request may see, padded: first tokens, the window before the prefix's end, the tree.
    most_s, most_w = min(s.sinks, max(m.prefix_lengths)), min(s.window - 1, max(m.prefix_lengths))
    a = torch.arange(most_s + most_w + most_t, device=_DEVICE)[None, :]
    from_window = torch.maximum(prefix - most_w, torch.clamp(prefix, max=most_s)) + a - most_s
    at = torch.where(a < most_s, a, from_window)
    node_at = a - most_s - most_w
    in_tree = node_at >= 0
    live = torch.where(in_tree, node_at < nodes, at < prefix)
    row = (start + node_at).clamp(0, m.total_queries - 1)
    page = m.block_tables.long().gather(1, (at // m.block_size).clamp(0, m.block_tables.shape[1] - 1))
    slot = torch.where(in_tree, m.tree_slots[row], page * m.block_size + at % m.block_size)
    slot = torch.where(live, slot, 0)
    key_at = torch.where(in_tree, s.positions[row], at)

    def rows(pool):
        return pool.view(-1, heads, dim)[slot].float() * live[:, :, None, None]

    # Queries padded to the longest tree: [requests, KV heads, nodes x group, head size].
    node = torch.arange(most_t, device=_DEVICE)[None, :]
    of = (start + node).clamp(max=m.total_queries - 1)
    q = s.q.float()[of].view(n, most_t, heads, s.groups, dim).permute(0, 2, 1, 3, 4).reshape(n, heads, most_t * s.groups, dim)
    scores = torch.matmul(q, rows(s.k).permute(0, 2, 3, 1).contiguous()) * s.scale
    where = m.qq_bias_offsets[:-1, None, None] + node[:, :, None] * nodes[:, :, None] + node_at[:, None, :]
    bias = m.qq_bias[where.clamp(0, m.qq_bias.numel() - 1)]
    near = (s.positions[of][:, :, None] - key_at[:, None, :] < s.window) | (key_at < s.sinks)[:, None, :]
    shown = live[:, None, :] & near & (node_at[:, None, :] <= node[:, :, None]) & (node < nodes)[:, :, None]
    bias = torch.where(shown, torch.where(in_tree[:, None, :], bias, 0.0), float("-inf"))
    scores = scores.view(n, heads, most_t, s.groups, -1) + bias[:, None, :, None, :]
    scores = torch.exp(scores - scores.amax(-1, keepdim=True))
    weight = (scores / scores.sum(-1, keepdim=True)).view(n, heads, most_t * s.groups, -1)
    out = torch.matmul(weight, rows(s.v).permute(0, 2, 1, 3).contiguous())
    out = out.view(n, heads, most_t, s.groups, dim).permute(0, 2, 1, 3, 4).reshape(n, most_t, heads * s.groups, dim)
    return out[m.query_to_request.long(), m.query_local_row.long()].to(s.out)


def _turned(s, x):
    angle = s.positions.double()[:, None] * s.frequencies
    cos, sin = (angle.cos() * s.gain).float()[:, None], (angle.sin() * s.gain).float()[:, None]
    n = s.frequencies.numel()
    x = x.float()
    out = x.clone()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if s.interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., first], x[..., second]
    out[..., first] = a * cos - b * sin
    out[..., second] = b * cos + a * sin
    return out


def _plain_rotary(s):
    s.out.copy_(_turned(s, s.q))
    s.k_pool.view(-1, *s.k_pool.shape[2:])[s.slots] = _turned(s, s.k).to(s.k_pool.dtype)
    s.v_pool.view(-1, *s.v_pool.shape[2:])[s.slots] = s.v


def _plain_logprobs(s):
    x = (s.logits if s.rows is None else s.logits[s.rows]).float()
    top = x.amax(-1, keepdim=True)
    z = x - top
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    entropy = (log_total - torch.where(e == 0, 0.0, e * z).sum(-1, keepdim=True) / total)[:, 0]
    del e, z
    given = s.tokens.view(x.shape[0], -1)
    logp = torch.where(given >= 0, x.gather(1, given.clamp(min=0)) - top - log_total, 0.0).view(s.tokens.shape)
    ids = torch.empty((x.shape[0], s.top), dtype=torch.int64, device=_DEVICE)
    values = torch.empty((x.shape[0], s.top), device=_DEVICE)
    index = torch.arange(x.shape[1], device=_DEVICE, dtype=torch.int32)
    left = torch.ones_like(x, dtype=torch.bool) if s.top else None
    x0 = x
    for i in range(s.top):   # the largest value that is left, at its lowest index
        best = torch.where(left, x0, -torch.inf).amax(-1, keepdim=True)
        first = torch.where(left & (x0 == best), index, x.shape[1]).amin(-1, keepdim=True).long()
        left.scatter_(1, first, False)
        ids[:, i:i + 1], values[:, i:i + 1] = first, best
    return logp, entropy, ids, values - top - log_total


def run(state):
    s = state
    if s.kind == "window":
        if own:
            return _package().packed_window_attention(s.q, s.k, s.v, s.metadata, s.positions, s.scale, s.groups,
                                                      window=s.window, sinks=s.sinks, output_dtype=s.out)
        return _plain_window(s)
    if s.kind == "logprobs":
        if own:
            return _package().token_logprobs(s.logits, s.tokens, top=s.top, rows=s.rows)
        return _plain_logprobs(s)
    if own:
        _package().rotary_scatter_prevalidated(s.q, s.k, s.v, s.positions, s.frequencies, s.k_pool, s.v_pool, s.slots,
                                               s.out, interleaved=s.interleaved, gain=s.gain)
    else:
        _plain_rotary(s)
    return [s.out, s.k_pool, s.v_pool]


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "window":
        pairs = keys = rows = 0
        for prefix, nodes, parents, depth in zip(*_trees(case)):
            seen, from_prefix, from_tree = _seen(int(prefix), parents, depth, case)
            pairs, keys, rows = pairs + seen, keys + from_prefix + from_tree, rows + int(nodes)
        hq, dim = case["kv_heads"] * case["groups"], case["head_dim"]
        return {"bytes": 2 * keys * case["kv_heads"] * dim * size + rows * (hq * dim * (size + (4 if case["out32"] else size)) + 8),
                "flops": 4 * hq * dim * pairs}
    if case["kind"] == "rotary":
        hq, hk, dim = case["q_heads"], case["kv_heads"], case["head_dim"]
        return {"bytes": case["rows"] * ((2 * hq + 4 * hk) * dim * size + 16) + 4 * case["turned"],
                "flops": case["rows"] * (hq + hk) * case["turned"] * 3}
    given = case["rows"] * case["tokens"]
    return {"bytes": case["rows"] * (case["vocab"] * size + 4 + 12 * case["top"]) + 12 * given,
            "flops": case["rows"] * case["vocab"] * 5}


# --------------------------------------------------------------------------- 64 bits
def _exact_window(case, seed):
    s = _prepare_window(case, seed)
    m = s.metadata
    heads, dim = s.k.shape[2], s.k.shape[3]
    out = torch.empty(s.q.shape, dtype=torch.float64, device=_DEVICE)
    first = 0
    for r, (prefix, nodes, table) in enumerate(zip(m.prefix_lengths, m.node_counts_host, m.block_tables_host)):
        rows = slice(m.query_offsets[r], m.query_offsets[r + 1])
        at = np.arange(prefix)
        at = at[(at < s.sinks) | (at > prefix - s.window)]   # what the earliest row sees
        mine = np.asarray(table, dtype=np.int64)[at // m.block_size] * m.block_size + at % m.block_size
        slots = torch.cat([_ints(mine, torch.int64), m.tree_slots[rows]])
        where = torch.cat([_ints(at, torch.int64), s.positions[rows]])
        bias = m.qq_bias[first:first + nodes * nodes].view(nodes, nodes).double()
        first += nodes * nodes
        mask = torch.cat([torch.zeros((nodes, len(at)), device=_DEVICE, dtype=torch.float64), bias.masked_fill(
            torch.triu(torch.ones_like(bias), 1) > 0, -torch.inf)], dim=1)
        hidden = (where[None, :] <= s.positions[rows][:, None] - s.window) & (where[None, :] >= s.sinks)
        mask = mask.masked_fill(hidden, -torch.inf).repeat_interleave(s.groups, dim=0)
        q = s.q[rows].double()
        for h in range(heads):
            k, v = s.k.view(-1, heads, dim)[slots, h].double(), s.v.view(-1, heads, dim)[slots, h].double()
            score = torch.mm(q[:, h * s.groups:(h + 1) * s.groups].reshape(-1, dim), k.t().contiguous()) * s.scale + mask
            out[rows, h * s.groups:(h + 1) * s.groups] = torch.mm(torch.softmax(score, -1), v).view(nodes, s.groups, dim)
    return out


def _exact_rotary(case, seed):
    s = _prepare_rotary(case, seed)
    n = s.frequencies.numel()
    turn = torch.polar(torch.full((case["rows"], n), s.gain, dtype=torch.float64, device=_DEVICE),
                       s.positions.double()[:, None] * s.frequencies)[:, None]

    def rotated(x):
        x = x.double()
        part = x[..., :2 * n]
        pairs = part.unflatten(-1, (n, 2)) if s.interleaved else part.unflatten(-1, (2, n)).transpose(-1, -2)
        z = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turn)
        z = z if s.interleaved else z.transpose(-1, -2)
        return torch.cat([z.flatten(-2), x[..., 2 * n:]], dim=-1)

    def put(pool, x):
        held = pool.double()
        held.view(-1, *pool.shape[2:])[s.slots] = x
        return held

    return [rotated(s.q), put(s.k_pool, rotated(s.k)), put(s.v_pool, s.v.double())]


def _exact_logprobs(case, seed):
    s = _prepare_logprobs(case, seed)
    kept = torch.arange(case["rows"], device=_DEVICE) if s.rows is None else s.rows
    given = s.tokens.view(case["rows"], -1)
    parts = []
    for at in range(0, case["rows"], 256):
        logp = torch.log_softmax(s.logits[kept[at:at + 256]].double(), -1)
        entropy = -torch.special.xlogy(logp.exp(), logp.exp()).sum(-1)
        ids = given[at:at + 256]
        chosen = torch.where(ids < 0, 0.0, logp.gather(1, ids.clamp(min=0)))
        order = torch.sort(s.logits[kept[at:at + 256]], dim=-1, descending=True, stable=True).indices[:, :s.top]
        parts.append((chosen, entropy, order, logp.gather(1, order)))
    logp, entropy, ids, values = (torch.cat(p) for p in zip(*parts))
    return logp.view(s.tokens.shape), entropy, ids, values


def exact(case, seed):
    return {"window": _exact_window, "rotary": _exact_rotary, "logprobs": _exact_logprobs}[case["kind"]](case, seed)
