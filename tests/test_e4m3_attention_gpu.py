"""The e4m3 tree attention on the GPU against 64 bits.

Tolerance, derived.  With normalised weights w_k and values u_k = vs_k V8_k, let S = sum_k w_k |u_k| per
output.  A probability times its scale is rounded to bf16 (2^-8 of it) or kept in two terms (2^-17,
f16 output) or three (2^-26, fp32 output).
Scores are sums of D exact products in fp32, scaled by two roundings: at most (D + 4) 2^-24 of
sum_d |q_d k_d| scale, and a bias adds its own rounding of the score; a probability is off by that
and by 2^-21 of its exponential, in the numerator and in the sum.  The sums over n keys and the joins
of up to 600 pieces add (n + 600) 2^-24 of S each.  The store adds half a step of its type.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import e4m3_helpers
from jetspec_amd import (PackedTreeMetadata, _lib, build_block_tables, commit_slots, copy_accepted_kv,
                         packed_slot_maps, packed_tree_attention, packed_tree_attention_e4m3, qk_norm_rope_scatter_prevalidated,
                         read_and_clear_status, store_kvcache_e4m3, workloads)

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class Batch:
    """A packed batch over a poisoned e4m3 pool: what no row may read holds NaN codes and scales."""

    def __init__(self, prefixes, trees, *, dim=128, kv_heads=2, groups=4, page=16, dtype=BF16, gain=1.0, seed=0):
        rng = np.random.default_rng(seed)
        gen = torch.Generator(device=DEV).manual_seed(seed)
        counts = [len(t) for t in trees]
        total = sum(counts)
        need = [-(-p // page) for p in prefixes]
        scratch = -(-total // page) + 1
        order = rng.permutation(sum(need) + scratch + 2)
        tables, at = [], 0
        for n in need:
            tables.append([int(x) for x in order[at:at + n]])
            at += n
        free = (order[at:at + scratch, None] * page + np.arange(page)).reshape(-1)
        slots = free[rng.permutation(free.size)[:total]]
        masks = [torch.as_tensor(workloads.ancestor_mask(t), device=DEV) for t in trees]
        self.meta = PackedTreeMetadata.build(prefixes, tables, [torch.as_tensor(s, device=DEV) for s in
                                                                np.split(slots, np.cumsum(counts)[:-1])], masks, page)
        self.prefixes, self.trees, self.counts, self.tables, self.groups = prefixes, trees, counts, tables, groups
        self.scale = dim ** -0.5
        shape = (order.size, page, kv_heads, dim)
        self.k, self.v = (torch.full(shape, 0x7F, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2))
        self.ks, self.vs = (torch.full(shape[:3], float("nan"), device=DEV) for _ in range(2))
        self.keys = [np.concatenate([np.asarray(tab, dtype=np.int64)[np.arange(p) // page] * page + np.arange(p) % page
                                     if p else np.zeros(0, np.int64), part])
                     for p, tab, part in zip(prefixes, tables, np.split(slots, np.cumsum(counts)[:-1]))]
        live = torch.as_tensor(np.concatenate(self.keys), device=DEV)
        rows = (live.numel(), kv_heads, dim)
        # Scales over a few octaves from key to key, as rows of different sizes have.
        sizes = torch.exp2(torch.randint(-2, 3, rows[:2], generator=gen, device=DEV)).unsqueeze(-1)
        store_kvcache_e4m3(torch.randn(rows, generator=gen, device=DEV),
                           torch.randn(rows, generator=gen, device=DEV) * sizes, self.k, self.v, self.ks, self.vs, live)
        self.q = (torch.randn((total, kv_heads * groups, dim), generator=gen, device=DEV) * gain).to(dtype)

    def run(self, out=None):
        return packed_tree_attention_e4m3(self.q, self.k, self.v, self.ks, self.vs, self.meta, self.scale, self.groups,
                                          output_dtype=out)

    def rows(self, pool, scale, keys, h):
        heads, dim = pool.shape[2:]
        codes = pool.contiguous().view(torch.uint8).view(-1, heads, dim)[keys, h].cpu().numpy()
        return torch.as_tensor(e4m3_helpers.VALUES[codes], device=DEV) * scale.reshape(-1, heads)[keys, h].double()[:, None]

    def check(self, out, requests=None):
        """Compares the rows of `requests` (all) with the formula in 64 bits."""
        got = self.run(out) if not isinstance(out, torch.Tensor) else out
        rounded = {BF16: 2.0 ** -8, F16: 2.0 ** -17, F32: 2.0 ** -26}[got.dtype]
        m = self.meta
        half_step = torch.finfo(got.dtype).eps / 2
        for r in range(len(self.prefixes)) if requests is None else requests:
            rows, prefix, n = m.request_slice(r), self.prefixes[r], self.counts[r]
            keys = torch.as_tensor(self.keys[r], device=DEV)
            first = int(m.qq_bias_offsets[r])
            bias = m.qq_bias[first:first + n * n].view(n, n).double()
            bias = torch.where(torch.tril(torch.ones_like(bias)) > 0, bias, -torch.inf).repeat_interleave(self.groups, 0)
            for h in range(self.k.shape[2]):
                mine = slice(h * self.groups, (h + 1) * self.groups)
                q = self.q[rows, mine].double().reshape(n * self.groups, -1)
                k, v = self.rows(self.k, self.ks, keys, h), self.rows(self.v, self.vs, keys, h)
                score = torch.mm(q, k.t().contiguous()) * self.scale
                size = torch.mm(q.abs(), k.abs().t().contiguous()) * abs(self.scale)
                score[:, prefix:] += bias
                size[:, prefix:] += torch.where(bias.isfinite(), bias.abs(), 0)
                seen = score > -torch.inf
                w = torch.softmax(score, -1)
                w = torch.where(seen.any(-1, keepdim=True), w, 0)
                expect, spread = torch.mm(w, v), torch.mm(w, v.abs())
                slack = ((q.shape[1] + 4) * 2.0 ** -24 * torch.where(seen, size, 0).amax(-1, keepdim=True) + 2.0 ** -21)
                relative = rounded + 2 * slack + 2 * (keys.numel() + 600) * 2.0 ** -24
                allowed = relative * spread * (1 + 2.0 ** -6)
                allowed = allowed + half_step * (expect.abs() + allowed) + (2.0 ** -25 if got.dtype == F16 else 0)
                off = (got[rows, mine].double().reshape(expect.shape) - expect).abs() - allowed
                assert bool((off <= 0).all()), (r, h, float(off.max()), float(allowed.max()))
        return got


def trees(sizes, seed=0, depth=8):
    rng = np.random.default_rng(seed)
    return [workloads.random_parents(int(n), depth, rng) for n in sizes]


EDGES = [0, 1, 31, 32, 33, 127, 128, 129, 200, 255, 256, 257, 383, 384, 1000]


@pytest.mark.parametrize("dtype, out", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("dim, kv_heads, groups, page", [
    (128, 2, 4, 16), (128, 1, 1, 48), (128, 3, 7, 256), (128, 1, 16, 1), (64, 2, 4, 16), (64, 1, 5, 7), (64, 2, 40, 32),
    (256, 2, 4, 16), (256, 1, 8, 100),
])
def test_single_tokens_at_every_edge(dim, kv_heads, groups, page, dtype, out):
    Batch(EDGES, [[-1]] * len(EDGES), dim=dim, kv_heads=kv_heads, groups=groups, page=page, dtype=dtype, gain=2.0).check(out)
    assert read_and_clear_status(DEV) == 0


@pytest.mark.parametrize("dtype, out", [(BF16, BF16), (BF16, F32), (F16, F16)])
@pytest.mark.parametrize("dim, kv_heads, groups, page, sizes", [
    (128, 2, 4, 16, [1, 2, 3, 5, 8, 13, 16, 10]), (128, 2, 4, 16, [16, 17, 30, 1, 32, 7, 20, 64]),
    (128, 2, 4, 256, [64, 65, 33, 1, 130, 64, 2, 40]), (128, 1, 3, 48, [100, 21, 86, 128, 129, 1, 255, 60]),
    (64, 2, 5, 16, [1, 40, 3, 5, 60, 13, 16, 33]), (64, 1, 8, 32, [64, 65, 127, 128, 129, 1, 20, 300]),
    (64, 8, 1, 16, [8, 40, 90, 200, 33, 1, 2, 64]),
    (256, 1, 4, 16, [1, 2, 3, 5, 8, 7, 6, 4]), (256, 2, 4, 48, [16, 1, 20, 9, 32, 7, 2, 11]),
    (256, 1, 6, 16, [64, 65, 33, 1, 130, 64, 2, 40]),
])
def test_trees(dim, kv_heads, groups, page, sizes, dtype, out):
    prefixes = [0, 5, 128, 300, 64, 257, 1023, 31]
    Batch(prefixes, trees(sizes), dim=dim, kv_heads=kv_heads, groups=groups, page=page, dtype=dtype, gain=1.5).check(out)
    assert read_and_clear_status(DEV) == 0


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_chunks_beside_trees(dim):
    parents = [workloads.chain_parents(n) for n in (512, 300, 129)] + trees([1, 64, 20])
    batch = Batch([0, 700, 127, 2000, 33, 0], parents, dim=dim, gain=2.0)
    batch.check(BF16)
    batch.check(F32)


@pytest.mark.parametrize("dim, groups, size", [(128, 4, 1), (128, 4, 16), (128, 4, 64), (64, 8, 4), (256, 4, 2), (256, 2, 40)])
def test_a_long_context_is_cut_and_joined(dim, groups, size):
    """One request of 40000 keys over the whole chip, beside one of a few keys."""
    batch = Batch([40001, 3], trees([size, size]), dim=dim, groups=groups, page=256, gain=3.0)
    first = batch.check(BF16)
    assert torch.equal(first, batch.run(BF16))   # no order of arrival in the result
    batch.check(F32)


@pytest.mark.parametrize("dim, groups, sizes", [(128, 4, [15, 1, 16, 3]), (64, 4, [60, 64, 2, 33]), (128, 3, [80, 60, 90, 1]),
                                                (256, 2, [9, 30, 7, 1])])
def test_requests_in_a_few_pieces_each(dim, groups, sizes):
    """Some rows are joined from a few pieces, others from more, by workgroups that share them out."""
    batch = Batch([9001, 300, 6000, 4097], trees(sizes), dim=dim, kv_heads=8, groups=groups, page=128, gain=2.0)
    first = batch.check(F32)
    assert torch.equal(first, batch.run(F32))


def test_many_requests():
    rng = np.random.default_rng(1)
    n = 900
    batch = Batch([int(x) for x in rng.integers(0, 90, n)], trees(rng.integers(1, 4, n)), kv_heads=1, page=16)
    batch.check(BF16, requests=range(0, n, 7))
    batch = Batch([int(x) for x in rng.integers(0, 300, n)], trees([1] * n), kv_heads=1, dim=64, page=16)
    batch.check(F32, requests=range(0, n, 13))


def test_every_code():
    """One key: the output is its V row, code by code, and K codes enter the score as their values."""
    batch = Batch([0, 0], [[-1], [-1, 0]], dim=256, kv_heads=1, groups=2)
    codes = torch.arange(256, dtype=torch.uint8, device=DEV)
    codes[codes & 127 == 127] = 0
    slots = batch.meta.tree_slots
    flat = [t.view(torch.uint8).view(-1, 256) for t in (batch.k, batch.v)]
    for t in flat:
        t[slots] = codes
    for s in (batch.ks, batch.vs):
        s.view(-1)[slots] = 1.0
    values = torch.as_tensor(e4m3_helpers.VALUES[codes.cpu().numpy()], device=DEV)
    assert torch.equal(batch.run(F32)[0, 0].double(), values)
    batch.q.zero_()
    for d in range(0, 256, 5):
        batch.q[2, 0, d] = 1 / 16
    batch.check(F32)


@pytest.mark.parametrize("size", [5, 40, 70])
def test_nan_and_infinity_stay_with_the_rows_that_see_them(size):
    """Node 1 is a leaf no other node descends from."""
    parents = [-1, 0] + [0] + list(range(2, size - 1))
    for where, value in (("ks", float("nan")), ("vs", float("nan")), ("vs", float("inf")), ("k", 0x7F), ("v", 0xFF)):
        batch = Batch([50, 7], [parents, parents], dim=128)
        clean = batch.run()
        slot = int(batch.meta.tree_slots[1])
        t = getattr(batch, where)
        if where in ("k", "v"):
            t.view(torch.uint8).view(-1, 2, 128)[slot, 0, 5] = value
        else:
            t.view(-1, 2)[slot, 0] = value
        got = batch.run()
        assert not bool(got[1, :4].isfinite().any()), where
        got[1, :4] = clean[1, :4]
        assert torch.equal(got, clean), where
    batch = Batch([50, 7], [parents, parents], dim=128)
    clean = batch.run()
    batch.q[3] = float("nan")
    got = batch.run()
    assert bool(got[3].isnan().all())
    got[3] = clean[3]
    assert torch.equal(got, clean)


def test_prefix_codes_that_are_nan():
    batch = Batch([300], [[-1, 0, 0]])
    clean = batch.run()
    page, offset = batch.tables[0][100 // 16], 100 % 16
    batch.v.view(torch.uint8)[page, offset, 0, 9] = 0x7F
    got = batch.run()
    assert bool(got[:, :4, 9].isnan().all()) and int(got.isnan().sum()) == 12
    got[:, :4, 9] = clean[:, :4, 9]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("size, groups", [(3, 4), (50, 4), (90, 3)])
def test_finite_biases_and_rows_that_see_nothing(size, groups):
    batch = Batch([0, 65, 0], trees([size, size, 2]), groups=groups, gain=2.0)
    gen = torch.Generator(device=DEV).manual_seed(3)
    bias = batch.meta.qq_bias
    shift = torch.randn(bias.shape, generator=gen, device=DEV) * 3
    bias.copy_(torch.where(bias == 0, shift, bias))
    bias[1] = 50.0                    # above the diagonal: never seen
    batch.check(BF16)
    batch.check(F32)
    # The last node of the first request sees nothing: no prefix, all of its row hidden.
    bias[size * (size - 1):size * size] = -float("inf")
    got = batch.check(F32)
    assert bool((got[size - 1] == 0).all())
    assert read_and_clear_status(DEV) == 0


def test_biases_of_the_lowest_value():
    lowest = torch.finfo(F32).min
    batch = Batch([0, 40], trees([6, 6]))
    n = 36
    for r in range(2):
        part = batch.meta.qq_bias[r * n:(r + 1) * n]
        part.copy_(torch.where(part == 0, lowest, part))
    got = batch.run(F32)
    # With a prefix the biased nodes weigh nothing; without one they weigh the same, the scores being
    # absorbed: the mean of the seen values.
    batch.meta.qq_bias.copy_(torch.where(batch.meta.qq_bias == lowest, -float("inf"), batch.meta.qq_bias))
    assert torch.equal(got[6:], batch.run(F32)[6:])
    seen = workloads.ancestor_mask(batch.trees[0])
    keys = torch.as_tensor(batch.keys[0], device=DEV)
    for h in range(2):
        v = batch.rows(batch.v, batch.vs, keys, h)
        for i in range(6):
            mine = v[torch.as_tensor(seen[i], device=DEV)]
            # Equal weights: the three-term probabilities and the quotient, and a sum of 6.
            allowed = (2.0 ** -26 + 10 * 2.0 ** -24) * mine.abs().mean(0)
            assert bool(((got[i, 4 * h].double() - mine.mean(0)).abs() <= allowed).all())


def test_layouts():
    """Views as a serving program has them: a layer of a stacked pool, columns of a projection."""
    batch = Batch([300, 0, 77], trees([20, 1, 9]), dim=128, kv_heads=2)
    expect = batch.run()
    stack = torch.zeros((2, 3, *batch.k.shape), dtype=torch.uint8, device=DEV).view(E4M3)
    scales = torch.zeros((2, 3, *batch.ks.shape), device=DEV)
    stack[0, 1], stack[1, 1], scales[0, 1], scales[1, 1] = batch.k, batch.v, batch.ks, batch.vs
    batch.k, batch.v, batch.ks, batch.vs = stack[0, 1], stack[1, 1], scales[0, 1], scales[1, 1]
    assert torch.equal(batch.run(), expect)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (batch.k, batch.v, batch.ks, batch.vs)]
    batch.k, batch.v, batch.ks, batch.vs = heads_first
    assert torch.equal(batch.run(), expect)
    q = batch.q
    for lead in (8, 3):   # rows that start at 16 bytes and rows that do not
        wide = torch.zeros((q.shape[0], q.shape[1] * 128 + 24), dtype=BF16, device=DEV)
        batch.q = wide[:, lead:lead + q.shape[1] * 128].unflatten(1, (q.shape[1], 128))
        batch.q.copy_(q)
        assert torch.equal(batch.run(), expect)
    batch.k = torch.zeros(batch.k.numel() + 8, dtype=torch.uint8, device=DEV).view(E4M3)[8:].view(heads_first[0].shape)
    with pytest.raises(ValueError, match="start at 16 bytes"):
        batch.run()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_layouts_of_large_pages(dim):
    """Pages of whole steps, read by the page where keys and values lie alike and key by key where not."""
    batch = Batch([700, 256, 255], trees([20, 1, 9]), dim=dim, page=256)
    expect = batch.check(BF16)
    plain = batch.k, batch.v, batch.ks, batch.vs
    stack = torch.zeros((2, 3, *batch.k.shape), dtype=torch.uint8, device=DEV).view(E4M3)
    stack[0, 1], stack[1, 1] = batch.k, batch.v
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in plain]
    wide = torch.zeros((*batch.ks.shape[:2], 5), device=DEV)[..., 1:3]
    wide.copy_(batch.vs)
    for batch.k, batch.v, batch.ks, batch.vs in ((stack[0, 1], stack[1, 1], *plain[2:]), heads_first,
                                                 (heads_first[0], *plain[1:]), (*plain[:2], heads_first[2], plain[3]),
                                                 (*plain[:3], wide)):
        assert torch.equal(batch.run(), expect)
    assert read_and_clear_status(DEV) == 0


@pytest.mark.parametrize("dim, page", [(64, 128), (128, 128), (128, 256), (256, 64), (256, 256)])
@pytest.mark.parametrize("bad", [-1, 10 ** 6, 2 ** 31 - 1])
def test_bad_large_pages_are_skipped_and_reported(dim, page, bad):
    batch = Batch([3 * page + 5, 90], trees([4, 4]), dim=dim, page=page)
    clean = batch.run()
    batch.meta.block_tables[0, 1] = bad
    got = batch.run()
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_PAGE
    assert torch.equal(got[4:], clean[4:])
    batch.keys[0] = np.delete(batch.keys[0], np.arange(page, 2 * page))
    batch.prefixes[0] -= page
    batch.check(got)


def test_scores_without_scale_and_with_a_negative_one():
    batch = Batch([130, 4], trees([9, 2]))
    for scale in (0.0, -0.2):
        batch.scale = scale
        batch.check(F32)


def test_bad_pages_are_skipped_and_reported():
    batch = Batch([100, 90], trees([4, 4]), page=16)
    clean = batch.run()
    batch.meta.block_tables[0, 2] = 10 ** 6
    got = batch.run()
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_PAGE
    assert torch.equal(got[4:], clean[4:]) and bool(got.isfinite().all())
    batch.keys[0] = np.delete(batch.keys[0], np.arange(32, 48))
    batch.prefixes[0] -= 16
    batch.check(got)
    batch = Batch([100, 90], trees([4, 4]), page=16)
    batch.meta.tree_slots[5] = -3
    got = batch.run()
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_PAGE
    assert torch.equal(got[:5], batch.run()[:5]) and bool(got.isfinite().all())
    read_and_clear_status(DEV)


@pytest.mark.parametrize("field, index, value", [
    ("prefix_lens", 0, 10 ** 6), ("prefix_lens", 0, -1), ("node_counts", 0, 100), ("node_counts", 0, -4),
    ("cu_seqlens_q", 0, 7), ("cu_seqlens_q", 0, -1), ("qq_bias_offsets", 0, 20), ("qq_bias_offsets", 0, -1),
])
def test_requests_outside_the_batch_are_left_out(field, index, value):
    batch = Batch([100, 90], trees([4, 4]), page=16)
    clean = batch.run()
    getattr(batch.meta, field)[index] = value
    got = batch.run()
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_REQUEST
    assert torch.equal(got[4:], clean[4:])


def test_a_request_without_nodes():
    batch = Batch([100, 90, 30], trees([4, 4, 4]), page=16)
    clean = batch.run()
    batch.meta.node_counts[1] = 0
    got = batch.run()
    assert torch.equal(got[:4], clean[:4]) and torch.equal(got[8:], clean[8:])
    assert read_and_clear_status(DEV) == 0


def test_pools_past_4_gib():
    page, heads, dim = 256, 8, 128
    pages = 20000
    batch = Batch([700, 300], trees([16, 3]), kv_heads=heads, page=page)
    expect = batch.run()
    moved = torch.as_tensor(np.random.default_rng(0).permutation(pages - 1)[:batch.k.shape[0]] + 1, device=DEV)
    moved[0], moved[1] = pages - 1, pages - 2
    assert torch.unique(moved).numel() == moved.numel()
    pools = [torch.empty((pages, page, heads, dim), dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2)]
    scales = [torch.empty((pages, page, heads), device=DEV) for _ in range(2)]
    for new, old in zip((*pools, *scales), (batch.k, batch.v, batch.ks, batch.vs)):
        new.view(torch.uint8)[moved] = old.view(torch.uint8)
    batch.k, batch.v, batch.ks, batch.vs = *pools, *scales
    tables = batch.meta.block_tables
    tables.copy_(torch.where(tables >= 0, moved[tables.clamp(min=0).long()].int(), tables))
    slots = batch.meta.tree_slots
    slots.copy_(moved[slots // page] * page + slots % page)
    assert torch.equal(batch.run(), expect)


def test_captured_replays_follow_the_metadata():
    batch = Batch([700, 300, 90], trees([16, 3, 8]), gain=2.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        batch.run()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):   # two graphs over the same metadata
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = batch.run()
        graphs.append((graph, out))
    for k, lengths in enumerate(([700, 300, 90], [1, 0, 17], [650, 299, 0], [700, 300, 90])):
        batch.meta.prefix_lens.copy_(torch.tensor(lengths))
        batch.q.normal_()
        for graph, out in graphs:
            out.fill_(7)
            graph.replay()
        torch.cuda.synchronize()
        eager = batch.run()
        assert all(torch.equal(out, eager) for _, out in graphs), k
    assert read_and_clear_status(DEV) == 0


def test_two_streams_at_once():
    batches = [Batch([5000, 90], trees([16, 8]), seed=s) for s in range(2)]
    expect = [b.run() for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    got = [[], []]
    for _ in range(5):
        for b, s, g in zip(batches, streams, got):
            with torch.cuda.stream(s):
                g.append(b.run())
    torch.cuda.synchronize()
    for e, g in zip(expect, got):
        assert all(torch.equal(e, x) for x in g)


def test_near_the_bf16_cache():
    """Against packed_tree_attention over the values the codes stand for, kept in bf16 pools."""
    batch = Batch([900, 40], trees([30, 64]), page=32, gain=1.0)
    read = [(t.float() * s.unsqueeze(-1)) for t, s in ((batch.k, batch.ks), (batch.v, batch.vs))]
    # Scales of 1 keep the values exact in bf16.
    batch.ks.fill_(1.0)
    batch.vs.fill_(1.0)
    for t in (batch.k, batch.v):
        t.view(torch.uint8)[t.view(torch.uint8) & 127 == 127] = 0
    batch.scale = 1e-4
    wide = [t.to(BF16) for t in (batch.k, batch.v)]
    theirs = packed_tree_attention(batch.q, *wide, batch.meta, batch.scale, 4)
    ours = batch.run()
    size = wide[1].float().abs().max()
    # Each is within 2^-8 (its probabilities) and 2^-8 (its store) of the largest value, and some fp32.
    assert float((theirs.float() - ours.float()).abs().max()) <= 4 * 2.0 ** -8 * 1.01 * float(size)


def test_a_round_from_lengths_to_commit():
    """Tables and maps from lengths, norm + rotation + quantised scatter, attention, commit of codes and
    scales: every operator on what the one before it made, and the next token over the committed cache."""
    page, heads, groups, dim, blocks, layers = 32, 2, 4, 128, 64, 2
    gen = torch.Generator(device=DEV).manual_seed(5)
    rng = np.random.default_rng(5)
    lengths = torch.tensor([70, 33, 0, 128], dtype=torch.int32, device=DEV)
    sizes = [9, 4, 16, 1]
    parents = trees(sizes, seed=4)
    pool = torch.zeros((2, layers, blocks, page, heads, dim), dtype=torch.uint8, device=DEV).view(E4M3)
    scale = torch.zeros((2, layers, blocks, page, heads), device=DEV)
    order = torch.as_tensor(rng.permutation(blocks), dtype=torch.int32, device=DEV)
    arena, free = order[:2], order[2:]
    tables, counts, taken = build_block_tables(lengths, free, page, 6)
    assert counts.tolist() == [3, 2, 0, 4] and taken.tolist() == [9]
    # The prompts.
    total = int(lengths.sum())
    _, _, _, _, slots = packed_slot_maps(torch.zeros_like(lengths), lengths, total, page, blocks, block_tables=tables)
    for layer in range(layers):
        rows = (torch.randn((2, total, heads, dim), generator=gen, device=DEV)).to(BF16)
        store_kvcache_e4m3(rows[0], rows[1], pool[0, layer], pool[1, layer], scale[0, layer], scale[1, layer], slots)
    # A round of trees in the arena.
    nodes = torch.tensor(sizes, dtype=torch.int32, device=DEV)
    depths = torch.as_tensor(np.concatenate([workloads.depths_of(t) for t in parents]), dtype=torch.int32, device=DEV)
    cu, _, _, positions, tree_slots = packed_slot_maps(lengths, nodes, sum(sizes), page, blocks, arena_pages=arena,
                                                       depths=depths)
    host_tables = [row[:n] for row, n in zip(tables.tolist(), counts.tolist())]
    meta = PackedTreeMetadata.build(lengths.tolist(), host_tables, list(torch.split(tree_slots, sizes)),
                                    [torch.as_tensor(workloads.ancestor_mask(t), device=DEV) for t in parents], page)
    angle = torch.arange(200, device=DEV).double()[:, None] * torch.logspace(0, -4, dim // 2, dtype=torch.float64, device=DEV)
    cache = torch.cat([angle.cos(), angle.sin()], 1).float()
    weight = torch.rand((2, dim), generator=gen, device=DEV).to(BF16) + 0.5
    for layer in range(layers):
        qkv = torch.randn((sum(sizes), heads * (groups + 2), dim), generator=gen, device=DEV).to(BF16)
        parts = torch.split(qkv, [heads * groups, heads, heads], 1)
        here = (pool[0, layer], pool[1, layer])
        q = qk_norm_rope_scatter_prevalidated(*parts, weight[0], weight[1], positions, cache, *here, tree_slots,
                                              torch.empty_like(parts[0], memory_format=torch.contiguous_format),
                                              k_scale=scale[0, layer], v_scale=scale[1, layer])
        batch = Batch.__new__(Batch)
        batch.meta, batch.prefixes, batch.counts, batch.groups, batch.scale = meta, lengths.tolist(), sizes, groups, dim ** -0.5
        batch.k, batch.v, batch.ks, batch.vs, batch.q = *here, scale[0, layer], scale[1, layer], q
        batch.keys = [np.concatenate([np.asarray(t, dtype=np.int64)[np.arange(p) // page] * page + np.arange(p) % page
                                      if p else np.zeros(0, np.int64), s.cpu().numpy()])
                      for t, p, s in zip(host_tables, batch.prefixes, torch.split(tree_slots, sizes))]
        batch.check(BF16)
    # Accept a root path each, grow the tables for it, move codes and scales.
    paths = []
    for t in parents:
        node = len(t) - 1
        path = [node]
        while t[node] >= 0:
            node = t[node]
            path.append(node)
        paths.append(path[::-1])
    taken_rows = torch.tensor([len(p) for p in paths], dtype=torch.int32, device=DEV)
    offsets = torch.nn.functional.pad(taken_rows.cumsum(0), (1, 0)).int()
    grown, counts, more = build_block_tables(lengths + taken_rows, free[int(taken):], page, 6, held_tables=tables,
                                             held_counts=counts)
    assert torch.equal(grown[tables >= 0], tables[tables >= 0])
    source, target = commit_slots(tree_slots, cu, torch.tensor(sum(paths, []), dtype=torch.int32, device=DEV), offsets, grown,
                                  lengths, page, blocks)
    before = [pool.view(torch.uint8).clone(), scale.clone()]
    copy_accepted_kv(pool, source, target, page)
    copy_accepted_kv(scale.unsqueeze(-1), source, target, page)
    for new, old in zip((pool.view(torch.uint8), scale), before):
        flat_new, flat_old = (t.reshape(2, layers, blocks * page, -1) for t in (new, old))
        assert torch.equal(flat_new[:, :, target], flat_old[:, :, source])
        rest = np.setdiff1d(np.arange(blocks * page), target.cpu().numpy())
        assert torch.equal(flat_new[:, :, rest], flat_old[:, :, rest])
    # The committed slots are where the maps put the next rows.
    _, _, _, _, again = packed_slot_maps(lengths, taken_rows, int(taken_rows.sum()), page, blocks, block_tables=grown)
    assert torch.equal(again, target)
    assert read_and_clear_status(DEV) == 0
