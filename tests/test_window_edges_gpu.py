"""The windowed tree attention: positions that int32 does not hold, requests of fewer nodes than rows, offsets at int32's ends,
infinities and NaN at every launch shape, unlike and overlapping requests (tolerances as derived in
test_window_attention_gpu.py)."""
from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from jetspec_amd import _lib, packed_window_attention, read_and_clear_status
from test_window_attention_gpu import BF16, DEV, F16, F32, attend, trees
from window_helpers import Batch, chain, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("position, nearest", [
    (2 ** 33 + 61, 62), (-2 ** 33 + 61, 60), (2 ** 31, 62), (2 ** 32, 62), (2 ** 32 - 1, 62), (-2 ** 31 - 1, 60), (-2 ** 63, 60),
    (2 ** 63 - 1, 62), (-1, 60), (2 ** 31 - 1, 62), (-2 ** 31, 60),
])
def test_int64_positions_outside_are_the_nearer_end(position, nearest):
    # Node 2 of a request over 60 keys.  A window of 2 tells 60, 61 and 62 apart, as the row's position and as the key's.
    b = Batch([50, 60, 70], [chain(5)] * 3, window=2, sinks=0, seed=7)
    p = b.positions.clone()
    p[7] = position
    read_and_clear_status(DEV)
    got = attend(b, positions=p)
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_POSITION
    p[7] = nearest
    assert torch.equal(got, attend(b, positions=p))
    assert read_and_clear_status(DEV) == 0
    p[7] = 122 - nearest    # the other end, which would show
    assert not torch.equal(got, attend(b, positions=p))


def staged(sizes, live, dim, seed, **options):
    """A batch packed for `sizes` nodes a request of which `live` are counted."""
    rng = np.random.default_rng(seed)
    b = Batch([int(rng.integers(0, 90)) for _ in sizes], trees(sizes, seed), window=30, sinks=2, seed=seed, dim=dim, **options)
    offsets = b.meta.qq_bias_offsets.tolist()
    left = []
    for r, (n, count) in enumerate(zip(sizes, live)):
        square = b.meta.qq_bias[offsets[r]:offsets[r + 1]].view(n, n)[:count, :count].clone()
        b.meta.qq_bias[offsets[r]:offsets[r + 1]].fill_(float("nan"))
        b.meta.qq_bias[offsets[r]:offsets[r] + count * count] = square.reshape(-1)
        left.append(torch.arange(n) >= count)
    b.meta.node_counts.copy_(torch.tensor(live, dtype=torch.int32))
    left = torch.cat(left).to(DEV)
    b.meta.tree_slots[left] = -1
    b.q[left] = float("nan")
    return b, left


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("sizes, live", [([5, 5], [5, 3]), ([5, 5], [1, 4]), ([64, 40, 64], [64, 1, 33]), ([200, 140], [3, 129]),
                                         ([6] * 70, [i % 7 for i in range(70)])])
def test_requests_of_fewer_nodes_than_rows(sizes, live, dim):
    b, left = staged(sizes, live, dim, len(sizes) + live[1])
    out = torch.full_like(b.q, 9.0)
    read_and_clear_status(DEV)
    attend(b, out=out)
    assert read_and_clear_status(DEV) == 0
    assert (out[left] == 9.0).all()
    # The rows that count, as a batch of their own for the 64-bit results.
    b.q = b.q[~left]
    b.keys = [(j, slots, own[:count]) for (j, slots, own), count in zip(b.keys, live)]
    b.depths = [depth[:count] for depth, count in zip(b.depths, live)]
    b.counts = live
    check(out[~left], b, f"{sizes[:3]} {live[:3]} {dim}")


VALUES = [(BF16, float("inf")), (BF16, float("nan")), (F16, float("-inf")), (F16, float("nan"))]
ODD_SHAPES = [
    # prefixes, trees, window, sinks, options: blocks of 32 to 256 rows, whole and in parts, one table of keys and many
    ([100, 0], [8, 5], 43, 0, {}),
    ([700], [200], 500, 4, dict(groups=1, kv_heads=2)),
    ([900, 333], [150, 130], 700, 20, dict(groups=4, kv_heads=2)),
    ([3000], [20], 2900, 8, dict(groups=4, kv_heads=2)),
    ([60 + 5 * i for i in range(140)], [1 + i % 5 for i in range(140)], 50, 3, dict(groups=2, kv_heads=8)),
]


@pytest.mark.parametrize("dtype, value", VALUES)
@pytest.mark.parametrize("dim", [64, 80, 128, 200, 256])
@pytest.mark.parametrize("case", range(len(ODD_SHAPES)))
def test_odd_keys_and_values_stay_with_the_rows_that_see_them(case, dim, dtype, value):
    prefixes, sizes, window, sinks, options = ODD_SHAPES[case]
    rng = np.random.default_rng(case)
    parents = trees(sizes, case)
    b, clean = (Batch(prefixes, parents, window=window, sinks=sinks, seed=case, dim=dim, dtype=dtype, **options) for _ in range(2))
    bias, offsets = b.meta.qq_bias.cpu().numpy(), b.meta.qq_bias_offsets.tolist()
    seen, k_pool, v_pool = [], b.k.view(-1, *b.k.shape[2:]), b.v.view(-1, *b.v.shape[2:])
    for r, (j, slots, own) in enumerate(b.keys):
        n, depth = sizes[r], b.depths[r]
        at = np.concatenate([j, prefixes[r] + depth])
        visible = np.concatenate([np.ones((n, len(j)), bool), bias[offsets[r]:offsets[r + 1]].reshape(n, n) == 0], 1)
        mine = prefixes[r] + depth
        visible &= (mine[:, None] - at[None] < window) | (at[None] < sinks)
        # The first key that some row has lost, and nodes early, in the middle and last but one, where not all see them.
        some = np.flatnonzero(~visible.all(0) & visible.any(0))
        odd = some[:1].tolist() + [int(x) for x in rng.choice(some, size=min(3, len(some)), replace=False)] if len(some) else []
        every = np.concatenate([slots, own])
        for key in odd:
            k_pool[int(every[key]), 1] = float("nan")
            v_pool[int(every[key]), 0, dim - 3] = value
        seen.append(visible[:, odd].any(1))
    seen = np.concatenate(seen)
    assert seen.any() and not seen.all()
    want, bound = clean.expected(dtype)
    groups = b.groups
    for _ in range(2):
        got = attend(b).double().cpu().numpy()
        assert not np.isfinite(got[seen][:, :groups, dim - 3]).any()        # KV head 0: the value row
        assert np.isnan(got[seen][:, groups:2 * groups]).all()              # KV head 1: the key row
        off = np.abs(got - want) / bound
        assert (off[~seen] <= 1).all() and (off[:, 2 * groups:] <= 1).all()


def test_offsets_of_rows_at_the_ends_of_int32():
    # A request's rows begin past the batch and end at int32's lowest: left out, whatever the difference wraps to.
    def fresh():
        read_and_clear_status(DEV)
        return Batch([50, 60, 70], trees([5, 5, 5]), window=30, seed=7)

    good = attend(fresh())
    for first, last in ((2 ** 30, -2 ** 31), (2 ** 31 - 1, -2 ** 31), (2 ** 31 - 1, 2 ** 31 - 1), (16, -2 ** 31 + 4), (5, -2 ** 31)):
        b = fresh()
        b.meta.cu_seqlens_q[1:3] = torch.tensor([first, last], dtype=torch.int32)
        out = torch.full_like(b.q, 9.0)
        attend(b, out=out)
        assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_REQUEST
        if first == 5:
            assert torch.equal(out[:5], good[:5])
        assert (out[0 if first != 5 else 5:] == 9.0).all(), (first, last)
    b = fresh()
    b.meta.node_counts[1] = 2 ** 31 - 1
    out = torch.full_like(b.q, 9.0)
    attend(b, out=out)
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_REQUEST
    assert torch.equal(out[:5], good[:5]) and torch.equal(out[10:], good[10:]) and (out[5:10] == 9.0).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("first", [True, False])
def test_single_tokens_and_a_chunk_in_one_call(dim, first):
    # The row blocks go by the average: a chunk among single tokens runs in blocks that are small for it.
    prefixes, sizes = [7 * i % 311 for i in range(63)], [1] * 63
    prefixes.insert(0 if first else 40, 900)
    sizes.insert(0 if first else 40, 512)
    for window, sinks in ((200, 4), (2 ** 20, 0)):
        b = Batch(prefixes, [chain(n) for n in sizes], window=window, sinks=sinks, dim=dim, kv_heads=8, groups=2, seed=dim)
        read_and_clear_status(DEV)
        check(attend(b), b, f"mixed {dim} {window}")
        assert read_and_clear_status(DEV) == 0


def test_requests_that_overlap_beyond_what_32_bits_count():
    # Every second request holds all rows (each tenth of them the first one only), and the others begin where they end:
    # 2.3 times 2^31 row blocks in all.  Which of them are computed is open, but with a window of one a row that is has its
    # own V row.
    requests, nodes, groups, dim = 106001, 1100, 3000, 8
    cu = torch.zeros(requests + 1, dtype=torch.int32)
    cu[1::2] = nodes
    counts = torch.full((requests,), nodes, dtype=torch.int32)
    counts[::20] = 1
    bias = torch.full((nodes, nodes), -torch.inf).triu(1).reshape(-1)
    gen = torch.Generator(DEV).manual_seed(1)
    k, v = (torch.randn((5, 256, 1, dim), generator=gen, device=DEV).to(BF16) for _ in range(2))
    q = torch.randn((nodes, groups, dim), generator=gen, device=DEV).to(BF16)
    slots = torch.randperm(5 * 256, generator=gen, device=DEV)[:nodes]
    meta = SimpleNamespace(cu_seqlens_q=cu.to(DEV), prefix_lens=torch.zeros(requests, dtype=torch.int32, device=DEV),
                           node_counts=counts.to(DEV), block_tables=torch.zeros((requests, 1), dtype=torch.int32, device=DEV),
                           tree_slots=slots, qq_bias=bias.to(DEV), block_size=256, num_requests=requests, total_queries=nodes,
                           qq_bias_offsets=torch.zeros(requests + 1, dtype=torch.int64, device=DEV))
    out = torch.full_like(q, 9.0)
    read_and_clear_status(DEV)
    packed_window_attention(q, k, v, meta, torch.arange(nodes, device=DEV), 0.3, groups, window=1, out=out)
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_REQUEST
    own = v.view(-1, 1, dim)[slots].expand_as(out)
    assert ((out == own) | (out == 9.0)).all()
