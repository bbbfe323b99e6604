"""The windowed tree attention on the GPU against 64 bits.

Tolerance, derived.  With normalised weights w_k, let S = sum_k w_k |V_k| per output.  A probability is
rounded to the operands' type (bf16 2^-8 of it, f16 2^-11), or for fp32 results kept in terms (bf16 three,
2^-24; f16 two, 2^-22).  f16 probabilities times 2^7, against a sum of at least 2^7, lose at most 2^-25
where they are below the smallest normal: 2^-32 of the sum a key, times the largest |V|.  Scores are sums
of D exact products in fp32, scaled by two roundings, and a bias adds its own rounding: at most
(D + 4) 2^-24 of sum_d |q_d k_d| scale + |bias|; a probability is off by that and by 2^-21 of its exponential, in
the numerator and in the sum.  The sums over n keys and the joins of up to 600 pieces add (n + 600) 2^-24 of S
each.  The store adds half a step of its type.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from jetspec_amd import (_lib, packed_tree_attention, packed_window_attention, read_and_clear_status)
from window_helpers import Batch, chain, check, random_tree

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def attend(b: Batch, **over):
    out_dtype = over.pop("output_dtype", None)
    return packed_window_attention(over.pop("q", b.q), over.pop("k", b.k), over.pop("v", b.v), b.meta,
                                   over.pop("positions", b.positions), b.scale, b.groups, window=b.window, sinks=b.sinks,
                                   output_dtype=out_dtype, **over)


def trees(sizes, seed=0):
    rng = np.random.default_rng(seed)
    return [random_tree(n, rng) for n in sizes]


SHAPES = [
    # prefixes, trees, window, sinks, options
    ([777], [[-1]], 128, 4, {}),
    ([0], [[-1]], 1, 0, {}),
    ([1], [[-1]], 1, 1, {}),
    ([130, 5, 64], trees([1, 1, 1]), 64, 3, {}),
    ([300, 0, 17, 1000], trees([5, 33, 16, 64]), 100, 2, dict(groups=4)),
    ([513], trees([200], 3), 37, 5, dict(groups=2, kv_heads=1)),
    ([90, 400], [chain(150), chain(70)], 40, 0, {}),
    ([90, 400], [chain(150), chain(70)], 40, 7, dict(groups=7, kv_heads=1)),
    ([3, 0], [chain(90), chain(40)], 8, 30, dict(groups=1)),
    ([260], trees([40], 5), 5000, 0, dict(groups=5)),
    ([260], trees([40], 5), 200, 300, dict(groups=16, kv_heads=1)),
    ([100] * 70, trees([1 + i % 5 for i in range(70)], 7), 20, 2, dict(groups=3, kv_heads=1)),
    ([10], [chain(400)], 2 ** 31 - 1, 2 ** 31 - 1, dict(kv_heads=1)),
]


@pytest.mark.parametrize("dim", [8, 64, 72, 128, 256])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_shapes_and_masks(case, dim):
    prefixes, nodes, window, sinks, options = SHAPES[case]
    b = Batch(prefixes, nodes, window=window, sinks=sinks, dim=dim, seed=case, page=[16, 48, 1, 256][case % 4], **options)
    read_and_clear_status(DEV)
    check(attend(b), b, f"case {case} dim {dim}")
    assert read_and_clear_status(DEV) == 0


@pytest.mark.parametrize("dtype, out", [(BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_types(dtype, out, dim):
    for gain, sizes in ((1.0, [1, 1, 1]), (4.0, [7, 64, 20]), (2.0, [90, 1, 70])):
        b = Batch([700, 90, 300], trees(sizes), window=150, sinks=4, dim=dim, dtype=dtype, gain=gain, seed=dim)
        check(attend(b, output_dtype=out), b, f"{dtype} {out} {dim} {sizes}")


@pytest.mark.parametrize("prefix", [31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257])
def test_lengths_around_tiles_and_steps(prefix):
    for window in (prefix - 1, prefix, prefix + 1, prefix + 2, 32, 64):
        for sinks in (0, 1, 32):
            b = Batch([prefix], trees([3]), window=window, sinks=sinks, seed=prefix, groups=2)
            check(attend(b), b, f"{prefix} {window} {sinks}")


@pytest.mark.parametrize("dim", [64, 128])
def test_every_shape_of_launch(dim):
    # Row blocks of 32 to 256, keys split over many workgroups, few and none.
    for requests, prefix, sizes, window in ((1, 9000, [1], 4096), (1, 20000, [30], 2 ** 20), (3, 5000, [40] * 3, 3000),
                                            (6, 2500, [100] * 6, 2000), (2, 40, [300] * 2, 64), (40, 600, [1] * 40, 512)):
        b = Batch([prefix] * requests, trees(sizes, requests), window=window, sinks=4, dim=dim, kv_heads=2, groups=4, page=48)
        check(attend(b), b, f"{requests} {prefix} {window} {dim}")


@pytest.mark.parametrize("dim, out", [(64, BF16), (64, F32), (128, BF16), (256, BF16), (256, F32)])
def test_many_short_requests(dim, out):
    # More blocks than the chip holds, of few rows.
    sizes, prefixes = [1 + i % 4 for i in range(140)], [(37 * i) % 170 for i in range(140)]
    b = Batch(prefixes, trees(sizes, 9), window=90, sinks=2, dim=dim, kv_heads=8, groups=2, seed=dim)
    check(attend(b, output_dtype=out), b, f"{dim} {out}")


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_parts_of_unlike_requests(dim):
    # Keys cut into parts by each request's length: up to 64 requests, above, and one long among short ones.
    for prefixes, sizes in (([5000, 1, 700, 33], [3, 9, 40, 1]), ([0] * 20 + [6000] + [3] * 20, [2] * 41),
                            ([300 + 13 * i for i in range(70)], [1 + i % 3 for i in range(70)]), ([9000, 9000], [150, 20])):
        b = Batch(prefixes, trees(sizes, 11), window=4000, sinks=4, dim=dim, kv_heads=1, groups=4, page=32, seed=dim)
        check(attend(b), b, f"{dim} {len(sizes)}")


@pytest.mark.parametrize("page", [1, 16, 48])
@pytest.mark.parametrize("groups", [1, 2, 3, 8])
def test_long_blocks(groups, page):
    # Keys of many tables, blocks of 128 nodes and of 256 rows, the first tokens before and inside the tree.
    for prefixes, sizes, window, sinks in (([2300], [300], 1500, 5), ([1200, 0], [300, 270], 2000, 1300), ([40], [600], 2 ** 20, 0)):
        b = Batch(prefixes, [chain(n) for n in sizes], window=window, sinks=sinks, groups=groups, kv_heads=1, dim=64, page=page,
                  seed=groups)
        check(attend(b), b, f"{groups} {page} {prefixes}")


@pytest.mark.parametrize("groups, dtype", [(1, BF16), (2, F16), (4, BF16)])
def test_finite_biases_in_long_trees(groups, dtype):
    # A few rows' biases are neither zero nor -inf, in tiles that are whole otherwise.
    sizes, rng = [300, 130], np.random.default_rng(groups)
    bias = []
    for n in sizes:
        x = np.where(np.tril(np.ones((n, n))) > 0, 0.0, -np.inf).astype(np.float32)
        x[::37] += np.where(rng.random(x[::37].shape) < 0.5, 0.0, rng.normal(size=x[::37].shape)).astype(np.float32)
        bias.append(x)
    for window, sinks in ((2000, 4), (90, 50)):
        b = Batch([1300, 20], [chain(n) for n in sizes], window=window, sinks=sinks, groups=groups, kv_heads=1, dtype=dtype,
                  seed=groups, bias=np.concatenate([x.reshape(-1) for x in bias]))
        check(attend(b), b, f"{groups} {window}")


def test_rows_that_see_nothing_and_finite_biases():
    sizes = [6, 40]
    rng = np.random.default_rng(1)
    bias = [np.where(rng.random((n, n)) < 0.4, -np.inf, rng.normal(size=(n, n)) * 3).astype(np.float32) for n in sizes]
    bias[0][3] = -np.inf     # with no prefix: row 3 sees nothing
    bias[1][7, :8] = np.finfo(np.float32).min
    b = Batch([0, 100], trees(sizes), window=9, sinks=0, seed=2, bias=np.concatenate([x.reshape(-1) for x in bias]))
    got = attend(b)
    check(got, b, "biases")
    assert torch.equal(got[3], torch.zeros_like(got[3]))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_infinities_and_nans_stay_with_the_rows_that_see_them(value, dtype):
    # Key 60 leaves the window of the later rows, node 2 is no ancestor of every node; both have such elements.
    b = Batch([100], [[-1, 0, 1, 0, 3, 4, 5, 6]], window=43, sinks=0, seed=3, dtype=dtype)
    j, slots, own = b.keys[0]
    for slot in (int(slots[list(j).index(60)]), int(own[2])):
        b.v.view(-1, *b.v.shape[2:])[slot, 0, 5] = value
        b.k.view(-1, *b.k.shape[2:])[slot, 1] = value
    got = attend(b).float().cpu().numpy()
    # Row at position P sees key 60 iff P - 60 < 43; node 2 is seen by itself alone.
    seen = np.array([100 + d - 60 < 43 for d in b.depths[0]])
    seen[2] = True
    assert not seen.all() and seen.any()
    finite = np.isfinite(got).all(-1)
    assert finite[~seen].all()
    assert not finite[seen][:, :4].any()       # KV head 0: the value row
    clean = Batch([100], [[-1, 0, 1, 0, 3, 4, 5, 6]], window=43, sinks=0, seed=3, dtype=dtype)
    want, bound = clean.expected(dtype)
    assert (np.abs(got - want) <= bound)[~seen].all()


def test_strides_types_of_positions_and_a_given_output():
    b = Batch([300, 77], trees([20, 9]), window=64, sinks=2, seed=4, dim=64)
    want = attend(b)
    rows, heads, dim = b.q.shape
    wide = torch.full((rows, heads + 3, dim + 16), 7.0, dtype=BF16, device=DEV)
    wide[:, 2:heads + 2, 8:dim + 8] = b.q
    k = torch.full((b.k.shape[0], b.k.shape[2], b.k.shape[1], dim + 8), float("nan"), dtype=BF16, device=DEV)
    v = k.clone()
    k[..., :dim], v[..., :dim] = b.k.transpose(1, 2), b.v.transpose(1, 2)
    out = torch.full((rows + 4, heads, dim + 8), 3.0, dtype=F32, device=DEV)
    apart = torch.zeros((rows, 3), dtype=torch.int32, device=DEV)
    apart[:, 1] = b.positions
    got = attend(b, q=wide[:, 2:heads + 2, 8:dim + 8], k=k[..., :dim].transpose(1, 2), v=v[..., :dim].transpose(1, 2),
                 positions=apart[:, 1], out=out[:rows, :, :dim], output_dtype=F32)
    assert got.data_ptr() == out.data_ptr()
    check(got, b, "strided")
    assert (out[rows:] == 3.0).all() and (out[:, :, dim:] == 3.0).all()
    shifted = torch.empty(b.q.numel() + 1, dtype=BF16, device=DEV)[1:].view(b.q.shape)   # off 16 bytes
    shifted.copy_(b.q)
    assert torch.equal(attend(b, q=shifted), want)


def test_a_window_over_everything_is_the_tree_attention():
    b = Batch([500, 40], trees([30, 64]), window=10 ** 6, seed=5, page=32)
    whole = packed_tree_attention(b.q, b.k, b.v, b.meta, b.scale, b.groups)
    check(whole, b, "tree attention")
    check(attend(b), b, "window")


def test_rows_that_no_request_counts_are_left_alone():
    b = Batch([50, 60], trees([5, 5]), window=30, seed=6)
    b.meta.node_counts.copy_(torch.tensor([5, 3], dtype=torch.int32))
    out = torch.full_like(b.q, 9.0)
    read_and_clear_status(DEV)
    # The bias of the second request keeps its rows of five.
    b.meta.node_counts.copy_(torch.tensor([5, 0], dtype=torch.int32))
    attend(b, out=out)
    assert (out[5:] == 9.0).all() and not (out[:5] == 9.0).all(-1).any()
    assert read_and_clear_status(DEV) == 0


def test_bad_requests_pages_and_positions_are_reported():
    def fresh():
        read_and_clear_status(DEV)
        return Batch([50, 60, 70], trees([5, 5, 5]), window=30, seed=7)

    good = attend(fresh())
    for field, value in (("prefix_lens", 10 ** 6), ("prefix_lens", -1), ("node_counts", -2), ("node_counts", 6)):
        b = fresh()
        getattr(b.meta, field)[1] = value
        out = torch.full_like(b.q, 9.0)
        attend(b, out=out)
        assert read_and_clear_status(DEV) & _lib.TV_STATUS_BAD_REQUEST, field
        assert torch.equal(out[:5], good[:5]) and torch.equal(out[10:], good[10:]) and (out[5:10] == 9.0).all()
    b = fresh()
    b.meta.qq_bias_offsets[1] = b.meta.qq_bias.numel() - 3
    attend(b)
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_REQUEST
    for page in (-1, b.k.shape[0], 2 ** 31 - 1):
        b = fresh()
        b.meta.block_tables[1, 3] = page       # keys 48 to 59, in the window
        got = attend(b)
        assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_PAGE
        assert torch.equal(got[:5], good[:5]) and torch.equal(got[10:], good[10:]) and got.isfinite().all()
        j, slots, own = b.keys[1]
        b.keys[1] = (j[j < 48], slots[j < 48], own)
        check(got, b, "a page less")
    for slot in (-5, 2 ** 40, b.k.shape[0] * 16):
        b = fresh()
        b.meta.tree_slots[7] = slot
        got = attend(b)
        assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_PAGE and got.isfinite().all()
    for position, nearest in ((-4, 60), (2 ** 33 + 61, 62), (2 ** 31 - 1, 62), (59, 60), (63, 62)):
        b = fresh()
        p = b.positions.clone()
        p[7] = position
        got = attend(b, positions=p)
        assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_POSITION
        assert torch.equal(got[:5], good[:5]) and got.isfinite().all()
        if position < 2 ** 32:
            p[7] = nearest
            assert torch.equal(got, attend(b, positions=p))


def test_empty_batches():
    b = Batch([5], [[-1]], window=3)
    b.meta.node_counts.zero_()
    out = torch.full_like(b.q, 9.0)
    attend(b, out=out)
    assert (out == 9.0).all()


def test_captured_calls_follow_the_staged_batch():
    sizes = [8, 8, 8]
    a = Batch([400, 30, 90], trees(sizes, 1), window=50, sinks=3, seed=8)
    rounds = [Batch([p, q, r], trees(sizes, s), window=50, sinks=3, seed=s) for s, (p, q, r) in
              enumerate([(400, 30, 90), (3, 399, 0), (128, 256, 64)], 20)]
    pages = max(x.k.shape[0] for x in (a, *rounds))
    width = max(x.meta.block_tables.shape[1] for x in (a, *rounds))
    pool = [torch.full((pages, *a.k.shape[1:]), float("nan"), dtype=BF16, device=DEV) for _ in range(2)]
    assert width == a.meta.block_tables.shape[1]

    def stage(x):
        for name in ("prefix_lens", "tree_slots", "qq_bias"):
            getattr(a.meta, name).copy_(getattr(x.meta, name))
        a.meta.block_tables.fill_(-1)
        a.meta.block_tables[:, :x.meta.block_tables.shape[1]].copy_(x.meta.block_tables)
        a.q.copy_(x.q)
        a.positions.copy_(x.positions)
        for mine, theirs in zip(pool, (x.k, x.v)):
            mine.fill_(float("nan"))
            mine[:theirs.shape[0]].copy_(theirs)

    stage(rounds[0])
    attend(a, k=pool[0], v=pool[1])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):   # two graphs beside each other
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(attend(a, k=pool[0], v=pool[1]))
        graphs.append(g)
    for x in rounds * 2:
        stage(x)
        eager = attend(a, k=pool[0], v=pool[1])
        for o in outs:
            o.fill_(5.0)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, eager) for o in outs)
        check(eager, x, "staged")


def test_two_streams_at_once():
    batches = [Batch([3000], trees([4], s), window=2500, sinks=4, seed=s) for s in (30, 31)]
    want = [attend(b) for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    for _ in range(5):
        got = []
        for b, s in zip(batches, streams):
            with torch.cuda.stream(s):
                got.append(attend(b))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_offsets_past_32_bits():
    # The pool's last pages lie 8 GiB from its start; the slots of the tree in its first.
    b = Batch([100], trees([6]), window=70, sinks=2, seed=9, kv_heads=2, dim=128)
    page_elems = b.k[0].numel()
    pages = (1 << 32) // page_elems + 8
    shift = pages - b.k.shape[0]
    big = [torch.empty((pages, *b.k.shape[1:]), dtype=BF16, device=DEV) for _ in range(2)]
    for mine, theirs in zip(big, (b.k, b.v)):
        mine[shift:].copy_(theirs)
        mine[:b.k.shape[0]].copy_(theirs)
    want = attend(b)
    t = b.meta.block_tables
    t.copy_(torch.where((t >= 0) & (t < b.k.shape[0]), t + shift, t))
    assert torch.equal(attend(b, k=big[0], v=big[1]), want)
    b.meta.tree_slots.add_(shift * b.page)
    assert torch.equal(attend(b, k=big[0], v=big[1]), want)
