"""The e4m3 tree attention where offsets pass 32 bits: biases of 2^31 elements and prefixes of millions of keys."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from jetspec_amd import PackedTreeMetadata, packed_tree_attention_e4m3, read_and_clear_status
from e4m3_helpers import VALUES

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn


def metadata(prefixes, counts, tables, slots, bias, page):
    """The fields of a batch whose masks are too large to validate on the host."""
    cu = np.concatenate([[0], np.cumsum(counts)])
    request = np.repeat(np.arange(len(counts)), counts)
    width = max(1, *map(len, tables))
    padded = np.full((len(tables), width), -1)
    for row, table in zip(padded, tables):
        row[:len(table)] = table

    def on(values, kind=torch.int32):
        return torch.as_tensor(np.asarray(values), dtype=kind, device=DEV)
    return PackedTreeMetadata(
        cu_seqlens_q=on(cu), query_to_request=on(request), query_local_row=on(np.arange(cu[-1]) - cu[request]),
        prefix_lens=on(prefixes), block_tables=on(padded), tree_slots=on(slots, torch.int64), qq_bias=bias,
        qq_bias_offsets=on(np.concatenate([[0], np.cumsum(np.square(np.asarray(counts, dtype=np.int64)))]), torch.int64),
        node_counts=on(counts), block_size=page, prefix_lengths=tuple(prefixes), query_offsets=tuple(map(int, cu)),
        node_counts_host=tuple(counts), block_tables_host=tuple(map(tuple, tables)), tree_slot_ids=tuple(map(int, slots)),
        request_ids=tuple(range(len(counts))))


def pools(gen, shape):
    codes = [torch.randint(0, 255, shape, generator=gen, dtype=torch.uint8, device=DEV) for _ in range(2)]
    for c in codes:
        c.masked_fill_((c & 127) == 127, 0x38)   # no NaN
    return [c.view(E4M3) for c in codes], [torch.rand(shape[:3], generator=gen, device=DEV) * 0.02 for _ in range(2)]


def check_row(got, q, codes, scales, slots, scale):
    """One row over its keys in 64 bits.  FP32 output: scores are off by (D + 4) 2^-24 of the sum of the sizes of
    their products, probabilities by twice that and 2^-21, sums over the keys and pieces by (n + 600) 2^-24."""
    heads, dim = codes[0].shape[2:]
    table = torch.as_tensor(VALUES, device=DEV)
    groups = q.shape[0] // heads
    for h in {0, heads - 1}:
        k, v = (table[c.view(torch.uint8).view(-1, heads, dim)[slots, h].long()] * s.view(-1, heads)[slots, h].double()[:, None]
                for c, s in zip(codes, scales))
        mine = q[h * groups:(h + 1) * groups].double()
        w = torch.softmax(torch.mm(mine, k.t().contiguous()) * scale, -1)
        size = torch.mm(mine.abs(), k.abs().t().contiguous()).amax(-1, keepdim=True) * scale
        slack = 2 * ((dim + 4) * 2.0 ** -24 * size + 2.0 ** -21) + 2.0 ** -26 + 2 * (slots.numel() + 600) * 2.0 ** -24
        off = (got[h * groups:(h + 1) * groups].double() - torch.mm(w, v)).abs()
        allowed = slack * torch.mm(w, v.abs()) * (1 + 2.0 ** -6) + 2.0 ** -24 * torch.mm(w, v).abs()
        assert bool((off <= allowed).all()), float((off - allowed).max())


def test_biases_past_two_to_the_31():
    page, counts, prefixes = 64, [46400, 60], [130, 70]
    assert counts[0] ** 2 > 2 ** 31
    gen = torch.Generator(device=DEV).manual_seed(0)
    blocks = -(-sum(counts) // page) + 6
    codes, scales = pools(gen, (blocks, page, 1, 64))
    slots = np.arange(sum(counts)) + 6 * page
    bias = torch.zeros(sum(n * n for n in counts), device=DEV)
    at = 0
    for n in counts:
        square = bias[at:at + n * n].view(n, n)
        square.masked_fill_(torch.ones((n, n), dtype=torch.bool, device=DEV).triu_(1), -torch.inf)
        square[:, 5::7] = -torch.inf
        at += n * n
        del square
    meta = metadata(prefixes, counts, [[0, 1, 2], [3, 4]], slots, bias, page)
    q = torch.randn((sum(counts), 2, 64), generator=gen, device=DEV).bfloat16()
    got = packed_tree_attention_e4m3(q, *codes, *scales, meta, 0.125, 2, output_dtype=torch.float32)
    assert read_and_clear_status(DEV) == 0
    for r, table in enumerate(([0, 1, 2], [3, 4])):
        for i in (0, 5, counts[r] // 2, counts[r] - 2, counts[r] - 1):
            p = np.arange(prefixes[r])
            nodes = np.arange(i + 1)
            nodes = nodes[nodes % 7 != 5]
            first = sum(counts[:r])
            keys = np.concatenate([np.asarray(table)[p // page] * page + p % page, slots[first + nodes]])
            check_row(got[first + i], q[first + i], codes, scales, torch.as_tensor(keys, device=DEV), 0.125)


@pytest.mark.parametrize("dim, page, nodes", [(128, 256, 1), (128, 16, 70), (64, 128, 70), (256, 64, 3)])
def test_prefixes_of_millions_of_keys(dim, page, nodes):
    gen = torch.Generator(device=DEV).manual_seed(1)
    prefix, heads = 1_500_007, 8 * 128 // dim
    blocks = -(-prefix // page) + 2 + -(-nodes // page)
    codes, scales = pools(gen, (blocks, page, heads, dim))
    assert codes[0].numel() > 1 << 30
    order = np.random.default_rng(0).permutation(blocks)
    table, scratch = order[:-(-prefix // page)], order[-(-nodes // page):]
    slots = (scratch[:, None] * page + np.arange(page)).reshape(-1)[:nodes]
    bias = torch.zeros((nodes, nodes), device=DEV).masked_fill_(
        torch.ones((nodes, nodes), dtype=torch.bool, device=DEV).triu_(1), -torch.inf)
    meta = metadata([prefix], [nodes], [table.tolist()], slots, bias.view(-1), page)
    q = torch.randn((nodes, 4 * heads, dim), generator=gen, device=DEV).bfloat16()
    got = packed_tree_attention_e4m3(q, *codes, *scales, meta, 0.1, 4, output_dtype=torch.float32)
    assert read_and_clear_status(DEV) == 0
    p = np.arange(prefix)
    for i in {0, nodes - 1}:
        keys = np.concatenate([table[p // page] * page + p % page, slots[:i + 1]])
        check_row(got[i], q[i], codes, scales, torch.as_tensor(keys, device=DEV), 0.1)
