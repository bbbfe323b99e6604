"""The fused norm and the e4m3 append where element offsets pass 32 bits: rows sampled against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import e4m3_helpers
from jetspec_amd import qk_norm_rope_scatter_prevalidated, read_and_clear_status, store_kvcache_e4m3
from test_qk_norm_gpu import BF16, DEV, E4M3, assert_near, turned

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim", [128, 90])
def test_offsets_past_two_to_the_31(dim, e4m3):
    rows, q_heads, kv_heads, page = 2 ** 22 // dim * 16 + 77, 32, 2, 16
    gen = torch.Generator(device=DEV).manual_seed(dim)
    qkv = torch.empty((rows, q_heads + 2 * kv_heads, dim), dtype=BF16, device=DEV)
    assert qkv.numel() > 2 ** 31
    qkv[:4096].normal_(generator=gen)
    qkv[4096:] = qkv[(torch.arange(4096, rows, device=DEV) * 7) % 4096]
    # A pool whose last pages lie past 2^32 bytes; only the sampled rows go there.
    pages = 2 ** 32 // (page * kv_heads * dim) + 9
    pool = [torch.zeros((pages, page, kv_heads, dim), dtype=torch.uint8 if e4m3 else BF16, device=DEV) for _ in range(2)]
    slots = torch.arange(rows, device=DEV)
    sample = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device=DEV)
    slots[sample] = pages * page - 1 - torch.arange(5, device=DEV) * 3
    q, k, v = qkv[:, :q_heads], qkv[:, q_heads:q_heads + kv_heads], qkv[:, q_heads + kv_heads:]
    angle = torch.arange(50, device=DEV).double()[:, None] * torch.logspace(0, -4, dim // 2, dtype=torch.float64, device=DEV)
    cache = torch.cat([angle.cos(), angle.sin()], 1).float()
    positions = torch.arange(rows, device=DEV) % 50
    weight = (1 + torch.rand((2, dim), generator=gen, device=DEV)).to(BF16)
    out = torch.zeros((rows, q_heads, dim), dtype=BF16, device=DEV)
    scales = [torch.zeros((pages, page, kv_heads), device=DEV) for _ in range(2)] if e4m3 else [None, None]
    pools = [p.view(E4M3) for p in pool] if e4m3 else pool
    qk_norm_rope_scatter_prevalidated(q, k, v, weight[0], weight[1], positions, cache, *pools, slots, out, k_scale=scales[0],
                                      v_scale=scales[1])
    at = slots[sample]
    assert_near(out[sample], *turned(q[sample], weight[0], cache, positions[sample], 1e-6), BF16)
    value, size = turned(k[sample], weight[1], cache, positions[sample], 1e-6)
    if not e4m3:
        assert_near(pools[0].view(-1, kv_heads, dim)[at], value, size, BF16)
        assert torch.equal(pools[1].view(-1, kv_heads, dim)[at], v[sample])
    else:
        def held(i):
            return e4m3_helpers.VALUES[pool[i].view(-1, kv_heads, dim)[at].cpu().numpy()], scales[i].view(-1, kv_heads)[at].cpu().numpy()
        codes, expect = e4m3_helpers.quantise(v[sample].float().cpu().numpy())
        np.testing.assert_array_equal(held(1)[0], e4m3_helpers.VALUES[codes])
        np.testing.assert_array_equal(held(1)[1], expect)
        got = held(0)[0] * held(0)[1][..., None].astype(np.float64)
        early = 20 * 2.0 ** -24 * size
        assert np.all(np.abs(got - value) <= (2.0 ** -4 + 2.0 ** -20) * (np.abs(value) + early) + early
                      + 2.0 ** -10 * held(0)[1][..., None])
        # The append into the same far slots.
        for p, s in zip(pool, scales):
            p.zero_()
            s.zero_()
        store_kvcache_e4m3(v, k, *pools, *scales, slots)
        for i, rows_ in enumerate((v, k)):
            codes, expect = e4m3_helpers.quantise(rows_[sample].float().cpu().numpy())
            np.testing.assert_array_equal(held(i)[0], e4m3_helpers.VALUES[codes])
            np.testing.assert_array_equal(held(i)[1], expect)
    assert read_and_clear_status(DEV) == 0
