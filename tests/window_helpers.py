"""Windowed tree attention in 64 bits and the batches that its tests share (no code of the package's kernels)."""
from __future__ import annotations

import numpy as np
import torch

from jetspec_amd import PackedTreeMetadata, workloads

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # half a step


def depths_of(parents) -> np.ndarray:
    depth = np.zeros(len(parents), dtype=np.int64)
    for node, up in enumerate(parents):
        depth[node] = 0 if up < 0 else depth[up] + 1
    return depth


def chain(n: int) -> list[int]:
    return list(range(-1, n - 1))


def random_tree(n: int, rng) -> list[int]:
    return [-1] + [int(rng.integers(max(0, node - 12), node)) for node in range(1, n)]


class Batch:
    """A packed batch: its pools hold NaN wherever no row may look, and table entries of pages that no row
    sees are no pages."""

    def __init__(self, prefixes, trees, *, window, sinks=0, dim=128, kv_heads=2, groups=4, page=16, dtype=torch.bfloat16,
                 gain=1.0, seed=0, device="cuda", bias=None):
        rng = np.random.default_rng(seed)
        gen = torch.Generator(device=device).manual_seed(seed)
        counts = [len(t) for t in trees]
        total = sum(counts)
        self.depths = [depths_of(t) for t in trees]
        self.window, self.sinks, self.groups, self.counts, self.prefixes, self.page = window, sinks, groups, counts, prefixes, page
        need = [-(-p // page) for p in prefixes]
        scratch = -(-total // page) + 1
        order = rng.permutation(sum(need) + scratch + 2)
        tables, at = [], 0
        for n in need:
            tables.append([int(x) for x in order[at:at + n]])
            at += n
        free = (order[at:at + scratch, None] * page + np.arange(page)).reshape(-1)
        slots = free[rng.permutation(free.size)[:total]]
        parts = np.split(slots, np.cumsum(counts)[:-1])
        masks = [torch.as_tensor(workloads.ancestor_mask(t), device=device) for t in trees]
        self.meta = PackedTreeMetadata.build(prefixes, tables, [torch.as_tensor(s, device=device) for s in parts], masks, page)
        if bias is not None:
            self.meta.qq_bias.copy_(torch.as_tensor(bias, device=device))
        self.positions = torch.as_tensor(np.concatenate([p + d for p, d in zip(prefixes, self.depths)]), device=device)
        # What some row sees: first tokens, and the prefix from its earliest row's window on.
        self.keys, entries = [], self.meta.block_tables.cpu().numpy().copy()
        for r, (p, tab, part, depth) in enumerate(zip(prefixes, tables, parts, self.depths)):
            j = np.arange(p)
            j = j[(j < sinks) | (j > p + depth.min() - window)]
            pages = np.asarray(tab, dtype=np.int64)
            self.keys.append((j, pages[j // page] * page + j % page if len(j) else j, part))
            unseen = np.setdiff1d(np.arange(len(tab)), j // page)
            entries[r, unseen] = rng.choice([-1, -7, 1 << 30], size=len(unseen))
        self.meta.block_tables.copy_(torch.as_tensor(entries, device=device))
        shape = (order.size, page, kv_heads, dim)
        self.k, self.v = (torch.full(shape, float("nan"), dtype=dtype, device=device) for _ in range(2))
        live = torch.as_tensor(np.concatenate([np.concatenate([s, part]) for _, s, part in self.keys]), device=device)
        for pool, size in ((self.k, 1.0), (self.v, 0.7)):
            rows = torch.randn((live.numel(), kv_heads, dim), generator=gen, device=device) * size
            pool.view(-1, kv_heads, dim)[live] = rows.to(dtype)
        self.q = (torch.randn((total, kv_heads * groups, dim), generator=gen, device=device) * gain).to(dtype)
        self.scale = dim ** -0.5

    def expected(self, out_dtype):
        """64-bit results [rows, heads, dim] and the bound of each, derived in test_window_attention_gpu.py."""
        heads, dim = self.k.shape[2:]
        bias, offsets = self.meta.qq_bias.cpu().numpy().astype(np.float64), self.meta.qq_bias_offsets.cpu().numpy()
        q = self.q.double().cpu().numpy()
        pools = [p.reshape(-1, heads, dim).double().cpu().numpy() for p in (self.k, self.v)]
        kind = self.q.dtype
        if out_dtype is kind:
            terms = STEP[kind]
        else:
            terms = 2.0 ** -24 if kind is torch.bfloat16 else 2.0 ** -22
        outs, bounds, row0 = [], [], 0
        for r, (n, (j, prefix_slots, own)) in enumerate(zip(self.counts, self.keys)):
            slots = np.concatenate([prefix_slots, own])
            at = np.concatenate([j, self.prefixes[r] + self.depths[r]])
            mine = self.prefixes[r] + self.depths[r]
            b = np.concatenate([np.zeros((n, len(j))), np.where(np.tril(np.ones((n, n))) > 0,
                                                                bias[offsets[r]:offsets[r] + n * n].reshape(n, n), -np.inf)], 1)
            seen = ((mine[:, None] - at[None] < self.window) | (at[None] < self.sinks)) & (b != -np.inf)
            b = np.where(seen, b, -np.inf)
            out, bound = np.zeros((n, heads * self.groups, dim)), np.zeros((n, heads * self.groups, dim))
            for h in range(heads * self.groups):
                k, v = (p[slots, h // self.groups] for p in pools)
                rows = q[row0:row0 + n, h]
                with np.errstate(all="ignore"):
                    score = np.where(seen, rows @ k.T * self.scale + np.where(seen, b, 0), -np.inf)
                    top = score.max(1, keepdims=True)
                    w = np.where(seen, np.exp(score - np.where(np.isfinite(top), top, 0)), 0)
                    total = w.sum(1, keepdims=True)
                    w = np.where(total > 0, w / np.where(total > 0, total, 1), 0)
                    clean = np.where(np.isfinite(v), v, 0)
                    out[:, h] = w @ clean
                    odd = (w > 0) @ (~np.isfinite(v)).any(1)   # rows that see a value row that is not finite
                    out[:, h][odd > 0] = np.nan
                    sums = w @ np.abs(clean)
                    delta = (dim + 4) * 2.0 ** -24 * (np.where(seen, (np.abs(rows) @ np.abs(k).T) * abs(self.scale) + np.abs(np.where(seen, b, 0)), 0)).max(1, keepdims=True)
                    relative = terms + 2 * (np.exp(2 * delta) - 1 + 2.0 ** -21) + 2 * (len(slots) + 600) * 2.0 ** -24
                    lost = len(slots) * 2.0 ** -32 * np.abs(clean).max() if kind is torch.float16 and len(slots) else 0.0
                    bound[:, h] = relative * sums + lost + STEP[out_dtype] * np.abs(out[:, h]) + 2.0 ** -126
            # A value below the type's smallest normal is rounded to its fixed steps.
            outs.append(out)
            bounds.append(bound + (2.0 ** -25 if out_dtype is torch.float16 else 0.0))
            row0 += n
        return np.concatenate(outs), np.concatenate(bounds)


def check(got: torch.Tensor, batch: Batch, label: str = "") -> None:
    want, bound = batch.expected(got.dtype)
    have = got.double().cpu().numpy()
    nans = np.isnan(want)
    assert np.array_equal(~np.isfinite(have), nans), f"{label}: NaN rows"
    worst = np.where(nans, 0, np.abs(have - np.where(nans, 0, want)) / bound).max()
    print(f"[{label}] worst error {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0, f"{label}: {worst} of the bound"
