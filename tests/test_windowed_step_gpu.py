"""A verification step of a windowed model: each layer rotates and appends its tree's keys and attends over its
window, then the accepted path's tokens get their log probabilities.  Each result is held to 64 bits with the
bounds that the operators' own tests derive, eager and replayed.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from jetspec_amd import (accept_batch_device, greedy_argmax, packed_window_attention, read_and_clear_status,
                         rotary_frequencies, rotary_scatter, rotary_scatter_prevalidated, token_logprobs)
from test_logprobs_gpu import check as check_logprobs
from test_rotary_gpu import close, turned
from window_helpers import Batch, check, depths_of, random_tree

pytestmark = pytest.mark.gpu
DEV = "cuda"
LAYERS, DEPTH = 2, 4


class Step:
    """Two layers' caches of one batch; the heads of the last layer's result are the logits."""

    def __init__(self, prefixes, sizes, seed, heads=(2, 4), interleaved=False):
        rng = np.random.default_rng(seed)
        self.trees = [random_tree(n, rng) for n in sizes]
        self.layers = [Batch(prefixes, self.trees, window=70, sinks=4, kv_heads=heads[0], groups=heads[1], seed=seed)
                       for _ in range(LAYERS)]
        for n, layer in enumerate(self.layers):     # one table of pages for all layers, as in an engine
            gen = torch.Generator(device=DEV).manual_seed(100 * seed + n)
            for pool in (layer.k, layer.v):
                pool.copy_(torch.where(pool.isnan(), pool, torch.randn(pool.shape, generator=gen, device=DEV).to(pool.dtype)))
        first = self.layers[0]
        self.meta, self.positions, self.interleaved = first.meta, first.positions, interleaved
        self.q = first.q.clone()
        self.kv = [[torch.randn((first.q.shape[0], heads[0], 128), generator=gen, device=DEV).to(first.q.dtype)
                    for _ in range(2)] for _ in range(LAYERS)]
        self.frequencies = rotary_frequencies(128, base=1e6, factor=4.0, original_length=256, device=DEV)
        self.parents = torch.as_tensor(np.concatenate(self.trees), device=DEV)
        self.depths = torch.as_tensor(np.concatenate([depths_of(t) for t in self.trees]), device=DEV)
        self.tokens = torch.full_like(self.parents, 3)
        self.starts = np.concatenate([[0], np.cumsum(sizes)[:-1]])

    def run(self, observe=None):
        x = self.q
        for layer, (k, v) in zip(self.layers, self.kv):
            args = (x, k, v, self.positions, self.frequencies, layer.k, layer.v, self.meta.tree_slots)
            if observe:
                q = rotary_scatter(*args, interleaved=self.interleaved)
            else:                                   # as a layer loop calls it
                q = torch.empty_like(x)
                rotary_scatter_prevalidated(*args, q, interleaved=self.interleaved, gain=1.0)
            out = packed_window_attention(q, layer.k, layer.v, self.meta, self.positions, layer.scale, layer.groups,
                                          window=layer.window, sinks=layer.sinks)
            if observe:
                observe(layer, x, k, v, q, out)
            x = out
        logits = x.view(x.shape[0], -1)
        cu = self.meta.cu_seqlens_q
        greedy, paths, lengths, bonus = accept_batch_device(logits, self.tokens, self.parents, self.depths, cu, DEPTH)
        rows = torch.where(paths >= 0, paths + cu[:-1, None], -1).view(-1)
        emitted = torch.where(rows >= 0, greedy[rows.clamp(min=0).long()], -1)
        return (logits, paths, lengths, emitted, *token_logprobs(logits, emitted, top=5, rows=rows))

    def draft(self):
        """Drafts what the model says for the first child of each node, so that paths are accepted."""
        greedy = greedy_argmax(self.run()[0]).cpu().numpy()
        tokens = np.full(greedy.shape, -5)
        for start, tree in zip(self.starts, self.trees):
            seen = set()
            for node, up in enumerate(tree):
                if up >= 0 and up not in seen:
                    seen.add(up)
                    tokens[start + node] = greedy[start + up]
        self.tokens.copy_(torch.as_tensor(np.maximum(tokens, 0), device=DEV))


@pytest.mark.parametrize("interleaved", [False, True])
def test_a_step_of_two_layers(interleaved):
    s = Step([300, 0, 41], [17, 5, 40], seed=3, interleaved=interleaved)
    read_and_clear_status(DEV)
    s.draft()

    def observe(layer, x, k, v, q, out):
        slots = s.meta.tree_slots.long()
        for got, given, moves in ((q, x, True), (layer.k.flatten(0, 1)[slots], k, True), (layer.v.flatten(0, 1)[slots], v, False)):
            if moves:
                close(got, turned(given, s.positions, s.frequencies, interleaved, 1.0), "rotation")
            else:
                assert torch.equal(got, given)
        layer.q = q
        check(out, layer, "attention")

    logits, paths, lengths, emitted, logp, entropy, ids, values = s.run(observe)
    assert read_and_clear_status(DEV) == 0
    assert int(lengths.max()) > 1    # something was accepted
    rows = torch.where(paths >= 0, paths + s.meta.cu_seqlens_q[:-1, None], -1).view(-1)
    live = rows >= 0
    check_logprobs(logits, emitted[live], 5, rows=rows[live], label="accepted")
    # Greedy decoding: the emitted token is the first alternative; padding is zero.
    assert torch.equal(ids[live, 0], emitted[live]) and torch.equal(values[live, 0], logp[live])
    assert (logp[~live] == 0).all() and (entropy[~live] == 0).all() and (ids[~live] == -1).all()


def test_a_captured_step_follows_its_inputs():
    s = Step([300, 90, 41], [16, 16, 16], seed=5)
    s.draft()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = s.run()
    for seed in (6, 7, 8):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        for x in (s.q, *[t for pair in s.kv for t in pair]):
            x.copy_(torch.randn(x.shape, generator=gen, device=DEV))
        s.draft()
        for layer in s.layers:      # what the step appends is written by the replay itself
            layer.k.flatten(0, 1)[s.meta.tree_slots.long()] = float("nan")
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in held]
        eager = s.run()
        assert all(torch.equal(a, b) for a, b in zip(replayed, eager)), seed
