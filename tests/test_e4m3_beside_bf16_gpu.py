"""The e4m3 tree attention beside the bf16 one, over the same values."""
from __future__ import annotations

import pytest
import torch

from jetspec_amd import packed_tree_attention, read_and_clear_status
from test_e4m3_attention_gpu import BF16, DEV, Batch, trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_agrees(dim):
    """packed_tree_attention over the same values in bf16 pools, with scores that spread over several units.

    Each result is within the formula's tolerance: ours as Batch.check derives it, theirs with a probability and
    the sum of the probabilities each off by half a bf16 step, 2^-8, at most.
    """
    batch = Batch([900, 40, 0], trees([30, 64, 9]), page=32, dim=dim)
    batch.ks.fill_(1.0)
    batch.vs.fill_(1.0)
    for t in (batch.k, batch.v):
        t.view(torch.uint8)[t.view(torch.uint8) & 127 == 127] = 0
    batch.scale = 0.012 / dim ** 0.5   # codes of a standard deviation of about 165
    wide = [t.to(BF16) for t in (batch.k, batch.v)]   # a code is a bf16 value exactly
    theirs = packed_tree_attention(batch.q, *wide, batch.meta, batch.scale, 4)
    ours = batch.check(BF16)
    heads = batch.k.shape[2]
    for r in range(3):
        rows, prefix, n = batch.meta.request_slice(r), batch.prefixes[r], batch.counts[r]
        keys = torch.as_tensor(batch.keys[r], device=DEV)
        first = int(batch.meta.qq_bias_offsets[r])
        bias = batch.meta.qq_bias[first:first + n * n].view(n, n).double().repeat_interleave(4, 0)
        for h in range(heads):
            mine = slice(4 * h, 4 * h + 4)
            q = batch.q[rows, mine].double().reshape(4 * n, -1)
            k, v = batch.rows(batch.k, batch.ks, keys, h), batch.rows(batch.v, batch.vs, keys, h)
            score = torch.mm(q, k.t().contiguous()) * batch.scale
            score[:, prefix:] += bias
            w = torch.softmax(score, -1)
            spread = torch.mm(w, v.abs())
            if r == 0:   # far from uniform: the largest weight of a typical row is many times the mean
                assert float((w.amax(-1) * keys.numel()).median()) > 8
            # Probability and store of ours; probability, sum and store of theirs; fp32 and second order.
            allowed = (2 + 3) * 2.0 ** -8 * 1.05 * spread
            apart = (ours[rows, mine].double() - theirs[rows, mine].double()).abs().reshape(spread.shape)
            assert bool((apart <= allowed).all()), (r, h, float((apart / spread).max()))
            # What the bound can tell: the same values under uniform weights, or under their neighbours' weights.
            if r == 0:
                for other in (v.mean(0, keepdim=True).expand_as(spread), torch.mm(w.roll(1, -1), v)):
                    assert float(((other - theirs[rows, mine].double().reshape(spread.shape)).abs() > allowed).double().mean()) > 0.5
    assert read_and_clear_status(DEV) == 0
