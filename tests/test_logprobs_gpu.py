"""token_logprobs on the GPU against 64 bits.

Tolerance, derived.  An exponent d = c x - R is one rounding of a number of at most max(|c x|, |R|) to 2^-24 of d, so a
term is off by 2^-24 |d| ln 2 + 2^-22 (the exponential) of itself, and terms with d < -24 are less than
2^-24 each of the largest: below |d| = 64 a term is within 2^-17.6 of itself.  A lane's chain of V / 64 terms in groups, and the joins, add
(V / 512 + 40) 2^-24 of the sum.  With r = 2^-17.6 + (V / 512 + 40) 2^-24: log Z is within r + 2^-22 |log2 Z'| (Z' = the
sum against R, 1 <= Z' <= 2^12 V), a log probability adds its own store, 2^-24 |log p|; R itself is carried exactly.
c as an fp32 number is off by 2^-25.4 of itself, which scales the exponents as a temperature would: 2^-25 |x - max x|
more.  The entropy is log Z' - E / Z' with E within r + 2^-24 |d| of its terms: (2 r + 2^-20) (1 + H + log V).
Ids are exact.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from jetspec_amd import (_lib, accept_batch_device, greedy_argmax, read_and_clear_status, token_logprobs)

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(rows, vocab, dtype=BF16, gain=2.5, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn((rows, vocab), generator=gen, device=DEV) * gain).to(dtype)


def expected(logits, tokens, top, rows=None):
    """64-bit results of each row: (log probabilities, entropy, ids, their log probabilities, bound, entropy's bound)."""
    x = (logits if rows is None else logits[rows.long()]).double().cpu()
    logp = torch.log_softmax(x, -1)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    entropy[torch.isnan(logp).all(-1)] = float("nan")
    t = tokens.cpu().long().view(x.shape[0], -1)
    given = torch.where(t < 0, 0.0, logp.gather(1, t.clamp(min=0)))
    order = torch.where(torch.isnan(x), torch.inf, x)
    # NaN above +inf: two stable sorts.
    by_value = torch.sort(order, descending=True, stable=True).indices
    nan = torch.isnan(x.gather(1, by_value))
    ids = by_value.gather(1, torch.sort((~nan).int(), stable=True).indices)[:, :top]
    v = x.shape[1]
    r = 2.0 ** -17.6 + (v / 512 + 40) * 2.0 ** -24
    base = r + 2.0 ** -22 * (12 + np.log2(v))
    spread = torch.where(x.isfinite(), x.amax(-1, keepdim=True) - x, 0.0).nan_to_num(0, 0, 0).abs()
    bound = base + 2.0 ** -24 * logp.nan_to_num(0, 0, 0).abs() + 2.0 ** -25 * spread
    h_bound = (2 * r + 2.0 ** -20) * (1 + entropy.nan_to_num(0) + np.log(v))
    return given, entropy, ids, logp.gather(1, ids), bound.gather(1, t.clamp(min=0)), h_bound, bound.gather(1, ids)


def near(got, want, bound, label):
    got, want = got.double().cpu(), want.double()
    assert torch.equal(got.isnan(), want.isnan()), label
    assert torch.equal(torch.where(got.isinf(), got, 0), torch.where(want.isinf(), want, 0)), label
    off = torch.where(want.isfinite(), (got - want).abs() / bound, 0.0)
    worst = float(off.max()) if off.numel() else 0.0
    print(f"[{label}] worst error {worst:.4f} of its bound", flush=True)
    assert worst <= 1.0, label


def check(logits, tokens, top, rows=None, label=""):
    logp, entropy, ids, values = token_logprobs(logits, tokens, top=top, rows=rows)
    want = expected(logits, tokens, top, rows)
    assert logp.shape == tokens.shape and logp.dtype is F32 and ids.dtype is torch.int64
    near(logp.view(want[0].shape), want[0], want[4], label + " given")
    near(entropy, want[1], want[5], label + " entropy")
    assert torch.equal(ids.cpu(), want[2]), label + ": ids"
    near(values, want[3], want[6], label + " top")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 63, 511, 513, 2048, 2049, 50257, 151936])
def test_vocabularies_and_types(vocab, dtype):
    for rows, top in ((1, 1), (3, 20), (17, 64)):
        logits = make(rows, vocab, dtype, seed=vocab + rows)
        tokens = torch.randint(0, vocab, (rows,), device=DEV)
        check(logits, tokens, min(top, vocab), label=f"{vocab} {rows} {top} {dtype}")


@pytest.mark.parametrize("top", [0, 1, 2, 31, 32, 33, 63, 64])
def test_tops(top):
    logits = make(5, 10007, seed=top)
    check(logits, torch.randint(0, 10007, (5, 3), device=DEV, dtype=torch.int32), top, label=f"top {top}")


def test_many_rows_take_one_workgroup_each():
    logits = make(3000, 4099, seed=1)
    check(logits, torch.randint(0, 4099, (3000,), device=DEV), 5, label="many rows")


def test_ties_go_to_the_lowest_index():
    x = torch.zeros((4, 30000), dtype=BF16, device=DEV)
    x[1] = torch.arange(30000, device=DEV) % 7
    x[2, ::2] = -0.0
    x[3] = -torch.inf
    x[3, 20000:] = 1.0
    for rows in (x, x.repeat(600, 1)):
        check(rows, torch.zeros(rows.shape[0], dtype=torch.int64, device=DEV), 64, label="ties")


def test_ascending_and_descending_rows():
    up = torch.arange(100000, device=DEV, dtype=F32) / 1000
    check(torch.stack([up, up.flip(0)]), torch.tensor([5, 99999], device=DEV), 64, label="sorted")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_masked_words(dtype):
    x = make(40, 5003, dtype, seed=2)
    x[:, ::2] = -torch.inf
    x[1] = -torch.inf                       # nothing is allowed
    x[2] = -torch.inf
    x[2, 4001] = -3.0                       # one word is
    x[3, 7] = torch.inf
    x[4, 4999] = torch.nan
    x[5, [9, 4000]] = torch.nan
    x[6, 0], x[6, 5002] = torch.nan, torch.inf
    x[7, :4096] = -torch.inf
    for rows in (x[:9], x.repeat(40, 1)):
        tokens = torch.full((rows.shape[0],), 4001, device=DEV)
        check(rows, tokens, 9, label=f"masked {dtype}")
        _, entropy, _, _ = token_logprobs(rows, tokens)
        assert entropy[2] == 0.0


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_lowest_and_highest_values_of_the_type(dtype):
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = make(12, 6001, dtype, seed=3)
    x[0] = low                              # the mask of a row that has nothing
    x[1, 1:] = low
    x[2, :3000] = low
    x[3, 17] = high
    x[4] = high
    x[5] = 1.95e38
    x[6, 5], x[6, 6] = 1.85e38, 2.5e38
    x[7] = low
    x[7, 100] = -2.0e38
    x[8] = -1.0e38
    x[9] = -1.0e9
    x[10, :] = 1.0e6
    x[10, ::3] = 1.0e6 - 8192
    x[11, 1:] = -1.0e9
    x[11, 3000:] = -65000.0
    for rows in (x, x.repeat(300, 1)):
        tokens = torch.full((rows.shape[0],), 17, device=DEV)
        check(rows, tokens, 5, label=f"extremes {dtype}")


def test_nearly_certain_and_flat_rows():
    x = torch.full((3, 151936), -20.0, device=DEV)
    x[0, 77] = 15.0
    x[1] = 3.0
    x[2, 77] = -3.0
    check(x, torch.tensor([77, 5, 6], device=DEV), 3, label="certain")


def test_layouts_of_logits_rows_and_tokens():
    wide = make(50, 4003, seed=4)
    tokens = torch.randint(0, 4001, (50, 6), device=DEV)
    check(wide[:, 1:4002], tokens[:, 0], 7, label="unaligned rows")
    check(wide[:, 3:4002].float()[:, ::2], tokens[:, ::3] % 2000, 7, label="strided columns")
    check(wide[:, :4001], tokens[:, :2], 7, label="column slice")
    check(wide.t().contiguous().t()[:, :4001], tokens, 3, label="transposed")
    check(wide[:1].expand(50, 4003), tokens, 3, label="broadcast")
    rows = torch.randint(0, 50, (120,), device=DEV, dtype=torch.int32)      # the same row again and again
    check(wide, torch.randint(0, 4003, (120, 2), device=DEV), 9, rows=rows, label="picked rows")
    check(wide, torch.randint(0, 4003, (25, 2), device=DEV), 9, rows=torch.arange(50, device=DEV)[::2], label="strided rows")
    empty = token_logprobs(wide, tokens[:0], top=2, rows=rows[:0])
    assert [tuple(t.shape) for t in empty] == [(0, 6), (0,), (0, 2), (0, 2)]
    none = token_logprobs(wide, tokens[:, :0], top=2)
    assert none[0].shape == (50, 0) and torch.equal(none[2][:, 0], greedy_argmax(wide))


@pytest.mark.parametrize("vocab", [300, 151936])
def test_padding_and_indices_outside(vocab):
    x = make(6, vocab, seed=5)
    tokens = torch.tensor([[3, -1], [vocab, 5], [-2, 0], [1, 1], [2, 2], [2 ** 40, 9]], device=DEV)
    rows = torch.tensor([0, 1, 2, -1, 6, 5], device=DEV)
    read_and_clear_status(DEV)
    logp, entropy, ids, values = token_logprobs(x, tokens, top=2, rows=rows)
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_REQUEST
    want = torch.log_softmax(x.double(), -1)
    assert logp[0, 1] == 0 and logp[1, 0].isnan() and logp[2, 0].isnan() and logp[5, 0].isnan()
    assert abs(float(logp[1, 1] - want[1, 5])) < 1e-4 and abs(float(logp[5, 1] - want[5, 9])) < 1e-4
    assert (logp[3] == 0).all() and entropy[3] == 0 and (ids[3] == -1).all() and (values[3] == 0).all()
    assert logp[4].isnan().all() and entropy[4].isnan() and (ids[4] == -1).all() and values[4].isnan().all()
    token_logprobs(x, tokens[:1].repeat(3, 1), rows=torch.tensor([0, -1, 2], device=DEV))
    assert read_and_clear_status(DEV) == 0


def test_the_first_alternative_is_the_greedy_one():
    x = make(64, 50257, seed=6)
    x[5, 40000] = torch.nan
    _, _, ids, _ = token_logprobs(x, torch.zeros(64, dtype=torch.int64, device=DEV), top=1)
    assert torch.equal(ids[:, 0], greedy_argmax(x))


def test_captured_replays_and_streams():
    x, tokens = make(4, 151936, seed=7), torch.randint(0, 151936, (4,), device=DEV)
    want = token_logprobs(x, tokens, top=8)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(token_logprobs(x, tokens, top=8))
        graphs.append(g)
    for seed in (7, 8, 9):
        x.copy_(make(4, 151936, seed=seed))
        eager = token_logprobs(x, tokens, top=8)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, eager))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(token_logprobs(x, tokens, top=8))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in got for a, b in zip(o, eager))


def test_offsets_past_32_bits():
    x = torch.empty((17000, 151936), dtype=BF16, device=DEV)      # 5.2 GB
    x[16999] = make(1, 151936, seed=10)[0]
    rows = torch.tensor([16999], device=DEV)
    tokens = torch.tensor([1234], device=DEV)
    got, want = token_logprobs(x, tokens, top=4, rows=rows), token_logprobs(x[16999:].clone(), tokens, top=4)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_accepted_path_of_a_round():
    # Two requests, a chain of three drafted tokens each; the second stops after one.
    logits = make(8, 1000, seed=11)
    greedy = greedy_argmax(logits).cpu()
    tokens = torch.tensor([7, int(greedy[0]), int(greedy[1]), int(greedy[2]),
                           9, int(greedy[4]), (int(greedy[5]) + 1) % 1000, 3], device=DEV)
    parents, depths = torch.tensor([-1, 0, 1, 2] * 2, device=DEV), torch.tensor([0, 1, 2, 3] * 2, device=DEV)
    cu = torch.tensor([0, 4, 8], dtype=torch.int32, device=DEV)
    greedy, paths, lengths, _ = accept_batch_device(logits, tokens, parents, depths, cu, 3)
    assert lengths.tolist() == [3, 1]
    # The emitted token after each accepted node is that row's own choice; -1 nodes are padding.
    rows = torch.where(paths >= 0, paths + cu[:2, None], -1).view(-1)
    emitted = torch.where(rows >= 0, greedy[rows.clamp(min=0).long()], -1)
    logp, entropy, ids, values = token_logprobs(logits, emitted, top=3, rows=rows)
    want = torch.log_softmax(logits.double(), -1).amax(-1)
    for i, row in enumerate(rows.tolist()):
        if row < 0:
            assert logp[i] == 0 and ids[i, 0] == -1
        else:
            assert abs(float(logp[i] - want[row])) < 1e-5 and ids[i, 0] == greedy[row] and values[i, 0] == logp[i]
