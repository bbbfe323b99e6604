"""token_logprobs where its sums change their reference, where a row is nearly certain, and single rows of any stride,
against 64 bits (tolerances as derived in test_logprobs_gpu.py)."""
from __future__ import annotations

import pytest
import torch

from jetspec_amd import token_logprobs
from test_logprobs_gpu import BF16, DEV, F16, F32, check, make

pytestmark = pytest.mark.gpu


def test_rows_that_rise_through_the_lowest_near_value():
    # Every lane's largest logit goes from -65536, which is summed against a far reference, over one that is 8 above
    # it or less to one that is more.
    x = torch.full((5, 6001), -65527.99, device=DEV)
    x[:, :1024] = -65536.0
    x[:, 1024:2048] = -65528.01
    x[1, 2048:] = -65528.01            # ... and stops there
    x[2, 2048:] = -65536.0 - 8         # ... and falls
    x[3, :3000] = -65536.0             # most of the row is lost where only what lies above it counts
    x[3, 3000:] = -65535.5
    x[4] = -65540.0
    x[4, 3001] = -65430.0              # the only word that counts
    for rows in (x, x.repeat(400, 1)):
        tokens = torch.full((rows.shape[0],), 1030, device=DEV)
        check(rows, tokens, 5, label="rising")


@pytest.mark.parametrize("centre", [-65536.0, 65536.0, -62383.0, 69315.0])
def test_rows_around_the_borders_of_far_values(centre):
    x = make(12, 9001, F32, gain=4.0, seed=1) + centre
    x[1] = x[1].sort().values
    x[2] = x[2].sort(descending=True).values
    x[3, :] = centre
    x[4, ::2] = -torch.inf
    x[5, ::3] = -1.0e9
    x[6] += torch.linspace(-30, 30, 9001, device=DEV)
    x[7] -= torch.linspace(-30, 30, 9001, device=DEV)
    x[8], x[9] = centre - 0.5, centre + 0.5
    x[8, 5000:], x[9, 5000:] = centre + 0.25, centre - 0.25
    x[10, 100:] = x[10, 100:].clamp(max=centre)
    for rows in (x, x.repeat(100, 1)):
        tokens = torch.randint(0, 9001, (rows.shape[0],), device=DEV, generator=torch.Generator(DEV).manual_seed(2))
        check(rows, tokens, 7, label=f"around {centre}")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_no_log_probability_is_above_zero(dtype):
    rows, vocab = 4096, 1009
    x = make(rows, vocab, dtype, gain=1.0, seed=3)
    largest = torch.arange(rows, device=DEV) % vocab
    margin = 18 + 20 * torch.rand(rows, device=DEV, generator=torch.Generator(DEV).manual_seed(4))
    x[torch.arange(rows, device=DEV), largest] = margin.to(dtype)
    x[7], x[7, 7] = -1.0e4, 0.0
    if dtype is not F16:
        x[8], x[8, 8] = -1.0e9, 3.0e6      # summed by differences
    logp, entropy, ids, values = token_logprobs(x, largest, top=3)
    assert (logp <= 0).all() and (values <= 0).all() and (entropy >= 0).all()
    assert torch.equal(ids[:, 0], largest) and torch.equal(values[:, 0], logp)
    check(x, largest, 3, label=f"certain {dtype}")


@pytest.mark.parametrize("vocab", [1, 9, 2049, 50257])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_row_of_any_row_stride(vocab, dtype):
    # A column of a product, transposed: [1, vocab] with strides (1, 1), which torch counts as contiguous.
    column = make(vocab, 1, dtype, seed=vocab)
    tokens = torch.tensor([[0, vocab - 1, vocab // 2]], device=DEV)
    row = column.t()
    assert row.stride() == (1, 1) and row.is_contiguous()
    check(row, tokens, min(vocab, 5), label="transposed column")
    same = row.clone(memory_format=torch.contiguous_format)
    assert all(torch.equal(a, b) for a, b in zip(token_logprobs(row, tokens, top=1), token_logprobs(same, tokens, top=1)))
    check(same.expand(4, vocab)[:1], tokens, 1, label="one of a broadcast row")      # a row stride of 0
    picked = torch.tensor([0, -1, 0], device=DEV)
    logp = token_logprobs(row, tokens.repeat(3, 1), rows=picked)[0]
    assert torch.equal(logp[0], logp[2]) and (logp[1] == 0).all()
    wide = make(vocab, 3, dtype, seed=7).t()[1:2]                                    # strides (1, 3)
    check(wide, tokens, 1, label="strided column")
