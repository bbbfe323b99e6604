"""token_logprobs where its sums change their reference, against 64 bits (tolerances as derived in test_logprobs_gpu.py)."""
from __future__ import annotations

import pytest
import torch

from test_logprobs_gpu import DEV, F32, check, make

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
