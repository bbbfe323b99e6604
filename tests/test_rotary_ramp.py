"""The two blends of rotary_frequencies against their formulas, pair by pair (CPU).

Tolerance: both sides are a handful of 64-bit operations, each within 2^-53, and the power is within 2^-52 times its
exponent's logarithm (at most 14): 1e-14.
"""
from __future__ import annotations

import math

import pytest

from jetspec_amd import rotary_frequencies


def by_pairs(dim, base, factor, length, slow, fast):
    index = [dim / 2 * math.log(length / (2 * math.pi * t), base) for t in (fast, slow)]
    first, last = math.floor(index[0]), math.ceil(index[1])
    values = []
    for p in range(dim // 2):
        plain = math.exp(-2 * p / dim * math.log(base))
        part = min(max((p - first) / (last - first), 0.0), 1.0)      # how much of it is divided
        values.append(plain * (1 - part) + plain / factor * part)
    return values


def by_turns(dim, base, factor, length, slow, fast):
    values = []
    for p in range(dim // 2):
        plain = math.exp(-2 * p / dim * math.log(base))
        part = min(max((fast - plain * length / (2 * math.pi)) / (fast - slow), 0.0), 1.0)
        values.append(plain * (1 - part) + plain / factor * part)
    return values


CASES = [(128, 1e6, 4.0, 32768, 1.0, 32.0), (64, 1e4, 8.0, 4096, 1.0, 4.0), (80, 5e5, 32.0, 8192, 0.5, 17.0), (36, 1e4, 2.0, 2048, 1.0, 32.0)]


@pytest.mark.parametrize("ramp, formula", [("turns", by_turns), ("pairs", by_pairs)])
@pytest.mark.parametrize("case", CASES)
def test_blends(case, ramp, formula):
    dim, base, factor, length, slow, fast = case
    got = rotary_frequencies(dim, base=base, factor=factor, original_length=length, slow=slow, fast=fast, ramp=ramp).tolist()
    assert got == pytest.approx(formula(*case), rel=1e-14, abs=0)


def test_a_ramp_over_pairs_by_hand():
    # Over 32768 positions pair 23.6 turns 32 times and pair 39.65 once: 23 stays, 40 is divided, 30 has 10 / 17 left.
    plain = rotary_frequencies(128, base=1e6).tolist()
    got = rotary_frequencies(128, base=1e6, factor=4.0, original_length=32768, ramp="pairs").tolist()
    assert got[:24] == plain[:24]
    assert got[40:] == pytest.approx([x / 4 for x in plain[40:]], rel=1e-14)
    assert got[30] == pytest.approx(plain[30] * (10 / 17 + 7 / 17 / 4), rel=1e-14)
    turns = rotary_frequencies(128, base=1e6, factor=4.0, original_length=32768).tolist()
    assert max(abs(a / b - 1) for a, b in zip(turns, got)) > 0.3       # not one for the other


def test_lengths_that_no_pair_or_every_pair_spans():
    plain = rotary_frequencies(16, base=1e4)
    assert rotary_frequencies(16, base=1e4, factor=4.0, original_length=3, ramp="pairs").tolist() == (plain / 4).tolist()
    assert rotary_frequencies(16, base=1e4, factor=4.0, original_length=10 ** 9, ramp="pairs").tolist() == plain.tolist()


@pytest.mark.parametrize("options", [dict(ramp="turn"), dict(ramp=None), dict(ramp="pairs", slow=0.0), dict(ramp="pairs", base=1.0),
                                     dict(ramp="pairs", base=0.5)])
def test_refusals(options):
    with pytest.raises(ValueError, match="ramp"):
        rotary_frequencies(64, original_length=4096, factor=2.0, **options)
