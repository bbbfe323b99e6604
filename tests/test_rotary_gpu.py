"""rotary_scatter on the GPU against 64 bits.

Tolerance, derived.  The angle is 64 bits but for the reduced turn's rounding to fp32 (at most an eighth of a
turn: 2^-28 turns, 2^-25.3 radians) and the 64-bit product's (position * 2^-52 turns at the positions here: nothing);
the library's sine and cosine add 2 units in the last place of fp32 (2^-22) and the gain half of one: a cosine is
within 2^-21 gain.  An output is two products and a sum, each rounded: |x1| and |x2| times (2^-21 + 2^-23) gain,
and the store's half step.  fp32 results below 2^-126 are not tested.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from jetspec_amd import (_lib, read_and_clear_status, rope_scatter, rotary_frequencies, rotary_scatter,
                         rotary_scatter_prevalidated)

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


class Rows:
    def __init__(self, rows=37, q_heads=8, kv_heads=2, dim=128, turned=128, dtype=BF16, page=16, length=10000, seed=0,
                 base=1e4, index=torch.int64):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.q, self.k, self.v = (torch.randn((rows, h, dim), generator=gen, device=DEV).to(dtype) for h in
                                  (q_heads, kv_heads, kv_heads))
        pages = -(-rows // page) + 1
        self.k_pool, self.v_pool = (torch.full((pages, page, kv_heads, dim), 5.0, dtype=dtype, device=DEV) for _ in range(2))
        self.slots = torch.as_tensor(rng.permutation(pages * page)[:rows], device=DEV).to(index)
        self.positions = torch.as_tensor(rng.integers(0, length, size=rows), device=DEV).to(index)
        self.frequencies = rotary_frequencies(turned, base=base, device=DEV)

    def args(self):
        return (self.q, self.k, self.v, self.positions, self.frequencies, self.k_pool, self.v_pool, self.slots)


def turned(x, positions, frequencies, interleaved, gain):
    """64-bit results and their bounds."""
    kind, x = x.dtype, x.double().cpu().numpy()
    f, n = frequencies.cpu().numpy(), frequencies.numel()
    angle = positions.cpu().numpy().astype(np.float64)[:, None, None] * f
    cos, sin = np.cos(angle) * gain, np.sin(angle) * gain
    out, size = x.copy(), np.zeros_like(x)
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    size[..., first] = size[..., second] = np.abs(a) + np.abs(b)
    bound = size * abs(gain) * (2.0 ** -21 + 2.0 ** -23)
    bound[..., :2 * n] += STEP[kind] * (np.abs(out[..., :2 * n]) + bound[..., :2 * n]) + (2.0 ** -25 if kind is F16 else 0)
    return out, bound


def close(got, want, label):
    have, (out, bound) = got.double().cpu().numpy(), want
    exact = bound == 0
    assert np.array_equal(have[exact], out[exact]), f"{label}: copied elements"
    worst = (np.abs(have - out)[~exact] / bound[~exact]).max() if (~exact).any() else 0
    print(f"[{label}] worst error {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0, label


def check(s, out, interleaved=False, gain=1.0, label=""):
    close(out, turned(s.q, s.positions, s.frequencies, interleaved, gain), label + " q")
    for pool, x in ((s.k_pool, turned(s.k, s.positions, s.frequencies, interleaved, gain)),
                    (s.v_pool, (s.v.double().cpu().numpy(), np.zeros(s.v.shape)))):
        flat = pool.reshape(-1, *pool.shape[2:])
        slots = s.slots.long()
        close(flat[slots], x, label + " pool")
        rest = torch.ones(flat.shape[0], dtype=torch.bool, device=DEV)
        rest[slots] = False
        assert (flat[rest] == 5.0).all(), label + ": other slots"


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim, part", [(2, 2), (6, 4), (64, 64), (64, 6), (80, 40), (96, 96), (96, 24), (128, 128), (128, 64),
                                       (128, 32), (250, 250), (256, 256), (256, 64)])
def test_layouts_types_and_parts(dim, part, interleaved, dtype):
    for rows, heads in ((1, (4, 1)), (67, (10, 5))):
        s = Rows(rows=rows, q_heads=heads[0], kv_heads=heads[1], dim=dim, turned=part, dtype=dtype, seed=dim + rows)
        out = rotary_scatter(*s.args(), interleaved=interleaved, gain=1.25)
        check(s, out, interleaved, 1.25, f"{dim} {part} {interleaved} {dtype} {rows}")


def test_far_positions_and_scaled_frequencies():
    s = Rows(dtype=F32, length=1 << 31, seed=1)
    s.positions[0], s.positions[1] = 2 ** 31 - 1, 0
    s.frequencies = rotary_frequencies(128, base=5e5, factor=32.0, original_length=8192, device=DEV)
    out = rotary_scatter(*s.args())
    # At 2^31 the product of position and frequency itself rounds at 2^-23 radians in both, and 1 / 2 pi's here: 2^-21.
    want, bound = turned(s.q, s.positions, s.frequencies, False, 1.0)
    have = out.double().cpu().numpy()
    assert (np.abs(have - want) <= bound + 2.0 ** -20 * np.abs(s.q.double().cpu().numpy()).max()).all()


def test_frequencies_of_stretched_contexts():
    plain = rotary_frequencies(64, base=1e6)
    assert plain.dtype is torch.float64 and plain[0] == 1.0 and plain.shape == (32,)
    np.testing.assert_allclose(plain.numpy(), 1e6 ** (-np.arange(32) / 32), rtol=1e-14)
    np.testing.assert_allclose(rotary_frequencies(64, base=1e6, factor=4.0).numpy(), plain.numpy() / 4, rtol=1e-15)
    scaled = rotary_frequencies(64, base=1e6, factor=8.0, original_length=4096, slow=1.0, fast=4.0).numpy()
    turns = plain.numpy() * 4096 / (2 * np.pi)
    assert np.array_equal(scaled[turns > 4], plain.numpy()[turns > 4])
    np.testing.assert_allclose(scaled[turns < 1], plain.numpy()[turns < 1] / 8, rtol=1e-15)
    between = (turns > 1) & (turns < 4)
    keep = (turns[between] - 1) / 3
    np.testing.assert_allclose(scaled[between], plain.numpy()[between] * (keep + (1 - keep) / 8), rtol=1e-14)


@pytest.mark.parametrize("interleaved", [False, True])
def test_strides_and_unaligned_starts(interleaved):
    for shift, dtype in ((1, BF16), (2, BF16), (4, F16), (1, F32), (2, F32)):
        s = Rows(rows=21, dtype=dtype, dim=64, turned=32, index=torch.int32, seed=shift)
        wide = torch.zeros((21, 20, 64 + 8), dtype=dtype, device=DEV)
        views = []
        for at, x in ((0, s.q), (8, s.k), (12, s.v)):
            view = wide[:, at:at + x.shape[1], shift:shift + 64]
            view.copy_(x)
            views.append(view)
        pools = []
        for pool in (s.k_pool, s.v_pool):
            held = torch.full((pool.shape[0], pool.shape[2], pool.shape[1], 64 + 8), 5.0, dtype=dtype, device=DEV)
            pools.append(held[..., shift:shift + 64].transpose(1, 2))
        apart = torch.zeros((21, 3), dtype=torch.int32, device=DEV)
        apart[:, 0], apart[:, 2] = s.positions, s.slots
        out = torch.empty((8, 21, 64), dtype=dtype, device=DEV).transpose(0, 1)
        got = rotary_scatter(*views, apart[:, 0], s.frequencies, *pools, apart[:, 2], interleaved=interleaved, out=out)
        assert got is out
        s.k_pool, s.v_pool = pools
        check(s, out, interleaved, 1.0, f"strided {shift} {dtype}")
    # A last dimension that is not contiguous.
    s = Rows(rows=5, dim=64, turned=64)
    s.q = s.q.transpose(1, 2).contiguous().transpose(1, 2)
    check(s, rotary_scatter(*s.args(), interleaved=interleaved), interleaved, 1.0, "columns")


def test_padding_and_rows_out_of_range():
    s = Rows(rows=9)
    s.slots[2], s.slots[3] = -1, -1
    s.positions[3] = -99
    out = torch.full_like(s.q, 3.0)
    read_and_clear_status(DEV)
    rotary_scatter_prevalidated(*s.args(), out)
    assert read_and_clear_status(DEV) == 0
    assert (out[2:4] == 3.0).all() and not (out[4] == 3.0).any()
    for field, value, bit in (("slots", s.k_pool.shape[0] * 16, _lib.TV_STATUS_BAD_SLOT), ("slots", -2, _lib.TV_STATUS_BAD_SLOT),
                              ("slots", 2 ** 40, _lib.TV_STATUS_BAD_SLOT), ("positions", -1, _lib.TV_STATUS_BAD_POSITION),
                              ("positions", 2 ** 31, _lib.TV_STATUS_BAD_POSITION)):
        s = Rows(rows=9)
        getattr(s, field)[4] = value
        out = torch.full_like(s.q, 3.0)
        rotary_scatter_prevalidated(*s.args(), out)
        assert read_and_clear_status(DEV) == bit, (field, value)
        assert (out[4] == 3.0).all() and not (out[5] == 3.0).any()
        with pytest.raises(ValueError):
            rotary_scatter(*s.args())
    s = Rows(rows=9)
    s.slots[1] = s.slots[0]
    with pytest.raises(ValueError, match="unique"):
        rotary_scatter(*s.args())
    with pytest.raises(ValueError, match="overlap"):
        rotary_scatter(*Rows(rows=9).args()[:5], s.k_pool, s.k_pool, Rows(rows=9).slots)
    with pytest.raises(ValueError, match="overlap"):
        s = Rows(rows=9)
        rotary_scatter(*s.args(), out=s.q)


def test_copied_parts_keep_infinities_and_nans():
    s = Rows(rows=3, dim=64, turned=16)
    s.q[1, 2, 16], s.q[1, 2, 63], s.v[0, 0, 7] = float("inf"), float("nan"), float("-inf")
    out = rotary_scatter(*s.args())
    assert torch.equal(out[..., 16:].view(torch.int16), s.q[..., 16:].view(torch.int16))
    assert out[..., :16].isfinite().all()
    assert torch.equal(s.v_pool.view(-1, 2, 64)[s.slots].view(torch.int16), s.v.view(torch.int16))


def test_whole_heads_in_halves_are_the_table_rotation():
    s, t = Rows(dtype=F32, seed=6), Rows(dtype=F32, seed=6)
    angle = torch.arange(10000, dtype=torch.float64, device=DEV)[:, None] * s.frequencies
    table = torch.cat([angle.cos(), angle.sin()], dim=1).float()
    out = rope_scatter(t.q, t.k, t.v, t.positions, table, t.k_pool, t.v_pool, t.slots)
    want, bound = turned(s.q, s.positions, s.frequencies, False, 1.0)
    assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()
    check(s, rotary_scatter(*s.args()), label="whole heads")


def test_many_rows_and_offsets_past_32_bits():
    s = Rows(rows=5001, q_heads=16, kv_heads=4, dim=64, turned=64, seed=7)
    check(s, rotary_scatter(*s.args(), interleaved=True), True, 1.0, "many rows")
    s = Rows(rows=40, kv_heads=2, dim=128, page=16, seed=8)
    pages = (1 << 32) // s.k_pool[0].numel() + 4
    shift = pages - s.k_pool.shape[0]
    big = [torch.empty((pages, *s.k_pool.shape[1:]), dtype=BF16, device=DEV) for _ in range(2)]
    for pool in big:
        pool[shift:].fill_(5.0)
    out = rotary_scatter(s.q, s.k, s.v, s.positions, s.frequencies, *big, s.slots + shift * 16)
    s.k_pool, s.v_pool = big[0][shift:], big[1][shift:]
    check(s, out, label="far pages")


def test_captured_replays_and_another_stream():
    s = Rows(rows=64, seed=9)
    out = torch.empty_like(s.q)
    rotary_scatter_prevalidated(*s.args(), out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rotary_scatter_prevalidated(*s.args(), out)
    for seed in (10, 11, 12):
        t = Rows(rows=64, seed=seed)
        for name in ("q", "k", "v", "positions", "slots"):
            getattr(s, name).copy_(getattr(t, name))
        s.k_pool.fill_(5.0), s.v_pool.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        check(s, out, label=f"replay {seed}")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = rotary_scatter_prevalidated(*s.args(), torch.empty_like(s.q))
    side.synchronize()
    assert torch.equal(other, out)
