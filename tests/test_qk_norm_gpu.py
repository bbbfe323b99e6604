"""The fused Q/K norm + rotation + scatter and the e4m3 append on the GPU, against 64 bits.

Tolerances, derived: the norm sums D squares in fp32, at most 16 in a lane and six steps over the
lanes, so its relative error is under 22 * 2^-24; its root halves that; mean, root, reciprocal, the two
products of the norm, the product of the rotation and its sum add at most 7 roundings.  So before
the store a value is within 18 * 2^-24, and a little more for second order, of the sum of the sizes
of its two terms: 20 * 2^-24 below.  The store adds half a step of its type.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import e4m3_helpers
from jetspec_amd import (_lib, qk_norm_rope_scatter, qk_norm_rope_scatter_prevalidated, read_and_clear_status,
                         store_kvcache_e4m3)

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def normal(gen, *shape, dtype=BF16, gain=2.0):
    return (torch.randn(shape, generator=gen, device=DEV) * gain).to(dtype)


def problem(rows, q_heads, kv_heads, dim, *, dtype=BF16, e4m3=False, cache_dtype=F32, weights=None, page=16, strided=False,
            seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    if strided:   # every second head and dimension of a wider projection
        base = normal(gen, rows, 2 * (q_heads + 2 * kv_heads), 2 * dim, dtype=dtype)[:, ::2, ::2]
    else:
        base = normal(gen, rows, q_heads + 2 * kv_heads, dim, dtype=dtype)
    pages = -(-rows // page) + 2
    angles = torch.arange(300, device=DEV).double()[:, None] * torch.logspace(0, -4, dim // 2, dtype=torch.float64, device=DEV)
    cache = torch.cat([angles.cos(), angles.sin()], 1).to(cache_dtype)
    pool = (pages, page, kv_heads, dim)

    def a_pool():
        return normal(gen, *pool, dtype=F32).to(E4M3 if e4m3 else dtype)
    call = dict(q=base[:, :q_heads], k=base[:, q_heads:q_heads + kv_heads], v=base[:, q_heads + kv_heads:],
                q_weight=normal(gen, dim, dtype=weights or dtype), k_weight=normal(gen, dim, dtype=weights or dtype),
                positions=torch.as_tensor(rng.integers(0, 300, rows), device=DEV), cos_sin_cache=cache, k_pool=a_pool(),
                v_pool=a_pool(), node_slots=torch.as_tensor(rng.permutation(pages * page)[:rows], device=DEV))
    if e4m3:
        call |= dict(k_scale=torch.ones(pool[:3], device=DEV), v_scale=torch.ones(pool[:3], device=DEV))
    return call


def host(t):
    return t.double().cpu().numpy()


def turned(x, weight, cache, positions, eps):
    """(value, sum of the sizes of its terms) in 64 bits."""
    x, weight, turn = host(x), host(weight), host(cache).reshape(cache.shape[0], -1)[positions.cpu().numpy()]
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    half = x.shape[-1] // 2
    a, b, cos, sin = y[..., :half], y[..., half:], turn[:, None, :half], turn[:, None, half:]
    return (np.concatenate([a * cos - b * sin, b * cos + a * sin], -1),
            np.concatenate([abs(a * cos) + abs(b * sin), abs(b * cos) + abs(a * sin)], -1))


def assert_near(got, value, size, dtype):
    got = host(got)
    early = 20 * 2.0 ** -24 * size
    half_step = torch.finfo(dtype).eps / 2
    allowed = early + half_step * (np.abs(value) + early) + (2.0 ** -25 if dtype == F16 else 0)
    worst = np.max(np.abs(got - value) - allowed)
    assert worst <= 0, worst


def check(call, eps=1e-6, validated=False):
    before = {name: call[name].clone() for name in ("k_pool", "v_pool", "k_scale", "v_scale") if name in call}
    dtype, dim = call["q"].dtype, call["q"].shape[-1]
    if validated:
        out = qk_norm_rope_scatter(**call, eps=eps)
    else:
        out = torch.full(call["q"].shape, float("nan"), dtype=dtype, device=DEV)
        assert qk_norm_rope_scatter_prevalidated(**call, out=out, eps=eps) is out
    assert_near(out, *turned(call["q"], call["q_weight"], call["cos_sin_cache"], call["positions"], eps), dtype)
    slots = call["node_slots"].cpu().numpy()
    heads = call["k"].shape[1]
    k, size = turned(call["k"], call["k_weight"], call["cos_sin_cache"], call["positions"], eps)
    untouched = np.setdiff1d(np.arange(call["k_pool"].shape[0] * call["k_pool"].shape[1]), slots)
    if "k_scale" in call:
        codes, scales = e4m3_helpers.quantise(call["v"].float().cpu().numpy())
        np.testing.assert_array_equal(e4m3_helpers.codes_of(call["v_pool"]).reshape(-1, heads, dim)[slots], codes)
        np.testing.assert_array_equal(call["v_scale"].reshape(-1, heads).cpu().numpy()[slots], scales)
        got = e4m3_helpers.dequantise(call["k_pool"], call["k_scale"]).reshape(-1, heads, dim)[slots]
        early = 20 * 2.0 ** -24 * size
        amax, scale = np.abs(k).max(-1), host(call["k_scale"]).reshape(-1, heads)[slots]
        assert np.all(np.abs(scale - np.maximum(amax / 448, 2.0 ** -100)) <= (early.max(-1) + 2.0 ** -23 * amax) / 448)
        # Half a code step (2^-4 of the value, or half the smallest code), and what the fp32 value is off.
        assert np.all(np.abs(got - k) <= (2.0 ** -4 + 2.0 ** -20) * (np.abs(k) + early) + early + 2.0 ** -10 * scale[..., None])
    else:
        flat = {name: call[name].reshape(-1, heads, dim)[call["node_slots"]] for name in ("k_pool", "v_pool")}
        assert_near(flat["k_pool"], k, size, dtype)
        assert torch.equal(flat["v_pool"], call["v"])
    for name, old in before.items():   # every other slot keeps its bytes
        new = call[name].contiguous().view(torch.uint8).reshape(-1, old[0, 0].numel() * old.element_size()).cpu()
        old = old.contiguous().view(torch.uint8).reshape(new.shape).cpu()
        assert torch.equal(new[untouched], old[untouched]), name
    assert read_and_clear_status(DEV) == 0


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows, q_heads, kv_heads, dim", [
    (1, 1, 1, 2), (1, 32, 8, 128), (3, 4, 2, 34), (7, 8, 2, 64), (5, 6, 3, 80), (9, 5, 5, 96), (65, 16, 2, 128),
    (33, 14, 2, 254), (40, 4, 1, 256), (5000, 3, 1, 32),
])
def test_against_64_bits(rows, q_heads, kv_heads, dim, dtype, e4m3):
    check(problem(rows, q_heads, kv_heads, dim, dtype=dtype, e4m3=e4m3, seed=rows + dim))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("change", [dict(cache_dtype=BF16), dict(weights=F32), dict(strided=True), dict(page=1), dict(page=48)])
def test_layouts(change, e4m3):
    call = problem(20, 8, 2, 128, e4m3=e4m3, **change)
    check(call)
    # Strided pools, addresses and angles (rank 3) give the same bytes.
    wide = {name: torch.zeros((*call[name].shape[:2], 2 * call[name].shape[2], *[2 * n for n in call[name].shape[3:]]),
                              device=DEV).to(call[name].dtype) for name in ("k_pool", "v_pool")}
    spread = dict(call)
    for name, t in wide.items():
        spread[name] = t[:, :, ::2, ::2]
    spread["positions"] = torch.stack([call["positions"], call["positions"]], 1).int()[:, 0]
    spread["node_slots"] = torch.stack([call["node_slots"], call["node_slots"]], 1).int()[:, 1]
    spread["cos_sin_cache"] = torch.stack([call["cos_sin_cache"]] * 2, -1)[..., 0].unsqueeze(1)
    check(spread, validated=True)
    at = call["node_slots"]
    for name in wide:
        a, b = (t.contiguous().view(torch.uint8).reshape(t.shape[0] * t.shape[1], -1)[at] for t in (call[name], spread[name]))
        if name == "v_pool":
            assert torch.equal(a, b)


def test_views_at_odd_offsets():
    """Rows and pools that start off 16 bytes."""
    for shift in (1, 2, 4):
        call = problem(6, 4, 2, 64)
        for name in ("k_pool", "v_pool"):
            t = call[name]
            call[name] = torch.zeros(t.numel() + shift, dtype=t.dtype, device=DEV)[shift:].view(t.shape)
        check(call)
        call = problem(6, 4, 2, 64, e4m3=True)
        for name in ("k_pool", "v_pool"):
            t = call[name]
            call[name] = torch.zeros(t.numel() + shift, device=DEV).to(E4M3)[shift:].view(t.shape)
        check(call)


def test_a_zero_row_and_a_large_eps():
    call = problem(4, 4, 2, 64)
    call["q"][1] = 0
    call["k"][2] = 0
    check(call)
    check(problem(4, 4, 2, 64, seed=1), eps=0.5)
    call = problem(4, 4, 2, 64, e4m3=True, seed=2)
    call["v"][1] = 0
    call["k"][2] = 0
    check(call)


def test_padding_rows_are_left_alone():
    call = problem(10, 4, 2, 128)
    call["node_slots"][3:7] = -1
    call["positions"][4] = 10 ** 9
    pools = [call["k_pool"].clone(), call["v_pool"].clone()]
    out = torch.full_like(call["q"], 7.0, memory_format=torch.contiguous_format)
    qk_norm_rope_scatter_prevalidated(**call, out=out)
    assert torch.all(out[3:7] == 7) and not torch.any(out[:3] == 7)
    kept = call["node_slots"][call["node_slots"] >= 0]
    for pool, old in zip((call["k_pool"], call["v_pool"]), pools):
        pool.view(-1, 256)[kept] = old.view(-1, 256)[kept]
        assert torch.equal(pool, old)
    assert read_and_clear_status(DEV) == 0
    assert torch.all(qk_norm_rope_scatter(**call)[3:7] == 0)


@pytest.mark.parametrize("rows", [12, 6000])
def test_bad_positions_and_slots_write_nothing(rows):
    call = problem(rows, 4, 2, 64)
    pools = [call["k_pool"].clone(), call["v_pool"].clone()]
    out = torch.full_like(call["q"], 7.0, memory_format=torch.contiguous_format)
    for name, bad, bit, message in (("positions", 300, _lib.TV_STATUS_BAD_POSITION, "positions lie outside"),
                                    ("positions", -1, _lib.TV_STATUS_BAD_POSITION, "positions lie outside"),
                                    ("node_slots", -2, _lib.TV_STATUS_BAD_SLOT, "slots lie outside"),
                                    ("node_slots", 10 ** 12, _lib.TV_STATUS_BAD_SLOT, "slots lie outside")):
        broken = call | {name: torch.full_like(call[name], bad)}
        qk_norm_rope_scatter_prevalidated(**broken, out=out)
        assert read_and_clear_status(DEV) == bit
        assert torch.all(out == 7) and torch.equal(call["k_pool"], pools[0]) and torch.equal(call["v_pool"], pools[1])
        with pytest.raises(ValueError, match=message):
            qk_norm_rope_scatter(**broken)
    with pytest.raises(ValueError, match="unique"):
        qk_norm_rope_scatter(**(call | dict(node_slots=torch.zeros_like(call["node_slots"]))))
    with pytest.raises(ValueError, match="overlap"):
        qk_norm_rope_scatter(**call, out=call["q"])
    with pytest.raises(ValueError, match="overlap"):
        qk_norm_rope_scatter(**(call | dict(v_pool=call["k_pool"])))
    assert torch.equal(call["k_pool"], pools[0])


def test_no_rows():
    call = problem(4, 4, 2, 64)
    empty = call | {n: call[n][:0] for n in ("q", "k", "v", "positions", "node_slots")}
    assert qk_norm_rope_scatter_prevalidated(**empty, out=empty["q"]).shape[0] == 0


def test_captured_replays_follow_the_inputs():
    call = problem(16, 8, 2, 128, e4m3=True)
    out = torch.empty_like(call["q"], memory_format=torch.contiguous_format)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qk_norm_rope_scatter_prevalidated(**call, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qk_norm_rope_scatter_prevalidated(**call, out=out)
    for seed in range(1, 4):
        fresh = problem(16, 8, 2, 128, e4m3=True, seed=seed)
        for name in ("q", "k", "v", "positions", "node_slots", "q_weight", "k_weight"):
            call[name].copy_(fresh[name])
        graph.replay()
        torch.cuda.synchronize()
        replayed = [out.clone(), *(call[n].clone() for n in ("k_pool", "v_pool", "k_scale", "v_scale"))]
        qk_norm_rope_scatter_prevalidated(**call, out=out)
        for a, b in zip(replayed, [out, *(call[n] for n in ("k_pool", "v_pool", "k_scale", "v_scale"))]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), seed


# --------------------------------------------------------------------------- append
def stored(key, value, slots, pages=4, page=16, layout=lambda t: t):
    heads, dim = key.shape[1:]
    pools = [layout(torch.full((pages, page, heads, dim), 3.0, device=DEV).to(E4M3)) for _ in range(2)]
    scales = [torch.full((pages, page, heads), 5.0, device=DEV) for _ in range(2)]
    store_kvcache_e4m3(key, value, *pools, *scales, slots)
    return pools, scales


def check_stored(key, value, slots, **kw):
    pools, scales = stored(key, value, slots, **kw)
    at = slots.cpu().numpy()
    heads, dim = key.shape[1:]
    for rows, pool, scale in zip((key, value), pools, scales):
        codes, expect = e4m3_helpers.quantise(rows.float().cpu().numpy())
        whole = np.full((pool.shape[0] * pool.shape[1], heads, dim), e4m3_helpers.encode(np.array([3.0]))[0])
        sized = np.full(whole.shape[:2], np.float32(5))
        whole[at[at >= 0]], sized[at[at >= 0]] = codes[at >= 0], expect[at >= 0]
        np.testing.assert_array_equal(e4m3_helpers.codes_of(pool).reshape(whole.shape), whole)
        np.testing.assert_array_equal(scale.cpu().numpy().reshape(sized.shape), sized)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows, heads, dim", [(1, 1, 2), (1, 8, 128), (17, 2, 64), (50, 5, 80), (30, 3, 34), (9000, 1, 128), (60, 2, 256)])
def test_append_is_the_definition_bit_for_bit(rows, heads, dim, dtype):
    gen = torch.Generator(device=DEV).manual_seed(rows)
    rng = np.random.default_rng(rows)
    key, value = normal(gen, rows, heads, dim, dtype=dtype), normal(gen, rows, heads, dim, dtype=dtype, gain=0.01)
    slots = torch.as_tensor(rng.permutation((-(-rows // 16) + 1) * 16)[:rows], device=DEV)
    slots[rng.random(rows) < 0.2] = -1
    check_stored(key, value, slots.int() if rows % 2 else slots, pages=-(-rows // 16) + 1)
    assert read_and_clear_status(DEV) == 0


def test_append_of_every_ratio_to_the_largest():
    """Rows whose first element is the largest and whose others cover the codes' borders and the subnormal ones."""
    x = torch.full((64, 1, 128), 448.0, device=DEV)
    ladder = torch.from_numpy(e4m3_helpers.VALUES[:127].copy()).to(DEV).float()
    middle = (ladder[1:] + ladder[:-1]) / 2
    zero = torch.zeros_like(middle)
    many = torch.cat([ladder, middle, torch.nextafter(middle, zero), torch.nextafter(middle, zero + 1e9), -middle])
    x[:5, 0, 1:] = torch.nn.functional.pad(many, (0, 5 * 127 - many.numel())).view(5, 127)
    x[5:10] = x[:5] * 2.0 ** -120
    x[10:15] = x[:5] * 2.0 ** 100
    x[15] = 1e-44
    x[16] = 0
    x[17:22] = x[:5] * 1.37
    check_stored(x, -x.flip(0), torch.arange(64, device=DEV))


@pytest.mark.parametrize("dtype, vector", [(BF16, True), (F32, True), (F16, False)])
def test_rows_with_infinities_and_nan_read_as_nan(dtype, vector):
    dim = 128 if vector else 70
    gen = torch.Generator(device=DEV).manual_seed(1)
    key, value = normal(gen, 6, 3, dim, dtype=dtype), normal(gen, 6, 3, dim, dtype=dtype)
    key[1, 2, 5], key[2, 0, dim - 1], value[4, 1, 0] = float("inf"), float("nan"), -float("inf")
    pools, scales = stored(key, value, torch.arange(6, device=DEV))
    bad = [torch.nonzero(s[0, :6].isnan()).tolist() for s in scales]
    assert bad == [[[1, 2], [2, 0]], [[4, 1]]]
    assert all(not (p.float().isnan().any()) for p in pools)
    check_stored(key, value, torch.arange(6, device=DEV))


def test_append_layouts_and_bad_slots():
    gen = torch.Generator(device=DEV).manual_seed(2)
    wide = normal(gen, 20, 8, 256)
    slots = torch.arange(40, device=DEV)[::2]
    check_stored(wide[:, ::2, ::2], wide[:, 1::2, 1::2], slots)
    check_stored(wide[:, :4, 1:129], wide[:, 4:, 1:129], slots)
    check_stored(wide[:, :4, :128], wide[:, 4:, 8:136], slots,
                 layout=lambda t: torch.zeros(2 * t.numel(), device=DEV).to(E4M3).view(*t.shape[:3], -1)[..., ::2].copy_(t))
    check_stored(wide[:, :4, :128], wide[:, 4:, :128], slots,
                 layout=lambda t: t.transpose(1, 2).contiguous().transpose(1, 2))
    pools, scales = stored(wide[:3], wide[:3], torch.tensor([64, -2, 10 ** 10], device=DEV))
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_SLOT
    assert all(torch.all(s == 5) for s in scales) and all(torch.all(p.float() == 3) for p in pools)
    stored(wide[:0], wide[:0], slots[:0])
