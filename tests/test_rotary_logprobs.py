"""Refusals of rotary_scatter and token_logprobs (CPU: nothing is launched)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from jetspec_amd import _lib, rotary_frequencies, rotary_scatter, rotary_scatter_prevalidated, token_logprobs

BF16 = torch.bfloat16


def rotary(**over):
    args = dict(q=torch.zeros((3, 4, 64), dtype=BF16), k=torch.zeros((3, 2, 64), dtype=BF16), v=torch.zeros((3, 2, 64), dtype=BF16),
                positions=torch.arange(3), frequencies=rotary_frequencies(64), k_pool=torch.zeros((2, 4, 2, 64), dtype=BF16),
                v_pool=torch.zeros((2, 4, 2, 64), dtype=BF16), node_slots=torch.arange(3), out=torch.zeros((3, 4, 64), dtype=BF16))
    return args | over


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.zeros((3, 64), dtype=BF16)), "rows,heads,dim"),
    (dict(q=torch.zeros((3, 3, 64), dtype=BF16)), "GQA"),
    (dict(k=torch.zeros((3, 2, 64))), "must share one of"),
    (dict(positions=torch.zeros(3)), "integer"),
    (dict(node_slots=torch.arange(4)), "integer"),
    (dict(frequencies=rotary_frequencies(64).float()), "float64"),
    (dict(frequencies=rotary_frequencies(66)), "float64"),
    (dict(frequencies=rotary_frequencies(64)[:0]), "float64"),
    (dict(frequencies=rotary_frequencies(64)[::2]), "float64"),
    (dict(k_pool=torch.zeros((2, 4, 2, 64))), "KV pools must match"),
    (dict(out=torch.zeros((3, 4, 64))), "output must match"),
    (dict(gain=float("nan")), "gain must be"),
    (dict(gain=1e39), "gain must be"),
    ({}, "requires GPU tensors"),
])
def test_rotary_refuses(change, message):
    for entry in (rotary_scatter, rotary_scatter_prevalidated):
        with pytest.raises(ValueError, match=message):
            entry(**rotary(**change))
    with pytest.raises(ValueError, match="given output"):
        rotary_scatter_prevalidated(**rotary(out=None))


@pytest.mark.parametrize("dim, options", [(0, {}), (3, {}), (True, {}), (4.0, {}), (8, dict(base=0)), (8, dict(factor=-1.0)),
                                          (8, dict(factor=float("inf"))), (8, dict(original_length=0)),
                                          (8, dict(original_length=9, slow=4.0, fast=4.0))])
def test_frequencies_refuse(dim, options):
    with pytest.raises(ValueError):
        rotary_frequencies(dim, **options)


@pytest.mark.parametrize("change, message", [
    (dict(logits=torch.zeros(5)), "rows, vocab"),
    (dict(logits=torch.zeros((3, 0))), "rows, vocab"),
    (dict(logits=torch.zeros((3, 10), dtype=torch.float64)), "BF16, FP16 or FP32"),
    (dict(token_ids=torch.zeros(3)), "token_ids"),
    (dict(token_ids=torch.zeros((3, 1, 1), dtype=torch.int64)), "token_ids"),
    (dict(token_ids=torch.zeros(4, dtype=torch.int64)), "one entry per logits row"),
    (dict(rows=torch.zeros(4, dtype=torch.int64)), "rows must be"),
    (dict(rows=torch.zeros(3)), "rows must be"),
    ({}, "requires GPU tensors"),
])
def test_logprobs_refuse(change, message):
    with pytest.raises(ValueError, match=message):
        token_logprobs(**(dict(logits=torch.zeros((3, 10)), token_ids=torch.zeros(3, dtype=torch.int64)) | change))


def test_entries_reject_bad_arguments_without_a_device():
    lib = _lib.library()
    assert lib.tv_rotary_scatter(None, None) == _lib.TV_ERR_INVALID
    assert lib.tv_token_logprobs(None, None, 0, None) == _lib.TV_ERR_INVALID
    assert lib.tv_token_logprobs_workspace_bytes(None) == _lib.TV_ERR_INVALID
    assert lib.tv_sizeof_rotary_args() == ctypes.sizeof(_lib.RotaryArgs)
    assert lib.tv_sizeof_token_logprobs_args() == ctypes.sizeof(_lib.TokenLogprobsArgs)

    def turn(**over):
        a = _lib.RotaryArgs()
        r = a.rope
        for name in ("q", "k", "v", "positions", "k_pool", "v_pool", "node_slots", "out"):
            setattr(r, name, 0x10000)
        for name in ("q_stride", "k_stride", "v_stride", "out_stride"):
            getattr(r, name)[:] = [256, 64, 1]
        r.k_pool_stride[:] = r.v_pool_stride[:] = [512, 128, 64, 1]
        r.positions_stride = r.slots_stride = r.pool_pages = r.page_size = 1
        r.rows, r.q_heads, r.kv_heads, r.head_dim, r.dtype = 2, 4, 2, 64, _lib.TV_BF16
        a.frequencies, a.num_frequencies, a.gain = 0x10000, 32, 1.0
        for name, value in over.items():
            setattr(a if hasattr(a, name) else r, name, value)
        return ctypes.byref(a)

    for over, code, message in [
        (dict(num_frequencies=33), _lib.TV_ERR_INVALID, b"33 frequencies"),
        (dict(num_frequencies=0), _lib.TV_ERR_INVALID, b"0 frequencies"),
        (dict(head_dim=258), _lib.TV_ERR_INVALID, b"head_dim 258"),
        (dict(q_heads=3), _lib.TV_ERR_INVALID, b"GQA"),
        (dict(dtype=9), _lib.TV_ERR_UNSUPPORTED, b"operands"),
        (dict(gain=float("inf")), _lib.TV_ERR_INVALID, b"gain"),
        (dict(rows=2 ** 31), _lib.TV_ERR_UNSUPPORTED, b"too many rows"),
        (dict(frequencies=None), _lib.TV_ERR_INVALID, b"null pointer"),
        (dict(frequencies=0x10004), _lib.TV_ERR_INVALID, b"unaligned"),
        (dict(page_size=0), _lib.TV_ERR_INVALID, b"empty KV pool"),
        (dict(slots_stride=0), _lib.TV_ERR_INVALID, b"positive"),
    ]:
        assert lib.tv_rotary_scatter(turn(**over), None) == code, over
        assert message in lib.tv_last_error(), (over, lib.tv_last_error())
    assert lib.tv_rotary_scatter(turn(rows=0), None) == _lib.TV_OK

    def say(**over):
        a = _lib.TokenLogprobsArgs()
        for name, kind in a._fields_:
            if kind is ctypes.c_void_p:
                setattr(a, name, 0x10000)
        a.logits_stride = a.vocab = 50000
        a.num_logits = a.num_rows = 2
        a.tokens, a.top, a.compute_units = 1, 5, 256
        for name, value in over.items():
            setattr(a, name, value)
        return ctypes.byref(a)

    for over, code, message in [
        (dict(vocab=0), _lib.TV_ERR_INVALID, b"invalid sizes"),
        (dict(logits_stride=49999), _lib.TV_ERR_INVALID, b"invalid sizes"),
        (dict(tokens=-1), _lib.TV_ERR_INVALID, b"invalid sizes"),
        (dict(dtype=4), _lib.TV_ERR_UNSUPPORTED, b"bf16, f16 or fp32"),
        (dict(vocab=2 ** 31, logits_stride=2 ** 31), _lib.TV_ERR_UNSUPPORTED, b"2^31 words"),
        (dict(top=65), _lib.TV_ERR_INVALID, b"65 alternatives"),
        (dict(top=5, vocab=4), _lib.TV_ERR_INVALID, b"5 alternatives"),
        (dict(rows=None, num_rows=3), _lib.TV_ERR_INVALID, b"more results"),
        (dict(num_rows=2 ** 25), _lib.TV_ERR_UNSUPPORTED, b"too many rows"),
        (dict(token_ids=None), _lib.TV_ERR_INVALID, b"null pointer"),
        (dict(top_ids=None), _lib.TV_ERR_INVALID, b"null pointer"),
    ]:
        assert lib.tv_token_logprobs(say(**over), 0x10000, 1 << 40, None) == code, over
        assert message in lib.tv_last_error(), (over, lib.tv_last_error())
    need = lib.tv_token_logprobs_workspace_bytes(say())
    assert need > 0 and lib.tv_token_logprobs(say(), 0x10000, need - 1, None) == _lib.TV_ERR_CAPACITY
    assert lib.tv_token_logprobs(say(num_rows=0), None, 0, None) == _lib.TV_OK
