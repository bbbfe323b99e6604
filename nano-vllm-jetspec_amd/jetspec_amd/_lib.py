"""ctypes binding of libtreeverify.so (the C ABI declared in include/treeverify.h).

The shared library is built in-tree by ``nano-vllm-jetspec_amd/build.py``.  There
is no fallback: if the library is missing or does not match this binding, every
device entry point raises ``RuntimeError`` naming the problem.
"""
from __future__ import annotations

import ctypes
import struct
from ctypes import POINTER, c_char_p, c_float, c_int32, c_int64, c_uint64, c_void_p
from pathlib import Path
import threading

LIBRARY_PATH = Path(__file__).resolve().parent / "libtreeverify.so"
ABI_VERSION = 5

TV_OK = 0
TV_ERR_INVALID = -1
TV_ERR_UNSUPPORTED = -2
TV_ERR_LAUNCH = -3
TV_ERR_CAPACITY = -4

TV_BF16 = 0
TV_F16 = 1
TV_F32 = 2

TV_STATUS_BAD_PAGE = 1
TV_STATUS_BAD_SLOT = 2
TV_STATUS_BAD_REQUEST = 4
TV_STATUS_BAD_POSITION = 8
TV_STATUS_BAD_DEPTH = 16
TV_STATUS_BAD_BIAS = 32
TV_STATUS_STALE_PLAN = 64
TV_STATUS_NO_PAGES = 128

TV_MAX_HOST_EOS = 8

# Every extern "C" symbol of include/treeverify.h.
EXPORTED_SYMBOLS = (
    "tv_abi_version",
    "tv_last_error",
    "tv_sizeof_tree_attention_args",
    "tv_store_kvcache",
    "tv_copy_accepted_kv_workspace_bytes",
    "tv_copy_accepted_kv",
    "tv_commit_slots",
    "tv_truncate_accepted",
    "tv_truncate_accepted_host_eos",
    "tv_tree_attention_plan",
    "tv_tree_attention_plan_slots",
    "tv_pack_ancestor_words",
    "tv_tree_attention",
    "tv_sizeof_rope_scatter_args",
    "tv_rope_scatter",
    "tv_argmax_rows",
    "tv_tree_accept",
    "tv_ancestor_words_from_parents",
    "tv_bias_from_ancestor_words",
    "tv_tree_attention_plan_capacity",
    "tv_tree_attention_plan_device",
    "tv_tree_attention_plan_capacity_packed",
    "tv_stream_capture_info",
    "tv_tree_attention_noalloc",
    "tv_tree_attention_noalloc_max_workspace",
    "tv_tree_attention_workspace_bytes",
    "tv_tree_attention_fp32",
    "tv_sizeof_tree_attention_fp32_args",
    "tv_tree_attention_fp32_split",
    "tv_tree_attention_fp32_workspace_bytes",
    "tv_tree_attention_fp32_chunk_keys",
    "tv_tree_attention_fp32_keys",
    "tv_tree_attention_fp32_keys_workspace_bytes",
    "tv_sizeof_qk_norm_args",
    "tv_qk_norm_rope_scatter",
    "tv_sizeof_store_e4m3_args",
    "tv_store_kvcache_e4m3",
    "tv_build_block_tables",
    "tv_packed_slot_maps",
    "tv_sizeof_tree_attention_e4m3_args",
    "tv_tree_attention_e4m3_workspace_bytes",
    "tv_tree_attention_e4m3",
    "tv_sizeof_window_attention_args",
    "tv_window_attention_workspace_bytes",
    "tv_window_attention",
    "tv_sizeof_rotary_args",
    "tv_rotary_scatter",
    "tv_sizeof_token_logprobs_args",
    "tv_token_logprobs_workspace_bytes",
    "tv_token_logprobs",
)


class PlanInfo(ctypes.Structure):
    _fields_ = [
        ("num_items", c_int32),
        ("num_groups", c_int32),
        ("num_partial_slots", c_int32),
        ("ancestor_words_per_row", c_int32),
        ("workspace_bytes", c_int64),
    ]


class TreeAttentionArgs(ctypes.Structure):
    _fields_ = [
        ("q", c_void_p),
        ("q_stride_row", c_int64),
        ("q_stride_head", c_int64),
        ("k_pool", c_void_p),
        ("v_pool", c_void_p),
        ("k_stride", c_int64 * 4),
        ("v_stride", c_int64 * 4),
        ("num_blocks", c_int64),
        ("in_dtype", c_int32),
        ("out", c_void_p),
        ("out_stride_row", c_int64),
        ("out_stride_head", c_int64),
        ("out_dtype", c_int32),
        ("cu_seqlens_q", c_void_p),
        ("prefix_lens", c_void_p),
        ("node_counts", c_void_p),
        ("block_tables", c_void_p),
        ("block_table_stride", c_int64),
        ("tree_slots", c_void_p),
        ("ancestor_words", c_void_p),
        ("ancestor_words_per_row", c_int32),
        ("num_requests", c_int32),
        ("total_queries", c_int32),
        ("num_q_heads", c_int32),
        ("num_kv_heads", c_int32),
        ("head_dim", c_int32),
        ("block_size", c_int32),
        ("scale", c_float),
        ("items", c_void_p),
        ("num_items", c_int32),
        ("groups", c_void_p),
        ("num_groups", c_int32),
        ("num_partial_slots", c_int32),
        ("workspace", c_void_p),
        ("workspace_bytes", c_int64),
        ("status", c_void_p),
        ("device_counts", c_void_p),
        ("prefix_slots", c_void_p),
        ("prefix_slots_stride", c_int64),
        ("prefix_slots_is_int64", c_int32),
        ("exact_probabilities", c_int32),
    ]


class TreeAttentionFp32Args(ctypes.Structure):
    _fields_ = [
        ("q", c_void_p),
        ("q_stride_row", c_int64),
        ("q_stride_head", c_int64),
        ("k_pool", c_void_p),
        ("v_pool", c_void_p),
        ("k_stride", c_int64 * 4),
        ("v_stride", c_int64 * 4),
        ("num_blocks", c_int64),
        ("in_dtype", c_int32),
        ("out", c_void_p),
        ("out_stride_row", c_int64),
        ("out_stride_head", c_int64),
        ("out_dtype", c_int32),
        ("cu_seqlens_q", c_void_p),
        ("query_to_request", c_void_p),
        ("query_local_row", c_void_p),
        ("prefix_lens", c_void_p),
        ("node_counts", c_void_p),
        ("block_tables", c_void_p),
        ("block_table_stride", c_int64),
        ("tree_slots", c_void_p),
        ("qq_bias", c_void_p),
        ("qq_bias_offsets", c_void_p),
        ("prefix_slots", c_void_p),
        ("prefix_slots_stride", c_int64),
        ("prefix_slots_is_int64", c_int32),
        ("num_requests", c_int32),
        ("total_queries", c_int32),
        ("num_q_heads", c_int32),
        ("num_kv_heads", c_int32),
        ("head_dim", c_int32),
        ("block_size", c_int32),
        ("scale", c_float),
        ("status", c_void_p),
    ]


class RopeScatterArgs(ctypes.Structure):
    _fields_ = [
        ("q", c_void_p), ("q_stride", c_int64 * 3),
        ("k", c_void_p), ("k_stride", c_int64 * 3),
        ("v", c_void_p), ("v_stride", c_int64 * 3),
        ("positions", c_void_p), ("positions_stride", c_int64), ("positions_is_int64", c_int32),
        ("cache", c_void_p), ("cache_rows", c_int64), ("cache_stride_row", c_int64), ("cache_stride_elem", c_int64),
        ("cache_dtype", c_int32),
        ("k_pool", c_void_p), ("k_pool_stride", c_int64 * 4),
        ("v_pool", c_void_p), ("v_pool_stride", c_int64 * 4),
        ("pool_pages", c_int64), ("page_size", c_int64),
        ("node_slots", c_void_p), ("slots_stride", c_int64), ("slots_is_int64", c_int32),
        ("out", c_void_p), ("out_stride", c_int64 * 3),
        ("rows", c_int64),
        ("q_heads", c_int32), ("kv_heads", c_int32), ("head_dim", c_int32), ("dtype", c_int32),
        ("status", c_void_p),
    ]


class QkNormArgs(ctypes.Structure):
    _fields_ = [
        ("rope", RopeScatterArgs),
        ("q_weight", c_void_p), ("k_weight", c_void_p),
        ("weight_dtype", c_int32), ("eps", c_float), ("pool_e4m3", c_int32),
        ("k_scale", c_void_p), ("k_scale_stride", c_int64 * 3),
        ("v_scale", c_void_p), ("v_scale_stride", c_int64 * 3),
    ]


class StoreE4m3Args(ctypes.Structure):
    _fields_ = [
        ("key", c_void_p), ("key_stride", c_int64 * 3),
        ("value", c_void_p), ("value_stride", c_int64 * 3),
        ("k_cache", c_void_p), ("k_cache_stride", c_int64 * 4),
        ("v_cache", c_void_p), ("v_cache_stride", c_int64 * 4),
        ("k_scale", c_void_p), ("k_scale_stride", c_int64 * 3),
        ("v_scale", c_void_p), ("v_scale_stride", c_int64 * 3),
        ("pool_pages", c_int64), ("page_size", c_int64),
        ("slots", c_void_p), ("slots_stride", c_int64), ("slots_is_int64", c_int32),
        ("rows", c_int64),
        ("kv_heads", c_int32), ("head_dim", c_int32), ("dtype", c_int32),
        ("status", c_void_p),
    ]


class TreeAttentionE4m3Args(ctypes.Structure):
    _fields_ = [
        ("q", c_void_p), ("q_stride_row", c_int64), ("q_stride_head", c_int64), ("in_dtype", c_int32),
        ("k_pool", c_void_p), ("v_pool", c_void_p), ("k_stride", c_int64 * 4), ("v_stride", c_int64 * 4),
        ("k_scale", c_void_p), ("v_scale", c_void_p), ("k_scale_stride", c_int64 * 3), ("v_scale_stride", c_int64 * 3),
        ("num_blocks", c_int64),
        ("out", c_void_p), ("out_stride_row", c_int64), ("out_stride_head", c_int64), ("out_dtype", c_int32),
        ("cu_seqlens_q", c_void_p), ("prefix_lens", c_void_p), ("node_counts", c_void_p),
        ("block_tables", c_void_p), ("block_table_stride", c_int64), ("block_table_width", c_int32),
        ("tree_slots", c_void_p), ("qq_bias", c_void_p), ("qq_bias_offsets", c_void_p), ("qq_bias_elems", c_int64),
        ("num_requests", c_int32), ("total_queries", c_int32), ("num_q_heads", c_int32), ("num_kv_heads", c_int32),
        ("head_dim", c_int32), ("block_size", c_int32),
        ("scale", c_float), ("compute_units", c_int32), ("status", c_void_p),
    ]


class WindowAttentionArgs(ctypes.Structure):
    _fields_ = [
        ("q", c_void_p), ("q_stride_row", c_int64), ("q_stride_head", c_int64), ("in_dtype", c_int32),
        ("k_pool", c_void_p), ("v_pool", c_void_p), ("k_stride", c_int64 * 4), ("v_stride", c_int64 * 4),
        ("num_blocks", c_int64),
        ("out", c_void_p), ("out_stride_row", c_int64), ("out_stride_head", c_int64), ("out_dtype", c_int32),
        ("cu_seqlens_q", c_void_p), ("prefix_lens", c_void_p), ("node_counts", c_void_p),
        ("block_tables", c_void_p), ("block_table_stride", c_int64), ("block_table_width", c_int32),
        ("tree_slots", c_void_p), ("qq_bias", c_void_p), ("qq_bias_offsets", c_void_p), ("qq_bias_elems", c_int64),
        ("positions", c_void_p), ("positions_is_int64", c_int32), ("window", c_int32), ("sinks", c_int32),
        ("num_requests", c_int32), ("total_queries", c_int32), ("num_q_heads", c_int32), ("num_kv_heads", c_int32),
        ("head_dim", c_int32), ("block_size", c_int32),
        ("scale", c_float), ("compute_units", c_int32), ("status", c_void_p),
    ]


class RotaryArgs(ctypes.Structure):
    _fields_ = [
        ("rope", RopeScatterArgs),
        ("frequencies", c_void_p), ("num_frequencies", c_int32), ("interleaved", c_int32), ("gain", c_float),
    ]


class TokenLogprobsArgs(ctypes.Structure):
    _fields_ = [
        ("logits", c_void_p), ("logits_stride", c_int64), ("num_logits", c_int64), ("vocab", c_int64), ("dtype", c_int32),
        ("rows", c_void_p), ("rows_is_int64", c_int32), ("token_ids", c_void_p), ("tokens_is_int64", c_int32),
        ("num_rows", c_int64), ("tokens", c_int32), ("top", c_int32),
        ("logprobs", c_void_p), ("entropy", c_void_p), ("top_ids", c_void_p), ("top_logprobs", c_void_p),
        ("compute_units", c_int32), ("status", c_void_p),
    ]


def _fields_format(structure, base: int = 0) -> list[tuple[int, str, int]]:
    """(offset, struct code, size) of every scalar of a structure, nested ones and arrays laid out flat."""
    codes = {c_void_p: "P", c_int64: "q", c_int32: "i", c_float: "f"}
    found = []
    for name, kind in structure._fields_:
        at = base + getattr(structure, name).offset
        if issubclass(kind, ctypes.Structure):
            found += _fields_format(kind, at)
        elif issubclass(kind, ctypes.Array):
            size = ctypes.sizeof(kind._type_)
            found += [(at + i * size, codes[kind._type_], size) for i in range(kind._length_)]
        else:
            found.append((at, codes[kind], ctypes.sizeof(kind)))
    return found


def packer(structure):
    """``pack(*values)`` of a structure's scalars in order, as the bytes an entry takes: filling a ctypes
    structure field by field costs more than a small kernel."""
    text, at = "=", 0
    for offset, code, size in _fields_format(structure):
        text += "x" * (offset - at) + {"P": "Q"}.get(code, code)
        at = offset + size
    return struct.Struct(text + "x" * (ctypes.sizeof(structure) - at)).pack


pack_qk_norm = packer(QkNormArgs)
pack_store_e4m3 = packer(StoreE4m3Args)
pack_tree_attention_e4m3 = packer(TreeAttentionE4m3Args)
pack_window_attention = packer(WindowAttentionArgs)
pack_rotary = packer(RotaryArgs)
pack_token_logprobs = packer(TokenLogprobsArgs)

_lock = threading.Lock()
_lib = None


def _declare(lib: ctypes.CDLL) -> None:
    lib.tv_abi_version.restype = c_int32
    lib.tv_abi_version.argtypes = []
    lib.tv_last_error.restype = c_char_p
    lib.tv_last_error.argtypes = []
    lib.tv_sizeof_tree_attention_args.restype = c_int64
    lib.tv_sizeof_tree_attention_args.argtypes = []
    lib.tv_store_kvcache.restype = c_int32
    lib.tv_store_kvcache.argtypes = [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_void_p, c_int64,
                                     c_void_p, c_int32, c_int64, c_int64, c_int32, c_void_p, c_void_p]
    lib.tv_copy_accepted_kv_workspace_bytes.restype = c_int64
    lib.tv_copy_accepted_kv_workspace_bytes.argtypes = [c_int64, c_int64, c_int64, c_int32]
    lib.tv_copy_accepted_kv.restype = c_int32
    lib.tv_copy_accepted_kv.argtypes = [c_void_p, POINTER(c_int64), POINTER(c_int64), c_int32, c_void_p,
                                        c_void_p, c_int64, c_void_p, c_int64, POINTER(c_int64), c_void_p,
                                        c_void_p]
    lib.tv_commit_slots.restype = c_int32
    lib.tv_commit_slots.argtypes = [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int32, c_void_p,
                                    c_int32, c_int32, c_int64, c_void_p, c_void_p, c_void_p, c_void_p]
    lib.tv_truncate_accepted.restype = c_int32
    lib.tv_truncate_accepted.argtypes = [c_void_p, c_int32, c_void_p, c_void_p, c_void_p, c_int32, c_void_p, c_int32,
                                         c_void_p, c_void_p, c_void_p, c_int32, c_void_p, c_void_p, c_void_p,
                                         c_void_p, c_void_p, c_void_p]
    lib.tv_truncate_accepted_host_eos.restype = c_int32
    lib.tv_truncate_accepted_host_eos.argtypes = [c_void_p, c_int32, c_void_p, c_void_p, c_void_p, c_int32, c_void_p,
                                                  c_int32, c_void_p, c_void_p, c_void_p, c_int32, c_void_p,
                                                  c_void_p, c_void_p, c_void_p, c_void_p, c_void_p]
    lib.tv_tree_attention_plan.restype = c_int32
    lib.tv_tree_attention_plan.argtypes = [POINTER(c_int32), POINTER(c_int32), c_int32, c_int32, c_int32,
                                           c_int32, c_int32, c_int32, POINTER(c_int32), POINTER(c_int32),
                                           POINTER(PlanInfo)]
    lib.tv_tree_attention_plan_slots.restype = c_int32
    lib.tv_tree_attention_plan_slots.argtypes = [POINTER(c_int32), POINTER(c_int32), c_int32, c_int32, c_int32,
                                                 c_int32, c_int32, POINTER(c_int32), POINTER(c_int32),
                                                 POINTER(PlanInfo)]
    lib.tv_pack_ancestor_words.restype = c_int32
    lib.tv_pack_ancestor_words.argtypes = [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32,
                                           c_int32, c_void_p, c_void_p, c_void_p]
    lib.tv_tree_attention.restype = c_int32
    lib.tv_tree_attention.argtypes = [POINTER(TreeAttentionArgs), c_void_p]
    lib.tv_tree_attention_noalloc.restype = c_int32
    lib.tv_tree_attention_noalloc.argtypes = [POINTER(TreeAttentionArgs), c_void_p]
    lib.tv_tree_attention_noalloc_max_workspace.restype = c_int64
    lib.tv_tree_attention_noalloc_max_workspace.argtypes = []
    lib.tv_tree_attention_workspace_bytes.restype = c_int64
    lib.tv_tree_attention_workspace_bytes.argtypes = [c_int32, c_int32]
    lib.tv_tree_attention_fp32.restype = c_int32
    lib.tv_tree_attention_fp32.argtypes = [POINTER(TreeAttentionFp32Args), c_void_p]
    lib.tv_tree_attention_fp32_split.restype = c_int32
    lib.tv_tree_attention_fp32_split.argtypes = [POINTER(TreeAttentionFp32Args), c_void_p, c_int64, c_void_p]
    lib.tv_tree_attention_fp32_workspace_bytes.restype = c_int64
    lib.tv_tree_attention_fp32_workspace_bytes.argtypes = [c_int32] * 5
    lib.tv_tree_attention_fp32_keys.restype = c_int32
    lib.tv_tree_attention_fp32_keys.argtypes = [POINTER(TreeAttentionFp32Args), c_int32, c_void_p, c_int64, c_void_p]
    lib.tv_tree_attention_fp32_keys_workspace_bytes.restype = c_int64
    lib.tv_tree_attention_fp32_keys_workspace_bytes.argtypes = [c_int32] * 7
    lib.tv_tree_attention_fp32_chunk_keys.restype = c_int32
    lib.tv_tree_attention_fp32_chunk_keys.argtypes = [POINTER(c_int32), POINTER(c_int32), *[c_int32] * 5,
                                                      POINTER(c_int32), POINTER(c_int32)]
    lib.tv_sizeof_tree_attention_fp32_args.restype = c_int64
    lib.tv_sizeof_tree_attention_fp32_args.argtypes = []
    lib.tv_sizeof_rope_scatter_args.restype = c_int64
    lib.tv_sizeof_rope_scatter_args.argtypes = []
    lib.tv_rope_scatter.restype = c_int32
    lib.tv_rope_scatter.argtypes = [POINTER(RopeScatterArgs), c_void_p]
    lib.tv_argmax_rows.restype = c_int32
    lib.tv_argmax_rows.argtypes = [c_void_p, c_int64, c_int64, c_int64, c_int32, c_void_p, c_void_p]
    lib.tv_ancestor_words_from_parents.restype = c_int32
    lib.tv_ancestor_words_from_parents.argtypes = [c_void_p, c_void_p, c_int32, c_int32, c_int32, c_void_p, c_void_p,
                                                   c_void_p]
    lib.tv_bias_from_ancestor_words.restype = c_int32
    lib.tv_bias_from_ancestor_words.argtypes = [c_void_p, c_int32, c_void_p, c_void_p, c_void_p, c_void_p, c_int32,
                                                c_void_p, c_void_p]
    lib.tv_tree_attention_plan_capacity.restype = c_int32
    lib.tv_tree_attention_plan_capacity.argtypes = [POINTER(c_int32), c_int32, c_int32, c_int32, c_int32, c_int32,
                                                    c_int32, c_int64, POINTER(PlanInfo)]
    lib.tv_tree_attention_plan_device.restype = c_int32
    lib.tv_tree_attention_plan_device.argtypes = [c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32, c_int32,
                                                  c_int32, c_int32, c_int32, c_int32, c_void_p, c_void_p, c_void_p,
                                                  c_void_p]
    lib.tv_tree_attention_plan_capacity_packed.restype = c_int32
    lib.tv_tree_attention_plan_capacity_packed.argtypes = [c_int32, c_int32, c_int64, c_int32, c_int32, c_int32,
                                                           c_int32, c_int32, c_int64, POINTER(PlanInfo)]
    lib.tv_stream_capture_info.restype = c_int32
    lib.tv_stream_capture_info.argtypes = [c_void_p, POINTER(c_int32), POINTER(c_uint64)]
    lib.tv_sizeof_qk_norm_args.restype = c_int64
    lib.tv_sizeof_qk_norm_args.argtypes = []
    lib.tv_qk_norm_rope_scatter.restype = c_int32
    lib.tv_qk_norm_rope_scatter.argtypes = [c_void_p, c_void_p]
    lib.tv_sizeof_store_e4m3_args.restype = c_int64
    lib.tv_sizeof_store_e4m3_args.argtypes = []
    lib.tv_store_kvcache_e4m3.restype = c_int32
    lib.tv_store_kvcache_e4m3.argtypes = [c_void_p, c_void_p]
    lib.tv_sizeof_tree_attention_e4m3_args.restype = c_int64
    lib.tv_sizeof_tree_attention_e4m3_args.argtypes = []
    lib.tv_tree_attention_e4m3_workspace_bytes.restype = c_int64
    lib.tv_tree_attention_e4m3_workspace_bytes.argtypes = [c_void_p]   # packed bytes or a structure by reference
    lib.tv_tree_attention_e4m3.restype = c_int32
    lib.tv_tree_attention_e4m3.argtypes = [c_void_p, c_void_p, c_int64, c_void_p]
    # Packed bytes or a structure by reference.
    for name in ("window_attention", "token_logprobs"):
        size, space, entry = (getattr(lib, f) for f in (f"tv_sizeof_{name}_args", f"tv_{name}_workspace_bytes", f"tv_{name}"))
        size.restype, size.argtypes = c_int64, []
        space.restype, space.argtypes = c_int64, [c_void_p]
        entry.restype, entry.argtypes = c_int32, [c_void_p, c_void_p, c_int64, c_void_p]
    lib.tv_sizeof_rotary_args.restype = c_int64
    lib.tv_sizeof_rotary_args.argtypes = []
    lib.tv_rotary_scatter.restype = c_int32
    lib.tv_rotary_scatter.argtypes = [c_void_p, c_void_p]
    lib.tv_build_block_tables.restype = c_int32
    lib.tv_build_block_tables.argtypes = [c_void_p, c_void_p, c_int64, c_int32, c_void_p, c_void_p, c_void_p,
                                          *[c_int32] * 4, *[c_void_p] * 5]
    lib.tv_packed_slot_maps.restype = c_int32
    lib.tv_packed_slot_maps.argtypes = [c_void_p, c_void_p, c_void_p, c_int64, c_int32, c_void_p, c_int32, c_void_p,
                                        c_int32, c_int64, c_int32, c_int64, *[c_void_p] * 7]
    lib.tv_tree_accept.restype = c_int32
    lib.tv_tree_accept.argtypes = [c_void_p, c_void_p, c_int32, c_void_p, c_int32, c_void_p, c_int32, c_void_p,
                                   c_int32, c_int32, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p]


def library() -> ctypes.CDLL:
    """The loaded library; raises RuntimeError if it is absent or mismatched."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not LIBRARY_PATH.exists():
            raise RuntimeError(
                f"{LIBRARY_PATH} is missing: build it with `python nano-vllm-jetspec_amd/build.py` "
                "(there is no non-HIP fallback)")
        lib = ctypes.CDLL(str(LIBRARY_PATH))
        missing = [name for name in EXPORTED_SYMBOLS if not hasattr(lib, name)]
        if missing:
            raise RuntimeError(f"{LIBRARY_PATH} lacks symbols {missing}; rebuild it")
        _declare(lib)
        version = lib.tv_abi_version()
        if version != ABI_VERSION:
            raise RuntimeError(f"libtreeverify ABI {version} != binding ABI {ABI_VERSION}; rebuild it")
        if lib.tv_sizeof_tree_attention_args() != ctypes.sizeof(TreeAttentionArgs):
            raise RuntimeError("tv_tree_attention_args layout differs between library and binding")
        if lib.tv_sizeof_rope_scatter_args() != ctypes.sizeof(RopeScatterArgs):
            raise RuntimeError("tv_rope_scatter_args layout differs between library and binding")
        if lib.tv_sizeof_qk_norm_args() != ctypes.sizeof(QkNormArgs):
            raise RuntimeError("tv_qk_norm_args layout differs between library and binding")
        if lib.tv_sizeof_store_e4m3_args() != ctypes.sizeof(StoreE4m3Args):
            raise RuntimeError("tv_store_e4m3_args layout differs between library and binding")
        if lib.tv_sizeof_tree_attention_e4m3_args() != ctypes.sizeof(TreeAttentionE4m3Args):
            raise RuntimeError("tv_tree_attention_e4m3_args layout differs between library and binding")
        for name, structure in (("window_attention", WindowAttentionArgs), ("rotary", RotaryArgs),
                                ("token_logprobs", TokenLogprobsArgs)):
            if getattr(lib, f"tv_sizeof_{name}_args")() != ctypes.sizeof(structure):
                raise RuntimeError(f"tv_{name}_args layout differs between library and binding")
        _lib = lib
        return lib


def check(code: int, what: str) -> None:
    """Raise for a nonzero C-ABI return code, with the library's message."""
    if code == TV_OK:
        return
    message = library().tv_last_error().decode(errors="replace")
    if code in (TV_ERR_INVALID, TV_ERR_UNSUPPORTED, TV_ERR_CAPACITY):
        raise ValueError(f"{what}: {message}")
    raise RuntimeError(f"{what}: {message} (code {code})")
