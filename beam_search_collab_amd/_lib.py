"""ctypes bindings of the two C-ABI libraries built in-tree.

libbs_hip.so  (include/bs_hip.h)   gfx950 search kernels
              (include/bs_embed.h) encoder operators
libbs_host.so (include/bs_host.h)  host formats, index construction, input preparation

Loading fails loudly when a library is missing: there is no CPU fallback for the
search path.
"""
from __future__ import annotations

import ctypes as C
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
HIP_LIB_PATH = os.path.join(_HERE, "libbs_hip.so")
# BS_HOST_LIB names another build of the host library (the sanitizer build: make sanitize-check)
HOST_LIB_PATH = os.environ.get("BS_HOST_LIB") or os.path.join(_HERE, "libbs_host.so")

u32, u64, i32, f32, f64 = C.c_uint32, C.c_uint64, C.c_int32, C.c_float, C.c_double
vp = C.c_void_p
P = C.POINTER


class SearchCfg(C.Structure):
    """bs_search_cfg (include/bs_hip.h)."""
    _fields_ = [
        ("mode", i32),
        ("queries_per_group", u32),
        ("K", u32),
        ("topk_size", u32),
        ("filter_capacity", u32),
        ("entry_point", u32),
        ("max_iterations", i32),
        ("reset_interval", i32),
    ]


class Stats(C.Structure):
    """bs_stats (include/bs_hip.h)."""
    _fields_ = [
        ("kernel_ms", f64),
        ("iterations", u64),
        ("expansions", u64),
        ("dist_evals", u64),
        ("est_evals", u64),
        ("rerank_evals", u64),
    ]

    def as_dict(self) -> dict:
        return {k: getattr(self, k) for k, _ in self._fields_}


i64 = C.c_int64


class AttentionArgs(C.Structure):
    """bs_attention_args (include/bs_embed.h)."""
    _fields_ = (
        [(n, vp) for n in ("q", "k", "v", "out", "lse", "q_offsets", "k_offsets")]
        + [(n, i64) for n in ("q_stride", "q_head_stride", "k_stride", "k_head_stride", "v_stride", "v_head_stride",
                              "out_stride", "out_head_stride")]
        + [(n, u32) for n in ("q_tokens", "k_tokens", "sequences", "heads", "kv_heads", "head_dim", "longest_q", "longest_k")]
        + [("type", i32), ("causal", i32), ("scale", f32)]
    )


class AttentionPrefix(C.Structure):
    """bs_attention_prefix (include/bs_embed.h)."""
    _fields_ = [("k", vp), ("v", vp), ("k_stride", i64), ("k_head_stride", i64), ("v_stride", i64), ("v_head_stride", i64),
                ("tokens", u32)]


class HeadNormRotaryArgs(C.Structure):
    """bs_head_norm_rotary_args (include/bs_embed.h)."""
    _fields_ = (
        [(n, vp) for n in ("q", "k", "q_grad", "k_grad", "q_out", "k_out", "q_weight", "k_weight", "q_weight_grad",
                           "k_weight_grad", "positions", "frequencies")]
        + [(n + e, i64) for n in ("q", "k", "q_grad", "k_grad", "q_out", "k_out") for e in ("_stride", "_head_stride")]
        + [(n, u32) for n in ("tokens", "heads", "kv_heads", "head_dim", "rotary")]
        + [(n, i32) for n in ("interleaved", "norm", "type", "wtype")]
        + [("eps", f32), ("magnitude", f32)]
    )


# name -> (restype, argtypes)
HIP_API = {
    "bs_index_create": (C.c_int, [vp, vp, u64, u32, u32, P(vp)]),
    "bs_index_attach_rabitq": (C.c_int, [vp, vp, vp, vp, u32]),
    "bs_search": (C.c_int, [vp, P(SearchCfg), vp, u64, vp, vp, P(Stats)]),
    "bs_search_device": (C.c_int, [vp, P(SearchCfg), vp, u64, vp, vp, vp, vp, C.c_int, P(Stats)]),
    "bs_search_device_noalloc": (C.c_int, [vp, P(SearchCfg), vp, u64, vp, vp, vp, vp]),
    "bs_index_info": (C.c_int, [vp, P(u64), P(u32), P(u32), P(u32), P(C.c_int)]),
    "bs_index_destroy": (None, [vp]),
    "bs_index_set_query_order": (C.c_int, [vp, C.c_int]),
    "bs_index_label_costs": (C.c_int, [vp, vp]),
    "bs_index_entry_point": (C.c_int, [vp, P(u32)]),
    "bs_index_build_rabitq": (C.c_int, [vp, u32, vp, vp, vp, P(u32)]),
    "bs_build_vamana_device": (C.c_int, [vp, u64, u32, u32, u32, f32, u32, vp, C.c_int]),
    "bs_last_error": (C.c_char_p, []),
    "bs_debug_l2": (C.c_int, [vp, vp, u64, vp, vp, u64, vp]),
    "bs_debug_fastscan": (C.c_int, [vp, vp, u32, u32, vp, vp, u32, u32, f32, vp, vp, vp, vp, vp]),
    "bs_debug_beam": (C.c_int, [u32, vp, u32, u32, u32, C.c_int, vp, vp]),
    "bs_debug_sort": (C.c_int, [vp, u32, vp]),
    "bs_debug_cost_order": (C.c_int, [vp, u64, vp, vp]),
    "bs_debug_label_order": (C.c_int, [vp, vp, u64, u32, u32, vp]),
    "bs_debug_filter": (C.c_int, [C.c_int, u32, vp, u32, u32, vp, vp, u32, vp]),
    "bs_index_groundtruth": (C.c_int, [vp, vp, u64, u32, vp, vp, P(u64)]),
    "bs_index_groundtruth_device": (C.c_int, [vp, vp, u64, u32, vp, vp, vp, P(u64)]),
    "bs_debug_mfma32": (C.c_int, [vp, vp, vp]),
    "bs_debug_mfma32_f16": (C.c_int, [vp, vp, vp]),
    "bs_debug_build_vamana": (C.c_int, [vp, u64, u32, u32, u32, f32, u32, u32, vp, vp]),
    "bs_debug_index_create_uncalibrated": (C.c_int, [vp, vp, u64, u32, u32, P(vp)]),
    "bs_debug_groundtruth": (C.c_int, [vp, vp, u64, u32, u64, vp, vp]),
    "bs_debug_gt_plan": (C.c_int, [u64, u64, u32, vp]),
    "bs_debug_gt_products": (C.c_int, [vp, u32, vp, u32, C.c_int, vp]),
}

# include/bs_embed.h, in libbs_hip.so too
EMBED_API = {
    "bs_layer_norm": (C.c_int, [vp, i64, vp, vp, C.c_int, f32, vp, i64, vp, vp, u64, u32, C.c_int, vp]),
    "bs_layer_norm_backward": (C.c_int, [vp, i64, vp, i64, vp, vp, vp, C.c_int, vp, i64, vp, vp, u64, u32, C.c_int, vp, u64, vp]),
    "bs_layer_norm_backward_workspace": (C.c_int, [u64, u32, C.c_int, P(u64)]),
    "bs_linear": (C.c_int, [vp, i64, vp, i64, vp, vp, i64, vp, i64, u64, u32, u32, C.c_int, C.c_int, C.c_int, vp, u64, vp]),
    "bs_linear_workspace": (C.c_int, [u64, u32, u32, P(u64)]),
    "bs_attention": (C.c_int, [P(AttentionArgs), vp, u64, vp]),
    "bs_attention_workspace": (C.c_int, [P(AttentionArgs), P(u64)]),
    "bs_attention_shared_prefix": (C.c_int, [P(AttentionArgs), P(AttentionPrefix), vp, u64, vp]),
    "bs_attention_shared_prefix_workspace": (C.c_int, [P(AttentionArgs), P(AttentionPrefix), P(u64)]),
    "bs_gated": (C.c_int, [vp, i64, vp, i64, vp, i64, vp, i64, vp, vp, u64, u32, u32, C.c_int, C.c_int, vp]),
    "bs_gated_backward": (C.c_int, [vp, i64] * 6 + [vp, vp, vp, u64, u32, u32, C.c_int, C.c_int, vp, u64, vp]),
    "bs_gated_backward_workspace": (C.c_int, [u64, u32, u32, P(u64)]),
    "bs_head_norm_rotary": (C.c_int, [P(HeadNormRotaryArgs), vp]),
    "bs_head_norm_rotary_backward": (C.c_int, [P(HeadNormRotaryArgs), vp, u64, vp]),
    "bs_head_norm_rotary_backward_workspace": (C.c_int, [P(HeadNormRotaryArgs), P(u64)]),
}

HOST_API = {
    "bs_host_last_error": (C.c_char_p, []),
    "bs_host_free": (None, [vp]),
    "bs_read_vecs": (C.c_int, [C.c_char_p, C.c_int, P(vp), P(u64), P(u32)]),
    "bs_write_vecs": (C.c_int, [C.c_char_p, C.c_int, vp, u64, u32]),
    "bs_read_graph": (C.c_int, [C.c_char_p, P(vp), P(u64), P(u32)]),
    "bs_write_graph": (C.c_int, [C.c_char_p, vp, u64, u32]),
    "bs_read_codebook": (C.c_int, [C.c_char_p, u64, u32, u32, P(u32), P(vp), P(vp), P(vp), P(u32)]),
    "bs_write_codebook": (C.c_int, [C.c_char_p, vp, vp, u64, u32, u32, u32, vp, vp, vp, u32]),
    "bs_entry_point": (u32, [vp, u64, u32]),
    "bs_recall": (f64, [vp, u64, u32, vp, u32, P(u64)]),
    "bs_gen_mixture": (C.c_int, [vp, u64, u32, u32, f32, f32, f32, f32, u64, u64]),
    "bs_gen_normalized": (C.c_int, [vp, u64, u32, u64]),
    "bs_groundtruth": (C.c_int, [vp, u64, vp, u64, u32, u32, vp, C.c_int]),
    "bs_groundtruth_refine": (C.c_int, [vp, u64, vp, u64, u32, vp, u32, u32, vp, C.c_int]),
    "bs_build_vamana": (C.c_int, [vp, u64, u32, u32, u32, f32, u32, C.c_int, C.c_int, vp, C.c_int]),
    "bs_build_rabitq": (C.c_int, [vp, vp, u64, u32, u32, u32, C.c_int, vp, vp, vp, P(u32)]),
    "bs_rabitq_padded_dim": (u32, [u32]),
}


def _bind(lib, api):
    for name, (res, args) in api.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    return lib


_hip = None
_host = None


def hip():
    """libbs_hip.so; raises if it was not built (no fallback exists)."""
    global _hip
    if _hip is None:
        if not os.path.exists(HIP_LIB_PATH):
            raise ImportError(
                f"{HIP_LIB_PATH} is missing: build it with "
                "`python -c 'import __graft_entry__ as g; g.build()'` (make -C beam_search_collab_amd/csrc)")
        _hip = _bind(C.CDLL(HIP_LIB_PATH), {**HIP_API, **EMBED_API})
    return _hip


def host():
    global _host
    if _host is None:
        if not os.path.exists(HOST_LIB_PATH):
            raise ImportError(f"{HOST_LIB_PATH} is missing: run make -C beam_search_collab_amd/csrc")
        _host = _bind(C.CDLL(HOST_LIB_PATH), HOST_API)
    return _host
