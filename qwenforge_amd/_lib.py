"""ctypes binding of the C ABI in ``include/qf_attn.h``, ``include/qf_step.h``,
``include/qf_wide.h``, ``include/qf_prefill.h``, ``include/qf_paged.h``,
``include/qf_prefix.h``, ``include/qf_verify.h``, ``include/qf_paged8.h`` and
``include/qf_probe.h``.

The shared object is built in-tree by ``qwenforge_amd.build``.  There is no
fallback: if it is missing or does not load, every op raises.
"""

from __future__ import annotations

import ctypes as C
import threading
from pathlib import Path

LIB_PATH = Path(__file__).resolve().with_name("_qf_attn.so")

_i64, _i32, _f32, _vp = C.c_int64, C.c_int, C.c_float, C.c_void_p


# name -> argument types, in header order.  Every entry point returns int.
SIGNATURES = {
    "qf_decode_attn": [
        _vp, _i64, _i64, _i64,          # q, q_sb, q_sh, q_sg
        _vp, _i64, _i64, _i64,          # k, k_sb, k_sh, k_sn
        _vp, _i64, _i64, _i64,          # v, v_sb, v_sh, v_sn
        _vp, _i64,                      # bias, bias_sb
        _vp, _i64,                      # kv_last, kv_last_sb
        _vp, _vp, _vp, _i32,            # acc, m, l, splits
        _vp,                            # ticket
        _vp, _i64, _i64, _i64,          # out, o_sb, o_sh, o_sg
        _i32, _i32, _i32, _i32, _i32,   # B, KVH, G, D, cap
        _f32, _vp,                      # scale, stream
    ],
    "qf_decode_waves": [_i32, _i32, _i32, _i32, _i32, _i32],   # B, KVH, G, cap, splits, fused
    "qf_decode_shares": [_i32, _i32, _i32, _i32, _i32],        # B, KVH, G, cap, splits
    "qf_decode_attn_noalloc": [
        _vp, _i64, _i64, _i64,          # q, q_sb, q_sh, q_sg
        _vp, _i64, _i64, _i64,          # k, k_sb, k_sh, k_sn
        _vp, _i64, _i64, _i64,          # v, v_sb, v_sh, v_sn
        _vp, _i64,                      # bias, bias_sb
        _vp, _i64,                      # kv_last, kv_last_sb
        _i32,                           # splits
        _vp, _i64, _i64, _i64,          # out, o_sb, o_sh, o_sg
        _i32, _i32, _i32, _i32, _i32,   # B, KVH, G, D, cap
        _f32, _vp,                      # scale, stream
    ],
    "qf_decode_split": [
        _vp, _i64, _i64, _i64,          # q
        _vp, _i64, _i64, _i64,          # k
        _vp, _i64, _i64, _i64,          # v
        _vp, _i64,                      # bias, bias_sb
        _vp, _i64,                      # kv_last, kv_last_sb
        _vp, _vp, _vp, _i32,            # acc, m, l, splits
        _i32, _i32, _i32, _i32, _i32,   # B, KVH, G, D, cap
        _f32, _vp,                      # scale, stream
    ],
    "qf_decode_split_capacity": [
        _vp, _i64, _i64, _i64,          # q
        _vp, _i64, _i64, _i64,          # k
        _vp, _i64, _i64, _i64,          # v
        _vp, _i64,                      # bias, bias_sb
        _vp, _i64,                      # kv_last, kv_last_sb
        _vp, _vp, _vp, _i32,            # acc, m, l, splits
        _i32, _i32, _i32, _i32, _i32,   # B, KVH, G, D, cap
        _f32, _vp,                      # scale, stream
    ],
    "qf_decode_combine": [
        _vp, _vp, _vp, _i32,            # acc, m, l, splits
        _vp, _i64, _i64, _i64,          # out, o_sb, o_sh, o_sg
        _i32, _i32, _i32, _i32,         # B, KVH, G, D
        _vp,                            # stream
    ],
    "qf_prefill_attn": [
        _vp, _i64, _i64, _i64,          # q
        _vp, _i64, _i64, _i64,          # k
        _vp, _i64, _i64, _i64,          # v
        _vp, _vp, _i64, _i64,           # cos, sin, cs_sb, cs_sn
        _vp, _i64, _i64, _i64,          # k_cache
        _vp, _i64, _i64, _i64,          # v_cache
        _i64, _i32,                     # start_pos, cap
        _vp, _i64, _i64, _i64,          # out
        _i32, _i32, _i32, _i32, _i32,   # B, QH, KVH, S, D
        _f32, _vp,                      # scale, stream
    ],
    "qf_prefill_varlen": [
        _vp, _i64, _i64,                # q, q_sh, q_sn
        _vp, _i64, _i64,                # k
        _vp, _i64, _i64,                # v
        _vp, _i32, _i32,                # cu_seqlens, total, max_seqlen
        _vp, _vp, _i64,                 # cos, sin, cs_sn
        _vp, _i64, _i64, _i64,          # k_cache
        _vp, _i64, _i64, _i64,          # v_cache
        _i64, _i32,                     # start_pos, cap
        _vp, _i64, _i64,                # out, o_sh, o_sn
        _i32, _i32, _i32, _i32,         # B, QH, KVH, D
        _f32, _vp,                      # scale, stream
    ],
    "qf_rope_append": [
        _vp, _i64, _i64,                # q, q_sb, q_sh
        _vp, _i64, _i64,                # k
        _vp, _i64, _i64,                # v
        _vp, _vp, _i64,                 # cos, sin, cs_sb
        _vp, _i64, _i64, _i64,          # k_cache
        _vp, _i64, _i64, _i64,          # v_cache
        _vp,                            # write_index
        _vp, _i64, _i64,                # q_out
        _i32, _i32, _i32, _i32, _i32,   # B, QH, KVH, D, cap
        _vp,                            # stream
    ],
    # include/qf_step.h
    "qf_rms_qkv_rope_append": [
        _vp, _i64, _vp,                 # x, x_sb, token
        _vp, _i64,                      # hidden_out, ho_sb
        _vp, _f32,                      # norm_w, eps
        _vp, _i32, _vp,                 # w_qkv, w_layout, bias
        _vp, _vp, _i64,                 # cos, sin, cs_sb
        _vp, _vp,                       # pos, inv_freq
        _vp, _i64, _i64, _i64,          # k_cache
        _vp, _i64, _i64, _i64,          # v_cache
        _vp,                            # write_index
        _vp, _i64, _i64,                # q_out, qo_sb, qo_sh
        _i32, _i32, _i32, _i32, _i32, _i32,  # B, hidden, QH, KVH, D, cap
        _vp,                            # stream
    ],
    "qf_gemv_residual": [
        _vp, _i64, _vp,                 # inp, in_sb, w
        _vp, _i64,                      # hidden, h_sb
        _i32, _i32, _i32,               # B, K, N
        _vp,                            # stream
    ],
    "qf_attn_merge_o_proj": [
        _vp, _vp, _vp, _i32,            # acc, m, l, splits
        _i32, _i32,                     # KVH, G
        _vp, _i32, _vp, _i64,           # w_o, w_layout, hidden, h_sb
        _i32, _i32,                     # B, N
        _vp,                            # stream
    ],
    "qf_rms_gate_up_swiglu": [
        _vp, _i64, _vp, _f32,           # x, x_sb, norm_w, eps
        _vp, _i32, _vp, _i64,           # w_gate_up, w_layout, h_out, ho_sb
        _i32, _i32, _i32,               # B, hidden, I
        _vp,                            # stream
    ],
    "qf_rms_lm_head": [
        _vp, _i64, _vp, _f32,           # x, x_sb, norm_w, eps
        _vp, _i32, _vp, _i64, _vp,      # w_lm, w_layout, logits, lg_sb, keys
        _i32, _i32, _i32, _i32,         # n_blocks, B, hidden, V
        _vp,                            # stream
    ],
    "qf_argmax_step": [
        _vp, _i32, _i32, _vp,           # keys, n_blocks, B, token
        _vp, _i64, _i32,                # rows, rows_sb, n_rows
        _vp, _vp, _vp,                  # step, write_index, pos
        _vp,                            # stream
    ],
    # include/qf_paged.h
    "qf_decode_attn_paged": [
        _vp, _i64, _i64, _i64,          # q, q_sb, q_sh, q_sg
        _vp, _i64, _i64, _i64,          # k_pool, kp_sp, kp_sh, kp_sn
        _vp, _i64, _i64, _i64,          # v_pool, vp_sp, vp_sh, vp_sn
        _vp, _i64, _i32, _i32, _i32,    # block_table, bt_sb, pages_per_row, n_pages, page_size
        _vp, _i64,                      # bias, bias_sb
        _vp, _i64,                      # kv_last, kv_last_sb
        _vp, _vp, _vp, _i32,            # acc, m, l, splits
        _vp,                            # ticket
        _vp, _i64, _i64, _i64,          # out, o_sb, o_sh, o_sg
        _i32, _i32, _i32, _i32,         # B, KVH, G, D
        _f32, _vp,                      # scale, stream
    ],
    "qf_decode_split_paged": [
        _vp, _i64, _i64, _i64,          # q
        _vp, _i64, _i64, _i64,          # k_pool
        _vp, _i64, _i64, _i64,          # v_pool
        _vp, _i64, _i32, _i32, _i32,    # block_table, bt_sb, pages_per_row, n_pages, page_size
        _vp, _i64,                      # bias, bias_sb
        _vp, _i64,                      # kv_last, kv_last_sb
        _vp, _vp, _vp, _i32,            # acc, m, l, splits
        _i32, _i32, _i32, _i32,         # B, KVH, G, D
        _f32, _vp,                      # scale, stream
    ],
    "qf_rope_append_paged": [
        _vp, _i64, _i64,                # q, q_sb, q_sh
        _vp, _i64, _i64,                # k
        _vp, _i64, _i64,                # v
        _vp, _vp, _i64,                 # cos, sin, cs_sb
        _vp, _i64, _i64, _i64,          # k_pool
        _vp, _i64, _i64, _i64,          # v_pool
        _vp, _i64, _i32, _i32, _i32,    # block_table, bt_sb, pages_per_row, n_pages, page_size
        _vp, _i64,                      # slots, slot_sb
        _vp, _i64, _i64,                # q_out
        _i32, _i32, _i32, _i32,         # B, QH, KVH, D
        _vp,                            # stream
    ],
    "qf_prefill_varlen_paged": [
        _vp, _i64, _i64,                # q, q_sh, q_sn
        _vp, _i64, _i64,                # k
        _vp, _i64, _i64,                # v
        _vp, _i32, _i32,                # cu_seqlens, total, max_seqlen
        _vp, _vp, _i64,                 # cos, sin, cs_sn
        _vp, _i64, _i64, _i64,          # k_pool
        _vp, _i64, _i64, _i64,          # v_pool
        _vp, _i64, _i32, _i32, _i32,    # block_table, bt_sb, pages_per_row, n_pages, page_size
        _i64,                           # start_pos
        _vp, _i64, _i64,                # out, o_sh, o_sn
        _i32, _i32, _i32, _i32,         # B, QH, KVH, D
        _f32, _vp,                      # scale, stream
    ],
    "qf_rms_qkv_rope_append_paged": [
        _vp, _i64, _vp,                 # x, x_sb, token
        _vp, _i64,                      # hidden_out, ho_sb
        _vp, _f32,                      # norm_w, eps
        _vp, _i32, _vp,                 # w_qkv, w_layout, bias
        _vp, _vp, _i64,                 # cos, sin, cs_sb
        _vp, _vp,                       # pos, inv_freq
        _vp, _i64, _i64, _i64,          # k_pool
        _vp, _i64, _i64, _i64,          # v_pool
        _vp, _i64, _i32, _i32, _i32,    # block_table, bt_sb, pages_per_row, n_pages, page_size
        _vp, _i64,                      # slots, slot_sb
        _vp, _i64, _i64,                # q_out, qo_sb, qo_sh
        _i32, _i32, _i32, _i32, _i32,   # B, hidden, QH, KVH, D
        _vp,                            # stream
    ],
    "qf_pack_weight": [
        _vp, _i64, _vp,                 # w, w_sb, packed
        _i32, _i32, _i32,               # N, K, layout
        _vp,                            # stream
    ],
    # include/qf_wide.h
    "qf_wide_qkv": [
        _vp, _i64, _vp, _f32,           # x, x_sb, norm_w, eps
        _vp, _vp, _vp, _vp,             # w_qkv, bias, pos, inv_freq
        _vp, _i64, _i64, _i64,          # k_cache
        _vp, _i64, _i64, _i64,          # v_cache
        _vp, _i64, _i32, _i32, _i32,    # block_table, bt_sb, pages_per_row, n_pages, page_size
        _vp, _i64,                      # slots, slot_sb
        _vp, _i64, _i64,                # q_out, qo_sb, qo_sh
        _i32, _i32, _i32, _i32, _i32, _i32,  # B, hidden, QH, KVH, D, cap
        _vp,                            # stream
    ],
    "qf_wide_splits": [_i32],           # K
    "qf_wide_gemv_residual": [
        _vp, _i64, _vp, _vp, _i64,      # inp, in_sb, w, hidden, h_sb
        _vp, _vp, _i32, _i32, _i32,     # part, ticket, B, K, N
        _vp,                            # stream
    ],
    "qf_wide_gate_up": [
        _vp, _i64, _vp, _f32, _vp,      # x, x_sb, norm_w, eps, w_gate_up
        _vp, _i64, _i32, _i32, _i32,    # h_out, ho_sb, B, hidden, I
        _vp,                            # stream
    ],
    "qf_wide_lm_head": [
        _vp, _i64, _vp, _f32, _vp,      # x, x_sb, norm_w, eps, w_lm
        _vp, _i64, _vp, _i32,           # logits, lg_sb, keys, n_blocks
        _i32, _i32, _i32, _vp,          # B, hidden, V, stream
    ],
    "qf_wide_argmax_step": [
        _vp, _i32, _i32, _vp,           # keys, n_blocks, B, token
        _vp, _i64, _i32,                # rows, rows_sb, n_rows
        _vp, _vp, _vp, _vp,             # step, write_index, pos, stream
    ],
    # include/qf_prefill.h
    "qf_prefill_layers_workspace": [_i32, _i32, _i32, _i32, _i32, _i32],  # T, hidden, QH, KVH, D, I
    "qf_extend_layers_workspace": [_i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32],  # ..., B, cap
    "qf_extend_layers": [
        _vp, _i32, _vp, _i32, _i32,     # layers, n_layers, hidden, T, B
        _vp, _vp, _i64, _i32, _vp,      # cu, context, ctx_sb, cap, inv_freq
        _vp, _i64, _i32, _i32, _i32,    # block_table, bt_sb, pages_per_row, n_pages, page_size
        _vp, _i64, _f32,                # ws, ws_bytes, eps
        _i32, _i32, _i32, _i32, _i32,   # hidden_size, QH, KVH, D, I
        _vp,                            # stream
    ],
    "qf_extend_layers_paged8_workspace": [_i32] * 9,  # T, hidden, QH, KVH, D, I, B, max_seqlen, cap
    "qf_extend_layers_paged8": [
        _vp, C.c_char_p, _i32, _vp,     # layers, pools, n_layers, hidden
        _i32, _i32, _i32,               # T, B, max_seqlen
        _vp, _vp, _i64, _i32, _vp,      # cu, context, ctx_sb, cap, inv_freq
        _vp, _i64, _f32,                # ws, ws_bytes, eps
        _i32, _i32, _i32, _i32, _i32,   # hidden_size, QH, KVH, D, I
        _vp,                            # stream
    ],
    "qf_prefill_layers": [
        _vp, _i32, _vp, _i32, _i32, _i32,  # layers, n_layers, hidden, T, B, S
        _vp, _vp,                       # cu, inv_freq
        _vp, _i64, _i32, _i32, _i32,    # block_table, bt_sb, pages_per_row, n_pages, page_size
        _vp, _i64, _f32,                # ws, ws_bytes, eps
        _i32, _i32, _i32, _i32, _i32,   # hidden_size, QH, KVH, D, I
        _vp,                            # stream
    ],
    # include/qf_prefix.h
    "qf_copy_pages": [
        C.POINTER(_vp), _i32, _i32, _i64,  # pools, n_pools, per, step
        _i64, _i64, _i64,               # sp, sh, sn
        _vp, _vp, _vp, _i32,            # src, dst, slots, n_pairs
        _i32, _i32, _i32, _i32, _vp,    # n_pages, KVH, page_size, D, stream
    ],
    "qf_decode_attn_prefix_workspace": [_i32, _i32, _i32, _i32, _i32],  # B, KVH, G, n_groups, cap
    "qf_decode_attn_prefix_paged": [
        _vp, _i64, _i64, _i64,          # q, q_sb, q_sh, q_sg
        _vp, _i64, _i64, _i64,          # k_pool, kp_sp, kp_sh, kp_sn
        _vp, _i64, _i64, _i64,          # v_pool, vp_sp, vp_sh, vp_sn
        _vp, _i64, _i32, _i32, _i32,    # block_table, bt_sb, pages_per_row, n_pages, page_size
        _vp, _vp, _i32,                 # prefix_rows, prefix_len, n_groups
        _vp, _i64, _i32,                # prefix_table, pt_sb, prefix_pages
        _vp, _i64,                      # kv_last, kv_last_sb
        _vp, _i64,                      # ws, ws_bytes
        _vp, _i64, _i64, _i64,          # out, o_sb, o_sh, o_sg
        _i32, _i32, _i32, _i32,         # B, KVH, G, D
        _f32, _vp,                      # scale, stream
    ],
    "qf_prefill_extend_workspace": [_i32, _i32, _i32, _i32, _i32],      # B, QH, KVH, total, cap
    "qf_prefill_extend_paged": [
        _vp, _i64, _i64,                # q, q_sh, q_sn
        _vp, _i64, _i64,                # k
        _vp, _i64, _i64,                # v
        _vp, _i32,                      # cu_seqlens, total
        _vp, _i64,                      # context, ctx_sb
        _vp, _vp, _i64,                 # cos, sin, cs_sn
        _vp, _i64, _i64, _i64,          # k_pool
        _vp, _i64, _i64, _i64,          # v_pool
        _vp, _i64, _i32, _i32, _i32,    # block_table, bt_sb, pages_per_row, n_pages, page_size
        _i32, _vp, _i64,                # cap, ws, ws_bytes
        _vp, _i64, _i64,                # out, o_sh, o_sn
        _i32, _i32, _i32, _i32,         # B, QH, KVH, D
        _f32, _vp,                      # scale, stream
    ],
    # include/qf_verify.h
    "qf_verify_workspace": [_i32, _i32, _i32],                          # T, B, V
    "qf_verify_drafts": [
        _vp, _i32, _i64, _vp, _vp,      # logits, dtype, lg_sn, tokens, cu_seqlens
        _vp, _vp, _vp, _i64, C.c_double,  # accept_u, sample_u, draft_probs, dp_sn, temperature
        _vp, _i32, _vp, _vp, _i64,      # out, width, count, ws, ws_bytes
        _i32, _i32, _i32, _vp,          # T, B, V, stream
    ],
    # include/qf_paged8.h
    "qf_append_paged8": [C.c_char_p, _vp],   # QfRows8, stream
    "qf_read_paged8": [C.c_char_p, _vp],     # QfRows8, stream
    "qf_copy_pages8": [
        _vp, _i32, _i64, _i64, _i64,    # store, layers, layer_step, step, bytes
        _vp, _vp, _i32, _i32, _vp,      # src, dst, n_pairs, n_pages, stream
    ],
    "qf_decode_attn_paged8_workspace": [_i32, _i32, _i32, _i32],        # B, KVH, G, cap
    "qf_decode_attn_paged8": [C.c_char_p, _vp],                         # QfDecode8, stream
    "qf_decode_split_paged8": [C.c_char_p, _vp, _vp, _vp, _i32, _vp],   # QfDecode8, acc, m, l, splits, stream
    "qf_prefill_extend_paged8_workspace": [_i32, _i32, _i32, _i32, _i32, _i32],  # B, QH, KVH, total, longest, cap
    "qf_prefill_extend_paged8": [C.c_char_p, _vp],                      # QfExtend8, stream
    # include/qf_probe.h
    "qf_stream_read": [_vp, _i64, _vp, _i32, _vp],   # src, bytes, sink, workgroups, stream
    "qf_launch_probe": [_vp, _i64, _vp, _vp,          # src, bytes, index, sink
                        _i32, _i32, _i32, _vp],      # workgroups, threads, round_trips, stream
    "qf_decode_split_valu": [
        _vp, _i64, _i64, _i64,          # q
        _vp, _i64, _i64, _i64,          # k
        _vp, _i64, _i64, _i64,          # v
        _vp, _i64,                      # kv_last, kv_last_sb
        _vp, _vp, _vp, _i32,            # acc, m, l, splits
        _i32, _i32, _i32, _i32, _i32,   # B, KVH, G, D, cap
        _f32, _vp,                      # scale, stream
    ],
    "qf_error_string": [_i32],
    "qf_abi_version": [],
}

# The same arguments as the calls that give every row the same splits.
for _name in ("qf_decode_attn", "qf_decode_attn_paged"):
    SIGNATURES[_name + "_shared"] = SIGNATURES[_name]

# Entry points that do not return an int status.
RESTYPES = {"qf_error_string": C.c_char_p, "qf_prefill_layers_workspace": _i64,
            "qf_decode_attn_prefix_workspace": _i64, "qf_prefill_extend_workspace": _i64,
            "qf_extend_layers_workspace": _i64, "qf_verify_workspace": _i64,
            "qf_extend_layers_paged8_workspace": _i64, "qf_decode_attn_paged8_workspace": _i64, "qf_prefill_extend_paged8_workspace": _i64}

_lock = threading.Lock()
_lib: C.CDLL | None = None


def load() -> C.CDLL:
    """Load ``_qf_attn.so`` once; raise ``RuntimeError`` if it is unavailable."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `python -m qwenforge_amd.build` "
                "(the HIP kernels have no fallback)"
            )
        lib = C.CDLL(str(LIB_PATH))
        for name, argtypes in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.argtypes = argtypes
            fn.restype = RESTYPES.get(name, C.c_int)
        _lib = lib
        return lib


def check(code: int, name: str) -> None:
    """Raise ``RuntimeError`` for a non-zero return code of entry point ``name``."""
    if code != 0:
        msg = load().qf_error_string(code).decode()
        raise RuntimeError(f"{name} failed with code {code}: {msg}")
