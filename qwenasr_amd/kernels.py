"""Host mirror of the reference's ``kernels::`` int8 hot-path API on the GPU.

Function names and argument meaning follow crates/qwen-asr/src/kernels/mod.rs;
buffers are :class:`qwenasr_amd.device.DeviceArray` instead of slices, and
every call runs the HIP kernels of libqasr_hip.so on the array's device
(asynchronously on its stream; reading a result back synchronises).
"""
import ctypes as C

from ._lib import QASR_GEMM_ADDTO, QASR_GEMM_PLAIN, QASR_GEMM_SWIGLU, QASR_ROUND_HALF_AWAY, P, check, lib


def _h(a):
    return a.dev.h


def quantize_bf16_weights_to_int8(w_bf16, out_dim, in_dim, q, scales, round_mode=QASR_ROUND_HALF_AWAY):
    """kernels/mod.rs:1805 — bf16 [out, in] -> int8 q [out, in] + f32 scales [out]."""
    check(lib().qasr_hip_pack_int8_rows(_h(w_bf16), w_bf16.ptr, out_dim, in_dim, round_mode,
                                        q.ptr, scales.ptr))


def quantize_f32_to_int8(x, q, scale):
    """kernels/mod.rs:1795 — x f32 [k] -> q int8 [k], scale f32 [1] (device)."""
    check(lib().qasr_hip_quantize_act(_h(x), x.ptr, x.shape[-1], q.ptr, scale.ptr))


def linear_int8(y, x, w, ws, bias, in_dim, out_dim):
    """int8_matvec_threaded (kernels/mod.rs:839) with optional bias."""
    check(lib().qasr_hip_linear_int8(_h(x), y.ptr, x.ptr, w.ptr, ws.ptr,
                                     bias.ptr if bias is not None else None, in_dim, out_dim))


def linear_nobias_int8_qkv(q, k, v, x, wq, sq, wk, sk, wv, sv, in_dim, q_dim, kv_dim,
                           norm_w=None, eps=1e-6):
    """kernels/mod.rs:884; with norm_w the rms_norm of decoder.rs:583 is fused in front."""
    if norm_w is None:
        check(lib().qasr_hip_linear_int8_qkv(_h(x), q.ptr, k.ptr, v.ptr, x.ptr, wq.ptr, sq.ptr,
                                             wk.ptr, sk.ptr, wv.ptr, sv.ptr, in_dim, q_dim, kv_dim))
    else:
        check(lib().qasr_hip_rmsnorm_linear_int8_qkv(_h(x), q.ptr, k.ptr, v.ptr, x.ptr, norm_w.ptr,
                                                     eps, wq.ptr, sq.ptr, wk.ptr, sk.ptr, wv.ptr,
                                                     sv.ptr, in_dim, q_dim, kv_dim))


def linear_nobias_int8_swiglu(ffn_out, x, w, ws, in_dim, intermediate, norm_w=None, eps=1e-6):
    """kernels/mod.rs:970 (interleaved gate/up rows); optional fused rms_norm."""
    if norm_w is None:
        check(lib().qasr_hip_linear_int8_swiglu(_h(x), ffn_out.ptr, x.ptr, w.ptr, ws.ptr, in_dim,
                                                intermediate))
    else:
        check(lib().qasr_hip_rmsnorm_linear_int8_swiglu(_h(x), ffn_out.ptr, x.ptr, norm_w.ptr, eps,
                                                        w.ptr, ws.ptr, in_dim, intermediate))


def linear_nobias_int8_addto(y, x, w, ws, in_dim, out_dim):
    """kernels/mod.rs:1030 — y += W x."""
    check(lib().qasr_hip_linear_int8_addto(_h(x), y.ptr, x.ptr, w.ptr, ws.ptr, in_dim, out_dim))


def argmax_matvec_int8(x, w, ws, in_dim, out_dim, out_idx, norm_w=None, eps=1e-6):
    """kernels/mod.rs:1832 — writes the index into out_idx (int32 device [1]) and returns it."""
    if norm_w is None:
        check(lib().qasr_hip_argmax_int8(_h(x), x.ptr, w.ptr, ws.ptr, in_dim, out_dim, out_idx.ptr))
    else:
        check(lib().qasr_hip_rmsnorm_argmax_int8(_h(x), x.ptr, norm_w.ptr, eps, w.ptr, ws.ptr,
                                                 in_dim, out_dim, out_idx.ptr))
    return int(out_idx.numpy().reshape(-1)[0])


def argmax_f32_rows(x, rows, cols, out_idx, ld=None):
    """align.rs:312-321 — per-row argmax of device logits x [rows][ld] into out_idx (int32 device [rows])."""
    check(lib().qasr_hip_argmax_f32_rows(_h(x), x.ptr, cols if ld is None else ld, rows, cols, out_idx.ptr))
    return out_idx.numpy().reshape(-1)[:rows].copy()


def rms_norm(out, x, weight, seq_len, hidden, eps):
    """kernels/mod.rs:1191."""
    check(lib().qasr_hip_rms_norm(_h(x), out.ptr, x.ptr, weight.ptr, seq_len, hidden, eps))


def rms_norm_per_head(x, weight, seq_len, n_heads, head_dim, eps):
    """kernels/mod.rs:1214 (in place)."""
    check(lib().qasr_hip_rms_norm_per_head(_h(x), x.ptr, weight.ptr, seq_len, n_heads, head_dim, eps))


def apply_rope_neox(x, cos_vals, sin_vals, seq, n_heads, head_dim):
    """kernels/mod.rs:1738 (in place)."""
    check(lib().qasr_hip_apply_rope_neox(_h(x), x.ptr, cos_vals.ptr, sin_vals.ptr, seq, n_heads,
                                         head_dim))


def causal_attention(out, q, k_base, v_base, head_stride, seq_q, seq_k, n_heads, n_kv_heads,
                     head_dim, scale, q_offset):
    """kernels/mod.rs:1663 — k_base/v_base are DeviceArrays or raw device pointers."""
    kp = k_base.ptr if hasattr(k_base, "ptr") else k_base
    vp = v_base.ptr if hasattr(v_base, "ptr") else v_base
    check(lib().qasr_hip_causal_attention(_h(q), out.ptr, q.ptr, kp, vp, head_stride, seq_q, seq_k,
                                          n_heads, n_kv_heads, head_dim, scale, q_offset))


def causal_attention_bf16kv(out, q, k_base, v_base, head_stride, seq_k, n_heads, n_kv_heads, head_dim,
                            scale, q_offset):
    """Single-query attention over a bf16 [kv_head][pos][head_dim] cache (config 3)."""
    kp = k_base.ptr if hasattr(k_base, "ptr") else k_base
    vp = v_base.ptr if hasattr(v_base, "ptr") else v_base
    check(lib().qasr_hip_causal_attention_bf16kv(_h(q), out.ptr, q.ptr, kp, vp, head_stride, seq_k, n_heads,
                                                 n_kv_heads, head_dim, scale, q_offset))


def linear(y, x, w_bf16, bias, seq_len, in_dim, out_dim, accumulate=False):
    """linear / linear_accumulate (kernels/mod.rs:550, 591) on bf16-valued weights."""
    check(lib().qasr_hip_linear_bf16w(_h(x), y.ptr, x.ptr, w_bf16.ptr, bias.ptr if bias is not None else None,
                                      seq_len, in_dim, out_dim, 1 if accumulate else 0))


def gemm_w8_bf16(y, a_bf16, w_int8, scales, M, N, K):
    """y[M, N] = (a_bf16 [M, K] . w_int8[N, K]^T) * scales[N] on MFMA."""
    check(lib().qasr_hip_gemm_w8_bf16(_h(a_bf16), y.ptr, a_bf16.ptr, w_int8.ptr, scales.ptr, M, N, K))


def layer_norm(out, x, weight, bias, seq_len, hidden, eps):
    """kernels/mod.rs:1160."""
    check(lib().qasr_hip_layer_norm(_h(x), out.ptr, x.ptr, weight.ptr, bias.ptr, seq_len, hidden, eps))


def bidirectional_attention(out, q, k, v, seq, n_heads, head_dim, scale, window_tokens):
    """kernels/mod.rs:1386 with windows of window_tokens positions."""
    check(lib().qasr_hip_bidirectional_attention(_h(q), out.ptr, q.ptr, k.ptr, v.ptr, seq, n_heads, head_dim,
                                                 scale, window_tokens))


# ---------------------------------------------------------------------------
# an 8-bit decoder layer over many rows and sequences (no counterpart in the
# reference): include/qasr_hip.h holds the definitions and the cache's layout
# ---------------------------------------------------------------------------

def _p(a):
    return a.ptr if a is not None else None


def add_rms_norm_int8(q, scales, x, norm_w, rows, hidden, res=None, sum_out=None, ld=None, eps=1e-6, bf16=False):
    """int8 rows q [rows][hidden] and scales [rows] of RMSNorm(x + res) * norm_w.

    res None: no addition; norm_w None: no norm.  sum_out receives x + res and
    may be x or res.  x, res, sum_out: f32 (or bf16) rows ld elements apart."""
    check(lib().qasr_hip_add_rms_norm_int8(_h(x), q.ptr, scales.ptr, _p(sum_out), x.ptr, _p(res), _p(norm_w), rows, hidden,
                                           hidden if ld is None else ld, eps, 1 if bf16 else 0))


def gemm_w8a8(y, a, a_scales, w, w_scales, M, N, K, bias=None, accumulate=False, swiglu=False, bf16=False):
    """y[M, N] = (a_int8 [M, K] . w_int8 [N, K]^T) * a_scales[M] * w_scales[N] (+ bias); y f32 or bf16.

    accumulate: y = (y + bias) + product; swiglu: interleaved gate / up rows,
    y [M, N / 2] = silu(gate) * up."""
    if accumulate and swiglu:
        raise ValueError("gemm_w8a8: accumulate and swiglu exclude each other")
    mode = QASR_GEMM_ADDTO if accumulate else QASR_GEMM_SWIGLU if swiglu else QASR_GEMM_PLAIN
    check(lib().qasr_hip_gemm_w8a8(_h(a), y.ptr, a.ptr, a_scales.ptr, w.ptr, w_scales.ptr, _p(bias), M, N, K, mode,
                                   1 if bf16 else 0))


def kv8_write(k8, v8, k_scales, v_scales, k, v, pos, n_rows, n_seq, max_rows, n_kv_heads, head_dim, capacity,
              row_start=None, ld=None, bf16=False):
    """Rows k, v of n_seq sequences into the int8 cache: row i of sequence j at position pos[j] + i.

    row_start (int32 [n_seq + 1]): the sequences' rows; None: max_rows each.
    ld: elements between rows (default n_kv_heads * head_dim)."""
    check(lib().qasr_hip_kv8_write(_h(k8), k8.ptr, v8.ptr, k_scales.ptr, v_scales.ptr, k.ptr, v.ptr,
                                   n_kv_heads * head_dim if ld is None else ld, _p(row_start), pos.ptr, n_rows, n_seq,
                                   max_rows, n_kv_heads, head_dim, capacity, 1 if bf16 else 0))


def kv8_read(k, v, k8, v8, k_scales, v_scales, pos, n_rows, n_seq, max_rows, n_kv_heads, head_dim, capacity,
             row_start=None, ld=None, bf16=False):
    """The int8 cache's values back into f32 (or bf16) rows k, v; arguments as kv8_write."""
    check(lib().qasr_hip_kv8_read(_h(k8), k.ptr, v.ptr, n_kv_heads * head_dim if ld is None else ld, k8.ptr, v8.ptr,
                                  k_scales.ptr, v_scales.ptr, _p(row_start), pos.ptr, n_rows, n_seq, max_rows, n_kv_heads,
                                  head_dim, capacity, 1 if bf16 else 0))


def attention_kv8(out, q, k8, v8, k_scales, v_scales, pos, n_rows, n_seq, max_rows, n_heads, n_kv_heads, head_dim,
                  capacity, scale, row_start=None, ldq=None, max_len=0, window=0, sinks=0, bf16=False):
    """softmax(scale q k) v over the int8 cache: row i of sequence j sees the positions up to pos[j] + i,
    with window > 0 the last `window` of those and the first `sinks`."""
    check(lib().qasr_hip_attention_kv8(_h(q), out.ptr, q.ptr, n_heads * head_dim if ldq is None else ldq, k8.ptr, v8.ptr,
                                       k_scales.ptr, v_scales.ptr, _p(row_start), pos.ptr, n_rows, n_seq, max_rows, max_len,
                                       n_heads, n_kv_heads, head_dim, capacity, scale, window, sinks, 1 if bf16 else 0))
