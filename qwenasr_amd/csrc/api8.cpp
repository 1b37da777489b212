// C-ABI of the 8-bit layer operators over many rows: int8 activation rows, the
// int8 x int8 product, the int8 KV cache and the attention over it.
#include "qasr_hip.h"
#include "kernels.h"
#include "model.h"

#include <climits>

using namespace qasr;

static int bad(const char *msg) { return qasr_fail(QASR_ERR_INVALID, msg); }

extern "C" int qasr_hip_add_rms_norm_int8(qasr_hip *h, int8_t *q, float *scales, void *sum, const void *x,
                                          const void *res, const float *norm_w, int64_t rows, int64_t hidden, int64_t ld,
                                          float eps, int bf16) {
    if (!q || !scales || !x) return bad("add_rms_norm_int8: null pointer");
    if (hidden <= 0 || hidden > QASR_ROWS8_MAX_HIDDEN) return bad("add_rms_norm_int8: hidden must be in [1, 16384]");
    if (rows < 0 || rows >= (1 << 22) || ld < hidden || ld > INT32_MAX)
        return bad("add_rms_norm_int8: rows or row stride out of range");
    if (!(eps >= 0.0f)) return bad("add_rms_norm_int8: eps must not be negative");
    CHECK_H(h);
    if (rows == 0) return QASR_OK;
    Rows8Args a{};
    a.x = x; a.res = res; a.sum = sum; a.norm_w = norm_w; a.q = q; a.scales = scales;
    a.rows = rows; a.ld = ld; a.H = (int)hidden; a.eps = eps;
    LAUNCHCHK(launch_add_rms_norm_int8(a, bf16 != 0, h->stream), "add_rms_norm_int8");
    return QASR_OK;
}

extern "C" int qasr_hip_gemm_w8a8(qasr_hip *h, void *y, const int8_t *a, const float *a_scales, const int8_t *w,
                                  const float *w_scales, const float *bias, int64_t M, int64_t N, int64_t K, int mode,
                                  int y_bf16) {
    if (!y || !a || !a_scales || !w || !w_scales) return bad("gemm_w8a8: null pointer");
    if (mode != QASR_GEMM_PLAIN && mode != QASR_GEMM_ADDTO && mode != QASR_GEMM_SWIGLU)
        return bad("gemm_w8a8: unknown mode");
    if (M < 0 || M > (1 << 22) || N <= 0 || N > (1 << 28) || K <= 0 || K >= 131072)
        return bad("gemm_w8a8: M must be in [0, 2^22], N in [1, 2^28], K in [1, 131071]");
    if (mode == QASR_GEMM_SWIGLU && N % 2 != 0) return bad("gemm_w8a8: SwiGLU needs an even N");
    CHECK_H(h);
    if (M == 0) return QASR_OK;
    Gemm8Args g{};
    g.a = a; g.as = a_scales; g.w = w; g.ws = w_scales; g.bias = bias; g.y = y; g.M = M; g.N = N; g.K = K;
    LAUNCHCHK(launch_gemm_w8a8(g, mode, y_bf16 != 0, h->stream), "gemm_w8a8");
    return QASR_OK;
}

// what the cache's three entry points share; fills the geometry
static int kv8_args(Kv8Args &c, const int8_t *k8, const int8_t *v8, const float *ks, const float *vs,
                    const int32_t *row_start, const int32_t *pos, int64_t n_rows, int64_t n_seq, int64_t max_rows,
                    int64_t n_kv_heads, int64_t head_dim, int64_t capacity) {
    if (!k8 || !v8 || !ks || !vs || !pos) return bad("kv8: null pointer");
    if (head_dim != 64 && head_dim != 128) return bad("kv8: head_dim must be 64 or 128");
    if (capacity <= 0 || capacity % QASR_KV8_TILE != 0 || capacity > (1 << 30))
        return bad("kv8: capacity must be a positive multiple of 64, at most 2^30");
    if (n_kv_heads <= 0 || n_kv_heads > 1024) return bad("kv8: n_kv_heads must be in [1, 1024]");
    if (n_seq < 0 || n_seq > 32767) return bad("kv8: n_seq must be in [0, 32767]");
    if (n_rows < 0 || n_rows > INT32_MAX || max_rows < 0 || max_rows > (1 << 24))
        return bad("kv8: n_rows or max_rows out of range");
    if (!row_start && n_seq * max_rows > n_rows) return bad("kv8: n_seq * max_rows rows need a larger n_rows");
    if ((((uintptr_t)k8) | (uintptr_t)v8) % 16 != 0) return bad("kv8: k8 and v8 must be 16-byte aligned");
    c.k8 = const_cast<int8_t *>(k8); c.v8 = const_cast<int8_t *>(v8);
    c.ks = const_cast<float *>(ks); c.vs = const_cast<float *>(vs);
    c.row_start = row_start; c.pos = pos; c.n_rows = n_rows; c.max_rows = max_rows; c.n_seq = (int)n_seq;
    c.Hkv = (int)n_kv_heads; c.hd = (int)head_dim; c.cap = (int)capacity;
    return QASR_OK;
}

extern "C" int qasr_hip_kv8_write(qasr_hip *h, int8_t *k8, int8_t *v8, float *k_scales, float *v_scales, const void *k,
                                  const void *v, int64_t ld, const int32_t *row_start, const int32_t *pos,
                                  int64_t n_rows, int64_t n_seq, int64_t max_rows, int64_t n_kv_heads, int64_t head_dim,
                                  int64_t capacity, int bf16) {
    Kv8Args a{};
    if (int rc = kv8_args(a, k8, v8, k_scales, v_scales, row_start, pos, n_rows, n_seq, max_rows, n_kv_heads, head_dim,
                          capacity))
        return rc;
    if (!k || !v) return bad("kv8_write: null pointer");
    if (ld < n_kv_heads * head_dim || ld > INT32_MAX) return bad("kv8_write: row stride out of range");
    CHECK_H(h);
    if (n_seq == 0 || n_rows == 0 || max_rows == 0) return QASR_OK;
    a.k = const_cast<void *>(k); a.v = const_cast<void *>(v); a.ld = ld;
    LAUNCHCHK(launch_kv8_write(a, bf16 != 0, h->stream), "kv8_write");
    return QASR_OK;
}

extern "C" int qasr_hip_kv8_read(qasr_hip *h, void *k, void *v, int64_t ld, const int8_t *k8, const int8_t *v8,
                                 const float *k_scales, const float *v_scales, const int32_t *row_start,
                                 const int32_t *pos, int64_t n_rows, int64_t n_seq, int64_t max_rows, int64_t n_kv_heads,
                                 int64_t head_dim, int64_t capacity, int bf16) {
    Kv8Args a{};
    if (int rc = kv8_args(a, k8, v8, k_scales, v_scales, row_start, pos, n_rows, n_seq, max_rows, n_kv_heads, head_dim,
                          capacity))
        return rc;
    if (!k || !v) return bad("kv8_read: null pointer");
    if (ld < n_kv_heads * head_dim || ld > INT32_MAX) return bad("kv8_read: row stride out of range");
    CHECK_H(h);
    if (n_seq == 0 || n_rows == 0 || max_rows == 0) return QASR_OK;
    a.k = k; a.v = v; a.ld = ld;
    LAUNCHCHK(launch_kv8_read(a, bf16 != 0, h->stream), "kv8_read");
    return QASR_OK;
}

extern "C" int qasr_hip_attention_kv8(qasr_hip *h, void *out, const void *q, int64_t ldq, const int8_t *k8,
                                      const int8_t *v8, const float *k_scales, const float *v_scales,
                                      const int32_t *row_start, const int32_t *pos, int64_t n_rows, int64_t n_seq,
                                      int64_t max_rows, int64_t max_len, int64_t n_heads, int64_t n_kv_heads,
                                      int64_t head_dim, int64_t capacity, float scale, int64_t window, int64_t sinks,
                                      int bf16) {
    AttnKv8Args a{};
    if (int rc = kv8_args(a.c, k8, v8, k_scales, v_scales, row_start, pos, n_rows, n_seq, max_rows, n_kv_heads, head_dim,
                          capacity))
        return rc;
    if (!out || !q) return bad("attention_kv8: null pointer");
    if (n_heads <= 0 || n_heads % n_kv_heads != 0 || n_heads > 65536)
        return bad("attention_kv8: n_heads must be a positive multiple of n_kv_heads");
    if (max_rows * (n_heads / n_kv_heads) > (1 << 30)) return bad("attention_kv8: max_rows x heads of a group out of range");
    if (ldq < n_heads * head_dim || ldq > INT32_MAX) return bad("attention_kv8: row stride out of range");
    if (window < 0 || sinks < 0 || max_len < 0) return bad("attention_kv8: window, sinks and max_len must not be negative");
    CHECK_H(h);
    if (n_seq == 0 || n_rows == 0 || max_rows == 0) return QASR_OK;
    a.q = q; a.ldq = ldq; a.out = out; a.Hq = (int)n_heads; a.G = (int)(n_heads / n_kv_heads); a.scale = scale;
    a.window = std::min<int64_t>(window, (int64_t)1 << 33);       // past any position
    a.sinks = (int)std::min<int64_t>(sinks, capacity);
    a.max_len = (int)(max_len > 0 ? std::min<int64_t>(max_len, capacity) : capacity);
    a.part = reinterpret_cast<float *>(h->scratch);
    LAUNCHCHK(launch_attention_kv8(a, bf16 != 0, h->stream), "attention_kv8");
    return QASR_OK;
}
