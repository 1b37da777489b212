// C-ABI of the operators for several hypotheses of one prompt: pages of a KV cache
// forked, compacted and written, the attention over them, log probabilities.
#include "qasr_hip.h"
#include "kernels.h"
#include "model.h"

#include <climits>
#include <cmath>

using namespace qasr;

static int bad(const char *msg) { return qasr_fail(QASR_ERR_INVALID, msg); }

static bool overlap(const void *a, int64_t na, const void *b, int64_t nb) {
    const char *x = (const char *)a, *y = (const char *)b;
    return a && b && na > 0 && nb > 0 && x < y + nb && y < x + na;
}

static bool off_type(const void *p, int bf16) { return (uintptr_t)p % (bf16 ? 2 : 4) != 0; }

// log2 of a page's positions, -1 for a size that is none
static int page_shift(int64_t page) {
    for (int s = 4; s <= 8; s++)
        if (page == (int64_t)1 << s) return s;
    return -1;
}

static int seq_args(int64_t n_seq, int64_t table_ld, int64_t n_pages, int64_t page) {
    if (page_shift(page) < 0) return bad("kvp: page must be 16, 32, 64, 128 or 256");
    if (n_pages <= 0 || n_pages > QASR_KVP_MAX_PAGES) return bad("kvp: n_pages must be in [1, 2^18]");
    if (n_seq < 0 || n_seq > QASR_KVP_MAX_SEQ) return bad("kvp: at most 2048 sequences");
    if (table_ld <= 0 || table_ld > (1 << 30) / page) return bad("kvp: table_ld x page must be in [1, 2^30]");
    return QASR_OK;
}

static int pool_args(KvpPools &p, void *pools, int64_t n_pools, int64_t pool_stride, int64_t n_pages, int64_t n_heads,
                     int64_t page, int64_t row_bytes) {
    if (!pools) return bad("kvp: null pointer");
    if (n_heads <= 0 || n_heads > 1024) return bad("kvp: n_heads must be in [1, 1024]");
    if (row_bytes <= 0 || row_bytes % 16 != 0 || row_bytes > 4096) return bad("kvp: row_bytes must be a multiple of 16 in [16, 4096]");
    if (n_pools <= 0 || n_pools > 65535) return bad("kvp: n_pools must be in [1, 65535]");
    if ((uintptr_t)pools % 16 != 0 || pool_stride % 16 != 0) return bad("kvp: pools must be 16-byte aligned");
    if (n_pools > 1 && pool_stride < n_pages * n_heads * page * row_bytes) return bad("kvp: pool_stride is smaller than a pool");
    p.base = (char *)pools; p.n_pools = n_pools; p.pool_stride = pool_stride; p.n_pages = (int)n_pages;
    p.heads = (int)n_heads; p.shift = page_shift(page); p.units = (int)(row_bytes / 16);
    return QASR_OK;
}

extern "C" int qasr_hip_kvp_fork(qasr_hip *h, int32_t *table_out, int32_t *pos_out, int32_t *len_out, int32_t *status,
                                 const int32_t *table, const int32_t *len, const int32_t *parent,
                                 const int32_t *row_start, int64_t max_rows, int64_t n_out, int64_t n_seq,
                                 int64_t table_ld, void *pools, int64_t n_pools, int64_t pool_stride, int64_t n_pages,
                                 int64_t n_heads, int64_t page, int64_t row_bytes) {
    KvpForkArgs a{};
    if (!table_out || !pos_out || !len_out || !status || !table || !len) return bad("kvp_fork: null pointer");
    if (int rc = seq_args(n_seq, table_ld, n_pages, page)) return rc;
    if (n_out < 0 || n_out > QASR_KVP_MAX_SEQ) return bad("kvp_fork: at most 2048 sequences");
    if (!parent && n_out > n_seq) return bad("kvp_fork: without parent n_out is at most n_seq");
    if (max_rows < 0 || max_rows > (1 << 24)) return bad("kvp_fork: max_rows must be in [0, 2^24]");
    if (int rc = pool_args(a.pools, pools, n_pools, pool_stride, n_pages, n_heads, page, row_bytes)) return rc;
    struct { const void *p; int64_t n; } out[] = {{table_out, n_out * table_ld * 4}, {pos_out, n_out * 4}, {len_out, n_out * 4}, {status, 8}},
        in[] = {{table, n_seq * table_ld * 4}, {len, n_seq * 4}, {parent, n_out * 4}, {row_start, (n_out + 1) * 4}};
    for (auto &o : out)
        for (auto &i : in)
            if (overlap(o.p, o.n, i.p, i.n)) return bad("kvp_fork: an output overlaps an input");
    for (int x = 0; x < 4; x++)
        for (int y = x + 1; y < 4; y++)
            if (overlap(out[x].p, out[x].n, out[y].p, out[y].n)) return bad("kvp_fork: outputs overlap");
    CHECK_H(h);
    a.table_out = table_out; a.pos_out = pos_out; a.len_out = len_out; a.status = status;
    a.table = table; a.len = len; a.parent = parent; a.row_start = row_start; a.max_rows = max_rows;
    a.n_out = (int)n_out; a.n_seq = (int)n_seq; a.table_ld = (int)table_ld;
    a.work = reinterpret_cast<int *>(h->scratch);
    LAUNCHCHK(launch_kvp_fork(a, h->stream), "kvp_fork");
    return QASR_OK;
}

extern "C" int qasr_hip_kvp_compact(qasr_hip *h, int32_t *table_out, int32_t *status, const int32_t *table,
                                    const int32_t *len, int64_t n_seq, int64_t table_ld, void *pools, int64_t n_pools,
                                    int64_t pool_stride, int64_t n_pages, int64_t n_heads, int64_t page,
                                    int64_t row_bytes) {
    KvpCompactArgs a{};
    if (!table_out || !status || !table || !len) return bad("kvp_compact: null pointer");
    if (int rc = seq_args(n_seq, table_ld, n_pages, page)) return rc;
    if (int rc = pool_args(a.pools, pools, n_pools, pool_stride, n_pages, n_heads, page, row_bytes)) return rc;
    const int64_t nt = n_seq * table_ld * 4, nl = n_seq * 4;
    if ((table_out != table && overlap(table_out, nt, table, nt)) || overlap(table_out, nt, len, nl) ||
        overlap(status, 8, table, nt) || overlap(status, 8, len, nl) || overlap(status, 8, table_out, nt))
        return bad("kvp_compact: an output overlaps an input");
    CHECK_H(h);
    a.table_out = table_out; a.status = status; a.table = table; a.len = len;
    a.n_seq = (int)n_seq; a.table_ld = (int)table_ld;
    a.work = reinterpret_cast<int *>(h->scratch);
    LAUNCHCHK(launch_kvp_compact(a, h->stream), "kvp_compact");
    return QASR_OK;
}

// what the write and the attention share; fills the geometry
static int row_args(KvpSeqs &s, const void *kp, const void *vp, int64_t n_pages, const int32_t *table, int64_t table_ld,
                    const int32_t *row_start, const int32_t *pos, int64_t n_rows, int64_t n_seq, int64_t max_rows,
                    int64_t n_kv_heads, int64_t head_dim, int64_t page) {
    if (!kp || !vp || !table || !pos) return bad("kvp: null pointer");
    if (int rc = seq_args(n_seq, table_ld, n_pages, page)) return rc;
    if (head_dim != 64 && head_dim != 128) return bad("kvp: head_dim must be 64 or 128");
    if (n_kv_heads <= 0 || n_kv_heads > 1024) return bad("kvp: n_kv_heads must be in [1, 1024]");
    if (n_rows < 0 || n_rows > INT32_MAX || max_rows < 0 || max_rows > (1 << 24))
        return bad("kvp: n_rows or max_rows out of range");
    if (!row_start && n_seq * max_rows > n_rows) return bad("kvp: n_seq * max_rows rows need a larger n_rows");
    if ((((uintptr_t)kp) | (uintptr_t)vp) % 16 != 0) return bad("kvp: pages must be 16-byte aligned");
    s.table = table; s.row_start = row_start; s.pos = pos; s.n_rows = n_rows; s.max_rows = std::min(max_rows, n_rows);
    s.n_seq = (int)n_seq; s.table_ld = (int)table_ld; s.n_pages = (int)n_pages; s.Hkv = (int)n_kv_heads;
    s.hd = (int)head_dim; s.shift = page_shift(page);
    return QASR_OK;
}

extern "C" int qasr_hip_kvp_write(qasr_hip *h, uint16_t *k_pages, uint16_t *v_pages, int64_t n_pages, const void *k,
                                  const void *v, int64_t ld, const int32_t *table, int64_t table_ld,
                                  const int32_t *row_start, const int32_t *pos, int64_t n_rows, int64_t n_seq,
                                  int64_t max_rows, int64_t n_kv_heads, int64_t head_dim, int64_t page, int bf16) {
    KvpWriteArgs a{};
    if (int rc = row_args(a.s, k_pages, v_pages, n_pages, table, table_ld, row_start, pos, n_rows, n_seq, max_rows,
                          n_kv_heads, head_dim, page))
        return rc;
    if (!k || !v) return bad("kvp_write: null pointer");
    if (off_type(k, bf16) || off_type(v, bf16)) return bad("kvp_write: k or v is not aligned to its type");
    if (ld < n_kv_heads * head_dim || ld > INT32_MAX) return bad("kvp_write: row stride out of range");
    CHECK_H(h);
    if (n_seq == 0 || n_rows == 0 || max_rows == 0) return QASR_OK;
    a.kp = k_pages; a.vp = v_pages; a.k = k; a.v = v; a.ld = ld;
    LAUNCHCHK(launch_kvp_write(a, bf16 != 0, h->stream), "kvp_write");
    return QASR_OK;
}

extern "C" int qasr_hip_attention_kvp(qasr_hip *h, void *out, const void *q, int64_t ldq, const uint16_t *k_pages,
                                      const uint16_t *v_pages, int64_t n_pages, const int32_t *table, int64_t table_ld,
                                      const int32_t *row_start, const int32_t *pos, int64_t n_rows, int64_t n_seq,
                                      int64_t max_rows, int64_t max_len, int64_t group, const int32_t *shared,
                                      int64_t max_own, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                                      int64_t page, float scale, int bf16) {
    AttnKvpArgs a{};
    if (int rc = row_args(a.s, k_pages, v_pages, n_pages, table, table_ld, row_start, pos, n_rows, n_seq, max_rows,
                          n_kv_heads, head_dim, page))
        return rc;
    if (!out || !q) return bad("attention_kvp: null pointer");
    if (off_type(out, bf16) || off_type(q, bf16)) return bad("attention_kvp: q or out is not aligned to its type");
    if (n_heads <= 0 || n_heads % n_kv_heads != 0 || n_heads > 65536)
        return bad("attention_kvp: n_heads must be a positive multiple of n_kv_heads");
    if (ldq < n_heads * head_dim || ldq > INT32_MAX) return bad("attention_kvp: row stride out of range");
    const int64_t es = bf16 ? 2 : 4, row = n_heads * head_dim;
    if ((out != q || ldq != row) && overlap(out, n_rows * row * es, q, n_rows > 0 ? ((n_rows - 1) * ldq + row) * es : 0))
        return bad("attention_kvp: out overlaps q and is not q");
    if (group < 1) return bad("attention_kvp: group must be positive");
    if (max_len < 0 || max_own < 0) return bad("attention_kvp: max_len and max_own must not be negative");
    if (!std::isfinite(scale * 1.4426950408889634f)) return bad("attention_kvp: scale x log2 e must be finite");
    if (a.s.max_rows * (n_heads / n_kv_heads) > (1 << 30))
        return bad("attention_kvp: rows x heads of a group out of range");
    CHECK_H(h);
    if (n_seq == 0 || n_rows == 0 || max_rows == 0) return QASR_OK;
    const int64_t cap = table_ld * page;
    a.kp = k_pages; a.vp = v_pages; a.q = q; a.out = out; a.ldq = ldq; a.scale = scale;
    a.group = (int)std::min<int64_t>(group, n_seq); a.shared = a.group > 1 ? shared : nullptr;
    a.Hq = (int)n_heads; a.G = (int)(n_heads / n_kv_heads);
    a.max_len = max_len > 0 ? std::min(max_len, cap) : cap;
    a.max_own = max_own > 0 ? std::min(max_own, a.max_len) : a.max_len;
    a.common = max_own > 0 ? a.max_len - a.max_own : -1;
    a.part = reinterpret_cast<float *>(h->scratch);
    LAUNCHCHK(launch_attention_kvp(a, bf16 != 0, h->stream), "attention_kvp");
    return QASR_OK;
}

extern "C" int qasr_hip_token_logprobs(qasr_hip *h, float *logp, float *entropy, int32_t *top_ids, float *top_logp,
                                       int64_t k, const void *logits, int64_t ld, const int32_t *targets, int64_t rows,
                                       int64_t cols, int bf16) {
    if (!logits) return bad("token_logprobs: null pointer");
    if (logp && !targets) return bad("token_logprobs: logp needs targets");
    if (cols <= 0 || cols > QASR_LOGP_MAX_COLS || ld < cols || ld > INT32_MAX) return bad("token_logprobs: cols must be in [1, 2^20], ld at least cols");
    if (rows < 0 || rows > (1 << 24)) return bad("token_logprobs: rows must be in [0, 2^24]");
    if (k < 0 || k > QASR_LOGP_MAX_K || k > cols) return bad("token_logprobs: k must be in [0, 32], at most cols");
    if (off_type(logits, bf16)) return bad("token_logprobs: logits are not aligned to their type");
    CHECK_H(h);
    if (k == 0) { top_ids = nullptr; top_logp = nullptr; }
    if (!top_ids && !top_logp) k = 0;
    if (rows == 0 || (!logp && !entropy && k == 0)) return QASR_OK;
    LogpArgs a{};
    a.logp = logp; a.entropy = entropy; a.top_ids = top_ids; a.top_logp = top_logp; a.targets = targets;
    a.x = logits; a.ld = ld; a.rows = rows; a.cols = (int)cols; a.k = (int)k;
    a.part = reinterpret_cast<char *>(h->scratch);
    LAUNCHCHK(launch_token_logprobs(a, bf16 != 0, h->stream), "token_logprobs");
    return QASR_OK;
}
