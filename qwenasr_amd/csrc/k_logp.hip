// Log probabilities of rows of logits: of given tokens, their entropy, the likeliest.
//
// A block takes a chunk of a row into registers and reads it once: its maximum M, the sum
// of e^(x - M) over the others, the sum of e^(x - M) (x - M), and its k largest.  A second
// launch joins a row's chunks.  Bound by the read; per value one subtraction, product,
// exponential, and three additions.
//
// The largest term of a row, 1, is not part of the sum (s): log p = x - M - log1p(s), so a
// probability next to 1 keeps the bits of its logarithm, where log(1 + s) would lose them.
//
// The k largest: 64 lanes' maxima (each over the chunk's values in that lane's places)
// as keys (value, then lowest index).  At least k values are not below the k-th
// largest of these keys T, and no value outside the k lanes whose key reaches it
// can be above T: what is not below T is at most k lanes' values, whatever the row holds,
// a few more than k as a rule, and is ranked by counting.
#include "kernels.h"
#include "gemm_common.h"

namespace qasr {

typedef unsigned long long u64;
#define LOGP_E 32                       // values a thread
// a row's chunks: those of 256 threads, and one more for what its first begins late by
#define LOGP_CHUNKS (QASR_LOGP_MAX_COLS / (256 * LOGP_E) + 1)
#define LOGP_LOG2E 1.4426950408889634f
#define LOGP_LN2 0.6931471805599453f

// bytes of a chunk's part: {maximum, sums}, then its k largest keys
__device__ __host__ __forceinline__ int64_t logp_part(int k) { return 16 + 16 * (int64_t)((k + 1) / 2); }
struct LogpPart { float m, s, h; };     // maximum, the others' sum, sum of e^(x - m) (x - m)

// larger value first, then lower index; NaN with -infinity, -0 with 0
__device__ __forceinline__ u64 logp_key(float x, int i) {
    const uint32_t u = __float_as_uint(fmaxf(x, -__builtin_inff()) + 0.0f);
    return (u64)((u >> 31) ? ~u : u | 0x80000000u) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ int logp_id(u64 key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float logp_value(u64 key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float((u >> 31) ? u & 0x7fffffffu : ~u);
}

__device__ __forceinline__ u64 shfl64(u64 v, int lane) {
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

// the row's results, by one block
__device__ __forceinline__ void logp_row(const LogpArgs &a, int64_t row, LogpPart p, float x_target, bool has_target) {
    // a row without any finite or infinite value above -infinity has no sum; NaN stays
    const float tail = p.m == -__builtin_inff() && !(p.s != p.s) ? 0.0f : log1pf(p.s);
    if (a.logp) a.logp[row] = !has_target ? __builtin_nanf("") : p.m == -__builtin_inff() ? (p.s != p.s ? p.s : p.m) : x_target - p.m - tail;
    if (a.entropy) a.entropy[row] = p.m == -__builtin_inff() && !(p.s != p.s) ? 0.0f : tail - p.h / (1.0f + p.s);
}
__device__ __forceinline__ void logp_top(const LogpArgs &a, int64_t row, int rank, u64 key, LogpPart p) {
    if (a.top_ids) a.top_ids[row * a.k + rank] = logp_id(key);
    if (a.top_logp) a.top_logp[row * a.k + rank] = p.m == -__builtin_inff() ? (p.s != p.s ? p.s : p.m) : logp_value(key) - p.m - log1pf(p.s);
}
template <bool BF16>
__device__ __forceinline__ float logp_at(const LogpArgs &a, int64_t row, int i) {
    const int64_t at = row * a.ld + i;
    return BF16 ? bf16_to_f32(reinterpret_cast<const uint16_t *>(a.x)[at]) : reinterpret_cast<const float *>(a.x)[at];
}

template <bool BF16, int W>
__global__ __launch_bounds__(64 * W) void k_logp(LogpArgs a, int64_t row0) {
    constexpr int V = BF16 ? 8 : 4, T = 64 * W, NV = LOGP_E / V, CH = T * LOGP_E;
    __shared__ float red[3][W];
    __shared__ u64 lane_key[W][64], limit;
    __shared__ u64 cand[QASR_LOGP_MAX_K * W * LOGP_E];
    __shared__ int n_cand;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const int64_t row = row0 + blockIdx.y;
    // chunks begin at 16-byte places: `off` values before the row's first are none of its
    const int64_t at = row * a.ld;
    constexpr int ES = BF16 ? 2 : 4;
    const char *row_p = reinterpret_cast<const char *>(a.x) + at * ES;
    const int off = (int)(((uintptr_t)row_p & 15) / ES);
    const int i0 = (int)blockIdx.x * CH - off;
    float x[LOGP_E];
    const float none = -__builtin_inff();
#pragma unroll
    for (int n = 0; n < NV; n++) {
        const int i = i0 + (n * T + t) * V;
        if (i >= 0 && i + V <= a.cols) {
            const uint4 u = *reinterpret_cast<const uint4 *>(row_p + (int64_t)i * ES);
            const uint32_t d[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < V; e++)
                x[n * V + e] = BF16 ? __uint_as_float((e & 1) ? d[e / 2] & 0xffff0000u : d[e / 2] << 16) : __uint_as_float(d[e]);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) x[n * V + e] = i + e >= 0 && i + e < a.cols ? logp_at<BF16>(a, row, i + e) : none;
        }
    }
    float tm = none;
#pragma unroll
    for (int e = 0; e < LOGP_E; e++) tm = fmaxf(tm, x[e]);
    float M = wave_max_f32(tm);
    if (W > 1) {
        if (lane == 0) red[0][w] = M;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < W; i++) M = fmaxf(M, red[0][i]);
    }
    // the sums; the terms of the maximum, exactly 1 each, are counted, all but one
    float s = 0.0f, h = 0.0f;
    int ones = 0;
    if (M == none) {
        // nothing above -infinity: NaN if there is one
#pragma unroll
        for (int e = 0; e < LOGP_E; e++) s += x[e] != x[e] ? x[e] : 0.0f;
    } else {
        const bool mine = tm == M;
        if (__any(mine)) {
#pragma unroll
            for (int e = 0; e < LOGP_E; e++) {
                const bool one = x[e] == M;
                const float d = (x[e] - M) * LOGP_LOG2E, p = __builtin_amdgcn_exp2f(d);
                h = fmaf(p, fmaxf(d, -200.0f), h);
                ones += one;
                s += one ? 0.0f : p;
            }
        } else {
#pragma unroll
            for (int e = 0; e < LOGP_E; e++) {
                const float d = (x[e] - M) * LOGP_LOG2E, p = __builtin_amdgcn_exp2f(d);
                h = fmaf(p, fmaxf(d, -200.0f), h);
                s += p;
            }
        }
        if (M == __builtin_inff()) s = __builtin_nanf("");
    }
    s = wave_sum_f32(s);
    h = wave_sum_f32(h);
    ones = wave_sum_i32(ones);
    if (W > 1) {
        if (lane == 0) {
            red[1][w] = s;
            red[2][w] = h;
            lane_key[w][0] = (u64)ones;
        }
        __syncthreads();
        s = h = 0.0f;
        ones = 0;
#pragma unroll
        for (int i = 0; i < W; i++) {
            s += red[1][i];
            h += red[2][i];
            ones += (int)lane_key[i][0];
        }
        __syncthreads();
    }
    const LogpPart part{M, s + (float)max(ones - 1, 0), h * LOGP_LN2};
    const bool only = a.chunks == 1;
    char *const base = a.part + ((int64_t)blockIdx.y * a.chunks + blockIdx.x) * logp_part(a.k);
    if (t == 0) {
        if (only) {
            const int g = a.logp ? a.targets[row] : -1;
            const bool has = (unsigned)g < (unsigned)a.cols;
            logp_row(a, row, part, has ? logp_at<BF16>(a, row, g) : 0.0f, has);
        } else {
            *reinterpret_cast<float4 *>(base) = make_float4(part.m, part.s, part.h, 0.0f);
        }
    }
    if (a.k == 0) return;

    // ---- the k largest
    u64 key = 0;                                  // 0: below the key of any value
    {
        int best = -1;
#pragma unroll
        for (int n = NV - 1; n >= 0; n--)
#pragma unroll
            for (int e = V - 1; e >= 0; e--) {
                const int i = i0 + (n * T + t) * V + e;
                if (fmaxf(x[n * V + e], none) == tm && i >= 0 && i < a.cols) best = i;
            }
        if (best >= 0) key = logp_key(tm, best);
    }
    lane_key[w][lane] = key;
    if (t == 0) n_cand = 0;
    __syncthreads();
    if (w == 0) {
        u64 g = 0;
#pragma unroll
        for (int i = 0; i < W; i++) g = max(g, lane_key[i][lane]);
        int above = 0;
        for (int i = 0; i < 64; i++) {
            const u64 o = shfl64(g, i);
            above += o > g || (o == g && i < lane);
        }
        if (above == a.k - 1) limit = g;
    }
    __syncthreads();
    const u64 lim = limit;
    if (key >= lim && key != 0) {
#pragma unroll
        for (int n = 0; n < NV; n++)
#pragma unroll
            for (int e = 0; e < V; e++) {
                const int i = i0 + (n * T + t) * V + e;
                const u64 y = logp_key(x[n * V + e], i);
                if (y >= lim && i >= 0 && i < a.cols) cand[atomicAdd(&n_cand, 1)] = y;
            }
    }
    __syncthreads();
    const int n = n_cand;
    u64 *top = reinterpret_cast<u64 *>(base + 16);
    for (int i = t; i < n; i += T) {
        const u64 y = cand[i];
        int rank = 0;
        for (int j = 0; j < n; j++) rank += cand[j] > y;
        if (rank < a.k) {
            if (only) logp_top(a, row, rank, y, part);
            else top[rank] = y;
        }
    }
    if (!only)
        for (int i = n + t; i < a.k; i += T) top[i] = 0;
}

// A row's chunks joined: one block a row.  A key can be among the k largest only if
// its place in its own list and the lists whose first key is larger are fewer than k.
template <bool BF16>
__global__ __launch_bounds__(256) void k_logp_join(LogpArgs a, int64_t row0) {
    __shared__ u64 cand[QASR_LOGP_MAX_K * QASR_LOGP_MAX_K], head[LOGP_CHUNKS];
    __shared__ float m_l[LOGP_CHUNKS], s_l[LOGP_CHUNKS], h_l[LOGP_CHUNKS];
    __shared__ int n_cand;
    const int t = threadIdx.x, n = a.chunks;
    const int64_t row = row0 + blockIdx.x, step = logp_part(a.k);
    const char *base = a.part + (int64_t)blockIdx.x * n * step;
    for (int i = t; i < n; i += 256) {
        const float4 p = *reinterpret_cast<const float4 *>(base + i * step);
        m_l[i] = p.x;
        s_l[i] = p.y;
        h_l[i] = p.z;
        head[i] = a.k > 0 ? *reinterpret_cast<const u64 *>(base + i * step + 16) : 0;
    }
    if (t == 0) n_cand = 0;
    __syncthreads();
    // in chunk order, by every thread alike
    LogpPart r{-__builtin_inff(), 0.0f, 0.0f};
    for (int i = 0; i < n; i++) r.m = fmaxf(r.m, m_l[i]);
    bool first = true;
    const float ref = r.m == -__builtin_inff() ? 0.0f : r.m;
    for (int i = 0; i < n; i++) {
        const float d = m_l[i] - ref, w = expf(d);       // a chunk of -infinity alone: 0
        const bool one = first && m_l[i] == r.m && r.m != -__builtin_inff();
        first = first && !one;
        r.s += one ? s_l[i] : w * s_l[i] + (m_l[i] == -__builtin_inff() ? 0.0f : w);
        r.h += w * (h_l[i] + (m_l[i] == -__builtin_inff() ? 0.0f : (1.0f + s_l[i]) * fmaxf(d, -200.0f)));
    }
    if (t == 0) {
        const int g = a.logp ? a.targets[row] : -1;
        const bool has = (unsigned)g < (unsigned)a.cols;
        logp_row(a, row, r, has ? logp_at<BF16>(a, row, g) : 0.0f, has);
    }
    if (a.k == 0) return;
    for (int i = t; i < n * a.k; i += 256) {
        const int c = i / a.k, place = i % a.k;
        const u64 y = *reinterpret_cast<const u64 *>(base + c * step + 16 + 8 * place);
        if (y == 0) continue;
        int above = place;
        for (int j = 0; j < n; j++) above += j != c && head[j] > y;
        if (above < a.k) cand[atomicAdd(&n_cand, 1)] = y;
    }
    __syncthreads();
    const int found = n_cand;
    for (int i = t; i < found; i += 256) {
        const u64 y = cand[i];
        int rank = 0;
        for (int j = 0; j < found; j++) rank += cand[j] > y;
        if (rank < a.k) logp_top(a, row, rank, y, r);
    }
}

template <bool BF16, int W>
static hipError_t go_logp(LogpArgs a, hipStream_t st) {
    constexpr int CH = 64 * W * LOGP_E, V = BF16 ? 8 : 4;
    a.chunks = (a.cols + V - 1 + CH - 1) / CH;           // up to V - 1 values before the row's first
    if (a.chunks > 1 && a.cols <= CH && (uintptr_t)a.x % 16 == 0 && a.ld % V == 0) a.chunks = 1;
    const int64_t per_row = a.chunks * logp_part(a.k);
    const int64_t rows = a.chunks == 1 ? 65535 : std::min<int64_t>(65535, QASR_LOGP_PART_BYTES / per_row);
    for (int64_t r = 0; r < a.rows; r += rows) {
        const unsigned n = (unsigned)std::min(rows, a.rows - r);
        hipLaunchKernelGGL((k_logp<BF16, W>), dim3((unsigned)a.chunks, n), dim3(64 * W), 0, st, a, r);
        if (a.chunks > 1) hipLaunchKernelGGL((k_logp_join<BF16>), dim3(n), dim3(256), 0, st, a, r);
    }
    return hipGetLastError();
}

hipError_t launch_token_logprobs(const LogpArgs &a, bool bf16, hipStream_t st) {
    if (a.k > QASR_LOGP_MAX_K || a.cols > QASR_LOGP_MAX_COLS) return hipErrorInvalidValue;
    // a wave a row where that holds it
    if (a.cols + 7 <= 64 * LOGP_E) return bf16 ? go_logp<true, 1>(a, st) : go_logp<false, 1>(a, st);
    return bf16 ? go_logp<true, 4>(a, st) : go_logp<false, 4>(a, st);
}

}  // namespace qasr
