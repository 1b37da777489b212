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
// The k largest: 64 lanes' maxima (each over the chunk's values in that lane's places).  At
// least k values are not below the k-th largest of these maxima, T, and what is not below
// T stands in the k lanes that reach it, a few more than k values as a rule: they are ranked
// by counting.  Where T is a value that many share (masked vocabularies, rows of one value)
// those above it are taken, and the first of those that have it.
#include "kernels.h"
#include "gemm_common.h"

namespace qasr {

typedef unsigned long long u64;
#define LOGP_E 32                       // values a thread
// a row's chunks: those of 256 threads, and one more for what its first begins late by
#define LOGP_CHUNKS (QASR_LOGP_MAX_COLS / (256 * LOGP_E) + 1)
#define LOGP_CAND 1024                  // values a chunk ranks by counting
#define LOGP_LANES 64                   // lanes whose values are looked through together
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

// W waves with E values a thread; five waves a SIMD (with four, f32 375 x 151936 52 us for 47), eight of short rows
template <bool BF16, int W, int E>
__global__ __launch_bounds__(64 * W, E == 8 ? 8 : W == 16 ? 4 : 5) void k_logp(LogpArgs a, int64_t row0) {
    constexpr int V = BF16 ? 8 : 4, T = 64 * W, NV = E / V, CH = T * E;
    __shared__ float red[3][W], lane_max[W][64], limit;
    constexpr bool SHARE = W > 2;                        // (with fewer waves the LDS that it takes holds blocks up)
    __shared__ int red_n[W], n_cand, n_lanes, lane_of[SHARE ? LOGP_LANES : 1], ranks[SHARE ? 64 : 1];
    __shared__ __attribute__((aligned(16))) float held[SHARE ? LOGP_LANES : 1][E + 4];
    constexpr int CAND = CH < LOGP_CAND ? CH : LOGP_CAND;
    __shared__ u64 cand[CAND], best_l[W];
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const int64_t row = row0 + blockIdx.y;
    // chunks begin at 16-byte places: `off` values before the row's first are none of its
    const int64_t at = row * a.ld;
    constexpr int ES = BF16 ? 2 : 4;
    const char *row_p = reinterpret_cast<const char *>(a.x) + at * ES;
    const int off = (int)(((uintptr_t)row_p & 15) / ES);
    const int i0 = (int)blockIdx.x * CH - off;
    float x[E];
    const float none = -__builtin_inff();
    if (i0 >= 0 && i0 + CH <= a.cols) {
#pragma unroll
        for (int n = 0; n < NV; n++) {
            const uint4 u = *reinterpret_cast<const uint4 *>(row_p + (int64_t)(i0 + (n * T + t) * V) * ES);
            const uint32_t d[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < V; e++)
                x[n * V + e] = BF16 ? __uint_as_float((e & 1) ? d[e / 2] & 0xffff0000u : d[e / 2] << 16) : __uint_as_float(d[e]);
        }
    } else {
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
    }
    float tm = none;
#pragma unroll
    for (int e = 0; e < E; e++) tm = fmaxf(tm, x[e]);
    float M = wave_max_f32(tm);
    if (t == 0) n_cand = n_lanes = 0;
    if (SHARE && t < 64) ranks[t] = 0;
    if (W > 1) {
        if (lane == 0) red[0][w] = M;
        lane_max[w][lane] = tm;
        __syncthreads();
#pragma unroll 4
        for (int i = 0; i < W; i++) M = fmaxf(M, red[0][i]);
    }
    // the k-th largest of the lanes' maxima, by the first wave, while the others go on
    if (a.k > 0 && w == 0) {
        float g = tm;
#pragma unroll 4
        for (int i = 1; i < W; i++) g = fmaxf(g, lane_max[i][lane]);
        float lim = M;
        // few: one after another, equal ones at once (375 x 151936, k 5: f32 47.2 -> 44.7 us, bf16 43.2 -> 39.2; 2000 x
        // 28000, k 8: 55.3 -> 53.5); more: by counting (8 x 151936, k 16: 12.9, one after another 13.8)
        if (a.k <= 8) {
            for (int n = __popcll(__ballot(g == lim)); n < a.k; n += __popcll(__ballot(g == lim))) {
                g = g == lim ? none : g;
                lim = wave_max_f32(g);
                if (lim == none) break;
            }
        } else {
            int above = 0;
#pragma unroll 16
            for (int i = 0; i < 64; i++) above += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(g), i)) > g;
            // the least of the maxima that fewer than k pass
            lim = -wave_max_f32(above < a.k ? -g : none);
        }
        if (lane == 0) limit = lim;
    }
    // the sums; the terms of the maximum, exactly 1 each, are counted, all but one
    float s = 0.0f, h = 0.0f;
    int ones = 0;
    if (M == none) {
        // nothing above -infinity: NaN if there is one
#pragma unroll
        for (int e = 0; e < E; e++) s += x[e] != x[e] ? x[e] : 0.0f;
    } else {
        const bool mine = tm == M;
        if (__any(mine)) {
#pragma unroll
            for (int e = 0; e < E; e++) {
                const bool one = x[e] == M;
                const float d = (x[e] - M) * LOGP_LOG2E, p = __builtin_amdgcn_exp2f(d);
                h = fmaf(p, fmaxf(d, -200.0f), h);
                ones += one;
                s += one ? 0.0f : p;
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; e++) {
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
    if (lane == 0) {
        red[1][w] = s;
        red[2][w] = h;
        red_n[w] = ones;
    }
    __syncthreads();
    s = h = 0.0f;
    ones = 0;
#pragma unroll 4
    for (int i = 0; i < W; i++) {
        s += red[1][i];
        h += red[2][i];
        ones += red_n[i];
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
    const float lim = limit;
    const bool hit = tm >= lim;
    const u64 hits = __ballot(hit);
    if (SHARE && hits) {
        // the values of the lanes that reach T, looked through by all threads: each lane its own is 50 instructions for four
        // values of which one is wanted (375 x 151936, k 32, bf16 71.7 -> 63.4 us)
        int slot = 0;
        if (lane == 0) slot = atomicAdd(&n_lanes, __popcll(hits));
        slot = __builtin_amdgcn_readfirstlane(slot) + __builtin_amdgcn_mbcnt_hi((unsigned)(hits >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)hits, 0));
        if (hit && slot < LOGP_LANES) {
            lane_of[slot] = t;
#pragma unroll
            for (int e = 0; e < E; e += 4) *reinterpret_cast<f32x4 *>(&held[slot][e]) = f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
        }
    }
    if (SHARE) __syncthreads();
    const int lanes = n_lanes;
    if (SHARE && lanes <= LOGP_LANES) {
        for (int u = t; u < lanes * E; u += T) {
            const int e = u % E, i = i0 + (e / V * T + lane_of[u / E]) * V + e % V;
            const float y = held[u / E][e];
            if (!(fmaxf(y, none) < lim) && i >= 0 && i < a.cols) {
                const int c = atomicAdd(&n_cand, 1);
                if (c < CAND) cand[c] = logp_key(y, i);
            }
        }
    } else if (hits) {
#pragma unroll
        for (int n = 0; n < NV; n++)
#pragma unroll
            for (int q = 0; q < V; q += 4) {
                const float *y = x + n * V + q;
                if (!__any(!(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) < lim))) continue;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = i0 + (n * T + t) * V + q + e;
                    if (!(fmaxf(y[e], none) < lim) && i >= 0 && i < a.cols) {
                        const int c = atomicAdd(&n_cand, 1);
                        if (c < CAND) cand[c] = logp_key(y[e], i);
                    }
                }
            }
    }
    __syncthreads();
    int n = n_cand;
    u64 *top = reinterpret_cast<u64 *>(base + 16);
    if (n > CAND) {
        // a value that many share: those above it, then as many of it as are wanted, in order
        __syncthreads();
        if (t == 0) n_cand = 0;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int i = i0 + (e / V * T + t) * V + e % V;
            if (x[e] > lim && i >= 0 && i < a.cols) {
                const int c = atomicAdd(&n_cand, 1);
                if (c < CAND) cand[c] = logp_key(x[e], i);
            }
        }
        __syncthreads();
        n = n_cand;
        if (n < a.k) {
#pragma unroll
            for (int v = 0; v < NV; v++) {
                if (n >= a.k) break;
                const int i = i0 + (v * T + t) * V;
                unsigned ties = 0;
#pragma unroll
                for (int e = 0; e < V; e++) ties |= (fmaxf(x[v * V + e], none) == lim && i + e >= 0 && i + e < a.cols ? 1u : 0u) << e;
                const int mine = __popc(ties);
                int before = mine;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int y = __shfl_up(before, o, 64);
                    before += lane >= o ? y : 0;
                }
                __syncthreads();
                if (lane == 63) red_n[w] = before;
                __syncthreads();
                before += n - mine;
#pragma unroll 4
                for (int u = 0; u < W; u++) {
                    before += u < w ? red_n[u] : 0;
                    n += red_n[u];
                }
                for (; ties && before < a.k; ties &= ties - 1, before++) cand[before] = logp_key(lim, i + __builtin_ctz(ties));
            }
            n = min(n, a.k);
            __syncthreads();
        }
    }
    if (SHARE && n > 8 && n <= 64) {
        // every wave compares all keys with some of them
        const u64 y = lane < n ? cand[lane] : ~0ull;
        int rank = 0;
        for (int j = w; j < n; j += W) rank += cand[j] > y;
        if (lane < n) atomicAdd(&ranks[lane], rank);
        __syncthreads();
        if (t < n) {
            const int r = ranks[t];
            if (r < a.k) {
                if (only) logp_top(a, row, r, y, part);
                else top[r] = y;
            }
        }
        if (!only)
            for (int i = n + t; i < a.k; i += T) top[i] = 0;
        return;
    }
    if (n <= CAND) {
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
        return;
    }
    // still more than there is room for, so more than k: the largest key below the last one, k times
    u64 last = ~0ull;
    for (int r = 0; r < a.k; r++) {
        u64 best = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int i = i0 + (e / V * T + t) * V + e % V;
            const u64 y = logp_key(x[e], i);
            if (i >= 0 && i < a.cols && y < last && y > best) best = y;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) best = max(best, (u64)__shfl_xor((unsigned long long)best, o, 64));
        if (lane == 0) best_l[w] = best;
        __syncthreads();
        last = 0;
#pragma unroll 4
        for (int i = 0; i < W; i++) last = max(last, best_l[i]);
        __syncthreads();
        if (t == 0) {
            if (only) logp_top(a, row, r, last, part);
            else top[r] = last;
        }
    }
}

// A row's chunks joined: one block a row, a lane of every wave a chunk or two.  A key can
// be among the k largest only if its place in its own list and the lists whose first key
// is larger are fewer than k.
template <bool BF16>
__global__ __launch_bounds__(256) void k_logp_join(LogpArgs a, int64_t row0) {
    constexpr int U = (LOGP_CHUNKS + 63) / 64, MAX_K = QASR_LOGP_MAX_K;
    extern __shared__ u64 keys[];                                // [chunks][k]
    __shared__ u64 cand[MAX_K * (MAX_K + 1) / 2];
    __shared__ int n_cand, list[MAX_K];
    const int t = threadIdx.x, lane = t & 63, n = a.chunks;
    const int64_t row = row0 + blockIdx.x, step = logp_part(a.k);
    const char *base = a.part + (int64_t)blockIdx.x * n * step;
    const int target = a.logp ? a.targets[row] : -1;
    float4 p[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = lane + 64 * u;
        p[u] = i < n ? *reinterpret_cast<const float4 *>(base + i * step) : make_float4(-__builtin_inff(), 0.0f, 0.0f, 0.0f);
    }
    const int at_once = a.k > 0 ? 256 / a.k : 1;                 // lists
    if (a.k > 0 && t < at_once * a.k)
        for (int c = t / a.k; c < n; c += at_once) keys[c * a.k + t % a.k] = *reinterpret_cast<const u64 *>(base + c * step + 16 + 8 * (t % a.k));
    if (t < MAX_K) list[t] = -1;
    if (t == 0) n_cand = 0;
    const bool has = (unsigned)target < (unsigned)a.cols;
    const float x_target = has ? logp_at<BF16>(a, row, target) : 0.0f;
    __syncthreads();
    LogpPart r{-__builtin_inff(), 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < U; u++) r.m = fmaxf(r.m, p[u].x);
    r.m = wave_max_f32(r.m);
    // the chunk whose largest term is the row's: the first of them
    int mine = 0x7fffffff;
#pragma unroll
    for (int u = U - 1; u >= 0; u--) mine = p[u].x == r.m && r.m != -__builtin_inff() ? lane + 64 * u : mine;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mine = min(mine, __shfl_xor(mine, o, 64));
    const float ref = r.m == -__builtin_inff() ? 0.0f : r.m;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const float d = p[u].x - ref, w = expf(d);       // a chunk of -infinity alone: 0
        const bool empty = p[u].x == -__builtin_inff();
        r.s += lane + 64 * u == mine ? p[u].y : w * p[u].y + (empty ? 0.0f : w);
        r.h += w * (p[u].z + (empty ? 0.0f : (1.0f + p[u].y) * fmaxf(d, -200.0f)));
    }
    r.s = wave_sum_f32(r.s);
    r.h = wave_sum_f32(r.h);
    if (t == 0) logp_row(a, row, r, x_target, has);
    if (a.k == 0) return;
    // the lists by their first keys, then of the r-th list the k - r first, if they are not below a key that k of them reach:
    // the k-th list's first; of fewer lists the least of those keys of which each has as many above it as make k
    const int deep = n < a.k ? (a.k - 1) / n : 0;
    for (int i = t; i < n; i += 256) {
        const u64 y = keys[i * a.k];
        int rank = 0;
        for (int j = 0; j < n; j++) rank += keys[j * a.k] > y;
        if (y != 0 && rank < a.k) list[rank] = i;
    }
    u64 least = ~0ull;
    if (deep > 0)
        for (int i = 0; i < n; i++) least = min(least, keys[i * a.k + deep]);
    __syncthreads();
    if (deep == 0) least = list[a.k - 1] >= 0 ? keys[list[a.k - 1] * a.k] : 0;
    least = max(least, 1ull);                                    // 0: no key
    for (int i = t; i < a.k * a.k; i += 256) {
        const int r = i / a.k, place = i % a.k;
        if (r + place >= a.k || list[r] < 0) continue;
        const u64 y = keys[list[r] * a.k + place];
        if (y >= least) cand[atomicAdd(&n_cand, 1)] = y;
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

template <bool BF16, int W, int E>
static hipError_t go_logp(LogpArgs a, hipStream_t st) {
    constexpr int CH = 64 * W * E, V = BF16 ? 8 : 4;
    a.chunks = (a.cols + V - 1 + CH - 1) / CH;           // up to V - 1 values before the row's first
    if (a.chunks > 1 && a.cols <= CH && (uintptr_t)a.x % 16 == 0 && a.ld % V == 0) a.chunks = 1;
    const int64_t per_row = a.chunks * logp_part(a.k);
    const int64_t rows = a.chunks == 1 ? 65535 : std::min<int64_t>(65535, QASR_LOGP_PART_BYTES / per_row);
    for (int64_t r = 0; r < a.rows; r += rows) {
        const unsigned n = (unsigned)std::min(rows, a.rows - r);
        hipLaunchKernelGGL((k_logp<BF16, W, E>), dim3((unsigned)a.chunks, n), dim3(64 * W), 0, st, a, r);
        if (a.chunks > 1) hipLaunchKernelGGL((k_logp_join<BF16>), dim3(n), dim3(256), (size_t)a.chunks * a.k * 8, st, a, r);
    }
    return hipGetLastError();
}

// The fewest waves that hold a row, as those of none cost what others do (4000 x 300 12.5 -> 9.7 us): one launch, while
// blocks of 8 or 16 waves are few enough not to wait for one another (us, chunks / one block: 8 waves, 8 x 12000 bf16 10.7 /
// 6.9, 2000 x 16000 f32 32.9 / 32.1, 4000 x 16000 55.6 / 56.5; 16 waves, 256 x 30000 f32 15.2 / 10.9, 512 x 20000 17.7 /
// 17.6, 600 x 20000 19.3 / 23.0).  Longer rows and more of them in chunks of four waves (of one, for few rows: 8 x 151936
// 16.9 us for 14.1; 64 values a thread: bf16 375 x 151936 47 for 43, and 16 waves of them spill).
template <bool BF16>
static hipError_t pick_logp(const LogpArgs &a, hipStream_t st) {
    const int n = a.cols + (BF16 ? 7 : 3);               // with what a row may begin behind a 16-byte place
    if (n <= 64 * 8) return go_logp<BF16, 1, 8>(a, st);
    if (n <= 64 * LOGP_E) return go_logp<BF16, 1, LOGP_E>(a, st);
    if (n <= 128 * LOGP_E) return go_logp<BF16, 2, LOGP_E>(a, st);
    if (n <= 192 * LOGP_E) return go_logp<BF16, 3, LOGP_E>(a, st);
    if (n > 256 * LOGP_E && n <= 512 * LOGP_E && a.rows <= 2048) return go_logp<BF16, 8, LOGP_E>(a, st);
    if (n > 512 * LOGP_E && n <= 1024 * LOGP_E && a.rows <= 512) return go_logp<BF16, 16, LOGP_E>(a, st);
    return go_logp<BF16, 4, LOGP_E>(a, st);
}

hipError_t launch_token_logprobs(const LogpArgs &a, bool bf16, hipStream_t st) {
    if (a.k > QASR_LOGP_MAX_K || a.cols > QASR_LOGP_MAX_COLS) return hipErrorInvalidValue;
    return bf16 ? pick_logp<true>(a, st) : pick_logp<false>(a, st);
}

}  // namespace qasr
