// Attention over a KV cache in pages, a prefix that a group of sequences shares read
// once for all of them.
//
// A wave takes 16 (or 32) query rows x heads of a group against 32 positions at a
// time, everything in registers: S^T = K Q^T leaves a lane (column c = its query, lane
// group g) positions 4 g + r of each half, r = 0..3.  O^T = V^T P^T may number its 32
// products' k as it likes, so k = 8 g + e is taken to be position 4 g + (e & 3) of
// half e / 4: the probabilities of a lane are its operand as they are, and no value
// crosses lanes between the two products.  V's operand is one dim of eight
// positions a lane, V's rows are eight dims of one position: each lane loads 16 bytes
// of its eight positions (16 lanes a whole row) and turns the 8 x 8 values by 32
// byte permutes, dim 8 m + t in row m of product t.  The output of a lane is then
// 8 consecutive dims a register, and running maximum and sum are one value a lane.
//
// All products take operands that lose nothing: K, V and bf16 rows of q are bf16,
// f32 rows of q three bf16 terms; weights are three terms for f32 rows (2^-24 of
// themselves) and two for bf16 rows (2^-17: with one term, 2^-9, the results' error was
// 1.4 times that of their own rounding).
//
// Positions that a row does not see: scores become -infinity by selection, and V of
// positions that no row of the wave sees is not read into a product.  A value that is
// not finite can still stand where one row sees it and another does not, and a weight's
// term of zero times infinity is NaN: a wave whose sums do not come out finite computes
// its rows again one position at a time in f32 (attn_kvp_again), with each row's own mask.
#include "kernels.h"
#include "gemm_common.h"
#include <type_traits>

namespace qasr {

#define KVP_NEG_INF (-__builtin_inff())
// a running maximum is moved only when it is passed by 2^8: weights stay below 2^8
#define KVP_SLACK 8.0f

template <int HD>
struct KvpDims {
    static constexpr int KC = HD / 32;       // k chunks of a score product
    static constexpr int VT = HD / 16;       // products of O, dims of a lane's V row
};

// one segment of positions: the whole sequence, or a group's shared prefix, or what a
// sequence has behind it
struct KvpSegment {
    const int32_t *table;
    int lo, hi;                // positions [lo, hi) at most
};

// terms of 8 values: x = o[0] + o[1] + .., each the rest rounded to bf16
template <int T>
__device__ __forceinline__ void kvp_terms(const float *x, bf16x8 *o) {
    uint32_t d[T][4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        float a = x[2 * e], b = x[2 * e + 1];
#pragma unroll
        for (int t = 0; t < T; t++) {
            const uint32_t h = cvt_pk_bf16(a, b);
            d[t][e] = h;
            if (t + 1 < T) {
                a = __fsub_rn(a, __uint_as_float(h << 16));
                b = __fsub_rn(b, __uint_as_float(h & 0xffff0000u));
            }
        }
    }
#pragma unroll
    for (int t = 0; t < T; t++) o[t] = __builtin_bit_cast(bf16x8, make_uint4(d[t][0], d[t][1], d[t][2], d[t][3]));
}

// `count` consecutive values of a row of q
template <bool BF16, int COUNT>
__device__ __forceinline__ void kvp_load_q(const void *q, int64_t at, bool vec, float *v) {
    if (BF16) {
        const uint16_t *p = reinterpret_cast<const uint16_t *>(q) + at;
#pragma unroll
        for (int i = 0; i < COUNT; i += 8) {
            if (vec) {
                const uint4 u = *reinterpret_cast<const uint4 *>(p + i);
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    v[i + 2 * e] = __uint_as_float(w[e] << 16);
                    v[i + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) v[i + e] = bf16_to_f32(p[i + e]);
            }
        }
    } else {
        const float *p = reinterpret_cast<const float *>(q) + at;
#pragma unroll
        for (int i = 0; i < COUNT; i += 4) {
            if (vec) {
                const f32x4 u = *reinterpret_cast<const f32x4 *>(p + i);
#pragma unroll
                for (int e = 0; e < 4; e++) v[i + e] = u[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) v[i + e] = p[i + e];
            }
        }
    }
}

// COUNT (4 or 8) consecutive results of a row
template <bool BF16, int COUNT>
__device__ __forceinline__ void kvp_store(void *out, int64_t at, bool vec, const float *v) {
    if (BF16) {
        uint16_t *p = reinterpret_cast<uint16_t *>(out) + at;
        uint32_t d[COUNT / 2];
#pragma unroll
        for (int e = 0; e < COUNT / 2; e++) d[e] = cvt_pk_bf16(v[2 * e], v[2 * e + 1]);
        if (vec) {
            if (COUNT == 8) *reinterpret_cast<uint4 *>(p) = make_uint4(d[0], d[1], d[COUNT / 2 - 2], d[COUNT / 2 - 1]);
            else *reinterpret_cast<uint2 *>(p) = make_uint2(d[0], d[1]);
        } else {
#pragma unroll
            for (int e = 0; e < COUNT; e++) p[e] = (uint16_t)(d[e / 2] >> (16 * (e & 1)));
        }
    } else {
        float *p = reinterpret_cast<float *>(out) + at;
#pragma unroll
        for (int i = 0; i < COUNT; i += 4) {
            if (vec) *reinterpret_cast<f32x4 *>(p + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
            else
#pragma unroll
                for (int e = 0; e < 4; e++) p[i + e] = v[i + e];
        }
    }
}

// the pages of a tile's two halves; -1: no page
struct KvpIds { int id[2]; };
__device__ __forceinline__ KvpIds kvp_ids(const AttnKvpArgs &a, const int32_t *table, int base) {
    KvpIds r;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int s = (base + 16 * h) >> a.s.shift;
        r.id[h] = s < a.s.table_ld ? __builtin_amdgcn_readfirstlane(table[s]) : -1;
        if ((unsigned)r.id[h] >= (unsigned)a.s.n_pages) r.id[h] = -1;
    }
    return r;
}
// first value of a half's 16 positions of head h
template <int HD>
__device__ __forceinline__ int64_t kvp_at(const AttnKvpArgs &a, int id, int h, int pos) {
    return ((((int64_t)max(id, 0) * a.s.Hkv + h) << a.s.shift) + (pos & ((1 << a.s.shift) - 1))) * HD;
}

// a value that all lanes hold alike, in a scalar register
__device__ __forceinline__ int kvp_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t kvp_uniform(int64_t v) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

template <int HD>
struct KvpK { bf16x8 k[2][HD / 32]; };
template <int HD>
__device__ __forceinline__ void kvp_load_k(const AttnKvpArgs &a, KvpIds ids, int h, int base, KvpK<HD> &o) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const uint16_t *p = a.kp + kvp_at<HD>(a, ids.id[x], h, base + 16 * x) + c * HD + 8 * g;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) o.k[x][i] = *reinterpret_cast<const bf16x8 *>(p + 32 * i);
    }
}
// row e of a lane: position 4 g + (e & 3) of half e / 4, dims HD / 16 * c ..
template <int HD>
struct KvpV { uint32_t v[8][HD / 32]; };
template <int HD>
__device__ __forceinline__ void kvp_load_v(const AttnKvpArgs &a, KvpIds ids, int h, int base, KvpV<HD> &o) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const uint16_t *p = a.vp + kvp_at<HD>(a, ids.id[x], h, base + 16 * x) + 4 * g * HD + HD / 16 * c;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (HD == 128) {
                const uint4 u = *reinterpret_cast<const uint4 *>(p + e * HD);
                o.v[4 * x + e][0] = u.x; o.v[4 * x + e][1] = u.y;
                o.v[4 * x + e][HD / 32 - 2] = u.z; o.v[4 * x + e][HD / 32 - 1] = u.w;
            } else {
                const uint2 u = *reinterpret_cast<const uint2 *>(p + e * HD);
                o.v[4 * x + e][0] = u.x; o.v[4 * x + e][1] = u.y;
            }
        }
    }
}

__device__ __forceinline__ float kvp_max_groups(float v) { return xhalf_max(xrow16_max(v)); }
__device__ __forceinline__ float kvp_sum_groups(float v) { return xhalf_sum(xrow16_sum(v)); }

// The rows of one tile of queries over the wave's positions again, one at a time: a
// lane holds the dims of its column's query that it holds in o, a quarter (16 columns) or
// a half (32) of them, RUN consecutive ones at a time.
template <bool BF16, int HD, int COLS>
__device__ __forceinline__ void attn_kvp_again(const AttnKvpArgs &a, const KvpSegment &sg, int h, int64_t q_at, bool live, int lim, int first,
                                            int end, int step, float kc, float *om) {
    constexpr int D = HD * COLS / 64, RUN = COLS == 16 ? D : HD / 8, STRIDE = 64 / COLS * RUN;
    const int lane = threadIdx.x & 63, g = lane / COLS * RUN;
    float q[D], o[D], m = KVP_NEG_INF, l = 0.0f;
#pragma unroll
    for (int d = 0; d < D; d++) q[d] = o[d] = 0.0f;
    if (live)
#pragma unroll
        for (int d = 0; d < D; d += RUN) kvp_load_q<BF16, RUN>(a.q, q_at + g + d / RUN * STRIDE, false, q + d);
    for (int base = first; base < end; base += step) {
        const KvpIds ids = kvp_ids(a, sg.table, base);
        for (int p = base; p < min(base + 32, end); p++) {
            const int id = p - base < 16 ? ids.id[0] : ids.id[1];
            if (id < 0 || p < sg.lo) continue;
            const int64_t at = kvp_at<HD>(a, id, h, p) + g;
            float s = 0.0f;
#pragma unroll
            for (int d = 0; d < D; d++) s = fmaf(q[d], bf16_to_f32(a.kp[at + d / RUN * STRIDE + d % RUN]), s);
            s = (COLS == 16 ? kvp_sum_groups(s) : xhalf_sum(s)) * kc;
            if (!live || p > lim) continue;
            const float mn = fmaxf(m, s), ref = mn == KVP_NEG_INF ? 0.0f : mn;
            const float al = __builtin_amdgcn_exp2f(m - ref), w = __builtin_amdgcn_exp2f(s - ref);
            m = mn;
            l = l * al + w;
#pragma unroll
            for (int d = 0; d < D; d++) o[d] = fmaf(w, bf16_to_f32(a.vp[at + d / RUN * STRIDE + d % RUN]), o[d] * al);
        }
    }
    if (m == __builtin_inff()) {                 // an infinite score: NaN, in every part
        m = 0.0f;
        l = __builtin_nanf("");
#pragma unroll
        for (int d = 0; d < D; d++) o[d] = l;
    }
#pragma unroll
    for (int d = 0; d < D; d++) om[d] = o[d];
    om[D] = m;
    om[D + 1] = l;
}

template <int HD>
constexpr int kvp_part = HD + 2;                 // floats of a query's part: O, maximum, sum

// blocks: h fastest, then the tile of rows, the split, the group or sequence; the
// prefixes' first
template <bool BF16, int HD, int NT, int WQ>
__global__ __launch_bounds__(256, 2) void k_attn_kvp(AttnKvpArgs a) {
    constexpr int KC = HD / 32, VT = HD / 16, QT = BF16 ? 1 : 3, PT = BF16 ? 2 : 3, WK = 4 / WQ, R = 16 * NT * WQ;
    __shared__ float o_l[WK == 1 ? 1 : WK][WK == 1 ? 1 : 16 * NT][HD + 4];
    __shared__ float ml_l[WK == 1 ? 1 : WK][2][16 * NT];
    __shared__ int64_t qi_l[WK == 1 ? 1 : 16 * NT];
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wq = wid / WK, wk = wid % WK;

    // ---- which rows, which positions
    unsigned b = blockIdx.x;
    const int h = b % a.s.Hkv;
    b /= a.s.Hkv;
    const int n_groups = a.prefix ? (a.s.n_seq + a.group - 1) / a.group : 0;
    const unsigned n_prefix = (unsigned)n_groups * a.sp * a.ptiles;
    const bool is_prefix = b < n_prefix;
    if (!is_prefix) b -= n_prefix;
    const int tiles = is_prefix ? a.ptiles : a.otiles, splits = is_prefix ? a.sp : a.so, chunk = is_prefix ? a.cp : a.co;
    const int tile = b % tiles, split = b / tiles % splits, unit = b / tiles / splits;
    const int cap = a.s.table_ld << a.s.shift;
    // a prefix takes max_rows rows of each member, those that a member does not have among them
    KvpSegment sg;
    const int j0 = is_prefix ? unit * a.group : unit;
    KvpRows sq{};
    unsigned n_flat;
    if (is_prefix) {
        sg.lo = 0;
        sg.hi = min(max(a.shared[unit], 0), cap);
        n_flat = (unsigned)min(a.group, a.s.n_seq - j0) * (unsigned)a.s.max_rows * (unsigned)a.G;
    } else {
        sq = kvp_rows(a.s, j0);
        sg.lo = a.prefix ? min(max(a.shared[j0 / a.group], 0), cap) : 0;
        sg.hi = (int)min((int64_t)cap, max((int64_t)sq.p0 + sq.n, (int64_t)0));
        n_flat = (unsigned)sq.n * (unsigned)a.G;
    }
    sg.table = a.s.table + (int64_t)j0 * a.s.table_ld;
    const unsigned f0 = (unsigned)tile * R;
    if (f0 >= n_flat) return;
    const int from = (sg.lo & ~31) + split * chunk;
    // an own part exists even if it is empty (it may be all that a row has); a prefix's only where there are positions
    if (split > 0 ? from >= sg.hi : is_prefix && sg.hi <= 0) return;
    const int upto = split + 1 < splits ? min(from + chunk, sg.hi) : sg.hi;

    // ---- the queries
    const unsigned fw = f0 + wq * 16 * NT;
    const float kc = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * 1.4426950408889634f;
    bf16x8 q[NT][QT][KC];
    int64_t q_at[NT], qi[NT];
    int lim[NT], wave_max = -1, wave_min = 0x7fffffff;
    bool live[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const unsigned f = fw + 16 * n + c, slot = f / (unsigned)a.G, head = h * a.G + f % (unsigned)a.G;
        KvpRows of = sq;
        int i = (int)slot;
        live[n] = f < n_flat;
        if (is_prefix && live[n]) {
            i = (int)(slot % (unsigned)a.s.max_rows);
            of = kvp_rows(a.s, j0 + (int)(slot / (unsigned)a.s.max_rows));
            live[n] = i < of.n;
        }
        q_at[n] = (of.r0 + i) * a.ldq + (int64_t)head * HD;
        qi[n] = (of.r0 + i) * a.Hq + head;
        const int at = is_prefix ? min(sg.hi - 1, of.p0 + i) : of.p0 + i;
        // rows past the end see everything, so that they ask for no mask: they are written nowhere
        lim[n] = live[n] ? min(at, cap - 1) : 0x7fffffff;
        wave_max = max(wave_max, live[n] ? lim[n] : -1);
        wave_min = min(wave_min, lim[n]);
        float x[KC][8];
#pragma unroll
        for (int i = 0; i < KC; i++) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[i][e] = 0.0f;
            if (live[n]) kvp_load_q<BF16, 8>(a.q, q_at[n] + 32 * i + 8 * g, a.vec_q, x[i]);
        }
#pragma unroll
        for (int i = 0; i < KC; i++) {
            // a negative scale is the queries', a zero one makes them zero
#pragma unroll
            for (int e = 0; e < 8; e++) x[i][e] = a.scale == 0.0f ? 0.0f : a.scale < 0.0f ? -x[i][e] : x[i][e];
            bf16x8 tr[QT];
            kvp_terms<QT>(x[i], tr);
#pragma unroll
            for (int t = 0; t < QT; t++) q[n][t][i] = tr[t];
        }
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        wave_max = max(wave_max, __shfl_xor(wave_max, o, 64));
        wave_min = min(wave_min, __shfl_xor(wave_min, o, 64));
    }
    wave_max = __builtin_amdgcn_readfirstlane(wave_max);
    wave_min = __builtin_amdgcn_readfirstlane(wave_min);

    // ---- the positions
    f32x4 o[NT][VT];
    float m[NT], l[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        m[n] = KVP_NEG_INF;
        l[n] = 0.0f;
#pragma unroll
        for (int t = 0; t < VT; t++) o[n][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    constexpr int STEP = 32 * WK;
    const int first = from + 32 * wk, end = min(upto, wave_max + 1);
    if (first < end) {
        KvpK<HD> k;
        KvpIds ids = kvp_ids(a, sg.table, first), next_ids = kvp_ids(a, sg.table, min(first + STEP, end - 1) & ~31);
        kvp_load_k<HD>(a, ids, h, first, k);
        for (int base = first; base < end; base += STEP) {
            KvpV<HD> v;
            kvp_load_v<HD>(a, ids, h, base, v);
            KvpK<HD> kn;
            const int nb = base + STEP < end ? base + STEP : base;
            const KvpIds now = ids;
            ids = base + STEP < end ? next_ids : ids;
            kvp_load_k<HD>(a, ids, h, nb, kn);
            next_ids = kvp_ids(a, sg.table, min(nb + STEP, end - 1) & ~31);

            const bool edge = base < sg.lo || base + 31 > wave_min || base + 32 > end || (now.id[0] | now.id[1]) < 0;
            bf16x8 p[NT][PT];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                f32x4 s[2];
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    s[x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < KC; i++)
#pragma unroll
                        for (int t = QT - 1; t >= 0; t--) s[x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k.k[x][i], q[n][t][i], s[x], 0, 0, 0);
                }
                if (edge) {
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int pos = base + 16 * x + 4 * g + r;
                            s[x][r] = pos >= sg.lo && pos <= min(lim[n], end - 1) && now.id[x] >= 0 ? s[x][r] : KVP_NEG_INF;
                        }
                }
                float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
                mx = kvp_max_groups(mx) * kc;
                if (__any(mx > m[n] + KVP_SLACK)) {
                    const float mn = fmaxf(m[n], mx), ref = mn == KVP_NEG_INF ? 0.0f : mn;
                    const float al = __builtin_amdgcn_exp2f(m[n] - ref);
                    m[n] = mn;
                    l[n] *= al;
#pragma unroll
                    for (int t = 0; t < VT; t++)
#pragma unroll
                        for (int r = 0; r < 4; r++) o[n][t][r] *= al;
                }
                const float ref = m[n] == KVP_NEG_INF ? 0.0f : m[n];
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; e++) w[e] = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], kc, -ref));
                l[n] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
                kvp_terms<PT>(w, p[n]);
            }
            if (edge) {
                // V of positions that no row here sees may hold anything
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int pos = base + 16 * (e >> 2) + 4 * g + (e & 3);
                    const bool seen = pos >= sg.lo && pos < end && now.id[e >> 2] >= 0;
#pragma unroll
                    for (int d = 0; d < HD / 32; d++) v.v[e][d] = seen ? v.v[e][d] : 0u;
                }
            }
#pragma unroll
            for (int t = 0; t < VT; t++) {
                // value t of the lane's eight rows
                uint32_t d[4];
#pragma unroll
                for (int e = 0; e < 4; e++) d[e] = __builtin_amdgcn_perm(v.v[2 * e + 1][t >> 1], v.v[2 * e][t >> 1], (t & 1) ? 0x07060302 : 0x05040100);
                const bf16x8 vt = __builtin_bit_cast(bf16x8, make_uint4(d[0], d[1], d[2], d[3]));
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int x = PT - 1; x >= 0; x--) o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, p[n][x], o[n][t], 0, 0, 0);
            }
            k = kn;
        }
        // sums that are not finite: again, row by row
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float z = l[n] * 0.0f;
#pragma unroll
            for (int t = 0; t < VT; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) z = fmaf(o[n][t][r], 0.0f, z);
            l[n] = kvp_sum_groups(l[n]);
            if (__any(live[n] && z != 0.0f)) {
                float om[HD / 4 + 2];
                attn_kvp_again<BF16, HD, 16>(a, sg, h, q_at[n], live[n], lim[n], first, end, STEP, a.scale * 1.4426950408889634f, om);
#pragma unroll
                for (int t = 0; t < VT; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) o[n][t][r] = om[VT * r + t];
                m[n] = om[HD / 4];
                l[n] = om[HD / 4 + 1];
            }
        }
    }

    // ---- out: the rows themselves, or their part
    const bool whole = !a.prefix && a.so == 1;
    const int P = (a.prefix ? a.sp : 0) + a.so, part_i = is_prefix ? split : (a.prefix ? a.sp : 0) + split;
    auto put = [&](int64_t qi, int d, float *v, auto count, float ll, float mm) {
        if (whole) {
            const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll
            for (int e = 0; e < decltype(count)::value; e++) v[e] *= inv;
            kvp_store<BF16, decltype(count)::value>(a.out, qi * HD + d, a.vec_o, v);
        } else {
            float *part = a.part + (qi * P + part_i) * kvp_part<HD>;
#pragma unroll
            for (int e = 0; e < decltype(count)::value; e += 2) *reinterpret_cast<float2 *>(part + d + e) = make_float2(v[e], v[e + 1]);
            if (d == 0) *reinterpret_cast<float2 *>(part + HD) = make_float2(mm, ll);
        }
    };
    if (WK == 1) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            if (!live[n]) continue;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float v[VT];
#pragma unroll
                for (int t = 0; t < VT; t++) v[t] = o[n][t][r];
                put(qi[n], VT * (4 * g + r), v, std::integral_constant<int, VT>{}, l[n], m[n]);
            }
        }
        return;
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
        if (g == 0) {
            ml_l[wk][0][16 * n + c] = m[n];
            ml_l[wk][1][16 * n + c] = l[n];
            if (wk == 0) qi_l[16 * n + c] = live[n] ? qi[n] : -1;
        }
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int t = 0; t < VT; t += 4)
                *reinterpret_cast<f32x4 *>(&o_l[wk][16 * n + c][VT * (4 * g + r) + t]) = f32x4{o[n][t][r], o[n][t + 1][r], o[n][t + 2][r], o[n][t + 3][r]};
    }
    __syncthreads();
    const int cols = (int)min((unsigned)R, n_flat - f0);
    for (int i = threadIdx.x; i < cols * (HD / 4); i += 256) {
        const int col = i / (HD / 4), d = 4 * (i % (HD / 4));
        if (qi_l[col] < 0) continue;
        float mm = KVP_NEG_INF, ll = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < WK; w++) mm = fmaxf(mm, ml_l[w][0][col]);
        const float ref = mm == KVP_NEG_INF ? 0.0f : mm;
#pragma unroll
        for (int w = 0; w < WK; w++) {
            const float e = __builtin_amdgcn_exp2f(ml_l[w][0][col] - ref);
            ll = fmaf(ml_l[w][1][col], e, ll);
            const f32x4 ow = *reinterpret_cast<const f32x4 *>(&o_l[w][col][d]);
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] = fmaf(ow[r], e, v[r]);
        }
        put(qi_l[col], d, v, std::integral_constant<int, 4>{}, ll, mm);
    }
}

// Many rows of a sequence: a block of four waves, 32 query columns each, goes through the
// positions together; K and V come 32 positions at a time through a ring of three LDS
// stages, so a block reads them once.  v_mfma 32x32x16: S^T leaves lane half hf of a
// column positions 8 (r / 4) + 4 hf + r % 4, and the second product's k is numbered like
// that, as above.  16-byte piece n of position r stands at n ^ (r & 15) (128 dims) or
// n ^ ((r / 2) & 7) (64), which spreads the 16 lanes that LDS serves at a time over all banks.
typedef float f32x16 __attribute__((ext_vector_type(16)));
template <bool BF16, int HD>
__global__ __launch_bounds__(256, 2) void k_attn_kvp_rows(AttnKvpArgs a) {
    constexpr int KC = HD / 16, DV = HD / 32, QT = BF16 ? 1 : 3, PT = BF16 ? 2 : 3, R = 128;
    constexpr int ROW = HD * 2, TB = 32 * ROW, NS = 3, NL = TB / 4096, PR = ROW / 16, RPL = 64 / PR;
    __shared__ __attribute__((aligned(1024))) char ring[NS * 2 * TB];
    const int lane = threadIdx.x & 63, c = lane & 31, hf = lane >> 5;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // ---- which rows, which positions; the tiles with the most positions first
    unsigned b = blockIdx.x;
    const int h = b % a.s.Hkv;
    b /= a.s.Hkv;
    const int tile = a.otiles - 1 - (int)(b % (unsigned)a.otiles), split = b / a.otiles % (unsigned)a.so, j = b / a.otiles / a.so;
    const int cap = a.s.table_ld << a.s.shift;
    const KvpRows sq = kvp_rows(a.s, j);
    const unsigned n_flat = (unsigned)sq.n * (unsigned)a.G, f0 = (unsigned)tile * R, fw = f0 + 32 * wid;
    if (f0 >= n_flat) return;
    KvpSegment sg;
    sg.table = a.s.table + (int64_t)j * a.s.table_ld;
    sg.lo = 0;
    sg.hi = (int)min((int64_t)cap, max((int64_t)sq.p0 + sq.n, (int64_t)0));
    const int from = split * a.co;
    if (split > 0 && from >= sg.hi) return;
    const int upto = split + 1 < a.so ? min(from + a.co, sg.hi) : sg.hi;
    auto last_seen = [&](unsigned f) { return min(sq.p0 + (int)((min(f, n_flat) - 1) / (unsigned)a.G), cap - 1); };
    const int block_end = min(upto, last_seen(f0 + R) + 1), n_it = kvp_uniform(block_end > from ? (block_end - from + 31) / 32 : 0);
    const int end = kvp_uniform(fw < n_flat ? min(upto, last_seen(fw + 32) + 1) : from);      // this wave's
    const int all_see = kvp_uniform(fw < n_flat ? sq.p0 + (int)(fw / (unsigned)a.G) : -1);    // what its first row sees

    // ---- a stage: each wave loads 8 positions of K and of V
    uint32_t src[NL];
#pragma unroll
    for (int i = 0; i < NL; i++) {
        const int r = 8 * wid + RPL * i + lane / PR, n = (lane % PR) ^ (HD == 128 ? r & 15 : (r >> 1) & 7);
        src[i] = (uint32_t)((r & 15) * ROW + 16 * n);
    }
    auto id_of = [&](int base) -> int {                          // the page of this wave's 8 positions
        const int s = (base + 16 * (wid >> 1)) >> a.s.shift;
        return s < a.s.table_ld ? __builtin_amdgcn_readfirstlane(sg.table[s]) : -1;
    };
    auto base_of = [&](int it) { return from + 32 * min(it, n_it - 1); };
    auto issue = [&](int slot, int base, int id) {
        const int64_t at = kvp_uniform(kvp_at<HD>(a, (unsigned)id < (unsigned)a.s.n_pages ? id : 0, h, base + 16 * (wid >> 1)));
        char *to = ring + slot * 2 * TB + 1024 * NL * wid;
#pragma unroll
        for (int i = 0; i < NL; i++) lds_dma16_s(a.kp + at, src[i], to + 1024 * i);
#pragma unroll
        for (int i = 0; i < NL; i++) lds_dma16_s(a.vp + at, src[i], to + TB + 1024 * i);
    };
    int id_next = 0;
    if (n_it > 0) {
        issue(0, base_of(0), id_of(base_of(0)));
        issue(1, base_of(1), id_of(base_of(1)));
        id_next = id_of(base_of(2));
    }

    // ---- the queries
    const float kc = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * 1.4426950408889634f;
    const unsigned f = fw + c;
    const bool live = f < n_flat;
    const unsigned i_row = live ? f / (unsigned)a.G : 0, head = h * a.G + (live ? f % (unsigned)a.G : 0);
    const int64_t q_at = (sq.r0 + i_row) * a.ldq + (int64_t)head * HD, qi = (sq.r0 + i_row) * a.Hq + head;
    const int lim = live ? min(sq.p0 + (int)i_row, cap - 1) : 0x7fffffff;
    bf16x8 q[QT][KC];
#pragma unroll
    for (int i = 0; i < KC; i++) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = 0.0f;
        if (live) kvp_load_q<BF16, 8>(a.q, q_at + 16 * i + 8 * hf, a.vec_q, x);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = a.scale == 0.0f ? 0.0f : a.scale < 0.0f ? -x[e] : x[e];
        bf16x8 tr[QT];
        kvp_terms<QT>(x, tr);
#pragma unroll
        for (int t = 0; t < QT; t++) q[t][i] = tr[t];
    }

    f32x16 o[DV];
    float m = KVP_NEG_INF, l = 0.0f;
#pragma unroll
    for (int t = 0; t < DV; t++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[t][r] = 0.0f;
    KvpIds ids = kvp_ids(a, sg.table, n_it > 0 ? base_of(0) : 0);
    for (int it = 0; it < n_it; it++) {
        wait_vmcnt<2 * NL>();                                    // this wave's loads of the stage have landed
        __syncthreads();                                         // ... and every wave's; the stage before is free
        issue((it + 2) % NS, base_of(it + 2), id_next);
        id_next = id_of(base_of(it + 3));
        const KvpIds now = ids;
        ids = kvp_ids(a, sg.table, base_of(it + 1));
        const int base = from + 32 * it;
        if (base >= end) continue;
        const char *ks = ring + it % NS * 2 * TB, *vs = ks + TB;
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < KC; i++) {
            const int n = (2 * i + hf) ^ (HD == 128 ? c & 15 : (c >> 1) & 7);
            const bf16x8 k = *reinterpret_cast<const bf16x8 *>(ks + c * ROW + 16 * n);
#pragma unroll
            for (int t = QT - 1; t >= 0; t--) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q[t][i], s, 0, 0, 0);
        }
        const bool edge = base + 31 > all_see || base + 32 > end || (now.id[0] | now.id[1]) < 0;
        if (edge) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int pos = base + 8 * (r >> 2) + 4 * hf + (r & 3);
                s[r] = pos <= min(lim, end - 1) && now.id[r >> 3] >= 0 ? s[r] : KVP_NEG_INF;
            }
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; r++) mx = fmaxf(mx, s[r]);
        mx = xhalf_max(mx) * kc;
        if (__any(mx > m + KVP_SLACK)) {
            const float mn = fmaxf(m, mx), ref = mn == KVP_NEG_INF ? 0.0f : mn;
            const float al = __builtin_amdgcn_exp2f(m - ref);
            m = mn;
            l *= al;
#pragma unroll
            for (int t = 0; t < DV; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[t][r] *= al;
        }
        const float ref = m == KVP_NEG_INF ? 0.0f : m;
        float w[16];
#pragma unroll
        for (int r = 0; r < 16; r++) w[r] = __builtin_amdgcn_exp2f(fmaf(s[r], kc, -ref));
        l += (((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]))) + (((w[8] + w[9]) + (w[10] + w[11])) + ((w[12] + w[13]) + (w[14] + w[15])));
#pragma unroll
        for (int x = 0; x < 2; x++) {
            bf16x8 p[PT];
            kvp_terms<PT>(w + 8 * x, p);
            uint32_t v[8][DV / 2];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int r = 16 * x + 8 * (e >> 2) + 4 * hf + (e & 3), swz = HD == 128 ? r & 15 : (r >> 1) & 7;
                const char *row = vs + r * ROW;
                if (HD == 128) {
                    const uint2 u = *reinterpret_cast<const uint2 *>(row + 16 * ((c >> 1) ^ swz) + 8 * (c & 1));
                    v[e][0] = u.x;
                    v[e][DV / 2 - 1] = u.y;
                } else {
                    v[e][0] = *reinterpret_cast<const uint32_t *>(row + 16 * ((c >> 2) ^ swz) + 4 * (c & 3));
                }
                if (edge) {
                    // V of positions that no row here sees may hold anything
#pragma unroll
                    for (int d = 0; d < DV / 2; d++) v[e][d] = base + r < end && now.id[x] >= 0 ? v[e][d] : 0u;
                }
            }
#pragma unroll
            for (int t = 0; t < DV; t++) {
                uint32_t d[4];
#pragma unroll
                for (int e = 0; e < 4; e++) d[e] = __builtin_amdgcn_perm(v[2 * e + 1][t >> 1], v[2 * e][t >> 1], (t & 1) ? 0x07060302 : 0x05040100);
                const bf16x8 vt = __builtin_bit_cast(bf16x8, make_uint4(d[0], d[1], d[2], d[3]));
#pragma unroll
                for (int y = PT - 1; y >= 0; y--) o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vt, p[y], o[t], 0, 0, 0);
            }
        }
    }
    wait_vmcnt<0>();                                             // no load may land in LDS after the block ends
    // sums that are not finite: again, row by row
    float z = l * 0.0f;
#pragma unroll
    for (int t = 0; t < DV; t++)
#pragma unroll
        for (int r = 0; r < 16; r++) z = fmaf(o[t][r], 0.0f, z);
    l = xhalf_sum(l);
    if (__any(live && z != 0.0f)) {
        float om[HD / 2 + 2];
        attn_kvp_again<BF16, HD, 32>(a, sg, h, q_at, live, lim, from, end, 32, a.scale * 1.4426950408889634f, om);
#pragma unroll
        for (int t = 0; t < DV; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[t][r] = om[4 * DV * (r >> 2) + DV * (r & 3) + t];
        m = om[HD / 2];
        l = om[HD / 2 + 1];
    }
    if (!live) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    float *part = a.part + (qi * a.so + split) * kvp_part<HD>;
#pragma unroll
    for (int x = 0; x < 4; x++) {
        float v[4 * DV];
        const int d = 4 * DV * (2 * x + hf);
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int t = 0; t < DV; t++) v[DV * r + t] = o[t][4 * x + r];
        if (a.so == 1) {
#pragma unroll
            for (int e = 0; e < 4 * DV; e++) v[e] *= inv;
#pragma unroll
            for (int e = 0; e < 4 * DV; e += 8) kvp_store<BF16, 8>(a.out, qi * HD + d + e, a.vec_o, v + e);
        } else {
#pragma unroll
            for (int e = 0; e < 4 * DV; e += 2) *reinterpret_cast<float2 *>(part + d + e) = make_float2(v[e], v[e + 1]);
        }
    }
    if (a.so > 1 && hf == 0) *reinterpret_cast<float2 *>(part + HD) = make_float2(m, l);
}

// The parts of each row and head, in order; a wave a head.  Each lane weighs one part,
// then the sums' loads do not wait for one another.
template <bool BF16, int HD>
__global__ __launch_bounds__(256) void k_attn_kvp_merge(AttnKvpArgs a) {
    const int lane = threadIdx.x & 63;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = blockIdx.y, i = blockIdx.x, head = blockIdx.z * 4 + wid;
    const KvpRows sq = kvp_rows(a.s, j);
    if (i >= sq.n || head >= a.Hq) return;
    const int cap = a.s.table_ld << a.s.shift, sp = a.prefix ? a.sp : 0, P = sp + a.so;
    const int sh = a.prefix ? min(max(a.shared[j / a.group], 0), cap) : 0;
    const int hi = (int)min((int64_t)cap, max((int64_t)sq.p0 + sq.n, (int64_t)0)), lo = sh & ~31;
    // the parts that the blocks wrote
    const int np = a.prefix ? min(sp, (sh + a.cp - 1) / a.cp) : 0, no = hi > lo ? min(a.so, (hi - lo + a.co - 1) / a.co) : 1;
    const int64_t qi = (sq.r0 + i) * a.Hq + head;
    const float *part = a.part + qi * P * kvp_part<HD>;
    const bool have = lane < sp ? lane < np : lane < sp + no;
    float2 ml = make_float2(KVP_NEG_INF, 0.0f);
    if (have) ml = *reinterpret_cast<const float2 *>(part + lane * kvp_part<HD> + HD);
    float mm = ml.x;
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) mm = fmaxf(mm, __shfl_xor(mm, s, 64));
    const float w = have ? __builtin_amdgcn_exp2f(ml.x - (mm == KVP_NEG_INF ? 0.0f : mm)) : 0.0f;
    const float ll = wave_sum_f32(ml.y * w);
    constexpr int E = HD / 64;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = 0.0f;
    for (int x = 0; x < P; x++) {
        if (x < sp ? x >= np : x >= sp + no) continue;
        const float wx = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), x));
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = fmaf(part[x * kvp_part<HD> + E * lane + e], wx, v[e]);
    }
    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int64_t at = qi * HD + E * lane + e;
        if (BF16) reinterpret_cast<__bf16 *>(a.out)[at] = (__bf16)(v[e] * inv);
        else reinterpret_cast<float *>(a.out)[at] = v[e] * inv;
    }
}

template <bool BF16, int HD>
static hipError_t go_merge(const AttnKvpArgs &a, hipStream_t st) {
    hipLaunchKernelGGL((k_attn_kvp_merge<BF16, HD>), dim3((unsigned)a.s.max_rows, (unsigned)a.s.n_seq, (unsigned)(a.Hq + 3) / 4), dim3(256), 0, st, a);
    return hipGetLastError();
}

// splits of `len` positions over blocks that take `step` of them a turn: up to 512 blocks
// (two a CU) at `units` tiles, each with `turns` turns at least
static void kvp_split(int64_t units, int64_t len, int64_t most, int step, int turns, int &s, int &chunk) {
    const int64_t tiles = (len + 31) / 32 + 1;
    const int64_t n = std::max<int64_t>(1, std::min({most, 512 / std::max<int64_t>(1, units), tiles * 32 / (step * turns)}));
    chunk = (int)((tiles + n - 1) / n * 32);
    s = (int)((tiles * 32 + chunk - 1) / chunk);
}

template <bool BF16, int HD>
static hipError_t go_rows(AttnKvpArgs &a, int64_t room, hipStream_t st) {
    const int64_t tiles = (a.s.max_rows * a.G + 127) / 128;
    // sequences shorter than max_rows leave tiles empty: counted are those that n_rows rows fill, half a one a sequence
    const int64_t units = std::min(tiles * a.s.n_seq, (a.s.n_rows * a.G / 64 + a.s.n_seq) / 2 + 1) * a.s.Hkv;
    kvp_split(units, a.max_len, std::max<int64_t>(1, room), 32, 4, a.so, a.co);
    a.otiles = (int)tiles;
    const int64_t blocks = (int64_t)a.s.n_seq * a.so * tiles * a.s.Hkv;
    if (blocks * 256 > UINT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_attn_kvp_rows<BF16, HD>), dim3((unsigned)blocks), dim3(256), 0, st, a);
    return a.so > 1 ? go_merge<BF16, HD>(a, st) : hipGetLastError();
}

template <bool BF16, int HD>
static hipError_t go_few(AttnKvpArgs &a, int64_t room, hipStream_t st) {
    constexpr int R = 16;
    const int64_t n_groups = a.prefix ? (a.s.n_seq + a.group - 1) / a.group : 0;
    const int64_t otiles = (a.s.max_rows * a.G + R - 1) / R, ptiles = a.prefix ? ((int64_t)a.group * a.s.max_rows * a.G + R - 1) / R : 0;
    a.otiles = (int)otiles;
    a.ptiles = (int)ptiles;
    a.sp = 1;
    a.cp = 1 << 30;
    if (a.prefix) kvp_split(n_groups * ptiles * a.s.Hkv, a.max_len, room / 2, 128, 1, a.sp, a.cp);
    kvp_split((int64_t)a.s.n_seq * a.s.Hkv * otiles, a.prefix ? a.max_own : a.max_len, a.prefix ? room - a.sp : std::max<int64_t>(1, room), 128, 1, a.so, a.co);
    const int64_t blocks = (n_groups * a.sp * ptiles + (int64_t)a.s.n_seq * a.so * otiles) * a.s.Hkv;
    if (blocks * 256 > UINT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_attn_kvp<BF16, HD, 1, 1>), dim3((unsigned)blocks), dim3(256), 0, st, a);
    return a.prefix || a.so > 1 ? go_merge<BF16, HD>(a, st) : hipGetLastError();
}

template <bool BF16, int HD>
static hipError_t go_attn_kvp(AttnKvpArgs &a, int64_t room, hipStream_t st) {
    return a.s.max_rows * a.G > 32 ? go_rows<BF16, HD>(a, room, st) : go_few<BF16, HD>(a, room, st);
}

hipError_t launch_attention_kvp(const AttnKvpArgs &a0, bool bf16, hipStream_t st) {
    AttnKvpArgs a = a0;
    if ((a.s.hd != 64 && a.s.hd != 128) || a.s.n_seq > 65535 || a.s.Hkv > 65535) return hipErrorInvalidValue;
    a.vec_q = (uintptr_t)a.q % 16 == 0 && (a.ldq * (bf16 ? 2 : 4)) % 16 == 0;
    a.vec_o = (uintptr_t)a.out % 16 == 0;
    // parts that fit the scratch area, for every row and head
    const int64_t room = std::min<int64_t>(64, (int64_t)QASR_KVP_PART_BYTES / (a.s.n_rows * a.Hq * (a.s.hd + 2) * 4));
    a.prefix = a.shared && a.s.max_rows * a.G <= 32 && room >= 2;
    if (bf16) return a.s.hd == 128 ? go_attn_kvp<true, 128>(a, room, st) : go_attn_kvp<true, 64>(a, room, st);
    return a.s.hd == 128 ? go_attn_kvp<false, 128>(a, room, st) : go_attn_kvp<false, 64>(a, room, st);
}

}  // namespace qasr
