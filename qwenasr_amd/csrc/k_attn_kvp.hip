// Attention over a KV cache in pages, a prefix that a group of sequences shares read
// for 16 rows x heads of theirs at a time.
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
// f32 rows of q three bf16 terms; weights are three terms (2^-24 of themselves), but two
// (2^-17) in tiles of many bf16 rows: the third costs 10 to 20% there (8 x 512 rows behind
// 3400 180 us, with three 217), and 0.2 to 2.7% of few rows (32 x 4000 73.6 / 73.9, 8
// hypotheses 9.1 / 9.3).  With two, results come out one step off the nearest bf16 value
// more often (2-norm of the difference 1.0e-4 of the results', with three 4e-5, of an f32
// form 5e-5); with one, 2^-9, their error was 1.4 times that of their own rounding.
//
// Positions that a row does not see: scores become -infinity by selection, and V of
// positions that no row of the wave sees is not read into a product.  A value that is
// not finite can still stand where one row sees it and another does not, and a weight's
// term of zero times infinity is NaN: a wave whose sums do not come out finite computes
// its rows again one position at a time in f32 (attn_kvp_again), with each row's own mask.
// So does one with a row that sees positions and found no score above -infinity: the tiles
// do not tell those from positions that it does not see.
#include "kernels.h"
#include "gemm_common.h"
#include "qasr_hip.h"
#include <type_traits>

namespace qasr {

#define KVP_NEG_INF (-__builtin_inff())
// the maximum where positions are seen whose scores are all -infinity, with a sum of 0: -infinity is where none is seen.
// The first gives 0 / 0, as the formula does, unless other positions join it, the second zeros
#define KVP_LOWEST (-__FLT_MAX__)
// a running maximum is moved only when it is passed by 2^8: weights stay below 2^8
#define KVP_SLACK 8.0f

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

// The pages of a tile's two halves; -1: no page.  A wave keeps 64 entries of the table,
// one a lane, and takes them out by lane: a load for each tile would be a wait for
// everything that is on its way.  For tiles in rising order.
struct KvpIds { int id[2]; };
struct KvpTable {
    const int32_t *table;
    int first, entry;
    __device__ __forceinline__ void load(const AttnKvpArgs &a, int s) {
        const int at = s + (int)(threadIdx.x & 63);
        first = s;
        entry = table[min(at, a.s.table_ld - 1)];
        if (at >= a.s.table_ld || (unsigned)entry >= (unsigned)a.s.n_pages) entry = -1;
    }
    __device__ __forceinline__ KvpTable(const AttnKvpArgs &a, const int32_t *t, int base) : table(t) { load(a, base >> a.s.shift); }
    __device__ __forceinline__ KvpIds at(const AttnKvpArgs &a, int base) {
        const int s0 = base >> a.s.shift, s1 = (base + 16) >> a.s.shift;
        if (s1 - first > 63) load(a, s0);
        return {{__builtin_amdgcn_readlane(entry, s0 - first), __builtin_amdgcn_readlane(entry, s1 - first)}};
    }
};
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

// 16 or 8 bytes; ONCE: not to be kept in the caches, as nobody else reads them
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <bool ONCE, typename T>
__device__ __forceinline__ T kvp_load(const uint16_t *p) {
    return ONCE ? __builtin_nontemporal_load(reinterpret_cast<const T *>(p)) : *reinterpret_cast<const T *>(p);
}
template <int HD>
struct KvpK { bf16x8 k[2][HD / 32]; };
template <int HD, bool ONCE>
__device__ __forceinline__ void kvp_load_k(const AttnKvpArgs &a, KvpIds ids, int h, int base, KvpK<HD> &o) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const uint16_t *p = a.kp + kvp_at<HD>(a, ids.id[x], h, base + 16 * x) + c * HD + 8 * g;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) o.k[x][i] = kvp_load<ONCE, bf16x8>(p + 32 * i);
    }
}
// row e of a lane: position 4 g + (e & 3) of half e / 4, dims HD / 16 * c ..
template <int HD>
struct KvpV { uint32_t v[8][HD / 32]; };
template <int HD, bool ONCE>
__device__ __forceinline__ void kvp_load_v(const AttnKvpArgs &a, KvpIds ids, int h, int base, KvpV<HD> &o) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const uint16_t *p = a.vp + kvp_at<HD>(a, ids.id[x], h, base + 16 * x) + 4 * g * HD + HD / 16 * c;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (HD == 128) {
                const u32x4 u = kvp_load<ONCE, u32x4>(p + e * HD);
                o.v[4 * x + e][0] = u[0]; o.v[4 * x + e][1] = u[1];
                o.v[4 * x + e][HD / 32 - 2] = u[2]; o.v[4 * x + e][HD / 32 - 1] = u[3];
            } else {
                const u32x2 u = kvp_load<ONCE, u32x2>(p + e * HD);
                o.v[4 * x + e][0] = u[0]; o.v[4 * x + e][1] = u[1];
            }
        }
    }
}

__device__ __forceinline__ float kvp_max_groups(float v) { return xhalf_max(xrow16_max(v)); }
__device__ __forceinline__ float kvp_sum_groups(float v) { return xhalf_sum(xrow16_sum(v)); }

// The rows of one tile of queries over the wave's positions again, one at a time: a
// lane holds the dims of its column's query that it holds in o, a quarter (16 columns) or
// a half (32) of them, RUN consecutive ones at a time.  first < end.
template <bool BF16, int HD, int COLS>
__device__ __forceinline__ void attn_kvp_again(const AttnKvpArgs &a, const KvpSegment &sg, int h, int64_t q_at, bool live, int lim, int first,
                                            int end, int step, float kc, float *om) {
    constexpr int D = HD * COLS / 64, RUN = COLS == 16 ? D : 8, STRIDE = 64 / COLS * RUN;
    const int lane = threadIdx.x & 63, g = lane / COLS * RUN;
    float q[D], o[D], m = KVP_NEG_INF, l = 0.0f;
#pragma unroll
    for (int d = 0; d < D; d++) q[d] = o[d] = 0.0f;
    if (live)
#pragma unroll
        for (int d = 0; d < D; d += RUN) kvp_load_q<BF16, RUN>(a.q, q_at + g + d / RUN * STRIDE, false, q + d);
    KvpTable table(a, sg.table, first);
    for (int base = first; base < end; base += step) {
        const KvpIds ids = table.at(a, base);
        for (int p = base; p < min(base + 32, end); p++) {
            const int id = p - base < 16 ? ids.id[0] : ids.id[1];
            if (id < 0 || p < sg.lo) continue;
            const int64_t at = kvp_at<HD>(a, id, h, p) + g;
            float s = 0.0f;
#pragma unroll
            for (int d = 0; d < D; d++) s = fmaf(q[d], bf16_to_f32(a.kp[at + d / RUN * STRIDE + d % RUN]), s);
            s = (COLS == 16 ? kvp_sum_groups(s) : xhalf_sum(s)) * kc;
            if (!live || p > lim) continue;
            const float mn = fmaxf(m, fmaxf(s, KVP_LOWEST));
            const float al = __builtin_amdgcn_exp2f(m - mn), w = __builtin_amdgcn_exp2f(s - mn);
            m = mn;
            l = l * al + w;
#pragma unroll
            for (int d = 0; d < D; d++) o[d] = fmaf(w, bf16_to_f32(a.vp[at + d / RUN * STRIDE + d % RUN]), o[d] * al);
        }
    }
    if (m == __builtin_inff() || l != l) {       // an infinite score, or one of NaN (no maximum knows of it): NaN, and a part that the merge takes
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

// Few rows of a sequence, and prefixes: a block of W waves takes 16 query columns, each
// wave every W-th 32 positions straight into registers, as no second tile shares them.
// Blocks: h fastest, then the tile of rows, the split, the group or sequence; the
// prefixes' first.  What bounds short ones is the chain rows -> table -> K -> products ->
// merge, so each load goes out as soon as its address is known: 8 hypotheses of 410 to 435
// positions 9.7 us (the first form 15.3).  Long ones are bound by memory: 32 sequences of up to 4000
// 74 us, 5.6 TB/s (four waves a block 81); four groups of 16 behind 4000 34.1 us (63), of
// which the merge is 4.7.
template <bool BF16, int HD, int W, bool ONCE, bool AHEAD>
__global__ __launch_bounds__(64 * W, 2) void k_attn_kvp(AttnKvpArgs a) {
    constexpr int KC = HD / 32, VT = HD / 16, QT = BF16 ? 1 : 3, PT = 3, R = 16, STEP = 32 * W;
    __shared__ float o_l[W][R][HD + 4];
    __shared__ float ml_l[W][2][R];
    __shared__ bf16x8 q_l[QT][KC][64];
    __shared__ int64_t qi_l[R];
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

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
    const int j0 = is_prefix ? unit * a.group : unit;
    // the lane's row: of a prefix one of max_rows of each member, which a member may not have
    const unsigned f = (unsigned)tile * R + c, slot = f / (unsigned)a.G, head = h * a.G + f % (unsigned)a.G;
    const int members = is_prefix ? min(a.group, a.s.n_seq - j0) : 1;
    const int k_row = is_prefix ? (int)(slot / (unsigned)a.s.max_rows) : 0, i_row = is_prefix ? (int)(slot % (unsigned)a.s.max_rows) : (int)slot;
    const KvpRows sq = kvp_rows(a.s, j0 + min(k_row, members - 1));
    const int sh = a.prefix ? min(max(a.shared[is_prefix ? unit : j0 / a.group], 0), cap) : 0;
    KvpSegment sg;
    sg.table = a.s.table + (int64_t)j0 * a.s.table_ld;
    sg.lo = is_prefix ? 0 : kvp_uniform(sh);
    sg.hi = kvp_uniform(is_prefix ? sh : (int)min((int64_t)cap, max((int64_t)sq.p0 + sq.n, (int64_t)0)));
    const bool live = k_row < members && i_row < sq.n;
    const int from = (sg.lo & ~31) + split * chunk;
    const int64_t qi = (sq.r0 + i_row) * a.Hq + head;
    const bool whole = !a.prefix && a.so == 1;
    const int P = (a.prefix ? a.sp : 0) + a.so, part_i = is_prefix ? split : (a.prefix ? a.sp : 0) + split;
    if (!__any(live)) return;
    if (!whole && from >= sg.hi) {                               // a part without positions
        if (live && threadIdx.x < 16) *reinterpret_cast<float2 *>(a.part + (qi * P + part_i) * kvp_part<HD> + HD) = make_float2(KVP_NEG_INF, 0.0f);
        return;
    }
    const int upto = split + 1 < splits ? min(from + chunk, sg.hi) : sg.hi;
    const int first = from + 32 * wid;
    KvpTable table(a, sg.table, min(first, cap - 1));

    // rows past the end see everything, so that they ask for no mask: they are written nowhere
    const int lim = live ? min(is_prefix ? min(sg.hi - 1, sq.p0 + i_row) : sq.p0 + i_row, cap - 1) : 0x7fffffff;
    int wave_max = live ? lim : -1, wave_min = lim;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        wave_max = max(wave_max, __shfl_xor(wave_max, o, 64));
        wave_min = min(wave_min, __shfl_xor(wave_min, o, 64));
    }
    wave_max = kvp_uniform(wave_max);
    wave_min = kvp_uniform(wave_min);
    const int end = min(upto, wave_max + 1);

    // ---- the first tiles, and the queries: each wave brings a chunk of their dims into terms, for all of them
    KvpK<HD> k0, k1;
    KvpV<HD> v0, v1;
    KvpIds id0, id1;
    if (first < end) {
        id0 = table.at(a, first);
        kvp_load_k<HD, ONCE>(a, id0, h, first, k0);
        kvp_load_v<HD, ONCE>(a, id0, h, first, v0);
    }
    const int64_t q_at = (sq.r0 + i_row) * a.ldq + (int64_t)head * HD;
    // a negative scale is the queries', a zero one makes them zero
    const float kc = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * 1.4426950408889634f, sign = a.scale == 0.0f ? 0.0f : a.scale < 0.0f ? -1.0f : 1.0f;
    for (int i = wid; i < KC; i += W) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = 0.0f;
        if (live) kvp_load_q<BF16, 8>(a.q, q_at + 32 * i + 8 * g, a.vec_q, x);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] *= sign;
        bf16x8 tr[QT];
        kvp_terms<QT>(x, tr);
#pragma unroll
        for (int t = 0; t < QT; t++) q_l[t][i][lane] = tr[t];
    }
    __syncthreads();

    // ---- the positions
    f32x4 o[VT];
    float m = KVP_NEG_INF, l = 0.0f;
#pragma unroll
    for (int t = 0; t < VT; t++) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (first < end) {
        // One tile.  AHEAD: the next one's K and V go out at once, into registers of their own; else into the same
        // ones as soon as the products have read them, and other waves are there to wait with
        auto turn = [&](int base, KvpK<HD> &k, KvpV<HD> &v, KvpIds now, KvpK<HD> &kn, KvpV<HD> &vn, KvpIds &next) {
            const bool more = base + STEP < end;
            if (more) next = table.at(a, base + STEP);
            if (AHEAD && more) {
                kvp_load_k<HD, ONCE>(a, next, h, base + STEP, kn);
                kvp_load_v<HD, ONCE>(a, next, h, base + STEP, vn);
            }
            const bool edge = base < sg.lo || base + 31 > wave_min || base + 32 > end || (now.id[0] | now.id[1]) < 0;
            f32x4 s[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
            int at = lane;
            asm volatile("" : "+v"(at));                 // q stays in LDS: kept over the turns it takes 48 registers
#pragma unroll
            for (int i = 0; i < KC; i++)
#pragma unroll
                for (int t = QT - 1; t >= 0; t--) {
                    const bf16x8 q = q_l[t][i][at];
#pragma unroll
                    for (int y = 0; y < 2; y++) s[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k.k[y][i], q, s[y], 0, 0, 0);
                }
            if (!AHEAD && more) kvp_load_k<HD, ONCE>(a, next, h, base + STEP, kn);
            if (edge) {
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int pos = base + 16 * y + 4 * g + r;
                        s[y][r] = pos >= sg.lo && pos <= min(lim, end - 1) && now.id[y] >= 0 ? s[y][r] : KVP_NEG_INF;
                    }
            }
            float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
            mx = kvp_max_groups(mx) * kc;
            if (__any(mx > m + KVP_SLACK)) {
                const float mn = fmaxf(m, mx), ref = mn == KVP_NEG_INF ? 0.0f : mn;
                const float al = __builtin_amdgcn_exp2f(m - ref);
                m = mn;
                l *= al;
#pragma unroll
                for (int t = 0; t < VT; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) o[t][r] *= al;
            }
            const float ref = m == KVP_NEG_INF ? 0.0f : m;
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], kc, -ref));
            l += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
            bf16x8 p[PT];
            kvp_terms<PT>(w, p);
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
                for (int y = PT - 1; y >= 0; y--) o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, p[y], o[t], 0, 0, 0);
            }
            if (!AHEAD && more) kvp_load_v<HD, ONCE>(a, next, h, base + STEP, vn);
        };
        if (AHEAD) {
            for (int base = first; base < end; base += 2 * STEP) {
                turn(base, k0, v0, id0, k1, v1, id1);
                if (base + STEP < end) turn(base + STEP, k1, v1, id1, k0, v0, id0);
            }
        } else {
            for (int base = first; base < end; base += STEP) {
                turn(base, k0, v0, id0, k0, v0, id1);
                id0 = id1;
            }
        }
        // sums that are not finite, or no score where positions are seen (or would be, on pages that are none): again, row by row
        float z4[4] = {l * 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < VT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) z4[r] = fmaf(o[t][r], 0.0f, z4[r]);
        const float z = (z4[0] + z4[1]) + (z4[2] + z4[3]);
        l = kvp_sum_groups(l);
        if (__any(live && (z != 0.0f || (m == KVP_NEG_INF && lim >= max(first, sg.lo))))) {
            float om[HD / 4 + 2];
            attn_kvp_again<BF16, HD, 16>(a, sg, h, q_at, live, lim, first, end, STEP, a.scale * 1.4426950408889634f, om);
#pragma unroll
            for (int t = 0; t < VT; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) o[t][r] = om[VT * r + t];
            m = om[HD / 4];
            l = om[HD / 4 + 1];
        }
    }

    // ---- the waves' parts together; out: the rows themselves, or their part
    if (live) {
        if (g == 0) {
            ml_l[wid][0][c] = m;
            ml_l[wid][1][c] = l;
        }
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int t = 0; t < VT; t += 4)
                *reinterpret_cast<f32x4 *>(&o_l[wid][c][VT * (4 * g + r) + t]) = f32x4{o[t][r], o[t + 1][r], o[t + 2][r], o[t + 3][r]};
    }
    if (wid == 0 && g == 0) qi_l[c] = live ? qi : -1;
    __syncthreads();
    for (int i = threadIdx.x; i < R * (HD / 4); i += 64 * W) {
        const int col = i / (HD / 4), d = 4 * (i % (HD / 4));
        const int64_t to = qi_l[col];
        if (to < 0) continue;
        float mm = KVP_NEG_INF, ll = 0.0f, r4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < W; w++) mm = fmaxf(mm, ml_l[w][0][col]);
        const float ref = mm == KVP_NEG_INF ? 0.0f : mm;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float e = __builtin_amdgcn_exp2f(ml_l[w][0][col] - ref);
            ll = fmaf(ml_l[w][1][col], e, ll);
            const f32x4 ow = *reinterpret_cast<const f32x4 *>(&o_l[w][col][d]);
#pragma unroll
            for (int r = 0; r < 4; r++) r4[r] = fmaf(ow[r], e, r4[r]);
        }
        if (whole) {
            const float inv = mm == KVP_NEG_INF ? 0.0f : 1.0f / ll;
#pragma unroll
            for (int r = 0; r < 4; r++) r4[r] *= inv;
            kvp_store<BF16, 4>(a.out, to * HD + d, a.vec_o, r4);
        } else {
            float *part = a.part + (to * P + part_i) * kvp_part<HD>;
            *reinterpret_cast<float2 *>(part + d) = make_float2(r4[0], r4[1]);
            *reinterpret_cast<float2 *>(part + d + 2) = make_float2(r4[2], r4[3]);
            if (d == 0) *reinterpret_cast<float2 *>(part + HD) = make_float2(mm, ll);
        }
    }
}

// The i-th of the tiles of R rows x heads that there are, those furthest back in their
// sequences first: those of the last index that a sequence has, in order of the sequences, and so
// on.  Blocks that have none (there are as many as the host can tell) come last: between
// the others they leave the CUs' registers in pieces (six prompts of up to 1337 rows: 400 of
// 512 blocks at a time).
// Sequences of max_rows rows each need no search, and of more sequences than a wave has
// lanes the tiles are counted once, into LDS: read again at each step of the search, 500
// sequences of 40 rows took 226 us.
struct KvpTile { int j, tile; };
template <int R>
__device__ __forceinline__ KvpTile kvp_tile(const AttnKvpArgs &a, int i, int *tiles_l) {
    const int lane = threadIdx.x & 63, n_seq = a.s.n_seq;
    if (a.uniform) return {i % n_seq, a.otiles - 1 - i / n_seq};
    auto tiles_of = [&](int j) { return j < n_seq ? (int)(((unsigned)kvp_rows(a.s, j).n * (unsigned)a.G + R - 1) / R) : 0; };
    if (n_seq == 1) return {0, tiles_of(0) - 1 - i};
    if (n_seq > 64) {
        for (int j = threadIdx.x; j < ((n_seq + 63) & ~63); j += blockDim.x) tiles_l[j] = tiles_of(j);
        __syncthreads();
    }
    const int mine = n_seq > 64 ? tiles_l[lane] : tiles_of(lane);
    // tiles of index t and more
    auto from = [&](int t) {
        int n = max(0, mine - t);
        for (int j = 64 + lane; j < n_seq; j += 64) n += max(0, tiles_l[j] - t);
        return wave_sum_i32(n);
    };
    KvpTile at{0, -1};
    if (i < from(0)) {
        int t = 0, end = a.otiles;               // from(t) > i >= from(end)
        while (end - t > 1) {
            const int mid = (t + end) / 2;
            if (from(mid) > i) t = mid;
            else end = mid;
        }
        int r = i - from(t + 1);                 // of the sequences that have it
        for (int j0 = 0; j0 < n_seq; j0 += 64) {
            const unsigned long long has = __ballot((j0 == 0 ? mine : tiles_l[j0 + lane]) > t);
            const int n = __popcll(has);
            if (r < n) {
                const int before = __builtin_amdgcn_mbcnt_hi((unsigned)(has >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)has, 0));
                at = {j0 + __ffsll((unsigned long long)__ballot(((has >> lane) & 1) && before == r)) - 1, t};
                break;
            }
            r -= n;
        }
    }
    if (n_seq > 64) __syncthreads();             // the counts make way for K and V
    return at;
}

// Many rows of a sequence: a block of RW x PG waves, RW of them side by side with 32 query
// columns each, PG groups of them over every PG-th 32 positions.  A group's K and V
// come through a ring of LDS stages, once for its RW waves; the groups' sums are joined at the
// end.  v_mfma 32x32x16: S^T leaves lane half hf of a
// column positions 8 (r / 4) + 4 hf + r % 4, and the second product's k is numbered like
// that, as above; product t of O has dims 32 t .., a lane of them eight at a time.  V's
// operand is turned as it is read: of 16 lanes that bring 16 dims of four positions, eight
// bytes each, every lane gets one dim of the four.  16-byte piece n of position r stands
// at n ^ kvp_place(r), which spreads over all banks both the 16 positions that K's lanes
// read a piece of and the four that V's read four pieces of (128 dims; 64: two positions
// fill the banks).
//
// Bound by the matrix instructions, three terms each of q and of the weights for f32 rows,
// and the chain between the two products that two waves a SIMD do not cover: 8 x 512 rows
// behind 2262 to 4000 positions, 16 heads, f32 318 us (1.05 PFLOP/s, every term counted; the
// library's bf16 product of 8192^3 reaches 1.41), bf16 199 (0.83); six prompts of up to 1337 rows, f32, 109 us
// (K and V straight into registers 272, V turned there 2% more).
template <int HD>
__device__ __forceinline__ int kvp_place(int r) {
    return HD == 128 ? (r & 3) << 2 | (r >> 2) : (r & 2) << 1 | (r >> 2);
}
__device__ __forceinline__ uint2 kvp_turned(char *p) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p));
}
typedef float f32x16 __attribute__((ext_vector_type(16)));
template <bool BF16, int HD, int RW, int PG>
__global__ __launch_bounds__(64 * RW * PG, 2) void k_attn_kvp_rows(AttnKvpArgs a) {
    constexpr int KC = HD / 16, DV = HD / 32, QT = BF16 ? 1 : 3, PT = BF16 ? 2 : 3, R = 32 * RW;
    // bytes of a position and of a tile (a ring of two: three held a CU to one block); loads of a wave for K of a tile; 16-byte pieces of a position, positions of a load
    constexpr int ROW = HD * 2, TB = 32 * ROW, NS = 2, NL = TB / 1024 / RW, PR = ROW / 16, RPL = 64 / PR;
    constexpr int RING = NS * 2 * TB, JOIN = (PG - 1) * RW * (16 * DV + 2) * 256;
    __shared__ __attribute__((aligned(1024))) char smem[PG * RING > JOIN ? PG * RING : JOIN];
    static_assert(sizeof smem >= 4 * QASR_KVP_MAX_SEQ, "a place for every sequence's count");
    const int lane = threadIdx.x & 63, c = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wid = wave % RW, grp = wave / RW;
    char *const ring = smem + grp * RING;

    // ---- which rows, which positions
    unsigned b = blockIdx.x;
    const int h = b % a.s.Hkv;
    b /= a.s.Hkv;
    const int split = b % (unsigned)a.so;
    const KvpTile at_tile = kvp_tile<R>(a, (int)(b / (unsigned)a.so), reinterpret_cast<int *>(smem));
    const int tile = at_tile.tile, j = at_tile.j;
    if (tile < 0) return;
    const int cap = a.s.table_ld << a.s.shift;
    const KvpRows sq = kvp_rows(a.s, j);
    const unsigned n_flat = (unsigned)sq.n * (unsigned)a.G, f0 = (unsigned)tile * R, fw = f0 + 32 * wid;
    if (f0 >= n_flat) return;
    KvpSegment sg;
    sg.table = a.s.table + (int64_t)j * a.s.table_ld;
    sg.lo = 0;
    sg.hi = (int)min((int64_t)cap, max((int64_t)sq.p0 + sq.n, (int64_t)0));
    const int from = split * a.co;
    if (split > 0 && from >= sg.hi) {                            // a part without positions
        const unsigned f = f0 + threadIdx.x;
        if (threadIdx.x < R && f < n_flat)
            *reinterpret_cast<float2 *>(a.part + (((sq.r0 + f / (unsigned)a.G) * a.Hq + h * a.G + f % (unsigned)a.G) * a.so + split) * kvp_part<HD> + HD) =
                make_float2(KVP_NEG_INF, 0.0f);
        return;
    }
    const int upto = split + 1 < a.so ? min(from + a.co, sg.hi) : sg.hi;
    auto last_seen = [&](unsigned f) { return min(sq.p0 + (int)((min(f, n_flat) - 1) / (unsigned)a.G), cap - 1); };
    const int block_end = min(upto, last_seen(f0 + R) + 1), n_it = kvp_uniform(block_end > from ? (block_end - from + 32 * PG - 1) / (32 * PG) : 0);
    const int end = kvp_uniform(fw < n_flat ? min(upto, last_seen(fw + 32) + 1) : from);      // this wave's
    const int all_see = kvp_uniform(fw < n_flat ? sq.p0 + (int)(fw / (unsigned)a.G) : -1);    // what its first row sees

    // ---- a stage: each wave of the group loads 32 / RW positions of K and of V
    uint32_t src[NL];
#pragma unroll
    for (int i = 0; i < NL; i++) {
        const int r = 32 / RW * wid + RPL * i + lane / PR, n = (lane % PR) ^ kvp_place<HD>(r & 15);
        src[i] = (uint32_t)((r & 15) * ROW + 16 * n);                // within a half of the tile
    }
    // the group's tiles; past its last one, that again: nothing sees it
    auto base_of = [&](int it) { return min(from + 32 * (PG * min(it, n_it - 1) + grp), (block_end - 1) & ~31); };
    const uint32_t page_bytes = (uint32_t)(a.s.Hkv << a.s.shift) * ROW, head_bytes = (uint32_t)(h << a.s.shift) * ROW;
    const char *const k_head = reinterpret_cast<const char *>(a.kp) + head_bytes, *const v_head = reinterpret_cast<const char *>(a.vp) + head_bytes;
    auto issue = [&](int slot, int base, KvpIds ids) {
        const int half = wid / (RW / 2);
        const uint64_t at = (uint64_t)(uint32_t)max(half ? ids.id[1] : ids.id[0], 0) * page_bytes + (uint32_t)(((base + 16 * half) & ((1 << a.s.shift) - 1)) * ROW);
        char *to = ring + slot + 1024 * NL * wid;
        const char *k_from = k_head + kvp_uniform((int64_t)at), *v_from = v_head + kvp_uniform((int64_t)at);
#pragma unroll
        for (int i = 0; i < NL; i++) lds_dma16_s(k_from, src[i], to + 1024 * i);
#pragma unroll
        for (int i = 0; i < NL; i++) lds_dma16_s(v_from, src[i], to + TB + 1024 * i);
    };
    KvpTable table(a, sg.table, n_it > 0 ? from : 0);
    KvpIds ids;
    if (n_it > 0) {
        ids = table.at(a, base_of(0));
        issue(0, base_of(0), ids);
    }

    // ---- the queries
    // a negative scale is the queries', a zero one makes them zero
    const float kc = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * 1.4426950408889634f, sign = a.scale == 0.0f ? 0.0f : a.scale < 0.0f ? -1.0f : 1.0f;
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
        for (int e = 0; e < 8; e++) x[e] *= sign;
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
    // where this lane reads in a stage: piece 2 i + hf of position c of K, half of piece 4 t + v_p of V's position 4 hf + v_r
    const int v_r = (lane >> 2) & 3, v_p = 2 * ((lane >> 4) & 1) + (lane & 1);
    int k_low = 16 * (hf ^ kvp_place<HD>(c & 15)), v_low = 16 * (v_p ^ kvp_place<HD>(4 * hf + v_r)) + 8 * ((lane >> 1) & 1);
    const int k_row = (int)(ring - smem) + c * ROW, v_row = (int)(ring - smem) + TB + (4 * hf + v_r) * ROW;
    int stage = 0;
    for (int it = 0; it < n_it; it++) {
        wait_vmcnt<0>();                                         // this wave's loads of the stage have landed
        __syncthreads();                                         // ... and every wave's; the other stage is free
        const KvpIds now = ids;
        ids = table.at(a, base_of(it + 1));
        const int ks = k_row + stage, vs = v_row + stage;
        asm volatile("" : "+v"(k_low), "+v"(v_low));             // kept over the turns the 16 addresses take registers that there are none of
        stage ^= 2 * TB;
        issue(stage, base_of(it + 1), ids);
        const int base = from + 32 * (PG * it + grp);
        if (base >= end) continue;
        // the tile's K first, all of it, and V as early as registers are free: LDS answers late
        bf16x8 k[KC];
#pragma unroll
        for (int i = 0; i < KC; i++) k[i] = *reinterpret_cast<const bf16x8 *>(smem + ((k_low ^ (32 * i)) + ks));
        uint2 v[2][DV][2];
        auto load_v = [&](int x) {
#pragma unroll
            for (int t = 0; t < DV; t++)
#pragma unroll
                for (int y = 0; y < 2; y++) v[x][t][y] = kvp_turned(smem + ((v_low ^ (64 * t + 32 * y)) + vs) + (16 * x + 8 * y) * ROW);
        };
        asm volatile("" ::: "memory");
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < KC; i++)
#pragma unroll
            for (int t = QT - 1; t >= 0; t--) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[i], q[t][i], s, 0, 0, 0);
        load_v(0);
        const bool edge = base + 31 > all_see || base + 32 > end || (now.id[0] | now.id[1]) < 0;
        if (edge) {
            const int upto_r = min(lim, end - 1) - base - 4 * hf;
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = 8 * (r >> 2) + (r & 3) <= upto_r && now.id[r >> 3] >= 0 ? s[r] : KVP_NEG_INF;
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
            if (x == 0) load_v(1);
            if (edge) {
                // V of positions that no row here sees may hold anything
                const int left = now.id[x] >= 0 ? end - base - 16 * x - 4 * hf : 0;
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const uint32_t m0 = (left > 8 * y ? 0xffffu : 0u) | (left > 8 * y + 1 ? 0xffff0000u : 0u);
                    const uint32_t m1 = (left > 8 * y + 2 ? 0xffffu : 0u) | (left > 8 * y + 3 ? 0xffff0000u : 0u);
#pragma unroll
                    for (int t = 0; t < DV; t++) v[x][t][y] = make_uint2(v[x][t][y].x & m0, v[x][t][y].y & m1);
                }
            }
#pragma unroll
            for (int t = 0; t < DV; t++) {
                const bf16x8 vt = __builtin_bit_cast(bf16x8, make_uint4(v[x][t][0].x, v[x][t][0].y, v[x][t][1].x, v[x][t][1].y));
#pragma unroll
                for (int y = PT - 1; y >= 0; y--) o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vt, p[y], o[t], 0, 0, 0);
            }
        }
    }
    wait_vmcnt<0>();                                             // no load may land in LDS after the block ends
    // sums that are not finite, or no score where positions are seen (or would be, on pages that are none): again, row by row
    float z = l * 0.0f;
#pragma unroll
    for (int t = 0; t < DV; t++)
#pragma unroll
        for (int r = 0; r < 16; r++) z = fmaf(o[t][r], 0.0f, z);
    l = xhalf_sum(l);
    const int first = from + 32 * grp;
    if (first < end && __any(live && (z != 0.0f || (m == KVP_NEG_INF && lim >= first)))) {
        float om[HD / 2 + 2];
        attn_kvp_again<BF16, HD, 32>(a, sg, h, q_at, live, lim, first, end, 32 * PG, a.scale * 1.4426950408889634f, om);
#pragma unroll
        for (int t = 0; t < DV; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[t][r] = om[16 * t + r];
        m = om[HD / 2];
        l = om[HD / 2 + 1];
    }
    // the groups' sums, in order, into the first's: every lane's from the same lane of the others
    if (PG > 1) __syncthreads();
    float *const join = reinterpret_cast<float *>(smem) + lane;
    auto join_at = [&](int g, int r) -> float & { return join[((g - 1) * RW + wid) * (16 * DV + 2) * 64 + r * 64]; };
    if (grp > 0) {
        join_at(grp, 0) = m;
        join_at(grp, 1) = l;
#pragma unroll
        for (int t = 0; t < DV; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) join_at(grp, 2 + 16 * t + r) = o[t][r];
    }
    if (PG > 1) __syncthreads();
    if (grp > 0 || !live) return;
    if (PG > 1) {
        float mm = m;
#pragma unroll
        for (int g = 1; g < PG; g++) mm = fmaxf(mm, join_at(g, 0));
        const float ref = mm == KVP_NEG_INF ? 0.0f : mm, own = __builtin_amdgcn_exp2f(m - ref);
        l *= own;
#pragma unroll
        for (int t = 0; t < DV; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[t][r] *= own;
#pragma unroll
        for (int g = 1; g < PG; g++) {
            const float w = __builtin_amdgcn_exp2f(join_at(g, 0) - ref);
            l = fmaf(join_at(g, 1), w, l);
#pragma unroll
            for (int t = 0; t < DV; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[t][r] = fmaf(join_at(g, 2 + 16 * t + r), w, o[t][r]);
        }
        m = mm;
    }
    const float inv = m == KVP_NEG_INF ? 0.0f : 1.0f / l;
    float *part = a.part + (qi * a.so + split) * kvp_part<HD>;
#pragma unroll
    for (int t = 0; t < DV; t++)
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const int d = 32 * t + 16 * x + 8 * hf;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = o[t][8 * x + e];
            if (a.so == 1) {
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] *= inv;
                kvp_store<BF16, 8>(a.out, qi * HD + d, a.vec_o, v);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e += 2) *reinterpret_cast<float2 *>(part + d + e) = make_float2(v[e], v[e + 1]);
            }
        }
    if (a.so > 1 && hf == 0) *reinterpret_cast<float2 *>(part + HD) = make_float2(m, l);
}

// The parts of each row and head, in order; a wave a head.  4.7 us for 64 rows x 16 heads, bound by its chain of loads: a
// part that has no positions says so by its maximum, -infinity (a part that is NaN has 0), so
// that nothing but the rows' places has to be known, and the first 24 parts are on their way
// with the weights.
template <bool BF16, int HD>
__global__ __launch_bounds__(256) void k_attn_kvp_merge(AttnKvpArgs a) {
    constexpr int E = HD / 64;
    const int lane = threadIdx.x & 63;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = blockIdx.y, i = blockIdx.x, head = blockIdx.z * 4 + wid;
    const KvpRows sq = kvp_rows(a.s, j);
    if (i >= sq.n || head >= a.Hq) return;
    const int P = (a.prefix ? a.sp : 0) + a.so;
    const int64_t qi = (sq.r0 + i) * a.Hq + head;
    const float *part = a.part + qi * P * kvp_part<HD>;
    const float2 ml = *reinterpret_cast<const float2 *>(part + min(lane, P - 1) * kvp_part<HD> + HD);
    float p0[8][E], p1[16][E];
    auto load = [&](auto &p, int x0, int count) {
#pragma unroll
        for (int u = 0; u < count; u++)
#pragma unroll
            for (int e = 0; e < E; e++) p[u][e] = part[min(x0 + u, P - 1) * kvp_part<HD> + E * lane + e];
    };
    load(p0, 0, 8);
    if (P > 16) load(p1, 8, 16);
    else if (P > 8) load(p1, 8, 8);
    const float mx = lane < P ? ml.x : KVP_NEG_INF;
    const float mm = wave_max_f32(mx);
    const float w = mx == KVP_NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(mx - mm);
    const float ll = wave_sum_f32(mx == KVP_NEG_INF ? 0.0f : ml.y * w);
    float v[E];
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = 0.0f;
    auto add = [&](const auto &p, int x0, int count) {
#pragma unroll
        for (int u = 0; u < count; u++) {
            const int x = min(x0 + u, 63);
            const float wx = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), x));
            const bool is = x0 + u < P && __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mx), x)) != KVP_NEG_INF;
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = is ? fmaf(p[u][e], wx, v[e]) : v[e];
        }
    };
    add(p0, 0, 8);
    if (P > 16)
        for (int x0 = 8; x0 < P; x0 += 16) {
            if (x0 > 8) load(p1, x0, 16);
            add(p1, x0, 16);
        }
    else if (P > 8) add(p1, 8, 8);
    const float inv = mm == KVP_NEG_INF ? 0.0f : 1.0f / ll;
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

// splits of `len` positions over blocks that take `step` of them a turn: up to `blocks` of
// them at `units` tiles, each with `turns` turns at least
static void kvp_split(int64_t units, int64_t len, int64_t most, int blocks, int step, int turns, int &s, int &chunk) {
    const int64_t tiles = (len + 31) / 32 + 1;
    const int64_t n = std::max<int64_t>(1, std::min({most, blocks / std::max<int64_t>(1, units), tiles * 32 / (step * turns)}));
    chunk = (int)((tiles + n - 1) / n * 32);
    s = (int)((tiles * 32 + chunk - 1) / chunk);
}

#define KVP_ROWS 64                             // rows x heads of a block's tile
template <bool BF16, int HD, int PG>
static hipError_t go_rows(AttnKvpArgs &a, int64_t units, int turns, int64_t room, hipStream_t st) {
    constexpr int RW = KVP_ROWS / 32;
    const int64_t tiles = (a.s.max_rows * a.G + KVP_ROWS - 1) / KVP_ROWS;
    kvp_split(units, a.max_len, std::max<int64_t>(1, room), 2048 / (RW * PG), 32 * PG, turns, a.so, a.co);
    a.otiles = (int)tiles;
    a.uniform = !a.s.row_start || a.s.n_rows == a.s.n_seq * a.s.max_rows;
    const int64_t blocks = std::min(tiles * a.s.n_seq, a.s.n_rows * a.G / KVP_ROWS + a.s.n_seq) * a.so * a.s.Hkv;
    if (blocks * 64 * RW * PG > UINT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_attn_kvp_rows<BF16, HD, RW, PG>), dim3((unsigned)blocks), dim3(64 * RW * PG), 0, st, a);
    return a.so > 1 ? go_merge<BF16, HD>(a, st) : hipGetLastError();
}

template <bool BF16, int HD, int W, bool ONCE, bool AHEAD>
static hipError_t run_few(const AttnKvpArgs &a, int64_t blocks, hipStream_t st) {
    if (blocks * 64 * W > UINT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_attn_kvp<BF16, HD, W, ONCE, AHEAD>), dim3((unsigned)blocks), dim3(64 * W), 0, st, a);
    return a.prefix || a.so > 1 ? go_merge<BF16, HD>(a, st) : hipGetLastError();
}

template <bool BF16, int HD>
static hipError_t go_few(AttnKvpArgs &a, int64_t room, hipStream_t st) {
    constexpr int R = 16;
    const int64_t otiles = (a.s.max_rows * a.G + R - 1) / R, own = (int64_t)a.s.n_seq * a.s.Hkv * otiles;
    // A prefix read for all members costs a merge and smaller blocks: it has to save 40 MB, counted as if one read were all
    // (every 16 rows x heads read it, most of them from the L2) (us, for all / by every member, 8 KV heads of
    // 128, bf16: 3 x 5 behind 939, 46 MB saved, 11.1 / 13.2, 2 x 19 of four rows behind 231, 34 MB, 13.4 / 9.1, 2 x 2 behind
    // 2877, 24 MB, 15.3 / 13.3; 2 x 27 behind 884 and 1011 of their own, 188 MB, 47 / 51), and short ones are in the
    // L2 for all that have a CU each
    const int64_t all_groups = (a.s.n_seq + a.group - 1) / a.group;
    const bool saves = a.common < 0 || (a.s.n_seq - all_groups) * a.common * a.s.Hkv * HD * 4 >= (int64_t)40 << 20;
    a.prefix = a.prefix && saves && (own > 256 || a.max_len > 640);
    const int64_t n_groups = a.prefix ? all_groups : 0, ptiles = a.prefix ? ((int64_t)a.group * a.s.max_rows * a.G + R - 1) / R : 0;
    a.otiles = (int)otiles;
    a.ptiles = (int)ptiles;
    a.sp = a.so = 1;
    a.cp = a.co = 1 << 30;
    const int64_t blocks_pre = n_groups * ptiles * a.s.Hkv;
    if (!a.prefix) {
        if (a.max_len > 512) kvp_split(own, a.max_len, room, 256, 256, 1, a.so, a.co);
        // Eight waves a block where every block has a CU of its own, or long to go; else four, and two of short contexts, as
        // waves and the LDS of their parts are what blocks wait for.  us, eight / four / two, 8 KV heads x 2 heads of 128, bf16,
        // sequences of half to all of the positions named (with weights of two terms; three add at most 0.4 us):
        // 48 sequences of 60 positions 10.3 / 6.8 / -, 250 of 120 46.2 / 25.1 / 24.1, of 500 77 / 67 / 72, 1000 of 32 141 / 53 /
        // 37, of 250 199 / 141 / 131, 128 of 4000 252 / 266 / 252.  (One wave: 1000 of 32 bf16 37.0, f32 48.5 against 48.0; 250 of
        // 1000 f32 150 / 144 with two / 132 with four.)
        const int w = own <= 256 || a.max_len > 2048 ? 8 : own <= 1024 || a.max_len > 384 ? 4 : 2;
        // K and V past the caches where there is more of them than those hold (250 of 250, 256 MB, two waves 43.2 / 39.7 us;
        // 64 of 500, 131 MB, 20.9 / 21.2; eight waves, which else ask for a tile ahead, 14 of 3786, 217 MB, 36.0 / 37.5)
        const bool once = otiles == 1 && (int64_t)a.s.n_seq * a.max_len * a.s.Hkv * HD * 4 >= (int64_t)(w == 8 ? 256 : 192) << 20;
        const int64_t blocks = own * a.so;
        if (w == 8) return once ? run_few<BF16, HD, 8, true, false>(a, blocks, st) : run_few<BF16, HD, 8, false, true>(a, blocks, st);
        if (w == 4) return once ? run_few<BF16, HD, 4, true, false>(a, blocks, st) : run_few<BF16, HD, 4, false, false>(a, blocks, st);
        return once ? run_few<BF16, HD, 2, true, false>(a, blocks, st) : run_few<BF16, HD, 2, false, false>(a, blocks, st);
    }
    kvp_split(own, a.max_own, room / 2, 768, 128, 1, a.so, a.co);
    // 128 positions a part at least, of long prefixes 256: parts cost the merge (5 behind 5204, 8 heads of 64, 21.4 -> 15.9 us)
    kvp_split(blocks_pre, a.max_len, room - a.so, (int)std::max<int64_t>(768 - own * a.so, 256), 128, a.max_len > 1024 ? 2 : 1, a.sp, a.cp);
    return run_few<BF16, HD, 4, false, false>(a, blocks_pre * a.sp + own * a.so, st);
}

template <bool BF16, int HD>
static hipError_t go_attn_kvp(AttnKvpArgs &a, int64_t room, hipStream_t st) {
    const int64_t rows = a.s.max_rows * a.G;
    if (rows <= 32) return go_few<BF16, HD>(a, room, st);
    // Tiles, by the rows there are: sequences shorter than max_rows leave some empty, counted is half a one a sequence
    const int64_t tiles = (rows + KVP_ROWS - 1) / KVP_ROWS * a.s.n_seq, full = a.s.n_rows * a.G * 2 / KVP_ROWS;
    const int64_t units = (a.s.n_rows >= a.s.n_seq * a.s.max_rows ? tiles : std::min(tiles, (full + a.s.n_seq) / 2 + 1)) * a.s.Hkv;
    // Four groups over the positions, one block a CU, or two and two blocks.  Four are for contexts that two would take long
    // over, where the tiles are one a CU at most and many enough that the parts of splits cost more; and for one prompt
    // with a bit more tiles, whose last ones see twice as much as its middle one.  us, two (not split) / four, 8 KV heads
    // x 2 heads of 128, behind half to all of what is named, bf16: 5 x 137 rows of 350 positions 13.7 / 13.8, of 600 17.8 /
    // 16.8; f32: 32 x 20 behind 1000 40.5 / 34.2, 2 x 512 behind 4000 105 / 96, 404 alone 16.8 / 17.2, 1337 alone 38.7 /
    // 35.2, 1750 alone 50.7 / 49.4; 2 x 900 alone 31.6 / 38.8, 6 x 404 20.2 / 27.7, 4 x 350 behind 1500 103 / 118, 8 x 512
    // behind 4000 317 / 338.  Fewer tiles, two (split) / four: bf16 1 x 200 behind 800 18.5 / 19.6, 2 x 137 behind 500 19.2 /
    // 15.9, 3 x 137 behind 8000 58 / 61; f32 2 x 137 behind 800 23.2 / 26.7, 1 x 400 behind 500 28.7 / 24.8.  A split of many
    // tiles has to save more than one of few (5 x 137 of 450, bf16, two groups: 25.7, not split 15.5; 1 x 67 behind 900: 15.1,
    // not split 18.8).  (Four side by side, two groups: 8 x 512 2% slower, but six ragged prompts of 1337 by 18%.)
    const int64_t many = BF16 ? 72 : 96;
    // One group, and four blocks a CU (128 dims), where tiles are more than two blocks a CU and short, or so many that the longest
    // is not what all wait for; and of a single tile of positions.  us, two / one: 16 x 32 rows of 32 positions bf16 7.7 / 6.8, of
    // 130 10.2 / 10.9, 64 x 32 of 32 11.7 / 10.4; bf16 128 x 17 alone 18.7 / 11.9, 500 x 40 alone 147 / 88, 16 x 200 behind
    // 1000 61.7 / 54.8, 8 x 512 behind 4000 214 / 199, 4 x 700 alone 27.0 / 27.6; f32 16 x 200 behind 100 34.1 / 28.4, 8 x 700
    // alone 68.0 / 61.3, 12 x 1000 alone 171 / 156, 16 x 512 behind 4000 634 / 644, 4 x 1000 alone 58.0 / 63.5; dim 64, bf16 128 x
    // 40 behind 1000 79 / 64, 4 x 1000 alone 22.8 / 29.1
    if (a.max_len <= 32 || (units > 512 && a.max_len <= 320) || units > (BF16 ? 800 : 1200) * (128 / HD)) return go_rows<BF16, HD, 1>(a, units, 8, room, st);
    const bool prompt = a.s.n_seq == 1 && a.max_len <= 2 * a.s.max_rows;
    if (units >= many && units <= (prompt ? 400 : 256) && a.max_len > 512 && (units >= 128 || a.max_len <= 4096))
        return go_rows<BF16, HD, 4>(a, units, 4, room, st);
    return go_rows<BF16, HD, 2>(a, units, units < many ? 4 : 8, room, st);
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
