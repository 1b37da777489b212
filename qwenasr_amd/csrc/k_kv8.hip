// The int8 KV cache: its write, its reading back and the attention over it.
//
// A block is 64 positions of one head with one scale for K and one for V; 64 is the
// K dimension of v_mfma_i32_16x16x64_i8.  The attention multiplies the cache's
// bytes as they are: scores S^T = K Q^T take K rows [position][dim] as the MFMA's
// rows, and leave position 16 t + 4 g + r of a block in lane group g (lane / 16),
// register r of product t.  The probabilities of one lane are then the 16
// consecutive K bytes that the second product O^T = V^T P^T takes from that lane if
// the bytes of a dim of V stand in the order (g, t, r): V is stored so, a block
// [dim][64], and no value crosses lanes or goes through LDS between the products.
#include "kernels.h"
#include "gemm_common.h"

namespace qasr {

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

// where position p of a block stands among a dim's 64 bytes of V
__device__ __forceinline__ int kv8_slot(int p) { return ((p >> 2) & 3) * 16 + (p >> 4) * 4 + (p & 3); }

struct Kv8Seq {
    int64_t r0;               // first row
    int n;                    // rows
    int p0;                   // position of the first row
};
// the rows and the place of sequence j, held to the buffers
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8Args &a, int j) {
    Kv8Seq s;
    int64_t r1;
    if (a.row_start) {
        s.r0 = min(max((int64_t)a.row_start[j], (int64_t)0), a.n_rows);
        r1 = min(max((int64_t)a.row_start[j + 1], s.r0), a.n_rows);
    } else {
        s.r0 = min((int64_t)j * a.max_rows, a.n_rows);
        r1 = min(s.r0 + a.max_rows, a.n_rows);
    }
    s.n = (int)min(r1 - s.r0, a.max_rows);
    s.p0 = min(max(a.pos[j], -(1 << 30)), 1 << 30);
    return s;
}

template <bool BF16>
__device__ __forceinline__ void kv8_load16(const void *base, int64_t at, bool vec, float *v) {
    if (BF16) {
        const uint16_t *p = reinterpret_cast<const uint16_t *>(base) + at;
        if (vec) {
            const u16x8 u0 = reinterpret_cast<const u16x8 *>(p)[0], u1 = reinterpret_cast<const u16x8 *>(p)[1];
#pragma unroll
            for (int i = 0; i < 8; i++) { v[i] = bf16_to_f32(u0[i]); v[8 + i] = bf16_to_f32(u1[i]); }
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) v[i] = bf16_to_f32(p[i]);
        }
    } else {
        const float *p = reinterpret_cast<const float *>(base) + at;
        if (vec) {
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const f32x4 u = reinterpret_cast<const f32x4 *>(p)[c];
#pragma unroll
                for (int i = 0; i < 4; i++) v[4 * c + i] = u[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) v[i] = p[i];
        }
    }
}

// 16 bytes of a row: 8 bf16 or 4 f32 values
template <bool BF16>
__device__ __forceinline__ void kv8_load(const void *base, int64_t at, bool vec, float *v) {
    if (BF16) {
        const uint16_t *p = reinterpret_cast<const uint16_t *>(base) + at;
        u16x8 u;
        if (vec) {
            u = *reinterpret_cast<const u16x8 *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) u[i] = p[i];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = bf16_to_f32(u[i]);
    } else {
        const float *p = reinterpret_cast<const float *>(base) + at;
        f32x4 u;
        if (vec) {
            u = *reinterpret_cast<const f32x4 *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) u[i] = p[i];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = u[i];
    }
}
template <bool BF16>
__device__ __forceinline__ void kv8_store(void *base, int64_t at, bool vec, const float *v) {
    if (BF16) {
        uint16_t *p = reinterpret_cast<uint16_t *>(base) + at;
        u16x8 u;
#pragma unroll
        for (int i = 0; i < 8; i++) u[i] = __builtin_bit_cast(uint16_t, (__bf16)v[i]);
        if (vec) {
            *reinterpret_cast<u16x8 *>(p) = u;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) p[i] = u[i];
        }
    } else {
        float *p = reinterpret_cast<float *>(base) + at;
        if (vec) {
            *reinterpret_cast<f32x4 *>(p) = f32x4{v[0], v[1], v[2], v[3]};
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = v[i];
        }
    }
}

__device__ __forceinline__ bool kv8_finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// A block's scale as its values meet it.  A multiple x / s is formed in f32, off by at
// most 2^-23 of itself, and decided exactly in f64 where that could matter: within
// 1e-4 of a half, and at scales whose inverse f32 does not hold well.  (The write of 8
// ragged prompts of up to 1337 bf16 rows, 8 heads of 128: 15 - 17 us, 17 - 20 with every
// value decided in f64.)
struct Kv8Scale {
    double s, inv;
    float inv_f;
    bool tiny;
    __device__ __forceinline__ explicit Kv8Scale(float sc)
        : s((double)sc), inv(sc > 0.0f ? 1.0 / (double)sc : 0.0), inv_f((float)inv), tiny(sc < 1e-30f) {}
    // 4 values' bytes: NaN 0, infinities +-127, everything 0 at scale 0
    __device__ __forceinline__ uint32_t round4(float x0, float x1, float x2, float x3) const {
        const float x[4] = {x0, x1, x2, x3};
        // 1.5 x 2^23: a sum's low byte is the nearest whole number's
        const float big = 12582912.0f;
        uint32_t n[4];
        bool near = tiny;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float u = x[i] * inv_f, t = u + big;
            n[i] = __float_as_uint(t);
            near |= !(fabsf(u - (t - big)) <= 0.4999f);          // also what is not finite
        }
        if (near) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int k = s == 0.0 || x[i] != x[i] ? 0 : kv8_finite(x[i]) ? round_ratio((double)fabsf(x[i]), s, inv) : 127;
                n[i] = (uint32_t)(x[i] < 0.0f ? -k : k);
            }
        }
        const uint32_t a = __builtin_amdgcn_perm(n[1], n[0], 0x0c0c0400), b = __builtin_amdgcn_perm(n[3], n[2], 0x04000c0c);
        return a | b;
    }
    // an earlier value q at scale `old`
    __device__ __forceinline__ int again(int q, double old) const {
        const int k = round_ratio((double)abs(q) * old, s, inv);
        return q < 0 ? -k : k;
    }
};

// How a block's 64 x HD values meet its 256 threads, in the write and the read: a
// thread has E consecutive dims (16 bytes of a row) of 4 consecutive positions 4 m ..
// 4 m + 3, for IT values of m.  A row is LPR lanes wide, so loads and stores cover whole
// rows; the 4 positions of one dim are one word of V's block.
template <bool BF16, int HD>
struct Kv8Map {
    static constexpr int E = BF16 ? 8 : 4, LPR = HD / E, RG = 256 / LPR, IT = RG < 16 ? 16 / RG : 1;
    int d, m0;
    __device__ __forceinline__ Kv8Map(int t) : d(t % LPR * E), m0(t / LPR) {}
    __device__ __forceinline__ int m(int i) const { return m0 + i * RG; }      // 16 and more: nothing
    // word of V's [dim][16 words] that holds positions 4 m .. 4 m + 3
    __device__ __forceinline__ static int word(int m) { return (m & 3) * 4 + (m >> 2); }
};
// V's block in LDS: rows of 17 words, for dims that lie LPR lanes apart
#define KV8_ROW 17

__device__ __forceinline__ uint32_t pack_bytes(const int *q) { return (uint32_t)pack4_i8(q[0], q[1], q[2], q[3]); }

// ---------------------------------------------------------------------------
// write: one block of 256 threads per (block of the sequence, head, sequence, K or V)
// ---------------------------------------------------------------------------
template <bool BF16, int HD>
__global__ __launch_bounds__(256) void k_kv8_write(Kv8Args a) {
    typedef Kv8Map<BF16, HD> Map;
    constexpr int E = Map::E, IT = Map::IT;
    __shared__ float red[4];
    __shared__ uint32_t tile[HD * KV8_ROW];
    const int t = threadIdx.x, lane = t & 63, wid = t >> 6;
    const bool is_v = blockIdx.z & 1;
    const int j = blockIdx.z >> 1, h = blockIdx.y;
    const Kv8Seq sq = kv8_seq(a, j);
    const int first = max(sq.p0, 0), end = min(sq.p0 + sq.n, a.cap);
    const int b = first / 64 + blockIdx.x;
    const int lo = max(first, b * 64), hi = min(end, b * 64 + 64);
    if (lo >= hi) return;
    const int64_t head = (int64_t)j * a.Hkv + h, blk = head * (a.cap / 64) + b;
    const void *src = is_v ? a.v : a.k;
    float *sp = (is_v ? a.vs : a.ks) + blk;
    int8_t *dst = (is_v ? a.v8 : a.k8) + blk * 64 * HD;
    const int keep = lo - b * 64, upto = hi - b * 64;            // positions held before, and behind the new ones
    const Map map(t);
    float x[IT][4][E];
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < IT; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int p = 4 * map.m(i) + r;
            if (p < keep || p >= upto) continue;                 // upto <= 64: m past 15 has none
            kv8_load<BF16>(src, (sq.r0 + (b * 64 + p - sq.p0)) * a.ld + h * HD + map.d, a.vec, x[i][r]);
#pragma unroll
            for (int e = 0; e < E; e++) m = fmaxf(m, fabsf(x[i][r][e]));     // NaN does not count
        }
    const float s_old = keep > 0 ? *sp : 0.0f;
    m = wave_max_f32(m);
    if (lane == 0) red[wid] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    if (!kv8_finite(m)) {                                        // nor do infinities
        m = 0.0f;
#pragma unroll
        for (int i = 0; i < IT; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int p = 4 * map.m(i) + r;
                if (p < keep || p >= upto) continue;
#pragma unroll
                for (int e = 0; e < E; e++) m = kv8_finite(x[i][r][e]) ? fmaxf(m, fabsf(x[i][r][e])) : m;
            }
        m = wave_max_f32(m);
        __syncthreads();
        if (lane == 0) red[wid] = m;
        __syncthreads();
        m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    }
    const float s = fmaxf(s_old, __fdiv_rn(m, 127.0f));
    const Kv8Scale sc(s);
    const bool grow = keep > 0 && s > s_old;
    auto again = [&](int q) { return sc.again(q, (double)s_old); };
    if (t == 0) *sp = s;
    if (!is_v) {
#pragma unroll
        for (int i = 0; i < IT; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int p = 4 * map.m(i) + r;
                uint32_t *o = reinterpret_cast<uint32_t *>(dst + p * HD + map.d);
                if (p >= keep && p < upto) {
#pragma unroll
                    for (int w = 0; w < E / 4; w++)
                        o[w] = sc.round4(x[i][r][4 * w], x[i][r][4 * w + 1], x[i][r][4 * w + 2], x[i][r][4 * w + 3]);
                } else if (p < keep && grow) {
#pragma unroll
                    for (int w = 0; w < E / 4; w++) {
                        const int v = (int)o[w], q[4] = {again((int8_t)v), again((int8_t)(v >> 8)), again((int8_t)(v >> 16)), again(v >> 24)};
                        o[w] = pack_bytes(q);
                    }
                }
            }
        return;
    }
    // V.  A few positions into a block that stays at its scale: their bytes alone
    if (!grow && upto - keep <= 4) {
#pragma unroll
        for (int i = 0; i < IT; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int p = 4 * map.m(i) + r;
                if (p < keep || p >= upto) continue;
#pragma unroll
                for (int w = 0; w < E / 4; w++) {
                    const uint32_t q = sc.round4(x[i][r][4 * w], x[i][r][4 * w + 1], x[i][r][4 * w + 2], x[i][r][4 * w + 3]);
#pragma unroll
                    for (int e = 0; e < 4; e++) dst[(map.d + 4 * w + e) * 64 + kv8_slot(p)] = (int8_t)(q >> (8 * e));
                }
            }
        return;
    }
    // else the stored block through LDS, where rows become words of a dim
    const bool part = keep > 0 || upto < 64;
    if (part) {
        for (int i = t; i < HD * 16; i += 256) tile[(i >> 4) * KV8_ROW + (i & 15)] = reinterpret_cast<const uint32_t *>(dst)[i];
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < IT; i++) {
        const int mm = map.m(i);
        if (mm >= 16 || 4 * mm >= upto || (!grow && 4 * mm + 3 < keep)) continue;
#pragma unroll
        for (int e = 0; e < E; e++) {
            uint32_t *w = &tile[(map.d + e) * KV8_ROW + Map::word(mm)];
            if (4 * mm >= keep && 4 * mm + 3 < upto) {           // all new
                *w = sc.round4(x[i][0][e], x[i][1][e], x[i][2][e], x[i][3][e]);
                continue;
            }
            const int v = (int)*w;                               // a whole block has none of these
            int q[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int p = 4 * mm + r, was = (int8_t)(v >> (8 * r));
                if (p >= upto) q[r] = was;
                else if (p >= keep) q[r] = (int8_t)sc.round4(x[i][r][e], 0.0f, 0.0f, 0.0f);
                else q[r] = grow ? again(was) : was;
            }
            *w = pack_bytes(q);
        }
    }
    __syncthreads();
    for (int i = t; i < HD * 16; i += 256) reinterpret_cast<uint32_t *>(dst)[i] = tile[(i >> 4) * KV8_ROW + (i & 15)];
}

template <bool BF16>
static hipError_t go_kv8_write(const Kv8Args &a, dim3 grid, hipStream_t st) {
    if (a.hd == 128) hipLaunchKernelGGL((k_kv8_write<BF16, 128>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_kv8_write<BF16, 64>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

// rows that 16-byte loads or stores can take
static int kv8_vec(const void *k, const void *v, int64_t ld, int es) {
    return ((uintptr_t)k | (uintptr_t)v) % 16 == 0 && (ld * es) % 16 == 0;
}

// blocks of 64 positions that max_rows rows from any position can touch
static int64_t kv8_blocks(const Kv8Args &a) { return std::min<int64_t>((a.max_rows + 62) / 64 + 1, a.cap / 64); }

hipError_t launch_kv8_write(const Kv8Args &a0, bool bf16, hipStream_t st) {
    Kv8Args a = a0;
    if ((a.hd != 64 && a.hd != 128) || a.n_seq > 32767 || a.Hkv > 65535) return hipErrorInvalidValue;
    a.vec = kv8_vec(a.k, a.v, a.ld, bf16 ? 2 : 4);
    const dim3 grid((unsigned)kv8_blocks(a), (unsigned)a.Hkv, (unsigned)(2 * a.n_seq));
    return bf16 ? go_kv8_write<true>(a, grid, st) : go_kv8_write<false>(a, grid, st);
}

// ---------------------------------------------------------------------------
// read: one block of 256 threads per (block of the sequence, head, sequence, K or V)
// ---------------------------------------------------------------------------
template <bool BF16, int HD>
__global__ __launch_bounds__(256) void k_kv8_read(Kv8Args a) {
    typedef Kv8Map<BF16, HD> Map;
    constexpr int E = Map::E, IT = Map::IT;
    __shared__ uint32_t tile[HD * KV8_ROW];
    const int t = threadIdx.x;
    const bool is_v = blockIdx.z & 1;
    const int j = blockIdx.z >> 1, h = blockIdx.y;
    const Kv8Seq sq = kv8_seq(a, j);
    const int first = max(sq.p0, 0), end = min(sq.p0 + sq.n, a.cap);
    const int b = first / 64 + blockIdx.x;
    const int lo = max(first, b * 64) - b * 64, hi = min(end, b * 64 + 64) - b * 64;
    if (lo >= hi) return;
    const int64_t head = (int64_t)j * a.Hkv + h, blk = head * (a.cap / 64) + b;
    const int8_t *src = (is_v ? a.v8 : a.k8) + blk * 64 * HD;
    const float s = is_v ? a.vs[blk] : a.ks[blk];
    const Map map(t);
    uint32_t k8[IT][4][E / 4];
    if (is_v) {
        for (int i = t; i < HD * 16; i += 256) tile[(i >> 4) * KV8_ROW + (i & 15)] = reinterpret_cast<const uint32_t *>(src)[i];
        __syncthreads();
    } else {
#pragma unroll
        for (int i = 0; i < IT; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int p = 4 * map.m(i) + r;
                if (p < lo || p >= hi) continue;
#pragma unroll
                for (int w = 0; w < E / 4; w++) k8[i][r][w] = reinterpret_cast<const uint32_t *>(src + p * HD + map.d)[w];
            }
    }
#pragma unroll
    for (int i = 0; i < IT; i++) {
        const int mm = map.m(i);
        if (mm >= 16 || 4 * mm >= hi || 4 * mm + 3 < lo) continue;
        uint32_t v8[E];
        if (is_v) {
#pragma unroll
            for (int e = 0; e < E; e++) v8[e] = tile[(map.d + e) * KV8_ROW + Map::word(mm)];
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int p = 4 * mm + r;
            if (p < lo || p >= hi) continue;
            float x[E];
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int q = is_v ? (int8_t)(v8[e] >> (8 * r)) : (int8_t)(k8[i][r][e >> 2] >> (8 * (e & 3)));
                x[e] = __fmul_rn((float)q, s);
            }
            kv8_store<BF16>(is_v ? a.v : a.k, (sq.r0 + (b * 64 + p - sq.p0)) * a.ld + h * HD + map.d, a.vec, x);
        }
    }
}

template <bool BF16>
static hipError_t go_kv8_read(const Kv8Args &a, dim3 grid, hipStream_t st) {
    if (a.hd == 128) hipLaunchKernelGGL((k_kv8_read<BF16, 128>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_kv8_read<BF16, 64>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_kv8_read(const Kv8Args &a0, bool bf16, hipStream_t st) {
    Kv8Args a = a0;
    if ((a.hd != 64 && a.hd != 128) || a.n_seq > 32767 || a.Hkv > 65535) return hipErrorInvalidValue;
    a.vec = kv8_vec(a.k, a.v, a.ld, bf16 ? 2 : 4);
    const dim3 grid((unsigned)kv8_blocks(a), (unsigned)a.Hkv, (unsigned)(2 * a.n_seq));
    return bf16 ? go_kv8_read<true>(a, grid, st) : go_kv8_read<false>(a, grid, st);
}

// ---------------------------------------------------------------------------
// attention
//
// Per tile of R flattened rows (query rows x heads of the group) and KV head:
// S = scale q.k over blocks of 64 positions with the running maximum and sum of the
// softmax, O += P V, both products on bf16 MFMA with operands that lose nothing:
//   K, V: an int8 value is a bf16 value; the block's scale joins the score's factor
//      (K) and the product's (V)
//   q: bf16 rows as they are, f32 rows in three bf16 terms, which hold all 24 bits
//   p: in three terms for f32 rows (a weight is off by 2^-24 of itself), in two for
//      bf16 rows (2^-17, their output is rounded to 2^-8 of itself)
// The weights are floating point, so small ones beside a large one keep all of their
// bits: where a position with next to nothing in V holds the maximum (a sink), the
// others alone are the result.  (Whole numbers of a block's largest weight, in base-256
// digits on the int8 MFMA, lose them: at 12 behind such a position 64 bf16 weights were
// 0, and f32 ones off by 3e-3.  That was faster, two or three products of half the
// length and no conversion: 1337 f32 rows 26 us, now 35; bf16 21, now 25; 4 x 67
// bf16 rows in a window of 8192 35, now 39, with the merge; one row a sequence as now.)
//
// The sums (O and the weights') count from a reference that moves only when a
// block's maximum is 2^16 above it: in f32 they lose nothing by that, and most
// blocks rescale nothing.
//
// What bounds it: the HBM reads where every sequence has one row.  Where rows share
// the positions, a wave's instructions: 384 vector ones to convert a block's K and V,
// 300 for 32 columns' weights and their terms, 64 for O; beside them 96 (f32) or 48
// matrix ones of 33 cycles, which let a vector one through in only 14 of them.
//
// R = 16: one tile a sequence and head, K and V straight into registers.  R = 32: two
// conversions' worth of tiles share one.  Each of a block's 4 waves takes every 4th
// block of positions, on its own: no barrier before their parts are joined.  K and V
// come through a slot each of the wave in LDS, direct from memory
// (global_load_lds_dwordx4), the next K's loads on their way during the weights and
// the second product, the next V's during the first one.  (Operands loaded straight
// into registers leave the four lanes of a quad in four rows: a 64-byte run is then
// asked for four times over, and 16 KB a tile and block at 5.3 TB/s was the end,
// cached or not.)  Other forms, 1337 f32 rows / 3 x 100 rows behind 8000: tiles of 16
// by two waves that share slots, 39 / 85 us; two tiles of 16 by one wave on 16 x 16 x
// 32 products, which hold vector instructions up longer, 41 / 63; the converted blocks
// in LDS for two or four tiles 41 / 74 and 42 / 81; q in four base-256 digits on the
// int8 MFMA, the weights as now, 39 / 67.  With `splits` > 1 several blocks share a
// tile's positions; a second launch merges their parts.
// ---------------------------------------------------------------------------

// 4 int8 values as bf16, which holds each: the upper halves of their floats
__device__ __forceinline__ void kv8_bf16(int w, uint32_t *o) {
    const float f0 = (float)(int8_t)w, f1 = (float)(int8_t)(w >> 8), f2 = (float)(int8_t)(w >> 16), f3 = (float)(w >> 24);
    o[0] = __builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), 0x07060302);
    o[1] = __builtin_amdgcn_perm(__float_as_uint(f3), __float_as_uint(f2), 0x07060302);
}
// 16 of them: the operands of two products
__device__ __forceinline__ void kv8_operand(i32x4 v, bf16x8 *o) {
    uint32_t d[8];
#pragma unroll
    for (int i = 0; i < 4; i++) kv8_bf16(v[i], d + 2 * i);
    o[0] = __builtin_bit_cast(bf16x8, make_uint4(d[0], d[1], d[2], d[3]));
    o[1] = __builtin_bit_cast(bf16x8, make_uint4(d[4], d[5], d[6], d[7]));
}
// 8 values in T bf16 terms, each the nearest to what the ones before it leave
template <int T>
__device__ __forceinline__ void kv8_terms(const float *x, bf16x8 *o) {
    if constexpr (T == 3) {
        split3(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]), o);
    } else {
        uint32_t c0, c1, hi[4], lo[4];                         // the residuals as split3 forms them
        if (T == 2) {
            asm("s_mov_b32 %0, 0xbf80" : "=s"(c0));
            asm("s_mov_b32 %0, 0xbf800000" : "=s"(c1));
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            hi[e] = cvt_pk_bf16(x[2 * e], x[2 * e + 1]);
            if (T == 2) {
                const bf16x2 h = __builtin_bit_cast(bf16x2, hi[e]);
                lo[e] = cvt_pk_bf16(__builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, c0), x[2 * e], false),
                                    __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, c1), x[2 * e + 1], false));
            }
        }
        o[0] = __builtin_bit_cast(bf16x8, make_uint4(hi[0], hi[1], hi[2], hi[3]));
        if (T == 2) o[T - 1] = __builtin_bit_cast(bf16x8, make_uint4(lo[0], lo[1], lo[2], lo[3]));
    }
}

// 4 output values of flattened row f, dims d .. d + 3, from O and the weights' sum
template <bool BF16, int HD>
__device__ __forceinline__ void kv8_put(const AttnKv8Args &a, const Kv8Seq &sq, int h, unsigned f, int d, f32x4 v, float l) {
#pragma unroll
    for (int r = 0; r < 4; r++) v[r] = l == 0.0f ? 0.0f : __fdiv_rn(v[r], l);
    const unsigned qi = f / (unsigned)a.G, qg = f - qi * (unsigned)a.G;
    const int64_t at = ((sq.r0 + qi) * a.Hq + (int64_t)h * a.G + qg) * HD + d;
    if (BF16) {
        typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
        u16x4 u;
#pragma unroll
        for (int r = 0; r < 4; r++) u[r] = __builtin_bit_cast(uint16_t, (__bf16)v[r]);
        uint16_t *p = reinterpret_cast<uint16_t *>(a.out) + at;
        if (a.vec_o) {
            *reinterpret_cast<u16x4 *>(p) = u;
        } else {
#pragma unroll
            for (int r = 0; r < 4; r++) p[r] = u[r];
        }
    } else {
        float *p = reinterpret_cast<float *>(a.out) + at;
        if (a.vec_o) {
            *reinterpret_cast<f32x4 *>(p) = v;
        } else {
#pragma unroll
            for (int r = 0; r < 4; r++) p[r] = v[r];
        }
    }
}

// one split's part of 16 rows in the scratch area: maxima and sums [2][16], then O [16][HD]
template <int HD> constexpr int kv8_part = 32 + 16 * HD;
#define KV8_WAVES 4           // of a block: each takes every 4th block of positions

// The products of an R x R tile.  Lane l has column l % R; with g = l / R and NG = 64 / R such groups it gives the 8 values
// of its group to the K dimension and receives rows 4 NG (i / 4) + 4 g + i % 4.
template <int R> struct Kv8Mfma;
template <> struct Kv8Mfma<16> {
    typedef f32x4 Acc;
    __device__ __forceinline__ static Acc mul(bf16x8 a, bf16x8 b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    __device__ __forceinline__ static float max(float v) { return xhalf_max(xrow16_max(v)); }      // over the groups
    __device__ __forceinline__ static float sum(float v) { return xhalf_sum(xrow16_sum(v)); }
};
template <> struct Kv8Mfma<32> {
    typedef float Acc __attribute__((ext_vector_type(16)));
    __device__ __forceinline__ static Acc mul(bf16x8 a, bf16x8 b, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    __device__ __forceinline__ static float max(float v) { return xhalf_max(v); }
    __device__ __forceinline__ static float sum(float v) { return xhalf_sum(v); }
};

template <bool BF16, int HD, int R>
__global__ __launch_bounds__(64 * KV8_WAVES, 2) void k_attn_kv8(AttnKv8Args a) {
    typedef Kv8Mfma<R> Mfma;
    constexpr bool LDS = R == 32;
    constexpr int PG = KV8_WAVES, NG = 64 / R, NA = R * R / 64, TB = 64 * HD, NL = TB / 1024;   // TB: bytes of a block; NL: loads of it into LDS
    constexpr int KT = 64 / R, KM = HD / (16 * NG), VT = HD / R, VM = 4 / NG;   // tiles of positions and dims; 16-byte operands of each
    constexpr int QT = BF16 ? 1 : 3, PT = BF16 ? 2 : 3;        // terms of q and of the weights
    constexpr int MERGE = PG * R * (HD + 4) * 4, SLOTS = LDS ? PG * 2 * TB : 0;
    __shared__ __attribute__((aligned(16))) char smem[MERGE > SLOTS ? MERGE : SLOTS];
    __shared__ float ml_l[PG][2][R];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane % R, g = lane / R;
    // Heads fastest: with 8 of them each XCD (blocks go to the 8 in turn) has one head's cache in its L2.  Tiles from
    // the longest on, but the `first` shortest ahead of all
    const int j = blockIdx.y, S = a.splits;
    const unsigned rest = blockIdx.x / (unsigned)a.c.Hkv;
    const int h = blockIdx.x - rest * a.c.Hkv, tx = rest / (unsigned)S, split = rest - tx * S;
    const int tile = tx < a.first ? tx : a.tiles - 1 - (tx - a.first);
    const Kv8Seq sq = kv8_seq(a.c, j);
    // flattened rows: fewer than 2^30 (the entry point)
    const unsigned n_flat = (unsigned)sq.n * (unsigned)a.G, f0 = (unsigned)tile * R;
    if (f0 >= n_flat) return;
    const unsigned f1 = n_flat - 1, fr = min(f0 + c, f1);      // a column past the last row repeats it
    const int i_lo = (int)(f0 / (unsigned)a.G), i_hi = (int)(min(f0 + R - 1, f1) / (unsigned)a.G);
    const int last = sq.p0 + (int)(fr / (unsigned)a.G);        // this column's own position, and its window's first
    auto low_of = [&](int i) { return a.window > 0 ? (int)min(max((int64_t)a.c.pos[j] + i - a.window + 1, (int64_t)0), (int64_t)1 << 30) : 0; };
    const int low = low_of((int)(fr / (unsigned)a.G)), low_hi = low_of(i_hi);

    // the blocks that some row of the tile sees: the sinks' and the window's; this split's run of them
    const int hi_pos = min(sq.p0 + i_hi, a.c.cap - 1), lo_blk = low_of(i_lo) / 64, n_sink = min((a.sinks + 63) / 64, lo_blk);
    const int n_blk = hi_pos < 0 ? 0 : n_sink + max(0, hi_pos / 64 - lo_blk + 1);
    const int per = n_blk / S, more = n_blk - per * S;         // the first `more` splits take one block more
    const int u0 = split * per + min(split, more), u1 = u0 + per + (split < more ? 1 : 0);
    auto block_of = [&](int u) { return u < n_sink ? u : lo_blk + u - n_sink; };

    const int64_t head = (int64_t)j * a.c.Hkv + h;
    const int8_t *kb = a.c.k8 + head * a.c.cap * HD, *vb = a.c.v8 + head * a.c.cap * HD;
    const float *ks = a.c.ks + head * (a.c.cap / 64), *vs = a.c.vs + head * (a.c.cap / 64);
    int u = u0 + wid;
    // LDS: the wave's own slots of K and V and this lane's bytes of a load, which fills 64 pieces of 16 bytes: 8 rows
    // of 128 bytes (the swizzle repeats every 16 rows) or 16 of 64
    char *kt = smem + wid * 2 * TB, *vt = kt + TB;
    const uint32_t v_src = (lane >> 2) * 64 + 16 * ((lane & 3) ^ lds_swz<64>(lane >> 2));
    const uint32_t k_src[2] = {HD == 64 ? v_src : (lane >> 3) * 128 + 16 * ((lane & 7) ^ lds_swz<128>(lane >> 3)),
                               HD == 64 ? v_src : (lane >> 3) * 128 + 16 * ((lane & 7) ^ lds_swz<128>(8 + (lane >> 3)))};
    auto issue_k = [&](int b) {
#pragma unroll
        for (int i = 0; i < NL; i++) lds_dma16_s(kb + (int64_t)b * TB + 1024 * i, k_src[i & 1], kt + 1024 * i);
    };
    auto issue_v = [&](int b) {
#pragma unroll
        for (int i = 0; i < NL; i++) lds_dma16_s(vb + (int64_t)b * TB + 1024 * i, v_src, vt + 1024 * i);
    };
    // otherwise the operands themselves, loaded again as soon as the products have read them
    i32x4 kr[KT][KM], vr[VT][VM];
    auto load_k = [&](int b) {
        const int8_t *p = kb + (int64_t)b * TB + c * HD + 16 * g;
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int m = 0; m < KM; m++) kr[t][m] = *reinterpret_cast<const i32x4 *>(p + R * t * HD + 16 * NG * m);
    };
    auto load_v = [&](int b) {
        const int8_t *p = vb + (int64_t)b * TB + c * 64 + 16 * g;
#pragma unroll
        for (int t = 0; t < VT; t++)
#pragma unroll
            for (int m = 0; m < VM; m++) vr[t][m] = *reinterpret_cast<const i32x4 *>(p + R * t * 64 + 16 * NG * m);
    };
    float ksl = 0.0f, vsl = 0.0f;                              // lane i: the scales of this wave's block `it` + i
    auto scales = [&]() {
        const int ul = u + lane * PG;
        ksl = ul < u1 ? ks[block_of(ul)] : 0.0f;
        vsl = ul < u1 ? vs[block_of(ul)] : 0.0f;
    };
    auto row_at = [&](unsigned f) {
        const unsigned i = f / (unsigned)a.G;
        return (sq.r0 + i) * a.ldq + (int64_t)(h * a.G + (int)(f - i * (unsigned)a.G)) * HD;
    };

    // The column's row, dims 16 (NG m + g) + 0..15 in x[m], the first blocks and their scales, at once.  LDS: the
    // rows come through the V slots, once a block and by whole rows (a lane's own loads, 64 bytes apart, for all
    // four waves: 1337 rows 44 -> 41 us), piece n of row r at n ^ (r & 15)
    constexpr int ES = BF16 ? 2 : 4, QR = HD * ES, QP = QR / 16, NQ = R * QR / 1024 / PG;
    float x[KM][16];
    const bool by_lds = LDS && a.vec_q;
    if (!by_lds) {
#pragma unroll
        for (int m = 0; m < KM; m++) kv8_load16<BF16>(a.q, row_at(fr) + 16 * (NG * m + g), a.vec_q, x[m]);
    }
    if constexpr (LDS) {
        static_assert(NQ >= 1 && R * QR <= PG * TB, "rows in the V slots");
        auto chunk = [&](int n) { return smem + TB + n / NL * 2 * TB + n % NL * 1024; };
        if (by_lds) {
#pragma unroll
            for (int i = 0; i < NQ; i++) {
                const int n = wid * NQ + i, r = (64 * n + lane) / QP, piece = ((64 * n + lane) % QP) ^ (r & 15 & (QP - 1));
                lds_dma16(reinterpret_cast<const char *>(a.q) + row_at(min(f0 + r, f1)) * ES + 16 * piece, chunk(n));
            }
        }
        if (u < u1) {
            issue_k(block_of(u));
            scales();
        }
        if (by_lds) {
            wait_vmcnt<0>();
            __syncthreads();
#pragma unroll
            for (int m = 0; m < KM; m++)
#pragma unroll
                for (int e = 0; e < ES; e++) {
                    const int at = c * QR + 16 * ((ES * (NG * m + g) + e) ^ (c & 15 & (QP - 1)));
                    const char *p = chunk(at / 1024) + at % 1024;
                    if constexpr (BF16) {
                        const u16x8 v = *reinterpret_cast<const u16x8 *>(p);
#pragma unroll
                        for (int i = 0; i < 8; i++) x[m][8 * e + i] = bf16_to_f32(v[i]);
                    } else {
                        const f32x4 v = *reinterpret_cast<const f32x4 *>(p);
#pragma unroll
                        for (int i = 0; i < 4; i++) x[m][4 * e + i] = v[i];
                    }
                }
            wait_lds();
            __syncthreads();                                   // every wave has its rows
        }
        if (u < u1) issue_v(block_of(u));
    } else if (u < u1) {
        load_k(block_of(u));
        load_v(block_of(u));
        scales();
    }
    __builtin_amdgcn_sched_barrier(0);

    // the row in bf16 terms
    bf16x8 qd[KM][2][QT];
    float qf;                                                  // score = sum x qf x the block's scale
    {
        float m = 0.0f, z = 0.0f;                              // z: NaN after a value that is not finite
#pragma unroll
        for (int k = 0; k < KM; k++)
#pragma unroll
            for (int e = 0; e < 16; e++) { m = fmaxf(m, fabsf(x[k][e])); z = fmaf(x[k][e], 0.0f, z); }
        m = Mfma::max(m);
        z = Mfma::sum(z);
        // rows whose sums f32 might not hold, or whose terms bf16, a power of two nearer to 1
        const int ex = (int)(__float_as_uint(m) >> 23) - 127, sh = z != 0.0f ? 0 : ex > 100 ? ex - 100 : ex < -60 ? ex + 60 : 0;
        const float f = __uint_as_float((uint32_t)(127 - sh) << 23);
        const float to = a.scale < 0.0f ? -f : f;              // the scores' factor is not negative
        if (__any(to != 1.0f)) {
#pragma unroll
            for (int k = 0; k < KM; k++)
#pragma unroll
                for (int e = 0; e < 16; e++) x[k][e] *= to;
        }
#pragma unroll
        for (int k = 0; k < KM; k++)
#pragma unroll
            for (int i = 0; i < 2; i++) kv8_terms<QT>(&x[k][8 * i], qd[k][i]);
        // a row that is not finite: NaN, in its own column alone
        qf = z != 0.0f ? __builtin_nanf("") : fabsf(a.scale) * 1.4426950408889634f * __uint_as_float((uint32_t)(127 + sh) << 23);
    }
    // waited for here and below: a wait at their use would drain the loads in flight in every turn
    asm volatile("" : "+v"(ksl), "+v"(vsl));

    float m = -__builtin_inff(), l = 0.0f;                     // m: what O and l count from
    typename Mfma::Acc o[VT];
#pragma unroll
    for (int t = 0; t < VT; t++)
#pragma unroll
        for (int i = 0; i < NA; i++) o[t][i] = 0.0f;

    for (int it = 0; u < u1; it++, u += PG) {
        if ((it & 63) == 0 && it > 0) {
            scales();
            asm volatile("" : "+v"(ksl), "+v"(vsl));
        }
        // the block behind the last one is the last one again: the waits count the same
        const int b = block_of(u), bn = block_of(min(u + PG, u1 - 1));
        const float ksb = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ksl), it & 63));
        const float vsb = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vsl), it & 63));
        if constexpr (LDS) wait_vmcnt<NL>();                   // K has landed; V's loads are behind it
        __builtin_amdgcn_sched_barrier(0);
        float s[KT * NA];
#pragma unroll
        for (int t = 0; t < KT; t++) {
            typename Mfma::Acc acc;
#pragma unroll
            for (int i = 0; i < NA; i++) acc[i] = 0.0f;
#pragma unroll
            for (int k = 0; k < KM; k++) {
                const int r = R * t + c;
                if constexpr (LDS) kr[t][k] = *reinterpret_cast<const i32x4 *>(kt + r * HD + 16 * ((NG * k + g) ^ lds_swz<HD>(r)));
                bf16x8 kv[2];
                kv8_operand(kr[t][k], kv);
#pragma unroll
                for (int e = QT - 1; e >= 0; e--)
#pragma unroll
                    for (int i = 0; i < 2; i++) acc = Mfma::mul(kv[i], qd[k][i][e], acc);
            }
#pragma unroll
            for (int i = 0; i < NA; i++) s[NA * t + i] = acc[i];
        }
        // one product, then its share of the next operands' conversion: the two run side by side
        constexpr int QN = KT * KM * 2 * QT;
        __builtin_amdgcn_sched_group_barrier(0x100, KT * KM, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 24, 0);
#pragma unroll
        for (int i = 0; i < QN; i++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, KT * KM * 24 / QN, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (LDS) wait_lds();                         // K has been read
        if constexpr (LDS) issue_k(bn);
        else load_k(bn);                                       // a whole block ahead of their use
        __builtin_amdgcn_sched_barrier(0);

        // mb: the block's maximum of what the column sees
        const float kf = ksb * qf;
        float mb, kc = kf;
        bool none = false;
        if (ksb >= 0.0f && b * 64 + 63 <= sq.p0 + i_lo && (b * 64 >= low_hi || b * 64 + 63 < a.sinks)) {
            // every row of the tile sees the whole block, and the largest sum is the largest score
            mb = s[0];
#pragma unroll
            for (int i = 1; i < KT * NA; i++) mb = fmaxf(mb, s[i]);
            mb = Mfma::max(mb) * kf;
        } else {
            mb = -__builtin_inff();
            kc = 1.0f;
#pragma unroll
            for (int i = 0; i < KT * NA; i++) {
                const int at = b * 64 + 4 * NG * (i >> 2) + 4 * g + (i & 3);
                const bool seen = (at <= last) & ((at >= low) | (at < a.sinks));
                s[i] = seen ? s[i] * kf : -__builtin_inff();
                mb = fmaxf(mb, s[i]);
            }
            mb = Mfma::max(mb);
            none = b * 64 > last || (min(b * 64 + 63, last) < low && b * 64 >= a.sinks);
        }
        // a column that sees none of this block takes nothing of it, its scale neither; one whose largest score f32
        // does not hold becomes NaN
        const float vf = none ? 0.0f : vsb;
        kc = none || kv8_finite(mb) ? kc : __builtin_nanf("");
        asm("" : "+v"(kc));                                    // else a select on every weight
        const bool up = mb > m + 16.0f;
        if (__any(up)) {
            const float al = up ? __builtin_amdgcn_exp2f(m - mb) : 1.0f;
            m = up ? mb : m;
            l *= al;
#pragma unroll
            for (int t = 0; t < VT; t++)
#pragma unroll
                for (int i = 0; i < NA; i++) o[t][i] *= al;
        }
        const float ref = m == -__builtin_inff() ? 0.0f : m;
        // the weights in the order of V's bytes: operand k's half i holds those of t = 2 i and 2 i + 1
        bf16x8 pd[VM][2][PT];
#pragma unroll
        for (int k = 0; k < VM; k++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; e++) p[e] = __builtin_amdgcn_exp2f(fmaf(s[4 * (4 / NG * (2 * i + (e >> 2)) + k) + (e & 3)], kc, -ref));
                l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                kv8_terms<PT>(p, pd[k][i]);
            }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (LDS) wait_vmcnt<NL>();                   // V has landed; the next K's loads are behind it
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < VT; t++) {
            typename Mfma::Acc acc;
#pragma unroll
            for (int i = 0; i < NA; i++) acc[i] = 0.0f;
#pragma unroll
            for (int k = 0; k < VM; k++) {
                const int r = R * t + c;
                if constexpr (LDS) vr[t][k] = *reinterpret_cast<const i32x4 *>(vt + r * 64 + 16 * ((NG * k + g) ^ lds_swz<64>(r)));
                bf16x8 vv[2];
                kv8_operand(vr[t][k], vv);
#pragma unroll
                for (int e = PT - 1; e >= 0; e--)
#pragma unroll
                    for (int i = 0; i < 2; i++) acc = Mfma::mul(vv[i], pd[k][i][e], acc);
            }
#pragma unroll
            for (int i = 0; i < NA; i++) o[t][i] = fmaf(acc[i], vf, o[t][i]);
        }
        constexpr int PN = VT * VM * 2 * PT;
        __builtin_amdgcn_sched_group_barrier(0x100, VT * VM, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 24, 0);
#pragma unroll
        for (int i = 0; i < PN; i++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, (VT * VM * 24 + VT * NA) / PN, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (LDS) wait_lds();                         // V has been read
        if constexpr (LDS) issue_v(bn);
        else load_v(bn);
        __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (LDS) wait_vmcnt<0>();                        // no load may land in LDS that the parts use
    l = Mfma::sum(l);

    const int cols = (int)min((unsigned)R, n_flat - f0);
    // the waves' parts of the tile, through the slots
    float (*o_l)[R][HD + 4] = reinterpret_cast<float (*)[R][HD + 4]>(smem);
    __syncthreads();
    if (g == 0) { ml_l[wid][0][c] = m; ml_l[wid][1][c] = l; }
#pragma unroll
    for (int t = 0; t < VT; t++)
#pragma unroll
        for (int i = 0; i < NA; i += 4)
            *reinterpret_cast<f32x4 *>(&o_l[wid][c][R * t + NG * i + 4 * g]) = f32x4{o[t][i], o[t][i + 1], o[t][i + 2], o[t][i + 3]};
    __syncthreads();
    for (int i = threadIdx.x; i < cols * (HD / 4); i += 64 * PG) {
        const int col = i / (HD / 4), d = 4 * (i % (HD / 4));
        float mm = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < PG; w++) mm = fmaxf(mm, ml_l[w][0][col]);
        const float ms = mm == -__builtin_inff() ? 0.0f : mm;
        float ll = 0.0f;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < PG; w++) {
            const float e = __builtin_amdgcn_exp2f(ml_l[w][0][col] - ms);
            ll = fmaf(ml_l[w][1][col], e, ll);
            const f32x4 ow = *reinterpret_cast<const f32x4 *>(&o_l[w][col][d]);
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] = fmaf(ow[r], e, v[r]);
        }
        if (S > 1) {
            const int at = tile * (R / 16) + (col >> 4), cc = col & 15;
            float *part = a.part + ((((int64_t)j * a.c.Hkv + h) * a.tiles * (R / 16) + at) * S + split) * kv8_part<HD>;
            if (d == 0) { part[cc] = mm; part[16 + cc] = ll; }
            *reinterpret_cast<f32x4 *>(part + 32 + cc * HD + d) = v;
        } else {
            kv8_put<BF16, HD>(a, sq, h, f0 + col, d, v, ll);
        }
    }
}

// The splits' parts of a tile, in split order; one block a tile: the parts' weights
// first, then sums whose loads do not wait for one another.  A launch of its own:
// handing the parts over inside the first one (a counter, the last block merging)
// cost 45 us at 512 blocks, each block's release writing its whole L2 back.
template <bool BF16, int HD>
__global__ __launch_bounds__(256) void k_attn_kv8_merge(AttnKv8Args a) {
    __shared__ float w_l[64][17], l_l[16];
    const int tile = blockIdx.x, h = blockIdx.y, j = blockIdx.z, S = a.splits;
    const Kv8Seq sq = kv8_seq(a.c, j);
    const unsigned n_flat = (unsigned)sq.n * (unsigned)a.G, f0 = (unsigned)tile * 16;
    if (f0 >= n_flat) return;
    const int cols = (int)min(16u, n_flat - f0);
    const float *part = a.part + (((int64_t)j * a.c.Hkv + h) * gridDim.x + tile) * S * kv8_part<HD>;
    // 16 lanes a column, each with the splits w, w + 16, ... (at most 4)
    const int col = threadIdx.x >> 4, w0 = threadIdx.x & 15;
    if (col < cols) {
        float mw[4], lw[4], mm = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int w = w0 + 16 * i;
            mw[i] = w < S ? part[w * kv8_part<HD> + col] : -__builtin_inff();
            lw[i] = w < S ? part[w * kv8_part<HD> + 16 + col] : 0.0f;
            mm = fmaxf(mm, mw[i]);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o, 64));
        const float ms = mm == -__builtin_inff() ? 0.0f : mm;
        float ll = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float e = __builtin_amdgcn_exp2f(mw[i] - ms);
            ll = fmaf(lw[i], e, ll);
            if (w0 + 16 * i < S) w_l[w0 + 16 * i][col] = e;
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) ll += __shfl_xor(ll, o, 64);
        if (w0 == 0) l_l[col] = ll;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < cols * (HD / 4); i += 256) {
        const int cc = i / (HD / 4), d = 4 * (i % (HD / 4));
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
        for (int w = 0; w < S; w++) {
            const f32x4 ow = *reinterpret_cast<const f32x4 *>(part + w * kv8_part<HD> + 32 + cc * HD + d);
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] = fmaf(ow[r], w_l[w][cc], v[r]);
        }
        kv8_put<BF16, HD>(a, sq, h, f0 + cc, d, v, l_l[cc]);
    }
}

template <bool BF16, int HD, int R>
static hipError_t go_attn_kv8(const AttnKv8Args &a, hipStream_t st) {
    const dim3 grid((unsigned)(a.tiles * a.splits * a.c.Hkv), (unsigned)a.c.n_seq);
    hipLaunchKernelGGL((k_attn_kv8<BF16, HD, R>), grid, dim3(64 * KV8_WAVES), 0, st, a);
    if (a.splits > 1)
        hipLaunchKernelGGL((k_attn_kv8_merge<BF16, HD>), dim3((unsigned)a.tiles * (R / 16), (unsigned)a.c.Hkv, (unsigned)a.c.n_seq), dim3(256), 0, st, a);
    return hipGetLastError();
}

template <int R>
static hipError_t pick_attn_kv8(AttnKv8Args &a, bool bf16, int splits, hipStream_t st) {
    const int64_t tiles = (a.c.max_rows * a.G + R - 1) / R, units = tiles * (R / 16) * a.c.Hkv * a.c.n_seq;
    // the splits' parts fit the scratch area
    int64_t s = std::min<int64_t>(splits, (int64_t)QASR_KV8_PART_BYTES / (units * (32 + 16 * a.c.hd) * 4));
    s = std::max<int64_t>(1, std::min<int64_t>(s, 64));
    if (tiles * s * a.c.Hkv * 64 * KV8_WAVES > UINT32_MAX || tiles * (R / 16) * 256 > UINT32_MAX) return hipErrorInvalidValue;   // the grid's limit
    a.tiles = (int)tiles;
    a.splits = (int)s;
    // 512 blocks are on the card at a time.  Some more: so many of the shortest go first, and those of middle length
    // follow them (1337 rows, 672 blocks: 37 us against 39 with the shortest last)
    const int64_t per_tile = s * a.c.Hkv * a.c.n_seq, over = (tiles * per_tile - 512 + per_tile - 1) / per_tile;
    a.first = over > 0 && 2 * over <= tiles ? (int)over : 0;
    if (bf16) return a.c.hd == 128 ? go_attn_kv8<true, 128, R>(a, st) : go_attn_kv8<true, 64, R>(a, st);
    return a.c.hd == 128 ? go_attn_kv8<false, 128, R>(a, st) : go_attn_kv8<false, 64, R>(a, st);
}

hipError_t launch_attention_kv8(const AttnKv8Args &a0, bool bf16, hipStream_t st) {
    AttnKv8Args a = a0;
    if ((a.c.hd != 64 && a.c.hd != 128) || a.c.n_seq > 65535 || a.c.Hkv > 65535) return hipErrorInvalidValue;
    a.vec_q = kv8_vec(a.q, nullptr, a.ldq, bf16 ? 2 : 4);
    a.vec_o = (uintptr_t)a.out % 16 == 0;
    const int64_t rows = a.c.max_rows * a.G;
    // blocks of positions that the longest sequence's rows see
    const int64_t seen = a.window > 0 ? std::min<int64_t>(a.max_len, a.window + a.sinks + a.c.max_rows) : a.max_len;
    const int64_t blocks = (seen + 63) / 64;
    if (rows <= 16) {
        // One tile a sequence and head (decoding): the operands straight into registers, as no
        // second tile shares them.  Positions are split over blocks of 4 waves up to 384 blocks,
        // a wave left with one block of positions at least; below 9 of them, 25 from 128 tiles on,
        // the merge costs what the split saves.  us, 1 split against these, 8 KV heads x 2 heads of
        // 128, bf16: one sequence at 404 positions 8.9 / 10.1 (2 splits), at 1000 11.5 -> 10.1, at
        // 4000 29 -> 10, at 60000 323 -> 33; 4 at 16000 98 -> 26; 8 at 1000 12.0 -> 11.1; 16 at 1500
        // 15.0 / 16.7 (3 splits); 32 at 4000 41 / 42.5 (2 splits).
        const int64_t units = a.c.Hkv * (int64_t)a.c.n_seq;
        const int splits = blocks <= (units < 128 ? 8 : 24) ? 1 : (int)std::min<int64_t>(384 / units, (blocks + 3) / 4);
        return pick_attn_kv8<16>(a, bf16, splits, st);
    }
    // Splits up to 512 blocks, which the card holds at a time; each wave left with two blocks of
    // positions at least.  us with the merge, 1 split against these: 4 x 67 bf16 rows, window 8192,
    // 70 -> 40; 3 x 100 f32 rows behind 8000 positions 97 -> 62; 67 f32 rows behind 20000 227 -> 52;
    // 20 bf16 rows behind 4000 37 -> 20; 404 f32 rows alone 13.7 with 1 and 21 with 2.
    // Sequences shorter than max_rows leave their last tiles' blocks empty: counted are the tiles
    // that n_rows rows fill, and half a tile a sequence (up to 67 rows each, window 8192: 40.2 + 5.3
    // -> 30.7 + 6.5; 6 sequences of up to 100 f32 rows behind 6000 positions 85.7 -> 51 + 5.4).
    const int64_t tiles = std::min((rows + 31) / 32 * a.c.n_seq, (a.c.n_rows * a.G / 16 + a.c.n_seq) / 2 + 1);
    const int64_t units = tiles * a.c.Hkv;
    if (units >= 384) return pick_attn_kv8<32>(a, bf16, 1, st);
    return pick_attn_kv8<32>(a, bf16, (int)std::min<int64_t>(512 / units, blocks / 8), st);
}

}  // namespace qasr
