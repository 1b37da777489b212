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
// Per tile of 16 query rows (row = query row x heads of the group, flattened) and
// KV head: S = scale q.k over blocks of 64 positions with the running maximum and
// sum of the softmax, O += P V.  Everything is exact integer products:
//   q: round(q c), c = N / max|q| of the row, in D signed base-256 digits, one MFMA
//      a digit
//   p: round(N p), p = 2^(s - the block's own maximum) in [0, 1], the same digits
// with N = 8e6 and D = 3 for f32 rows (a value is off by at most 6e-8 of the largest
// of its row or block) and N = 32000, D = 2 for bf16 rows (1.6e-5; their output is
// rounded to 2^-8 of itself).  p is counted from the block's maximum and not the
// running one: where one position far back holds the maximum (a sink), what is left
// of every other block would otherwise vanish in the rounding, and the loss would
// grow with the context.  A block's scale is the same for all of its 64 positions:
// it joins the score's factor (K) and the product's (V).
//
// The sums (O and the weights') count from a reference that moves only when a
// block's maximum is 2^16 above it: in f32 they lose nothing by that, and most
// blocks rescale nothing.
//
// What bounds it: the HBM reads where every sequence has one row; vector
// instructions where rows share the positions (a score's way from the integer sums
// to the digits is about 14 instructions, a product's value 5; three in bf16).
//
// A block takes CG tiles (CG x 16 flattened rows) with CG x PG waves: PG groups of
// waves take every PG-th block of positions each, the CG waves of a group one tile
// each.  SHARED: a group's K and V blocks come through one slot each in LDS, direct
// from memory (global_load_lds_dwordx4), K while the block before is multiplied by
// its weights, V during the scores.  (Operands loaded straight into registers leave
// the four lanes of a quad in four rows: a 64-byte run is then asked for four times
// over, and 16 KB a tile and block at 5.3 TB/s was the end, cached or not.  Two slots
// each, a whole block ahead: 36 us for 29 at 1337 rows; the waves that the LDS then
// keeps out are worth more.)  With `splits` > 1 several blocks share a tile's
// positions; a second launch merges their parts.
// ---------------------------------------------------------------------------

// Digit dwords: digit d of 4 values in one dword, a byte each.  Signed base-256
// digits are the bytes of (n + 0x..8080) ^ 0x..8080; the highest of a value that is
// not negative needs no offset.  v holds the sums in its low bytes.
template <int D, bool SIGNED>
__device__ __forceinline__ void digits4(const uint32_t *v, uint32_t *d) {
    const uint32_t a = __builtin_amdgcn_perm(v[1], v[0], 0x05010400), b = __builtin_amdgcn_perm(v[3], v[2], 0x05010400);
    d[0] = __builtin_amdgcn_perm(b, a, 0x05040100) ^ 0x80808080u;
    d[1] = __builtin_amdgcn_perm(b, a, 0x07060302);
    if (D == 3 || SIGNED) d[1] ^= 0x80808080u;
    if (D == 3) {
        const uint32_t e = __builtin_amdgcn_perm(v[1], v[0], 0x0c0c0602), f = __builtin_amdgcn_perm(v[3], v[2], 0x06020c0c);
        d[D - 1] = e | f;
        if (SIGNED) d[D - 1] ^= 0x80808080u;
    }
}
// the value of a product's digit sums
template <int D>
__device__ __forceinline__ float digit_sum(const i32x4 *acc, int r) {
    if (D == 2) return (float)(acc[1][r] * 256 + acc[0][r]);
    return fmaf((float)(acc[D - 1][r] * 256 + acc[1][r]), 256.0f, (float)acc[0][r]);
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

// one split's part of a tile in the scratch area: maxima and sums [2][16], then O [16][HD]
template <int HD> constexpr int kv8_part = 32 + 16 * HD;

template <bool BF16, int HD, int CG, int PG, bool SHARED>
__global__ __launch_bounds__(64 * CG * PG, SHARED ? 4 : 2) void k_attn_kv8(AttnKv8Args a) {
    constexpr int KS = HD / 64, DT = HD / 16, D = BF16 ? 2 : 3, TB = 64 * HD, LD = HD / 8 / CG;   // bytes of a block; a wave's loads of K and V
    constexpr float N = BF16 ? 32000.0f : 8.0e6f;
    static_assert(SHARED || CG == 1, "waves that share a block's positions share its bytes in LDS");
    constexpr int MERGE = CG * PG * 16 * (HD + 4) * 4, SLOTS = SHARED ? PG * 2 * TB : 0;
    __shared__ __attribute__((aligned(16))) char smem[MERGE > SLOTS ? MERGE : SLOTS];
    __shared__ float ml_l[CG * PG][2][16];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cg = wid % CG, pg = wid / CG;
    const int c = lane & 15, g = lane >> 4;
    // Heads fastest: with 8 of them each XCD (blocks go to the 8 in turn) has one head's
    // cache in its L2.  Tiles from the longest on, but every second 256 blocks the other way
    // round: a CU that has a long tile gets a short one next (1337 rows 29.3 -> 28.2 us).
    const int j = blockIdx.y, S = a.splits;
    const unsigned rest = blockIdx.x / (unsigned)a.c.Hkv;
    const int h = blockIdx.x - rest * a.c.Hkv, tx = rest / (unsigned)S, split = rest - tx * S;
    const int run = max(1, 256 / (a.c.Hkv * S)), turn = tx / run;
    const int back = (turn & 1) && (turn + 1) * run <= a.tiles ? (2 * turn + 1) * run - 1 - tx : tx;
    const int tile0 = (a.tiles - 1 - back) * CG, tile = tile0 + cg;
    const Kv8Seq sq = kv8_seq(a.c, j);
    // flattened rows: fewer than 2^30 (the entry point)
    const unsigned n_flat = (unsigned)sq.n * (unsigned)a.G;
    if ((unsigned)tile0 * 16 >= n_flat) return;
    const unsigned f0 = (unsigned)tile * 16, f1 = n_flat - 1;      // a tile past the last row repeats it
    const unsigned fr = min(f0 + c, f1);
    const int qi = (int)(fr / (unsigned)a.G), qg = (int)(fr - (unsigned)qi * (unsigned)a.G);
    const int i_lo = (int)(min(f0, f1) / (unsigned)a.G), i_hi = (int)(min(f0 + 15, f1) / (unsigned)a.G);
    const int last = sq.p0 + qi;                               // this column's own position, and its window's first
    const int low = a.window > 0 ? last - a.window + 1 : INT32_MIN;

    // the blocks that some row of the block's tiles sees: the sinks' and the window's; this split's run of them
    const int hi_pos = min(sq.p0 + (int)(min((unsigned)(tile0 + CG) * 16 - 1, f1) / (unsigned)a.G), a.c.cap - 1);
    int lo_pos = 0, n_sink = 0;
    if (a.window > 0) {
        lo_pos = max(0, sq.p0 + (int)((unsigned)tile0 * 16 / (unsigned)a.G) - a.window + 1);
        n_sink = min((a.sinks + 63) / 64, lo_pos / 64);
    }
    const int lo_blk = lo_pos / 64;
    const int n_blk = hi_pos < 0 ? 0 : n_sink + max(0, hi_pos / 64 - lo_blk + 1);
    const int per = n_blk / S, more = n_blk - per * S;         // the first `more` splits take one block more
    const int u0 = split * per + min(split, more), u1 = u0 + per + (split < more ? 1 : 0);
    auto block_of = [&](int u) { return u < n_sink ? u : lo_blk + u - n_sink; };

    const int64_t head = (int64_t)j * a.c.Hkv + h;
    const int8_t *kb = a.c.k8 + head * a.c.cap * HD, *vb = a.c.v8 + head * a.c.cap * HD;
    const float *ks = a.c.ks + head * (a.c.cap / 64), *vs = a.c.vs + head * (a.c.cap / 64);
    int u = u0 + pg;
    // SHARED: this lane's bytes of the wave's loads
    char *kt = smem + pg * 2 * TB, *vt = kt + TB;
    // a load fills 64 slots: 8 rows of 128 bytes (the swizzle repeats every 16 rows) or 16 of 64
    const uint32_t v_src = (lane >> 2) * 64 + 16 * ((lane & 3) ^ lds_swz<64>(lane >> 2));
    const uint32_t k_src[2] = {HD == 64 ? v_src : (lane >> 3) * 128 + 16 * ((lane & 7) ^ lds_swz<128>(lane >> 3)),
                               HD == 64 ? v_src : (lane >> 3) * 128 + 16 * ((lane & 7) ^ lds_swz<128>(8 + (lane >> 3)))};
    static_assert(LD % 4 == 0 || HD == 64, "pairs of loads a wave");
    auto issue_k = [&](int b) {
#pragma unroll
        for (int i = 0; i < LD / 2; i++) {
            const int at = 1024 * (cg * (LD / 2) + i);
            lds_dma16_s(kb + (int64_t)b * TB + at, k_src[i & 1], kt + at);
        }
    };
    auto issue_v = [&](int b) {
#pragma unroll
        for (int i = 0; i < LD / 2; i++) {
            const int at = 1024 * (cg * (LD / 2) + i);
            lds_dma16_s(vb + (int64_t)b * TB + at, v_src, vt + at);
        }
    };
    // otherwise the operands themselves, loaded again as soon as the products have read them
    i32x4 kr[4][KS], vr[DT];
    auto load_k = [&](int b) {
        const int8_t *p = kb + (int64_t)b * TB + c * HD + 16 * g;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int k = 0; k < KS; k++) kr[t][k] = *reinterpret_cast<const i32x4 *>(p + 16 * t * HD + 64 * k);
    };
    auto load_v = [&](int b) {
        const int8_t *p = vb + (int64_t)b * TB + c * 64 + 16 * g;
#pragma unroll
        for (int d = 0; d < DT; d++) vr[d] = *reinterpret_cast<const i32x4 *>(p + 16 * d * 64);
    };
    // the column's row, ahead of the first block: it is turned into digits while that is on its way
    float x[KS][16];
#pragma unroll
    for (int s = 0; s < KS; s++)
        kv8_load16<BF16>(a.q, (sq.r0 + qi) * a.ldq + (int64_t)(h * a.G + qg) * HD + 64 * s + 16 * g, a.vec_q, x[s]);
    __builtin_amdgcn_sched_barrier(0);
    if (u < u1) {
        if constexpr (SHARED) {
            issue_k(block_of(u));
        } else {
            load_k(block_of(u));
            load_v(block_of(u));
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // the column's row in signed digits: dims 64 s + 16 g + 0..15 of product s
    i32x4 qd[KS][D];
    float qf;                                                  // score = integer sum x qf x the block's scale
    {
        float m = 0.0f;
        bool bad = false;
#pragma unroll
        for (int s = 0; s < KS; s++) {
#pragma unroll
            for (int e = 0; e < 16; e++) x[s][e] = a.scale < 0.0f ? -x[s][e] : x[s][e];   // the scores' factor is not negative
#pragma unroll
            for (int e = 0; e < 16; e++) { m = fmaxf(m, fabsf(x[s][e])); bad |= !kv8_finite(x[s][e]); }
        }
        m = xhalf_max(xrow16_max(m));
        float nf = bad ? 1.0f : 0.0f;
        nf = xhalf_max(xrow16_max(nf));
        // a row below 1e-30 multiplies by the largest factor that stays finite with it
        const float f = __fdiv_rn(N, fmaxf(m, 1e-30f));
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint32_t n[4], d[D];
#pragma unroll
                for (int i = 0; i < 4; i++) n[i] = (uint32_t)(int)rintf(x[s][4 * e + i] * f) + 0x80808080u;
                digits4<D, true>(n, d);
#pragma unroll
                for (int i = 0; i < D; i++) qd[s][i][e] = (int)d[i];
            }
        qf = nf > 0.0f ? __builtin_nanf("") : fabsf(a.scale) * 1.4426950408889634f * __fdiv_rn(1.0f, f);
    }

    float m = -__builtin_inff(), l = 0.0f;                     // m: what O and l count from
    f32x4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    float ksl = 0.0f, vsl = 0.0f;                              // lane i: the scales of this group's block `it` + i
    const int n_it = (u1 - u0 + PG - 1) / PG;
    for (int it = 0; it < n_it; it++, u += PG) {
        if ((it & 63) == 0) {
            const int ul = u + lane * PG;
            ksl = ul < u1 ? ks[block_of(ul)] : 0.0f;
            vsl = ul < u1 ? vs[block_of(ul)] : 0.0f;
            // waited for here: a wait at their use would drain the loads in flight in every turn
            asm volatile("" : "+v"(ksl), "+v"(vsl));
        }
        const bool live = u < u1;
        const int b = block_of(u), bn = block_of(min(u + PG, u1 - 1));
        if constexpr (SHARED) {
            wait_vmcnt<0>();                                   // this wave's part of the block's K has landed
            __syncthreads();                                   // ... and every wave's; V of the block before has been read
            if (live) issue_v(b);
        }
        if (!live) {                                           // the other groups' last block
            if (SHARED) __syncthreads();
            continue;
        }
        const float ksb = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ksl), it & 63));
        const float vsb = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vsl), it & 63));
        // a product's sums are read behind the next product's issue
        float s[16];
        {
            i32x4 acc[2][D];
#pragma unroll
            for (int t = 0; t <= 4; t++) {
                if (t < 4) {
#pragma unroll
                    for (int d = 0; d < D; d++) acc[t & 1][d] = i32x4{0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < KS; k++) {
                        const int r = 16 * t + c;
                        if (SHARED) kr[t][k] = *reinterpret_cast<const i32x4 *>(kt + r * HD + 16 * ((4 * k + g) ^ lds_swz<HD>(r)));
#pragma unroll
                        for (int d = 0; d < D; d++)
                            acc[t & 1][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kr[t][k], qd[k][d], acc[t & 1][d], 0, 0, 0);
                    }
                }
                if (t > 0) {
#pragma unroll
                    for (int r = 0; r < 4; r++) s[4 * (t - 1) + r] = digit_sum<D>(acc[(t - 1) & 1], r);
                }
            }
        }
        if constexpr (!SHARED) {
            __builtin_amdgcn_sched_barrier(0);
            load_k(bn);                                        // a whole block ahead of their use
            __builtin_amdgcn_sched_barrier(0);
        }
        // p from the integer sums; mb: the block's maximum
        const float kf = ksb * qf;
        float mb, p[16];
        if (ksb >= 0.0f && b * 64 + 63 <= sq.p0 + i_lo &&
            (a.window == 0 || b * 64 > sq.p0 + i_hi - a.window || b * 64 + 63 < a.sinks)) {
            // every row of the tile sees the whole block
            mb = s[0];
#pragma unroll
            for (int i = 1; i < 16; i++) mb = fmaxf(mb, s[i]);
            mb = xhalf_max(xrow16_max(mb)) * kf;
#pragma unroll
            for (int i = 0; i < 16; i++) p[i] = __builtin_amdgcn_exp2f(s[i] * kf - mb);   // two roundings: at most 1, as the digits hold
        } else {
            mb = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int at = b * 64 + 16 * (i >> 2) + 4 * g + (i & 3);
                const bool seen = (at <= last) & ((at >= low) | (at < a.sinks));
                s[i] = seen ? s[i] * kf : -__builtin_inff();
                mb = fmaxf(mb, s[i]);
            }
            mb = xhalf_max(xrow16_max(mb));
            const float ref = mb == -__builtin_inff() ? 0.0f : mb;
#pragma unroll
            for (int i = 0; i < 16; i++) p[i] = __builtin_amdgcn_exp2f(s[i] - ref);
        }
        const bool up = mb > m + 16.0f;
        if (__any(up)) {
            const float al = up ? __builtin_amdgcn_exp2f(m - mb) : 1.0f;
            m = up ? mb : m;
            l *= al;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int r = 0; r < 4; r++) o[dt][r] *= al;
        }
        // a column that sees none of this block takes nothing of it, its scale neither
        const float eb = mb == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(mb - m);
        const float vf = mb == -__builtin_inff() ? 0.0f : vsb * eb * (1.0f / N);
        i32x4 pd[D];
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            uint32_t n[4], d[D];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                sum += p[4 * t + r];
                // 2^23 + the lower digits' offset: the sum's low bytes are round(N p) + that offset
                n[r] = __float_as_uint(fmaf(p[4 * t + r], N, 8388608.0f + (D == 2 ? 128.0f : 32896.0f)));
            }
            digits4<D, false>(n, d);
#pragma unroll
            for (int e = 0; e < D; e++) pd[e][t] = (int)d[e];
        }
        l = fmaf(sum, eb, l);
        if constexpr (SHARED) {
            wait_vmcnt<0>();                                   // V has landed, and every wave has read K
            __syncthreads();
            if (u + PG < u1) issue_k(bn);
        }
        {
            i32x4 acc[2][D];
#pragma unroll
            for (int dt = 0; dt <= DT; dt++) {
                if (dt < DT) {
                    const int vrow = 16 * dt + c;
                    if (SHARED) vr[dt] = *reinterpret_cast<const i32x4 *>(vt + vrow * 64 + 16 * (g ^ lds_swz<64>(vrow)));
#pragma unroll
                    for (int e = 0; e < D; e++) {
                        const i32x4 z = {0, 0, 0, 0};
                        acc[dt & 1][e] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vr[dt], pd[e], z, 0, 0, 0);
                    }
                }
                if (dt > 0) {
#pragma unroll
                    for (int r = 0; r < 4; r++) o[dt - 1][r] = fmaf(digit_sum<D>(acc[(dt - 1) & 1], r), vf, o[dt - 1][r]);
                }
                // one product, then its share of the last one's vector instructions: the two run side by side
                if (dt > 0 && dt < DT) {
#pragma unroll
                    for (int e = 0; e < D; e++) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x002, D == 3 ? 7 : 6, 0);
                    }
                }
            }
        }
        if constexpr (!SHARED) {
            __builtin_amdgcn_sched_barrier(0);
            load_v(bn);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    l = xhalf_sum(xrow16_sum(l));

    const int cols = f0 < n_flat ? (int)min(16u, n_flat - f0) : 0;
    float *part = a.part + ((((int64_t)j * a.c.Hkv + h) * a.tiles * CG + tile) * S + split) * kv8_part<HD>;
    // the groups' parts of each tile, through the ring's LDS (every load into it has landed and been read)
    float (*o_l)[16][HD + 4] = reinterpret_cast<float (*)[16][HD + 4]>(smem);
    __syncthreads();
    if (g == 0) { ml_l[wid][0][c] = m; ml_l[wid][1][c] = l; }
#pragma unroll
    for (int dt = 0; dt < DT; dt++) *reinterpret_cast<f32x4 *>(&o_l[wid][c][16 * dt + 4 * g]) = o[dt];
    __syncthreads();
    for (int i = lane + 64 * pg; i < cols * (HD / 4); i += 64 * PG) {
        const int col = i / (HD / 4), d = 4 * (i % (HD / 4));
        float mm = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < PG; w++) mm = fmaxf(mm, ml_l[w * CG + cg][0][col]);
        const float ms = mm == -__builtin_inff() ? 0.0f : mm;
        float ll = 0.0f;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < PG; w++) {
            const float e = __builtin_amdgcn_exp2f(ml_l[w * CG + cg][0][col] - ms);
            ll = fmaf(ml_l[w * CG + cg][1][col], e, ll);
            const f32x4 ow = *reinterpret_cast<const f32x4 *>(&o_l[w * CG + cg][col][d]);
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] = fmaf(ow[r], e, v[r]);
        }
        if (S > 1) {
            if (d == 0) { part[col] = mm; part[16 + col] = ll; }
            *reinterpret_cast<f32x4 *>(part + 32 + col * HD + d) = v;
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

template <bool BF16, int HD, int CG, int PG, bool SHARED>
static hipError_t go_attn_kv8(const AttnKv8Args &a, hipStream_t st) {
    const dim3 grid((unsigned)(a.tiles * a.splits * a.c.Hkv), (unsigned)a.c.n_seq);
    hipLaunchKernelGGL((k_attn_kv8<BF16, HD, CG, PG, SHARED>), grid, dim3(64 * CG * PG), 0, st, a);
    if (a.splits > 1)
        hipLaunchKernelGGL((k_attn_kv8_merge<BF16, HD>), dim3((unsigned)a.tiles * CG, (unsigned)a.c.Hkv, (unsigned)a.c.n_seq), dim3(256), 0, st, a);
    return hipGetLastError();
}

template <int CG, int PG, bool SHARED>
static hipError_t pick_attn_kv8(AttnKv8Args &a, bool bf16, int splits, hipStream_t st) {
    const int64_t tiles = (a.c.max_rows * a.G + 16 * CG - 1) / (16 * CG), units = tiles * CG * a.c.Hkv * a.c.n_seq;
    // the splits' parts fit the scratch area
    int64_t s = std::min<int64_t>(splits, (int64_t)QASR_KV8_PART_BYTES / (units * (32 + 16 * a.c.hd) * 4));
    s = std::max<int64_t>(1, std::min<int64_t>(s, 64));
    if (tiles * s * a.c.Hkv * 64 * CG * PG > UINT32_MAX || tiles * CG * 256 > UINT32_MAX) return hipErrorInvalidValue;   // the grid's limit
    a.tiles = (int)tiles;
    a.splits = (int)s;
    if (bf16) return a.c.hd == 128 ? go_attn_kv8<true, 128, CG, PG, SHARED>(a, st) : go_attn_kv8<true, 64, CG, PG, SHARED>(a, st);
    return a.c.hd == 128 ? go_attn_kv8<false, 128, CG, PG, SHARED>(a, st) : go_attn_kv8<false, 64, CG, PG, SHARED>(a, st);
}

hipError_t launch_attention_kv8(const AttnKv8Args &a0, bool bf16, hipStream_t st) {
    AttnKv8Args a = a0;
    if ((a.c.hd != 64 && a.c.hd != 128) || a.c.n_seq > 65535 || a.c.Hkv > 65535) return hipErrorInvalidValue;
    a.vec_q = kv8_vec(a.q, nullptr, a.ldq, bf16 ? 2 : 4);
    a.vec_o = (uintptr_t)a.out % 16 == 0;
    const int64_t rows = a.c.max_rows * a.G;
    // blocks of positions that the longest sequence's rows see
    const int64_t seen = a.window > 0 ? std::min<int64_t>(a.max_len, (int64_t)a.window + a.sinks + a.c.max_rows) : a.max_len;
    const int64_t blocks = (seen + 63) / 64;
    if (rows <= 16) {
        // One tile a sequence and head (decoding): the operands straight into registers, as no
        // second tile shares them.  Positions are split over blocks of 4 waves up to 384 blocks,
        // a wave left with one block of positions at least; below 25 of them the merge costs what
        // the split saves.  us, 1 split against these, 8 KV heads x 2 heads of 128, bf16: one
        // sequence at 4000 positions 25.2 -> 9.9, at 60000 323 -> 30, 4 at 16000 90 -> 24; at 1000
        // positions 10.9 against 12.2; 32 at 4000 40.3 against 42.5 (2 splits), so one there.
        const int64_t units = a.c.Hkv * (int64_t)a.c.n_seq;
        const int splits = blocks <= 24 ? 1 : (int)std::min<int64_t>(384 / units, (blocks + 3) / 4);
        return pick_attn_kv8<1, 4, false>(a, bf16, splits, st);
    }
    // Two tiles a block.  2 groups of waves a block where 384 blocks are there, else 4 groups
    // and splits up to 512 blocks, each wave left with 4 blocks of positions at least.  us, 2
    // groups against 4: 1337 rows 29.4 / 32.4, with bf16 22.6 / 26.6; 404 rows 12.5 / 12.2; 2 x
    // 300 rows behind 3000 positions 45 / 41; 4 x 67 rows, window 8192: 87 / 61, with 3 splits
    // 43 + 5 / 38 + 5.
    // Sequences shorter than max_rows leave their last tiles' blocks empty: counted are the tiles
    // that n_rows rows fill, and half a tile a sequence (up to 67 rows each, window 8192: 40.2 + 5.3
    // -> 30.7 + 6.5; 6 sequences of up to 100 f32 rows behind 6000 positions 85.7 -> 51 + 5.4).
    const int64_t tiles = std::min((rows + 31) / 32 * a.c.n_seq, (a.c.n_rows * a.G / 16 + a.c.n_seq) / 2 + 1);
    const int64_t units = tiles * a.c.Hkv;
    if (units >= 384) return pick_attn_kv8<2, 2, true>(a, bf16, 1, st);
    return pick_attn_kv8<2, 4, true>(a, bf16, (int)std::min<int64_t>(512 / units, blocks / 16), st);
}

}  // namespace qasr
