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

__device__ __forceinline__ bool kv8_finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// x at scale s (inv about 1 / s): NaN 0, infinities +-127, everything 0 at scale 0
__device__ __forceinline__ int kv8_round(float x, double s, double inv) {
    if (!(fabsf(x) >= 0.0f) || s == 0.0) return 0;
    const int k = kv8_finite(x) ? round_ratio((double)fabsf(x), s, inv) : 127;
    return x < 0.0f ? -k : k;
}

// ---------------------------------------------------------------------------
// write: one block of 256 threads per (block of the sequence, head, sequence, K or V)
// ---------------------------------------------------------------------------
template <bool BF16, int HD>
__global__ __launch_bounds__(256) void k_kv8_write(Kv8Args a) {
    constexpr int CH = HD / 16, RP = 256 / CH, IT = 64 / RP;     // 16-value chunks a row, rows a pass, passes
    __shared__ float red[4];
    __shared__ __attribute__((aligned(16))) int8_t tile[HD][64 + 16];
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
    const int ch = t % CH, rr = t / CH;
    float x[IT][16];
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < IT; i++) {
        const int p = i * RP + rr;
        if (p < keep || p >= upto) continue;
        kv8_load16<BF16>(src, (sq.r0 + (b * 64 + p - sq.p0)) * a.ld + h * HD + ch * 16, a.vec, x[i]);
#pragma unroll
        for (int e = 0; e < 16; e++) m = kv8_finite(x[i][e]) ? fmaxf(m, fabsf(x[i][e])) : m;
    }
    m = wave_max_f32(m);
    if (lane == 0) red[wid] = m;
    const float s_old = keep > 0 ? *sp : 0.0f;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float s = fmaxf(s_old, __fdiv_rn(m, 127.0f));
    const double sd = (double)s, inv = s > 0.0f ? 1.0 / sd : 0.0, od = (double)s_old;
    const bool grow = keep > 0 && s > s_old;
    auto again = [&](int q) {                                    // an earlier value at the raised scale
        const int k = round_ratio((double)abs(q) * od, sd, inv);
        return q < 0 ? -k : k;
    };
    if (t == 0) *sp = s;
    if (!is_v) {
#pragma unroll
        for (int i = 0; i < IT; i++) {
            const int p = i * RP + rr;
            i32x4 *o = reinterpret_cast<i32x4 *>(dst + p * HD + ch * 16);
            if (p >= keep && p < upto) {
                int q[16];
#pragma unroll
                for (int e = 0; e < 16; e++) q[e] = kv8_round(x[i][e], sd, inv);
                *o = i32x4{pack4_i8(q[0], q[1], q[2], q[3]), pack4_i8(q[4], q[5], q[6], q[7]),
                           pack4_i8(q[8], q[9], q[10], q[11]), pack4_i8(q[12], q[13], q[14], q[15])};
            } else if (p < keep && grow) {
                i32x4 v = *o;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    v[e] = pack4_i8(again((int8_t)v[e]), again((int8_t)(v[e] >> 8)), again((int8_t)(v[e] >> 16)), again(v[e] >> 24));
                *o = v;
            }
        }
        return;
    }
    // V: the stored block goes through LDS, where rows become bytes of a dim
    if (keep > 0 || upto < 64) {
        for (int i = t; i < HD * 4; i += 256) *reinterpret_cast<i32x4 *>(&tile[i >> 2][16 * (i & 3)]) = reinterpret_cast<const i32x4 *>(dst)[i];
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < IT; i++) {
        const int p = i * RP + rr, sl = kv8_slot(p);
        if (p >= keep && p < upto) {
#pragma unroll
            for (int e = 0; e < 16; e++) tile[ch * 16 + e][sl] = (int8_t)kv8_round(x[i][e], sd, inv);
        } else if (p < keep && grow) {
#pragma unroll
            for (int e = 0; e < 16; e++) tile[ch * 16 + e][sl] = (int8_t)again(tile[ch * 16 + e][sl]);
        }
    }
    __syncthreads();
    for (int i = t; i < HD * 4; i += 256) reinterpret_cast<i32x4 *>(dst)[i] = *reinterpret_cast<const i32x4 *>(&tile[i >> 2][16 * (i & 3)]);
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
    constexpr int CH = HD / 16, RP = 256 / CH, IT = 64 / RP;
    __shared__ __attribute__((aligned(16))) int8_t tile[HD][64 + 16];
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
    if (is_v) {
        for (int i = t; i < HD * 4; i += 256) *reinterpret_cast<i32x4 *>(&tile[i >> 2][16 * (i & 3)]) = reinterpret_cast<const i32x4 *>(src)[i];
        __syncthreads();
    }
    const int ch = t % CH, rr = t / CH;
#pragma unroll
    for (int i = 0; i < IT; i++) {
        const int p = i * RP + rr;
        if (p < lo || p >= hi) continue;
        float x[16];
        if (is_v) {
            const int sl = kv8_slot(p);
#pragma unroll
            for (int e = 0; e < 16; e++) x[e] = __fmul_rn((float)tile[ch * 16 + e][sl], s);
        } else {
            const i32x4 v = *reinterpret_cast<const i32x4 *>(src + p * HD + ch * 16);
#pragma unroll
            for (int e = 0; e < 16; e++) x[e] = __fmul_rn((float)(int8_t)(v[e >> 2] >> (8 * (e & 3))), s);
        }
        const int64_t at = (sq.r0 + (b * 64 + p - sq.p0)) * a.ld + h * HD + ch * 16;
        if (BF16) {
            uint16_t *o = reinterpret_cast<uint16_t *>(is_v ? a.v : a.k) + at;
            u16x8 u[2];
#pragma unroll
            for (int e = 0; e < 16; e++) u[e >> 3][e & 7] = __builtin_bit_cast(uint16_t, (__bf16)x[e]);
            if (a.vec) {
                reinterpret_cast<u16x8 *>(o)[0] = u[0];
                reinterpret_cast<u16x8 *>(o)[1] = u[1];
            } else {
#pragma unroll
                for (int e = 0; e < 16; e++) o[e] = u[e >> 3][e & 7];
            }
        } else {
            float *o = reinterpret_cast<float *>(is_v ? a.v : a.k) + at;
            if (a.vec) {
#pragma unroll
                for (int c = 0; c < 4; c++) reinterpret_cast<f32x4 *>(o)[c] = f32x4{x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]};
            } else {
#pragma unroll
                for (int e = 0; e < 16; e++) o[e] = x[e];
            }
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
//   q: round(q c) with c = 8e6 / max|q| of the row, three signed base-256 digits
//      (24 bits: a row's error is 6e-8 of its largest value), three MFMAs a product
//   p: round(2^30 p), p = 2^(s - max) in [0, 1], four digits.  30 bits and not 24:
//      a sink that holds the maximum leaves every other p small, and what a long
//      context loses by rounding them grows with its length
// The digits of a value n come out together: the bytes of (n + 0x80808080) ^
// 0x80808080 are its signed base-256 digits.
// A block's scale is the same for all of its 64 positions: it joins the score's
// factor (K) and the product's (V).
// ---------------------------------------------------------------------------

// 4 values' digit dwords -> digit d of the 4 values in one dword (a 4 x 4 byte transpose)
__device__ __forceinline__ void digits4(uint32_t n0, uint32_t n1, uint32_t n2, uint32_t n3, uint32_t *d) {
    const uint32_t a = __builtin_amdgcn_perm(n1, n0, 0x05010400), b = __builtin_amdgcn_perm(n1, n0, 0x07030602);
    const uint32_t c = __builtin_amdgcn_perm(n3, n2, 0x05010400), e = __builtin_amdgcn_perm(n3, n2, 0x07030602);
    d[0] = __builtin_amdgcn_perm(c, a, 0x05040100);
    d[1] = __builtin_amdgcn_perm(c, a, 0x07060302);
    d[2] = __builtin_amdgcn_perm(e, b, 0x05040100);
    d[3] = __builtin_amdgcn_perm(e, b, 0x07060302);
}
__device__ __forceinline__ uint32_t signed_digits(int n) { return ((uint32_t)n + 0x80808080u) ^ 0x80808080u; }

#define QASR_KV8_WAVES 4
template <bool BF16, int HD>
__global__ __launch_bounds__(64 * QASR_KV8_WAVES) void k_attn_kv8(AttnKv8Args a) {
    constexpr int KS = HD / 64, DT = HD / 16, W = QASR_KV8_WAVES;
    __shared__ float o_l[W][16][HD + 4];
    __shared__ float ml_l[W][2][16];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int h = blockIdx.y, j = blockIdx.z;
    const Kv8Seq sq = kv8_seq(a.c, j);
    const int64_t n_flat = (int64_t)sq.n * a.G, f0 = (int64_t)blockIdx.x * 16;
    if (f0 >= n_flat) return;
    const int64_t fr = min(f0 + c, n_flat - 1);
    const int qi = (int)(fr / a.G), qg = (int)(fr % a.G);
    const int i_lo = (int)(f0 / a.G), i_hi = (int)(min(f0 + 15, n_flat - 1) / a.G);
    const int last = sq.p0 + qi;                               // this column's own position

    // the column's row in signed digits: dims 64 s + 16 g + 0..15 of product s
    i32x4 qd[KS][3];
    float qf;                                                  // score = integer sum x qf x the block's scale
    {
        const int64_t at = (sq.r0 + qi) * a.ldq + (int64_t)(h * a.G + qg) * HD;
        float x[KS][16], m = 0.0f;
        bool bad = false;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            kv8_load16<BF16>(a.q, at + 64 * s + 16 * g, a.vec_q, x[s]);
#pragma unroll
            for (int e = 0; e < 16; e++) { m = fmaxf(m, fabsf(x[s][e])); bad |= !kv8_finite(x[s][e]); }
        }
        m = xhalf_max(xrow16_max(m));
        float nf = bad ? 1.0f : 0.0f;
        nf = xhalf_max(xrow16_max(nf));
        // a row below 1e-30 multiplies by the largest factor that stays finite with it
        const float f = __fdiv_rn(8.0e6f, fmaxf(m, 1e-30f));
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint32_t d[4];
                digits4(signed_digits((int)rintf(x[s][4 * e] * f)), signed_digits((int)rintf(x[s][4 * e + 1] * f)),
                        signed_digits((int)rintf(x[s][4 * e + 2] * f)), signed_digits((int)rintf(x[s][4 * e + 3] * f)), d);
                qd[s][0][e] = (int)d[0];
                qd[s][1][e] = (int)d[1];
                qd[s][2][e] = (int)d[2];
            }
        qf = nf > 0.0f ? __builtin_nanf("") : a.scale * 1.4426950408889634f * __fdiv_rn(1.0f, f);
    }

    // the blocks that some row of the tile sees: the sinks' and the window's
    const int hi_pos = min(sq.p0 + i_hi, a.c.cap - 1);
    int lo_pos = 0, n_sink = 0;
    if (a.window > 0) {
        lo_pos = max(0, sq.p0 + i_lo - a.window + 1);
        n_sink = min((min(a.sinks, a.c.cap) + 63) / 64, lo_pos / 64);
    }
    const int lo_blk = lo_pos / 64;
    const int n_blk = hi_pos < 0 ? 0 : n_sink + max(0, hi_pos / 64 - lo_blk + 1);

    const int64_t head = (int64_t)j * a.c.Hkv + h;
    const int8_t *kb = a.c.k8 + head * a.c.cap * HD, *vb = a.c.v8 + head * a.c.cap * HD;
    const float *ks = a.c.ks + head * (a.c.cap / 64), *vs = a.c.vs + head * (a.c.cap / 64);
    float m = -__builtin_inff(), l = 0.0f;
    f32x4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    for (int u = wid; u < n_blk; u += W) {
        const int b = u < n_sink ? u : lo_blk + u - n_sink;
        const int8_t *kt = kb + (int64_t)b * 64 * HD, *vt = vb + (int64_t)b * 64 * HD;
        const float kf = ks[b] * qf;
        float s[16];
        float mx = -__builtin_inff();
#pragma unroll
        for (int t = 0; t < 4; t++) {
            i32x4 acc[3] = {};
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const i32x4 ka = *reinterpret_cast<const i32x4 *>(kt + (16 * t + c) * HD + 64 * k + 16 * g);
#pragma unroll
                for (int d = 0; d < 3; d++) acc[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(ka, qd[k][d], acc[d], 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int p = b * 64 + 16 * t + 4 * g + r;
                const float v = fmaf((float)(acc[2][r] * 256 + acc[1][r]), 256.0f, (float)acc[0][r]) * kf;
                const bool seen = p <= last && (a.window == 0 || p > last - a.window || p < a.sinks);
                s[4 * t + r] = seen ? v : -__builtin_inff();
                mx = fmaxf(mx, s[4 * t + r]);
            }
        }
        mx = xhalf_max(xrow16_max(mx));
        const float mn = fmaxf(m, mx), ms = mn == -__builtin_inff() ? 0.0f : mn;
        const float al = __builtin_amdgcn_exp2f(m - ms);
        m = mn;
        // a column that sees none of this block takes nothing of it, its scale neither
        const float vf = mx == -__builtin_inff() ? 0.0f : vs[b] * 0x1p-30f;
        i32x4 pd[4];
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            uint32_t n[4], d[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float p = __builtin_amdgcn_exp2f(s[4 * t + r] - ms);
                sum += p;
                n[r] = signed_digits((int)rintf(p * 0x1p30f));
            }
            digits4(n[0], n[1], n[2], n[3], d);
#pragma unroll
            for (int e = 0; e < 4; e++) pd[e][t] = (int)d[e];
        }
        l = fmaf(l, al, sum);
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            const i32x4 va = *reinterpret_cast<const i32x4 *>(vt + (16 * dt + c) * 64 + 16 * g);
            i32x4 acc[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const i32x4 z = {0, 0, 0, 0};
                acc[e] = __builtin_amdgcn_mfma_i32_16x16x64_i8(va, pd[e], z, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float pv = fmaf((float)(acc[3][r] * 256 + acc[2][r]), 65536.0f, (float)(acc[1][r] * 256 + acc[0][r]));
                o[dt][r] = fmaf(o[dt][r], al, pv * vf);
            }
        }
    }
    l = xhalf_sum(xrow16_sum(l));

    // the waves' parts
    if (g == 0) { ml_l[wid][0][c] = m; ml_l[wid][1][c] = l; }
#pragma unroll
    for (int dt = 0; dt < DT; dt++) *reinterpret_cast<f32x4 *>(&o_l[wid][c][16 * dt + 4 * g]) = o[dt];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (HD / 4); i += 64 * W) {
        const int col = i / (HD / 4), d = 4 * (i % (HD / 4));
        const int64_t f = f0 + col;
        if (f >= n_flat) continue;
        float mm = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < W; w++) mm = fmaxf(mm, ml_l[w][0][col]);
        const float ms = mm == -__builtin_inff() ? 0.0f : mm;
        float ll = 0.0f;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float e = __builtin_amdgcn_exp2f(ml_l[w][0][col] - ms);
            ll = fmaf(ml_l[w][1][col], e, ll);
            const f32x4 ow = *reinterpret_cast<const f32x4 *>(&o_l[w][col][d]);
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] = fmaf(ow[r], e, v[r]);
        }
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = ll == 0.0f ? 0.0f : __fdiv_rn(v[r], ll);
        const int64_t at = ((sq.r0 + f / a.G) * a.Hq + (int64_t)h * a.G + f % a.G) * HD + d;
        if (BF16) {
            uint16_t *p = reinterpret_cast<uint16_t *>(a.out) + at;
#pragma unroll
            for (int r = 0; r < 4; r++) p[r] = __builtin_bit_cast(uint16_t, (__bf16)v[r]);
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
}

hipError_t launch_attention_kv8(const AttnKv8Args &a0, bool bf16, hipStream_t st) {
    AttnKv8Args a = a0;
    if ((a.c.hd != 64 && a.c.hd != 128) || a.c.n_seq > 65535 || a.c.Hkv > 65535) return hipErrorInvalidValue;
    a.vec_q = kv8_vec(a.q, nullptr, a.ldq, bf16 ? 2 : 4);
    a.vec_o = (uintptr_t)a.out % 16 == 0;
    const int64_t tiles = (a.c.max_rows * a.G + 15) / 16;
    if (tiles > INT32_MAX) return hipErrorInvalidValue;
    const dim3 grid((unsigned)tiles, (unsigned)a.c.Hkv, (unsigned)a.c.n_seq), blk(64 * QASR_KV8_WAVES);
    if (bf16) {
        if (a.c.hd == 128) hipLaunchKernelGGL((k_attn_kv8<true, 128>), grid, blk, 0, st, a);
        else hipLaunchKernelGGL((k_attn_kv8<true, 64>), grid, blk, 0, st, a);
    } else {
        if (a.c.hd == 128) hipLaunchKernelGGL((k_attn_kv8<false, 128>), grid, blk, 0, st, a);
        else hipLaunchKernelGGL((k_attn_kv8<false, 64>), grid, blk, 0, st, a);
    }
    return hipGetLastError();
}

}  // namespace qasr
