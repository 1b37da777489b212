// int8 x int8 products with a scale for each row and each column:
//
//   y[m, n] = ((float)(sum_k a[m, k] w[n, k]) * as[m]) * ws[n] (+ bias[n])
//
// on v_mfma_i32_16x16x64_i8.  The weights are the MFMA's rows and the activations
// its columns, so a lane ends with four consecutive n of one m: interleaved gate
// and up rows meet in one lane, and a row's stores are 16 bytes wide.
#include "kernels.h"
#include "gemm_common.h"

namespace qasr {

// y's types; 4 values at a time at any element's address, which the hardware takes (2021
// x 4999 x 1024 to bf16: 21.0 us, 25.9 with the odd rows stored value by value).  STREAM:
// past the caches
template <typename YT>
struct Gemm8Io;
template <>
struct Gemm8Io<float> {
    typedef float Any4 __attribute__((ext_vector_type(4), aligned(4)));
    __device__ __forceinline__ static float in(const float *p) { return *p; }
    __device__ __forceinline__ static f32x4 in4(const float *p) { return *reinterpret_cast<const Any4 *>(p); }
    __device__ __forceinline__ static void out(float *p, float v) { *p = v; }
    template <bool STREAM>
    __device__ __forceinline__ static void out4(float *p, f32x4 v) {
        if (STREAM) __builtin_nontemporal_store((Any4)v, reinterpret_cast<Any4 *>(p));
        else *reinterpret_cast<Any4 *>(p) = v;
    }
};
template <>
struct Gemm8Io<uint16_t> {
    typedef uint16_t Any4 __attribute__((ext_vector_type(4), aligned(2)));
    __device__ __forceinline__ static float in(const uint16_t *p) { return bf16_to_f32(*p); }
    __device__ __forceinline__ static f32x4 in4(const uint16_t *p) {
        const Any4 u = *reinterpret_cast<const Any4 *>(p);
        return f32x4{bf16_to_f32(u[0]), bf16_to_f32(u[1]), bf16_to_f32(u[2]), bf16_to_f32(u[3])};
    }
    __device__ __forceinline__ static void out(uint16_t *p, float v) { *p = __builtin_bit_cast(uint16_t, (__bf16)v); }
    template <bool STREAM>
    __device__ __forceinline__ static void out4(uint16_t *p, f32x4 v) {
        Any4 u;
#pragma unroll
        for (int r = 0; r < 4; r++) u[r] = __builtin_bit_cast(uint16_t, (__bf16)v[r]);
        if (STREAM) __builtin_nontemporal_store(u, reinterpret_cast<Any4 *>(p));
        else *reinterpret_cast<Any4 *>(p) = u;
    }
};

// what 4 consecutive columns of a row give: 4 results, for SwiGLU 2 in front; ADDTO
// without bias, which belongs to the old value
template <int MODE>
__device__ __forceinline__ f32x4 gemm8_value(i32x4 acc, float as, f32x4 ws, f32x4 bias) {
    f32x4 v;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        v[r] = __fmul_rn(__fmul_rn((float)acc[r], as), ws[r]);
        if (MODE != G8_ADDTO) v[r] = __fadd_rn(v[r], bias[r]);
    }
    if (MODE == G8_SWIGLU) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const float gt = v[2 * e], up = v[2 * e + 1];
            v[e] = __fmul_rn(__fdiv_rn(gt, __fadd_rn(1.0f, expf(-gt))), up);
        }
    }
    return v;
}

// 16 bytes of a row from byte k on, `left` of them before the row's end (K bytes), zeros
// behind it; rows begin at any address, which the hardware's vector loads take
__device__ __forceinline__ i32x4 gemm8_row16(const int8_t *p, int left, int K) {
    typedef int Any __attribute__((ext_vector_type(4), aligned(1)));
    if (left >= 16) return *reinterpret_cast<const Any *>(p);
    i32x4 v = {0, 0, 0, 0};
    if (left <= 0) return v;
    if (K >= 16) {                                           // the row's last 16, moved down
        v = *reinterpret_cast<const Any *>(p + left - 16);
        const int sh = 8 * (16 - left);
        uint64_t lo = (uint32_t)v[0] | (uint64_t)(uint32_t)v[1] << 32, hi = (uint32_t)v[2] | (uint64_t)(uint32_t)v[3] << 32;
        lo = sh < 64 ? lo >> sh | hi << (64 - sh) : hi >> (sh - 64);
        hi = sh < 64 ? hi >> sh : 0;
        return i32x4{(int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32)};
    }
#pragma unroll
    for (int i = 0; i < 15; i++)
        if (i < left) v[i >> 2] |= (int)(uint8_t)p[i] << (8 * (i & 3));
    return v;
}

// BM x BN tiles fed by direct global -> LDS loads through rings of two
// stages of BK = 128 bytes of K, one in flight while one is multiplied.  KP groups of
// WM x WN waves each take every KP-th K-step through a ring of their own and add up in
// LDS at the end (int32: exact in any order): a short grid or few rows leave a CU few
// waves otherwise, and a long chain of K-steps for each.
//
// What bounds it is the way from the caches into LDS.  Such loads, with nothing else
// running, bring 34 TB/s when a row gives 128 bytes and lies in the XCD's L2, 20 when it
// gives 64, 7-8 when it comes from the cache behind the L2s (375 x 151936 x 1024, 192 x
// 128 tiles: 142 us with 64-byte steps and three stages, 107 with these; more stages or
// larger tiles leave too few waves on a CU).  Hence also the order of the tiles, below.
//
// A stage holds the tile's activation rows, then its weight rows, in 16-byte slots;
// slot q of row r stands at q ^ lds_swz(r).  A load fills 64 slots in lane order.
// K-steps past the end load zeros, so every wait counts the same.
//
// ANY: K % 16 != 0 or operands that are not 16-byte aligned, which the direct loads do
// not take: the same slots through registers, a step ahead.
__device__ __attribute__((aligned(256))) int4 g_gemm8_zero16[16];

template <int MODE, typename YT, int BM, int BN, int WM, int WN, int KP, bool STREAM, bool ANY>
__global__ __launch_bounds__(64 * WM * WN * KP, KP == 1 ? 4 : 2) void k_gemm8(Gemm8Args g) {
    constexpr int BK = 128, NS = 2, W = WM * WN, MT = BM / WM / 16, NT = BN / WN / 16, RPL = 1024 / BK, SPR = BK / 16;
    constexpr int LA = BM / RPL / W, LB = BN / RPL / W, STG = (BM + BN) * BK;
    static_assert(BM % (RPL * W) == 0 && BN % (RPL * W) == 0 && BM % (16 * WM) == 0 && BN % (16 * WN) == 0, "tile");
    // after the K loop: the groups' partial sums, then 16 rows of each wave's results
    constexpr int RED = (KP - 1) * W * MT * NT * 4 * 64 * 4, OC = BN / WN / (MODE == G8_SWIGLU ? 2 : 1), OP = OC + 4;
    constexpr int END = RED + W * 16 * OP * 4;
    __shared__ __attribute__((aligned(16))) char smem[KP * NS * STG > END ? KP * NS * STG : END];
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6), grp = wave / W, w = wave % W, wm = w % WM, wn = w / WM;
    const int fr = lane & 15, fg = lane >> 4;
    const int64_t M = g.M, N = g.N, K = g.K;
    // blocks go to the 8 XCDs in turn: the row tiles of a strip of weights follow one
    // another on one XCD, whose L2 then holds the strip once.  (Row tiles that begin at
    // different K-steps, for weights past the caches, gain 4% at 375 x 151936 x 1024 and 2000 x
    // 60000 x 2048 and lose 9% at 404 x 20000 x 6144, 6% at 1337 x 24576 x 6144, 3% at 250 x
    // 151936 x 2048: left out.)
    const unsigned rows = (unsigned)((M + BM - 1) / BM), xcd = blockIdx.x & 7, q = blockIdx.x >> 3;
    const unsigned strip = q / rows * 8 + xcd;
    const unsigned row = q - q / rows * rows;
    const int64_t m0 = (int64_t)row * BM, n0 = (int64_t)strip * BN;
    if (n0 >= N) return;
    char *ring = smem + grp * NS * STG;
    const int nk = (int)((K + BK - 1) / BK), nit = (nk + KP - 1) / KP;
    // the epilogue's operands, ahead of the ring's loads
    f32x4 ws[NT], bias[NT];
    float as[MT];
    const bool sv = ((uintptr_t)g.ws & 15) == 0, bv = ((uintptr_t)g.bias & 15) == 0;
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int64_t n = n0 + wn * (BN / WN) + 16 * j + 4 * fg;
        const int nn = (int)min(n, N - 1);
        ws[j] = gemm_load4(g.ws, nn, (int)N, sv && nn == n);
        bias[j] = g.bias ? gemm_load4(g.bias, nn, (int)N, bv && nn == n) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll
    for (int i = 0; i < MT; i++) as[i] = g.as[min(m0 + wm * (BM / WM) + 16 * i + fr, M - 1)];
    // this lane's row and 16-byte slot in each of the wave's loads
    const int lr = lane / SPR, lq = lane % SPR;
    const int8_t *src[LA + LB];
    int sq[LA + LB];
#pragma unroll
    for (int u = 0; u < LA + LB; u++) {
        const int r = (u < LA ? w * LA + u : w * LB + u - LA) * RPL + lr;
        sq[u] = 16 * (lq ^ lds_swz<BK>(r));
        src[u] = (u < LA ? g.a + min(m0 + r, M - 1) * K : g.w + min(n0 + r, N - 1) * K) + sq[u];
    }
    const int8_t *zero = reinterpret_cast<const int8_t *>(g_gemm8_zero16);
    // the byte of K that this group's step begins with; past the end: K, nothing but zeros
    auto step = [&](int it) {
        const int kt = grp + KP * it;
        return kt < nk ? kt * BK : (int)K;
    };
    auto issue = [&](int stage, int it) {
        char *st = ring + stage * STG;
        const int k0 = step(it);
        const bool whole = k0 + BK <= K;
#pragma unroll
        for (int u = 0; u < LA + LB; u++) {
            char *to = st + (u < LA ? 1024 * (w * LA + u) : BM * BK + 1024 * (w * LB + u - LA));
            lds_dma16(whole || k0 + sq[u] < K ? src[u] + k0 : zero, to);
        }
    };
    // ANY: the step's slots into registers, and from there into a stage
    i32x4 held[LA + LB];
    auto load = [&](int it) {
        const int k0 = step(it);
#pragma unroll
        for (int u = 0; u < LA + LB; u++) {
            typedef int Any __attribute__((ext_vector_type(4), aligned(1)));
            if (k0 + BK <= K) held[u] = *reinterpret_cast<const Any *>(src[u] + k0);
            else held[u] = gemm8_row16(src[u] + k0, (int)K - k0 - sq[u], (int)K);
        }
    };
    auto store = [&](int stage) {
        char *st = ring + stage * STG + 16 * lane;
#pragma unroll
        for (int u = 0; u < LA + LB; u++)
            *reinterpret_cast<i32x4 *>(st + (u < LA ? 1024 * (w * LA + u) : BM * BK + 1024 * (w * LB + u - LA))) = held[u];
    };
    i32x4 acc[NT][MT] = {};
    if constexpr (ANY) {
        load(0);
        store(0);
        load(1);
    } else {
        issue(0, 0);
    }
    for (int it = 0; it < nit; it++) {
        if constexpr (!ANY) wait_vmcnt<0>();                 // this wave's loads of the stage have landed
        __syncthreads();                                     // ... and every wave's; the stage before is free
        if constexpr (!ANY) issue((it + 1) % NS, it + 1);
        const char *at = ring + (it % NS) * STG, *wt = at + BM * BK;
#pragma unroll
        for (int s = 0; s < BK / 64; s++) {
            i32x4 af[MT], wf[NT];
#pragma unroll
            for (int i = 0; i < MT; i++) {
                const int r = wm * (BM / WM) + 16 * i + fr;
                af[i] = *reinterpret_cast<const i32x4 *>(at + r * BK + 16 * ((4 * s + fg) ^ lds_swz<BK>(r)));
            }
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const int r = wn * (BN / WN) + 16 * j + fr;
                wf[j] = *reinterpret_cast<const i32x4 *>(wt + r * BK + 16 * ((4 * s + fg) ^ lds_swz<BK>(r)));
            }
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int i = 0; i < MT; i++) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], af[i], acc[j][i], 0, 0, 0);
        }
        if constexpr (ANY) {
            store((it + 1) % NS);
            load(it + 2);
        }
    }
    wait_vmcnt<0>();                                         // no load may land in LDS after the block ends
    __syncthreads();
    if constexpr (KP > 1) {
        int *red = reinterpret_cast<int *>(smem);
        if (grp > 0) {
            int *dst = red + ((grp - 1) * W + w) * MT * NT * 256 + lane;
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) dst[((j * MT + i) * 4 + r) * 64] = acc[j][i][r];
        }
        __syncthreads();
        if (grp > 0) return;
#pragma unroll
        for (int p = 1; p < KP; p++) {
            const int *from = red + ((p - 1) * W + w) * MT * NT * 256 + lane;
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[j][i][r] += from[((j * MT + i) * 4 + r) * 64];
        }
    }
    // 16 rows at a time through the wave's own LDS, so that a store covers whole runs of a
    // row: lanes as the products leave them hold 64 bytes of each of 16 rows
    float *tr = reinterpret_cast<float *>(smem + RED) + w * 16 * OP;
    const int64_t cols = MODE == G8_SWIGLU ? N >> 1 : N, c0 = (n0 + wn * (BN / WN)) / (MODE == G8_SWIGLU ? 2 : 1);
    YT *y = reinterpret_cast<YT *>(g.y);
#pragma unroll
    for (int i = 0; i < MT; i++) {
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const f32x4 v = gemm8_value<MODE>(acc[j][i], as[i], ws[j], bias[j]);
            if constexpr (MODE == G8_SWIGLU) *reinterpret_cast<f32x2 *>(tr + fr * OP + 8 * j + 2 * fg) = f32x2{v[0], v[1]};
            else *reinterpret_cast<f32x4 *>(tr + fr * OP + 16 * j + 4 * fg) = v;
        }
        wave_lds_fence();                                    // the rows change lanes
        const int64_t m = m0 + wm * (BM / WM) + 16 * i;
        if (n0 + BN <= N) {
#pragma unroll
            for (int e = lane; e < 16 * (OC / 4); e += 64) {
                const int r = e / (OC / 4), cc = 4 * (e % (OC / 4));
                f32x4 v = *reinterpret_cast<const f32x4 *>(tr + r * OP + cc);
                if (m + r < M) {
                    YT *p = y + (m + r) * cols + c0 + cc;
                    if constexpr (MODE == G8_ADDTO) {
                        const f32x4 y0 = Gemm8Io<YT>::in4(p);
#pragma unroll
                        for (int k = 0; k < 4; k++) v[k] = __fadd_rn(__fadd_rn(y0[k], g.bias ? g.bias[c0 + cc + k] : 0.0f), v[k]);
                    }
                    Gemm8Io<YT>::template out4<STREAM>(p, v);
                }
            }
        } else {                                         // the last strip of columns: 4 or what is left of them
#pragma unroll
            for (int e = lane; e < 16 * (OC / 4); e += 64) {
                const int r = e / (OC / 4), cc = 4 * (e % (OC / 4)), n = (int)min(cols - c0 - cc, (int64_t)4);
                f32x4 v = *reinterpret_cast<const f32x4 *>(tr + r * OP + cc);
                if (m + r >= M || n <= 0) continue;
                YT *p = y + (m + r) * cols + c0 + cc;
                if constexpr (MODE == G8_ADDTO) {
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (k < n) v[k] = __fadd_rn(__fadd_rn(Gemm8Io<YT>::in(p + k), g.bias ? g.bias[c0 + cc + k] : 0.0f), v[k]);
                }
                if (n == 4) {
                    Gemm8Io<YT>::template out4<STREAM>(p, v);
                } else {
#pragma unroll
                    for (int k = 0; k < 3; k++)
                        if (k < n) Gemm8Io<YT>::out(p + k, v[k]);
                }
            }
        }
        wave_lds_fence();                                    // read, before the next 16 rows come
    }
}

template <int MODE, typename YT, int BM, int BN, int WM, int WN, int KP, bool STREAM = false, bool ANY = false>
static hipError_t go_gemm8_tile(const Gemm8Args &g, hipStream_t st) {
    const int64_t gx = (g.N + BN - 1) / BN, gy = (g.M + BM - 1) / BM;
    const int64_t blocks = (gx + 7) / 8 * 8 * gy;
    if (blocks * 64 * WM * WN * KP > UINT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_gemm8<MODE, YT, BM, BN, WM, WN, KP, STREAM, ANY>), dim3((unsigned)blocks), dim3(64 * WM * WN * KP), 0, st, g);
    return hipGetLastError();
}

// The form with the least estimated time: ns for the first round of tiles over the 256 CUs
// (fixed, and for each 64 of K), and for each further round.  Fits to 257 shapes, M 1 ...
// 2000, N 512 ... 151936, K 320 ... 6144; of nine forms and 290 shapes the choice is 2.5%
// behind the best on average, 50% at worst (1 x 60000 x 512: 12.4 us, 8.1 with 64 x 128
// tiles, which elsewhere gain too little to be told apart).  us, in the order of the list:
// 32 x 2048 x 6144 8.0, 10.3, 17.5, 31, 37; 32 x 12288 x 2048 12.4, 7.3, 9.2, 13, 16; 404 x
// 4096 x 1024 34, 17.0, 8.2, 9.9, 12.2; 2000 x 4096 x 1024 155, 68, 25.8, 17.8, 18.0; 1337 x
// 12288 x 2048 409, 208, 78, 49.5, 42.7; 375 x 151936 x 1024 1153, 562, 217, 120, 109.
struct Gemm8Form { int bm, bn, one, one_k, more, more_k; };
static const Gemm8Form g8_forms[] = {{16, 32, 3531, 47, 1969, 42},
                                     {16, 32, 2908, 70, 792, 20},
                                     {64, 64, 3529, 141, 1877, 70},
                                     {128, 128, 4831, 297, 2450, 218},
                                     {192, 128, 6170, 381, 3731, 256}};
// the same where operands come through registers; 169 shapes, K 319 ... 6143: 1% behind the
// best of the four on average, 11% at worst (64 x 4096 x 319).  16 x 2048 x 6143 12.6, 13.4,
// 23.5, 44; 404 x 4096 x 1023 71, 38, 12.8, 12.8; 2000 x 4999 x 1023 420, 195, 55, 34.5
static const Gemm8Form g8_any_forms[] = {{16, 32, 5771, 73, 4046, 78},
                                         {16, 32, 5320, 84, 1037, 60},
                                         {64, 64, 5453, 169, 1625, 195},
                                         {128, 128, 5859, 401, 3659, 428}};
static int gemm8_form(const Gemm8Form *f, int n, const Gemm8Args &g) {
    const int64_t nk = (g.K + 63) / 64;
    int best = 0;
    int64_t best_ns = INT64_MAX;
    for (int i = 0; i < n; i++) {
        const int64_t tiles = (g.M + f[i].bm - 1) / f[i].bm * ((g.N + f[i].bn - 1) / f[i].bn), rounds = (tiles + 255) / 256;
        const int64_t ns = f[i].one + f[i].one_k * nk + (rounds - 1) * (f[i].more + f[i].more_k * nk);
        if (ns < best_ns) { best_ns = ns; best = i; }
    }
    return best;
}

template <int MODE, typename YT>
static hipError_t go_gemm8(const Gemm8Args &g, hipStream_t st) {
    if (g.K % 16 != 0 || ((uintptr_t)g.a | (uintptr_t)g.w) % 16 != 0) {
        switch (gemm8_form(g8_any_forms, 4, g)) {
            case 0: return go_gemm8_tile<MODE, YT, 16, 32, 1, 1, 8, false, true>(g, st);
            case 1: return go_gemm8_tile<MODE, YT, 16, 32, 1, 1, 4, false, true>(g, st);
            case 2: return go_gemm8_tile<MODE, YT, 64, 64, 2, 2, 2, false, true>(g, st);
            default: return go_gemm8_tile<MODE, YT, 128, 128, 2, 4, 1, false, true>(g, st);
        }
    }
    // Results of 32 MB and more whose rows are whole 64-byte pieces go past the caches: f32,
    // 1337 x 12288 x 2048 50.0 -> 43.0 us, 404 x 60000 x 512 43 -> 32, 1000 x 60000 x 512 90 -> 64,
    // 375 x 151936 x 1024 110 -> 107.  A smaller result is better left for its reader (a layer of
    // 404 rows 77.0 us in all, 78.3 with every result past the caches); rows in odd pieces have to
    // meet in a cache (2021 x 4999 bf16 18.8 us, 24.5).
    constexpr bool CAN = MODE != G8_ADDTO;      // which gains nothing: its result was read just before
    const int64_t row = (MODE == G8_SWIGLU ? g.N / 2 : g.N) * (int64_t)sizeof(YT);
    const bool stream = g.M * row >= (1 << 25) && row % 64 == 0 && (uintptr_t)g.y % 64 == 0;
    switch (gemm8_form(g8_forms, 5, g)) {
        case 0: return go_gemm8_tile<MODE, YT, 16, 32, 1, 1, 8>(g, st);
        case 1: return go_gemm8_tile<MODE, YT, 16, 32, 1, 1, 4>(g, st);
        case 2: return go_gemm8_tile<MODE, YT, 64, 64, 2, 2, 2>(g, st);
        case 3: return stream ? go_gemm8_tile<MODE, YT, 128, 128, 2, 4, 1, CAN>(g, st) : go_gemm8_tile<MODE, YT, 128, 128, 2, 4, 1>(g, st);
        default: return stream ? go_gemm8_tile<MODE, YT, 192, 128, 2, 4, 1, CAN>(g, st) : go_gemm8_tile<MODE, YT, 192, 128, 2, 4, 1>(g, st);
    }
}

hipError_t launch_gemm_w8a8(const Gemm8Args &g, int mode, bool y_bf16, hipStream_t st) {
    if (g.M <= 0 || g.N <= 0 || g.K <= 0 || g.K >= 131072) return hipErrorInvalidValue;
    switch (mode) {
#define QG(MODE) \
    case MODE: return y_bf16 ? go_gemm8<MODE, uint16_t>(g, st) : go_gemm8<MODE, float>(g, st);
        QG(G8_PLAIN) QG(G8_ADDTO) QG(G8_SWIGLU)
#undef QG
        default: return hipErrorInvalidValue;
    }
}

}  // namespace qasr
