// int8 activation rows: the residual's addition, RMSNorm and the rounding to
// int8 with one scale a row, in one pass.
//
//   s = x + res,  n = s / rms(s) * g,  scale = max|n| / 127,  q = round(n / scale)
//
// 1 / rms(s) is common to a row and cancels in q: q = round(127 t / max|t|) with
// t = s g, so one pass over the registers decides q from the row's maximum alone
// and the sum of squares only enters the scale.  Memory bound: x and res read
// once, s and q written once (13 bytes a value in f32, 7 in bf16), the row held in
// registers between the reductions and the stores.  Sums and decisions are in f64:
// the vector unit runs f64 at the f32 rate, and int8 values then do not depend on
// the order of a sum (next to a half an f32 product rounds either way).
#include "kernels.h"

namespace qasr {

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, QASR_WAVE);
    return v;
}
__device__ __forceinline__ double wave_max_f64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o, QASR_WAVE));
    return v;
}

// 8 consecutive values of a row from element e on (those past H: 0)
template <bool BF16, bool VEC>
__device__ __forceinline__ void load8(const void *base, int64_t row0, int e, int H, float *v) {
    if (BF16) {
        const uint16_t *p = reinterpret_cast<const uint16_t *>(base) + row0 + e;
        if (VEC) {
            const u16x8 u = *reinterpret_cast<const u16x8 *>(p);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = bf16_to_f32(u[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = e + i < H ? bf16_to_f32(p[i]) : 0.0f;
        }
    } else {
        const float *p = reinterpret_cast<const float *>(base) + row0 + e;
        if (VEC) {
            const f32x4 a = reinterpret_cast<const f32x4 *>(p)[0], b = reinterpret_cast<const f32x4 *>(p)[1];
#pragma unroll
            for (int i = 0; i < 4; i++) { v[i] = a[i]; v[4 + i] = b[i]; }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = e + i < H ? p[i] : 0.0f;
        }
    }
}

// f32 -> bf16, nearest even, any input
__device__ __forceinline__ uint16_t to_bf16(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }

// STREAM: past the caches
template <bool STREAM, typename V>
__device__ __forceinline__ void put(V *p, V v) {
    if (STREAM) __builtin_nontemporal_store(v, p);
    else *p = v;
}

template <bool BF16, bool VEC, bool STREAM>
__device__ __forceinline__ void store8(void *base, int64_t row0, int e, int H, const float *v) {
    if (BF16) {
        uint16_t *p = reinterpret_cast<uint16_t *>(base) + row0 + e;
        if (VEC) {
            u16x8 u;
#pragma unroll
            for (int i = 0; i < 8; i++) u[i] = to_bf16(v[i]);
            put<STREAM>(reinterpret_cast<u16x8 *>(p), u);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (e + i < H) p[i] = to_bf16(v[i]);
        }
    } else {
        float *p = reinterpret_cast<float *>(base) + row0 + e;
        if (VEC) {
            put<STREAM>(reinterpret_cast<f32x4 *>(p), f32x4{v[0], v[1], v[2], v[3]});
            put<STREAM>(reinterpret_cast<f32x4 *>(p) + 1, f32x4{v[4], v[5], v[6], v[7]});
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (e + i < H) p[i] = v[i];
        }
    }
}

// One block of T threads a row; thread t holds the 8-value chunks t, t + T, ...
// (C of them).  VEC: H and ld multiples of 8, 16-byte aligned buffers.
template <bool BF16, bool VEC, bool STREAM, int T, int C>
__global__ __launch_bounds__(T) void k_add_rms_norm_int8(Rows8Args a) {
    constexpr int W = T / 64;
    __shared__ double red[2][W];
    __shared__ int bad_l[W];
    const int t = threadIdx.x, lane = t & 63, wid = t >> 6;
    const int64_t row = blockIdx.x;
    const int H = a.H;
    const int64_t r0 = row * a.ld;
    double tv[C][8];
    double ss = 0.0, mx = 0.0;
    bool bad = false;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int e = (c * T + t) * 8;
#pragma unroll
        for (int i = 0; i < 8; i++) tv[c][i] = 0.0;
        if (e >= H) continue;
        float x[8], r[8], g[8], s[8];
        load8<BF16, VEC>(a.x, r0, e, H, x);
        if (a.res) load8<BF16, VEC>(a.res, r0, e, H, r);
        if (a.norm_w) load8<false, VEC>(a.norm_w, 0, e, H, g);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // f32 operands: the f64 sum is exact unless their exponents are 30 apart
            const double sd = a.res ? (double)x[i] + (double)r[i] : (double)x[i];
            s[i] = (float)sd;
            ss = fma(sd, sd, ss);
            const double td = a.norm_w ? sd * (double)g[i] : sd;
            tv[c][i] = td;
            bad |= !(fabs(td) <= 1.7976931348623157e308) || !(fabs(sd) <= 1.7976931348623157e308);
            mx = fmax(mx, fabs(td));
        }
        if (a.sum) store8<BF16, VEC, STREAM>(a.sum, r0, e, H, s);
    }
    ss = wave_sum_f64(ss);
    mx = wave_max_f64(mx);
    bad = __any(bad);
    if (W > 1) {
        if (lane == 0) { red[0][wid] = ss; red[1][wid] = mx; bad_l[wid] = bad; }
        __syncthreads();
        ss = 0.0;
        mx = 0.0;
        bad = false;
#pragma unroll
        for (int w = 0; w < W; w++) { ss += red[0][w]; mx = fmax(mx, red[1][w]); bad |= bad_l[w] != 0; }
    }
    if (t == 0) {
        double sc = mx / 127.0;
        if (a.norm_w) sc = sc / sqrt(ss / (double)H + (double)a.eps);
        a.scales[row] = bad ? __builtin_nanf("") : mx > 0.0 ? (float)sc : 1.0f;
    }
    const double inv = !bad && mx > 0.0 ? 127.0 / mx : 0.0;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int e = (c * T + t) * 8;
        if (e >= H) continue;
        int q[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int k = round_ratio(127.0 * fabs(tv[c][i]), mx, inv * (1.0 / 127.0));
            q[i] = inv == 0.0 ? 0 : tv[c][i] < 0.0 ? -k : k;
        }
        int8_t *p = a.q + row * H + e;
        if (VEC) {
            typedef int i32x2 __attribute__((ext_vector_type(2)));
            put<STREAM>(reinterpret_cast<i32x2 *>(p), i32x2{pack4_i8(q[0], q[1], q[2], q[3]), pack4_i8(q[4], q[5], q[6], q[7])});
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (e + i < H) p[i] = (int8_t)q[i];
        }
    }
}

// As many threads as the row has chunks, half as many in bf16, whose chunks are 16
// bytes: a wave then keeps as much in flight (12120 x 2048 bf16 with 256 and 128
// threads 42.6 and 39.6 us; f32 5000 x 2048 27.5 and 30.7).  From 2^23 values on the
// results go past the caches, which do not hold them until they are read (that case
// 45.5 -> 42.6 us with 256 threads).
template <bool BF16, bool VEC, bool STREAM>
static hipError_t go_rows8(const Rows8Args &a, hipStream_t st) {
    constexpr int C = BF16 ? 2 : 1;
    const dim3 grid((unsigned)a.rows);
    const int n = (a.H + 8 * C - 1) / (8 * C);
#define QR(T, CC) hipLaunchKernelGGL((k_add_rms_norm_int8<BF16, VEC, STREAM, T, CC>), grid, dim3(T), 0, st, a)
    if (n <= 64) QR(64, C);
    else if (n <= 128) QR(128, C);
    else if (n <= 256) QR(256, C);
    else if (n <= 512) QR(512, C);
    else if (n <= 1024) QR(1024, C);
    else QR(1024, 2);
#undef QR
    return hipGetLastError();
}

template <bool BF16, bool VEC>
static hipError_t pick_rows8(const Rows8Args &a, hipStream_t st) {
    if constexpr (VEC)
        if (a.rows * a.H >= (1 << 23)) return go_rows8<BF16, VEC, true>(a, st);
    return go_rows8<BF16, VEC, false>(a, st);
}

hipError_t launch_add_rms_norm_int8(const Rows8Args &a, bool bf16, hipStream_t st) {
    if (a.rows <= 0 || a.rows >= (1 << 22) || a.H <= 0 || a.H > QASR_ROWS8_MAX_HIDDEN) return hipErrorInvalidValue;
    const uintptr_t ptrs = (uintptr_t)a.x | (uintptr_t)a.res | (uintptr_t)a.sum | (uintptr_t)a.norm_w;
    const bool vec = a.H % 8 == 0 && a.ld % 8 == 0 && ptrs % 16 == 0 && (uintptr_t)a.q % 8 == 0;
    if (bf16) return vec ? pick_rows8<true, true>(a, st) : pick_rows8<true, false>(a, st);
    return vec ? pick_rows8<false, true>(a, st) : pick_rows8<false, false>(a, st);
}

}  // namespace qasr
