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

// the value of 4 consecutive columns n .. n + 3 of row m (n % 4 == 0) and its store
template <int MODE, typename YT>
struct Gemm8Out {
    const Gemm8Args &g;
    bool vec;                                        // y rows hold aligned runs of 4
    __device__ __forceinline__ static float in(const float *p) { return *p; }
    __device__ __forceinline__ static float in(const uint16_t *p) { return bf16_to_f32(*p); }
    __device__ __forceinline__ static void out(float *p, float v) { *p = v; }
    __device__ __forceinline__ static void out(uint16_t *p, float v) { *p = __builtin_bit_cast(uint16_t, (__bf16)v); }
    __device__ __forceinline__ void operator()(int64_t m, int64_t n, i32x4 acc, float as, f32x4 ws, f32x4 bias) const {
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = __fmul_rn(__fmul_rn((float)acc[r], as), ws[r]);
        YT *y = reinterpret_cast<YT *>(g.y);
        if constexpr (MODE == G8_SWIGLU) {
            y += m * (g.N >> 1) + (n >> 1);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float gt = __fadd_rn(v[2 * e], bias[2 * e]), up = __fadd_rn(v[2 * e + 1], bias[2 * e + 1]);
                if (n + 2 * e < g.N) out(y + e, __fmul_rn(__fdiv_rn(gt, __fadd_rn(1.0f, expf(-gt))), up));
            }
        } else {
            y += m * g.N + n;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                if (n + r >= g.N) continue;
                if constexpr (MODE == G8_ADDTO) v[r] = __fadd_rn(__fadd_rn(in(y + r), bias[r]), v[r]);
                else v[r] = __fadd_rn(v[r], bias[r]);
                out(y + r, v[r]);
            }
        }
    }
};

// The general form: 64 x 64 tiles, four waves of 32 x 32, K-steps of 64 through a
// pair of LDS buffers; every size and alignment (rows that are not 16-byte
// aligned and the last K-step are read byte by byte).
template <int MODE, typename YT>
__global__ __launch_bounds__(256) void k_gemm8_any(Gemm8Args g, int vec_k) {
    constexpr int BK = 64, LDK = BK + 16;
    __shared__ __attribute__((aligned(16))) int8_t As[2][64][LDK], Ws[2][64][LDK];
    const int t = threadIdx.x, lane = t & 63;
    const int wid = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = (wid & 1) * 32, wn = (wid >> 1) * 32;
    const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
    const int64_t K = g.K;
    const int lr = t >> 2, lk = (t & 3) * 16;        // this thread's 16 bytes of a 64 x 64 tile
    const int8_t *ap = g.a + min(m0 + lr, g.M - 1) * K, *wp = g.w + min(n0 + lr, g.N - 1) * K;
    i32x4 ar, wr;
    auto load16 = [&](const int8_t *p, int64_t k) {
        i32x4 v = {0, 0, 0, 0};
        if (vec_k && k + 16 <= K) return *reinterpret_cast<const i32x4 *>(p + k);
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (k + i < K) v[i >> 2] |= (int)(uint8_t)p[k + i] << (8 * (i & 3));
        return v;
    };
    ar = load16(ap, lk);
    wr = load16(wp, lk);
    i32x4 acc[2][2] = {};
    const int fr = lane & 15, fg = lane >> 4;
    const int64_t nk = (K + BK - 1) / BK;
    for (int64_t kt = 0; kt < nk; kt++) {
        const int b = kt & 1;
        *reinterpret_cast<i32x4 *>(&As[b][lr][lk]) = ar;
        *reinterpret_cast<i32x4 *>(&Ws[b][lr][lk]) = wr;
        __syncthreads();
        if (kt + 1 < nk) {
            ar = load16(ap, (kt + 1) * BK + lk);
            wr = load16(wp, (kt + 1) * BK + lk);
        }
        i32x4 af[2], wf[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            af[i] = *reinterpret_cast<const i32x4 *>(&As[b][wm + 16 * i + fr][16 * fg]);
            wf[i] = *reinterpret_cast<const i32x4 *>(&Ws[b][wn + 16 * i + fr][16 * fg]);
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], af[i], acc[i][j], 0, 0, 0);
    }
    const Gemm8Out<MODE, YT> put{g, false};
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int64_t n = n0 + wn + 16 * j + 4 * fg;
        if (n >= g.N) continue;
        f32x4 ws, bias = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < 4; r++) {
            ws[r] = g.ws[min(n + r, g.N - 1)];
            if (g.bias) bias[r] = g.bias[min(n + r, g.N - 1)];
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int64_t m = m0 + wm + 16 * i + fr;
            if (m < g.M) put(m, n, acc[i][j], g.as[m], ws, bias);
        }
    }
}

template <int MODE, typename YT>
static hipError_t go_gemm8(const Gemm8Args &g, hipStream_t st) {
    const int vec_k = g.K % 16 == 0 && ((uintptr_t)g.a | (uintptr_t)g.w) % 16 == 0;
    const int64_t gx = (g.N + 63) / 64, gy = (g.M + 63) / 64;
    if (gy > 65535 || gx > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_gemm8_any<MODE, YT>), dim3((unsigned)gx, (unsigned)gy), dim3(256), 0, st, g, vec_k);
    return hipGetLastError();
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
