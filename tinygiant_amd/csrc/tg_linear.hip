// tg_linear.hip -- int8 matrix product with a scale per token and per
// channel: activations quantised on the way (after an RMS norm where one is
// given), v_mfma_i32_16x16x64_i8 tiles, scales and residual in the epilogue.
#include "tg_device.h"
#include "tg_internal.h"

#include "../../include/tinygiant.h"

namespace tg {

typedef int i32x4 __attribute__((ext_vector_type(4)));

TG_DEV float lin_get(const void *p, int type, int64_t i) {
    if (type == TG_T_F32) return static_cast<const float *>(p)[i];
    const uint16_t v = static_cast<const uint16_t *>(p)[i];
    return type == TG_T_F16 ? h2f(v) : __uint_as_float((uint32_t)v << 16);
}

TG_DEV void lin_put(void *p, int type, int64_t i, float v) {
    if (type == TG_T_F32) static_cast<float *>(p)[i] = v;
    else static_cast<uint16_t *>(p)[i] = type == TG_T_F16 ? f2h(v) : __builtin_bit_cast(uint16_t, (__bf16)v);
}

constexpr int LIN_K = 64;  // columns per step: rows of codes are padded to it with zeros

static int lin_kp(int K) { return (K + LIN_K - 1) / LIN_K * LIN_K; }

// ================================================================ quantise
// q = rint(127 x / a) of one value, decided by the exact quotient: half the
// row's largest value lies on a border (63.5).  t is within 1e-4 of the
// quotient (its two fp32 roundings are 2^-23 of at most 127).
TG_DEV int code_of(double x, double a, float inv) {
    const float t = (float)x * inv;
    const float r = __builtin_rintf(t);
    if (fabsf(t - r) < 0.4998f) return (int)r;
    return (int)__builtin_rint(127.0 * x / a);
}

// One block per row: mean square and largest magnitude in 64 bits (the
// codes do not depend on the order of the sum), codes and scale.
__global__ __launch_bounds__(256) void k_lin_quant(MatmulI8Args a, int Kp, int8_t *xq, float *xs) {
    __shared__ double red[4];
    const int row = blockIdx.x, tid = threadIdx.x;
    const int64_t x0 = (int64_t)row * a.x_stride;
    double r = 1.0;
    if (a.norm_w) {
        double ss = 0.0;
        for (int k = tid; k < a.K; k += 256) {
            const double x = lin_get(a.x, a.x_type, x0 + k);
            ss += x * x;
        }
        for (int m = 1; m < 64; m *= 2) ss += __shfl_xor(ss, m);
        if (tid % 64 == 0) red[tid / 64] = ss;
        __syncthreads();
        r = 1.0 / __builtin_sqrt((red[0] + red[1] + red[2] + red[3]) / a.K + a.eps);
        __syncthreads();
    }
    auto at = [&](int k) {
        const double x = lin_get(a.x, a.x_type, x0 + k);
        return a.norm_w ? x * r * (double)a.norm_w[k] : x;
    };
    double top = 0.0;
    for (int k = tid; k < a.K; k += 256) {
        const double v = fabs(at(k));
        top = fmax(top, v < INFINITY ? v : INFINITY);  // NaN counts as infinite
    }
    for (int m = 1; m < 64; m *= 2) top = fmax(top, __shfl_xor(top, m));
    if (tid % 64 == 0) red[tid / 64] = top;
    __syncthreads();
    top = fmax(fmax(red[0], red[1]), fmax(red[2], red[3]));
    const bool bad = !(top < INFINITY);
    const float inv = bad || top == 0.0 ? 0.0f : (float)(127.0 / top);
    for (int k = tid; k < Kp; k += 256)
        xq[(size_t)row * Kp + k] = (int8_t)(k < a.K && inv != 0.0f ? code_of(at(k), top, inv) : 0);
    if (tid == 0) xs[row] = bad ? __builtin_nanf("") : (float)(top / 127.0);
}

// ================================================================ product
// 64 channels x 64 rows per block, 4 waves of 32 x 32.
__global__ __launch_bounds__(256) void k_lin_mm(MatmulI8Args a, int Kp, const int8_t *xq, const float *xs) {
    __shared__ __align__(16) int8_t sw[64][80], sx[64][80];
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int n0 = blockIdx.x * 64, m0 = blockIdx.y * 64;
    const int r = tid / 4, c = (tid % 4) * 16;
    const int8_t *wp = a.w + (size_t)min(n0 + r, a.N - 1) * a.K, *xp = xq + (size_t)min(m0 + r, a.M - 1) * Kp;
    const int wn = (wave % 2) * 32, wm = (wave / 2) * 32;
    i32x4 acc[2][2] = {};
    for (int k = 0; k < Kp; k += 64) {
        i32x4 vw = {0, 0, 0, 0};
        if (k + c < a.K) vw = *reinterpret_cast<const i32x4 *>(wp + k + c);
        const i32x4 vx = *reinterpret_cast<const i32x4 *>(xp + k + c);
        __syncthreads();
        *reinterpret_cast<i32x4 *>(&sw[r][c]) = vw;
        *reinterpret_cast<i32x4 *>(&sx[r][c]) = vx;
        __syncthreads();
        i32x4 fw[2], fx[2];
        for (int i = 0; i < 2; i++) {
            fw[i] = *reinterpret_cast<const i32x4 *>(&sw[wn + 16 * i + lane % 16][16 * (lane / 16)]);
            fx[i] = *reinterpret_cast<const i32x4 *>(&sx[wm + 16 * i + lane % 16][16 * (lane / 16)]);
        }
        for (int i = 0; i < 2; i++)
            for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[i], fx[j], acc[i][j], 0, 0, 0);
    }
    for (int j = 0; j < 2; j++) {
        const int m = m0 + wm + 16 * j + lane % 16;
        if (m >= a.M) continue;
        const float s = xs[m];
        for (int i = 0; i < 2; i++)
            for (int e = 0; e < 4; e++) {
                const int n = n0 + wn + 16 * i + 4 * (lane / 16) + e;
                if (n >= a.N) continue;
                float v = (float)acc[i][j][e] * s * a.w_scale[n];
                if (a.res) v += lin_get(a.res, a.out_type, (int64_t)m * a.res_stride + n);
                lin_put(a.out, a.out_type, (int64_t)m * a.out_stride + n, v);
            }
    }
}

// ================================================================ launchers
size_t matmul_i8_workspace(int M, int N, int K) { return (size_t)M * lin_kp(K) + 4 * (size_t)M + 16; }

hipError_t launch_matmul_i8(const MatmulI8Args &a, void *ws, hipStream_t st) {
    const int Kp = lin_kp(a.K);
    float *xs = reinterpret_cast<float *>(static_cast<uint8_t *>(ws) + (size_t)a.M * Kp);
    int8_t *xq = static_cast<int8_t *>(ws);
    TG_LAUNCH(k_lin_quant, dim3((unsigned)a.M), dim3(256), 0, st, a, Kp, xq, xs);
    TG_LAUNCH(k_lin_mm, dim3((unsigned)((a.N + 63) / 64), (unsigned)((a.M + 63) / 64)), dim3(256), 0, st, a, Kp, xq, xs);
    return hipGetLastError();
}

}  // namespace tg
