// tg_linear.hip -- int8 matrix product with a scale per token and per
// channel: activations quantised on the way (after an RMS norm where one is
// given), v_mfma_i32_16x16x64_i8 tiles, scales and residual in the epilogue.
#include "tg_device.h"
#include "tg_internal.h"

#include "../../include/tinygiant.h"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace tg {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

TG_DEV float lin_bf(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }

template <int TYPE>
TG_DEV float lin_get(const void *p, int64_t i) {
    if constexpr (TYPE == TG_T_F32) return static_cast<const float *>(p)[i];
    const uint16_t v = static_cast<const uint16_t *>(p)[i];
    return TYPE == TG_T_F16 ? h2f(v) : lin_bf(v);
}

// Four elements of memory that is aligned to one: still one access.
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4_u __attribute__((ext_vector_type(4), aligned(2)));

template <int TYPE>
TG_DEV f32x4 lin_get4(const void *p, int64_t i) {
    if constexpr (TYPE == TG_T_F32) {
        return *reinterpret_cast<const f32x4_u *>(static_cast<const float *>(p) + i);
    } else {
        const u16x4 v = *reinterpret_cast<const u16x4_u *>(static_cast<const uint16_t *>(p) + i);
        f32x4 r;
#pragma unroll
        for (int e = 0; e < 4; e++) r[e] = TYPE == TG_T_F16 ? h2f(v[e]) : lin_bf(v[e]);
        return r;
    }
}

template <int TYPE>
TG_DEV void lin_put(void *p, int64_t i, float v) {
    if constexpr (TYPE == TG_T_F32) static_cast<float *>(p)[i] = v;
    else static_cast<uint16_t *>(p)[i] = TYPE == TG_T_F16 ? f2h(v) : __builtin_bit_cast(uint16_t, (__bf16)v);
}

template <int TYPE>
TG_DEV void lin_put4(void *p, int64_t i, f32x4 v) {
    if constexpr (TYPE == TG_T_F32) {
        *reinterpret_cast<f32x4_u *>(static_cast<float *>(p) + i) = v;
    } else {
        u16x4 r;
#pragma unroll
        for (int e = 0; e < 4; e++) r[e] = TYPE == TG_T_F16 ? f2h(v[e]) : __builtin_bit_cast(uint16_t, (__bf16)v[e]);
        *reinterpret_cast<u16x4_u *>(static_cast<uint16_t *>(p) + i) = r;
    }
}

TG_DEV int lin_fours(int N) { return (N + 3) / 4 * 4; }

// Channel n of row m.
template <int OT>
TG_DEV void lin_out1(const MatmulI8Args &a, int m, int n, float v) {
    float y = v * a.w_scale[n];
    if (a.res) y += lin_get<OT>(a.res, (int64_t)m * a.res_stride + n);
    lin_put<OT>(a.out, (int64_t)m * a.out_stride + n, y);
}

// Channels n .. n + 3 of row m: sums times the row's scale to the output; sw: their scales where all four are there.
template <int OT>
TG_DEV void lin_out(const MatmulI8Args &a, int m, int n, f32x4 v, f32x4 sw) {
    if (n + 4 <= a.N) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = v[e] * sw[e];
        if (a.res) v += lin_get4<OT>(a.res, (int64_t)m * a.res_stride + n);
        lin_put4<OT>(a.out, (int64_t)m * a.out_stride + n, v);
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (n + e >= a.N) return;
        lin_out1<OT>(a, m, n + e, v[e]);
    }
}

constexpr int LIN_K = 128;  // rows of codes are padded to it with zeros

static int lin_kp(int K) { return (K + LIN_K - 1) / LIN_K * LIN_K; }

// ================================================================ quantise
// v from the lane that a DPP control names (0 where there is none)
template <class T, int CTRL, int ROWS, bool ZERO>
TG_DEV T dpp(T v) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, ZERO));
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, ZERO);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, ZERO);
        return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
    }
}

// Sums and maxima (of values of at least 0) over the TPR threads of one row; red: a value per wave.
template <int TPR, class T, class F>
TG_DEV T row_reduce(T v, T *red, F op) {
    v = op(v, dpp<T, 0x111, 0xF, true>(v));
    v = op(v, dpp<T, 0x112, 0xF, true>(v));
    v = op(v, dpp<T, 0x114, 0xF, true>(v));
    v = op(v, dpp<T, 0x118, 0xF, true>(v));
    v = op(v, dpp<T, 0x142, 0xA, false>(v));
    v = op(v, dpp<T, 0x143, 0xC, false>(v));
    if constexpr (TPR > 64) {
        if (threadIdx.x % 64 == 63) red[threadIdx.x / 64] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < TPR / 64; i++) v = op(v, red[i]);
    } else {
        v = __shfl(v, 63);
    }
    return v;
}

struct QuantLds {
    double sum[4];
    uint32_t mag[4];
    unsigned long long top[4];
};

// One row's codes q = rint(127 xn / a), a = max |xn|, and its scale a / 127 by
// TPR threads, which hold the row (NV vectors of 4 each; NV 0: a row too long
// for that is read once per pass).  The mean square is summed in 64 bits; then
// fp32 does: xn is off by at most 3 roundings and t = xn * (127 / a) by 5, so t is the quotient to
// within 127 * 5 * 2^-24 < 5e-5, and what that leaves open is worked out in 64 bits:
// which value is the largest (those within 2^-20 of it), and codes that near a
// border.  Half the largest value lies on one (63.5), and no order of the sum
// shows.  put(k, four codes) for every k below Kp.  A barrier at least lies between the last look at
// `l` and the return, none behind a second row's first write to it: callers with two rows put one there.
template <int TYPE, int TPR, int NV, class P>
TG_DEV float quant_row(const MatmulI8Args &a, int Kp, int row, QuantLds &l, P put) {
    const int tid = threadIdx.x % TPR;
    const int64_t x0 = (int64_t)row * a.x_stride;
    constexpr int NH = NV ? NV : 1;
    f32x4 h[NH], g[NH];
    auto load = [&](int k) { return k < a.K ? lin_get4<TYPE>(a.x, x0 + k) : f32x4{0, 0, 0, 0}; };
    auto weight = [&](int k) { return a.norm_w && k < a.K ? lin_get4<TG_T_F32>(a.norm_w, k) : f32x4{1, 1, 1, 1}; };
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; i++) h[i] = load(4 * (tid + i * TPR));
    }
    // f(i, k, x) for each four of the row
    auto pass = [&](int limit, auto f) {
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; i++) f(i, 4 * (tid + i * TPR), h[i]);
        } else {
            for (int k = 4 * tid; k < limit; k += 4 * TPR) f(0, k, load(k));
        }
    };
    unsigned long long *slot = &l.top[TPR == 64 ? threadIdx.x / 64 : 0];
    if (tid == 0) *slot = 0;
    double r = 1.0;
    if (a.norm_w) {
        double ss = 0.0;
        pass(a.K, [&](int, int, f32x4 x) {
#pragma unroll
            for (int e = 0; e < 4; e++) ss = __builtin_fma((double)x[e], (double)x[e], ss);
        });
        r = 1.0 / __builtin_sqrt(row_reduce<TPR>(ss, l.sum, [](double x, double y) { return x + y; }) / a.K + (double)a.eps);
    }
    const float r32 = (float)r;
    auto normed = [&](int k, f32x4 x) {
        if (!a.norm_w) return x;
        const f32x4 w = weight(k);
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = x[e] * r32 * w[e];
        return x;
    };
    auto exact = [&](float x, float w) { return a.norm_w ? (double)x * r * (double)w : (double)x; };
    // the largest magnitude, as the integers that magnitudes order as (NaN above infinity above all others)
    uint32_t mag = 0;
    pass(a.K, [&](int i, int k, f32x4 x) {
        g[i] = normed(k, x);
#pragma unroll
        for (int e = 0; e < 4; e++) mag = max(mag, __float_as_uint(g[i][e]) & 0x7FFFFFFFu);
    });
    const float mine = __uint_as_float(mag);
    const float top32 = __uint_as_float(row_reduce<TPR>(mag, l.mag, [](uint32_t x, uint32_t y) { return max(x, y); }));
    const bool bad = !(top32 < INFINITY);
    // r or the largest value near the ends of fp32's range: everything in 64 bits
    const bool wild = a.norm_w && (r32 < 1e-30f || top32 < 1e-30f);
    double top = top32;
    if (a.norm_w) {
        const float from = wild ? 0.0f : top32 * (1.0f - 0x1p-20f);
        if (mine >= from) {
            double t = 0.0;
            pass(a.K, [&](int, int k, f32x4 x) {
                const f32x4 w = weight(k);
#pragma unroll
                for (int e = 0; e < 4; e++) t = fmax(t, fabs(exact(x[e], w[e])));
            });
            __hip_atomic_fetch_max(slot, __builtin_bit_cast(unsigned long long, t), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
        if (TPR > 64) __syncthreads();
        else wave_lds_sync();
        top = __builtin_bit_cast(double, *slot);
    }
    const float inv = bad || top == 0.0 ? 0.0f : (float)(127.0 / top);
    pass(Kp, [&](int i, int k, f32x4 x) {
        const f32x4 n = NV > 0 ? g[i] : normed(k, x);
        uint32_t q = 0;
        float off = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float t = n[e] * inv, c = __builtin_rintf(t);
            off = fmaxf(off, fabsf(t - c));
            q |= ((uint32_t)(int)c & 255) << (8 * e);
        }
        if ((wild || !(off < 0.49995f) || !(inv < INFINITY)) && inv != 0.0f) {
            const f32x4 w = weight(k);
            q = 0;
            for (int e = 0; e < 4; e++) q |= ((uint32_t)(int)__builtin_rint(127.0 * exact(x[e], w[e]) / top) & 255) << (8 * e);
        }
        if (NV == 0 || k < Kp) put(k, q);
    });
    return bad ? __builtin_nanf("") : (float)(top / 127.0);
}

// A launch of its own for the codes: 8192 x 4096 fp32 with norm 42 us, 4.0 TB/s, bound by bytes; 1999 x 4096
// bf16 11 us, 2.2 TB/s, of which 5 are what 7 rows take too.
template <int TYPE, int TPR, int NV>
__global__ __launch_bounds__(256) void k_lin_quant(MatmulI8Args a, int Kp, int8_t *xq, float *xs) {
    __shared__ QuantLds l;
    const int row = blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    if (row >= a.M) return;  // whole waves
    const float s = quant_row<TYPE, TPR, NV>(a, Kp, row, l, [&](int k, uint32_t q) {
        *reinterpret_cast<uint32_t *>(xq + (size_t)row * Kp + k) = q;
    });
    if (threadIdx.x % TPR == 0) xs[row] = s;
}

// ================================================================ few rows
// Up to 16 MT rows: bound by the weights' bytes, each read once, 16 bytes of
// a channel per lane straight into the matrix instruction's operand.  A block takes 16 R channels, its
// four waves every fourth step of 64 columns, two batches of U steps under
// way in each; the waves' int32 sums meet in LDS.  XT >= 0: up to 4 rows (4096 columns together) are
// quantised by every block for itself, the codes in LDS, while its first
// weights are on their way, which saves a launch.  7 rows by 151936 x 2048: 66 us, 4.7 TB/s of the 6
// that reading reaches; 1 by 5120 x 2048: 8.1, its latency.
constexpr int LIN_FUSE_M = 4, LIN_FUSE = 4096;

template <int MT, int R, int U, int OT, int XT>
__global__ __launch_bounds__(256) void k_lin_few(MatmulI8Args a, int Kp, const int8_t *xq, const float *xs) {
    constexpr bool FUSE = XT >= 0;
    __shared__ __align__(16) i32x4 part[4][R * MT][64];
    __shared__ float scale[LIN_FUSE_M];
    __shared__ QuantLds ql;
    extern __shared__ __align__(16) uint8_t codes[];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), r16 = lane % 16, h16 = lane / 16 * 16;
    const int n0 = blockIdx.x * 16 * R, m0 = blockIdx.y * 16 * MT;
    const int8_t *wp[R];
#pragma unroll
    for (int i = 0; i < R; i++) wp[i] = a.w + (size_t)min(n0 + 16 * i + r16, a.N - 1) * a.K;
    const int8_t *xp[MT];
#pragma unroll
    for (int j = 0; j < MT; j++) xp[j] = (FUSE ? reinterpret_cast<const int8_t *>(codes) : xq) + (size_t)min(m0 + 16 * j + r16, a.M - 1) * Kp;
    const int nk = Kp / 64;
    struct Batch {
        i32x4 w[U][R], x[U][MT];
    };
    auto load_w = [&](Batch &b, int k) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int kk = min(k + 4 * u, nk - 1) * 64 + h16;
#pragma unroll
            for (int i = 0; i < R; i++) b.w[u][i] = *reinterpret_cast<const i32x4 *>(wp[i] + (kk < a.K ? kk : 0));  // beyond: any
        }
    };
    auto load_x = [&](Batch &b, int k) {  // zeros for the steps behind the last
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < MT; j++) {
                b.x[u][j] = *reinterpret_cast<const i32x4 *>(xp[j] + min(k + 4 * u, nk - 1) * 64 + h16);
                if (k + 4 * u >= nk) b.x[u][j] = i32x4{0, 0, 0, 0};
            }
    };
    Batch cur, nxt;
    load_w(nxt, wave);
    if constexpr (FUSE) {
        for (int m = 0; m < a.M; m++) {
            const auto put = [&](int k, uint32_t q) { *reinterpret_cast<uint32_t *>(codes + (size_t)m * Kp + k) = q; };
            float s;
            if (Kp <= 2048) s = quant_row<XT, 256, 2>(a, Kp, m, ql, put);
            else s = quant_row<XT, 256, 4>(a, Kp, m, ql, put);
            if (threadIdx.x == 0) scale[m] = s;
            __syncthreads();
        }
    }
    load_x(nxt, wave);
    i32x4 acc[R][MT] = {};
    for (int k = wave; k < nk; k += 4 * U) {
        cur = nxt;
        load_w(nxt, k + 4 * U);
        load_x(nxt, k + 4 * U);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < R; i++)
#pragma unroll
                for (int j = 0; j < MT; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(cur.w[u][i], cur.x[u][j], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) part[wave][i * MT + j][lane] = acc[i][j];
    __syncthreads();
#pragma unroll
    for (int t = 0; t < (R * MT + 3) / 4; t++) {
        const int ij = t * 4 + wave;
        if (ij >= R * MT) break;
        i32x4 v = part[0][ij][lane];
#pragma unroll
        for (int w = 1; w < 4; w++) v += part[w][ij][lane];
        const int m = m0 + ij % MT * 16 + r16;
        const int n = n0 + ij / MT * 16 + h16 / 4;
        if (m >= a.M) continue;
        const float s = FUSE ? scale[m & 3] : xs[m];
        f32x4 y, sw = {0, 0, 0, 0};
        if (n + 4 <= a.N) sw = *reinterpret_cast<const f32x4_u *>(a.w_scale + n);
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = (float)v[e] * s;
        lin_out<OT>(a, m, n, y, sw);
    }
}

// ================================================================ large products
// BN channels x BM rows per block, WN x WM waves, ST stages of 128 columns in
// LDS.  A stage is (BN + BM) rows of 128 bytes (whole cache lines), the
// 16-byte chunk c of row r at place c ^ (r % 8) of it, so that the 8 lanes
// that LDS serves together read 8 different places; it is loaded straight to
// LDS (8 rows per instruction, the swizzle done by which chunk a lane asks
// for).  The operands of half a stage are held in registers while those of the
// next half are read, so LDS reads run beside the matrix instructions.  One
// barrier per stage, in its middle: behind it every wave holds the rest of
// stage k in registers, so k's place is loaded with stage k + ST, and stage k
// + 1 has landed for every wave.
//
// 8192 x 9216 x 4096 in tiles of 256 x 256: 310 us, 2.0 POP/s, matrix units busy 41%, vector instructions 20%; by
// count, not by a counter, the tiles' bytes come to 2.4 GB, 7.8 TB/s out of the caches.  1999 x 2048 x 4096 in tiles of
// 128 x 128: 32 us, 1.0; its 256 blocks, one to a CU, are one round, whose start and way out nothing covers.
//
// Where the tiles are too few for the device's CUs the columns are split: a block takes `stages` of
// them and leaves its int32 sums in part [split][row][N in fours] (OT LIN_PART), which
// k_lin_sum adds.
constexpr int LIN_PART = -1;

template <int BN, int BM, int WN, int WM, int ST, int OT>
__global__ __launch_bounds__(64 * WN * WM, 2) void k_lin_tile(MatmulI8Args a, int Kp, const int8_t *xq, const float *xs, int tiles_n,
                                                              int tiles_m, int stages, int32_t *part) {
    constexpr int NW = WN * WM, PER = (BN + BM) / 8 / NW, TN = BN / WN / 16, TM = BM / WM / 16;
    constexpr int STAGE = (BN + BM) * 128;
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    // blocks of one XCD (every eighth) take neighbouring tiles, in bands of 8 tiles of channels
    const int total = tiles_n * tiles_m, id = blockIdx.x, q8 = gridDim.x / 8, r8 = gridDim.x % 8, xcd = id % 8;
    const int item = xcd * q8 + min(xcd, r8) + id / 8, split = OT == LIN_PART ? item / total : 0, t = item - split * total;
    constexpr int BAND = 8;
    const int band = t / (BAND * tiles_m), wide = min(BAND, tiles_n - band * BAND), in = t - band * BAND * tiles_m;
    const int n0 = (band * BAND + in % wide) * BN, m0 = in / wide * BM;

    const int8_t *w0 = a.w + (size_t)n0 * a.K, *x0 = xq + (size_t)m0 * Kp;
    const int chunk = ((lane % 8) ^ (lane / 8)) * 16;
    uint32_t at[PER];  // the rows that this lane loads, from w0 or x0
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int r0 = (wave * PER + i) * 8, r = r0 + lane / 8;
        at[i] = r0 < BN ? (uint32_t)min(r, a.N - 1 - n0) * a.K : (uint32_t)min(r - BN, a.M - 1 - m0) * Kp;
    }
    const int last = Kp / 128 - 1, from = split * stages, nk = OT == LIN_PART ? min(stages, last + 1 - from) : last + 1;
    auto load = [&](int k) {
        const uint32_t kx = min(from + k, last) * 128 + chunk, kw = kx < (uint32_t)a.K ? kx : 0;  // columns of w behind its last meet zeros: any
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const bool w = (wave * PER + i) * 8 < BN;
            const int8_t *p = (w ? w0 : x0) + (at[i] + (w ? kw : kx));
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)p,
                                             (__attribute__((address_space(3))) void *)(lds + k % ST * STAGE + (wave * PER + i) * 1024), 16, 0, 0);
        }
    };
    const int wn = wave % WN * (BN / WN), wm = wave / WN * (BM / WM);
    const int r16 = lane % 16, place = ((lane / 16) ^ (r16 % 8)) * 16;  // of the first half's chunk; the second's is 4 further, xor 64
    i32x4 acc[TN][TM] = {};
    i32x4 fw[2][TN], fx[2][TM];
    auto read = [&](int k, int half) {
        const uint8_t *st = lds + k % ST * STAGE + (place ^ (half * 64)) + r16 * 128;
#pragma unroll
        for (int i = 0; i < TN; i++) fw[half][i] = *reinterpret_cast<const i32x4 *>(st + (wn + 16 * i) * 128);
#pragma unroll
        for (int i = 0; i < TM; i++) fx[half][i] = *reinterpret_cast<const i32x4 *>(st + (BN + wm + 16 * i) * 128);
    };
    auto meet = [&](auto left) {  // vmcnt: all but `left` loads have landed; lgkmcnt(0): this wave's reads are done
        constexpr int N = decltype(left)::value;
        __builtin_amdgcn_s_waitcnt((N & 15) | 0x70 | (N >> 4 << 14));
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto mul = [&](int half) {
#pragma unroll
        for (int i = 0; i < TN; i++)
#pragma unroll
            for (int j = 0; j < TM; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[half][i], fx[half][j], acc[i][j], 0, 0, 0);
    };
#pragma unroll
    for (int k = 0; k < ST; k++) load(k);
    meet(std::integral_constant<int, PER * (ST - 1)>{});
    read(0, 0);
    for (int k = 0; k < nk; k++) {
        read(k, 1);
        mul(0);
        meet(std::integral_constant<int, PER * (ST - 2)>{});
        load(k + ST);
        read(k + 1, 0);
        mul(1);
    }
    // Out through LDS: 16 rows of the wave's channels at a time, so that a row
    // leaves as whole lines.  First nothing may still be on its way to LDS, or be read there.
    meet(std::integral_constant<int, 0>{});
    constexpr int CN = BN / WN, LD = CN + 4, L = CN / 4, RW = 64 / L;  // channels of the wave, lanes of a row, rows at once
    float *so = reinterpret_cast<float *>(lds) + wave * 16 * LD;
    const int n = n0 + wn + 4 * (lane % L);
    f32x4 sw = {0, 0, 0, 0};
    if (OT != LIN_PART && n + 4 <= a.N) sw = *reinterpret_cast<const f32x4_u *>(a.w_scale + n);
#pragma unroll
    for (int j = 0; j < TM; j++) {
        const int mj = m0 + wm + 16 * j;
        const float s = xs[min(mj + r16, a.M - 1)];
#pragma unroll
        for (int i = 0; i < TN; i++) {
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = OT == LIN_PART ? __int_as_float(acc[i][j][e]) : (float)acc[i][j][e] * s;
            *reinterpret_cast<f32x4 *>(so + r16 * LD + 16 * i + 4 * (lane / 16)) = v;
        }
        wave_lds_sync();
#pragma unroll
        for (int q = 0; q < 16 / RW; q++) {
            const int r = q * RW + lane / L, m = mj + r;
            const f32x4 v = *reinterpret_cast<const f32x4 *>(so + r * LD + 4 * (lane % L));
            if constexpr (OT == LIN_PART) {
                if (m < a.M && n < a.N) *reinterpret_cast<f32x4 *>(part + ((size_t)split * a.M + m) * lin_fours(a.N) + n) = v;
            } else {
                if (m < a.M) lin_out<OT>(a, m, n, v, sw);
            }
        }
        wave_lds_sync();
    }
}

// Four channels of a row: the splits' sums, exact, and what follows them.
template <int OT>
__global__ __launch_bounds__(256) void k_lin_sum(MatmulI8Args a, const float *xs, const int32_t *part, int splits) {
    const int ld = lin_fours(a.N), m = blockIdx.y, n = 4 * (blockIdx.x * 256 + threadIdx.x);
    if (n >= a.N) return;
    const int32_t *p = part + (size_t)m * ld + n;
    i32x4 v = *reinterpret_cast<const i32x4 *>(p);
    for (int i = 1; i < splits; i++) v += *reinterpret_cast<const i32x4 *>(p + (size_t)i * a.M * ld);
    const float s = xs[m];
    f32x4 y, sw = {0, 0, 0, 0};
    if (n + 4 <= a.N) sw = *reinterpret_cast<const f32x4_u *>(a.w_scale + n);
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = (float)v[e] * s;
    lin_out<OT>(a, m, n, y, sw);
}

// ================================================================ launchers
// The dynamic-LDS limit of kernel fn raised to `bytes` on the current device, once per (kernel, device).
static hipError_t lin_lds(const void *fn, size_t bytes, std::atomic<uint64_t> &done) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
    if (bit && (done.load(std::memory_order_relaxed) & bit)) return hipSuccess;
    e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == hipSuccess && bit) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

#define TG_BY_TYPE(T, NAME, ...)                                                        \
    do {                                                                                \
        if ((T) == TG_T_F32) { constexpr int NAME = TG_T_F32; __VA_ARGS__; }            \
        else if ((T) == TG_T_F16) { constexpr int NAME = TG_T_F16; __VA_ARGS__; }       \
        else { constexpr int NAME = TG_T_BF16; __VA_ARGS__; }                           \
    } while (0)

// 64 channels to a block, not 16: 4 rows by 151936 x 2048 58 us (16: 72), 32768 x 2048 18 (21), 9216 x 4096 22 (19).
static bool lin_wide_n(int N) { return N >= 32768; }
// One launch, not two: 1 row by 5120 x 2048 8.7 us (12.4), by 2048 x 4096 8.7 (12.2); 2 rows by 5120 x 2048 7.9 (11.6).
static bool lin_fused(int M, int N, int Kp) { return !lin_wide_n(N) && M <= LIN_FUSE_M && M * Kp <= LIN_FUSE; }

// Which kernel, and how many stages of 128 columns a block takes (0: all).
struct LinPlan {
    bool few, big;
    int stages, splits;
};
static LinPlan lin_plan(int M, int N, int Kp) {
    const int64_t tiles = (int64_t)((N + 127) / 128) * ((M + 127) / 128);
    // Up to 32 rows the weights' bytes count, above them the operands' way through LDS (64 rows: 2048 x 4096 16.4 us by
    // tiles, 20.6 as few rows; 9216 x 4096 29 and 37; 33 rows: 27 and 30).  The large tiles halve that way, where they are
    // enough for the CUs and rows fill them (8192 x 9216 x 4096: 310 us; 4096 rows 201, 234 by the small ones; 128 rows by
    // 151936 x 2048: 121 and 99).
    LinPlan p{M <= 32, M > 128 && (int64_t)((N + 255) / 256) * ((M + 255) / 256) >= 256, 0, 1};
    const int nk = Kp / 128;
    // Tiles for half the CUs or fewer: a block to a CU by splitting the columns, 8 stages to a block at the least
    // (4: 30 us for 200 x 130 x 16384, 28 with 8, 68 as few rows; 300 x 2048 x 4096 25, 21 and 28), where there are more than
    // 2560 of them (300 x 256 x 2048: 16 us split, 13 as few rows).
    if (!p.few && tiles <= 128 && nk > 20) {
        p.stages = std::max(8, (int)((nk * tiles + 255) / 256));
        p.splits = (nk + p.stages - 1) / p.stages;
    }
    // Short columns and next to no tiles: the few rows' kernel, 16 channels to a block (500 x 1024 x 1024: 12 us, 14 by tiles).
    if (p.splits == 1 && tiles <= 40) p.few = true;
    return p;
}
static int lin_quant_threads(int Kp) { return Kp <= 512 ? 64 : 256; }  // of a row
static size_t lin_codes(int M, int Kp) { return ((size_t)M * Kp + 4 * (size_t)M + 15) / 16 * 16; }

// A launch has fewer than 2^32 threads.  Rows and channels up to 2^30, so that indexes of tiles that pass the last one
// stay within 32 bits.
bool matmul_i8_fits(int M, int N, int K) {
    if (M > 1 << 30 || N > 1 << 30) return false;
    const int Kp = lin_kp(K), few_n = M <= 32 && lin_wide_n(N) ? 64 : 16;
    const LinPlan p = lin_plan(M, N, Kp);
    const int64_t codes = lin_fused(M, N, Kp) ? 0 : ((int64_t)M * lin_quant_threads(Kp) + 255) / 256;
    const int64_t tiles = p.big ? 2 * (int64_t)((N + 255) / 256) * ((M + 255) / 256)  // of 512 threads
                                : (int64_t)((N + 127) / 128) * ((M + 127) / 128) * p.splits;
    return std::max(codes, p.few ? (int64_t)(N + few_n - 1) / few_n : tiles) * 256 <= UINT32_MAX;
}

size_t matmul_i8_workspace(int M, int N, int K) {
    const int Kp = lin_kp(K);
    if (lin_fused(M, N, Kp)) return 0;
    const LinPlan p = lin_plan(M, N, Kp);
    return lin_codes(M, Kp) + (p.splits > 1 ? (size_t)p.splits * M * ((N + 3) / 4 * 4) * 4 : 0) + 16;
}

template <int TYPE>
static void quant_launch(const MatmulI8Args &a, int Kp, int8_t *xq, float *xs, hipStream_t st) {
#define TG_QUANT(TPR, NV) TG_LAUNCH((k_lin_quant<TYPE, TPR, NV>), dim3((unsigned)((a.M + 256 / TPR - 1) / (256 / TPR))), dim3(256), 0, st, a, Kp, xq, xs)
    if (Kp <= 256) TG_QUANT(64, 1);
    else if (Kp <= 512) TG_QUANT(64, 2);
    else if (Kp <= 1024) TG_QUANT(256, 1);
    else if (Kp <= 2048) TG_QUANT(256, 2);
    else if (Kp <= 4096) TG_QUANT(256, 4);
    else if (Kp <= 8192) TG_QUANT(256, 8);
    else TG_QUANT(256, 0);
#undef TG_QUANT
}

template <int BN, int BM, int WN, int WM, int ST, int OT>
static hipError_t tile_launch(const MatmulI8Args &a, int Kp, const int8_t *xq, const float *xs, const LinPlan &p, int32_t *part, hipStream_t st) {
    static std::atomic<uint64_t> done{0};
    constexpr size_t bytes = (size_t)ST * (BN + BM) * 128;
    const hipError_t e = lin_lds((const void *)k_lin_tile<BN, BM, WN, WM, ST, OT>, bytes, done);
    if (e != hipSuccess) return e;
    const int tn = (a.N + BN - 1) / BN, tm = (a.M + BM - 1) / BM;
    TG_LAUNCH((k_lin_tile<BN, BM, WN, WM, ST, OT>), dim3((unsigned)(tn * tm * p.splits)), dim3(64 * WN * WM), bytes, st, a, Kp, xq, xs, tn, tm, p.stages, part);
    return hipSuccess;
}

template <int MT, int R, int U, int OT>
static void few_launch(const MatmulI8Args &a, int Kp, const int8_t *xq, const float *xs, hipStream_t st) {
    const dim3 grid((unsigned)((a.N + 16 * R - 1) / (16 * R)), (unsigned)((a.M + 16 * MT - 1) / (16 * MT)));
    if constexpr (MT == 1 && R == 1) {  // the only one that lin_fused's N and M come to
        if (lin_fused(a.M, a.N, Kp)) {
            TG_BY_TYPE(a.x_type, XT, TG_LAUNCH((k_lin_few<MT, R, U, OT, XT>), grid, dim3(256), (size_t)a.M * Kp, st, a, Kp, xq, xs));
            return;
        }
    }
    TG_LAUNCH((k_lin_few<MT, R, U, OT, -1>), grid, dim3(256), 0, st, a, Kp, xq, xs);
}

hipError_t launch_matmul_i8(const MatmulI8Args &a, void *ws, hipStream_t st) {
    const int Kp = lin_kp(a.K);
    int8_t *xq = static_cast<int8_t *>(ws);
    float *xs = reinterpret_cast<float *>(xq + (size_t)a.M * Kp);
    if (!lin_fused(a.M, a.N, Kp)) TG_BY_TYPE(a.x_type, XT, quant_launch<XT>(a, Kp, xq, xs, st));
    const bool wide = lin_wide_n(a.N);
    const LinPlan p = lin_plan(a.M, a.N, Kp);
    int32_t *part = reinterpret_cast<int32_t *>(xq + lin_codes(a.M, Kp));
    hipError_t e = hipSuccess;
    if (p.splits > 1) e = tile_launch<128, 128, 2, 2, 4, LIN_PART>(a, Kp, xq, xs, p, part, st);
    if (e != hipSuccess) return e;
    TG_BY_TYPE(a.out_type, OT, {
        if (p.splits > 1) {
            TG_LAUNCH((k_lin_sum<OT>), dim3((unsigned)((a.N + 1023) / 1024), (unsigned)a.M), dim3(256), 0, st, a, xs, part, p.splits);
        } else if (p.few) {
            if (a.M <= 16 && wide) few_launch<1, 4, 2, OT>(a, Kp, xq, xs, st);
            else if (a.M <= 16) few_launch<1, 1, 8, OT>(a, Kp, xq, xs, st);
            else if (a.M <= 32 && wide) few_launch<2, 4, 2, OT>(a, Kp, xq, xs, st);
            else if (a.M <= 32) few_launch<2, 1, 4, OT>(a, Kp, xq, xs, st);
            else few_launch<4, 1, 2, OT>(a, Kp, xq, xs, st);
        } else if (p.big) e = tile_launch<256, 256, 2, 4, 2, OT>(a, Kp, xq, xs, p, part, st);
        else e = tile_launch<128, 128, 2, 2, 4, OT>(a, Kp, xq, xs, p, part, st);
    });
    return e != hipSuccess ? e : hipGetLastError();
}

}  // namespace tg
