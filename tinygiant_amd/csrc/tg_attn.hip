// tg_attn.hip -- a paged Q4_0 KV cache on the device: new rows into it (head
// norm, rotation, quantisation), reading it back, and causal grouped-query
// attention over it (the roles of engine.py:199-227 and
// csrc/libtinygiant.c:365-456 for ragged batches).
//
// A sequence's tokens sit in pages, a page's in tiles of 16 tokens of one key
// head: K codes (8 D bytes), V codes (8 D), K scales (D), V scales (D), as
// include/tinygiant.h lays them out.
#include "tg_device.h"
#include "tg_internal.h"

#include "../../include/tinygiant.h"

namespace tg {

// ================================================================ the batch
// byte of a page's tile for one key head
template <int D>
TG_DEV size_t tile_at(const KvBatch &b, int page, int head, int tile) {
    return (((size_t)page * b.n_kv + head) * (b.page_tokens / 16) + tile) * (size_t)(18 * D);
}

// rows [lo, hi) of sequence s, kept inside the row tensors whatever cu holds
struct SeqRows {
    int lo, hi, len;
};
TG_DEV SeqRows seq_rows(const KvBatch &b, int s) {
    SeqRows r;
    const int lo = b.cu[s], hi = b.cu[s + 1], len = b.kv_len[s];
    r.lo = min(max(lo, 0), b.n_tokens);
    r.hi = min(max(hi, r.lo), b.n_tokens);
    r.len = max(len, 0);
    return r;
}

// the page of position p of sequence s, or -1
TG_DEV int page_of(const KvBatch &b, int s, int p) {
    const int c = p / b.page_tokens;
    if (p < 0 || c >= b.table_cols) return -1;
    const int page = b.table[(size_t)s * b.table_stride + c];
    return page >= 0 && page < b.n_pages ? page : -1;
}

// The sequence of row t: the number of j with cu[j + 1] <= t, counted by L
// neighbouring lanes (li: lane among them); n_seqs for padding rows.
template <int L>
TG_DEV int seq_of(const KvBatch &b, int t, int li) {
    int c = 0;
    for (int j = li; j < b.n_seqs; j += L) c += b.cu[j + 1] <= t;
#pragma unroll
    for (int m = 1; m < L; m *= 2) c += __shfl_xor(c, m);
    return c;
}

// ================================================================ element types
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

TG_DEV float bf2f(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
TG_DEV uint16_t f2bf(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }

template <int TYPE>
TG_DEV f32x4 load4(const void *p, int64_t i) {
    if constexpr (TYPE == TG_T_F32) {
        return *reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + i);
    } else {
        const u16x4 v = *reinterpret_cast<const u16x4 *>(static_cast<const uint16_t *>(p) + i);
        f32x4 r;
#pragma unroll
        for (int e = 0; e < 4; e++) r[e] = TYPE == TG_T_F16 ? h2f(v[e]) : bf2f(v[e]);
        return r;
    }
}

template <int TYPE>
TG_DEV void store4(void *p, int64_t i, f32x4 v) {
    if constexpr (TYPE == TG_T_F32) {
        *reinterpret_cast<f32x4 *>(static_cast<float *>(p) + i) = v;
    } else {
        u16x4 r;
#pragma unroll
        for (int e = 0; e < 4; e++) r[e] = TYPE == TG_T_F16 ? f2h(v[e]) : f2bf(v[e]);
        *reinterpret_cast<u16x4 *>(static_cast<uint16_t *>(p) + i) = r;
    }
}

// ================================================================ append
// Q4_0 of 32 values held 4 to a lane by 8 neighbouring lanes: the scale as a
// half, the four codes.  m = the value of largest magnitude (the first on
// ties), d = m / -8, code = min(15, trunc(x / d + 8.5)) by the reciprocal of
// the unrounded d.
TG_DEV uint16_t quant4(f32x4 x, int li, int code[4]) {
    float top = 0.0f, val = 0.0f;
    bool nan = false;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        x[e] = x[e] > 65504.0f ? 65504.0f : x[e] < -65504.0f ? -65504.0f : x[e];  // NaN stays
        nan |= x[e] != x[e];
        if (top < fabsf(x[e])) top = fabsf(x[e]), val = x[e];
    }
#pragma unroll
    for (int m = 1; m < 8; m *= 2) {
        const float ot = __shfl_xor(top, m), ov = __shfl_xor(val, m);
        if (ot > top || (ot == top && (li & m))) top = ot, val = ov;
        nan |= __shfl_xor((int)nan, m) != 0;
    }
    const float d = nan ? __builtin_nanf("") : val / -8.0f;
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float c = x[e] * id + 8.5f;
        code[e] = c < 15.0f ? (int)(c > 0.0f ? c : 0.0f) : 15;  // NaN: 15, next to a NaN scale
    }
    return f2h(d);
}

// One unit = one head of one row of q, k or v: D / 8 lanes, lane i holding
// dims 4 i .. 4 i + 3 and the same of the upper half, so that a rotation pair
// is one lane's and 8 lanes hold one Q4_0 block of each half.
//
// Bound by bytes (rows in, q out, 72 bytes per token, head and K or V at 128).
template <int D, int TYPE>
__global__ __launch_bounds__(256) void k_kv_append(KvBatch b, AppendArgs a) {
    constexpr int L = D / 8, NG = D / 32;
    const int units = a.n_heads + 2 * b.n_kv;
    const int li = threadIdx.x % L;
    const int64_t u = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const bool live = u < (int64_t)b.n_tokens * units;
    const int t = live ? (int)(u / units) : 0, slot = live ? (int)(u % units) : 0;
    const bool is_q = slot < a.n_heads, is_v = slot >= a.n_heads + b.n_kv;
    const int head = is_q ? slot : is_v ? slot - a.n_heads - b.n_kv : slot - a.n_heads;
    const KvRows src = is_q ? a.q : is_v ? a.v : a.k;
    f32x4 lo = load4<TYPE>(src.p, (int64_t)t * src.stride + head * D + 4 * li);
    f32x4 hi = load4<TYPE>(src.p, (int64_t)t * src.stride + head * D + D / 2 + 4 * li);

    const int s = seq_of<L>(b, t, li);
    const bool row = live && s < b.n_seqs;
    int pos = -1, page = -1;
    if (row) {
        const SeqRows r = seq_rows(b, s);
        pos = r.len - r.hi + t;
        if (pos >= a.max_pos) pos = -1;
        page = page_of(b, s, pos);
    }

    const float *nw = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
    if (nw) {
        // the mean square in 64 bits, rounded once: the row's scale does not
        // depend on the order of the sum
        double ss = 0.0;
#pragma unroll
        for (int e = 0; e < 4; e++) ss += (double)lo[e] * (double)lo[e] + (double)hi[e] * (double)hi[e];
#pragma unroll
        for (int m = 1; m < L; m *= 2) ss += __shfl_xor(ss, m);
        const float r = 1.0f / __builtin_sqrtf((float)(ss / D) + a.eps);
        const f32x4 wl = *reinterpret_cast<const f32x4 *>(nw + 4 * li), wh = *reinterpret_cast<const f32x4 *>(nw + D / 2 + 4 * li);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            lo[e] = lo[e] * r * wl[e];
            hi[e] = hi[e] * r * wh[e];
        }
    }
    if (!is_v && a.cos && pos >= 0) {
        const f32x4 c = *reinterpret_cast<const f32x4 *>(a.cos + (size_t)pos * (D / 2) + 4 * li);
        const f32x4 sn = *reinterpret_cast<const f32x4 *>(a.sin + (size_t)pos * (D / 2) + 4 * li);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float x = lo[e] * c[e] - hi[e] * sn[e], y = hi[e] * c[e] + lo[e] * sn[e];
            lo[e] = x;
            hi[e] = y;
        }
    }
    if (is_q) {
        if (row) {
            const f32x4 nan = {__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
            const int64_t o = (int64_t)t * a.q_out_stride + head * D + 4 * li;
            store4<TYPE>(a.q_out, o, page >= 0 ? lo : nan);
            store4<TYPE>(a.q_out, o + D / 2, page >= 0 ? hi : nan);
        }
    }
    // q's lanes take part in the exchanges below: units of one wave differ in kind
    int cl[4], ch[4];
    const uint16_t dl = quant4(lo, li, cl), dh = quant4(hi, li, ch);
    const bool put = row && !is_q && page >= 0;
    const int r = pos & 15;
    uint8_t *tile = b.pages + (put ? tile_at<D>(b, page, head, (pos % b.page_tokens) / 16) : 0);
    // K: slots 0..7 of block g, piece h are lanes 2 h, 2 h + 1 of the block's 8; slot 2 n + p is nibble n of halfword p
    uint32_t kl = cl[0] | cl[1] << 16 | cl[2] << 4 | cl[3] << 20, kh = ch[0] | ch[1] << 16 | ch[2] << 4 | ch[3] << 20;
    if (li & 1) kl <<= 8, kh <<= 8;
    kl |= __shfl_xor(kl, 1);
    kh |= __shfl_xor(kh, 1);
    // V: dim 16 (4 b + n) + c is nibble n of halfword (c, b): the four lanes (two at D = 64) that hold dims c + 16 n
    uint32_t v0[2], v1[2];  // [lower, upper half of dims]: c pairs (0, 1) and (2, 3) of this lane's four
    const int nl = (li / 4) % 4, nh = (D == 64 ? 2 + li / 4 : li / 4) % 4;
    v0[0] = (uint32_t)(cl[0] | cl[1] << 16) << (4 * nl);
    v1[0] = (uint32_t)(cl[2] | cl[3] << 16) << (4 * nl);
    v0[1] = (uint32_t)(ch[0] | ch[1] << 16) << (4 * nh);
    v1[1] = (uint32_t)(ch[2] | ch[3] << 16) << (4 * nh);
    if (D == 64) {
        v0[0] |= v0[1];
        v1[0] |= v1[1];
    }
#pragma unroll
    for (int m = 4; m < (D == 64 ? 8 : 16); m *= 2) {
#pragma unroll
        for (int i = 0; i < (D == 64 ? 1 : 2); i++) {
            v0[i] |= __shfl_xor(v0[i], m);
            v1[i] |= __shfl_xor(v1[i], m);
        }
    }
    if (!put) return;
    if (!is_v) {
        const int g = li / 8, h = (li % 8) / 2;
        if (!(li & 1)) {
            uint32_t *kc = reinterpret_cast<uint32_t *>(tile);
            kc[(h * 16 + r) * NG + g] = kl;
            kc[(h * 16 + r) * NG + NG / 2 + g] = kh;
        }
        if (li % 8 == 0) {
            uint16_t *ks = reinterpret_cast<uint16_t *>(tile + 16 * D);
            ks[r * NG + g] = dl;
            ks[r * NG + NG / 2 + g] = dh;
        }
    } else {
        uint16_t *vc = reinterpret_cast<uint16_t *>(tile + 8 * D);
        uint16_t *vs = reinterpret_cast<uint16_t *>(tile + 17 * D);
        const int at = ((r / 4) * 16) * 2 + (r % 4) / 2;  // (c = 0) of this token
        // each of the lanes that now hold the same halfwords writes one of the four c
        const int e = (li / 4) % 4, c = 4 * (li % 4) + e;
        const int bq = D == 256 ? li / 16 : 0;
        if (D == 64) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int ee = 2 * (li / 4) + i;
                const uint32_t w = ee < 2 ? v0[0] : v1[0];
                vc[(at + 2 * (4 * (li % 4) + ee)) * NG + r % 2] = (uint16_t)(ee & 1 ? w >> 16 : w);
            }
        } else {
            const uint32_t w0 = e < 2 ? v0[0] : v1[0], w1 = e < 2 ? v0[1] : v1[1];
            vc[(at + 2 * c) * NG + 2 * bq + r % 2] = (uint16_t)(e & 1 ? w0 >> 16 : w0);
            vc[(at + 2 * c) * NG + 2 * (bq + NG / 4) + r % 2] = (uint16_t)(e & 1 ? w1 >> 16 : w1);
        }
        if (li % 8 == 0) {
            vs[((r / 2) * NG + li / 8) * 2 + r % 2] = dl;
            vs[((r / 2) * NG + NG / 2 + li / 8) * 2 + r % 2] = dh;
        }
    }
}

// ================================================================ read
// 8 consecutive dims (8 i ..) of one token's K and V from its tile, as halves
template <int D>
TG_DEV void held8(const uint8_t *tile, int r, int i, f16x8 &k, f16x8 &v) {
    constexpr int NG = D / 32;
    const int g = i / 4, h = i % 4;
    const uint32_t w = reinterpret_cast<const uint32_t *>(tile)[(h * 16 + r) * NG + g];
    const _Float16 dk = reinterpret_cast<const _Float16 *>(tile + 16 * D)[r * NG + g];
    const _Float16 dv = reinterpret_cast<const _Float16 *>(tile + 17 * D)[((r / 2) * NG + g) * 2 + r % 2];
    const uint16_t *vc = reinterpret_cast<const uint16_t *>(tile + 8 * D);
    const int j = i / 2, c0 = 8 * (i % 2);
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int kc = (w >> (16 * (e & 1) + 4 * (e / 2))) & 15;
        const uint16_t vw = vc[(((r / 4) * 16 + c0 + e) * 2 + (r % 4) / 2) * NG + 2 * (j / 4) + r % 2];
        const int vn = (vw >> (4 * (j % 4))) & 15;
        k[e] = (_Float16)((float)dk * (float)(kc - 8));
        v[e] = (_Float16)((float)dv * (float)(vn - 8));
    }
}

template <int D>
__global__ __launch_bounds__(256) void k_kv_read(KvBatch b, _Float16 *k, _Float16 *v) {
    constexpr int L = D / 8;
    const int li = threadIdx.x % L;
    const int64_t u = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const bool live = u < (int64_t)b.n_tokens * b.n_kv;
    const int t = live ? (int)(u / b.n_kv) : 0, head = live ? (int)(u % b.n_kv) : 0;
    const int s = seq_of<L>(b, t, li);
    if (!live || s >= b.n_seqs) return;
    const SeqRows r = seq_rows(b, s);
    const int pos = r.len - r.hi + t, page = page_of(b, s, pos);
    f16x8 kk, vv;
    if (page >= 0) {
        held8<D>(b.pages + tile_at<D>(b, page, head, (pos % b.page_tokens) / 16), pos & 15, li, kk, vv);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) kk[e] = vv[e] = (_Float16)__builtin_nanf("");
    }
    const size_t o = ((size_t)t * b.n_kv + head) * D + 8 * li;
    *reinterpret_cast<f16x8 *>(k + o) = kk;
    *reinterpret_cast<f16x8 *>(v + o) = vv;
}

// ================================================================ attention
// One wave per (row, head): a lane scores one of 64 tokens, then holds D / 64
// dims of the output while the 64 weights pass by.
template <int D, bool BF>
__global__ __launch_bounds__(64) void k_attn_rows(KvBatch b, KvRows q, int n_heads, float scale, void *out,
                                                  int64_t out_stride) {
    constexpr int E = D / 64;
    __shared__ float sq[D], sp[64];
    const int t = blockIdx.x / n_heads, hq = blockIdx.x % n_heads, lane = threadIdx.x;
    const int s = seq_of<64>(b, t, lane);
    if (s >= b.n_seqs) return;
    const SeqRows r = seq_rows(b, s);
    const int pos = r.len - r.hi + t, hk = hq / (n_heads / b.n_kv);
    const uint16_t *qp = static_cast<const uint16_t *>(q.p) + (int64_t)t * q.stride + hq * D;
    for (int i = lane; i < D; i += 64) sq[i] = (BF ? bf2f(qp[i]) : h2f(qp[i])) * scale;
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[E] = {};
    for (int p0 = 0; p0 <= pos; p0 += 64) {
        const int p = p0 + lane;
        float sc = -INFINITY;
        const int page = p <= pos ? page_of(b, s, p) : 0;
        if (p <= pos) {
            sc = 0.0f;
            if (page >= 0) {
                const uint8_t *tile = b.pages + tile_at<D>(b, page, hk, (p % b.page_tokens) / 16);
                for (int i = 0; i < D / 8; i++) {
                    f16x8 kk, vv;
                    held8<D>(tile, p & 15, i, kk, vv);
                    for (int e = 0; e < 8; e++) sc += sq[8 * i + e] * (float)kk[e];
                }
            } else {
                sc = __builtin_nanf("");
            }
        }
        float top = sc;
        for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
        const float m2 = fmaxf(m, top), f = m2 > -INFINITY ? __expf(m - m2) : 1.0f;
        const float w = p <= pos ? __expf(sc - m2) : 0.0f;
        float sum = w;
        for (int x = 1; x < 64; x *= 2) sum += __shfl_xor(sum, x);
        l = l * f + sum;
        m = m2;
        sp[lane] = w;
        __syncthreads();
        for (int e = 0; e < E; e++) o[e] *= f;
        for (int j = 0; j < 64 && p0 + j <= pos; j++) {
            const int pg = page_of(b, s, p0 + j);
            if (pg < 0) continue;
            const uint8_t *tile = b.pages + tile_at<D>(b, pg, hk, ((p0 + j) % b.page_tokens) / 16);
            for (int e = 0; e < E; e++) {
                const int d = 64 * e + lane;
                f16x8 kk, vv;
                held8<D>(tile, (p0 + j) & 15, d / 8, kk, vv);
                o[e] += sp[j] * (float)vv[d % 8];
            }
        }
        __syncthreads();
    }
    for (int e = 0; e < E; e++) {
        const float v = pos < 0 ? 0.0f : o[e] / l;
        static_cast<uint16_t *>(out)[(int64_t)t * out_stride + hq * D + 64 * e + lane] = BF ? f2bf(v) : f2h(v);
    }
}

// ================================================================ launchers
#define TG_BY_DIM(D, ...)                                                     \
    do {                                                                      \
        if ((D) == 64) { constexpr int DIM = 64; __VA_ARGS__; }               \
        else if ((D) == 128) { constexpr int DIM = 128; __VA_ARGS__; }        \
        else { constexpr int DIM = 256; __VA_ARGS__; }                        \
    } while (0)

hipError_t launch_kv_append(const KvBatch &b, int type, const AppendArgs &a, hipStream_t st) {
    const int64_t units = (int64_t)b.n_tokens * (a.n_heads + 2 * b.n_kv);
    const int64_t grid = (units + 256 / (b.D / 8) - 1) / (256 / (b.D / 8));
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    TG_BY_DIM(b.D, {
        if (type == TG_T_F32) TG_LAUNCH((k_kv_append<DIM, TG_T_F32>), dim3((unsigned)grid), dim3(256), 0, st, b, a);
        else if (type == TG_T_F16) TG_LAUNCH((k_kv_append<DIM, TG_T_F16>), dim3((unsigned)grid), dim3(256), 0, st, b, a);
        else TG_LAUNCH((k_kv_append<DIM, TG_T_BF16>), dim3((unsigned)grid), dim3(256), 0, st, b, a);
    });
    return hipGetLastError();
}

hipError_t launch_kv_read(const KvBatch &b, void *k, void *v, hipStream_t st) {
    const int64_t units = (int64_t)b.n_tokens * b.n_kv;
    const int64_t grid = (units + 256 / (b.D / 8) - 1) / (256 / (b.D / 8));
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    TG_BY_DIM(b.D, TG_LAUNCH(k_kv_read<DIM>, dim3((unsigned)grid), dim3(256), 0, st, b, static_cast<_Float16 *>(k),
                             static_cast<_Float16 *>(v)));
    return hipGetLastError();
}

size_t attn_workspace(const KvBatch &b, int n_heads, int max_len) { return 0; }

hipError_t launch_attn(const KvBatch &b, int type, KvRows q, int n_heads, float scale, void *out, int64_t out_stride,
                       int max_len, void *ws, hipStream_t st) {
    const int64_t grid = (int64_t)b.n_tokens * n_heads;
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    TG_BY_DIM(b.D, {
        if (type == TG_T_F16) TG_LAUNCH((k_attn_rows<DIM, false>), dim3((unsigned)grid), dim3(64), 0, st, b, q, n_heads, scale, out, out_stride);
        else TG_LAUNCH((k_attn_rows<DIM, true>), dim3((unsigned)grid), dim3(64), 0, st, b, q, n_heads, scale, out, out_stride);
    });
    return hipGetLastError();
}

}  // namespace tg
