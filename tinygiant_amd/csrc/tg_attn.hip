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

#include <algorithm>

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
// Columns.  A sequence's rows and the G query heads of one key head are laid
// out as columns f = row * G + head, 16 of which make a column tile, the
// width of v_mfma_f32_16x16x32_f16.  Column tiles of all sequences are
// numbered so that a launch needs no look at cu: sequence s starts at
// cu[s] * G / 16 + s, at or behind the last tile of the sequence before it.
//
// Scores.  S^T = K Q^T with keys as the A operand: lane (c = lane % 16, h =
// lane / 16) supplies key token c (16 bytes of a tile: its codes 8 h .. 8 h +
// 7 of each block) and receives column c of tokens 4 h .. 4 h + 3, which is
// just the layout the weights need as the B operand of O^T = V^T P^T.
// The codes stay integers: a nibble masked in place is the fp16 subnormal
// code * 2^-24 (bits 0..3) or code * 2^-20 (bits 4..7), which the matrix
// instructions take exactly; the query operand carries the factor 16 between
// the two, the sum starts at -8 times the query's block sum, and the block's
// scale multiplies the fp32 sum.  So keys and queries are exact: a query row
// is scaled by a power of two to below 2^15 (its largest value in 2^10 ..
// 2^11), which drops nothing above 2^-24 of that.
//
// Weights are exp2(s - m + 4) with m raised (and the sums rescaled) only
// where a score passes m + 11: they stay below 2^15 as fp16 operands, and
// with m at most 11 below the largest score a weight is a normal fp16 down to
// 2^-18 of it.  Values are dequantised to fp16 (one rounding, 2^-11), the
// weights rounded to fp16 (2^-11); sums, maxima and outputs are fp32.
//
// A value block that is not finite makes the token's scores NaN and its values 0, so
// that rows which see the token are NaN and rows which do not are as ever.
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float AT_NONE = -3.402823466e38f;  // m of a column that has seen nothing
constexpr float AT_LIFT = 4.0f, AT_ROOM = 11.0f;

TG_DEV f16x2 as_h2(uint32_t v) { return __builtin_bit_cast(f16x2, v); }
TG_DEV uint32_t as_u(f16x2 v) { return __builtin_bit_cast(uint32_t, v); }
TG_DEV f16x8 as_h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const u32x4 v = {a, b, c, d};
    return __builtin_bit_cast(f16x8, v);
}
TG_DEV uint32_t pack_h2(float a, float b) {
    const f32x2 v = {a, b};
    return as_u(__builtin_convertvector(v, f16x2));
}

// a half whose exponent is all ones, in either half of v
TG_DEV bool odd_half(uint32_t v) { return (v & 0x7C00u) == 0x7C00u || (v & 0x7C000000u) == 0x7C000000u; }

// Column tile `z` of the launch: its sequence (or -1) and its number there.
struct ColTile {
    int seq, tile, lo, n, len;
};
TG_DEV ColTile col_tile(const KvBatch &b, int G, int cols, int z, int lane) {
    ColTile r{-1, 0, 0, 0, 0};
    for (int j0 = 0; j0 < b.n_seqs; j0 += 64) {
        const int j = j0 + lane;
        const bool in = j < b.n_seqs;
        const int lo = in ? min(max(b.cu[j], 0), b.n_tokens) : 0;
        const int hi = in ? min(max(b.cu[j + 1], lo), b.n_tokens) : 0;
        const int len = in ? max(b.kv_len[j], 0) : 0;
        const int first = (int)((int64_t)lo * G / cols) + j;
        const uint64_t m = __ballot(in && first <= z);
        if (m) {
            // cu does not decrease, so neither does first: the last lane of m
            const int k = 63 - __builtin_clzll(m);
            r.seq = j0 + k;
            r.tile = z - __builtin_amdgcn_readlane(first, k);
            r.lo = __builtin_amdgcn_readlane(lo, k);
            r.n = __builtin_amdgcn_readlane(hi, k) - r.lo;
            r.len = __builtin_amdgcn_readlane(len, k);
        }
        if (m != ~0ull) break;
    }
    if (r.seq >= 0 && (int64_t)r.tile * cols >= (int64_t)r.n * G) r.seq = -1;
    return r;
}

// How many tokens row i of the sequence sees.  One beyond the table is
// enough to make NaN of it, so a length that no table holds costs no more.
TG_DEV int tokens_seen(const KvBatch &b, const ColTile &ct, int i) {
    return max(0, min(ct.len - ct.n + i + 1, b.table_cols * b.page_tokens + 1));
}

// One step of 32 tokens of one key head as a lane holds it: tiles x = 0, 1
template <int D>
struct KvStep {
    static constexpr int NG = D / 32, SW = D / 64;  // scale words per lane and step
    uint32_t k[2][NG], v[2][2][NG / 2], s[SW];
    bool bad[2];
};

template <int N>
TG_DEV void load_words(const void *p, uint32_t *w) {
    if constexpr (N == 2) {
        const u32x2 v = *static_cast<const u32x2 *>(p);
        w[0] = v[0], w[1] = v[1];
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const u32x4 v = *reinterpret_cast<const u32x4 *>(static_cast<const uint32_t *>(p) + i);
#pragma unroll
            for (int e = 0; e < 4; e++) w[i + e] = v[e];
        }
    }
}

// Few columns: split over the tokens.  A block holds one column tile of one
// key head and a chunk of tokens, its four waves every fourth step of 32; the
// packed bytes go from memory to registers one step ahead and are unpacked
// there (each is used by one wave, so LDS would only add a trip), the scales
// through a wave's corner of LDS because 16 lanes need the same ones.  Chunks
// of one column tile are joined by k_attn_join, or written out at once where
// one chunk is all.
struct AttnOut {
    void *p;
    int64_t stride;
    float *part;  // [column tile][key head][split][16][D + 2]
};

template <int D, bool BF>
__global__ __launch_bounds__(256, 2) void k_attn_split(KvBatch b, KvRows q, int G, float scale, int chunk, int nsplit,
                                                       AttnOut o) {
    constexpr int NG = D / 32, ND = D / 16, SW = D / 64;
    __shared__ __align__(16) uint8_t sm[4 * 16 * D * 4 + 4 * 16 * 8];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int c = lane % 16, h = lane / 16;
    const int z = blockIdx.x, hk = blockIdx.y, split = blockIdx.z;
    const ColTile ct = col_tile(b, G, 16, z, lane);
    if (ct.seq < 0) return;
    // this lane's column
    const int f = ct.tile * 16 + c, last = min(ct.n * G - 1, ct.tile * 16 + 15);
    const bool col = f < ct.n * G;
    const int row = ct.lo + (col ? f / G : 0), head = hk * G + (col ? f % G : 0);
    const int pos = col ? ct.len - ct.n + f / G : -1;
    const int seen = tokens_seen(b, ct, last / G);
    const int t0 = split * chunk, t1 = split == nsplit - 1 ? seen : min(seen, t0 + chunk);
    if (t0 >= t1 && split > 0) return;  // a column tile that sees nothing is split 0's to write

    // queries: operand slots 8 h .. 8 h + 7 of each block, and the start of the sums
    f16x8 qf[NG];
    f32x4 start[NG];
    float cs;
    {
        const uint16_t *qp = static_cast<const uint16_t *>(q.p) + (int64_t)row * q.stride + (int64_t)head * D;
        float x[NG][8], top = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            uint32_t w[4];
            load_words<4>(qp + 32 * g + 8 * h, w);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint16_t u = (uint16_t)(w[e / 2] >> (16 * (e % 2)));
                x[g][e] = col ? (BF ? bf2f(u) : h2f(u)) : 0.0f;
                top = fmaxf(top, fabsf(x[g][e]));
            }
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        int e2 = 0;
        (void)frexpf(top, &e2);  // top = m 2^e2, m in [0.5, 1)
        const int a = top > 0.0f && top < INFINITY ? 11 - e2 : 0;
        cs = ldexpf(scale * 1.44269504f, 20 - a);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const _Float16 v = (_Float16)ldexpf(x[g][e], a + ((e / 2) % 2 ? 0 : 4));
                qf[g][e] = v;
                sum += (e / 2) % 2 ? (float)v * 16.0f : (float)v;
            }
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            const float st = sum * (-8.0f / 16777216.0f);
            start[g] = f32x4{st, st, st, st};
        }
    }

    uint32_t *sl = reinterpret_cast<uint32_t *>(sm) + wave * (16 * D);  // this wave's corner
    f32x4 acc[ND] = {};
    float m = AT_NONE, l = 0.0f;
    const int ptok = b.page_tokens, span = min(chunk, 63 * ptok & ~31);
    for (int c0 = t0; c0 < t1; c0 += span) {
        const int c1 = min(t1, c0 + span);
        // this stretch's pages, one to a lane
        const int page0 = c0 / ptok;
        const int mine = c0 / ptok * ptok + lane * ptok < c1 ? page_of(b, ct.seq, (page0 + lane) * ptok) : 0;
        auto load = [&](int st, KvStep<D> &k) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                int t = st * 32 + 16 * x;
                t = t < c1 ? t : c0;  // behind the end: any tile, its tokens are masked
                const int pg = __builtin_amdgcn_readlane(mine, t / ptok - page0);
                k.bad[x] = pg < 0;
                const uint8_t *p = b.pages + tile_at<D>(b, max(pg, 0), hk, (t % ptok) / 16);
                load_words<NG>(p + lane * (NG * 4), k.k[x]);
                load_words<NG>(p + 8 * D + lane * (NG * 4), &k.v[x][0][0]);
                // lane's share of the scales: the step's 4 D bytes over 64 lanes
                if (SW == 1) {
                    if (lane / 32 == x) k.s[0] = reinterpret_cast<const uint32_t *>(p + 16 * D)[lane % 32];
                } else {
#pragma unroll
                    for (int i = 0; i < SW / 2; i++)
                        k.s[x * (SW / 2) + i] = reinterpret_cast<const uint32_t *>(p + 16 * D)[lane * (SW / 2) + i];
                }
            }
        };
        const int s1 = (c1 + 31) / 32;
        int st = c0 / 32 + wave;
        KvStep<D> cur, nxt;
        if (st < s1) load(st, nxt);
        for (; st < s1; st += 4) {
            cur = nxt;
            if (st + 4 < s1) load(st + 4, nxt);
            const bool edge = st * 32 + 31 > ct.len - ct.n + (ct.tile * 16) / G;  // some column does not see all of it
            // scales to LDS as the tiles hold them; what no column sees is zero
            bool oddv = false;
#pragma unroll
            for (int i = 0; i < SW; i++) {
                const int w = SW == 1 ? lane % 32 : lane * (SW / 2) + i % (SW / 2);  // word of the tile's 2 D bytes
                const int x = SW == 1 ? lane / 32 : i / (SW / 2);
                uint32_t v = cur.s[i];
                const bool isv = w >= D / 4;
                if (edge) {
                    const int t = st * 32 + 16 * x;
                    if (!isv) {
                        if (t + w / (NG / 2) >= seen) v = 0;
                    } else {
                        const int tp = t + (w - D / 4) / NG * 2;
                        if (tp + 1 >= seen) v &= 0xFFFFu;
                        if (tp >= seen) v = 0;
                    }
                }
                oddv |= isv && odd_half(v);
                sl[x * (D / 2) + w] = v;
            }
            const bool odd = __ballot(oddv) != 0 || cur.bad[0] || cur.bad[1];
            wave_lds_sync();
            float s[2][4];
#pragma unroll
            for (int x = 0; x < 2; x++) {
                uint32_t kd[2 * NG];  // halves [token i][block g]
                load_words<2 * NG>(sl + x * (D / 2) + h * (2 * NG), kd);
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    const uint32_t w = cur.k[x][g], w8 = w >> 8;
                    const f16x8 kf = as_h8(w & 0x000F000Fu, w & 0x00F000F0u, w8 & 0x000F000Fu, w8 & 0x00F000F0u);
                    const f32x4 r = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[g], start[g], 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float d = (float)as_h2(kd[(i * NG + g) / 2])[g % 2];
                        s[x][i] = g == 0 ? d * r[i] : __builtin_fmaf(d, r[i], s[x][i]);
                    }
                }
            }
            if (odd) {
                // NaN for the tokens of a bad page and of value blocks that are not finite; those blocks become 0
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    uint32_t vd[2 * NG];
                    load_words<2 * NG>(sl + x * (D / 2) + D / 4 + h * (2 * NG), vd);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        bool n = cur.bad[x];
#pragma unroll
                        for (int g = 0; g < NG; g++) n |= ((vd[(i / 2) * NG + g] >> (16 * (i % 2))) & 0x7C00u) == 0x7C00u;
                        if (n) s[x][i] = __builtin_nanf("");
                    }
                }
                wave_lds_sync();
#pragma unroll
                for (int i = 0; i < SW; i++) {
                    const int w = SW == 1 ? lane % 32 : lane * (SW / 2) + i % (SW / 2);
                    const int x = SW == 1 ? lane / 32 : i / (SW / 2);
                    if (w >= D / 4) {
                        uint32_t v = sl[x * (D / 2) + w];
                        if ((v & 0x7C00u) == 0x7C00u) v &= 0xFFFF0000u;
                        if ((v & 0x7C000000u) == 0x7C000000u) v &= 0xFFFFu;
                        sl[x * (D / 2) + w] = v;
                    }
                }
                wave_lds_sync();
            }
            if (edge) {
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (st * 32 + 16 * x + 4 * h + i > pos) s[x][i] = -INFINITY;
            }
            // cs > 0, so the largest s is the largest score
            float top = s[0][0];
#pragma unroll
            for (int i = 1; i < 8; i++) top = fmaxf(top, s[i / 4][i % 4]);
            if (__ballot(top * cs > m + AT_ROOM)) {
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float m2 = fmaxf(m, top * cs), r = __builtin_amdgcn_exp2f(m - m2);
                l *= r;
#pragma unroll
                for (int j = 0; j < ND; j++) acc[j] *= r;
                m = m2;
            }
            const float off = AT_LIFT - m;
            float p[2][4];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                p[i / 4][i % 4] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 4][i % 4], cs, off));
                l += p[i / 4][i % 4];
            }
            const f16x8 pf = as_h8(pack_h2(p[0][0], p[0][1]), pack_h2(p[0][2], p[0][3]), pack_h2(p[1][0], p[1][1]),
                                   pack_h2(p[1][2], p[1][3]));
            // values: words [token pair][block] of each tile's scales
            uint32_t vd[2][2 * NG];
#pragma unroll
            for (int x = 0; x < 2; x++) load_words<2 * NG>(sl + x * (D / 2) + D / 4 + h * (2 * NG), vd[x]);
#pragma unroll
            for (int bq = 0; bq < NG / 2; bq++) {
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    uint32_t w[4];
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        const uint32_t raw = cur.v[y / 2][y % 2][bq], sh = n < 2 ? raw : raw >> 8;
                        f16x2 t;
                        if (n % 2 == 0) t = as_h2((sh & 0x000F000Fu) | 0x64006400u) - f16x2{(_Float16)1032.0f, (_Float16)1032.0f};
                        else t = as_h2((sh & 0x00F000F0u) | 0x54005400u) - f16x2{(_Float16)72.0f, (_Float16)72.0f};
                        w[y] = as_u(t * as_h2(vd[y / 2][(y % 2) * NG + 2 * bq + n / 2]));
                    }
                    acc[4 * bq + n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(w[0], w[1], w[2], w[3]), pf, acc[4 * bq + n], 0, 0, 0);
                }
            }
            wave_lds_sync();
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // the waves' shares joined in order: O[wave][column][D], m and l [wave][column]
    __syncthreads();
    float *so = reinterpret_cast<float *>(sm) + wave * 16 * D, *sml = reinterpret_cast<float *>(sm + 4 * 16 * D * 4);
#pragma unroll
    for (int j = 0; j < ND; j++) *reinterpret_cast<f32x4 *>(so + c * D + 16 * j + 4 * h) = acc[j];
    if (h == 0) sml[(wave * 16 + c) * 2] = m, sml[(wave * 16 + c) * 2 + 1] = l;
    __syncthreads();
    const int active = (seen + chunk - 1) / chunk;
    const bool whole = active <= 1 || nsplit == 1;
    for (int i = threadIdx.x; i < 16 * D / 4; i += 256) {
        const int cc = i / (D / 4), d = (i % (D / 4)) * 4, ff = ct.tile * 16 + cc;
        if (ff >= ct.n * G) break;
        float mm = AT_NONE, ll = 0.0f;
        f32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; w++) mm = fmaxf(mm, sml[(w * 16 + cc) * 2]);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float r = __builtin_amdgcn_exp2f(sml[(w * 16 + cc) * 2] - mm);
            ll += sml[(w * 16 + cc) * 2 + 1] * r;
            v += *reinterpret_cast<const f32x4 *>(reinterpret_cast<float *>(sm) + (w * 16 + cc) * D + d) * r;
        }
        if (whole) {
            const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
            store4<BF ? TG_T_BF16 : TG_T_F16>(o.p, (int64_t)(ct.lo + ff / G) * o.stride + (int64_t)(hk * G + ff % G) * D + d, v * inv);
        } else {
            float *pp = o.part + ((((size_t)z * b.n_kv + hk) * nsplit + split) * 16 + cc) * (D + 2);
            pp[d] = v[0], pp[d + 1] = v[1], pp[d + 2] = v[2], pp[d + 3] = v[3];
            if (d == 0) pp[D] = mm, pp[D + 1] = ll;
        }
    }
}

// The splits of one column tile, joined in order.
template <int D, bool BF>
__global__ __launch_bounds__(256) void k_attn_join(KvBatch b, int G, int chunk, int nsplit, AttnOut o) {
    const int hk = blockIdx.y, z = blockIdx.x;
    const ColTile ct = col_tile(b, G, 16, z, threadIdx.x % 64);
    if (ct.seq < 0) return;
    const int last = min(ct.n * G - 1, ct.tile * 16 + 15), seen = tokens_seen(b, ct, last / G);
    const int active = min(nsplit, (seen + chunk - 1) / chunk);
    if (active <= 1) return;
    const float *part = o.part + ((size_t)z * b.n_kv + hk) * nsplit * 16 * (D + 2);
    for (int i = threadIdx.x; i < 16 * D; i += 256) {
        const int cc = i / D, d = i % D, ff = ct.tile * 16 + cc;
        if (ff >= ct.n * G) break;
        float mm = AT_NONE, ll = 0.0f, v = 0.0f;
        for (int s = 0; s < active; s++) mm = fmaxf(mm, part[(s * 16 + cc) * (D + 2) + D]);
        for (int s = 0; s < active; s++) {
            const float *pp = part + (s * 16 + cc) * (D + 2);
            const float r = __builtin_amdgcn_exp2f(pp[D] - mm);
            ll += pp[D + 1] * r;
            v += pp[d] * r;
        }
        v *= ll == 0.0f ? 0.0f : 1.0f / ll;
        static_cast<uint16_t *>(o.p)[(int64_t)(ct.lo + ff / G) * o.stride + (int64_t)(hk * G + ff % G) * D + d] = BF ? f2bf(v) : f2h(v);
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

// Splits of one launch: chunks of a power of two of 128 tokens or more, so
// many that about 1024 blocks of the longest sequences share the device.
struct AttnPlan {
    int64_t tiles;
    int chunk, nsplit;
};
static AttnPlan attn_plan(const KvBatch &b, int n_heads, int max_len) {
    const int G = n_heads / b.n_kv;
    AttnPlan p;
    p.tiles = (int64_t)b.n_tokens * G / 16 + b.n_seqs;
    p.chunk = 128;
    while (p.chunk < 4096 && (int64_t)p.chunk * 2048 < (int64_t)max_len * p.tiles * b.n_kv) p.chunk *= 2;
    while (max_len / p.chunk >= 4096) p.chunk *= 2;
    p.nsplit = std::max(1, (max_len + p.chunk - 1) / p.chunk);
    return p;
}

size_t attn_workspace(const KvBatch &b, int n_heads, int max_len) {
    const AttnPlan p = attn_plan(b, n_heads, max_len);
    return p.nsplit == 1 ? 0 : (size_t)p.tiles * b.n_kv * p.nsplit * 16 * (b.D + 2) * sizeof(float);
}

hipError_t launch_attn(const KvBatch &b, int type, KvRows q, int n_heads, float scale, void *out, int64_t out_stride,
                       int max_len, void *ws, hipStream_t st) {
    const AttnPlan p = attn_plan(b, n_heads, max_len);
    if (p.tiles > INT32_MAX) return hipErrorInvalidValue;
    const int G = n_heads / b.n_kv;
    const AttnOut o{out, out_stride, static_cast<float *>(ws)};
    const dim3 grid((unsigned)p.tiles, (unsigned)b.n_kv, (unsigned)p.nsplit), join((unsigned)p.tiles, (unsigned)b.n_kv);
    TG_BY_DIM(b.D, {
        if (type == TG_T_F16) TG_LAUNCH((k_attn_split<DIM, false>), grid, dim3(256), 0, st, b, q, G, scale, p.chunk, p.nsplit, o);
        else TG_LAUNCH((k_attn_split<DIM, true>), grid, dim3(256), 0, st, b, q, G, scale, p.chunk, p.nsplit, o);
        if (p.nsplit > 1) {
            if (type == TG_T_F16) TG_LAUNCH((k_attn_join<DIM, false>), join, dim3(256), 0, st, b, G, p.chunk, p.nsplit, o);
            else TG_LAUNCH((k_attn_join<DIM, true>), join, dim3(256), 0, st, b, G, p.chunk, p.nsplit, o);
        }
    });
    return hipGetLastError();
}

}  // namespace tg
