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
#include <atomic>
#include <type_traits>

namespace tg {

// ================================================================ the batch
// byte of a page's tile for one key head
template <int D>
TG_DEV size_t tile_at(const KvBatch &b, int page, int head, int tile) {
    return (((size_t)page * b.n_kv + head) * (b.page_tokens / 16) + tile) * (size_t)(18 * D);
}

// Rows [lo, hi) of a sequence, kept inside the row tensors whatever cu holds,
// and the tokens up to row hi - 1: its length less the rows behind the
// tensors' end (so below 0 where those are more than its tokens).
struct SeqRows {
    int lo, hi, len;
};
TG_DEV SeqRows seq_rows(const KvBatch &b, int c0, int c1, int len) {
    SeqRows r;
    r.lo = min(max(c0, 0), b.n_tokens);
    const int end = max(c1, r.lo);
    r.hi = min(end, b.n_tokens);
    r.len = max(len, 0) - (end - r.hi);
    return r;
}
TG_DEV SeqRows seq_rows(const KvBatch &b, int s) { return seq_rows(b, b.cu[s], b.cu[s + 1], b.kv_len[s]); }

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
// Three prompts of 3001, 2965 and 1819 tokens, fp32, 32 heads of 64 over 8: 40 us, 4.0 TB/s
// (50 where waves of q alone went through the quantising too and rows were
// found by 64-bit divisions); one token 4.1, 61 tokens 5.4, which are their latency.
template <int D, int TYPE>
__global__ __launch_bounds__(256) void k_kv_append(KvBatch b, AppendArgs a) {
    constexpr int L = D / 8, NG = D / 32;
    const uint32_t units = a.n_heads + 2 * b.n_kv;
    const int li = threadIdx.x % L;
    const uint32_t u = blockIdx.x * (256 / L) + threadIdx.x / L;  // below 2^32 / L, as the launch checks
    const bool live = u < (uint64_t)b.n_tokens * units;
    const int t = live ? (int)(u / units) : 0, slot = live ? (int)(u - (uint32_t)t * units) : 0;
    const bool is_q = slot < a.n_heads, is_v = slot >= a.n_heads + b.n_kv;
    const int head = is_q ? slot : is_v ? slot - a.n_heads - b.n_kv : slot - a.n_heads;
    const KvRows src = is_q ? a.q : is_v ? a.v : a.k;
    f32x4 lo = load4<TYPE>(src.p, (int64_t)t * src.stride + head * D + 4 * li);
    f32x4 hi = load4<TYPE>(src.p, (int64_t)t * src.stride + head * D + D / 2 + 4 * li);

    const int s = seq_of<L>(b, t, li);
    const bool row = live && s < b.n_seqs;
    int pos = -1, page = -1, turn = -1;  // place, its page, the position that it is rotated by
    if (row) {
        const SeqRows r = seq_rows(b, s);
        pos = turn = r.len - r.hi + t;
        // a node of a draft tree has its own place but stands as many steps behind the sequence as it is deep
        if (a.depth) {
            const int depth = a.depth[t];
            turn = depth < 0 ? -1 : r.len - r.hi + r.lo + depth;
        }
        if (turn < 0 || turn >= a.max_pos) pos = -1;
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
        const f32x4 c = *reinterpret_cast<const f32x4 *>(a.cos + (size_t)turn * (D / 2) + 4 * li);
        const f32x4 sn = *reinterpret_cast<const f32x4 *>(a.sin + (size_t)turn * (D / 2) + 4 * li);
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
    // q's lanes take part in the exchanges below where units of one wave differ in kind
    if (!__ballot(row && !is_q)) return;
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
    const uint32_t u = blockIdx.x * (256 / L) + threadIdx.x / L;
    const bool live = u < (uint64_t)b.n_tokens * b.n_kv;
    const int t = live ? (int)(u / (uint32_t)b.n_kv) : 0, head = live ? (int)(u - (uint32_t)t * b.n_kv) : 0;
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

// ================================================================ keep
// The token that a walk through a draft tree kept as its i-th to place i of the tree, codes and scales as they are.  A
// wave has one key head of one sequence in KEEP_LAYERS layers and goes through the places in order: entry i comes from
// path[i] >= i, so no place is written before what it held is read.
//
// Bound by latency: cu and kv_len, path and count, the table, and then the entries, those of all its layers at once but
// one after the other, 0.6 us each: 1 user, 48 layers of 4 heads of 128, 4 entries moved 5.8 us, 16 13, 64 44, 256 166.
// 64 users with a few each, a layer to a wave 18.2 us (more waves than the card holds at once, entries four at a time),
// four layers 10.5; 1 user 4.6 either way.  The lengths by a launch of their own: 1 user 10.1 us a call, 6.6 so.
constexpr int KEEP_LAYERS = 4;
template <int D>
__global__ __launch_bounds__(256) void k_kv_keep(KvBatch b, KeepArgs a) {
    constexpr int NG = D / 32, KW = D / 8, VH = D / 4, ITEMS = KW + VH + 2 * NG;  // K words, V halfwords, scales of a token
    constexpr int PER = (ITEMS + 63) / 64;
    const int lane = threadIdx.x % 64;
    const uint32_t unit = blockIdx.x * 4 + uni(threadIdx.x / 64), pair = unit / b.n_kv;  // below 2^26, as the launch checks
    const int hk = unit - pair * b.n_kv, group = pair / b.n_seqs, s = pair - group * b.n_seqs;
    const int layer = group * KEEP_LAYERS, layers = min(KEEP_LAYERS, a.n_layers - layer);
    if (layers <= 0) return;
    const int lo = max(b.cu[s], 0), n = max(b.cu[s + 1], lo) - lo, base = max(b.kv_len[s], 0) - n;
    const int count = min(max(a.count[s], 0), min(n, a.path_cols));
    if (a.kv_len && a.kv_len != b.kv_len && layer == 0 && hk == 0 && lane == 0) a.kv_len[s] = max(base + count, 0);
    uint8_t *pages = b.pages + layer * a.layer_bytes;
    // bytes of this lane's items in token r's tile: V's as halfwords, K's as words
    auto at = [&](int item, int r) {
        if (item < KW) return ((item / NG * 16 + r) * NG + item % NG) * 4;
        item -= KW;
        if (item < VH) return 8 * D + ((((r / 4) * 16 + item / (NG / 2)) * 2 + r % 4 / 2) * NG + 2 * (item % (NG / 2)) + r % 2) * 2;
        item -= VH;
        if (item < NG) return 16 * D + (r * NG + item) * 2;
        return 17 * D + ((r / 2 * NG + item - NG) * 2 + r % 2) * 2;
    };
    for (int i0 = 0; i0 < count; i0 += 64) {
        // lane i finds entry i0 + i's places
        const int i = i0 + lane, from = i < count ? a.path[(int64_t)s * a.path_stride + i] : i;
        const int to_page = i < count && from != i ? page_of(b, s, base + i) : -1;
        const int from_page = to_page >= 0 && from > i && from < n ? page_of(b, s, base + from) : -1;
        for (uint64_t todo = __ballot(to_page >= 0); todo; todo &= todo - 1) {
            const int e = __builtin_ctzll(todo);
            const int tp = __builtin_amdgcn_readlane(to_page, e), fp = __builtin_amdgcn_readlane(from_page, e);
            const int t = base + i0 + e, f = fp < 0 ? t : base + __builtin_amdgcn_readlane(from, e);
            uint8_t *tt = pages + tile_at<D>(b, tp, hk, t % b.page_tokens / 16);
            const uint8_t *ft = pages + tile_at<D>(b, fp < 0 ? tp : fp, hk, f % b.page_tokens / 16);
            uint32_t v[KEEP_LAYERS][PER];
#pragma unroll
            for (int q = 0; q < KEEP_LAYERS; q++)
#pragma unroll
                for (int k = 0; k < PER; k++) {
                    const int item = min(lane + 64 * k, ITEMS - 1);
                    const uint8_t *p = ft + min(q, layers - 1) * a.layer_bytes + at(item, f % 16);
                    if (item < KW) v[q][k] = *reinterpret_cast<const uint32_t *>(p);
                    else v[q][k] = *reinterpret_cast<const uint16_t *>(p);
                    if (fp < 0 && item >= KW + VH) v[q][k] = 0x7E00;  // an entry that is none: NaN for scales
                }
#pragma unroll
            for (int q = 0; q < KEEP_LAYERS; q++) {
                if (q >= layers) break;
#pragma unroll
                for (int k = 0; k < PER; k++) {
                    const int item = lane + 64 * k;
                    if (item >= ITEMS) break;
                    uint8_t *p = tt + q * a.layer_bytes + at(item, t % 16);
                    if (item < KW) *reinterpret_cast<uint32_t *>(p) = v[q][k];
                    else *reinterpret_cast<uint16_t *>(p) = (uint16_t)v[q][k];
                }
            }
        }
    }
}

// The lengths where they take the place of the ones before, which every other block reads: a launch of their own.
__global__ __launch_bounds__(256) void k_kv_keep_len(KvBatch b, KeepArgs a) {
    const int s = blockIdx.x * 256 + threadIdx.x;
    if (s >= b.n_seqs) return;
    const int lo = max(b.cu[s], 0), n = max(b.cu[s + 1], lo) - lo;
    a.kv_len[s] = max(max(b.kv_len[s], 0) - n + min(max(a.count[s], 0), min(n, a.path_cols)), 0);
}

// ================================================================ attention
// Columns.  A sequence's rows and the G query heads of one key head are laid
// out as columns f = row * G + head, 16 of which make a column tile, the
// width of v_mfma_f32_16x16x32_f16.  Which blocks do which tiles and tokens is worked out on the
// device from cu and kv_len (Cut and col_tile, below); the launch knows only how many there can be.
//
// Scores.  S^T = K Q^T with keys as the A operand: lane (c = lane % 16, h =
// lane / 16) supplies key token c (16 bytes of a tile: its codes 8 h .. 8 h +
// 7 of each block) and receives column c of tokens 4 h .. 4 h + 3, which is
// just the layout the weights need as the B operand of O^T = V^T P^T.
// The codes stay integers: a nibble shifted to bits 2..5 or 6..9 of a half and
// masked is the fp16 subnormal code * 2^-22 or code * 2^-18, which the matrix
// instructions take; the query operand carries the factor 16 between the
// two, the sum starts at -8 times the query's block sum, and the block's
// scale multiplies the fp32 sum.  So keys and queries are exact: a query row
// is scaled by a power of two to below 2^15 (its largest value in 2^10 ..
// 2^11), which drops nothing above 2^-24 of that.  What the instruction adds up
// is aligned to its largest product, a subnormal counting as 2^-14, and cut
// 2^-24 below it: 32 addends lose at most 2^-11 of the largest query value times one
// step of the block (measured: a tenth of it).  Unshifted nibbles (bits
// 0..3 and 4..7) would lose four times that and save one shift in 5 operations.
//
// Weights and values.  A value block's scale d multiplies the weight, p' =
// exp2(s - m + A) d, one rounding to fp16, once for its two column tiles, and
// the codes stay the integers they are, again as subnormals; a constant operand of -8
// takes the codes' offset off within the same step, so no sum grows with it.
// A = 9 - e where every scale so far is below 2^e (2^(e - 1) when A was set: one bit of room), and m is raised
// (and the sums rescaled) only where a score passes m + 6: p' stays below 2^15, 2^15.25 with m's own rounding
// (coarse, below), and next to the largest weight on the largest scale, 2^7 or more when A was set, it is a normal
// fp16 down to 2^-21, the smallest subnormal at 2^-31.  Sums, maxima and outputs are fp32.
//
// A value block that is not finite makes the token's scores NaN and its values 0, so
// that rows which see the token are NaN and rows which do not are as ever; its scales do not count for A.
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float AT_NONE = -3.402823466e38f;  // m of a column that has seen nothing
constexpr uint32_t AT_EVEN = 0x003C003Cu, AT_ODD = 0x03C003C0u;  // codes in bits 2..5, 6..9 of both halves
constexpr float AT_LEAST = 1e-37f;           // of the factor on scores: times it -inf stays -inf, and finite sums vanish
constexpr float AT_MOST = 3.402823466e38f;   // ... and +-0 stays 0
constexpr float AT_ROOM = 6.0f;
constexpr float AT_FINE = 4194304.0f;        // up to this m (2^22) a score's product, m and A fit one multiply-add
constexpr int AT_TOP = 9;                    // A + e, and A of the wide tiles

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

// The maximum of v over the four lanes that share a column (lane % 16)
TG_DEV float col_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
TG_DEV float col_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// What a score's fp32 sum is multiplied by, scale log2(e) 2^e.  Between its bounds: beyond them, scores that fp32 holds
// differ by so much, or so little, that the weights are the same.
TG_DEV float score_factor(float scale, int e) {
    return fminf(fmaxf(ldexpf(scale, e) * 1.44269504f, AT_LEAST), AT_MOST);
}

// Is some m so large that exponents have to be formed in two steps?  exp2(s cs + (A - m)) as one multiply-add is exact
// in s cs, but m and A - m are rounded, together by 2^(k - 24) where m is below 2^k: a factor on all of a column's
// weights, which falls out in the end if fp16 holds them.  Up to 2^22 it is below 2^0.25, and p' below 2^15.25;
// beyond 2^26 it could be 2^8.  In two steps, s cs - m and then A, the largest weight is 2^A again, and a score is
// off by the rounding of its product.
TG_DEV bool coarse(float m) { return __ballot(fabsf(m) > AT_FINE && m != AT_NONE) != 0; }

// One sequence as a lane of the planning scan holds it
struct SeqWork {
    int lo, n, len, tiles, steps;
};
template <int COLS>
TG_DEV SeqWork seq_work(const KvBatch &b, int G, int j) {
    const bool in = j < b.n_seqs;
    const int jj = in ? j : 0;  // three loads side by side, not one behind the other
    const int c0 = b.cu[jj], c1 = b.cu[jj + 1], cl = b.kv_len[jj];
    const SeqRows r = seq_rows(b, c0, c1, cl);
    SeqWork w;
    w.lo = r.lo;
    w.n = in ? r.hi - r.lo : 0;
    w.len = r.len;
    const int64_t cols = (int64_t)w.n * G;
    w.tiles = cols >= b.cols_from && cols < b.cols_to ? (int)((cols + COLS - 1) / COLS) : 0;
    w.steps = max(1, (min(w.len, b.table_cols * b.page_tokens + 1) + 31) / 32);
    return w;
}

// Inclusive sums over the wave's lanes (rows of 16 by shifts, then across rows)
template <class T>
TG_DEV T wave_scan(T v) {
    auto from = [&](auto ctrl, auto rows, auto zero) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value,
                                                                 decltype(rows)::value, 0xF, decltype(zero)::value));
    };
    using std::integral_constant;
    constexpr integral_constant<int, 0xF> all{};
    constexpr std::true_type zero{};
    v += from(integral_constant<int, 0x111>{}, all, zero);
    v += from(integral_constant<int, 0x112>{}, all, zero);
    v += from(integral_constant<int, 0x114>{}, all, zero);
    v += from(integral_constant<int, 0x118>{}, all, zero);
    v += from(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{}, std::false_type{});
    v += from(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{}, std::false_type{});
    return v;
}
template <class T>
TG_DEV T wave_sum(T v) { return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_scan(v)), 63)); }

// How a launch of wide column tiles is cut.  Sequence s has `tiles` of them of
// `steps` steps of 32 tokens.  A block takes at most `each` steps of one tile, the fewest
// (from an even share on, an eighth more at a time, 16 times at the most) with which all the pieces of a key head are
// `share` blocks or less, so that one round of the device's CUs does them
// all and the longest block is as short as that allows, and AT_WIDE at the least: what a piece costs
// beside its steps (its start, 128 KB of partial sums written and read) is as long as 16.  A tile is one piece at the
// least, so next to `share` short tiles a long one leaves up to share / 6.6 pieces for a second round.
// Every block works this out for itself from cu and kv_len (a wave's
// scan), so a launch follows lengths that only the device knows.
constexpr int AT_WIDE = 32;
struct ColTile {
    int seq, tile, lo, n, len;
    int split, splits, per;  // this split of the tile's, tokens of one split
    int part;                // the tile's first partial result (splits > 1)
    int join, joins;         // its place among the tiles that are split, and how many those are
};
// splits of `steps` steps where a block takes 1 / inv of them (the same in every block; per covers them all)
TG_DEV int splits_of(int steps, float inv) { return max(1, (int)ceilf((float)steps * inv)); }

// 1 / (the most steps of one block)
template <int COLS>
TG_DEV float block_share(const KvBatch &b, int G, int share, int lane, const SeqWork &w0) {
    if (share == 0) return 0.0f;  // no splits
    float all = (float)w0.tiles * (float)w0.steps;
    for (int j = lane + 64; j < (b.n_seqs + 63) / 64 * 64; j += 64) {
        const SeqWork w = seq_work<COLS>(b, G, j);
        all += (float)w.tiles * (float)w.steps;
    }
    float each = fmaxf((float)AT_WIDE, wave_sum(all) / (float)share);
    if (b.n_seqs > 64) return 1.0f / (each * 1.5f);
    for (int i = 0; i < 16 && wave_sum(w0.tiles * splits_of(w0.steps, 1.0f / each)) > share; i++) each *= 1.125f;
    return 1.0f / each;
}

// Block x of the launch; seq -1 where there is none.
template <int COLS>
TG_DEV ColTile col_tile(const KvBatch &b, int G, int share, int x, int lane) {
    const SeqWork w0 = seq_work<COLS>(b, G, lane);
    const float inv = block_share<COLS>(b, G, share, lane, w0);
    ColTile r{-1, 0, 0, 0, 0, 0, 1, 0, 0, 0, 0};
    int before = 0, parts = 0, joins = 0;
    for (int j0 = 0; j0 < b.n_seqs; j0 += 64) {
        const SeqWork w = j0 == 0 ? w0 : seq_work<COLS>(b, G, j0 + lane);
        const int splits = splits_of(w.steps, inv);
        const int mine = w.tiles * splits, mparts = splits > 1 ? mine : 0;
        const int items = wave_scan(mine), ps = wave_scan(mparts);
        const int mjoins = splits > 1 ? w.tiles : 0, js = wave_scan(mjoins);
        const uint64_t m = __ballot(before + items > x);
        if (m && before <= x) {
            const int k = __builtin_ctzll(m);
            const int sp = __builtin_amdgcn_readlane(splits, k), st = __builtin_amdgcn_readlane(w.steps, k);
            const int local = x - before - __builtin_amdgcn_readlane(items, k) + __builtin_amdgcn_readlane(mine, k);
            r.seq = j0 + k;
            r.tile = local / sp;
            r.split = local - r.tile * sp;
            r.lo = __builtin_amdgcn_readlane(w.lo, k);
            r.n = __builtin_amdgcn_readlane(w.n, k);
            r.len = __builtin_amdgcn_readlane(w.len, k);
            r.splits = sp;
            r.per = (st + 2 * sp - 1) / (2 * sp) * 64;
            r.part = parts + __builtin_amdgcn_readlane(ps, k) - __builtin_amdgcn_readlane(mparts, k) + r.tile * sp;
            r.join = joins + __builtin_amdgcn_readlane(js, k) - __builtin_amdgcn_readlane(mjoins, k) + r.tile;
        }
        before += __builtin_amdgcn_readlane(items, 63);
        parts += __builtin_amdgcn_readlane(ps, 63);
        joins += __builtin_amdgcn_readlane(js, 63);
    }
    // what follows from these is scalar work and real branches
    r.seq = uni(r.seq), r.tile = uni(r.tile), r.lo = uni(r.lo), r.n = uni(r.n), r.len = uni(r.len);
    r.split = uni(r.split), r.splits = uni(r.splits), r.per = uni(r.per), r.part = uni(r.part);
    r.join = uni(r.join), r.joins = joins;
    return r;
}

// How a launch of narrow column tiles is cut.  The column tiles of a key head
// stand in a row, each as long as its steps of 32 tokens (in units of `unit`)
// and AT_OVER units more for what beginning it costs, and the row is cut into `share`
// equal lengths (fewer where there are fewer units), one to a block, which does the
// pieces of tiles that it holds one after the other.  share 0: a tile is one
// unit, a block one tile.  64 sequences of up to 8192 tokens, 32 heads of 128 over 4: 40 us
// (AT_OVER 3 .. 6; 8: 41), with tiles cut into even parts of their own, a block to a part: 45.
constexpr uint32_t AT_OVER = 4;
struct Spot {
    int seq, tile, lo, n, len;
    int place;           // the tile's among all
    uint32_t at, units;  // units into the tile, and its length
};
struct Cut {
    SeqWork w;  // of the lane's sequence among the first 64
    uint32_t mine, upto, total, share, each, more;  // the first `more` blocks have each + 1 units
    int unit, tiles;
    TG_DEV uint32_t length(const SeqWork &s) const { return share ? ((uint32_t)s.steps + unit - 1) / unit + AT_OVER : 1; }
    TG_DEV Cut(const KvBatch &b, int G, int share_, int unit_, int lane) : w(seq_work<16>(b, G, lane)), share(share_), unit(unit_) {
        mine = (uint32_t)w.tiles * length(w), upto = wave_scan(mine);
        total = __builtin_amdgcn_readlane(upto, 63), tiles = wave_sum(w.tiles);
        if (!share) return;
        for (int j = lane + 64; j < (b.n_seqs + 63) / 64 * 64; j += 64) {
            const SeqWork s = seq_work<16>(b, G, j);
            total += wave_sum((uint32_t)s.tiles * length(s)), tiles += wave_sum(s.tiles);
        }
        total = uni(total), tiles = uni(tiles);
        share = min(share, max(total, 1u));
        each = total / share, more = total - each * share;
    }
    TG_DEV uint32_t begin(uint32_t x) const { return share ? x * each + min(x, more) : x; }
    TG_DEV uint32_t block_of(uint32_t u) const {  // share only
        const uint32_t w = more * (each + 1);
        return min(u < w ? u / (each + 1) : more + (u - w) / max(each, 1u), share - 1);
    }
    TG_DEV Spot at(const KvBatch &b, int G, uint32_t u, int lane) const {
        uint32_t before = 0;
        int tiles_before = 0;
        for (int j0 = 0; j0 < b.n_seqs; j0 += 64) {
            const SeqWork s = j0 == 0 ? w : seq_work<16>(b, G, j0 + lane);
            const uint32_t m = j0 == 0 ? mine : (uint32_t)s.tiles * length(s), up = j0 == 0 ? upto : wave_scan(m);
            const uint64_t found = __ballot(before + up > u);
            if (found) {
                const int k = __builtin_ctzll(found);
                Spot r;
                r.units = __builtin_amdgcn_readlane(length(s), k);
                const uint32_t local = u - before - __builtin_amdgcn_readlane(up, k) + __builtin_amdgcn_readlane(m, k);
                r.seq = j0 + k, r.tile = uni(local / r.units), r.at = local - r.tile * r.units;
                r.place = tiles_before + wave_sum(lane < k ? s.tiles : 0) + r.tile;
                r.lo = __builtin_amdgcn_readlane(s.lo, k), r.n = __builtin_amdgcn_readlane(s.n, k), r.len = __builtin_amdgcn_readlane(s.len, k);
                if ((uint32_t)r.tile >= (uint32_t)__builtin_amdgcn_readlane(s.tiles, k)) r.seq = -1;  // rows counted twice, sums that wrapped
                return r;
            }
            before += __builtin_amdgcn_readlane(up, 63), tiles_before += wave_sum(s.tiles);
        }
        return Spot{-1, 0, 0, 0, 0, 0, 0, 0};
    }
};

// How many tokens row i of the sequence sees.  One beyond the table is
// enough to make NaN of it, so a length that no table holds costs no more.
template <class T>
TG_DEV int tokens_seen(const KvBatch &b, const T &ct, int i) {
    return max(0, min(ct.len - ct.n + i + 1, b.table_cols * b.page_tokens + 1));
}

// Draft trees.  Behind the tokens that all rows of a sequence see, row i sees token base + j where bit j of its words
// is set.  tree_window: those of 32 tokens from token base + j on (j may be below 0: those before the tree are seen).
TG_DEV uint32_t tree_word(const uint32_t *bits, int words, int w) {
    const uint32_t v = bits[min(max(w, 0), words - 1)];
    return w < 0 ? ~0u : w < words ? v : 0u;
}
TG_DEV uint32_t tree_window(const uint32_t *bits, int words, int j) {
    const int w = j >> 5;
    return __builtin_amdgcn_alignbit(tree_word(bits, words, w + 1), tree_word(bits, words, w), j & 31);
}
// The last place that a row at place p visits.  Rows of a tree that are behind the table visit the first place there,
// as far as tokens_seen goes: unlike causal ones they need not see the token that is missing there.
template <bool TREE>
TG_DEV int last_place(const KvBatch &b, int p) {
    return TREE ? min(p, b.table_cols * b.page_tokens) : p;
}
// A token that a row of a tree does not see.  Its last place, if it does not see that, says that the row is no node of
// the tree or that its own token is behind the table, and makes NaN of it.
TG_DEV float tree_hides(float s, bool seen, int t, int last) {
    return t > last ? -INFINITY : seen ? s : t == last ? __builtin_nanf("") : -INFINITY;
}

// One step of 32 tokens of one key head as a lane holds it: tiles x = 0, 1
template <int D>
struct KvStep {
    static constexpr int NG = D / 32, SW = D / 64;  // scale words per lane and step
    uint32_t k[2][NG], v[2][2][NG / 2], s[SW];
    bool bad[2];  // the tile's page is none (D = 64: of the lane's own tile)
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

// What k_attn_join needs of one column tile that is split: its first column
// (row * G + head of the key head's), how many, its first partial result (of
// narrow tiles: the block that began it), and how many to join (0: none is split).
struct JoinTile {
    int col, cols, part, splits;
};
struct AttnOut {
    void *p;
    int64_t stride;
    JoinTile *join;  // [joins][key head]
    int joins;       // no more tiles than this are split
    float *part;     // [split][key head] of COLS x D sums, then COLS pairs (m, l); narrow tiles: two to a block, that of the
                     // tile it goes on with and that of the tile it leaves
};
template <int D, int COLS>
constexpr int AT_PART = COLS * (D + 2);  // floats of one split

// Few columns: split over the tokens.  A block goes through pieces of column
// tiles (as Cut says), its four waves every fourth step of 32 tokens; the
// packed bytes go from memory to registers one step ahead and are unpacked
// there (each is used by one wave, so LDS would only add a trip), the scales
// through a wave's corner of LDS because 16 lanes need the same ones.  The pieces
// of one column tile are joined by k_attn_join, or written out at once where
// one is all.  64 sequences of up to 8192 tokens, 32 heads of 128 over 4: 40 us, 3.8 TB/s; two of up to 200003,
// 64 heads over 4: 52 us, 4.4.  No unit is busy throughout: vector instructions, which unpack codes and weigh scores, take
// 40 to 46% of a SIMD's clocks, matrix ones 11 to 14%.  What is left is waiting: a step is a chain (scales to LDS and
// back, matrix, exponents, matrix), and two waves to a SIMD are few to cover it.
template <int D, bool BF, bool TREE>
__global__ __launch_bounds__(256, D == 64 ? 3 : D == 128 ? 2 : 1) void k_attn_split(KvBatch b, KvRows q, int G, float scale, int share,
                                                                      int unit, FastDiv tpp, AttnOut o) {
    constexpr int NG = D / 32, ND = D / 16, SW = D / 64;
    // Steps held: one at work, the others on their way.  Heads of 256 take all of a CU's registers for a block; in
    // half of them, 120 a lane spilled: 64 sequences of up to 4096 tokens, 32 heads over 4: 58 us, 113 so.
    constexpr int NB = D == 256 ? 2 : 3;
    __shared__ __align__(16) uint8_t sm[4 * 16 * D * 4 + 4 * 16 * 8];
    const int lane = threadIdx.x % 64, wave = uni(threadIdx.x / 64);
    const int c = lane % 16, h = lane / 16;
    const int hk = blockIdx.y;
    const Cut cut(b, G, share, unit, lane);
    // what is to be joined stands at the tile's place where places are few, at that of the block that begins it otherwise
    const bool by_tile = o.joins < share;
    JoinTile left{0, 0, 0, 0};  // the tile that the block begins and does not end
    uint32_t u = cut.begin(blockIdx.x);
    const uint32_t u1 = cut.share && blockIdx.x >= cut.share ? u : cut.begin(blockIdx.x + 1);
    while (u < u1) {
        const Spot ct = cut.at(b, G, u, lane);
        if (ct.seq < 0) break;
        const uint32_t over = cut.share ? AT_OVER : 0, end = min(ct.at + (u1 - u), ct.units);
        const uint32_t tile_u = u - ct.at;
        u = tile_u + end;
        if (end <= over && end < ct.units) break;  // the block ends before the tile's first step
        // this lane's column
        const int f = ct.tile * 16 + c, last = min(ct.n * G - 1, ct.tile * 16 + 15);
        const bool col = f < ct.n * G;
        const int row = ct.lo + (col ? f / G : 0), head = hk * G + (col ? f % G : 0);
        const int pos = col ? last_place<TREE>(b, ct.len - ct.n + f / G) : -1;
        // what every column sees ends at the first one's position, of trees before their first node
        const int seen = uni(tokens_seen(b, ct, last / G)), all = uni(ct.len - ct.n + (TREE ? -1 : (ct.tile * 16) / G));
        const bool first = ct.at <= over;
        const int t0 = first ? 0 : (int)(ct.at - over) * cut.unit * 32;
        const int t1 = end == ct.units ? seen : min(seen, (int)(end - over) * cut.unit * 32);
        const bool whole = first && t1 == seen;
        if (first && !whole) {
            const uint32_t last_u = tile_u + over + ((uint32_t)seen + 32 * cut.unit - 1) / (32 * cut.unit) - 1;
            left = JoinTile{ct.lo * G + ct.tile * 16, last - ct.tile * 16 + 1, (int)blockIdx.x, (int)(cut.block_of(last_u) - blockIdx.x) + 1};
        }
        if (first && by_tile && ct.place < o.joins && threadIdx.x == 0) o.join[(size_t)ct.place * b.n_kv + hk] = left;
        if (t0 >= t1) {
            // nothing to see here; a column tile that sees nothing at all is its first piece's to write
            if (first) {
                for (int i = threadIdx.x; i < 16 * D / 4; i += 256) {
                    const int ff = ct.tile * 16 + i / (D / 4);
                    if (ff >= ct.n * G) break;
                    store4<BF ? TG_T_BF16 : TG_T_F16>(o.p, (int64_t)(ct.lo + ff / G) * o.stride + (int64_t)(hk * G + ff % G) * D + i % (D / 4) * 4, f32x4{0, 0, 0, 0});
                }
            }
            continue;
        }

        uint32_t qw[NG][4];
        {
            const uint16_t *qp = static_cast<const uint16_t *>(q.p) + (int64_t)row * q.stride + (int64_t)head * D;
#pragma unroll
            for (int g = 0; g < NG; g++) load_words<4>(qp + 32 * g + 8 * h, qw[g]);
        }

        // a stretch of tokens c0 .. c1 - 1 whose pages the lanes hold, one each
        const int ntile = (int)tpp.d, span = 63 * 16 * ntile & ~31;
        const size_t head_bytes = (size_t)ntile * (18 * D), page_bytes = head_bytes * b.n_kv;
        const uint8_t *base = b.pages + hk * head_bytes;
        int c0 = t0, c1 = 0, page0 = 0, mine = 0, st = 0, s1 = 0;
        KvStep<D> k[NB];
        auto load = [&](KvStep<D> &k, int step) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                int t = step * 2 + x;
                t = (t * 16 < c1 ? t : c0 / 16) - page0 * ntile;  // behind the end: any tile, its tokens are masked
                const int pi = (int)fdiv((uint32_t)t, tpp), pg = __builtin_amdgcn_readlane(mine, pi);
                const uint8_t *p = base + (size_t)max(pg, 0) * page_bytes + (size_t)(t - pi * ntile) * (18 * D);
                load_words<NG>(p + lane * (NG * 4), k.k[x]);
                load_words<NG>(p + 8 * D + lane * (NG * 4), &k.v[x][0][0]);
                // lane's share of the scales: the step's 4 D bytes over 64 lanes; a page that is none has NaN ones
                const uint32_t *sp = reinterpret_cast<const uint32_t *>(p + 16 * D);
                if (SW == 1) {
                    const uint32_t v = sp[lane % 32];
                    if (lane / 32 == x) k.s[0] = v, k.bad[0] = pg < 0;
                } else {
                    k.bad[x] = pg < 0;
#pragma unroll
                    for (int i = 0; i < SW / 2; i++) k.s[x * (SW / 2) + i] = sp[lane * (SW / 2) + i];
                }
            }
            // loads leave in the order of their steps, so that the wait for one step leaves those behind it under way
            asm volatile("" ::: "memory");
        };
        auto begin = [&]() {
            c1 = min(t1, c0 + span);
            page0 = uni(c0 / 16 / ntile);
            mine = (page0 + lane) * 16 * ntile < c1 ? page_of(b, ct.seq, (page0 + lane) * 16 * ntile) : 0;
            s1 = (c1 + 31) / 32;
            st = c0 / 32 + wave;
#pragma unroll
            for (int i = 0; i < NB - 1; i++) load(k[i], st + 4 * i);
        };
        begin();

        // queries: operand slots 8 h .. 8 h + 7 of each block, and the start of the sums
        f16x8 qf[NG];
        f32x4 start[NG];
        float cs;
        {
            uint32_t mag = 0;  // magnitudes order as the integers they are stored as
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (!col) qw[g][e] = 0;
                    mag = max(mag, max(qw[g][e] & 0x7FFFu, (qw[g][e] >> 16) & 0x7FFFu));
                }
            mag = max(mag, (uint32_t)__shfl_xor((int)mag, 16));
            mag = max(mag, (uint32_t)__shfl_xor((int)mag, 32));
            const float top = BF ? bf2f((uint16_t)mag) : h2f((uint16_t)mag);
            int e2 = 0;
            (void)frexpf(top, &e2);  // top = m 2^e2, m in [0.5, 1)
            const int a = top > 0.0f && top < INFINITY ? 11 - e2 : 0;
            cs = score_factor(scale, 18 - a);
#pragma unroll
            for (int g = 0; g < NG; g++) {
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint16_t u = (uint16_t)(qw[g][e / 2] >> (16 * (e % 2)));
                    const _Float16 v = (_Float16)ldexpf(BF ? bf2f(u) : h2f(u), a + ((e / 2) % 2 ? 0 : 4));
                    qf[g][e] = v;
                    sum += (e / 2) % 2 ? (float)v * 16.0f : (float)v;
                }
                sum = col_sum(sum);
                const float s0 = sum * (-8.0f / 4194304.0f);
                start[g] = f32x4{s0, s0, s0, s0};
            }
        }

        uint32_t *sl = reinterpret_cast<uint32_t *>(sm) + wave * (16 * D);  // this wave's corner
        // word w of a tile's 2 D bytes of scales that this lane's i-th word is, and its tile
        auto word_of = [&](int i) { return SW == 1 ? lane % 32 : lane * (SW / 2) + i % (SW / 2); };
        auto tile_of = [&](int i) { return SW == 1 ? lane / 32 : i / (SW / 2); };
        const uint32_t vmask = word_of(0) >= D / 4 ? 0x7FFF7FFFu : 0u;  // this lane's words are value scales
        const f16x8 off_even = as_h8(0x80208020u, 0x80208020u, 0x80208020u, 0x80208020u);  // -8 as the subnormals the
        const f16x8 off_odd = as_h8(0x82008200u, 0x82008200u, 0x82008200u, 0x82008200u);   // two kinds of codes are
        f32x4 acc[ND] = {};
        float m = AT_NONE, l = 0.0f;
        float A = 0.0f;           // the same in all lanes of a wave
        uint32_t below = 0u;      // pairs of halves: the largest scale that A allows for
        bool rough = false;       // as coarse(m) says
        auto work = [&](KvStep<D> &k, int step) {
            const bool edge = step * 32 + 31 > all;  // some column does not see all of it
            // scales to LDS as the tiles hold them; what no column sees is zero
            uint32_t big = below, vs[SW];  // value scales
#pragma unroll
            for (int i = 0; i < SW; i++) {
                const int w = word_of(i), x = tile_of(i);
                uint32_t v = k.bad[SW == 1 ? 0 : x] ? 0x7E007E00u : k.s[i];  // a page that is none has NaN scales
                if (edge) {
                    const int t = step * 32 + 16 * x;
                    if (w < D / 4) {
                        if (t + w / (NG / 2) >= seen) v = 0;
                    } else {
                        const int tp = t + (w - D / 4) / NG * 2;
                        if (tp + 1 >= seen) v &= 0xFFFFu;
                        if (tp >= seen) v = 0;
                    }
                }
                typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
                vs[i] = v & vmask;
                big = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, big), __builtin_bit_cast(u16x2, vs[i])));
                sl[x * (D / 2) + w] = v;
            }
            bool odd = false;
            if (__ballot(big != below)) {
                // a scale at or above the bound: a new one, or a block that is not finite, which is left out by itself
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < SW; i++) {
                    const uint32_t lo = vs[i] & 0xFFFFu, hi = vs[i] >> 16;
                    odd = odd || max(lo, hi) >= 0x7C00u;
                    top = max(top, max(lo < 0x7C00u ? lo : 0u, hi < 0x7C00u ? hi : 0u));
                }
                odd = __ballot(odd) != 0;
#pragma unroll
                for (int i = 1; i < 64; i *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, i));
                if (top > (below & 0xFFFFu)) {
                    const int e = min(16, max((int)(top >> 10), 1) - 15 + 2);  // top is below 2^(e - 1): one bit of room; e is -12 or more
                    below = e > 15 ? 0x7BFF7BFFu : (uint32_t)(((e + 15) << 10) - 1) * 0x10001u;
                    const float r = ldexpf(1.0f, AT_TOP - e - (int)A);
                    A = (float)(AT_TOP - e);
                    l *= r;
#pragma unroll
                    for (int j = 0; j < ND; j++) acc[j] *= r;
                }
            }
            wave_lds_sync();
            f32x4 r[2][NG];
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    const uint32_t w = k.k[x][g] << 2, w2 = k.k[x][g] >> 6;
                    const f16x8 kf = as_h8(w & AT_EVEN, w & AT_ODD, w2 & AT_EVEN, w2 & AT_ODD);
                    r[x][g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[g], start[g], 0, 0, 0);
                }
            if (D <= 128) __builtin_amdgcn_sched_barrier(0);  // all of them under way before the first is waited for
            float s[2][4];
#pragma unroll
            for (int x = 0; x < 2; x++) {
                uint32_t kd[2 * NG];  // halves [token i][block g]
                load_words<2 * NG>(sl + x * (D / 2) + h * (2 * NG), kd);
#pragma unroll
                for (int g = 0; g < NG; g++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        s[x][i] = __builtin_fmaf((float)as_h2(kd[(i * NG + g) / 2])[g % 2], r[x][g][i], g == 0 ? 0.0f : s[x][i]);
            }
            if (odd) {
                // NaN for the tokens of value blocks that are not finite; those blocks become 0
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    uint32_t vd[2 * NG];
                    load_words<2 * NG>(sl + x * (D / 2) + D / 4 + h * (2 * NG), vd);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        bool n = false;
#pragma unroll
                        for (int g = 0; g < NG; g++) n |= ((vd[(i / 2) * NG + g] >> (16 * (i % 2))) & 0x7C00u) == 0x7C00u;
                        if (n) s[x][i] = __builtin_nanf("");
                    }
                }
                wave_lds_sync();
#pragma unroll
                for (int i = 0; i < SW; i++) {
                    if (vmask) {
                        uint32_t *at = sl + tile_of(i) * (D / 2) + word_of(i), v = *at;
                        if ((v & 0x7C00u) == 0x7C00u) v &= 0xFFFF0000u;
                        if ((v & 0x7C000000u) == 0x7C000000u) v &= 0xFFFFu;
                        *at = v;
                    }
                }
                wave_lds_sync();
            }
            if (edge) {
                if (TREE) {
                    const uint32_t w = tree_window(b.bits + (size_t)row * b.words, b.words, step * 32 - all - 1) >> 4 * h;
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            s[x][i] = tree_hides(s[x][i], w >> (16 * x + i) & 1, step * 32 + 16 * x + 4 * h + i, pos);
                } else {
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (step * 32 + 16 * x + 4 * h + i > pos) s[x][i] = -INFINITY;
                }
            }
            // cs > 0, so the largest s is the largest score
            float top = s[0][0];
#pragma unroll
            for (int i = 1; i < 8; i++) top = __builtin_elementwise_maximum(top, s[i / 4][i % 4]);  // a NaN stays one
            if (__ballot(top * cs > m + AT_ROOM)) {
                top = col_max(top);
                const float m2 = fmaxf(m, top * cs), r = __builtin_amdgcn_exp2f(m - m2);
                l *= r;
#pragma unroll
                for (int j = 0; j < ND; j++) acc[j] *= r;
                m = m2;
                rough = coarse(m);
            }
            float by = cs, off = A - m;
            if (rough) {
#pragma unroll
                for (int i = 0; i < 8; i++) s[i / 4][i % 4] = s[i / 4][i % 4] * cs - m;
                by = 1.0f, off = A;
            }
            float p[2][4];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                p[i / 4][i % 4] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 4][i % 4], by, off));
                l += p[i / 4][i % 4];
            }
            // value scales: words [token pair][block] of each tile
            uint32_t vd[2][2 * NG];
#pragma unroll
            for (int x = 0; x < 2; x++) load_words<2 * NG>(sl + x * (D / 2) + D / 4 + h * (2 * NG), vd[x]);
#pragma unroll
            for (int g = 0; g < NG; g++) {
                uint32_t w[4];
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const f16x2 d = as_h2(vd[y / 2][(y % 2) * NG + g]);
                    const f16x2 v = {(_Float16)__builtin_fmaf(p[y / 2][2 * (y % 2)], (float)d[0], 0.0f),
                                     (_Float16)__builtin_fmaf(p[y / 2][2 * (y % 2) + 1], (float)d[1], 0.0f)};
                    w[y] = as_u(v);
                }
                const f16x8 pf = as_h8(w[0], w[1], w[2], w[3]);
                uint32_t r[4];  // the block's two column tiles are nibbles 2 (g % 2) and 2 (g % 2) + 1
#pragma unroll
                for (int y = 0; y < 4; y++) r[y] = g % 2 ? k.v[y / 2][y % 2][g / 2] >> 6 : k.v[y / 2][y % 2][g / 2] << 2;
                const f16x8 even = as_h8(r[0] & AT_EVEN, r[1] & AT_EVEN, r[2] & AT_EVEN, r[3] & AT_EVEN);
                const f16x8 odd8 = as_h8(r[0] & AT_ODD, r[1] & AT_ODD, r[2] & AT_ODD, r[3] & AT_ODD);
                acc[2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, pf, acc[2 * g], 0, 0, 0);
                acc[2 * g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd8, pf, acc[2 * g + 1], 0, 0, 0);
                acc[2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(off_even, pf, acc[2 * g], 0, 0, 0);
                acc[2 * g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(off_odd, pf, acc[2 * g + 1], 0, 0, 0);
            }
            wave_lds_sync();
        };
        while (c0 < t1) {
            // loads ahead of the last step too (of a tile that is there): were they conditional, the wait for a
            // step's bytes would have to take in those of the steps behind it
            while (st < s1) {
#pragma unroll
                for (int i = 0; i < NB; i++) {
                    load(k[(i + NB - 1) % NB], st + 4 * (NB - 1));
                    work(k[i], st);
                    st += 4;
                    if (st >= s1) break;
                }
            }
            c0 += span;
            if (c0 < t1) begin();
        }
        // weights were exp2(score - m + A), and m may be too large to take A up
        const float unit = ldexpf(1.0f, -(int)A);
        l = col_sum(l) * unit;

        // the waves' shares joined in order: O[wave][column][D], m and l [wave][column]
        __syncthreads();
        float *so = reinterpret_cast<float *>(sm) + wave * 16 * D, *sml = reinterpret_cast<float *>(sm + 4 * 16 * D * 4);
#pragma unroll
        for (int j = 0; j < ND; j++) *reinterpret_cast<f32x4 *>(so + c * D + 16 * j + 4 * h) = acc[j] * (unit * (j % 2 ? 262144.0f : 4194304.0f));
        if (h == 0) sml[(wave * 16 + c) * 2] = m, sml[(wave * 16 + c) * 2 + 1] = l;
        __syncthreads();
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
                float *pp = o.part + ((size_t)(2 * blockIdx.x + first) * b.n_kv + hk) * AT_PART<D, 16>;
                *reinterpret_cast<f32x4 *>(pp + cc * D + d) = v;
                if (d == 0) pp[16 * D + 2 * cc] = mm, pp[16 * D + 2 * cc + 1] = ll;
            }
        }
        if (u < u1) __syncthreads();  // before the next piece's scales go where the sums were
    }
    if (share && threadIdx.x == 0) {
        if (!by_tile) o.join[(size_t)blockIdx.x * b.n_kv + hk] = left;
        else for (int i = cut.tiles + blockIdx.x; i < o.joins; i += gridDim.x) o.join[(size_t)i * b.n_kv + hk] = JoinTile{0, 0, 0, 0};
    }
}

// Many columns: a block of 8 waves holds 256 columns of one key head (heads of 256: 128), 32 to a
// wave, and goes through the tokens in steps of 64, which it dequantises to
// fp16 once for all of them: half the waves take a tile's keys, half its
// values, ahead of their use (the packed bytes a phase before that), and leave
// them in LDS as whole operands of the matrix instructions, 16 bytes to a
// lane, which every wave then reads without conflict.
//
// The two waves of a SIMD (w and w + 4) take turns: a step is a matrix phase
// (the output of step t - 1, the scores of step t) and a vector phase (the
// weights of step t, dequantising a later one) with a barrier behind each,
// and the second four waves run one phase behind, so that one wave's vector work
// hides under the other's matrix work.  In intervals between barriers: waves
// 0..3 have M(t) in 2 t and V(t) in 2 t + 1, where they write step t + 1;
// waves 4..7 have M(t) in 2 t + 1 and V(t) in 2 t + 2, where they write step t +
// 2.  K(t) is read in 2 t and 2 t + 1, V(t) in 2 t + 2 and 2 t + 3: two places for
// keys and three for values keep every write behind the last reading.
//
// Keys and values rounded to fp16 (2^-11 of each at the most) buy scores and
// weights without a scale to apply.  For bf16 rows that stays under the rounding
// of the result, 2^-9; fp16 rows, whose results show it (2.1 times the error of one
// rounding), take the roundings' remainders, which fp16 holds exactly, as a second
// operand of every product.  The weights' sum is a matrix product with
// ones.  Scores and bounds as in k_attn_split, A = 9 throughout.
//
// Bound: at D = 128, bf16, a phase of a wave is 66 matrix instructions (1056 clocks)
// behind 32 KB of operands from LDS (1024 for the four waves that read), about 1750
// together, against 32 exponentials and what surrounds them (1200) and the
// dequantising of a sixteenth of the step (900); the two overlap in part (the longer of two such
// streams alone takes 290 us, both at once 406).  Three prompts of 4096, 4046 and
// 2482 tokens, 32 heads over 4: 390 us, 0.83 PFLOP/s; all waves in step, one
// barrier to a step: 422; heads one after the other instead of side by side: 455, since
// the longest blocks of the last head start late.  fp16, D = 64, 500 tokens each of two prompts of
// 16001, 32 heads over 8: 250 us, without the remainders 186, with those of the keys and of the weights
// (more vector work, less of LDS) 284.
//
// Heads of 256: 128 columns to a block, and both waves of a SIMD hold the same 32, each with half of the output's dims; the
// scores and weights they form twice, which keeps them from having to meet.  A prompt of 4096, bf16, 32 heads
// over 8: 445 us, 0.62 PFLOP/s (by few columns 1133).
template <int D>
constexpr int AT_COLS = D == 256 ? 128 : 256;

template <int D, bool BF, bool TREE>
__global__ __launch_bounds__(512, 2) void k_attn_tile(KvBatch b, KvRows q, int G, float scale, int share, FastDiv tpp, AttnOut o) {
    constexpr int NG = D / 32, ND = D / 16, NC = 2, COLS = AT_COLS<D>, BUF = 64 * D * 2;  // keys or values of a step
    constexpr int DW = COLS * D / 256, NJ = DW / 16;  // dims of the output that are a wave's
    constexpr int REST = BF ? 0 : 5 * BUF;  // where the roundings' remainders are
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x % 64, wave = uni(threadIdx.x / 64), c16 = lane % 16, h = lane / 16;
    // all heads of a tile side by side, and the late tiles of a sequence, which see the most tokens, first
    const int x = blockIdx.x / (unsigned)b.n_kv, hk = blockIdx.x - x * b.n_kv;
    const ColTile ct = col_tile<COLS>(b, G, share, gridDim.x / (unsigned)b.n_kv - 1 - x, lane);
    if (x >= ct.joins && x < o.joins && threadIdx.x == 0)
        o.join[(size_t)x * b.n_kv + hk] = JoinTile{0, 0, 0, 0};
    if (ct.seq < 0) return;
    const int ncol = ct.n * G, col0 = ct.tile * COLS, last = min(ncol - 1, col0 + COLS - 1);
    const int seen = uni(tokens_seen(b, ct, last / G));
    const int t0 = ct.split * ct.per, t1 = min(seen, t0 + ct.per);
    if (ct.splits > 1 && ct.split == 0 && threadIdx.x == 0)
        o.join[(size_t)ct.join * b.n_kv + hk] = JoinTile{ct.lo * G + col0, last - col0 + 1, ct.part, seen <= ct.per ? 0 : (seen + ct.per - 1) / ct.per};
    if (t0 >= t1 && ct.split > 0) return;

    // this lane's columns, one of each column tile of the wave
    const int f0 = col0 + wave % (COLS / (16 * NC)) * 16 * NC, dim0 = wave / (COLS / (16 * NC)) * DW;
    int pos[NC];
    uint32_t qw[NC][NG][4];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int f = f0 + 16 * c + c16;
        const bool col = f < ncol;
        pos[c] = col ? last_place<TREE>(b, ct.len - ct.n + f / G) : -1;
        const uint16_t *qp = static_cast<const uint16_t *>(q.p) + (int64_t)(ct.lo + (col ? f / G : 0)) * q.stride +
                             (int64_t)(hk * G + (col ? f % G : 0)) * D;
#pragma unroll
        for (int g = 0; g < NG; g++) load_words<4>(qp + 32 * g + 8 * h, qw[c][g]);
    }
    // position of the wave's first column; of trees the one before their first node
    const int first = uni(ct.len - ct.n + (TREE ? -1 : min(f0, last) / G));

    // this wave's share of a step: the keys (even) or values (odd) of its tile wave / 2
    const int ntile = (int)tpp.d, span = min(ct.per, 63 * 16 * ntile & ~63);
    const size_t head_bytes = (size_t)ntile * (18 * D), page_bytes = head_bytes * b.n_kv;
    const uint8_t *base = b.pages + hk * head_bytes;
    const bool is_v = wave % 2;
    const int xt = wave / 2;
    int mine = 0, page0 = 0, from = t0 - span;
    // codes; scales.  Values: words [token pair][block].  Keys: those of token c16 (and what follows them), then
    // the value scales of it and its neighbour.  The same loads for either, so that no branch waits for one.
    uint32_t raw[NG], sc[2 * NG];
    const uint32_t code_at = (is_v ? 8 * D : 0) + lane * (NG * 4), scale_at = is_v ? 17 * D + h * (8 * NG) : 16 * D + c16 * (2 * NG);
    const uint32_t more_at = is_v ? scale_at + 4 * NG : 17 * D + c16 / 2 * (4 * NG);
    bool bad = false;
    auto pages = [&](int step) {  // those of the stretch that holds it
        const int t = t0 + 64 * step;
        if (t >= from + span && t < t1) {
            from = t;
            page0 = uni(from / 16 / ntile);
            mine = (page0 + lane) * 16 * ntile < t1 ? page_of(b, ct.seq, (page0 + lane) * 16 * ntile) : 0;
        }
    };
    auto fetch = [&](int step) {  // tile xt of it, or any behind the end, whose scales become 0
        int t = t0 + 64 * step + 16 * xt;
        t = t < t1 ? t : from;
        const int tt = t / 16 - page0 * ntile, pi = (int)fdiv((uint32_t)tt, tpp), pg = __builtin_amdgcn_readlane(mine, pi);
        bad = pg < 0;
        const uint8_t *p = base + (size_t)max(pg, 0) * page_bytes + (size_t)(tt - pi * ntile) * (18 * D);
        load_words<NG>(p + code_at, raw);
        load_words<NG>(p + scale_at, sc);
        load_words<NG>(p + more_at, sc + NG);
    };
    // codes n of the four-code halfwords of w, less 8, times d, and the rounding's remainder; one of the two
    // constants in a scalar register and one in a vector register make a single instruction of the mask and what
    // makes a number of it
    uint32_t lo = 0x000F000Fu, hi = 0x00F000F0u, k1024 = 0x64006400u, k64 = 0x54005400u;
    asm("" : "+s"(lo), "+s"(hi), "+v"(k1024), "+v"(k64));
    auto unpack = [&](uint32_t w, int n, f16x2 d, uint32_t &rest) {
        const uint32_t v = n < 2 ? w : w >> 8;
        const f16x2 t = n % 2 == 0 ? as_h2((v & lo) | k1024) - f16x2{(_Float16)1032.0f, (_Float16)1032.0f}
                                   : as_h2((v & hi) | k64) - f16x2{(_Float16)72.0f, (_Float16)72.0f};
        const f16x2 v16 = t * d;
        rest = as_u(__builtin_elementwise_fma(t, d, -v16));
        return as_u(v16);
    };
    auto spread = [&](int step) __attribute__((always_inline)) {  // what fetch(step) brought, to LDS
        const int t = t0 + 64 * step + 16 * xt;
        uint8_t *buf = lds + (is_v ? 2 + step % 3 : step % 2) * BUF + lane * 16;
        // an infinity or NaN among the value scales makes the sum of products with 0 a NaN; so does, for the
        // remainders, a scale whose values fp16 does not hold
        f16x2 odd = {0, 0}, over = {0, 0};
#pragma unroll
        for (int i = 0; i < NG; i++) {
            if (is_v) odd = __builtin_elementwise_fma(as_h2(sc[i]), f16x2{0, 0}, odd);
            odd = __builtin_elementwise_fma(as_h2(sc[NG + i]), f16x2{0, 0}, odd);
            if (REST && (is_v || i < NG / 2)) over = __builtin_elementwise_fma(as_h2(sc[i]) * (_Float16)8.0f, f16x2{0, 0}, over);
            if (REST && is_v) over = __builtin_elementwise_fma(as_h2(sc[NG + i]) * (_Float16)8.0f, f16x2{0, 0}, over);
        }
        const bool plain = !bad && t + 16 <= seen && !__ballot(as_u(odd) & 0x7C007C00u);
        const bool rests = REST && !__ballot(as_u(over) & 0x7C007C00u);
        auto keys = [&](auto with) __attribute__((always_inline)) {
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const _Float16 d = as_h2(sc[g / 2])[g % 2];
                u32x4 v, r;
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    uint32_t lo2 = 0;
                    v[n] = unpack(raw[g], n, f16x2{d, d}, lo2);
                    r[n] = decltype(with)::value ? lo2 : 0;
                }
                *reinterpret_cast<u32x4 *>(buf + (xt * NG + g) * 1024) = v;
                if (REST) *reinterpret_cast<u32x4 *>(buf + REST + (xt * NG + g) * 1024) = r;
            }
        };
        auto values = [&](auto with) __attribute__((always_inline)) {
#pragma unroll
            for (int bq = 0; bq < NG / 2; bq++)
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    uint32_t r0, r1;
                    const u32x2 v = {unpack(raw[bq], n, as_h2(sc[2 * bq + n / 2]), r0), unpack(raw[NG / 2 + bq], n, as_h2(sc[NG + 2 * bq + n / 2]), r1)};
                    uint8_t *p = buf + (xt / 2 * ND + 4 * bq + n) * 1024 + xt % 2 * 8;
                    *reinterpret_cast<u32x2 *>(p) = v;
                    if (REST) *reinterpret_cast<u32x2 *>(p + REST) = decltype(with)::value ? u32x2{r0, r1} : u32x2{0, 0};
                }
        };
        if (!is_v) {
            if (!plain) {
                uint32_t inf = 0;
#pragma unroll
                for (int g = 0; g < NG; g++) inf |= ((sc[NG + g] >> (16 * (c16 % 2))) & 0x7C00u) == 0x7C00u;
                const bool poison = bad || inf, none = t + c16 >= seen;
#pragma unroll
                for (int g = 0; g < NG / 2; g++) sc[g] = none ? 0u : poison ? 0x7E007E00u : sc[g];
            }
            if (rests) keys(std::true_type{});
            else keys(std::false_type{});
        } else {
            if (!plain) {
#pragma unroll
                for (int i = 0; i < 2 * NG; i++) {
                    const int tp = t + 4 * h + 2 * (i / NG);
                    uint32_t d = bad ? 0u : sc[i];
                    if ((d & 0x7C00u) == 0x7C00u || tp >= seen) d &= 0xFFFF0000u;
                    if ((d & 0x7C000000u) == 0x7C000000u || tp + 1 >= seen) d &= 0xFFFFu;
                    sc[i] = d;
                }
            }
            if (rests) values(std::true_type{});
            else values(std::false_type{});
        }
    };

    const int steps = (t1 - t0 + 63) / 64;
    if (steps > 0) {
        pages(0);
        fetch(0);  // before the conversions that follow
    }
    f16x8 qf[NC][NG];
    float cs[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        uint32_t mag = 0;
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (pos[c] < 0) qw[c][g][e] = 0;
                mag = max(mag, max(qw[c][g][e] & 0x7FFFu, (qw[c][g][e] >> 16) & 0x7FFFu));
            }
        mag = max(mag, (uint32_t)__shfl_xor((int)mag, 16));
        mag = max(mag, (uint32_t)__shfl_xor((int)mag, 32));
        const float top = BF ? bf2f((uint16_t)mag) : h2f((uint16_t)mag);
        int e2 = 0;
        (void)frexpf(top, &e2);
        const int a = top > 0.0f && top < INFINITY ? 14 - e2 : 0;  // the row's largest value to 2^13 .. 2^14
        cs[c] = score_factor(scale, -a);
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint16_t u = (uint16_t)(qw[c][g][e / 2] >> (16 * (e % 2)));
                qf[c][g][e] = (_Float16)ldexpf(BF ? bf2f(u) : h2f(u), a);
            }
    }

    f32x4 acc[NC][NJ] = {}, sum[NC] = {};
    float m[NC];
    bool rough[NC];  // as coarse(m) says
#pragma unroll
    for (int c = 0; c < NC; c++) m[c] = AT_NONE, rough[c] = false;
    const f16x8 ones = as_h8(0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u);
    f32x4 s[NC][4];
    f16x8 pf[NC][2];
    const bool late = wave >= 4;
    auto matrix = [&](int step, auto with_pv, auto with_qk) __attribute__((always_inline)) {
        constexpr bool PV = decltype(with_pv)::value, QK = decltype(with_qk)::value;
        const int next = step + (late ? 2 : 1);
        if (QK) pages(next);
        if (QK) fetch(next);
        if (PV) {
            const uint8_t *vb = lds + (2 + (step - 1) % 3) * BUF + dim0 * 64 + lane * 16;
#pragma unroll
            for (int p = 0; p < 2; p++) {
#pragma unroll
                for (int c = 0; c < NC; c++) sum[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pf[c][p], sum[c], 0, 0, 0);
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    const f16x8 vf = *reinterpret_cast<const f16x8 *>(vb + (p * ND + j) * 1024);
#pragma unroll
                    for (int c = 0; c < NC; c++) acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[c][p], acc[c][j], 0, 0, 0);
                    if (REST) {
                        const f16x8 vr = *reinterpret_cast<const f16x8 *>(vb + REST + (p * ND + j) * 1024);
#pragma unroll
                        for (int c = 0; c < NC; c++) acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vr, pf[c][p], acc[c][j], 0, 0, 0);
                    }
                }
            }
        }
        if (QK) {
            const uint8_t *kb = lds + step % 2 * BUF + lane * 16;
#pragma unroll
            for (int x = 0; x < 4; x++)
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    const f16x8 kf = *reinterpret_cast<const f16x8 *>(kb + (x * NG + g) * 1024);
#pragma unroll
                    for (int c = 0; c < NC; c++)
                        s[c][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[c][g], g == 0 ? f32x4{0, 0, 0, 0} : s[c][x], 0, 0, 0);
                    if (REST) {
                        const f16x8 kr = *reinterpret_cast<const f16x8 *>(kb + REST + (x * NG + g) * 1024);
#pragma unroll
                        for (int c = 0; c < NC; c++) s[c][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kr, qf[c][g], s[c][x], 0, 0, 0);
                    }
                }
        }
    };
    auto vector = [&](int step) __attribute__((always_inline)) {
        const int t = t0 + 64 * step;
        if (TREE && t + 63 > first) {
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const int f = f0 + 16 * c + c16;
                const uint32_t *bits = b.bits + (size_t)(ct.lo + (f < ncol ? f / G : 0)) * b.words;
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const uint32_t w = tree_window(bits, b.words, t + 32 * y - first - 1) >> 4 * h;
#pragma unroll
                    for (int x = 2 * y; x < 2 * y + 2; x++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            s[c][x][i] = tree_hides(s[c][x][i], w >> (16 * (x % 2) + i) & 1, t + 16 * x + 4 * h + i, pos[c]);
                }
            }
        } else if (!TREE && t + 63 > first) {
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int x = 0; x < 4; x++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (t + 16 * x + 4 * h + i > pos[c]) s[c][x][i] = -INFINITY;
        }
#pragma unroll
        for (int c = 0; c < NC; c++) {
            float top = s[c][0][0];
#pragma unroll
            for (int i = 1; i < 16; i++) top = __builtin_elementwise_maximum(top, s[c][i / 4][i % 4]);  // a NaN stays one
            if (__ballot(top * cs[c] > m[c] + AT_ROOM)) {
                const float m2 = fmaxf(m[c], col_max(top) * cs[c]), r = __builtin_amdgcn_exp2f(m[c] - m2);
                sum[c] *= r;
#pragma unroll
                for (int j = 0; j < NJ; j++) acc[c][j] *= r;
                m[c] = m2;
                rough[c] = coarse(m2);
            }
            float by = cs[c], off = (float)AT_TOP - m[c];
            if (rough[c]) {
#pragma unroll
                for (int i = 0; i < 16; i++) s[c][i / 4][i % 4] = s[c][i / 4][i % 4] * cs[c] - m[c];
                by = 1.0f, off = (float)AT_TOP;
            }
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; i++)
                w[i] = pack_h2(__builtin_amdgcn_exp2f(__builtin_fmaf(s[c][i / 2][i % 2 * 2], by, off)),
                               __builtin_amdgcn_exp2f(__builtin_fmaf(s[c][i / 2][i % 2 * 2 + 1], by, off)));
            pf[c][0] = as_h8(w[0], w[1], w[2], w[3]);
            pf[c][1] = as_h8(w[4], w[5], w[6], w[7]);
        }
        const int ahead = step + (late ? 2 : 1);
        if (ahead < steps) spread(ahead);
    };
    if (steps > 0) {
        using std::true_type, std::false_type;
        spread(0);
        lds_barrier();
        if (late) {
            if (steps > 1) {
                pages(1);
                fetch(1);
                spread(1);
            }
            lds_barrier();
        }
        // a wave without columns, of which trees leave many, does its share of the codes alone: 16 trees of 16 nodes,
        // half a tile each, after 8000 tokens 71 us, 84 with all of the products
        if (TREE && f0 >= ncol) {
            for (int i = 0; i < steps; i++) {
                const int next = i + (late ? 2 : 1);
                pages(next);
                fetch(next);
                lds_barrier();
                if (next < steps) spread(next);
                lds_barrier();
            }
        } else {
            matrix(0, false_type{}, true_type{});
            lds_barrier();
            vector(0);
            lds_barrier();
            for (int i = 1; i < steps; i++) {
                matrix(i, true_type{}, true_type{});
                lds_barrier();
                vector(i);
                lds_barrier();
            }
            matrix(steps, true_type{}, false_type{});
        }
        if (!late) lds_barrier();
        lds_barrier();
    }
    const bool whole = seen <= ct.per;
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int f = f0 + 16 * c + c16;
        if (whole) {
            // through LDS, 16 columns of the wave at a time, so that a head leaves as whole lines
            uint16_t *so = reinterpret_cast<uint16_t *>(lds) + wave * 16 * (DW + 8);
            const float inv = sum[c][0] == 0.0f ? 0.0f : 1.0f / sum[c][0];
#pragma unroll
            for (int j = 0; j < NJ; j++) store4<BF ? TG_T_BF16 : TG_T_F16>(so, c16 * (DW + 8) + 16 * j + 4 * h, acc[c][j] * inv);
            wave_lds_sync();
            constexpr int L = DW / 8;  // lanes of one head
#pragma unroll
            for (int i = 0; i < 16 * L / 64; i++) {
                const int cc = i * (64 / L) + lane / L, ff = f0 + 16 * c + cc;
                const u32x4 v = *reinterpret_cast<const u32x4 *>(so + cc * (DW + 8) + 8 * (lane % L));
                if (ff < ncol)
                    *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(o.p) + (int64_t)(ct.lo + ff / G) * o.stride + (int64_t)(hk * G + ff % G) * D + dim0 + 8 * (lane % L)) = v;
            }
            wave_lds_sync();
        } else if (f < ncol) {
            float *pp = o.part + ((size_t)(ct.part + ct.split) * b.n_kv + hk) * AT_PART<D, COLS>;
            const int cc = f - col0;
#pragma unroll
            for (int j = 0; j < NJ; j++) *reinterpret_cast<f32x4 *>(pp + (size_t)cc * D + dim0 + 16 * j + 4 * h) = acc[c][j];
            if (h == 0 && dim0 == 0) pp[COLS * D + 2 * cc] = m[c], pp[COLS * D + 2 * cc + 1] = sum[c][0];
        }
    }
}

// The splits of one column, joined in order: TC threads per column, D / 4
// lanes side by side for one split, each group of them every GR-th split.  A
// block per column where few tiles have many splits, four columns to a block otherwise.
template <int D, bool BF, int TC>
__global__ __launch_bounds__(256) void k_attn_join(KvBatch b, int G, AttnOut o) {
    constexpr int L = D / 4, GR = TC / L > 0 ? TC / L : 1, NC = 256 / TC, W = TC / 64;
    static_assert(TC >= L, "");
    __shared__ float sm_m[4], sm_l[4], sw[256];
    __shared__ __align__(16) f32x4 so[256];
    const int hk = blockIdx.y, tid = threadIdx.x % TC, ci = threadIdx.x / TC, cc = blockIdx.z * NC + ci;
    const JoinTile jt = o.join[(size_t)blockIdx.x * b.n_kv + hk];
    if (!jt.splits || (int)blockIdx.z * NC >= jt.cols) return;
    const size_t step = (size_t)b.n_kv * AT_PART<D, 16>;
    const float *part = o.part + ((size_t)(2 * jt.part) * b.n_kv + hk) * AT_PART<D, 16>;
    auto piece = [&](int i) { return i == 0 ? step : 2 * i * step; };  // from there
    // all of a thread's sums (those of the first 8 turns) and its (m, l) are asked for before the first is
    // waited for; columns behind the last hold zeros
    const float *mine = part + cc * D + 4 * (tid % L), *ml = part + 16 * D + 2 * cc;
    f32x4 first[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const int i = tid / L + k * GR;
        first[k] = f32x4{0, 0, 0, 0};
        if (i < jt.splits && cc < jt.cols) first[k] = *reinterpret_cast<const f32x4 *>(mine + piece(i));
    }
    float mm = AT_NONE;
    for (int s = tid; s < jt.splits && cc < jt.cols; s += TC) mm = fmaxf(mm, ml[piece(s)]);
    mm = col_max(mm);
#pragma unroll
    for (int i = 1; i < 16; i *= 2) mm = fmaxf(mm, __shfl_xor(mm, i));
    if (tid % 64 == 0) sm_m[threadIdx.x / 64] = mm;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; i++) mm = fmaxf(mm, sm_m[ci * W + i]);
    float ll = 0.0f;
    f32x4 v = {0, 0, 0, 0};
    for (int s0 = 0; s0 < jt.splits; s0 += TC) {
        float w = 0.0f;
        if (s0 + tid < jt.splits && cc < jt.cols) {
            const float *p = ml + piece(s0 + tid);
            w = __builtin_amdgcn_exp2f(p[0] - mm);
            ll += p[1] * w;
        }
        __syncthreads();
        sw[threadIdx.x] = w;
        __syncthreads();
        const int n = min(TC, jt.splits - s0);
        int i = tid / L;
        if (s0 == 0) {
#pragma unroll
            for (int k = 0; k < 8; k++, i += GR)
                if (i < n) v += first[k] * sw[ci * TC + i];
        }
        for (; i < n && cc < jt.cols; i += GR) v += *reinterpret_cast<const f32x4 *>(mine + piece(s0 + i)) * sw[ci * TC + i];
    }
    ll = wave_sum(ll);
    if (tid % 64 == 0) sm_l[threadIdx.x / 64] = ll;
    so[threadIdx.x] = v;
    __syncthreads();
    if (tid >= L || cc >= jt.cols) return;
    ll = 0.0f;
#pragma unroll
    for (int i = 0; i < W; i++) ll += sm_l[ci * W + i];
#pragma unroll
    for (int i = 1; i < GR; i++) v += so[ci * TC + i * L + tid];
    const int f = jt.col + cc, row = f / G;
    store4<BF ? TG_T_BF16 : TG_T_F16>(o.p, (int64_t)row * o.stride + (int64_t)(hk * G + f - row * G) * D + 4 * tid,
                                      v * (ll == 0.0f ? 0.0f : 1.0f / ll));
}

// The same for the wide column tiles, which have few splits: a thread to four
// dims of a column, which goes through them alone.
template <int D, bool BF, int COLS>
__global__ __launch_bounds__(256) void k_attn_join_wide(KvBatch b, int G, AttnOut o) {
    constexpr int L = D / 4, NC = 256 / L;
    const int hk = blockIdx.y, d = threadIdx.x % L * 4, cc = blockIdx.z * NC + threadIdx.x / L;
    const JoinTile jt = o.join[(size_t)blockIdx.x * b.n_kv + hk];
    if (!jt.splits || cc >= jt.cols) return;
    const size_t step = (size_t)b.n_kv * AT_PART<D, COLS>;
    const float *part = o.part + ((size_t)jt.part * b.n_kv + hk) * AT_PART<D, COLS>, *ml = part + COLS * D + 2 * cc, *mine = part + (size_t)cc * D + d;
    float mm = AT_NONE, ll = 0.0f;
    f32x4 v = {0, 0, 0, 0};
    for (int s = 0; s < jt.splits; s++) mm = fmaxf(mm, ml[s * step]);
#pragma unroll 4
    for (int s = 0; s < jt.splits; s++) {
        const float w = __builtin_amdgcn_exp2f(ml[s * step] - mm);
        ll += ml[s * step + 1] * w;
        v += *reinterpret_cast<const f32x4 *>(mine + s * step) * w;
    }
    const int f = jt.col + cc, row = f / G;
    store4<BF ? TG_T_BF16 : TG_T_F16>(o.p, (int64_t)row * o.stride + (int64_t)(hk * G + f - row * G) * D + d,
                                      v * (ll == 0.0f ? 0.0f : 1.0f / ll));
}

// ================================================================ launchers
// The dynamic-LDS limit of kernel fn raised to `bytes` (above 64 KB) on the
// current device, once per (kernel, device): `done` holds a bit per device.
static hipError_t attn_lds(const void *fn, size_t bytes, std::atomic<uint64_t> &done) {
    if (bytes <= 65536) return hipSuccess;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
    if (bit && (done.load(std::memory_order_relaxed) & bit)) return hipSuccess;
    e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == hipSuccess && bit) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

#define TG_BY_DIM(D, ...)                                                     \
    do {                                                                      \
        if ((D) == 64) { constexpr int DIM = 64; __VA_ARGS__; }               \
        else if ((D) == 128) { constexpr int DIM = 128; __VA_ARGS__; }        \
        else { constexpr int DIM = 256; __VA_ARGS__; }                        \
    } while (0)

hipError_t launch_kv_append(const KvBatch &b, int type, const AppendArgs &a, hipStream_t st) {
    const int64_t units = (int64_t)b.n_tokens * (a.n_heads + 2 * b.n_kv);
    const int64_t grid = (units + 256 / (b.D / 8) - 1) / (256 / (b.D / 8));
    if (grid > UINT32_MAX / 256) return hipErrorInvalidValue;
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
    if (grid > UINT32_MAX / 256) return hipErrorInvalidValue;
    TG_BY_DIM(b.D, TG_LAUNCH(k_kv_read<DIM>, dim3((unsigned)grid), dim3(256), 0, st, b, static_cast<_Float16 *>(k),
                             static_cast<_Float16 *>(v)));
    return hipGetLastError();
}

hipError_t launch_kv_keep(const KvBatch &b, const KeepArgs &a, hipStream_t st) {
    const int64_t grid = ((int64_t)b.n_seqs * b.n_kv * ((a.n_layers + KEEP_LAYERS - 1) / KEEP_LAYERS) + 3) / 4;
    if (grid > UINT32_MAX / 256) return hipErrorInvalidValue;
    if (a.n_layers) TG_BY_DIM(b.D, TG_LAUNCH(k_kv_keep<DIM>, dim3((unsigned)grid), dim3(256), 0, st, b, a));
    if (a.kv_len && (a.kv_len == b.kv_len || !a.n_layers)) TG_LAUNCH(k_kv_keep_len, dim3((b.n_seqs + 255) / 256), dim3(256), 0, st, b, a);
    return hipGetLastError();
}

// Blocks of one launch.  Narrow column tiles: `share` per key head, or one for each tile.  Wide ones, of which there are
// `share` at most: one for each tile and `share` per key head more.  That is enough for their pieces: where an even
// share is taken as it is there are as many at the most (a piece more than its part of them for each tile), and a
// larger one makes fewer.  Of split tiles alone there are 2 share pieces at the most, which is what `parts` holds.
struct AttnPlan {
    int64_t tiles;
    int cols, share, joins, unit;
    int64_t blocks, parts;  // of a key head
    int from, to;           // columns of the sequences that it is for
};
static AttnPlan attn_plan(const KvBatch &b, int n_heads, int max_len, bool many, int from, int to) {
    const int64_t all = (int64_t)b.n_tokens * (n_heads / b.n_kv);
    AttnPlan p;
    p.from = from, p.to = to;
    p.cols = !many ? 16 : b.D == 256 ? AT_COLS<256> : AT_COLS<128>;
    p.tiles = all / p.cols + std::min<int64_t>(b.n_seqs, from ? all / from : b.n_seqs);
    if (to != INT32_MAX) p.tiles = std::min(p.tiles, (int64_t)b.n_seqs * ((to + p.cols - 2) / p.cols));
    // one block of wide tiles or of heads of 256 fits a CU, two of the others
    p.share = std::max(1, (many || b.D == 256 ? 256 : 512) / b.n_kv);
    // Nothing to split where no sequence is longer than a block should take, or there are tiles enough: narrow ones
    // for four rounds; wide ones for one (4 prompts of 447 tokens, 64 heads of 128 over 8: 51 us, split over two rounds 85;
    // one of 2000, 32 heads over 4: 77, split 84).
    if (max_len <= 32 * (many ? 2 * AT_WIDE : 4) || p.tiles > (many ? 1 : 4) * p.share) p.share = 0;
    p.unit = 4;  // a step for each wave; more only where their number would not stay below 2^30
    if (many) {
        p.joins = p.share ? (int)p.tiles : 0;
        p.blocks = p.tiles + p.share, p.parts = 2 * p.share;
    } else {
        p.joins = (int)std::min<int64_t>(p.tiles, p.share), p.blocks = p.share ? p.share : p.tiles, p.parts = 2 * p.share;
        const int64_t steps = (int64_t)b.table_cols * b.page_tokens / 32 + 1;
        while (p.share && p.tiles * (steps / p.unit + 1 + AT_OVER) >= 1 << 30) p.unit *= 2;
    }
    return p;
}

// The launches of a call, one or two.  The mean number of columns of a sequence says which kernel takes all of them.
// 16 sequences of up to 4096 tokens, D = 128, few against many: 64 columns 42 and 50 us, 96 51 and 52, 128 53 and 54,
// 256 88 and 59; one of 16000: 128 43 and 56, 256 51 and 61; 200 of up to 1000: 128 117 and 129, 256 203 and 127; D =
// 64, 16 of up to 8192: 64 72 and 88, 128 87 and 89.  fp16, whose many take longer: D = 128, 128 columns 56 and 74, 192
// 73 and 74, 256 88 and 76; D = 64 128 88 and 109, 192 114 and 111, 256 137 and 114.  D = 256, bf16, 16 of up to 4096:
// 64 columns 55 and 72, 128 78 and 78, 192 103 and 83; fp16 has no wide tiles, its remainders do not fit LDS.
//
// Where that is many, and the rows are so few next to the lengths that not all of more than 8 sequences can be prompts,
// single tokens may be among them, to which a wide tile is a waste: each kernel takes those that are its.  A prompt of
// 2000 and 32 single tokens after 8192, 32 heads over 4: 133 us, 274 in one launch; after 4000 122 and 147; 8 chunks of
// 128, where the second launch finds nothing to do: 84 and 79.  So a row's roundings are those of the kernel that its
// call's numbers choose, not of the row alone.
//
// Trees have few rows next to long sequences, and rarely fill the card: what counts is the longest block of either
// kernel, in narrow steps of 32 tokens, of which a wide one of 64 takes 7 (fp16 10, at heads of 64 6.5; heads of 256
// 8).  A narrow tile costs 12 steps beside its own, a wide block 6, and 16 of its steps at the least.  Of 519 sizes (1
// to 48 sequences of 8 to 200 nodes after 500 to 30000 tokens, all head sizes, 1 to 16 heads to a key head) that chose
// the faster but for 1% of the time in the mean and 1.5 times at the most.  D = 128, bf16, 32 heads over 4, few and
// many: 1 tree of 16 nodes after 2000 21 and 58 us, after 8000 27 and 43; 1 of 200 after 8000 99 and 60; 4 of 64 after
// 2000 36 and 71, after 8000 99 and 58; 48 of 8 after 8000 171 and 232, of 31 509 and 262.  One launch for all: 32
// trees of 16 nodes in the mean after 4200 123 us, each by the kernel that suits it, in two launches, 129; 64 of 32
// after 1000 154 and 187.
static bool tree_wide(const KvBatch &b, int n_heads, int max_len, bool bf16) {
    const AttnPlan few = attn_plan(b, n_heads, max_len, false, 0, INT32_MAX), many = attn_plan(b, n_heads, max_len, true, 0, INT32_MAX);
    const double width = b.D == 256 ? 8 : bf16 ? 7 : b.D == 64 ? 6.5 : 10;
    const double all = (double)b.n_tokens * (n_heads / b.n_kv), seqs = 0.5 * b.n_seqs;
    const double blocks = std::max(1, (b.D == 256 ? 256 : 512) / b.n_kv), wide_blocks = std::max(1, 256 / b.n_kv);
    const double narrow = (all / few.cols + seqs) * (max_len / 32.0 + 12.0) / blocks;
    const double steps = max_len / 64.0, rounds = (all / many.cols + seqs) / wide_blocks;
    return narrow > width * (many.share ? std::max(16.0, rounds * steps) : std::max(1.0, rounds) * steps) + 6.0;
}

static int attn_plans(const KvBatch &b, int n_heads, int max_len, bool bf16, bool tree, AttnPlan p[2]) {
    const int64_t all = (int64_t)b.n_tokens * (n_heads / b.n_kv);
    if (tree) {
        p[0] = attn_plan(b, n_heads, max_len, (b.D < 256 || bf16) && tree_wide(b, n_heads, max_len, bf16), 0, INT32_MAX);
        return 1;
    }
    const int few = bf16 ? 128 : 192;
    const bool many = (b.D < 256 || bf16) && all >= few * (int64_t)b.n_seqs;
    const bool both = many && b.n_seqs > 8 && 2 * (int64_t)b.n_tokens < (int64_t)b.n_seqs * max_len;
    p[0] = attn_plan(b, n_heads, max_len, many, both ? few : 0, INT32_MAX);
    if (both) p[1] = attn_plan(b, n_heads, max_len, false, 0, few);
    return both ? 2 : 1;
}

static size_t attn_join_bytes(const KvBatch &b, const AttnPlan &p) {
    return ((size_t)p.joins * b.n_kv * sizeof(JoinTile) + 255) / 256 * 256;
}

// Enough for rows of either type; a call's launches use it one after the other.
size_t attn_workspace(const KvBatch &b, int n_heads, int max_len, bool tree) {
    size_t most = 0;
    for (const bool bf16 : {false, true}) {
        AttnPlan p[2];
        for (int i = attn_plans(b, n_heads, max_len, bf16, tree, p) - 1; i >= 0; i--)
            if (p[i].share) most = std::max(most, attn_join_bytes(b, p[i]) + (size_t)p[i].parts * b.n_kv * (p[i].cols * (b.D + 2)) * sizeof(float));
    }
    return most;
}

template <int D, bool BF, bool TREE>
static hipError_t attn_launch(const KvBatch &b, KvRows q, int G, float scale, const AttnPlan &p, const AttnOut &o, hipStream_t st) {
    static std::atomic<uint64_t> done{0};
    const dim3 grid((unsigned)p.blocks, (unsigned)b.n_kv);
    const FastDiv tpp = make_fastdiv((uint32_t)(b.page_tokens / 16));
    if constexpr (D < 256 || BF) {
        if (p.cols != 16) {
            constexpr size_t LDS = (BF ? 5 : 10) * 64 * D * 2;
            const hipError_t e = attn_lds((const void *)k_attn_tile<D, BF, TREE>, LDS, done);
            if (e != hipSuccess) return e;
            TG_LAUNCH((k_attn_tile<D, BF, TREE>), dim3(grid.x * grid.y), dim3(512), LDS, st, b, q, G, scale, p.share, tpp, o);
            if (p.share)
                TG_LAUNCH((k_attn_join_wide<D, BF, AT_COLS<D>>), dim3(p.joins, b.n_kv, AT_COLS<D> * D / 1024), dim3(256), 0, st, b, G, o);
            return hipSuccess;
        }
    }
    TG_LAUNCH((k_attn_split<D, BF, TREE>), grid, dim3(256), 0, st, b, q, G, scale, p.share, p.unit, tpp, o);
    if (!p.share) return hipSuccess;
    if (p.joins * b.n_kv <= 64) TG_LAUNCH((k_attn_join<D, BF, 256>), dim3(p.joins, b.n_kv, 16), dim3(256), 0, st, b, G, o);
    else TG_LAUNCH((k_attn_join<D, BF, 64>), dim3(p.joins, b.n_kv, 4), dim3(256), 0, st, b, G, o);
    return hipSuccess;
}

hipError_t launch_attn(const KvBatch &b, int type, KvRows q, int n_heads, float scale, void *out, int64_t out_stride,
                       int max_len, void *ws, hipStream_t st) {
    AttnPlan plans[2];
    const int n = attn_plans(b, n_heads, max_len, type == TG_T_BF16, b.bits, plans), G = n_heads / b.n_kv;
    hipError_t e = hipSuccess;
    for (int i = 0; i < n && e == hipSuccess; i++) {
        const AttnPlan &p = plans[i];
        // threads of the launch's first dimension
        if (p.blocks * (p.cols != 16 ? 512 * b.n_kv : 256) > UINT32_MAX) return hipErrorInvalidValue;
        KvBatch kb = b;
        kb.cols_from = p.from, kb.cols_to = p.to;
        const AttnOut o{out, out_stride, static_cast<JoinTile *>(ws), p.joins,
                        reinterpret_cast<float *>(static_cast<uint8_t *>(ws) + attn_join_bytes(b, p))};
        TG_BY_DIM(b.D, {
            const bool bf = type != TG_T_F16;
            if (b.bits) e = bf ? attn_launch<DIM, true, true>(kb, q, G, scale, p, o, st) : attn_launch<DIM, false, true>(kb, q, G, scale, p, o, st);
            else e = bf ? attn_launch<DIM, true, false>(kb, q, G, scale, p, o, st) : attn_launch<DIM, false, false>(kb, q, G, scale, p, o, st);
        });
    }
    return e != hipSuccess ? e : hipGetLastError();
}

}  // namespace tg
