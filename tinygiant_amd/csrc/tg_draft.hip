// tg_draft.hip -- trees of drafted tokens on the device: which nodes each one sees and how deep it stands, and which of
// the drafts a target's probabilities keep.
//
// Node j of a sequence is row cu[s] + j of the batch; its parent is a node before it, so a walk towards the root only
// goes down in j.
#include "tg_device.h"
#include "tg_internal.h"

#include "../../include/tinygiant.h"

#include <algorithm>
#include <type_traits>

namespace tg {

constexpr int DT_NODES = 1024;  // of one sequence at the most
constexpr int DT_NONE = -1, DT_BAD = -2;

// rows of sequence s, kept inside the row tensors whatever cu holds
struct TreeRows {
    int lo, n;
};
TG_DEV TreeRows tree_rows(const DraftTrees &t, int s) {
    const int lo = min(max(t.cu[s], 0), t.n_tokens), hi = min(max(t.cu[s + 1], lo), t.n_tokens);
    return {lo, hi - lo};
}
TG_DEV int parent_of(const DraftTrees &t, int lo, int j) {
    const int p = t.parent ? t.parent[lo + j] : j - 1;
    return p >= DT_NONE && p < j ? p : DT_BAD;
}

// A block per sequence, a thread per node, which walks to its root through the parents in LDS and sets the bits of what
// it meets, one word after the other.  Bound by latency: the rows' bounds, the parents, then a dependent read of LDS a
// step, so by the depth, and from 257 nodes on by the depths of the up to four nodes of a thread and the words that it
// writes.  One tree of 16 nodes, 4 deep, 2.0 us (a launch that does nothing takes 1.7); 37 of up to 61, 7 deep, 3.3;
// one of 512, 9 deep, 7.0, of 1024 21.6.  Chains, with parents or without: 5 nodes 1.9 us, 16 2.6, 64 7.5, 256 30, 1024
// 291.
__global__ __launch_bounds__(256) void k_draft_tree(DraftTrees t, uint32_t *bits, int32_t *depth, int32_t *links) {
    __shared__ int16_t par[DT_NODES];
    __shared__ uint8_t kids[DT_NODES];
    const TreeRows r = tree_rows(t, blockIdx.x);
    const int n = min(r.n, t.max_nodes), words = (t.max_nodes + 31) / 32;
    for (int j = threadIdx.x; j < n; j += 256) par[j] = (int16_t)parent_of(t, r.lo, j), kids[j] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += 256)
        if (par[j] >= 0) kids[par[j]] = 1;
    __syncthreads();
    // rows before the first and behind the last sequence are no nodes either
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < r.lo; i += 256) links[i] = -1;
    if (blockIdx.x == gridDim.x - 1)
        for (int i = r.lo + r.n + threadIdx.x; i < t.n_tokens; i += 256) links[i] = -1;
    for (int j = threadIdx.x; j < r.n; j += 256) {
        uint32_t *out = bits + (size_t)(r.lo + j) * words;
        int d = -1, a = j < n ? j : DT_BAD, w = words;  // words from w on are written
        uint32_t v = 0;
        for (; a >= 0; a = par[a], d++) {
            if (a / 32 < w) {
                if (w < words) out[w] = v;
                while (--w > a / 32) out[w] = 0;
                v = 0;
            }
            v |= 1u << (a % 32);
        }
        if (a == DT_NONE) {
            out[w] = v;
            while (w > 0) out[--w] = 0;
        } else {
            for (w = 0; w < words; w++) out[w] = 0;
            d = -1;
        }
        depth[r.lo + j] = d;
        links[r.lo + j] = d < 0 ? -1 : 2 * (int)blockIdx.x + kids[j];
    }
}

hipError_t launch_draft_tree(const DraftTrees &t, uint32_t *bits, int32_t *depth, int32_t *links, hipStream_t st) {
    TG_LAUNCH(k_draft_tree, dim3((unsigned)t.n_seqs), dim3(256), 0, st, t, bits, depth, links);
    return hipGetLastError();
}

// ================================================================ verification
// One sequence's walk.  At a node, p = softmax(target's logits / T) and q the same of the draft's.  Its children x were
// drawn from q, one after the other: x stays with probability r(x) / q(x) at the most 1, where r = p for the first, and
// each one that does not stay leaves max(r - q, 0) / its sum for the next, so that whichever stays, or the token that
// is drawn of what is left in the end, is distributed as p.  In closed form r = max(p - c q, 0) / Z with c = 0, Z = 1
// at first; one that does not stay makes c + Z of c, and Z the sum of max(p - c q, 0) for the new c: one number is kept
// of all that were asked.  Without q the children are candidates that no one drew, kept with probability p(x) / (1 -
// what those before them had), and what is left is p without them.
//
// Whatever a random number decides is decided in 64 bits: probabilities, their sums and running sums.
constexpr int V_CHUNK = 4096;  // values of a row to a block of the first launch
constexpr int V_PIECE = 2048;  // ... whose sum is kept
constexpr int V_PER = V_CHUNK / V_PIECE;
constexpr int V_ROUNDS = 12;     // sweeps that have launches of their own

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int TYPE>
TG_DEV float load1(const void *p, int64_t i) {
    if constexpr (TYPE == TG_T_F32) return static_cast<const float *>(p)[i];
    const uint16_t v = static_cast<const uint16_t *>(p)[i];
    return TYPE == TG_T_F16 ? h2f(v) : __uint_as_float((uint32_t)v << 16);
}
// 8 values of a row from i on: rows of any alignment, global loads of 16 bytes need that of their elements
template <int TYPE>
TG_DEV void load8(const void *row, int i, float v[8]) {
    if constexpr (TYPE == TG_T_F32) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            f32x4 x;
            __builtin_memcpy(&x, static_cast<const float *>(row) + i + 4 * h, 16);
#pragma unroll
            for (int e = 0; e < 4; e++) v[4 * h + e] = x[e];
        }
    } else {
        u32x4 x;
        __builtin_memcpy(&x, static_cast<const uint16_t *>(row) + i, 16);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint16_t b = (uint16_t)(x[e / 2] >> (16 * (e % 2)));
            v[e] = TYPE == TG_T_F16 ? h2f(b) : __uint_as_float((uint32_t)b << 16);
        }
    }
}
// N times 8 values, STEP apart, of a stretch of the row that ends at `end`: one branch around all of the loads, and a
// value at a time, -inf behind the row's end, where the stretch passes it
template <int TYPE, int N, int STEP>
TG_DEV void load_stretch(const void *row, int i, int end, int V, float v[N][8]) {
    if (end <= V) {
#pragma unroll
        for (int k = 0; k < N; k++) load8<TYPE>(row, i + k * STEP, v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int at = i + k * STEP + e;
                const float x = load1<TYPE>(row, min(at, V - 1));
                v[k][e] = at < V ? x : -INFINITY;
            }
    }
}
template <int TYPE>
TG_DEV const void *row_of(const void *p, int64_t stride, int row) {
    return static_cast<const uint8_t *>(p) + (int64_t)row * stride * (TYPE == TG_T_F32 ? 4 : 2);
}

// Exponentials of what is 0 or below, to some 2^-51: exp(d / T) = 2^(y / 32), y = d 32 log2(e) / T, is 2^(j / 32) from
// a table times the power of 2 that the nearest whole number n = 32 i + j of y gives, times 2^(f / 32) for the rest f,
// at most 1/2, by the polynomial of degree 5 that has its values at the six Chebyshev nodes (off by 2^-52.6, the
// constant rounded to 1).  Below 2^-1021 the result is 0.  13 operations on doubles; by the remainder of ln 2 and
// Taylor's polynomial 26.
constexpr int V_TABLE = 32;
struct Exp64 {
    double by, least;     // 32 log2(e) / T; the least d whose exponential is not 0
    const uint64_t *two;  // 2^(j / 32), its exponent's half less what n brings into it of j
    TG_DEV double operator()(double d) const {
        constexpr double ONES = 6755399441055744.0;  // 1.5 2^52: its unit is 1
        const double t = __builtin_fma(d, by, ONES), f = __builtin_fma(d, by, -(t - ONES));
        const int n = (int)__builtin_bit_cast(uint64_t, t);
        double p = 3.9737266313166245e-11;
        p = __builtin_fma(p, f, 9.172616498159851e-09);
        p = __builtin_fma(p, f, 1.6938509724215757e-06);
        p = __builtin_fma(p, f, 0.0002345961981972034);
        p = __builtin_fma(p, f, 0.02166084939249829);
        p = __builtin_fma(p, f, 1.0);
        const uint64_t w = two[n & (V_TABLE - 1)];
        const uint32_t hi = (uint32_t)(w >> 32) + ((uint32_t)n << 15);
        const double r = __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)w) * p;
        return d > least ? r : 0.0;
    }
};
TG_DEV Exp64 exp_of(double by, const uint64_t *two) { return {by, -32.0 * 1021.0 / by, two}; }
// the table, by repeated square roots of 2: 2^(j / 32) is the product of those of j's bits
TG_DEV void exp_table(uint64_t *two, int j) {
    double r = 1.0;
    if (j & 16) r *= 1.4142135623730951;
    if (j & 8) r *= 1.189207115002721;
    if (j & 4) r *= 1.0905077326652577;
    if (j & 2) r *= 1.0442737824274138;
    if (j & 1) r *= 1.0218971486541166;
    two[j] = __builtin_bit_cast(uint64_t, r) - ((uint64_t)j << 47);
}

// the sequence's temperature; 32 log2(e) / T, so that -inf times it stays -inf
TG_DEV float temperature_of(const VerifyArgs &a, int s) { return a.temps ? a.temps[s] : a.temp; }
TG_DEV double factor_of(float t) { return fmax(46.16624130844683 / (double)t, 1e-300); }

TG_DEV float uni(float v) { return __int_as_float(uni(__float_as_int(v))); }
// what is true or not in all lanes of a wave, told to the compiler
TG_DEV bool sure(bool c) { return __ballot(c) != 0; }

// What a lane gets from `CTRL` lanes further down (DPP: row_shr 1, 2, 4, 8, row_bcast 15, 31 for rows ROWS), or `none`
template <int CTRL, int ROWS>
TG_DEV float from_below(float v, float none) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), CTRL, ROWS, 0xF, false));
}
template <int CTRL, int ROWS>
TG_DEV double from_below(double v, double none) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v), o = __builtin_bit_cast(uint64_t, none);
    const uint32_t lo = __builtin_amdgcn_update_dpp((int)o, (int)b, CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp((int)(o >> 32), (int)(b >> 32), CTRL, ROWS, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// over the lanes up to each (half: of its half of the wave), in a fixed order
template <class T, class F>
TG_DEV T wave_upto(T v, T none, bool half, F f) {
    v = f(v, from_below<0x111, 0xF>(v, none));
    v = f(v, from_below<0x112, 0xF>(v, none));
    v = f(v, from_below<0x114, 0xF>(v, none));
    v = f(v, from_below<0x118, 0xF>(v, none));
    v = f(v, from_below<0x142, 0xA>(v, none));
    return half ? v : f(v, from_below<0x143, 0xC>(v, none));
}
TG_DEV double of_lane(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)b, lane), hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
TG_DEV float of_lane(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }
constexpr auto v_plus = [](auto x, auto y) { return x + y; };
constexpr auto v_most = [](float x, float y) { return fmaxf(x, y); };
TG_DEV double sums_upto(double v) { return wave_upto(v, 0.0, false, v_plus); }
TG_DEV double wave_add(double v) { return of_lane(sums_upto(v), 63); }
TG_DEV float wave_max(float v) { return of_lane(wave_upto(v, -INFINITY, false, v_most), 63); }
// of the half of the wave that a lane is in
template <class T>
TG_DEV T half_of(T v, int lane) {
    const T a = of_lane(v, 31), b = of_lane(v, 63);
    return lane < 32 ? a : b;
}
TG_DEV double half_add(double v, int lane) { return half_of(wave_upto(v, 0.0, true, v_plus), lane); }
TG_DEV float half_max(float v, int lane) { return half_of(wave_upto(v, -INFINITY, true, v_most), lane); }
// over the four waves of a block, in order; `sm` is 4 values that nothing else uses until the next barrier
TG_DEV double block_add(double v, double *sm) {
    v = wave_add(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) sm[threadIdx.x / 64] = v;
    __syncthreads();
    return ((sm[0] + sm[1]) + sm[2]) + sm[3];
}
TG_DEV float block_max(float v, float *sm) {
    v = wave_max(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) sm[threadIdx.x / 64] = v;
    __syncthreads();
    return fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
}

// The largest value of each chunk of the rows that a walk may ask (those that something follows, of greedy sequences
// all), of the chunk and its pieces the sums of exp((v - largest) / T), or the place of the first of the largest.  NaN
// or +inf: the largest is +inf.
//
// Bound by reading where there are rows enough: 64 chains of up to 7 nodes, 151936 tokens, fp32, target's and draft's
// rows: 33 us, 5 TB/s; 5 rows of 304 KB of each 5.4 us, launch, load and two joins.  Chunks of 4096 against 2048 and
// 8192: 35.4, 43.6 and 36.7 us, 5.2, 4.6 and 6.9.  Rows loaded before it is known whether they are asked for: chains of
// 5, 13 and 54, bf16, 5.4, 8.4 and 20.0 us, 5.3, 7.7 and 20.2 so; trees of 13 and 54, fp32, most of whose nodes nothing
// follows, 6.3 and 15.2, 5.5 and 13.4 so.
template <int TYPE>
__global__ __launch_bounds__(256) void k_verify_rows(VerifyArgs a) {
    __shared__ float sm[4];
    __shared__ double smd[4][V_PER];
    __shared__ uint64_t two[V_TABLE];
    __shared__ int first;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks, of = blockIdx.y;
    const void *p = of ? row_of<TYPE>(a.draft, a.draft_stride, row) : row_of<TYPE>(a.logits, a.stride, row);
    float v[V_PER][8], m = -INFINITY;
    if (threadIdx.x < V_TABLE) exp_table(two, threadIdx.x);
    const int link = uni(a.links[row]);  // twice the sequence, and whether something follows
    if (link < 0 || link / 2 >= a.t.n_seqs) return;
    const float t = uni(temperature_of(a, link / 2));
    const bool greedy = !(t > 0.0f);
    if (greedy ? of : !(link & 1)) return;
    load_stretch<TYPE, V_PER, V_PIECE>(p, chunk * V_CHUNK + threadIdx.x * 8, (chunk + 1) * V_CHUNK, a.vocab, v);
    bool bad = false;
#pragma unroll
    for (int k = 0; k < V_PER; k++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            m = fmaxf(m, v[k][e]);
            bad |= !(v[k][e] < INFINITY);
        }
    m = block_max(bad ? INFINITY : m, sm);
    const size_t at_row = (size_t)row * 2 + of;
    if (threadIdx.x == 0) a.top[at_row * a.chunks + chunk] = m;
    if (greedy) {
        if (threadIdx.x == 0) first = INT32_MAX;
        __syncthreads();
        int at = INT32_MAX;
#pragma unroll
        for (int k = V_PER - 1; k >= 0; k--)
#pragma unroll
            for (int e = 7; e >= 0; e--) at = v[k][e] == m ? chunk * V_CHUNK + k * V_PIECE + (int)threadIdx.x * 8 + e : at;
        if (at != INT32_MAX) atomicMin(&first, at);
        __syncthreads();
        if (threadIdx.x == 0) a.arg[(size_t)row * a.chunks + chunk] = first;
        return;
    }
    if (m == INFINITY) return;
    const Exp64 exp64 = exp_of(factor_of(t), two);
#pragma unroll
    for (int k = 0; k < V_PER; k++) {
        double sum = 0.0;
        if (m > -INFINITY)
#pragma unroll
            for (int e = 0; e < 8; e++) sum += exp64((double)v[k][e] - m);
        sum = wave_add(sum);
        if (lane == 0) smd[wave][k] = sum;
    }
    __syncthreads();
    if (threadIdx.x < V_PER) {
        const int k = threadIdx.x;
        double z = ((smd[0][k] + smd[1][k]) + smd[2][k]) + smd[3][k];
        if (chunk * V_PER + k < a.pieces) a.sum[at_row * a.pieces + chunk * V_PER + k] = z;
#pragma unroll
        for (int m = 1; m < V_PER; m *= 2) z += __shfl_xor(z, m);
        if (k == 0) a.whole[at_row * a.chunks + chunk] = z;
    }
}

// One piece of a sweep, by a block: the sum of max(p - c q, 0) over it, or (leaf) its largest value and the sum of
// exp((v - largest) / T).
template <int TYPE>
struct Pieces {
    const void *logits, *draft;
    int64_t stride, draft_stride;
    int vocab;
    Exp64 exp64;
    float *smf;
    double *smd;
    TG_DEV Pieces(const VerifyArgs &a, const Exp64 &e, float *f, double *d)
        : logits(a.logits), draft(a.draft), stride(a.stride), draft_stride(a.draft_stride), vocab(a.vocab), exp64(e), smf(f), smd(d) {}
    TG_DEV const void *row_p(int row) const { return row_of<TYPE>(logits, stride, row); }
    TG_DEV const void *row_q(int row) const { return row_of<TYPE>(draft, draft_stride, row); }
    TG_DEV void load(const void *row, int k, float v[1][8]) const {
        load_stretch<TYPE, 1, 0>(row, k * V_PIECE + (int)threadIdx.x * 8, (k + 1) * V_PIECE, vocab, v);
    }
    TG_DEV void load_both(int row, int k, float v[2][8]) const {
        const int i = k * V_PIECE + (int)threadIdx.x * 8;
        if ((k + 1) * V_PIECE <= vocab) {  // one branch around the loads of both
            load8<TYPE>(row_p(row), i, v[0]);
            load8<TYPE>(row_q(row), i, v[1]);
        } else {
            load(row_p(row), k, v);
            load(row_q(row), k, v + 1);
        }
    }
    TG_DEV double rest(const WalkState &w, float v, float q) const {
        return fmax(exp64((double)v - w.Mp) * w.ip - exp64((double)q - w.Mq) * w.iq, 0.0);
    }
    TG_DEV void operator()(const WalkState &w, int k, double &sum, float &top) const {
        float v[2][8];
        double z = 0.0;
        if (!uni(w.leaf)) {
            load_both(uni(w.row), k, v);
#pragma unroll
            for (int e = 0; e < 8; e++) z += rest(w, v[0][e], v[1][e]);
        } else {
            load(row_p(uni(w.row)), k, v);
            float m = -INFINITY;
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                bad |= !(v[0][e] < INFINITY);
                m = fmaxf(m, v[0][e]);
            }
            top = block_max(bad ? INFINITY : m, smf);
            if (top > -INFINITY && top < INFINITY)
#pragma unroll
                for (int e = 0; e < 8; e++) z += exp64((double)v[0][e] - top);
        }
        sum = block_add(z, smd);
    }
};

// What blocks hand to each other goes past the caches of an XCD, and what is to be seen first is waited for (a release
// at the device's scope writes back a whole L2).
template <class T>
TG_DEV T seen_now(const T *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <class T>
TG_DEV void show(T *p, T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
TG_DEV void shown() { __builtin_amdgcn_s_waitcnt(0x0F70); }  // vmcnt 0: this thread's stores are acknowledged

// LDS of a walk, for `nodes` of them and rows of `pieces`
struct WalkNodes {
    double *u;        // random numbers
    double *e, *inv;  // the nodes' logits at their parents, then exponentials of those; 1 / the rows' sums of exponentials
    double *weight;   // of the pieces of what is left
    float *top;       // the rows' largest values (e, inv, top: target's, then draft's)
    float *most;      // of a sweep's pieces
    uint16_t *list;   // in its place: pieces to be summed again
    int *tok;
    int16_t *par, *way;
    uint8_t *again;   // an earlier sibling has the same token
    TG_DEV WalkNodes(uint8_t *lds, int nodes, int pieces) {
        u = reinterpret_cast<double *>(lds), e = u + nodes, inv = e + 2 * nodes, weight = inv + 2 * nodes;
        top = reinterpret_cast<float *>(weight + pieces), most = top + 2 * nodes, list = reinterpret_cast<uint16_t *>(most);
        tok = reinterpret_cast<int *>(most + pieces);
        par = reinterpret_cast<int16_t *>(tok + nodes), way = par + nodes;
        again = reinterpret_cast<uint8_t *>(way + nodes);
    }
    static constexpr size_t bytes(int nodes, int pieces) { return ((size_t)nodes * (5 * 8 + 3 * 4 + 2 * 2 + 1) + (size_t)pieces * (8 + 4) + 15) / 16 * 16; }
};

// A sequence's walk, by one block, up to the next sum over a whole row that it needs (what rejected siblings drawn from
// q leave, the row of a leaf): it asks for a sweep of it and leaves what it knows in memory.  The next launch has a
// block to each piece, and the last of them to be done goes on with the walk: no block waits for another.  With `alone`
// the block does its sweeps itself, a piece after the other.  What decides where the walk goes is the same in all of
// its lanes, and told so to the compiler (uni, sure), and every loop has a counter that is the same in all of them
// (each, by_lanes): with loops that lanes left one after the other, what it moved between registers behind such a loop
// was moved with all lanes off, and lost (rejected tokens were drawn).
template <int TYPE>
TG_DEV void walk(const VerifyArgs &a, int s, WalkState w, const Pieces<TYPE> &piece_of, bool begin, bool alone) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ int hits[4], lasts[4];
    __shared__ uint8_t inner[4][64];
    __shared__ int listed;
    const int tid = threadIdx.x, lane = tid % 64, wave = uni(tid / 64), V = a.vocab, N = a.t.max_nodes;
    const TreeRows r = tree_rows(a.t, s);
    const bool greedy = !(uni(temperature_of(a, s)) > 0.0f), with_q = a.draft && !greedy;
    const Exp64 exp64 = piece_of.exp64;
    double *smd = piece_of.smd;
    const int n = uni(min(r.n, N)), lo = uni(r.lo);
    const WalkNodes d(lds, N, a.pieces);
    u32x4 *held = reinterpret_cast<u32x4 *>(a.held + (size_t)s * a.held_bytes);
    // f(i) for each i below n, by the block, or from `first` on by `width` lanes: the loop itself is the same in all
    // lanes
    auto each = [&](int n, auto f) {
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += 256)
            if (i0 + tid < n) f(i0 + tid);
    };
    auto by_lanes = [&](int first, int n, int lane, int width, auto f) {
#pragma unroll 1
        for (int i0 = first; i0 < n; i0 += width)
            if (i0 + lane < n) f(i0 + lane);
    };
    auto copy = [&](u32x4 *to, const u32x4 *from) { each((int)(a.held_bytes / 16), [&](int i) { to[i] = from[i]; }); };

    // Largest values and sums of the rows of nodes j0 .. j0 + 63, from those of their chunks: half a wave to a row,
    // four rows at a time.  For a greedy sequence the first of the largest stands in the place of the draft's logits.
    auto join = [&](int j0) {
        // those that something follows, of greedy sequences all
        const int link = j0 + lane < n ? a.links[lo + j0 + lane] : -1;
        const bool asked = link >= 0 && (greedy || link & 1);
        const uint64_t asks = __ballot(asked);
        if (asked) inner[wave][__builtin_popcountll(asks & ((1ull << lane) - 1))] = (uint8_t)lane;
        wave_lds_sync();
        const int l = lane % 32, two_rows = with_q, units = __builtin_popcountll(asks) << two_rows;
        // of the unit that a half wave has: its place among the rows' parts; among the nodes'
        auto row_at = [&](int i) { return ((size_t)(lo + j0 + inner[wave][i >> two_rows]) * 2 + (i & two_rows)) * a.chunks; };
        auto node_at = [&](int i) { return j0 + inner[wave][i >> two_rows] + (i & two_rows) * N; };
        if (greedy) {
#pragma unroll 1
            for (int i0 = 2 * wave; i0 < units; i0 += 8) {
                const int i = min(i0 + lane / 32, units - 1);
                const float *top = a.top + row_at(i);
                float m = -INFINITY;
                by_lanes(0, a.chunks, l, 32, [&](int k) { m = fmaxf(m, top[k]); });
                m = half_max(m, lane);
                int best = INT32_MAX;
                by_lanes(0, a.chunks, l, 32, [&](int k) {
                    if (top[k] == m) best = min(best, a.arg[row_at(i) / 2 + k]);
                });
#pragma unroll
                for (int k = 1; k < 32; k *= 2) best = min(best, __shfl_xor(best, k));
                if (l == 0) d.top[node_at(i)] = m, d.e[N + node_at(i)] = best;
            }
            __syncthreads();
            return;
        }
        constexpr int B = 4;
#pragma unroll 1
        for (int i0 = 2 * wave; i0 < units; i0 += 8 * B) {
            float m[B][2];
            double z[B][2];
#pragma unroll
            for (int b = 0; b < B; b++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const size_t at = row_at(min(i0 + 8 * b + lane / 32, units - 1)) + min(l + 32 * h, a.chunks - 1);
                    m[b][h] = a.top[at];
                    z[b][h] = l + 32 * h < a.chunks ? a.whole[at] : 0.0;
                }
#pragma unroll
            for (int b = 0; b < B; b++) {
                if (i0 + 8 * b >= units) break;
                const int i = min(i0 + 8 * b + lane / 32, units - 1);
                float t = fmaxf(m[b][0], m[b][1]);
                by_lanes(64, a.chunks, l, 32, [&](int k) { t = fmaxf(t, a.top[row_at(i) + k]); });
                t = half_max(t, lane);
                double y = z[b][0] * exp64((double)m[b][0] - t) + z[b][1] * exp64((double)m[b][1] - t);
                by_lanes(64, a.chunks, l, 32, [&](int k) { y += a.whole[row_at(i) + k] * exp64((double)a.top[row_at(i) + k] - t); });
                y = half_add(y, lane);
                if (l == 0) d.top[node_at(i)] = t, d.inv[node_at(i)] = 1.0 / y;
            }
        }
        __syncthreads();
        each(n, [&](int j) {
            const int p = d.par[j];
            if (p < j0 || p >= j0 + 64) return;
            d.e[j] = exp64(d.e[j] - d.top[p]);
            if (with_q) d.e[N + j] = exp64(d.e[N + j] - d.top[N + p]);
        });
        __syncthreads();
    };
    bool none = !n;  // or node 0 is no node, so that none of the rows was summed
    if (begin) {
        none = none || a.links[lo] < 0;
        each(n, [&](int j) {
            const int p = parent_of(a.t, lo, j), x = a.tokens[lo + j];
            const bool ok = p >= 0 && x >= 0 && x < V;
            d.par[j] = (int16_t)p, d.tok[j] = x, d.u[j] = a.u[lo + j];
            if (!greedy) {
                d.e[j] = ok ? load1<TYPE>(piece_of.row_p(lo + p), x) : -INFINITY;
                if (with_q) d.e[N + j] = ok ? load1<TYPE>(piece_of.row_q(lo + p), x) : -INFINITY;
            }
        });
        if (tid == 0) d.way[0] = 0;
    } else {
        copy(reinterpret_cast<u32x4 *>(lds), held);
        __syncthreads();
        each(a.pieces, [&](int k) {
            d.weight[k] = seen_now(a.swept_sum + (size_t)s * a.pieces + k);
            if (w.leaf) d.most[k] = seen_now(a.swept_top + (size_t)s * a.pieces + k);
        });
    }
    __syncthreads();
    // the next child of `node` behind j, or -1: the same in every wave, like all that follows
    auto child = [&](int node, int j) {
        for (int k = j + 1; k < n; k += 64) {
            const uint64_t m = __ballot(k + lane < n && d.par[min(k + lane, n - 1)] == node);
            if (m) return k + __builtin_ctzll(m);
        }
        return -1;
    };
    auto no_number = [](float m) { return m == INFINITY || m == -INFINITY; };
    auto total_of = [&]() {  // of the pieces' weights
        double z = 0.0;
        by_lanes(0, a.pieces, lane, 64, [&](int k) { z += d.weight[k]; });
        return wave_add(z);
    };

    int at = begin ? 0 : uni(w.at), kept = begin ? 1 : uni(w.kept), joined = begin ? 0 : uni(w.joined), next = -1;
    bool swept = !begin;  // this launch goes on behind a sweep
    none = sure(none);
    for (; kept <= n && !none;) {
        const int row = lo + at, kid = child(at, at);
        int yes = -1;
        if (at >= joined) {
            join(at);
            joined = at + 64;
        }
        if (greedy) {
            if (no_number(uni(d.top[at]))) break;
            next = uni((int)d.e[N + at]);
            for (int k = at + 1; k < n && yes < 0; k += 64) {
                const int j = min(k + lane, n - 1);
                const uint64_t m = __ballot(k + lane < n && d.par[j] == at && d.tok[j] == next);
                if (m) yes = k + __builtin_ctzll(m);
            }
            if (yes >= 0) next = -1;
        } else {
            w.row = row, w.leaf = kid < 0;
            w.Mp = 0.0, w.ip = 1.0, w.Mq = 0.0;
            double iq = 1.0;
            if (kid >= 0) {
                w.Mp = d.top[at], w.ip = d.inv[at];
                if (with_q) w.Mq = d.top[N + at], iq = d.inv[N + at];
                if (no_number(uni((float)w.Mp)) || no_number(uni((float)w.Mq))) break;
            }
            if (with_q || kid < 0) {
                // each child that is rejected leaves a sweep's sums, by pieces: to the next one, or to be drawn from;
                // as does the row of a leaf
                double c = swept ? w.c : 0.0, left = 1.0;
                int k = swept ? uni(w.k) : kid;
                for (;;) {
                    if (!swept) {
                        if (k >= 0) {
                            const double px = d.e[k] * w.ip, qx = d.e[N + k] * iq;
                            if (sure(d.u[k] * left * qx < px - c * qx)) {
                                yes = k;
                                break;
                            }
                            c += left;
                            k = child(at, k);
                        }
                        w.iq = c * iq;
                        if (!alone) {
                            __syncthreads();
                            copy(held, reinterpret_cast<u32x4 *>(lds));
                            w.c = c, w.k = k, w.at = at, w.kept = kept, w.joined = joined, w.asks = 1;
                            if (tid == 0) a.states[s] = w;
                            return;
                        }
                        for (int i = 0; i < a.pieces; i++) {
                            double z;
                            float m;
                            piece_of(w, i, z, m);
                            if (tid == 0) d.weight[i] = z, d.most[i] = m;
                        }
                        __syncthreads();
                    }
                    swept = false;
                    w.iq = c * iq;
                    if (k < 0) break;
                    left = total_of();
                }
            } else {
                // side by side: each candidate with what those before it have left; one whose token was asked before,
                // or is none, has nothing
                double left = 1.0;
                for (int k = at + 1; k < n && yes < 0; k += 64) {
                    const int j = min(k + lane, n - 1), x = d.tok[j];
                    const bool mine = k + lane < n && d.par[j] == at;
                    bool again = x < 0 || x >= V;
                    for (int i = at + 1; i <= k; i += 64) {
                        const int y = d.tok[min(i + lane, n - 1)];
                        for (uint64_t m = __ballot(i + lane < n && d.par[min(i + lane, n - 1)] == at); m; m &= m - 1) {
                            const int f = __builtin_ctzll(m);
                            again |= i + f < k + lane && __builtin_amdgcn_readlane(y, f) == x;
                        }
                    }
                    if (mine) d.again[j] = again;
                    const double px = mine && !again ? d.e[j] * w.ip : 0.0, up = sums_upto(px);
                    const uint64_t m = __ballot(px > 0.0 && d.u[j] * (left - (up - px)) < px);
                    if (m) yes = k + __builtin_ctzll(m);
                    left -= of_lane(up, 63);
                }
                __syncthreads();
            }
            if (yes < 0) {
                if (!sure(d.u[0] >= 0.0 && d.u[0] < 1.0)) break;
                // what is left, by pieces: a sweep's sums, or the row's own
                bool of_rest = with_q && kid >= 0, without = !with_q && kid >= 0;
                // A piece's sum is relative to its chunk's largest value: one that is next to nothing may be of
                // elements that are each 0 next to the row's largest.  From 2^-1000 on it has one of 2^-1011 at least,
                // and, where less than 15 / 16 are taken off below, of 2^-1015, which Exp64 does not make 0.
                auto own_weights = [&]() {
                    __syncthreads();
                    each(a.pieces, [&](int k) {
                        const double z = a.sum[(size_t)row * 2 * a.pieces + k] * exp64((double)a.top[(size_t)row * 2 * a.chunks + k / V_PER] - w.Mp);
                        d.weight[k] = z < 0x1p-1000 ? 0.0 : z;
                    });
                    __syncthreads();
                };
                // the candidates that were rejected (all), one after the other: their tokens and exponentials
                auto rejected = [&](auto f) {
                    for (int k = at + 1; k < n; k += 64) {
                        const int j = min(k + lane, n - 1), x = d.tok[j];
                        const double e = d.e[j];
                        for (uint64_t m = __ballot(k + lane < n && d.par[j] == at && !d.again[j]); m; m &= m - 1) {
                            const int i = __builtin_ctzll(m);
                            f(__builtin_amdgcn_readlane(x, i), of_lane(e, i));
                        }
                    }
                };
                if (kid < 0) {
                    float m = -INFINITY;
                    by_lanes(0, a.pieces, lane, 64, [&](int k) { m = fmaxf(m, d.most[k]); });
                    m = uni(wave_max(m));
                    if (no_number(m)) break;
                    w.Mp = m;
                    each(a.pieces, [&](int k) { d.weight[k] *= exp64((double)d.most[k] - w.Mp); });
                    __syncthreads();
                } else if (without) {
                    // without the rejected tokens, which are taken off.  A piece of which less than a 16th is left, so
                    // that what is left could be off by more than 2^-48, is summed again without them, by one wave.
                    own_weights();
                    if (tid == 0) listed = 0;
                    __syncthreads();
                    for (int k0 = 0; k0 < a.pieces; k0 += 256) {
                        const int k = min(k0 + tid, a.pieces - 1);
                        const double z = d.weight[k];
                        double y = z;
                        rejected([&](int x, double e) { y -= x / V_PIECE == k ? e : 0.0; });
                        if (k0 + tid < a.pieces) {
                            d.weight[k] = y;
                            if (y < z / 16) d.list[atomicAdd(&listed, 1)] = (uint16_t)k;
                        }
                    }
                    __syncthreads();
                    const int lists = uni(listed);
                    for (int i = wave; i < lists; i += 4) {
                        const int k = uni(d.list[i]);
                        double z = 0.0;
#pragma unroll 1
                        for (int h = 0; h < 4; h++) {
                            float v[1][8];
                            load_stretch<TYPE, 1, 0>(piece_of.row_p(row), k * V_PIECE + h * 512 + lane * 8, (k + 1) * V_PIECE, V, v);
                            uint32_t o = 0;
                            rejected([&](int x, double) {
                                x -= k * V_PIECE + h * 512;
                                o |= x >= 0 && x >> 3 == lane ? 1u << (x & 7) : 0u;
                            });
#pragma unroll
                            for (int e = 0; e < 8; e++) z += o >> e & 1 ? 0.0 : exp64((double)v[0][e] - w.Mp);
                        }
                        z = wave_add(z);
                        if (lane == 0) d.weight[k] = z;
                    }
                    __syncthreads();
                }
                double total = total_of();
                if (kid >= 0 && !sure(total > 0.0)) {  // nothing left: of all that there was
                    of_rest = without = false;
                    own_weights();
                    total = total_of();
                }
                // the piece in which the running sum passes the target, and the sum before it
                const double target = d.u[0] * total;
                double before = 0.0, start = 0.0;
                int piece = -1, last = 0;
                for (int k0 = 0; k0 < a.pieces && piece < 0; k0 += 64) {
                    const double z = k0 + lane < a.pieces ? d.weight[k0 + lane] : 0.0, up = sums_upto(z);
                    const uint64_t past = __ballot(before + up > target && z > 0.0), some = __ballot(z > 0.0);
                    if (some) last = k0 + 63 - __builtin_clzll(some);
                    if (past) {
                        const int k = __builtin_ctzll(past);
                        piece = k0 + k, start = before + of_lane(up - z, k);
                    }
                    before += of_lane(up, 63);
                }
                const bool behind = piece < 0;  // by a rounding: the last token there is
                if (behind) piece = last;
                float v[1][8], q[1][8];
                double z[8], mine = 0.0;
                piece_of.load(piece_of.row_p(row), piece, v);
                if (of_rest) piece_of.load(piece_of.row_q(row), piece, q);
                uint32_t o = 0;
                if (without)
                    rejected([&](int x, double) {
                        x -= piece * V_PIECE;
                        o |= x >= 0 && x >> 3 == tid ? 1u << (x & 7) : 0u;
                    });
                if (of_rest) {
#pragma unroll
                    for (int e = 0; e < 8; e++) z[e] = piece_of.rest(w, v[0][e], q[0][e]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) z[e] = o >> e & 1 ? 0.0 : exp64((double)v[0][e] - w.Mp);
                }
#pragma unroll
                for (int e = 0; e < 8; e++) mine += z[e];
                const double up = sums_upto(mine);
                if (lane == 63) smd[wave] = up;
                __syncthreads();
                double sum = start + (up - mine);
                for (int k = 0; k < wave; k++) sum += smd[k];
                int hit = INT32_MAX, most = -1;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    sum += z[e];
                    if (z[e] > 0.0) {
                        most = piece * V_PIECE + tid * 8 + e;
                        if (sum > target && hit == INT32_MAX) hit = most;
                    }
                }
                const uint64_t past = __ballot(hit != INT32_MAX), some = __ballot(most >= 0);
                if (lane == 0) {
                    hits[wave] = past ? __builtin_amdgcn_readlane(hit, __builtin_ctzll(past)) : INT32_MAX;
                    lasts[wave] = some ? __builtin_amdgcn_readlane(most, 63 - __builtin_clzll(some)) : -1;
                }
                __syncthreads();
                next = min(min(hits[0], hits[1]), min(hits[2], hits[3]));
                if (behind || next == INT32_MAX) next = max(max(lasts[0], lasts[1]), max(lasts[2], lasts[3]));
                next = uni(next);
            }
        }
        if (yes < 0) break;
        at = yes;
        if (tid == 0) d.way[kept] = (int16_t)at;
        kept++;
    }
    __syncthreads();
    if (tid == 0) a.states[s].asks = 0;
    if (none) kept = 0;
    int32_t *out = a.out + (size_t)s * N, *path = a.path + (size_t)s * N;
    each(N, [&](int j) {
        path[j] = j < kept ? d.way[j] : -1;
        out[j] = j + 1 < kept ? d.tok[d.way[j + 1]] : j + 1 == kept ? next : -1;
    });
    if (tid == 0) a.count[s] = kept;
}

template <int TYPE>
__global__ __launch_bounds__(256, 2) void k_verify_walk(VerifyArgs a) {
    __shared__ float smf[4];
    __shared__ double smd[4];
    __shared__ uint64_t two[V_TABLE];
    const int s = blockIdx.x;
    if (threadIdx.x < V_TABLE) exp_table(two, threadIdx.x);
    if (threadIdx.x == 0) a.swept[s] = 0;
    walk<TYPE>(a, s, WalkState{}, Pieces<TYPE>(a, exp_of(factor_of(uni(temperature_of(a, s))), two), smf, smd), true, false);
}

// The sweeps that the walks of the last launch ask for, a block to a piece of a sequence's row, and the walks behind
// them.  Bound by latencies, the state, the rows, two joins, the count and then the walk's own: 11 us of a sweep of 4
// sequences, 28 of one of 32 pairs of rows of 151936 (17.5 alone, and the walk's launch behind it 9).  Four blocks to a
// CU in place of three put 16 registers to scratch: 4 drawn trees 118 us, 82 so.
template <int TYPE>
__global__ __launch_bounds__(256, 3) void k_verify_sweep(VerifyArgs a, bool alone) {
    __shared__ float smf[4];
    __shared__ double smd[4];
    __shared__ uint64_t two[V_TABLE];
    __shared__ int last;
    const int k = blockIdx.x / a.t.n_seqs, s = blockIdx.x - k * a.t.n_seqs;
    const WalkState w = a.states[s];
    if (!uni(w.asks)) return;
    if (threadIdx.x < V_TABLE) exp_table(two, threadIdx.x);
    __syncthreads();
    const Pieces<TYPE> piece_of(a, exp_of(factor_of(uni(temperature_of(a, s))), two), smf, smd);
    double z;
    float m;
    piece_of(w, k, z, m);
    if (threadIdx.x == 0) {
        show(a.swept_sum + (size_t)s * a.pieces + k, z);
        if (w.leaf) show(a.swept_top + (size_t)s * a.pieces + k, m);
        shown();
        last = __hip_atomic_fetch_add(a.swept + s, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.pieces - 1;
        if (last) a.swept[s] = 0;  // for the next launch
    }
    __syncthreads();
    if (uni(last)) walk<TYPE>(a, s, w, piece_of, false, alone);
}

static size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// Where the workspace's parts are; its size.
static size_t verify_layout(VerifyArgs &a, uint8_t *ws) {
    a.chunks = (a.vocab + V_CHUNK - 1) / V_CHUNK, a.pieces = (a.vocab + V_PIECE - 1) / V_PIECE;
    size_t n = 0;
    auto part = [&](auto *&p, size_t count) {
        p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(ws + n);
        n += round256(count * sizeof(*p));
    };
    part(a.sum, (size_t)a.t.n_tokens * 2 * a.pieces);
    part(a.whole, (size_t)a.t.n_tokens * 2 * a.chunks);
    part(a.top, (size_t)a.t.n_tokens * 2 * a.chunks);
    part(a.arg, (size_t)a.t.n_tokens * a.chunks);
    part(a.swept_sum, (size_t)a.t.n_seqs * a.pieces);
    part(a.swept_top, (size_t)a.t.n_seqs * a.pieces);
    part(a.swept, (size_t)a.t.n_seqs);
    part(a.states, (size_t)a.t.n_seqs);
    a.held_bytes = WalkNodes::bytes(a.t.max_nodes, a.pieces);
    part(a.held, (size_t)a.t.n_seqs * a.held_bytes);
    return n;
}

bool verify_fits(const DraftTrees &t, int vocab) {
    return (int64_t)t.n_tokens * ((vocab + V_CHUNK - 1) / V_CHUNK) <= UINT32_MAX / 256 &&
           (int64_t)t.n_seqs * ((vocab + V_PIECE - 1) / V_PIECE) <= UINT32_MAX / 256;
}

static_assert(WalkNodes::bytes(DT_NODES, (1 << 20) / V_PIECE) + 768 <= 65536, "a walk's LDS");

size_t verify_workspace(const DraftTrees &t, int vocab) {
    VerifyArgs a{};
    a.t = t, a.vocab = vocab;
    return verify_layout(a, nullptr);
}

hipError_t launch_verify(VerifyArgs a, int type, void *ws, hipStream_t st) {
    verify_layout(a, static_cast<uint8_t *>(ws));
    const dim3 grid((unsigned)(a.t.n_tokens * a.chunks), a.draft ? 2 : 1);
    // Sweeps: none where all are greedy; one where a walk ends with its first, as every one without a draft model's
    // logits and every chain's does; of trees as many as a walk may have, but V_ROUNDS at the most, the rest by the
    // walk's block alone, which takes a tenth of a ms each.  What 40 calls each need, with siblings drawn from a draft
    // model: 4 trees of 26 nodes 4 in the mean, 9 at the most; one of 26 2 and 6; one of 5 1 and 2; 64 of 16 8 and 9;
    // 16 of 64 9 and 13, one more than there are launches in 4 of the 40.  An idle launch takes 1.7 us: the first of
    // these would take 60 us with 4 where those are enough, and takes 66 to 90, by its inputs, with 12.
    const int rounds = !grid.x || (!a.temps && !(a.temp > 0.0f)) ? 0 : !a.draft || !a.t.parent ? 1 : std::min(V_ROUNDS, a.t.max_nodes);
    auto launch = [&](auto T) {
        constexpr int TYPE = decltype(T)::value;
        const size_t lds = WalkNodes::bytes(a.t.max_nodes, a.pieces);
        if (grid.x) TG_LAUNCH(k_verify_rows<TYPE>, grid, dim3(256), 0, st, a);
        TG_LAUNCH(k_verify_walk<TYPE>, dim3((unsigned)a.t.n_seqs), dim3(256), lds, st, a);
        for (int i = 1; i <= rounds; i++) TG_LAUNCH(k_verify_sweep<TYPE>, dim3((unsigned)(a.t.n_seqs * a.pieces)), dim3(256), lds, st, a, i == rounds);
    };
    if (type == TG_T_F32) launch(std::integral_constant<int, TG_T_F32>{});
    else if (type == TG_T_F16) launch(std::integral_constant<int, TG_T_F16>{});
    else launch(std::integral_constant<int, TG_T_BF16>{});
    return hipGetLastError();
}

}  // namespace tg
