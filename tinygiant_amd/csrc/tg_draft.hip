// tg_draft.hip -- trees of drafted tokens on the device: which nodes each one
// sees and how deep it stands, and which of the drafts a target's
// probabilities keep.
//
// Node j of a sequence is row cu[s] + j of the batch; its parent is a node
// before it, so a walk towards the root only goes down in j.
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

// A block per sequence, a thread per node, which walks to its root through the parents in LDS and sets the bits of what it
// meets, one word after the other.  Bound by latency: the rows' bounds, the parents, then a read of LDS a step, 1 us for
// trees of ordinary depth.
__global__ __launch_bounds__(256) void k_draft_tree(DraftTrees t, uint32_t *bits, int32_t *depth) {
    __shared__ int16_t par[DT_NODES];
    const TreeRows r = tree_rows(t, blockIdx.x);
    const int n = min(r.n, t.max_nodes), words = (t.max_nodes + 31) / 32;
    for (int j = threadIdx.x; j < n; j += 256) par[j] = (int16_t)parent_of(t, r.lo, j);
    __syncthreads();
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
    }
}

hipError_t launch_draft_tree(const DraftTrees &t, uint32_t *bits, int32_t *depth, hipStream_t st) {
    TG_LAUNCH(k_draft_tree, dim3((unsigned)t.n_seqs), dim3(256), 0, st, t, bits, depth);
    return hipGetLastError();
}

// ================================================================ verification
// One sequence's walk.  At a node, p = softmax(target's logits / T) and q the same of the draft's.  Its children x were
// drawn from q, one after the other: x stays with probability r(x) / q(x) at the most 1, where r = p for the first, and
// each one that does not stay leaves max(r - q, 0) / its sum for the next, so that whichever stays, or the token that is
// drawn of what is left in the end, is distributed as p.  In closed form r = max(p - c q, 0) / Z with c = 0, Z = 1 at
// first; one that does not stay makes c + Z of c, and Z the sum of max(p - c q, 0) for the new c: one number is kept of all
// that were asked.  Without q the children are candidates that no one drew, kept with probability p(x) / (1 - what those
// before them had), and what is left is p without them.
//
// Whatever a random number decides is decided in 64 bits: probabilities, their sums and running sums.
constexpr int V_CHUNK = 8192;  // values of a row to a block of the first launch
constexpr int V_PIECE = 2048;  // ... whose sum is kept
constexpr int V_PER = V_CHUNK / V_PIECE;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int TYPE>
TG_DEV float load1(const void *p, int64_t i) {
    if constexpr (TYPE == TG_T_F32) return static_cast<const float *>(p)[i];
    const uint16_t v = static_cast<const uint16_t *>(p)[i];
    return TYPE == TG_T_F16 ? h2f(v) : __uint_as_float((uint32_t)v << 16);
}
// 8 values of a row from i on, -inf behind its end.  Rows of any alignment: global loads of 16 bytes need that of their elements.
template <int TYPE>
TG_DEV void load8(const void *row, int i, int V, float v[8]) {
    if (i + 8 <= V) {
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
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = i + e < V ? load1<TYPE>(row, i + e) : -INFINITY;
    }
}
template <int TYPE>
TG_DEV const void *row_of(const void *p, int64_t stride, int row) {
    return static_cast<const uint8_t *>(p) + (int64_t)row * stride * (TYPE == TG_T_F32 ? 4 : 2);
}

// Exponentials of what is 0 or below, to some 2^-50: exp(d / T) = 2^(y / 32), y = d 32 log2(e) / T, by the nearest whole
// number n of y from a table of 2^(j / 32) and the power of 2, and the rest f, at most 1/2, by the Taylor polynomial of
// 2^(f / 32) of degree 6 (what it leaves out is below 2^-57).  Below 2^-1021 the result is 0.  14 operations on doubles; without the
// table, by the remainder of ln 2 and degree 13, 26.
constexpr int V_TABLE = 32;
struct Exp64 {
    double by;          // 32 log2(e) / T
    const double *two;  // 2^(j / 32)
    TG_DEV double operator()(double d) const {
        const double y = d * by, t = y + 6755399441055744.0, f = y - (t - 6755399441055744.0);  // 1.5 2^52: its unit is 1
        const int n = (int)__builtin_bit_cast(uint64_t, t);
        double p = 1.4345655584131934e-13;  // (ln 2 / 32)^i / i!
        p = __builtin_fma(p, f, 3.973709984549416e-11);
        p = __builtin_fma(p, f, 9.172562701824643e-09);
        p = __builtin_fma(p, f, 1.693850972437182e-06);
        p = __builtin_fma(p, f, 0.0002345961982022468);
        p = __builtin_fma(p, f, 0.02166084939249829);
        p = __builtin_fma(p, f, 1.0);
        const uint64_t w = __builtin_bit_cast(uint64_t, two[n & (V_TABLE - 1)]) + ((uint64_t)(uint32_t)(n >> 5) << 52);
        const double r = __builtin_bit_cast(double, w) * p;
        return y > -32.0 * 1021.0 ? r : 0.0;
    }
};
// the table, by repeated square roots of 2: 2^(j / 32) is the product of those of j's bits
TG_DEV void exp_table(double *two, int j) {
    double r = 1.0;
    if (j & 16) r *= 1.4142135623730951;
    if (j & 8) r *= 1.189207115002721;
    if (j & 4) r *= 1.0905077326652577;
    if (j & 2) r *= 1.0442737824274138;
    if (j & 1) r *= 1.0218971486541166;
    two[j] = r;
}

// the sequence's temperature; 32 log2(e) / T, so that -inf times it stays -inf
TG_DEV float temperature_of(const VerifyArgs &a, int s) { return a.temps ? a.temps[s] : a.temp; }
TG_DEV double factor_of(float t) { return fmax(46.16624130844683 / (double)t, 1e-300); }

TG_DEV float uni(float v) { return __int_as_float(uni(__float_as_int(v))); }
// what is true or not in all lanes of a wave, told to the compiler
TG_DEV bool sure(bool c) { return __ballot(c) != 0; }

template <class T>
TG_DEV T wave_max(T v) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const T o = __shfl_xor(v, m);
        v = v > o ? v : o;
    }
    return v;
}
template <class T>
TG_DEV T wave_add(T v) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m);
    return v;
}
// inclusive sums over the lanes
TG_DEV double wave_upto(double v, int lane) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const double o = __shfl_up(v, m);
        if (lane >= m) v += o;
    }
    return v;
}
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
// or +inf: the largest is +inf.  The first blocks also clear what the walks' blocks meet by.
template <int TYPE>
__global__ __launch_bounds__(256) void k_verify_rows(VerifyArgs a) {
    __shared__ float sm[4];
    __shared__ double smd[4][V_PER], two[V_TABLE];
    __shared__ int first;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks, of = blockIdx.y;
    const void *p = of ? row_of<TYPE>(a.draft, a.draft_stride, row) : row_of<TYPE>(a.logits, a.stride, row);
    float v[V_PER][8], m = -INFINITY;
    auto load = [&]() {
#pragma unroll
        for (int k = 0; k < V_PER; k++) load8<TYPE>(p, chunk * V_CHUNK + k * V_PIECE + threadIdx.x * 8, a.vocab, v[k]);
    };
    if (a.early) load();
    if (!of)
        for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < a.meet_words; i += (size_t)gridDim.x * 256) a.meet[i] = 0;
    if (threadIdx.x < V_TABLE) exp_table(two, threadIdx.x);
    int s = 0;
    for (int j = lane; j < a.t.n_seqs; j += 64) s += a.t.cu[j + 1] <= row;
    s = uni(wave_add(s));
    if (s >= a.t.n_seqs) return;
    const TreeRows r = tree_rows(a.t, s);
    const float t = uni(temperature_of(a, s));
    const int node = row - r.lo, n = min(r.n, a.t.max_nodes);
    if (node < 0 || node >= n) return;
    const bool greedy = !(t > 0.0f);
    if (greedy) {
        if (of) return;
    } else {
        bool kid = false;
        for (int j = node + 1 + lane; j < n; j += 64) kid |= parent_of(a.t, r.lo, j) == node;
        if (!__ballot(kid)) return;
    }
    if (!a.early) load();
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
    const Exp64 exp64{factor_of(t), two};
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
        static_assert(V_PER == 4, "");
        z += __shfl_xor(z, 1);
        z += __shfl_xor(z, 2);
        if (k == 0) a.whole[at_row * a.chunks + chunk] = z;
    }
}

// What a walk asks of all the pieces of a row at once
struct Sweep {
    uint64_t row;           // times 2; + 1: sums of max(p - c q, 0); else of exp((v - largest) / T), each piece by itself
    double Mp, ip, Mq, iq;  // p = exp((v - Mp) / T) ip, c q likewise
};
// How the blocks of one sequence's walk meet: the first to begin leads, the others help with its sweeps.  The leader
// writes what a sweep is, then its number to `number`; every block that sees it (the leader too) takes pieces from its
// counter until there are none, and counts those it has done.  Only the leader waits for something that others do, and only for
// pieces that running blocks have taken; helpers wait for the leader, which runs.  So a walk ends however few of its blocks the
// device runs at a time.
struct Meeting {
    uint32_t ticket, number;
    Sweep sweep;
    uint32_t taken_done[];  // [max_nodes + 2][2]
};
constexpr uint32_t V_END = ~0u;
// What blocks hand to each other goes past the caches of an XCD, and what is to be seen first is waited for (a release at
// the device's scope writes back a whole L2).
template <class T>
TG_DEV T seen_now(const T *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <class T>
TG_DEV void show(T *p, T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
TG_DEV void shown() { __builtin_amdgcn_s_waitcnt(0x0F70); }  // vmcnt 0: this thread's stores are acknowledged

template <int TYPE>
struct Walk {
    const VerifyArgs &a;
    int helpers;
    Exp64 exp64;
    Meeting *meet;
    float *top;   // of a sweep's pieces: the largest value of each
    double *sum;  // ... the sums
    float *smf;
    double *smd;
    uint32_t *smu;

    // piece k of a sweep, by one block
    TG_DEV void piece(const Sweep &w, int k) {
        const int row = uni((int)(w.row >> 1));
        const void *pr = row_of<TYPE>(a.logits, a.stride, row);
        float v[8], q[8];
        load8<TYPE>(pr, k * V_PIECE + threadIdx.x * 8, a.vocab, v);
        double z = 0.0;
        if (uni((int)w.row & 1)) {
            load8<TYPE>(row_of<TYPE>(a.draft, a.draft_stride, row), k * V_PIECE + threadIdx.x * 8, a.vocab, q);
#pragma unroll
            for (int e = 0; e < 8; e++) z += rest(w, v[e], q[e]);
        } else {
            float m = -INFINITY;
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                bad |= !(v[e] < INFINITY);
                m = fmaxf(m, v[e]);
            }
            m = block_max(bad ? INFINITY : m, smf);
            if (m > -INFINITY && m < INFINITY)
#pragma unroll
                for (int e = 0; e < 8; e++) z += exp64((double)v[e] - m);
            if (threadIdx.x == 0) show(top + k, m);
        }
        z = block_add(z, smd);
        if (threadIdx.x == 0) show(sum + k, z);
    }
    TG_DEV double rest(const Sweep &w, float v, float q) const {
        return fmax(exp64((double)v - w.Mp) * w.ip - exp64((double)q - w.Mq) * w.iq, 0.0);
    }
    // takes pieces of sweep `number` until there are none
    TG_DEV void take(const Sweep &w, uint32_t number) {
        uint32_t *taken = meet->taken_done + 2 * number;
        for (;;) {
            __syncthreads();
            if (threadIdx.x == 0) *smu = __hip_atomic_fetch_add(taken, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            const uint32_t k = uni((int)*smu);
            if (k >= (uint32_t)a.pieces) return;
            piece(w, (int)k);
            if (threadIdx.x == 0) {
                shown();
                __hip_atomic_fetch_add(taken + 1, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
    }
    TG_DEV void help() {
        for (uint32_t number = 0;;) {
            __syncthreads();
            if (threadIdx.x == 0) {
                uint32_t now;
                while ((now = seen_now(&meet->number)) == number) __builtin_amdgcn_s_sleep(4);
                *smu = now;
            }
            __syncthreads();
            number = uni((int)*smu);
            if (number == V_END) return;
            // this sweep's as long as pieces of it can be taken: a later one's is not worked on
            const Sweep w{seen_now(&meet->sweep.row), seen_now(&meet->sweep.Mp), seen_now(&meet->sweep.ip), seen_now(&meet->sweep.Mq),
                          seen_now(&meet->sweep.iq)};
            take(w, number);
        }
    }
    // the leader's: a whole sweep
    TG_DEV void lead(const Sweep &w, uint32_t number) {
        __syncthreads();
        if (!helpers) {
            for (int k = 0; k < a.pieces; k++) piece(w, k);
            shown();
            __syncthreads();
            return;
        }
        if (threadIdx.x == 0) {
            show(&meet->sweep.row, w.row), show(&meet->sweep.Mp, w.Mp), show(&meet->sweep.ip, w.ip);
            show(&meet->sweep.Mq, w.Mq), show(&meet->sweep.iq, w.iq);
            shown();
            show(&meet->number, number);
        }
        take(w, number);
        if (threadIdx.x == 0)
            while (seen_now(meet->taken_done + 2 * number + 1) != (uint32_t)a.pieces) __builtin_amdgcn_s_sleep(1);
        __syncthreads();
    }
};

// LDS of a walk, for `nodes` of them
struct WalkNodes {
    double *u, *sum[2];    // random numbers; the rows' sums of exponentials, target's and draft's
    float *x[2], *top[2];  // the nodes' logits at their parents; the rows' largest values
    int *tok;
    int16_t *par, *way;
    uint8_t *kids;
    TG_DEV WalkNodes(uint8_t *lds, int nodes) {
        u = reinterpret_cast<double *>(lds), sum[0] = u + nodes, sum[1] = sum[0] + nodes;
        x[0] = reinterpret_cast<float *>(sum[1] + nodes), x[1] = x[0] + nodes, top[0] = x[1] + nodes, top[1] = top[0] + nodes;
        tok = reinterpret_cast<int *>(top[1] + nodes);
        par = reinterpret_cast<int16_t *>(tok + nodes), way = par + nodes;
        kids = reinterpret_cast<uint8_t *>(way + nodes);
    }
    static size_t bytes(int nodes) { return (size_t)nodes * (3 * 8 + 5 * 4 + 2 * 2 + 1); }
};

// A sequence's walk: one block leads, the others help with sums over whole rows.  What decides where the leader goes is the
// same in all of its lanes, and told so to the compiler (uni, sure): with branches by lanes, what it moved between registers behind
// a loop was moved with all lanes off, and lost (rejected tokens of some waves were drawn).
template <int TYPE>
__global__ __launch_bounds__(256, 3) void k_verify_walk(VerifyArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ double smd[4], two[V_TABLE];
    __shared__ float smf[4];
    __shared__ uint32_t gone[4][V_PIECE / 32];  // a wave's: tokens of a piece that were rejected
    __shared__ uint32_t smu;
    __shared__ int found;
    const int tid = threadIdx.x, lane = tid % 64, wave = uni(tid / 64), s = blockIdx.x % a.t.n_seqs, V = a.vocab;
    const float t = uni(temperature_of(a, s));
    const bool greedy = !(t > 0.0f), with_q = a.draft && !greedy;
    if (tid < V_TABLE) exp_table(two, tid);
    const Exp64 exp64{factor_of(t), two};
    Walk<TYPE> walk{a, a.team - 1, exp64, reinterpret_cast<Meeting *>(a.meet + s * (a.meet_words / a.t.n_seqs)),
                    a.swept_top + (size_t)s * a.pieces, a.swept_sum + (size_t)s * a.pieces, smf, smd, &smu};
    if (a.team > 1) {
        if (tid == 0) smu = __hip_atomic_fetch_add(&walk.meet->ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (uni((int)smu)) {
            walk.help();
            return;
        }
    }
    const TreeRows r = tree_rows(a.t, s);
    const int n = uni(min(r.n, a.t.max_nodes)), lo = uni(r.lo);
    const WalkNodes d(lds, a.t.max_nodes);
    for (int j = tid; j < n; j += 256) d.kids[j] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += 256) {
        const int p = parent_of(a.t, lo, j), x = a.tokens[lo + j];
        const bool ok = p >= 0 && x >= 0 && x < V;
        if (p >= 0) d.kids[p] = 1;
        d.par[j] = (int16_t)p, d.tok[j] = x, d.u[j] = a.u[lo + j];
        d.x[0][j] = ok ? load1<TYPE>(row_of<TYPE>(a.logits, a.stride, lo + p), x) : -INFINITY;
        d.x[1][j] = ok && with_q ? load1<TYPE>(row_of<TYPE>(a.draft, a.draft_stride, lo + p), x) : -INFINITY;
    }
    __syncthreads();
    // the next child of `node` behind j, or -1: the same in every wave, like all that follows
    auto child = [&](int node, int j) {
        for (int k = j + 1; k < n; k += 64) {
            const uint64_t m = __ballot(k + lane < n && d.par[k + lane < n ? k + lane : 0] == node);
            if (m) return k + __builtin_ctzll(m);
        }
        return -1;
    };
    // is there a child of `node` before j whose token `same` takes for j's
    auto earlier = [&](int node, int j, auto same) {
        for (int k = node + 1; k < j; k += 64)
            if (__ballot(k + lane < j && d.par[k + lane < j ? k + lane : 0] == node && same(d.tok[k + lane < j ? k + lane : 0]))) return true;
        return false;
    };
    // Largest values and sums of the rows of nodes j0 .. j0 + 63, from those of their chunks: half a wave to a row.  For a
    // greedy sequence the first of the largest stands in the place of the draft's logits.
    auto join = [&](int j0) {
        const int each = with_q ? 2 : 1, units = min(n - j0, 64) * each, l = lane % 32;
        for (int i = tid / 32; i < units; i += 8) {
            const int j = j0 + i / each, of = i % each;
            if (!greedy && !d.kids[j]) continue;
            const size_t at = ((size_t)(lo + j) * 2 + of) * a.chunks;
            float m = -INFINITY;
            for (int k = l; k < a.chunks; k += 32) m = fmaxf(m, a.top[at + k]);
#pragma unroll
            for (int k = 1; k < 32; k *= 2) m = fmaxf(m, __shfl_xor(m, k));
            if (l == 0) d.top[of][j] = m;
            if (m == INFINITY || m == -INFINITY) continue;
            if (greedy) {
                int best = INT32_MAX;
                for (int k = l; k < a.chunks; k += 32)
                    if (a.top[at + k] == m) best = min(best, a.arg[(size_t)(lo + j) * a.chunks + k]);
#pragma unroll
                for (int k = 1; k < 32; k *= 2) best = min(best, __shfl_xor(best, k));
                if (l == 0) d.x[1][j] = __int_as_float(best);
            } else {
                double z = 0.0;
                for (int k = l; k < a.chunks; k += 32) z += a.whole[at + k] * exp64((double)a.top[at + k] - m);
#pragma unroll
                for (int k = 1; k < 32; k *= 2) z += __shfl_xor(z, k);
                if (l == 0) d.sum[of][j] = z;
            }
        }
        __syncthreads();
    };
    auto swept = [&]() {  // the sum over a sweep's pieces
        double z = 0.0;
        for (int k = lane; k < a.pieces; k += 64) z += seen_now(walk.sum + k);
        return wave_add(z);
    };
    auto no_number = [](float m) { return m == INFINITY || m == -INFINITY; };

    int at = 0, kept = 1, next = -1, joined = 0;
    uint32_t sweeps = 0;
    if (tid == 0) d.way[0] = 0;
    while (n) {
        const int row = lo + at, kid = child(at, at);  // all of these are the same in every lane
        int yes = -1;
        if (at >= joined) {
            join(at);
            joined = at + 64;
        }
        if (greedy) {
            if (no_number(uni(d.top[0][at]))) break;
            const int best = uni(__float_as_int(d.x[1][at]));
            for (int k = kid; k >= 0 && yes < 0; k = child(at, k))
                if (uni(d.tok[k]) == best) yes = k;
            if (yes < 0) next = best;
        } else {
            double Mp = 0, Zp = 1, Mq = 0, Zq = 1, c = 0;
            if (kid >= 0) {
                Mp = d.top[0][at], Zp = d.sum[0][at];
                if (with_q) Mq = d.top[1][at], Zq = d.sum[1][at];
                if (no_number(uni((float)Mp)) || no_number(uni((float)Mq))) break;
                double left = 1.0;
                for (int k = kid, after; k >= 0; k = after) {
                    after = child(at, k);
                    double px = exp64((double)d.x[0][k] - Mp) / Zp;
                    if (with_q) {
                        const double qx = exp64((double)d.x[1][k] - Mq) / Zq;
                        if (sure(d.u[k] * left * qx < px - c * qx)) {
                            yes = k;
                            break;
                        }
                        c += left;
                        if (after >= 0) {
                            walk.lead({2 * (uint64_t)row + 1, Mp, 1.0 / Zp, Mq, c / Zq}, ++sweeps);
                            left = swept();
                        }
                    } else {
                        if (earlier(at, k, [&](int x) { return x == d.tok[k]; })) px = 0.0;  // rejected already
                        if (sure(px > 0.0 && d.u[k] * left < px)) {
                            yes = k;
                            break;
                        }
                        left -= px;
                    }
                }
            }
            if (yes < 0) {
                if (!sure(d.u[0] >= 0.0 && d.u[0] < 1.0)) break;
                // weights of the pieces of what is left: a sweep's sums, or those times exp((largest - M) / T)
                Sweep w{2 * (uint64_t)row, Mp, 1.0 / Zp, Mq, c / Zq};
                bool of_rest = with_q && kid >= 0;
                if (of_rest) {
                    w.row++;
                    walk.lead(w, ++sweeps);
                    of_rest = sure(swept() > 0.0);  // nothing: of all that there was
                } else if (kid < 0) {
                    walk.lead(w, ++sweeps);
                    float m = -INFINITY;
                    for (int k = lane; k < a.pieces; k += 64) m = fmaxf(m, seen_now(walk.top + k));
                    m = uni(wave_max(m));
                    if (no_number(m)) break;
                    w.Mp = m;
                }
                // the row's own sums, and of pieces that hold rejected tokens those without them
                const bool own = kid >= 0 && !of_rest;
                const double *own_sum = a.sum + (size_t)row * 2 * a.pieces;
                const float *own_top = a.top + (size_t)row * 2 * a.chunks;
                double *less = a.own_sum + (size_t)s * a.pieces;
                // piece k's rejected tokens as bits of the wave's `gone`
                auto mark = [&](int k) {
                    wave_lds_sync();
                    gone[wave][lane] = 0;
                    wave_lds_sync();
                    for (int j = at + 1 + lane; j < n; j += 64) {
                        const int x = d.tok[j] - k * V_PIECE;
                        if (d.par[j] == at && x >= 0 && x < V_PIECE) atomicOr(&gone[wave][x / 32], 1u << (x % 32));
                    }
                    wave_lds_sync();
                };
                const void *pr = row_of<TYPE>(a.logits, a.stride, row);
                bool without = !with_q && kid >= 0;
                if (without) {
                    for (int k = tid; k < a.pieces; k += 256) less[k] = own_sum[k];
                    __syncthreads();
                    // pieces that hold rejected tokens again, without those: each of them by one wave
                    int i = 0;
                    for (int j = kid; j >= 0; j = child(at, j)) {
                        const int x = uni(d.tok[j]), k = x / V_PIECE;
                        if (x < 0 || x >= V || earlier(at, j, [&](int y) { return y >= 0 && y / V_PIECE == k; })) continue;
                        if (i++ % 4 != wave) continue;
                        float v[4][8];
#pragma unroll
                        for (int h = 0; h < 4; h++) load8<TYPE>(pr, k * V_PIECE + h * 512 + lane * 8, V, v[h]);
                        mark(k);
                        double z = 0.0;
                        const double m = own_top[k / V_PER];
#pragma unroll
                        for (int h = 0; h < 4; h++) {
                            const uint32_t o = gone[wave][h * 16 + lane / 4] >> (8 * (lane % 4));
#pragma unroll
                            for (int e = 0; e < 8; e++) z += o >> e & 1 ? 0.0 : exp64((double)v[h][e] - m);
                        }
                        z = wave_add(z);
                        if (lane == 0) less[k] = z;
                    }
                    __syncthreads();
                }
                auto weight_of = [&](int k) {
                    if (own) return (without ? less : own_sum)[k] * exp64((double)own_top[k / V_PER] - w.Mp);
                    const double z = seen_now(walk.sum + k);
                    return of_rest ? z : z * exp64((double)seen_now(walk.top + k) - w.Mp);
                };
                auto all = [&]() {
                    double z = 0.0;
                    for (int k = lane; k < a.pieces; k += 64) z += weight_of(k);
                    return wave_add(z);
                };
                double total = all();
                if (without && !sure(total > 0.0)) {  // nothing left: of all that there was
                    without = false;
                    total = all();
                }
                // the piece in which the running sum passes the target, and the sum before it
                const double target = d.u[0] * total;
                double before = 0.0, start = 0.0;
                int piece = -1, last = 0;
                for (int k0 = 0; k0 < a.pieces && piece < 0; k0 += 64) {
                    const double z = k0 + lane < a.pieces ? weight_of(k0 + lane) : 0.0, up = wave_upto(z, lane);
                    const uint64_t past = __ballot(before + up > target && z > 0.0), some = __ballot(z > 0.0);
                    if (some) last = k0 + 63 - __builtin_clzll(some);
                    if (past) {
                        const int k = __builtin_ctzll(past);
                        piece = k0 + k, start = before + __shfl(up - z, k);
                    }
                    before += __shfl(up, 63);
                }
                const bool behind = piece < 0;  // by a rounding: the last token there is
                if (behind) piece = last;
                float v[8], q[8];
                double z[8], mine = 0.0;
                load8<TYPE>(pr, piece * V_PIECE + tid * 8, V, v);
                if (of_rest) load8<TYPE>(row_of<TYPE>(a.draft, a.draft_stride, row), piece * V_PIECE + tid * 8, V, q);
                uint32_t o = 0;
                if (without) {
                    mark(piece);
                    o = gone[wave][tid / 4] >> (8 * (tid % 4));
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    z[e] = o >> e & 1 ? 0.0 : of_rest ? walk.rest(w, v[e], q[e]) : exp64((double)v[e] - w.Mp);
                    mine += z[e];
                }
                const double up = wave_upto(mine, lane);
                __syncthreads();
                if (lane == 63) smd[wave] = up;
                if (tid == 0) found = INT32_MAX;
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
                if (hit != INT32_MAX && !behind) atomicMin(&found, hit);
                __syncthreads();
                next = uni(found);
                if (next == INT32_MAX) {
                    __syncthreads();
                    if (tid == 0) found = -1;
                    __syncthreads();
                    if (most >= 0) atomicMax(&found, most);
                    __syncthreads();
                    next = uni(found);
                }
            }
        }
        if (yes < 0) break;
        at = yes;
        if (tid == 0) d.way[kept] = (int16_t)at;
        kept++;
    }
    __syncthreads();
    if (a.team > 1 && tid == 0) show(&walk.meet->number, V_END);
    if (!n) kept = 0;
    int32_t *out = a.out + (size_t)s * a.t.max_nodes, *path = a.path + (size_t)s * a.t.max_nodes;
    for (int j = tid; j < a.t.max_nodes; j += 256) {
        path[j] = j < kept ? d.way[j] : -1;
        out[j] = j + 1 < kept ? d.tok[d.way[j + 1]] : j + 1 == kept ? next : -1;
    }
    if (tid == 0) a.count[s] = kept;
}

static size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// Where the workspace's parts are; its size.
static size_t verify_layout(VerifyArgs &a, uint8_t *ws) {
    a.chunks = (a.vocab + V_CHUNK - 1) / V_CHUNK, a.pieces = (a.vocab + V_PIECE - 1) / V_PIECE;
    // 8-byte aligned words of one sequence
    a.meet_words = (sizeof(Meeting) / 4 + 2 * (a.t.max_nodes + 2) + 1) / 2 * 2 * (size_t)a.t.n_seqs;
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
    part(a.own_sum, (size_t)a.t.n_seqs * a.pieces);
    part(a.swept_top, (size_t)a.t.n_seqs * a.pieces);
    part(a.meet, a.meet_words);
    return n;
}

bool verify_fits(const DraftTrees &t, int vocab) {
    return (int64_t)t.n_tokens * ((vocab + V_CHUNK - 1) / V_CHUNK) <= UINT32_MAX / 256;
}

size_t verify_workspace(const DraftTrees &t, int vocab) {
    VerifyArgs a{};
    a.t = t, a.vocab = vocab;
    return verify_layout(a, nullptr);
}

hipError_t launch_verify(VerifyArgs a, int type, void *ws, hipStream_t st) {
    verify_layout(a, static_cast<uint8_t *>(ws));
    const dim3 grid((unsigned)(a.t.n_tokens * a.chunks), a.draft ? 2 : 1);
    // blocks to a walk: as many as the row has pieces, but what the device holds at once for all walks at the most; one
    // where nothing is swept
    a.team = grid.x && (a.temps || a.temp > 0.0f) ? std::max(1, std::min(a.pieces, 768 / a.t.n_seqs)) : 1;
    a.early = grid.x * grid.y <= 1024;
    auto launch = [&](auto T) {
        constexpr int TYPE = decltype(T)::value;
        if (grid.x) TG_LAUNCH(k_verify_rows<TYPE>, grid, dim3(256), 0, st, a);
        TG_LAUNCH(k_verify_walk<TYPE>, dim3((unsigned)(a.t.n_seqs * a.team)), dim3(256), WalkNodes::bytes(a.t.max_nodes), st, a);
    };
    if (type == TG_T_F32) launch(std::integral_constant<int, TG_T_F32>{});
    else if (type == TG_T_F16) launch(std::integral_constant<int, TG_T_F16>{});
    else launch(std::integral_constant<int, TG_T_BF16>{});
    return hipGetLastError();
}

}  // namespace tg
