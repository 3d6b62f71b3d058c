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

// exp(x) for x <= 0: x = n ln 2 + r, |r| <= ln 2 / 2, the Taylor polynomial of degree 13 (its rest is below 2^-57), times
// 2^n.  Below -745 it is 0, as the result would be.
TG_DEV double exp64(double x) {
    x = x < -800.0 ? -800.0 : x;
    const double n = __builtin_rint(x * 1.4426950408889634);
    double r = __builtin_fma(n, -0.6931471805599453, x);  // ln 2, and what its double leaves out
    r = __builtin_fma(n, -2.3190468138462996e-17, r);
    double p = 1.0 / 6227020800.0;
    p = __builtin_fma(p, r, 1.0 / 479001600.0);
    p = __builtin_fma(p, r, 1.0 / 39916800.0);
    p = __builtin_fma(p, r, 1.0 / 3628800.0);
    p = __builtin_fma(p, r, 1.0 / 362880.0);
    p = __builtin_fma(p, r, 1.0 / 40320.0);
    p = __builtin_fma(p, r, 1.0 / 5040.0);
    p = __builtin_fma(p, r, 1.0 / 720.0);
    p = __builtin_fma(p, r, 1.0 / 120.0);
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_ldexp(p, (int)n);
}

// the sequence's temperature; 1 / T, so that -inf times it stays -inf
TG_DEV float temperature_of(const VerifyArgs &a, int s) { return a.temps ? a.temps[s] : a.temp; }
TG_DEV double inverse_of(float t) { return fmax(1.0 / (double)t, 1e-300); }

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
// all), and of its pieces the sums of exp((v - largest) / T), or the place of the first of the largest.  NaN or +inf:
// the largest is +inf.  The first blocks also clear what the walks' blocks meet by.
template <int TYPE>
__global__ __launch_bounds__(256) void k_verify_rows(VerifyArgs a) {
    __shared__ float sm[4];
    __shared__ double smd[4][V_PER];
    __shared__ int first;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks, of = blockIdx.y;
    if (!of)
        for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < a.meet_words; i += (size_t)gridDim.x * 256) a.meet[i] = 0;
    int s = 0;
    for (int j = lane; j < a.t.n_seqs; j += 64) s += a.t.cu[j + 1] <= row;
    s = wave_add(s);
    if (s >= a.t.n_seqs) return;
    const TreeRows r = tree_rows(a.t, s);
    const int node = row - r.lo, n = min(r.n, a.t.max_nodes);
    if (node < 0 || node >= n) return;
    const float t = temperature_of(a, s);
    const bool greedy = !(t > 0.0f);
    if (greedy) {
        if (of) return;
    } else {
        bool kid = false;
        for (int j = node + 1 + lane; j < n; j += 64) kid |= parent_of(a.t, r.lo, j) == node;
        if (!__ballot(kid)) return;
    }
    const void *p = of ? row_of<TYPE>(a.draft, a.draft_stride, row) : row_of<TYPE>(a.logits, a.stride, row);
    float v[V_PER][8], m = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int k = 0; k < V_PER; k++) load8<TYPE>(p, chunk * V_CHUNK + k * V_PIECE + threadIdx.x * 8, a.vocab, v[k]);
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
    const double inv = inverse_of(t);
#pragma unroll
    for (int k = 0; k < V_PER; k++) {
        double sum = 0.0;
        if (m > -INFINITY)
#pragma unroll
            for (int e = 0; e < 8; e++) sum += exp64(((double)v[k][e] - m) * inv);
        sum = wave_add(sum);
        if (lane == 0) smd[wave][k] = sum;
    }
    __syncthreads();
    if (threadIdx.x < V_PER && chunk * V_PER + (int)threadIdx.x < a.pieces) {
        const int k = threadIdx.x;
        a.sum[at_row * a.pieces + chunk * V_PER + k] = ((smd[0][k] + smd[1][k]) + smd[2][k]) + smd[3][k];
    }
}

// What a walk asks of all the pieces of a row at once
struct Sweep {
    int of_rest;  // sums of max(p - c q, 0); else of exp((v - largest) / T), each piece by itself
    int row;
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
TG_DEV uint32_t seen_now(const uint32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

template <int TYPE>
struct Walk {
    const VerifyArgs &a;
    int s, helpers;
    double inv;
    Meeting *meet;
    float *top;   // of a sweep's pieces: the largest value of each
    double *sum;  // ... the sums
    float *smf;
    double *smd;
    uint32_t *smu;

    // piece k of a sweep, by one block
    TG_DEV void piece(const Sweep &w, int k) {
        const void *pr = row_of<TYPE>(a.logits, a.stride, w.row);
        float v[8], q[8];
        load8<TYPE>(pr, k * V_PIECE + threadIdx.x * 8, a.vocab, v);
        double z = 0.0;
        if (w.of_rest) {
            load8<TYPE>(row_of<TYPE>(a.draft, a.draft_stride, w.row), k * V_PIECE + threadIdx.x * 8, a.vocab, q);
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
                for (int e = 0; e < 8; e++) z += exp64(((double)v[e] - m) * inv);
            if (threadIdx.x == 0) top[k] = m;
        }
        z = block_add(z, smd);
        if (threadIdx.x == 0) sum[k] = z;
    }
    TG_DEV double rest(const Sweep &w, float v, float q) const {
        return fmax(exp64(((double)v - w.Mp) * inv) * w.ip - exp64(((double)q - w.Mq) * inv) * w.iq, 0.0);
    }
    // takes pieces of sweep `number` until there are none
    TG_DEV void take(uint32_t number) {
        uint32_t *taken = meet->taken_done + 2 * number;
        for (;;) {
            __syncthreads();
            if (threadIdx.x == 0) *smu = __hip_atomic_fetch_add(taken, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            const uint32_t k = *smu;
            if (k >= (uint32_t)a.pieces) return;
            const Sweep w = meet->sweep;  // this sweep's, as long as a piece of it is not done
            piece(w, (int)k);
            if (threadIdx.x == 0) __hip_atomic_fetch_add(taken + 1, 1u, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    TG_DEV void help() {
        for (uint32_t number = 0;;) {
            __syncthreads();
            if (threadIdx.x == 0) {
                uint32_t now;
                while ((now = seen_now(&meet->number)) == number) __builtin_amdgcn_s_sleep(8);
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
                *smu = now;
            }
            __syncthreads();
            number = *smu;
            if (number == V_END) return;
            take(number);
        }
    }
    // the leader's: a whole sweep
    TG_DEV void lead(const Sweep &w, uint32_t number) {
        __syncthreads();
        if (!helpers) {
            for (int k = 0; k < a.pieces; k++) piece(w, k);
            __syncthreads();
            return;
        }
        if (threadIdx.x == 0) {
            meet->sweep = w;
            __hip_atomic_store(&meet->number, number, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_AGENT);
        }
        take(number);
        if (threadIdx.x == 0) {
            while (seen_now(meet->taken_done + 2 * number + 1) != (uint32_t)a.pieces) __builtin_amdgcn_s_sleep(2);
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
        }
        __syncthreads();
    }
};

// A sequence's walk: one block leads, the others help with sums over whole rows.
template <int TYPE>
__global__ __launch_bounds__(256) void k_verify_walk(VerifyArgs a) {
    __shared__ int16_t par[DT_NODES], way[DT_NODES];
    __shared__ int tok[DT_NODES];
    __shared__ float lp[DT_NODES], lq[DT_NODES];  // the children's logits at their parents
    __shared__ double uu[DT_NODES], smd[4], joint[4];
    __shared__ float smf[4];
    __shared__ uint32_t gone[V_PIECE / 32];       // tokens of a piece that were rejected
    __shared__ uint32_t smu;
    __shared__ int found;
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, s = blockIdx.x % a.t.n_seqs, V = a.vocab;
    const float t = temperature_of(a, s);
    const bool greedy = !(t > 0.0f), with_q = a.draft && !greedy;
    const double inv = inverse_of(t);
    Walk<TYPE> walk{a, s, a.team - 1, inv, reinterpret_cast<Meeting *>(a.meet + s * (a.meet_words / a.t.n_seqs)),
                    a.swept_top + (size_t)s * a.pieces, a.swept_sum + (size_t)s * a.pieces, smf, smd, &smu};
    if (a.team > 1) {
        if (tid == 0) smu = __hip_atomic_fetch_add(&walk.meet->ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (smu) {
            walk.help();
            return;
        }
    }
    const TreeRows r = tree_rows(a.t, s);
    const int n = min(r.n, a.t.max_nodes), lo = r.lo;
    int32_t *out = a.out + (size_t)s * a.t.max_nodes, *path = a.path + (size_t)s * a.t.max_nodes;
    for (int j = tid; j < n; j += 256) {
        const int p = parent_of(a.t, lo, j), x = a.tokens[lo + j];
        const bool ok = p >= 0 && x >= 0 && x < V;
        par[j] = (int16_t)p, tok[j] = x, uu[j] = a.u[lo + j];
        lp[j] = ok ? load1<TYPE>(row_of<TYPE>(a.logits, a.stride, lo + p), x) : -INFINITY;
        lq[j] = ok && with_q ? load1<TYPE>(row_of<TYPE>(a.draft, a.draft_stride, lo + p), x) : -INFINITY;
    }
    __syncthreads();
    // the next child of `node` behind j, or -1: the same in every wave, like all that follows
    auto child = [&](int node, int j) {
        for (int k = j + 1; k < n; k += 64) {
            const uint64_t m = __ballot(k + lane < n && par[k + lane < n ? k + lane : 0] == node);
            if (m) return k + __builtin_ctzll(m);
        }
        return -1;
    };
    // is there a child of `node` before j whose token `same` takes for j's
    auto earlier = [&](int node, int j, auto same) {
        for (int k = node + 1; k < j; k += 64)
            if (__ballot(k + lane < j && par[k + lane < j ? k + lane : 0] == node && same(tok[k + lane < j ? k + lane : 0]))) return true;
        return false;
    };
    // largest value and sum of a row, of the target (wave 0) and the draft (wave 1), from those of its chunks and pieces
    auto join = [&](int row, double &Mp, double &Zp, double &Mq, double &Zq) {
        __syncthreads();
        if (wave < (with_q ? 2 : 1)) {
            const size_t at = (size_t)row * 2 + wave;
            const float *top = a.top + at * a.chunks;
            const double *sum = a.sum + at * a.pieces;
            float m = -INFINITY;
            for (int k = lane; k < a.chunks; k += 64) m = fmaxf(m, top[k]);
            const double M = wave_max(m);
            double z = 0.0;
            if (M < INFINITY && M > -INFINITY)
                for (int k = lane; k < a.pieces; k += 64) z += sum[k] * exp64(((double)top[k / V_PER] - M) * inv);
            z = wave_add(z);
            if (lane == 0) joint[2 * wave] = M, joint[2 * wave + 1] = z;
        }
        __syncthreads();
        Mp = joint[0], Zp = joint[1], Mq = with_q ? joint[2] : 0.0, Zq = with_q ? joint[3] : 1.0;
        return Mp < INFINITY && Mp > -INFINITY && Mq < INFINITY && Mq > -INFINITY;
    };
    auto swept = [&]() {  // the sum over a sweep's pieces
        double z = 0.0;
        for (int k = lane; k < a.pieces; k += 64) z += walk.sum[k];
        return wave_add(z);
    };

    int at = 0, kept = 1, next = -1;
    uint32_t sweeps = 0;
    if (tid == 0) way[0] = 0;
    while (n) {
        const int row = lo + at, kid = child(at, at);
        int yes = -1;
        if (greedy) {
            const float *top = a.top + (size_t)row * 2 * a.chunks;
            float m = -INFINITY;
            for (int k = lane; k < a.chunks; k += 64) m = fmaxf(m, top[k]);
            m = wave_max(m);
            if (m == INFINITY || m == -INFINITY) break;
            int best = INT32_MAX;
            for (int k = lane; k < a.chunks; k += 64)
                if (top[k] == m) best = min(best, a.arg[(size_t)row * a.chunks + k]);
            best = -wave_max(-best);
            for (int k = kid; k >= 0 && yes < 0; k = child(at, k))
                if (tok[k] == best) yes = k;
            if (yes < 0) next = best;
        } else {
            double Mp = 0, Zp = 1, Mq = 0, Zq = 1, c = 0;
            if (kid >= 0) {
                if (!join(row, Mp, Zp, Mq, Zq)) break;
                double left = 1.0;
                for (int k = kid, after; k >= 0; k = after) {
                    after = child(at, k);
                    double px = exp64(((double)lp[k] - Mp) * inv) / Zp;
                    if (with_q) {
                        const double qx = exp64(((double)lq[k] - Mq) * inv) / Zq;
                        if (uu[k] * left * qx < px - c * qx) {
                            yes = k;
                            break;
                        }
                        c += left;
                        if (after >= 0) {
                            walk.lead({1, row, Mp, 1.0 / Zp, Mq, c / Zq}, ++sweeps);
                            left = swept();
                        }
                    } else {
                        if (earlier(at, k, [&](int x) { return x == tok[k]; })) px = 0.0;  // rejected already
                        if (px > 0.0 && uu[k] * left < px) {
                            yes = k;
                            break;
                        }
                        left -= px;
                    }
                }
            }
            if (yes < 0) {
                if (!(uu[0] >= 0.0 && uu[0] < 1.0)) break;
                // weights of the pieces of what is left: a sweep's sums, or those times exp((largest - M) / T)
                Sweep w{0, row, Mp, 1.0 / Zp, Mq, c / Zq};
                const float *top = walk.top;
                int per = 1;  // pieces to a largest value
                if (with_q && kid >= 0) {
                    w.of_rest = 1;
                    walk.lead(w, ++sweeps);
                    if (!(swept() > 0.0)) w.of_rest = 0;  // nothing: of all that there was
                } else if (kid < 0) {
                    walk.lead(w, ++sweeps);
                    float m = -INFINITY;
                    for (int k = lane; k < a.pieces; k += 64) m = fmaxf(m, walk.top[k]);
                    w.Mp = wave_max(m);
                    if (w.Mp == INFINITY || w.Mp == -INFINITY) break;
                }
                if (kid >= 0 && !w.of_rest) {
                    // the row's own sums, in pieces that hold rejected tokens without those
                    __syncthreads();
                    for (int k = tid; k < a.pieces; k += 256) walk.sum[k] = a.sum[(size_t)row * 2 * a.pieces + k];
                    top = a.top + (size_t)row * 2 * a.chunks, per = V_PER;
                    __syncthreads();
                }
                // bits of this thread's values of a piece that are out of the draw
                auto out_of = [&](int k) -> uint32_t {
                    __syncthreads();
                    if (tid < V_PIECE / 32) gone[tid] = 0;
                    __syncthreads();
                    for (int j = tid; j < n; j += 256) {
                        const int x = tok[j] - k * V_PIECE;
                        if (par[j] == at && x >= 0 && x < V_PIECE) atomicOr(&gone[x / 32], 1u << (x % 32));
                    }
                    __syncthreads();
                    return gone[tid / 4] >> (8 * (tid % 4)) & 255;
                };
                bool without = !with_q && kid >= 0;
                if (without) {
                    const void *pr = row_of<TYPE>(a.logits, a.stride, row);
                    for (int j = kid; j >= 0; j = child(at, j)) {
                        const int k = tok[j] / V_PIECE;
                        if (tok[j] < 0 || tok[j] >= V || earlier(at, j, [&](int x) { return x >= 0 && x / V_PIECE == k; })) continue;
                        const uint32_t o = out_of(k);
                        float v[8];
                        load8<TYPE>(pr, k * V_PIECE + tid * 8, V, v);
                        double z = 0.0;
#pragma unroll
                        for (int e = 0; e < 8; e++) z += o >> e & 1 ? 0.0 : exp64(((double)v[e] - top[k / per]) * inv);
                        z = block_add(z, smd);
                        if (tid == 0) walk.sum[k] = z;
                    }
                    __syncthreads();
                }
                auto weight_of = [&](int k) { return w.of_rest ? walk.sum[k] : walk.sum[k] * exp64(((double)top[k / per] - w.Mp) * inv); };
                auto all = [&]() {
                    double z = 0.0;
                    for (int k = lane; k < a.pieces; k += 64) z += weight_of(k);
                    return wave_add(z);
                };
                double total = all();
                if (without && !(total > 0.0)) {  // nothing left: of all that there was
                    __syncthreads();
                    for (int k = tid; k < a.pieces; k += 256) walk.sum[k] = a.sum[(size_t)row * 2 * a.pieces + k];
                    __syncthreads();
                    without = false, total = all();
                }
                // the piece in which the running sum passes the target, and the sum before it
                const double target = uu[0] * total;
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
                load8<TYPE>(row_of<TYPE>(a.logits, a.stride, row), piece * V_PIECE + tid * 8, V, v);
                if (w.of_rest) load8<TYPE>(row_of<TYPE>(a.draft, a.draft_stride, row), piece * V_PIECE + tid * 8, V, q);
                const uint32_t o = without ? out_of(piece) : 0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    z[e] = o >> e & 1 ? 0.0 : w.of_rest ? walk.rest(w, v[e], q[e]) : exp64(((double)v[e] - w.Mp) * inv);
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
                next = found;
                if (next == INT32_MAX) {
                    __syncthreads();
                    if (tid == 0) found = -1;
                    __syncthreads();
                    if (most >= 0) atomicMax(&found, most);
                    __syncthreads();
                    next = found;
                }
            }
        }
        if (yes < 0) break;
        at = yes;
        if (tid == 0) way[kept] = (int16_t)at;
        kept++;
    }
    __syncthreads();
    if (a.team > 1 && tid == 0) __hip_atomic_store(&walk.meet->number, V_END, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (!n) kept = 0;
    for (int j = tid; j < a.t.max_nodes; j += 256) {
        path[j] = j < kept ? way[j] : -1;
        out[j] = j + 1 < kept ? tok[way[j + 1]] : j + 1 == kept ? next : -1;
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
    part(a.top, (size_t)a.t.n_tokens * 2 * a.chunks);
    part(a.arg, (size_t)a.t.n_tokens * a.chunks);
    part(a.swept_sum, (size_t)a.t.n_seqs * a.pieces);
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
    // blocks to a walk: as many as the row has pieces, but two rounds of the device's CUs for all walks at the most; one
    // where nothing is swept
    a.team = grid.x && (a.temps || a.temp > 0.0f) ? std::max(1, std::min(a.pieces, 512 / a.t.n_seqs)) : 1;
    auto launch = [&](auto T) {
        constexpr int TYPE = decltype(T)::value;
        if (grid.x) TG_LAUNCH(k_verify_rows<TYPE>, grid, dim3(256), 0, st, a);
        TG_LAUNCH(k_verify_walk<TYPE>, dim3((unsigned)(a.t.n_seqs * a.team)), dim3(256), 0, st, a);
    };
    if (type == TG_T_F32) launch(std::integral_constant<int, TG_T_F32>{});
    else if (type == TG_T_F16) launch(std::integral_constant<int, TG_T_F16>{});
    else launch(std::integral_constant<int, TG_T_BF16>{});
    return hipGetLastError();
}

}  // namespace tg
