// tg_draft.hip -- trees of drafted tokens on the device: which nodes each one
// sees and how deep it stands, and which of the drafts a target's
// probabilities keep.
//
// Node j of a sequence is row cu[s] + j of the batch; its parent is a node
// before it, so a walk towards the root only goes down in j.
#include "tg_device.h"
#include "tg_internal.h"

#include "../../include/tinygiant.h"

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
// Whatever a random number decides is decided as in 64 bits.  The rows' sums of exponentials are formed in fp32 first:
// a term's exponent d log2(e) / T is off by 3 2^-24 of itself, a weighted mean of at most log2(V) + 2 <= 26 binary digits over
// the terms that count, its exponential by 2^-23, and the sums by 48 2^-24 at the most, together below 2^-16.  Where two
// sides are nearer than V_NEAR, and wherever something is drawn, the row is summed again in fp64.
constexpr int V_CHUNK = 8192;          // values of a row to a block of the first launch
constexpr int V_PIECE = 2048;          // ... that are summed in fp64 at a time
constexpr double V_NEAR = 1.0 / 32768;

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

TG_DEV float wave_max(float v) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}
TG_DEV double wave_max(double v) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) v = fmax(v, __shfl_xor(v, m));
    return v;
}
template <class T>
TG_DEV T wave_add(T v) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m);
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

// The largest value and the sum of exponentials of each chunk of the rows that a walk may ask: those that something
// follows, of greedy sequences all (and the place of the first of the largest).  NaN or +inf: the largest is +inf.
template <int TYPE>
__global__ __launch_bounds__(256) void k_verify_rows(VerifyArgs a) {
    __shared__ float sm[4];
    __shared__ double smd[4];
    __shared__ int first;
    const int lane = threadIdx.x % 64;
    const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks, of = blockIdx.y;
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
    constexpr int PER = V_CHUNK / 2048;
    float v[PER][8], m = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int k = 0; k < PER; k++) load8<TYPE>(p, chunk * V_CHUNK + k * 2048 + threadIdx.x * 8, a.vocab, v[k]);
#pragma unroll
    for (int k = 0; k < PER; k++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            m = fmaxf(m, v[k][e]);
            bad |= !(v[k][e] < INFINITY);
        }
    m = block_max(bad ? INFINITY : m, sm);
    float sum = 0.0f;
    if (greedy) {
        if (threadIdx.x == 0) first = INT32_MAX;
        __syncthreads();
        int at = INT32_MAX;
#pragma unroll
        for (int k = PER - 1; k >= 0; k--)
#pragma unroll
            for (int e = 7; e >= 0; e--) at = v[k][e] == m ? chunk * V_CHUNK + k * 2048 + (int)threadIdx.x * 8 + e : at;
        if (at != INT32_MAX) atomicMin(&first, at);
        __syncthreads();
        if (threadIdx.x == 0) a.arg[(size_t)row * a.chunks + chunk] = first;
    } else if (m > -INFINITY && m < INFINITY) {
        const float by = fminf(fmaxf((float)(1.4426950408889634 * inverse_of(t)), 1e-37f), 3.402823466e38f);
#pragma unroll
        for (int k = 0; k < PER; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) sum += __builtin_amdgcn_exp2f((v[k][e] - m) * by);
        sum = (float)block_add((double)sum, smd);
    }
    if (threadIdx.x == 0) a.rows[((size_t)row * 2 + of) * a.chunks + chunk] = {m, sum};
}

// A block per sequence: its walk, and the fp64 sums that this asks for.
template <int TYPE>
__global__ __launch_bounds__(256) void k_verify_walk(VerifyArgs a) {
    __shared__ int16_t par[DT_NODES], way[DT_NODES];
    __shared__ int tok[DT_NODES];
    __shared__ float lp[DT_NODES], lq[DT_NODES];  // the children's logits at their parents
    __shared__ double uu[DT_NODES], smd[4];
    __shared__ float smf[4];
    __shared__ uint32_t gone[V_PIECE / 32];       // tokens of a piece that were rejected
    __shared__ int found;
    const int tid = threadIdx.x, lane = tid % 64, s = blockIdx.x, V = a.vocab;
    const TreeRows r = tree_rows(a.t, s);
    const int n = min(r.n, a.t.max_nodes), lo = r.lo;
    const float t = temperature_of(a, s);
    const bool greedy = !(t > 0.0f), with_q = a.draft && !greedy;
    const double inv = inverse_of(t);
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
    // largest value and sum of a row from the chunks'
    auto joined = [&](int row, int of, double &M, double &S) {
        const RowPart *c = a.rows + ((size_t)row * 2 + of) * a.chunks;
        float m = -INFINITY;
        for (int k = lane; k < a.chunks; k += 64) m = fmaxf(m, c[k].m);
        M = wave_max(m);
        S = 0.0;
        if (!(M < INFINITY) || M == -INFINITY) return false;
        for (int k = lane; k < a.chunks; k += 64) S += (double)c[k].s * exp64(((double)c[k].m - M) * inv);
        S = wave_add(S);
        return true;
    };
    PieceSums *ps = a.sums + (size_t)s * a.pieces;
    // sums of exponentials of a piece relative to its largest value, without the tokens of `but`'s children
    auto sum_piece = [&](const void *row, int piece, int but, double &m_out, double &s_out) {
        float v[8];
        load8<TYPE>(row, piece * V_PIECE + tid * 8, V, v);
        uint32_t out8 = 0;
        if (but >= 0) {
            __syncthreads();
            if (tid < V_PIECE / 32) gone[tid] = 0;
            __syncthreads();
            for (int j = tid; j < n; j += 256) {
                const int x = tok[j] - piece * V_PIECE;
                if (par[j] == but && x >= 0 && x < V_PIECE) atomicOr(&gone[x / 32], 1u << (x % 32));
            }
            __syncthreads();
            out8 = gone[tid / 4] >> (8 * (tid % 4)) & 255;
        }
        float m = -INFINITY;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            bad |= !(v[e] < INFINITY);
            if (out8 >> e & 1) v[e] = -INFINITY;
            m = fmaxf(m, v[e]);
        }
        m = block_max(bad ? INFINITY : m, smf);
        double sum = 0.0;
        if (m > -INFINITY && m < INFINITY)
#pragma unroll
            for (int e = 0; e < 8; e++) sum += exp64(((double)v[e] - m) * inv);
        m_out = m, s_out = block_add(sum, smd);
    };
    auto rest_piece = [&](const void *pr, const void *qr, int piece, double c, double Mp, double Zp, double Mq, double Zq) {
        const double ip = 1.0 / Zp, iq = c / Zq;
        float v[8], w[8];
        load8<TYPE>(pr, piece * V_PIECE + tid * 8, V, v);
        load8<TYPE>(qr, piece * V_PIECE + tid * 8, V, w);
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < 8; e++) sum += fmax(exp64(((double)v[e] - Mp) * inv) * ip - exp64(((double)w[e] - Mq) * inv) * iq, 0.0);
        return block_add(sum, smd);
    };
    // sums of a whole row's pieces, p's or q's
    auto sum_row = [&](const void *row, int of, int but, double &M, double &Z) {
        for (int k = 0; k < a.pieces; k++) {
            double m, z;
            sum_piece(row, k, but, m, z);
            if (tid == 0) ps[k].m[of] = m, ps[k].z[of] = z;
        }
        __syncthreads();
        M = -INFINITY;
        for (int k = lane; k < a.pieces; k += 64) M = fmax(M, ps[k].m[of]);
        M = wave_max(M);
        Z = 0.0;
        if (!(M < INFINITY) || M == -INFINITY) return false;
        for (int k = lane; k < a.pieces; k += 64) Z += ps[k].z[of] * exp64((ps[k].m[of] - M) * inv);
        Z = wave_add(Z);
        return true;
    };

    int at = 0, kept = 1, next = -1;
    if (tid == 0) way[0] = 0;
    while (n) {
        const int row = lo + at, kid = child(at, at);
        int yes = -1;
        if (greedy) {
            const RowPart *c = a.rows + (size_t)row * 2 * a.chunks;
            float m = -INFINITY;
            for (int k = lane; k < a.chunks; k += 64) m = fmaxf(m, c[k].m);
            m = wave_max(m);
            if (!(m < INFINITY) || m == -INFINITY) break;
            int best = INT32_MAX;
            for (int k = lane; k < a.chunks; k += 64)
                if (c[k].m == m) best = min(best, a.arg[(size_t)row * a.chunks + k]);
#pragma unroll
            for (int k = 1; k < 64; k *= 2) best = min(best, __shfl_xor(best, k));
            for (int k = kid; k >= 0 && yes < 0; k = child(at, k))
                if (tok[k] == best) yes = k;
            if (yes < 0) next = best;
        } else {
            const void *pr = row_of<TYPE>(a.logits, a.stride, row), *qr = with_q ? row_of<TYPE>(a.draft, a.draft_stride, row) : nullptr;
            double Mp = 0, Zp = 1, Mq = 0, Zq = 1, c = 0;
            bool exact = false;
            if (kid >= 0) {
                if (!joined(row, 0, Mp, Zp) || (with_q && !joined(row, 1, Mq, Zq))) break;
                auto sum_again = [&]() {
                    sum_row(pr, 0, -1, Mp, Zp);
                    if (with_q) sum_row(qr, 1, -1, Mq, Zq);
                    exact = true;
                };
                bool near;
                do {
                    near = false;
                    c = 0.0;
                    double left = 1.0;
                    for (int k = kid, after; k >= 0; k = after) {
                        after = child(at, k);
                        double px = exp64(((double)lp[k] - Mp) * inv) / Zp;
                        if (with_q) {
                            const double qx = exp64(((double)lq[k] - Mq) * inv) / Zq, x = uu[k] * left * qx, y = px - c * qx;
                            near = !exact && fabs(x - y) < V_NEAR * (x + px + c * qx);
                            if (near) break;
                            if (x < y) {
                                yes = k;
                                break;
                            }
                            c += left;
                            if (after >= 0) {
                                if (!exact) sum_again();
                                left = 0.0;
                                for (int i = 0; i < a.pieces; i++) left += rest_piece(pr, qr, i, c, Mp, Zp, Mq, Zq);
                            }
                        } else {
                            for (int j = kid; j < k; j = child(at, j))
                                if (tok[j] == tok[k]) px = 0.0;  // rejected already
                            near = !exact && px > 0.0 && fabs(uu[k] * left - px) < V_NEAR * (uu[k] + px);
                            if (near) break;
                            if (px > 0.0 && uu[k] * left < px) {
                                yes = k;
                                break;
                            }
                            left -= px;
                        }
                    }
                    if (near) sum_again();
                } while (near);
            }
            if (yes < 0) {
                if (!(uu[0] >= 0.0 && uu[0] < 1.0)) break;
                // what is left, piece by piece
                bool rest = with_q && kid >= 0;
                int but = !with_q && kid >= 0 ? at : -1;
                double total = 0.0;
                if (rest) {
                    if (!exact) {
                        sum_row(pr, 0, -1, Mp, Zp);
                        sum_row(qr, 1, -1, Mq, Zq);
                    }
                    for (int k = 0; k < a.pieces; k++) {
                        const double z = rest_piece(pr, qr, k, c, Mp, Zp, Mq, Zq);
                        if (tid == 0) ps[k].rest = z;
                        total += z;
                    }
                    rest = total > 0.0;  // else of all that there was
                } else if (!sum_row(pr, 0, but, Mp, Zp)) {
                    if (Mp == INFINITY || but < 0) break;
                    but = -1;
                    if (!sum_row(pr, 0, -1, Mp, Zp)) break;
                }
                __syncthreads();
                auto weight_of = [&](int k) { return rest ? ps[k].rest : ps[k].z[0] * exp64((ps[k].m[0] - Mp) * inv); };
                if (!rest) total = Zp;
                // the piece in which the running sum passes the target, and the sum before it
                const double target = uu[0] * total;
                double before = 0.0, start = 0.0;
                int piece = -1, last = 0;
                for (int k0 = 0; k0 < a.pieces && piece < 0; k0 += 64) {
                    const double w = k0 + lane < a.pieces ? weight_of(k0 + lane) : 0.0;
                    double up = w;
#pragma unroll
                    for (int m = 1; m < 64; m *= 2) {
                        const double o = __shfl_up(up, m);
                        if (lane >= m) up += o;
                    }
                    const uint64_t past = __ballot(before + up > target && w > 0.0), some = __ballot(w > 0.0);
                    if (some) last = k0 + 63 - __builtin_clzll(some);
                    if (past) {
                        const int k = __builtin_ctzll(past);
                        piece = k0 + k, start = before + __shfl(up - w, k);
                    }
                    before += __shfl(up, 63);
                }
                const bool behind = piece < 0;  // by a rounding: the last token there is
                if (behind) piece = last;
                const double ip = 1.0 / Zp, iq = c / Zq;
                float v[8], q8[8];
                double w[8], mine = 0.0;
                load8<TYPE>(pr, piece * V_PIECE + tid * 8, V, v);
                if (rest) load8<TYPE>(qr, piece * V_PIECE + tid * 8, V, q8);
                uint32_t out8 = 0;
                if (but >= 0) {
                    __syncthreads();
                    if (tid < V_PIECE / 32) gone[tid] = 0;
                    __syncthreads();
                    for (int j = tid; j < n; j += 256) {
                        const int x = tok[j] - piece * V_PIECE;
                        if (par[j] == but && x >= 0 && x < V_PIECE) atomicOr(&gone[x / 32], 1u << (x % 32));
                    }
                    __syncthreads();
                    out8 = gone[tid / 4] >> (8 * (tid % 4)) & 255;
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    w[e] = out8 >> e & 1 ? 0.0 : exp64(((double)v[e] - Mp) * inv);
                    if (rest) w[e] = fmax(w[e] * ip - exp64(((double)q8[e] - Mq) * inv) * iq, 0.0);
                    mine += w[e];
                }
                double up = mine;
#pragma unroll
                for (int m = 1; m < 64; m *= 2) {
                    const double o = __shfl_up(up, m);
                    if (lane >= m) up += o;
                }
                __syncthreads();
                if (lane == 63) smd[tid / 64] = up;
                if (tid == 0) found = INT32_MAX;
                __syncthreads();
                double sum = start + (up - mine);
                for (int k = 0; k < tid / 64; k++) sum += smd[k];
                int hit = INT32_MAX, most = -1;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    sum += w[e];
                    if (w[e] > 0.0) {
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
    const size_t rows = round256((size_t)a.t.n_tokens * 2 * a.chunks * sizeof(RowPart));
    const size_t args = round256((size_t)a.t.n_tokens * a.chunks * sizeof(int));
    a.rows = reinterpret_cast<RowPart *>(ws);
    a.arg = reinterpret_cast<int *>(ws + rows);
    a.sums = reinterpret_cast<PieceSums *>(ws + rows + args);
    return rows + args + (size_t)a.t.n_seqs * a.pieces * sizeof(PieceSums);
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
    auto launch = [&](auto T) {
        constexpr int TYPE = decltype(T)::value;
        if (grid.x) TG_LAUNCH(k_verify_rows<TYPE>, grid, dim3(256), 0, st, a);
        TG_LAUNCH(k_verify_walk<TYPE>, dim3((unsigned)a.t.n_seqs), dim3(256), 0, st, a);
    };
    if (type == TG_T_F32) launch(std::integral_constant<int, TG_T_F32>{});
    else if (type == TG_T_F16) launch(std::integral_constant<int, TG_T_F16>{});
    else launch(std::integral_constant<int, TG_T_BF16>{});
    return hipGetLastError();
}

}  // namespace tg
