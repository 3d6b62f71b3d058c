// tg_draft.hip -- trees of drafted tokens on the device: which nodes each one
// sees and how deep it stands.
//
// Node j of a sequence is row cu[s] + j of the batch; its parent is a node
// before it, so a walk towards the root only goes down in j.
#include "tg_device.h"
#include "tg_internal.h"

#include "../../include/tinygiant.h"

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

}  // namespace tg
