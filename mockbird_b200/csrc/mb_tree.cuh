// The tree of drafted tokens that mb_tree_attend and mb_tree_commit take
// (mb_tree.cu): a node's parent is an earlier node, -1 (it follows the ring's
// last position) or -2 (absent).
#pragma once

#include "mb_internal.cuh"

namespace mb {

constexpr int TREE_MAX_NODES = 64;  // one bit of an ancestor mask per node
constexpr int TREE_ABSENT = -2;

// Topology of one item's tree in shared memory.
struct TreeShape {
    unsigned long long path[TREE_MAX_NODES];  // bit u: u lies on the path root..t, t included; 0: absent
    int link[TREE_MAX_NODES];                 // scratch of tree_shape
    int max_depth;                            // proper ancestors of the deepest node; -1: no node is present
    int bad;                                  // a parent that is neither -2, -1 nor an earlier present node
};

// Fills `sh` from parents[0, nodes), by one full warp (two nodes per lane).
// Pointer doubling: after round i a node's mask holds its nearest 2^i ancestors
// (itself included) and its link the node 2^i steps up, so log2(nodes) rounds
// of one warp replace a walk of up to `nodes` dependent loads.  Reads only
// indices checked against [0, t).
__device__ __forceinline__ void tree_shape(TreeShape& sh, const int32_t* __restrict__ parents, int nodes, int lane) {
    int par[2];
    unsigned long long mask[2];
    int link[2];
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const int t = lane + 32 * e;
        par[e] = t < nodes ? parents[t] : TREE_ABSENT;
        if (par[e] < TREE_ABSENT || par[e] >= t) {
            if (t < nodes) bad = true;
            par[e] = TREE_ABSENT;
        }
        mask[e] = par[e] == TREE_ABSENT ? 0ull : 1ull << t;
        link[e] = par[e] < 0 ? -1 : par[e];
        sh.path[t] = mask[e];
        sh.link[t] = link[e];
    }
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 2; e++)
        if (link[e] >= 0 && sh.path[link[e]] == 0ull) bad = true;  // the parent is absent
    for (int span = 1; span < nodes; span <<= 1) {
        unsigned long long m[2] = {0ull, 0ull};
        int l[2] = {-1, -1};
#pragma unroll
        for (int e = 0; e < 2; e++)
            if (link[e] >= 0) m[e] = sh.path[link[e]], l[e] = sh.link[link[e]];
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 2; e++) {
            mask[e] |= m[e];
            link[e] = l[e];
            sh.path[lane + 32 * e] = mask[e];
            sh.link[lane + 32 * e] = link[e];
        }
        __syncwarp();
    }
    const int deep = max(__popcll(mask[0]), __popcll(mask[1])) - 1;
    const int all_deep = __reduce_max_sync(0xffffffffu, deep);
    const bool any_bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) sh.max_depth = all_deep, sh.bad = any_bad;
    __syncwarp();
}

// Why an item's tree cannot follow position base - 1 of stream s (0: it can).
__device__ __forceinline__ int tree_reject(const RingView& r, const TreeShape& sh, int s, int base) {
    if (sh.bad) return DERR_TREE;
    if (s < 0 || s >= r.streams) return DERR_STREAM;
    if (base < 0 || base >= r.max_position - sh.max_depth) return DERR_POSITION;
    if (!r.wrap && base >= r.capacity - sh.max_depth) return DERR_CAPACITY;
    return 0;
}

}  // namespace mb
