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
    int max_depth;                            // proper ancestors of the deepest node; -1: no node is present
    int bad;                                  // a parent that is neither -2, -1 nor an earlier present node
};

// Fills `sh` from par = (parents[lane], parents[lane + 32]) (tree_parents), by one
// full warp.  Pointer doubling: after round i a node's mask holds its nearest 2^i
// ancestors (itself included) and its link the node 2^i steps up, so log2(nodes)
// rounds of one warp replace a walk of up to `nodes` dependent loads.  Follows
// only links checked against [0, t).
__device__ __forceinline__ int2 tree_parents(const int32_t* __restrict__ parents, int nodes, int lane) {
    return make_int2(lane < nodes ? parents[lane] : TREE_ABSENT, lane + 32 < nodes ? parents[lane + 32] : TREE_ABSENT);
}

__device__ __forceinline__ void tree_shape(TreeShape& sh, int2 parent, int nodes, int lane) {
    constexpr unsigned ALL = 0xffffffffu;
    const bool bad0 = parent.x < TREE_ABSENT || parent.x >= lane, bad1 = parent.y < TREE_ABSENT || parent.y >= lane + 32;
    const int par0 = bad0 ? TREE_ABSENT : parent.x, par1 = bad1 ? TREE_ABSENT : parent.y;
    // nodes 0..31 descend from nodes below 32 alone
    uint32_t low0 = par0 == TREE_ABSENT ? 0u : 1u << lane, low1 = 0u, high1 = par1 == TREE_ABSENT ? 0u : 1u << lane;
    int link0 = par0 < 0 ? -1 : par0, link1 = par1 < 0 ? -1 : par1;
    const uint32_t there0 = __ballot_sync(ALL, low0 != 0u), there1 = __ballot_sync(ALL, high1 != 0u);
    bool bad = bad0 || bad1;  // or the parent is absent
    if (link0 >= 0) bad |= !((there0 >> link0) & 1u);
    if (link1 >= 0) bad |= !(((link1 < 32 ? there0 : there1) >> (link1 & 31)) & 1u);
    for (int span = 1; span < nodes; span <<= 1) {
        const uint32_t a0 = __shfl_sync(ALL, low0, link0 & 31);
        const int n0 = __shfl_sync(ALL, link0, link0 & 31);
        if (nodes > 32) {
            const uint32_t b0 = __shfl_sync(ALL, low0, link1 & 31), b1 = __shfl_sync(ALL, low1, link1 & 31);
            const uint32_t b2 = __shfl_sync(ALL, high1, link1 & 31);
            const int m0 = __shfl_sync(ALL, link0, link1 & 31), m1 = __shfl_sync(ALL, link1, link1 & 31);
            if (link1 >= 32)
                low1 |= b1, high1 |= b2, link1 = m1;
            else if (link1 >= 0)
                low1 |= b0, link1 = m0;
        }
        if (link0 >= 0) low0 |= a0, link0 = n0;
    }
    sh.path[lane] = low0;
    sh.path[lane + 32] = (unsigned long long)high1 << 32 | low1;
    const int deep = max(__popc(low0), __popc(low1) + __popc(high1)) - 1;
    const int all_deep = __reduce_max_sync(ALL, deep);
    const bool any_bad = __any_sync(ALL, bad);
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
