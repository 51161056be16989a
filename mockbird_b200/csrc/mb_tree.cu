// Attention of a tree of drafted tokens over the ring, and the commit of an
// accepted path.  No counterpart in the reference, which decodes one token per
// step: they verify several drafted continuations of a stream in one pass.
//
//   node t of an item at base position b, with d_t proper ancestors:
//     q_t = rope(q, b + d_t)   k_t = round(rope(k, b + d_t))   v_t = round(v)
//     out_t = sum_j softmax_j(0.125 q_t . k_j) v_j
//   over the ring's slots with 0 <= slot_pos < b and b + d_t - slot_pos < C, and
//   the nodes u on the path root..t with d_t - d_u < C; round() is the rounding to
//   the ring's storage type.  That is what mb_append_attend gives for t when the
//   nodes of its path are appended one after another.
#include "mb_tree.cuh"

namespace mb {

namespace {

template <typename T>
__device__ __forceinline__ float to_f(T v) {
    return static_cast<float>(v);
}
template <typename T>
__device__ __forceinline__ T from_f(float v) {
    return static_cast<T>(v);
}

// One warp per node, one slot per lane: every lane keeps the running maximum,
// sum and context of its slots, and the warp joins them at the end.
template <typename T>
__global__ void __launch_bounds__(128) tree_attend_kernel(RingView r, int nodes, const int32_t* __restrict__ streams,
                                                          const int32_t* __restrict__ positions,
                                                          const int32_t* __restrict__ parents,
                                                          const float* __restrict__ qkv, float* __restrict__ out) {
    __shared__ TreeShape sh;
    __shared__ __align__(16) float sq[4][HD];
    const int H = r.heads, C = r.capacity, item = blockIdx.x / H, h = blockIdx.x % H;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 0) tree_shape(sh, parents + (size_t)item * nodes, nodes, lane);
    __syncthreads();
    if (!sh.bad && sh.max_depth < 0) return;
    const int s = streams[item], base = positions[item];
    if (const int why = tree_reject(r, sh, s, base)) {
        if (threadIdx.x == 0 && h == 0) atomicOr(r.err, why);
        return;
    }
    const T* K = reinterpret_cast<const T*>(r.kv) + (((size_t)s * 2 + 0) * H + h) * (size_t)C * HD;
    const T* V = K + (size_t)H * C * HD;
    const int32_t* sp = r.slot_pos + (size_t)s * C;
    const size_t row = (size_t)3 * H * HD;
    const float* rows = qkv + (size_t)item * nodes * row + h * HD;
    const int window = min(base, C);
    for (int t = warp; t < nodes; t += 4) {
        const unsigned long long path = sh.path[t];
        if (!path) continue;
        const int depth = __popcll(path) - 1, pos = base + depth;
        __syncwarp();
        {
            const float2 q = reinterpret_cast<const float2*>(rows + t * row)[lane];
            reinterpret_cast<float2*>(sq[warp])[lane] = rope_pair(q, r.rope[(size_t)pos * 32 + lane]);
        }
        __syncwarp();
        float m = -INFINITY, l = 0.f, o[HD];
#pragma unroll
        for (int d = 0; d < HD; d++) o[d] = 0.f;
        for (int j = lane; j < window + nodes; j += 32) {
            float k[HD], v[HD];
            if (j < window) {
                const int p = sp[j];
                if (p < 0 || p >= base || pos - p >= C) continue;
#pragma unroll
                for (int d = 0; d < HD; d++) k[d] = to_f(K[(size_t)j * HD + d]), v[d] = to_f(V[(size_t)j * HD + d]);
            } else {
                const int u = j - window;
                if (!((path >> u) & 1ull)) continue;
                const int du = __popcll(sh.path[u]) - 1;
                if (depth - du >= C) continue;
                const float2* kr = reinterpret_cast<const float2*>(rows + u * row + (size_t)H * HD);
                const float* vr = rows + u * row + (size_t)2 * H * HD;
#pragma unroll
                for (int d = 0; d < HD / 2; d++) {
                    const float2 kk = rope_pair(kr[d], r.rope[(size_t)(base + du) * 32 + d]);
                    k[2 * d] = to_f(from_f<T>(kk.x)), k[2 * d + 1] = to_f(from_f<T>(kk.y));
                    v[2 * d] = to_f(from_f<T>(vr[2 * d])), v[2 * d + 1] = to_f(from_f<T>(vr[2 * d + 1]));
                }
            }
            float x = 0.f;
#pragma unroll
            for (int d = 0; d < HD; d++) x = fmaf(sq[warp][d], k[d], x);
            x *= SCALE * LOG2E;
            const float mn = fmaxf(m, x), a = exp2f(m - mn), p = exp2f(x - mn);
            m = mn;
            l = l * a + p;
#pragma unroll
            for (int d = 0; d < HD; d++) o[d] = o[d] * a + p * v[d];
        }
        const float M = [&] {
            float g = m;
            for (int i = 16; i > 0; i >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, i));
            return g;
        }();
        const float a = m == -INFINITY ? 0.f : exp2f(m - M);  // a lane without a visible slot
        float L = l * a;
        for (int i = 16; i > 0; i >>= 1) L += __shfl_xor_sync(0xffffffffu, L, i);
        float* dst = out + ((size_t)item * nodes + t) * H * HD + h * HD;
#pragma unroll
        for (int d = 0; d < HD; d++) {
            float g = o[d] * a;
            for (int i = 16; i > 0; i >>= 1) g += __shfl_xor_sync(0xffffffffu, g, i);
            if (lane == (d & 31)) dst[d] = g / L;
        }
    }
}

// grid (node groups, items, layers), heads * 16 threads: each thread ropes and
// stores four dims of one head, for the accepted nodes of its group.
constexpr int COMMIT_NODES = 4;

template <typename T>
__global__ void __launch_bounds__(1024) tree_commit_kernel(RingView r, int n, int nodes,
                                                           const int32_t* __restrict__ streams,
                                                           const int32_t* __restrict__ positions,
                                                           const int32_t* __restrict__ parents,
                                                           const int32_t* __restrict__ leaves,
                                                           const float* __restrict__ qkv,
                                                           int32_t* __restrict__ next_positions) {
    __shared__ TreeShape sh;
    const int H = r.heads, HID = H * HD, C = r.capacity, item = blockIdx.y, layer = blockIdx.z;
    if (threadIdx.x < 32) tree_shape(sh, parents + (size_t)item * nodes, nodes, threadIdx.x);
    __syncthreads();
    const int s = streams[item], base = positions[item], leaf = leaves[item];
    const bool first = threadIdx.x == 0 && blockIdx.x == 0 && layer == 0;
    if (leaf == -1) {  // nothing accepted: the ring and the position stay
        if (first && next_positions) next_positions[item] = base;
        return;
    }
    int why = leaf < -1 || leaf >= nodes || sh.path[leaf & (TREE_MAX_NODES - 1)] == 0ull ? DERR_TREE : 0;
    if (!why) why = tree_reject(r, sh, s, base);
    if (why) {
        if (first) atomicOr(r.err, why);
        return;
    }
    const unsigned long long path = sh.path[leaf];
    const int len = __popcll(path);
    if (first && next_positions) next_positions[item] = base + len;
    const int t0 = blockIdx.x * COMMIT_NODES, h = threadIdx.x >> 4, d4 = (threadIdx.x & 15) * 4;
    T* kv = reinterpret_cast<T*>(r.kv) + (size_t)layer * r.kv_layer;
    int32_t* sp = r.slot_pos + (size_t)layer * r.slot_layer + (size_t)s * C;
    for (int t = t0; t < min(t0 + COMMIT_NODES, nodes); t++) {
        if (!((path >> t) & 1ull)) continue;
        const int d = __popcll(path & ((1ull << t) - 1ull));  // t's proper ancestors: they come before it
        if (len - d > C) continue;                            // the path's later nodes take this slot
        const int pos = base + d, slot = pos % C;
        const float* src = qkv + (((size_t)layer * n + item) * nodes + t) * 3 * HID + h * HD + d4;
        const float4 k = *reinterpret_cast<const float4*>(src + HID), v = *reinterpret_cast<const float4*>(src + 2 * HID);
        const float4 cs = *reinterpret_cast<const float4*>(r.rope + (size_t)pos * 32 + d4 / 2);
        const float2 k0 = rope_pair(make_float2(k.x, k.y), make_float2(cs.x, cs.y));
        const float2 k1 = rope_pair(make_float2(k.z, k.w), make_float2(cs.z, cs.w));
        T* kd = kv + ((((size_t)s * 2 + 0) * H + h) * C + slot) * HD + d4;
        T* vd = kd + (size_t)H * C * HD;
        alignas(16) T kq[4] = {from_f<T>(k0.x), from_f<T>(k0.y), from_f<T>(k1.x), from_f<T>(k1.y)};
        alignas(16) T vq[4] = {from_f<T>(v.x), from_f<T>(v.y), from_f<T>(v.z), from_f<T>(v.w)};
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(kd) = *reinterpret_cast<const float4*>(kq);
            *reinterpret_cast<float4*>(vd) = *reinterpret_cast<const float4*>(vq);
        } else {
            *reinterpret_cast<uint2*>(kd) = *reinterpret_cast<const uint2*>(kq);
            *reinterpret_cast<uint2*>(vd) = *reinterpret_cast<const uint2*>(vq);
        }
        if (threadIdx.x == 0) sp[slot] = pos;
    }
}

template <typename T>
cudaError_t attend_t(const RingView& r, int n, int nodes, const int32_t* streams, const int32_t* positions,
                     const int32_t* parents, const float* qkv, float* out, cudaStream_t st) {
    tree_attend_kernel<T><<<n * r.heads, 128, 0, st>>>(r, nodes, streams, positions, parents, qkv, out);
    return cudaGetLastError();
}

template <typename T>
cudaError_t commit_t(const RingView& r, int layers, int n, int nodes, const int32_t* streams,
                     const int32_t* positions, const int32_t* parents, const int32_t* leaves, const float* qkv,
                     int32_t* next_positions, cudaStream_t st) {
    const dim3 grid((nodes + COMMIT_NODES - 1) / COMMIT_NODES, n, layers);
    tree_commit_kernel<T><<<grid, r.heads * 16, 0, st>>>(r, n, nodes, streams, positions, parents, leaves, qkv,
                                                         next_positions);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_tree_attend(int dtype, const RingView& r, int n, int nodes, const int32_t* streams,
                               const int32_t* positions, const int32_t* parents, const float* qkv, float* out,
                               cudaStream_t st) {
    switch (dtype) {
        case MB_F32: return attend_t<float>(r, n, nodes, streams, positions, parents, qkv, out, st);
        case MB_BF16: return attend_t<__nv_bfloat16>(r, n, nodes, streams, positions, parents, qkv, out, st);
        default: return attend_t<__half>(r, n, nodes, streams, positions, parents, qkv, out, st);
    }
}

cudaError_t launch_tree_commit(int dtype, const RingView& r, int layers, int n, int nodes, const int32_t* streams,
                               const int32_t* positions, const int32_t* parents, const int32_t* leaves,
                               const float* qkv, int32_t* next_positions, cudaStream_t st) {
    switch (dtype) {
        case MB_F32:
            return commit_t<float>(r, layers, n, nodes, streams, positions, parents, leaves, qkv, next_positions, st);
        case MB_BF16:
            return commit_t<__nv_bfloat16>(r, layers, n, nodes, streams, positions, parents, leaves, qkv,
                                           next_positions, st);
        default:
            return commit_t<__half>(r, layers, n, nodes, streams, positions, parents, leaves, qkv, next_positions,
                                    st);
    }
}

}  // namespace mb
