// Beam search over the rings: the selection over beams and codes, and the
// reordering of the beams' ring state.  No counterpart in the reference, whose
// decoder is greedy (ARGMAX_PENALTY, liyu1981/mockbird
// src/lib/tts/engine/kernels-decode.ts:428-485): beam_select takes the place of
// that argmax when several hypotheses of an utterance are kept.
#include <math.h>

#include "mb_internal.cuh"

namespace mb {

namespace {

constexpr int BEAM_MAX = 16;

struct BeamArgs {
    int beams, codes, end_id;
    long long stride;       // elements between two rows of logits
    const void* logits;     // [groups][beams], rows `stride` apart
    const float* scores;    // [groups][beams]
    float* scores_out;      // may be `scores`
    const int32_t* finished;  // or null
    int32_t* finished_out;    // may be `finished`
    uint32_t* seen;         // [groups][beams][codes / 32] or null
    float penalty;
    int32_t *parents, *tokens;  // [groups][beams]
};

template <typename T>
__device__ __forceinline__ float to_f(T v) {
    return static_cast<float>(v);
}

__device__ __forceinline__ float penalised(float x, bool on, float penalty) {
    return on ? (x >= 0.f ? x / penalty : x * penalty) : x;
}

// (value, id) a before b: larger value first, lower id among equals
__device__ __forceinline__ bool before(double av, int ai, double bv, int bi) {
    return av > bv || (av == bv && ai < bi);
}

// One block per group; B passes over the candidates, each for the best one
// behind the last pick.
template <typename T>
__global__ void __launch_bounds__(256) beam_select_kernel(BeamArgs a) {
    __shared__ double s_red[8], s_lse[BEAM_MAX], s_val;
    __shared__ int s_id[8], s_pick[BEAM_MAX], s_last;
    __shared__ float s_score[BEAM_MAX];
    __shared__ int s_done[BEAM_MAX];
    const int g = blockIdx.x, B = a.beams, V = a.codes, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const T* logits = static_cast<const T*>(a.logits) + (long long)g * B * a.stride;
    uint32_t* seen = a.seen ? a.seen + (size_t)g * B * (V / 32) : nullptr;
    if (tid < B) {
        s_score[tid] = a.scores[g * B + tid];
        s_done[tid] = a.finished ? a.finished[g * B + tid] : 0;
    }
    auto logit = [&](int b, int j) {
        const float x = to_f(logits[b * a.stride + j]);
        return seen ? penalised(x, (seen[(size_t)b * (V / 32) + (j >> 5)] >> (j & 31)) & 1u, a.penalty) : x;
    };
    for (int b = 0; b < B; b++) {
        float m = -INFINITY;
        bool nan = false;
        for (int j = tid; j < V; j += 256) {
            const float x = logit(b, j);
            nan |= x != x;
            m = fmaxf(m, x);
        }
        for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
        if (lane == 0) s_red[warp] = m;
        nan = __syncthreads_or(nan);
        for (int i = 0; i < 8; i++) m = fmaxf(m, (float)s_red[i]);
        __syncthreads();
        double sum = 0;
        for (int j = tid; j < V; j += 256) sum += exp((double)logit(b, j) - (double)m);
        for (int i = 16; i > 0; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
        if (lane == 0) s_red[warp] = sum;
        __syncthreads();
        if (tid == 0) {
            double t = 0;
            for (int i = 0; i < 8; i++) t += s_red[i];
            s_lse[b] = nan ? (double)NAN : (double)m + log(t);
        }
        __syncthreads();
    }
    double lastv = INFINITY;
    int last = -1;
    for (int k = 0; k < B; k++) {
        double bv = -INFINITY;
        int bi = INT_MAX;
        for (int b = 0; b < B; b++)
            for (int j = tid; j < V; j += 256) {
                double v;
                if (s_done[b]) {
                    if (j != a.end_id) continue;
                    v = s_score[b];
                } else {
                    v = (double)s_score[b] + ((double)logit(b, j) - s_lse[b]);
                }
                const int id = b * V + j;
                if (!isfinite((float)v) || !before(lastv, last, v, id)) continue;
                if (before(v, id, bv, bi)) bv = v, bi = id;
            }
        for (int i = 16; i > 0; i >>= 1) {
            const double ov = __shfl_xor_sync(0xffffffffu, bv, i);
            const int oi = __shfl_xor_sync(0xffffffffu, bi, i);
            if (before(ov, oi, bv, bi)) bv = ov, bi = oi;
        }
        if (lane == 0) s_red[warp] = bv, s_id[warp] = bi;
        __syncthreads();
        if (tid == 0) {
            for (int i = 1; i < 8; i++)
                if (before(s_red[i], s_id[i], bv, bi)) bv = s_red[i], bi = s_id[i];
            s_val = bv, s_last = s_pick[k] = bi == INT_MAX ? -1 : bi;
            const bool there = bi != INT_MAX;
            a.parents[g * B + k] = there ? bi / V : -1;
            a.tokens[g * B + k] = there ? bi % V : -1;
            a.scores_out[g * B + k] = there ? (float)bv : -INFINITY;
            if (a.finished_out)
                a.finished_out[g * B + k] = there ? (s_done[bi / V] || bi % V == a.end_id) : s_done[k];
        }
        __syncthreads();
        lastv = s_val, last = s_last;
        if (last < 0) lastv = -INFINITY, last = INT_MAX;  // nothing is behind this
        if (s_last < 0 && tid == 0) s_last = INT_MAX;
        __syncthreads();
    }
    if (seen)
        for (int w = tid; w < V / 32; w += 256) {
            uint32_t word[BEAM_MAX];
#pragma unroll
            for (int k = 0; k < BEAM_MAX; k++) {
                if (k >= B) break;
                const int p = s_pick[k], from = p < 0 ? k : p / V, j = p < 0 ? 0 : p % V;
                word[k] = seen[(size_t)from * (V / 32) + w];
                if (p >= 0 && !s_done[from] && (j >> 5) == w) word[k] |= 1u << (j & 31);
            }
#pragma unroll
            for (int k = 0; k < BEAM_MAX; k++) {
                if (k >= B) break;
                seen[(size_t)k * (V / 32) + w] = word[k];
            }
        }
}

// ---------------------------------------------------------------- ring reorder

// Stream k of a group takes the state of stream parents[k] of the group.  A
// block owns REORDER_SLOTS slots of one layer and group, for K and V of every
// head, so no other block touches what it reads or writes; a thread carries one
// 16-byte piece of all the group's rows, and reads them all before it writes.
constexpr int REORDER_SLOTS = 16;

template <int B>
__global__ void __launch_bounds__(256) ring_reorder_kernel(RingView r, int beams, int row16,
                                                           const int32_t* __restrict__ streams,
                                                           const int32_t* __restrict__ parents) {
    __shared__ int s_stream[BEAM_MAX], s_from[BEAM_MAX], s_pos[BEAM_MAX][REORDER_SLOTS];
    const int C = r.capacity, g = blockIdx.y, j0 = blockIdx.x * REORDER_SLOTS, tid = threadIdx.x;
    char* kv = reinterpret_cast<char*>(r.kv) + (size_t)blockIdx.z * r.kv_layer * (row16 * 16 / HD);
    int32_t* slot_pos = r.slot_pos + (size_t)blockIdx.z * r.slot_layer;
    int why = 0;
    if (tid < beams) {
        const int s = streams[g * beams + tid], p = parents[g * beams + tid];
        s_stream[tid] = s;
        s_from[tid] = p < 0 ? tid : p;
        if (s < 0 || s >= r.streams) why = DERR_STREAM;
        if (p < -1 || p >= beams) why = DERR_PARENT;
    }
    __syncthreads();
    if (tid < beams)
        for (int k = 0; k < tid; k++)
            if (s_stream[k] == s_stream[tid]) why = DERR_STREAM;  // two beams on one ring
    if (__syncthreads_or(why)) {
        if (why && blockIdx.x == 0 && blockIdx.z == 0) atomicOr(r.err, why);
        return;
    }
    const int slots = min(REORDER_SLOTS, C - j0);
    for (int i = tid; i < beams * REORDER_SLOTS; i += 256) {
        const int k = i / REORDER_SLOTS, j = i % REORDER_SLOTS;
        s_pos[k][j] = j < slots ? slot_pos[(size_t)s_stream[k] * C + j0 + j] : -1;
    }
    __syncthreads();
    const size_t stream16 = (size_t)2 * r.heads * C * row16;  // 16-byte pieces of one stream and layer
    uint4* base = reinterpret_cast<uint4*>(kv);
    const int per = slots * row16;
    for (int i = tid; i < 2 * r.heads * per; i += 256) {
        const int hv = i / per, x = i % per, j = x / row16;
        const size_t at = ((size_t)hv * C + j0) * row16 + x;
        uint4 v[B];
#pragma unroll
        for (int k = 0; k < B; k++)
            if (k < beams && s_from[k] != k && s_pos[s_from[k]][j] >= 0)
                v[k] = base[s_stream[s_from[k]] * stream16 + at];
#pragma unroll
        for (int k = 0; k < B; k++)
            if (k < beams && s_from[k] != k && s_pos[s_from[k]][j] >= 0) base[s_stream[k] * stream16 + at] = v[k];
    }
    for (int i = tid; i < beams * REORDER_SLOTS; i += 256) {
        const int k = i / REORDER_SLOTS, j = i % REORDER_SLOTS;
        if (j < slots && s_from[k] != k) slot_pos[(size_t)s_stream[k] * C + j0 + j] = s_pos[s_from[k]][j];
    }
}

cudaError_t launch_select(int dtype, int groups, const BeamArgs& a, cudaStream_t st) {
    switch (dtype) {
        case MB_F32: beam_select_kernel<float><<<groups, 256, 0, st>>>(a); break;
        case MB_BF16: beam_select_kernel<__nv_bfloat16><<<groups, 256, 0, st>>>(a); break;
        default: beam_select_kernel<__half><<<groups, 256, 0, st>>>(a); break;
    }
    return cudaGetLastError();
}

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

}  // namespace

cudaError_t launch_ring_reorder(int dtype, const RingView& r, int layers, int groups, int beams,
                                const int32_t* streams, const int32_t* parents, cudaStream_t st) {
    const int row16 = dtype == MB_F32 ? 16 : 8;
    const dim3 grid((r.capacity + REORDER_SLOTS - 1) / REORDER_SLOTS, groups, layers);
    if (beams <= 4)
        ring_reorder_kernel<4><<<grid, 256, 0, st>>>(r, beams, row16, streams, parents);
    else if (beams <= 8)
        ring_reorder_kernel<8><<<grid, 256, 0, st>>>(r, beams, row16, streams, parents);
    else
        ring_reorder_kernel<16><<<grid, 256, 0, st>>>(r, beams, row16, streams, parents);
    return cudaGetLastError();
}

}  // namespace mb

extern "C" {

MB_API int mb_beam_select(int32_t groups, int32_t beams, int32_t codes, int32_t dtype, const void* logits,
                          int64_t row_stride, const float* scores, float* scores_out, const int32_t* finished,
                          int32_t* finished_out, int32_t end_id, uint32_t* seen, float penalty, int32_t* parents,
                          int32_t* tokens, void* cuda_stream) {
    if (groups < 0 || groups > 65535 || beams < 1 || beams > mb::BEAM_MAX || codes < 1 || codes > (1 << 24) ||
        dtype < MB_F32 || dtype > MB_F16 || row_stride < codes || row_stride > (1ll << 32) || end_id < -1 ||
        end_id >= codes)
        return MB_ERR_ARG;
    if ((finished != nullptr) != (finished_out != nullptr) || (finished && end_id < 0)) return MB_ERR_ARG;
    if (seen && (codes % 32 || !(penalty > 0.f) || !isfinite(penalty))) return MB_ERR_ARG;
    if (groups == 0) return MB_OK;
    if (!logits || !scores || !scores_out || !parents || !tokens) return MB_ERR_ARG;
    if (!mb::aligned(logits, dtype == MB_F32 ? 4 : 2)) return MB_ERR_ARG;
    for (const void* p : {(const void*)scores, (const void*)scores_out, (const void*)finished,
                          (const void*)finished_out, (const void*)seen, (const void*)parents, (const void*)tokens})
        if (!mb::aligned(p, 4)) return MB_ERR_ARG;
    mb::BeamArgs a{};
    a.beams = beams, a.codes = codes, a.end_id = end_id, a.stride = row_stride;
    a.logits = logits, a.scores = scores, a.scores_out = scores_out;
    a.finished = finished, a.finished_out = finished_out;
    a.seen = seen, a.penalty = penalty, a.parents = parents, a.tokens = tokens;
    return mb::launch_select(dtype, groups, a, static_cast<cudaStream_t>(cuda_stream)) == cudaSuccess ? MB_OK
                                                                                                       : MB_ERR_CUDA;
}

}  // extern "C"
