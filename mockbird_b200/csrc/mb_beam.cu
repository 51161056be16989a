// Beam search over the rings: the selection over beams and codes, and the
// reordering of the beams' ring state.  No counterpart in the reference, whose
// decoder is greedy (ARGMAX_PENALTY, liyu1981/mockbird
// src/lib/tts/engine/kernels-decode.ts:428-485): beam_select takes the place of
// that argmax when several hypotheses of an utterance are kept.
#include <cooperative_groups.h>
#include <limits.h>
#include <math.h>
#include <stdlib.h>

#include "mb_internal.cuh"

namespace mb {

namespace {

constexpr int BEAM_MAX = 16;
#ifndef FLIGHT
#define FLIGHT 8
#define BMIN 1
#endif
#ifdef TUNE
static int tune(const char* n, int d) { const char* v = getenv(n); return v ? atoi(v) : d; }
#define SEGMENT tune("SEGMENT", 256)
#else
constexpr int SEGMENT = 256;
#endif

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
__device__ __forceinline__ bool before(float av, int ai, float bv, int bi) {
    return av > bv || (av == bv && ai < bi);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A double as an integer of the same order, so that a warp finds the largest of 32
// with integer reductions (-0 counts as 0).
__device__ __forceinline__ unsigned long long order_key(double v) {
    const long long k = __double_as_longlong(v + 0.0);
    return (unsigned long long)(k ^ ((k >> 63) & 0x7fffffffffffffffll)) ^ 0x8000000000000000ull;
}

// ---------------------------------------------------------------- selection
//
// One pass over the logits.  A cluster of blocks takes a group, a warp of it one
// segment of one row: it keeps the segment's sum of exponentials and its `beams`
// best codes (which are the row's best candidates too, since a row's values differ
// from its logits by one number).  The first block then knows every row's
// log-sum-exp, turns the lists into values and merges them.
//
// The sum: exponentials in fp32 against a reference that the warp's maximum exceeds
// by at most 8, batches of 16 added in fp32 and then in fp64.  An exponent x - ref
// is off by at most 2^-23 of itself, whose mean under the softmax is at most
// ln(codes) + 8 < 25, ex2 by 2^-22 and a batch's sum by 2^-22, so the log-sum-exp is
// off by less than 3.5e-6 -- near the rounding of the returned score, but enough to
// exchange two candidates of different beams that differ by less than 7e-6.  Such
// neighbours (NEAR) at or above the last pick are rare; then the group's sums are taken again
// in fp64, by the same warps, and the merge repeated, so the order is always that of
// the values in 64 bits.  (All sums in fp64 would cost 14 fp64 operations per logit:
// 1.4e12 logits/s on this part's fp64 units, against the 1.6e12 fp32 logits/s of HBM.)
constexpr int BEAM_WARPS = 16, BEAM_CLUSTER = 8, UNITS = BEAM_WARPS * BEAM_CLUSTER;
constexpr int CELLS = 12;  // per warp and lane
constexpr double NEAR = 8e-6;
constexpr float ABOVE = 8.f;  // how far the warp's maximum may exceed its reference

struct BeamSmem {
    float value[BEAM_WARPS][BEAM_MAX];  // a warp's list: logits, best first (-inf: none)
    int id[BEAM_WARPS][BEAM_MAX];       // codes
    double sum[BEAM_WARPS];             // of exp(x - top)
    float top[BEAM_WARPS];              // the reference
    float row_top[BEAM_MAX];
    int again;
    union {
        float cell[BEAM_WARPS][CELLS][32];  // the pass: largest values
        struct {                            // the first block's merge
            double cand[UNITS * BEAM_MAX];
            int cand_id[UNITS * BEAM_MAX];
        };
    };
    double lse[BEAM_MAX];
    int pick[BEAM_MAX];
    float score[BEAM_MAX];
    int done[BEAM_MAX];
};

template <typename T, bool SEEN>
struct Row {
    const T* p;
    const uint32_t* seen;
    float penalty;
    __device__ __forceinline__ float one(T v, int j) const {
        const float x = to_f(v);
        if constexpr (SEEN) return penalised(x, (seen[j >> 5] >> (j & 31)) & 1u, penalty);
        return x;
    }
};

// A segment of a row, codes [e0, e1): 16-byte vectors from code `body` on, and up to
// a vector's codes before and behind them.  A batch is 16 codes of every lane: batch
// q's vector v (of VECS) of lane l is vector l + 32 (q VECS + v).
template <typename T>
struct Segment {
    static constexpr int E = 16 / sizeof(T), VECS = 16 / E;
    int e0, head, body, nvec, tail0, tail;
    __device__ __forceinline__ Segment(const T* row, int from, int to) : e0(from) {
        const int off = (int)((reinterpret_cast<uintptr_t>(row + from) & 15) / sizeof(T));
        head = min((E - off) % E, to - from);
        body = from + head;
        nvec = (to - body) / E;
        tail0 = body + nvec * E;
        tail = to - tail0;
    }
    __device__ __forceinline__ int batches() const { return (nvec + 32 * VECS - 1) / (32 * VECS); }
    __device__ __forceinline__ int code(int q, int l, int e) const {  // of value e of a lane's batch
        return body + (l + 32 * (q * VECS + e / E)) * E + e % E;
    }
    // lane's code of the head (lanes 0..) or tail (lanes 16..), -1: none
    __device__ __forceinline__ int edge(int lane) const {
        return lane < head ? e0 + lane : lane >= 16 && lane - 16 < tail ? tail0 + lane - 16 : -1;
    }
};

template <typename T>
__device__ __forceinline__ void load_batch(const T* row, const Segment<T>& sg, int q, int l, uint4* raw) {
    const uint4* vp = reinterpret_cast<const uint4*>(row + sg.body);
#pragma unroll
    for (int v = 0; v < Segment<T>::VECS; v++) {
        const int at = l + 32 * (q * Segment<T>::VECS + v);
        if (at < sg.nvec) raw[v] = vp[at];
    }
}

// the batch's values, -inf behind the segment's last vector
template <typename T, bool SEEN>
__device__ __forceinline__ void batch_values(const Row<T, SEEN>& row, const Segment<T>& sg, int q, int l,
                                             const uint4* raw, float (&x)[16]) {
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const bool in = l + 32 * (q * Segment<T>::VECS + e / Segment<T>::E) < sg.nvec;
        x[e] = in ? row.one(reinterpret_cast<const T*>(raw)[e], sg.code(q, l, e)) : -INFINITY;
    }
}

template <int N>
__device__ __forceinline__ float tree_max(const float (&x)[N]) {
    float m = x[0];
#pragma unroll
    for (int e = 1; e < N; e++) m = fmaxf(m, x[e]);
    return m;
}

template <typename T, bool SEEN>
__global__ void __launch_bounds__(32 * BEAM_WARPS, BMIN) beam_select_kernel(BeamArgs a, int blocks) {
    __shared__ BeamSmem sm;
    constexpr unsigned ALL = 0xffffffffu;
    namespace cg = cooperative_groups;
    const int B = a.beams, V = a.codes, g = blockIdx.x / blocks, rank = blockIdx.x % blocks;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int segs = blocks * BEAM_WARPS / B, unit = rank * BEAM_WARPS + warp, units = segs * B;
    const int b = unit / segs, seg = unit % segs;
    const int e0 = (int)((long long)V * seg / segs), e1 = (int)((long long)V * (seg + 1) / segs);
    auto sync = [&] {
        if (blocks > 1)
            cg::this_cluster().sync();
        else
            __syncthreads();
    };

    Row<T, SEEN> row{};
    bool live = false;
    if (unit < units) {
        const float score = a.scores[g * B + b];
        live = isfinite(score) && !(a.finished && a.finished[g * B + b]);
        row.p = static_cast<const T*>(a.logits) + ((long long)g * B + b) * a.stride;
        if constexpr (SEEN) row.seen = a.seen + ((size_t)g * B + b) * (V / 32);
        row.penalty = a.penalty;
    }
    if (rank == 0 && tid < B) {
        sm.score[tid] = a.scores[g * B + tid];
        sm.done[tid] = a.finished ? a.finished[g * B + tid] : 0;
    }

    const Segment<T> sg(row.p, e0, e1);
    float top = -INFINITY;  // the warp's reference, and a lane's sum of exp(x - top)
    double sum = 0;
    if (live) {
        // The pass: sums, and the largest value of every cell (CELL consecutive batches of a lane).
        constexpr int VECS = Segment<T>::VECS, AHEAD = FLIGHT / VECS;  // batches in flight
        const int nb = sg.batches(), cell = (nb + CELLS - 1) / CELLS;
        float cell_max = -INFINITY, lane_max = -INFINITY;
        auto add = [&](auto& x, float m) {
            constexpr int N = sizeof(x) / sizeof(float);
            if (__any_sync(ALL, m > top + ABOVE)) {
                float w = m;
                for (int i = 16; i > 0; i >>= 1) w = fmaxf(w, __shfl_xor_sync(ALL, w, i));
                if (top > -INFINITY) sum *= exp((double)top - (double)w);
                top = w;
            }
            const float ref = top == -INFINITY ? 0.f : top;
            float s[N];
#pragma unroll
            for (int e = 0; e < N; e++) s[e] = ex2((x[e] - ref) * LOG2E);
#pragma unroll
            for (int w = N / 2; w > 0; w >>= 1)
#pragma unroll
                for (int e = 0; e < w; e++) s[e] += s[e + w];
            sum += (double)s[0];
        };
        uint4 raw[AHEAD][VECS];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) load_batch(row.p, sg, i, lane, raw[i]);
        int in_cell = 0;
        for (int q0 = 0; q0 < nb; q0 += AHEAD)
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const int q = q0 + i;
                if (q >= nb) break;
                float x[16];
                batch_values(row, sg, q, lane, raw[i], x);
                load_batch(row.p, sg, q + AHEAD, lane, raw[i]);
                const float m = tree_max(x);
                add(x, m);
                cell_max = fmaxf(cell_max, m);
                if (++in_cell == cell || q == nb - 1) {
                    sm.cell[warp][q / cell][lane] = cell_max;
                    lane_max = fmaxf(lane_max, cell_max);
                    cell_max = -INFINITY, in_cell = 0;
                }
            }
        const int ej = sg.edge(lane);
        float edge[1] = {ej >= 0 ? row.one(row.p[ej], ej) : -INFINITY};
        add(edge, edge[0]);

        // The list, entry k in lane k.  At least `beams` values are no less than `need`, the beams-th largest of
        // the lanes' maxima, and few more than that are: those in the cells that reach it, which are read again.
        float lv = -INFINITY, need = -INFINITY;
        int li = INT_MAX, need_id = INT_MAX, place = 0;
#pragma unroll
        for (int i = 0; i < 32; i++) place += before(__shfl_sync(ALL, lane_max, i), i, lane_max, lane);
        const unsigned at = __ballot_sync(ALL, place == B - 1);
        if (at) need = __shfl_sync(ALL, lane_max, __ffs(at) - 1);
        auto insert = [&](auto& x, auto&& id) {
            constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
            for (int e = 0; e < N; e++)
                while (true) {
                    const int j = id(e);
                    const unsigned in = __ballot_sync(ALL, x[e] > -INFINITY && before(x[e], j, need, need_id));
                    if (!in) break;
                    const int src = __ffs(in) - 1;
                    const float v = __shfl_sync(ALL, x[e], src);
                    const int vj = __shfl_sync(ALL, j, src);
                    if (lane == src) x[e] = -INFINITY;
                    const int to = __popc(__ballot_sync(ALL, before(lv, li, v, vj)));
                    const float uv = __shfl_up_sync(ALL, lv, 1);
                    const int ui = __shfl_up_sync(ALL, li, 1);
                    if (lane >= to) lv = lane == to ? v : uv, li = lane == to ? vj : ui;
                    const float kv = __shfl_sync(ALL, lv, B - 1);
                    const int ki = __shfl_sync(ALL, li, B - 1);
                    if (kv > -INFINITY) need = kv, need_id = ki;
                }
        };
        insert(edge, [&](int) { return ej; });
        // The cells that reach `need`, 32 at a time, one to a lane.
        const int used = nb ? (nb - 1) / cell + 1 : 0;
        int mine = -1, taken = 0;  // this lane's: cell * 32 + its lane
        auto flush = [&] {
            for (int g = 0; g < cell; g++) {
                const int q = mine < 0 ? nb : (mine >> 5) * cell + g, l = mine & 31;
                uint4 again[VECS];
                float x[16];
                load_batch(row.p, sg, q, l, again);
                batch_values(row, sg, q, l, again, x);
                if (q >= nb)
#pragma unroll
                    for (int e = 0; e < 16; e++) x[e] = -INFINITY;
                if (__any_sync(ALL, tree_max(x) >= need)) insert(x, [&](int e) { return sg.code(q, l, e); });
            }
            mine = -1, taken = 0;
        };
        for (int k = 0; k < used; k++) {
            const float c = sm.cell[warp][k][lane];
            unsigned in = __ballot_sync(ALL, c >= need && c > -INFINITY);
            while (in) {
                const int fit = min(__popc(in), 32 - taken);
                // the fit lowest lanes of `in` go to lanes taken .. taken + fit - 1
                const int want = lane - taken;
                const int src = want >= 0 && want < fit ? (int)__fns(in, 0, want + 1) : -1;
                if (src >= 0) mine = k * 32 + src;
                taken += fit;
                for (int i = 0; i < fit; i++) in &= in - 1u;
                if (taken == 32) flush();
            }
        }
        if (taken) flush();
        if (lane < B) sm.value[warp][lane] = lv, sm.id[warp][lane] = li;
    } else if (lane < B) {
        sm.value[warp][lane] = -INFINITY, sm.id[warp][lane] = INT_MAX;
    }
    auto put_sum = [&] {
        double s = sum;
        for (int i = 16; i > 0; i >>= 1) s += __shfl_xor_sync(ALL, s, i);
        if (lane == 0) sm.top[warp] = top, sm.sum[warp] = s;
    };
    put_sum();
    sync();

    // an object of the cluster's block r
    auto at_block = [&](auto* p, int r) {
        return blocks > 1 ? cg::this_cluster().map_shared_rank(p, r) : p;
    };
    // The first block: every row's log-sum-exp, every candidate's value, the best `beams`.
    // Returns whether two of different beams, a pick and another, are too near to be told apart.
    auto merge = [&]() -> bool {
        for (int r = warp; r < B; r += BEAM_WARPS) {
            float m = -INFINITY, x = -INFINITY;  // the largest reference, the largest logit
            for (int i = lane; i < segs; i += 32) {
                const int u = r * segs + i;
                m = fmaxf(m, *at_block(&sm.top[u % BEAM_WARPS], u / BEAM_WARPS));
                x = fmaxf(x, *at_block(&sm.value[u % BEAM_WARPS][0], u / BEAM_WARPS));
            }
            for (int i = 16; i > 0; i >>= 1) {
                m = fmaxf(m, __shfl_xor_sync(ALL, m, i));
                x = fmaxf(x, __shfl_xor_sync(ALL, x, i));
            }
            double s = 0;
            for (int i = lane; i < segs; i += 32) {
                const int u = r * segs + i;
                const float t = *at_block(&sm.top[u % BEAM_WARPS], u / BEAM_WARPS);
                const double p = *at_block(&sm.sum[u % BEAM_WARPS], u / BEAM_WARPS);
                s += t == -INFINITY ? p : p * exp((double)t - (double)m);
            }
            for (int i = 16; i > 0; i >>= 1) s += __shfl_xor_sync(ALL, s, i);
            if (lane == 0) sm.row_top[r] = x, sm.lse[r] = (double)m + log(s);
        }
        __syncthreads();
        for (int i = tid; i < units * B; i += 32 * BEAM_WARPS) {
            const int u = i / B, k = i % B, r = u / segs;
            float x = *at_block(&sm.value[u % BEAM_WARPS][k], u / BEAM_WARPS);
            int j = *at_block(&sm.id[u % BEAM_WARPS][k], u / BEAM_WARPS);
            double v = (double)sm.score[r] + ((double)x - sm.lse[r]);
            if (sm.done[r]) {  // goes on as it is, once
                v = u % segs == 0 && k == 0 ? (double)sm.score[r] : -INFINITY;
                j = a.end_id;
            }
            if (!isfinite((float)v)) v = -INFINITY;
            sm.cand[u * B + k] = v;
            sm.cand_id[u * B + k] = v > -INFINITY ? r * V + j : INT_MAX;
        }
        __syncthreads();
        bool near = false;
        if (warp == 0) {
            // lane l merges the lists of units l, l + 32, ..: sorted, so only their heads compete
            constexpr int L = UNITS / 32;
            double head[L];
            int head_id[L], pos[L];
#pragma unroll
            for (int i = 0; i < L; i++) {
                const int u = lane + 32 * i;
                pos[i] = 0;
                head[i] = u < units ? sm.cand[u * B] : -INFINITY;
                head_id[i] = u < units ? sm.cand_id[u * B] : INT_MAX;
            }
            // Pick k in lane k; behind the last one, those so near to it that they may belong before it.
            double pv = -INFINITY, least = -INFINITY;
            int pi = INT_MAX, k = 0;
            for (; k < 32; k++) {
                double v = -INFINITY;
                int id = INT_MAX, from = 0;
#pragma unroll
                for (int i = 0; i < L; i++)
                    if (head[i] > v || (head[i] == v && head_id[i] < id)) v = head[i], id = head_id[i], from = i;
                const unsigned long long key = order_key(v);
                const unsigned hi = __reduce_max_sync(ALL, (unsigned)(key >> 32));
                bool in = (unsigned)(key >> 32) == hi;
                const unsigned lo = __reduce_max_sync(ALL, in ? (unsigned)key : 0u);
                in = in && (unsigned)key == lo;
                const int best = (int)__reduce_min_sync(ALL, in ? (unsigned)id : 0xffffffffu);
                const int src = __ffs(__ballot_sync(ALL, in && id == best)) - 1;
                const double bv = __shfl_sync(ALL, v, src);
                if (bv == -INFINITY || (k >= B && least - bv >= NEAR)) break;
                if (lane == k) pv = bv, pi = best;
                if (k == B - 1) least = bv;
                if (lane == src) {
#pragma unroll
                    for (int i = 0; i < L; i++)
                        if (i == from) {
                            const int u = lane + 32 * i;
                            pos[i]++;
                            head[i] = pos[i] < B ? sm.cand[u * B + pos[i]] : -INFINITY;
                            head_id[i] = pos[i] < B ? sm.cand_id[u * B + pos[i]] : INT_MAX;
                        }
                }
            }
            const double nv = __shfl_down_sync(ALL, pv, 1);
            const int ni = __shfl_down_sync(ALL, pi, 1);
            near = k == 32 || __any_sync(ALL, lane < 31 && nv > -INFINITY && pv - nv < NEAR && pi / V != ni / V);
            if (lane < B) {
                sm.pick[lane] = pi;
                sm.lse[lane] = pv;  // (the log-sum-exps are used up: the picks' values)
            }
        }
        return __syncthreads_or(near);
    };
    bool again = false;
    if (rank == 0) {
        again = merge();
        if (tid < blocks) *at_block(&sm.again, tid) = again;  // (to each block: this one may leave first)
    }
    sync();
    again = sm.again;
    if (again) {  // the sums once more, in fp64 against the row's maximum
        if (live) {
            // (every row in the same order, whatever its alignment: equal rows have equal sums)
            top = *at_block(&sm.row_top[b], 0);
            sum = 0;
            for (int j = e0 + lane; j < e1; j += 32) {
                const float x = row.one(row.p[j], j);
                if (!(x == -INFINITY)) sum += exp((double)x - (double)top);
            }
            put_sum();
        }
        sync();
        if (rank == 0) merge();
        sync();  // no block leaves while the first one reads its shared memory
    }
    if (rank != 0) return;

    if (tid < B) {
        const int p = sm.pick[tid];
        const bool there = p != INT_MAX;
        const int from = there ? p / V : -1, j = there ? p % V : -1;
        a.parents[g * B + tid] = from;
        a.tokens[g * B + tid] = j;
        a.scores_out[g * B + tid] = there ? (float)sm.lse[tid] : -INFINITY;
        if (a.finished_out) a.finished_out[g * B + tid] = there ? (sm.done[from] || j == a.end_id) : sm.done[tid];
    }
    if constexpr (SEEN) {  // a thread carries one word of every row: all read before any is written
        uint32_t* seen = a.seen + (size_t)g * B * (V / 32);
        for (int w = tid; w < V / 32; w += 32 * BEAM_WARPS) {
            uint32_t word[BEAM_MAX];
#pragma unroll
            for (int k = 0; k < BEAM_MAX; k++)
                if (k < B) {
                    const int p = sm.pick[k], from = p == INT_MAX ? k : p / V, j = p == INT_MAX ? 0 : p % V;
                    word[k] = seen[(size_t)from * (V / 32) + w];
                    if (p != INT_MAX && !sm.done[from] && (j >> 5) == w) word[k] |= 1u << (j & 31);
                }
#pragma unroll
            for (int k = 0; k < BEAM_MAX; k++)
                if (k < B) seen[(size_t)k * (V / 32) + w] = word[k];
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

template <typename T, bool SEEN>
cudaError_t launch_select_t(int groups, const BeamArgs& a, cudaStream_t st) {
    // blocks per group: enough for the SMs, a warp's segment no shorter than SEGMENT codes
    int blocks = 1;
    while (blocks < BEAM_CLUSTER && groups * blocks < 2 * 148 &&
           (long long)a.beams * a.codes >= 2ll * blocks * BEAM_WARPS * SEGMENT)
        blocks *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(groups * blocks);
    cfg.blockDim = dim3(32 * BEAM_WARPS);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {(unsigned)blocks, 1, 1};
    cfg.attrs = &attr;
    cfg.numAttrs = blocks > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, beam_select_kernel<T, SEEN>, a, blocks);
}

template <typename T>
cudaError_t launch_select_s(int groups, const BeamArgs& a, cudaStream_t st) {
    return a.seen ? launch_select_t<T, true>(groups, a, st) : launch_select_t<T, false>(groups, a, st);
}

cudaError_t launch_select(int dtype, int groups, const BeamArgs& a, cudaStream_t st) {
    switch (dtype) {
        case MB_F32: return launch_select_s<float>(groups, a, st);
        case MB_BF16: return launch_select_s<__nv_bfloat16>(groups, a, st);
        default: return launch_select_s<__half>(groups, a, st);
    }
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
