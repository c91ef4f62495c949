// experts.cu -- the row operations of a routed (mixture-of-experts)
// feed-forward: the router's top-k of a softmax, the stable sort of the
// (token, slot) pairs by expert, the copy of token rows to their experts'
// rows and the weighted sum on the way back, each with its gradient.  No
// counterpart in the reference (its DAG has no routed layer).
//
// All of them are bound by memory traffic or, for a few tokens, by launch
// latency.  Sums are f32 in slot order, so results do not depend on timing;
// the only atomics are integer counts in shared memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <climits>
#include <type_traits>

#include "common.cuh"

namespace chelis {

extern std::atomic<uint64_t> g_launches;

namespace experts {

constexpr int MAX_EXPERTS = 1024;
constexpr int MAX_K = 32;  // slots of a token: one lane of the router's warp each

// ---- element access -------------------------------------------------------
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// V consecutive elements as one access: 16 bytes when VEC, one element
// otherwise (a width or a base that 16 bytes do not divide).
template <typename T, bool VEC>
struct Pack {
    static constexpr int N = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
    T v[N];
};
template <typename T, bool VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T *p) {
    Pack<T, VEC> r;
    if constexpr (VEC) *reinterpret_cast<uint4 *>(&r) = __ldg(reinterpret_cast<const uint4 *>(p));
    else r.v[0] = p[0];
    return r;
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, VEC> &r) {
    if constexpr (VEC) *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(&r);
    else p[0] = r.v[0];
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// ---- router ---------------------------------------------------------------
// A number's bits as an unsigned integer that orders as the number does; -0
// and +0 alike.  0 stands for "not to be chosen": -inf (a masked expert), a
// NaN and what was already chosen; every other number is above 0.
__device__ __forceinline__ uint32_t order_key(float l) {
    if (!(l > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(l + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// One warp a token, expert v * 32 + lane in the lane's value v: k rounds of a
// warp maximum over the keys, then over the indices that hold it (the lowest
// wins).  The softmax is taken against the first chosen logit, the largest.
// 16384 x 64, k = 8 in 9.5 us: bound by the rounds' instructions (about 350 a
// token, ALU 71 % busy), not by its 5 MB; 8 tokens take 2.8 us, a launch.
template <typename T, int NV>
__global__ void route_kernel(const T *__restrict__ logits, int64_t tokens, int experts, int k,
                             int renormalize, float *__restrict__ weights, int32_t *__restrict__ ids) {
    const int lane = threadIdx.x & 31;
    const int64_t t = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    if (t >= tokens) return;
    float l[NV];
    uint32_t key[NV];
    bool nan = false;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int i = v * 32 + lane;
        l[v] = i < experts ? to_f32(logits[t * experts + i]) : -INFINITY;
        nan |= l[v] != l[v];
        key[v] = order_key(l[v]);
    }
    nan = __any_sync(0xffffffffu, nan);
    int id = -1;  // lane j: the expert chosen in round j
    for (int j = 0; j < k; ++j) {
        uint32_t best = 0;
        int at = 0;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (key[v] > best) {
                best = key[v];
                at = v * 32 + lane;
            }
        const uint32_t most = __reduce_max_sync(0xffffffffu, best);
        if (most == 0) break;  // nothing left to choose
        const int which = __reduce_min_sync(0xffffffffu, best == most ? at : INT_MAX);
        if (lane == j) id = which;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (which == v * 32 + lane) key[v] = 0;
    }
    // the chosen logits, read again (from L1) rather than carried through the rounds
    const float mine = id >= 0 ? to_f32(logits[t * experts + id]) : -INFINITY;
    const float top = __shfl_sync(0xffffffffu, mine, 0);
    const float e = id >= 0 ? expf(mine - top) : 0.0f;
    float z = e;
    if (!renormalize) {
        z = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) z += l[v] > -INFINITY ? expf(l[v] - top) : 0.0f;
    }
    z = warp_sum(z);
    if (lane < k) {
        float w = id >= 0 ? e / z : 0.0f;
        if (nan) w = __int_as_float(0x7fc00000);
        weights[t * k + lane] = w;
        ids[t * k + lane] = id;
    }
}

// dl_i = p_i (g_i - sum_j p_j g_j): over the chosen experts when the weights
// were renormalised (p their softmax alone), over all of them otherwise (g_i
// = 0 off the chosen).  16384 x 64, k = 8 in 6.6 us, bound as route_kernel.
template <typename T, int NV>
__global__ void route_bwd_kernel(const T *__restrict__ logits, const int32_t *__restrict__ ids,
                                 const float *__restrict__ dweights, int64_t tokens, int experts,
                                 int k, int renormalize, T *__restrict__ dlogits) {
    const int lane = threadIdx.x & 31;
    const int64_t t = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    if (t >= tokens) return;
    float p[NV], g[NV];
    bool in[NV];
    bool nan = false;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int i = v * 32 + lane;
        p[v] = i < experts ? to_f32(logits[t * experts + i]) : -INFINITY;
        nan |= p[v] != p[v];
        g[v] = 0.0f;
        in[v] = !renormalize;
    }
    nan = __any_sync(0xffffffffu, nan);
    int my_id = -1;
    float my_g = 0.0f;
    if (lane < k) {
        my_id = ids[t * k + lane];
        my_g = dweights[t * k + lane];
        if (my_id < -1 || my_id >= experts) {
            report_device_error(DEVERR_BAD_INDEX);
            my_id = -1;
        }
    }
    for (int j = 0; j < k; ++j) {
        const int id = __shfl_sync(0xffffffffu, my_id, j);
        const float gj = __shfl_sync(0xffffffffu, my_g, j);
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (id == v * 32 + lane) {
                g[v] += gj;
                in[v] = true;
            }
    }
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v)
        if (in[v]) top = fmaxf(top, p[v]);
    top = warp_max(top);
    float z = 0.0f, inner = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        p[v] = in[v] && p[v] > -INFINITY ? expf(p[v] - top) : 0.0f;
        z += p[v];
    }
    z = warp_sum(z);
    const bool none = z == 0.0f;  // no expert to choose from
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        p[v] = none ? 0.0f : p[v] / z;
        inner += p[v] * g[v];
    }
    inner = warp_sum(inner);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int i = v * 32 + lane;
        float d = p[v] != 0.0f ? p[v] * (g[v] - inner) : 0.0f;
        if (nan) d = __int_as_float(0x7fc00000);
        if (i < experts) dlogits[t * experts + i] = from_f32<T>(d);
    }
}

// ---- sort by expert -------------------------------------------------------
// A stable counting sort of the n = tokens * k pairs.  sort_count_kernel
// counts each segment's pairs by expert; sort_place_kernel adds up the
// segments before its own, ranks its pairs in order and writes the places.
// One segment (n <= SEGMENT) needs that kernel alone; from SCAN_FROM counts on
// sort_scan_kernel adds them up in between.  Latency bounds them: 8 x 2 pairs
// by 8 experts 2.8 us, 16384 x 2 by 8 5.3 us, 16384 x 8 by 64 9.3 us, by 1024
// 10.7 us; 131072 x 8 by 64 20 us.  Shorter segments read too many others' counts, longer
// ones leave the machine idle (512 / 1024 / 2048 pairs, before the counts were
// shared out among the threads: 9.1 / 7.5 / 8.9 us for the first of these).
constexpr int SORT_THREADS = 256;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SEGMENT = 1024;
constexpr int PER_WARP = SEGMENT / SORT_WARPS;  // consecutive pairs of a warp

__device__ __forceinline__ int sort_id(const int32_t *ids, int64_t i, int64_t n, int experts) {
    if (i >= n) return -1;
    const int id = ids[i];
    if (id >= -1 && id < experts) return id;
    report_device_error(DEVERR_BAD_INDEX);  // taken as not routed
    return -1;
}

__global__ void __launch_bounds__(SORT_THREADS)
    sort_count_kernel(const int32_t *__restrict__ ids, int64_t n, int experts,
                      int32_t *__restrict__ counts) {
    __shared__ int hist[MAX_EXPERTS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int e = threadIdx.x; e < experts; e += SORT_THREADS) hist[e] = 0;
    __syncthreads();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * SEGMENT;
    for (int i = threadIdx.x; i < SEGMENT; i += SORT_THREADS) {
        const int id = sort_id(ids, first + i, n, experts);
        if (id >= 0) atomicAdd(&hist[id], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += SORT_THREADS)
        counts[static_cast<int64_t>(blockIdx.x) * experts + e] = hist[e];
}

// For many segments or experts, where each segment adding up all the others'
// counts is what costs (with the scan and without: 32 segments of 64 experts
// 8.5 and 6.7 us, of 256 8.8 and 9.9; 128 of 64 9.3 and 11.0, of 1024 10.7 and
// 78; 1024 of 64 20 and 72, of 1024 25 and 1050): counts[s][e] becomes the pairs of e in the segments before s, and
// one more row, counts[segments], each expert's total.  A block has SCAN_WIDTH
// experts (a 32-byte sector of a row), its threads consecutive shares of the
// segments.
constexpr int SCAN_THREADS = 1024;
constexpr int SCAN_WIDTH = 8;
constexpr int SCAN_SHARES = SCAN_THREADS / SCAN_WIDTH;
constexpr int SCAN_DEEP = 8;  // counts in flight a thread
constexpr int64_t SCAN_FROM = 8192;  // counts from which the scan pays for its launch

__global__ void __launch_bounds__(SCAN_THREADS)
    sort_scan_kernel(int32_t *__restrict__ counts, int64_t segments, int experts) {
    __shared__ int part[SCAN_WIDTH][SCAN_SHARES];
    const int col = threadIdx.x % SCAN_WIDTH, share = threadIdx.x / SCAN_WIDTH;
    const int e = blockIdx.x * SCAN_WIDTH + col;
    const int64_t per = (segments + SCAN_SHARES - 1) / SCAN_SHARES;
    const int64_t first = share * per;
    int64_t last = first + per < segments ? first + per : segments;
    if (e >= experts) last = first;  // no expert, nothing to add up
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int sum = 0;
#pragma unroll SCAN_DEEP
    for (int64_t s = first; s < last; ++s) sum += counts[s * experts + e];
    part[col][share] = sum;
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp < SCAN_WIDTH) {  // an expert's shares, each to the sum of those before it
        constexpr int EACH = SCAN_SHARES / 32;
        int own[EACH], all = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            own[i] = part[warp][lane * EACH + i];
            all += own[i];
        }
        int scan = all;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, scan, off);
            if (lane >= off) scan += o;
        }
        const int expert = blockIdx.x * SCAN_WIDTH + warp;
        if (lane == 31 && expert < experts) counts[segments * experts + expert] = scan;
        scan -= all;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            part[warp][lane * EACH + i] = scan;
            scan += own[i];
        }
    }
    __syncthreads();
    int before = part[col][share];
    for (int64_t s = first; s < last; s += SCAN_DEEP) {
        int c[SCAN_DEEP];
#pragma unroll
        for (int i = 0; i < SCAN_DEEP; ++i) c[i] = s + i < last ? counts[(s + i) * experts + e] : 0;
#pragma unroll
        for (int i = 0; i < SCAN_DEEP; ++i) {
            if (s + i < last) counts[(s + i) * experts + e] = before;
            before += c[i];
        }
    }
}

// `counts` is still being written while this kernel's first part runs, so it is
// neither const nor __restrict__: as such its loads could take the read-only
// path or be moved above the wait.
__global__ void __launch_bounds__(SORT_THREADS)
    sort_place_kernel(const int32_t *__restrict__ ids, int64_t n, int experts,
                      int32_t *counts, int scanned, int32_t *__restrict__ offsets,
                      int32_t *__restrict__ position, int32_t *__restrict__ source) {
    extern __shared__ int sort_smem[];
    int *next = sort_smem;                      // [SORT_WARPS][experts]: a warp's next place
    int *total = next + SORT_WARPS * experts;   // [experts]: pairs of the expert, then its start
    __shared__ int routed, warp_part[SORT_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int segments = gridDim.x, seg = blockIdx.x;
    int *earlier = total + experts;             // [experts]: pairs of earlier segments
    for (int i = threadIdx.x; i < (SORT_WARPS + 2) * experts; i += SORT_THREADS) next[i] = 0;
    __syncthreads();
    // pairs of each warp by expert
    const int64_t first = static_cast<int64_t>(seg) * SEGMENT + warp * PER_WARP;
    int mine[PER_WARP / 32];
#pragma unroll
    for (int c = 0; c < PER_WARP / 32; ++c) {
        mine[c] = sort_id(ids, first + c * 32 + lane, n, experts);
        if (mine[c] >= 0) atomicAdd(&next[warp * experts + mine[c]], 1);
    }
    __syncthreads();
    // before[w] = pairs of earlier segments and earlier warps, once those are counted
    if (segments > 1) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (scanned) {
        for (int e = threadIdx.x; e < experts; e += SORT_THREADS) {
            earlier[e] = counts[static_cast<int64_t>(seg) * experts + e];
            total[e] = counts[static_cast<int64_t>(segments) * experts + e];
        }
    } else if (segments > 1) {
        // `shares` threads add up an expert's segments, every shares-th each
        const int shares = experts < SORT_THREADS ? SORT_THREADS / experts : 1;
        for (int i = threadIdx.x; i < shares * experts; i += SORT_THREADS) {
            const int e = i % experts;
            int before = 0, all = 0;
#pragma unroll 8
            for (int s = i / experts; s < segments; s += shares) {
                const int c = counts[static_cast<int64_t>(s) * experts + e];
                if (s < seg) before += c;
                all += c;
            }
            atomicAdd(&total[e], all);
            atomicAdd(&earlier[e], before);
        }
        __syncthreads();
    }
    for (int e = threadIdx.x; e < experts; e += SORT_THREADS) {
        int before = earlier[e];
#pragma unroll
        for (int w = 0; w < SORT_WARPS; ++w) {
            const int c = next[w * experts + e];
            next[w * experts + e] = before;
            before += c;
        }
        if (segments == 1) total[e] = before;
    }
    __syncthreads();
    // exclusive scan over experts: SORT_THREADS chunks of consecutive experts
    const int per = (experts + SORT_THREADS - 1) / SORT_THREADS;
    int sum = 0;
    for (int c = 0; c < per; ++c) {
        const int e = threadIdx.x * per + c;
        if (e < experts) sum += total[e];
    }
    int scan = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, scan, off);
        if (lane >= off) scan += o;
    }
    if (lane == 31) warp_part[warp] = scan;
    __syncthreads();
    int start = scan - sum;
    for (int w = 0; w < warp; ++w) start += warp_part[w];
    for (int c = 0; c < per; ++c) {
        const int e = threadIdx.x * per + c;
        if (e < experts) {
            const int cnt = total[e];
            total[e] = start;
            if (seg == 0) offsets[e] = start;
            start += cnt;
        }
    }
    if (threadIdx.x == SORT_THREADS - 1) {
        routed = start;
        if (seg == 0) offsets[experts] = start;
    }
    __syncthreads();
    // places, 32 pairs at a time in order
#pragma unroll
    for (int c = 0; c < PER_WARP / 32; ++c) {
        const int64_t i = first + c * 32 + lane;
        const int id = mine[c];
        const unsigned same = __match_any_sync(0xffffffffu, id);
        const int rank = __popc(same & ((1u << lane) - 1u));
        int place = -1;
        if (id >= 0) place = total[id] + next[warp * experts + id] + rank;
        __syncwarp();
        if (id >= 0 && rank == 0) next[warp * experts + id] += __popc(same);
        __syncwarp();
        if (i < n) {
            position[i] = place;
            if (place >= 0) source[place] = static_cast<int32_t>(i);
        }
    }
    // places that no pair takes
    for (int64_t i = routed + static_cast<int64_t>(seg) * SORT_THREADS + threadIdx.x; i < n;
         i += static_cast<int64_t>(segments) * SORT_THREADS)
        source[i] = -1;
}

// ---- rows to their experts, and back --------------------------------------
// xs[position[t, j]] = x[t]: one read of a token's row, k writes.  A warp
// moves WIDE packs a lane of one row at a time.  Rows that no pair takes
// (from *routed on) are written as zeros.  Bound by memory: 16384 tokens of
// 1024 f32 to two rows each in 32 us (6.3 TB/s), of 1024 bf16 to eight 54 us
// (5.6 TB/s, eight writes to a read).
constexpr int ROW_THREADS = 256;
constexpr int WIDE = 4;

template <typename T, bool VEC>
__global__ void __launch_bounds__(ROW_THREADS)
    spread_kernel(const T *__restrict__ x, const int32_t *__restrict__ position,
                  const int32_t *__restrict__ routed, int64_t tokens, int k, int64_t hidden,
                  T *__restrict__ xs) {
    using P = Pack<T, VEC>;
    const int lane = threadIdx.x & 31;
    const int64_t span = static_cast<int64_t>(32) * WIDE * P::N;
    const int64_t pieces = (hidden + span - 1) / span;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (ROW_THREADS / 32);
    const int64_t warp0 = (static_cast<int64_t>(blockIdx.x) * ROW_THREADS + threadIdx.x) >> 5;
    const int64_t rows = tokens * k;
    for (int64_t w = warp0; w < tokens * pieces; w += warps) {
        const int64_t t = w / pieces, c0 = (w - t * pieces) * span + lane * P::N;
        P r[WIDE];
#pragma unroll
        for (int u = 0; u < WIDE; ++u) {
            const int64_t c = c0 + u * 32 * P::N;
            if (c < hidden) r[u] = load_pack<T, VEC>(x + t * hidden + c);
        }
        for (int j = 0; j < k; ++j) {
            const int64_t at = position[t * k + j];
            if (at < 0) continue;
            if (at >= rows) {
                report_device_error(DEVERR_BAD_INDEX);
                continue;
            }
#pragma unroll
            for (int u = 0; u < WIDE; ++u) {
                const int64_t c = c0 + u * 32 * P::N;
                if (c < hidden) store_pack<T, VEC>(xs + at * hidden + c, r[u]);
            }
        }
    }
    int64_t used = *routed;
    used = used < 0 ? 0 : (used > rows ? rows : used);
    P zero{};
    for (int64_t w = warp0; w < (rows - used) * pieces; w += warps) {
        const int64_t r = w / pieces, c0 = (w - r * pieces) * span + lane * P::N;
#pragma unroll
        for (int u = 0; u < WIDE; ++u) {
            const int64_t c = c0 + u * 32 * P::N;
            if (c < hidden) store_pack<T, VEC>(xs + (used + r) * hidden + c, zero);
        }
    }
}

// y[t] = sum_j w[t, j] ys[position[t, j]] in f32, slot order, rounded once.
// Without weights it is the gradient of spread_kernel.  A warp takes DEEP
// packs a lane of one token; its lanes hold the token's positions and weights.
// Bound by memory: 16384 tokens of 1024 f32 from two rows each 35 us (5.8 TB/s;
// one pack 37), of 1024 bf16 from eight 56 us (5.4 TB/s).  Loading four rows
// before adding the first took 61 to 86 us: the registers cost more resident
// warps than the loads in flight gained.
constexpr int DEEP = 2;

template <typename T, bool VEC>
__global__ void __launch_bounds__(ROW_THREADS)
    combine_kernel(const T *__restrict__ ys, const float *__restrict__ weights,
                   const int32_t *__restrict__ position, int64_t tokens, int k, int64_t hidden,
                   T *__restrict__ y) {
    using P = Pack<T, VEC>;
    const int lane = threadIdx.x & 31;
    const int64_t span = static_cast<int64_t>(32) * DEEP * P::N;
    const int64_t pieces = (hidden + span - 1) / span;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (ROW_THREADS / 32);
    const int64_t rows = tokens * k;
    for (int64_t w = (static_cast<int64_t>(blockIdx.x) * ROW_THREADS + threadIdx.x) >> 5;
         w < tokens * pieces; w += warps) {
        const int64_t t = w / pieces, c0 = (w - t * pieces) * span + lane * P::N;
        int at_lane = -1;
        float w_lane = 0.0f;
        if (lane < k) {
            at_lane = position[t * k + lane];
            w_lane = weights ? weights[t * k + lane] : 1.0f;
            if (at_lane >= rows) {
                report_device_error(DEVERR_BAD_INDEX);
                at_lane = -1;
            }
        }
        float acc[DEEP][P::N] = {};
#pragma unroll 2
        for (int j = 0; j < k; ++j) {
            const int64_t at = __shfl_sync(0xffffffffu, at_lane, j);
            const float wj = __shfl_sync(0xffffffffu, w_lane, j);
            if (at < 0) continue;
            P r[DEEP];
#pragma unroll
            for (int u = 0; u < DEEP; ++u) {
                r[u] = P{};
                if (c0 + u * 32 * P::N < hidden) r[u] = load_pack<T, VEC>(ys + at * hidden + c0 + u * 32 * P::N);
            }
#pragma unroll
            for (int u = 0; u < DEEP; ++u)
#pragma unroll
                for (int i = 0; i < P::N; ++i) acc[u][i] = fmaf(wj, to_f32(r[u].v[i]), acc[u][i]);
        }
#pragma unroll
        for (int u = 0; u < DEEP; ++u) {
            const int64_t c = c0 + u * 32 * P::N;
            P out;
#pragma unroll
            for (int i = 0; i < P::N; ++i) out.v[i] = from_f32<T>(acc[u][i]);
            if (c < hidden) store_pack<T, VEC>(y + t * hidden + c, out);
        }
    }
}

// dys[position[t, j]] = w[t, j] dy[t] and dw[t, j] = <dy[t], ys[position[t, j]]>:
// one block a token, the k dot products reduced by warp, then over warps (a
// fixed order).  dy stays in L1 over the slots.  Bound by memory: 16384 tokens
// of 1024 bf16, k = 8, 95 us (6.0 TB/s); four rows at a time halved the
// resident blocks and took 132 us.
constexpr int BWD_THREADS = 128;

template <typename T, bool VEC>
__global__ void __launch_bounds__(BWD_THREADS)
    combine_bwd_kernel(const T *__restrict__ dy, const T *__restrict__ ys,
                       const float *__restrict__ weights, const int32_t *__restrict__ position,
                       const int32_t *__restrict__ routed, int64_t tokens, int k, int64_t hidden,
                       T *__restrict__ dys, float *__restrict__ dweights) {
    using P = Pack<T, VEC>;
    __shared__ float part[BWD_THREADS / 32][MAX_K];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t rows = tokens * k;
    for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
        for (int j = 0; j < k; ++j) {
            const int64_t at = position[t * k + j];
            const bool ok = at >= 0 && at < rows;
            if (at >= rows) report_device_error(DEVERR_BAD_INDEX);
            const float wj = weights[t * k + j];
            float dot = 0.0f;
            if (ok)
                for (int64_t c = threadIdx.x * P::N; c < hidden; c += BWD_THREADS * P::N) {
                    const P d = load_pack<T, VEC>(dy + t * hidden + c);
                    const P r = load_pack<T, VEC>(ys + at * hidden + c);
                    P out;
#pragma unroll
                    for (int i = 0; i < P::N; ++i) {
                        const float g = to_f32(d.v[i]);
                        dot = fmaf(g, to_f32(r.v[i]), dot);
                        out.v[i] = from_f32<T>(wj * g);
                    }
                    store_pack<T, VEC>(dys + at * hidden + c, out);
                }
            dot = warp_sum(dot);
            if (lane == 0) part[warp][j] = dot;
        }
        __syncthreads();
        if (threadIdx.x < k) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < BWD_THREADS / 32; ++w) s += part[w][threadIdx.x];
            dweights[t * k + threadIdx.x] = s;
        }
        __syncthreads();
    }
    int64_t used = *routed;
    used = used < 0 ? 0 : (used > rows ? rows : used);
    P zero{};
    for (int64_t r = used + blockIdx.x; r < rows; r += gridDim.x)
        for (int64_t c = threadIdx.x * P::N; c < hidden; c += BWD_THREADS * P::N)
            store_pack<T, VEC>(dys + r * hidden + c, zero);
}

// ---- host side ------------------------------------------------------------
bool is_act(int32_t dtype) {
    return dtype == CHELIS_DTYPE_F32 || dtype == CHELIS_DTYPE_BF16 || dtype == CHELIS_DTYPE_F16;
}
int64_t width(int32_t dtype) { return dtype == CHELIS_DTYPE_F32 ? 4 : 2; }
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_route(const char *op, int32_t dtype, int64_t tokens, int32_t experts, int32_t k) {
    if (!is_act(dtype)) return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "%s takes f32, bf16 or f16", op);
    if (tokens < 0 || experts < 1 || k < 1 || k > experts)
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "%s: tokens >= 0 and 1 <= k <= experts", op);
    if (experts > MAX_EXPERTS || k > MAX_K)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "%s admits %d experts and k = %d at most", op,
                         MAX_EXPERTS, MAX_K);
    if (tokens * k > INT32_MAX || tokens > INT32_MAX)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "%s: tokens * k above 2^31 - 1", op);
    return CHELIS_CUDA_OK;
}

int check_rows(const char *op, int32_t dtype, int64_t tokens, int32_t k, int64_t hidden) {
    CHELIS_TRY(check_route(op, dtype, tokens, MAX_EXPERTS, k));
    if (hidden < 0) return set_error(CHELIS_CUDA_ERR_DOMAIN, "%s: hidden >= 0", op);
    return CHELIS_CUDA_OK;
}

unsigned row_grid(int64_t warps) {
    const int64_t g = (warps + ROW_THREADS / 32 - 1) / (ROW_THREADS / 32);
    const int64_t cap = static_cast<int64_t>(sm_count()) * 8;
    return static_cast<unsigned>(g < 1 ? 1 : (g > cap ? cap : g));
}

template <typename T, int NV>
void launch_route(const void *logits, const int32_t *in_ids, const float *dw, int64_t tokens,
                  int experts, int k, int renorm, float *w, int32_t *ids, void *dl, cudaStream_t s) {
    const unsigned grid = static_cast<unsigned>((tokens + 7) / 8);
    if (dl)
        route_bwd_kernel<T, NV><<<grid, 256, 0, s>>>(static_cast<const T *>(logits), in_ids, dw, tokens,
                                                     experts, k, renorm, static_cast<T *>(dl));
    else
        route_kernel<T, NV><<<grid, 256, 0, s>>>(static_cast<const T *>(logits), tokens, experts, k,
                                                 renorm, w, ids);
}
template <typename T>
void pick_route(const void *logits, const int32_t *in_ids, const float *dw, int64_t tokens,
                int experts, int k, int renorm, float *w, int32_t *ids, void *dl, cudaStream_t s) {
    auto go = [&](auto f) { f(logits, in_ids, dw, tokens, experts, k, renorm, w, ids, dl, s); };
    if (experts <= 32) go(launch_route<T, 1>);
    else if (experts <= 64) go(launch_route<T, 2>);
    else if (experts <= 128) go(launch_route<T, 4>);
    else if (experts <= 256) go(launch_route<T, 8>);
    else go(launch_route<T, 32>);
}
int run_route(int32_t dtype, const void *logits, const int32_t *in_ids, const float *dw,
              int64_t tokens, int experts, int k, int renorm, float *w, int32_t *ids, void *dl) {
    cudaStream_t s = current_stream();
    auto go = [&](auto f) { f(logits, in_ids, dw, tokens, experts, k, renorm, w, ids, dl, s); };
    if (dtype == CHELIS_DTYPE_F32) go(pick_route<float>);
    else if (dtype == CHELIS_DTYPE_BF16) go(pick_route<__nv_bfloat16>);
    else go(pick_route<__half>);
    g_launches++;
    CHELIS_LAUNCH_CHECK("experts::route_kernel");
    return CHELIS_CUDA_OK;
}

// Run f<T, VEC> for the element type, in 16-byte packs where the row width
// and every base allow them.
template <typename F>
void by_type(int32_t dtype, bool vec, F f) {
    if (dtype == CHELIS_DTYPE_F32) vec ? f(float{}, std::true_type{}) : f(float{}, std::false_type{});
    else if (dtype == CHELIS_DTYPE_BF16)
        vec ? f(__nv_bfloat16{}, std::true_type{}) : f(__nv_bfloat16{}, std::false_type{});
    else vec ? f(__half{}, std::true_type{}) : f(__half{}, std::false_type{});
}

}  // namespace experts
}  // namespace chelis

using namespace chelis;

extern "C" int chelis_cuda_expert_route(int32_t dtype, const void *logits, int64_t tokens,
                                        int32_t n_experts, int32_t k, int renormalize,
                                        float *weights, int32_t *ids) {
    CHELIS_TRY(experts::check_route("expert_route", dtype, tokens, n_experts, k));
    if (tokens == 0) return CHELIS_CUDA_OK;
    if (!logits || !weights || !ids)
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "expert_route: null operand");
    return experts::run_route(dtype, logits, nullptr, nullptr, tokens, n_experts, k, renormalize != 0,
                              weights, ids, nullptr);
}

extern "C" int chelis_cuda_expert_route_bwd(int32_t dtype, const void *logits, const int32_t *ids,
                                            const float *dweights, int64_t tokens,
                                            int32_t n_experts, int32_t k, int renormalize,
                                            void *dlogits) {
    CHELIS_TRY(experts::check_route("expert_route_bwd", dtype, tokens, n_experts, k));
    if (tokens == 0) return CHELIS_CUDA_OK;
    if (!logits || !ids || !dweights || !dlogits)
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "expert_route_bwd: null operand");
    return experts::run_route(dtype, logits, ids, dweights, tokens, n_experts, k, renormalize != 0,
                              nullptr, nullptr, dlogits);
}

extern "C" int chelis_cuda_expert_sort(const int32_t *ids, int64_t tokens, int32_t k,
                                       int32_t n_experts, int32_t *offsets, int32_t *position,
                                       int32_t *source) {
    if (tokens < 0 || k < 1 || n_experts < 1)
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "expert_sort: tokens >= 0, k >= 1, experts >= 1");
    if (n_experts > experts::MAX_EXPERTS || k > experts::MAX_K)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "expert_sort admits %d experts and k = %d at most",
                         experts::MAX_EXPERTS, experts::MAX_K);
    const int64_t n = tokens * k;
    if (tokens > INT32_MAX || n > INT32_MAX)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "expert_sort: tokens * k above 2^31 - 1");
    if (!offsets) return set_error(CHELIS_CUDA_ERR_DOMAIN, "expert_sort: null operand");
    cudaStream_t s = current_stream();
    if (n == 0)
        return check_cuda(cudaMemsetAsync(offsets, 0, (n_experts + 1) * sizeof(int32_t), s), "memset");
    if (!ids || !position || !source)
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "expert_sort: null operand");
    const unsigned segments = static_cast<unsigned>((n + experts::SEGMENT - 1) / experts::SEGMENT);
    void *counts = nullptr;
    if (segments > 1) {
        CHELIS_TRY(scratch_alloc(&counts, sizeof(int32_t) * (segments + 1) * n_experts, s));
        experts::sort_count_kernel<<<segments, experts::SORT_THREADS, 0, s>>>(
            ids, n, n_experts, static_cast<int32_t *>(counts));
        g_launches++;
    }
    cudaLaunchAttribute early{};  // the next kernel's blocks start while the last of this one's run
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    const bool scanned = static_cast<int64_t>(segments) * n_experts >= experts::SCAN_FROM;
    if (scanned) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((n_experts + experts::SCAN_WIDTH - 1) / experts::SCAN_WIDTH);
        cfg.blockDim = dim3(experts::SCAN_THREADS);
        cfg.stream = s;
        cfg.attrs = &early;
        cfg.numAttrs = 1;
        const int rc = check_cuda(cudaLaunchKernelEx(&cfg, experts::sort_scan_kernel, static_cast<int32_t *>(counts),
                                                     static_cast<int64_t>(segments), static_cast<int>(n_experts)),
                                  "experts::sort_scan_kernel");
        if (rc != CHELIS_CUDA_OK) {
            scratch_free(counts, s);
            return rc;
        }
        g_launches++;
    }
    const size_t smem = sizeof(int) * (experts::SORT_WARPS + 2) * n_experts;
    // the last kernel counts its own pairs while the one before it finishes
    // (16384 x 2 by 8 6.8 us against 7.6; with more segments its waiting blocks
    // are in the way, 16384 x 8 by 64 12.4 against 11.0 without the scan)
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(segments);
    cfg.blockDim = dim3(experts::SORT_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = &early;
    cfg.numAttrs = segments > 1 && segments <= 64 ? 1 : 0;
    const int rc = check_cuda(cudaLaunchKernelEx(&cfg, experts::sort_place_kernel, ids, n, static_cast<int>(n_experts),
                                                 static_cast<int32_t *>(counts), static_cast<int>(scanned),
                                                 offsets, position, source),
                              "experts::sort_place_kernel");
    g_launches++;
    scratch_free(counts, s);
    return rc;
}

extern "C" int chelis_cuda_expert_spread(int32_t dtype, const void *x, const int32_t *position,
                                         const int32_t *routed, int64_t tokens, int32_t k,
                                         int64_t hidden, void *xs) {
    CHELIS_TRY(experts::check_rows("expert_spread", dtype, tokens, k, hidden));
    if (tokens == 0 || hidden == 0) return CHELIS_CUDA_OK;
    if (!x || !position || !routed || !xs)
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "expert_spread: null operand");
    cudaStream_t s = current_stream();
    const bool vec = hidden * experts::width(dtype) % 16 == 0 && experts::aligned16(x) &&
                     experts::aligned16(xs);
    experts::by_type(dtype, vec, [&](auto t, auto v) {
        using T = decltype(t);
        constexpr bool VEC = decltype(v)::value;
        const int64_t span = static_cast<int64_t>(32) * experts::WIDE * experts::Pack<T, VEC>::N;
        experts::spread_kernel<T, VEC>
            <<<experts::row_grid(tokens * ((hidden + span - 1) / span)), experts::ROW_THREADS, 0, s>>>(
                static_cast<const T *>(x), position, routed, tokens, k, hidden, static_cast<T *>(xs));
    });
    g_launches++;
    CHELIS_LAUNCH_CHECK("experts::spread_kernel");
    return CHELIS_CUDA_OK;
}

extern "C" int chelis_cuda_expert_combine(int32_t dtype, const void *ys, const float *weights,
                                          const int32_t *position, int64_t tokens, int32_t k,
                                          int64_t hidden, void *y) {
    CHELIS_TRY(experts::check_rows("expert_combine", dtype, tokens, k, hidden));
    if (tokens == 0 || hidden == 0) return CHELIS_CUDA_OK;
    if (!ys || !position || !y) return set_error(CHELIS_CUDA_ERR_DOMAIN, "expert_combine: null operand");
    cudaStream_t s = current_stream();
    const bool vec = hidden * experts::width(dtype) % 16 == 0 && experts::aligned16(ys) &&
                     experts::aligned16(y);
    experts::by_type(dtype, vec, [&](auto t, auto v) {
        using T = decltype(t);
        constexpr bool VEC = decltype(v)::value;
        const int64_t span = static_cast<int64_t>(32) * experts::DEEP * experts::Pack<T, VEC>::N;
        experts::combine_kernel<T, VEC>
            <<<experts::row_grid(tokens * ((hidden + span - 1) / span)), experts::ROW_THREADS, 0, s>>>(
                static_cast<const T *>(ys), weights, position, tokens, k, hidden, static_cast<T *>(y));
    });
    g_launches++;
    CHELIS_LAUNCH_CHECK("experts::combine_kernel");
    return CHELIS_CUDA_OK;
}

extern "C" int chelis_cuda_expert_combine_bwd(int32_t dtype, const void *dy, const void *ys,
                                              const float *weights, const int32_t *position,
                                              const int32_t *routed, int64_t tokens, int32_t k,
                                              int64_t hidden, void *dys, float *dweights) {
    CHELIS_TRY(experts::check_rows("expert_combine_bwd", dtype, tokens, k, hidden));
    if (tokens == 0) return CHELIS_CUDA_OK;
    if (!weights || !position || !routed || !dweights || (hidden > 0 && (!dy || !ys || !dys)))
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "expert_combine_bwd: null operand");
    cudaStream_t s = current_stream();
    const bool vec = hidden * experts::width(dtype) % 16 == 0 && experts::aligned16(dy) &&
                     experts::aligned16(ys) && experts::aligned16(dys);
    const int64_t cap = static_cast<int64_t>(sm_count()) * 16;
    const unsigned grid = static_cast<unsigned>(tokens < cap ? tokens : cap);
    experts::by_type(dtype, vec, [&](auto t, auto v) {
        using T = decltype(t);
        constexpr bool VEC = decltype(v)::value;
        experts::combine_bwd_kernel<T, VEC><<<grid, experts::BWD_THREADS, 0, s>>>(
            static_cast<const T *>(dy), static_cast<const T *>(ys), weights, position, routed, tokens,
            k, hidden, static_cast<T *>(dys), dweights);
    });
    g_launches++;
    CHELIS_LAUNCH_CHECK("experts::combine_bwd_kernel");
    return CHELIS_CUDA_OK;
}
