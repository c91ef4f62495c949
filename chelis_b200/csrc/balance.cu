// balance.cu -- how evenly a router deals its tokens out:
//
//   loss = E / (k N^2) sum_e c_e P_e,   P_e = sum_t softmax(l_t)_e
//   dl_te = E / (k N^2) p_te (c_e - sum_f p_tf c_f)
//
// over the N tokens that count, c_e their pairs of expert e (held constant by
// the gradient).  A warp takes a token, expert v * 32 + lane in the lane's value
// v, and keeps its lanes' sums of p over all of its tokens; blocks' sums and
// counts are added up in order by the last launch, so the loss does not depend
// on timing.  16384 x 64 with its gradient 14 us, 18 with eight warps a block and a
// token loaded as it was wanted; 64 x 8 6.2 us.  Bound by the launches: the host's two
// calls take longer (25 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "common.cuh"

namespace chelis {

extern std::atomic<uint64_t> g_launches;

namespace balance {

using experts::from_f32;
using experts::to_f32;
using experts::warp_sum;

constexpr int THREADS = 256, WARPS = THREADS / 32;  // of the gradient
// Warps of a block of partial_kernel, as many as its shared sums allow.
constexpr int block_warps(int nv) { return nv <= 2 ? 32 : nv <= 8 ? 16 : 8; }
constexpr int FOLD_THREADS = 1024;

// The lane's probabilities of a token, 0 for experts at -inf (NaN where a logit
// is NaN or +inf).
template <typename T, int NV>
__device__ __forceinline__ void load_row(const T *row, int experts, int lane, float (&p)[NV]) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int i = v * 32 + lane;
        p[v] = i < experts ? to_f32(row[i]) : -INFINITY;
    }
}
template <int NV>
__device__ __forceinline__ void softmax(float (&p)[NV]) {
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v) top = fmaxf(top, p[v]);
    top = warp_max(top);
    const float base = top > -INFINITY ? top : 0.0f;  // a row of -inf: all 0
    float z = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        p[v] = expf(p[v] - base);
        z += p[v];
    }
    z = warp_sum(z);
    const float r = z != 0.0f ? 1.0f / z : 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) p[v] *= r;
}

// The loss from P and c, by one block: thread sums in order, then a tree.
__device__ void finish(const float *probs, const int32_t *counts, int experts, int tokens, int k, float *loss) {
    __shared__ double part[32];
    double s = 0.0;
    for (int e = threadIdx.x; e < experts; e += blockDim.x) s += static_cast<double>(probs[e]) * counts[e];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int w = 0; w < static_cast<int>(blockDim.x) / 32; ++w) s += part[w];
        const double n = tokens > 0 ? tokens : 1;
        *loss = static_cast<float>(s * experts / (k * n * n));
    }
}

// probs [blocks][experts], counts [blocks][experts + 1]; of one block: the results.
// A token's logits and ids are read while the one before it is worked on.
template <typename T, int NV>
__global__ void __launch_bounds__(32 * block_warps(NV))
    partial_kernel(const T *__restrict__ logits, const int32_t *__restrict__ ids, const uint8_t *__restrict__ mask,
                   int64_t tokens, int experts, int k, float *probs, int32_t *counts, float *loss) {
    constexpr int WARPS = block_warps(NV), THREADS = 32 * WARPS;
    extern __shared__ float shared_sums[];  // [WARPS][experts]
    __shared__ int hist[experts::MAX_EXPERTS], live;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int e = threadIdx.x; e < experts; e += THREADS) hist[e] = 0;
    if (threadIdx.x == 0) live = 0;
    __syncthreads();
    float sum[NV], next[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) sum[v] = 0.0f;
    int mine = 0, next_id = -1;
    bool next_live = false;
    const int64_t step = static_cast<int64_t>(gridDim.x) * WARPS;
    auto load = [&](int64_t t) {
        next_live = t < tokens && (!mask || mask[t]);
        if (!next_live) return;
        load_row<T, NV>(logits + t * experts, experts, lane, next);
        next_id = lane < k ? ids[t * k + lane] : -1;
    };
    int64_t t = static_cast<int64_t>(blockIdx.x) * WARPS + warp;
    load(t);
    for (; t < tokens; t += step) {
        const bool counted = next_live;
        const int id = next_id;
        float p[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) p[v] = next[v];
        load(t + step);
        if (!counted) continue;
        ++mine;
        if (id >= 0 && id < experts) atomicAdd(&hist[id], 1);
        else if (id != -1) report_device_error(DEVERR_BAD_INDEX);
        softmax<NV>(p);
#pragma unroll
        for (int v = 0; v < NV; ++v) sum[v] += p[v];
    }
    if (lane == 0 && mine) atomicAdd(&live, mine);
#pragma unroll
    for (int v = 0; v < NV; ++v)
        if (v * 32 + lane < experts) shared_sums[warp * experts + v * 32 + lane] = sum[v];
    __syncthreads();
    float *out = gridDim.x > 1 ? probs + static_cast<int64_t>(blockIdx.x) * experts : shared_sums;
    int32_t *c = gridDim.x > 1 ? counts + static_cast<int64_t>(blockIdx.x) * (experts + 1) : counts;
    for (int e = threadIdx.x; e < experts; e += THREADS) {
        float s = 0.0f;
#pragma unroll 8
        for (int w = 0; w < WARPS; ++w) s += shared_sums[w * experts + e];
        out[e] = s;
        c[e] = hist[e];
    }
    if (threadIdx.x == 0) c[experts] = live;
    if (gridDim.x == 1) {
        __syncthreads();
        finish(shared_sums, hist, experts, live, k, loss);
    }
}

// The blocks' sums in order: `slices` threads an expert take consecutive shares.
__global__ void __launch_bounds__(FOLD_THREADS)
    fold_kernel(const float *probs, const int32_t *parts, int blocks, int experts, int slices, int k, int32_t *counts,
                float *loss) {
    extern __shared__ float fold_smem[];  // probs, then counts: [slices][experts + 1] each
    const int width = experts + 1;
    int *csum = reinterpret_cast<int *>(fold_smem + slices * width);
    const int per = (blocks + slices - 1) / slices;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int i = threadIdx.x; i < slices * width; i += FOLD_THREADS) {
        const int slice = i / width, e = i - slice * width;
        const int first = slice * per, last = min(blocks, first + per);
        float s = 0.0f;
        int c = 0;
#pragma unroll 8
        for (int b = first; b < last; ++b) {
            if (e < experts) s += probs[b * experts + e];
            c += parts[b * width + e];
        }
        fold_smem[i] = s;
        csum[i] = c;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < width; e += FOLD_THREADS) {
        float s = 0.0f;
        int c = 0;
        for (int i = 0; i < slices; ++i) s += fold_smem[i * width + e], c += csum[i * width + e];
        fold_smem[e] = s;
        csum[e] = c;
        counts[e] = c;
    }
    __syncthreads();
    finish(fold_smem, csum, experts, csum[experts], k, loss);
}

template <typename T, int NV>
__global__ void __launch_bounds__(THREADS)
    bwd_kernel(const T *__restrict__ logits, const int32_t *__restrict__ counts, const uint8_t *__restrict__ mask,
               int64_t tokens, int experts, int k, float weight, const float *__restrict__ dloss, const T *add,
               T *dlogits) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float c[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) c[v] = v * 32 + lane < experts ? static_cast<float>(counts[v * 32 + lane]) : 0.0f;
    const float n = fmaxf(static_cast<float>(counts[experts]), 1.0f);
    const float each = weight * (dloss ? *dloss : 1.0f) * (static_cast<float>(experts) / (static_cast<float>(k) * n)) / n;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * WARPS + warp; t < tokens; t += static_cast<int64_t>(gridDim.x) * WARPS) {
        float p[NV];
        const bool counted = !mask || mask[t];
        if (counted) {
            load_row<T, NV>(logits + t * experts, experts, lane, p);
            softmax<NV>(p);
            float inner = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v) inner = fmaf(p[v], c[v], inner);
            inner = warp_sum(inner);
#pragma unroll
            for (int v = 0; v < NV; ++v) p[v] = each * (p[v] * (c[v] - inner));
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int i = v * 32 + lane;
            if (i < experts) {
                const float d = counted ? p[v] : 0.0f;
                dlogits[t * experts + i] = from_f32<T>(add ? to_f32(add[t * experts + i]) + d : d);
            }
        }
    }
}

// f(T, NV)
template <typename F>
void by_experts(int32_t dtype, int experts, F f) {
    experts::by_type(dtype, true, [&](auto t, auto) {
        if (experts <= 32) f(t, std::integral_constant<int, 1>{});
        else if (experts <= 64) f(t, std::integral_constant<int, 2>{});
        else if (experts <= 128) f(t, std::integral_constant<int, 4>{});
        else if (experts <= 256) f(t, std::integral_constant<int, 8>{});
        else f(t, std::integral_constant<int, 32>{});
    });
}

}  // namespace balance
}  // namespace chelis

using namespace chelis;

extern "C" int chelis_cuda_expert_balance(int32_t dtype, const void *logits, const int32_t *ids, const uint8_t *mask,
                                          int64_t tokens, int32_t n_experts, int32_t k, float *loss, int32_t *counts) {
    CHELIS_TRY(experts::check_route("expert_balance", dtype, tokens, n_experts, k));
    if (!loss || !counts || (tokens > 0 && (!logits || !ids)))
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "expert_balance: null operand");
    cudaStream_t s = current_stream();
    // one block where its warps have few tokens each
    const int64_t warps = balance::block_warps(n_experts <= 64 ? 1 : n_experts <= 256 ? 8 : 32);
    int64_t blocks = tokens <= 4 * warps ? 1 : (tokens + warps - 1) / warps;
    if (blocks > sm_count()) blocks = sm_count();
    void *scratch = nullptr;
    const size_t probs_n = static_cast<size_t>(blocks) * n_experts, counts_n = static_cast<size_t>(blocks) * (n_experts + 1);
    if (blocks > 1) CHELIS_TRY(scratch_alloc(&scratch, (probs_n + counts_n) * 4, s));
    float *probs = static_cast<float *>(scratch);
    int32_t *parts = blocks > 1 ? reinterpret_cast<int32_t *>(probs + probs_n) : counts;
    balance::by_experts(dtype, n_experts, [&](auto t, auto nv) {
        using T = decltype(t);
        balance::partial_kernel<T, decltype(nv)::value>
            <<<static_cast<unsigned>(blocks), static_cast<unsigned>(32 * warps), warps * n_experts * 4, s>>>(
                static_cast<const T *>(logits), ids, mask, tokens, n_experts, k, probs, parts, loss);
    });
    g_launches++;
    int rc = check_cuda(cudaGetLastError(), "balance::partial_kernel");
    if (rc == CHELIS_CUDA_OK && blocks > 1) {
        int slices = balance::FOLD_THREADS / (n_experts + 1);
        slices = slices < 1 ? 1 : (slices > blocks ? static_cast<int>(blocks) : slices);
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(1);
        cfg.blockDim = dim3(balance::FOLD_THREADS);
        cfg.dynamicSmemBytes = static_cast<size_t>(slices) * (n_experts + 1) * 8;
        cfg.stream = s;
        cudaLaunchAttribute attr[1]{};
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        rc = check_cuda(cudaLaunchKernelEx(&cfg, balance::fold_kernel, static_cast<const float *>(probs),
                                           static_cast<const int32_t *>(parts), static_cast<int>(blocks),
                                           static_cast<int>(n_experts), slices, static_cast<int>(k), counts, loss),
                        "balance::fold_kernel");
        g_launches++;
    }
    scratch_free(scratch, s);
    return rc;
}

extern "C" int chelis_cuda_expert_balance_bwd(int32_t dtype, const void *logits, const int32_t *counts,
                                              const uint8_t *mask, int64_t tokens, int32_t n_experts, int32_t k,
                                              float weight, const float *dloss, const void *add, void *dlogits) {
    CHELIS_TRY(experts::check_route("expert_balance_bwd", dtype, tokens, n_experts, k));
    if (tokens == 0) return CHELIS_CUDA_OK;
    if (!logits || !counts || !dlogits) return set_error(CHELIS_CUDA_ERR_DOMAIN, "expert_balance_bwd: null operand");
    balance::by_experts(dtype, n_experts, [&](auto t, auto nv) {
        using T = decltype(t);
        balance::bwd_kernel<T, decltype(nv)::value>
            <<<blocks8::grid_for((tokens + balance::WARPS - 1) / balance::WARPS, 8), balance::THREADS, 0, current_stream()>>>(
                static_cast<const T *>(logits), counts, mask, tokens, n_experts, k, weight, dloss,
                static_cast<const T *>(add), static_cast<T *>(dlogits));
    });
    g_launches++;
    CHELIS_LAUNCH_CHECK("balance::bwd_kernel");
    return CHELIS_CUDA_OK;
}
