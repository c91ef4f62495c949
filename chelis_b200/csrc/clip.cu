// clip.cu -- the norm of all gradients of a step and their scaling to a bound:
//
//   norm = sqrt(sum_i sum g_i^2),   out_i = g_i min(1, max_norm / norm)
//
// over many tensors of f32, bf16 or f16 in two launches.  The tensors' table
// travels with the launch; the numbers are dealt out in chunks that no tensor's
// end is cut across, so that a block has the same amount to do whether the
// tensors are a few large ones or hundreds of small ones.  A thread squares and
// adds a few numbers in f32 and keeps their sum in f64, or all of it in f64 where
// the squares leave f32; blocks' sums are added up in order, so the norm does not
// depend on timing.  Memory bounds it; in the second launch each block goes through
// its chunks backwards, from what the first has left in L2.  240 tensors of 1e8 numbers,
// bf16 to f32: 150 us on the device (40 for the norm, 200 MB at 5.0 TB/s, and 110, 600 MB at
// 5.4), behind a call that takes 172 of the host, 142 of them for the list of 480 tensors.
// 16-byte halves of a sector a lane took 155 for the 110.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <new>
#include <vector>

#include "common.cuh"

namespace chelis {

extern std::atomic<uint64_t> g_launches;

namespace clip {

constexpr int THREADS = 512;
constexpr int CHUNK = 32768;   // numbers of a chunk
constexpr int FEW = 32, MANY = 768;  // tensors of a launch: two sizes of table

struct Entry {
    const void *src;
    void *dst;
    int64_t count;
    int32_t first;  // chunks before this tensor's
    uint8_t in, out, pad[2];
};
template <int N>
struct Table {
    Entry t[N];
    int32_t n, chunks;
};
static_assert(sizeof(Table<MANY>) < 32000, "kernel parameters");

template <typename T>
__device__ __forceinline__ void wide(uint4 u, float (&v)[16 / sizeof(T)]) {
    const T *p = reinterpret_cast<const T *>(&u);
#pragma unroll
    for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) v[i] = experts::to_f32(p[i]);
}

// Squares of a few numbers: in f32, or in f64 where that over- or underflows
// (below 2^-100 a square may have lost digits).
template <int N>
__device__ __forceinline__ double squares(const float (&v)[N]) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(v[i], v[i], s);
    if (s > 0x1p-100f && s < 0x1p126f) return s;
    double d = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) d = fma(static_cast<double>(v[i]), static_cast<double>(v[i]), d);
    return d;
}

// `count` numbers by THREADS threads: single ones up to 16 bytes' alignment, packs,
// single ones.  READ_ONLY: no one writes them in this launch.
template <bool READ_ONLY>
__device__ __forceinline__ uint4 load_packed(const uint4 *p) {
    if constexpr (READ_ONLY) return __ldg(p);
    else return *p;
}
template <int THREADS, bool READ_ONLY, typename T>
__device__ __forceinline__ double chunk_squares(const T *p, int64_t count, int thread) {
    constexpr int N = 16 / sizeof(T), DEEP = 8;
    double sum = 0.0;
    const int64_t skew = (16 - (reinterpret_cast<uintptr_t>(p) & 15)) % 16 / sizeof(T);
    const int64_t head = skew < count ? skew : count, packs = (count - head) / N;
    const uint4 *q = reinterpret_cast<const uint4 *>(p + head);
    int64_t i = thread;
    for (; i + (DEEP - 1) * THREADS < packs; i += DEEP * THREADS) {
        uint4 u[DEEP];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) u[d] = load_packed<READ_ONLY>(q + i + d * THREADS);
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            float v[N];
            wide<T>(u[d], v);
            sum += squares(v);
        }
    }
    for (; i < packs; i += THREADS) {
        float v[N];
        wide<T>(load_packed<READ_ONLY>(q + i), v);
        sum += squares(v);
    }
    const int64_t tail = head + packs * N;
    if (thread < head) {
        const double v = experts::to_f32(p[thread]);
        sum = fma(v, v, sum);
    }
    if (tail + thread < count) {
        const double v = experts::to_f32(p[tail + thread]);
        sum = fma(v, v, sum);
    }
    return sum;
}

template <int THREADS, bool READ_ONLY>
__device__ __forceinline__ double squares_part(const Entry &e, int64_t at, int64_t count, int thread) {
    if (e.in == CHELIS_DTYPE_F32) return chunk_squares<THREADS, READ_ONLY>(static_cast<const float *>(e.src) + at, count, thread);
    if (e.in == CHELIS_DTYPE_BF16)
        return chunk_squares<THREADS, READ_ONLY>(static_cast<const __nv_bfloat16 *>(e.src) + at, count, thread);
    return chunk_squares<THREADS, READ_ONLY>(static_cast<const __half *>(e.src) + at, count, thread);
}

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[THREADS / 32];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) v += part[w];
    __syncthreads();
    return v;
}

// A block takes consecutive chunks: looking for each chunk's tensor in the table,
// which the constant cache does not hold, had cost as much as reading the chunk.
__device__ __forceinline__ int block_first(int chunks, unsigned block) {
    return static_cast<int>(static_cast<int64_t>(chunks) * block / gridDim.x);
}
template <int N>
__device__ __forceinline__ int tensor_of(const Table<N> &table, int chunk) {
    int lo = 0, hi = table.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (table.t[mid].first <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <int N>
__global__ void __launch_bounds__(THREADS, 2)
    norm_kernel(const __grid_constant__ Table<N> table, double *sums) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    double sum = 0.0;
    const int first = block_first(table.chunks, blockIdx.x), last = block_first(table.chunks, blockIdx.x + 1);
    int tensor = tensor_of(table, first);
    for (int c = first; c < last; ++c) {
        while (tensor + 1 < table.n && table.t[tensor + 1].first <= c) ++tensor;
        const Entry &e = table.t[tensor];
        const int64_t at = static_cast<int64_t>(c - e.first) * CHUNK;
        const int64_t count = e.count - at < CHUNK ? e.count - at : CHUNK;
        sum += squares_part<THREADS, true>(e, at, count, threadIdx.x);
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// The blocks' sums in order of the threads: every block comes to the same norm.
__device__ __forceinline__ double total_norm(const double *sums, int n) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += THREADS) v += sums[i];
    return sqrt(block_sum(v));
}
__global__ void __launch_bounds__(THREADS)
    total_kernel(const double *sums, int n, float *norm) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const double v = total_norm(sums, n);
    if (threadIdx.x == 0) *norm = static_cast<float>(v);
}

// What the numbers are multiplied by.
struct Factor {
    float f;
    double tiny;  // f itself where it is below 2^-126, of which f32 lacks digits; else 0
};

template <int THREADS, typename T, typename U>
__device__ __forceinline__ void scale_chunk(const T *p, U *o, int64_t count, Factor factor, int thread) {
    constexpr int N = 16 / sizeof(T), DEEP = 8;
    if (factor.tiny != 0.0) {
        for (int64_t i = thread; i < count; i += THREADS)
            o[i] = experts::from_f32<U>(static_cast<float>(static_cast<double>(experts::to_f32(p[i])) * factor.tiny));
        return;
    }
    const float c = factor.f;
    const int64_t skew = (16 - (reinterpret_cast<uintptr_t>(p) & 15)) % 16 / sizeof(T);
    int64_t head = skew < count ? skew : count;
    // packs want the result aligned as well as the source
    const bool packed = (reinterpret_cast<uintptr_t>(o + head) & (N * sizeof(U) - 1)) == 0;
    if (!packed) {
        for (int64_t i = thread; i < count; i += THREADS) o[i] = experts::from_f32<U>(experts::to_f32(p[i]) * c);
        return;
    }
    const int64_t packs = (count - head) / N;
    const uint4 *q = reinterpret_cast<const uint4 *>(p + head);
    auto put = [&](int64_t i, uint4 u) {
        float v[N];
        wide<T>(u, v);
        struct alignas(N * sizeof(U)) Out {
            U v[N];
        } r;
#pragma unroll
        for (int j = 0; j < N; ++j) r.v[j] = experts::from_f32<U>(v[j] * c);
        // 16 bits to f32: a whole sector at once
        if constexpr (sizeof(r) == 32) gemm8::store32(o + head + i * N, reinterpret_cast<const uint32_t(&)[8]>(r));
        else *reinterpret_cast<Out *>(o + head + i * N) = r;
    };
    int64_t i = thread;
    for (; i + (DEEP - 1) * THREADS < packs; i += DEEP * THREADS) {
        uint4 u[DEEP];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) u[d] = q[i + d * THREADS];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) put(i + d * THREADS, u[d]);
    }
    for (; i < packs; i += THREADS) put(i, q[i]);
    const int64_t tail = head + packs * N;
    if (thread < head) o[thread] = experts::from_f32<U>(experts::to_f32(p[thread]) * c);
    if (tail + thread < count)
        o[tail + thread] = experts::from_f32<U>(experts::to_f32(p[tail + thread]) * c);
}
template <int THREADS, typename T>
__device__ __forceinline__ void scale_as(const Entry &e, int64_t at, int64_t count, Factor c, int thread) {
    const T *p = static_cast<const T *>(e.src) + at;
    if (e.out == CHELIS_DTYPE_F32) scale_chunk<THREADS>(p, static_cast<float *>(e.dst) + at, count, c, thread);
    else if (e.out == CHELIS_DTYPE_BF16) scale_chunk<THREADS>(p, static_cast<__nv_bfloat16 *>(e.dst) + at, count, c, thread);
    else scale_chunk<THREADS>(p, static_cast<__half *>(e.dst) + at, count, c, thread);
}

template <int THREADS>
__device__ __forceinline__ void scale_part(const Entry &e, int64_t at, int64_t count, Factor c, int thread) {
    if (e.in == CHELIS_DTYPE_F32) scale_as<THREADS, float>(e, at, count, c, thread);
    else if (e.in == CHELIS_DTYPE_BF16) scale_as<THREADS, __nv_bfloat16>(e, at, count, c, thread);
    else scale_as<THREADS, __half>(e, at, count, c, thread);
}

// A norm that is reported as infinite or NaN changes nothing.
__device__ __forceinline__ Factor factor(double norm, float max_norm) {
    if (!(norm > max_norm && static_cast<float>(norm) < INFINITY)) return {1.0f, 0.0};
    const double c = max_norm / norm;
    return {static_cast<float>(c), c < 0x1p-126 ? c : 0.0};
}

template <int N>
__global__ void __launch_bounds__(THREADS, 2)
    scale_kernel(const __grid_constant__ Table<N> table, const double *sums, int n, float max_norm, float *norm) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const double v = total_norm(sums, n);
    if (blockIdx.x == 0 && threadIdx.x == 0 && norm) *norm = static_cast<float>(v);
    const Factor c = factor(v, max_norm);
    const int first = block_first(table.chunks, blockIdx.x), last = block_first(table.chunks, blockIdx.x + 1);
    int tensor = first < last ? tensor_of(table, last - 1) : 0;
    for (int chunk = last - 1; chunk >= first; --chunk) {
        while (table.t[tensor].first > chunk) --tensor;
        const Entry &e = table.t[tensor];
        if (c.f == 1.0f && e.src == e.dst) continue;  // as they are
        const int64_t at = static_cast<int64_t>(chunk - e.first) * CHUNK;
        const int64_t count = e.count - at < CHUNK ? e.count - at : CHUNK;
        scale_part<THREADS>(e, at, count, c, threadIdx.x);
    }
}

// Few numbers: all of them by one block, which needs no scratch and no second
// launch; a warp takes a chunk.
constexpr int64_t FEW_NUMBERS = 65536;
constexpr int FEW_CHUNK = 1024;

template <bool SCALE>
__global__ void __launch_bounds__(THREADS)
    small_kernel(const __grid_constant__ Table<FEW> table, float max_norm, float *norm) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    double sum = 0.0;
    for (int c = warp; c < table.chunks; c += THREADS / 32) {
        const Entry &e = table.t[tensor_of(table, c)];
        const int64_t at = static_cast<int64_t>(c - e.first) * FEW_CHUNK;
        sum += squares_part<32, !SCALE>(e, at, e.count - at < FEW_CHUNK ? e.count - at : FEW_CHUNK, lane);
    }
    const double v = sqrt(block_sum(sum));
    if (threadIdx.x == 0) *norm = static_cast<float>(v);
    if (!SCALE) return;
    const Factor c = factor(v, max_norm);
    for (int chunk = warp; chunk < table.chunks; chunk += THREADS / 32) {
        const Entry &e = table.t[tensor_of(table, chunk)];
        if (c.f == 1.0f && e.src == e.dst) continue;
        const int64_t at = static_cast<int64_t>(chunk - e.first) * FEW_CHUNK;
        scale_part<32>(e, at, e.count - at < FEW_CHUNK ? e.count - at : FEW_CHUNK, c, lane);
    }
}

// ---- host side ------------------------------------------------------------
int check(const char *op, int32_t n, const void *const *data, const int64_t *counts, const int32_t *dtypes) {
    if (n < 0) return set_error(CHELIS_CUDA_ERR_DOMAIN, "%s: tensors >= 0", op);
    if (n > 0 && (!data || !counts || !dtypes)) return set_error(CHELIS_CUDA_ERR_DOMAIN, "%s: null operand", op);
    for (int32_t i = 0; i < n; ++i) {
        if (!experts::is_act(dtypes[i])) return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "%s takes f32, bf16 or f16", op);
        if (counts[i] < 0) return set_error(CHELIS_CUDA_ERR_DOMAIN, "%s: counts >= 0", op);
        if (counts[i] > 0 && !data[i]) return set_error(CHELIS_CUDA_ERR_DOMAIN, "%s: null operand", op);
        if (counts[i] > (static_cast<int64_t>(INT32_MAX) - MANY) / MANY * CHUNK)
            return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "%s: a tensor of more than 4e10 numbers", op);
        if (reinterpret_cast<uintptr_t>(data[i]) % experts::width(dtypes[i]) != 0)
            return set_error(CHELIS_CUDA_ERR_DOMAIN, "%s: a tensor that does not lie on its numbers' size", op);
    }
    return CHELIS_CUDA_OK;
}

struct Span {
    uintptr_t lo, hi;
    int32_t i;
};
// Outputs lie apart from one another, and from the inputs but their own.
int check_spans(int32_t n, const void *const *data, const int64_t *counts, const int32_t *dtypes, void *const *out,
                const int32_t *out_dtypes) {
    std::vector<Span> spans;
    try {
        spans.reserve(static_cast<size_t>(n));
        for (int32_t i = 0; i < n; ++i)
            if (counts[i] > 0) {
                const uintptr_t at = reinterpret_cast<uintptr_t>(out[i]);
                spans.push_back({at, at + static_cast<uintptr_t>(counts[i] * experts::width(out_dtypes[i])), i});
            }
    } catch (const std::bad_alloc &) {
        return set_error(CHELIS_CUDA_ERR_FAIL, "clip_grads: out of host memory");
    }
    std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.lo < b.lo; });
    for (size_t i = 1; i < spans.size(); ++i)
        if (spans[i].lo < spans[i - 1].hi)
            return set_error(CHELIS_CUDA_ERR_DOMAIN, "clip_grads: results %d and %d overlap", spans[i - 1].i, spans[i].i);
    for (int32_t i = 0; i < n; ++i) {
        if (counts[i] == 0) continue;
        const uintptr_t lo = reinterpret_cast<uintptr_t>(data[i]), hi = lo + static_cast<uintptr_t>(counts[i] * experts::width(dtypes[i]));
        if (data[i] == out[i] && dtypes[i] == out_dtypes[i]) continue;  // then no other result is there
        auto it = std::lower_bound(spans.begin(), spans.end(), lo, [](const Span &s, uintptr_t v) { return s.hi <= v; });
        if (it != spans.end() && it->lo < hi)
            return set_error(CHELIS_CUDA_ERR_DOMAIN, "clip_grads: result %d overlaps tensor %d", it->i, i);
    }
    return CHELIS_CUDA_OK;
}

unsigned grid_of(int32_t chunks, int per_sm) {
    const int64_t cap = static_cast<int64_t>(sm_count()) * per_sm;
    return static_cast<unsigned>(chunks < 1 ? 1 : (chunks > cap ? cap : chunks));
}

template <typename... Args, typename... Given>
int launch_after(void (*kernel)(Args...), unsigned grid, const char *name, Given... given) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = current_stream();
    cudaLaunchAttribute attr[1]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CHELIS_TRY(check_cuda(cudaLaunchKernelEx(&cfg, kernel, given...), name));
    g_launches++;
    return CHELIS_CUDA_OK;
}

constexpr int NORM_BLOCKS = 2, SCALE_BLOCKS = 2;  // a multiprocessor

// f(table) for tensors `first` on, as many as a table has; the next first.
template <int N, int CHUNK, typename F>
int with_table(int32_t *first, int32_t n, const void *const *data, const int64_t *counts, const int32_t *dtypes,
               void *const *out, const int32_t *out_dtypes, F f) {
    Table<N> table;
    table.n = 0;
    int64_t chunks = 0;
    while (*first < n && table.n < N) {
        const int32_t i = (*first)++;
        if (counts[i] == 0) continue;
        Entry &e = table.t[table.n++];
        e = Entry{data[i], out ? out[i] : nullptr, counts[i], static_cast<int32_t>(chunks), static_cast<uint8_t>(dtypes[i]),
                  static_cast<uint8_t>(out ? out_dtypes[i] : 0), {}};
        chunks += (counts[i] + CHUNK - 1) / CHUNK;
    }
    table.chunks = static_cast<int32_t>(chunks);
    return f(table);
}

template <int N>
int run(int32_t n, const void *const *data, const int64_t *counts, const int32_t *dtypes, void *const *out,
        const int32_t *out_dtypes, float max_norm, float *norm) {
    cudaStream_t s = current_stream();
    if constexpr (N == FEW) {
        int64_t numbers = 0;
        for (int32_t i = 0; i < n && numbers <= FEW_NUMBERS; ++i) numbers += counts[i];
        if (numbers <= FEW_NUMBERS) {
            int32_t first = 0;
            return with_table<FEW, FEW_CHUNK>(&first, n, data, counts, dtypes, out, out_dtypes, [&](const Table<FEW> &table) -> int {
                if (out) small_kernel<true><<<1, THREADS, 0, s>>>(table, max_norm, norm);
                else small_kernel<false><<<1, THREADS, 0, s>>>(table, max_norm, norm);
                g_launches++;
                CHELIS_LAUNCH_CHECK("clip::small_kernel");
                return CHELIS_CUDA_OK;
            });
        }
    }
    const int64_t tables = (static_cast<int64_t>(n) + N - 1) / N, most = sm_count() * NORM_BLOCKS;
    void *scratch = nullptr;
    CHELIS_TRY(scratch_alloc(&scratch, static_cast<size_t>((tables < 1 ? 1 : tables) * most) * sizeof(double), s));
    double *sums = static_cast<double *>(scratch);
    auto body = [&]() -> int {
        int blocks = 0;
        for (int32_t first = 0; first < n;)
            CHELIS_TRY((with_table<N, CHUNK>(&first, n, data, counts, dtypes, out, out_dtypes, [&](const Table<N> &table) -> int {
                if (table.chunks == 0) return CHELIS_CUDA_OK;
                const unsigned grid = grid_of(table.chunks, NORM_BLOCKS);
                norm_kernel<N><<<grid, THREADS, 0, s>>>(table, sums + blocks);
                g_launches++;
                CHELIS_LAUNCH_CHECK("clip::norm_kernel");
                blocks += static_cast<int>(grid);
                return CHELIS_CUDA_OK;
            })));
        if (!out || blocks == 0)
            return launch_after(total_kernel, 1, "clip::total_kernel", static_cast<const double *>(sums), blocks, norm);
        float *report = norm;  // by the first launch alone
        for (int32_t first = 0; first < n;)
            CHELIS_TRY((with_table<N, CHUNK>(&first, n, data, counts, dtypes, out, out_dtypes, [&](const Table<N> &table) -> int {
                if (table.chunks == 0) return CHELIS_CUDA_OK;
                CHELIS_TRY(launch_after(scale_kernel<N>, grid_of(table.chunks, SCALE_BLOCKS), "clip::scale_kernel", table,
                                        static_cast<const double *>(sums), blocks, max_norm, report));
                report = nullptr;
                return CHELIS_CUDA_OK;
            })));
        return CHELIS_CUDA_OK;
    };
    const int rc = body();
    scratch_free(scratch, s);
    return rc;
}

}  // namespace clip
}  // namespace chelis

using namespace chelis;

extern "C" int chelis_cuda_grad_norm(int32_t n, const void *const *data, const int64_t *counts, const int32_t *dtypes,
                                     float *norm) {
    CHELIS_TRY(clip::check("grad_norm", n, data, counts, dtypes));
    if (!norm) return set_error(CHELIS_CUDA_ERR_DOMAIN, "grad_norm: null operand");
    if (n <= clip::FEW) return clip::run<clip::FEW>(n, data, counts, dtypes, nullptr, nullptr, 0.0f, norm);
    return clip::run<clip::MANY>(n, data, counts, dtypes, nullptr, nullptr, 0.0f, norm);
}

extern "C" int chelis_cuda_clip_grads(int32_t n, const void *const *data, const int64_t *counts, const int32_t *dtypes,
                                      void *const *out, const int32_t *out_dtypes, float max_norm, float *norm) {
    CHELIS_TRY(clip::check("clip_grads", n, data, counts, dtypes));
    if (!norm || (n > 0 && !out)) return set_error(CHELIS_CUDA_ERR_DOMAIN, "clip_grads: null operand");
    CHELIS_TRY(clip::check("clip_grads", n, const_cast<const void *const *>(out), counts, out_dtypes));
    if (!(max_norm >= 0.0f)) return set_error(CHELIS_CUDA_ERR_DOMAIN, "clip_grads: max_norm >= 0");
    CHELIS_TRY(clip::check_spans(n, data, counts, dtypes, out, out_dtypes));
    if (n <= clip::FEW) return clip::run<clip::FEW>(n, data, counts, dtypes, out, out_dtypes, max_norm, norm);
    return clip::run<clip::MANY>(n, data, counts, dtypes, out, out_dtypes, max_norm, norm);
}
