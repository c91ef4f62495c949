// blocks8.cu -- matrices in 8-bit floating point with one scale for each
// block of 128, quantised from f32, bf16 or f16.  No counterpart in the
// reference (its dtypes end at 16 bits).
//
// A block's scale is the least power of two s = 2^e (e >= -126) with
// max|x| / s <= the format's largest value (448 for e4m3, 57344 for e5m2),
// 1 for a block of zeros.  Dividing by a power of two is exact, so a number
// is rounded once, to nearest even, and the same bits come out whatever the
// order or the width of the arithmetic.  Infinities and NaNs do not enter the
// maximum: a NaN stays a NaN, an infinity stays one in e5m2 and is a NaN in
// e4m3, which has none.
//
// Three layouts (ld = the contiguous extent rounded up to 16, the rest zero):
//   rows        data [rows][ld(cols)], scales [ceil(cols/128)][rows]
//   tiles       data [batch][rows][ld(cols)], scales [batch][ceil(rows/128)][ceil(cols/128)]
//   transposed  data [cols][places], scales [places/128][cols]: x's rows along
//               the contiguous axis, every expert's rows starting on a block
//               of 128 (the places in between hold zero)
// Each is one pass over x: read once, 1 byte an element written.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "common.cuh"

namespace chelis {

namespace blocks8 {

constexpr int BLOCK = 128;
constexpr int THREADS = 256;
constexpr int MAX_GROUPS = experts::MAX_EXPERTS;

using experts::Pack;
using experts::to_f32;

// 8 consecutive elements from p[0..valid), zeros beyond.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *p, int64_t valid, float (&v)[8]) {
    if (VEC && valid >= 8) {
        constexpr int N = 16 / static_cast<int>(sizeof(T));
#pragma unroll
        for (int u = 0; u < 8 / N; ++u) {
            const Pack<T, true> r = experts::load_pack<T, true>(p + u * N);
#pragma unroll
            for (int i = 0; i < N; ++i) v[u * N + i] = to_f32(r.v[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < valid ? to_f32(p[i]) : 0.0f;
    }
}

__device__ __forceinline__ float finite_abs(float v) {
    const float a = fabsf(v);
    return a < INFINITY ? a : 0.0f;
}

// Exponent of the scale from the block's largest finite magnitude.  The
// largest value is 1.75 * 2^TOP in both formats, so amax = m * 2^x needs
// x - TOP, one more when m > 1.75.
template <bool E5M2>
__device__ __forceinline__ int scale_exponent(float amax) {
    constexpr int TOP = E5M2 ? 15 : 8;
    if (amax == 0.0f) return 0;
    const uint32_t b = __float_as_uint(amax);
    const int e = static_cast<int>(b >> 23) - 127 - TOP + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;
}
__device__ __forceinline__ float power2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// 8 numbers times inv to 8 bytes (element 0 lowest).
template <bool E5M2>
__device__ __forceinline__ uint2 convert8(const float (&v)[8], float inv) {
    uint16_t h[4];
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float lo = v[2 * i] * inv, hi = v[2 * i + 1] * inv;
        odd |= !(fabsf(lo) < INFINITY) || !(fabsf(hi) < INFINITY);
        if (E5M2) asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(h[i]) : "f"(hi), "f"(lo));
        else asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h[i]) : "f"(hi), "f"(lo));
    }
    uint2 r = make_uint2(h[0] | (static_cast<uint32_t>(h[1]) << 16), h[2] | (static_cast<uint32_t>(h[3]) << 16));
    if (odd) {  // the conversion saturates infinities: put them right
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (fabsf(v[i]) < INFINITY) continue;
            uint32_t code = (E5M2 && v[i] == v[i]) ? 0x7cu : 0x7fu;
            if (v[i] < 0.0f) code |= 0x80u;
            uint32_t &w = i < 4 ? r.x : r.y;
            w = (w & ~(0xffu << (8 * (i & 3)))) | (code << (8 * (i & 3)));
        }
    }
    return r;
}

// Blocks of a row: 16 lanes hold one, 8 elements a lane; a thread block takes
// 16 rows of one column block, so a warp reads two rows' 128 elements and
// the 16 scales go out together.
template <typename T, bool E5M2, bool VEC>
__global__ void __launch_bounds__(THREADS)
    rows_kernel(const T *__restrict__ x, int64_t rows, int64_t cols, int64_t ld, int64_t kb,
                uint8_t *__restrict__ q, float *__restrict__ scales) {
    const int part = threadIdx.x & 15, sub = threadIdx.x >> 4;
    const int64_t row_tiles = (rows + 15) / 16;
    for (int64_t w = blockIdx.x; w < row_tiles * kb; w += gridDim.x) {
        const int64_t row = (w / kb) * 16 + sub, b = w % kb;
        const int64_t col = b * BLOCK + part * 8;
        float v[8] = {};
        if (row < rows && col < cols) load8<T, VEC>(x + row * cols + col, cols - col, v);
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, finite_abs(v[i]));
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        const int e = scale_exponent<E5M2>(amax);
        if (row < rows) {
            if (part == 0) scales[b * rows + row] = power2(e);
            if (col < ld) *reinterpret_cast<uint2 *>(q + row * ld + col) = convert8<E5M2>(v, power2(-e));
        }
    }
}

// A 128 x 128 tile a thread block: 8 rows a thread, 8 elements of each.
template <typename T, bool E5M2, bool VEC>
__global__ void __launch_bounds__(THREADS)
    tiles_kernel(const T *__restrict__ x, int64_t batch, int64_t rows, int64_t cols, int64_t ld,
                 uint8_t *__restrict__ q, float *__restrict__ scales) {
    __shared__ float warp_amax[THREADS / 32];
    const int part = threadIdx.x & 15, sub = threadIdx.x >> 4;
    const int64_t rb = (rows + BLOCK - 1) / BLOCK, kb = (cols + BLOCK - 1) / BLOCK;
    for (int64_t w = blockIdx.x; w < batch * rb * kb; w += gridDim.x) {
        const int64_t b = w / (rb * kb), in = w - b * rb * kb;
        const int64_t row0 = (in / kb) * BLOCK + sub, col = (in % kb) * BLOCK + part * 8;
        float v[8][8];
        float amax = 0.0f;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int64_t row = row0 + r * 16;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[r][i] = 0.0f;
            if (row < rows && col < cols) load8<T, VEC>(x + (b * rows + row) * cols + col, cols - col, v[r]);
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, finite_abs(v[r][i]));
        }
        amax = warp_max(amax);
        __syncthreads();  // the previous tile's maxima have been read
        if ((threadIdx.x & 31) == 0) warp_amax[threadIdx.x >> 5] = amax;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < THREADS / 32; ++i) amax = fmaxf(amax, warp_amax[i]);
        const int e = scale_exponent<E5M2>(amax);
        if (threadIdx.x == 0) scales[w] = power2(e);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int64_t row = row0 + r * 16;
            if (row < rows && col < ld)
                *reinterpret_cast<uint2 *>(q + (b * rows + row) * ld + col) = convert8<E5M2>(v[r], power2(-e));
        }
    }
}

// The rows [row, row + len) of x that place block `b` holds (len 0: none):
// groups' rows in order, each group from a block of 128 on.  Offsets outside
// [0, rows] are held to it.
__device__ __forceinline__ void block_rows(const int32_t *offsets, int groups, int64_t rows, int64_t b,
                                           int64_t *row, int *len) {
    if (!offsets) {
        *row = b * BLOCK;
        const int64_t left = rows - *row;
        *len = static_cast<int>(left < 0 ? 0 : (left > BLOCK ? BLOCK : left));
        return;
    }
    *row = 0;
    *len = 0;
    int64_t at = 0;  // first block of the group
    for (int g = 0; g < groups; ++g) {
        int64_t lo = offsets[g], hi = offsets[g + 1];
        lo = lo < 0 ? 0 : (lo > rows ? rows : lo);
        hi = hi < lo ? lo : (hi > rows ? rows : hi);
        const int64_t nb = (hi - lo + BLOCK - 1) / BLOCK;
        if (b < at + nb) {
            *row = lo + (b - at) * BLOCK;
            const int64_t left = hi - *row;
            *len = static_cast<int>(left > BLOCK ? BLOCK : left);
            return;
        }
        at += nb;
    }
}

// 128 rows x 128 columns a thread block, turned over in shared memory as
// bytes.  A thread holds rows 8 sub .. 8 sub + 7 of 8 columns: its 8 bytes of
// a column are consecutive places.
template <typename T, bool E5M2, bool VEC>
__global__ void __launch_bounds__(THREADS)
    transposed_kernel(const T *__restrict__ x, const int32_t *__restrict__ offsets, int groups,
                      int64_t rows, int64_t cols, int64_t blocks, uint8_t *__restrict__ q,
                      float *__restrict__ scales) {
    constexpr int PITCH = BLOCK + 16;
    __shared__ __align__(16) uint8_t tile[BLOCK * PITCH];
    __shared__ float amax_part[16][BLOCK];
    __shared__ int64_t row_s;
    __shared__ int len_s;
    const int part = threadIdx.x & 15, sub = threadIdx.x >> 4;
    const int64_t cb = (cols + BLOCK - 1) / BLOCK, places = blocks * BLOCK;
    for (int64_t w = blockIdx.x; w < blocks * cb; w += gridDim.x) {
        const int64_t b = w / cb, col0 = (w % cb) * BLOCK;
        __syncthreads();
        if (threadIdx.x == 0) block_rows(offsets, groups, rows, b, &row_s, &len_s);
        __syncthreads();
        const int64_t row0 = row_s, col = col0 + part * 8;
        const int len = len_s;
        float v[8][8], amax[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) amax[i] = 0.0f;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int in = sub * 8 + r;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[r][i] = 0.0f;
            if (in < len && col < cols) load8<T, VEC>(x + (row0 + in) * cols + col, cols - col, v[r]);
#pragma unroll
            for (int i = 0; i < 8; ++i) amax[i] = fmaxf(amax[i], finite_abs(v[r][i]));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) amax_part[sub][part * 8 + i] = amax[i];
        __syncthreads();
        if (threadIdx.x < BLOCK) {
            float a = 0.0f;
#pragma unroll
            for (int s = 0; s < 16; ++s) a = fmaxf(a, amax_part[s][threadIdx.x]);
            amax_part[0][threadIdx.x] = a;
            if (col0 + threadIdx.x < cols)
                scales[b * cols + col0 + threadIdx.x] = power2(scale_exponent<E5M2>(a));
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float c[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) c[r] = v[r][i];
            const int e = scale_exponent<E5M2>(amax_part[0][part * 8 + i]);
            *reinterpret_cast<uint2 *>(tile + (part * 8 + i) * PITCH + sub * 8) = convert8<E5M2>(c, power2(-e));
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < BLOCK * BLOCK / (16 * THREADS); ++u) {
            const int i = u * THREADS + threadIdx.x, c = i >> 3, o = (i & 7) * 16;
            if (col0 + c < cols)
                *reinterpret_cast<uint4 *>(q + (col0 + c) * places + b * BLOCK + o) =
                    *reinterpret_cast<const uint4 *>(tile + c * PITCH + o);
        }
    }
}

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

int check_format(const char *op, int32_t format) {
    if (format != CHELIS_FORMAT_E4M3 && format != CHELIS_FORMAT_E5M2)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "%s: 8-bit formats are e4m3 and e5m2", op);
    return CHELIS_CUDA_OK;
}

unsigned grid_for(int64_t work, int per_sm) {
    const int64_t cap = static_cast<int64_t>(sm_count()) * per_sm;
    return static_cast<unsigned>(work < 1 ? 1 : (work > cap ? cap : work));
}

template <typename F>
void by_format(int32_t dtype, int32_t format, bool vec, F f) {
    experts::by_type(dtype, vec, [&](auto t, auto v) {
        if (format == CHELIS_FORMAT_E5M2) f(t, std::true_type{}, v);
        else f(t, std::false_type{}, v);
    });
}

}  // namespace blocks8
}  // namespace chelis

using namespace chelis;

extern "C" int chelis_cuda_quantize8(int32_t dtype, int32_t format, int32_t layout, const void *x,
                                     int64_t batch, int64_t rows, int64_t cols, uint8_t *data,
                                     float *scales) {
    if (!experts::is_act(dtype))
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "quantize8 takes f32, bf16 or f16");
    CHELIS_TRY(blocks8::check_format("quantize8", format));
    if (layout != CHELIS_BLOCKS_ROWS && layout != CHELIS_BLOCKS_TILES)
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "quantize8: layout %d", layout);
    if (batch < 0 || rows < 0 || cols < 0 || (layout == CHELIS_BLOCKS_ROWS && batch != 1))
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "quantize8: extents >= 0, and batch 1 for rows");
    if (batch == 0 || rows == 0 || cols == 0) return CHELIS_CUDA_OK;
    if (!x || !data || !scales) return set_error(CHELIS_CUDA_ERR_DOMAIN, "quantize8: null operand");
    if (!experts::aligned16(data))
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "quantize8: data must lie on 16 bytes");
    cudaStream_t s = current_stream();
    const int64_t ld = blocks8::round16(cols), kb = (cols + blocks8::BLOCK - 1) / blocks8::BLOCK;
    const bool vec = cols * experts::width(dtype) % 16 == 0 && experts::aligned16(x);
    blocks8::by_format(dtype, format, vec, [&](auto t, auto f, auto v) {
        using T = decltype(t);
        constexpr bool E5M2 = decltype(f)::value, VEC = decltype(v)::value;
        if (layout == CHELIS_BLOCKS_ROWS)
            blocks8::rows_kernel<T, E5M2, VEC>
                <<<blocks8::grid_for((rows + 15) / 16 * kb, 32), blocks8::THREADS, 0, s>>>(
                    static_cast<const T *>(x), rows, cols, ld, kb, data, scales);
        else
            blocks8::tiles_kernel<T, E5M2, VEC>
                <<<blocks8::grid_for(batch * ((rows + blocks8::BLOCK - 1) / blocks8::BLOCK) * kb, 8),
                   blocks8::THREADS, 0, s>>>(static_cast<const T *>(x), batch, rows, cols, ld, data,
                                             scales);
    });
    g_launches++;
    CHELIS_LAUNCH_CHECK("blocks8::quantize");
    return CHELIS_CUDA_OK;
}

extern "C" int64_t chelis_cuda_quantize8_places(int64_t rows, int32_t groups) {
    if (rows < 0 || groups < 0) return -1;
    const int64_t blocks = groups > 0 ? rows / blocks8::BLOCK + groups
                                      : (rows + blocks8::BLOCK - 1) / blocks8::BLOCK;
    return blocks * blocks8::BLOCK;
}

extern "C" int chelis_cuda_quantize8_transposed(int32_t dtype, int32_t format, const void *x,
                                                const int32_t *offsets, int32_t groups, int64_t rows,
                                                int64_t cols, uint8_t *data, float *scales) {
    if (!experts::is_act(dtype))
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "quantize8_transposed takes f32, bf16 or f16");
    CHELIS_TRY(blocks8::check_format("quantize8_transposed", format));
    if (rows < 0 || cols < 0 || groups < 0 || (groups > 0) != (offsets != nullptr))
        return set_error(CHELIS_CUDA_ERR_DOMAIN,
                         "quantize8_transposed: extents >= 0, offsets exactly with groups");
    if (groups > blocks8::MAX_GROUPS)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "quantize8_transposed admits %d groups at most",
                         blocks8::MAX_GROUPS);
    const int64_t places = chelis_cuda_quantize8_places(rows, groups);
    if (places == 0 || cols == 0) return CHELIS_CUDA_OK;
    if ((rows > 0 && !x) || !data || !scales)
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "quantize8_transposed: null operand");
    if (!experts::aligned16(data))
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "quantize8_transposed: data must lie on 16 bytes");
    cudaStream_t s = current_stream();
    const int64_t blocks = places / blocks8::BLOCK;
    const bool vec = cols * experts::width(dtype) % 16 == 0 && experts::aligned16(x);
    blocks8::by_format(dtype, format, vec, [&](auto t, auto f, auto v) {
        using T = decltype(t);
        constexpr bool E5M2 = decltype(f)::value, VEC = decltype(v)::value;
        blocks8::transposed_kernel<T, E5M2, VEC>
            <<<blocks8::grid_for(blocks * ((cols + blocks8::BLOCK - 1) / blocks8::BLOCK), 8),
               blocks8::THREADS, 0, s>>>(static_cast<const T *>(x), offsets, groups, rows, cols, blocks,
                                         data, scales);
    });
    g_launches++;
    CHELIS_LAUNCH_CHECK("blocks8::transposed_kernel");
    return CHELIS_CUDA_OK;
}
