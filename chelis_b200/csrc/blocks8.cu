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

// 8 consecutive elements, held as they were loaded (16-bit ones in half the
// registers, so that more thread blocks are resident) and read as f32.
template <typename T, bool VEC>
struct Eight {
    static constexpr int N = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
    Pack<T, VEC> r[8 / N];
    __device__ __forceinline__ float operator[](int i) const { return to_f32(r[i / N].v[i % N]); }
};
// From p[0..valid), zeros beyond.  VEC: in 16-byte packs, none of which
// straddles the end (the width is a multiple of one).
template <typename T, bool VEC>
__device__ __forceinline__ Eight<T, VEC> load8(const T *p, int valid) {
    using E = Eight<T, VEC>;
    E v{};
#pragma unroll
    for (int u = 0; u < 8 / E::N; ++u)
        if (u * E::N < valid) v.r[u] = experts::load_pack<T, VEC>(p + u * E::N);
    return v;
}

// Magnitudes are compared as bits, which order as the numbers do, 16-bit ones
// two at a time: nothing is converted before the scale is known, so a block
// waits for it in the registers that it was loaded into (as f32 it took twice
// as many, and spilled).  A running maximum holds bits of T (two halves of it
// for a 16-bit T), magnitude_key turns it into f32 bits.
template <typename T, bool VEC>
__device__ __forceinline__ uint32_t max8(const Eight<T, VEC> &v, uint32_t most) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
    } else if constexpr (VEC) {
        const uint4 w = *reinterpret_cast<const uint4 *>(&v);
        most = __vmaxu2(most, w.x & 0x7fff7fffu);
        most = __vmaxu2(most, w.y & 0x7fff7fffu);
        most = __vmaxu2(most, w.z & 0x7fff7fffu);
        most = __vmaxu2(most, w.w & 0x7fff7fffu);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            most = max(most, static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(&v.r[i].v[0])) & 0x7fffu);
    }
    return most;
}
template <typename T>
__device__ __forceinline__ uint32_t key_of_bits(uint32_t bits) {
    if constexpr (sizeof(T) == 4) {
        return bits;
    } else {
        const uint16_t h = static_cast<uint16_t>(bits);
        return __float_as_uint(to_f32(*reinterpret_cast<const T *>(&h)));
    }
}
template <typename T>
__device__ __forceinline__ uint32_t magnitude_key(uint32_t most) {
    return sizeof(T) == 4 ? most : key_of_bits<T>(max(most & 0xffffu, most >> 16));
}
// An infinity or a NaN is among them: the block goes the slow way.
__device__ __forceinline__ bool special(uint32_t key) { return key >= 0x7f800000u; }

// Exponent of the scale from the bits of the block's largest finite magnitude.  The
// largest value is 1.75 * 2^TOP in both formats, so amax = m * 2^x needs
// x - TOP, one more when m > 1.75.
template <bool E5M2>
__device__ __forceinline__ int scale_exponent(uint32_t b) {
    constexpr int TOP = E5M2 ? 15 : 8;
    if (b == 0) return 0;
    const int e = static_cast<int>(b >> 23) - 127 - TOP + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;
}
__device__ __forceinline__ float power2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// 8 numbers times inv to 8 bytes (element 0 lowest).  The conversion keeps
// NaNs; a block with an infinity, which it would saturate, does not come here.
template <bool E5M2, typename V>
__device__ __forceinline__ uint2 convert8(const V &v, float inv) {
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float lo = v[2 * i] * inv, hi = v[2 * i + 1] * inv;
        if (E5M2) asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(h[i]) : "f"(hi), "f"(lo));
        else asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h[i]) : "f"(hi), "f"(lo));
    }
    return make_uint2(h[0] | (static_cast<uint32_t>(h[1]) << 16), h[2] | (static_cast<uint32_t>(h[3]) << 16));
}
// Blocks with an infinity or a NaN are done again one number at a time, from
// memory, by functions of their own: kept out of line and called last, they
// cost the usual blocks no registers (inlined, or called where a block is
// held, they made the kernels below spill).
template <bool E5M2>
__device__ __forceinline__ uint8_t convert1(float v, float inv) {
    uint16_t h;
    const float x = v * inv;
    if (E5M2) asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(h) : "f"(0.0f), "f"(x));
    else asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(0.0f), "f"(x));
    if (fabsf(v) == INFINITY) h = (E5M2 ? 0x7c : 0x7f) | (v < 0.0f ? 0x80 : 0);
    return static_cast<uint8_t>(h);
}
__device__ __forceinline__ uint32_t finite_key(float v, uint32_t most) {
    const uint32_t key = __float_as_uint(fabsf(v));
    return special(key) ? most : max(most, key);
}
// One thread, up to 128 numbers `step` apart.
template <typename T, bool E5M2>
__device__ __noinline__ void slow_block(const T *x, int64_t step, int n, uint8_t *q, float *scale) {
    uint32_t key = 0;
    for (int i = 0; i < n; ++i) key = finite_key(to_f32(x[i * step]), key);
    const int e = scale_exponent<E5M2>(key);
    *scale = power2(e);
    for (int i = 0; i < n; ++i) q[i] = convert1<E5M2>(to_f32(x[i * step]), power2(-e));
}

// Blocks of a row: LANES lanes hold one, 8 elements a lane at a time; a thread
// block takes ROWS rows of RUN consecutive column blocks, whose loads are all
// in flight before the first maximum is formed, and the rows' scales of a
// block go out together.  f32 is bound by memory with 16 lanes and runs of 4
// (16384 x 4096 in 50.5 us, 6.7 TB/s; runs of 2 54.5).  16-bit types were bound
// by the ALU's work around each maximum (71 % busy, 48 us) and take 8 lanes of
// 16 elements, which halves it, and runs of 2, which leave more blocks resident
// (41 us, 4.9 TB/s; runs of 4 44 us); latency is what is left.
template <typename T>
struct RowShape {
    static constexpr int RUN = sizeof(T) == 2 ? 2 : 4;
    static constexpr int LANES = sizeof(T) == 2 ? 8 : 16;
    static constexpr int EIGHTS = 16 / LANES;  // of a lane
    static constexpr int ROWS = THREADS / LANES;
};

template <typename T, bool E5M2, bool VEC>
__global__ void __launch_bounds__(THREADS)
    rows_kernel(const T *__restrict__ x, int64_t rows, int64_t cols, int64_t ld, int64_t kb,
                uint8_t *__restrict__ q, float *__restrict__ scales) {
    constexpr int LANES = RowShape<T>::LANES, EIGHTS = RowShape<T>::EIGHTS, ROWS = RowShape<T>::ROWS;
    constexpr int RUN = RowShape<T>::RUN;
    const int part = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const int64_t row_tiles = (rows + ROWS - 1) / ROWS, runs = (kb + RUN - 1) / RUN;
    for (int64_t w = blockIdx.x; w < row_tiles * runs; w += gridDim.x) {
        const int64_t tile = w / runs, b0 = (w - tile * runs) * RUN;
        const int64_t row = tile * ROWS + sub, col0 = b0 * BLOCK;
        const bool in = row < rows;
        const T *src = x + row * cols + col0 + part * 8;
        uint8_t *dst = q + row * ld + col0 + part * 8;
        // columns from this lane's first on, of the data and of its padded row
        const int left = in ? static_cast<int>(cols - col0 < RUN * BLOCK ? cols - col0 : RUN * BLOCK) - part * 8 : 0;
        const int wide = in ? static_cast<int>(ld - col0 < RUN * BLOCK ? ld - col0 : RUN * BLOCK) - part * 8 : 0;
        Eight<T, VEC> v[RUN][EIGHTS];
#pragma unroll
        for (int u = 0; u < RUN; ++u)
#pragma unroll
            for (int h = 0; h < EIGHTS; ++h) {
                const int o = u * BLOCK + h * LANES * 8;
                v[u][h] = load8<T, VEC>(src + o, left - o);
            }
        uint32_t odd = 0;
#pragma unroll
        for (int u = 0; u < RUN; ++u) {
            uint32_t most = 0;
#pragma unroll
            for (int h = 0; h < EIGHTS; ++h) most = max8(v[u][h], most);
            uint32_t key = magnitude_key<T>(most);
#pragma unroll
            for (int off = LANES / 2; off > 0; off >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, off));
            if (special(key)) {
                odd |= 1u << u;
                continue;
            }
            const int e = scale_exponent<E5M2>(key);
            if (part == 0 && in && b0 + u < kb) scales[(b0 + u) * rows + row] = power2(e);
            const float inv = power2(-e);
#pragma unroll
            for (int h = 0; h < EIGHTS; ++h) {
                const int o = u * BLOCK + h * LANES * 8;
                if (wide > o) *reinterpret_cast<uint2 *>(dst + o) = convert8<E5M2>(v[u][h], inv);
            }
        }
        if (odd && part == 0 && in)
            for (int u = 0; u < RUN; ++u)
                if (odd >> u & 1) {
                    const int64_t col = col0 + u * BLOCK;
                    const int n = static_cast<int>(cols - col < BLOCK ? cols - col : BLOCK);
                    slow_block<T, E5M2>(x + row * cols + col, 1, n, q + row * ld + col, scales + (b0 + u) * rows + row);
                    for (int64_t c = cols; c < ld && c < col + BLOCK; ++c) q[row * ld + c] = 0;
                }
    }
}

// The largest of the thread block's numbers.
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t *warp_part) {
    v = __reduce_max_sync(0xffffffffu, v);
    __syncthreads();  // the last use of warp_part is over
    if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) v = max(v, warp_part[i]);
    return v;
}

template <typename T, bool E5M2>
__device__ __noinline__ void slow_tile(const T *x, int64_t rows, int64_t cols, int64_t ld, int64_t row0,
                                       int64_t col0, uint8_t *q, float *scale, uint32_t *warp_part) {
    uint32_t key = 0;
    for (int i = threadIdx.x; i < BLOCK * BLOCK; i += THREADS) {
        const int64_t row = row0 + i / BLOCK, col = col0 + i % BLOCK;
        if (row < rows && col < cols) key = finite_key(to_f32(x[row * cols + col]), key);
    }
    const int e = scale_exponent<E5M2>(block_max(key, warp_part));
    if (threadIdx.x == 0) *scale = power2(e);
    for (int i = threadIdx.x; i < BLOCK * BLOCK; i += THREADS) {
        const int64_t row = row0 + i / BLOCK, col = col0 + i % BLOCK;
        if (row < rows && col < ld)
            q[row * ld + col] = col < cols ? convert1<E5M2>(to_f32(x[row * cols + col]), power2(-e)) : 0;
    }
}

// A 128 x 128 tile a thread block: 8 rows a thread, 8 elements of each, all
// loaded before the block's maximum is formed.  Memory bounds f32 (16384 x 4096
// in 52.7 us, 6.4 TB/s); a 16-bit tile is half the bytes behind the same two
// barriers, and three resident blocks a multiprocessor do not hide them (53 us,
// 3.8 TB/s; two 98 us, four spill: 69 us).
template <typename T, bool E5M2, bool VEC>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 2 ? 3 : 2)
    tiles_kernel(const T *__restrict__ x, int64_t batch, int64_t rows, int64_t cols, int64_t ld,
                 uint8_t *__restrict__ q, float *__restrict__ scales) {
    __shared__ uint32_t warp_most[THREADS / 32];
    const int part = threadIdx.x & 15, sub = threadIdx.x >> 4;
    const int64_t rb = (rows + BLOCK - 1) / BLOCK, kb = (cols + BLOCK - 1) / BLOCK;
    for (int64_t w = blockIdx.x; w < batch * rb * kb; w += gridDim.x) {
        const int64_t b = w / (rb * kb), in = w - b * rb * kb;
        const int64_t trow = in / kb, row0 = trow * BLOCK + sub, col = (in - trow * kb) * BLOCK + part * 8;
        const T *src = x + (b * rows + row0) * cols + col;
        uint8_t *dst = q + (b * rows + row0) * ld + col;
        const int64_t src_step = 16 * cols, dst_step = 16 * ld;
        const int high = static_cast<int>(rows - row0 < BLOCK ? rows - row0 : BLOCK);  // rows from this one on
        const int left = static_cast<int>(cols - col < 8 ? cols - col : 8);
        const bool store = col < ld;
        Eight<T, VEC> v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = load8<T, VEC>(src + r * src_step, r * 16 < high ? left : 0);
        uint32_t most = 0;
#pragma unroll
        for (int r = 0; r < 8; ++r) most = max8(v[r], most);
        const uint32_t key = block_max(magnitude_key<T>(most), warp_most);
        if (!special(key)) {
            const int e = scale_exponent<E5M2>(key);
            if (threadIdx.x == 0) scales[w] = power2(e);
            const float inv = power2(-e);
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r * 16 < high && store)
                    *reinterpret_cast<uint2 *>(dst + r * dst_step) = convert8<E5M2>(v[r], inv);
        } else {  // the whole block
            slow_tile<T, E5M2>(x + b * rows * cols, rows, cols, ld, trow * BLOCK, (in - trow * kb) * BLOCK,
                               q + b * rows * ld, scales + w, warp_most);
        }
    }
}

// Rows of group g, held to [0, rows].
__device__ __forceinline__ void group_rows(const int32_t *offsets, int g, int64_t rows, int64_t *lo, int64_t *hi) {
    const int64_t a = offsets[g], b = offsets[g + 1];
    *lo = a < 0 ? 0 : (a > rows ? rows : a);
    *hi = b < *lo ? *lo : (b > rows ? rows : b);
}
// start[g], one warp: the place blocks before group g, each group's rows from a
// block of 128 on; held to `blocks`, which ordered offsets do not pass.
__device__ __forceinline__ void block_starts(const int32_t *offsets, int groups, int64_t rows, int64_t blocks, int lane,
                                             int64_t *start) {
    int64_t base = 0;
    for (int g0 = 0; g0 < groups; g0 += 32) {
        int64_t sum = 0;
        if (g0 + lane < groups) {
            int64_t lo, hi;
            group_rows(offsets, g0 + lane, rows, &lo, &hi);
            sum = (hi - lo + BLOCK - 1) / BLOCK;
        }
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, sum, off);
            if (lane >= off) sum += o;
        }
        sum += base;
        if (sum > blocks) sum = blocks;
        if (g0 + lane < groups) start[g0 + lane + 1] = sum;
        base = __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) start[0] = 0;
}
// The rows [row, row + len) of x that place block `b` holds (len 0: none).  By
// every thread, from the groups' first blocks in shared memory: 16384 x 4096 bf16
// by 64 experts in 72 us and by 1024 in 427 (nine times the tiles, most of each
// empty), where one thread going through the offsets took 119 and 4499.
__device__ __forceinline__ void block_rows(const int32_t *offsets, const int64_t *start, int groups, int64_t rows,
                                           int64_t b, int64_t *row, int *len) {
    int64_t lo = 0, hi = rows, in = b;  // without offsets: one group
    if (offsets) {
        int first = 0, last = groups;  // the last group that starts at or before b
        while (last - first > 1) {
            const int mid = (first + last) >> 1;
            if (start[mid] <= b) first = mid;
            else last = mid;
        }
        group_rows(offsets, first, rows, &lo, &hi);
        in = b - start[first];
    }
    const int64_t left = hi - lo - in * BLOCK;
    *row = left > 0 ? lo + in * BLOCK : 0;
    *len = static_cast<int>(left <= 0 ? 0 : (left > BLOCK ? BLOCK : left));
}

// f32 bits of the largest magnitude in each of the 8 columns of 8 rows.
template <typename T, bool VEC>
__device__ __forceinline__ void column_keys(const Eight<T, VEC> (&v)[8], uint32_t (&key)[8]) {
    if constexpr (sizeof(T) == 2 && VEC) {
        uint4 m = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const uint4 w = *reinterpret_cast<const uint4 *>(&v[r]);
            m.x = __vmaxu2(m.x, w.x & 0x7fff7fffu);
            m.y = __vmaxu2(m.y, w.y & 0x7fff7fffu);
            m.z = __vmaxu2(m.z, w.z & 0x7fff7fffu);
            m.w = __vmaxu2(m.w, w.w & 0x7fff7fffu);
        }
        const uint32_t w[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) key[i] = key_of_bits<T>((w[i >> 1] >> (16 * (i & 1))) & 0xffffu);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            key[i] = 0;
#pragma unroll
            for (int r = 0; r < 8; ++r) key[i] = max(key[i], __float_as_uint(fabsf(v[r][i])));
        }
    }
}

// 128 rows x 128 columns a thread block, turned over in shared memory as
// bytes.  A thread holds rows 8 sub .. 8 sub + 7 of 8 columns: its 8 bytes of
// a column are consecutive places.  16384 x 4096: bf16 48 us (4.2 TB/s), f32 57
// us (5.9 TB/s), bound by the barriers between load, maximum and store; before
// the bytes were swizzled bank conflicts made it 64 and 71 us.
template <typename T, bool E5M2, bool VEC>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 2 ? 3 : 2)
    transposed_kernel(const T *__restrict__ x, const int32_t *__restrict__ offsets, int groups,
                      int64_t rows, int64_t cols, int64_t blocks, uint8_t *__restrict__ q,
                      float *__restrict__ scales) {
    // column c's eight bytes of rows 8 s .. 8 s + 7 lie in slot s ^ (c / 8 mod
    // 16) of its 128, so that neither the threads' stores nor the loads collide
    constexpr int PITCH = BLOCK + 16;
    __shared__ __align__(16) uint8_t tile[BLOCK * PITCH];
    __shared__ __align__(16) uint32_t most_part[16][BLOCK];
    __shared__ int64_t start[MAX_GROUPS + 1];
    const int part = threadIdx.x & 15, sub = threadIdx.x >> 4;
    const int64_t cb = (cols + BLOCK - 1) / BLOCK, places = blocks * BLOCK;
    if (offsets) {
        if (threadIdx.x < 32) block_starts(offsets, groups, rows, blocks, threadIdx.x, start);
        __syncthreads();
    }
    for (int64_t w = blockIdx.x; w < blocks * cb; w += gridDim.x) {
        // (the last turn's reads of shared memory end at its last barrier)
        const int64_t b = w / cb, col0 = (w % cb) * BLOCK, col = col0 + part * 8;
        int64_t row0;
        int len;
        block_rows(offsets, start, groups, rows, b, &row0, &len);
        const T *src = x + (row0 + sub * 8) * cols + col;
        const int left = static_cast<int>(cols - col < 8 ? cols - col : 8);
        Eight<T, VEC> v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int in = sub * 8 + r;
            v[r] = load8<T, VEC>(src + r * cols, in < len ? left : 0);
        }
        {
            uint32_t key[8];
            column_keys(v, key);
            uint4 *to = reinterpret_cast<uint4 *>(&most_part[sub][part * 8]);
            to[0] = make_uint4(key[0], key[1], key[2], key[3]);
            to[1] = make_uint4(key[4], key[5], key[6], key[7]);
        }
        __syncthreads();
        bool odd = false;  // this thread's column
        if (threadIdx.x < BLOCK) {
            uint32_t a = 0;
#pragma unroll
            for (int s = 0; s < 16; ++s) a = max(a, most_part[s][threadIdx.x]);
            const int e = special(a) ? 0 : scale_exponent<E5M2>(a);
            most_part[0][threadIdx.x] = static_cast<uint32_t>(127 - e) << 23;  // bits of 1 / scale
            odd = special(a);
            if (col0 + threadIdx.x < cols) scales[b * cols + col0 + threadIdx.x] = power2(e);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float c[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) c[r] = v[r][i];
            uint8_t *to = tile + (part * 8 + i) * PITCH + (sub ^ part) * 8;
            *reinterpret_cast<uint2 *>(to) = convert8<E5M2>(c, __uint_as_float(most_part[0][part * 8 + i]));
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < BLOCK * BLOCK / (16 * THREADS); ++u) {
            const int i = u * THREADS + threadIdx.x, c = i >> 3, pair = i & 7, turn = (c >> 3) & 15;
            uint4 w = *reinterpret_cast<const uint4 *>(tile + c * PITCH + (pair ^ (turn >> 1)) * 16);
            if (turn & 1) w = make_uint4(w.z, w.w, w.x, w.y);
            if (col0 + c < cols) *reinterpret_cast<uint4 *>(q + (col0 + c) * places + b * BLOCK + pair * 16) = w;
        }
        if (__syncthreads_or(odd)) {  // columns done again, over what was just written
            const int64_t c = col0 + threadIdx.x;
            if (odd && c < cols)
                slow_block<T, E5M2>(x + row0 * cols + c, cols, len, q + c * places + b * BLOCK, scales + b * cols + c);
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
                <<<blocks8::grid_for((rows + blocks8::RowShape<T>::ROWS - 1) / blocks8::RowShape<T>::ROWS *
                                        ((kb + blocks8::RowShape<T>::RUN - 1) / blocks8::RowShape<T>::RUN), 32), blocks8::THREADS, 0, s>>>(
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
