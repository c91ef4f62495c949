// gemm_few8.cu -- the layer product of gemm_blocks8.cu for few rows: a token
// or a handful for each matrix, as in serving.  Such a product reads the
// weights once and does little with them, so memory bounds it, not the tensor
// core: the weights go straight from global memory into registers, 16 bytes a
// lane, and warp-level MMAs (m16n8k32) multiply 16 of their rows by 8 tokens.
// A tcgen05 tile would put 128 rows of a beside them, all but a few empty.
//
// A warp takes 16 rows of one expert's matrix.  `share` warps of a block split
// its contraction block by block (block b to warp b mod share) and are added
// up in that order; the fewer strips of 16 rows there are, the more warps
// share one, so that enough loads are in flight.  In a block of 128, lane
// (g, t) = (lane / 4, lane % 4) takes bytes 16 t .. 16 t + 15 and 64 + 16 t ..
// of weight rows g and g + 8 and of token g: the MMA wants other bytes of K in
// a lane, but the same ones of both operands, and a sum does not mind their
// order.
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "common.cuh"

namespace chelis {

extern std::atomic<uint64_t> g_launches;

namespace few8 {

using gemm8::Params;
using gemm8::group_span;

constexpr int WARPS = 8, STRIP = 16, COLS = 8;

template <bool E5A, bool E5B>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    // a: weights (format b of the product), b: tokens (format a)
#define CHELIS_MMA8(TA, TB)                                                                      \
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32." TA "." TB ".f32 "                     \
                 "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"                       \
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                              \
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1))
    if (E5B) {
        if (E5A) CHELIS_MMA8("e5m2", "e5m2");
        else CHELIS_MMA8("e5m2", "e4m3");
    } else {
        if (E5A) CHELIS_MMA8("e4m3", "e5m2");
        else CHELIS_MMA8("e4m3", "e4m3");
    }
#undef CHELIS_MMA8
}

__device__ __forceinline__ uint4 load16(const uint8_t *p, bool ok) {
    return ok ? __ldg(reinterpret_cast<const uint4 *>(p)) : make_uint4(0, 0, 0, 0);
}

// v s w in 64 bits, where no pair of them leaves the range.
__device__ __forceinline__ float scaled(float v, float s, float w) {
    return static_cast<float>(static_cast<double>(v) * static_cast<double>(s) * static_cast<double>(w));
}

// NT: tokens of one pass over the weights, in eights.
// Three blocks a multiprocessor with two blocks of K in flight a warp: 9.8 us for
// 16 rows by 8 matrices of 4096 x 1024 out of memory (3.4 TB/s); two with four
// took 10 % longer.  What is left is latency (a strip's loads start
// once its expert's rows are known) and the 8-bit MMA itself, which this
// machine runs by converting its operands to 16 bits (ALU 36 % busy).
template <bool E5A, bool E5B, int NT>
__global__ void __launch_bounds__(WARPS * 32, NT == 1 ? 3 : 1)
    few8_kernel(const Params p, const uint8_t *__restrict__ a, const uint8_t *__restrict__ w, int64_t ld,
                int share) {
    __shared__ float part[WARPS * NT * COLS * STRIP];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int strips = WARPS / share, mine = warp / share, turn = warp - mine * share;
    const int group = blockIdx.y;
    const int64_t n_first = static_cast<int64_t>(blockIdx.x) * (strips * STRIP);
    if (group == p.groups) {  // rows that no group holds
        int64_t lo, hi, first, last;
        group_span(p, p.rows, 0, &first, &hi);
        group_span(p, p.rows, p.groups - 1, &lo, &last);
        const int64_t loose = first + p.rows - last, wide = strips * STRIP;
        for (int64_t i = threadIdx.x; i < loose * wide; i += WARPS * 32) {
            const int64_t r = i / wide, n = n_first + i % wide;
            if (n >= p.n) continue;
            const int64_t o = (r < first ? r : last + r - first) * p.n + n;
            if (p.out_dtype == CHELIS_DTYPE_F32) static_cast<float *>(p.out)[o] = 0.0f;
            else static_cast<uint16_t *>(p.out)[o] = 0;
        }
        return;
    }
    int64_t row0, row_end;
    group_span(p, p.rows, group, &row0, &row_end);
    const int64_t n0 = n_first + mine * STRIP;
    const bool live = n0 < p.n;  // a warp past the matrix's last strip only keeps the barriers
    // rows and tokens past the end read the last one; they are not stored
    const int64_t last_n = p.n - 1;
    const uint8_t *wg = w + group * p.n * ld;
    const uint8_t *w0 = wg + (n0 + g < last_n ? n0 + g : last_n) * ld;
    const uint8_t *w1 = wg + (n0 + g + 8 < last_n ? n0 + g + 8 : last_n) * ld;
    const float *sb = p.sb + group * p.sb_group + ((live ? n0 : last_n) / 128) * p.sb_n;
    const bool any = p.any_scales != 0;
    const uint32_t sign = any ? 0x7fffffffu : 0xffffffffu;  // a negative scale is far where it is not admitted
    for (; row0 < row_end; row0 += NT * COLS) {
        const int64_t last_r = row_end - 1;
        float run[NT][4];
        const uint8_t *tok[NT];
        int64_t col[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int64_t r = row0 + j * COLS;
            tok[j] = a + (r + g < last_r ? r + g : last_r) * ld;
#pragma unroll
            for (int i = 0; i < 2; ++i) col[j][i] = r + 2 * t + i < last_r ? r + 2 * t + i : last_r;
#pragma unroll
            for (int i = 0; i < 4; ++i) run[j][i] = 0.0f;
        }
        // The scales are looked at as they pass, without a branch that would
        // keep the next block's loads behind it; where one is not admitted or
        // far from 1 the strip is done again.  16 rows by 8 matrices of 4096 x
        // 1024 take 7 % longer for it (looked up before the loop or after it 14 to 18).
        uint32_t far = 0, bits = 0;
        auto look = [&](float scale) {
            const uint32_t b = __float_as_uint(scale) & sign;
            far = max(far, b - gemm8::NEAR_LOW);
            bits |= b;
        };
        auto strip = [&](auto odd) {
            constexpr bool ODD = decltype(odd)::value;
            bool bad = false;
#pragma unroll(ODD ? 1 : 2)
            for (int kb = turn; kb < p.kblocks; kb += share) {
                const int64_t k = static_cast<int64_t>(kb) * 128 + t * 16;
                const bool ok0 = k < ld, ok1 = k + 64 < ld;
                const uint4 x0 = load16(w0 + k, ok0), x1 = load16(w1 + k, ok0);
                const uint4 y0 = load16(w0 + k + 64, ok1), y1 = load16(w1 + k + 64, ok1);
                const float s = __ldg(sb + kb);
                if (!ODD) look(s);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const uint4 u = load16(tok[j] + k, ok0), v = load16(tok[j] + k + 64, ok1);
                    const float a0 = __ldg(p.sa + kb * p.rows + col[j][0]);
                    const float a1 = __ldg(p.sa + kb * p.rows + col[j][1]);
                    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma<E5A, E5B>(d, {x0.x, x1.x, x0.y, x1.y}, u.x, u.y);
                    mma<E5A, E5B>(d, {x0.z, x1.z, x0.w, x1.w}, u.z, u.w);
                    mma<E5A, E5B>(d, {y0.x, y1.x, y0.y, y1.y}, v.x, v.y);
                    mma<E5A, E5B>(d, {y0.z, y1.z, y0.w, y1.w}, v.z, v.w);
                    if (ODD) {
                        bad |= !any && !(gemm8::power_of_two(__float_as_uint(s)) && gemm8::power_of_two(__float_as_uint(a0)) &&
                                         gemm8::power_of_two(__float_as_uint(a1)));
                        const float sw = gemm8::admitted(s, any), c0 = gemm8::admitted(a0, any), c1 = gemm8::admitted(a1, any);
#pragma unroll
                        for (int i = 0; i < 4; ++i) run[j][i] += scaled(d[i], i & 1 ? c1 : c0, sw);
                    } else {
                        look(a0);
                        look(a1);
                        const float s0 = s * a0, s1 = s * a1;
                        run[j][0] = fmaf(d[0], s0, run[j][0]);
                        run[j][1] = fmaf(d[1], s1, run[j][1]);
                        run[j][2] = fmaf(d[2], s0, run[j][2]);
                        run[j][3] = fmaf(d[3], s1, run[j][3]);
                    }
                }
            }
            if (bad) report_device_error(DEVERR_SCALE);
        };
        if (live) {
            strip(std::false_type{});
            if (__any_sync(0xffffffffu, far > gemm8::NEAR_SPAN || (!any && (bits & 0x7fffffu) != 0))) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) run[j][i] = 0.0f;
                strip(std::true_type{});
            }
        }
        // part[warp][token][weight row]
        if (share > 1) __syncthreads();  // the last pass has been read
        else __syncwarp();
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float *q = part + (warp * (NT * COLS) + j * COLS + 2 * t) * STRIP + g;
            q[0] = run[j][0];
            q[STRIP] = run[j][1];
            q[8] = run[j][2];
            q[STRIP + 8] = run[j][3];
        }
        if (share > 1) __syncthreads();
        else __syncwarp();
        // a strip's sums, by the warps that share it
        const float *sum = part + mine * share * (NT * COLS * STRIP);
        for (int i = turn * 32 + lane; i < NT * COLS * STRIP; i += share * 32) {
            const int64_t row = row0 + i / STRIP, n = n0 + i % STRIP;
            if (row >= row_end || n >= p.n) continue;
            float v = sum[i];
            for (int x = 1; x < share; ++x) v += sum[x * (NT * COLS * STRIP) + i];
            const int64_t o = row * p.n + n;
            if (p.out_dtype == CHELIS_DTYPE_F32) static_cast<float *>(p.out)[o] = v;
            else if (p.out_dtype == CHELIS_DTYPE_BF16)
                static_cast<__nv_bfloat16 *>(p.out)[o] = __float2bfloat16_rn(v);
            else static_cast<__half *>(p.out)[o] = __float2half_rn(v);
        }
    }
}

template <bool E5A, bool E5B>
void launch(const uint8_t *a, const uint8_t *w, const Params &p, int64_t ld, bool wide, int share, dim3 grid,
            cudaStream_t s) {
    if (wide) few8_kernel<E5A, E5B, 4><<<grid, WARPS * 32, 0, s>>>(p, a, w, ld, share);
    else few8_kernel<E5A, E5B, 1><<<grid, WARPS * 32, 0, s>>>(p, a, w, ld, share);
}

int run(const uint8_t *a, const uint8_t *w, const Params &p, int64_t ld, int32_t fa, int32_t fb) {
    // measured with 2048 strips 4 against 8 warps a strip 10.4 and 12.1 us, with
    // 256 strips of 64 rows 10.9 and 9.0, of one row and K = 4096 10.1 and 7.4
    const int64_t strips = (p.n + STRIP - 1) / STRIP * p.groups;
    int share = strips <= 512 ? 8 : 4;
    while (share > p.kblocks) share /= 2;
    const int64_t per = WARPS / share * STRIP;
    const dim3 grid(static_cast<unsigned>((p.n + per - 1) / per),
                    static_cast<unsigned>(p.groups + (p.offsets ? 1 : 0)));
    cudaStream_t s = current_stream();
    const bool ea = fa == CHELIS_FORMAT_E5M2, eb = fb == CHELIS_FORMAT_E5M2;
    const bool wide = p.rows > COLS * static_cast<int64_t>(p.groups);
    if (ea && eb) launch<true, true>(a, w, p, ld, wide, share, grid, s);
    else if (ea) launch<true, false>(a, w, p, ld, wide, share, grid, s);
    else if (eb) launch<false, true>(a, w, p, ld, wide, share, grid, s);
    else launch<false, false>(a, w, p, ld, wide, share, grid, s);
    g_launches++;
    CHELIS_LAUNCH_CHECK("few8::few8_kernel");
    return CHELIS_CUDA_OK;
}

}  // namespace few8
}  // namespace chelis
