// gemm_blocks8.cu -- products of 8-bit matrices with a scale for each block
// of 128 (blocks8.cu) on the sm_100a tensor cores, dense or by expert.
//
//   y[t, n]    = sum_b sa[b, t] sb[n / 128, b] sum_{k in b} a[t, k] w[n, k]
//   dx[t, k]   = sum_b sa[b, t] sb[b, k / 128] sum_{n in b} a[t, n] w[n, k]
//   dw[n, k]   = sum_b sa[b, n] sx[b, k]       sum_{t in b} a[n, t] x[k, t]
//
// The first two take row blocks (a) and tiles (w); the second reads the same
// bytes of w with the contraction along its rows (an MN-major operand), so
// no transposed copy is made.  The third takes two transposed operands.  By
// expert, the rows [offsets[e], offsets[e + 1]) of a meet matrix e of w, and
// dw has one matrix an expert, summed over that expert's blocks.
//
// One thread block works on 128 x 256 tiles of the result, one after the
// other (320 threads):
//   warp 0      TMA producer (one elected lane)
//   warp 1      TMEM allocator + tcgen05.mma kind::f8f6f4 issuer (one lane)
//   warps 2-9   fold: the block's sum in tensor memory times its scales into
//               f32 registers, then the store
// The scales differ from block to block, so the tensor core sums one block
// of 128 (four MMAs of K = 32) from a fresh start, alternating between two
// 256-column accumulators, and the fold adds it in IEEE f32 while the next
// block runs.  That also keeps the sum as exact as f32: one long TMEM
// accumulator truncates, and its error grows with K.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "common.cuh"

namespace chelis {

extern std::atomic<uint64_t> g_launches;

namespace gemm8 {

constexpr int BM = 128, BN = 256, BK = 128;  // one scale block of K = 128 bytes = one swizzle row
constexpr int STAGES = 4;
constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK;
constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int FOLD_WARPS = 8;
constexpr int THREADS = 64 + 32 * FOLD_WARPS;
constexpr uint32_t ACC_COLS = 256, TMEM_COLS = 512;
constexpr int MAX_GROUPS = experts::MAX_EXPERTS;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 /*align*/ + 256 /*barriers*/ +
                           FOLD_WARPS * BK * 4 /*column scales*/ + (MAX_GROUPS + 1) * 4 /*tile starts*/;

struct Params {
    int64_t rows;     // rows of a: tokens (forward, input gradient), outputs (weight gradient)
    int64_t n;        // columns of the result
    int32_t kblocks;  // blocks of the contraction (weight gradient: of all groups)
    int32_t groups;   // experts; 1 without offsets
    const int32_t *offsets;
    int64_t group_rows;  // weight gradient: rows that the offsets count
    const float *sa;     // [kblocks][rows]
    const float *sb;     // tiles, or [kblocks][n] (weight gradient)
    int64_t sb_group, sb_n, sb_k;  // tiles: strides of expert, column block, contraction block
    void *out;
    int32_t out_dtype;
    uint32_t idesc;
};

__device__ __forceinline__ void mma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// MN-major 8-bit operand: boxes of 128 (MN) x 128 (K) bytes, one 128-byte row
// along MN for each k, 8-row swizzle atoms.  LBO = the next 128 of MN (the
// next box), SBO = the next 8 of K (1024 B).
__device__ __forceinline__ uint64_t mnmajor_desc(uint32_t addr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>((128u * 128u) >> 4) << 16;
    d |= static_cast<uint64_t>(1024u >> 4) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    d |= static_cast<uint64_t>(2u) << 61;
    return d;
}

// First and last + 1 row of group g, held to [0, rows].
__device__ __forceinline__ void group_span(const Params &p, int64_t rows, int g, int64_t *lo, int64_t *hi) {
    if (!p.offsets) {
        *lo = 0;
        *hi = rows;
        return;
    }
    int64_t a = p.offsets[g], b = p.offsets[g + 1];
    a = a < 0 ? 0 : (a > rows ? rows : a);
    b = b < a ? a : (b > rows ? rows : b);
    *lo = a;
    *hi = b;
}

// One tile of the result.
struct Tile {
    int group;
    int64_t m0, m_end;  // rows of the result, this tile's first and the group's last + 1
    int64_t n0;
    int kb0, kbs;       // contraction blocks
};

// `start` is, by group, the prefix of row tiles (forward, input gradient) or
// of contraction blocks (weight gradient).
template <bool WG>
__device__ __forceinline__ Tile tile_at(const Params &p, const int32_t *start, int64_t L) {
    const int64_t nt = (p.n + BN - 1) / BN;
    Tile t;
    if (WG) {
        const int64_t mt = (p.rows + BM - 1) / BM;
        t.group = static_cast<int>(L / (mt * nt));
        const int64_t in = L - t.group * mt * nt;
        t.m0 = (in % mt) * BM;
        t.n0 = (in / mt) * BN;
        t.m_end = p.rows;
        t.kb0 = start[t.group];
        t.kbs = start[t.group + 1] - t.kb0;
    } else {
        int lo = 0, hi = p.groups;  // the last group whose first tile is at or before L
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start[mid] * nt <= L) lo = mid;
            else hi = mid;
        }
        t.group = lo;
        const int64_t in = L - start[lo] * nt, mt = start[lo + 1] - start[lo];
        int64_t a, b;
        group_span(p, p.rows, lo, &a, &b);
        t.m0 = a + (in % mt) * BM;
        t.n0 = (in / mt) * BN;
        t.m_end = b;
        t.kb0 = 0;
        t.kbs = p.kblocks;
    }
    return t;
}

__device__ __forceinline__ void store_row(const Params &p, const float (&run)[128], int64_t index,
                                          int64_t left) {
    if (p.out_dtype == CHELIS_DTYPE_F32) {
        float *o = static_cast<float *>(p.out) + index;
        if (left >= 128 && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
#pragma unroll
            for (int j = 0; j < 128; j += 4)
                *reinterpret_cast<float4 *>(o + j) = make_float4(run[j], run[j + 1], run[j + 2], run[j + 3]);
        } else {
#pragma unroll
            for (int j = 0; j < 128; ++j)
                if (j < left) o[j] = run[j];
        }
        return;
    }
    const bool bf = p.out_dtype == CHELIS_DTYPE_BF16;
    uint16_t *o = static_cast<uint16_t *>(p.out) + index;
    const bool vec = left >= 128 && (reinterpret_cast<uintptr_t>(o) & 15) == 0;
#pragma unroll
    for (int j = 0; j < 128; j += 8) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float lo = run[j + 2 * i], hi = run[j + 2 * i + 1];
            if (bf) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __half2 h = __floats2half2_rn(lo, hi);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        if (vec) {
            *reinterpret_cast<uint4 *>(o + j) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (j + i < left) o[j + i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
        }
    }
}

// BMN: b is read with its rows along the contraction (the input gradient).
// WG: the weight gradient (groups along the contraction, scales on both sides).
template <bool BMN, bool WG>
__global__ void __launch_bounds__(THREADS, 1)
    gemm8_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const Params p) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + STAGES * STAGE_BYTES);
    uint64_t *empty = full + STAGES;
    uint64_t *acc_full = empty + STAGES;   // [2]
    uint64_t *acc_empty = acc_full + 2;    // [2]
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
    volatile uint32_t *abort_flag = tmem_slot + 1;
    volatile int32_t *consumed = reinterpret_cast<volatile int32_t *>(tmem_slot + 2);
    float *col_scale = reinterpret_cast<float *>(smem + STAGES * STAGE_BYTES + 256);
    int32_t *start = reinterpret_cast<int32_t *>(col_scale + FOLD_WARPS * BK);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], FOLD_WARPS);
        }
        *abort_flag = 0;
        *consumed = 0;
        fence_mbarrier_init();
        prefetch_tensormap(&map_a);
        prefetch_tensormap(&map_b);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, TMEM_COLS);
        tmem_relinquish();
    }
    if (warp == 2) {
        // prefix over groups of row tiles or contraction blocks (both of 128),
        // held to what ordered offsets give at most
        const int64_t count = WG ? p.group_rows : p.rows;
        const int most = WG ? p.kblocks : static_cast<int>((count + 127) / 128) + p.groups;
        int base = 0;
        for (int g0 = 0; g0 < p.groups; g0 += 32) {
            int c = 0;
            if (g0 + lane < p.groups) {
                int64_t lo, hi;
                group_span(p, count, g0 + lane, &lo, &hi);
                c = static_cast<int>((hi - lo + 127) / 128);
            }
            int sum = c;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, sum, off);
                if (lane >= off) sum += o;
            }
            if (g0 + lane < p.groups) start[g0 + lane + 1] = min(base + sum, most);
            base = min(base + __shfl_sync(0xffffffffu, sum, 31), most);
        }
        if (lane == 0) start[0] = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int64_t nt = (p.n + BN - 1) / BN;
    const int64_t tiles = WG ? p.groups * nt * ((p.rows + BM - 1) / BM) : start[p.groups] * nt;
    int32_t issued = 0;

    if (warp == 0) {
        if (lane == 0) {
            int32_t it = 0;
            bool ok = true;
            for (int64_t L = blockIdx.x; ok && L < tiles; L += gridDim.x) {
                const Tile t = tile_at<WG>(p, start, L);
                for (int i = 0; i < t.kbs; ++i, ++it) {
                    const int s = it % STAGES;
                    if (!mbar_wait_bounded(&empty[s], ((it / STAGES) & 1) ^ 1, DEVERR_TIMEOUT_PRODUCER)) {
                        *abort_flag = 1;
                        ok = false;
                        break;
                    }
                    unsigned char *st = smem + s * STAGE_BYTES;
                    mbar_arrive_expect_tx(&full[s], STAGE_BYTES);
                    const int32_t k0 = (t.kb0 + i) * BK;
                    tma_load_2d(st, &map_a, &full[s], k0, static_cast<int32_t>(t.m0));
#pragma unroll
                    for (int h = 0; h < BN / 128; ++h) {
                        unsigned char *dst = st + A_BYTES + h * (128 * BK);
                        const int32_t n0 = static_cast<int32_t>(t.n0) + h * 128;
                        if (WG) tma_load_2d(dst, &map_b, &full[s], k0, n0);
                        else if (BMN) tma_load_3d(dst, &map_b, &full[s], n0, k0, t.group);
                        else tma_load_3d(dst, &map_b, &full[s], k0, n0, t.group);
                    }
                    issued = it + 1;
                }
                if (*abort_flag) ok = false;
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int32_t it = 0;
            int cur = 0;
            bool ok = true;
            for (int64_t L = blockIdx.x; ok && L < tiles; L += gridDim.x) {
                const Tile t = tile_at<WG>(p, start, L);
                for (int i = 0; i < t.kbs; ++i, ++it) {
                    cur = it & 1;
                    if (it >= 2) {
                        if (!mbar_wait_bounded(&acc_empty[cur], ((it >> 1) - 1) & 1, DEVERR_TIMEOUT_MMA)) {
                            *abort_flag = 1;
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                    }
                    const int s = it % STAGES;
                    if (!mbar_wait_bounded(&full[s], (it / STAGES) & 1, DEVERR_TIMEOUT_MMA)) {
                        *abort_flag = 1;
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = smem_u32(smem + s * STAGE_BYTES), b = a + A_BYTES;
                    const uint32_t d = tmem_base + static_cast<uint32_t>(cur) * ACC_COLS;
#pragma unroll
                    for (int kk = 0; kk < BK / 32; ++kk)
                        mma_f8(d, sw128_kmajor_desc(a + kk * 32),
                               BMN ? mnmajor_desc(b + kk * 32 * 128) : sw128_kmajor_desc(b + kk * 32),
                               p.idesc, kk != 0);
                    mma_commit(&empty[s]);
                    *consumed = it + 1;
                    mma_commit(&acc_full[cur]);
                }
                if (*abort_flag) ok = false;
            }
            if (*abort_flag) mma_commit(&acc_full[cur]);  // let the fold see the flag
        }
    } else {
        const int quad = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        float *cs = col_scale + (warp - 2) * BK;
        int32_t it = 0;
        bool ok = true;
        for (int64_t L = blockIdx.x; ok && L < tiles; L += gridDim.x) {
            const Tile t = tile_at<WG>(p, start, L);
            const int64_t row = t.m0 + quad * 32 + lane, col0 = t.n0 + half * 128;
            const int64_t srow = row < p.rows ? row : p.rows - 1;
            float run[128];
#pragma unroll
            for (int j = 0; j < 128; ++j) run[j] = 0.0f;
            for (int i = 0; i < t.kbs; ++i, ++it) {
                const int64_t kb = t.kb0 + i;
                float s = p.sa[kb * p.rows + srow];
                if (WG) {
                    __syncwarp();
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int64_t c = col0 + u * 32 + lane;
                        cs[u * 32 + lane] = c < p.n ? p.sb[kb * p.n + c] : 0.0f;
                    }
                    __syncwarp();
                } else if (col0 < p.n) {
                    s *= p.sb[t.group * p.sb_group + (col0 / 128) * p.sb_n + kb * p.sb_k];
                }
                const int b = it & 1;
                if (!mbar_wait_bounded(&acc_full[b], (it >> 1) & 1, DEVERR_TIMEOUT_EPILOGUE)) {
                    *abort_flag = 1;
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (*abort_flag) {
                    ok = false;
                    break;
                }
                const uint32_t acc = tmem_base + lanes + static_cast<uint32_t>(b) * ACC_COLS + half * 128;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t r[32];
                    tmem_ld_32x32b_x32(acc + j * 32, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < 32; ++c) {
                        float v = __uint_as_float(r[c]);
                        if (WG) v *= cs[j * 32 + c];
                        run[j * 32 + c] = fmaf(v, s, run[j * 32 + c]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&acc_empty[b]);
            }
            if (ok && row < t.m_end && col0 < p.n) {
                const int64_t base = WG ? t.group * p.rows * p.n : 0;
                store_row(p, run, base + row * p.n + col0, p.n - col0);
            }
        }
        // rows of the result that no group holds
        if (!WG && p.offsets) {
            int64_t a, b, first, last;
            group_span(p, p.rows, 0, &first, &b);
            group_span(p, p.rows, p.groups - 1, &a, &last);
            const int64_t bytes = p.out_dtype == CHELIS_DTYPE_F32 ? 4 : 2;
            unsigned char *o = static_cast<unsigned char *>(p.out);
            const int64_t who = static_cast<int64_t>(blockIdx.x) * (FOLD_WARPS * 32) + threadIdx.x - 64;
            const int64_t step = static_cast<int64_t>(gridDim.x) * (FOLD_WARPS * 32);
            const int64_t loose = (first + p.rows - last) * p.n;
            for (int64_t i = who; i < loose; i += step) {
                const int64_t e = i < first * p.n ? i : last * p.n + (i - first * p.n);
                if (bytes == 4) reinterpret_cast<float *>(o)[e] = 0.0f;
                else reinterpret_cast<uint16_t *>(o)[e] = 0;
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    // after an abort, copies that were issued but not consumed land first
    if (warp == 0 && lane == 0 && *abort_flag)
        for (int32_t it = *consumed; it < issued; ++it)
            mbar_wait_bounded(&full[it % STAGES], (it / STAGES) & 1, DEVERR_TIMEOUT_PRODUCER);
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
}

// 8-bit tensor [batch][rows][ld] -> boxes of 128 (contiguous axis) x 128 rows;
// what lies past cols or rows reads as zero.
int make_map(CUtensorMap *map, const void *base, int64_t cols, int64_t ld, int64_t rows, int64_t batch,
             bool rank3) {
    tf32x3::EncodeTiledFn fn = tf32x3::encode_fn();
    if (!fn) return set_error(CHELIS_CUDA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows),
                          static_cast<cuuint64_t>(batch)};
    cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld), static_cast<cuuint64_t>(ld * rows)};
    cuuint32_t box[3] = {128, 128, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank3 ? 3 : 2, const_cast<void *>(base), dims,
                    strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return set_error(CHELIS_CUDA_ERR_CUDA, "cuTensorMapEncodeTiled(8-bit) failed (%d)", (int)r);
    return CHELIS_CUDA_OK;
}

uint32_t instruction(int32_t format_a, int32_t format_b, bool bmn) {
    return (1u << 4) |                                            // f32 sums
           (format_a == CHELIS_FORMAT_E5M2 ? 1u << 7 : 0u) |      // 0 e4m3, 1 e5m2
           (format_b == CHELIS_FORMAT_E5M2 ? 1u << 10 : 0u) |
           (bmn ? 1u << 16 : 0u) |                                // b MN-major
           (static_cast<uint32_t>(BN >> 3) << 17) | (static_cast<uint32_t>(BM >> 4) << 24);
}

template <bool BMN, bool WG>
int launch(const CUtensorMap &ma, const CUtensorMap &mb, const Params &p, int64_t most_tiles) {
    CHELIS_TRY(check_cuda(cudaFuncSetAttribute(gemm8_kernel<BMN, WG>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES),
                          "cudaFuncSetAttribute"));
    const int64_t sms = sm_count();
    const unsigned grid = static_cast<unsigned>(most_tiles < sms ? (most_tiles < 1 ? 1 : most_tiles) : sms);
    gemm8_kernel<BMN, WG><<<grid, THREADS, SMEM_BYTES, current_stream()>>>(ma, mb, p);
    g_launches++;
    CHELIS_LAUNCH_CHECK("gemm8::gemm8_kernel");
    return CHELIS_CUDA_OK;
}

int check_common(const char *op, int32_t fa, int32_t fb, int32_t out_dtype, int64_t rows, int64_t n,
                 int64_t k, const int32_t *offsets, int32_t groups) {
    CHELIS_TRY(blocks8::check_format(op, fa));
    CHELIS_TRY(blocks8::check_format(op, fb));
    if (!experts::is_act(out_dtype))
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "%s gives f32, bf16 or f16", op);
    if (rows < 0 || n < 0 || k < 0 || groups < 1 || (!offsets && groups != 1))
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "%s: extents >= 0, groups >= 1, more than one with offsets", op);
    if (groups > MAX_GROUPS)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "%s admits %d groups at most", op, MAX_GROUPS);
    // tensor-map coordinates and the counts of tiles are 32-bit
    if (rows > INT32_MAX - 512 || n > INT32_MAX - 512 || k > INT32_MAX - 512)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "%s: an extent above 2^31", op);
    return CHELIS_CUDA_OK;
}

int zero_out(void *out, int32_t dtype, int64_t count) {
    return check_cuda(cudaMemsetAsync(out, 0, static_cast<size_t>(count * experts::width(dtype)),
                                      current_stream()), "memset");
}

}  // namespace gemm8
}  // namespace chelis

using namespace chelis;

extern "C" int chelis_cuda_matmul8(int32_t format_a, int32_t format_b, int trans_b, int64_t rows,
                                   int64_t n, int64_t k, const uint8_t *a, const float *scales_a,
                                   const uint8_t *b, const float *scales_b, const int32_t *offsets,
                                   int32_t groups, int32_t out_dtype, void *out) {
    CHELIS_TRY(gemm8::check_common("matmul8", format_a, format_b, out_dtype, rows, n, k, offsets, groups));
    if (rows == 0 || n == 0) return CHELIS_CUDA_OK;
    if (!out) return set_error(CHELIS_CUDA_ERR_DOMAIN, "matmul8: null operand");
    if (k == 0) return gemm8::zero_out(out, out_dtype, rows * n);
    if (!a || !scales_a || !b || !scales_b)
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "matmul8: null operand");
    if (!experts::aligned16(a) || !experts::aligned16(b))
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "matmul8: 8-bit data must lie on 16 bytes");
    const int64_t kblocks = (k + 127) / 128, nblocks = (n + 127) / 128;
    CUtensorMap ma, mb;
    CHELIS_TRY(gemm8::make_map(&ma, a, k, blocks8::round16(k), rows, 1, false));
    if (trans_b) CHELIS_TRY(gemm8::make_map(&mb, b, k, blocks8::round16(k), n, groups, true));
    else CHELIS_TRY(gemm8::make_map(&mb, b, n, blocks8::round16(n), k, groups, true));
    gemm8::Params p{};
    p.rows = rows;
    p.n = n;
    p.kblocks = static_cast<int32_t>(kblocks);
    p.groups = groups;
    p.offsets = offsets;
    p.sa = scales_a;
    p.sb = scales_b;
    p.sb_group = kblocks * nblocks;
    p.sb_n = trans_b ? kblocks : 1;
    p.sb_k = trans_b ? 1 : nblocks;
    p.out = out;
    p.out_dtype = out_dtype;
    p.idesc = gemm8::instruction(format_a, format_b, !trans_b);
    const int64_t most = ((rows + 127) / 128 + (offsets ? groups : 0)) * ((n + gemm8::BN - 1) / gemm8::BN);
    return trans_b ? gemm8::launch<false, false>(ma, mb, p, most) : gemm8::launch<true, false>(ma, mb, p, most);
}

extern "C" int chelis_cuda_matmul8_wgrad(int32_t format_a, int32_t format_b, int64_t n, int64_t k,
                                         int64_t places, const uint8_t *a, const float *scales_a,
                                         const uint8_t *b, const float *scales_b,
                                         const int32_t *offsets, int32_t groups, int32_t out_dtype,
                                         void *out) {
    CHELIS_TRY(gemm8::check_common("matmul8_wgrad", format_a, format_b, out_dtype, places, n, k, offsets, groups));
    if (places % 128 != 0) return set_error(CHELIS_CUDA_ERR_DOMAIN, "matmul8_wgrad: places in blocks of 128");
    if (n == 0 || k == 0) return CHELIS_CUDA_OK;
    if (!out) return set_error(CHELIS_CUDA_ERR_DOMAIN, "matmul8_wgrad: null operand");
    if (places == 0) return gemm8::zero_out(out, out_dtype, groups * n * k);
    if (!a || !scales_a || !b || !scales_b)
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "matmul8_wgrad: null operand");
    if (!experts::aligned16(a) || !experts::aligned16(b))
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "matmul8_wgrad: 8-bit data must lie on 16 bytes");
    CUtensorMap ma, mb;
    CHELIS_TRY(gemm8::make_map(&ma, a, places, places, n, 1, false));
    CHELIS_TRY(gemm8::make_map(&mb, b, places, places, k, 1, false));
    gemm8::Params p{};
    p.rows = n;
    p.n = k;
    p.kblocks = static_cast<int32_t>(places / 128);
    p.groups = groups;
    p.offsets = offsets;
    p.group_rows = places;  // the rows are no more
    p.sa = scales_a;
    p.sb = scales_b;
    p.out = out;
    p.out_dtype = out_dtype;
    p.idesc = gemm8::instruction(format_a, format_b, false);
    const int64_t most = groups * ((n + 127) / 128) * ((k + gemm8::BN - 1) / gemm8::BN);
    return gemm8::launch<false, true>(ma, mb, p, most);
}
