// linear16.cu -- products of bf16 or f16 matrices with f32 sums and what
// follows them in the same kernel, and what their gradients need besides:
//
//   z = op(a) . op(b) + bias,   y = act(z) + residual      (z stored on request)
//   y = (op(a) . op(b)) * act'(through)                    (a gradient's product)
//   dz = dy * act'(z);  column sums                        (act_bwd, column_sums)
//
// act is none, relu, gelu or silu (linear16.cuh); every result is rounded once,
// from f32, and act is taken of the sum before z is rounded.
//
// pair_kernel: a pair of thread blocks (cta_group::2) works on a 256 x 256 tile,
// each with its 128 rows of a and half of b's columns in shared memory (stages
// of 64 along the contraction, 128 bytes, TMA) and its 128 rows of the f32 sums
// in tensor memory, which holds two such tiles: warps 4 to 19 read one, 32 rows
// and 64 columns each, finish and store it while the tensor core fills the other.
// Either operand may lie with its rows along the contraction (a descriptor bit),
// so no product of a layer or of its gradients turns a matrix over.
//
// What bounds it: at the tensor core's full rate a multiprocessor takes 64 bytes a
// clock of operands into shared memory and reads 64 out again, which is all that
// shared memory does; the issuer waits for a stage 3700 of the 10400 clocks of a
// tile of K = 1024 (8192 at full rate).  16384 x 4096 x 1024 without any epilogue 91
// us (1510 TFLOP/s), with the plain one 103 to 107, with bias, gelu and pre 134;
// 16384 x 1024 x 4096 with bias and residual 105 (256 tiles on 74 pairs: 3.5 rounds
// of 4); 8192^3 720 (1528 TFLOP/s).  The card is at its power cap in these (1.4 GHz).
// Stages of 5, 6 and 7: no change.  Eight warps of 128 columns in place of sixteen of
// 64: 184 for 143 us at the time.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "linear16.cuh"

namespace chelis {

extern std::atomic<uint64_t> g_launches;

namespace linear16 {

using gemm8::all;
using gemm8::arrive_relaxed;
using gemm8::band_order;
using gemm8::elect_one;
using gemm8::landed;
using gemm8::probe;
using gemm8::round2;
using gemm8::store_box;
using gemm8::uniform;
using gemm8::wait;

constexpr uint64_t DRAIN_NS = 200000;   // bounded drain of an aborted pair's second block
constexpr int BM = 128, TM = 256, TN = 256, BK = 64;
constexpr int BOX_BYTES = 128 * BK * 2;  // 128 rows or columns of one stage
constexpr int HALF_BOX = BOX_BYTES / 2;  // MN-major: 64 of them
constexpr int STAGE = 2 * BOX_BYTES, STAGES = 5;
constexpr int OUT_WARPS = 16, THREADS = 128 + 32 * OUT_WARPS;
// Registers: the launch's 640 x 96, of which the first warpgroup gives some up.
constexpr int LAUNCH_REGS = 96, FEW_REGS = 40, FINISH_REGS = 104;
static_assert(128 * FEW_REGS + 32 * OUT_WARPS * FINISH_REGS <= THREADS * LAUNCH_REGS, "register split");
constexpr int PIECE = 16;                // columns finished at once
constexpr int BOX = 2048, BOXES = 2;     // 32 rows x 64 bytes, two a warp
constexpr int SMEM_BYTES = STAGES * STAGE + OUT_WARPS * BOXES * BOX + 1024 /*align*/ + 512 /*barriers*/;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");

constexpr int32_t ANY_ACT = -1;          // of the kernels that are compiled for no one activation
enum : int32_t { AUX_NONE = 0, AUX_RESIDUAL = 1, AUX_THROUGH = 2 };

// What follows the sums.
struct Finish {
    const void *bias;     // [n] or NULL
    const void *aux;      // [m][n] of the result's type: residual or through
    void *out, *pre;      // [m][n]; pre may be NULL
    int32_t dtype;        // of out, pre and aux
    int32_t bias_dtype;
    int32_t bias_vec;     // 8 of them load as 16 bytes
    int32_t act, aux_kind;
};

struct Params {
    int64_t m, n;
    int32_t kblocks, parts;
    int32_t tn;           // columns of a tile: 256, or 128
    uint32_t idesc;
    int32_t vec;          // rows of the results start on 16 (1) or 32 bytes (2)
    int32_t aux_tma;      // aux, of 16 bits, comes by TMA
    int32_t amn, bmn;     // the operand's rows lie along the contraction
    Finish f;
};

__device__ __forceinline__ float load_f32(const void *p, int64_t i, int32_t dtype) {
    if (dtype == CHELIS_DTYPE_F32) return static_cast<const float *>(p)[i];
    if (dtype == CHELIS_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    return __half2float(static_cast<const __half *>(p)[i]);
}
__device__ __forceinline__ void store_f32(void *p, int64_t i, int32_t dtype, float v) {
    if (dtype == CHELIS_DTYPE_F32) static_cast<float *>(p)[i] = v;
    else if (dtype == CHELIS_DTYPE_BF16) static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half *>(p)[i] = __float2half_rn(v);
}
template <bool BF>
__device__ __forceinline__ f32x2 wide2(uint32_t w) {
    if (BF) return gemm8::pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    return gemm8::pack2(f.x, f.y);
}
// One element's way from its sum to memory (the kernels without tiles).
__device__ __forceinline__ void finish_one(const Finish &f, float z, int64_t row, int64_t col, int64_t n) {
    const int64_t i = row * n + col;
    if (f.bias) z += load_f32(f.bias, col, f.bias_dtype);
    if (f.pre) store_f32(f.pre, i, f.dtype, z);
    float y;
    if (f.aux_kind == AUX_THROUGH) {
        y = slope_times(z, load_f32(f.aux, i, f.dtype), f.act);
    } else {
        y = value(z, f.act);
        if (f.aux_kind == AUX_RESIDUAL) y += load_f32(f.aux, i, f.dtype);
    }
    store_f32(f.out, i, f.dtype, y);
}

// A piece's biases from `col` on, added to its sums; past n there are none.
template <bool BF>
__device__ __forceinline__ void add_bias(const Finish &f, int col, int n, f32x2 (&v)[PIECE / 2]) {
    if (f.bias_vec && col + PIECE <= n) {
        if (f.bias_dtype == CHELIS_DTYPE_F32) {
            const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(f.bias) + col);
#pragma unroll
            for (int c = 0; c < PIECE / 4; ++c) {
                const float4 u = __ldg(p + c);
                v[2 * c] = add2(v[2 * c], gemm8::pack2(u.x, u.y));
                v[2 * c + 1] = add2(v[2 * c + 1], gemm8::pack2(u.z, u.w));
            }
        } else {
            const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(f.bias) + col);
#pragma unroll
            for (int c = 0; c < PIECE / 8; ++c) {
                const uint4 u = __ldg(p + c);
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * c + i] = add2(v[4 * c + i], wide2<BF>(w[i]));
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < PIECE / 2; ++c) {
            const int at = col + 2 * c;
            v[c] = add2(v[c], gemm8::pack2(at < n ? load_f32(f.bias, at, f.bias_dtype) : 0.0f,
                                           at + 1 < n ? load_f32(f.bias, at + 1, f.bias_dtype) : 0.0f));
        }
    }
}

__device__ __forceinline__ void mma_f16_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// An operand's descriptor but for its address: K-major rows as sw128_kmajor_desc
// has them, or MN-major boxes of 64 (MN) x 64 (K), one 128-byte row along MN for
// each k, 8-row swizzle atoms (LBO = the next 64 of MN, the next box; SBO = the next
// 8 of K).  An MMA's 16 of K are 32 bytes or 16 rows further on.
__device__ __forceinline__ uint64_t operand_desc(bool mn) {
    return static_cast<uint64_t>(mn ? HALF_BOX >> 4 : 1) << 16 | static_cast<uint64_t>(1024u >> 4) << 32 |
           static_cast<uint64_t>(1u) << 46 | static_cast<uint64_t>(2u) << 61;
}
__device__ __forceinline__ uint64_t at_address(uint64_t desc, uint32_t addr) {
    return desc | static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
}

struct Tile {
    int m0, n0, part, kb0, kbs;
};
__device__ __forceinline__ Tile tile_at(const Params &p, int mt, int nt, int L) {
    Tile t;
    t.part = 0;
    t.kb0 = 0;
    t.kbs = p.kblocks;
    if (p.parts > 1) {
        t.part = L / (mt * nt);
        L -= t.part * (mt * nt);
        t.kb0 = static_cast<int>(static_cast<int64_t>(p.kblocks) * t.part / p.parts);
        t.kbs = static_cast<int>(static_cast<int64_t>(p.kblocks) * (t.part + 1) / p.parts) - t.kb0;
    }
    int m, n;
    band_order(L, mt, nt, &m, &n);
    t.m0 = m * TM;
    t.n0 = n * p.tn;
    return t;
}

// ---- between a warp's registers and its rows of the results -----------------
// A lane has a row.  Where rows start on 16 bytes, out goes through the warp's two
// boxes (32 rows x 64 bytes) by TMA, and 16-bit aux has come to them by TMA before
// the sums were ready.  pre goes from the registers to the lane's row, whole
// sectors: that takes the load and store unit 64 clocks a KB, which it has to spare
// once, not twice (16384 x 4096 x 1024, us: out alone 106 and 103 directly, f32 121
// and 137), and the boxes are too few for both.  Other rows go through a box, so that
// neighbouring lanes write neighbouring units.
__device__ __forceinline__ void wait_reads_all() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void wait_reads_but_last() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }

// 16-byte piece c of the lane's row of a box, in TMA's 64-byte swizzle.
__device__ __forceinline__ uint4 *box_at(unsigned char *box, int lane, int c) {
    return reinterpret_cast<uint4 *>(box + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4));
}
// The lane's 16 values as they are stored: 8 words, or 16 of f32.
template <bool F32, bool BF>
__device__ __forceinline__ void to_words(const f32x2 (&v)[PIECE / 2], uint32_t (&w)[F32 ? 16 : 8]) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        const float2 f = gemm8::unpack2(v[c]);
        if constexpr (F32) w[2 * c] = __float_as_uint(f.x), w[2 * c + 1] = __float_as_uint(f.y);
        else w[c] = round2(f, BF);
    }
}
template <bool F32, bool BF>
__device__ __forceinline__ void to_values(const uint32_t (&w)[F32 ? 16 : 8], f32x2 (&x)[PIECE / 2]) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        if constexpr (F32) x[c] = gemm8::pack2(__uint_as_float(w[2 * c]), __uint_as_float(w[2 * c + 1]));
        else x[c] = wide2<BF>(w[c]);
    }
}

// A piece to [m][n] at dst: columns `col` on of row `row` + lane, `rows` of the
// warp's 32 being there.
template <bool F32, bool BF>
__device__ __forceinline__ void put_piece(const Params &p, void *dst, unsigned char *box, int lane, const f32x2 (&v)[PIECE / 2],
                                          int row, int rows, int col, int part) {
    constexpr int W = F32 ? 4 : 2, WORDS = F32 ? 16 : 8;
    uint32_t w[WORDS];
    to_words<F32, BF>(v, w);
    const int left = static_cast<int>(p.n) - col;
    unsigned char *first = static_cast<unsigned char *>(dst) + ((part * p.m + row) * p.n + col) * W;
    if (p.vec) {
        if (lane >= rows) return;
        unsigned char *o = first + lane * p.n * W;
        if (p.vec == 2 && left >= PIECE) {
#pragma unroll
            for (int c = 0; c < WORDS; c += 8) {
                const uint32_t u[8] = {w[c], w[c + 1], w[c + 2], w[c + 3], w[c + 4], w[c + 5], w[c + 6], w[c + 7]};
                gemm8::store32(o + 4 * c, u);
            }
        } else {
#pragma unroll
            for (int c = 0; c < WORDS; c += 4)
                if (c * 4 < left * W) *reinterpret_cast<uint4 *>(o + 4 * c) = make_uint4(w[c], w[c + 1], w[c + 2], w[c + 3]);
        }
        return;
    }
    __syncwarp();
#pragma unroll
    for (int c = 0; c < WORDS; c += 4) *box_at(box, lane, c / 4) = make_uint4(w[c], w[c + 1], w[c + 2], w[c + 3]);
    __syncwarp();
    const int64_t ld = p.n * W;
    const int bytes = min(left, PIECE) * W;
    if (((reinterpret_cast<uintptr_t>(first) | ld) & 3) == 0) store_box<uint32_t>(box, lane, first, ld, rows, bytes);
    else store_box<uint16_t>(box, lane, first, ld, rows, bytes);
}
// A piece of aux, where TMA has not brought it.
template <bool F32, bool BF>
__device__ __forceinline__ void get_piece(const Params &p, unsigned char *box, int lane, int row, int rows, int col,
                                          f32x2 (&x)[PIECE / 2]) {
    using U = typename std::conditional<F32, uint32_t, uint16_t>::type;
    constexpr int W = F32 ? 4 : 2, WORDS = F32 ? 16 : 8;
    const int left = static_cast<int>(p.n) - col;
    uint32_t w[WORDS];
    if (p.vec) {
        const unsigned char *at = static_cast<const unsigned char *>(p.f.aux) + ((static_cast<int64_t>(row) + lane) * p.n + col) * W;
#pragma unroll
        for (int c = 0; c < WORDS; c += 4) {
            const bool in = lane < rows && c * 4 < left * W;
            const uint4 u = in ? *reinterpret_cast<const uint4 *>(at + 4 * c) : make_uint4(0, 0, 0, 0);
            w[c] = u.x, w[c + 1] = u.y, w[c + 2] = u.z, w[c + 3] = u.w;
        }
    } else {
        __syncwarp();
        const int c = lane % PIECE;
#pragma unroll 8
        for (int r0 = 0; r0 < 32; r0 += 2) {
            const int r = r0 + lane / PIECE, byte = c * W;
            const bool in = r < rows && c < left;
            const U v = in ? static_cast<const U *>(p.f.aux)[static_cast<int64_t>(row + r) * p.n + col + c] : U(0);
            *reinterpret_cast<U *>(box + r * 64 + (((byte >> 4) ^ ((r >> 1) & 3)) << 4) + (byte & 15)) = v;
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < WORDS; i += 4) {
            const uint4 u = *box_at(box, lane, i / 4);
            w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
        }
    }
    to_values<F32, BF>(w, x);
}

template <bool HOLD>
__device__ __forceinline__ void act_piece(const GeluConstants<HOLD> &k, f32x2 (&v)[PIECE / 2], const f32x2 (&x)[PIECE / 2],
                                          int32_t aux_kind, int32_t act) {
    if (aux_kind == AUX_THROUGH) {
#pragma unroll
        for (int c = 0; c < PIECE / 2; ++c) v[c] = slope_times(k, v[c], x[c], act);
        return;
    }
#pragma unroll
    for (int c = 0; c < PIECE / 2; ++c) v[c] = value(k, v[c], act);
    if (aux_kind == AUX_RESIDUAL)
#pragma unroll
        for (int c = 0; c < PIECE / 2; ++c) v[c] = add2(v[c], x[c]);
}

// ---- long contractions ------------------------------------------------------
// The tensor core's sum loses what lies below its last place at every 16 of k, so it
// drifts towards 0: by 1e-6 of it at k = 1024, 4.4e-6 at 4096, 1.9e-5 at 16384, 7.6e-5 at
// 65536 (normal numbers; 8e-5 at 16384 where all products have one sign).  In an f32
// result, such as a weight gradient over many tokens, that is far more than f32's own
// roundings.  So the kernels without an activation, whose contraction may be the long
// one (the f32 kernel also makes the parts), cut a tile's contraction into chunks, which
// take the two accumulators in turn, and their finishing warps add them up in registers,
// rounding as f32 does.  f32 results by chunks of 1024 at most: 1e-6 at any k, 1024 x 4096 x
// 16384 108 us for 105, 4096 x 4096 x 65536 1640 for 1630 (chunks of 4096, 4.4e-6: 106 and
// 1600).  16-bit results by chunks of 16384, whose drift is below half a step of f16 by a
// factor of 3 even where all products have one sign; smaller ones would not show, at 130
// us for 109 (16384 x 1024 x 4096, chunks of 2048).  With an activation there are no 64
// registers to spare.
constexpr int CHUNK_F32 = 16, CHUNK_16 = 256;  // blocks of the contraction
constexpr bool adds_chunks(int32_t act) { return act == CHELIS_ACT_NONE; }
constexpr int MOST_PIECES = TN / (4 * PIECE);
struct Chunks {
    int count, blocks;  // of a tile, of a chunk (the last one may have fewer)
};
template <bool LONG, bool F32>
__device__ __forceinline__ Chunks chunks_of(int kbs) {
    if constexpr (!LONG) return {1, kbs};
    constexpr int MOST = F32 ? CHUNK_F32 : CHUNK_16;
    const int count = (kbs + MOST - 1) / MOST;
    return {count, (kbs + count - 1) / count};
}
__device__ __forceinline__ int pieces_of(const Params &p, int col0) {
    return min((static_cast<int>(p.n) - col0 + PIECE - 1) / PIECE, p.tn / (4 * PIECE));
}
// A warp's sums of one chunk on top of those before.
__device__ __forceinline__ void add_chunk(uint32_t acc, int pieces, f32x2 (&sum)[MOST_PIECES][PIECE / 2]) {
#pragma unroll
    for (int i = 0; i < MOST_PIECES; ++i)
        if (i < pieces) {
            uint32_t r[PIECE];
            tmem_ld_32x32b_x16(acc + i * PIECE, r);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < PIECE / 2; ++c)
                sum[i][c] = add2(sum[i][c], gemm8::pack2(__uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1])));
        }
}

// One warp's piece i of its 32 rows and a quarter of the columns of a tile, from the
// sums, which sums(v) gives, to the results.  `used` counts the boxes that TMA has
// stored.
template <bool F32, bool BF, int32_t ACT, bool HOLD, typename Sums>
__device__ __forceinline__ void finish_piece(const Params &p, const CUtensorMap *map_out, unsigned char *boxes, unsigned char *&box,
                                             int &used, int lane, int row, int rows, int col0, int part, bool aux_here,
                                             const GeluConstants<HOLD> &constants, int i, int pieces, Sums sums) {
    constexpr int PER_BOX = F32 ? 1 : 2, WORDS = F32 ? 16 : 8;
    const int n = static_cast<int>(p.n), col = col0 + i * PIECE, odd = F32 ? 0 : i & 1;
    f32x2 v[PIECE / 2], x[PIECE / 2];
    if (p.vec && odd == 0) {
        if (aux_here) {
            box = boxes + i / 2 * BOX;
        } else {
            box = boxes + (used & 1) * BOX;
            if (lane == 0) wait_reads_but_last();
            __syncwarp();
        }
        ++used;
    }
    if (aux_here) {
        if constexpr (!F32) {
            uint32_t w[8];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint4 u = *box_at(box, lane, odd * 2 + c);
                w[4 * c] = u.x, w[4 * c + 1] = u.y, w[4 * c + 2] = u.z, w[4 * c + 3] = u.w;
            }
            to_values<F32, BF>(w, x);
        }
    } else if (p.f.aux_kind != AUX_NONE) {
        get_piece<F32, BF>(p, boxes, lane, row, rows, col, x);
    }
    sums(v);
    if (p.f.bias) add_bias<BF>(p.f, col, n, v);
    if (p.f.pre) put_piece<F32, BF>(p, p.f.pre, boxes, lane, v, row, rows, col, 0);
    act_piece(constants, v, x, p.f.aux_kind, ACT == ANY_ACT ? p.f.act : ACT);
    if (!p.vec) {
        put_piece<F32, BF>(p, p.f.out, boxes, lane, v, row, rows, col, part);
        return;
    }
    uint32_t w[WORDS];
    to_words<F32, BF>(v, w);
#pragma unroll
    for (int c = 0; c < WORDS; c += 4)
        *box_at(box, lane, odd * 2 + c / 4) = make_uint4(w[c], w[c + 1], w[c + 2], w[c + 3]);
    if (odd == PER_BOX - 1 || i + 1 == pieces) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            scaled8::tma_store_3d(map_out, smem_u32(box), col - odd * PIECE, row, part);
            scaled8::store_commit();
        }
    }
}
// All of its pieces from tensor memory, the next one's sums loading meanwhile.
template <bool F32, bool BF, int32_t ACT, bool HOLD, typename Release>
__device__ __forceinline__ void finish_tile(const Params &p, const CUtensorMap *map_out, unsigned char *boxes, int &used, int lane,
                                            uint32_t acc, int row, int rows, int col0, int part, bool aux_here,
                                            const GeluConstants<HOLD> &constants, Release release) {
    const int pieces = pieces_of(p, col0);
    uint32_t r[PIECE];
    unsigned char *box = boxes;
    tmem_ld_32x32b_x16(acc, r);
#pragma unroll 2
    for (int i = 0; i < pieces; ++i)
        finish_piece<F32, BF, ACT>(p, map_out, boxes, box, used, lane, row, rows, col0, part, aux_here, constants, i, pieces,
                                   [&](f32x2 (&v)[PIECE / 2]) {
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < PIECE / 2; ++c)
                v[c] = gemm8::pack2(__uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1]));
            if (i + 1 < pieces) tmem_ld_32x32b_x16(acc + (i + 1) * PIECE, r);
            else release();  // all of the sums have been read: the next tile but one may have them
        });
}

// BF: bf16 operands, else f16.  F32: f32 results, else the operands' type; ACT is
// the activation, or any of them (f32 results are rarely activations).  Each has a
// kernel of its own: one that branched to them had no registers left for any.
template <bool BF, bool F32, int32_t ACT>
__global__ void __launch_bounds__(THREADS, 1)
    pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_aux, const Params p) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    unsigned char *out_stage = smem + STAGES * STAGE;
    uint64_t *full = reinterpret_cast<uint64_t *>(out_stage + OUT_WARPS * BOXES * BOX);
    uint64_t *empty = full + STAGES;
    uint64_t *acc_full = empty + STAGES;   // [2]
    uint64_t *acc_empty = acc_full + 2;    // [2]: of a pair, the first block's
    uint64_t *aux_full = acc_empty + 2;    // [OUT_WARPS]
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(aux_full + OUT_WARPS);
    volatile uint32_t *abort_flag = tmem_slot + 1;
    volatile int32_t *consumed = reinterpret_cast<volatile int32_t *>(tmem_slot + 2);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t tries = *static_cast<volatile uint32_t *>(&g_wait_tries);
    const uint32_t rank = cluster_ctarank();
    const int worker = static_cast<int>(blockIdx.x >> 1), workers = static_cast<int>(gridDim.x >> 1);
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 2 * OUT_WARPS);
        }
        for (int w = 0; w < OUT_WARPS; ++w) mbar_init(&aux_full[w], 1);
        *abort_flag = 0;
        *consumed = 0;
        fence_mbarrier_init();
        prefetch_tensormap(&map_a);
        prefetch_tensormap(&map_b);
        if (p.vec) prefetch_tensormap(&map_out);
        if (p.aux_tma) prefetch_tensormap(&map_aux);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 2 * TN);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int mt = static_cast<int>((p.m + TM - 1) / TM), nt = static_cast<int>((p.n + p.tn - 1) / p.tn);
    const int tiles = uniform(mt * nt * p.parts);
    constexpr bool LONG = adds_chunks(ACT);
    int32_t issued = 0;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FEW_REGS));
        if (warp == 0) {
            // ---------------- TMA producer ----------------
            int stage = 0;
            uint32_t phase = 1;
            bool ok = true;
            for (int L = worker; ok && L < tiles; L += workers) {
                const Tile t = tile_at(p, mt, nt, L);
                const int kbs = uniform(t.kbs);
                const int32_t m0 = uniform(t.m0) + static_cast<int32_t>(rank) * BM;
                const int32_t n0 = uniform(t.n0) + static_cast<int32_t>(rank) * (p.tn / 2);
                int32_t k0 = uniform(t.kb0) * BK;
                for (int i = 0; i < kbs; ++i) {
                    ok = all(wait(&empty[stage], phase, tries, abort_flag, DEVERR_TIMEOUT_PRODUCER));
                    if (!ok) break;
                    unsigned char *st = smem + stage * STAGE;
                    uint64_t *bar = &full[stage];
                    if (elect_one()) {
                        const uint32_t bar0 = mapa_shared(smem_u32(bar), 0);
                        if (rank == 0) mbar_arrive_expect_tx(bar, 2 * BOX_BYTES + p.tn * (BK * 2));
                        if (p.amn) {
                            tma_load_2d_pair(st, &map_a, bar0, m0, k0);
                            tma_load_2d_pair(st + HALF_BOX, &map_a, bar0, m0 + 64, k0);
                        } else {
                            tma_load_2d_pair(st, &map_a, bar0, k0, m0);
                        }
                        if (p.bmn) {
                            tma_load_2d_pair(st + BOX_BYTES, &map_b, bar0, n0, k0);
                            if (p.tn == TN) tma_load_2d_pair(st + BOX_BYTES + HALF_BOX, &map_b, bar0, n0 + 64, k0);
                        } else {
                            tma_load_2d_pair(st + BOX_BYTES, &map_b, bar0, k0, n0);
                        }
                    }
                    ++issued;
                    k0 += BK;
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        } else if (warp == 1 && rank == 0) {
            // ---------------- MMA issuer ----------------
            const uint32_t tb = uniform(static_cast<int>(tmem_base));
            const uint64_t desc_a = operand_desc(p.amn), desc_b = operand_desc(p.bmn);
            const uint32_t step_a = p.amn ? 16 * 128 : 32, step_b = p.bmn ? 16 * 128 : 32;
            int32_t it = 0, use = 0;  // stages, accumulators taken
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true, ready = false;
            // `blocks` stages into the next accumulator
            const auto chunk = [&](int blocks) {
                const int cur = use & 1;
                const uint32_t d = tb + (cur ? static_cast<uint32_t>(TN) : 0u);
                // what it held before has been read
                if (use >= 2) ok = all(wait<true>(&acc_empty[cur], ((use >> 1) - 1) & 1, tries, abort_flag, DEVERR_TIMEOUT_MMA));
                if (!ok) return;
                ++use;
                for (int i = 0; i < blocks; ++i, ++it) {
                    if (!ready) ok = all(wait(&full[stage], phase, tries, abort_flag, DEVERR_TIMEOUT_MMA));
                    if (!ok) return;
                    tc_fence_after();
                    // ask for the next stage now, read the answer after this one's instructions
                    const int next = stage + 1 == STAGES ? 0 : stage + 1;
                    const uint32_t next_phase = next ? phase : phase ^ 1;
                    const bool peek = probe(&full[next], next_phase);
                    const uint32_t a = smem_u32(smem) + stage * STAGE, b = a + BOX_BYTES;
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < BK / 16; ++kk)
                            mma_f16_pair(d, at_address(desc_a, a + kk * step_a), at_address(desc_b, b + kk * step_b), p.idesc,
                                         !(i == 0 && kk == 0));
                        mma_commit_pair(&empty[stage], 0x3);
                        if (i == blocks - 1) mma_commit_pair(&acc_full[cur], 0x3);
                    }
                    __syncwarp();
                    ready = all(peek);
                    stage = next;
                    phase = next_phase;
                }
            };
            for (int L = worker; ok && L < tiles; L += workers) {
                const int kbs = p.parts > 1 ? uniform(tile_at(p, mt, nt, L).kbs) : p.kblocks;
                if constexpr (LONG) {
                    const int most = uniform(chunks_of<LONG, F32>(kbs).blocks);
                    for (int left = kbs; ok && left > 0; left -= most) chunk(min(left, most));
                } else {
                    chunk(kbs);
                }
            }
            if (lane == 0) *consumed = it;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(FINISH_REGS));
        // ---------------- finish and store ----------------
        const int quad = warp & 3, side = (warp - 4) >> 2, span = p.tn / 4;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        unsigned char *boxes = out_stage + (warp - 4) * (BOXES * BOX);
        uint64_t *aux_bar = &aux_full[warp - 4];
        const bool aux_tma = !F32 && p.aux_tma;
        const GeluConstants<!F32 && ACT == CHELIS_ACT_GELU> constants;
        int32_t use = 0, aux_count = 0, used = 0;  // use: accumulators read
        bool ok = true;
        auto sums_at = [&] { return tmem_base + lanes + (use & 1 ? static_cast<uint32_t>(TN) : 0u) + side * span; };
        auto landed_sums = [&] {
            return all(wait(&acc_full[use & 1], (use >> 1) & 1, tries, abort_flag, DEVERR_TIMEOUT_EPILOGUE));
        };
        auto release = [&] {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_relaxed(mapa_shared(smem_u32(&acc_empty[use & 1]), 0));
        };
        // taken on an abort too: the copies land before the block leaves
        auto aux_landed = [&] {
            if (ok) ok = all(wait(aux_bar, (aux_count - 1) & 1, tries, abort_flag, DEVERR_TIMEOUT_EPILOGUE));
            else landed(aux_bar, (aux_count - 1) & 1, tries);
        };
        for (int L = worker; ok && L < tiles; L += workers, ++use) {
            const Tile t = tile_at(p, mt, nt, L);
            const int row0 = t.m0 + static_cast<int>(rank) * BM + quad * 32, col0 = t.n0 + side * span;
            const bool live = row0 < p.m && col0 < p.n;  // else nothing to read or store
            const int rows = min(static_cast<int>(p.m) - row0, 32);
            if (aux_tma && live) {
                if (lane == 0) {
                    wait_reads_all();  // the last tile's have left
                    const int count = span > 32 && p.n - col0 > 32 ? 2 : 1;
                    mbar_arrive_expect_tx(aux_bar, count * BOX);
                    for (int n = 0; n < count; ++n)
                        tma_load_3d(boxes + n * BOX, &map_aux, aux_bar, col0 + n * 32, row0, 0);
                }
                __syncwarp();
                ++aux_count;
            }
            if constexpr (LONG) {
                const int chunks = chunks_of<LONG, F32>(t.kbs).count;
                if (chunks > 1) {
                    f32x2 sum[MOST_PIECES][PIECE / 2] = {};
                    const int pieces = pieces_of(p, col0);
                    for (int c = 0; c < chunks; ++c) {
                        if (c) ++use;
                        ok = landed_sums();
                        if (!ok) break;
                        tc_fence_after();
                        if (live) add_chunk(sums_at(), pieces, sum);
                        release();
                    }
                    if (aux_tma && live) aux_landed();
                    if (!ok) break;
                    unsigned char *box = boxes;
                    if (live)
#pragma unroll
                        for (int i = 0; i < MOST_PIECES; ++i)
                            if (i < pieces)
                                finish_piece<F32, BF, ACT>(p, &map_out, boxes, box, used, lane, row0, rows, col0, t.part, aux_tma,
                                                           constants, i, pieces, [&](f32x2 (&v)[PIECE / 2]) {
#pragma unroll
                                    for (int c = 0; c < PIECE / 2; ++c) v[c] = sum[i][c];
                                });
                    continue;
                }
            }
            ok = landed_sums();
            if (aux_tma && live) aux_landed();
            if (!ok) break;
            tc_fence_after();
            if (live)
                finish_tile<F32, BF, ACT>(p, &map_out, boxes, used, lane, sums_at(), row0, rows, col0, t.part, aux_tma, constants,
                                          release);
            else release();
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }

    tc_fence_before();
    __syncthreads();
    // after an abort, copies that were issued but not consumed land first
    if (warp == 0 && lane == 0 && *abort_flag) {
        if (rank == 0) {
            for (int32_t it = *consumed; it < issued; ++it)
                landed(&full[it % STAGES], (it / STAGES) & 1, tries);
        } else if (issued > 0) {
            const uint64_t t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < DRAIN_NS) __nanosleep(1000);
        }
    }
    // neither block leaves while the other may use its memory
    tc_fence_before();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 2 * TN);
    }
}

// ---- parts ----------------------------------------------------------------
// Fewer tiles than half the machine: the contraction is cut into parts, each
// with an f32 result, which join_kernel adds up in order and finishes.  It also
// finishes a product with no contraction (no parts).
template <int N>
__global__ void __launch_bounds__(256)
    join_kernel(const float *__restrict__ parts, int32_t count, int64_t m, int64_t n, const Finish f) {
    const int64_t matrix = m * n, step = static_cast<int64_t>(gridDim.x) * 256 * N;
    for (int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * N; i < matrix; i += step) {
        float sum[N] = {};
#pragma unroll 4
        for (int s = 0; s < count; ++s) {
            if constexpr (N == 4) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(parts + s * matrix + i));
                sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w;
            } else {
                sum[0] += __ldg(parts + s * matrix + i);
            }
        }
        const int64_t row = i / n, col = i - row * n;
#pragma unroll
        for (int c = 0; c < N; ++c) finish_one(f, sum[c], row, col + c, n);
    }
}

// ---- unaligned operands ---------------------------------------------------
// [rows][cols] to rows of ld = cols rounded up to 8 (TMA's 16 bytes); the last
// columns are never read as the map ends at cols.  Both operands' copies in one
// launch.
struct Repack {
    const uint16_t *src;
    uint16_t *dst;      // NULL: none
    int64_t rows, cols, ld;
};
__global__ void __launch_bounds__(256)
    repack_kernel(const Repack a, const Repack b) {
    const int64_t first = a.dst ? a.rows * (a.ld / 8) : 0, all = first + (b.dst ? b.rows * (b.ld / 8) : 0);
    for (int64_t j = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; j < all; j += static_cast<int64_t>(gridDim.x) * 256) {
        const Repack &p = j < first ? a : b;
        const int64_t i = j < first ? j : j - first, groups = p.ld / 8, row = i / groups, c = (i - row * groups) * 8;
        const uint16_t *s = p.src + row * p.cols + c;
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t lo = c + 2 * k < p.cols ? __ldg(s + 2 * k) : 0, hi = c + 2 * k + 1 < p.cols ? __ldg(s + 2 * k + 1) : 0;
            w[k] = lo | hi << 16;
        }
        *reinterpret_cast<uint4 *>(p.dst + row * p.ld + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// ---- few rows -------------------------------------------------------------
// A token or a handful, as in serving: the product reads the weights once and
// does little with them, so memory and latency bound it, not the tensor core.
// The weights go from global memory into registers, 16 bytes a lane, and warp
// MMAs (m16n8k16: 16 of the weights' n, 8 tokens) take them there.
//
// The eight warps of a block share a strip of n and split its contraction; a
// cluster of blocks splits it further where there are few strips.  Their sums
// are added up in order, through the cluster's shared memory.
//   K-major weights (few_kernel<.., false>): a strip is 16 of n.  In a step of 32
// of k, lane (g, t) = (lane / 4, lane % 4) takes k = 8 t .. 8 t + 7 of weight rows
// g and g + 8 and of token g: the MMA wants other k in a lane, but the same ones
// of both operands, and a sum does not mind their order.
//   MN-major weights: a strip is 64 of n.  In a step of 16 of k, lane (g, t) takes
// n = 8 g .. 8 g + 7 of rows k = 4 t .. 4 t + 3; pairs of k are put together from
// two rows (PRMT), and MMA j of four has n = 8 g + 2 j and 8 g + 2 j + 1.
constexpr int FEW_WARPS = 8;

// Whether few_kernel takes a product: up to 16 rows it reads the weights once, and
// does so faster than the pairs fill their tiles, of which rows are mostly missing;
// more rows read them again, which pays while that costs less than the pairs' set-up.
// us in a graph, pairs and few: 8 rows 1024 x 1024 10.6, 4.8, of [n][k] 10.5, 3.6;
// 4096 x 4096 20.5, 12.0; 16 rows 16384 x 4096 30.8, 32.7; 32 rows 4096 x 1024 11.4,
// 10.1, 4096 x 4096 19.8, 19.4, 16384 x 1024 14.9, 21.9; 64 rows 1024 x 1024 10.6, 7.8,
// 4096 x 1024 11.5, 11.7.
bool few_rows(int64_t m, int64_t n, int64_t k) {
    const int64_t passes = (m + 15) / 16;
    return passes == 1 || (passes <= 4 && n <= (int64_t{1} << 23) / passes / k);
}

__device__ __forceinline__ uint4 load8(const uint16_t *p, int64_t left, bool vec) {
    if (left <= 0) return make_uint4(0, 0, 0, 0);
    if (vec) return __ldg(reinterpret_cast<const uint4 *>(p));
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t lo = 2 * j < left ? __ldg(p + 2 * j) : 0, hi = 2 * j + 1 < left ? __ldg(p + 2 * j + 1) : 0;
        w[j] = lo | hi << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint2 load4(const uint16_t *p, int64_t left, bool vec) {
    if (left <= 0) return make_uint2(0, 0);
    if (vec) return __ldg(reinterpret_cast<const uint2 *>(p));
    uint32_t w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t lo = 2 * j < left ? __ldg(p + 2 * j) : 0, hi = 2 * j + 1 < left ? __ldg(p + 2 * j + 1) : 0;
        w[j] = lo | hi << 16;
    }
    return make_uint2(w[0], w[1]);
}

// TG: groups of 8 tokens.  blockIdx.x: (strip, block of the cluster), blockIdx.y:
// groups of 8 * TG tokens.
template <bool BF16, bool BMN, int TG, bool VEC>
__global__ void __launch_bounds__(32 * FEW_WARPS)
    few_kernel(int64_t m, int64_t n, int64_t k, const uint16_t *__restrict__ a, const uint16_t *__restrict__ b,
               int32_t split, const Finish f) {
    constexpr int STRIP = BMN ? 64 : 16, TOKENS = 8 * TG, MMAS = BMN ? 4 : 1;
    constexpr int STEP = BMN ? 16 : 32, DEEP = BMN ? (TG > 2 ? 2 : 4) : (TG > 2 ? 2 : 4);
    __shared__ float red[FEW_WARPS][STRIP * TOKENS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t strip = blockIdx.x / split;
    const int rank = static_cast<int>(blockIdx.x % split);
    const int64_t n0 = strip * STRIP, m0 = static_cast<int64_t>(blockIdx.y) * TOKENS;
    float acc[MMAS][TG][4] = {};
    const int64_t steps = (k + STEP - 1) / STEP;
    const int64_t stride = static_cast<int64_t>(split) * FEW_WARPS;
    const uint16_t *at[TG];
    bool has[TG];
#pragma unroll
    for (int u = 0; u < TG; ++u) {
        has[u] = m0 + u * 8 + g < m;
        at[u] = a + (has[u] ? (m0 + u * 8 + g) * k : 0);
    }
    for (int64_t s0 = rank * FEW_WARPS + warp; s0 < steps; s0 += stride * DEEP) {
        if constexpr (!BMN) {
            uint4 w0[DEEP], w1[DEEP], x[DEEP][TG];
            const bool r0 = n0 + g < n, r1 = n0 + g + 8 < n;
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
                const int64_t k0 = (s0 + d * stride) * STEP + 8 * t, left = k - k0;
                w0[d] = load8(b + (n0 + g) * k + k0, r0 ? left : 0, VEC);
                w1[d] = load8(b + (n0 + g + 8) * k + k0, r1 ? left : 0, VEC);
#pragma unroll
                for (int u = 0; u < TG; ++u) x[d][u] = load8(at[u] + k0, has[u] ? left : 0, VEC);
            }
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
                const uint32_t lo[4] = {w0[d].x, w1[d].x, w0[d].y, w1[d].y}, hi[4] = {w0[d].z, w1[d].z, w0[d].w, w1[d].w};
#pragma unroll
                for (int u = 0; u < TG; ++u) {
                    g16::mma_16816<BF16>(acc[0][u], lo, x[d][u].x, x[d][u].y);
                    g16::mma_16816<BF16>(acc[0][u], hi, x[d][u].z, x[d][u].w);
                }
            }
        } else {
            uint4 w[DEEP][4];
            uint2 x[DEEP][TG];
            const int64_t col = n0 + 8 * g;
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
                const int64_t k0 = (s0 + d * stride) * STEP + 4 * t;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[d][i] = load8(b + (k0 + i) * n + col, k0 + i < k ? n - col : 0, VEC);
#pragma unroll
                for (int u = 0; u < TG; ++u) x[d][u] = load4(at[u] + k0, has[u] ? k - k0 : 0, VEC);
            }
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    auto word = [&](int i) { return j == 0 ? w[d][i].x : j == 1 ? w[d][i].y : j == 2 ? w[d][i].z : w[d][i].w; };
                    const uint32_t q[4] = {__byte_perm(word(0), word(1), 0x5410), __byte_perm(word(0), word(1), 0x7632),
                                           __byte_perm(word(2), word(3), 0x5410), __byte_perm(word(2), word(3), 0x7632)};
#pragma unroll
                    for (int u = 0; u < TG; ++u) g16::mma_16816<BF16>(acc[j][u], q, x[d][u].x, x[d][u].y);
                }
            }
        }
    }
    // [token][n] of this warp
#pragma unroll
    for (int j = 0; j < MMAS; ++j)
#pragma unroll
        for (int u = 0; u < TG; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int token = u * 8 + 2 * t + (i & 1);
                const int col = BMN ? 8 * g + 2 * j + (i >> 1) : g + 8 * (i >> 1);
                red[warp][token * STRIP + col] = acc[j][u][i];
            }
    __syncthreads();
    if (split == 1) {
        for (int e = threadIdx.x; e < STRIP * TOKENS; e += 32 * FEW_WARPS) {
            float z = 0.0f;
#pragma unroll
            for (int w = 0; w < FEW_WARPS; ++w) z += red[w][e];
            const int64_t row = m0 + e / STRIP, col = n0 + e % STRIP;
            if (row < m && col < n) finish_one(f, z, row, col, n);
        }
        return;
    }
    // the block's sums to its first warp's place, then each block adds up a share
    // of the strip over the cluster
    for (int e = threadIdx.x; e < STRIP * TOKENS; e += 32 * FEW_WARPS) {
        float z = 0.0f;
#pragma unroll
        for (int w = 0; w < FEW_WARPS; ++w) z += red[w][e];
        red[0][e] = z;
    }
    cluster_sync_all();
    const uint32_t base = smem_u32(&red[0][0]);
    for (int e = rank * 32 * FEW_WARPS + threadIdx.x; e < STRIP * TOKENS; e += split * 32 * FEW_WARPS) {
        float z = 0.0f;
        for (int c = 0; c < split; ++c) {
            float v;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(base + e * 4, c)) : "memory");
            z += v;
        }
        const int64_t row = m0 + e / STRIP, col = n0 + e % STRIP;
        if (row < m && col < n) finish_one(f, z, row, col, n);
    }
    cluster_sync_all();  // no block leaves while another reads its sums
}

// ---- activation's gradient, column sums -----------------------------------
// dz may be dy: plain loads of it, each before its own store.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    act_bwd_kernel(const T *dy, const T *__restrict__ z, int64_t count, int32_t act, T *dz) {
    using P = experts::Pack<T, VEC>;
    const int64_t step = static_cast<int64_t>(gridDim.x) * 256 * P::N;
    for (int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * P::N; i < count; i += step) {
        const P x = experts::load_pack<T, VEC>(z + i);
        P g, o;
        if constexpr (VEC) *reinterpret_cast<uint4 *>(&g) = *reinterpret_cast<const uint4 *>(dy + i);
        else g.v[0] = dy[i];
#pragma unroll
        for (int c = 0; c < P::N; ++c)
            o.v[c] = experts::from_f32<T>(slope_times(experts::to_f32(g.v[c]), experts::to_f32(x.v[c]), act));
        experts::store_pack<T, VEC>(dz + i, o);
    }
}

// Column sums of [rows][cols], f32: a block has 32 lanes of packs side by side
// and 8 warps of rows; blocks along y take equal shares of the rows, whose sums
// a second launch adds up in order.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    column_sums_kernel(const T *__restrict__ x, int64_t rows, int64_t cols, float *__restrict__ out) {
    using P = experts::Pack<T, VEC>;
    __shared__ float part[8][32 * P::N];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t col = (static_cast<int64_t>(blockIdx.x) * 32 + lane) * P::N;
    const int64_t per = (rows + gridDim.y - 1) / gridDim.y;
    const int64_t first = blockIdx.y * per, last = first + per < rows ? first + per : rows;
    float sum[P::N] = {};
    if (col < cols) {
#pragma unroll 4
        for (int64_t r = first + warp; r < last; r += 8) {
            const P v = experts::load_pack<T, VEC>(x + r * cols + col);
#pragma unroll
            for (int c = 0; c < P::N; ++c) sum[c] += experts::to_f32(v.v[c]);
        }
    }
#pragma unroll
    for (int c = 0; c < P::N; ++c) part[warp][lane * P::N + c] = sum[c];
    __syncthreads();
    for (int e = threadIdx.x; e < 32 * P::N; e += 256) {
        const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 * P::N + e;
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) s += part[w][e];
        if (c < cols) out[blockIdx.y * cols + c] = s;
    }
}

// The shares' sums in order: 32 columns a block, 32 threads of each.
__global__ void __launch_bounds__(1024)
    fold_columns_kernel(const float *__restrict__ parts, int count, int64_t cols, float *__restrict__ out) {
    __shared__ float part[32][32];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float s = 0.0f;
    if (col < cols)
#pragma unroll 8
        for (int i = slice; i < count; i += 32) s += __ldg(parts + i * cols + col);
    part[slice][lane] = s;
    __syncthreads();
    if (slice == 0 && col < cols) {
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += part[i][lane];
        out[col] = s;
    }
}

// ---- host side ------------------------------------------------------------
int64_t round8(int64_t v) { return (v + 7) / 8 * 8; }

// [rows][ld] -> boxes of 64 (contiguous axis) x `high` rows; what lies past cols
// or rows reads as zero.
int make_map(CUtensorMap *map, const void *base, int64_t cols, int64_t ld, int64_t rows, int high, bool bf) {
    tf32x3::EncodeTiledFn fn = tf32x3::encode_fn();
    if (!fn) return set_error(CHELIS_CUDA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
    cuuint32_t box[2] = {64, static_cast<cuuint32_t>(high)};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                    const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return set_error(CHELIS_CUDA_ERR_CUDA, "cuTensorMapEncodeTiled(16-bit) failed (%d)", (int)r);
    return CHELIS_CUDA_OK;
}

// An operand as TMA can read it: itself, or a copy whose rows start on 16 bytes.
Repack repack_of(const void *src, int64_t rows, int64_t cols) {
    Repack r{static_cast<const uint16_t *>(src), nullptr, rows, cols, cols};
    if (cols % 8 != 0 || !experts::aligned16(src)) r.ld = round8(cols);
    return r;
}
bool needs_copy(const Repack &r) { return r.ld != r.cols || !experts::aligned16(r.src); }

int join(const float *parts, int32_t count, int64_t m, int64_t n, const Finish &f, cudaStream_t s) {
    if (n % 4 == 0)
        join_kernel<4><<<blocks8::grid_for((m * n / 4 + 255) / 256, 8), 256, 0, s>>>(parts, count, m, n, f);
    else
        join_kernel<1><<<blocks8::grid_for((m * n + 255) / 256, 8), 256, 0, s>>>(parts, count, m, n, f);
    g_launches++;
    return check_cuda(cudaGetLastError(), "linear16::join_kernel");
}

template <bool BF>
auto kernel_for(const Finish &f) {
    if (f.dtype == CHELIS_DTYPE_F32)
        return f.act == CHELIS_ACT_NONE ? pair_kernel<BF, true, CHELIS_ACT_NONE> : pair_kernel<BF, true, ANY_ACT>;
    switch (f.act) {
        case CHELIS_ACT_RELU: return pair_kernel<BF, false, CHELIS_ACT_RELU>;
        case CHELIS_ACT_GELU: return pair_kernel<BF, false, CHELIS_ACT_GELU>;
        case CHELIS_ACT_SILU: return pair_kernel<BF, false, CHELIS_ACT_SILU>;
        default: return pair_kernel<BF, false, CHELIS_ACT_NONE>;
    }
}
int launch_pairs(bool bf, const CUtensorMap &ma, const CUtensorMap &mb, Params p, cudaStream_t s) {
    CUtensorMap mo{}, mx{};
    const uintptr_t lie = reinterpret_cast<uintptr_t>(p.f.out) | reinterpret_cast<uintptr_t>(p.f.pre) |
                          static_cast<uintptr_t>(p.n * experts::width(p.f.dtype));
    p.vec = lie % 32 == 0 ? 2 : lie % 16 == 0 ? 1 : 0;
    if (!experts::aligned16(p.f.aux)) p.vec = 0;
    p.aux_tma = p.vec && p.f.aux && p.f.dtype != CHELIS_DTYPE_F32;
    if (p.vec) CHELIS_TRY(scaled8::make_out_map(&mo, p.f.out, p.f.dtype, p.n, p.m, p.parts));
    if (p.aux_tma) CHELIS_TRY(scaled8::make_out_map(&mx, const_cast<void *>(p.f.aux), p.f.dtype, p.n, p.m, 1));
    auto kernel = bf ? kernel_for<true>(p.f) : kernel_for<false>(p.f);
    CHELIS_TRY(check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES),
                          "cudaFuncSetAttribute"));
    const int64_t tiles = ((p.m + TM - 1) / TM) * ((p.n + p.tn - 1) / p.tn) * p.parts, workers = sm_count() / 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * (tiles < workers ? tiles : workers)));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM_BYTES;
    cfg.stream = s;
    cudaLaunchAttribute attr[1]{};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CHELIS_TRY(check_cuda(cudaLaunchKernelEx(&cfg, kernel, ma, mb, mo, mx, p), "linear16::pair_kernel"));
    g_launches++;
    return CHELIS_CUDA_OK;
}

int run_pairs(bool bf, bool amn, bool bmn, int64_t m, int64_t n, int64_t k, const void *a, const void *b, const Finish &f) {
    cudaStream_t s = current_stream();
    Params p{};
    p.m = m;
    p.n = n;
    p.kblocks = static_cast<int32_t>((k + BK - 1) / BK);
    p.f = f;
    p.amn = amn;
    p.bmn = bmn;
    // tiles of 256 x 128 where those of 256 x 256 leave half the machine idle
    const int64_t mt = (m + TM - 1) / TM;
    p.tn = 2 * mt * ((n + TN - 1) / TN) <= sm_count() / 2 ? TN / 2 : TN;
    p.idesc = (1u << 4) | (bf ? (1u << 7) | (1u << 10) : 0u) | (amn ? 1u << 15 : 0u) | (bmn ? 1u << 16 : 0u) |
              (static_cast<uint32_t>(p.tn >> 3) << 17) | (static_cast<uint32_t>(TM >> 4) << 24);
    const int64_t tiles = mt * ((n + p.tn - 1) / p.tn);
    if (tiles > INT32_MAX / 256)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "matmul16: more than 2^23 tiles of 256 x 256");
    p.parts = gemm8::part_count(tiles, p.kblocks, sm_count() / 2, 4, 16);
    Repack ra = repack_of(a, amn ? k : m, amn ? m : k), rb = repack_of(b, bmn ? k : n, bmn ? n : k);
    void *scratch = nullptr;
    auto body = [&]() -> int {
        // scratch: the operands' copies, the parts' results
        const size_t size_a = needs_copy(ra) ? static_cast<size_t>(ra.rows) * ra.ld * 2 : 0;
        const size_t size_b = needs_copy(rb) ? static_cast<size_t>(rb.rows) * rb.ld * 2 : 0;
        const size_t size_sums = p.parts > 1 ? static_cast<size_t>(p.parts) * m * n * sizeof(float) : 0;
        CHELIS_TRY(scratch_alloc(&scratch, size_a + size_b + size_sums, s));  // the sizes are multiples of 16
        unsigned char *at = static_cast<unsigned char *>(scratch);
        if (size_a) ra.dst = reinterpret_cast<uint16_t *>(at);
        if (size_b) rb.dst = reinterpret_cast<uint16_t *>(at + size_a);
        if (size_a + size_b) {
            repack_kernel<<<blocks8::grid_for(static_cast<int64_t>((size_a + size_b) / 16 + 255) / 256, 16), 256, 0, s>>>(ra, rb);
            g_launches++;
            CHELIS_LAUNCH_CHECK("linear16::repack_kernel");
        }
        const void *pa = ra.dst ? ra.dst : a, *pb = rb.dst ? rb.dst : b;
        CUtensorMap ma, mb;
        CHELIS_TRY(amn ? make_map(&ma, pa, m, ra.ld, k, 64, bf) : make_map(&ma, pa, k, ra.ld, m, 128, bf));
        CHELIS_TRY(bmn ? make_map(&mb, pb, n, rb.ld, k, 64, bf) : make_map(&mb, pb, k, rb.ld, n, p.tn / 2, bf));
        void *sums = at + size_a + size_b;
        if (p.parts > 1) {
            p.f = Finish{};
            p.f.out = sums;
            p.f.dtype = CHELIS_DTYPE_F32;
        }
        CHELIS_TRY(launch_pairs(bf, ma, mb, p, s));
        if (p.parts > 1) CHELIS_TRY(join(static_cast<const float *>(sums), p.parts, m, n, f, s));
        return CHELIS_CUDA_OK;
    };
    const int rc = body();
    scratch_free(scratch, s);
    return rc;
}

template <bool BF16, bool BMN, int TG, bool VEC>
int launch_few(int64_t m, int64_t n, int64_t k, const void *a, const void *b, const Finish &f) {
    constexpr int64_t STRIP = BMN ? 64 : 16, STEP = BMN ? 16 : 32;
    const int64_t strips = (n + STRIP - 1) / STRIP, groups = (m + 8 * TG - 1) / (8 * TG);
    // blocks for every multiprocessor, while each warp has two steps
    int32_t split = 1;
    while (split < 8 && strips * groups * split < sm_count() && (k + STEP - 1) / STEP >= 4 * split * FEW_WARPS) split *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(strips * split), static_cast<unsigned>(groups));
    cfg.blockDim = dim3(32 * FEW_WARPS);
    cfg.stream = current_stream();
    cudaLaunchAttribute attr[1]{};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(split);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
    CHELIS_TRY(check_cuda(cudaLaunchKernelEx(&cfg, few_kernel<BF16, BMN, TG, VEC>, m, n, k,
                                             static_cast<const uint16_t *>(a), static_cast<const uint16_t *>(b), split, f),
                          "linear16::few_kernel"));
    g_launches++;
    return CHELIS_CUDA_OK;
}
template <bool BF16, bool BMN>
int run_few(int64_t m, int64_t n, int64_t k, const void *a, const void *b, const Finish &f) {
    const bool vec = k % 8 == 0 && (!BMN || n % 8 == 0) && experts::aligned16(a) && experts::aligned16(b);
    if (m <= 8) return vec ? launch_few<BF16, BMN, 1, true>(m, n, k, a, b, f) : launch_few<BF16, BMN, 1, false>(m, n, k, a, b, f);
    return vec ? launch_few<BF16, BMN, 2, true>(m, n, k, a, b, f) : launch_few<BF16, BMN, 2, false>(m, n, k, a, b, f);
}

template <typename F>
void by_half(int32_t dtype, bool vec, F f) {
    if (dtype == CHELIS_DTYPE_BF16) vec ? f(__nv_bfloat16{}, std::true_type{}) : f(__nv_bfloat16{}, std::false_type{});
    else vec ? f(__half{}, std::true_type{}) : f(__half{}, std::false_type{});
}

int check_half(const char *op, int32_t dtype) {
    if (dtype != CHELIS_DTYPE_BF16 && dtype != CHELIS_DTYPE_F16)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "%s takes bf16 or f16", op);
    return CHELIS_CUDA_OK;
}
int check_act(const char *op, int32_t act) {
    if (act < CHELIS_ACT_NONE || act > CHELIS_ACT_SILU)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "%s: unknown activation %d", op, act);
    return CHELIS_CUDA_OK;
}

}  // namespace linear16
}  // namespace chelis

using namespace chelis;

extern "C" int chelis_cuda_matmul16(int32_t dtype, int trans_a, int trans_b, int64_t m, int64_t n, int64_t k,
                                    const void *a, const void *b, const void *bias, int32_t bias_dtype,
                                    int32_t activation, const void *residual, const void *through, void *pre,
                                    int32_t out_dtype, void *out) {
    CHELIS_TRY(linear16::check_half("matmul16", dtype));
    CHELIS_TRY(linear16::check_act("matmul16", activation));
    if (out_dtype != CHELIS_DTYPE_F32 && out_dtype != dtype)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "matmul16 gives f32 or its operands' type");
    if (bias && bias_dtype != CHELIS_DTYPE_F32 && bias_dtype != dtype)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "matmul16: bias is f32 or of the operands' type");
    if (m < 0 || n < 0 || k < 0) return set_error(CHELIS_CUDA_ERR_DOMAIN, "matmul16: extents >= 0");
    if (m > INT32_MAX - 512 || n > INT32_MAX - 512 || k > INT32_MAX - 512)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "matmul16: an extent above 2^31");
    if (through && (bias || residual || pre))
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "matmul16: through goes with no bias, residual or pre");
    if (m == 0 || n == 0) return CHELIS_CUDA_OK;
    if (!out || (k > 0 && (!a || !b))) return set_error(CHELIS_CUDA_ERR_DOMAIN, "matmul16: null operand");
    linear16::Finish f{};
    f.bias = bias;
    f.bias_dtype = bias_dtype;
    f.bias_vec = bias && experts::aligned16(bias);
    f.out = out;
    f.pre = pre;
    f.dtype = out_dtype;
    f.act = activation;
    f.aux = residual ? residual : through;
    f.aux_kind = residual ? linear16::AUX_RESIDUAL : through ? linear16::AUX_THROUGH : linear16::AUX_NONE;
    if (k == 0) return linear16::join(nullptr, 0, m, n, f, current_stream());
    const bool bf = dtype == CHELIS_DTYPE_BF16;
    if (!trans_a && linear16::few_rows(m, n, k)) {
        if (trans_b) return bf ? linear16::run_few<true, false>(m, n, k, a, b, f) : linear16::run_few<false, false>(m, n, k, a, b, f);
        return bf ? linear16::run_few<true, true>(m, n, k, a, b, f) : linear16::run_few<false, true>(m, n, k, a, b, f);
    }
    return linear16::run_pairs(bf, trans_a != 0, trans_b == 0, m, n, k, a, b, f);
}

extern "C" int chelis_cuda_activation16_bwd(int32_t dtype, int32_t activation, const void *dy, const void *pre,
                                            int64_t count, void *dz) {
    CHELIS_TRY(linear16::check_half("activation16_bwd", dtype));
    CHELIS_TRY(linear16::check_act("activation16_bwd", activation));
    if (count < 0) return set_error(CHELIS_CUDA_ERR_DOMAIN, "activation16_bwd: extents >= 0");
    if (count == 0) return CHELIS_CUDA_OK;
    if (!dy || !pre || !dz) return set_error(CHELIS_CUDA_ERR_DOMAIN, "activation16_bwd: null operand");
    const bool vec = count % 8 == 0 && experts::aligned16(dy) && experts::aligned16(pre) && experts::aligned16(dz);
    linear16::by_half(dtype, vec, [&](auto t, auto v) {
        using T = decltype(t);
        constexpr bool VEC = decltype(v)::value;
        linear16::act_bwd_kernel<T, VEC><<<blocks8::grid_for((count / (VEC ? 8 : 1) + 255) / 256, 8), 256, 0, current_stream()>>>(
            static_cast<const T *>(dy), static_cast<const T *>(pre), count, activation, static_cast<T *>(dz));
    });
    g_launches++;
    CHELIS_LAUNCH_CHECK("linear16::act_bwd_kernel");
    return CHELIS_CUDA_OK;
}

extern "C" int chelis_cuda_column_sums16(int32_t dtype, const void *x, int64_t rows, int64_t cols, float *out) {
    CHELIS_TRY(linear16::check_half("column_sums16", dtype));
    if (rows < 0 || cols < 0) return set_error(CHELIS_CUDA_ERR_DOMAIN, "column_sums16: extents >= 0");
    if (cols == 0) return CHELIS_CUDA_OK;
    if (!out || (rows > 0 && !x)) return set_error(CHELIS_CUDA_ERR_DOMAIN, "column_sums16: null operand");
    cudaStream_t s = current_stream();
    if (rows == 0) return check_cuda(cudaMemsetAsync(out, 0, static_cast<size_t>(cols) * 4, s), "memset");
    const bool vec = cols % 8 == 0 && experts::aligned16(x);
    const int64_t wide = (cols / (vec ? 8 : 1) + 31) / 32;
    if (wide > INT32_MAX) return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "column_sums16: an extent above 2^31");
    // shares of the rows: eight blocks a multiprocessor, 32 rows at least, and one
    // where going through all of them takes no longer than a second launch
    int64_t shares = static_cast<int64_t>(sm_count()) * 8 / wide;
    if (shares > (rows + 31) / 32) shares = (rows + 31) / 32;
    if (shares < 1 || rows <= 256) shares = 1;
    void *parts = nullptr;
    if (shares > 1) CHELIS_TRY(scratch_alloc(&parts, static_cast<size_t>(shares) * cols * 4, s));
    float *first = shares > 1 ? static_cast<float *>(parts) : out;
    linear16::by_half(dtype, vec, [&](auto t, auto v) {
        using T = decltype(t);
        constexpr bool VEC = decltype(v)::value;
        linear16::column_sums_kernel<T, VEC><<<dim3(static_cast<unsigned>(wide), static_cast<unsigned>(shares)), 256, 0, s>>>(
            static_cast<const T *>(x), rows, cols, first);
    });
    g_launches++;
    int rc = check_cuda(cudaGetLastError(), "linear16::column_sums_kernel");
    if (rc == CHELIS_CUDA_OK && shares > 1) {
        linear16::fold_columns_kernel<<<static_cast<unsigned>((cols + 31) / 32), 1024, 0, s>>>(
            first, static_cast<int>(shares), cols, out);
        g_launches++;
        rc = check_cuda(cudaGetLastError(), "linear16::fold_columns_kernel");
    }
    scratch_free(parts, s);
    return rc;
}
