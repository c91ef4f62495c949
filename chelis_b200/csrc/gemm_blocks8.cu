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
// This file has what the three product kernels share, and the one that takes
// any f32 scales: gemm8_kernel, one thread block for a 128 x 256 tile of the
// result at a time, 384 threads:
//   warp 0      TMA producer
//   warp 1      TMEM allocator + tcgen05.mma kind::f8f6f4 issuer
//   warp 2      the blocks' scales into a ring of their own (cp.async)
//   warp 3      looks at them: not admitted or far from 1?
//   warps 4-11  fold: a block's sum in tensor memory times its scales into
//               f32 registers, then the store
// The scales differ from block to block, so the tensor core sums one block
// of 128 (four MMAs of K = 32) from a fresh start, alternating between two
// 256-column accumulators, and the fold adds it in IEEE f32 while the next
// block runs.  The round trip between the two, about twice a block's 512
// clocks of MMAs, is what bounds it; gemm_scaled8.cu has none.
// Scales that are powers of two come here too where the product is too small
// for that kernel's second launch (see gemm_scaled8.cu's one_by_one).  Without
// any_scales another scale is made NaN and reported.  The fold multiplies the
// two scales, or one of them and the sum, first; where a block has one so far
// from 1 that this may leave f32 although the result does not, it takes them by
// halves of their exponents.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>

#include "common.cuh"

namespace chelis {

extern std::atomic<uint64_t> g_launches;

namespace gemm8 {

constexpr int BM = 128, BN = 256, BK = 128;  // one scale block of K = 128 bytes = one swizzle row
constexpr int BOX_BYTES = 128 * BK;          // 128 rows or columns of one block
constexpr int STAGES = 4, STAGE_BYTES = 3 * BOX_BYTES;
constexpr int RING_BYTES = STAGES * STAGE_BYTES;
constexpr int SCALE_SLOTS = 8;
constexpr int SLOT_FLOATS = BM + BN;  // row scales, then column scales (or one for each 128 columns)
constexpr int FOLD_WARPS = 8;
constexpr int THREADS = 128 + 32 * FOLD_WARPS;
// Registers: a launch of 384 threads at 168 gives the first warpgroup's share
// to the fold (128 x 40 + 256 x 232 = 384 x 168), which keeps 128 sums and
// two 16-column loads of tensor memory in flight.  With 56 and 224 the fold
// spilled in its loop (8192 x 4096 x 1024 with any scales 71 us against 60).
constexpr int LAUNCH_REGS = 168, FEW_REGS = 40, FOLD_REGS = 232;
static_assert(128 * FEW_REGS + 32 * FOLD_WARPS * FOLD_REGS <= THREADS * LAUNCH_REGS, "register split");
constexpr uint32_t ACC_COLS = 256, TMEM_COLS = 512;
constexpr int MAX_GROUPS = experts::MAX_EXPERTS;
constexpr int OUT_BOX = 2048;  // 32 rows x 64 bytes of a fold warp on the way out
constexpr int SMEM_BYTES = RING_BYTES + 1024 /*align*/ + 512 /*barriers*/ + SCALE_SLOTS * SLOT_FLOATS * 4 +
                           FOLD_WARPS * OUT_BOX + (MAX_GROUPS + 1) * 4 /*tile starts*/;

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
    int32_t parts;       // of the contraction, each with a result of its own (part_sums)
    int32_t any_scales;  // admit scales that are no powers of two
    uint32_t idesc;
};

// ---- scales ---------------------------------------------------------------
// A normal power of two, what a product takes without any_scales.
__device__ __forceinline__ bool power_of_two(uint32_t bits) {
    return (bits & 0x7fffffu) == 0 && bits - (1u << 23) < (254u << 23);
}
// Magnitude from 2^-60 to 2^60: a block's sum (below 2^39) times two of them
// leaves f32 only where the result does, in any order.  look() gathers scales,
// odd() says whether one of them is further off or not admitted.
constexpr uint32_t NEAR_LOW = 67u << 23, NEAR_SPAN = 120u << 23;
__device__ __forceinline__ void look(float scale, uint32_t *span, uint32_t *bits) {
    const uint32_t b = __float_as_uint(scale);
    *span = max(*span, 2 * b - 2 * NEAR_LOW);  // without the sign
    *bits |= b;
}
__device__ __forceinline__ bool odd(uint32_t span, uint32_t bits, bool any) {
    return span > 2 * NEAR_SPAN || (!any && (bits & 0x807fffffu) != 0);
}
// NaN for a scale that is not admitted.
__device__ __forceinline__ float admitted(float scale, bool any) {
    return any || power_of_two(__float_as_uint(scale)) ? scale : __int_as_float(0x7fc00000);
}
// v s w where a scale is far from 1: each as two factors of half its exponent
// (exact, the first a power of two), multiplied in an order in which nothing
// leaves f32 that is not on its way out: no factor is infinite, and the
// magnitude moves one way once s1 w1 is in.
struct Halves {
    float one, two;
};
__device__ __forceinline__ Halves halves(float scale) {
    const uint32_t h = (__float_as_uint(scale) >> 24 & 0x7fu) + 63u;  // half the exponent, in [2^-64, 2^63]
    return {__uint_as_float(h << 23), scale * __uint_as_float((254u - h) << 23)};
}
__device__ __forceinline__ float scaled(float v, const Halves &s, const Halves &w) {
    return v * (s.one * w.one) * s.two * w.two;
}

__device__ __forceinline__ void mma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 4 bytes from global to shared memory.
__device__ __forceinline__ void cp_async4(float *dst, const float *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// Arrive once this thread's cp.async so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Two f32 at a time: (lo, hi) in one 64-bit register pair.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 unpack2(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
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

// start[g], one warp: the row tiles (or contraction blocks) of HIGH rows before
// group g, held to what ordered offsets give at most (`most`, or the tiles).
template <int HIGH>
__device__ __forceinline__ void group_starts(const Params &p, int64_t rows, int lane, int32_t *start,
                                             int most = -1) {
    if (most < 0) most = static_cast<int>((rows + HIGH - 1) / HIGH) + p.groups;
    int base = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
        int c = 0;
        if (g0 + lane < p.groups) {
            int64_t lo, hi;
            group_span(p, rows, g0 + lane, &lo, &hi);
            c = static_cast<int>((hi - lo + HIGH - 1) / HIGH);
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

// One tile of the result.  Extents are below 2^31 and so are the tiles that
// fit any memory: 32 bits, as the fold has no register to spare.
struct Tile {
    int group;
    int m_tile;         // its row tile, counted over all groups (weight gradient: in its matrix)
    int m0, m_end;      // rows of the result, this tile's first and the group's last + 1
    int n0;
    int kb0, kbs;       // contraction blocks
    int in_group;       // of them before kb0 in the group
    int matrix;         // of the result: a group's (weight gradient), a part's
};

// Blocks of part `part` of a contraction, in whole units of UNIT.
template <int UNIT>
__device__ __forceinline__ void take_part(const Params &p, int part, Tile *t) {
    const int64_t units = (t->kbs + UNIT - 1) / UNIT;
    const int lo = static_cast<int>(units * part / p.parts) * UNIT, hi = static_cast<int>(units * (part + 1) / p.parts) * UNIT;
    t->kbs = min(hi, t->kbs) - lo;
    t->kb0 += lo;
    t->in_group = lo;
}

// Tiles of one group's matrix (mt x nt) in bands of BAND row tiles, column by
// column within a band: the tiles in flight then share a few panels of a and
// b in L2 however tall the matrix is (8192^3 by pairs: bands of 4, 8 and 16
// tiles 390, 372 and 379 us; 32768 x 1024 x 4096 102, 104 and 102, 16384 x 4096 x
// 1024 63, 64 and 63).
constexpr int BAND = 8;
__device__ __forceinline__ void band_order(int in, int mt, int nt, int *m, int *n) {
    const int band = in / (BAND * nt), first = band * BAND;
    const int high = min(mt - first, BAND), r = in - band * (BAND * nt);
    *n = r / high;
    *m = first + (r - *n * high);
}

// `start` is, by group, the prefix of row tiles of TM rows (forward, input
// gradient) or of contraction blocks (weight gradient).
template <bool WG, int TM, int UNIT>
__device__ __forceinline__ Tile tile_at(const Params &p, const int32_t *start, int L) {
    const int nt = static_cast<int>((p.n + BN - 1) / BN);
    Tile t;
    t.in_group = 0;
    int m, n;
    if (WG) {
        const int mt = static_cast<int>((p.rows + TM - 1) / TM);
        t.matrix = L / (mt * nt);
        band_order(L - t.matrix * (mt * nt), mt, nt, &m, &n);
        t.group = p.parts > 1 ? t.matrix / p.parts : t.matrix;
        t.m_tile = m;
        t.m0 = m * TM;
        t.m_end = static_cast<int>(p.rows);
        t.kb0 = start[t.group];
        t.kbs = start[t.group + 1] - t.kb0;
        if (p.parts > 1) take_part<UNIT>(p, t.matrix - t.group * p.parts, &t);
    } else {
        t.matrix = 0;
        if (p.parts > 1) {
            const int tiles = start[p.groups] * nt;
            t.matrix = L / tiles;
            L -= t.matrix * tiles;
        }
        int lo = 0, hi = p.groups;  // the last group whose first tile is at or before L
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start[mid] * nt <= L) lo = mid;
            else hi = mid;
        }
        t.group = lo;
        band_order(L - start[lo] * nt, start[lo + 1] - start[lo], nt, &m, &n);
        int64_t a, b;
        group_span(p, p.rows, lo, &a, &b);
        t.m_tile = start[lo] + m;
        t.m0 = static_cast<int>(a) + m * TM;
        t.m_end = static_cast<int>(b);
        t.kb0 = 0;
        t.kbs = p.kblocks;
        if (p.parts > 1) take_part<UNIT>(p, t.matrix, &t);
    }
    t.n0 = n * BN;
    return t;
}

// 32 bytes at once (a whole sector of a row).
__device__ __forceinline__ void store32(void *p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
                 "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
__device__ __forceinline__ uint32_t round2(float2 v, bool bf) {
    if (bf) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __half2 h = __floats2half2_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// 64 bytes of this lane's row into the warp's 32 x 64 byte box, 16-byte pieces
// in the order of TMA's 64-byte swizzle.
__device__ __forceinline__ void stage_box(unsigned char *box, int lane, const uint32_t (&w)[16]) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
        *reinterpret_cast<uint4 *>(box + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)) =
            make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
}
// Columns N * 64 bytes on of this thread's row, as they are stored.
template <int N>
__device__ __forceinline__ void box_words(const f32x2 (&run)[64], int32_t dtype, uint32_t (&w)[16]) {
    if (N >= 4 || dtype == CHELIS_DTYPE_F32) {  // 16 bits fill four boxes
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const float2 v = unpack2(run[(N * 8 + c) & 63]);
            w[2 * c] = __float_as_uint(v.x);
            w[2 * c + 1] = __float_as_uint(v.y);
        }
    } else {
#pragma unroll
        for (int c = 0; c < 16; ++c) w[c] = round2(unpack2(run[(N * 16 + c) & 63]), dtype == CHELIS_DTYPE_BF16);
    }
}

__device__ __forceinline__ uint32_t load_shared(uint32_t at, uint32_t) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint16_t load_shared(uint32_t at, uint16_t) {
    uint16_t v;
    asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void store_if(bool ok, void *p, uint32_t v) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p st.global.b32 [%0], %1;\n\t}" ::"l"(p), "r"(v),
                 "r"(static_cast<int>(ok))
                 : "memory");
}
__device__ __forceinline__ void store_if(bool ok, void *p, uint16_t v) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p st.global.b16 [%0], %1;\n\t}" ::"l"(p), "h"(v),
                 "r"(static_cast<int>(ok))
                 : "memory");
}
// The rows of a box to global memory from `out`, U at a time: two rows (32-bit
// units) or one (16-bit) by the warp's 32 lanes, sixteen loads before their
// stores.  The loads are asm because the compiler, depending on what else is in
// the file, moved each one under its store's condition, which made the stores
// wait for one load after another (6718 x 2335 x 656 by 26 experts 54 against
// 47 us).
template <typename U>
__device__ __forceinline__ void store_box(const unsigned char *box, int lane, unsigned char *out, int64_t ld, int rows,
                                          int bytes) {
    constexpr int WIDE = 64 / static_cast<int>(sizeof(U)), ROWS = 32 / WIDE, DEEP = 16;
    const int byte = lane % WIDE * static_cast<int>(sizeof(U)), row = lane / WIDE;
    rows = byte < bytes ? rows - row : 0;
    out += row * ld + byte;
    const uint32_t at = smem_u32(box) + row * 64 + (byte & 15), piece = byte >> 4;
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += DEEP * ROWS) {
        U v[DEEP];
#pragma unroll
        for (int i = 0; i < DEEP; ++i) {
            const int r = r0 + i * ROWS;  // its bits 1 and 2 alone turn the pieces round
            v[i] = load_shared(at + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4), U{});
        }
#pragma unroll
        for (int i = 0; i < DEEP; ++i) {
            store_if(r0 + i * ROWS < rows, out, v[i]);
            out += ROWS * ld;
        }
    }
}
template <int N>
__device__ __forceinline__ void store_boxes(const f32x2 (&run)[64], int32_t dtype, unsigned char *box, int lane,
                                            unsigned char *out, int64_t ld, int rows, int bytes) {
    if (N * 64 >= bytes) return;
    uint32_t w[16];
    box_words<N>(run, dtype, w);
    __syncwarp();
    stage_box(box, lane, w);
    __syncwarp();
    if (((reinterpret_cast<uintptr_t>(out) | ld) & 3) == 0)
        store_box<uint32_t>(box, lane, out + N * 64, ld, rows, bytes - N * 64);
    else
        store_box<uint16_t>(box, lane, out + N * 64, ld, rows, bytes - N * 64);
    if constexpr (N < 7) store_boxes<N + 1>(run, dtype, box, lane, out, ld, rows, bytes);
}

// 32 rows x 128 columns of a warp from element `index` on, of which `rows` and
// `left` lie in the result.  Whole columns of rows that start on 32 bytes go
// from each thread's registers, a sector at a time; others through the warp's
// box, so that neighbouring lanes write neighbouring units.  One element at
// a time from the registers touched 32 sectors a store: 8941 x 3329 x 144 by
// 11 experts to f16 334 us, so 46; 20930 x 263 x 135 by 19 115 and 20.  Tiles of
// a few rows lose up to 1.2 us by it, and wide f32 results of few blocks more: the
// weight gradient 2433 x 1747 by 31 experts from 898 rows took 240 us one element
// at a time and takes 252, 1520 x 2529 by 16 from 4838 118 and 121.
__device__ __forceinline__ void store_rows(const Params &p, const f32x2 (&run)[64], unsigned char *box, int lane,
                                           int64_t index, int rows, int64_t left) {
    const int w = p.out_dtype == CHELIS_DTYPE_F32 ? 4 : 2;
    unsigned char *first = static_cast<unsigned char *>(p.out) + index * w;
    if (left < 128 || p.n * w % 32 != 0 || (reinterpret_cast<uintptr_t>(first) & 31) != 0) {
        store_boxes<0>(run, p.out_dtype, box, lane, first, p.n * w, rows, static_cast<int>(left < 128 ? left : 128) * w);
        return;
    }
    if (lane >= rows) return;
    unsigned char *o = first + lane * p.n * w;
    if (p.out_dtype == CHELIS_DTYPE_F32) {
#pragma unroll
        for (int j = 0; j < 64; j += 4) {
            uint32_t v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = unpack2(run[j + i]);
                v[2 * i] = __float_as_uint(f.x);
                v[2 * i + 1] = __float_as_uint(f.y);
            }
            store32(o + 8 * j, v);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 64; j += 8) {
            uint32_t v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = round2(unpack2(run[j + i]), p.out_dtype == CHELIS_DTYPE_BF16);
            store32(o + 4 * j, v);
        }
    }
}

// Arrive on the pair's first block's barrier.  What it orders is the read of
// tensor memory, which the tcgen05 fences around it carry, so it releases
// nothing: a release at cluster scope waits for all of the thread's memory
// traffic (with it the pair kernel took 2700 clocks a block, without it 1300).
__device__ __forceinline__ void arrive_relaxed(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr)
                 : "memory");
}
// A suspended try at cluster scope for the pair's arrivals (relaxed: see
// arrive_relaxed).
__device__ __forceinline__ bool try_wait_relaxed(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(1000u)
        : "memory");
    return ok != 0;
}
// One look at an mbarrier's phase, without suspending.
__device__ __forceinline__ bool probe(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// The bounded wait of common.cuh with the limit held in a register: reading
// it anew costs a trip to L2 at every wait, more than a block's MMAs take.
// False on the limit, or once another role of the block has given up.
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, uint32_t tries,
                                     volatile uint32_t *abort_flag, unsigned int code) {
    for (uint32_t i = 0; i < tries; ++i) {
        if (CLUSTER ? try_wait_relaxed(bar, parity) : mbar_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
    }
    report_device_error(code);
    *abort_flag = 1;
    return false;
}

// One lane of a converged warp.  The producer's and the issuer's loops run in
// the whole warp, with only the instructions themselves under this predicate:
// their descriptors and coordinates then live in uniform registers.  In code
// under `lane == 0` each MMA took about 80 clocks to issue, more than half of
// what it runs.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// The result of a wait as a vote, so that the branch on it is uniform too.
__device__ __forceinline__ bool all(bool ok) { return __all_sync(0xffffffffu, ok); }
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// Rows of the result that no group holds, by all blocks' fold warps.
__device__ __forceinline__ void zero_loose_rows(const Params &p) {
    int64_t a, b, first, last;
    group_span(p, p.rows, 0, &first, &b);
    group_span(p, p.rows, p.groups - 1, &a, &last);
    const int64_t who = static_cast<int64_t>(blockIdx.x) * (FOLD_WARPS * 32) + threadIdx.x - (THREADS - FOLD_WARPS * 32);
    const int64_t step = static_cast<int64_t>(gridDim.x) * (FOLD_WARPS * 32);
    const int64_t loose = (first + p.rows - last) * p.n;
    for (int64_t i = who; i < loose * p.parts; i += step) {
        const int64_t part = p.parts > 1 ? i / loose : 0, j = i - part * loose;
        const int64_t e = part * p.rows * p.n + (j < first * p.n ? j : last * p.n + (j - first * p.n));
        if (p.out_dtype == CHELIS_DTYPE_F32) static_cast<float *>(p.out)[e] = 0.0f;
        else static_cast<uint16_t *>(p.out)[e] = 0;
    }
}
// Copies that were issued but not consumed land before an aborted block leaves.
__device__ __forceinline__ void landed(uint64_t *bar, uint32_t parity, uint32_t tries) {
    for (uint32_t i = 0; i < tries; ++i)
        if (mbar_try_wait(bar, parity)) return;
}

// One block's scales, by one warp, before the fold sees them: true where one is
// far from 1.  Those that are not admitted become NaN and are reported, where
// `rows` and `cols` have them in the result (what lies past its end repeats the
// last).  The usual block takes few instructions, as the fold needs the issue
// slots: the weight gradient of 2048 rows by 8 experts of 1024 x 1024 takes 23.4
// us with this and the fold's branch, 20.9 without.
template <bool WG>
__device__ __forceinline__ bool check_scales(float *slot, int lane, int rows, int cols, bool any) {
    uint32_t span = 0, bits = 0;
    auto look4 = [&](int at) {
        const float4 v = *reinterpret_cast<const float4 *>(slot + at + 4 * lane);
        look(v.x, &span, &bits);
        look(v.y, &span, &bits);
        look(v.z, &span, &bits);
        look(v.w, &span, &bits);
    };
    look4(0);
    if (WG) {
        look4(BM);
        look4(BM + 128);
    } else {
        look(slot[BM + (cols > 128 ? lane & 1 : 0)], &span, &bits);
    }
    if (!__any_sync(0xffffffffu, odd(span, bits, any))) return false;
    if (!any) {
        bool bad = false;
        auto look_again = [&](float *at) {
            if (!power_of_two(__float_as_uint(*at))) {
                bad = true;
                *at = __int_as_float(0x7fc00000);
            }
        };
        for (int i = lane; i < min(rows, BM); i += 32) look_again(slot + i);
        for (int i = lane; i < (WG ? min(cols, BN) : (cols > 128 ? 2 : 1)); i += 32) look_again(slot + BM + i);
        if (bad) report_device_error(DEVERR_SCALE);
    }
    return true;
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
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + RING_BYTES);
    uint64_t *empty = full + STAGES;
    uint64_t *acc_full = empty + STAGES;  // [2]
    uint64_t *acc_empty = acc_full + 2;   // [2]
    uint64_t *scale_full = acc_empty + 2;
    uint64_t *scale_empty = scale_full + SCALE_SLOTS;
    uint64_t *scale_landed = scale_empty + SCALE_SLOTS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(scale_landed + SCALE_SLOTS);
    volatile uint32_t *abort_flag = tmem_slot + 1;
    volatile int32_t *consumed = reinterpret_cast<volatile int32_t *>(tmem_slot + 2);
    uint32_t *far = tmem_slot + 3;  // [SCALE_SLOTS]: a scale of the block is far from 1 or not admitted
    float *scales = reinterpret_cast<float *>(smem + RING_BYTES + 512);
    unsigned char *out_stage = reinterpret_cast<unsigned char *>(scales + SCALE_SLOTS * SLOT_FLOATS);
    int32_t *start = reinterpret_cast<int32_t *>(out_stage + FOLD_WARPS * OUT_BOX);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t tries = *static_cast<volatile uint32_t *>(&g_wait_tries);
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], FOLD_WARPS);
        }
        for (int q = 0; q < SCALE_SLOTS; ++q) {
            mbar_init(&scale_landed[q], 32);
            mbar_init(&scale_full[q], 1);
            mbar_init(&scale_empty[q], FOLD_WARPS);
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
    if (warp == 2) group_starts<WG ? BK : BM>(p, WG ? p.group_rows : p.rows, lane, start, WG ? p.kblocks : -1);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int64_t nt = (p.n + BN - 1) / BN;
    const int tiles = uniform(static_cast<int>(p.parts * (WG ? p.groups * nt * ((p.rows + BM - 1) / BM) : start[p.groups] * nt)));
    const int first = static_cast<int>(blockIdx.x), step = static_cast<int>(gridDim.x);
    int32_t issued = 0;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FEW_REGS));
        if (warp == 0) {
            // ---------------- TMA producer ----------------
            int stage = 0;
            uint32_t phase = 1;
            bool ok = true;
            for (int L = first; ok && L < tiles; L += step) {
                const Tile t = tile_at<WG, BM, 1>(p, start, L);
                const int group = uniform(t.group), kbs = uniform(t.kbs);
                const int32_t m0 = uniform(t.m0), n0 = uniform(t.n0);
                int32_t k0 = uniform(t.kb0) * BK;
                for (int i = 0; i < kbs; ++i, k0 += BK) {
                    ok = all(wait(&empty[stage], phase, tries, abort_flag, DEVERR_TIMEOUT_PRODUCER));
                    if (!ok) break;
                    unsigned char *st = smem + stage * STAGE_BYTES;
                    uint64_t *bar = &full[stage];
                    if (elect_one()) {
                        mbar_arrive_expect_tx(bar, STAGE_BYTES);
                        tma_load_2d(st, &map_a, bar, k0, m0);
#pragma unroll
                        for (int h = 0; h < BN / 128; ++h) {
                            unsigned char *dst = st + (1 + h) * BOX_BYTES;
                            if (WG) tma_load_2d(dst, &map_b, bar, k0, n0 + h * 128);
                            else if (BMN) tma_load_3d(dst, &map_b, bar, n0 + h * 128, k0, group);
                            else tma_load_3d(dst, &map_b, bar, k0, n0 + h * 128, group);
                        }
                    }
                    ++issued;
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        } else if (warp == 1) {
            // ---------------- MMA issuer ----------------
            const uint32_t tb = uniform(static_cast<int>(tmem_base));
            int32_t it = 0;
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int L = first; ok && L < tiles; L += step) {
                const int kbs = WG || p.parts > 1 ? uniform(tile_at<WG, BM, 1>(p, start, L).kbs) : p.kblocks;
                for (int i = 0; i < kbs; ++i, ++it) {
                    const int cur = it & 1;
                    if (it >= 2)
                        ok = all(wait(&acc_empty[cur], ((it >> 1) - 1) & 1, tries, abort_flag, DEVERR_TIMEOUT_MMA));
                    if (ok) ok = all(wait(&full[stage], phase, tries, abort_flag, DEVERR_TIMEOUT_MMA));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t a = smem_u32(smem) + stage * STAGE_BYTES, b = a + BOX_BYTES;
                    const uint32_t d = tb + static_cast<uint32_t>(cur) * ACC_COLS;
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < BK / 32; ++kk)
                            mma_f8(d, sw128_kmajor_desc(a + kk * 32),
                                   BMN ? mnmajor_desc(b + kk * 32 * 128) : sw128_kmajor_desc(b + kk * 32), p.idesc,
                                   kk != 0);
                        mma_commit(&empty[stage]);
                        mma_commit(&acc_full[cur]);
                    }
                    __syncwarp();
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            if (lane == 0) *consumed = it;
        } else if (warp == 2) {
            // ---------------- scales ----------------
            int32_t it = 0;
            bool ok = true;
            for (int L = first; ok && L < tiles; L += step) {
                const Tile t = tile_at<WG, BM, 1>(p, start, L);
                const float *tile_sb = p.sb + t.group * p.sb_group + (t.n0 / 128) * p.sb_n;
                for (int i = 0; i < t.kbs; ++i, ++it) {
                    const int q = it % SCALE_SLOTS;
                    ok = all(wait(&scale_empty[q], ((it / SCALE_SLOTS) & 1) ^ 1, tries, abort_flag,
                                  DEVERR_TIMEOUT_PRODUCER));
                    if (!ok) break;
                    float *slot = scales + q * SLOT_FLOATS;
                    const int64_t kb = t.kb0 + i;
#pragma unroll
                    for (int u = 0; u < BM / 32; ++u) {
                        const int64_t row = t.m0 + u * 32 + lane;
                        cp_async4(slot + u * 32 + lane, p.sa + kb * p.rows + (row < p.rows ? row : p.rows - 1));
                    }
                    if (WG) {
#pragma unroll
                        for (int u = 0; u < BN / 32; ++u) {
                            const int64_t c = t.n0 + u * 32 + lane;
                            cp_async4(slot + BM + u * 32 + lane, p.sb + kb * p.n + (c < p.n ? c : p.n - 1));
                        }
                    } else if (lane < 2 && t.n0 + lane * 128 < p.n) {
                        cp_async4(slot + BM + lane, tile_sb + lane * p.sb_n + kb * p.sb_k);
                    }
                    cp_async_arrive(&scale_landed[q]);
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else {
            // ---------------- check of the scales ----------------
            int32_t it = 0;
            bool ok = true;
            for (int L = first; ok && L < tiles; L += step) {
                const Tile t = tile_at<WG, BM, 1>(p, start, L);
                const int rows = t.m_end - t.m0, cols = static_cast<int>(p.n) - t.n0;
                for (int i = 0; i < t.kbs; ++i, ++it) {
                    const int q = it % SCALE_SLOTS;
                    ok = all(wait(&scale_landed[q], (it / SCALE_SLOTS) & 1, tries, abort_flag, DEVERR_TIMEOUT_PRODUCER));
                    if (!ok) break;
                    const bool distant = check_scales<WG>(scales + q * SLOT_FLOATS, lane, rows, cols, p.any_scales != 0);
                    if (lane == 0) far[q] = distant;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&scale_full[q]);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(FOLD_REGS));
        // ---------------- fold and store ----------------
        const int quad = warp & 3, half = (warp - 4) >> 2;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        int32_t it = 0;
        bool ok = true;
        for (int L = first; ok && L < tiles; L += step) {
            const Tile t = tile_at<WG, BM, 1>(p, start, L);
            const int row0 = t.m0 + quad * 32, col0 = t.n0 + half * 128;
            const bool live = row0 < t.m_end && col0 < p.n;  // else nothing to read or store
            f32x2 run[64];
#pragma unroll
            for (int j = 0; j < 64; ++j) run[j] = 0ull;
            for (int i = 0; i < t.kbs; ++i, ++it) {
                const int b = it & 1, q = it % SCALE_SLOTS;
                const float *slot = scales + q * SLOT_FLOATS;
                ok = wait(&scale_full[q], (it / SCALE_SLOTS) & 1, tries, abort_flag, DEVERR_TIMEOUT_EPILOGUE) &&
                     wait(&acc_full[b], (it >> 1) & 1, tries, abort_flag, DEVERR_TIMEOUT_EPILOGUE);
                ok = all(ok);
                if (!ok) break;
                tc_fence_after();
                auto release = [&] {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&acc_empty[b]);
                };
                if (!live) {
                    release();
                    if (lane == 0) mbar_arrive(&scale_empty[q]);
                    continue;
                }
                float s = slot[quad * 32 + lane];
                const float4 *cs = reinterpret_cast<const float4 *>(slot + BM + half * 128);
                const uint32_t acc = tmem_base + lanes + static_cast<uint32_t>(b) * ACC_COLS + half * 128;
                if (far[q]) {  // unrolled like the usual fold: it must leave the sums in their registers
                    const Halves hs = halves(s), hw = halves(WG ? 1.0f : slot[BM + half]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        uint32_t r[16];
                        tmem_ld_32x32b_x16(acc + j * 16, r);
                        tmem_wait_ld();
#pragma unroll
                        for (int c = 0; c < 16; c += 4) {
                            const float4 w = WG ? cs[j * 4 + c / 4] : float4{};
                            const int o = j * 8 + c / 2;
                            run[o] = add2(run[o], pack2(scaled(__uint_as_float(r[c]), hs, WG ? halves(w.x) : hw),
                                                        scaled(__uint_as_float(r[c + 1]), hs, WG ? halves(w.y) : hw)));
                            run[o + 1] = add2(run[o + 1], pack2(scaled(__uint_as_float(r[c + 2]), hs, WG ? halves(w.z) : hw),
                                                                scaled(__uint_as_float(r[c + 3]), hs, WG ? halves(w.w) : hw)));
                        }
                    }
                    release();
                    if (lane == 0) mbar_arrive(&scale_empty[q]);
                    continue;
                }
                if (!WG) s *= slot[BM + half];
                const f32x2 s2 = pack2(s, s);
                // 16 columns are added while the next 16 load
                uint32_t r[2][16];
                tmem_ld_32x32b_x16(acc, r[0]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    tmem_wait_ld();
                    if (j < 7) tmem_ld_32x32b_x16(acc + (j + 1) * 16, r[(j + 1) & 1]);
                    else release();  // the accumulator has been read: the next block may have it
#pragma unroll
                    for (int c = 0; c < 16; c += 4) {
                        f32x2 v0 = pack2(__uint_as_float(r[j & 1][c]), __uint_as_float(r[j & 1][c + 1]));
                        f32x2 v1 = pack2(__uint_as_float(r[j & 1][c + 2]), __uint_as_float(r[j & 1][c + 3]));
                        if (WG) {
                            const float4 w = cs[j * 4 + c / 4];
                            v0 = mul2(v0, pack2(w.x, w.y));
                            v1 = mul2(v1, pack2(w.z, w.w));
                        }
                        const int o = j * 8 + c / 2;
                        run[o] = fma2(v0, s2, run[o]);
                        run[o + 1] = fma2(v1, s2, run[o + 1]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&scale_empty[q]);
            }
            if (ok && live)
                store_rows(p, run, out_stage + (warp - 4) * OUT_BOX, lane,
                           (t.matrix * p.rows + row0) * p.n + col0, min(t.m_end - row0, 32), p.n - col0);
        }
        if (!WG && p.offsets) zero_loose_rows(p);
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 0 && lane == 0 && *abort_flag)
        for (int32_t it = *consumed; it < issued; ++it)
            landed(&full[it % STAGES], (it / STAGES) & 1, tries);
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

// Tiles of `high` rows that the groups have at most.
int64_t row_tiles(int64_t rows, int32_t groups, bool offsets, int64_t high) {
    return (rows + high - 1) / high + (offsets ? groups : 0);
}

// ---- parts ----------------------------------------------------------------
// Fewer tiles than half the machine: the contraction is cut into parts, each
// tile of each part its own piece of work with its own f32 result, which
// part_sums_kernel adds up in order (us, whole and in parts): weight gradients
// 256 x 256 from 8192 rows 77 and 17, 1024 x 256 from 131072 rows 339 and 48,
// products 512 x 1024 x 16384 47 and 22, input gradient 16 x 1024 x 4096 30 and
// 11.  Each part costs a result written and read and the join its launch: with
// 6 blocks saved of 12, 1369 x 1013 x 1507 by 4 experts took 21 us and whole 17.
constexpr int PART_BLOCKS = 2;   // that a part has at least (2, 4, 8: 169 x 133 from 3332 rows by 2 22, 27, 45 us)
constexpr int SAVED_BLOCKS = 8;  // one after another, from which the second launch pays

template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    part_sums_kernel(const float *__restrict__ parts, int32_t count, int64_t matrix, int64_t all, T *__restrict__ out) {
    constexpr int N = VEC ? 4 : 1;
    const int64_t step = static_cast<int64_t>(gridDim.x) * 256 * N;
    for (int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * N; i < all; i += step) {
        const int64_t g = i / matrix;
        const float *src = parts + g * count * matrix + (i - g * matrix);
        float sum[N] = {};
#pragma unroll 4
        for (int s = 0; s < count; ++s) {
            if constexpr (VEC) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(src + s * matrix));
                sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w;
            } else {
                sum[0] += __ldg(src + s * matrix);
            }
        }
#pragma unroll
        for (int c = 0; c < N; ++c) out[i + c] = experts::from_f32<T>(sum[c]);
    }
}

int32_t part_count(int64_t tiles, int64_t blocks, int64_t workers, int64_t least, int64_t saved) {
    if (2 * tiles > workers) return 1;
    const int64_t most = workers / tiles, parts = blocks / least < most ? blocks / least : most;
    return parts < 2 || blocks - (blocks + parts - 1) / parts < saved ? 1 : static_cast<int32_t>(parts);
}

// f(p) with p.parts results in scratch and their sums into p.out; f(p) itself
// for one part.
template <typename F>
int in_parts(Params p, int32_t parts, int64_t matrices, F f) {
    p.parts = parts;
    if (parts == 1) return f(p);
    cudaStream_t s = current_stream();
    const int64_t matrix = p.rows * p.n, all = matrices * matrix;
    void *out = p.out, *sums = nullptr;
    const int32_t dtype = p.out_dtype;
    CHELIS_TRY(scratch_alloc(&sums, static_cast<size_t>(parts) * all * sizeof(float), s));
    p.out = sums;
    p.out_dtype = CHELIS_DTYPE_F32;
    int rc = f(p);
    if (rc == CHELIS_CUDA_OK) {
        const bool vec = matrix % 4 == 0;
        experts::by_type(dtype, vec, [&](auto t, auto v) {
            using T = decltype(t);
            constexpr bool VEC = decltype(v)::value;
            part_sums_kernel<T, VEC><<<blocks8::grid_for((all / (VEC ? 4 : 1) + 255) / 256, 8), 256, 0, s>>>(
                static_cast<const float *>(sums), parts, matrix, all, static_cast<T *>(out));
        });
        g_launches++;
        rc = check_cuda(cudaGetLastError(), "gemm8::part_sums_kernel");
    }
    scratch_free(sums, s);
    return rc;
}

// Tiles at most, and the parts that they are cut into.
template <bool WG>
int64_t tiles_of(const Params &p) {
    return (WG ? p.groups * row_tiles(p.rows, 0, false, BM) : row_tiles(p.rows, p.groups, p.offsets != nullptr, BM)) *
           ((p.n + BN - 1) / BN);
}
template <bool WG>
int32_t parts_of(const Params &p) {
    return part_count(tiles_of<WG>(p), WG ? p.kblocks / p.groups : p.kblocks, sm_count(), PART_BLOCKS, SAVED_BLOCKS);
}
// Experts that have rows, about: as many as rows dealt out at random reach.
inline double used_groups(const Params &p) {
    return p.offsets ? -p.groups * std::expm1(-static_cast<double>(p.rows) / p.groups) : 1.0;
}
// The tiles of `high` rows that each of `workers` goes through one after another,
// about: an expert's rows end half a tile early on average, but each has a tile.
template <bool WG>
int64_t rounds(const Params &p, int64_t high, int64_t workers) {
    double tiles = static_cast<double>((p.rows + high - 1) / high);
    if (WG) tiles *= p.groups;
    else if (p.offsets) tiles = std::fmax(static_cast<double>(p.rows) / high + 0.5 * used_groups(p), std::ceil(used_groups(p)));
    return static_cast<int64_t>(std::ceil(tiles * static_cast<double>((p.n + BN - 1) / BN) / workers));
}
// gemm8_kernel's time for a layer product or an input gradient, about (us).
inline double forward_us(const Params &p, int64_t *serial) {
    const int64_t parts = parts_of<false>(p);
    *serial = rounds<false>(p, BM, sm_count()) * ((p.kblocks + parts - 1) / parts);
    return 6.0 + 0.62 * *serial + (parts > 1 ? 3.5 : 0.0);
}

template <bool BMN, bool WG>
int run(const CUtensorMap &ma, const CUtensorMap &mb, Params p, int32_t fa, int32_t fb) {
    p.idesc = (1u << 4) |                                    // f32 sums
              (fa == CHELIS_FORMAT_E5M2 ? 1u << 7 : 0u) |    // 0 e4m3, 1 e5m2
              (fb == CHELIS_FORMAT_E5M2 ? 1u << 10 : 0u) |
              (BMN ? 1u << 16 : 0u) |                        // b MN-major
              (static_cast<uint32_t>(BN >> 3) << 17) | (static_cast<uint32_t>(BM >> 4) << 24);
    const int64_t most = tiles_of<WG>(p);
    auto kernel = gemm8_kernel<BMN, WG>;
    CHELIS_TRY(check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES),
                          "cudaFuncSetAttribute"));
    const int64_t sms = sm_count();
    const int32_t parts = parts_of<WG>(p);
    return in_parts(p, parts, WG ? p.groups : 1, [&](const Params &q) -> int {
        const int64_t grid = parts * most < sms ? parts * most : sms;
        kernel<<<static_cast<unsigned>(grid), THREADS, SMEM_BYTES, current_stream()>>>(ma, mb, q);
        g_launches++;
        CHELIS_LAUNCH_CHECK("gemm8::gemm8_kernel");
        return CHELIS_CUDA_OK;
    });
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
