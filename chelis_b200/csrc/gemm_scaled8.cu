// gemm_scaled8.cu -- the products of gemm_blocks8.cu for scales that are
// powers of two (what quantize8 makes): the tensor core applies them itself
// (tcgen05.mma kind::mxf8f6f4.block_scale), so the sums stay in tensor memory
// over many blocks and nothing but the result is read back.
//
// The hardware's scale is one 8-bit exponent for 32 of K, four of them in a
// 32-bit word of tensor memory of which an MMA names one byte.  A block of 128
// has one exponent, so a word holds those of four blocks (a quad) and a
// block's four MMAs name the same byte.  pack_scales_kernel writes the words
// from the f32 scales in the order in which tcgen05.cp takes them: 512 bytes
// for 128 rows of a quad, row r's word at 16 (r mod 32) + 4 (r / 32).
//
// A pair of thread blocks (cta_group::2) works on a 256 x 256 tile of the
// result, each with its 128 rows of a and half of b's columns in shared memory
// and its 128 rows of the sums in tensor memory: a block of 128 x 256 alone
// loads half as much again (16384 x 4096 x 1024 91 us against 82, 8192^3 485
// against 408).  Warp roles are gemm8_kernel's, but warp 0 loads the packed
// scales with the operands, warp 1 of the first block copies them to tensor
// memory ahead of a quad's MMAs, and the fold runs once in CHUNK blocks.
//
// CHUNK: the accumulator truncates where IEEE rounds, and its error grows with
// the number of MMAs on it, so after 32 blocks (128 MMAs) it is added to f32
// registers.  Tensor memory has 512 columns and the scales need some, so the
// two 256-column accumulators overlap by 32 columns: the fold reads those
// first, and the other accumulator's MMAs start behind them.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "common.cuh"

namespace chelis {

extern std::atomic<uint64_t> g_launches;

namespace scaled8 {

using namespace gemm8;

constexpr uint64_t DRAIN_NS = 200000;     // bounded drain of an aborted pair's second block
constexpr int PAIR_FEW_REGS = 56, PAIR_FOLD_REGS = 224;  // 128 x 56 + 256 x 224 = 384 x 168
static_assert(128 * PAIR_FEW_REGS + 32 * FOLD_WARPS * PAIR_FOLD_REGS <= THREADS * LAUNCH_REGS, "register split");
constexpr int CHUNK = 32;
constexpr int QUAD = 4;                   // blocks of K in one packed scale word
constexpr int SF_BYTES = 512;             // packed scales of 128 rows, four blocks
constexpr int SF_SLOT = 3 * SF_BYTES;     // a's 128 rows, b's 256 columns
constexpr uint32_t ACC1 = 224;            // first column of the second accumulator
constexpr uint32_t SF_COL = 480;          // two slots of 12 columns of scales
constexpr int OUT_BUFS = 1;               // boxes of a warp on the way out
constexpr int OUT_BYTES = FOLD_WARPS * OUT_BUFS * OUT_BOX;

constexpr int TM = 2 * BM;                // rows of a pair's tile
constexpr int PAIR_STAGE = 2 * BOX_BYTES;  // a block's rows of a, its columns of b
constexpr int PAIR_STAGES = 6;
// scales lie beside the stage of their quad's first block
constexpr int PAIR_SMEM = PAIR_STAGES * (PAIR_STAGE + SF_SLOT) + OUT_BYTES + 1024 /*align*/ + 512 /*barriers*/ +
                          2 * (MAX_GROUPS + 1) * 4;

struct Params8 {
    Params p;
    int32_t m_atoms;          // 128-row scale atoms of a in one quad
    int32_t quads;            // of the contraction (weight gradient: of all groups at most)
    int32_t sfb_group;        // rows of the packed scales of b: an expert's, a quad's
    int32_t sfb_k;
    int32_t tma_out;          // the result can be stored by TMA
};

// ---- scales ---------------------------------------------------------------
// The exponent byte of a power of two, NaN (0xff) for anything else.
__device__ __forceinline__ uint32_t exponent_byte(uint32_t bits) { return power_of_two(bits) ? bits >> 23 : 0xffu; }

constexpr int PACK_THREADS = 256;

// start[g]: quads of the groups before g, from their blocks' prefix.
__device__ __forceinline__ void quad_starts(const Params &p, int lane, const int32_t *blocks, int32_t *quads) {
    int base = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
        int sum = g0 + lane < p.groups ? (blocks[g0 + lane + 1] - blocks[g0 + lane] + QUAD - 1) / QUAD : 0;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, sum, off);
            if (lane >= off) sum += o;
        }
        if (g0 + lane < p.groups) quads[g0 + lane + 1] = base + sum;
        base += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) quads[0] = 0;
}
// The last group that starts at or before v.
__device__ __forceinline__ int group_of(const int32_t *start, int groups, int v) {
    int lo = 0, hi = groups;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

// A warp a packed atom (128 rows of a quad): lane l writes the words of rows
// l, l + 32, l + 64, l + 96.  a's atoms first ([quads][m_atoms]), then b's
// ([groups][quads][ceil(n/128)], or [quads][ceil(n/128)] for the weight
// gradient, whose quads are counted through the groups).  Rows that a tile
// does not have, and blocks past the last, get 1.  Latency bounds it (a few
// hundred KB): one atom a warp, its sixteen loads in flight together.
template <bool WG>
__global__ void __launch_bounds__(PACK_THREADS)
    pack_scales_kernel(const Params p, int32_t quads, int32_t m_atoms, uint4 *__restrict__ sfa,
                       uint4 *__restrict__ sfb) {
    __shared__ int32_t start[MAX_GROUPS + 1], quad_start[MAX_GROUPS + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp == 0) {
        group_starts<WG ? BK : TM>(p, WG ? p.group_rows : p.rows, lane, start, WG ? p.kblocks : -1);
        __syncwarp();
        if (WG) quad_starts(p, lane, start, quad_start);
    }
    __syncthreads();
    const int64_t nb = (p.n + 127) / 128;
    const int64_t a_items = static_cast<int64_t>(quads) * m_atoms;
    const int64_t b_items = (WG ? 1 : p.groups) * quads * nb;
    for (int64_t w = static_cast<int64_t>(blockIdx.x) * (PACK_THREADS / 32) + warp; w < a_items + b_items;
         w += static_cast<int64_t>(gridDim.x) * (PACK_THREADS / 32)) {
        const bool is_a = w < a_items;
        const int64_t i = is_a ? w : w - a_items, per = is_a ? m_atoms : nb;
        int64_t quad = i / per;
        const int64_t atom = i - quad * per;
        const float *src;                  // row 0 of the atom, the quad's first block
        int64_t row_step = 1, kb_step;     // between rows and blocks
        int rows = 128;                    // rows that the atom has
        int kb0, kbs;                      // the quad's blocks
        if (WG) {
            if (quad >= quad_start[p.groups]) continue;
            const int g = group_of(quad_start, p.groups, static_cast<int>(quad));
            kb0 = start[g] + static_cast<int>(quad - quad_start[g]) * QUAD;
            kbs = start[g + 1] - kb0;
            const int64_t extent = is_a ? p.rows : p.n;
            src = (is_a ? p.sa : p.sb) + kb0 * extent + atom * 128;
            kb_step = extent;
            if (extent - atom * 128 < 128) rows = static_cast<int>(extent - atom * 128);
        } else {
            int64_t g = 0;
            if (!is_a) {
                g = quad / quads;
                quad -= g * quads;
                if (start[g + 1] == start[g]) continue;  // no rows: nothing reads them
            }
            kb0 = static_cast<int>(quad) * QUAD;
            kbs = p.kblocks - kb0;
            if (is_a) {
                const int tile = static_cast<int>(atom) / (TM / 128);
                if (tile >= start[p.groups]) continue;
                const int group = group_of(start, p.groups, tile);
                int64_t first, end;
                group_span(p, p.rows, group, &first, &end);
                const int64_t row0 =
                    first + static_cast<int64_t>(tile - start[group]) * TM + (atom % (TM / 128)) * 128;
                src = p.sa + kb0 * p.rows + row0;
                kb_step = p.rows;
                rows = static_cast<int>(end - row0 < 128 ? end - row0 : 128);
            } else {
                src = p.sb + g * p.sb_group + atom * p.sb_n + kb0 * p.sb_k;
                row_step = 0;
                kb_step = p.sb_k;
            }
        }
        // all loads first: a report between them would make each wait for the last
        constexpr uint32_t ONE = 127u << 23;
        uint32_t bits[4][QUAD];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < QUAD; ++j) {
                const bool in = j < kbs && (row_step ? u * 32 + lane < rows : u == 0);
                bits[u][j] = in ? __float_as_uint(src[(u * 32 + lane) * row_step + j * kb_step]) : ONE;
            }
        uint32_t r[4];
        bool bad = false;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            r[u] = 0;
#pragma unroll
            for (int j = 0; j < QUAD; ++j) {
                const uint32_t e = exponent_byte(bits[u][j]);
                bad |= e == 0xffu;
                r[u] |= e << (8 * j);
            }
        }
        if (!row_step) r[1] = r[2] = r[3] = r[0];
        if (bad) report_device_error(DEVERR_SCALE);
        (is_a ? sfa : sfb)[i * 32 + lane] = make_uint4(r[0], r[1], r[2], r[3]);
    }
}

// 512 bytes of scales to 4 columns of tensor memory (every lane quadrant).
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t smem) {
    // 32 rows of 16 bytes, 8-row groups 128 bytes apart, no swizzle
    const uint64_t d = static_cast<uint64_t>((smem >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128u >> 4) << 32) |
                       (static_cast<uint64_t>(1u) << 46);
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
}
__device__ __forceinline__ void mma_scaled(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                           uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X "
        "[%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// ---- fold -----------------------------------------------------------------
// This warp's 128 columns 16 at a time, from the FIRST of the eight pieces on,
// the next loading while one is added; `first` runs once two pieces have been
// read, `last` once all.  (32 at a time need 32 registers more and spilled.)
template <int FIRST, typename F, typename G>
__device__ __forceinline__ void fold128(f32x2 (&run)[64], uint32_t acc, F first, G last) {
    uint32_t r[2][16];
    tmem_ld_32x32b_x16(acc + FIRST * 16, r[0]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int piece = (FIRST + j) % 8, next = (FIRST + j + 1) % 8;
        tmem_wait_ld();
        if (j == 1) first();
        if (j == 7) last();
        else tmem_ld_32x32b_x16(acc + next * 16, r[(j + 1) & 1]);
#pragma unroll
        for (int c = 0; c < 8; ++c)
            run[piece * 8 + c] = add2(run[piece * 8 + c], pack2(__uint_as_float(r[j & 1][2 * c]),
                                                                __uint_as_float(r[j & 1][2 * c + 1])));
    }
}

// ---- the way out ----------------------------------------------------------
__device__ __forceinline__ void tma_store_3d(const CUtensorMap *map, uint32_t src, int32_t x, int32_t y,
                                             int32_t z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(src), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void store_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(OUT_BUFS - 1) : "memory");
}

// 32 rows x 128 columns of a warp, 64 bytes of each row at a time through its
// boxes of shared memory: each box is stored by TMA while the next is filled.
__device__ __forceinline__ void store_tma(const Params &p, const CUtensorMap *map, const f32x2 (&run)[64],
                                          unsigned char *stage, int lane, int64_t col0, int64_t row0, int group) {
    const int32_t x = static_cast<int32_t>(col0), y = static_cast<int32_t>(row0);
    const bool f32 = p.out_dtype == CHELIS_DTYPE_F32, bf = p.out_dtype == CHELIS_DTYPE_BF16;
    auto box = [&](int n, int cols, const uint32_t(&w)[16]) {
        unsigned char *dst = stage + (n % OUT_BUFS) * OUT_BOX;
        if (lane == 0) store_wait_read();
        __syncwarp();
        stage_box(dst, lane, w);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            if (col0 + n * cols < p.n) tma_store_3d(map, smem_u32(dst), x + n * cols, y, group);
            store_commit();
        }
    };
    if (f32) {
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            uint32_t w[16];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float2 v = unpack2(run[n * 8 + c]);
                w[2 * c] = __float_as_uint(v.x);
                w[2 * c + 1] = __float_as_uint(v.y);
            }
            box(n, 16, w);
        }
    } else {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            uint32_t w[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) w[c] = round2(unpack2(run[n * 16 + c]), bf);
            box(n, 32, w);
        }
    }
}

template <bool BMN, bool WG>
__global__ void __launch_bounds__(THREADS, 1)
    scaled8_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ CUtensorMap map_sfa, const __grid_constant__ CUtensorMap map_sfb,
                   const __grid_constant__ CUtensorMap map_out, const Params8 q) {
    constexpr int STAGES = PAIR_STAGES, STAGE = PAIR_STAGE;
    const Params &p = q.p;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    unsigned char *out_stage = smem + STAGES * STAGE, *sf_ring = out_stage + OUT_BYTES;
    uint64_t *full = reinterpret_cast<uint64_t *>(sf_ring + STAGES * SF_SLOT);
    uint64_t *empty = full + STAGES;
    uint64_t *acc_full = empty + STAGES;  // [2]
    uint64_t *acc_empty = acc_full + 2;   // [2]: of a pair, the first block's
    uint64_t *shared_cols = acc_empty + 2;  // the overlapping columns have been read
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(shared_cols + 1);
    volatile uint32_t *abort_flag = tmem_slot + 1;
    volatile int32_t *consumed = reinterpret_cast<volatile int32_t *>(tmem_slot + 2);
    int32_t *start = reinterpret_cast<int32_t *>(sf_ring + STAGES * SF_SLOT + 512);
    int32_t *quad_start = start + MAX_GROUPS + 1;  // weight gradient

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
            mbar_init(&acc_empty[b], 2 * FOLD_WARPS);
        }
        mbar_init(shared_cols, FOLD_WARPS);  // half of each block's
        *abort_flag = 0;
        *consumed = 0;
        fence_mbarrier_init();
        prefetch_tensormap(&map_a);
        prefetch_tensormap(&map_b);
        prefetch_tensormap(&map_sfa);
        prefetch_tensormap(&map_sfb);
        if (q.tma_out) prefetch_tensormap(&map_out);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, TMEM_COLS);
        tmem_relinquish_pair();
    }
    if (warp == 2) {
        group_starts<WG ? BK : TM>(p, WG ? p.group_rows : p.rows, lane, start, WG ? p.kblocks : -1);
        __syncwarp();
        if (WG) quad_starts(p, lane, start, quad_start);
    }
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int64_t nt = (p.n + BN - 1) / BN;
    const int64_t tiles = p.parts * (WG ? p.groups * nt * ((p.rows + TM - 1) / TM) : start[p.groups] * nt);
    const int all_tiles = uniform(static_cast<int>(tiles));
    int32_t issued = 0;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PAIR_FEW_REGS));
        if (warp == 0) {
            // ---------------- TMA producer ----------------
            int stage = 0;
            uint32_t phase = 1;
            bool ok = true;
            asm volatile("griddepcontrol.wait;" ::: "memory");  // the packed scales are written
            for (int L = worker; ok && L < all_tiles; L += workers) {
                const Tile t = tile_at<WG, TM, QUAD>(p, start, L);
                const int group = uniform(t.group), kbs = uniform(t.kbs), kb0 = uniform(t.kb0);
                const int32_t m0 = uniform(t.m0) + static_cast<int32_t>(rank) * BM;
                const int32_t n_tile = uniform(t.n0);
                const int32_t n0 = n_tile + static_cast<int32_t>(rank) * 128;
                const int quad0 = uniform((WG ? quad_start[group] : 0) + t.in_group / QUAD);
                int32_t sfa = uniform(t.m_tile) * (TM / 128) + static_cast<int32_t>(rank) + quad0 * q.m_atoms;
                int32_t sfb = (WG ? 0 : group * q.sfb_group) + n_tile / 128 + quad0 * q.sfb_k;
                int32_t k0 = kb0 * BK;
                for (int i = 0; i < kbs; ++i) {
                    ok = all(wait(&empty[stage], phase, tries, abort_flag, DEVERR_TIMEOUT_PRODUCER));
                    if (!ok) break;
                    unsigned char *st = smem + stage * STAGE, *sf = sf_ring + stage * SF_SLOT;
                    uint64_t *bar = &full[stage];
                    const bool quad = i % QUAD == 0;
                    const uint32_t bytes = STAGE + (quad ? SF_SLOT : 0);
                    if (elect_one()) {
                        const uint32_t bar0 = mapa_shared(smem_u32(bar), 0);
                        if (rank == 0) mbar_arrive_expect_tx(bar, 2 * bytes);
                        tma_load_2d_pair(st, &map_a, bar0, k0, m0);
                        if (WG) tma_load_2d_pair(st + BOX_BYTES, &map_b, bar0, k0, n0);
                        else if (BMN) tma_load_3d_pair(st + BOX_BYTES, &map_b, bar0, n0, k0, group);
                        else tma_load_3d_pair(st + BOX_BYTES, &map_b, bar0, k0, n0, group);
                        if (quad) {
                            tma_load_2d_pair(sf, &map_sfa, bar0, 0, sfa);
                            tma_load_2d_pair(sf + SF_BYTES, &map_sfb, bar0, 0, sfb);
                        }
                    }
                    ++issued;
                    k0 += BK;
                    if (quad) {
                        sfa += q.m_atoms;
                        sfb += q.sfb_k;
                    }
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        } else if (warp == 1 && rank == 0) {
            // ---------------- MMA issuer ----------------
            const uint32_t tb = uniform(static_cast<int>(tmem_base));
            int32_t it = 0, chunk = 0;
            int stage = 0, slot = 0;
            uint32_t phase = 0;
            bool ok = true, ready = false;
            for (int L = worker; ok && L < all_tiles; L += workers) {
                const int kbs = WG || p.parts > 1 ? uniform(tile_at<WG, TM, QUAD>(p, start, L).kbs) : p.kblocks;
                uint32_t d = 0;
                int cur = 0;
                for (int i = 0; i < kbs; ++i, ++it) {
                    const bool first = i % CHUNK == 0;
                    if (first) {
                        cur = chunk & 1;
                        d = tb + (cur ? ACC1 : 0u);
                        // this accumulator's last chunk but one has been read,
                        // and of the other's the columns they share
                        if (chunk >= 2)
                            ok = all(wait<true>(&acc_empty[cur], ((chunk >> 1) - 1) & 1, tries, abort_flag,
                                                DEVERR_TIMEOUT_MMA));
                        if (!ok) break;
                        if (chunk >= 1)
                            ok = all(wait<true>(shared_cols, (chunk - 1) & 1, tries, abort_flag,
                                                DEVERR_TIMEOUT_MMA));
                        if (!ok) break;
                    }
                    if (!ready) ok = all(wait(&full[stage], phase, tries, abort_flag, DEVERR_TIMEOUT_MMA));
                    if (!ok) break;
                    tc_fence_after();
                    // ask for the next block now, read the answer after this
                    // one's instructions
                    const int next = stage + 1 == STAGES ? 0 : stage + 1;
                    const uint32_t next_phase = next ? phase : phase ^ 1;
                    const bool peek = probe(&full[next], next_phase);
                    const uint32_t a = smem_u32(smem) + stage * STAGE, b = a + BOX_BYTES;
                    if (i % QUAD == 0) slot ^= 1;
                    const uint32_t sf = smem_u32(sf_ring) + stage * SF_SLOT;
                    const uint32_t sfa = tb + SF_COL + slot * 12, sfb = sfa + 4;
                    // the block's byte of the quad's words
                    const uint32_t idesc = p.idesc | (static_cast<uint32_t>(i % QUAD) << 4) |
                                           (static_cast<uint32_t>(i % QUAD) << 29);
                    const bool end = i % CHUNK == CHUNK - 1 || i == kbs - 1;
                    if (elect_one()) {
                        if (i % QUAD == 0) {
                            copy_scales(sfa, sf);
                            copy_scales(sfb, sf + SF_BYTES);
                            copy_scales(sfb + 4, sf + 2 * SF_BYTES);
                        }
#pragma unroll
                        for (int kk = 0; kk < BK / 32; ++kk)
                            mma_scaled(d, sw128_kmajor_desc(a + kk * 32),
                                             BMN ? mnmajor_desc(b + kk * 32 * 128) : sw128_kmajor_desc(b + kk * 32),
                                             idesc, sfa, sfb, !(first && kk == 0));
                        mma_commit_pair(&empty[stage], 0x3);
                        if (end) mma_commit_pair(&acc_full[cur], 0x3);
                    }
                    __syncwarp();
                    if (end) ++chunk;
                    ready = all(peek);
                    stage = next;
                    phase = next_phase;
                }
            }
            if (lane == 0) *consumed = it;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PAIR_FOLD_REGS));
        // ---------------- fold and store ----------------
        const int quad = warp & 3, half = (warp - 4) >> 2;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        unsigned char *stage = out_stage + (warp - 4) * (OUT_BUFS * OUT_BOX);
        int32_t chunk = 0;
        bool ok = true;
        for (int L = worker; ok && L < all_tiles; L += workers) {
            const Tile t = tile_at<WG, TM, QUAD>(p, start, L);
            const int row0 = t.m0 + static_cast<int>(rank) * BM + quad * 32, col0 = t.n0 + half * 128;
            const bool live = row0 < t.m_end && col0 < p.n;  // else nothing to read or store
            f32x2 run[64];
#pragma unroll
            for (int j = 0; j < 64; ++j) run[j] = 0ull;
            for (int i = 0; i < t.kbs; i += CHUNK, ++chunk) {
                const int b = chunk & 1;
                ok = wait(&acc_full[b], (chunk >> 1) & 1, tries, abort_flag, DEVERR_TIMEOUT_EPILOGUE);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t acc = tmem_base + lanes + (b ? ACC1 : 0u) + half * 128;
                auto arrive = [&](uint64_t *bar) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_relaxed(mapa_shared(smem_u32(bar), 0));
                };
                // accumulator 0 shares its last 32 columns, 1 its first
                auto none = [] {};
                auto shared = [&] { arrive(shared_cols); };
                auto done = [&] { arrive(&acc_empty[b]); };
                if (!live) {
                    if (half != b) arrive(shared_cols);
                    arrive(&acc_empty[b]);
                } else if (b == 0 && half == 1) fold128<6>(run, acc, shared, done);
                else if (b == 1 && half == 0) fold128<0>(run, acc, shared, done);
                else fold128<0>(run, acc, none, done);
            }
            if (!ok || !live) continue;
            // whole rows of 32 by TMA (which cuts at the result's own edge); a
            // group's last rows one by one
            if (q.tma_out && (WG || row0 + 32 <= t.m_end)) {
                store_tma(p, &map_out, run, stage, lane, col0, row0, t.matrix);
            } else {
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the box is free
                store_rows(p, run, stage, lane, (t.matrix * p.rows + row0) * p.n + col0, min(t.m_end - row0, 32),
                           p.n - col0);
            }
        }
        if (!WG && p.offsets) zero_loose_rows(p);
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
        tmem_dealloc_pair(tmem_base, TMEM_COLS);
    }
}

// ---- host side ------------------------------------------------------------
// Packed scales [atoms][512 bytes] -> boxes of `atoms` rows.
int make_scale_map(CUtensorMap *map, const void *base, int64_t atoms, int box) {
    tf32x3::EncodeTiledFn fn = tf32x3::encode_fn();
    if (!fn) return set_error(CHELIS_CUDA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    cuuint64_t dims[2] = {SF_BYTES / 4, static_cast<cuuint64_t>(atoms)};
    cuuint64_t strides[1] = {SF_BYTES};
    cuuint32_t boxes[2] = {SF_BYTES / 4, static_cast<cuuint32_t>(box)};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void *>(base), dims, strides, boxes, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return set_error(CHELIS_CUDA_ERR_CUDA, "cuTensorMapEncodeTiled(scales) failed (%d)", (int)r);
    return CHELIS_CUDA_OK;
}
// The result [groups][rows][n] -> boxes of 32 rows x 64 bytes.
int make_out_map(CUtensorMap *map, void *base, int32_t dtype, int64_t n, int64_t rows, int64_t groups) {
    tf32x3::EncodeTiledFn fn = tf32x3::encode_fn();
    if (!fn) return set_error(CHELIS_CUDA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    const cuuint64_t w = static_cast<cuuint64_t>(experts::width(dtype));
    cuuint64_t dims[3] = {static_cast<cuuint64_t>(n), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(groups)};
    cuuint64_t strides[2] = {n * w, n * rows * w};
    cuuint32_t box[3] = {static_cast<cuuint32_t>(64 / w), 32, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = fn(map, w == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, base, dims,
                    strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                    CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return set_error(CHELIS_CUDA_ERR_CUDA, "cuTensorMapEncodeTiled(result) failed (%d)", (int)r);
    return CHELIS_CUDA_OK;
}

uint32_t instruction(int32_t format_a, int32_t format_b, bool bmn) {
    return (format_a == CHELIS_FORMAT_E5M2 ? 1u << 7 : 0u) |  // 0 e4m3, 1 e5m2
           (format_b == CHELIS_FORMAT_E5M2 ? 1u << 10 : 0u) |
           (bmn ? 1u << 16 : 0u) |                             // b MN-major
           (static_cast<uint32_t>(BN >> 3) << 17) | (1u << 23) |  // scales are exponents
           (static_cast<uint32_t>(TM >> 7) << 27);
}

template <bool BMN, bool WG>
int run_parts(const CUtensorMap &ma, const CUtensorMap &mb, const Params &p, int32_t fa, int32_t fb) {
    cudaStream_t s = current_stream();
    const int64_t nt = (p.n + BN - 1) / BN, nb = (p.n + 127) / 128;
    const int64_t mt = WG ? (p.rows + TM - 1) / TM : row_tiles(p.rows, p.groups, p.offsets != nullptr, TM);
    Params8 q{};
    q.p = p;
    q.p.idesc = instruction(fa, fb, BMN);
    q.m_atoms = static_cast<int32_t>(mt * (TM / 128));
    // by expert, each group's last quad may be a short one
    q.quads = (p.kblocks + QUAD - 1) / QUAD + (WG && p.offsets ? p.groups : 0);
    q.sfb_k = static_cast<int32_t>(nb);
    const int64_t a_atoms = static_cast<int64_t>(q.quads) * q.m_atoms;
    const int64_t b_atoms = (WG ? 1 : p.groups) * q.quads * nb;
    q.sfb_group = static_cast<int32_t>(q.quads * nb);
    if (a_atoms > INT32_MAX || b_atoms > INT32_MAX)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "matmul8: more than 2^31 blocks of scales");
    void *scratch = nullptr;
    CHELIS_TRY(scratch_alloc(&scratch, static_cast<size_t>(a_atoms + b_atoms) * SF_BYTES, s));
    unsigned char *sfb = static_cast<unsigned char *>(scratch) + a_atoms * SF_BYTES;
    auto body = [&]() -> int {
        CUtensorMap msa, msb, mo{};
        CHELIS_TRY(make_scale_map(&msa, scratch, a_atoms, 1));
        CHELIS_TRY(make_scale_map(&msb, sfb, b_atoms, 2));
        q.tma_out = p.n * experts::width(p.out_dtype) % 16 == 0 && experts::aligned16(p.out);
        if (q.tma_out) CHELIS_TRY(make_out_map(&mo, p.out, p.out_dtype, p.n, p.rows, (WG ? p.groups : 1) * p.parts));
        pack_scales_kernel<WG><<<blocks8::grid_for((a_atoms + b_atoms + 7) / 8, 8), PACK_THREADS, 0, s>>>(
            q.p, q.quads, q.m_atoms, static_cast<uint4 *>(scratch), reinterpret_cast<uint4 *>(sfb));
        g_launches++;
        CHELIS_LAUNCH_CHECK("scaled8::pack_scales_kernel");
        auto kernel = scaled8_kernel<BMN, WG>;
        CHELIS_TRY(check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   PAIR_SMEM), "cudaFuncSetAttribute"));
        const int64_t most = (WG ? p.groups : 1) * mt * nt * p.parts;
        const int64_t workers = sm_count() / 2;
        const int64_t used = most < workers ? (most < 1 ? 1 : most) : workers;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(static_cast<unsigned>(2 * used));
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = PAIR_SMEM;
        cfg.stream = s;
        // the set-up of the product's blocks overlaps the packing of the scales,
        // which only its producer waits for
        cudaLaunchAttribute attr[2]{};
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        CHELIS_TRY(check_cuda(cudaLaunchKernelEx(&cfg, kernel, ma, mb, msa, msb, mo, q), "scaled8::scaled8_kernel"));
        g_launches++;
        return CHELIS_CUDA_OK;
    };
    const int rc = body();
    scratch_free(scratch, s);
    return rc;
}
template <bool WG>
int32_t pair_parts_of(const Params &p) {
    const int64_t tiles = (WG ? p.groups * row_tiles(p.rows, 0, false, TM)
                              : row_tiles(p.rows, p.groups, p.offsets != nullptr, TM)) * ((p.n + BN - 1) / BN);
    return part_count(tiles, WG ? p.kblocks / p.groups : p.kblocks, sm_count() / 2, QUAD,
                      2 * SAVED_BLOCKS);  // a block takes half as long here
}
template <bool BMN, bool WG>
int run(const CUtensorMap &ma, const CUtensorMap &mb, const Params &p, int32_t fa, int32_t fb) {
    return in_parts(p, pair_parts_of<WG>(p), WG ? p.groups : 1,
                    [&](const Params &q) { return run_parts<BMN, WG>(ma, mb, q, fa, fb); });
}

}  // namespace scaled8
}  // namespace chelis

using namespace chelis;

namespace {
// The kernel for a product, by what each is estimated to take: few8's time goes
// with the weights that it reads, once for 8 or 32 rows, gemm8's with the blocks
// of 128 x 256 x 128 that a multiprocessor goes through one after another, and
// scaled8's too, at about half as much for a block after a launch more.  The
// estimates' constants are from runs of all three over sizes and experts, of
// which (us in a graph, the weights rotated through memory):
//   few8 and gemm8: 8 rows 1024 x 1024 2.8 and 9.6, 4096 x 4096 8.1 and 13.3,
//   16384 x 4096 22.8 and 22.5; 32 rows 2048 x 4096 8.7 and 12.4, 8192 x 1024 12.6
//   and 10.8; 64 rows 1024 x 4096 11.4 and 11.9, 8192 x 512 11.6 and 8.1; 16 rows by
//   8 experts of 4096 x 1024 12.8 and 13.5, by 64 26.8 and 20.1, of 1024 x 4096 20.1
//   and 28.8.
//   gemm8 and scaled8, and called among others, host included: 512 x 1024 x 512
//   (4 blocks) 8.4, 8.8 and 11.3, 15.2; 2048 x 1024 x 1024 (8) 11.5, 10.2 and 13.5,
//   15.3; 1024 x 1024 x 2048 (16) 14.8, 12.3 and 20.7, 16.4; 6144 x 1024 x 1024 by 8
//   experts (16) 21, 15; 4096 x 1024 x 1024 by 64 21.0, 24.2 and 22.7, 27.9.  Weight
//   gradients: 256 x 256 from 256 rows 10.3, 9.2 and 11.3, 14.7; 1024 x 1024 from
//   512 13.0, 10.1 and 14.5, 15.0, from 2048 17.5, 13.6 and 23.6, 16.7; 1111 x 179
//   from 250 by 64 experts 25.5 and 31.3.
// 128 rows at most for few8, as one expert may hold them all (of 64 of 1024 x
// 1024: 30 and 12.5).
bool few_rows(const gemm8::Params &p) {
    if (p.rows > 128 || p.kblocks > 64) return false;
    const bool wide = p.rows > 8 * static_cast<int64_t>(p.groups);  // as few8::run takes them
    const double each = static_cast<double>(p.rows) / p.groups / (wide ? 32 : 8);
    const double passes = p.offsets ? std::fmax(1.0, each + 0.5) : std::ceil(each);
    if (passes > 2.0) return false;
    const double mb = static_cast<double>(p.n) * p.kblocks * 128 / (1 << 20) * gemm8::used_groups(p);
    const double rate = !wide ? (p.offsets ? 0.26 : 0.33) : (p.kblocks <= 8 ? 1.2 : 0.75);  // us a MB and pass
    int64_t serial;
    return passes * (2.0 + rate * mb) < gemm8::forward_us(p, &serial);
}

// gemm8 for powers of two too: few blocks one after another, or experts with so
// few rows that a pair's tiles of 256 are mostly empty and its blocks no fewer.
bool one_by_one(const gemm8::Params &p) {
    int64_t serial;
    gemm8::forward_us(p, &serial);
    return serial <= 8 || (p.offsets && p.rows <= 64 * static_cast<int64_t>(p.groups) &&
                           2 * gemm8::rounds<false>(p, scaled8::TM, sm_count() / 2) * p.kblocks >= 3 * serial);
}
// The same for a weight gradient, whose f32 result costs gemm8 as much as three
// blocks more a tile and scaled8 a little less, the most where TMA cannot store it.
bool one_by_one_wgrad(const gemm8::Params &p) {
    const double blocks = static_cast<double>((p.kblocks + p.groups - 1) / p.groups);
    const int64_t parts = gemm8::parts_of<true>(p), pair_parts = scaled8::pair_parts_of<true>(p);
    const double one = parts > 1 ? 7.1 + blocks / parts : gemm8::rounds<true>(p, gemm8::BM, sm_count()) * (blocks + 3.4);
    const double store = p.n * experts::width(p.out_dtype) % 16 == 0 ? 2.9 : 4.0;
    const int64_t rounds = gemm8::rounds<true>(p, scaled8::TM, sm_count() / 2);
    const double pairs = pair_parts > 1 ? 9.3 + 0.25 * blocks / pair_parts : 2.7 + rounds * (0.25 * blocks + store);
    return one <= pairs;
}
}  // namespace

extern "C" int chelis_cuda_matmul8(int32_t format_a, int32_t format_b, int trans_b, int64_t rows,
                                   int64_t n, int64_t k, const uint8_t *a, const float *scales_a,
                                   const uint8_t *b, const float *scales_b, const int32_t *offsets,
                                   int32_t groups, int any_scales, int32_t out_dtype, void *out) {
    CHELIS_TRY(gemm8::check_common("matmul8", format_a, format_b, out_dtype, rows, n, k, offsets, groups));
    if (rows == 0 || n == 0) return CHELIS_CUDA_OK;
    if (!out) return set_error(CHELIS_CUDA_ERR_DOMAIN, "matmul8: null operand");
    if (k == 0) return gemm8::zero_out(out, out_dtype, rows * n);
    if (!a || !scales_a || !b || !scales_b)
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "matmul8: null operand");
    if (!experts::aligned16(a) || !experts::aligned16(b))
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "matmul8: 8-bit data must lie on 16 bytes");
    const int64_t kblocks = (k + 127) / 128, nblocks = (n + 127) / 128;
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
    p.any_scales = any_scales != 0;
    if (trans_b && few_rows(p)) return few8::run(a, b, p, blocks8::round16(k), format_a, format_b);
    CUtensorMap ma, mb;
    CHELIS_TRY(gemm8::make_map(&ma, a, k, blocks8::round16(k), rows, 1, false));
    if (trans_b) CHELIS_TRY(gemm8::make_map(&mb, b, k, blocks8::round16(k), n, groups, true));
    else CHELIS_TRY(gemm8::make_map(&mb, b, n, blocks8::round16(n), k, groups, true));
    if (any_scales || one_by_one(p))
        return trans_b ? gemm8::run<false, false>(ma, mb, p, format_a, format_b)
                       : gemm8::run<true, false>(ma, mb, p, format_a, format_b);
    return trans_b ? scaled8::run<false, false>(ma, mb, p, format_a, format_b)
                   : scaled8::run<true, false>(ma, mb, p, format_a, format_b);
}

extern "C" int chelis_cuda_matmul8_wgrad(int32_t format_a, int32_t format_b, int64_t n, int64_t k,
                                         int64_t places, const uint8_t *a, const float *scales_a,
                                         const uint8_t *b, const float *scales_b,
                                         const int32_t *offsets, int32_t groups, int any_scales, int32_t out_dtype,
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
    p.any_scales = any_scales != 0;
    if (any_scales || one_by_one_wgrad(p))
        return gemm8::run<false, true>(ma, mb, p, format_a, format_b);
    return scaled8::run<false, true>(ma, mb, p, format_a, format_b);
}
