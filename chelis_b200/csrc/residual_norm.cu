// residual_norm.cu -- what stands between two blocks, one pass over a row:
//
//   u = N(branch) g1 + b1,   y = scale x + gate u,   h = N(y) g2 + b2
//
// and its gradients.  N is layer_norm's or the root-mean-square norm; every part
// is optional; rows are f32, bf16 or f16, everything between is f32.  With n1, n2
// the normalised rows, r1, r2 what they were multiplied by:
//
//   q  = dh g2,             dt = dy + r2 (q - mean(q) - n2 mean(q n2)),  dx = scale dt
//   w  = dt gate g1,        dbranch = r1 (w - mean(w) - n1 mean(w n1))
//   dg2 = sum dh n2,  db2 = sum dh,  s1 = sum dt n1,  s0 = sum dt over a gate's rows,
//   dgate = g1 s1 + b1 s0,  dg1 = sum gate s1,  db1 = sum gate s0
//
// (the rms norm without the means of q and w; without a first norm dgate = sum
// dt branch, kept as s1).  A row's values are taken about its warps' own means, which
// are put together exactly, so a mean far from 0 costs no digits but those of its sum.
//
// 16384 x 1024 bf16, both norms, gate and residual: 35 us (134 MB, 3.9 TB/s; the
// floor is 20): bound by a row's chain of sums at 16 warps a multiprocessor.  With 8
// values a thread it took 62 (84 instructions a value, most of them a row's fixed
// ones), with 32 and IEEE divisions away 44, with the parameters in shared memory 34.
// 16384 x 1024 f32 54 us (268 MB, 5.0 TB/s), 16384 x 4096 f32 183 (5.9 TB/s), though of
// f32 rows of 1024, 2048, 4096 and 8192 shared memory holds no more than those at work.
// Gradients of 16384 x 4096 f32 with 8 gates: 298 us (1.61 GB, 5.4 TB/s; the floor is
// 246), 643 with rows loaded as they were wanted, 461 through the ring of bulk copies,
// 291 by reciprocals, sums of two at once, pointers carried along and packed
// instructions, the last 7 for the mean's second part.  16384 x 1024 bf16, one norm 42 us
// (134 MB, 3.2 TB/s), both 76 (2.6 TB/s): instructions and a row's chains of sums at 16
// warps a multiprocessor; 64 to 86 and 107 with every team's sums written out and folded
// by few warps.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "common.cuh"

namespace chelis {

extern std::atomic<uint64_t> g_launches;

namespace rnorm {

using experts::from_f32;
using experts::load_pack;
using experts::Pack;
using experts::store_pack;
using experts::to_f32;
using experts::warp_sum;

constexpr int MAX_HIDDEN = 8192;

// Two values at a time where packs have pairs (packed f32 instructions): v + s, v a +
// s, v a + w of N of them.
using gemm8::f32x2;
using gemm8::pack2;
using gemm8::unpack2;
template <int N>
__device__ __forceinline__ void affine(float (&v)[N], float a, float s) {
    if constexpr (N % 2 == 0) {
        const f32x2 a2 = pack2(a, a), s2 = pack2(s, s);
#pragma unroll
        for (int c = 0; c < N; c += 2) {
            const float2 r = unpack2(gemm8::fma2(pack2(v[c], v[c + 1]), a2, s2));
            v[c] = r.x, v[c + 1] = r.y;
        }
    } else {
#pragma unroll
        for (int c = 0; c < N; ++c) v[c] = fmaf(v[c], a, s);
    }
}
template <int N>
__device__ __forceinline__ void multiply_add(float (&v)[N], const float (&a)[N], const float (&s)[N]) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int c = 0; c < N; c += 2) {
            const float2 r = unpack2(gemm8::fma2(pack2(v[c], v[c + 1]), pack2(a[c], a[c + 1]), pack2(s[c], s[c + 1])));
            v[c] = r.x, v[c + 1] = r.y;
        }
    } else {
#pragma unroll
        for (int c = 0; c < N; ++c) v[c] = fmaf(v[c], a[c], s[c]);
    }
}
// Sum of v; v less `centre`, in place, and the sum of its squares.
template <int N>
__device__ __forceinline__ float values_sum(const float *v) {
    if constexpr (N % 2 == 0) {
        f32x2 s = pack2(v[0], v[1]);
#pragma unroll
        for (int c = 2; c < N; c += 2) s = gemm8::add2(s, pack2(v[c], v[c + 1]));
        const float2 r = unpack2(s);
        return r.x + r.y;
    } else {
        float s = v[0];
#pragma unroll
        for (int c = 1; c < N; ++c) s += v[c];
        return s;
    }
}
template <int N>
__device__ __forceinline__ float centre_squares(float *v, float centre) {
    if constexpr (N % 2 == 0) {
        const f32x2 m = pack2(-centre, -centre);
        f32x2 q = 0ull;
#pragma unroll
        for (int c = 0; c < N; c += 2) {
            const f32x2 d = gemm8::add2(pack2(v[c], v[c + 1]), m);
            const float2 r = unpack2(d);
            v[c] = r.x, v[c + 1] = r.y;
            q = gemm8::fma2(d, d, q);
        }
        const float2 r = unpack2(q);
        return r.x + r.y;
    } else {
        float q = 0.0f;
#pragma unroll
        for (int c = 0; c < N; ++c) {
            v[c] -= centre;
            q = fmaf(v[c], v[c], q);
        }
        return q;
    }
}
// sum / n by the reciprocal of n, rounded once.
__device__ __forceinline__ float quotient(float sum, float n, float inv) {
    const float m = sum * inv;
    return fmaf(fmaf(-m, n, sum), inv, m);
}

// to = a b, sum += a b, sum += a, of N of them; the sum of a b; a =
// (a + b w + c0) s (rounded so, a row that cancels gives 0).
template <int N>
__device__ __forceinline__ void product(float *to, const float *a, const float *b) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int c = 0; c < N; c += 2) {
            const float2 r = unpack2(gemm8::mul2(pack2(a[c], a[c + 1]), pack2(b[c], b[c + 1])));
            to[c] = r.x, to[c + 1] = r.y;
        }
    } else {
#pragma unroll
        for (int c = 0; c < N; ++c) to[c] = a[c] * b[c];
    }
}
template <int N>
__device__ __forceinline__ void accumulate(float *sum, const float *a, const float *b) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int c = 0; c < N; c += 2) {
            const float2 r = unpack2(gemm8::fma2(pack2(a[c], a[c + 1]), pack2(b[c], b[c + 1]), pack2(sum[c], sum[c + 1])));
            sum[c] = r.x, sum[c + 1] = r.y;
        }
    } else {
#pragma unroll
        for (int c = 0; c < N; ++c) sum[c] = fmaf(a[c], b[c], sum[c]);
    }
}
template <int N>
__device__ __forceinline__ void accumulate(float *sum, const float *a) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int c = 0; c < N; c += 2) {
            const float2 r = unpack2(gemm8::add2(pack2(sum[c], sum[c + 1]), pack2(a[c], a[c + 1])));
            sum[c] = r.x, sum[c + 1] = r.y;
        }
    } else {
#pragma unroll
        for (int c = 0; c < N; ++c) sum[c] += a[c];
    }
}
template <int N>
__device__ __forceinline__ float products_sum(const float *a, const float *b) {
    if constexpr (N % 2 == 0) {
        f32x2 s = gemm8::mul2(pack2(a[0], a[1]), pack2(b[0], b[1]));
#pragma unroll
        for (int c = 2; c < N; c += 2) s = gemm8::fma2(pack2(a[c], a[c + 1]), pack2(b[c], b[c + 1]), s);
        const float2 r = unpack2(s);
        return r.x + r.y;
    } else {
        float s = a[0] * b[0];
#pragma unroll
        for (int c = 1; c < N; ++c) s = fmaf(a[c], b[c], s);
        return s;
    }
}
template <int N>
__device__ __forceinline__ void combine(float *a, const float *b, float w, float c0, float s) {
    if constexpr (N % 2 == 0) {
        const f32x2 s2 = pack2(s, s), w2 = pack2(w, w), c2 = pack2(c0, c0);
#pragma unroll
        for (int c = 0; c < N; c += 2) {
            const f32x2 t = gemm8::fma2(pack2(b[c], b[c + 1]), w2, c2);
            const float2 r = unpack2(gemm8::mul2(gemm8::add2(pack2(a[c], a[c + 1]), t), s2));
            a[c] = r.x, a[c + 1] = r.y;
        }
    } else {
#pragma unroll
        for (int c = 0; c < N; ++c) a[c] = (a[c] + fmaf(b[c], w, c0)) * s;
    }
}

struct Params {
    int64_t rows;
    int32_t hidden, rms;
    const void *x, *branch;
    const float *post_gamma, *post_beta, *gate, *pre_gamma, *pre_beta;
    int64_t per_gate;  // rows that share a gate
    float scale, eps;
    void *y, *h;
    int32_t staged;    // the parameters fit in shared memory beside the ring
};

// V consecutive f32 parameters.
template <int N>
__device__ __forceinline__ void load_params(const float *p, float (&v)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 f = __ldg(reinterpret_cast<const float4 *>(p + i));
            v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __ldg(p + i);
    }
}

template <int N>
__device__ __forceinline__ void store_sums(float *p, const float *v) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) *reinterpret_cast<float4 *>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = v[i];
    }
}

// The threads of one row: W warps, TEAMS of them in a block.
//
// Rows come through shared memory: a team's first lane copies the next STAGES
// rows of every operand there in bulk while this one is worked on (operands whose
// rows no 16 bytes divide are read from global memory where they are wanted).
// Each thread keeps E values of a row, in packs of N, pack i from column
// (t + i THREADS) N on, and reads its parameters once for all of its rows.
constexpr int THREADS = 512;
constexpr int MAX_STAGES = 4;
constexpr int MAX_ARRAYS = 4;

__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

template <int W>
struct Shared {
    static constexpr int TEAMS = THREADS / (32 * W);
    float2 slots[TEAMS][2][2][W];  // of each team two in turn, for one row's sums and another's
    uint64_t landed[TEAMS][MAX_STAGES];
};

// A row's operands; NULL: not there.
struct Rows {
    const void *of[MAX_ARRAYS];
    int32_t arrays;     // that are there
    int32_t row_bytes;  // rounded up to 16
    int32_t stages;
};

template <typename T, bool VEC, int W, int PACKS>
struct Team {
    static constexpr int TEAMS = Shared<W>::TEAMS, SPAN = W * 32, N = Pack<T, VEC>::N, E = PACKS * N;
    Shared<W> &shared;
    const int t, id, warp, lane, hidden;
    const bool second;        // the half of the warp that looks after the second of two sums
    const uint32_t tries;
    float inv, own, own_inv;  // 1 / hidden; values of this warp's, 1 / them (0 for none)
    float slot_own, slot_inv;  // of the warp whose slot this lane reads
    int turn = 0;
    bool in[PACKS];
    // the ring
    unsigned char *ring, *at;
    int stage_bytes, stage = 0;
    uint32_t phase = 0;
    bool dead = false;  // a wait ran out: reported, no more waits

    __device__ __forceinline__ Team(Shared<W> &sh, unsigned char *smem, const Rows &rows, int h)
        : shared(sh), t(threadIdx.x % SPAN), id(threadIdx.x / SPAN), warp(threadIdx.x / 32 % W), lane(threadIdx.x & 31),
          hidden(h), second((threadIdx.x & 16) != 0), tries(*static_cast<volatile uint32_t *>(&g_wait_tries)),
          stage_bytes(rows.arrays * rows.row_bytes) {
        const int mine = values_of(warp), other = values_of(lane % W);
        inv = 1.0f / static_cast<float>(h);
        own = static_cast<float>(mine);
        own_inv = mine ? 1.0f / own : 0.0f;
        slot_own = static_cast<float>(other);
        slot_inv = other ? 1.0f / static_cast<float>(other) : 0.0f;
#pragma unroll
        for (int i = 0; i < PACKS; ++i) in[i] = col(i) < hidden;
        ring = smem + static_cast<size_t>(id) * rows.stages * stage_bytes;
        at = ring + t * N * sizeof(T);
        if (threadIdx.x == 0) {
            for (int k = 0; k < TEAMS; ++k)
                for (int s = 0; s < MAX_STAGES; ++s) mbar_init(&sh.landed[k][s], 1);
            fence_mbarrier_init();
        }
        __syncthreads();
    }
    __device__ __forceinline__ int values_of(int w) const {
        int n = 0;
#pragma unroll
        for (int i = 0; i < PACKS; ++i) n += min(max(hidden - (w * 32 + i * SPAN) * N, 0), 32 * N);
        return n;
    }
    __device__ __forceinline__ int col(int i) const { return (t + i * SPAN) * N; }
    __device__ __forceinline__ void barrier() const {
        if constexpr (W > 1) asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "n"(SPAN) : "memory");
        else __syncwarp();
    }
    // Row `row` on its way to stage `s`, by one thread.
    __device__ __forceinline__ void fetch(const Rows &rows, int64_t row, int s) {
        if (dead) return;
        unsigned char *dst = ring + s * stage_bytes;
        uint64_t *bar = &shared.landed[id][s];
        mbar_arrive_expect_tx(bar, stage_bytes);
#pragma unroll
        for (int a = 0; a < MAX_ARRAYS; ++a)
            if (rows.of[a]) {
                bulk_load(dst, static_cast<const unsigned char *>(rows.of[a]) + row * rows.row_bytes, rows.row_bytes, bar);
                dst += rows.row_bytes;
            }
    }
    __device__ __forceinline__ bool wait_for(uint64_t *bar) const {
        for (uint32_t i = 0; i < tries; ++i)
            if (mbar_try_wait(bar, phase)) return true;
        report_device_error(DEVERR_TIMEOUT_PRODUCER);
        return false;
    }
    __device__ __forceinline__ void wait() {
        if (VEC && !dead) dead = !wait_for(&shared.landed[id][stage]);
    }
    __device__ __forceinline__ void next(int stages) {
        at += stage_bytes;
        if (++stage == stages) {
            at -= stages * stage_bytes;
            stage = 0;
            phase ^= 1;
        }
    }
    // Pack i of operand `a`, the `place`th of those that are there.
    __device__ __forceinline__ void value(const Rows &rows, int a, int place, int64_t row, int i, float (&v)[N]) const {
        Pack<T, VEC> k;
        if constexpr (VEC)
            *reinterpret_cast<uint4 *>(&k) =
                *reinterpret_cast<const uint4 *>(at + place * rows.row_bytes + i * (SPAN * N * static_cast<int>(sizeof(T))));
        else
            k = load_pack<T, false>(static_cast<const T *>(rows.of[a]) + row * hidden + col(i));
#pragma unroll
        for (int c = 0; c < N; ++c) v[c] = to_f32(k.v[c]);
    }
    template <typename F>
    __device__ __forceinline__ void store(void *to, int64_t row, int i, F f) const {
        Pack<T, VEC> o;
#pragma unroll
        for (int c = 0; c < N; ++c) o.v[c] = from_f32<T>(f(i * N + c));
        store_pack<T, VEC>(static_cast<T *>(to) + row * hidden + t * N + i * (SPAN * N), o);
    }
    // This thread's parameters, `absent` where there are none.
    __device__ __forceinline__ void params(const float *p, float absent, float (&v)[E]) const {
#pragma unroll
        for (int i = 0; i < PACKS; ++i) params(p, absent, i, *reinterpret_cast<float(*)[N]>(&v[i * N]));
    }
    __device__ __forceinline__ void params(const float *p, float absent, int i, float (&v)[N]) const {
#pragma unroll
        for (int c = 0; c < N; ++c) v[c] = absent;
        if (p && in[i]) load_params<N>(p + col(i), v);
    }
    // The same of a copy in shared memory (stage_params): of each 8 the first four
    // lie in one half, the others in the other, so that a warp reads whole lines.
    __device__ __forceinline__ void staged(const float *p, int i, float (&v)[N]) const {
        if constexpr (N == 8) {
            const float4 *f = reinterpret_cast<const float4 *>(p) + t + i * SPAN;
            const float4 a = f[0], b = f[hidden / 8];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else if constexpr (N == 4) {
            const float4 a = reinterpret_cast<const float4 *>(p)[t + i * SPAN];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        }
    }

    // Sums over the team, the same bits in every thread, two at a time: the lower
    // half of a warp adds up the first, the upper half the second.  One barrier;
    // the slots are taken in turn, so the next sum's need not wait for this one's
    // readers.
    __device__ __forceinline__ float2 (*slot())[W] {
        turn ^= 1;
        return shared.slots[id][turn];
    }
    // The warp's sum of a in its lower half, of b in its upper.
    __device__ __forceinline__ float halves_sum(float a, float b) const {
        float v = (second ? b : a) + __shfl_xor_sync(0xffffffffu, second ? a : b, 16);
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
        return v;
    }
    __device__ __forceinline__ static float slots_sum(float v) {
#pragma unroll
        for (int off = W / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
        return v;
    }
    __device__ __forceinline__ static void both(float v, float &a, float &b) {
        a = __shfl_sync(0xffffffffu, v, 0);
        b = __shfl_sync(0xffffffffu, v, 16);
    }
    __device__ __forceinline__ void sum2(float &a, float &b) {
        float v = halves_sum(a, b);
        if constexpr (W > 1) {
            float2(*s)[W] = slot();
            if ((lane & 15) == 0) s[second][warp].x = v;
            barrier();
            v = slots_sum(s[second][lane % W].x);
        }
        both(v, a, b);
    }
    // Reciprocal root, one Newton step past the hardware's.
    __device__ __forceinline__ static float root(float v) {
        const float r = rsqrtf(v);
        return v < INFINITY ? fmaf(0.5f * r, fmaf(-v * r, r, 1.0f), r) : r;
    }
    // Rows u and v at once (or one: two false): their values less the warp's own mean,
    // in place, and what takes them to the normalised row, n = u r + shift: the
    // reciprocal root of the variance and the rest of the mean.  Each warp's sum, its
    // squares about its mean, then the team's.  The difference comes before the product:
    // as u r - mean r the rounding of mean r is left, 1e-3 of a constant row of 100s.
    // The mean is carried in two parts, so a row whose sum f32 holds is off by no more
    // than its products' roundings.
    __device__ __forceinline__ void stats2(float (&u)[E], float (&v)[E], bool two, bool rms, float eps, float *shift_u,
                                           float *r_u, float *shift_v, float *r_v) {
        float su = 0.0f, sv = 0.0f, sum = 0.0f, centre = 0.0f, cu = 0.0f, cv = 0.0f;
        if (!rms) {
            su = values_sum<E>(u);
            if (two) sv = values_sum<E>(v);
            sum = halves_sum(su, sv);
            centre = quotient(sum, own, own_inv);
            both(centre, cu, cv);
        }
        float qu = 0.0f, qv = 0.0f;
#pragma unroll
        for (int i = 0; i < PACKS; ++i)
            if (in[i]) {
                qu += centre_squares<N>(u + i * N, cu);
                if (two) qv += centre_squares<N>(v + i * N, cv);
            }
        float q = halves_sum(qu, qv), rest;
        if constexpr (W > 1) {
            float2(*s)[W] = slot();
            if ((lane & 15) == 0) s[second][warp] = make_float2(sum, q);
            barrier();
            const float2 o = s[second][lane % W];
            const float all = static_cast<float>(hidden), total = slots_sum(o.x), mean = quotient(total, all, inv);
            const float d = rms ? 0.0f : quotient(o.x, slot_own, slot_inv) - mean;
            q = slots_sum(fmaf(slot_own * d, d, o.y));
            rest = (mean - centre) + fmaf(-mean, all, total) * inv;
        } else {
            rest = fmaf(-centre, own, sum) * own_inv;
        }
        const float r = root(fmaf(q, inv, eps));
        both(-rest * r, *shift_u, *shift_v);
        both(r, *r_u, *r_v);
    }
    // Copies that a wait gave up on get another 200 us to land before the block
    // leaves; none are issued after one was.
    __device__ __forceinline__ void drain() const {
        if (!VEC || !dead || t != 0) return;
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000) __nanosleep(1000);
    }
};

// By the whole block: parameters as Team::staged takes them, times `factor`'s if
// that is given, `absent` where there are none.  Whether all that this thread put
// there is finite.
template <int N>
__device__ __forceinline__ bool stage_params(float *to, const float *p, const float *factor, float absent, int hidden) {
    bool finite = true;
    for (int c = threadIdx.x; c < hidden; c += THREADS) {
        const int at = N == 8 ? (c / 8 * 4 + c % 4) + (c & 4 ? hidden / 2 : 0) : c;
        to[at] = (p ? __ldg(p + c) : absent) * (factor ? __ldg(factor + c) : 1.0f);
        finite &= fabsf(to[at]) < INFINITY;
    }
    return finite;
}

// y = scale x + N1(branch) c1 + c0 with c1 = gate g1, c0 = gate b1, h = N2(y) g2 + b2.
template <typename T, bool VEC, int W, int PACKS>
__global__ void __launch_bounds__(THREADS, 1)
    fwd_kernel(const Params p, const Rows in) {
    using G = Team<T, VEC, W, PACKS>;
    constexpr int N = G::N, E = G::E;
    extern __shared__ __align__(128) unsigned char rows_smem[];
    __shared__ Shared<W> shared;
    G team(shared, rows_smem, in, p.hidden);
    const int64_t teams = static_cast<int64_t>(gridDim.x) * G::TEAMS;
    const int64_t me = static_cast<int64_t>(blockIdx.x) * G::TEAMS + team.id;
    const int64_t first = p.rows * me / teams, last = p.rows * (me + 1) / teams;
    if (VEC && team.t == 0)
        for (int s = 0; s < in.stages && first + s < last; ++s) team.fetch(in, first + s, s);
    const bool rms = p.rms != 0, post = p.post_gamma != nullptr, pre = p.pre_gamma != nullptr, branch = p.branch != nullptr;
    // one gate at most: it goes into c1 and c0, unless that leaves f32: gate (n g1 +
    // b1) is an infinity where gate g1 n + gate b1 may be the difference of two
    bool staged = VEC && p.staged;
    const bool one_gate = p.per_gate >= p.rows;
    float *const c1 =
        reinterpret_cast<float *>(rows_smem + static_cast<size_t>(G::TEAMS) * in.stages * in.arrays * in.row_bytes);
    float *const c0 = c1 + p.hidden, *const g2 = c0 + p.hidden, *const b2 = g2 + p.hidden;
    if (staged) {
        const float *g = one_gate ? p.gate : nullptr;
        bool finite = stage_params<N>(c1, p.post_gamma, g, 1.0f, p.hidden);
        finite &= stage_params<N>(c0, p.post_beta, g, 0.0f, p.hidden);
        stage_params<N>(g2, p.pre_gamma, nullptr, 1.0f, p.hidden);
        stage_params<N>(b2, p.pre_beta, nullptr, 0.0f, p.hidden);
        staged = __syncthreads_and(finite);
    }
    const float *gate = nullptr;
    int64_t gate_end = first;
    for (int64_t row = first; row < last; ++row) {
        if (p.gate && !(staged && one_gate) && row >= gate_end) {
            const int64_t group = row / p.per_gate;
            gate = p.gate + group * p.hidden;
            gate_end = (group + 1) * p.per_gate;
        }
        team.wait();
        float v[E], shift = 0.0f, r = 1.0f, none;
#pragma unroll
        for (int i = 0; i < PACKS; ++i) {
            float u[N] = {};
            if (team.in[i]) team.value(in, branch ? 1 : 0, branch ? 1 : 0, row, i, u);
#pragma unroll
            for (int c = 0; c < N; ++c) v[i * N + c] = u[c];
        }
        if (branch) {
            if (post) team.stats2(v, v, false, rms, p.eps, &shift, &r, &none, &none);
#pragma unroll
            for (int i = 0; i < PACKS; ++i)
                if (team.in[i]) {
                    float x[N], k[N];
                    float(&w)[N] = *reinterpret_cast<float(*)[N]>(&v[i * N]);
                    if (staged) {
                        float z[N];
                        team.staged(c1, i, k);
                        team.staged(c0, i, z);
                        affine<N>(w, r, shift);
                        multiply_add<N>(w, k, z);
                    } else if (post) {
                        team.params(p.post_gamma, 1.0f, i, k);
#pragma unroll
                        for (int c = 0; c < N; ++c) v[i * N + c] = fmaf(v[i * N + c], r, shift) * k[c];
                        if (p.post_beta) {
                            team.params(p.post_beta, 0.0f, i, k);
#pragma unroll
                            for (int c = 0; c < N; ++c) v[i * N + c] += k[c];
                        }
                    }
                    if (gate) {
                        team.params(gate, 1.0f, i, k);
#pragma unroll
                        for (int c = 0; c < N; ++c) v[i * N + c] *= k[c];
                    }
                    team.value(in, 0, 0, row, i, x);
                    float scale[N];
#pragma unroll
                    for (int c = 0; c < N; ++c) scale[c] = p.scale;
                    multiply_add<N>(x, scale, w);
#pragma unroll
                    for (int c = 0; c < N; ++c) w[c] = x[c];
                    team.store(p.y, row, i, [&](int e) { return v[e]; });
                }
        }
        if (pre) {
            team.stats2(v, v, false, rms, p.eps, &shift, &r, &none, &none);
#pragma unroll
            for (int i = 0; i < PACKS; ++i)
                if (team.in[i]) {
                    float g[N], k[N];
                    if (staged) {
                        team.staged(g2, i, g);
                        team.staged(b2, i, k);
                    } else {
                        team.params(p.pre_gamma, 0.0f, i, g);
                        team.params(p.pre_beta, 0.0f, i, k);
                    }
                    float(&w)[N] = *reinterpret_cast<float(*)[N]>(&v[i * N]);
                    affine<N>(w, r, shift);
                    multiply_add<N>(w, g, k);
                    team.store(p.h, row, i, [&](int e) { return v[e]; });
                }
        }
        if (VEC) {
            // every thread has read the row once the last statistics' barrier is
            // passed (of the second norm: they need all of y)
            if (!pre || W == 1) team.barrier();
            if (team.t == 0 && row + in.stages < last) team.fetch(in, row + in.stages, team.stage);
            team.next(in.stages);
        }
    }
    team.drain();
}

// ---- backward -------------------------------------------------------------
// A team's rows are consecutive, in units that lie within one gate's rows; the
// sums over them (s1, s0 of a unit, dg2, db2 of the team) stay in registers.  A
// block's teams are put together in shared memory (with more than one gate only dg2
// and db2), and fold_kernel adds up the blocks', or units', sums in order.
struct Backward {
    int64_t rows;
    int32_t hidden, rms;
    const float *post_gamma, *gate, *pre_gamma;
    int64_t per_gate, groups, chunks;  // units = groups * chunks
    float scale, eps;
    void *dx, *dbranch;
    float *unit_sums;  // [units][2][hidden], with one gate [blocks][2][hidden]: s1, s0; NULL: not needed
    float *pre_sums;   // [blocks][2][hidden]: dg2, db2; NULL: not needed
    int32_t staged;    // the parameters lie in shared memory beside the ring
};
enum { DY = 0, DH = 1, Y = 2, BRANCH = 3 };  // of Rows
// What a kernel is made for: the second norm, the branch, or whichever is there.
enum { PRE = 1, POST = 2, ANY = 3 };

template <typename T, bool VEC, int W, int PACKS, int PARTS>
__global__ void __launch_bounds__(THREADS, 1)
    bwd_kernel(const Backward p, const Rows in) {
    using G = Team<T, VEC, W, PACKS>;
    constexpr int N = G::N, E = G::E;
    constexpr bool HOLD = E <= 8 && PARTS == ANY;  // parameters stay in registers
    extern __shared__ __align__(128) unsigned char rows_smem[];
    __shared__ Shared<W> shared;
    G team(shared, rows_smem, in, p.hidden);
    const int64_t teams = static_cast<int64_t>(gridDim.x) * G::TEAMS;
    const int64_t me = static_cast<int64_t>(blockIdx.x) * G::TEAMS + team.id;
    const int64_t units = p.groups * p.chunks;
    // (With fewer and 32-bit divisions here the compiler lays them into every row's
    // path: 16384 x 4096 f32 with 8 gates then takes 318 us for 291.)
    auto unit_rows = [&](int64_t u, int64_t *first, int64_t *last) {
        *first = u / p.chunks * p.per_gate + p.per_gate * (u % p.chunks) / p.chunks;
        *last = u / p.chunks * p.per_gate + p.per_gate * (u % p.chunks + 1) / p.chunks;
    };
    // the row after the last one on its way
    int64_t ahead_unit = me, ahead = 0, ahead_last = 0;
    if (me < units) unit_rows(me, &ahead, &ahead_last);
    auto fetch = [&](int s) {
        while (ahead == ahead_last) {
            ahead_unit += teams;
            if (ahead_unit >= units) return;
            unit_rows(ahead_unit, &ahead, &ahead_last);
        }
        team.fetch(in, ahead++, s);
    };
    if (VEC && team.t == 0 && me < units)
        for (int s = 0; s < in.stages; ++s) fetch(s);

    const bool rms = p.rms != 0, has_dy = in.of[DY] != nullptr;
    const bool pre = PARTS == ANY ? in.of[DH] != nullptr : PARTS == PRE;
    const bool has_branch = PARTS == ANY ? in.of[BRANCH] != nullptr : PARTS == POST;
    const bool post = PARTS != PRE && p.post_gamma != nullptr;
    const int at_dh = has_dy ? 1 : 0, at_y = at_dh + 1, at_b = at_dh + (pre ? 2 : 0);
    const float inv = team.inv;
    float s1[E], s0[E], dg2[E], db2[E], g2[HOLD ? E : 1], c1[HOLD ? E : 1];
#pragma unroll
    for (int e = 0; e < E; ++e) s1[e] = s0[e] = dg2[e] = db2[e] = 0.0f;
    if constexpr (HOLD) team.params(p.pre_gamma, 0.0f, g2);
    const bool staged = !HOLD && VEC && p.staged;
    float *const held =
        reinterpret_cast<float *>(rows_smem + static_cast<size_t>(G::TEAMS) * in.stages * in.arrays * in.row_bytes);
    if (staged) {  // the second norm's gamma, or the first's times the gate
        if (pre) stage_params<N>(held, p.pre_gamma, nullptr, 1.0f, p.hidden);
        else stage_params<N>(held, p.post_gamma, p.gate, 1.0f, p.hidden);
        __syncthreads();
    }
    for (int64_t unit = me; unit < units; unit += teams) {
#pragma unroll
        for (int e = 0; e < E; ++e) s1[e] = s0[e] = 0.0f;
        const float *gate = p.gate ? p.gate + unit / p.chunks * p.hidden : nullptr;
        if constexpr (HOLD) {  // gate times gamma
            float g[E];
            team.params(p.post_gamma, 1.0f, c1);
            team.params(gate, 1.0f, g);
#pragma unroll
            for (int e = 0; e < E; ++e) c1[e] *= g[e];
        }
        int64_t row, last;
        for (unit_rows(unit, &row, &last); row < last; ++row) {
            team.wait();
            float v[E], b[E], dt[E], shift2, r2, shift1 = 0.0f, r1 = 1.0f;
#pragma unroll
            for (int i = 0; i < PACKS; ++i) {
                float u[N] = {}, w[N] = {};
                if (pre && team.in[i]) team.value(in, Y, at_y, row, i, u);
                if (has_branch && team.in[i]) team.value(in, BRANCH, at_b, row, i, w);
#pragma unroll
                for (int c = 0; c < N; ++c) v[i * N + c] = u[c], b[i * N + c] = w[c];
            }
            if (pre) {
                team.stats2(v, b, post, rms, p.eps, &shift2, &r2, &shift1, &r1);
                float sq = 0.0f, sqn = 0.0f;
#pragma unroll
                for (int i = 0; i < PACKS; ++i)
                    if (team.in[i]) {
                        float d[N], g[N];
                        team.value(in, DH, at_dh, row, i, d);
                        if constexpr (!HOLD) {
                            if (staged) team.staged(held, i, g);
                            else load_params<N>(p.pre_gamma + team.col(i), g);
                        }
                        float(&n)[N] = *reinterpret_cast<float(*)[N]>(&v[i * N]);
                        affine<N>(n, r2, shift2);
                        accumulate<N>(dg2 + i * N, d, n);
                        accumulate<N>(db2 + i * N, d);
                        product<N>(dt + i * N, d, HOLD ? g2 + i * N : g);
                        sq += values_sum<N>(dt + i * N);
                        sqn += products_sum<N>(dt + i * N, n);
                    }
                team.sum2(sq, sqn);
                sq = rms ? 0.0f : sq * inv;
                sqn *= inv;
#pragma unroll
                for (int i = 0; i < PACKS; ++i) combine<N>(dt + i * N, v + i * N, -sqn, -sq, r2);
            } else {
                if (post) team.stats2(b, b, false, rms, p.eps, &shift1, &r1, &shift2, &r2);
#pragma unroll
                for (int e = 0; e < E; ++e) dt[e] = 0.0f;
            }
            if (!post) shift1 = 0.0f, r1 = 1.0f;
#pragma unroll
            for (int i = 0; i < PACKS; ++i)
                if (team.in[i]) {
                    if (has_dy) {
                        float d[N];
                        team.value(in, DY, 0, row, i, d);
                        accumulate<N>(dt + i * N, d);
                    }
                    float scaled[N];
#pragma unroll
                    for (int c = 0; c < N; ++c) scaled[c] = p.scale;
                    product<N>(scaled, scaled, dt + i * N);
                    team.store(p.dx, row, i, [&](int e) { return scaled[e - i * N]; });
                }
            if (PARTS == ANY ? p.dbranch != nullptr : has_branch) {
                float sw = 0.0f, swn = 0.0f;
#pragma unroll
                for (int i = 0; i < PACKS; ++i)
                    if (team.in[i]) {
                        float g[N];
#pragma unroll
                        for (int c = 0; c < N; ++c) g[c] = 1.0f;
                        if constexpr (!HOLD) {
                            if (staged && !pre) team.staged(held, i, g);
                            else if (post) load_params<N>(p.post_gamma + team.col(i), g);
                            if (gate && !(staged && !pre)) {
                                float k[N];
                                load_params<N>(gate + team.col(i), k);
#pragma unroll
                                for (int c = 0; c < N; ++c) g[c] *= k[c];
                            }
                        }
                        float(&n)[N] = *reinterpret_cast<float(*)[N]>(&b[i * N]);
                        affine<N>(n, r1, shift1);  // the branch itself without a norm
                        accumulate<N>(s1 + i * N, dt + i * N, n);
                        accumulate<N>(s0 + i * N, dt + i * N);
                        product<N>(dt + i * N, dt + i * N, HOLD ? c1 + i * N : g);
                        sw += values_sum<N>(dt + i * N);
                        swn += products_sum<N>(dt + i * N, n);
                    }
                if (post) {
                    team.sum2(sw, swn);
                    sw = rms ? 0.0f : sw * inv;
                    swn *= inv;
#pragma unroll
                    for (int i = 0; i < PACKS; ++i) combine<N>(dt + i * N, b + i * N, -swn, -sw, r1);
                }
#pragma unroll
                for (int i = 0; i < PACKS; ++i)
                    if (team.in[i]) team.store(p.dbranch, row, i, [&](int e) { return dt[e]; });
            }
            if (VEC) {
                // the last sum's barrier says that every thread has read the row
                if (!post || W == 1) team.barrier();
                if (team.t == 0) fetch(team.stage);
                team.next(in.stages);
            }
        }
        if (p.unit_sums && p.groups > 1) {
            float *dst = p.unit_sums + unit * 2 * p.hidden;
#pragma unroll
            for (int i = 0; i < PACKS; ++i)
                if (team.in[i]) {
                    store_sums<N>(dst + team.col(i), s1 + i * N);
                    store_sums<N>(dst + p.hidden + team.col(i), s0 + i * N);
                }
        }
    }
    team.drain();
    // The teams' sums put together in order, in the ring's memory.
    const auto join = [&](float *to, const float (&a)[E], const float (&b)[E]) {
        float *const all = reinterpret_cast<float *>(rows_smem);
        float *const dst = to + static_cast<int64_t>(blockIdx.x) * 2 * p.hidden;
        float *const mine = G::TEAMS > 1 ? all + team.id * 2 * p.hidden : dst;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PACKS; ++i)
            if (team.in[i]) {
                store_sums<N>(mine + team.col(i), a + i * N);
                store_sums<N>(mine + p.hidden + team.col(i), b + i * N);
            }
        if (G::TEAMS == 1) return;
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * p.hidden; c += THREADS) {
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < G::TEAMS; ++k) sum += all[k * 2 * p.hidden + c];
            dst[c] = sum;
        }
    };
    if (p.unit_sums && p.groups == 1) join(p.unit_sums, s1, s0);
    if (p.pre_sums) join(p.pre_sums, dg2, db2);
}

// Sums of `count` rows of [..][2][hidden], both halves, in a fixed order: 32
// columns a block, its warps taking a row each in turn.  FEW warps where there are
// blocks enough for the machine (8 groups of 16384 x 4096 rows took 30 us with 32,
// the blocks' own launch most of it), MANY where there are not (the 592 rows of 1024
// of one group: 12 us with FEW).
constexpr int FEW_WARPS = 8, MANY_WARPS = 32;
__device__ __forceinline__ void fold2(const float *src, int64_t count, int hidden, float (*part)[2][32], float *a, float *b) {
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, slices = blockDim.x >> 5, col = blockIdx.x * 32 + lane;
    float u = 0.0f, v = 0.0f;
    if (col < hidden) {
        const float *at = src + static_cast<int64_t>(slice) * 2 * hidden + col;
        const int64_t step = static_cast<int64_t>(slices) * 2 * hidden;
        int64_t i = slice;
        for (; i + 7 * slices < count; i += 8 * slices, at += 8 * step) {  // all loads first
            float x[8], y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = __ldg(at + k * step), y[k] = __ldg(at + k * step + hidden);
#pragma unroll
            for (int k = 0; k < 8; ++k) u += x[k], v += y[k];
        }
        float x[7], y[7];
#pragma unroll
        for (int k = 0; k < 7; ++k) {
            const bool there = i + k * slices < count;
            x[k] = there ? __ldg(at + k * step) : 0.0f, y[k] = there ? __ldg(at + k * step + hidden) : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 7; ++k) u += x[k], v += y[k];
    }
    part[slice][0][lane] = u;
    part[slice][1][lane] = v;
    __syncthreads();
    *a = *b = 0.0f;
    if (slice == 0)
#pragma unroll 8
        for (int s = 0; s < slices; ++s) *a += part[s][0][lane], *b += part[s][1][lane];
}
inline int fold_warps(int64_t blocks) { return blocks < 2 * sm_count() ? MANY_WARPS : FEW_WARPS; }
struct Fold {
    const float *unit_sums, *pre_sums;
    int64_t groups, chunks, blocks;  // partial sums of a group, of the second norm
    int32_t hidden;
    const float *post_gamma, *post_beta, *gate;
    float *dgate, *dpost_gamma, *dpost_beta, *dpre_gamma, *dpre_beta;
    float *by_group;  // [groups][2][hidden]: gate times s1, s0 (more than one group)
};
__global__ void __launch_bounds__(32 * MANY_WARPS)
    fold_kernel(const Fold p) {
    __shared__ float part[MANY_WARPS][2][32];
    const int lane = threadIdx.x & 31, col = blockIdx.x * 32 + lane;
    const int64_t groups = p.unit_sums ? p.groups : 0, all = groups + (p.pre_sums ? 1 : 0);
    const bool writes = threadIdx.x < 32 && col < p.hidden;
    for (int64_t group = blockIdx.y; group < all; group += gridDim.y, __syncthreads()) {
        float a, b;
        const bool second = group == groups;  // the second norm's, over all teams
        fold2(second ? p.pre_sums : p.unit_sums + group * p.chunks * 2 * p.hidden, second ? p.blocks : p.chunks, p.hidden,
              part, &a, &b);
        if (second) {
            if (writes && p.dpre_gamma) p.dpre_gamma[col] = a;
            if (writes && p.dpre_beta) p.dpre_beta[col] = b;
            continue;
        }
        if (!writes) continue;
        const int64_t at = group * p.hidden + col;
        if (p.dgate) {
            float d = a;
            if (p.post_gamma) d = p.post_beta ? fmaf(p.post_gamma[col], a, p.post_beta[col] * b) : p.post_gamma[col] * a;
            p.dgate[at] = d;
        }
        if (!p.post_gamma) continue;
        const float g = p.gate ? p.gate[at] : 1.0f;
        if (p.by_group) {
            p.by_group[group * 2 * p.hidden + col] = g * a;
            p.by_group[(group * 2 + 1) * p.hidden + col] = g * b;
        } else {
            if (p.dpost_gamma) p.dpost_gamma[col] = g * a;
            if (p.dpost_beta) p.dpost_beta[col] = g * b;
        }
    }
}
__global__ void __launch_bounds__(32 * MANY_WARPS)
    fold_groups_kernel(const float *__restrict__ by_group, int64_t groups, int hidden, float *__restrict__ dgamma,
                       float *__restrict__ dbeta) {
    __shared__ float part[MANY_WARPS][2][32];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31);
    float a, b;
    fold2(by_group, groups, hidden, part, &a, &b);
    if (threadIdx.x < 32 && col < hidden) {
        if (dgamma) dgamma[col] = a;
        if (dbeta) dbeta[col] = b;
    }
}

// The shared memory that a launch may have.  The attribute that admits it belongs to the
// kernel, which serves rows of many lengths on many host threads, so it is set to one
// value for all of them: with each launch's own, two threads' calls could set it and
// launch by turns, and the longer rows' launch was refused.
constexpr int MOST_SHARED = 208 * 1024;

// The ring's shape and the grid for f(T, VEC, W, PACKS, grid, shared memory): MOST
// values a thread (8 where one warp can take the row so), the fewest warps a team.
// `params`: bytes of parameters that would lie beside the ring; *staged, whether they do.
template <int MOST, typename F>
void launch(int32_t dtype, bool vec, int64_t hidden, Rows &in, int64_t rows, int64_t params, int32_t *staged, F f) {
    const int each = hidden <= 256 ? 8 : (MOST == 8 && hidden > 4096 ? 16 : MOST);
    int warps = 1;
    while (warps < 16 && hidden > static_cast<int64_t>(warps) * 32 * each) warps *= 2;
    const int teams = 16 / warps;
    in.row_bytes = static_cast<int32_t>((hidden * experts::width(dtype) + 15) / 16 * 16);
    const int64_t stage = static_cast<int64_t>(in.arrays) * in.row_bytes * teams;
    // the parameters, where that leaves two stages, or the one that there is
    const int64_t room = MOST_SHARED, beside = vec ? (room - params) / stage : 0;
    *staged = params > 0 && (beside >= 2 || (beside == 1 && room / stage == 1));
    const int64_t stages = vec ? (*staged ? beside : room / stage) : 0;
    in.stages = static_cast<int32_t>(stages > MAX_STAGES ? MAX_STAGES : stages);
    int64_t grid = sm_count();
    if (grid > (rows + teams - 1) / teams) grid = (rows + teams - 1) / teams;
    const size_t smem = static_cast<size_t>(stage) * in.stages + (*staged ? params : 0);
    experts::by_type(dtype, vec, [&](auto t, auto v) {
        constexpr int N = experts::Pack<decltype(t), decltype(v)::value>::N;
        const unsigned g = static_cast<unsigned>(grid);
        auto with = [&](auto w, auto e) { f(t, v, w, std::integral_constant<int, decltype(e)::value / N>{}, g, smem); };
        using E = std::integral_constant<int, MOST>;
        if (each == 8 && warps == 1) with(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
        else if (warps == 16) {
            if constexpr (MOST == 8) {
                if (each == 16) with(std::integral_constant<int, 16>{}, std::integral_constant<int, 16>{});
                else with(std::integral_constant<int, 16>{}, E{});
            } else if constexpr (MOST == 16) with(std::integral_constant<int, 16>{}, E{});
        } else if (warps == 8) with(std::integral_constant<int, 8>{}, E{});
        else if (warps == 4) with(std::integral_constant<int, 4>{}, E{});
        else if (warps == 2) with(std::integral_constant<int, 2>{}, E{});
        else with(std::integral_constant<int, 1>{}, E{});
    });
}

int check(const char *op, int32_t dtype, int32_t kind, int64_t rows, int64_t hidden, int64_t groups) {
    if (!experts::is_act(dtype)) return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "%s takes f32, bf16 or f16", op);
    if (kind != CHELIS_NORM_LAYER && kind != CHELIS_NORM_RMS)
        return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "%s: unknown norm %d", op, kind);
    if (rows < 0 || hidden < 0) return set_error(CHELIS_CUDA_ERR_DOMAIN, "numeric trap: domain in %s at i64", op);
    if (hidden > MAX_HIDDEN) return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "%s admits rows of <= %d", op, MAX_HIDDEN);
    if (groups < 1 || rows % groups != 0)
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "%s: the gate's groups divide the rows", op);
    return CHELIS_CUDA_OK;
}
bool aligned(std::initializer_list<const void *> ps) {
    for (const void *p : ps)
        if (!experts::aligned16(p)) return false;
    return true;
}

}  // namespace rnorm
}  // namespace chelis

using namespace chelis;

extern "C" int chelis_cuda_residual_norm(int32_t dtype, int32_t kind, int64_t rows, int64_t hidden, const void *x,
                                         const void *branch, const float *post_gamma, const float *post_beta,
                                         const float *gate, int64_t groups, float scale, const float *pre_gamma,
                                         const float *pre_beta, float eps, void *y, void *h) {
    CHELIS_TRY(rnorm::check("residual_norm", dtype, kind, rows, hidden, groups));
    if (rows == 0 || hidden == 0) return CHELIS_CUDA_OK;
    if (!branch && (post_gamma || gate || y || scale != 1.0f))
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "residual_norm: without a branch there is the second norm alone");
    if ((post_beta && !post_gamma) || (pre_beta && !pre_gamma))
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "residual_norm: a beta without its gamma");
    if (!x || (branch && !y) || (pre_gamma && !h) || (!branch && !pre_gamma))
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "residual_norm: null operand");
    rnorm::Params p{rows, static_cast<int32_t>(hidden), kind == CHELIS_NORM_RMS, x, branch, post_gamma, post_beta, gate,
                    pre_gamma, pre_beta, rows / groups, scale, eps, y, h, 0};
    const bool vec = hidden * experts::width(dtype) % 16 == 0 &&
                     rnorm::aligned({x, branch, post_gamma, post_beta, gate, pre_gamma, pre_beta, y, h});
    rnorm::Rows in{{x, branch, nullptr, nullptr}, branch ? 2 : 1, 0, 0};
    int rc = CHELIS_CUDA_OK;
    const auto run = [&](auto t, auto v, auto w, auto packs, unsigned grid, size_t smem) {
        auto kernel = rnorm::fwd_kernel<decltype(t), decltype(v)::value, decltype(w)::value, decltype(packs)::value>;
        rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, rnorm::MOST_SHARED),
                        "cudaFuncSetAttribute");
        if (rc == CHELIS_CUDA_OK) kernel<<<grid, rnorm::THREADS, smem, current_stream()>>>(p, in);
    };
    // Few rows: eight values a thread, a row over as many warps as there are; more: 32,
    // which have fewer instructions a number and a longer chain of sums.  us with 8 and
    // with 32, bf16: 148 x 1024 5.4, 8.2, 600 x 1024 6.7, 8.2, 1200 x 1024 9.1, 8.5, 16384 x 1024
    // 60, 35; 200 x 4096 8.2, 9.3, 300 x 4096 10.4, 9.3; 148 x 8192 7.2, 9.5, 149 x 8192 11.0, 9.7;
    // f32 200 x 4096 8.7, 9.5, 300 x 4096 11.0, 9.7.  So the rows of 8192 are parted where the
    // two meet; shorter ones meet at a million numbers, and from 149 rows to there take up
    // to 3 us more than they would with 8.
    if (rows <= sm_count()) rnorm::launch<8>(dtype, vec, hidden, in, rows, 0, &p.staged, run);
    else rnorm::launch<32>(dtype, vec, hidden, in, rows, 16 * hidden, &p.staged, run);
    CHELIS_TRY(rc);
    g_launches++;
    CHELIS_LAUNCH_CHECK("rnorm::fwd_kernel");
    return CHELIS_CUDA_OK;
}

extern "C" int chelis_cuda_residual_norm_bwd(int32_t dtype, int32_t kind, int64_t rows, int64_t hidden, const void *dy,
                                             const void *dh, const void *y, const void *branch, const float *post_gamma,
                                             const float *post_beta, const float *gate, int64_t groups, float scale,
                                             const float *pre_gamma, float eps, void *dx, void *dbranch,
                                             float *dpost_gamma, float *dpost_beta, float *dgate, float *dpre_gamma,
                                             float *dpre_beta) {
    CHELIS_TRY(rnorm::check("residual_norm_bwd", dtype, kind, rows, hidden, groups));
    if (hidden == 0) return CHELIS_CUDA_OK;
    cudaStream_t s = current_stream();
    if ((!post_gamma && (post_beta || dpost_gamma || dpost_beta)) || (!gate && dgate) ||
        (!pre_gamma && (dpre_gamma || dpre_beta)))
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "residual_norm_bwd: a gradient of what is not there");
    if (rows == 0) {
        auto zero = [&](float *p, int64_t n) {
            return p ? check_cuda(cudaMemsetAsync(p, 0, static_cast<size_t>(n) * 4, s), "memset") : CHELIS_CUDA_OK;
        };
        CHELIS_TRY(zero(dpost_gamma, hidden));
        CHELIS_TRY(zero(dpost_beta, hidden));
        CHELIS_TRY(zero(dgate, groups * hidden));
        CHELIS_TRY(zero(dpre_gamma, hidden));
        return zero(dpre_beta, hidden);
    }
    const bool needs_branch = post_gamma || gate;
    if (!dx || (!dy && !dh) || (pre_gamma && !y) || (dh != nullptr) != (pre_gamma != nullptr) ||
        (needs_branch && (!branch || !dbranch)))
        return set_error(CHELIS_CUDA_ERR_DOMAIN, "residual_norm_bwd: null operand");
    const bool vec = hidden * experts::width(dtype) % 16 == 0 &&
                     rnorm::aligned({dy, dh, y, branch, post_gamma, gate, pre_gamma, dx, dbranch});
    rnorm::Rows in{{dy, dh, dh ? y : nullptr, needs_branch ? branch : nullptr},
                   (dy ? 1 : 0) + (dh ? 2 : 0) + (needs_branch ? 1 : 0), 0, 0};
    rnorm::Backward p{};
    p.rows = rows;
    p.hidden = static_cast<int32_t>(hidden);
    p.rms = kind == CHELIS_NORM_RMS;
    p.post_gamma = post_gamma;
    p.gate = gate;
    p.pre_gamma = pre_gamma;
    p.per_gate = rows / groups;
    p.groups = groups;
    p.scale = scale;
    p.eps = eps;
    p.dx = dx;
    p.dbranch = dbranch;
    const bool unit_sums = dpost_gamma || dpost_beta || dgate, pre_sums = dpre_gamma || dpre_beta;
    const bool by_group = groups > 1 && (dpost_gamma || dpost_beta);
    void *scratch = nullptr;
    auto body = [&]() -> int {
        int rc = CHELIS_CUDA_OK;
        float *sums = nullptr;
        size_t unit_n = 0, pre_n = 0;
        int64_t blocks = 0;
        const auto run = [&](auto parts, auto t, auto v, auto w, auto packs, unsigned grid, size_t smem) {
            constexpr int W = decltype(w)::value, TEAMS = rnorm::THREADS / (32 * W);
            const int64_t teams = static_cast<int64_t>(grid) * TEAMS;
            blocks = grid;
            p.chunks = teams / groups < 1 ? 1 : teams / groups;
            if (p.chunks > p.per_gate) p.chunks = p.per_gate;
            unit_n = unit_sums ? static_cast<size_t>(groups > 1 ? groups * p.chunks : blocks) * 2 * hidden : 0;
            pre_n = pre_sums ? static_cast<size_t>(blocks) * 2 * hidden : 0;
            // the teams' sums, put together there
            if (TEAMS > 1) smem = std::max(smem, static_cast<size_t>(TEAMS) * 2 * hidden * sizeof(float));
            const size_t group_n = by_group ? static_cast<size_t>(groups) * 2 * hidden : 0;
            rc = scratch_alloc(&scratch, (unit_n + pre_n + group_n) * sizeof(float), s);
            if (rc != CHELIS_CUDA_OK) return;
            sums = static_cast<float *>(scratch);
            p.unit_sums = unit_sums ? sums : nullptr;
            p.pre_sums = pre_sums ? sums + unit_n : nullptr;
            auto kernel = rnorm::bwd_kernel<decltype(t), decltype(v)::value, W, decltype(packs)::value, decltype(parts)::value>;
            rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, rnorm::MOST_SHARED),
                            "cudaFuncSetAttribute");
            if (rc == CHELIS_CUDA_OK) kernel<<<grid, rnorm::THREADS, smem, s>>>(p, in);
        };
        using Any = std::integral_constant<int, rnorm::ANY>;
        using Pre = std::integral_constant<int, rnorm::PRE>;
        using Post = std::integral_constant<int, rnorm::POST>;
        // Where there are more rows than teams of 8 values a thread, one norm's gradients
        // in 16, which its sums leave registers for: 4800 x 1024 bf16 18.7 us for 22.5 with
        // 8, 300 x 1024 9.7 for 8.6 (both some 4 % less, before means had two parts).  Both
        // norms' in 8.
        const bool many = vec && hidden > 256 && rows * hidden > sm_count() * 4096ll;
        if (many && dh && !needs_branch && !dbranch)
            rnorm::launch<16>(dtype, vec, hidden, in, rows, 4 * hidden, &p.staged, [&](auto t, auto v, auto... rest) {
                if constexpr (decltype(v)::value) run(Pre{}, t, v, rest...);
            });
        else if (many && !dh && needs_branch)
            rnorm::launch<16>(dtype, vec, hidden, in, rows, groups == 1 ? 4 * hidden : 0, &p.staged,
                              [&](auto t, auto v, auto... rest) {
                                  if constexpr (decltype(v)::value) run(Post{}, t, v, rest...);
                              });
        else
            rnorm::launch<8>(dtype, vec, hidden, in, rows, 0, &p.staged, [&](auto... shape) { run(Any{}, shape...); });
        CHELIS_TRY(rc);
        g_launches++;
        CHELIS_LAUNCH_CHECK("rnorm::bwd_kernel");
        if (!unit_sums && !pre_sums) return CHELIS_CUDA_OK;
        rnorm::Fold f{p.unit_sums, p.pre_sums, groups, groups > 1 ? p.chunks : blocks, blocks, p.hidden, post_gamma, post_beta,
                      gate, dgate, dpost_gamma, dpost_beta, dpre_gamma, dpre_beta,
                      by_group ? sums + unit_n + pre_n : nullptr};
        int64_t high = (unit_sums ? groups : 0) + (pre_sums ? 1 : 0);
        if (high > 65535) high = 65535;
        const unsigned wide = static_cast<unsigned>((hidden + 31) / 32);
        rnorm::fold_kernel<<<dim3(wide, static_cast<unsigned>(high)), 32 * rnorm::fold_warps(wide * high), 0, s>>>(f);
        g_launches++;
        CHELIS_LAUNCH_CHECK("rnorm::fold_kernel");
        if (by_group) {
            rnorm::fold_groups_kernel<<<wide, 32 * rnorm::fold_warps(wide), 0, s>>>(f.by_group, groups, p.hidden, dpost_gamma,
                                                                                    dpost_beta);
            g_launches++;
            CHELIS_LAUNCH_CHECK("rnorm::fold_groups_kernel");
        }
        return CHELIS_CUDA_OK;
    };
    const int rc = body();
    scratch_free(scratch, s);
    return rc;
}
