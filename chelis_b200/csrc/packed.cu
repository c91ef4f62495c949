// packed.cu -- the 16-bit sublayer's entries with their arguments in an array,
// for bindings that pay by the argument (ctypes: 1.9 us for seventeen, 0.5 packed,
// of the 9 to 11 that a small call takes).
#include <cstring>

#include "common.cuh"

using namespace chelis;

namespace {
struct Packed {
    const int64_t *at;
    int64_t integer() { return *at++; }
    int32_t small() { return static_cast<int32_t>(*at++); }
    template <typename T = void>
    T *pointer() { return reinterpret_cast<T *>(static_cast<uintptr_t>(*at++)); }
    float real() {
        double v;
        std::memcpy(&v, at++, sizeof v);
        return static_cast<float>(v);
    }
};
}  // namespace

extern "C" int chelis_cuda_call_packed(int32_t entry, const int64_t *args) {
    if (!args) return set_error(CHELIS_CUDA_ERR_DOMAIN, "call_packed: null operand");
    Packed p{args};
    CHELIS_TRY(chelis_cuda_set_stream(p.pointer()));
    // the arguments are read one after another: braces order them
    switch (entry) {
        case CHELIS_PACKED_MATMUL16: {
            const int32_t dtype = p.small(), ta = p.small(), tb = p.small();
            const int64_t m = p.integer(), n = p.integer(), k = p.integer();
            const void *a = p.pointer(), *b = p.pointer(), *bias = p.pointer();
            const int32_t bias_dtype = p.small(), act = p.small();
            const void *residual = p.pointer(), *through = p.pointer();
            void *pre = p.pointer();
            const int32_t out_dtype = p.small();
            return chelis_cuda_matmul16(dtype, ta, tb, m, n, k, a, b, bias, bias_dtype, act, residual, through, pre, out_dtype,
                                        p.pointer());
        }
        case CHELIS_PACKED_ACTIVATION16_BWD: {
            const int32_t dtype = p.small(), act = p.small();
            const void *dy = p.pointer(), *pre = p.pointer();
            const int64_t count = p.integer();
            return chelis_cuda_activation16_bwd(dtype, act, dy, pre, count, p.pointer());
        }
        case CHELIS_PACKED_COLUMN_SUMS16: {
            const int32_t dtype = p.small();
            const void *x = p.pointer();
            const int64_t rows = p.integer(), cols = p.integer();
            return chelis_cuda_column_sums16(dtype, x, rows, cols, p.pointer<float>());
        }
        case CHELIS_PACKED_RESIDUAL_NORM: {
            const int32_t dtype = p.small(), kind = p.small();
            const int64_t rows = p.integer(), hidden = p.integer();
            const void *x = p.pointer(), *branch = p.pointer();
            const float *g1 = p.pointer<float>(), *b1 = p.pointer<float>(), *gate = p.pointer<float>();
            const int64_t groups = p.integer();
            const float scale = p.real();
            const float *g2 = p.pointer<float>(), *b2 = p.pointer<float>();
            const float eps = p.real();
            void *y = p.pointer(), *h = p.pointer();
            return chelis_cuda_residual_norm(dtype, kind, rows, hidden, x, branch, g1, b1, gate, groups, scale, g2, b2, eps, y, h);
        }
        case CHELIS_PACKED_RESIDUAL_NORM_BWD: {
            const int32_t dtype = p.small(), kind = p.small();
            const int64_t rows = p.integer(), hidden = p.integer();
            const void *dy = p.pointer(), *dh = p.pointer(), *y = p.pointer(), *branch = p.pointer();
            const float *g1 = p.pointer<float>(), *b1 = p.pointer<float>(), *gate = p.pointer<float>();
            const int64_t groups = p.integer();
            const float scale = p.real();
            const float *g2 = p.pointer<float>();
            const float eps = p.real();
            void *dx = p.pointer(), *dbranch = p.pointer();
            float *dg1 = p.pointer<float>(), *db1 = p.pointer<float>(), *dgate = p.pointer<float>(), *dg2 = p.pointer<float>(),
                  *db2 = p.pointer<float>();
            return chelis_cuda_residual_norm_bwd(dtype, kind, rows, hidden, dy, dh, y, branch, g1, b1, gate, groups, scale, g2,
                                                 eps, dx, dbranch, dg1, db1, dgate, dg2, db2);
        }
        case CHELIS_PACKED_EXPERT_BALANCE: {
            const int32_t dtype = p.small();
            const void *logits = p.pointer();
            const int32_t *ids = p.pointer<int32_t>();
            const uint8_t *mask = p.pointer<uint8_t>();
            const int64_t tokens = p.integer();
            const int32_t experts = p.small(), k = p.small();
            float *loss = p.pointer<float>();
            return chelis_cuda_expert_balance(dtype, logits, ids, mask, tokens, experts, k, loss, p.pointer<int32_t>());
        }
        case CHELIS_PACKED_EXPERT_BALANCE_BWD: {
            const int32_t dtype = p.small();
            const void *logits = p.pointer();
            const int32_t *counts = p.pointer<int32_t>();
            const uint8_t *mask = p.pointer<uint8_t>();
            const int64_t tokens = p.integer();
            const int32_t experts = p.small(), k = p.small();
            const float weight = p.real(), *dloss = p.pointer<float>();
            const void *add = p.pointer();
            return chelis_cuda_expert_balance_bwd(dtype, logits, counts, mask, tokens, experts, k, weight, dloss, add, p.pointer());
        }
        case CHELIS_PACKED_GRAD_NORM: {
            const int32_t n = p.small();
            const void *const *data = p.pointer<const void *const>();
            const int64_t *counts = p.pointer<int64_t>();
            const int32_t *dtypes = p.pointer<int32_t>();
            return chelis_cuda_grad_norm(n, data, counts, dtypes, p.pointer<float>());
        }
        case CHELIS_PACKED_CLIP_GRADS: {
            const int32_t n = p.small();
            const void *const *data = p.pointer<const void *const>();
            const int64_t *counts = p.pointer<int64_t>();
            const int32_t *dtypes = p.pointer<int32_t>();
            void *const *out = p.pointer<void *const>();
            const int32_t *out_dtypes = p.pointer<int32_t>();
            const float max_norm = p.real();
            return chelis_cuda_clip_grads(n, data, counts, dtypes, out, out_dtypes, max_norm, p.pointer<float>());
        }
        default:
            return set_error(CHELIS_CUDA_ERR_UNSUPPORTED, "call_packed: unknown entry %d", entry);
    }
}
