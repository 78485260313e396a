// matmul.hip -- entry points of the products with packed weights (include/ggq.h): argument checks and launches.
#include "../../include/ggq.h"
#include "internal.h"
#include "launch.h"
#include "route.h"

#include <algorithm>

using namespace ggq;

namespace {

// a sum of nothing
static __global__ __launch_bounds__(MV_THREADS) void fill_zero(MatvecArgs a) {
    const uint64_t r = (uint64_t)blockIdx.x * MV_THREADS + threadIdx.x;
    if (r >= a.rows) return;
    for (uint32_t t = 0; t < a.tokens; ++t) store_elem(a.y, t * a.y_stride + r, a.y_kind, 0.0f);
}

#define HIP_TRY(call)                                       \
    do {                                                    \
        if (!report_hip((call), #call)) return GGQ_DEVICE;  \
    } while (0)

// CASE(F) for the block type `ty`, otherwise GGQ_UNSUPPORTED
#define GGQ_FOR_TYPE(ty, CASE)                                    \
    switch (ty) {                                                 \
    case GGQ_TYPE_F16: CASE(WF16); break;                         \
    case GGQ_TYPE_BF16: CASE(WBF16); break;                       \
    case GGQ_TYPE_Q4_0: CASE(Q4_0); break;                        \
    case GGQ_TYPE_Q4_1: CASE(Q4_1); break;                        \
    case GGQ_TYPE_Q5_0: CASE(Q5_0); break;                        \
    case GGQ_TYPE_Q5_1: CASE(Q5_1); break;                        \
    case GGQ_TYPE_Q8_0: CASE(Q8_0); break;                        \
    case GGQ_TYPE_Q8_1: CASE(Q8_1); break;                        \
    case GGQ_TYPE_Q2K: CASE(Q2K); break;                          \
    case GGQ_TYPE_Q3K: CASE(Q3K); break;                          \
    case GGQ_TYPE_Q4K: CASE(Q4K); break;                          \
    case GGQ_TYPE_Q5K: CASE(Q5K); break;                          \
    case GGQ_TYPE_Q6K: CASE(Q6K); break;                          \
    case GGQ_TYPE_Q8K: CASE(Q8K); break;                          \
    case GGQ_TYPE_IQ4NL: CASE(IQ4NL); break;                      \
    case GGQ_TYPE_IQ4XS: CASE(IQ4XS); break;                      \
    default: return GGQ_UNSUPPORTED;                              \
    }

bool elem_kind(uint32_t ty, uint32_t *kind, uint32_t *bytes) {
    switch (ty) {
    case GGQ_TYPE_F32: *kind = EK_F32; *bytes = 4; return true;
    case GGQ_TYPE_F16: *kind = EK_F16; *bytes = 2; return true;
    case GGQ_TYPE_BF16: *kind = EK_BF16; *bytes = 2; return true;
    }
    return false;
}

// Sizes beyond these have no use and would let products of sizes wrap.
constexpr uint64_t MAX_DIM = 1ull << 30;
// Workgroups of one launch along y
constexpr uint64_t MAX_GRID_Y = 65535;

bool strides_ok(uint64_t stride, uint64_t width, uint64_t tokens) {
    return stride < (1ull << 40) && (tokens <= 1 || stride >= width);
}

}  // namespace

// ---- mixture of experts ---------------------------------------------------------------------------------
namespace {

bool is_float(uint32_t type) { return type == GGQ_TYPE_F16 || type == GGQ_TYPE_BF16; }
// rows of 16-bit floats that are shorter than a piece of an image
bool short_rows(uint32_t type, uint64_t cols) { return is_float(type) && cols < 8; }

uint64_t up256(uint64_t v) { return (v + 255) & ~255ull; }

ggq_status check_moe(const ggq_moe *m, uint64_t tokens) {
    if (!m) return GGQ_INVALID;
    uint32_t kind, bytes;
    const uint64_t ub = ggq_block_elems(m->up_type), db = ggq_block_elems(m->down_type);
    if (!ub || !db || !elem_kind(m->router_type, &kind, &bytes)) return GGQ_UNSUPPORTED;
    if (m->hidden >= MAX_COLS || m->ff >= MAX_COLS || m->hidden == 0 || m->ff == 0) return GGQ_INVALID;
    if (m->hidden % ub != 0 || m->ff % db != 0) return GGQ_INDIVISIBLE;
    if (m->experts == 0 || m->experts > GGQ_MOE_MAX_EXPERTS || m->top_k == 0 || m->top_k > m->experts || m->top_k > GGQ_MOE_MAX_TOP_K)
        return GGQ_INVALID;
    if (m->reserved || m->gating > 1 || m->normalize > 1 || m->activation > 1) return GGQ_INVALID;
    if (tokens > GGQ_MOE_MAX_TOKENS) return GGQ_TOO_LARGE;
    return GGQ_OK;
}

// byte offsets of the workspace's parts
struct MoeSpace {
    uint64_t ids, weights, table, h, o, end;
    MoeSpace(const ggq_moe &m, uint64_t tokens) {
        ids = up256(4 * tokens * m.experts);
        weights = ids + up256(4 * tokens * m.top_k);
        table = weights + up256(4 * tokens * m.top_k);
        h = table + up256(sizeof(Slot) * tokens * m.top_k);
        o = h + up256(4 * tokens * m.top_k * m.ff);
        end = o + up256(4 * tokens * m.top_k * m.hidden);
    }
};

}  // namespace

extern "C" {

ggq_status ggq_matvec_device(uint32_t ty, uint64_t rows, uint64_t cols, const void *d_w, uint32_t x_type, const void *d_x,
                             uint64_t x_stride, uint64_t tokens, uint32_t y_type, void *d_y, uint64_t y_stride,
                             void *hip_stream) {
    MatvecArgs a{};
    uint32_t xb, yb;
    const uint64_t be = ggq_block_elems(ty);
    if (be == 0 || !elem_kind(x_type, &a.x_kind, &xb) || !elem_kind(y_type, &a.y_kind, &yb)) return GGQ_UNSUPPORTED;
    if (cols % be != 0) return GGQ_INDIVISIBLE;
    if (rows >= MAX_DIM || cols >= MAX_COLS || tokens >= MAX_DIM) return GGQ_INVALID;
    if (!strides_ok(y_stride, rows, tokens) || x_stride >= (1ull << 40)) return GGQ_INVALID;
    if (rows == 0 || tokens == 0) return GGQ_OK;
    if (!d_y || (cols && (!d_w || !d_x))) return GGQ_INVALID;
    if ((uintptr_t)d_y % yb != 0 || (uintptr_t)d_x % xb != 0) return GGQ_MISALIGNED;
    a.w = (const uint8_t *)d_w;
    a.rows = rows;
    a.cols = cols;
    a.x_stride = x_stride;
    a.y_stride = y_stride;
    hipStream_t st = (hipStream_t)hip_stream;
    for (uint64_t t = 0, done = 0; t < tokens; t += done) {
        a.x = (const uint8_t *)d_x + t * x_stride * xb;
        a.y = (uint8_t *)d_y + t * y_stride * yb;
        if (cols == 0) {
            done = a.tokens = (uint32_t)std::min<uint64_t>(4, tokens - t);
            fill_zero<<<(uint32_t)((rows + MV_THREADS - 1) / MV_THREADS), MV_THREADS, 0, st>>>(a);
            continue;
        }
#define CASE(F) done = Launch<F>::matvec(a, tokens - t, st)
        GGQ_FOR_TYPE(ty, CASE)
#undef CASE
    }
    HIP_TRY(hipGetLastError());
    return GGQ_OK;
}

ggq_status ggq_get_rows_device(uint32_t ty, uint64_t rows, uint64_t cols, const void *d_w, uint32_t id_type,
                               const void *d_ids, uint64_t n, uint32_t y_type, void *d_y, uint64_t y_stride,
                               void *hip_stream) {
    RowsArgs a{};
    uint32_t y_kind, yb;
    const uint64_t be = ggq_block_elems(ty);
    const uint32_t idb = id_type == 26 ? 4 : id_type == 27 ? 8 : 0;     // GGmlType I32, I64
    if (be == 0 || idb == 0 || !elem_kind(y_type, &y_kind, &yb)) return GGQ_UNSUPPORTED;
    if (cols % be != 0) return GGQ_INDIVISIBLE;
    if (rows >= MAX_DIM || cols >= MAX_COLS || n >= MAX_DIM || !strides_ok(y_stride, cols, n)) return GGQ_INVALID;
    if (cols == 0 || n == 0) return GGQ_OK;
    if (!d_y || !d_ids || (rows && !d_w)) return GGQ_INVALID;
    if ((uintptr_t)d_y % yb != 0 || (uintptr_t)d_ids % idb != 0) return GGQ_MISALIGNED;
    a.w = (const uint8_t *)d_w;
    a.ids = d_ids;
    a.y = d_y;
    a.rows = rows;
    a.cols = cols;
    a.n = n;
    a.y_stride = y_stride;
    a.row_bytes = cols / be * ggq_block_bytes(ty);
    a.wide_ids = idb == 8;
    for (; a.first < n; a.first += MAX_GRID_Y) {
        const uint32_t now = (uint32_t)std::min<uint64_t>(MAX_GRID_Y, n - a.first);
#define CASE(F) Launch<F>::rows(a, y_kind, now, (hipStream_t)hip_stream)
        GGQ_FOR_TYPE(ty, CASE)
#undef CASE
    }
    HIP_TRY(hipGetLastError());
    return GGQ_OK;
}

// ---- mixture of experts ---------------------------------------------------------------------------------
ggq_status ggq_moe_workspace_bytes(const ggq_moe *m, uint64_t tokens, size_t *bytes_out) {
    const ggq_status st = check_moe(m, tokens);
    if (st != GGQ_OK) return st;
    if (!bytes_out) return GGQ_INVALID;
    *bytes_out = tokens ? MoeSpace(*m, tokens).end : 0;
    return GGQ_OK;
}

ggq_status ggq_moe_device(const ggq_moe *m, uint32_t x_type, const void *d_x, uint64_t x_stride, uint64_t tokens,
                          uint32_t y_type, void *d_y, uint64_t y_stride, int32_t *d_ids, float *d_weights,
                          void *d_workspace, size_t workspace_bytes, void *hip_stream) {
    ggq_status rc = check_moe(m, tokens);
    if (rc != GGQ_OK) return rc;
    MoeArgs a{};
    uint32_t xb, yb, rb;
    if (!elem_kind(x_type, &a.x_kind, &xb) || !elem_kind(y_type, &a.y_kind, &yb)) return GGQ_UNSUPPORTED;
    elem_kind(m->router_type, &a.router_kind, &rb);
    if (!strides_ok(y_stride, m->hidden, tokens) || x_stride >= (1ull << 40)) return GGQ_INVALID;
    if (tokens == 0) return GGQ_OK;
    const MoeSpace ws(*m, tokens);
    if (!d_x || !d_y || !m->d_router || !m->d_gate || !m->d_up || !m->d_down || !d_workspace || workspace_bytes < ws.end) return GGQ_INVALID;
    if ((uintptr_t)d_x % xb || (uintptr_t)d_y % yb || (uintptr_t)m->d_router % rb || (uintptr_t)d_workspace % 256 ||
        (uintptr_t)d_ids % 4 || (uintptr_t)d_weights % 4)
        return GGQ_MISALIGNED;
    uint8_t *space = (uint8_t *)d_workspace;
    a.gate = (const uint8_t *)m->d_gate;
    a.up = (const uint8_t *)m->d_up;
    a.down = (const uint8_t *)m->d_down;
    a.router = m->d_router;
    a.x = d_x;
    a.y = d_y;
    a.logits = (float *)space;
    a.ids = (int32_t *)(space + ws.ids);
    a.weights = (float *)(space + ws.weights);
    a.table = (Slot *)(space + ws.table);
    a.h = (float *)(space + ws.h);
    a.o = (float *)(space + ws.o);
    a.out_ids = d_ids;
    a.out_weights = d_weights;
    a.hidden = m->hidden;
    a.ff = m->ff;
    a.x_stride = x_stride;
    a.y_stride = y_stride;
    a.tokens = (uint32_t)tokens;
    a.experts = m->experts;
    a.top_k = m->top_k;
    a.sigmoid = m->gating;
    a.normalize = m->normalize;
    a.gelu = m->activation;
    a.scale = m->scale;
    hipStream_t st = (hipStream_t)hip_stream;
    if (tokens == 1) moe_logits<1><<<m->experts, MV_THREADS, 0, st>>>(a);
    else moe_logits<LOGIT_TOKENS><<<dim3(m->experts, ((uint32_t)tokens + LOGIT_TOKENS - 1) / LOGIT_TOKENS), MV_THREADS, 0, st>>>(a);
    // groups of pairs with the same expert: one for each pair, or one for each expert and one more for each slot_tokens pairs.
    // Shared memory is kept for as many tokens: where experts have four on average, or fewer, more than eight are rare (128
    // experts, 8 chosen, 2048/768 by 16 tokens: 102 us, with room for 16 110).
    const uint32_t pairs = (uint32_t)tokens * m->top_k, in_use = std::min(m->experts, pairs);
    a.slot_tokens = std::min((uint32_t)tokens, pairs > 4 * m->experts ? SLOT_TOKENS : SLOT_TOKENS / 2);
    a.slots = std::min(pairs, in_use + (pairs - in_use) / a.slot_tokens);
    double unused = 1.0;
    for (uint64_t t = 0; t < tokens; ++t) unused *= 1.0 - (double)m->top_k / m->experts;
    a.slots_expected = std::max(1u, std::min(a.slots, (uint32_t)(m->experts * (1.0 - unused) + 0.5)));
    // one token of packed codes: the kernel of gate and up makes the choice
    if (tokens > 1 || is_float(m->up_type) || is_float(m->down_type)) moe_route<<<1, ROUTE_WAVES * 64, 0, st>>>(a);
#define CASE(F) Launch<F>::up(a, st)
    GGQ_FOR_TYPE(m->up_type, CASE)
#undef CASE
#define CASE(F) Launch<F>::down(a, st)
    GGQ_FOR_TYPE(m->down_type, CASE)
#undef CASE
    if ((tokens > 1 || is_float(m->down_type)) && !short_rows(m->down_type, m->ff))
        moe_sum<<<dim3((uint32_t)((a.hidden + MV_THREADS - 1) / MV_THREADS), a.tokens), MV_THREADS, 0, st>>>(a);
    HIP_TRY(hipGetLastError());
    return GGQ_OK;
}

}  // extern "C"
