// matmul.hip -- entry points of the products with packed weights (include/ggq.h): argument checks and launches.
#include "../../include/ggq.h"
#include "internal.h"
#include "dense.h"
#include "matmul.h"
#include "moe.h"

#include <algorithm>

using namespace ggq;

namespace {

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
// Columns: eight packed rows of any type are within 32-bit offsets.
constexpr uint64_t MAX_COLS = 1ull << 26;
// Workgroups of one launch: the grid's threads are counted in 32 bits
constexpr uint64_t MAX_GRID = 1ull << 22;
// ... and along y
constexpr uint64_t MAX_GRID_Y = 65535;

bool strides_ok(uint64_t stride, uint64_t width, uint64_t tokens) {
    return stride < (1ull << 40) && (tokens <= 1 || stride >= width);
}

// Shared memory of one workgroup for x, beside its waves' images.
constexpr uint32_t X_LDS = 64 << 10;

// The shape of a launch over `tiles` wave tiles, each of which takes `turns` turns: how many waves share a tile's turns,
// the turns staged at a time (equal chunks, whole rounds of the waves), the shared memory.
struct Shape {
    uint32_t ksplit = 1, groups;
    // `waves`: of a workgroup that may share a tile's turns; x_bytes: shared memory of a turn of x
    Shape(uint64_t tiles, uint32_t turns, uint32_t waves, uint32_t x_bytes) {
        // few rows: the columns are shared out, until there are 8 waves for each of 256 CUs
        while (ksplit < waves && ksplit < turns && tiles * ksplit < 2048 && 2 * ksplit * x_bytes <= X_LDS) ksplit *= 2;
        groups = waves / ksplit;
    }
    template <class M> uint32_t chunk(uint32_t turns) const {
        const uint32_t rounds = (turns + ksplit - 1) / ksplit, most = std::max(1u, X_LDS / (M::X_BYTES * ksplit)), chunks = (rounds + most - 1) / most;
        return (rounds + chunks - 1) / chunks * ksplit;
    }
    template <class M> uint32_t bytes(uint32_t turns) const {
        return TILE_WAVES * M::WAVE_BYTES + M::CLEAR + std::max<uint32_t>(std::min(chunk<M>(turns), turns) * M::X_BYTES, TILE_WAVES * M::TOKENS * M::ROWS * 4);
    }
};
template <class M> constexpr uint32_t turns_of(uint64_t cols) { return (uint32_t)((cols + M::ELEMS - 1) / M::ELEMS); }

template <class F, class M>
uint64_t launch_tiles(MatvecArgs a, uint64_t tokens, hipStream_t st) {
    a.tokens = (uint32_t)std::min<uint64_t>(tokens, M::TOKENS);
    const uint64_t tiles = (a.rows + M::ROWS - 1) / M::ROWS;
    const uint32_t turns = turns_of<M>(a.cols);
    const Shape sh(tiles, turns, TILE_WAVES, M::X_BYTES);
    a.ksplit = sh.ksplit;
    a.chunk = sh.chunk<M>(turns);
    for (a.first_tile = 0; a.first_tile < tiles; a.first_tile += MAX_GRID * sh.groups) {
        const dim3 grid((uint32_t)std::min<uint64_t>(MAX_GRID, (tiles - a.first_tile + sh.groups - 1) / sh.groups));
        matvec_tiles<F, M><<<grid, TILE_THREADS, sh.bytes<M>(turns), st>>>(a);
    }
    return a.tokens;
}

// x is taken to 16 bits below an element, or the largest of 32, where the result is rounded to a 16-bit float anyway.
bool to_16_bits(uint32_t x_kind, uint32_t y_kind) { return x_kind != EK_F32 && y_kind != EK_F32; }

// One launch over the first of the tokens.  Returns how many it takes.
template <class F>
uint64_t launch_some(MatvecArgs a, uint64_t tokens, hipStream_t st) {
    if constexpr (is_float_type<F>) {
        if (a.cols < 8) {
            a.tokens = (uint32_t)std::min<uint64_t>(tokens, 64);
            matvec_short<F><<<(uint32_t)((a.rows + MV_THREADS - 1) / MV_THREADS), MV_THREADS, 0, st>>>(a);
            return a.tokens;
        }
        if (tokens == 1) {
            if (a.x_kind == EK_BF16) return launch_tiles<F, FloatTile<F, 1>>(a, 1, st);
            if (a.x_kind == EK_F16) return launch_tiles<F, FloatTile<F, 2>>(a, 1, st);
            return launch_tiles<F, FloatTile<F, 3>>(a, 1, st);
        }
    } else if (tokens == 1) {
        return to_16_bits(a.x_kind, a.y_kind) ? launch_tiles<F, CodeTile<F, 1>>(a, 1, st) : launch_tiles<F, CodeTile<F, 2>>(a, 1, st);
    }
    if (a.x_kind == EK_BF16) return launch_tiles<F, DenseTile<F, 1>>(a, tokens, st);
    if (a.x_kind == EK_F16) return launch_tiles<F, DenseTile<F, 2>>(a, tokens, st);
    return launch_tiles<F, DenseTile<F, 3>>(a, tokens, st);
}

template <class F, class O>
void launch_rows_as(const RowsArgs &a, uint32_t n, hipStream_t st) {
    const uint64_t piece = WG_THREADS * STORES_PER_THREAD * O::EPL;
    get_rows<F, O><<<dim3((uint32_t)((a.cols + piece - 1) / piece), n), WG_THREADS, 0, st>>>(a);
}
template <class F>
void launch_rows(const RowsArgs &a, uint32_t y_kind, uint32_t n, hipStream_t st) {
    if (y_kind == EK_F32) launch_rows_as<F, OutF32>(a, n, st);
    else if (y_kind == EK_F16) launch_rows_as<F, OutF16>(a, n, st);
    else launch_rows_as<F, OutBF16>(a, n, st);
}

}  // namespace

// ---- mixture of experts ---------------------------------------------------------------------------------
namespace {

// rows of 16-bit floats that are shorter than a piece of an image
bool short_rows(uint32_t type, uint64_t cols) { return (type == GGQ_TYPE_F16 || type == GGQ_TYPE_BF16) && cols < 8; }

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
    uint64_t ids, weights, h, o, end;
    MoeSpace(const ggq_moe &m, uint64_t tokens) {
        ids = up256(4 * tokens * m.experts);
        weights = ids + up256(4 * tokens * m.top_k);
        h = weights + up256(4 * tokens * m.top_k);
        o = h + up256(4 * tokens * m.top_k * m.ff);
        end = o + (tokens > 4 ? up256(4 * tokens * m.top_k * m.hidden) : 0);
    }
};

// One: the tile of experts with one token, Many: of the others
template <class F, class One, class Many>
void launch_up(MoeArgs a, hipStream_t st) {
    const uint32_t tiles = (uint32_t)((a.ff + Many::ROWS - 1) / Many::ROWS);
    static_assert(One::ROWS == Many::ROWS, "one grid for both");
    const uint32_t one = turns_of<One>(a.hidden), many = turns_of<Many>(a.hidden);
    const Shape sh(2 * (uint64_t)tiles * a.slots, std::min(one, many), TILE_WAVES / 2, std::max(One::X_BYTES, Many::X_BYTES));
    a.ksplit = sh.ksplit;
    a.chunk_one = sh.chunk<One>(one);
    a.chunk = sh.chunk<Many>(many);
    moe_up<F, One, Many><<<dim3((tiles + sh.groups - 1) / sh.groups, a.slots), TILE_THREADS, std::max(sh.bytes<One>(one), sh.bytes<Many>(many)), st>>>(a);
}

template <class F>
void launch_up_of(MoeArgs a, hipStream_t st) {
    if constexpr (is_float_type<F>) {
        if (a.hidden < 8) {
            moe_up_short<F><<<dim3((uint32_t)((a.ff + MV_THREADS - 1) / MV_THREADS), a.tokens * a.top_k), MV_THREADS, 0, st>>>(a);
        } else if (a.x_kind == EK_BF16) {
            launch_up<F, DenseTile<F, 1>, DenseTile<F, 1>>(a, st);
        } else if (a.x_kind == EK_F16) {
            launch_up<F, DenseTile<F, 2>, DenseTile<F, 2>>(a, st);
        } else {
            launch_up<F, DenseTile<F, 3>, DenseTile<F, 3>>(a, st);
        }
    } else if (a.tokens == 1) {
        if (to_16_bits(a.x_kind, a.y_kind)) launch_up<F, CodeTile<F, 1>, CodeTile<F, 1>>(a, st);
        else launch_up<F, CodeTile<F, 2>, CodeTile<F, 2>>(a, st);
    } else {
        if (a.x_kind == EK_BF16) launch_up<F, CodeTile<F, 2>, DenseTile<F, 1>>(a, st);
        else if (a.x_kind == EK_F16) launch_up<F, CodeTile<F, 2>, DenseTile<F, 2>>(a, st);
        else launch_up<F, CodeTile<F, 2>, DenseTile<F, 3>>(a, st);
    }
}

template <class F, class M>
void launch_down_few(MoeArgs a, hipStream_t st) {
    const uint32_t tiles = (uint32_t)((a.hidden + M::ROWS - 1) / M::ROWS), turns = turns_of<M>(a.ff) * a.tokens * a.top_k;
    const Shape sh(tiles, turns, TILE_WAVES, M::X_BYTES);
    a.ksplit = sh.ksplit;
    a.chunk = sh.chunk<M>(turns);
    moe_down_few<F, M><<<(tiles + sh.groups - 1) / sh.groups, TILE_THREADS, sh.bytes<M>(turns), st>>>(a);
}

template <class F, class One, class Many>
void launch_down_many(MoeArgs a, hipStream_t st) {
    const uint32_t tiles = (uint32_t)((a.hidden + Many::ROWS - 1) / Many::ROWS), one = turns_of<One>(a.ff), many = turns_of<Many>(a.ff);
    const Shape sh((uint64_t)tiles * a.slots, std::min(one, many), TILE_WAVES, std::max(One::X_BYTES, Many::X_BYTES));
    a.ksplit = sh.ksplit;
    a.chunk_one = sh.chunk<One>(one);
    a.chunk = sh.chunk<Many>(many);
    moe_down_many<F, One, Many><<<dim3((tiles + sh.groups - 1) / sh.groups, a.slots), TILE_THREADS, std::max(sh.bytes<One>(one), sh.bytes<Many>(many)), st>>>(a);
    moe_sum<<<dim3((uint32_t)((a.hidden + MV_THREADS - 1) / MV_THREADS), a.tokens), MV_THREADS, 0, st>>>(a);
}

template <class F>
void launch_down_of(MoeArgs a, hipStream_t st) {
    if constexpr (is_float_type<F>) {
        if (a.ff < 8) {
            moe_down_short<F><<<dim3((uint32_t)((a.hidden + MV_THREADS - 1) / MV_THREADS), a.tokens), MV_THREADS, 0, st>>>(a);
        } else if (a.tokens <= 4) {
            launch_down_few<F, DenseTile<F, 3>>(a, st);
        } else {
            launch_down_many<F, DenseTile<F, 3>, DenseTile<F, 3>>(a, st);
        }
    } else if (to_16_bits(a.x_kind, a.y_kind)) {
        if (a.tokens == 1) launch_down_few<F, CodeTile<F, 1>>(a, st);
        else if (a.tokens <= 4) launch_down_few<F, DenseTile<F, 2>>(a, st);
        else launch_down_many<F, CodeTile<F, 1>, DenseTile<F, 2>>(a, st);
    } else {
        if (a.tokens == 1) launch_down_few<F, CodeTile<F, 2>>(a, st);
        else if (a.tokens <= 4) launch_down_few<F, DenseTile<F, 3>>(a, st);
        else launch_down_many<F, CodeTile<F, 2>, DenseTile<F, 3>>(a, st);
    }
}

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
#define CASE(F) done = launch_some<F>(a, tokens - t, st)
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
#define CASE(F) launch_rows<F>(a, y_kind, now, (hipStream_t)hip_stream)
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
    moe_logits<<<dim3(m->experts, ((uint32_t)tokens + LOGIT_TOKENS - 1) / LOGIT_TOKENS), MV_THREADS, 0, st>>>(a);
    // Comparing each expert with each is on every workgroup's way; the launch that it saves takes about 2.5 us.
    a.choose = tokens <= CHOOSE_TOKENS && m->experts <= 128 && !short_rows(m->up_type, m->hidden);
    if (!a.choose) moe_route<<<(uint32_t)tokens, MV_THREADS, 0, st>>>(a);
    // groups of up to 16 pairs with the same expert: one for each pair, or one for each expert and one more for each 16 pairs
    const uint32_t pairs = (uint32_t)tokens * m->top_k, in_use = std::min(m->experts, pairs);
    a.slots = std::min(pairs, in_use + (pairs - in_use) / SLOT_TOKENS);
#define CASE(F) launch_up_of<F>(a, st)
    GGQ_FOR_TYPE(m->up_type, CASE)
#undef CASE
#define CASE(F) launch_down_of<F>(a, st)
    GGQ_FOR_TYPE(m->down_type, CASE)
#undef CASE
    HIP_TRY(hipGetLastError());
    return GGQ_OK;
}

}  // extern "C"
