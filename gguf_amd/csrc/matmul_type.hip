// matmul_type.hip -- the launches of the products with packed weights for one block type: compiled once for each, with
// GGQ_FORMAT its struct in formats.h, so that they build side by side.
#include "launch.h"
#include "moe.h"

#include <algorithm>

namespace ggq {
namespace {

// Workgroups of one launch: the grid's threads are counted in 32 bits
constexpr uint64_t MAX_GRID = 1ull << 22;
// Shared memory of one workgroup for one token's x, beside its waves' images.  Less means more chunks, more fewer workgroups on a
// CU: with 32 / 64 / 128 KiB q4_k 28672 x 8192 by an f32 token takes 28.2 / 26.8 / 31.3 us, a layer of 64 experts, 8 chosen,
// 2048/1024 24.2 / 20.7 / 20.1.
constexpr uint32_t X_LDS = 64 << 10;
// ... of one workgroup for several tokens: what a CU has, less the kernel's own
constexpr uint32_t DENSE_LDS = 152 << 10;

// ... of one workgroup in all, so that two fit a CU.  Where there are more of them than CUs and shorter chunks are enough for that,
// those are taken: q5_0 11008 x 4096 11.3 instead of 13.5 us, q2_k 28672 x 8192 25.0 instead of 31.1.  With one workgroup for a CU
// they only cost: q5_0 8192 x 28672 45 instead of 38 us.
constexpr uint32_t HALF_CU = 80 << 10;

// The shape of a launch over `tiles` wave tiles, each of which takes `turns` turns: how many waves share a tile's turns,
// the turns staged at a time (equal chunks, whole rounds of the waves), the shared memory.
struct Shape {
    uint32_t ksplit = 1, groups;
    bool two;             // more workgroups than CUs
    // `waves`: of a workgroup that may share a tile's turns; x_bytes: shared memory of a turn of x
    Shape(uint64_t tiles, uint32_t turns, uint32_t waves, uint32_t x_bytes) {
        // few rows: the columns are shared out, until there are 8 waves for each of 256 CUs (up to 32: q6_k 32000 x 4096 32.4
        // instead of 26.8 us, q4_k 28672 x 8192 36.5 instead of 26.8; up to 16: the same within 1 % for all that were tried)
        while (ksplit < waves && ksplit < turns && tiles * ksplit < 2048 && 2 * ksplit * x_bytes <= X_LDS) ksplit *= 2;
        groups = waves / ksplit;
        two = tiles * ksplit > 256 * TILE_WAVES;
    }
    template <class M> uint32_t chunk(uint32_t turns) const {
        const uint32_t each = M::X_BYTES * ksplit, rounds = (turns + ksplit - 1) / ksplit, own = TILE_WAVES * M::WAVE_BYTES + M::CLEAR;
        auto in_chunks = [&](uint32_t most) { const uint32_t chunks = (rounds + most - 1) / most; return (rounds + chunks - 1) / chunks; };
        uint32_t take = in_chunks(std::max(1u, X_LDS / each));
        if (two && own + take * each > HALF_CU && own + each <= HALF_CU) take = in_chunks((HALF_CU - own) / each);
        return take * ksplit;
    }
    template <class M> uint32_t bytes(uint32_t turns) const {
        return TILE_WAVES * M::WAVE_BYTES + M::CLEAR + std::max<uint32_t>(std::min(chunk<M>(turns), turns) * M::X_BYTES, TILE_WAVES * M::ROWS * 4);
    }
};
template <class M> constexpr uint32_t turns_of(uint64_t cols) { return (uint32_t)((cols + M::ELEMS - 1) / M::ELEMS); }

template <class F, class M>
uint64_t launch_tiles(MatvecArgs a, hipStream_t st) {
    const uint64_t tiles = (a.rows + M::ROWS - 1) / M::ROWS;
    const uint32_t turns = turns_of<M>(a.cols);
    const Shape sh(tiles, turns, TILE_WAVES, M::X_BYTES);
    a.ksplit = sh.ksplit;
    a.chunk = sh.chunk<M>(turns);
    for (a.first_tile = 0; a.first_tile < tiles; a.first_tile += MAX_GRID * sh.groups) {
        const dim3 grid((uint32_t)std::min<uint64_t>(MAX_GRID, (tiles - a.first_tile + sh.groups - 1) / sh.groups));
        matvec_tiles<F, M><<<grid, TILE_THREADS, sh.bytes<M>(turns), st>>>(a);
    }
    return 1;
}

// Waves that share the columns of R tiles: no more than `most`, or turns, or fit; all with as many turns or one less.
template <class M>
uint32_t dense_waves(uint32_t most, uint32_t turns, uint32_t tokens) {
    most = std::min(std::min(most, turns), DENSE_LDS / M::wave_bytes(tokens));
    const uint32_t rounds = (turns + most - 1) / most;
    return (turns + rounds - 1) / rounds;
}
// How a dense product is cut: R tiles of rows for a workgroup, waves that share their columns.
struct DenseCut {
    uint64_t cost = ~0ull;
    uint32_t R = 0, waves = 0;
    // `groups`: of waves that share columns.  They run in rounds of what 256 CUs hold; in each, waves take their turns, whose x
    // costs as much as half a tile, and what a tile takes to begin and end; some of the work of a CU and of a SIMD is not hidden
    // by that, and a wave has a price.  The weights were fitted to nine ways to cut each of eight products (4096 x 4096 to
    // 32000 x 4096, 4 to 16 tokens, two types of x, three block types) and three or four of four MoE products: the way with the
    // least cost is the fastest of them, or within 8 %.  q6_k 32000 x 4096 by 16 tokens: 37 us with two tiles and two waves, 48
    // with three and eight; 11008 x 4096: 29 and 16.
    template <class M>
    void consider(uint64_t groups, uint32_t turns, uint32_t tokens) {
        for (uint32_t most = TILE_WAVES; most; most /= 2) {
            const uint32_t w = dense_waves<M>(most, turns, tokens), turn = 2 * M::TILES + 1, each = (turns + w - 1) / w * turn;
            const uint32_t fit = std::max(1u, std::min<uint32_t>(dense_waves_per_cu(M::TILES) / w, DENSE_LDS / (w * M::wave_bytes(tokens))));
            const uint64_t of_cu = (groups + 255) / 256, rounds = (of_cu + fit - 1) / fit, of_simd = (of_cu * w + 3) / 4;
            const uint64_t c = rounds * (160 * each + 320) + of_simd * each * 40 + of_cu * (turns * turn * 5 + w * 16);
            if (c < cost) cost = c, R = M::TILES, waves = w;
        }
    }
};
template <class F, int X, int R>
void launch_dense_tiles(MatvecArgs a, uint64_t tiles, uint32_t waves, hipStream_t st) {
    typedef DenseTile<F, X, R> M;
    static_assert(M::wave_bytes(M::TOKENS) <= DENSE_LDS, "a wave's shared memory");
    for (a.first_tile = 0; a.first_tile < tiles; a.first_tile += MAX_GRID * R) {
        const uint32_t grid = (uint32_t)std::min<uint64_t>(MAX_GRID, (tiles - a.first_tile + R - 1) / R);
        matvec_dense<F, X, R><<<grid, waves * 64, waves * M::wave_bytes(a.tokens), st>>>(a);
    }
}
template <class F, int X>
uint64_t launch_dense(MatvecArgs a, uint64_t tokens, hipStream_t st) {
    a.tokens = (uint32_t)std::min<uint64_t>(tokens, 16);
    const uint64_t tiles = (a.rows + 15) / 16;
    const uint32_t turns = (uint32_t)((a.cols + 255) / 256);
    DenseCut cut;
    cut.consider<DenseTile<F, X, 1>>(tiles, turns, a.tokens);
    cut.consider<DenseTile<F, X, 2>>((tiles + 1) / 2, turns, a.tokens);
    cut.consider<DenseTile<F, X, 3>>((tiles + 2) / 3, turns, a.tokens);
    if (cut.R == 1) launch_dense_tiles<F, X, 1>(a, tiles, cut.waves, st);
    else if (cut.R == 2) launch_dense_tiles<F, X, 2>(a, tiles, cut.waves, st);
    else launch_dense_tiles<F, X, 3>(a, tiles, cut.waves, st);
    return a.tokens;
}

}  // namespace

// One token is left to the digits, which need fewer instructions: q4_k 28672 x 8192 26.8 us (as several tokens 33.1 by bf16 x, 59 by
// f32), 11008 x 4096 9.1 (9.6, 13.1), q6_k 32000 x 4096 24.5 (29.4, 44.5).  Few rows with long columns are slower so by 16-bit x
// (q4_k 8192 x 28672 31.7, 30.8; 4096 x 11008 10.6, 8.4), but not for all types (q4_0 1024 x 8192 6.8, 7.9).  One launch over the
// first of the tokens.  Returns how many it takes.
template <class F>
uint64_t Launch<F>::matvec(MatvecArgs a, uint64_t tokens, hipStream_t st) {
    if constexpr (is_float_type<F>) {
        if (a.cols < 8) {
            a.tokens = (uint32_t)std::min<uint64_t>(tokens, 64);
            matvec_short<F><<<(uint32_t)((a.rows + MV_THREADS - 1) / MV_THREADS), MV_THREADS, 0, st>>>(a);
            return a.tokens;
        }
        if (tokens == 1) {
            if (a.x_kind == EK_BF16) return launch_tiles<F, FloatTile<F, 1>>(a, st);
            if (a.x_kind == EK_F16) return launch_tiles<F, FloatTile<F, 2>>(a, st);
            return launch_tiles<F, FloatTile<F, 3>>(a, st);
        }
    } else if (tokens == 1) {
        return launch_tiles<F, CodeTile<F>>(a, st);
    }
    if (a.x_kind == EK_BF16) return launch_dense<F, X_BF16>(a, tokens, st);
    if (a.x_kind == EK_F16) return launch_dense<F, X_F16>(a, tokens, st);
    return launch_dense<F, X_F32>(a, tokens, st);
}

template <class F, class O>
void launch_rows_as(const RowsArgs &a, uint32_t n, hipStream_t st) {
    const uint64_t piece = WG_THREADS * STORES_PER_THREAD * O::EPL;
    get_rows<F, O><<<dim3((uint32_t)((a.cols + piece - 1) / piece), n), WG_THREADS, 0, st>>>(a);
}
template <class F>
void Launch<F>::rows(const RowsArgs &a, uint32_t y_kind, uint32_t n, hipStream_t st) {
    if (y_kind == EK_F32) launch_rows_as<F, OutF32>(a, n, st);
    else if (y_kind == EK_F16) launch_rows_as<F, OutF16>(a, n, st);
    else launch_rows_as<F, OutBF16>(a, n, st);
}

// ---- mixture of experts ---------------------------------------------------------------------------------
namespace {
// one token
template <class F, class M>
void launch_up(MoeArgs a, hipStream_t st) {
    const uint32_t tiles = (uint32_t)((a.ff + M::ROWS - 1) / M::ROWS), turns = turns_of<M>(a.hidden);
    const Shape sh(2 * (uint64_t)tiles * a.top_k, turns, TILE_WAVES / 2, M::X_BYTES);
    a.ksplit = sh.ksplit;
    a.chunk = sh.chunk<M>(turns);
    moe_up<F, M><<<dim3((tiles + sh.groups - 1) / sh.groups, a.top_k), TILE_THREADS, sh.bytes<M>(turns), st>>>(a);
}
template <class F, int X>
void launch_up_dense(MoeArgs a, hipStream_t st) {
    typedef DenseTile<F, X, 2> M;
    const uint32_t tiles = (uint32_t)((a.ff + 15) / 16);
    DenseCut cut;
    cut.consider<M>((uint64_t)tiles * a.slots_expected, turns_of<M>(a.hidden), a.slot_tokens);
    moe_up_dense<F, X><<<dim3(tiles, a.slots), cut.waves * 64, cut.waves * M::wave_bytes(a.slot_tokens), st>>>(a);
}
template <class F, int X>
void launch_down_dense(MoeArgs a, hipStream_t st) {
    typedef DenseTile<F, X, DOWN_TILES> M;
    const uint32_t tiles = (uint32_t)((a.hidden + 16 * DOWN_TILES - 1) / (16 * DOWN_TILES));
    DenseCut cut;
    cut.consider<M>((uint64_t)tiles * a.slots_expected, turns_of<M>(a.ff), a.slot_tokens);
    moe_down_dense<F, X><<<dim3(tiles, a.slots), cut.waves * 64, cut.waves * M::wave_bytes(a.slot_tokens), st>>>(a);
}
template <class F, class M>
void launch_down_one(MoeArgs a, hipStream_t st) {
    const uint32_t tiles = (uint32_t)((a.hidden + M::ROWS - 1) / M::ROWS), turns = turns_of<M>(a.ff) * a.top_k;
    const Shape sh(tiles, turns, TILE_WAVES, M::X_BYTES);
    a.ksplit = sh.ksplit;
    a.chunk = sh.chunk<M>(turns);
    moe_down_one<F, M><<<(tiles + sh.groups - 1) / sh.groups, TILE_THREADS, sh.bytes<M>(turns), st>>>(a);
}
}  // namespace

template <class F>
void Launch<F>::up(MoeArgs a, hipStream_t st) {
    if constexpr (is_float_type<F>) {
        if (a.hidden < 8) {
            moe_up_short<F><<<dim3((uint32_t)((a.ff + MV_THREADS - 1) / MV_THREADS), a.tokens * a.top_k), MV_THREADS, 0, st>>>(a);
            return;
        }
    } else if (a.tokens == 1) {
        launch_up<F, CodeTile<F>>(a, st);
        return;
    }
    if (a.x_kind == EK_BF16) launch_up_dense<F, X_BF16>(a, st);
    else if (a.x_kind == EK_F16) launch_up_dense<F, X_F16>(a, st);
    else launch_up_dense<F, X_F32>(a, st);
}

template <class F>
void Launch<F>::down(MoeArgs a, hipStream_t st) {
    if constexpr (is_float_type<F>) {
        if (a.ff < 8) {
            moe_down_short<F><<<dim3((uint32_t)((a.hidden + MV_THREADS - 1) / MV_THREADS), a.tokens), MV_THREADS, 0, st>>>(a);
            return;
        }
    } else if (a.tokens == 1) {
        launch_down_one<F, CodeTile<F>>(a, st);
        return;
    }
    launch_down_dense<F, X_F32>(a, st);
}

template struct Launch<GGQ_FORMAT>;

}  // namespace ggq
