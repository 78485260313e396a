// moe.h -- a mixture-of-experts layer with packed experts, for few tokens.
//
//     l = router x;  the top_k experts of each token;  h_e = act(gate_e x) * (up_e x);  y = sum of w_e down_e h_e
//
// One token: the logits; gate and up, whose workgroups find the choice themselves; down, with the sum over the experts in it.
// Several: the logits; the choice and the table of slots (route.h); gate and up, slot by slot; down, slot by slot; the sum.
// An expert's bytes are read once for each slot: for up to 16 of its tokens, or 8.
//
// Bound, for one token and large experts, by the bytes of the experts in use and by x, which each workgroup turns into digits (8
// experts, 2 chosen, 4096/11008: gate and up 101 MB in 27 us, down 74 MB in 24.7; 344 and 256 workgroups for 256 CUs); for small
// ones by the time that three launches take to begin and end (64, 8, 2048/1024: 20.6 us for 29 MB); for several tokens by the
// instructions that unpack (128, 8, 2048/768 by 16 tokens: 102 us for 235 MB, vector units busy for 51 and 65 % of gate / up and down).
#pragma once
#include "choice.h"
#include "dense.h"

namespace ggq {

// SiLU, or GELU's tanh form, (1 + tanh z) / 2 = 1 / (1 + exp(-2 z)): 1 + tanh z itself has no bits left for z below -9
__device__ __forceinline__ float moe_act(float g, uint32_t gelu) {
    const float z = gelu ? 1.5957691216057308f * (g + 0.044715f * g * g * g) : g;
    return g / (1.0f + expf(-z));
}

// ---- gate and up ----------------------------------------------------------------------------------------
// One token.  As matvec_tiles; half of a workgroup's waves take gate's rows, the others the same rows of up.  Each workgroup finds
// the choice by itself, which costs less than one more launch; one hands it on.  Grid: (row groups, top_k).
template <class F, class M>
__global__ __launch_bounds__(TILE_THREADS) void moe_up(MoeArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ int32_t chosen[MOE_MAX_TOP_K];
    typedef typename M::I I;
    static_assert(TILE_WAVES * M::WAVE_BYTES >= MOE_MAX_EXPERTS * 4, "room for the keys");
    choose(a.logits, a.experts, a.top_k, threadIdx.x, TILE_THREADS, (uint32_t *)lds, chosen, [] { __syncthreads(); });
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 64) put_choice(a, 0, chosen, threadIdx.x);
    const uint32_t expert = __builtin_amdgcn_readfirstlane((uint32_t)chosen[blockIdx.y]);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t second = wave / (TILE_WAVES / 2), group = wave % (TILE_WAVES / 2) / a.ksplit, groups = TILE_WAVES / 2 / a.ksplit;
    const uint32_t row_bytes = (uint32_t)(a.hidden / F::N * F::BYTES), turns = (uint32_t)((a.hidden + M::ELEMS - 1) / M::ELEMS);
    const uint32_t ff = (uint32_t)a.ff, first_row = blockIdx.x * groups * M::ROWS, row = first_row + group * M::ROWS;
    const RowTile<uint32_t> tile = tile_at<M::ROWS>(row, ff);
    const uint32_t own = tile.own, rows = tile.rows;
    const uint8_t *w = (second ? a.up : a.gate) + ((uint64_t)expert * ff + own) * row_bytes;
    const uint64_t behind = ((uint64_t)(a.experts - expert) * ff - own - 1) * row_bytes;
    uint8_t *clear = lds + TILE_WAVES * M::WAVE_BYTES;
    typename M::Sums acc = no_sums<M>();
    run_turns<M>(lds + wave * M::WAVE_BYTES, clear, typename I::Places(threadIdx.x % 64, rows, row_bytes), I::reach(rows, row_bytes),
                 Share{wave % a.ksplit, a.ksplit, a.chunk, turns},
                 [&](uint32_t turn) {
                     const uint32_t off = turn * I::TURN_BYTES;
                     return Turn{w + off, row_bytes - off, behind + row_bytes - off};
                 },
                 [&](uint32_t turn, uint32_t c, float (&v)[8]) { load8(a.x, 0, (uint64_t)turn * M::ELEMS + c, a.hidden, a.x_kind, v); },
                 acc);
    float *part = (float *)(clear + M::CLEAR);
    put_parts<M>(part, wave, acc);
    for (uint32_t r = threadIdx.x; r < groups * M::ROWS; r += TILE_THREADS) {
        const uint32_t g = r / M::ROWS;
        float v[2] = {0.0f, 0.0f};
        for (uint32_t k = 0; k < a.ksplit; ++k)
#pragma unroll
            for (uint32_t m = 0; m < 2; ++m) v[m] += part[(m * TILE_WAVES / 2 + g * a.ksplit + k) * M::ROWS + r % M::ROWS];
        if (first_row + r < ff) a.h[(uint64_t)blockIdx.y * ff + first_row + r] = moe_act(v[0], a.gelu) * v[1];
    }
}

// Several tokens.  As matvec_dense: a wave's two tiles are the same rows of gate and of up.  Grid: (tiles, slots).
template <class F, int X>
__global__ __launch_bounds__(TILE_THREADS) void moe_up_dense(MoeArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    typedef DenseTile<F, X, 2> M;
    typedef typename M::I I;
    const Slot &slot = a.table[blockIdx.y];
    const uint32_t expert = slot.expert, count = slot.count;
    if (count == 0) return;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), waves = blockDim.x / 64, wave_bytes = M::wave_bytes(a.slot_tokens);
    const uint32_t row_bytes = (uint32_t)(a.hidden / F::N * F::BYTES), turns = (uint32_t)((a.hidden + M::ELEMS - 1) / M::ELEMS);
    const uint32_t ff = (uint32_t)a.ff, row = blockIdx.x * M::ROWS;
    const RowTile<uint32_t> tile = full_tile_at<M::ROWS>(row, ff);
    const uint32_t own = tile.own, rows = tile.rows;
    const uint64_t at_row = (uint64_t)expert * ff + own, behind = ((uint64_t)a.experts * ff - at_row) * row_bytes;
    const uint8_t *w[2] = {a.gate + at_row * row_bytes, a.up + at_row * row_bytes};
    dense_turns<M, 2, true>(lds + wave * wave_bytes, typename I::Places(threadIdx.x % 64, rows, row_bytes), I::reach(rows, row_bytes), wave, waves, turns, count,
                             (uint32_t)a.hidden,
                             [&](uint32_t turn, int r) {
                                 const uint32_t off = turn * I::TURN_BYTES;
                                 return Turn{w[r] + off, row_bytes - off, behind - off};
                             },
                             [&](uint32_t t) { return (const uint8_t *)a.x + slot.pair[t] / a.top_k * a.x_stride * M::X_SIZE; });
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < M::ROWS * count; i += blockDim.x) {
        const uint32_t n = i % M::ROWS, t = i / M::ROWS, at = own + n;
        if (at < row || at >= ff) continue;
        float v[2] = {0.0f, 0.0f};
        for (uint32_t k = 0; k < waves; ++k)
#pragma unroll
            for (uint32_t m = 0; m < 2; ++m) v[m] += M::part(lds + k * wave_bytes, m, t, n);
        a.h[(uint64_t)slot.pair[t] * ff + at] = moe_act(v[0], a.gelu) * v[1];
    }
}

// ---- down -----------------------------------------------------------------------------------------------
// One token: the rows of its experts, one behind the other, are one long row times the experts' h, each times its weight; the sum
// over the experts is the sum over the row.
template <class F, class M>
__global__ __launch_bounds__(TILE_THREADS) void moe_down_one(MoeArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ uint32_t experts[MOE_MAX_TOP_K];
    __shared__ float weights[MOE_MAX_TOP_K];
    typedef typename M::I I;
    if (threadIdx.x < a.top_k) {
        experts[threadIdx.x] = (uint32_t)a.ids[threadIdx.x];
        weights[threadIdx.x] = a.weights[threadIdx.x];
    }
    __syncthreads();
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t group = wave / a.ksplit, groups = TILE_WAVES / a.ksplit;
    const uint32_t row_bytes = (uint32_t)(a.ff / F::N * F::BYTES), each = (uint32_t)((a.ff + M::ELEMS - 1) / M::ELEMS);
    const uint32_t hidden = (uint32_t)a.hidden, first_row = blockIdx.x * groups * M::ROWS, row = first_row + group * M::ROWS;
    const RowTile<uint32_t> tile = tile_at<M::ROWS>(row, hidden);
    const uint32_t own = tile.own, rows = tile.rows;
    uint8_t *clear = lds + TILE_WAVES * M::WAVE_BYTES;
    typename M::Sums acc = no_sums<M>();
    run_turns<M>(lds + wave * M::WAVE_BYTES, clear, typename I::Places(lane, rows, row_bytes), I::reach(rows, row_bytes),
                 Share{wave % a.ksplit, a.ksplit, a.chunk, each * a.top_k},
                 [&](uint32_t turn) {
                     const uint32_t item = turn / each, off = (turn - item * each) * I::TURN_BYTES;
                     const uint64_t e = __builtin_amdgcn_readfirstlane(experts[item]);
                     return Turn{a.down + (e * hidden + own) * row_bytes + off, row_bytes - off, ((a.experts - e) * hidden - own) * row_bytes - off};
                 },
                 [&](uint32_t turn, uint32_t c, float (&v)[8]) {
                     const uint32_t item = turn / each;
                     load8(a.h, item * a.ff, (uint64_t)(turn - item * each) * M::ELEMS + c, a.ff, EK_F32, v);
#pragma unroll
                     for (int j = 0; j < 8; ++j) v[j] *= weights[item];
                 },
                 acc);
    float *part = (float *)(clear + M::CLEAR);
    put_parts<M>(part, wave, acc);
    for (uint32_t r = threadIdx.x; r < groups * M::ROWS; r += TILE_THREADS) {
        const uint32_t g = r / M::ROWS;
        float v = 0.0f;
        for (uint32_t k = 0; k < a.ksplit; ++k) v += part[(g * a.ksplit + k) * M::ROWS + r % M::ROWS];
        if (first_row + r < hidden) store_elem(a.y, first_row + r, a.y_kind, v);
    }
}

// Several tokens: expert by expert, into o[pair]; grid: (tiles, slots).
constexpr int DOWN_TILES = 2;
template <class F, int X>
__global__ __launch_bounds__(TILE_THREADS) void moe_down_dense(MoeArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    typedef DenseTile<F, X, DOWN_TILES> M;
    typedef typename M::I I;
    const Slot &slot = a.table[blockIdx.y];
    const uint32_t expert = slot.expert, count = slot.count;
    if (count == 0) return;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), waves = blockDim.x / 64, wave_bytes = M::wave_bytes(a.slot_tokens);
    const uint32_t row_bytes = (uint32_t)(a.ff / F::N * F::BYTES), turns = (uint32_t)((a.ff + M::ELEMS - 1) / M::ELEMS);
    const uint32_t hidden = (uint32_t)a.hidden, first_row = blockIdx.x * DOWN_TILES * M::ROWS, rows = full_tile_at<M::ROWS>(first_row, hidden).rows;
    auto begin = [&](uint32_t nominal) { return full_tile_at<M::ROWS>(nominal, hidden).own; };
    dense_turns<M, DOWN_TILES, true>(lds + wave * wave_bytes, typename I::Places(threadIdx.x % 64, rows, row_bytes), I::reach(rows, row_bytes), wave, waves, turns, count,
                                      (uint32_t)a.ff,
                                      [&](uint32_t turn, int r) {
                                          const uint64_t row = (uint64_t)expert * hidden + begin(first_row + r * M::ROWS);
                                          const uint32_t off = turn * I::TURN_BYTES;
                                          return Turn{a.down + row * row_bytes + off, row_bytes - off, ((uint64_t)a.experts * hidden - row) * row_bytes - off};
                                      },
                                      [&](uint32_t t) { return (const uint8_t *)a.h + slot.pair[t] * a.ff * M::X_SIZE; });
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < DOWN_TILES * M::ROWS * count; i += blockDim.x) {
        const uint32_t r = i % (DOWN_TILES * M::ROWS), t = i / (DOWN_TILES * M::ROWS), tile = r / M::ROWS;
        const uint32_t nominal = first_row + tile * M::ROWS, at = begin(nominal) + r % M::ROWS;
        if (at < nominal || at >= hidden) continue;
        float v = 0.0f;
        for (uint32_t k = 0; k < waves; ++k) v += M::part(lds + k * wave_bytes, tile, t, r % M::ROWS);
        a.o[(uint64_t)slot.pair[t] * hidden + at] = v;
    }
}

// Experts with rows of 16-bit floats shorter than a piece of an image: a thread per output.
template <class F>
__device__ __forceinline__ float short_dot(const uint8_t *row, uint32_t cols, const void *x, uint64_t at, uint32_t kind) {
    float sum = 0.0f;
    for (uint32_t c = 0; c < cols; ++c) {
        const uint32_t b = ld2(row + 2 * c);
        sum = __builtin_fmaf(__is_same(F, WF16) ? h2f(b) : bf2f(b), load_elem(x, at + c, kind), sum);
    }
    return sum;
}
template <class F>
__global__ __launch_bounds__(MV_THREADS) void moe_up_short(MoeArgs a) {
    const uint64_t r = (uint64_t)blockIdx.x * MV_THREADS + threadIdx.x;
    if (r >= a.ff) return;
    const uint32_t pair = blockIdx.y, cols = (uint32_t)a.hidden;
    const uint64_t at = ((uint64_t)a.ids[pair] * a.ff + r) * cols * 2, x = pair / a.top_k * a.x_stride;
    a.h[pair * a.ff + r] = moe_act(short_dot<F>(a.gate + at, cols, a.x, x, a.x_kind), a.gelu) * short_dot<F>(a.up + at, cols, a.x, x, a.x_kind);
}
template <class F>
__global__ __launch_bounds__(MV_THREADS) void moe_down_short(MoeArgs a) {
    const uint64_t r = (uint64_t)blockIdx.x * MV_THREADS + threadIdx.x;
    if (r >= a.hidden) return;
    const uint32_t t = blockIdx.y, cols = (uint32_t)a.ff;
    float y = 0.0f;
    for (uint32_t j = 0; j < a.top_k; ++j) {
        const uint64_t pair = t * a.top_k + j;
        y = __builtin_fmaf(a.weights[pair], short_dot<F>(a.down + ((uint64_t)a.ids[pair] * a.hidden + r) * cols * 2, cols, a.h, pair * a.ff, EK_F32), y);
    }
    store_elem(a.y, t * a.y_stride + r, a.y_kind, y);
}

}  // namespace ggq
