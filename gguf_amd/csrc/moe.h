// moe.h -- a mixture-of-experts layer with packed experts, for few tokens.
//
//     l = router x;  the top_k experts of each token;  h_e = act(gate_e x) * (up_e x);  y = sum of w_e down_e h_e
//
// The launches: logits; the choice, where it is not found on the way; gate and up of the experts in use; down with the sum
// over a token's experts (for more than four tokens down and the sum apart).  Bound by the bytes of the experts in use: each is read once for up to 16 of its
// tokens, and once more for each further 16.
#pragma once
#include "choice.h"
#include "dense.h"

namespace ggq {

__device__ __forceinline__ float moe_act(float g, uint32_t gelu) {
    if (!gelu) return g / (1.0f + expf(-g));
    const float z = 0.7978845608028654f * (g + 0.044715f * g * g * g);
    return 0.5f * g * (1.0f + tanhf(z));
}


// ---- which expert, and which tokens ----------------------------------------------------------------------
// Experts in use, in the order of their index, each with its tokens a few at a time (a.slot_tokens): a slot is one such group.
struct Slot {
    uint32_t expert, count;       // of tokens; 0: no such slot
};
struct SlotSpace {
    uint32_t low[MOE_MAX_EXPERTS], high[MOE_MAX_EXPERTS];         // masks of tokens, by expert
    uint32_t pair[SLOT_TOKENS];   // of the slot's tokens: token * top_k + place
};
__device__ __forceinline__ uint32_t nth_bit(uint64_t m, uint32_t n) {
    for (; n; --n) m &= m - 1;
    return (uint32_t)__builtin_ctzll(m);
}
// All threads of the workgroup; ids: the choices of all tokens.  The same answer in all of them.
__device__ __forceinline__ Slot find_slot(SlotSpace &s, const MoeArgs &a, const int32_t *ids, uint32_t slot) {
    const uint32_t lane = threadIdx.x % 64;
    for (uint32_t e = threadIdx.x; e < a.experts; e += blockDim.x) s.low[e] = s.high[e] = 0;
    __syncthreads();
    for (uint32_t p = threadIdx.x; p < a.tokens * a.top_k; p += blockDim.x) {
        const uint32_t t = p / a.top_k;
        atomicOr(t < 32 ? &s.low[ids[p]] : &s.high[ids[p]], 1u << (t & 31));
    }
    __syncthreads();
    uint32_t seen = 0, expert = 0, count = 0;
    for (uint32_t base = 0; base < a.experts; base += 64) {
        const uint32_t e = base + lane;
        const uint32_t tokens = e < a.experts ? (uint32_t)__popc(s.low[e]) + (uint32_t)__popc(s.high[e]) : 0u, mine = (tokens + a.slot_tokens - 1) / a.slot_tokens;
        uint32_t upto = mine;                                     // slots of the lanes up to this one
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_up(upto, d);
            upto += lane >= (uint32_t)d ? o : 0u;
        }
        const uint64_t here = __ballot(slot < seen + upto);
        if (here) {
            const uint32_t l = (uint32_t)__builtin_ctzll(here);
            const uint32_t group = __builtin_amdgcn_readfirstlane(slot - seen - __shfl(upto - mine, l));
            expert = base + l;
            const uint32_t low = __builtin_amdgcn_readfirstlane(s.low[expert]), high = __builtin_amdgcn_readfirstlane(s.high[expert]);
            const uint64_t mask = low | ((uint64_t)high << 32);
            const uint32_t n = (uint32_t)__popcll(mask) - group * a.slot_tokens;
            count = n < a.slot_tokens ? n : a.slot_tokens;
            if (threadIdx.x < count) {
                const uint32_t first = nth_bit(mask, group * a.slot_tokens + threadIdx.x) * a.top_k;
                uint32_t pair = first;
                for (uint32_t j = 0; j < a.top_k; ++j) pair = (uint32_t)ids[first + j] == expert ? first + j : pair;
                s.pair[threadIdx.x] = pair;
            }
            break;
        }
        seen += __builtin_amdgcn_readfirstlane(__shfl(upto, 63));
    }
    __syncthreads();
    return {(uint32_t)__builtin_amdgcn_readfirstlane(expert), (uint32_t)__builtin_amdgcn_readfirstlane(count)};
}

// ---- gate and up ----------------------------------------------------------------------------------------
// The choice of all tokens: already there, or found by each workgroup with few tokens and experts, a wave for each token, which
// costs it less than one more launch; one workgroup hands it on.  `space`: wave_bytes of shared memory for each wave.
constexpr uint32_t MOE_KEYS = MOE_MAX_EXPERTS * 4;
struct Chosen { int32_t ids[CHOOSE_TOKENS * MOE_MAX_TOP_K]; };
__device__ __forceinline__ const int32_t *choices(const MoeArgs &a, Chosen &chosen, uint8_t *space, uint32_t wave_bytes) {
    if (!a.choose) return a.ids;
    const uint32_t lane = threadIdx.x % 64, waves = blockDim.x / 64, wave = threadIdx.x / 64;
    for (uint32_t t = wave; t < a.tokens; t += waves) {
        int32_t *ids = chosen.ids + t * a.top_k;
        choose(a.logits + (uint64_t)t * a.experts, a.experts, a.top_k, lane, 64, (uint32_t *)(space + wave * wave_bytes), ids, [] { wave_order(); });
        if (blockIdx.x == 0 && blockIdx.y == 0) put_choice(a, t, ids, lane);
    }
    __syncthreads();
    return chosen.ids;
}

// One token.  As matvec_tiles; half of a workgroup's waves take gate's rows, the others the same rows of up.  Grid: (row groups, slots).
template <class F, class M>
__global__ __launch_bounds__(TILE_THREADS) void moe_up(MoeArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ Chosen chosen;
    typedef typename M::I I;
    static_assert(M::WAVE_BYTES >= MOE_KEYS, "room for the keys");
    const uint32_t expert = __builtin_amdgcn_readfirstlane((uint32_t)choices(a, chosen, lds, M::WAVE_BYTES)[blockIdx.y]);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t second = wave / (TILE_WAVES / 2), group = wave % (TILE_WAVES / 2) / a.ksplit, groups = TILE_WAVES / 2 / a.ksplit;
    const uint32_t row_bytes = (uint32_t)(a.hidden / F::N * F::BYTES), turns = (uint32_t)((a.hidden + M::ELEMS - 1) / M::ELEMS);
    const uint32_t ff = (uint32_t)a.ff, first_row = blockIdx.x * groups * M::ROWS, row = first_row + group * M::ROWS, own = row < ff ? row : ff - 1;
    const uint32_t rows = ff - own < M::ROWS ? ff - own : M::ROWS;
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

// Several tokens.  As matvec_dense: a wave's two tiles are the same rows of gate and of up; a workgroup has several groups of
// waves.  Grid: (row groups, slots).
template <class F, int X>
__global__ __launch_bounds__(TILE_THREADS) void moe_up_dense(MoeArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ SlotSpace space;
    __shared__ Chosen chosen;
    typedef DenseTile<F, X, 2> M;
    typedef typename M::I I;
    static_assert(M::AT_X >= MOE_KEYS, "room for the keys");
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wave_bytes = M::wave_bytes(a.slot_tokens);
    const Slot slot = find_slot(space, a, choices(a, chosen, lds, wave_bytes), blockIdx.y);
    if (slot.count == 0) return;
    const uint32_t group = wave / a.ksplit, groups = blockDim.x / 64 / a.ksplit;
    const uint32_t row_bytes = (uint32_t)(a.hidden / F::N * F::BYTES), turns = (uint32_t)((a.hidden + M::ELEMS - 1) / M::ELEMS);
    const uint32_t ff = (uint32_t)a.ff, rows = ff < M::ROWS ? ff : M::ROWS, first_row = blockIdx.x * groups * M::ROWS, row = first_row + group * M::ROWS;
    const uint32_t own = row < ff - rows ? row : ff - rows;
    const uint64_t at_row = (uint64_t)slot.expert * ff + own, behind = ((uint64_t)a.experts * ff - at_row) * row_bytes;
    const uint8_t *w[2] = {a.gate + at_row * row_bytes, a.up + at_row * row_bytes};
    if (row < ff)
        dense_turns<M, 2, false>(lds + wave * wave_bytes, typename I::Places(threadIdx.x % 64, rows, row_bytes), I::reach(rows, row_bytes), wave % a.ksplit, a.ksplit, turns,
                                 slot.count, (uint32_t)a.hidden,
                                 [&](uint32_t turn, int r) {
                                     const uint32_t off = turn * I::TURN_BYTES;
                                     return Turn{w[r] + off, row_bytes - off, behind - off};
                                 },
                                 [&](uint32_t, uint32_t t) { return (const uint8_t *)a.x + space.pair[t] / a.top_k * a.x_stride * M::X_SIZE; },
                                 [](uint32_t turn) { return turn * M::ELEMS; }, [](uint32_t, uint32_t) { return Factor{}; });
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < groups * M::ROWS * slot.count; i += blockDim.x) {
        const uint32_t r = i % (groups * M::ROWS), t = i / (groups * M::ROWS), g = r / M::ROWS;
        const uint32_t nominal = first_row + g * M::ROWS, begin = nominal < ff - rows ? nominal : ff - rows, at = begin + r % M::ROWS;
        if (at < nominal || at >= ff) continue;
        float v[2] = {0.0f, 0.0f};
        for (uint32_t k = 0; k < a.ksplit; ++k)
#pragma unroll
            for (uint32_t m = 0; m < 2; ++m) v[m] += M::part(lds + (g * a.ksplit + k) * wave_bytes, m, t, r % M::ROWS);
        a.h[(uint64_t)space.pair[t] * ff + at] = moe_act(v[0], a.gelu) * v[1];
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
    const uint32_t hidden = (uint32_t)a.hidden, first_row = blockIdx.x * groups * M::ROWS, row = first_row + group * M::ROWS, own = row < hidden ? row : hidden - 1;
    const uint32_t rows = hidden - own < M::ROWS ? hidden - own : M::ROWS;
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

constexpr uint32_t FEW_PAIRS = FEW_TOKENS * MOE_MAX_TOP_K;
// Up to FEW_TOKENS: the same with the rows of all experts in use; a token that did not choose an expert meets zeros.
template <class F, int X>
__global__ __launch_bounds__(TILE_THREADS) void moe_down_few(MoeArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ uint32_t items[FEW_PAIRS];          // experts in use, in the order of their first pair
    __shared__ int32_t pair_at[FEW_PAIRS][FEW_TOKENS];      // the pair of item and token, or -1
    __shared__ int32_t ids[FEW_PAIRS];
    __shared__ uint64_t fresh_of[2];
    typedef DenseTile<F, X, 1> M;
    typedef typename M::I I;
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), waves = blockDim.x / 64, wave_bytes = M::wave_bytes(a.tokens);
    const uint32_t pairs = a.tokens * a.top_k, me_pair = threadIdx.x;      // at most 128: the first two waves
    if (me_pair < FEW_PAIRS) {
        ids[me_pair] = me_pair < pairs ? a.ids[me_pair] : -1;
#pragma unroll
        for (int t = 0; t < (int)FEW_TOKENS; ++t) pair_at[me_pair][t] = -1;
    }
    __syncthreads();
    uint32_t front = me_pair;                              // the first pair with the same expert
    if (me_pair < pairs)
        for (uint32_t q = me_pair; q-- > 0;) front = ids[q] == ids[me_pair] ? q : front;
    const uint64_t fresh = __ballot(me_pair < pairs && front == me_pair);
    if (lane == 0 && wave < 2) fresh_of[wave] = fresh;
    __syncthreads();
    if (me_pair < pairs) {
        const uint32_t below = (uint32_t)__popcll(fresh_of[front / 64] & ((1ull << (front % 64)) - 1));
        const uint32_t place = below + (front >= 64 ? (uint32_t)__popcll(fresh_of[0]) : 0u);
        if (front == me_pair) items[place] = (uint32_t)ids[me_pair];
        pair_at[place][me_pair / a.top_k] = (int32_t)me_pair;
    }
    __syncthreads();
    const uint32_t count = __builtin_amdgcn_readfirstlane((uint32_t)(__popcll(fresh_of[0]) + __popcll(fresh_of[1])));
    const uint32_t row_bytes = (uint32_t)(a.ff / F::N * F::BYTES), each = (uint32_t)((a.ff + M::ELEMS - 1) / M::ELEMS);
    const uint32_t hidden = (uint32_t)a.hidden, rows = hidden < M::ROWS ? hidden : M::ROWS, row = blockIdx.x * M::ROWS, own = row < hidden - rows ? row : hidden - rows;
    dense_turns<M, 1, true>(lds + wave * wave_bytes, typename I::Places(lane, rows, row_bytes), I::reach(rows, row_bytes), wave, waves, each * count, a.tokens, (uint32_t)a.ff,
                            [&](uint32_t turn, int) {
                                const uint32_t item = turn / each, off = (turn - item * each) * I::TURN_BYTES;
                                const uint64_t e = __builtin_amdgcn_readfirstlane(items[item]);
                                return Turn{a.down + (e * hidden + own) * row_bytes + off, row_bytes - off, ((a.experts - e) * hidden - own) * row_bytes - off};
                            },
                            [&](uint32_t turn, uint32_t t) {
                                const int32_t pair = pair_at[turn / each][t];
                                return (const uint8_t *)a.h + (pair < 0 ? 0 : pair) * a.ff * M::X_SIZE;
                            },
                            [&](uint32_t turn) { return turn % each * M::ELEMS; },
                            [&](uint32_t turn, uint32_t t) {
                                const int32_t pair = pair_at[turn / each][t];
                                return pair < 0 ? Factor{0.0f, 0u} : Factor{a.weights[pair], ~0u};
                            });
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < M::ROWS * a.tokens; i += blockDim.x) {
        const uint32_t n = i % M::ROWS, t = i / M::ROWS, at = own + n;
        if (at < row || at >= hidden) continue;
        float v = 0.0f;
        for (uint32_t k = 0; k < waves; ++k) v += M::part(lds + k * wave_bytes, 0, t, n);
        store_elem(a.y, t * a.y_stride + at, a.y_kind, v);
    }
}

// More tokens: expert by expert, into o[pair]; grid: (row groups, slots).
constexpr int DOWN_TILES = 2;
template <class F, int X>
__global__ __launch_bounds__(TILE_THREADS) void moe_down_dense(MoeArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ SlotSpace space;
    typedef DenseTile<F, X, DOWN_TILES> M;
    typedef typename M::I I;
    constexpr uint32_t ROWS = DOWN_TILES * M::ROWS;
    const Slot slot = find_slot(space, a, a.ids, blockIdx.y);
    if (slot.count == 0) return;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wave_bytes = M::wave_bytes(a.slot_tokens);
    const uint32_t group = wave / a.ksplit, groups = blockDim.x / 64 / a.ksplit;
    const uint32_t row_bytes = (uint32_t)(a.ff / F::N * F::BYTES), turns = (uint32_t)((a.ff + M::ELEMS - 1) / M::ELEMS);
    const uint32_t hidden = (uint32_t)a.hidden, rows = hidden < M::ROWS ? hidden : M::ROWS, first_row = blockIdx.x * groups * ROWS;
    auto begin = [&](uint32_t nominal) { return nominal < hidden - rows ? nominal : hidden - rows; };
    if (first_row + group * ROWS < hidden)
        dense_turns<M, DOWN_TILES, false>(lds + wave * wave_bytes, typename I::Places(threadIdx.x % 64, rows, row_bytes), I::reach(rows, row_bytes), wave % a.ksplit, a.ksplit,
                                          turns, slot.count, (uint32_t)a.ff,
                                          [&](uint32_t turn, int r) {
                                              const uint64_t row = (uint64_t)slot.expert * hidden + begin(first_row + group * ROWS + r * M::ROWS);
                                              const uint32_t off = turn * I::TURN_BYTES;
                                              return Turn{a.down + row * row_bytes + off, row_bytes - off, ((uint64_t)a.experts * hidden - row) * row_bytes - off};
                                          },
                                          [&](uint32_t, uint32_t t) { return (const uint8_t *)a.h + space.pair[t] * a.ff * M::X_SIZE; },
                                          [](uint32_t turn) { return turn * M::ELEMS; }, [](uint32_t, uint32_t) { return Factor{}; });
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < groups * ROWS * slot.count; i += blockDim.x) {
        const uint32_t r = i % (groups * ROWS), t = i / (groups * ROWS), g = r / ROWS, tile = r % ROWS / M::ROWS;
        const uint32_t nominal = first_row + r / M::ROWS * M::ROWS, at = begin(nominal) + r % M::ROWS;
        if (at < nominal || at >= hidden) continue;
        float v = 0.0f;
        for (uint32_t k = 0; k < a.ksplit; ++k) v += M::part(lds + (g * a.ksplit + k) * wave_bytes, tile, t, r % M::ROWS);
        a.o[(uint64_t)space.pair[t] * hidden + at] = v;
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
