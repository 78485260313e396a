// moe.h -- a mixture-of-experts layer with packed experts, for few tokens.
//
//     l = router x;  the top_k experts of each token;  h_e = act(gate_e x) * (up_e x);  y = sum of w_e down_e h_e
//
// The launches: logits, choice, gate and up of the experts in use, down with the sum over a token's experts (for more than
// four tokens down and the sum apart).  Bound by the bytes of the experts in use: each is read once for up to four of its
// tokens, and once more for each further four.
#pragma once
#include "matmul.h"

namespace ggq {

struct MoeArgs {
    const uint8_t *gate, *up, *down;
    const void *router, *x;
    void *y;
    float *logits;        // [tokens][experts]
    int32_t *ids;         // [tokens][top_k]
    float *weights;       // [tokens][top_k]
    float *h;             // [tokens * top_k][ff]
    float *o;             // [tokens * top_k][hidden], where tokens > 4
    int32_t *out_ids;     // the caller's, or null
    float *out_weights;
    uint64_t hidden, ff, x_stride, y_stride;
    uint32_t tokens, experts, top_k, router_kind, x_kind, y_kind;
    uint32_t sigmoid, normalize, gelu;
    uint32_t parts, chunk, ksplit;            // as in MatvecArgs, of the launch
    uint32_t slots;                           // experts that may be in use: workgroups along y
    float scale;
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

// one workgroup per expert; a product of two f32 values is exact in 64 bits
__global__ __launch_bounds__(MV_THREADS) static void moe_logits(MoeArgs a) {
    __shared__ double part[MV_THREADS / 64];
    const uint32_t e = blockIdx.x;
    for (uint32_t t = 0; t < a.tokens; ++t) {
        double s = 0.0;
        for (uint64_t c = threadIdx.x; c < a.hidden; c += MV_THREADS)
            s = __builtin_fma((double)load_elem(a.router, e * a.hidden + c, a.router_kind), (double)load_elem(a.x, t * a.x_stride + c, a.x_kind), s);
        s = wave_sum(s);
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (uint32_t w = 1; w < MV_THREADS / 64; ++w) s += part[w];
            a.logits[(uint64_t)t * a.experts + e] = (float)s;
        }
        __syncthreads();
    }
}

// an order-preserving key of a logit: larger logit, larger key; NaN below everything; -0 equals +0
__device__ __forceinline__ uint32_t logit_key(float v) {
    if (v != v) return 0u;
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// ---- the choice -----------------------------------------------------------------------------------------
constexpr uint32_t MOE_MAX_EXPERTS = 512, MOE_MAX_TOP_K = 32, MOE_MAX_TOKENS = 64;

// One wave: the top_k experts of a token, ids[j] = the j-th.  An expert's place is the number of experts in front of it
// (a larger key, or the same and a lower index), so all places are found at once, without a chain of k maxima; keys are
// read four at a time, the same for all lanes.  `keys`: the wave's own, room for 512.
__device__ __forceinline__ void choose(const float *logits, uint32_t experts, uint32_t top_k, uint32_t lane, uint32_t *keys, int32_t *ids) {
    const uint32_t padded = (experts + 3) & ~3u;
    for (uint32_t e = lane; e < padded; e += 64) keys[e] = e < experts ? logit_key(logits[e]) : 0u;
    wave_order();
    for (uint32_t e = lane; e < experts; e += 64) {
        const uint32_t key = keys[e];
        uint32_t place = 0;
        for (uint32_t q = 0; q < padded; q += 4) {
            const u32x4 k = *(const u32x4 *)(keys + q);
#pragma unroll
            for (int i = 0; i < 4; ++i) place += (k[i] > key) || (k[i] == key && q + i < e);
        }
        if (place < top_k) ids[place] = (int32_t)e;
    }
    wave_order();
}

// One wave: the weights of a token's chosen experts, weight j in lane j.
__device__ __forceinline__ float choice_weight(const float *l, const MoeArgs &a, const int32_t *ids, uint32_t lane) {
    float top = -__builtin_inff(), total = 0.0f;
    if (!a.sigmoid) {
        for (uint32_t e = lane; e < a.experts; e += 64) top = __builtin_fmaxf(top, l[e]);
#pragma unroll
        for (int m = 32; m; m >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, m));
        for (uint32_t e = lane; e < a.experts; e += 64) total += expf(l[e] - top);
        total = wave_sum(total);
    }
    float mine = 0.0f;
    if (lane < a.top_k) {
        const float v = l[ids[lane]];
        mine = a.sigmoid ? 1.0f / (1.0f + expf(-v)) : expf(v - top) / total;
    }
    const float sum = wave_sum(mine);
    return (a.normalize ? mine / sum : mine) * a.scale;
}

// The choice of all tokens, a wave per token; `out`: what the caller gets as well
__global__ __launch_bounds__(64) static void moe_route(MoeArgs a) {
    __shared__ uint32_t keys[MOE_MAX_EXPERTS];
    __shared__ int32_t ids[MOE_MAX_TOP_K];
    const uint32_t t = blockIdx.x, lane = threadIdx.x;
    const float *l = a.logits + (uint64_t)t * a.experts;
    choose(l, a.experts, a.top_k, lane, keys, ids);
    const float w = choice_weight(l, a, ids, lane);
    if (lane < a.top_k) {
        const uint32_t at = t * a.top_k + lane;
        a.ids[at] = ids[lane];
        a.weights[at] = w;
        if (a.out_ids) a.out_ids[at] = ids[lane];
        if (a.out_weights) a.out_weights[at] = w;
    }
}

__device__ __forceinline__ float moe_act(float g, uint32_t gelu) {
    if (!gelu) return g / (1.0f + expf(-g));
    const float z = 0.7978845608028654f * (g + 0.044715f * g * g * g);
    return 0.5f * g * (1.0f + tanhf(z));
}


// ---- which expert, and which tokens ----------------------------------------------------------------------
// The tokens that chose the slot-th expert in use (experts in use in order of their index).
struct Slot {
    uint32_t expert, count;
    uint64_t mask;                // bit t: token t
};
struct SlotSpace {
    uint32_t low[MOE_MAX_EXPERTS], high[MOE_MAX_EXPERTS];         // masks of tokens, by expert
};
__device__ __forceinline__ uint32_t nth_bit(uint64_t m, uint32_t n) {
    for (; n; --n) m &= m - 1;
    return (uint32_t)__builtin_ctzll(m);
}
// All threads of the workgroup; ids: the choices of all tokens.
__device__ __forceinline__ Slot find_slot(SlotSpace &s, const int32_t *ids, const MoeArgs &a, uint32_t slot) {
    for (uint32_t e = threadIdx.x; e < a.experts; e += blockDim.x) s.low[e] = s.high[e] = 0;
    __syncthreads();
    for (uint32_t p = threadIdx.x; p < a.tokens * a.top_k; p += blockDim.x) {
        const uint32_t t = p / a.top_k;
        atomicOr(t < 32 ? &s.low[ids[p]] : &s.high[ids[p]], 1u << (t & 31));
    }
    __syncthreads();
    const uint32_t lane = threadIdx.x % 64;
    Slot r{0, 0, 0};
    uint32_t seen = 0;
    for (uint32_t base = 0; base < a.experts; base += 64) {
        const uint32_t e = base + lane;
        const uint64_t used = __ballot(e < a.experts && (s.low[e < a.experts ? e : 0] | s.high[e < a.experts ? e : 0]));
        const uint32_t n = (uint32_t)__popcll(used);
        if (slot < seen + n) {
            r.expert = base + nth_bit(used, slot - seen);
            r.mask = s.low[r.expert] | ((uint64_t)s.high[r.expert] << 32);
            r.expert = __builtin_amdgcn_readfirstlane(r.expert);
            r.count = (uint32_t)__popcll(r.mask);
            return r;
        }
        seen += n;
    }
    return r;
}

// the pair of a token and an expert that it chose
__device__ __forceinline__ uint32_t pair_with(const MoeArgs &a, uint32_t token, uint32_t expert) {
    uint32_t pair = token * a.top_k;
    for (uint32_t j = 0; j < a.top_k; ++j) pair = (uint32_t)a.ids[token * a.top_k + j] == expert ? token * a.top_k + j : pair;
    return pair;
}

// ---- gate and up ----------------------------------------------------------------------------------------
// As matvec_quads, with a tile of gate's rows and the same rows of up in each wave; grid: (row groups, slots).
template <class F, int NC, int CHAIN>
__global__ __launch_bounds__(QD_THREADS) void moe_up(MoeArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ SlotSpace space;
    __shared__ uint32_t pairs[MOE_MAX_TOKENS];
    typedef Slice<F> S;
    typedef XStep<F, NC, CHAIN> X;
    typedef Image<F, 1> I;
    const Slot slot = find_slot(space, a.ids, a, blockIdx.y);
    if (slot.count == 0) return;
    if (threadIdx.x < slot.count) pairs[threadIdx.x] = pair_with(a, nth_bit(slot.mask, threadIdx.x), slot.expert);
    __syncthreads();
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), quad = lane / 4;
    const uint32_t kp = wave % a.ksplit, group = wave / a.ksplit, groups = QD_WAVES / a.ksplit;
    const uint32_t row_bytes = (uint32_t)(a.hidden / F::N * F::BYTES), steps = (uint32_t)((a.hidden + 1023) / 1024);
    const uint32_t ff = (uint32_t)a.ff, first_row = blockIdx.x * groups * 4, row = first_row + group * 4, own = row < ff ? row : ff - 1;
    const uint32_t rows = ff - own < 4 ? ff - own : 4;
    const uint64_t at_row = ((uint64_t)slot.expert * ff + own) * row_bytes;
    const uint32_t reach = (rows - 1) * row_bytes + (S::UNITS - 1) * S::UNIT + I::UNIT;
    const uint64_t behind = ((uint64_t)(a.experts - slot.expert) * ff - own - 1) * row_bytes;
    const typename S::Lane me(quad);
    uint8_t *image = lds + wave * 2 * I::BYTES, *xs = lds + QD_WAVES * 2 * I::BYTES;
    const uint8_t *x = xs + (quad * NC + (lane % 4 < NC ? lane % 4 : NC - 1)) * 16, *sums = xs + X::SUMS + quad * NC * 4;
    const typename I::Places places(lane, rows, row_bytes);
    I gate, up;
    const uint32_t most = NC / a.parts;

    for (uint32_t done = 0; done < slot.count; done += most) {
        const uint32_t tokens = slot.count - done < most ? slot.count - done : most;
        float acc[2][NC];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int c = 0; c < NC; ++c) acc[t][c] = 0.0f;
        uint64_t off = at_row + (uint64_t)kp * S::STEP;
        uint32_t left = row_bytes - (kp < steps ? kp : steps - 1) * S::STEP, step = kp;
        if (kp < steps) {
            gate.fetch(places, a.gate + off, behind + left, reach);
            up.fetch(places, a.up + off, behind + left, reach);
        }
        for (uint32_t first = 0; first < steps; first += a.chunk) {
            const uint32_t now = first + a.chunk < steps ? a.chunk : steps - first, end = first + now;
            if (first || done) __syncthreads();
            stage_x<F, NC, CHAIN>(xs, now, tokens, a.parts, [&](uint32_t n, uint32_t t, uint32_t f, float (&v)[8]) {
                load8(a.x, pairs[done + t] / a.top_k * a.x_stride, ((uint64_t)(first + n) * 128 + f) * 8, a.hidden, a.x_kind, v);
            });
            __syncthreads();
            for (; step < end; step += a.ksplit) {
                wave_order();
                gate.put(places, image);
                up.put(places, image + I::BYTES);
                wave_order();
                const uint32_t here = left;
                if (step + a.ksplit < steps) {
                    off += (uint64_t)a.ksplit * S::STEP;
                    left -= a.ksplit * S::STEP;
                    gate.fetch(places, a.gate + off, behind + left, reach);
                    up.fetch(places, a.up + off, behind + left, reach);
                }
                const uint32_t at = (step - first) * X::BYTES;
                if constexpr (S::STEP <= 640) {
                    typename S::Raw raw[2];
                    raw[0].load(image + lane % 4 * I::ROW, me, here);
                    raw[1].load(image + I::BYTES + lane % 4 * I::ROW, me, here);
                    add_slices<F, NC, CHAIN, 2>(raw, me, x + at, sums + at, acc);
                } else {
#pragma unroll
                    for (int m = 0; m < 2; ++m) {          // one after the other: their bytes would not fit in registers
                        typename S::Raw raw[1];
                        raw[0].load(image + m * I::BYTES + lane % 4 * I::ROW, me, here);
                        add_slices<F, NC, CHAIN, 1>(raw, me, x + at, sums + at, *(float (*)[1][NC])&acc[m]);
                        wave_order();
                    }
                }
            }
        }
        __syncthreads();
        float *part = (float *)xs;                         // [wave][gate, up][column][row]
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float v = quads_sum(acc[t][c]);
                if (lane < 4) part[((wave * 2 + t) * NC + c) * 4 + lane] = v;
            }
        __syncthreads();
        if (threadIdx.x < groups * 4 * tokens) {
            const uint32_t r = threadIdx.x % (groups * 4), t = threadIdx.x / (groups * 4), g = r / 4;
            float v[2] = {0.0f, 0.0f};
            for (uint32_t k = 0; k < a.ksplit; ++k)
                for (uint32_t p = 0; p < a.parts; ++p)
#pragma unroll
                    for (int m = 0; m < 2; ++m) v[m] += part[(((g * a.ksplit + k) * 2 + m) * NC + t * a.parts + p) * 4 + r % 4];
            if (first_row + r < ff) a.h[(uint64_t)pairs[done + t] * ff + first_row + r] = moe_act(v[0], a.gelu) * v[1];
        }
    }
}

// ---- down -----------------------------------------------------------------------------------------------
// Up to four tokens: the rows of all experts in use, one behind the other, are one long row times the tokens' h, each
// times its weight (0 for a token that did not choose the expert); the sum over a token's experts is the sum over the
// row.  NC columns are the three pieces of the only token's h, or the tokens, whose pieces follow each other.
template <class F, int NC, int CHAIN, int RT>
__global__ __launch_bounds__(QD_THREADS) void moe_down_few(MoeArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ uint32_t items[4 * MOE_MAX_TOP_K];          // experts in use, in the order of their first pair
    __shared__ int32_t pair_of[4 * MOE_MAX_TOP_K][4];      // the pair of item and token, or -1
    __shared__ int32_t ids[4 * MOE_MAX_TOP_K];
    __shared__ uint64_t fresh_of[2];
    typedef Slice<F> S;
    typedef XStep<F, NC, CHAIN> X;
    typedef Image<F, RT> I;
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), quad = lane / 4;
    const uint32_t pairs = a.tokens * a.top_k, me_pair = threadIdx.x;      // at most 128: the first two waves
    if (me_pair < 4 * MOE_MAX_TOP_K) {
        ids[me_pair] = me_pair < pairs ? a.ids[me_pair] : -1;
#pragma unroll
        for (int t = 0; t < 4; ++t) pair_of[me_pair][t] = -1;
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
        pair_of[place][me_pair / a.top_k] = (int32_t)me_pair;
    }
    __syncthreads();
    const uint32_t count = __builtin_amdgcn_readfirstlane((uint32_t)(__popcll(fresh_of[0]) + __popcll(fresh_of[1])));
    const uint32_t kp = wave % a.ksplit, group = wave / a.ksplit, groups = QD_WAVES / a.ksplit;
    const uint32_t row_bytes = (uint32_t)(a.ff / F::N * F::BYTES), each = (uint32_t)((a.ff + 1023) / 1024), steps = each * count;
    const uint32_t hidden = (uint32_t)a.hidden, first_row = blockIdx.x * groups * I::ROWS, row = first_row + group * I::ROWS, own = row < hidden ? row : hidden - 1;
    const uint32_t rows = hidden - own < I::ROWS ? hidden - own : I::ROWS;
    const uint32_t reach = (rows - 1) * row_bytes + (S::UNITS - 1) * S::UNIT + I::UNIT;
    const typename S::Lane me(quad);
    uint8_t *image = lds + wave * I::BYTES, *xs = lds + QD_WAVES * I::BYTES;
    const uint8_t *x = xs + (quad * NC + (lane % 4 < NC ? lane % 4 : NC - 1)) * 16, *sums = xs + X::SUMS + quad * NC * 4;
    float acc[RT][NC];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[t][c] = 0.0f;

    const typename I::Places places(lane, rows, row_bytes);
    I in;
    uint32_t item = kp / each, local = kp % each;          // of the step that is fetched
    auto fetch = [&]() {
        const uint64_t e = __builtin_amdgcn_readfirstlane(items[item]);
        const uint32_t left = row_bytes - local * S::STEP;
        in.fetch(places, a.down + (e * hidden + own) * row_bytes + (uint64_t)local * S::STEP, ((a.experts - e) * hidden - own - 1) * row_bytes + left, reach);
        return left;
    };
    uint32_t left = 0, step = kp;
    if (kp < steps) left = fetch();
    for (uint32_t first = 0; first < steps; first += a.chunk) {
        const uint32_t now = first + a.chunk < steps ? a.chunk : steps - first, end = first + now;
        if (first) __syncthreads();
        stage_x<F, NC, CHAIN>(xs, now, a.tokens, a.parts, [&](uint32_t n, uint32_t t, uint32_t f, float (&v)[8]) {
            const uint32_t i = (first + n) / each, s = (first + n) % each;
            const int32_t pair = pair_of[i][t];
            const uint32_t from = pair < 0 ? 0u : (uint32_t)pair;
            const float w = pair < 0 ? 0.0f : a.weights[from];
            load8(a.h, from * a.ff, ((uint64_t)s * 128 + f) * 8, a.ff, EK_F32, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = pair < 0 ? 0.0f : v[j] * w;
        });
        __syncthreads();
        for (; step < end; step += a.ksplit) {
            wave_order();
            in.put(places, image);
            wave_order();
            const uint32_t here = left;
            if (step + a.ksplit < steps) {
                for (local += a.ksplit; local >= each; local -= each) ++item;
                left = fetch();
            }
            typename S::Raw raw[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t) raw[t].load(image + (t * 4 + lane % 4) * I::ROW, me, here);
            const uint32_t at = (step - first) * X::BYTES;
            add_slices<F, NC, CHAIN, RT>(raw, me, x + at, sums + at, acc);
        }
    }
    __syncthreads();
    float *part = (float *)xs;                             // [wave][column][row]
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const float v = quads_sum(acc[t][c]);
            if (lane < 4) part[(wave * NC + c) * I::ROWS + t * 4 + lane] = v;
        }
    __syncthreads();
    if (threadIdx.x < groups * I::ROWS * a.tokens) {
        const uint32_t r = threadIdx.x % (groups * I::ROWS), t = threadIdx.x / (groups * I::ROWS), g = r / I::ROWS;
        float v = 0.0f;
        for (uint32_t k = 0; k < a.ksplit; ++k)
            for (uint32_t p = 0; p < a.parts; ++p) v += part[((g * a.ksplit + k) * NC + t * a.parts + p) * I::ROWS + r % I::ROWS];
        if (first_row + r < hidden) store_elem(a.y, t * a.y_stride + first_row + r, a.y_kind, v);
    }
}

// More tokens: expert by expert, four of its tokens at a time, into o[pair]; grid: (row groups, slots).
template <class F, int RT>
__global__ __launch_bounds__(QD_THREADS) void moe_down_many(MoeArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ SlotSpace space;
    __shared__ uint32_t pairs[MOE_MAX_TOKENS];
    constexpr int NC = 4, CHAIN = 3;
    typedef Slice<F> S;
    typedef XStep<F, NC, CHAIN> X;
    typedef Image<F, RT> I;
    const Slot slot = find_slot(space, a.ids, a, blockIdx.y);
    if (slot.count == 0) return;
    if (threadIdx.x < slot.count) pairs[threadIdx.x] = pair_with(a, nth_bit(slot.mask, threadIdx.x), slot.expert);
    __syncthreads();
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), quad = lane / 4;
    const uint32_t kp = wave % a.ksplit, group = wave / a.ksplit, groups = QD_WAVES / a.ksplit;
    const uint32_t row_bytes = (uint32_t)(a.ff / F::N * F::BYTES), steps = (uint32_t)((a.ff + 1023) / 1024);
    const uint32_t hidden = (uint32_t)a.hidden, first_row = blockIdx.x * groups * I::ROWS, row = first_row + group * I::ROWS, own = row < hidden ? row : hidden - 1;
    const uint32_t rows = hidden - own < I::ROWS ? hidden - own : I::ROWS;
    const uint64_t at_row = ((uint64_t)slot.expert * hidden + own) * row_bytes;
    const uint32_t reach = (rows - 1) * row_bytes + (S::UNITS - 1) * S::UNIT + I::UNIT;
    const uint64_t behind = ((uint64_t)(a.experts - slot.expert) * hidden - own - 1) * row_bytes;
    const typename S::Lane me(quad);
    uint8_t *image = lds + wave * I::BYTES, *xs = lds + QD_WAVES * I::BYTES;
    const uint8_t *x = xs + (quad * NC + lane % 4) * 16, *sums = xs + X::SUMS + quad * NC * 4;
    const typename I::Places places(lane, rows, row_bytes);
    I in;
    for (uint32_t done = 0; done < slot.count; done += NC) {
        const uint32_t tokens = slot.count - done < NC ? slot.count - done : NC;
        float acc[RT][NC];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int c = 0; c < NC; ++c) acc[t][c] = 0.0f;
        uint64_t off = at_row + (uint64_t)kp * S::STEP;
        uint32_t left = row_bytes - (kp < steps ? kp : steps - 1) * S::STEP, step = kp;
        if (kp < steps) in.fetch(places, a.down + off, behind + left, reach);
        for (uint32_t first = 0; first < steps; first += a.chunk) {
            const uint32_t now = first + a.chunk < steps ? a.chunk : steps - first, end = first + now;
            if (first || done) __syncthreads();
            stage_x<F, NC, CHAIN>(xs, now, tokens, 1, [&](uint32_t n, uint32_t t, uint32_t f, float (&v)[8]) {
                load8(a.h, pairs[done + t] * a.ff, ((uint64_t)(first + n) * 128 + f) * 8, a.ff, EK_F32, v);
            });
            __syncthreads();
            for (; step < end; step += a.ksplit) {
                wave_order();
                in.put(places, image);
                wave_order();
                const uint32_t here = left;
                if (step + a.ksplit < steps) {
                    off += (uint64_t)a.ksplit * S::STEP;
                    left -= a.ksplit * S::STEP;
                    in.fetch(places, a.down + off, behind + left, reach);
                }
                typename S::Raw raw[RT];
#pragma unroll
                for (int t = 0; t < RT; ++t) raw[t].load(image + (t * 4 + lane % 4) * I::ROW, me, here);
                const uint32_t at = (step - first) * X::BYTES;
                add_slices<F, NC, CHAIN, RT>(raw, me, x + at, sums + at, acc);
            }
        }
        __syncthreads();
        float *part = (float *)xs;
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float v = quads_sum(acc[t][c]);
                if (lane < 4) part[(wave * NC + c) * I::ROWS + t * 4 + lane] = v;
            }
        __syncthreads();
        if (threadIdx.x < groups * I::ROWS * tokens) {
            const uint32_t r = threadIdx.x % (groups * I::ROWS), t = threadIdx.x / (groups * I::ROWS), g = r / I::ROWS;
            float v = 0.0f;
            for (uint32_t k = 0; k < a.ksplit; ++k) v += part[((g * a.ksplit + k) * NC + t) * I::ROWS + r % I::ROWS];
            if (first_row + r < hidden) a.o[(uint64_t)pairs[done + t] * hidden + first_row + r] = v;
        }
    }
}
// ... and the sum over a token's experts, in order
__global__ __launch_bounds__(MV_THREADS) static void moe_sum(MoeArgs a) {
    const uint64_t r = (uint64_t)blockIdx.x * MV_THREADS + threadIdx.x;
    if (r >= a.hidden) return;
    const uint32_t t = blockIdx.y;
    float y = 0.0f;
    for (uint32_t j = 0; j < a.top_k; ++j) {
        const uint64_t pair = t * a.top_k + j;
        y = __builtin_fmaf(a.weights[pair], a.o[pair * a.hidden + r], y);
    }
    store_elem(a.y, t * a.y_stride + r, a.y_kind, y);
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
