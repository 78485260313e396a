// choice.h -- a mixture-of-experts layer (moe.h): what its kernels share, and the choice of experts.
#pragma once
#include "matmul.h"

namespace ggq {

constexpr uint32_t MOE_MAX_EXPERTS = 512, MOE_MAX_TOP_K = 32, MOE_MAX_TOKENS = 64;
constexpr uint32_t SLOT_TOKENS = 16;          // most tokens of one expert that a workgroup takes

// Experts in use, in the order of their index, each with its tokens a few at a time (MoeArgs::slot_tokens): a slot is one such
// group.
struct Slot {
    uint32_t expert, count;           // of tokens; 0: no such slot
    uint32_t pair[SLOT_TOKENS];       // of the tokens, in order: token * top_k + place
};

struct MoeArgs {
    const uint8_t *gate, *up, *down;
    const void *router, *x;
    void *y;
    float *logits;        // [tokens][experts]
    int32_t *ids;         // [tokens][top_k]
    float *weights;       // [tokens][top_k]
    float *h;             // [tokens * top_k][ff]
    float *o;             // [tokens * top_k][hidden]
    Slot *table;          // [slots]
    int32_t *out_ids;     // the caller's, or null
    float *out_weights;
    uint64_t hidden, ff, x_stride, y_stride;
    uint32_t tokens, experts, top_k, router_kind, x_kind, y_kind;
    uint32_t sigmoid, normalize, gelu;
    uint32_t ksplit, chunk;                   // as in MatvecArgs, of the launch
    uint32_t slots, slot_tokens;              // of the table: most there may be; most tokens of one
    uint32_t slots_expected;                  // where every expert is as likely
    float scale;
};

// an order-preserving key of a logit: larger logit, larger key; NaN below everything; -0 equals +0
__device__ __forceinline__ uint32_t logit_key(float v) {
    if (v != v) return 0u;
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// ---- the choice -----------------------------------------------------------------------------------------
// The top_k experts of a token, ids[j] = the j-th.  An expert's place is the number of experts in front of it (a larger key,
// or the same and a lower index), so all places are found at once, without a chain of k maxima; keys are read four at a
// time, the same for all lanes.  Threads `me`, me + threads, ... of `threads` share the work; `keys`: theirs, room for 512;
// order(): what makes their writes to shared memory seen.
template <class Order>
__device__ __forceinline__ void choose(const float *logits, uint32_t experts, uint32_t top_k, uint32_t me, uint32_t threads, uint32_t *keys, int32_t *ids,
                                       Order order) {
    const uint32_t padded = (experts + 3) & ~3u;
    for (uint32_t e = me; e < padded; e += threads) keys[e] = e < experts ? logit_key(logits[e]) : 0u;
    order();
    for (uint32_t e = me; e < experts; e += threads) {
        const uint32_t key = keys[e];
        uint32_t place = 0;
#pragma unroll 4
        for (uint32_t q = 0; q < padded; q += 4) {
            const u32x4 k = *(const u32x4 *)(keys + q);
#pragma unroll
            for (int i = 0; i < 4; ++i) place += (k[i] > key) || (k[i] == key && q + i < e);
        }
        if (place < top_k) ids[place] = (int32_t)e;
    }
    order();
}

__device__ __forceinline__ float wave_max(float v) {
    v = __builtin_fmaxf(v, dpp<QUAD_XOR1>(v));
    v = __builtin_fmaxf(v, dpp<QUAD_XOR2>(v));
    v = __builtin_fmaxf(v, dpp<ROW_ROR4>(v));
    v = __builtin_fmaxf(v, dpp<ROW_ROR8>(v));
    v = __builtin_fmaxf(v, __shfl_xor(v, 16));
    return __builtin_fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float wave_total(float v) {
    v += dpp<QUAD_XOR1>(v);
    v += dpp<QUAD_XOR2>(v);
    v += dpp<ROW_ROR4>(v);
    v += dpp<ROW_ROR8>(v);
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
// One wave: the choice of token t and its weights to the workspace and to the caller.
__device__ __forceinline__ void put_choice(const MoeArgs &a, uint32_t t, const int32_t *ids, uint32_t lane) {
    const float *l = a.logits + (uint64_t)t * a.experts;
    float top = -__builtin_inff(), total = 0.0f;
    if (!a.sigmoid) {
        for (uint32_t e = lane; e < a.experts; e += 64) top = __builtin_fmaxf(top, l[e]);
        top = wave_max(top);
        for (uint32_t e = lane; e < a.experts; e += 64) total += expf(l[e] - top);
        total = wave_total(total);
    }
    float p = 0.0f;
    if (lane < a.top_k) {
        const float v = l[ids[lane]];
        p = a.sigmoid ? 1.0f / (1.0f + expf(-v)) : expf(v - top) / total;
    }
    const float sum = wave_total(p);
    if (lane < a.top_k) {
        const uint32_t at = t * a.top_k + lane;
        const float w = (a.normalize ? p / sum : p) * a.scale;
        a.ids[at] = ids[lane];
        a.weights[at] = w;
        if (a.out_ids) a.out_ids[at] = ids[lane];
        if (a.out_weights) a.out_weights[at] = w;
    }
}

}  // namespace ggq
