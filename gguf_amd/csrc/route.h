// route.h -- a mixture-of-experts layer (moe.h): the kernels that have nothing to do with packed weights.
#pragma once
#include "choice.h"

namespace ggq {

// ---- logits ---------------------------------------------------------------------------------------------
// four elements from c on, 0 past the end
__device__ __forceinline__ void floats4(const void *p, uint64_t at, uint32_t c, uint32_t n, uint32_t kind, float (&v)[4]) {
    if (c + 4 <= n && kind == EK_F32) {
        const f32x4 a = __builtin_bit_cast(f32x4, ld16((const uint8_t *)p + 4 * (at + c)));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i];
    } else if (c + 4 <= n) {
        const uint8_t *q = (const uint8_t *)p + 2 * (at + c);
        const uint32_t a = ld4(q), b = ld4(q + 4);
        v[0] = kind == EK_F16 ? h2f(a & 0xFFFFu) : bf2f(a & 0xFFFFu);
        v[1] = kind == EK_F16 ? h2f(a >> 16) : bf2f(a >> 16);
        v[2] = kind == EK_F16 ? h2f(b & 0xFFFFu) : bf2f(b & 0xFFFFu);
        v[3] = kind == EK_F16 ? h2f(b >> 16) : bf2f(b >> 16);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = c + i < n ? load_elem(p, at + c + i, kind) : 0.0f;
    }
}
// ... as they lie in memory (16-bit ones in the first two words), and the values of those
__device__ __forceinline__ u32x4 load4(const void *p, uint64_t at, uint32_t c, uint32_t n, uint32_t kind) {
    u32x4 v = {0, 0, 0, 0};
    if (kind == EK_F32) {
        const uint8_t *q = (const uint8_t *)p + 4 * (at + c);
        if (c + 4 <= n) return ld16(q);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) v[i] = c + i < n ? ld4(q + 4 * i) : 0u;
    } else {
        const uint8_t *q = (const uint8_t *)p + 2 * (at + c);
        if (c + 4 <= n) {
            v[0] = ld4(q);
            v[1] = ld4(q + 4);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) v[i / 2] |= c + i < n ? ld2(q + 2 * i) << (16 * (i % 2)) : 0u;
        }
    }
    return v;
}
__device__ __forceinline__ void values4(const u32x4 &w, uint32_t kind, double (&v)[4]) {
    const uint32_t w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3], h[4] = {w0 & 0xFFFFu, w0 >> 16, w1 & 0xFFFFu, w1 >> 16}, f[4] = {w0, w1, w2, w3};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (double)(kind == EK_F32 ? __builtin_bit_cast(float, f[i]) : kind == EK_F16 ? h2f(h[i]) : bf2f(h[i]));
}
// One expert and T tokens a workgroup; grid: (experts, tokens / T).  The choice hangs on the order of the logits, so
// products (exact in 64 bits) are summed in 64 bits and rounded once.  Bound by its latency: 4 KiB of the router are on the
// way at once in each workgroup, and as much of each token's x.  128 experts of 2048 by 16 tokens, T = 4: 7.4 us (9.0 with one
// token's x on the way after the other's); 64 by one token, T = 1: 4.3.
constexpr uint32_t LOGIT_TOKENS = 4;
template <uint32_t T>
__global__ __launch_bounds__(MV_THREADS) void moe_logits(MoeArgs a) {
    __shared__ double part[T][MV_THREADS];
    const uint32_t e = blockIdx.x, first = blockIdx.y * T, n = (uint32_t)a.hidden;
    const uint32_t tokens = a.tokens - first < T ? a.tokens - first : T;
    double sum[T] = {};
    for (uint32_t c = threadIdx.x * 4; c < n; c += MV_THREADS * 16) {
        if constexpr (T == 1) {
            // values as they are loaded: by way of the words, as below, a layer's call takes 0.3 to 0.5 us more (20.6 -> 20.9, 56.1 -> 56.6)
            float w[4][4], x[4][4];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) floats4(a.router, e * a.hidden, c + k * MV_THREADS * 4, n, a.router_kind, w[k]);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) floats4(a.x, first * a.x_stride, c + k * MV_THREADS * 4, n, a.x_kind, x[k]);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[0] = __builtin_fma((double)w[k][i], (double)x[k][i], sum[0]);
        } else {
            // all tokens' x on the way before the first is used
            u32x4 w[4], x[T][4];
            const uint32_t parts = (n - c + MV_THREADS * 4 - 1) / (MV_THREADS * 4);      // of this thread; beyond: nothing to load
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
                if (k < parts) {
                    w[k] = load4(a.router, e * a.hidden, c + k * MV_THREADS * 4, n, a.router_kind);
#pragma unroll
                    for (uint32_t t = 0; t < T; ++t)
                        if (t < tokens) x[t][k] = load4(a.x, (first + t) * a.x_stride, c + k * MV_THREADS * 4, n, a.x_kind);
                }
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
                if (k < parts) {
                    double wv[4], xv[4];
                    values4(w[k], a.router_kind, wv);
#pragma unroll
                    for (uint32_t t = 0; t < T; ++t)
                        if (t < tokens) {
                            values4(x[t][k], a.x_kind, xv);
#pragma unroll
                            for (int i = 0; i < 4; ++i) sum[t] = __builtin_fma(wv[i], xv[i], sum[t]);
                        }
                }
        }
    }
#pragma unroll
    for (uint32_t t = 0; t < T; ++t) part[t][threadIdx.x] = sum[t];
    __syncthreads();
    const uint32_t t = threadIdx.x / 64, lane = threadIdx.x % 64;         // a wave for each token
    if (t >= tokens) return;
    double s = (part[t][lane] + part[t][lane + 64]) + (part[t][lane + 128] + part[t][lane + 192]);
#pragma unroll
    for (int m = 32; m; m >>= 1) s += __shfl_xor(s, m);
    if (lane == 0) a.logits[(uint64_t)(first + t) * a.experts + e] = (float)s;
}

// ---- several tokens: the choices and the slots --------------------------------------------------------------
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    auto larger = [](uint32_t p, uint32_t q) { return p > q ? p : q; };
    v = larger(v, dpp<QUAD_XOR1>(v));
    v = larger(v, dpp<QUAD_XOR2>(v));
    v = larger(v, dpp<ROW_ROR4>(v));
    v = larger(v, dpp<ROW_ROR8>(v));
    v = larger(v, (uint32_t)__shfl_xor((int)v, 16));
    return larger(v, (uint32_t)__shfl_xor((int)v, 32));
}
// As choose, by one wave with the keys in its registers: a maximum after the other.  With the waves of 16 tokens on one CU the
// chains hide each other, while comparing each expert with each keeps its vector units busy: with 128 experts, 8 chosen, the launch
// takes 9.0 us instead of 14.5.
__device__ __forceinline__ void choose_maxima(const float *logits, uint32_t experts, uint32_t top_k, uint32_t lane, int32_t *ids) {
    constexpr uint32_t EACH = MOE_MAX_EXPERTS / 64;
    uint32_t key[EACH];                                    // of expert 64 i + lane; 0: taken, or none
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) {
        const uint32_t e = 64 * i + lane;
        key[i] = 0;
        if (e < experts) {
            const uint32_t k = logit_key(logits[e]);
            key[i] = k ? k : 1u;                           // NaN; the key of -infinity is larger
        }
    }
    for (uint32_t j = 0; j < top_k; ++j) {
        uint32_t best = key[0], at = 0;
#pragma unroll
        for (uint32_t i = 1; i < EACH; ++i) {
            at = key[i] > best ? i : at;
            best = key[i] > best ? key[i] : best;
        }
        const uint32_t top = wave_max_u32(best);
        // the lowest index among equals
        const uint32_t mine = best == top ? ~(64 * at + lane) : 0u, e = ~wave_max_u32(mine);
#pragma unroll
        for (uint32_t i = 0; i < EACH; ++i) key[i] = 64 * i + lane == e ? 0u : key[i];
        if (lane == 0) ids[j] = (int32_t)e;
    }
    wave_order();
}
// One workgroup: its waves take the tokens, then its threads the experts and the pairs.  The kernels of gate, up and down find
// their slot in a table.  Where each of their workgroups looked for its own, down of 128 experts, 8 chosen, 2048/768 by 16 tokens
// took 51 us instead of 39 (with three pieces of h, as now, 45).
constexpr uint32_t ROUTE_WAVES = 16;
__global__ __launch_bounds__(ROUTE_WAVES * 64) static void moe_route(MoeArgs a) {
    __shared__ int32_t ids[MOE_MAX_TOKENS * MOE_MAX_TOP_K];
    __shared__ uint32_t low[MOE_MAX_EXPERTS], high[MOE_MAX_EXPERTS], first[MOE_MAX_EXPERTS], of_wave[ROUTE_WAVES];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, pairs = a.tokens * a.top_k;
    static_assert(ROUTE_WAVES * 64 >= MOE_MAX_EXPERTS, "a thread for each expert");
    if (threadIdx.x < MOE_MAX_EXPERTS) low[threadIdx.x] = high[threadIdx.x] = 0;
    for (uint32_t t = wave; t < a.tokens; t += ROUTE_WAVES) {
        int32_t *of_token = ids + t * a.top_k;
        choose_maxima(a.logits + (uint64_t)t * a.experts, a.experts, a.top_k, lane, of_token);
        put_choice(a, t, of_token, lane);
    }
    __syncthreads();
    for (uint32_t p = threadIdx.x; p < pairs; p += ROUTE_WAVES * 64) {
        const uint32_t t = p / a.top_k;
        atomicOr(t < 32 ? &low[ids[p]] : &high[ids[p]], 1u << (t & 31));
    }
    __syncthreads();
    // slots in front of each expert's
    const uint32_t tokens = threadIdx.x < MOE_MAX_EXPERTS ? (uint32_t)__popc(low[threadIdx.x]) + (uint32_t)__popc(high[threadIdx.x]) : 0u;
    const uint32_t mine = (tokens + a.slot_tokens - 1) / a.slot_tokens;
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(upto, d);
        upto += lane >= (uint32_t)d ? o : 0u;
    }
    if (lane == 63) of_wave[wave] = upto;
    __syncthreads();
    uint32_t front = upto - mine, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < ROUTE_WAVES; ++w) {
        front += w < wave ? of_wave[w] : 0u;
        total += of_wave[w];
    }
    if (threadIdx.x < MOE_MAX_EXPERTS) first[threadIdx.x] = front;
    for (uint32_t k = 0; k < mine; ++k) {
        a.table[front + k].expert = threadIdx.x;
        a.table[front + k].count = tokens - k * a.slot_tokens < a.slot_tokens ? tokens - k * a.slot_tokens : a.slot_tokens;
    }
    for (uint32_t k = total + threadIdx.x; k < a.slots; k += ROUTE_WAVES * 64) a.table[k].count = 0;
    __syncthreads();
    for (uint32_t p = threadIdx.x; p < pairs; p += ROUTE_WAVES * 64) {
        const uint32_t t = p / a.top_k, e = (uint32_t)ids[p];
        const uint64_t mask = low[e] | ((uint64_t)high[e] << 32);
        const uint32_t place = (uint32_t)__popcll(mask & ((1ull << t) - 1));
        a.table[first[e] + place / a.slot_tokens].pair[place % a.slot_tokens] = p;
    }
}

// ---- the sum over a token's experts, in order; where down left it apart ---------------------------------------
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

}  // namespace ggq
