// route.h -- a mixture-of-experts layer (moe.h): the kernels that have nothing to do with packed weights.
#pragma once
#include "choice.h"

namespace ggq {

// ---- logits ---------------------------------------------------------------------------------------------
// four elements from c on, 0 past the end
__device__ __forceinline__ void load4(const void *p, uint64_t at, uint32_t c, uint32_t n, uint32_t kind, float (&v)[4]) {
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
// One expert and four tokens a workgroup; grid: (experts, tokens / 4).  The choice hangs on the order of the logits, so
// products (exact in 64 bits) are summed in 64 bits and rounded once.  Bound by its latency: 4 KiB of the router are on the
// way at once in each workgroup, and the token's x with them.
constexpr uint32_t LOGIT_TOKENS = 4;
__global__ __launch_bounds__(MV_THREADS) static void moe_logits(MoeArgs a) {
    __shared__ double part[LOGIT_TOKENS][MV_THREADS];
    const uint32_t e = blockIdx.x, first = blockIdx.y * LOGIT_TOKENS, n = (uint32_t)a.hidden;
    const uint32_t tokens = a.tokens - first < LOGIT_TOKENS ? a.tokens - first : LOGIT_TOKENS;
    double sum[LOGIT_TOKENS] = {0.0, 0.0, 0.0, 0.0};
    for (uint32_t c = threadIdx.x * 4; c < n; c += MV_THREADS * 16) {
        float w[4][4];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) load4(a.router, e * a.hidden, c + k * MV_THREADS * 4, n, a.router_kind, w[k]);
#pragma unroll
        for (uint32_t t = 0; t < LOGIT_TOKENS; ++t) {
            if (t >= tokens) break;
            float x[4][4];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) load4(a.x, (first + t) * a.x_stride, c + k * MV_THREADS * 4, n, a.x_kind, x[k]);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[t] = __builtin_fma((double)w[k][i], (double)x[k][i], sum[t]);
        }
    }
#pragma unroll
    for (uint32_t t = 0; t < LOGIT_TOKENS; ++t) part[t][threadIdx.x] = sum[t];
    __syncthreads();
    const uint32_t t = threadIdx.x / 64, lane = threadIdx.x % 64;         // a wave for each token
    if (t >= tokens) return;
    double s = (part[t][lane] + part[t][lane + 64]) + (part[t][lane + 128] + part[t][lane + 192]);
#pragma unroll
    for (int m = 32; m; m >>= 1) s += __shfl_xor(s, m);
    if (lane == 0) a.logits[(uint64_t)(first + t) * a.experts + e] = (float)s;
}

// The choice of all tokens, a workgroup for each
__global__ __launch_bounds__(MV_THREADS) static void moe_route(MoeArgs a) {
    __shared__ uint32_t keys[MOE_MAX_EXPERTS];
    __shared__ int32_t ids[MOE_MAX_TOP_K];
    const uint32_t t = blockIdx.x;
    choose(a.logits + (uint64_t)t * a.experts, a.experts, a.top_k, threadIdx.x, MV_THREADS, keys, ids, [] { __syncthreads(); });
    if (threadIdx.x < 64) put_choice(a, t, ids, threadIdx.x);
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
