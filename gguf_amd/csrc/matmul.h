// matmul.h -- products with packed weights: the kernels.
//
//     y[t][r] = sum over c of W[r][c] * x[t][c]        W packed blocks (formats.h), x and y f32 / f16 / bf16
//
// and what surrounds them in a decoding step: rows of a packed table by id, and a mixture-of-experts layer.
#pragma once
#include "formats.h"

namespace ggq {

// ---- packed bytes in global memory, at any alignment -----------------------------------------------------
// The same interface as LdsBytes, reading exactly the bytes that are asked for: the last block of a tensor may end
// at the end of an allocation.
typedef uint32_t u32_any __attribute__((aligned(1), may_alias));
typedef uint16_t u16_any __attribute__((aligned(1), may_alias));
struct GlobalBytes {
    const uint8_t *p;
    __device__ __forceinline__ uint32_t u32(uint32_t off) const { return *(const u32_any *)(p + off); }
    __device__ __forceinline__ uint32_t u16(uint32_t off) const { return *(const u16_any *)(p + off); }
    __device__ __forceinline__ uint32_t u8(uint32_t off) const { return p[off]; }
    template <int G>
    __device__ __forceinline__ void words(uint32_t off, uint32_t (&out)[G]) const {
#pragma unroll
        for (int g = 0; g < G; ++g) out[g] = u32(off + 4 * g);
    }
};

// The 16-bit floats as one-element block types
struct WF16 { static constexpr uint32_t N = 1, BYTES = 2; };
struct WBF16 { static constexpr uint32_t N = 1, BYTES = 2; };
template <class F> constexpr bool is_float_type = false;
template <> constexpr bool is_float_type<WF16> = true;
template <> constexpr bool is_float_type<WBF16> = true;

__device__ __forceinline__ float bf2f(uint32_t bits16) { return __builtin_bit_cast(float, bits16 << 16); }

enum ElemKind : uint32_t { EK_F32 = 0, EK_F16 = 1, EK_BF16 = 2 };

__device__ __forceinline__ float load_elem(const void *p, uint64_t i, uint32_t kind) {
    if (kind == EK_F32) return ((const float *)p)[i];
    const uint32_t b = ((const uint16_t *)p)[i];
    return kind == EK_F16 ? h2f(b) : bf2f(b);
}
// f32 to the output type, rounded to nearest even
__device__ __forceinline__ void store_elem(void *p, uint64_t i, uint32_t kind, float v) {
    if (kind == EK_F32) ((float *)p)[i] = v;
    else if (kind == EK_F16) ((_Float16 *)p)[i] = (_Float16)v;
    else ((__bf16 *)p)[i] = (__bf16)v;
}

// elements [c, c + 4) of a packed row of `cols` elements (c % 4 == 0; past the end of a float row: 0)
template <class F>
__device__ __forceinline__ void row4(const uint8_t *row, uint64_t c, uint64_t cols, float (&w)[4]) {
    if constexpr (is_float_type<F>) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t b = c + i < cols ? *(const u16_any *)(row + 2 * (c + i)) : 0u;
            w[i] = sizeof(F) && __is_same(F, WF16) ? h2f(b) : bf2f(b);
        }
    } else {
        const uint64_t b = c / F::N;
        F::dec4(GlobalBytes{row + b * F::BYTES}, 0u, (uint32_t)(c % F::N), w);
    }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

struct MatvecArgs {
    const uint8_t *w;
    const void *x;
    void *y;
    uint64_t rows, cols, tokens, x_stride, y_stride;
    uint32_t x_kind, y_kind;
};

constexpr uint32_t MV_THREADS = 256;

// one wave per row and token
template <class F>
__global__ __launch_bounds__(MV_THREADS) void matvec_rows(MatvecArgs a, uint64_t first_token) {
    const uint64_t r = (uint64_t)blockIdx.x * (MV_THREADS / 64) + threadIdx.x / 64;
    const uint64_t t = first_token + blockIdx.y;
    if (r >= a.rows) return;
    const uint8_t *row = a.w + r * (a.cols / F::N * F::BYTES);
    float sum = 0.0f;
    for (uint64_t c = 4 * (threadIdx.x % 64); c < a.cols; c += 256) {
        float w[4];
        row4<F>(row, c, a.cols, w);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < a.cols) sum = __builtin_fmaf(w[i], load_elem(a.x, t * a.x_stride + c + i, a.x_kind), sum);
    }
    sum = wave_sum(sum);
    if (threadIdx.x % 64 == 0) store_elem(a.y, t * a.y_stride + r, a.y_kind, sum);
}

// ---- rows by id -----------------------------------------------------------------------------------------
struct RowsArgs {
    const uint8_t *w;
    const void *ids;
    void *y;
    uint64_t rows, cols, n, y_stride, row_bytes;
    uint32_t y_kind, wide_ids;
};

__device__ __forceinline__ int64_t id_at(const RowsArgs &a, uint64_t i) {
    return a.wide_ids ? ((const int64_t *)a.ids)[i] : (int64_t)((const int32_t *)a.ids)[i];
}

// one thread per 4 elements
template <class F>
__global__ __launch_bounds__(MV_THREADS) void get_rows(RowsArgs a, uint64_t first, uint64_t pieces) {
    const uint64_t p = first + (uint64_t)blockIdx.x * MV_THREADS + threadIdx.x;
    const uint64_t i = p / pieces, c = (p - i * pieces) * 4;
    if (i >= a.n) return;
    const int64_t id = id_at(a, i);
    float w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (id >= 0 && (uint64_t)id < a.rows) row4<F>(a.w + (uint64_t)id * a.row_bytes, c, a.cols, w);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (c + j < a.cols) store_elem(a.y, i * a.y_stride + c + j, a.y_kind, w[j]);
}

// ---- mixture of experts ---------------------------------------------------------------------------------
struct MoeArgs {
    const uint8_t *gate, *up, *down;
    const void *router, *x;
    void *y;
    float *logits;        // [tokens][experts]
    int32_t *ids;         // [tokens][top_k]
    float *weights;       // [tokens][top_k]
    float *h;             // [tokens * top_k][ff]
    int32_t *out_ids;     // the caller's, or null
    float *out_weights;
    uint64_t hidden, ff, x_stride, y_stride;
    uint32_t tokens, experts, top_k, router_kind, x_kind, y_kind;
    uint32_t sigmoid, normalize, gelu;
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

// one wave per token
__global__ __launch_bounds__(64) static void moe_route(MoeArgs a) {
    const uint32_t t = blockIdx.x, lane = threadIdx.x;
    const float *l = a.logits + (uint64_t)t * a.experts;
    float top = -__builtin_inff();
    for (uint32_t e = lane; e < a.experts; e += 64) top = __builtin_fmaxf(top, l[e]);
    for (int m = 32; m; m >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, m));
    float total = 0.0f;
    if (!a.sigmoid) {
        for (uint32_t e = lane; e < a.experts; e += 64) total += expf(l[e] - top);
        total = wave_sum(total);
    }
    uint64_t last = ~0ull;
    float sum = 0.0f, mine = 0.0f;
    for (uint32_t j = 0; j < a.top_k; ++j) {
        uint64_t best = 0;
        for (uint32_t e = lane; e < a.experts; e += 64) {
            const uint64_t key = ((uint64_t)logit_key(l[e]) << 32) | (0xFFFFFFFFu - e);
            if (key < last && key > best) best = key;
        }
        for (int m = 32; m; m >>= 1) {
            const uint64_t other = __shfl_xor(best, m);
            if (other > best) best = other;
        }
        last = best;
        const uint32_t e = 0xFFFFFFFFu - (uint32_t)best;
        const float v = l[e], p = a.sigmoid ? 1.0f / (1.0f + expf(-v)) : expf(v - top) / total;
        sum += p;
        if (lane == j) mine = p;
        if (lane == 0) {
            a.ids[t * a.top_k + j] = (int32_t)e;
            if (a.out_ids) a.out_ids[t * a.top_k + j] = (int32_t)e;
        }
    }
    if (lane < a.top_k) {
        const float w = (a.normalize ? mine / sum : mine) * a.scale;
        a.weights[t * a.top_k + lane] = w;
        if (a.out_weights) a.out_weights[t * a.top_k + lane] = w;
    }
}

__device__ __forceinline__ float moe_act(float g, uint32_t gelu) {
    if (!gelu) return g / (1.0f + expf(-g));
    const float z = 0.7978845608028654f * (g + 0.044715f * g * g * g);
    return 0.5f * g * (1.0f + tanhf(z));
}

template <class F>
__device__ __forceinline__ float row_dot(const uint8_t *row, uint64_t cols, const void *x, uint64_t at, uint32_t kind) {
    float sum = 0.0f;
    for (uint64_t c = 4 * (threadIdx.x % 64); c < cols; c += 256) {
        float w[4];
        row4<F>(row, c, cols, w);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < cols) sum = __builtin_fmaf(w[i], load_elem(x, at + c + i, kind), sum);
    }
    return wave_sum(sum);
}

template <class F>
__global__ __launch_bounds__(MV_THREADS) void moe_up(MoeArgs a) {
    const uint64_t r = (uint64_t)blockIdx.x * (MV_THREADS / 64) + threadIdx.x / 64;
    if (r >= a.ff) return;
    const uint32_t pair = blockIdx.y, t = pair / a.top_k;
    const uint64_t e = (uint64_t)a.ids[pair];
    const float g = row_dot<F>(a.gate + (e * a.ff + r) * (a.hidden / F::N * F::BYTES), a.hidden, a.x, t * a.x_stride, a.x_kind);
    const float u = row_dot<F>(a.up + (e * a.ff + r) * (a.hidden / F::N * F::BYTES), a.hidden, a.x, t * a.x_stride, a.x_kind);
    if (threadIdx.x % 64 == 0) a.h[pair * a.ff + r] = moe_act(g, a.gelu) * u;
}

template <class FD>
__global__ __launch_bounds__(MV_THREADS) void moe_down(MoeArgs a) {
    const uint64_t r = (uint64_t)blockIdx.x * (MV_THREADS / 64) + threadIdx.x / 64;
    if (r >= a.hidden) return;
    const uint32_t t = blockIdx.y;
    float y = 0.0f;
    for (uint32_t j = 0; j < a.top_k; ++j) {
        const uint32_t pair = t * a.top_k + j;
        const uint64_t e = (uint64_t)a.ids[pair];
        const float d = row_dot<FD>(a.down + (e * a.hidden + r) * (a.ff / FD::N * FD::BYTES), a.ff, a.h, pair * a.ff, EK_F32);
        y = __builtin_fmaf(a.weights[pair], d, y);
    }
    if (threadIdx.x % 64 == 0) store_elem(a.y, t * a.y_stride + r, a.y_kind, y);
}

}  // namespace ggq
