// dense.h -- two to sixteen tokens at once: products with packed weights (matmul.h).
//
// With several tokens the matrix unit's rows are tokens: v_mfma_f32_16x16x32_bf16 multiplies 32 codes of 16 rows, one
// sub-block, with 16 tokens (16x16x16 for sub-blocks of 16).  Codes are turned into bf16, which holds every code exactly (two at
// a time by v_cvt_scalef32_pk_bf16_fp8 where they are below 16: an e4m3 byte of 0..15 times 2^9 is itself).  x goes in as bf16,
// in pieces where its type is wider: three of f32, exactly; f16 goes in as it is, with codes as f16.  Lane (n, g), n = lane % 16,
// g = lane / 16, brings the codes k = 8 g .. 8 g + 7 (4 g .. 4 g + 3) of row n and receives the sums of tokens 4 g .. 4 g + 3,
// which it scales: a multiply-add for each eight codes and token.  The offsets' part, sum over sub-blocks of c times the sum of x,
// is a product too: the sums come from a multiplication with ones, and v_mfma_f32_16x16x4_f32 adds them up in f32.  The scales of
// 256 columns are unpacked once, each lane a quarter of its row's, and handed round through shared memory.
//
// Bound by the vector instructions that unpack and scale (about 150 for 256 columns of 16 rows), and for few rows by the time
// that a workgroup takes to begin and end.  Against all waves of a workgroup staging x for each other: q4_k 11008 x 4096 by 16
// tokens (bf16) 11.4 against 20.5 us, q6_k 15.5 against 36.8.  Against one token's digits (matmul.h): q4_k 28672 x 8192 by one
// token 33 (bf16) and 59 (f32) against 27 us, so one token is left to those.
#pragma once
#include "matmul.h"

namespace ggq {

// A format's step (256 elements of a row, its image in shared memory) as this tile takes it:
//     SUB, OFFSET       elements of a sub-block, whether c can differ from zero
//     scale(row, g, left, out)   {a, c} of the sub-blocks g * N .. g * N + N - 1, N = 64 / SUB; 0 behind the row's end
//     codes(row, s, g, b)        sub-block s: the lane's 8 codes (SUB 32) or 4 (SUB 16) as bf16
template <class F> struct Step;

// four codes (bytes of w) -> two words of two bf16, or of two f16 (H): both hold every code exactly
template <bool H>
__device__ __forceinline__ uint32_t pair_of(float lo, float hi) {
    if constexpr (H) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(lo, hi));
    else return upper_halves(lo, hi);
}
// ... below 16
template <bool H>
__device__ __forceinline__ void small_codes(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if constexpr (H) {
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 512.0f, false));
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 512.0f, true));
    } else {
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 512.0f, false));
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 512.0f, true));
    }
}
template <bool H>
__device__ __forceinline__ void byte_codes(uint32_t w, uint32_t &lo, uint32_t &hi) {
    w = opaque(w);
    lo = pair_of<H>(ub<0>(w), ub<1>(w));
    hi = pair_of<H>(ub<2>(w), ub<3>(w));
}
template <bool H>
__device__ __forceinline__ void signed_codes(uint32_t w, uint32_t &lo, uint32_t &hi) {
    w = opaque(w);
    lo = pair_of<H>(sb<0>(w), sb<1>(w));
    hi = pair_of<H>(sb<2>(w), sb<3>(w));
}
template <bool H>
__device__ __forceinline__ void iq4_codes(uint32_t nibbles, uint32_t &lo, uint32_t &hi) { signed_codes<H>(iq4_lookup4(nibbles) ^ 0x80808080u, lo, hi); }

// ---- 32-element formats: sub-block s is block s of the step, at byte s * B -----------------------------------
template <uint32_t B>
struct StepOfBlocks {
    static constexpr int SUB = 32;
    static __device__ __forceinline__ uint32_t live(uint32_t s, uint32_t left) { return in_row((s + 1) * B, left); }
    // the words at bytes AT and AT + 4 of block s; s is a constant once the loop over it is unrolled
    static __device__ __forceinline__ void two_words(const uint8_t *row, uint32_t at, bool odd, uint32_t (&w)[2]) {
        if (!odd) {
            w[0] = al4(row + at);
            w[1] = al4(row + at + 4);
        } else {                                   // two bytes beyond a whole word
            const uint32_t a = al4(row + at - 2), b = al4(row + at + 2), c = al4(row + at + 6);
            w[0] = funnel16(b, a);
            w[1] = funnel16(c, b);
        }
    }
    // bytes 8 (g % 2) .. of the nibbles at byte HEAD of the block, the half of each that lane g's codes are in
    template <uint32_t HEAD>
    static __device__ __forceinline__ void nibbles(const uint8_t *row, uint32_t s, uint32_t g, uint32_t (&w)[2]) {
        two_words(row, s * B + HEAD + 8 * (g & 1), (s * B + HEAD) % 4 != 0, w);
#pragma unroll
        for (int i = 0; i < 2; ++i) w[i] = (w[i] >> (4 * (g >> 1))) & LOW4;
    }
    // the fifth bits of lane g's codes
    template <uint32_t HEAD>
    static __device__ __forceinline__ void with_fifth(const uint8_t *row, uint32_t s, uint32_t g, uint32_t (&w)[2]) {
        nibbles<HEAD + 4>(row, s, g, w);
        const uint32_t bits = row[s * B + HEAD + g];
        w[0] |= spread4(bits) << 4;
        w[1] |= spread4(bits >> 4) << 4;
    }
};
#define GGQ_STEP_SCALES(N) static __device__ __forceinline__ void scale(const uint8_t *row, uint32_t g, uint32_t left, SubScale (&out)[N])
#define GGQ_STEP_CODES(N) template <bool H> static __device__ __forceinline__ void codes(const uint8_t *row, uint32_t s, uint32_t g, uint32_t (&b)[N])
// {d, c(d)} of blocks 2 g and 2 g + 1 with a half at their begin; {d, m} with two
#define GGQ_BLOCK_SCALES(EXPR_C)                                                        \
    GGQ_STEP_SCALES(2) {                                                                \
        _Pragma("unroll") for (uint32_t k = 0; k < 2; ++k) {                            \
            const uint32_t s = 2 * g + k, on = live(s, left);                           \
            const uint8_t *p = row + s * BYTES;                                         \
            const float d = h2f(al2(p) & on);                                           \
            out[k] = {d, EXPR_C};                                                       \
        }                                                                               \
    }
template <> struct Step<Q4_0> : StepOfBlocks<18> {
    static constexpr bool OFFSET = true;
    static constexpr uint32_t BYTES = 18;
    GGQ_BLOCK_SCALES(8.0f * d)
    GGQ_STEP_CODES(4) {
        uint32_t w[2];
        nibbles<2>(row, s, g, w);
        small_codes<H>(w[0], b[0], b[1]);
        small_codes<H>(w[1], b[2], b[3]);
    }
};
template <> struct Step<Q4_1> : StepOfBlocks<20> {
    static constexpr bool OFFSET = true;
    static constexpr uint32_t BYTES = 20;
    GGQ_BLOCK_SCALES(-h2f(al2(p + 2) & on))
    GGQ_STEP_CODES(4) {
        uint32_t w[2];
        nibbles<4>(row, s, g, w);
        small_codes<H>(w[0], b[0], b[1]);
        small_codes<H>(w[1], b[2], b[3]);
    }
};
template <> struct Step<Q5_0> : StepOfBlocks<22> {
    static constexpr bool OFFSET = true;
    static constexpr uint32_t BYTES = 22;
    GGQ_BLOCK_SCALES(16.0f * d)
    GGQ_STEP_CODES(4) {
        uint32_t w[2];
        with_fifth<2>(row, s, g, w);
        byte_codes<H>(w[0], b[0], b[1]);
        byte_codes<H>(w[1], b[2], b[3]);
    }
};
template <> struct Step<Q5_1> : StepOfBlocks<24> {
    static constexpr bool OFFSET = true;
    static constexpr uint32_t BYTES = 24;
    GGQ_BLOCK_SCALES(-h2f(al2(p + 2) & on))
    GGQ_STEP_CODES(4) {
        uint32_t w[2];
        with_fifth<4>(row, s, g, w);
        byte_codes<H>(w[0], b[0], b[1]);
        byte_codes<H>(w[1], b[2], b[3]);
    }
};
template <uint32_t B, uint32_t HEAD>
struct StepOfBytes : StepOfBlocks<B> {
    static constexpr uint32_t BYTES = B;
    template <bool H>
    static __device__ __forceinline__ void codes(const uint8_t *row, uint32_t s, uint32_t g, uint32_t (&b)[4]) {
        uint32_t w[2];
        StepOfBlocks<B>::two_words(row, s * B + HEAD + 8 * g, (s * B + HEAD) % 4 != 0, w);
        signed_codes<H>(w[0], b[0], b[1]);
        signed_codes<H>(w[1], b[2], b[3]);
    }
};
template <> struct Step<Q8_0> : StepOfBytes<34, 2> {
    static constexpr bool OFFSET = false;
    GGQ_BLOCK_SCALES(0.0f)
};
template <> struct Step<Q8_1> : StepOfBytes<36, 4> {
    static constexpr bool OFFSET = false;
    GGQ_BLOCK_SCALES(0.0f)
};
template <> struct Step<IQ4NL> : StepOfBlocks<18> {
    static constexpr bool OFFSET = false;
    static constexpr uint32_t BYTES = 18;
    GGQ_BLOCK_SCALES(0.0f)
    GGQ_STEP_CODES(4) {
        uint32_t w[2];
        nibbles<2>(row, s, g, w);
        iq4_codes<H>(w[0], b[0], b[1]);
        iq4_codes<H>(w[1], b[2], b[3]);
    }
};

// ---- 256-element formats: the step is a block ----------------------------------------------------------------
template <> struct Step<Q4K> {
    static constexpr bool OFFSET = true;
    static constexpr int SUB = 32;
    GGQ_STEP_SCALES(2) {
        const u32x4 h = al16(row);
        const uint32_t dm = h[0] & in_row(144, left);
        const PairOfK4 k = scales_k4(h[1], h[2], h[3], g);
        const float d = h2f(dm & 0xFFFFu), m = h2f(dm >> 16);
        out[0] = {d * ub<0>(k.sc), m * ub<0>(k.mn)};
        out[1] = {d * ub<1>(k.sc), m * ub<1>(k.mn)};
    }
    GGQ_STEP_CODES(4) {
        const u32x2 q = al8(row + 16 + 32 * (s >> 1) + 8 * g);
        small_codes<H>((q[0] >> (4 * (s & 1))) & LOW4, b[0], b[1]);
        small_codes<H>((q[1] >> (4 * (s & 1))) & LOW4, b[2], b[3]);
    }
};
template <> struct Step<Q5K> {
    static constexpr bool OFFSET = true;
    static constexpr int SUB = 32;
    GGQ_STEP_SCALES(2) {
        const u32x4 h = al16(row);
        const uint32_t dm = h[0] & in_row(176, left);
        const PairOfK4 k = scales_k4(h[1], h[2], h[3], g);
        const float d = h2f(dm & 0xFFFFu), m = h2f(dm >> 16);
        out[0] = {d * ub<0>(k.sc), m * ub<0>(k.mn)};
        out[1] = {d * ub<1>(k.sc), m * ub<1>(k.mn)};
    }
    GGQ_STEP_CODES(4) {
        const u32x2 q = al8(row + 48 + 32 * (s >> 1) + 8 * g), f = al8(row + 16 + 8 * g);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            byte_codes<H>(((q[i] >> (4 * (s & 1))) & LOW4) | (((f[i] >> s) & 0x01010101u) << 4), b[2 * i], b[2 * i + 1]);
    }
};
template <> struct Step<IQ4XS> {
    static constexpr bool OFFSET = false;
    static constexpr int SUB = 32;
    GGQ_STEP_SCALES(2) {
        const u32x2 h = al8(row);
        const float d = h2f(h[0] & 0xFFFFu & in_row(136, left));
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k) {
            const uint32_t ls = ((h[1] >> (8 * g + 4 * k)) & 0xFu) | (((h[0] >> (16 + 4 * g + 2 * k)) & 3u) << 4);
            out[k] = {d * (float)((int)ls - 32), 0.0f};
        }
    }
    GGQ_STEP_CODES(4) {
        const u32x2 q = al8(row + 8 + 16 * s + 8 * (g & 1));
        iq4_codes<H>((q[0] >> (4 * (g >> 1))) & LOW4, b[0], b[1]);
        iq4_codes<H>((q[1] >> (4 * (g >> 1))) & LOW4, b[2], b[3]);
    }
};
template <> struct Step<Q8K> {
    static constexpr bool OFFSET = false;
    static constexpr int SUB = 32;
    GGQ_STEP_SCALES(2) {
        const float d = h2f(al2(row) & in_row(290, left));
        out[0] = out[1] = {d, 0.0f};
    }
    GGQ_STEP_CODES(4) {
        const uint8_t *p = row + 32 * s + 8 * g;             // the codes begin two bytes behind
        const u32x2 q = al8(p);
        const uint32_t over = al4(p + 8);
        signed_codes<H>(funnel16(q[1], q[0]), b[0], b[1]);
        signed_codes<H>(funnel16(over, q[1]), b[2], b[3]);
    }
};
// sub-blocks of 16: s = 8 n + 2 p + h, elements 128 n + 32 p + 16 h + 0..15; lane g the elements 4 g .. of them
template <> struct Step<Q6K> {
    static constexpr bool OFFSET = true;
    static constexpr int SUB = 16;
    GGQ_STEP_SCALES(4) {
        const float d = h2f(al2(row + 208) & in_row(210, left));
        const uint32_t sc = al4(row + 192 + 4 * g);
        const float a[4] = {d * sb<0>(sc), d * sb<1>(sc), d * sb<2>(sc), d * sb<3>(sc)};
#pragma unroll
        for (int k = 0; k < 4; ++k) out[k] = {a[k], 32.0f * a[k]};
    }
    GGQ_STEP_CODES(2) {
        const uint32_t n = s >> 3, p = (s >> 1) & 3, h = s & 1;
        const uint32_t low = (al4(row + 64 * n + 32 * (p & 1) + 16 * h + 4 * g) >> (4 * (p >> 1))) & LOW4;
        const uint32_t high = (al4(row + 128 + 32 * n + 16 * h + 4 * g) >> (2 * p)) & 0x03030303u;
        byte_codes<H>(low | (high << 4), b[0], b[1]);
    }
};
template <> struct Step<Q2K> {
    static constexpr bool OFFSET = true;
    static constexpr int SUB = 16;
    GGQ_STEP_SCALES(4) {
        const uint32_t dm = al4(row + 80) & in_row(84, left), sc = al4(row + 4 * g);
        const float d = h2f(dm & 0xFFFFu), m = h2f(dm >> 16);
        const uint32_t lo = sc & LOW4, hi = (sc >> 4) & LOW4;
        out[0] = {d * ub<0>(lo), m * ub<0>(hi)};
        out[1] = {d * ub<1>(lo), m * ub<1>(hi)};
        out[2] = {d * ub<2>(lo), m * ub<2>(hi)};
        out[3] = {d * ub<3>(lo), m * ub<3>(hi)};
    }
    GGQ_STEP_CODES(2) {
        const uint32_t n = s >> 3, p = (s >> 1) & 3, h = s & 1;
        small_codes<H>((al4(row + 16 + 32 * n + 16 * h + 4 * g) >> (2 * p)) & 0x03030303u, b[0], b[1]);
    }
};
template <> struct Step<Q3K> {
    static constexpr bool OFFSET = true;
    static constexpr int SUB = 16;
    GGQ_STEP_SCALES(4) {
        const float d = h2f(al2(row + 108) & in_row(110, left));
        // scales 4 g .. 4 g + 3: nibbles of word g % 2 (high ones for g >= 2), top bits 2 g.. of the third word's bytes
        const uint32_t lo = (al4(row + 96 + 4 * (g & 1)) >> (4 * (g >> 1))) & LOW4, hi = (al4(row + 104) >> (2 * g)) & 0x03030303u;
        const uint32_t sc = lo | (hi << 4);
        const float a[4] = {d * (ub<0>(sc) - 32.0f), d * (ub<1>(sc) - 32.0f), d * (ub<2>(sc) - 32.0f), d * (ub<3>(sc) - 32.0f)};
#pragma unroll
        for (int k = 0; k < 4; ++k) out[k] = {a[k], 4.0f * a[k]};
    }
    GGQ_STEP_CODES(2) {
        const uint32_t n = s >> 3, p = (s >> 1) & 3, h = s & 1;
        const uint32_t low = (al4(row + 32 + 32 * n + 16 * h + 4 * g) >> (2 * p)) & 0x03030303u;
        const uint32_t high = (al4(row + 16 * h + 4 * g) >> (4 * n + p)) & 0x01010101u;
        small_codes<H>(low | (high << 2), b[0], b[1]);
    }
};

// ---- 16-bit floats: no scales; a half in two pieces ----------------------------------------------------------
template <class F>
struct StepOfFloats {
    static constexpr int SUB = 32;
    static constexpr bool OFFSET = false;
    // elements 32 s + 8 g .. + 7; what lies behind the row may be anything, an infinity too
    static __device__ __forceinline__ u32x4 load(const uint8_t *row, uint32_t s, uint32_t g, uint32_t left) {
        const uint32_t at = 64 * s + 16 * g;
        u32x4 v = al16(row + at);
        if (left < 512) {
            const uint32_t n = left > at ? (left - at) / 2 : 0;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) v[i] &= 2 * i + 1 < n ? ~0u : 2 * i < n ? 0xFFFFu : 0u;
        }
        return v;
    }
};
template <> struct Step<WF16> : StepOfFloats<WF16> {};
template <> struct Step<WBF16> : StepOfFloats<WBF16> {};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// How x goes into the matrix unit: its type, and the bf16 pieces that a value is cut into
enum XForm : int { X_BF16, X_F16, X_F32 };

// Up to 16 tokens times R tiles of 16 rows.  A wave takes whole turns, 256 columns of all its rows and tokens, and nobody else
// needs that part of x: it lies in the wave's own shared memory, as it comes from global memory, beside the images of its
// tiles, and the waves of a workgroup meet only to add up their sums.  A fragment of x is read and cut into pieces once for
// the R tiles.
template <class F, int X, int R>
struct DenseTile {
    typedef Step<F> S;
    static constexpr uint32_t TILES = R, ROWS = 16, ELEMS = 256, TOKENS = 16;
    typedef Image<F, ROWS, 1> I;
    static constexpr bool WIDE = X == X_F32;
    static constexpr bool H = X == X_F16 && !__is_same(F, WBF16);                           // f16 as it is
    static constexpr int P = X == X_BF16 || H ? 1 : WIDE ? 3 : 2;
    static constexpr uint32_t SUBS = 256 / S::SUB, EACH = SUBS / 4, N = S::SUB / 4;        // N: elements of a lane's fragment
    static constexpr uint32_t X_SIZE = WIDE ? 4 : 2, X_ROW = 256 * X_SIZE + 16;              // an odd number of 16-byte places
    static constexpr uint32_t X_LOADS = WIDE ? TOKENS : TOKENS / 2, X_EACH = 16 / X_SIZE;
    static constexpr uint32_t SCALES = is_float_type<F> ? 0 : SUBS * ROWS * 4, PART = TOKENS * ROWS * 4;
    static_assert(I::BYTES >= PART, "the sums take the place of the images");
    // shared memory of a wave: images, scales [tile][4 sub-blocks][row][sub-block], x [token]
    static constexpr uint32_t AT_X = R * (I::BYTES + SCALES);
    static constexpr __host__ __device__ __forceinline__ uint32_t wave_bytes(uint32_t tokens) { return AT_X + (tokens + 1) / 2 * 2 * X_ROW; }

    // a sum of the wave's, after dense_turns
    static __device__ __forceinline__ float part(const uint8_t *space, uint32_t tile, uint32_t token, uint32_t row) {
        return *(const float *)(space + tile * PART + (token * ROWS + row) * 4);
    }
    typedef float Values[N];
    // N elements as pieces, in words of two: cut off behind eight bits each, which three pieces hold exactly (two, of f16)
    static __device__ __forceinline__ void cut(Values &v, uint32_t (&out)[P][N / 2]) {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (uint32_t i = 0; i < N; i += 2) {
                out[p][i / 2] = upper_halves(v[i], v[i + 1]);
                v[i] = below_bf16(v[i]);
                v[i + 1] = below_bf16(v[i + 1]);
            }
    }
    // the fragment of sub-block s: elements SUB s + N g ..
    static __device__ __forceinline__ void fragment(const uint8_t *x, uint32_t s, uint32_t g, uint32_t (&out)[P][N / 2]) {
        const uint8_t *at = x + (S::SUB * s + N * g) * X_SIZE;
        if constexpr (X == X_BF16 || H) {
            if constexpr (N == 8) {
                const u32x4 w = al16(at);
#pragma unroll
                for (int i = 0; i < 4; ++i) out[0][i] = w[i];
            } else {
                const u32x2 w = al8(at);
                out[0][0] = w[0];
                out[0][1] = w[1];
            }
        } else {
            Values v;
            if constexpr (X == X_F16) {
#pragma unroll
                for (uint32_t i = 0; i < N; i += 4) {
                    const u32x2 w = al8(at + 2 * i);
                    const uint32_t w0 = w[0], w1 = w[1];
                    v[i] = h2f(w0 & 0xFFFFu);
                    v[i + 1] = h2f(w0 >> 16);
                    v[i + 2] = h2f(w1 & 0xFFFFu);
                    v[i + 3] = h2f(w1 >> 16);
                }
            } else {
#pragma unroll
                for (uint32_t i = 0; i < N; i += 4) {
                    const f32x4 w = *(const f32x4 *)(at + 4 * i);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[i + j] = w[j];
                }
            }
            cut(v, out);
        }
    }
    static __device__ __forceinline__ f32x4 multiply(const uint32_t (&a)[N / 2], const uint32_t (&b)[N / 2], f32x4 d) {
        if constexpr (N == 8) {
            const u32x4 va = {a[0], a[1], a[2], a[3]}, vb = {b[0], b[1], b[2], b[3]};
            if constexpr (H) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, va), __builtin_bit_cast(f16x8, vb), d, 0, 0, 0);
            else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, va), __builtin_bit_cast(bf16x8, vb), d, 0, 0, 0);
        } else {
            const u32x2 va = {a[0], a[1]}, vb = {b[0], b[1]};
            if constexpr (H) return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, va), __builtin_bit_cast(f16x4, vb), d, 0, 0, 0);
            else return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, va), __builtin_bit_cast(s16x4, vb), d, 0, 0, 0);
        }
    }
    // the products of one turn; `space`: the wave's shared memory, x: of the lane's token
    static __device__ __forceinline__ void add(uint8_t *space, const uint8_t *x, uint32_t n, uint32_t g, uint32_t left, f32x4 (&acc)[R]) {
        const uint8_t *row = space + n * I::ROW;
        if constexpr (is_float_type<F>) {
#pragma unroll
            for (uint32_t s = 0; s < SUBS; ++s) {
                uint32_t a[P][N / 2];
                fragment(x, s, g, a);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const u32x4 w = S::load(row + r * I::BYTES, s, g, left);
                    uint32_t b[4] = {w[0], w[1], w[2], w[3]}, low[4];
                    if constexpr (__is_same(F, WF16) && !H) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float v0 = h2f(b[i] & 0xFFFFu), v1 = h2f(b[i] >> 16);
                            b[i] = upper_halves(v0, v1);
                            low[i] = upper_halves(below_bf16(v0), below_bf16(v1));
                        }
                    }
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        acc[r] = multiply(a[p], b, acc[r]);
                        if constexpr (__is_same(F, WF16) && !H) acc[r] = multiply(a[p], low, acc[r]);
                    }
                }
            }
        } else {
            float *scales = (float *)(space + R * I::BYTES);
            float offset[R][EACH], sums[EACH];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                SubScale mine[EACH];
                S::scale(row + r * I::BYTES, g, left, mine);
                float *to = scales + r * (SCALES / 4);
                if constexpr (EACH == 2) *(f32x2 *)(to + (g / 2 * ROWS + n) * 4 + g % 2 * 2) = f32x2{mine[0].a, mine[1].a};
                else *(f32x4 *)(to + (g * ROWS + n) * 4) = f32x4{mine[0].a, mine[1].a, mine[2].a, mine[3].a};
#pragma unroll
                for (uint32_t k = 0; k < EACH; ++k) offset[r][k] = -mine[k].c;
            }
            wave_order();
            f32x4 scale[R];
#pragma unroll
            for (uint32_t s = 0; s < SUBS; ++s) {
                uint32_t a[P][N / 2];
                fragment(x, s, g, a);
                if constexpr (S::OFFSET) {
                    // times ones: the sum of the lane's token, in all four of D's rows
                    uint32_t ones[N / 2];
#pragma unroll
                    for (uint32_t i = 0; i < N / 2; ++i) ones[i] = H ? 0x3C003C00u : 0x3F803F80u;
                    f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int p = 0; p < P; ++p) d = multiply(ones, a[p], d);
                    sums[s % EACH] = s / EACH == 0 || g == s / EACH ? d[0] : sums[s % EACH];
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (s % 4 == 0) scale[r] = *(const f32x4 *)(scales + r * (SCALES / 4) + (s / 4 * ROWS + n) * 4);
                    uint32_t b[N / 2];
                    S::template codes<H>(row + r * I::BYTES, s, g, b);
                    f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int p = 0; p < P; ++p) d = multiply(a[p], b, d);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[r][i] = __builtin_fmaf(scale[r][s % 4], d[i], acc[r][i]);
                }
            }
            if constexpr (S::OFFSET) {
                // the offsets of a lane's row and sub-blocks meet the sums of its token and the same sub-blocks, in f32
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (uint32_t k = 0; k < EACH; ++k) acc[r] = __builtin_amdgcn_mfma_f32_16x16x4f32(sums[k], offset[r][k], acc[r], 0, 0, 0);
            }
        }
    }
};

// The wave's turns kp, kp + waves, ..., the next one's bytes on the way while one is multiplied; then its sums, in the place of
// the images, [tile][token][row].
//     at(turn, r)        the packed bytes of tile r, as in run_turns
//     src(t)             the first element of token t's row of `cols`; KEEP: not found by arithmetic alone
template <class M, int R, bool KEEP, class At, class Src>
__device__ __forceinline__ void dense_turns(uint8_t *space, const typename M::I::Places &places, uint32_t reach, uint32_t kp, uint32_t waves, uint32_t turns, uint32_t tokens,
                                            uint32_t cols, At at, Src src) {
    const uint32_t lane = threadIdx.x % 64, n = lane % 16, g = lane / 16;
    uint8_t *xs = space + M::AT_X;
    const uint32_t token = n < tokens ? n : tokens - 1;
    const uint8_t *x = xs + token * M::X_ROW;
    typename M::I in[R];
    u32x4 xr[M::X_LOADS];
    uint64_t room[R];
    uint32_t left = 0, column = 0;
    const uint32_t x_need = M::WIDE ? tokens : (tokens + 1) / 2, x_slot = M::WIDE ? 0 : lane / 32, x_at = (M::WIDE ? lane : lane % 32) * M::X_EACH;
    const uint8_t *x_row[KEEP ? M::X_LOADS : 1];
    auto of = [&](uint32_t i) {
        const uint32_t slot = M::WIDE ? i : 2 * i + x_slot;
        return src(slot < tokens ? slot : tokens - 1);
    };
    if constexpr (KEEP) {
#pragma unroll
        for (uint32_t i = 0; i < M::X_LOADS; ++i)
            if (i < x_need) x_row[i] = of(i);
    }
    // 16 bytes of x that would end behind the row are moved back to end with it, and shifted when they are put
    const uint32_t x_last = cols - M::X_EACH;
    auto fetch = [&](uint32_t turn) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const Turn t = at(turn, r);
            in[r].fetch(places, t.base, t.room);
            room[r] = t.room;
            left = t.left;
        }
        column = turn * M::ELEMS;
        const uint32_t from = (column + x_at < x_last ? column + x_at : x_last) * M::X_SIZE;
#pragma unroll
        for (uint32_t i = 0; i < M::X_LOADS; ++i)
            if (i < x_need) xr[i] = ld16((KEEP ? x_row[KEEP ? i : 0] : of(i)) + from);
    };
    f32x4 acc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (kp < turns) fetch(kp);
    for (uint32_t turn = kp; turn < turns; turn += waves) {
        wave_order();
#pragma unroll
        for (int r = 0; r < R; ++r) in[r].put(places, space + r * M::I::BYTES, room[r], reach);
        if (column + M::ELEMS <= cols) {
#pragma unroll
            for (uint32_t i = 0; i < M::X_LOADS; ++i)
                if (i < x_need) *(u32x4 *)(xs + (M::WIDE ? i : 2 * i + x_slot) * M::X_ROW + x_at * M::X_SIZE) = xr[i];
        } else {                                          // behind the row: zeros
            const uint32_t c = column + x_at, back = c > x_last ? (c - x_last) * M::X_SIZE : 0u;
#pragma unroll
            for (uint32_t i = 0; i < M::X_LOADS; ++i)
                if (i < x_need) *(u32x4 *)(xs + (M::WIDE ? i : 2 * i + x_slot) * M::X_ROW + x_at * M::X_SIZE) = back < 16 ? M::I::shifted(xr[i], back) : u32x4{0, 0, 0, 0};
        }
        wave_order();
        const uint32_t here = left;
        if (turn + waves < turns) fetch(turn + waves);
        M::add(space, x, n, g, here, acc);
    }
    wave_order();
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) *(float *)(space + r * M::PART + ((4 * g + i) * M::ROWS + n) * 4) = acc[r][i];
}

// Waves of a CU that the registers of R tiles leave room for.
constexpr int dense_waves_per_cu(int R) { return R == 1 ? 12 : 8; }

// ---- one matrix, several tokens ---------------------------------------------------------------------------------
// A workgroup takes R tiles of rows, its waves share their columns.
template <class F, int X, int R>
__global__ __launch_bounds__(TILE_THREADS) __attribute__((amdgpu_waves_per_eu(dense_waves_per_cu(R) / 4))) void matvec_dense(MatvecArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    typedef DenseTile<F, X, R> M;
    typedef typename M::I I;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), waves = blockDim.x / 64, wave_bytes = M::wave_bytes(a.tokens);
    const uint32_t row_bytes = (uint32_t)(a.cols / F::N * F::BYTES), turns = (uint32_t)((a.cols + M::ELEMS - 1) / M::ELEMS);
    const uint64_t first_row = (a.first_tile + (uint64_t)blockIdx.x * R) * M::ROWS;
    const uint32_t rows = full_tile_at<M::ROWS>(first_row, a.rows).rows;
    auto begin = [&](int r) { return full_tile_at<M::ROWS>(first_row + r * M::ROWS, a.rows).own; };
    dense_turns<M, R, false>(lds + wave * wave_bytes, typename I::Places(threadIdx.x % 64, rows, row_bytes), I::reach(rows, row_bytes), wave, waves, turns, a.tokens,
                             (uint32_t)a.cols,
                             [&](uint32_t turn, int r) {
                                 const uint64_t row = begin(r);
                                 const uint32_t off = turn * I::TURN_BYTES;
                                 return Turn{a.w + row * row_bytes + off, row_bytes - off, (a.rows - row) * row_bytes - off};
                             },
                             [&](uint32_t t) { return (const uint8_t *)a.x + t * a.x_stride * M::X_SIZE; });
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < R * M::ROWS * a.tokens; i += blockDim.x) {
        const uint32_t r = i % (R * M::ROWS) / M::ROWS, n = i % M::ROWS, t = i / (R * M::ROWS);
        const uint64_t row = begin(r) + n;
        float v = 0.0f;
        for (uint32_t k = 0; k < waves; ++k) v += M::part(lds + k * wave_bytes, r, t, n);
        if (row >= first_row + r * M::ROWS && row < a.rows) store_elem(a.y, t * a.y_stride + row, a.y_kind, v);
    }
}

}  // namespace ggq
