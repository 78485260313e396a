// slices.h -- a lane's share of a packed row, for the products with packed weights (matmul.h).
//
// A row is cut into slices of 64 elements.  One lane loads the packed bytes of one slice and turns them into whole-number
// codes in bf16, which holds every code exactly (at most 8 significant bits), so that products with bf16 pieces of x are
// exact.  Elements that share a scale form a sub-block of SUB = 16, 32 or 64:
//     w = a * q - c      q: code, a: scale of the sub-block, c: its offset
// and the product needs a and c once per sub-block:  sum of w x = a * (sum of q x) - c * (sum of x).
//
// 16 neighbouring slices are a step: what the 16 quads of a wave take at a time.
//
// Per format:
//     NSUB, SUB       sub-blocks of a slice and their elements (NSUB * SUB = 64)
//     OFFSET          whether c can differ from zero
//     PLANES          the sub-blocks of a slice are 16 elements each, 32 elements apart (two-level formats of 16-element
//                     sub-blocks: the codes of elements l, l + 32, l + 64 and l + 96 share a byte); otherwise the slice is 64
//                     consecutive elements
//     STEP            packed bytes of a step
//     UNIT, UNITS     the bytes of a row's step come into shared memory as UNITS pieces of UNIT bytes, each at a 16-byte
//                     aligned place: whole blocks of the 256-element formats, so that their parts can be read with wide
//                     aligned loads; everything at once for the others, whose slices are whole words
//     Lane            what a lane knows of its place: made of its quad (its slice within a step)
//     Raw             the packed bytes of a slice in registers; load(row, lane, left): from the row's image in shared memory,
//                     `left` bytes of the row from this step on.  Blocks behind the row's end hold anything there: they get
//                     the scale 0
//     codes<S>(r, l, b)  the codes of sub-block S as pairs of bf16, elements in order
//     scale<S>(r, l)     {a, c} of sub-block S
//
// Codes below 16 become bf16 two at a time by v_cvt_scalef32_pk_bf16_fp8: an e4m3 byte of 0..15 is a subnormal or in the
// first binade, both of which step by 2^-9, so with a scale of 2^9 its value is the byte itself (one full-rate instruction
// for two codes; by way of f32 it is three).  Wider codes go through f32.
#pragma once
#include "formats.h"

namespace ggq {

typedef uint32_t u32_any __attribute__((aligned(1), may_alias));
typedef uint16_t u16_any __attribute__((aligned(1), may_alias));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_any __attribute__((aligned(1), may_alias));
typedef u32x2 u32x2_any __attribute__((aligned(1), may_alias));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ u32x4 ld16(const uint8_t *p) { return *(const u32x4_any *)p; }
__device__ __forceinline__ u32x2 ld8(const uint8_t *p) { return *(const u32x2_any *)p; }
__device__ __forceinline__ uint32_t ld4(const uint8_t *p) { return *(const u32_any *)p; }
__device__ __forceinline__ uint32_t ld2(const uint8_t *p) { return *(const u16_any *)p; }

// four codes below 16 (bytes of w) -> two words of two bf16
__device__ __forceinline__ void small_codes(uint32_t w, uint32_t &lo, uint32_t &hi) {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 512.0f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 512.0f, true));
}
// the upper halves of two f32 that bf16 holds exactly
__device__ __forceinline__ uint32_t upper_halves(float lo, float hi) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u);
}
__device__ __forceinline__ void byte_codes(uint32_t w, uint32_t &lo, uint32_t &hi) {
    w = opaque(w);
    lo = upper_halves(ub<0>(w), ub<1>(w));
    hi = upper_halves(ub<2>(w), ub<3>(w));
}
__device__ __forceinline__ void signed_codes(uint32_t w, uint32_t &lo, uint32_t &hi) {
    w = opaque(w);
    lo = upper_halves(sb<0>(w), sb<1>(w));
    hi = upper_halves(sb<2>(w), sb<3>(w));
}

struct SubScale { float a, c; };

// aligned loads, from shared memory
__device__ __forceinline__ u32x4 al16(const uint8_t *p) { return *(const u32x4 *)p; }
__device__ __forceinline__ u32x2 al8(const uint8_t *p) { return *(const u32x2 *)p; }
__device__ __forceinline__ uint32_t al4(const uint8_t *p) { return *(const uint32_t *)p; }
// ~0 where a block that ends at byte `end` is part of the row, otherwise 0
__device__ __forceinline__ uint32_t in_row(uint32_t end, uint32_t left) { return end <= left ? ~0u : 0u; }
__device__ __forceinline__ uint32_t funnel16(uint32_t hi, uint32_t lo) { return __builtin_amdgcn_alignbit(hi, lo, 16); }

// ---- 32-element formats: a slice is two blocks; the second may be missing at the end of a row --------------
// The two blocks are a whole number of words and lie at a whole word, so they are read as words.
template <uint32_t B>
struct SliceOfTwo {
    static constexpr bool PLANES = false;
    static constexpr int NSUB = 2, SUB = 32;
    static constexpr uint32_t STEP = 32 * B, UNIT = STEP, UNITS = 1;
    struct Lane {
        uint32_t at;
        __device__ __forceinline__ explicit Lane(uint32_t quad) : at(2 * quad * B) {}
    };
    struct Raw {
        uint32_t w[B / 2], live[2];
        __device__ __forceinline__ void load(const uint8_t *row, const Lane &l, uint32_t left) {
#pragma unroll
            for (uint32_t i = 0; i < B / 2; ++i) w[i] = al4(row + l.at + 4 * i);
            live[0] = in_row(l.at + B, left);
            live[1] = in_row(l.at + 2 * B, left);
        }
        // the word at byte `off` of block S; both are whole words, or off + S * B is two bytes beyond one
        template <int S, uint32_t OFF>
        __device__ __forceinline__ uint32_t word() const {
            constexpr uint32_t at = S * B + OFF;
            if constexpr (at % 4 == 0) return w[at / 4];
            else return funnel16(w[at / 4 + 1], w[at / 4]);
        }
        template <int S>
        __device__ __forceinline__ uint32_t half() const {          // the first two bytes of block S, 0 behind the row
            constexpr uint32_t at = S * B;
            return (at % 4 ? w[at / 4] >> 16 : w[at / 4] & 0xFFFFu) & live[S];
        }
    };
};

template <class F> struct Slice;

// the 16-bit floats as one-element block types
struct WF16 { static constexpr uint32_t N = 1, BYTES = 2; };
struct WBF16 { static constexpr uint32_t N = 1, BYTES = 2; };
template <class F> constexpr bool is_float_type = false;
template <> constexpr bool is_float_type<WF16> = true;
template <> constexpr bool is_float_type<WBF16> = true;

// a template's loop over words whose places are constants: BODY(i) for i < N
#define GGQ_WORDS4(BODY) BODY(0) BODY(1) BODY(2) BODY(3)
#define GGQ_WORDS8(BODY) GGQ_WORDS4(BODY) BODY(4) BODY(5) BODY(6) BODY(7)

// 16 bytes of nibbles behind HEAD bytes: word i holds elements 4 i.. in its low and 16 + 4 i.. in its high nibbles
template <class Raw, int S, uint32_t HEAD>
__device__ __forceinline__ void nibble_codes(const Raw &r, uint32_t (&b)[16]) {
#define ONE(i)                                                                        \
    {                                                                                 \
        const uint32_t q = r.template word<S, HEAD + 4 * i>();                        \
        small_codes(q & 0x0F0F0F0Fu, b[2 * i], b[2 * i + 1]);                         \
        small_codes((q >> 4) & 0x0F0F0F0Fu, b[8 + 2 * i], b[9 + 2 * i]);              \
    }
    GGQ_WORDS4(ONE)
#undef ONE
}
template <class Raw, int S, uint32_t HEAD>
__device__ __forceinline__ void iq4_codes(const Raw &r, uint32_t (&b)[16]) {
#define ONE(i)                                                                                              \
    {                                                                                                       \
        const uint32_t q = r.template word<S, HEAD + 4 * i>();                                              \
        signed_codes(iq4_lookup4(q & 0x0F0F0F0Fu) ^ 0x80808080u, b[2 * i], b[2 * i + 1]);                   \
        signed_codes(iq4_lookup4((q >> 4) & 0x0F0F0F0Fu) ^ 0x80808080u, b[8 + 2 * i], b[9 + 2 * i]);        \
    }
    GGQ_WORDS4(ONE)
#undef ONE
}
// ... with a word of fifth bits in front of the nibbles
template <class Raw, int S, uint32_t HEAD>
__device__ __forceinline__ void five_codes(const Raw &r, uint32_t (&b)[16]) {
    const uint32_t hi = r.template word<S, HEAD>();
#define ONE(i)                                                                                                              \
    {                                                                                                                       \
        const uint32_t q = r.template word<S, HEAD + 4 + 4 * i>();                                                          \
        byte_codes((q & 0x0F0F0F0Fu) | (spread4(hi >> (4 * i)) << 4), b[2 * i], b[2 * i + 1]);                              \
        byte_codes(((q >> 4) & 0x0F0F0F0Fu) | (spread4(hi >> (16 + 4 * i)) << 4), b[8 + 2 * i], b[9 + 2 * i]);              \
    }
    GGQ_WORDS4(ONE)
#undef ONE
}
template <class Raw, int S, uint32_t HEAD>
__device__ __forceinline__ void signed_byte_codes(const Raw &r, uint32_t (&b)[16]) {
#define ONE(i) signed_codes(r.template word<S, HEAD + 4 * i>(), b[2 * i], b[2 * i + 1]);
    GGQ_WORDS8(ONE)
#undef ONE
}

#define GGQ_CODES(N) template <int S> static __device__ __forceinline__ void codes(const Raw &r, const Lane &l, uint32_t (&b)[N])
#define GGQ_SCALE template <int S> static __device__ __forceinline__ SubScale scale(const Raw &r, const Lane &l)
template <> struct Slice<Q4_0> : SliceOfTwo<18> {
    static constexpr bool OFFSET = true;
    GGQ_CODES(16) { nibble_codes<Raw, S, 2>(r, b); }
    GGQ_SCALE { const float d = h2f(r.half<S>()); return {d, 8.0f * d}; }
};
template <> struct Slice<IQ4NL> : SliceOfTwo<18> {
    static constexpr bool OFFSET = false;
    GGQ_CODES(16) { iq4_codes<Raw, S, 2>(r, b); }
    GGQ_SCALE { return {h2f(r.half<S>()), 0.0f}; }
};
template <> struct Slice<Q4_1> : SliceOfTwo<20> {
    static constexpr bool OFFSET = true;
    GGQ_CODES(16) { nibble_codes<Raw, S, 4>(r, b); }
    GGQ_SCALE { return {h2f(r.half<S>()), -h2f((r.word<S, 0>() & r.live[S]) >> 16)}; }
};
template <> struct Slice<Q5_0> : SliceOfTwo<22> {
    static constexpr bool OFFSET = true;
    GGQ_CODES(16) { five_codes<Raw, S, 2>(r, b); }
    GGQ_SCALE { const float d = h2f(r.half<S>()); return {d, 16.0f * d}; }
};
template <> struct Slice<Q5_1> : SliceOfTwo<24> {
    static constexpr bool OFFSET = true;
    GGQ_CODES(16) { five_codes<Raw, S, 4>(r, b); }
    GGQ_SCALE { return {h2f(r.half<S>()), -h2f((r.word<S, 0>() & r.live[S]) >> 16)}; }
};
template <> struct Slice<Q8_0> : SliceOfTwo<34> {
    static constexpr bool OFFSET = false;
    GGQ_CODES(16) { signed_byte_codes<Raw, S, 2>(r, b); }
    GGQ_SCALE { return {h2f(r.half<S>()), 0.0f}; }
};
template <> struct Slice<Q8_1> : SliceOfTwo<36> {
    static constexpr bool OFFSET = false;
    GGQ_CODES(16) { signed_byte_codes<Raw, S, 4>(r, b); }
    GGQ_SCALE { return {h2f(r.half<S>()), 0.0f}; }
};

// ---- 256-element formats: four slices a block ------------------------------------------------------------
template <uint32_t B>
struct SliceOfQuarter {
    static constexpr uint32_t STEP = 4 * B, UNIT = B, UNITS = 4;
    struct Lane {
        uint32_t at, end, j;          // its block's image, the block's end in the packed step, which quarter of the block
        __device__ __forceinline__ explicit Lane(uint32_t quad) : at((quad >> 2) * ((B + 15) / 16 * 16)), end((quad >> 2) * B + B), j(quad & 3) {}
    };
};

// 6-bit scale and minimum of sub-blocks 2j and 2j + 1 (j = 0..3) from the twelve bytes in words s0, s1, s2: for j < 2 the
// first two words' low six bits, for j >= 2 the third word's nibbles under the first two words' top two bits
struct PairOfK4 { uint32_t sc[2], mn[2]; };
__device__ __forceinline__ PairOfK4 scales_k4(uint32_t s0, uint32_t s1, uint32_t s2, uint32_t j) {
    const uint32_t sh = 16 * (j & 1);            // two bytes of each word
    const uint32_t a = s0 >> sh, b = s1 >> sh, c = s2 >> sh;
    const uint32_t low = j < 2 ? 0x3F3Fu : 0u, high = 0x3F3Fu ^ low;        // a mask: lanes of one wave are in all quarters
    const uint32_t sc = (a & low) | (((c & 0x0F0Fu) | ((a >> 2) & 0x3030u)) & high);
    const uint32_t mn = (b & low) | ((((c >> 4) & 0x0F0Fu) | ((b >> 2) & 0x3030u)) & high);
    return {{sc & 0xFFu, (sc >> 8) & 0xFFu}, {mn & 0xFFu, (mn >> 8) & 0xFFu}};
}
template <> struct Slice<Q4K> : SliceOfQuarter<144> {
    static constexpr bool PLANES = false, OFFSET = true;
    static constexpr int NSUB = 2, SUB = 32;
    struct Raw {
        u32x4 h, q[2];
        uint32_t live;
        __device__ __forceinline__ void load(const uint8_t *row, const Lane &l, uint32_t left) {
            const uint8_t *p = row + l.at;
            live = in_row(l.end, left);
            h = al16(p);
            q[0] = al16(p + 16 + 32 * l.j);
            q[1] = al16(p + 32 + 32 * l.j);
        }
    };
    GGQ_CODES(16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) small_codes((r.q[i / 4][i % 4] >> (4 * S)) & 0x0F0F0F0Fu, b[2 * i], b[2 * i + 1]);
    }
    GGQ_SCALE {
        const PairOfK4 k = scales_k4(r.h[1], r.h[2], r.h[3], l.j);
        return {h2f(r.h[0] & r.live & 0xFFFFu) * (float)k.sc[S], h2f((r.h[0] & r.live) >> 16) * (float)k.mn[S]};
    }
};
template <> struct Slice<Q5K> : SliceOfQuarter<176> {
    static constexpr bool PLANES = false, OFFSET = true;
    static constexpr int NSUB = 2, SUB = 32;
    struct Raw {
        u32x4 h, q[2], f[2];
        uint32_t live;
        __device__ __forceinline__ void load(const uint8_t *row, const Lane &l, uint32_t left) {
            const uint8_t *p = row + l.at;
            live = in_row(l.end, left);
            h = al16(p);
            f[0] = al16(p + 16);
            f[1] = al16(p + 32);
            q[0] = al16(p + 48 + 32 * l.j);
            q[1] = al16(p + 64 + 32 * l.j);
        }
    };
    GGQ_CODES(16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t five = (r.f[i / 4][i % 4] >> (2 * l.j + S)) & 0x01010101u;
            byte_codes(((r.q[i / 4][i % 4] >> (4 * S)) & 0x0F0F0F0Fu) | (five << 4), b[2 * i], b[2 * i + 1]);
        }
    }
    GGQ_SCALE {
        const PairOfK4 k = scales_k4(r.h[1], r.h[2], r.h[3], l.j);
        return {h2f(r.h[0] & r.live & 0xFFFFu) * (float)k.sc[S], h2f((r.h[0] & r.live) >> 16) * (float)k.mn[S]};
    }
};
template <> struct Slice<IQ4XS> : SliceOfQuarter<136> {
    static constexpr bool PLANES = false, OFFSET = false;
    static constexpr int NSUB = 2, SUB = 32;
    struct Raw {
        u32x2 h;
        u32x4 q[2];
        uint32_t live;
        __device__ __forceinline__ void load(const uint8_t *row, const Lane &l, uint32_t left) {
            const uint8_t *p = row + l.at;
            live = in_row(l.end, left);
            h = al8(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) {                    // 8-byte aligned
                const u32x2 v = al8(p + 8 + 32 * l.j + 8 * i);
                q[i / 2][2 * (i & 1)] = v[0];
                q[i / 2][2 * (i & 1) + 1] = v[1];
            }
        }
    };
    GGQ_CODES(16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            signed_codes(iq4_lookup4(r.q[S][i] & 0x0F0F0F0Fu) ^ 0x80808080u, b[2 * i], b[2 * i + 1]);
            signed_codes(iq4_lookup4((r.q[S][i] >> 4) & 0x0F0F0F0Fu) ^ 0x80808080u, b[8 + 2 * i], b[9 + 2 * i]);
        }
    }
    GGQ_SCALE {
        const uint32_t ls = ((r.h[1] >> (8 * l.j + 4 * S)) & 0xFu) | (((r.h[0] >> (16 + 4 * l.j + 2 * S)) & 3u) << 4);
        return {h2f(r.h[0] & r.live & 0xFFFFu) * (float)((int)ls - 32), 0.0f};
    }
};

// Slice s = (block, half n, 16-element column h): sub-block p = elements 128 n + 32 p + 16 h + 0..15 of the block.
template <uint32_t B>
struct SliceOfPlanes : SliceOfQuarter<B> {
    static constexpr bool PLANES = true;
    static constexpr int NSUB = 4, SUB = 16;
};
template <> struct Slice<Q6K> : SliceOfPlanes<210> {
    static constexpr bool OFFSET = true;
    struct Raw {
        u32x4 lo[2], f;
        u32x2 sc;
        uint32_t d, live;
        __device__ __forceinline__ void load(const uint8_t *row, const Lane &l, uint32_t left) {
            const uint8_t *p = row + l.at;
            live = in_row(l.end, left);
            lo[0] = al16(p + 64 * (l.j >> 1) + 16 * (l.j & 1));
            lo[1] = al16(p + 64 * (l.j >> 1) + 32 + 16 * (l.j & 1));
            f = al16(p + 128 + 16 * l.j);
            sc = al8(p + 192 + 8 * (l.j >> 1));
            d = *(const uint16_t *)(p + 208);
        }
    };
    GGQ_CODES(8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t low = (r.lo[S & 1][i] >> (4 * (S >> 1))) & 0x0F0F0F0Fu;
            byte_codes(low | (((r.f[i] >> (2 * S)) & 0x03030303u) << 4), b[2 * i], b[2 * i + 1]);
        }
    }
    GGQ_SCALE {
        const int sc = (int)(int8_t)(r.sc[S >> 1] >> (16 * (S & 1) + 8 * (l.j & 1)));
        const float a = h2f(r.d & r.live) * (float)sc;
        return {a, 32.0f * a};
    }
};
template <> struct Slice<Q2K> : SliceOfPlanes<84> {
    static constexpr bool OFFSET = true;
    struct Raw {
        u32x4 q;
        u32x2 sc;
        uint32_t dm, live;
        __device__ __forceinline__ void load(const uint8_t *row, const Lane &l, uint32_t left) {
            const uint8_t *p = row + l.at;
            live = in_row(l.end, left);
            sc = al8(p + 8 * (l.j >> 1));
            q = al16(p + 16 + 16 * l.j);
            dm = al4(p + 80);
        }
    };
    GGQ_CODES(8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) small_codes((r.q[i] >> (2 * S)) & 0x03030303u, b[2 * i], b[2 * i + 1]);
    }
    GGQ_SCALE {
        const uint32_t sc = (r.sc[S >> 1] >> (16 * (S & 1) + 8 * (l.j & 1))) & 0xFFu;
        return {h2f(r.dm & r.live & 0xFFFFu) * (float)(sc & 0xFu), h2f((r.dm & r.live) >> 16) * (float)(sc >> 4)};
    }
};
template <> struct Slice<Q3K> : SliceOfPlanes<110> {
    static constexpr bool OFFSET = true;
    struct Raw {
        u32x4 q, f, s;               // s: three words of scales, then the block's scale
        uint32_t live;
        __device__ __forceinline__ void load(const uint8_t *row, const Lane &l, uint32_t left) {
            const uint8_t *p = row + l.at;
            live = in_row(l.end, left);
            f = al16(p + 16 * (l.j & 1));
            q = al16(p + 32 + 16 * l.j);
            s = al16(p + 96);
        }
    };
    GGQ_CODES(8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t high = (r.f[i] >> (4 * (l.j >> 1) + S)) & 0x01010101u;
            small_codes(((r.q[i] >> (2 * S)) & 0x03030303u) | (high << 2), b[2 * i], b[2 * i + 1]);
        }
    }
    // sub-block g = 8 n + 2 S + h of 16: low nibble g % 8 of bytes 0..7 (high nibble for n = 1), top bits g / 4 of byte g % 4
    GGQ_SCALE {
        const uint32_t w = S < 2 ? r.s[0] : r.s[1], sh = 16 * (S & 1) + 8 * (l.j & 1);
        const uint32_t low = (w >> (sh + 4 * (l.j >> 1))) & 0xFu, top = (r.s[2] >> (sh + 4 * (l.j >> 1) + 2 * (S >> 1))) & 3u;
        const float a = h2f(r.s[3] & 0xFFFFu & r.live) * (float)((int)(low | (top << 4)) - 32);
        return {a, 4.0f * a};
    }
};
template <> struct Slice<Q8K> : SliceOfQuarter<290> {
    static constexpr bool PLANES = false, OFFSET = false;
    static constexpr int NSUB = 2, SUB = 32;
    struct Raw {
        u32x4 q[4];                  // the codes begin two bytes behind a whole word
        uint32_t over, d, live;
        __device__ __forceinline__ void load(const uint8_t *row, const Lane &l, uint32_t left) {
            const uint8_t *p = row + l.at;
            live = in_row(l.end, left);
            d = *(const uint16_t *)p;
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = al16(p + 64 * l.j + 16 * i);
            over = al4(p + 64 * l.j + 64);
        }
    };
    GGQ_CODES(16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            constexpr int from = 8 * S;
            const uint32_t lo = r.q[(from + i) / 4][(from + i) % 4], hi = from + i == 15 ? r.over : r.q[(from + i + 1) / 4 % 4][(from + i + 1) % 4];
            signed_codes(funnel16(hi, lo), b[2 * i], b[2 * i + 1]);
        }
    }
    GGQ_SCALE { return {h2f(r.d & r.live), 0.0f}; }
};

// ---- 16-bit floats: rows of any length, 64 elements a slice ------------------------------------------------
// The weights are their own codes; a half has eleven significant bits and becomes two bf16 (WP pieces).
struct SliceOfFloats {
    static constexpr bool PLANES = false, OFFSET = false;
    static constexpr int NSUB = 2, SUB = 32;
    static constexpr uint32_t STEP = 2048, UNIT = STEP, UNITS = 1;
    struct Lane {
        uint32_t at;
        __device__ __forceinline__ explicit Lane(uint32_t quad) : at(128 * quad) {}
    };
    struct Raw {
        u32x4 q[8];
        __device__ __forceinline__ void load(const uint8_t *row, const Lane &l, uint32_t left) {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = al16(row + l.at + 16 * i);
            if (left < STEP) {       // what lies behind the row may be anything, an infinity too
                const uint32_t n = left > l.at ? (left - l.at) / 2 : 0;
#pragma unroll
                for (uint32_t i = 0; i < 32; ++i) q[i / 4][i % 4] &= 2 * i + 1 < n ? ~0u : 2 * i < n ? 0xFFFFu : 0u;
            }
        }
    };
    GGQ_SCALE { return {1.0f, 0.0f}; }
};
// v minus its upper 16 bits as a bf16, exactly; a NaN where v is not finite
__device__ __forceinline__ float below_bf16(float v) {
    return v - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & 0xFFFF0000u);
}
template <> struct Slice<WBF16> : SliceOfFloats {
    static constexpr int WP = 1;
    template <int S> static __device__ __forceinline__ void codes(const Raw &r, const Lane &, uint32_t (&b)[16], int) {
#pragma unroll
        for (int i = 0; i < 16; ++i) b[i] = r.q[4 * S + i / 4][i % 4];
    }
};
template <> struct Slice<WF16> : SliceOfFloats {
    static constexpr int WP = 2;
    template <int S> static __device__ __forceinline__ void codes(const Raw &r, const Lane &, uint32_t (&b)[16], int piece) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t w = r.q[4 * S + i / 4][i % 4];
            const float v0 = h2f(w & 0xFFFFu), v1 = h2f(w >> 16);
            b[i] = piece == 0 ? upper_halves(v0, v1) : upper_halves(below_bf16(v0), below_bf16(v1));
        }
    }
};

}  // namespace ggq
