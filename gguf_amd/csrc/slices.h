// slices.h -- a lane's share of a packed row, for the products with packed weights (matmul.h).
//
// A row is cut into slices of 64 elements, four to a step (256 elements).  One lane takes the packed bytes of one slice and
// turns them into whole-number codes.  Elements that share a scale form a sub-block of SUB = 16 or 32:
//     w = a * q - c      q: code, a: scale of the sub-block, c: its offset
// and the product needs a and c once per sub-block:  sum of w x = a * (sum of q x) - c * (sum of x).
//
// Codes go into the matrix unit as e4m3 bytes without any conversion: a byte of 0..15 is a subnormal or in the first
// binade, both of which step by 2^-9, so its value is the byte times 2^-9, and the unit's block scale takes that factor
// back.  Codes of more than four bits are two planes of bytes, q = low + 16 * high, the second with its own block scale.
// Signed codes: an IQ4 codebook can hold sign and magnitude, the sign goes into both planes; 8-bit codes are counted from -128 on,
// and a third plane, the constant -128, takes that back in the same sums.
//
// Per format:
//     NSUB, SUB       sub-blocks of a slice and their elements (NSUB * SUB = 64)
//     PLANES          the sub-blocks of a slice are 16 elements each, 32 elements apart (two-level formats of 16-element
//                     sub-blocks: the codes of elements l, l + 32, l + 64 and l + 96 share a byte); otherwise the slice is 64
//                     consecutive elements
//     HIGH            codes have a second plane
//     OFFSET          whether c can differ from zero
//     STEP            packed bytes of a step
//     TURN            steps that a wave takes at a time
//     BLOCKS          the steps of a turn come into shared memory at 16-byte aligned places, each a block of a 256-element
//                     format, whose parts can then be read with wide aligned loads; otherwise a turn is one run of bytes,
//                     whose slices are whole words
//     Raw             the packed bytes of slice g of a step in registers; load(row, step, g, left): from the row's image in
//                     shared memory, `left` bytes of the row from this turn on.  Blocks behind the row's end hold anything
//                     there: they get the scale 0
//     low<S>(r, b), high<S>(r, b)   the planes of sub-block S, elements in order
//     LOW_EXP<S>, HIGH_EXP<S>       ... are to be multiplied by 2 to this
//     scale<S>(r)     {a, c} of sub-block S
#pragma once
#include "formats.h"

namespace ggq {

typedef uint32_t u32_any __attribute__((aligned(1), may_alias));
typedef uint16_t u16_any __attribute__((aligned(1), may_alias));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_any __attribute__((aligned(1), may_alias));

// global memory, any alignment
__device__ __forceinline__ u32x4 ld16(const uint8_t *p) { return *(const u32x4_any *)p; }
// 16 bytes that nothing reads soon
template <class V> __device__ __forceinline__ void st16_streaming(void *p, V v) { __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), (u32x4_any *)p); }
__device__ __forceinline__ uint32_t ld4(const uint8_t *p) { return *(const u32_any *)p; }
__device__ __forceinline__ uint32_t ld2(const uint8_t *p) { return *(const u16_any *)p; }
// shared memory, aligned
__device__ __forceinline__ u32x4 al16(const uint8_t *p) { return *(const u32x4 *)p; }
__device__ __forceinline__ u32x2 al8(const uint8_t *p) { return *(const u32x2 *)p; }
__device__ __forceinline__ uint32_t al4(const uint8_t *p) { return *(const uint32_t *)p; }
__device__ __forceinline__ uint32_t al2(const uint8_t *p) { return *(const uint16_t *)p; }

// the upper halves of two f32 as two bf16
__device__ __forceinline__ uint32_t upper_halves(float lo, float hi) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u);
}
// v minus its upper 16 bits as a bf16, exactly; a NaN where v is not finite
__device__ __forceinline__ float below_bf16(float v) {
    return v - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & 0xFFFF0000u);
}

struct SubScale { float a, c; };

// ~0 where a block that ends at byte `end` is part of the row, otherwise 0
__device__ __forceinline__ uint32_t in_row(uint32_t end, uint32_t left) { return end <= left ? ~0u : 0u; }
__device__ __forceinline__ uint32_t funnel16(uint32_t hi, uint32_t lo) { return __builtin_amdgcn_alignbit(hi, lo, 16); }
constexpr uint32_t LOW4 = 0x0F0F0F0Fu;

template <class F> struct Slice;

// the 16-bit floats as one-element block types
struct WF16 { static constexpr uint32_t N = 1, BYTES = 2; };
struct WBF16 { static constexpr uint32_t N = 1, BYTES = 2; };
template <class F> constexpr bool from_minus_128 = false;             // codes are counted from there on
template <> inline constexpr bool from_minus_128<Q8_0> = true;
template <> inline constexpr bool from_minus_128<Q8_1> = true;
template <> inline constexpr bool from_minus_128<Q8K> = true;
template <class F> constexpr bool is_float_type = false;
template <> inline constexpr bool is_float_type<WF16> = true;
template <> inline constexpr bool is_float_type<WBF16> = true;

#define GGQ_LOW(N) template <int S> static __device__ __forceinline__ void low(const Raw &r, uint32_t (&b)[N])
#define GGQ_HIGH(N) template <int S> static __device__ __forceinline__ void high(const Raw &r, uint32_t (&b)[N])
#define GGQ_SCALE template <int S> static __device__ __forceinline__ SubScale scale(const Raw &r)
#define GGQ_EXP(name, value) template <int S> static constexpr int name = value

// ---- 32-element formats: a slice is two blocks; the second may be missing at the end of a row --------------
// The two blocks are a whole number of words and lie at a whole word, so they are read as words.
template <uint32_t B, uint32_t T>
struct SliceOfTwo {
    static constexpr bool PLANES = false;
    static constexpr int NSUB = 2, SUB = 32;
    static constexpr uint32_t STEP = 8 * B, TURN = T;
    static constexpr bool BLOCKS = false;
    GGQ_EXP(LOW_EXP, 9);
    GGQ_EXP(HIGH_EXP, 13);
    struct Raw {
        uint32_t w[B / 2], live[2];
        __device__ __forceinline__ void load(const uint8_t *row, uint32_t step, uint32_t g, uint32_t left) {
            const uint32_t at = step * STEP + 2 * g * B;
#pragma unroll
            for (uint32_t i = 0; i < B / 2; ++i) w[i] = al4(row + at + 4 * i);
            live[0] = in_row(at + B, left);
            live[1] = in_row(at + 2 * B, left);
        }
        // the word at byte OFF of block S; it is a whole word, or begins two bytes behind one
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
#define GGQ_WORDS4(BODY) BODY(0) BODY(1) BODY(2) BODY(3)
#define GGQ_WORDS8(BODY) GGQ_WORDS4(BODY) BODY(4) BODY(5) BODY(6) BODY(7)

// 16 bytes of nibbles at OFF: word i holds elements 4 i.. in its low and 16 + 4 i.. in its high nibbles
template <int S, uint32_t OFF, class Raw>
__device__ __forceinline__ void nibbles(const Raw &r, uint32_t (&b)[8]) {
#define ONE(i)                                                  \
    {                                                           \
        const uint32_t q = r.template word<S, OFF + 4 * i>();   \
        b[i] = q & LOW4;                                        \
        b[4 + i] = (q >> 4) & LOW4;                             \
    }
    GGQ_WORDS4(ONE)
#undef ONE
}
// a word of fifth bits -> a byte for each
__device__ __forceinline__ void fifth_bits(uint32_t w, uint32_t (&b)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = __umul24((w >> (4 * i)) & 0xFu, 0x204081u) & 0x01010101u;
}
// 8-bit codes counted from -128 on
template <int S, uint32_t OFF, int SHIFT, class Raw>
__device__ __forceinline__ void byte_plane(const Raw &r, uint32_t (&b)[8]) {
#define ONE(i) b[i] = ((r.template word<S, OFF + 4 * i>() ^ 0x80808080u) >> SHIFT) & LOW4;
    GGQ_WORDS8(ONE)
#undef ONE
}
// The IQ4 codebook (iq4_lookup4) as sign and magnitude, 0..127, without further operations for the low plane and one for the high
// one: the constant plane would take iq4_xs 28672 x 8192 from 37.8 to 40.8 us, this takes it to 39.4.
__device__ __forceinline__ uint32_t iq4_signed4(uint32_t nibs) {
    const uint32_t sel = nibs & 0x07070707u;                           // the lower eight values are negative
    const uint32_t lo = __builtin_amdgcn_perm(0x8A96A3B1u, 0xC1D3E8FFu, sel), hi = __builtin_amdgcn_perm(0x71594535u, 0x26190D01u, sel);
    const uint32_t mask = ((nibs >> 3) & 0x01010101u) * 0xFFu;
    return (hi & mask) | (lo & ~mask);
}
template <int SHIFT>
__device__ __forceinline__ uint32_t signed_plane(uint32_t v) { return SHIFT ? ((v >> 4) & 0x07070707u) | (v & 0x80808080u) : v & 0x8F8F8F8Fu; }
// the codebook's values of 16 bytes of nibbles in four words
template <int SHIFT>
__device__ __forceinline__ void codebook_plane(uint32_t q, uint32_t &first, uint32_t &second) {
    first = signed_plane<SHIFT>(iq4_signed4(q & LOW4));
    second = signed_plane<SHIFT>(iq4_signed4((q >> 4) & LOW4));
}

template <> struct Slice<Q4_0> : SliceOfTwo<18, 2> {
    static constexpr bool HIGH = false, OFFSET = true;
    GGQ_LOW(8) { nibbles<S, 2>(r, b); }
    GGQ_SCALE { const float d = h2f(r.half<S>()); return {d, 8.0f * d}; }
};
template <> struct Slice<Q4_1> : SliceOfTwo<20, 2> {
    static constexpr bool HIGH = false, OFFSET = true;
    GGQ_LOW(8) { nibbles<S, 4>(r, b); }
    GGQ_SCALE { return {h2f(r.half<S>()), -h2f((r.word<S, 0>() & r.live[S]) >> 16)}; }
};
template <> struct Slice<Q5_0> : SliceOfTwo<22, 2> {
    static constexpr bool HIGH = true, OFFSET = true;
    GGQ_LOW(8) { nibbles<S, 6>(r, b); }
    GGQ_HIGH(8) { fifth_bits(r.word<S, 2>(), b); }
    GGQ_SCALE { const float d = h2f(r.half<S>()); return {d, 16.0f * d}; }
};
template <> struct Slice<Q5_1> : SliceOfTwo<24, 1> {
    static constexpr bool HIGH = true, OFFSET = true;
    GGQ_LOW(8) { nibbles<S, 8>(r, b); }
    GGQ_HIGH(8) { fifth_bits(r.word<S, 4>(), b); }
    GGQ_SCALE { return {h2f(r.half<S>()), -h2f((r.word<S, 0>() & r.live[S]) >> 16)}; }
};
template <> struct Slice<Q8_0> : SliceOfTwo<34, 1> {
    static constexpr bool HIGH = true, OFFSET = false;
    GGQ_LOW(8) { byte_plane<S, 2, 0>(r, b); }
    GGQ_HIGH(8) { byte_plane<S, 2, 4>(r, b); }
    GGQ_SCALE { return {h2f(r.half<S>()), 0.0f}; }
};
template <> struct Slice<Q8_1> : SliceOfTwo<36, 1> {
    static constexpr bool HIGH = true, OFFSET = false;
    GGQ_LOW(8) { byte_plane<S, 4, 0>(r, b); }
    GGQ_HIGH(8) { byte_plane<S, 4, 4>(r, b); }
    GGQ_SCALE { return {h2f(r.half<S>()), 0.0f}; }
};
template <> struct Slice<IQ4NL> : SliceOfTwo<18, 2> {
    static constexpr bool HIGH = true, OFFSET = false;
#define ONE(i) codebook_plane<0>(r.word<S, 2 + 4 * i>(), b[i], b[4 + i]);
    GGQ_LOW(8) { GGQ_WORDS4(ONE) }
#undef ONE
#define ONE(i) codebook_plane<4>(r.word<S, 2 + 4 * i>(), b[i], b[4 + i]);
    GGQ_HIGH(8) { GGQ_WORDS4(ONE) }
#undef ONE
    GGQ_SCALE { return {h2f(r.half<S>()), 0.0f}; }
};

// ---- 256-element formats: a block is a step, a lane's slice a quarter of it ----------------------------------
template <uint32_t B, uint32_t T>
struct SliceOfQuarter {
    static constexpr uint32_t STEP = B, TURN = T;
    static constexpr bool BLOCKS = true;
    GGQ_EXP(LOW_EXP, 9);
    GGQ_EXP(HIGH_EXP, 13);
    // the block's image and whether there is such a block
    static __device__ __forceinline__ const uint8_t *block(const uint8_t *row, uint32_t step) { return row + step * ((B + 15) / 16 * 16); }
    static __device__ __forceinline__ uint32_t live(uint32_t step, uint32_t left) { return in_row((step + 1) * B, left); }
};

// 6-bit scale and minimum of sub-blocks 2j and 2j + 1 (j = 0..3) from the twelve bytes in words s0, s1, s2: for j < 2 the
// first two words' low six bits, for j >= 2 the third word's nibbles under the first two words' top two bits
struct PairOfK4 { uint32_t sc, mn; };            // bytes 0 and 1
__device__ __forceinline__ PairOfK4 scales_k4(uint32_t s0, uint32_t s1, uint32_t s2, uint32_t j) {
    const uint32_t sh = 16 * (j & 1);            // two bytes of each word
    const uint32_t a = s0 >> sh, b = s1 >> sh, c = s2 >> sh;
    const uint32_t low = j < 2 ? 0x3F3Fu : 0u, high = 0x3F3Fu ^ low;        // a mask: lanes of one wave are in all quarters
    return {(a & low) | (((c & 0x0F0Fu) | ((a >> 2) & 0x3030u)) & high), (b & low) | ((((c >> 4) & 0x0F0Fu) | ((b >> 2) & 0x3030u)) & high)};
}
template <> struct Slice<Q4K> : SliceOfQuarter<144, 2> {
    static constexpr bool PLANES = false, HIGH = false, OFFSET = true;
    static constexpr int NSUB = 2, SUB = 32;
    struct Raw {
        u32x4 q[2];
        PairOfK4 k;
        uint32_t dm;
        __device__ __forceinline__ void load(const uint8_t *row, uint32_t step, uint32_t g, uint32_t left) {
            const uint8_t *p = block(row, step);
            const u32x4 h = al16(p);
            q[0] = al16(p + 16 + 32 * g);
            q[1] = al16(p + 32 + 32 * g);
            dm = h[0] & SliceOfQuarter::live(step, left);
            k = scales_k4(h[1], h[2], h[3], g);
        }
    };
    GGQ_LOW(8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = (r.q[i / 4][i % 4] >> (4 * S)) & LOW4;
    }
    GGQ_SCALE { return {h2f(r.dm & 0xFFFFu) * ub<S>(r.k.sc), h2f(r.dm >> 16) * ub<S>(r.k.mn)}; }
};
template <> struct Slice<Q5K> : SliceOfQuarter<176, 1> {
    static constexpr bool PLANES = false, HIGH = true, OFFSET = true;
    static constexpr int NSUB = 2, SUB = 32;
    struct Raw {
        u32x4 q[2], f[2];
        PairOfK4 k;
        uint32_t dm;
        __device__ __forceinline__ void load(const uint8_t *row, uint32_t step, uint32_t g, uint32_t left) {
            const uint8_t *p = block(row, step);
            const u32x4 h = al16(p);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                q[i] = al16(p + 48 + 32 * g + 16 * i);
                f[i] = al16(p + 16 + 16 * i);
#pragma unroll
                for (int n = 0; n < 4; ++n) f[i][n] >>= 2 * g;
            }
            dm = h[0] & SliceOfQuarter::live(step, left);
            k = scales_k4(h[1], h[2], h[3], g);
        }
    };
    GGQ_LOW(8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = (r.q[i / 4][i % 4] >> (4 * S)) & LOW4;
    }
    // bit S of each byte, where it is
    GGQ_HIGH(8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = r.f[i / 4][i % 4] & (0x01010101u << S);
    }
    GGQ_EXP(HIGH_EXP, 13 - S);
    GGQ_SCALE { return {h2f(r.dm & 0xFFFFu) * ub<S>(r.k.sc), h2f(r.dm >> 16) * ub<S>(r.k.mn)}; }
};
template <> struct Slice<IQ4XS> : SliceOfQuarter<136, 2> {
    static constexpr bool PLANES = false, HIGH = true, OFFSET = false;
    static constexpr int NSUB = 2, SUB = 32;
    struct Raw {
        uint32_t q[8], d, ls;         // ls: the two scales' low nibbles and top bits, each S-th in place
        __device__ __forceinline__ void load(const uint8_t *row, uint32_t step, uint32_t g, uint32_t left) {
            const uint8_t *p = block(row, step);
            const u32x2 h = al8(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u32x2 v = al8(p + 8 + 32 * g + 8 * i);      // 8-byte aligned
                q[2 * i] = v[0];
                q[2 * i + 1] = v[1];
            }
            d = h[0] & 0xFFFFu & SliceOfQuarter::live(step, left);
            ls = ((h[1] >> (8 * g)) & 0xFFu) | ((h[0] >> (16 + 4 * g)) & 0xFu) << 8;
        }
    };
    GGQ_LOW(8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) codebook_plane<0>(r.q[4 * S + i], b[i], b[4 + i]);
    }
    GGQ_HIGH(8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) codebook_plane<4>(r.q[4 * S + i], b[i], b[4 + i]);
    }
    GGQ_SCALE {
        const uint32_t ls = ((r.ls >> (4 * S)) & 0xFu) | (((r.ls >> (8 + 2 * S)) & 3u) << 4);
        return {h2f(r.d) * (float)((int)ls - 32), 0.0f};
    }
};
template <> struct Slice<Q8K> : SliceOfQuarter<290, 1> {
    static constexpr bool PLANES = false, HIGH = true, OFFSET = false;
    static constexpr int NSUB = 2, SUB = 32;
    struct Raw {
        uint32_t q[16], d;
        __device__ __forceinline__ void load(const uint8_t *row, uint32_t step, uint32_t g, uint32_t left) {
            const uint8_t *p = block(row, step);
            d = al2(p) & SliceOfQuarter::live(step, left);
            uint32_t w[17];           // the codes begin two bytes behind a whole word
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u32x4 v = al16(p + 64 * g + 16 * i);
#pragma unroll
                for (int n = 0; n < 4; ++n) w[4 * i + n] = v[n];
            }
            w[16] = al4(p + 64 * g + 64);
#pragma unroll
            for (int i = 0; i < 16; ++i) q[i] = funnel16(w[i + 1], w[i]) ^ 0x80808080u;
        }
    };
    GGQ_LOW(8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = r.q[8 * S + i] & LOW4;
    }
    GGQ_HIGH(8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = (r.q[8 * S + i] >> 4) & LOW4;
    }
    GGQ_SCALE { return {h2f(r.d), 0.0f}; }
};

// Slice g = (half n, 16-element column h) of a block: sub-block S = elements 128 n + 32 S + 16 h + 0..15.
template <uint32_t B, uint32_t T>
struct SliceOfPlanes : SliceOfQuarter<B, T> {
    static constexpr bool PLANES = true, OFFSET = true;
    static constexpr int NSUB = 4, SUB = 16;
};
template <> struct Slice<Q6K> : SliceOfPlanes<210, 1> {
    static constexpr bool HIGH = true;
    struct Raw {
        u32x4 lo[2], f;
        uint32_t sc[2], d;            // sc: scale S at bits 16 (S & 1) of word S >> 1
        __device__ __forceinline__ void load(const uint8_t *row, uint32_t step, uint32_t g, uint32_t left) {
            const uint8_t *p = block(row, step);
            const uint32_t n = g >> 1, h = g & 1;
            lo[0] = al16(p + 64 * n + 16 * h);
            lo[1] = al16(p + 64 * n + 32 + 16 * h);
            f = al16(p + 128 + 16 * g);
            const u32x2 s = al8(p + 192 + 8 * n);
            sc[0] = s[0] >> (8 * h);
            sc[1] = s[1] >> (8 * h);
            d = al2(p + 208) & SliceOfQuarter::live(step, left);
        }
    };
    GGQ_LOW(4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = (r.lo[S & 1][i] >> (4 * (S >> 1))) & LOW4;
    }
    // two bits of each byte; the odd sub-blocks' stay two places up
    GGQ_HIGH(4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = (r.f[i] >> (4 * (S >> 1))) & (S & 1 ? 0x0C0C0C0Cu : 0x03030303u);
    }
    GGQ_EXP(HIGH_EXP, S & 1 ? 11 : 13);
    GGQ_SCALE {
        const float a = h2f(r.d) * (float)(int)(int8_t)(r.sc[S >> 1] >> (16 * (S & 1)));
        return {a, 32.0f * a};
    }
};
template <> struct Slice<Q2K> : SliceOfPlanes<84, 4> {
    static constexpr bool HIGH = false;
    struct Raw {
        u32x4 q;
        uint32_t sc[2], dm;           // sc as in Q6_K
        __device__ __forceinline__ void load(const uint8_t *row, uint32_t step, uint32_t g, uint32_t left) {
            const uint8_t *p = block(row, step);
            const u32x2 s = al8(p + 8 * (g >> 1));
            sc[0] = s[0] >> (8 * (g & 1));
            sc[1] = s[1] >> (8 * (g & 1));
            q = al16(p + 16 + 16 * g);
            dm = al4(p + 80) & SliceOfQuarter::live(step, left);
        }
    };
    GGQ_LOW(4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = (r.q[i] >> (4 * (S >> 1))) & (S & 1 ? 0x0C0C0C0Cu : 0x03030303u);
    }
    GGQ_EXP(LOW_EXP, S & 1 ? 7 : 9);
    GGQ_SCALE {
        const uint32_t sc = r.sc[S >> 1] >> (16 * (S & 1));
        return {h2f(r.dm & 0xFFFFu) * (float)(sc & 0xFu), h2f(r.dm >> 16) * (float)((sc >> 4) & 0xFu)};
    }
};
template <> struct Slice<Q3K> : SliceOfPlanes<110, 2> {
    static constexpr bool HIGH = false;
    struct Raw {
        u32x4 q, f;
        uint32_t lo, hi, d;           // lo: the low nibble of scale S at bits 8 S; hi: its top bits at bits 16 (S & 1) + 2 (S >> 1)
        __device__ __forceinline__ void load(const uint8_t *row, uint32_t step, uint32_t g, uint32_t left) {
            const uint8_t *p = block(row, step);
            const uint32_t n = g >> 1, h = g & 1;
            f = al16(p + 16 * h);
            q = al16(p + 32 + 16 * g);
            const u32x4 s = al16(p + 96);                    // three words of scales, then the block's scale
            // scale 8 n + 2 S + h: low nibble in byte (2 S + h) % 8 of the first two words (n = 1: its high nibble)
            const uint32_t a = s[0] >> (8 * h + 4 * n), b = s[1] >> (8 * h + 4 * n);
            lo = __builtin_amdgcn_perm(b, a, 0x06040200u) & LOW4;
            hi = s[2] >> (8 * h + 4 * n);
            d = s[3] & 0xFFFFu & SliceOfQuarter::live(step, left);
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] >>= 4 * n;
        }
    };
    GGQ_LOW(4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            b[i] = ((r.q[i] >> (2 * S)) & 0x03030303u) | ((S == 3 ? r.f[i] >> 1 : r.f[i] << (S == 3 ? 0 : 2 - S)) & 0x04040404u);
    }
    GGQ_SCALE {
        const uint32_t sc = ((r.lo >> (8 * S)) & 0xFu) | (((r.hi >> (16 * (S & 1) + 2 * (S >> 1))) & 3u) << 4);
        const float a = h2f(r.d) * (float)((int)sc - 32);
        return {a, 4.0f * a};
    }
};

// ---- 16-bit floats: rows of any length; a lane takes 64 elements ---------------------------------------------
// The weights are their own codes, in bf16; a half has eleven significant bits and becomes two of them (WP pieces).
struct SliceOfFloats {
    static constexpr uint32_t STEP = 512, TURN = 4;       // a turn of 16 slices
    static constexpr bool BLOCKS = false;
    struct Raw {
        u32x4 q[8];
        __device__ __forceinline__ void load(const uint8_t *row, uint32_t quad, uint32_t left) {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = al16(row + 128 * quad + 16 * i);
            if (left < STEP * TURN) {      // what lies behind the row may be anything, an infinity too
                const uint32_t n = left > 128 * quad ? (left - 128 * quad) / 2 : 0;
#pragma unroll
                for (uint32_t i = 0; i < 32; ++i) q[i / 4][i % 4] &= 2 * i + 1 < n ? ~0u : 2 * i < n ? 0xFFFFu : 0u;
            }
        }
    };
};
template <> struct Slice<WBF16> : SliceOfFloats {
    static constexpr int WP = 1;
    // elements [32 S, 32 S + 32) of the slice
    static __device__ __forceinline__ void codes(const Raw &r, int S, int, uint32_t (&b)[16]) {
#pragma unroll
        for (int i = 0; i < 16; ++i) b[i] = r.q[4 * S + i / 4][i % 4];
    }
};
template <> struct Slice<WF16> : SliceOfFloats {
    static constexpr int WP = 2;
    static __device__ __forceinline__ void codes(const Raw &r, int S, int piece, uint32_t (&b)[16]) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t w = r.q[4 * S + i / 4][i % 4];
            const float v0 = h2f(w & 0xFFFFu), v1 = h2f(w >> 16);
            b[i] = piece == 0 ? upper_halves(v0, v1) : upper_halves(below_bf16(v0), below_bf16(v1));
        }
    }
};

}  // namespace ggq
