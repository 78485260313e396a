// matmul.h -- products with packed weights: the kernels.
//
//     y[t][r] = sum over c of W[r][c] * x[t][c]        W packed blocks (formats.h), x and y f32 / f16 / bf16
//
// and what surrounds them in a decoding step: rows of a packed table by id, and a mixture-of-experts layer.
#pragma once
#include "kernels.h"
#include "slices.h"

namespace ggq {

// ---- packed bytes in global memory, at any alignment -----------------------------------------------------
// The same interface as LdsBytes, reading exactly the bytes that are asked for: the last block of a tensor may end
// at the end of an allocation.
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

// ---- shared by the products -------------------------------------------------------------------------------
struct MatvecArgs {
    const uint8_t *w;
    const void *x;
    void *y;
    uint64_t rows, cols, x_stride, y_stride;
    uint64_t first_tile;      // wave tiles before this launch's
    uint32_t tokens;          // of this launch's group
    uint32_t x_kind, y_kind;
    uint32_t chunk;           // turns staged at a time, a multiple of ksplit
    uint32_t ksplit;          // waves that share a tile's columns: 1, 2, 4 or 8
};

constexpr uint32_t MV_THREADS = 256;      // the small kernels here
constexpr uint32_t TILE_WAVES = 8, TILE_THREADS = 64 * TILE_WAVES;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int QUAD_XOR1 = 0xB1, QUAD_XOR2 = 0x4E, ROW_ROR4 = 0x124, ROW_ROR8 = 0x128;
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) { return __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(uint32_t, v))); }

// Orders a wave's own accesses to shared memory (its lanes read what others of the wave wrote).
__device__ __forceinline__ void wave_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// eight elements of x from c on, 0 past the end
__device__ __forceinline__ void load8(const void *x, uint64_t at, uint64_t c, uint64_t cols, uint32_t kind, float (&v)[8]) {
    if (c + 8 <= cols) {
        if (kind == EK_F32) {
            const uint8_t *p = (const uint8_t *)x + 4 * (at + c);
            const f32x4 a = __builtin_bit_cast(f32x4, ld16(p)), b = __builtin_bit_cast(f32x4, ld16(p + 16));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = a[i];
                v[4 + i] = b[i];
            }
        } else {
            const u32x4 a = ld16((const uint8_t *)x + 2 * (at + c));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = kind == EK_F16 ? h2f(a[i] & 0xFFFFu) : bf2f(a[i] & 0xFFFFu);
                v[2 * i + 1] = kind == EK_F16 ? h2f(a[i] >> 16) : bf2f(a[i] >> 16);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? load_elem(x, at + c + i, kind) : 0.0f;
    }
}

// Columns: the sixteen packed rows of a tile are within the offsets that Image::last can bound, whatever their type.
constexpr uint64_t MAX_COLS = 1ull << 26;

// A wave's packed bytes of one turn.  Lanes that multiply together hold different rows, so loads straight into their
// registers would touch a line per lane: the memory pipeline takes about two cycles for each, which held the products at
// 4.1 TB/s whatever the format's arithmetic.  Instead neighbouring lanes load neighbouring 16-byte pieces into registers,
// one turn ahead, and hand them over through the wave's own part of shared memory.
template <class F, uint32_t ROWS, uint32_t TURN>
struct Image {
    typedef Slice<F> S;
    static constexpr uint32_t TURN_BYTES = S::STEP * TURN;             // packed, of a row
    static constexpr uint32_t UNITS = S::BLOCKS ? TURN : 1, UNIT_BYTES = TURN_BYTES / UNITS;
    static constexpr uint32_t PIECES = (UNIT_BYTES + 15) / 16, PER_ROW = PIECES * UNITS, LOADS = (PER_ROW * ROWS + 63) / 64;
    // an odd number of 16-byte places from row to row: the rows' parts of one column lie in different banks
    static constexpr uint32_t UNIT = PIECES * 16, ROW = 16 * (PER_ROW | 1);
    static constexpr uint32_t BYTES = ROW * ROWS;
    static_assert((ROWS - 1) * (MAX_COLS / F::N * F::BYTES) + TURN_BYTES + 32 <= (1ull << 31), "offsets in a tile");
    // where this lane's pieces are
    struct Places {
        uint32_t src[LOADS], dst[LOADS];      // from the tile's first row on; in the image
        // `rows` of the tile's rows exist; the others are the last one again
        __host__ __device__ __forceinline__ Places(uint32_t lane, uint32_t rows, uint32_t row_bytes) {
#pragma unroll
            for (uint32_t i = 0; i < LOADS; ++i) {
                uint32_t p = i * 64 + lane;
                if (p >= PER_ROW * ROWS) p = PER_ROW * ROWS - 1;
                const uint32_t r = p / PER_ROW, u = p % PER_ROW / PIECES, c = p % PIECES * 16;
                src[i] = (r < rows ? r : rows - 1) * row_bytes + u * UNIT_BYTES + c;
                dst[i] = r * ROW + u * UNIT + c;
            }
        }
    };
    // bytes from a turn's begin in the tile's first row to the end of its furthest piece
    static __host__ __device__ __forceinline__ uint32_t reach(uint32_t rows, uint32_t row_bytes) { return (rows - 1) * row_bytes + (UNITS - 1) * UNIT_BYTES + UNIT; }
    u32x4 v[LOADS];

    // The turn that begins at `base` (in the tile's first row).  A unit's last piece and a row's last turn may reach beyond
    // them, into whatever follows in the tensor; `room` bytes of the tensor are left from base on, and pieces that would end
    // behind them are moved back to end with it.  put shifts those into place: without a second way through fetch the loads
    // in flight keep their registers.  A turn begins with a whole block, so that only blocks of less than 16 bytes, the 16-bit
    // floats, may leave less room than a piece takes; then all pieces begin in front of base, in the same row, which has 16 bytes.
    static constexpr bool SHORT = F::BYTES < 16;
    // the last place from base on where a piece may begin
    static __host__ __device__ __forceinline__ int32_t last(uint64_t room) { return room < (1u << 31) ? (int32_t)room - 16 : (int32_t)((1u << 31) - 16); }
    // where a piece begins, and how far that is in front of its place
    static __host__ __device__ __forceinline__ uint32_t begin(uint32_t src, int32_t last) {
        const uint32_t most = SHORT && last < 0 ? 0u : (uint32_t)last;
        return src < most ? src : most;
    }
    static __host__ __device__ __forceinline__ int32_t begin_of_turn(int32_t last) { return SHORT && last < 0 ? last : 0; }       // from base on
    static __host__ __device__ __forceinline__ uint32_t moved(uint32_t src, int32_t last) { return (int32_t)src > last ? (uint32_t)((int32_t)src - last) : 0u; }
    __device__ __forceinline__ void fetch(const Places &at, const uint8_t *base, uint64_t room) {
        const int32_t end = last(room);
        const uint8_t *from = base + begin_of_turn(end);
#pragma unroll
        for (uint32_t i = 0; i < LOADS; ++i) {
            uint32_t o = begin(at.src[i], end);
            asm("" : "+v"(o));                // keeps the offset 32 bits wide, for a load with a scalar base
            v[i] = ld16(from + o);
        }
    }
    static __device__ __forceinline__ u32x4 shifted(u32x4 a, uint32_t bytes) {
        const uint32_t b = (bytes & 3) * 8;
        uint32_t w[8] = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = bytes < 4 ? w[i] : bytes < 8 ? w[i + 1] : bytes < 12 ? w[i + 2] : w[i + 3];
            const uint32_t hi = bytes < 4 ? w[i + 1] : bytes < 8 ? w[i + 2] : bytes < 12 ? w[i + 3] : w[i + 4];
            o[i] = __builtin_amdgcn_alignbit(hi, lo, b);
        }
        return {o[0], o[1], o[2], o[3]};
    }
    __device__ __forceinline__ void put(const Places &at, uint8_t *image, uint64_t room, uint32_t reach) const {
        if (room >= reach) {
#pragma unroll
            for (uint32_t i = 0; i < LOADS; ++i) *(u32x4 *)(image + at.dst[i]) = v[i];
        } else {
            const int32_t end = last(room);
#pragma unroll
            for (uint32_t i = 0; i < LOADS; ++i) {
                const uint32_t back = moved(at.src[i], end);
                *(u32x4 *)(image + at.dst[i]) = shifted(v[i], back < 15 ? back : 15);
            }
        }
    }
};

// A wave's tile of at most N rows, from `row` on, in a matrix of `total` rows
template <class T>
struct RowTile {
    T own;                // its first row
    uint32_t rows;
};
// ... of one token: fewer rows at the matrix' end; a wave that has nothing to do takes the last row
template <uint32_t N, class T>
__host__ __device__ __forceinline__ RowTile<T> tile_at(T row, T total) {
    const T own = row < total ? row : total - 1;
    return {own, total - own < N ? (uint32_t)(total - own) : N};
}
// ... of several: moved back to end with the matrix
template <uint32_t N, class T>
__host__ __device__ __forceinline__ RowTile<T> full_tile_at(T row, T total) {
    const uint32_t rows = total < N ? (uint32_t)total : N;
    return {row < total - rows ? row : total - rows, rows};
}

// What a wave does with a tile of rows and one token.  Two kinds, with the same members:
//     ROWS, ELEMS       rows of the tile, elements of a turn
//     X_BYTES           shared memory of a turn of x
//     CLEAR             bytes of zeros in front of the staged x
//     WAVE_BYTES        shared memory of a wave: its image
//     stage             puts turns of x into shared memory
//     Me                what a lane knows of its place
//     add               the products of one turn
//     put               the wave's sums to part[row]

// ---- packed whole-number codes, one token: x in digits ------------------------------------------------------
// The matrix unit multiplies e4m3 bytes with a block scale for each 32 of them.  Codes are such bytes already (slices.h),
// and so are the digits of x: 32 neighbouring elements share an exponent e, the largest one's; each becomes a whole number
// of 32 bits (rounded, to 2^-32 of the largest element) and that eight hexadecimal digits, each a byte 0..15 with x's sign, in
// two chains of four.  All products are exact, and a chain's sums over a sub-block are whole numbers below 2^13 for each plane;
// the two chains, 2^-16 apart, and the four digits are joined in f32.  Sixteen bits, one chain, would do for 16-bit results of
// ordinary x (q6_k 32000 x 4096 22.8 instead of 24.0 us), but beside an outlier small elements would lose bits that the caller gave.
//
// v_mfma_scale_f32_16x16x128: A is x, B the codes of 16 rows.  Lane (n, g), n = lane % 16, g = lane / 16, brings 32 codes of
// row n, slice g.  Row m of A is digit m % 4 of the slices g = m / 4 and zero for the other slices, so that D's rows
// 4 g .. 4 g + 3, which lane (n, g) receives, are the four digits' sums of the lane's own codes: slices are kept apart, and
// the scale that a lane has unpacked is applied where it is.  The lanes of A whose slice is not m / 4's read zeros.  A's block
// scale is e, whatever it is; the second chain's weight 2^-16 is in B's, and the digits' weights 16^-d are applied when a
// sub-block's four sums are joined.
//
// Codes that are counted from -128 on: the constant is a third plane.  With 128 a (sum of x) as the offset instead, the f32 sums
// carried it and lost it again: by codes that were small beside their range, next to an outlier, the result was 2^-13 off.  The
// matrix unit has room for it (q8_0 11008 x 4096 12.5 instead of 12.3 us; codes by sign and magnitude 13.5).
//
// Codes need no conversion, and a sub-block's four digits a multiply-add each: q6_k 4096 x 11008 takes 12.1 us, q5_k 11008 x 4096
// 9.6; with codes in bf16 (x as three pieces, v_mfma_f32_4x4x4, what 16-bit float weights take below) 12.6 and 11.4.  Pieces of x
// as e5m2, which would be exact too, are no way out: the unit keeps sums of such bytes only to some 2^-11 of the largest product.
// Large matrices are bound by the bytes that the loads in flight bring (q4_k 28672 x 8192, f32: 26.5 us, 5.0 TB/s of 7.05, vector
// units busy for 46 % of it), small ones by the way from the launch to the staged x (q4_0 256 x 2048: 4.2 us, an empty kernel 2.5).
//
// Staged x, per turn: [step][chain][block of 32][half][digit][16 bytes], then [step][block] e as a byte, then
// the sums of x, f32, where the format has an offset: [step][slice][sub-block].
template <class F>
struct CodeTile {
    typedef Slice<F> S;
    static constexpr uint32_t ROWS = 16, ELEMS = 256 * S::TURN, CHAINS = 2;
    typedef Image<F, ROWS, S::TURN> I;
    static constexpr uint32_t DIGITS = CHAINS * 1024, EXPS = DIGITS * S::TURN, SUMS = EXPS + 8 * S::TURN + 8 * (S::TURN & 1);
    static constexpr uint32_t X_BYTES = SUMS + (S::OFFSET ? 16 * S::NSUB * S::TURN : 0), CLEAR = DIGITS, WAVE_BYTES = I::BYTES;

    template <class Load>
    static __device__ __forceinline__ void stage(uint8_t *lds, uint32_t turns, Load load) {
        constexpr uint32_t FRAGS = 32 * S::TURN;               // of eight elements; four lanes side by side have a block
        for (uint32_t i = threadIdx.x; i < FRAGS * turns; i += TILE_THREADS) {
            const uint32_t turn = i / FRAGS, f = i % FRAGS;
            const uint32_t step = f / 32, block = f / 4 % 8, half = f / 2 % 2;
            uint8_t *to = lds + turn * X_BYTES;
            float v[8];
            load(turn, f * 8, v);
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t b = __builtin_bit_cast(uint32_t, v[k]) & 0x7FFFFFFFu;
                top = b > top ? b : top;
            }
            const uint32_t o1 = dpp<QUAD_XOR1>(top);
            top = o1 > top ? o1 : top;
            const uint32_t o2 = dpp<QUAD_XOR2>(top);
            top = o2 > top ? o2 : top;
            uint32_t e = top >> 23;                            // biased
            e = e < 1 ? 1 : e;
            const uint32_t bad = e == 255 ? 0x7F7F7F7Fu : 0u;  // an infinity or NaN among them: e4m3's NaN
            e = e > 254 ? 254 : e;
            if (f % 4 == 0) to[EXPS + step * 8 + block] = (uint8_t)e;
            const int up = 158 - (int)e;
            uint32_t whole[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[k] = __builtin_rintf(__builtin_amdgcn_ldexpf(v[k], up));          // what is taken of x, times 2^up
                whole[k] = (uint32_t)__builtin_fabsf(v[k]);
            }
            if constexpr (S::OFFSET) {
                float sum = __builtin_amdgcn_ldexpf(((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])), -up);
                sum += dpp<QUAD_XOR1>(sum);
                float *sums = (float *)(to + SUMS) + step * 4 * S::NSUB;
                if constexpr (S::PLANES) {                     // 16 elements: column `half` of sub-block block % 4
                    if (f % 2 == 0) sums[(block / 4 * 2 + half) * 4 + block % 4] = sum;
                } else {
                    sum += dpp<QUAD_XOR2>(sum);
                    if (f % 4 == 0) sums[block] = sum;
                }
            }
            uint8_t *digits = to + step * DIGITS + block * 128 + half * 64 + f % 2 * 8;
            uint32_t sign[2], plane[2][4];                     // four elements a word; byte p of the whole numbers
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const uint32_t *n = whole + 4 * q;
                const float *x = v + 4 * q;
                const uint32_t s0 = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, x[1]), __builtin_bit_cast(uint32_t, x[0]), 0x0C0C0703u);
                const uint32_t s1 = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, x[3]), __builtin_bit_cast(uint32_t, x[2]), 0x07030C0Cu);
                sign[q] = ((s0 | s1) & 0x80808080u) | bad;
                const uint32_t a = __builtin_amdgcn_perm(n[1], n[0], 0x05010400u), b = __builtin_amdgcn_perm(n[3], n[2], 0x05010400u);
                plane[q][0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
                plane[q][1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
                const uint32_t c = __builtin_amdgcn_perm(n[1], n[0], 0x07030602u), d = __builtin_amdgcn_perm(n[3], n[2], 0x07030602u);
                plane[q][2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
                plane[q][3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
            }
#pragma unroll
            for (int p = 0; p < 4; ++p) {                      // the highest byte first: digits 2 p and 2 p + 1
                uint8_t *d = digits + p / 2 * 1024 + p % 2 * 32;
                const uint32_t w0 = plane[0][3 - p], w1 = plane[1][3 - p];
                *(u32x2 *)d = u32x2{((w0 >> 4) & LOW4) | sign[0], ((w1 >> 4) & LOW4) | sign[1]};
                *(u32x2 *)(d + 16) = u32x2{(w0 & LOW4) | sign[0], (w1 & LOW4) | sign[1]};
            }
        }
    }
    struct Me {
        uint32_t g, row;              // the lane's slice, its row's image
        uint32_t own, digits, exps;   // ~0 where the lane's part of A is not zero; its place in a step's digits; of its row's exponents
        // zeros: in shared memory, in front of the staged x
        __device__ __forceinline__ Me(uint32_t lane, const uint8_t *) {
            const uint32_t m = lane % 16, p = m % 4, gm = m / 4;
            g = lane / 16;
            row = m * I::ROW;
            own = gm == g ? ~0u : 0u;
            digits = S::PLANES ? (g / 2 * 4) * 128 + g % 2 * 64 + p * 16 : g * 256 + p * 16;
            exps = S::PLANES ? gm / 2 * 4 : gm * 2;
        }
    };
    struct Sums { float v[1]; };

    static __device__ __forceinline__ i32x8 join(u32x4 a, u32x4 b) {
        return {(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
    }
    template <int SB>
    static __device__ __forceinline__ f32x4 multiply(const i32x8 &x, uint32_t x_exp, const i32x8 &w, int w_exp, f32x4 d) {
        // a byte n is n 2^-9, and the first digit's unit 2^(e - 130): 6 in front of e - 127 and w_exp
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, w, d, 0, 0, SB, (int)x_exp, 0, w_exp + 127 + 6);
    }
    // `x`: the step's digits of the token, or the zeros; `exps`: the step's exponents
    template <int SB>
    static __device__ __forceinline__ f32x4 sub_block(const i32x8 &lo, const i32x8 &hi, const uint8_t *x, uint32_t exps) {
        f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t c = 0; c < CHAINS; ++c) {
            const uint8_t *at = x + c * 1024 + SB * 128;
            const u32x4 none = {0, 0, 0, 0};
            const i32x8 a = join(al16(at), S::PLANES ? none : al16(at + 64));
            d = multiply<SB>(a, exps, lo, S::template LOW_EXP<SB> - 16 * (int)c, d);
            if constexpr (S::HIGH) d = multiply<SB>(a, exps, hi, S::template HIGH_EXP<SB> - 16 * (int)c, d);
            if constexpr (from_minus_128<F>) {                 // -8 times 16 for each code, before the next chain is added
                constexpr int k = (int)0x88888888u;
                d = multiply<SB>(a, exps, i32x8{k, k, k, k, k, k, k, k}, S::template HIGH_EXP<SB> - 16 * (int)c, d);
            }
        }
        return d;
    }
    // the four digits' sums, each 16 times the next one's weight
    static __device__ __forceinline__ float joined(const f32x4 &d) {
        return __builtin_fmaf(__builtin_fmaf(d[3], 0.0625f, d[2]), 0.00390625f, __builtin_fmaf(d[1], 0.0625f, d[0]));
    }
    template <int SB>
    static __device__ __forceinline__ void add_sub(const typename S::Raw &raw, const Me &me, const uint8_t *clear, const uint8_t *x, uint32_t step,
                                                   Sums &acc) {
        constexpr int WORDS = S::SUB / 4;
        uint32_t b[WORDS], h[WORDS];
        S::template low<SB>(raw, b);
        if constexpr (S::HIGH) S::template high<SB>(raw, h);
        i32x8 lo, hi;
#pragma unroll
        for (int i = 0; i < 8; ++i) {                          // 16 codes: the second half meets zeros
            lo[i] = (int)b[i % WORDS];
            hi[i] = S::HIGH ? (int)h[i % WORDS] : 0;
        }
        const SubScale s = S::template scale<SB>(raw);
        const uint32_t exps = (S::PLANES ? al4(x + EXPS + step * 8 + me.exps) : al2(x + EXPS + step * 8 + me.exps));
        const uint8_t *digits = clear + ((uint32_t)(x + step * DIGITS + me.digits - clear) & me.own);
        const f32x4 d = sub_block<SB>(lo, hi, digits, exps);
        acc.v[0] = __builtin_fmaf(s.a, joined(d), acc.v[0]);
        if constexpr (S::OFFSET) {
            const float sum = ((const float *)(x + SUMS))[(step * 4 + me.g) * S::NSUB + SB];
            acc.v[0] = __builtin_fmaf(-s.c, sum, acc.v[0]);
        }
    }
    // one turn: `image` the wave's bytes, `x` the turn's staged x, `clear` the zeros, `left` bytes of the row from the turn on
    static __device__ __forceinline__ void add(const uint8_t *image, const Me &me, const uint8_t *clear, const uint8_t *x, uint32_t left,
                                               Sums &acc) {
#pragma unroll
        for (uint32_t step = 0; step < S::TURN; ++step) {
            typename S::Raw raw;
            raw.load(image + me.row, step, me.g, left);
            // one sub-block after the other: scheduled into each other they take the registers of more waves
            add_sub<0>(raw, me, clear, x, step, acc);
            __builtin_amdgcn_sched_barrier(0);
            add_sub<1>(raw, me, clear, x, step, acc);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (S::NSUB == 4) {
                add_sub<2>(raw, me, clear, x, step, acc);
                __builtin_amdgcn_sched_barrier(0);
                add_sub<3>(raw, me, clear, x, step, acc);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    static __device__ __forceinline__ void put(float *part, uint32_t lane, const Sums &acc) {
        float v = acc.v[0];
        v += __shfl_xor(v, 16);
        v += __shfl_xor(v, 32);
        if (lane < ROWS) part[lane] = v;
    }
};

// ---- 16-bit float weights, one token: bf16 pieces ------------------------------------------------------------
// x in CH bf16 pieces (bf16 one, f16 two, f32 three, exactly), the weights in one or two: products are exact, sums f32.
// A wave takes four rows; its quads (four neighbouring lanes, one lane per row) take 16 neighbouring slices at a time, and
// v_mfma_f32_4x4x4 with 16 blocks multiplies, in each quad, the four rows with the x that the quad's lanes hold, the same in
// all four: a lane's result is its row's.
// Staged x, per turn: [piece][k][slice] fragments of eight bf16, k = the fragment's place in its slice; the quads
// read the same k of neighbouring slices, so their addresses are consecutive; 16 bytes between one k and the next keep the
// staging threads, which run along k first, out of each other's banks.
template <class F, int CH>
struct FloatTile {
    typedef Slice<F> S;
    static constexpr uint32_t ROWS = 4, ELEMS = 1024;
    typedef Image<F, ROWS, S::TURN> I;
    static constexpr uint32_t K = 256 + 16, X_BYTES = CH * 8 * K, CLEAR = 0, WAVE_BYTES = I::BYTES;

    template <class Load>
    static __device__ __forceinline__ void stage(uint8_t *lds, uint32_t turns, Load load) {
        for (uint32_t i = threadIdx.x; i < 128 * turns; i += TILE_THREADS) {
            const uint32_t turn = i / 128, f = i % 128;
            float v[8];
            load(turn, f * 8, v);
            uint8_t *to = lds + turn * X_BYTES + f % 8 * K + f / 8 * 16;
#pragma unroll
            for (int p = 0; p < CH; ++p) {
                *(u32x4 *)(to + p * 8 * K) = u32x4{upper_halves(v[0], v[1]), upper_halves(v[2], v[3]), upper_halves(v[4], v[5]), upper_halves(v[6], v[7])};
                if (p + 1 < CH)
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = below_bf16(v[k]);
            }
        }
    }
    struct Me {
        uint32_t quad, row, x;
        __device__ __forceinline__ Me(uint32_t lane, const uint8_t *) : quad(lane / 4), row(lane % 4 * I::ROW), x(lane / 4 * 16) {}
    };
    struct Sums { float v[1]; };
    static __device__ __forceinline__ void add(const uint8_t *image, const Me &me, const uint8_t *, const uint8_t *x, uint32_t left, Sums &acc) {
        typename S::Raw raw;
        raw.load(image + me.row, me.quad, left);
        f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int piece = 0; piece < S::WP; ++piece) {
                uint32_t b[16];
                S::codes(raw, s, piece, b);
#pragma unroll
                for (int p = 0; p < CH; ++p)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const u32x4 a = al16(x + me.x + (p * 8 + 4 * s + k) * K);
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const u32x2 av = {a[2 * half], a[2 * half + 1]}, bv = {b[4 * k + 2 * half], b[4 * k + 2 * half + 1]};
                            d = __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(__builtin_bit_cast(s16x4, av), __builtin_bit_cast(s16x4, bv), d, 0, 0, 0);
                        }
                    }
            }
        acc.v[0] += d[0];
    }
    static __device__ __forceinline__ void put(float *part, uint32_t lane, const Sums &acc) {
        float v = acc.v[0];
        v += dpp<ROW_ROR8>(v);
        v += dpp<ROW_ROR4>(v);
        v += __shfl_xor(v, 16);
        v += __shfl_xor(v, 32);
        if (lane < ROWS) part[lane] = v;
    }
};

// ---- the loop over a row ----------------------------------------------------------------------------------------
// The wave's part of a tile: turns kp, kp + ksplit, ... of `turns`, the next one's bytes on the way while one is multiplied.
// All waves of the workgroup call this together, since they stage x for each other, `chunk` turns at a time.
//     at(turn)           {where the turn begins in the tile's first row, bytes of the row and of the tensor from there on}
//     load(turn, c, v)   elements [c, c + 8) of x in that turn
struct Turn {
    const uint8_t *base;
    uint32_t left;
    uint64_t room;
};
struct Share { uint32_t kp, ksplit, chunk, turns; };
template <class M, class At, class Load>
__device__ __forceinline__ void run_turns(uint8_t *image, uint8_t *clear, const typename M::I::Places &places, uint32_t reach, const Share &sh, At at, Load load,
                                          typename M::Sums &acc) {
    const uint32_t lane = threadIdx.x % 64;
    uint8_t *xs = clear + M::CLEAR;
    const typename M::Me me(lane, clear);
    typename M::I in;
    Turn next{};
    uint32_t turn = sh.kp;
    auto fetch = [&](uint32_t n) {
        next = at(n);
        in.fetch(places, next.base, next.room);
    };
    if (turn < sh.turns) fetch(turn);
    for (uint32_t i = threadIdx.x * 16; i < M::CLEAR; i += TILE_THREADS * 16) *(u32x4 *)(clear + i) = u32x4{0, 0, 0, 0};
    for (uint32_t first = 0; first < sh.turns; first += sh.chunk) {
        const uint32_t now = first + sh.chunk < sh.turns ? sh.chunk : sh.turns - first, end = first + now;
        if (first) __syncthreads();
        M::stage(xs, now, [&](uint32_t n, uint32_t c, float (&v)[8]) { load(first + n, c, v); });
        __syncthreads();
        for (; turn < end; turn += sh.ksplit) {
            wave_order();
            in.put(places, image, next.room, reach);
            wave_order();
            const uint32_t here = next.left;
            if (turn + sh.ksplit < sh.turns) fetch(turn + sh.ksplit);
            M::add(image, me, clear, xs + (turn - first) * M::X_BYTES, here, acc);
        }
    }
}
// The waves' sums to part[wave][row].
template <class M>
__device__ __forceinline__ void put_parts(float *part, uint32_t wave, const typename M::Sums &acc) {
    __syncthreads();                                   // the staged x is no longer needed
    M::put(part + wave * M::ROWS, threadIdx.x % 64, acc);
    __syncthreads();
}
template <class M>
__device__ __forceinline__ typename M::Sums no_sums() {
    typename M::Sums s;
#pragma unroll
    for (uint32_t t = 0; t < sizeof(s.v) / 4; ++t) s.v[t] = 0.0f;
    return s;
}

// ---- one matrix -----------------------------------------------------------------------------------------------
// One token.  A wave owns a tile of rows, or shares it with others that take other turns of its columns.
template <class F, class M>
__global__ __launch_bounds__(TILE_THREADS) void matvec_tiles(MatvecArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    typedef typename M::I I;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t group = wave / a.ksplit, groups = TILE_WAVES / a.ksplit;
    const uint32_t row_bytes = (uint32_t)(a.cols / F::N * F::BYTES), turns = (uint32_t)((a.cols + M::ELEMS - 1) / M::ELEMS);
    const uint64_t first_row = (a.first_tile + (uint64_t)blockIdx.x * groups) * M::ROWS;      // of the workgroup
    const uint64_t row = first_row + group * M::ROWS;                                         // of the wave
    const RowTile<uint64_t> tile = tile_at<M::ROWS>(row, a.rows);
    const uint64_t own = tile.own;
    const uint32_t rows = tile.rows;
    const uint8_t *w = a.w + own * row_bytes;
    const uint64_t behind = (a.rows - own - 1) * row_bytes;                                   // of the tensor, behind the row
    uint8_t *clear = lds + TILE_WAVES * M::WAVE_BYTES;
    typename M::Sums acc = no_sums<M>();
    run_turns<M>(lds + wave * M::WAVE_BYTES, clear, typename I::Places(threadIdx.x % 64, rows, row_bytes), I::reach(rows, row_bytes),
                 Share{wave % a.ksplit, a.ksplit, a.chunk, turns},
                 [&](uint32_t turn) {
                     const uint32_t off = turn * I::TURN_BYTES;
                     return Turn{w + off, row_bytes - off, behind + row_bytes - off};
                 },
                 [&](uint32_t turn, uint32_t c, float (&v)[8]) { load8(a.x, 0, (uint64_t)turn * M::ELEMS + c, a.cols, a.x_kind, v); },
                 acc);
    float *part = (float *)(clear + M::CLEAR);
    put_parts<M>(part, wave, acc);
    for (uint32_t r = threadIdx.x; r < groups * M::ROWS; r += TILE_THREADS) {
        const uint32_t g = r / M::ROWS;
        float v = 0.0f;
        for (uint32_t k = 0; k < a.ksplit; ++k) v += part[(g * a.ksplit + k) * M::ROWS + r % M::ROWS];
        if (first_row + r < a.rows) store_elem(a.y, first_row + r, a.y_kind, v);
    }
}

// Rows of 16-bit floats shorter than a piece of an image: a thread each.
template <class F>
__global__ __launch_bounds__(MV_THREADS) void matvec_short(MatvecArgs a) {
    const uint64_t r = (uint64_t)blockIdx.x * MV_THREADS + threadIdx.x;
    if (r >= a.rows) return;
    for (uint32_t t = 0; t < a.tokens; ++t) {
        float sum = 0.0f;
        for (uint32_t c = 0; c < a.cols; ++c) {
            const uint32_t b = ld2(a.w + 2 * (r * a.cols + c));
            sum = __builtin_fmaf(__is_same(F, WF16) ? h2f(b) : bf2f(b), load_elem(a.x, t * a.x_stride + c, a.x_kind), sum);
        }
        store_elem(a.y, t * a.y_stride + r, a.y_kind, sum);
    }
}

// ---- rows by id -----------------------------------------------------------------------------------------
struct RowsArgs {
    const uint8_t *w;
    const void *ids;
    void *y;
    uint64_t rows, cols, n, y_stride, row_bytes;
    uint64_t first;           // ids before this launch's
    uint32_t wide_ids;
};

// elements [c, c + N) of a packed row of `cols` elements; what is past the end of a float row: 0
template <class F, uint32_t N>
__device__ __forceinline__ void row_part(const uint8_t *row, uint32_t c, uint32_t cols, float (&v)[N]) {
    if constexpr (is_float_type<F>) {
#pragma unroll
        for (uint32_t i = 0; i < N; i += 2) {
            uint32_t w;
            if (c + i + 2 <= cols) w = ld4(row + 2 * (uint64_t)(c + i));
            else w = c + i < cols ? ld2(row + 2 * (uint64_t)(c + i)) : 0u;
            v[i] = __is_same(F, WF16) ? h2f(w & 0xFFFFu) : bf2f(w & 0xFFFFu);
            v[i + 1] = __is_same(F, WF16) ? h2f(w >> 16) : bf2f(w >> 16);
        }
    } else {
        const GlobalBytes at{row + (uint64_t)(c / F::N) * F::BYTES};
        F::template vals<N / 4>(at, 0u, c % F::N, F::scale(at, 0u, c % F::N), v);
    }
}

// A workgroup takes a piece of one row, as large as a tile of the decode kernels (kernels.h); each thread decodes what fills a
// 16-byte store, straight from the packed bytes: neighbouring threads read neighbouring words, and what they share of a block
// comes from the cache.  Bound by the bytes written.  2049 rows of 8192 q6_k elements to f32: 13.4 us, 6.0 TB/s; with stores
// that stay in the caches 18.8 us (a contiguous decode of as much, by way of shared memory, takes 14.4).
template <class F, class O>
__global__ __launch_bounds__(WG_THREADS) void get_rows(RowsArgs a) {
    typedef typename O::T T;
    const uint64_t i = a.first + blockIdx.y;
    const int64_t id = a.wide_ids ? ((const int64_t *)a.ids)[i] : (int64_t)((const int32_t *)a.ids)[i];
    const bool in_table = id >= 0 && (uint64_t)id < a.rows;
    const uint8_t *row = a.w + (in_table ? (uint64_t)id : 0) * a.row_bytes;
    T *y = (T *)a.y + i * a.y_stride;
    const uint32_t cols = (uint32_t)a.cols;
#pragma unroll
    for (uint32_t k = 0; k < STORES_PER_THREAD; ++k) {
        const uint32_t c = ((blockIdx.x * STORES_PER_THREAD + k) * WG_THREADS + threadIdx.x) * O::EPL;
        if (c >= cols) return;
        float v[O::EPL] = {};
        if (in_table) row_part<F>(row, c, cols, v);
        uint4v out;
        O::template store<false>((T *)&out, v);
        if (c + O::EPL <= cols) {
            st16_streaming(y + c, out);
        } else {
            for (uint32_t j = 0; c + j < cols; ++j) y[c + j] = ((const T *)&out)[j];
        }
    }
}

}  // namespace ggq
