// matmul.h -- products with packed weights: the kernels.
//
//     y[t][r] = sum over c of W[r][c] * x[t][c]        W packed blocks (formats.h), x and y f32 / f16 / bf16
//
// and what surrounds them in a decoding step: rows of a packed table by id, and a mixture-of-experts layer.
#pragma once
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

// ---- the product ----------------------------------------------------------------------------------------
struct MatvecArgs {
    const uint8_t *w;
    const void *x;
    void *y;
    uint64_t rows, cols, x_stride, y_stride;
    uint64_t first_tile;      // groups of four rows before this launch's
    uint32_t tokens;          // of this launch's group: at most NC / parts
    uint32_t x_kind, y_kind;
    uint32_t parts;           // columns that a token takes: its bf16 pieces, or 1 where they follow each other
    uint32_t chunk;           // steps staged at a time, a multiple of ksplit
    uint32_t ksplit;          // waves that share a row group's columns: 1, 2, 4 or 8
};

constexpr uint32_t MV_THREADS = 256;      // the other kernels here
constexpr uint32_t QD_WAVES = 8, QD_THREADS = 64 * QD_WAVES;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// x in shared memory, as the matrix unit takes it: fragments of eight bf16 (16 bytes).  A step (16 slices, 1024 elements)
// is [chain][k][slice][column], k = the fragment's place in its slice: the 16 quads of a wave read the same k of 16
// neighbouring slices, so their addresses are consecutive and all other parts of the address are constants.  16 bytes
// between one k and the next keep the staging threads, which run along k first, out of each other's banks.  Behind the
// fragments, for formats with an offset, the sum of x over each sub-block: [sub-block][slice][column], f32, a token's whole
// sum in the first of its columns and zero in the others.
//   NC columns: tokens times their pieces side by side; CHAIN: pieces one after the other into the same columns.
template <class F, int NC, int CHAIN>
struct XStep {
    typedef Slice<F> S;
    static constexpr uint32_t K = 256 * NC + 16;
    static constexpr uint32_t SUMS = CHAIN * 8 * K;
    static constexpr uint32_t BYTES = SUMS + (S::OFFSET ? S::NSUB * 64 * NC : 0);
};

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
constexpr int QUAD_XOR1 = 0xB1, QUAD_XOR2 = 0x4E, ROW_ROR4 = 0x124, ROW_ROR8 = 0x128;

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

// Stages `steps` steps of x.  load(step, t, f, v): the eight elements of fragment f (of 128) of that step, for token t.
template <class F, int NC, int CHAIN, class Load>
__device__ __forceinline__ void stage_x(uint8_t *lds, uint32_t steps, uint32_t tokens, uint32_t parts, Load load) {
    typedef Slice<F> S;
    typedef XStep<F, NC, CHAIN> X;
    const uint32_t frags = steps * 128;
    for (uint32_t i = threadIdx.x; i < frags * tokens; i += blockDim.x) {       // whole waves: frags is a multiple of 64
        const uint32_t t = NC == 1 || tokens == 1 ? 0 : i / frags, f = (i - t * frags) & 127u, n = (i - t * frags) >> 7;
        uint32_t sl, k;
        if constexpr (S::PLANES) {
            sl = ((f >> 3) & 12u) | ((f >> 3) & 2u) | ((f >> 1) & 1u);
            k = ((f >> 1) & 6u) | (f & 1u);
        } else {
            sl = f >> 3;
            k = f & 7u;
        }
        uint8_t *step = lds + n * X::BYTES;
        float v[8];
        load(n, t, f, v);
        const uint32_t col = t * parts;
        if constexpr (S::OFFSET) {
            float sum = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
            sum += dpp<QUAD_XOR1>(sum);
            if (S::SUB == 32) sum += dpp<QUAD_XOR2>(sum);
            if (f % (S::SUB / 8) == 0) {
                float *to = (float *)(step + X::SUMS) + (k / (S::SUB / 8) * 16 + sl) * NC + col;
                to[0] = sum;
                for (uint32_t p = 1; p < parts; ++p) to[p] = 0.0f;
            }
        }
        uint8_t *to = step + k * X::K + (sl * NC + col) * 16;
        const uint32_t pieces = CHAIN > 1 ? CHAIN : parts, stride = CHAIN > 1 ? 8 * X::K : 16;
        for (uint32_t p = 0; p < pieces; ++p, to += stride) {
            const u32x4 w = {upper_halves(v[0], v[1]), upper_halves(v[2], v[3]), upper_halves(v[4], v[5]), upper_halves(v[6], v[7])};
            *(u32x4 *)to = w;
            if (p + 1 < pieces)
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = below_bf16(v[j]);
        }
    }
}

// acc[t][c] += sub-block S of the lane's slice of its row in tile t, times column c of x, for RT tiles of four rows that
// share the fragments.  `x`: the step's fragments, from the lane's own on; `sums`: the step's sums from the lane's slice on.
template <class F, int NC, int CHAIN, int RT, int S>
__device__ __forceinline__ void add_sub(const typename Slice<F>::Raw (&raw)[RT], const typename Slice<F>::Lane &lane, const uint8_t *x,
                                        const uint8_t *sums, float (&acc)[RT][NC]) {
    typedef Slice<F> T;
    typedef XStep<F, NC, CHAIN> X;
    constexpr int FRAGS = T::SUB / 8, WORDS = T::SUB / 2;
    constexpr int WP = [] { if constexpr (is_float_type<F>) return T::WP; else return 1; }();
    f32x4 d[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) d[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int piece = 0; piece < WP; ++piece) {
        uint32_t b[RT][WORDS];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            if constexpr (is_float_type<F>) T::template codes<S>(raw[t], lane, b[t], piece);
            else T::template codes<S>(raw[t], lane, b[t]);
        }
#pragma unroll
        for (int p = 0; p < CHAIN; ++p)
#pragma unroll
            for (int k = 0; k < FRAGS; ++k) {
                const u32x4 a = al16(x + (p * 8 + S * FRAGS + k) * X::K);
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int t = 0; t < RT; ++t) {
                        const u32x2 av = {a[2 * half], a[2 * half + 1]}, bv = {b[t][4 * k + 2 * half], b[t][4 * k + 2 * half + 1]};
                        d[t] = __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(__builtin_bit_cast(s16x4, av), __builtin_bit_cast(s16x4, bv), d[t], 0, 0, 0);
                    }
            }
    }
    float sum[NC];
    if constexpr (T::OFFSET) {
#pragma unroll
        for (int c = 0; c < NC; ++c) sum[c] = ((const float *)(sums + S * 64 * NC))[c];
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const SubScale s = T::template scale<S>(raw[t], lane);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            acc[t][c] = __builtin_fmaf(s.a, d[t][c], acc[t][c]);
            if constexpr (T::OFFSET) acc[t][c] = __builtin_fmaf(-s.c, sum[c], acc[t][c]);
        }
    }
}
template <class F, int NC, int CHAIN, int RT>
__device__ __forceinline__ void add_slices(const typename Slice<F>::Raw (&raw)[RT], const typename Slice<F>::Lane &lane, const uint8_t *x,
                                           const uint8_t *sums, float (&acc)[RT][NC]) {
    add_sub<F, NC, CHAIN, RT, 0>(raw, lane, x, sums, acc);
    add_sub<F, NC, CHAIN, RT, 1>(raw, lane, x, sums, acc);
    if constexpr (Slice<F>::NSUB == 4) {
        add_sub<F, NC, CHAIN, RT, 2>(raw, lane, x, sums, acc);
        add_sub<F, NC, CHAIN, RT, 3>(raw, lane, x, sums, acc);
    }
}

// A wave's packed bytes of one step: 4 * RT rows.  Lanes that multiply together hold different rows, so loads straight
// into their registers would touch a line per lane: the memory pipeline takes about two cycles for each, which held the
// products at 4.1 TB/s whatever the format's arithmetic.  Instead neighbouring lanes load neighbouring 16-byte pieces into
// registers, one step ahead, and hand them over through the wave's own part of shared memory.
template <class F, int RT>
struct Image {
    typedef Slice<F> S;
    static constexpr uint32_t ROWS = 4 * RT, PIECES = (S::UNIT + 15) / 16, PER_ROW = PIECES * S::UNITS, LOADS = (PER_ROW * ROWS + 63) / 64;
    static constexpr uint32_t UNIT = PIECES * 16, ROW = UNIT * S::UNITS + (UNIT * S::UNITS % 64 == 32 ? 32 : 0) + 16 * (UNIT * S::UNITS % 32 / 16);
    static constexpr uint32_t BYTES = ROW * ROWS;
    // where this lane's pieces are
    struct Places {
        uint32_t src[LOADS], dst[LOADS];      // from the tile's first row on; in the image
        // `rows` of the tile's rows exist; the others are the last one again
        __device__ __forceinline__ Places(uint32_t lane, uint32_t rows, uint32_t row_bytes) {
#pragma unroll
            for (uint32_t i = 0; i < LOADS; ++i) {
                uint32_t p = i * 64 + lane;
                if (p >= PER_ROW * ROWS) p = PER_ROW * ROWS - 1;
                const uint32_t r = p / PER_ROW, u = p % PER_ROW / PIECES, c = p % PIECES * 16;
                src[i] = (r < rows ? r : rows - 1) * row_bytes + u * S::UNIT + c;
                dst[i] = r * ROW + u * UNIT + c;
            }
        }
    };
    u32x4 v[LOADS];

    // The step that begins at `base` (in the tile's first row).  A unit's last piece and a row's last step may reach beyond
    // them, into whatever follows in the tensor; `room` bytes of the tensor are left from base on, and where the furthest
    // piece would end behind them (`reach`), pieces are moved back to end with it and shifted into place.
    __device__ __forceinline__ void fetch(const Places &at, const uint8_t *base, uint64_t room, uint32_t reach) {
        if (room >= reach) {
#pragma unroll
            for (uint32_t i = 0; i < LOADS; ++i) v[i] = ld16(base + at.src[i]);
        } else {
            const int32_t limit = (int32_t)room - 16;
#pragma unroll
            for (uint32_t i = 0; i < LOADS; ++i) {
                const int32_t from = (int32_t)at.src[i] < limit ? (int32_t)at.src[i] : limit;
                const uint32_t back = at.src[i] - (uint32_t)from;
                v[i] = shifted(ld16(base + from), back < 15 ? back : 15);
            }
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
    __device__ __forceinline__ void put(const Places &at, uint8_t *image) const {
#pragma unroll
        for (uint32_t i = 0; i < LOADS; ++i) *(u32x4 *)(image + at.dst[i]) = v[i];
    }
};

// Orders a wave's own accesses to shared memory (its lanes read what others of the wave wrote).
__device__ __forceinline__ void wave_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// Sum over the 16 quads of a wave: afterwards every lane holds its row's total.
__device__ __forceinline__ float quads_sum(float v) {
    v += dpp<ROW_ROR8>(v);
    v += dpp<ROW_ROR4>(v);
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
    return v;
}

// One to four tokens.  A wave owns four rows; its quads (four neighbouring lanes, one lane per row) take 16 neighbouring
// slices at a time, each lane the packed bytes of its row's slice.  v_mfma_f32_4x4x4 with 16 blocks multiplies, in each
// quad, the four rows' codes with up to four columns of x that the quad's lanes hold: every lane ends with its own row's
// products, so that the sub-block's scale is applied in the lane that loaded it.  Columns are tokens, or the bf16 pieces
// of a token (f32 = three pieces, exactly; products with codes are exact, sums are f32).
template <class F, int NC, int CHAIN, int RT>
__global__ __launch_bounds__(QD_THREADS) void matvec_quads(MatvecArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    typedef Slice<F> S;
    typedef XStep<F, NC, CHAIN> X;
    typedef Image<F, RT> I;
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), quad = lane / 4;
    const uint32_t kp = wave % a.ksplit, group = wave / a.ksplit, groups = QD_WAVES / a.ksplit;
    const uint32_t row_bytes = (uint32_t)(a.cols / F::N * F::BYTES), steps = (uint32_t)((a.cols + 1023) / 1024);
    const uint64_t first_row = (a.first_tile + (uint64_t)blockIdx.x * groups) * I::ROWS;      // of the workgroup
    const uint64_t row = first_row + group * I::ROWS;                                         // of the wave
    const uint64_t own = row < a.rows ? row : a.rows - 1;
    const uint32_t rows = a.rows - own < I::ROWS ? (uint32_t)(a.rows - own) : I::ROWS;
    const uint8_t *w = a.w + own * row_bytes + (uint64_t)kp * S::STEP;
    uint32_t left = row_bytes - (kp < steps ? kp : steps - 1) * S::STEP;       // of each row, from w on
    const uint32_t reach = (rows - 1) * row_bytes + (S::UNITS - 1) * S::UNIT + I::UNIT;
    const uint64_t behind = (a.rows - own - 1) * row_bytes;                    // of the tensor, behind the tile's first row
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
    if (kp < steps) in.fetch(places, w, behind + left, reach);
    uint32_t step = kp;
    for (uint32_t first = 0; first < steps; first += a.chunk) {
        const uint32_t now = first + a.chunk < steps ? a.chunk : steps - first, end = first + now;
        if (first) __syncthreads();
        stage_x<F, NC, CHAIN>(xs, now, a.tokens, a.parts, [&](uint32_t n, uint32_t t, uint32_t f, float (&v)[8]) {
            load8(a.x, t * a.x_stride, ((uint64_t)(first + n) * 128 + f) * 8, a.cols, a.x_kind, v);
        });
        __syncthreads();
        for (; step < end; step += a.ksplit) {
            wave_order();
            in.put(places, image);
            wave_order();
            const uint32_t here = left;
            if (step + a.ksplit < steps) {
                w += (uint64_t)a.ksplit * S::STEP;
                left -= a.ksplit * S::STEP;
                in.fetch(places, w, behind + left, reach);
            }
            typename S::Raw raw[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t) raw[t].load(image + (t * 4 + lane % 4) * I::ROW, me, here);
            const uint32_t at = (step - first) * X::BYTES;
            add_slices<F, NC, CHAIN, RT>(raw, me, x + at, sums + at, acc);
        }
    }
    __syncthreads();                                   // the staged x is no longer needed
    float *part = (float *)xs;                         // [wave][column][row]
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const float v = quads_sum(acc[t][c]);
            if (lane < 4) part[(wave * NC + c) * I::ROWS + t * 4 + lane] = v;
        }
    __syncthreads();
    // one thread per row and token: the waves' parts, and the token's pieces
    if (threadIdx.x < groups * I::ROWS * a.tokens) {
        const uint32_t r = threadIdx.x % (groups * I::ROWS), t = threadIdx.x / (groups * I::ROWS), g = r / I::ROWS;
        const uint64_t out = first_row + r;
        float v = 0.0f;
        for (uint32_t k = 0; k < a.ksplit; ++k)
            for (uint32_t p = 0; p < a.parts; ++p) v += part[((g * a.ksplit + k) * NC + t * a.parts + p) * I::ROWS + r % I::ROWS];
        if (out < a.rows) store_elem(a.y, t * a.y_stride + out, a.y_kind, v);
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

// a sum of nothing
static __global__ __launch_bounds__(MV_THREADS) void fill_zero(MatvecArgs a) {
    const uint64_t r = (uint64_t)blockIdx.x * MV_THREADS + threadIdx.x;
    if (r >= a.rows) return;
    for (uint32_t t = 0; t < a.tokens; ++t) store_elem(a.y, t * a.y_stride + r, a.y_kind, 0.0f);
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

}  // namespace ggq
