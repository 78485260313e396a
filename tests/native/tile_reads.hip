// Where the products with packed weights read (matmul.h, dense.h), followed on the host with the kernels' own functions: every
// 16 bytes lie in the tensor, and what put shifts into place is what belongs there.  Prints the number of pieces that do not,
// for each kind of tile; with an argument, the number with every `last` below 0 taken as a far one (a plant: must not be 0).
#include "../../gguf_amd/csrc/dense.h"

#include <algorithm>
#include <cstdio>

using namespace ggq;

static bool plant;

template <class F, class I, uint32_t ROWS, uint32_t ELEMS>
static void turns(uint64_t own, uint32_t rows, uint64_t total, uint32_t cols, uint64_t &bad, uint64_t &pieces) {
    const uint32_t row_bytes = cols / F::N * F::BYTES;
    const int64_t end = (int64_t)(total * row_bytes);
    for (uint32_t turn = 0; turn * ELEMS < cols; ++turn) {
        const int64_t base = (int64_t)(own * row_bytes) + turn * I::TURN_BYTES;
        const uint64_t room = (uint64_t)(end - base);
        int32_t last = I::last(room);
        if (plant && last < 0) last = 1 << 30;
        const uint32_t left = row_bytes - turn * I::TURN_BYTES, reach = I::reach(rows, row_bytes);
        for (uint32_t lane = 0; lane < 64; ++lane) {
            const typename I::Places at(lane, rows, row_bytes);
            for (uint32_t i = 0; i < I::LOADS; ++i) {
                const uint32_t src = at.src[i], moved = room >= reach ? 0u : I::moved(src, last);
                const int64_t begin = base + I::begin_of_turn(last) + I::begin(src, last);
                bool ok = begin >= 0 && begin + 16 <= end;
                // bytes that are used: of the row, in front of its end; shifts of 15 and more leave one byte
                const uint32_t of_row = src % row_bytes;
                if (of_row < left || src / row_bytes) ok = ok && (src >= room || (begin + moved == base + src && moved < 16));
                bad += !ok;
                ++pieces;
            }
        }
    }
}

// one token: tiles of `N` rows and waves that have none; several: tiles moved back
template <class F, class I, uint32_t ELEMS, bool FULL, uint32_t ROWS>
static void kind(const char *name, uint32_t step, uint32_t least, uint32_t most) {
    uint64_t bad = 0, pieces = 0;
    for (uint64_t total : {1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 21, 33})
        for (uint32_t cols = least; cols <= most; cols += step) {
            if (cols > 2 * ELEMS + 8 && cols % ELEMS > 8 && cols % ELEMS + 8 < ELEMS && step < 8) continue;
            for (uint64_t row = 0; row < (FULL ? total + 2 * ROWS : total + 8 * ROWS); row += ROWS) {
                const RowTile<uint64_t> t = FULL ? full_tile_at<ROWS>(row, total) : tile_at<ROWS>(row, total);
                turns<F, I, ROWS, ELEMS>(t.own, t.rows, total, cols, bad, pieces);
            }
        }
    std::printf("%s %s %llu %llu\n", name, FULL ? "several" : "one", (unsigned long long)bad, (unsigned long long)pieces);
}

template <class F>
static void packed(const char *name) {
    typedef CodeTile<F> C;
    typedef DenseTile<F, X_F32, 1> D;
    kind<F, typename C::I, C::ELEMS, false, C::ROWS>(name, F::N, F::N, 9 * 256);
    kind<F, typename D::I, D::ELEMS, true, D::ROWS>(name, F::N, F::N, 9 * 256);
}
template <class F>
static void floats(const char *name) {
    typedef FloatTile<F, 3> C;
    typedef DenseTile<F, X_F32, 1> D;
    kind<F, typename C::I, C::ELEMS, false, C::ROWS>(name, 1, 8, 4104);
    kind<F, typename D::I, D::ELEMS, true, D::ROWS>(name, 1, 8, 1300);
}

int main(int argc, char **) {
    plant = argc > 1;
    floats<WF16>("f16");
    floats<WBF16>("bf16");
    packed<Q4_0>("q4_0");
    packed<Q4_1>("q4_1");
    packed<Q5_0>("q5_0");
    packed<Q5_1>("q5_1");
    packed<Q8_0>("q8_0");
    packed<Q8_1>("q8_1");
    packed<IQ4NL>("iq4_nl");
    packed<Q2K>("q2_k");
    packed<Q3K>("q3_k");
    packed<Q4K>("q4_k");
    packed<Q5K>("q5_k");
    packed<Q6K>("q6_k");
    packed<Q8K>("q8_k");
    packed<IQ4XS>("iq4_xs");
}
