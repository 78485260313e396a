// launch.h -- the launches of the products with packed weights, block type by block type (matmul_type.hip), for their entry
// points (matmul.hip).
#pragma once
#include "choice.h"

namespace ggq {

template <class F>
struct Launch {
    static uint64_t matvec(MatvecArgs a, uint64_t tokens, hipStream_t st);                            // returns how many tokens it took
    static void rows(const RowsArgs &a, uint32_t y_kind, uint32_t n, hipStream_t st);                 // n: ids of this launch
    static void up(MoeArgs a, hipStream_t st);
    static void down(MoeArgs a, hipStream_t st);
};

}  // namespace ggq
