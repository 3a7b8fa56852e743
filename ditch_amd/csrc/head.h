// head.h — what the head's losses (head.hip) and their gradients
// (head_grad.hip) share: pieces of the vocabulary, the logits' product.
#pragma once
#include "rows_gemm.h"

namespace ditch {

__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(__fmul_rn(x, 1.4426950408889634f)); }


// Words of a piece: what is held for one (d, and the weight's planes where they
// are decoded) stays within about 256 MB, the size of the last cache; pieces of
// whole 256-row tiles, alike in size.
inline int64_t piece_rows(int64_t vocab, int64_t per_row) {
    const int64_t most = ((int64_t)256 << 20) / (per_row > 0 ? per_row : 1);
    int64_t pieces = most >= vocab ? 1 : ceil_div(vocab, most < 256 ? 256 : most);
    return ceil_div(ceil_div(vocab, pieces), 256) * 256;
}

inline int64_t weight_row_bytes(const TileView &w) {
    return weight_is_planes(w) ? 0 : weight_planes_shape(w, 16).plane_bytes() * weight_terms(w) / 16;
}
inline int order_of(int a, int b) { return a > b ? a : b; }
inline RowsGemm logits_gemm(const Planes &wp, const Planes &x, const Planes *second) {
    RowsGemm g;
    g.a = rows_inner(wp);
    g.b = rows_inner(x);
    if (second) {
        g.b.paired = 1;
        g.b.pair = second->p - x.p;
    }
    g.k32 = (int32_t)x.units;
    rows_pairs(g, wp, x, order_of(wp.terms, x.terms));
    return g;
}

inline int logits_tile(const TileView &w, int64_t rows, const Planes &x, int64_t nblocks) {
    const int a = weight_terms(w);
    return rows_tiling(ceil_div(rows, 16), nblocks, x.units, a, x.terms, order_of(a, x.terms), 1, false).tile;
}

}  // namespace ditch
