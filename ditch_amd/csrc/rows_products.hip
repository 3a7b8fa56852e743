// rows_products.hip — the products that gradients end in: d W as partial sums,
// d^T x as the caller's rows.
#include "rows_gemm.h"

namespace ditch {

void launch_rows_parts(int tile, const RowsGemm &g, float *part, int64_t ld, int64_t n, int64_t m, bool add, hipStream_t s) {
    const EpiParts epi{part, n * ld, ld, n, m, add};
    with_terms(g.terms, [&](auto terms) {
        launch_rows_gemm<true, false, decltype(terms)::value>(tile, g, ceil_div(m, 16), ceil_div(n, 64) * 4, epi, s);
    });
}

// Both operands are read transposed, k is the rows of x, and what is written
// weighs more. One term: 256 x 128, two workgroups a CU, of which one multiplies while
// the other begins or ends (128256 x 4096 of 4096 rows 3.40 ms, 256 x 256 3.55; of
// 60 rows 319 us, 256 x 256 373, 128 x 128 385), or 128 x 128 where those are few (4864 x
// 896 of 1000 rows 20 us, 23, 33). Several terms: 256 x 256 or 128 x 128, by what
// they pad (of f16, 1000 rows: 128256 x 4096 2.73 and 3.18 ms, 151936 x 896 1.00 and
// 0.82) and again by how many there are.
static int rows_out_tile(int64_t mb, int64_t nb, int terms) {
    auto tiles = [&](int64_t bm, int64_t bn) { return ceil_div(mb, bm) * ceil_div(nb, bn); };
    if (terms == 1) return tiles(16, 8) < 300 ? 1 : 5;
    return tiles(16, 16) < 512 || 256 * tiles(16, 16) > 72 * tiles(8, 8) ? 1 : 0;
}

void launch_rows_out(const RowsGemm &g, RowsArg out, RowsArg second, int32_t dtype, int64_t n, int64_t m, hipStream_t s) {
    const int64_t mb = ceil_div(m, 16), nb = second.p ? 2 * ceil_div(ceil_div(n, 16), 2) * 2 : ceil_div(n, 16);
    const int tile = rows_out_tile(mb, nb, g.terms);
    const bool wide = rows_wide(out.p, out.stride, dtype) && (!second.p || rows_wide(second.p, second.stride, dtype));
    const EpiRows epi{out.p, second.p, out.stride, second.stride, n, m, dtype, wide};
    with_terms(g.terms, [&](auto terms) {
        launch_rows_gemm<true, true, decltype(terms)::value>(tile, g, mb, nb, epi, s);
    });
}

}  // namespace ditch
