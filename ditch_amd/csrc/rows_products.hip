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

void launch_rows_out(const RowsGemm &g, RowsArg out, RowsArg second, int32_t dtype, int64_t n, int64_t m, hipStream_t s) {
    const int64_t mb = ceil_div(m, 16), nb = second.p ? 2 * ceil_div(ceil_div(n, 16), 2) * 2 : ceil_div(n, 16);
    int tile = rows_tiling(mb, nb, g.k32, g.nseg, g.terms, g.count[0], 1, false).tile;
    // Large products of one term in 256 x 128, two workgroups a CU, of which one
    // multiplies while the other begins or ends: 3.40 ms against 3.55 in 256 x 256 for
    // 128256 x 4096 x 4096 (x W^T, read without transposing, keeps 256 x 256: 6.61 ms
    // against 6.94 for 8192 rows; the chip holds its clock longer for fewer LDS copies).
    if (tile == 0 && g.terms == 1) tile = 5;
    const bool wide = rows_wide(out.p, out.stride, dtype) && (!second.p || rows_wide(second.p, second.stride, dtype));
    const EpiRows epi{out.p, second.p, out.stride, second.stride, n, m, dtype, wide};
    with_terms(g.terms, [&](auto terms) {
        launch_rows_gemm<true, true, decltype(terms)::value>(tile, g, mb, nb, epi, s);
    });
}

}  // namespace ditch
