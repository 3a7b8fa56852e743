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

void launch_rows_out(const RowsGemm &g, void *out, int32_t dtype, int64_t stride, int64_t n, int64_t m, hipStream_t s) {
    const int64_t mb = ceil_div(m, 16), nb = ceil_div(n, 16);
    const int tile = rows_tiling(mb, nb, g.k32, g.nseg, g.terms, g.count[0], 1, false).tile;
    const EpiRows epi{out, stride, n, m, dtype, rows_wide(out, stride, dtype)};
    with_terms(g.terms, [&](auto terms) {
        launch_rows_gemm<true, true, decltype(terms)::value>(tile, g, mb, nb, epi, s);
    });
}

}  // namespace ditch
