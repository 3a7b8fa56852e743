// glu_coded.hip — the gated block's product of few rows on weights that are not
// planes (rows_coded.h).
#include "glu.h"

namespace ditch {

void launch_glu_coded(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks, const EpiGlu &epi,
                      hipStream_t s) {
    with_terms(terms, [&](auto t) { launch_rows_coded<decltype(t)::value>(tile, p, mblocks, nblocks, epi, s); });
}

}  // namespace ditch
