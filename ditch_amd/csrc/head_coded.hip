// head_coded.hip — the head's products of few rows on weights that are not
// planes (rows_coded.h).
#include "head.h"

namespace ditch {

#ifdef CODED_KL
void launch_kl_coded(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks, const EpiKlStats &epi,
                     hipStream_t s) {
    with_terms(terms, [&](auto t) { launch_rows_coded<decltype(t)::value>(tile, p, mblocks, nblocks, epi, s); });
}
#else
void launch_loss_coded(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks, const EpiLossStats &epi,
                       hipStream_t s) {
    with_terms(terms, [&](auto t) { launch_rows_coded<decltype(t)::value>(tile, p, mblocks, nblocks, epi, s); });
}
#endif

}  // namespace ditch
