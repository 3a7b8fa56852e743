// glu_coded.hip — the gated block's products of few rows on weights that are not
// planes (rows_coded.h). An object a direction (CODED_GRAD), they compile in parallel.
#include "glu.h"

namespace ditch {

#ifndef CODED_GRAD
void launch_glu_coded(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks, const EpiGlu &epi,
                      hipStream_t s) {
    with_terms(terms, [&](auto t) { launch_rows_coded<decltype(t)::value>(tile, p, mblocks, nblocks, epi, s); });
}
#else
template <int T>
void launch_glu_grad_coded(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks,
                           const EpiGluGrad<T> &epi, hipStream_t s) {
    launch_rows_coded_grad<T>(tile, p, terms, mblocks, nblocks, epi, s);
}
#define OF_TERMS(T) template void launch_glu_grad_coded<T>(int, const RowsCoded &, int, int64_t, int64_t, const EpiGluGrad<T> &, hipStream_t);
OF_TERMS(1)
OF_TERMS(2)
OF_TERMS(3)
#endif

}  // namespace ditch
