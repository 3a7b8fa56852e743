// head_coded.hip — the head's products of few rows on weights that are not
// planes (rows_coded.h). An object an epilogue (CODED), they compile in parallel.
#include "head.h"

namespace ditch {

#ifndef CODED
#error "compiled once for each epilogue"
#endif

#if CODED < 2
#if CODED == 0
void launch_loss_coded(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks, const EpiLossStats &epi,
                       hipStream_t s) {
#else
void launch_kl_coded(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks, const EpiKlStats &epi,
                     hipStream_t s) {
#endif
    with_terms(terms, [&](auto t) { launch_rows_coded<decltype(t)::value>(tile, p, mblocks, nblocks, epi, s); });
}
#else
#if CODED == 2
template <int T>
void launch_loss_grad_coded(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks,
                            const EpiLossGrad<T> &epi, hipStream_t s) {
    launch_rows_coded_grad<T>(tile, p, terms, mblocks, nblocks, epi, s);
}
#define OF_TERMS(T) template void launch_loss_grad_coded<T>(int, const RowsCoded &, int, int64_t, int64_t, const EpiLossGrad<T> &, hipStream_t);
#else
template <int T>
void launch_kl_grad_coded(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks,
                          const EpiKlGrad<T> &epi, hipStream_t s) {
    launch_rows_coded_grad<T>(tile, p, terms, mblocks, nblocks, epi, s);
}
#define OF_TERMS(T) template void launch_kl_grad_coded<T>(int, const RowsCoded &, int, int64_t, int64_t, const EpiKlGrad<T> &, hipStream_t);
#endif
OF_TERMS(1)
OF_TERMS(2)
OF_TERMS(3)
#endif

}  // namespace ditch
