// head_grad.hip — the gradients of the head's losses (head.hip has the
// formulas). The logits are formed again, a piece of the vocabulary at a time;
// the epilogue leaves d = dloss/dlogits of the piece as bf16 terms, [row][word],
// and two products over them give the piece's share of dx = d W and its rows of
// dW = d^T x.
#include "head.h"

namespace ditch {

struct HeadGradPlan {
    Planes x[2], d;
    int64_t piece = 0, nblocks = 0, ld = 0;
    RowsTiling tiling;
    int order = 1;  // of the products with d
    int w_terms = 1;  // rows_weight_terms: what the planes are for
    int coded = 0;  // the tile of rows_coded.h's product, 0: planes
    char *room = nullptr;
    float *part = nullptr;
    size_t bytes = 0;
};
static HeadGradPlan head_grad_plan(const TileView &w, int64_t n, int32_t dtype, bool kl, void *ws) {
    HeadGradPlan p;
    Carver c(ws);
    const int terms = row_terms(dtype);
    for (int i = 0; i < (kl ? 2 : 1); i++) {
        p.x[i] = row_planes(n, w.cols, terms);
        p.x[i].p = c.take(p.x[i].bytes());
    }
    p.nblocks = grad_blocks(n);
    const int td = grad_term_count(terms, n), wt = rows_weight_terms(w, terms);
    p.coded = rows_coded_tile(w, ceil_div(w.rows, 16), (kl ? 2 : 1) * p.nblocks, true);
    p.w_terms = kl ? ROWS_MAX_TERMS : terms;
    const int64_t held = p.coded ? 0 : weight_row_bytes(w, p.w_terms);
    p.piece = piece_rows(w.rows, p.nblocks * 32 * td + held);
    if (p.piece > ceil_div(w.rows, 64) * 64) p.piece = ceil_div(w.rows, 64) * 64;
    p.d = Planes{nullptr, p.nblocks, p.piece / 32, td};
    p.d.p = c.take(p.d.bytes());
    p.ld = ceil_div(w.cols, 4) * 4;
    p.order = rows_order_of(wt, td);
    if (p.coded) p.tiling.parts = coded_parts_count(w, p.piece, n, 1);
    else p.tiling = rows_tiling(ceil_div(w.cols, 16), p.nblocks, p.piece / 32, wt, td, p.order, 1, true, false);
    p.part = c.take<float>((size_t)p.tiling.parts * n * p.ld);
    if (held) p.room = c.take(weight_planes_shape(w, p.piece, p.w_terms).bytes());
    p.bytes = c.at;
    return p;
}

size_t head_loss_grad_workspace(const TileView &w, int64_t n, int32_t dtype, bool dw) {
    return head_grad_plan(w, n, dtype, false, nullptr).bytes;
}
size_t head_kl_grad_workspace(const TileView &w, int64_t n, int32_t dtype) {
    return head_grad_plan(w, n, dtype, true, nullptr).bytes;
}

// `fill` launches the product that leaves a piece's d.
template <typename Fill>
static void head_grad(const HeadGradPlan &p, int32_t dtype, RowsArg dx, RowsArg dw, int64_t n, const TileView &w,
                      hipStream_t s, Fill &&fill) {
    for (int64_t r = 0; r < w.rows; r += p.piece) {
        const int64_t rows = w.rows - r < p.piece ? w.rows - r : p.piece;
        const Planes wp = p.coded ? Planes{} : weight_planes(w, r, rows, p.w_terms, p.room, s);
        Planes d = p.d;
        d.units = ceil_div(rows, 64) * 2;
        fill(wp, d, r, rows);
        if (dx.p && p.coded) {
            CodedParts g;
            g.w[0] = w;
            g.d[0] = d.p;
            g.d_groups = (int32_t)d.groups;
            g.d_units = d.units;
            g.d_plane = d.plane_bytes();
            g.first = (int32_t)(r / 16);
            g.blocks = (int32_t)ceil_div(rows, 16);
            g.steps = (int32_t)ceil_div(rows, 32);
            g.parts = p.tiling.parts;
            launch_coded_parts(g, d.terms, p.part, p.ld, n, r > 0, s);
        } else if (dx.p) {
            RowsGemm g;
            g.a = rows_outer(wp);
            g.b = rows_inner(d);
            g.k32 = (int32_t)d.units;
            g.parts = p.tiling.parts;
            rows_pairs(g, wp, d, p.order);
            launch_rows_parts(p.tiling.tile, g, p.part, p.ld, n, w.cols, r > 0, s);
        }
        if (dw.p) {
            RowsGemm g;
            g.a = rows_outer(p.x[0]);
            g.b = rows_outer(d);
            g.k32 = (int32_t)(d.groups / 2);
            rows_pairs(g, p.x[0], d, d.terms);
            const RowsArg out{(char *)dw.p + r * dw.stride * (int64_t)row_size(dtype), dw.stride};
            launch_rows_out(g, out, RowsArg{}, dtype, rows, w.cols, s);
        }
    }
    if (dx.p) launch_join_parts(dx.p, dtype, dx.stride, p.part, p.tiling.parts, n * p.ld, p.ld, n, w.cols, s);
}

template <int TB, int T>
static void fill_loss(const HeadGradPlan &p, const RowsIn &in, const TileView &w, const Planes &wp, const Planes &d, int64_t row0,
                      int64_t rows, int64_t n, const int32_t *targets, const float *lse, const float *dloss, hipStream_t s) {
    const EpiLossGrad<T> epi{d, targets, lse, dloss, n, rows, row0, w.rows};
    if (p.coded) {
        RowsCoded c = coded_product(w, in);
        c.first = (int32_t)(row0 / 16);
        c.blocks = (int32_t)ceil_div(rows, 16);
        launch_loss_grad_coded<T>(p.coded, c, TB, d.units * 2, p.nblocks, epi, s);
        return;
    }
    launch_rows_gemm<false, false, TB>(logits_tile(w, rows, p.x[0], p.nblocks, false), logits_gemm(wp, in, false),
                                      d.units * 2, p.nblocks, epi, s);
}
template <int TB, int T>
static void fill_kl(const HeadGradPlan &p, const RowsIn &in, const TileView &w, const Planes &wp, const Planes &d, int64_t row0,
                    int64_t rows, int64_t n, const float *lse_base, const float *lse_trial,
                    const float *dkl, hipStream_t s) {
    const EpiKlGrad<T> epi{d, lse_base, lse_trial, dkl, n, rows};
    if (p.coded) {
        RowsCoded c = coded_product(w, in);
        c.first = (int32_t)(row0 / 16);
        c.blocks = (int32_t)ceil_div(rows, 16);
        launch_kl_grad_coded<T>(p.coded, c, TB, d.units * 2, 2 * p.nblocks, epi, s);
        return;
    }
    launch_rows_gemm<false, false, TB>(logits_tile(w, rows, p.x[0], 2 * p.nblocks, true), logits_gemm(wp, in, true),
                                      d.units * 2, 2 * p.nblocks, epi, s);
}

void launch_head_loss_grad(int32_t dtype, RowsArg dx, RowsArg dw, RowsArg x, int64_t n, const TileView &w,
                           const int32_t *targets, const float *lse, const float *dloss, void *ws, hipStream_t s) {
    const HeadGradPlan p = head_grad_plan(w, n, dtype, false, ws);
    // (rows without a target are zeros in d^T x, where an infinity or NaN times their zero d would stay)
    const RowsIn in = rows_in(dtype, n, w.cols, x, nullptr, p.x, s, targets);
    if (dw.p && in.x.p != p.x[0].p) launch_pack_rows(p.x[0], x.p, dtype, n, w.cols, x.stride, s, targets);  // (read transposed)
    head_grad(p, dtype, dx, dw, n, w, s, [&](const Planes &wp, const Planes &d, int64_t row0, int64_t rows) {
        auto f = p.x[0].terms == 3 ? fill_loss<3, 3> : p.x[0].terms == 2 ? fill_loss<2, 2> : p.d.terms == 2 ? fill_loss<1, 2> : fill_loss<1, 1>;
        f(p, in, w, wp, d, row0, rows, n, targets, lse, dloss, s);
    });
}

void launch_head_kl_grad(int32_t dtype, RowsArg dx, RowsArg base, RowsArg trial, int64_t n, const TileView &w,
                         const float *lse_base, const float *lse_trial, const float *dkl, void *ws, hipStream_t s) {
    const HeadGradPlan p = head_grad_plan(w, n, dtype, true, ws);
    const RowsIn in = rows_in(dtype, n, w.cols, base, &trial, p.x, s);
    head_grad(p, dtype, dx, RowsArg{}, n, w, s, [&](const Planes &wp, const Planes &d, int64_t row0, int64_t rows) {
        auto f = p.x[0].terms == 3 ? fill_kl<3, 3> : p.x[0].terms == 2 ? fill_kl<2, 2> : p.d.terms == 2 ? fill_kl<1, 2> : fill_kl<1, 1>;
        f(p, in, w, wp, d, row0, rows, n, lse_base, lse_trial, dkl, s);
    });
}

}  // namespace ditch
