// glu.hip — the gated block over rows, y = act(x Wg^T) * (x Wu^T), and its
// gradient.
//
// One product over both matrices, their 16-row blocks interleaved, so that a
// lane holds a gate and the up value beside it: y is formed in registers and is
// all that is written. Gradient: the same product again, its epilogue reads dy and
// leaves dg = dy u act'(g) and du = dy act(g) as bf16 terms; then dx = dg Wg +
// du Wu is one product over both pairs, and dWg = dg^T x, dWu = du^T x.
#include "glu.h"

namespace ditch {

// x and both matrices as planes, one operand after the other.
struct GluPlan {
    Planes x, dg, du;
    char *room[2] = {nullptr, nullptr};
    int64_t ld = 0, nblocks = 0;
    int order = 1, tile = 0, coded = 0;  // coded: the tile of rows_coded.h's product, 0: planes
    RowsTiling back;
    int back_order = 1;  // of the product with d
    float *part = nullptr;
    size_t bytes = 0;
};
static GluPlan glu_plan(const TileView &w, const TileView &up, int64_t n, int32_t dtype, bool grad, void *ws) {
    GluPlan p;
    Carver c(ws);
    const int64_t nblocks = p.nblocks = grad ? grad_blocks(n) : row_blocks(n);
    const int terms = row_terms(dtype), wt = rows_weight_terms(w, terms);
    p.order = rows_order_of(wt, terms);
    p.x = row_planes(n, w.cols, terms);
    p.x.p = c.take(p.x.bytes());
    if (rows_coded_pair(w, up)) p.coded = rows_coded_tile(w, 2 * ceil_div(w.rows, 16), nblocks, grad);
    if (!weight_is_planes(w) && !p.coded)
        for (int i = 0; i < 2; i++) p.room[i] = c.take(weight_planes_shape(w, w.rows, terms).bytes());
    if (grad) {
        const int td = grad_term_count(terms, n);
        p.back_order = rows_order_of(wt, td);
        for (Planes *d : {&p.dg, &p.du}) {
            *d = Planes{nullptr, nblocks, ceil_div(w.rows, 64) * 2, td};
            d->p = c.take(d->bytes());
        }
        p.ld = ceil_div(w.cols, 4) * 4;
        if (p.coded) p.back.parts = coded_parts_count(w, w.rows, n, 2);
        else p.back = rows_tiling(ceil_div(w.cols, 16), nblocks, p.dg.units, wt, td, p.back_order, 2, true, false);
        p.part = c.take<float>((size_t)p.back.parts * n * p.ld);
    }
    p.tile = rows_tiling(2 * ceil_div(w.rows, 16), nblocks, ceil_div(w.cols, 64) * 2, wt, terms, p.order, 1, false, true).tile;
    p.bytes = c.at;
    return p;
}

size_t glu_rows_workspace(const TileView &gate, const TileView &up, int64_t n, int32_t dtype) {
    return glu_plan(gate, up, n, dtype, false, nullptr).bytes;
}
size_t glu_rows_grad_workspace(const TileView &gate, const TileView &up, int64_t n, int32_t dtype, bool dw) {
    return glu_plan(gate, up, n, dtype, true, nullptr).bytes;
}

static RowsCoded glu_coded(const RowsIn &in, const TileView &gate, const TileView &up) {
    RowsCoded c;
    c.w[0] = gate;
    c.w[1] = up;
    c.paired = 1;
    c.b = in.op;
    c.x = in.x.p;
    c.x_plane = in.x.plane_bytes();
    c.blocks = (int32_t)ceil_div(gate.rows, 16);
    c.stages = (int32_t)gate.units_k;
    return c;
}
static RowsGemm glu_gemm(const GluPlan &p, const RowsIn &in, const Planes &wg, const Planes &wu) {
    RowsGemm g;
    g.a = rows_inner(wg);
    g.a.paired = 1;
    g.a.pair = wu.p - wg.p;
    g.b = in.op;
    g.k32 = (int32_t)ceil_div(wg.units, 2) * 2;
    rows_pairs(g, wg, in.x, p.order);
    return g;
}

void launch_glu_rows(int32_t dtype, RowsArg out, RowsArg x, int64_t n, const TileView &gate, const TileView &up,
                     uint32_t act, void *ws, hipStream_t s) {
    const GluPlan p = glu_plan(gate, up, n, dtype, false, ws);
    const RowsIn in = rows_in(dtype, n, gate.cols, x, nullptr, &p.x, s);
    const EpiGlu epi{out.p, out.stride, n, gate.rows, dtype, rows_wide(out.p, out.stride, dtype), act};
    if (p.coded) {
        const RowsCoded c = glu_coded(in, gate, up);
        launch_glu_coded(p.coded, c, p.x.terms, 2 * c.blocks, p.nblocks, epi, s);
        return;
    }
    const Planes wg = weight_planes(gate, 0, gate.rows, p.x.terms, p.room[0], s),
                 wu = weight_planes(up, 0, up.rows, p.x.terms, p.room[1], s);
    with_terms(p.x.terms, [&](auto terms) {
        launch_rows_gemm<false, false, decltype(terms)::value>(p.tile, glu_gemm(p, in, wg, wu), 2 * wg.groups, p.nblocks, epi, s);
    });
}

template <int TB, int T>
static void fill_glu(const GluPlan &p, const RowsIn &in, const Planes &wg, const Planes &wu, const TileView &gate,
                     const TileView &up, int32_t dtype, RowsArg dout, int64_t n, uint32_t act, hipStream_t s) {
    const EpiGluGrad<T> epi{p.dg, p.du, dout.p, dout.stride, n, gate.rows, dtype, act};
    if (p.coded) launch_glu_grad_coded<T>(p.coded, glu_coded(in, gate, up), TB, 4 * p.dg.units, p.nblocks, epi, s);
    else launch_rows_gemm<false, false, TB>(p.tile, glu_gemm(p, in, wg, wu), 4 * p.dg.units, p.nblocks, epi, s);
}

void launch_glu_rows_grad(int32_t dtype, RowsArg dx, RowsArg dgate, RowsArg dup, RowsArg dout, RowsArg x, int64_t n,
                          const TileView &gate, const TileView &up, uint32_t act, void *ws, hipStream_t s) {
    const GluPlan p = glu_plan(gate, up, n, dtype, true, ws);
    const RowsIn in = rows_in(dtype, n, gate.cols, x, nullptr, &p.x, s);
    if ((dgate.p || dup.p) && in.x.p != p.x.p) launch_pack_rows(p.x, x.p, dtype, n, gate.cols, x.stride, s);  // (read transposed)
    Planes wg, wu;
    if (!p.coded) {
        wg = weight_planes(gate, 0, gate.rows, p.x.terms, p.room[0], s);
        wu = weight_planes(up, 0, up.rows, p.x.terms, p.room[1], s);
    }
    auto fill = p.x.terms == 3 ? fill_glu<3, 3> : p.x.terms == 2 ? fill_glu<2, 2> : p.dg.terms == 2 ? fill_glu<1, 2> : fill_glu<1, 1>;
    fill(p, in, wg, wu, gate, up, dtype, dout, n, act, s);
    if (dx.p) {
        if (p.coded) {
            CodedParts g;
            g.w[0] = gate;
            g.w[1] = up;
            g.d[0] = p.dg.p;
            g.d[1] = p.du.p;
            g.d_groups = (int32_t)p.dg.groups;
            g.d_units = p.dg.units;
            g.d_plane = p.dg.plane_bytes();
            g.blocks = (int32_t)ceil_div(gate.rows, 16);
            g.steps = (int32_t)ceil_div(gate.rows, 32);
            g.sets = 2;
            g.parts = p.back.parts;
            launch_coded_parts(g, p.dg.terms, p.part, p.ld, n, false, s);
        } else {
            RowsGemm g;
            g.a = rows_outer(wg);
            g.b = rows_inner(p.dg);
            g.k32 = (int32_t)p.dg.units;
            g.parts = p.back.parts;
            rows_pairs(g, wg, p.dg, p.back_order);
            rows_pairs(g, wu, p.du, p.back_order);
            launch_rows_parts(p.back.tile, g, p.part, p.ld, n, gate.cols, false, s);
        }
        launch_join_parts(dx.p, dtype, dx.stride, p.part, p.back.parts, n * p.ld, p.ld, n, gate.cols, s);
    }
    if (!dgate.p && !dup.p) return;
    const Planes &d = dgate.p ? p.dg : p.du;
    RowsGemm g;
    g.a = rows_outer(p.x);
    g.b = rows_outer(d);
    if (dgate.p && dup.p) {
        g.b.paired = 1;
        g.b.pair = p.du.p - p.dg.p;
    }
    g.k32 = (int32_t)(p.nblocks / 2);
    rows_pairs(g, p.x, d, d.terms);
    launch_rows_out(g, dgate.p ? dgate : dup, dgate.p ? dup : RowsArg{}, dtype, gate.rows, gate.cols, s);
}

}  // namespace ditch
