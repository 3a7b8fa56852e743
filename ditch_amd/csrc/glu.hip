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

template <int T>
struct EpiGluGrad {
    Planes dg, du;
    const void *dout;
    int64_t stride, n, rows;
    int32_t dtype;
    uint32_t act;
    __device__ __forceinline__ float dout_at(int64_t i) const {
        if (dtype == DITCH_F32) return ((const float *)dout)[i];
        const uint16_t b = ((const uint16_t *)dout)[i];
        return dtype == DITCH_F16 ? f16_to_f32_hw(b) : bf16_to_f32(b);
    }
    template <int A, int MI, int NJ>
    __device__ __forceinline__ void store(floatx4 (&acc)[MI][NJ], int mb, int nb, int lane) const {
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            if (nb + j >= dg.groups) continue;
            const int64_t tok = (int64_t)(nb + j) * 16 + (lane & 15);
#pragma unroll
            for (int i = 0; i < MI; i += 2) {
                const int wb = (mb + i) / 2;
                if ((wb >> 1) >= dg.units) continue;
                const int64_t c = (int64_t)wb * 16 + 4 * (lane >> 4);
                float a[4], b[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float y, dy;
                    act_both<A>(acc[i][j][r], y, dy);
                    const bool in = tok < n && c + r < rows;
                    const float d = in ? dout_at(tok * stride + c + r) : 0.f;
                    a[r] = in ? d * acc[i + 1][j][r] * dy : 0.f;
                    b[r] = in ? d * y : 0.f;
                }
                put_grad_terms<T>(dg, wb, nb + j, lane, a);
                put_grad_terms<T>(du, wb, nb + j, lane, b);
            }
        }
    }
    template <int MI, int NJ>
    __device__ __forceinline__ void operator()(floatx4 (&acc)[MI][NJ], int mb, int nb, int lane) const {
        switch (act) {
        case 0: store<0>(acc, mb, nb, lane); break;
        case 1: store<1>(acc, mb, nb, lane); break;
        case 2: store<2>(acc, mb, nb, lane); break;
        case 3: store<3>(acc, mb, nb, lane); break;
        case 4: store<4>(acc, mb, nb, lane); break;
        default: store<5>(acc, mb, nb, lane); break;
        }
    }
};

// x and both matrices as planes, one operand after the other.
struct GluPlan {
    Planes x, dg, du;
    char *room[2] = {nullptr, nullptr};
    int64_t ld = 0;
    int order = 1, tile = 0, coded = 0;  // coded: the tile of rows_coded.h's product, 0: planes
    RowsTiling back;
    int back_order = 1;  // of the product with d
    float *part = nullptr;
    size_t bytes = 0;
};
static GluPlan glu_plan(const TileView &w, const TileView &up, int64_t n, int32_t dtype, bool grad, void *ws) {
    GluPlan p;
    Carver c(ws);
    const int terms = row_terms(dtype), wt = rows_weight_terms(w, terms);
    p.order = rows_order_of(wt, terms);
    p.x = row_planes(n, w.cols, terms);
    p.x.p = c.take(p.x.bytes());
    p.coded = grad || !rows_coded_pair(w, up) ? 0 : rows_coded_tile(w, 2 * ceil_div(w.rows, 16), p.x.groups, terms);
    if (!weight_is_planes(w) && !p.coded)
        for (int i = 0; i < 2; i++) p.room[i] = c.take(weight_planes_shape(w, w.rows, terms).bytes());
    if (grad) {
        const int td = grad_term_count(terms, n);
        p.back_order = rows_order_of(wt, td);
        for (Planes *d : {&p.dg, &p.du}) {
            *d = Planes{nullptr, p.x.groups, ceil_div(w.rows, 64) * 2, td};
            d->p = c.take(d->bytes());
        }
        p.ld = ceil_div(w.cols, 4) * 4;
        p.back = rows_tiling(ceil_div(w.cols, 16), p.x.groups, p.dg.units, wt, td, p.back_order, 2, true, false);
        p.part = c.take<float>((size_t)p.back.parts * n * p.ld);
    }
    p.tile = rows_tiling(2 * ceil_div(w.rows, 16), p.x.groups, ceil_div(w.cols, 64) * 2, wt, terms, p.order, 1, false, true).tile;
    p.bytes = c.at;
    return p;
}

size_t glu_rows_workspace(const TileView &gate, const TileView &up, int64_t n, int32_t dtype) {
    return glu_plan(gate, up, n, dtype, false, nullptr).bytes;
}
size_t glu_rows_grad_workspace(const TileView &gate, const TileView &up, int64_t n, int32_t dtype, bool dw) {
    return glu_plan(gate, up, n, dtype, true, nullptr).bytes;
}

static RowsGemm glu_gemm(const GluPlan &p, const Planes &wg, const Planes &wu) {
    RowsGemm g;
    g.a = rows_inner(wg);
    g.a.paired = 1;
    g.a.pair = wu.p - wg.p;
    g.b = rows_inner(p.x);
    g.k32 = (int32_t)ceil_div(wg.units, 2) * 2;
    rows_pairs(g, wg, p.x, p.order);
    return g;
}

void launch_glu_rows(int32_t dtype, RowsArg out, RowsArg x, int64_t n, const TileView &gate, const TileView &up,
                     uint32_t act, void *ws, hipStream_t s) {
    const GluPlan p = glu_plan(gate, up, n, dtype, false, ws);
    launch_pack_rows(p.x, x.p, dtype, n, gate.cols, x.stride, s);
    const EpiGlu epi{out.p, out.stride, n, gate.rows, dtype, rows_wide(out.p, out.stride, dtype), act};
    if (p.coded) {
        RowsCoded c;
        c.w[0] = gate;
        c.w[1] = up;
        c.paired = 1;
        c.b = rows_inner(p.x);
        c.x = p.x.p;
        c.x_plane = p.x.plane_bytes();
        c.blocks = (int32_t)ceil_div(gate.rows, 16);
        c.stages = (int32_t)gate.units_k;
        launch_glu_coded(p.coded, c, p.x.terms, 2 * c.blocks, p.x.groups, epi, s);
        return;
    }
    const Planes wg = weight_planes(gate, 0, gate.rows, p.x.terms, p.room[0], s),
                 wu = weight_planes(up, 0, up.rows, p.x.terms, p.room[1], s);
    with_terms(p.x.terms, [&](auto terms) {
        launch_rows_gemm<false, false, decltype(terms)::value>(p.tile, glu_gemm(p, wg, wu), 2 * wg.groups, p.x.groups, epi, s);
    });
}

template <int TB, int T>
static void fill_glu(const GluPlan &p, const RowsGemm &g, int32_t dtype, RowsArg dout, int64_t n, int64_t rows,
                     uint32_t act, hipStream_t s) {
    const EpiGluGrad<T> epi{p.dg, p.du, dout.p, dout.stride, n, rows, dtype, act};
    launch_rows_gemm<false, false, TB>(p.tile, g, 4 * p.dg.units, p.x.groups, epi, s);
}

void launch_glu_rows_grad(int32_t dtype, RowsArg dx, RowsArg dgate, RowsArg dup, RowsArg dout, RowsArg x, int64_t n,
                          const TileView &gate, const TileView &up, uint32_t act, void *ws, hipStream_t s) {
    const GluPlan p = glu_plan(gate, up, n, dtype, true, ws);
    launch_pack_rows(p.x, x.p, dtype, n, gate.cols, x.stride, s);
    const Planes wg = weight_planes(gate, 0, gate.rows, p.x.terms, p.room[0], s),
                 wu = weight_planes(up, 0, up.rows, p.x.terms, p.room[1], s);
    auto fill = p.x.terms == 3 ? fill_glu<3, 3> : p.x.terms == 2 ? fill_glu<2, 2> : p.dg.terms == 2 ? fill_glu<1, 2> : fill_glu<1, 1>;
    fill(p, glu_gemm(p, wg, wu), dtype, dout, n, gate.rows, act, s);
    if (dx.p) {
        RowsGemm g;
        g.a = rows_outer(wg);
        g.b = rows_inner(p.dg);
        g.k32 = (int32_t)p.dg.units;
        g.parts = p.back.parts;
        rows_pairs(g, wg, p.dg, p.back_order);
        rows_pairs(g, wu, p.du, p.back_order);
        launch_rows_parts(p.back.tile, g, p.part, p.ld, n, gate.cols, false, s);
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
    g.k32 = (int32_t)(p.x.groups / 2);
    rows_pairs(g, p.x, d, d.terms);
    launch_rows_out(g, dgate.p ? dgate : dup, dgate.p ? dup : RowsArg{}, dtype, gate.rows, gate.cols, s);
}

}  // namespace ditch
