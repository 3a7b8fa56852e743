// head_grad.hip — the gradients of the head's losses (head.hip has the
// formulas). The logits are formed again, a piece of the vocabulary at a time;
// the epilogue leaves d = dloss/dlogits of the piece as bf16 terms, [row][word],
// and two products over them give the piece's share of dx = d W and its rows of
// dW = d^T x.
//
// The divergence's d = g (q - p) is made with log sums that its caller holds in f32, so
// that c = lse_trial - lse_base is off by up to 2^-20 (log sums of 8 to 16), and dx by
// that times sum q w, along the head's mean direction. For 70 f32 rows over 128256 x
// 512, the mean as strong as the words' own parts, that was 1.4e-5, 4e-4 and 6e-3 of
// the gradient at divergences of 0.16, 2e-4 and 6e-7. But sum q = sum p, so what the d
// of all words sum to is that error, epsilon, and dx - epsilon g sum p w is without
// it (3e-7, 1e-6 and 1.6e-5): one more product, of p as one term, whose own rounding
// weighs epsilon 2^-9. 64 f32 rows over 128256 x 4096 take 820 us instead of 620, 1000
// 8.3 ms instead of 7.3. (c in 64 bits would take the logits twice, two products.)
// bf16 rows do without: it shows below divergences of 1e-5 only (2.3e-3 instead of
// 1.7e-3 of the gradient at 5e-6), and is a fifth of their time.
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
    // what mends the divergence's log sums
    Planes p;
    RowsTiling p_tiling;
    float *p_part = nullptr, *sums = nullptr, *times = nullptr;
    int64_t npad = 0, strips = 0;
    size_t bytes = 0;
};
constexpr int P_ORDER = 2;  // of the product with p: the weight in 16 bits
static int64_t grad_strips(const HeadGradPlan &p, const TileView &w, int64_t rows) {
    return strips_of(ceil_div(rows, 64) * 64, p.coded ? p.coded : logits_tile(w, rows, p.x[0], 2 * p.nblocks, true));
}
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
    if (kl && dtype != DITCH_BF16) {
        p.p = Planes{nullptr, p.nblocks, p.piece / 32, 1};
        p.p.p = c.take(p.p.bytes());
        if (p.coded) p.p_tiling.parts = coded_parts_count(w, p.piece, n, 1);
        else p.p_tiling = rows_tiling(ceil_div(w.cols, 16), p.nblocks, p.piece / 32, wt, 1, P_ORDER, 1, true, false);
        p.p_part = c.take<float>((size_t)p.p_tiling.parts * n * p.ld);
        p.npad = n < 32 ? n : ceil_div(n, 32) * 32;
        for (int64_t r = 0; r < w.rows; r += p.piece) p.strips += grad_strips(p, w, w.rows - r < p.piece ? w.rows - r : p.piece);
        p.sums = c.take<float>((size_t)p.strips * p.npad);
        p.times = c.take<float>(n);
    }
    p.bytes = c.at;
    return p;
}

size_t head_loss_grad_workspace(const TileView &w, int64_t n, int32_t dtype, bool dw) {
    return head_grad_plan(w, n, dtype, false, nullptr).bytes;
}
size_t head_kl_grad_workspace(const TileView &w, int64_t n, int32_t dtype) {
    return head_grad_plan(w, n, dtype, true, nullptr).bytes;
}

// A piece's share of d W, to the parts `part`.
static void add_parts(const HeadGradPlan &p, const Planes &d, const Planes &wp, const RowsTiling &tiling, int order, float *part,
                      int64_t r, int64_t rows, int64_t n, const TileView &w, hipStream_t s) {
    if (p.coded) {
        CodedParts g;
        g.w[0] = w;
        g.d[0] = d.p;
        g.d_groups = (int32_t)d.groups;
        g.d_units = d.units;
        g.d_plane = d.plane_bytes();
        g.first = (int32_t)(r / 16);
        g.blocks = (int32_t)ceil_div(rows, 16);
        g.steps = (int32_t)ceil_div(rows, 32);
        g.parts = tiling.parts;
        launch_coded_parts(g, d.terms, part, p.ld, n, r > 0, s);
    } else {
        RowsGemm g;
        g.a = rows_outer(wp);
        g.b = rows_inner(d);
        g.k32 = (int32_t)d.units;
        g.parts = tiling.parts;
        rows_pairs(g, wp, d, order);
        launch_rows_parts(tiling.tile, g, part, p.ld, n, w.cols, r > 0, s);
    }
}

// `fill` launches the product that leaves a piece's d (and p); `mended` what makes p.times of all pieces' sums.
template <typename Fill, typename Mended>
static void head_grad(const HeadGradPlan &p, int32_t dtype, RowsArg dx, RowsArg dw, int64_t n, const TileView &w,
                      hipStream_t s, Fill &&fill, Mended &&mended) {
    for (int64_t r = 0; r < w.rows; r += p.piece) {
        const int64_t rows = w.rows - r < p.piece ? w.rows - r : p.piece;
        const Planes wp = p.coded ? Planes{} : weight_planes(w, r, rows, p.w_terms, p.room, s);
        Planes d = p.d, q = p.p;
        d.units = q.units = ceil_div(rows, 64) * 2;
        fill(wp, d, q, r, rows);
        if (dx.p) add_parts(p, d, wp, p.tiling, p.order, p.part, r, rows, n, w, s);
        if (q.p) add_parts(p, q, wp, p.p_tiling, P_ORDER, p.p_part, r, rows, n, w, s);
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
    if (!dx.p) return;
    MoreParts more;
    if (p.p.p) {
        mended();
        more = MoreParts{p.p_part, p.times, p.p_tiling.parts};
    }
    launch_join_parts(dx.p, dtype, dx.stride, p.part, p.tiling.parts, n * p.ld, p.ld, n, w.cols, s, more);
}

// times[i] = -g epsilon, of the strips' sums of q - p. (Only what rounding leaves of
// log sums is mended: of others the gradient is what the formula says.)
template <int TOK>
__global__ __launch_bounds__(512) void kl_times_kernel(float *times, const float *sums, const float *lse_base,
                                                       const float *lse_trial, const float *dkl, int64_t n, int64_t npad,
                                                       int64_t strips) {
    constexpr int SL = 512 / TOK;
    __shared__ double dl[8 * TOK];
    const int c = threadIdx.x % TOK, sl = threadIdx.x / TOK;
    const int64_t tok = (int64_t)blockIdx.x * TOK + c;
    double sum = 0;
    if (tok < n)
#pragma unroll 4
        for (int64_t k = sl; k < strips; k += SL) sum += (double)sums[k * npad + tok];
    sum = block_sum<TOK>(sum, dl);
    if (sl != 0 || tok >= n) return;
    const double most = 0x1p-20 * (4 + fabs((double)lse_base[tok]) + fabs((double)lse_trial[tok]));
    times[tok] = fabs(sum) <= most ? (float)(-(double)dkl[tok] * sum / (1 + sum)) : 0.f;
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
    launch_rows_gemm<false, false, TB>(logits_tile(w, rows, p.x[0], p.nblocks, false), logits_gemm(wp, in),
                                      d.units * 2, p.nblocks, epi, s);
}
template <int TB, int T>
static void fill_kl(const HeadGradPlan &p, const RowsIn &in, const TileView &w, const Planes &wp, const Planes &d, const Planes &q,
                    int64_t strip0, int64_t row0, int64_t rows, int64_t n, const float *lse_base, const float *lse_trial,
                    const float *dkl, hipStream_t s) {
    const EpiKlGrad<T> epi{d, q, p.sums, lse_base, lse_trial, dkl, n, rows, p.npad, strip0};
    if (p.coded) {
        RowsCoded c = coded_product(w, in);
        c.first = (int32_t)(row0 / 16);
        c.blocks = (int32_t)ceil_div(rows, 16);
        launch_kl_grad_coded<T>(p.coded, c, TB, d.units * 2, 2 * p.nblocks, epi, s);
        return;
    }
    launch_rows_gemm<false, false, TB>(logits_tile(w, rows, p.x[0], 2 * p.nblocks, true), logits_gemm(wp, in),
                                      d.units * 2, 2 * p.nblocks, epi, s);
}

void launch_head_loss_grad(int32_t dtype, RowsArg dx, RowsArg dw, RowsArg x, int64_t n, const TileView &w,
                           const int32_t *targets, const float *lse, const float *dloss, void *ws, hipStream_t s) {
    const HeadGradPlan p = head_grad_plan(w, n, dtype, false, ws);
    // (rows without a target are zeros in d^T x, where an infinity or NaN times their zero d would stay)
    const RowsIn in = rows_in(dtype, n, w.cols, x, nullptr, p.x, s, targets);
    if (dw.p && in.x.p != p.x[0].p) launch_pack_rows(p.x[0], x.p, dtype, n, w.cols, x.stride, s, targets);  // (read transposed)
    head_grad(p, dtype, dx, dw, n, w, s, [&](const Planes &wp, const Planes &d, const Planes &, int64_t row0, int64_t rows) {
        auto f = p.x[0].terms == 3 ? fill_loss<3, 3> : p.x[0].terms == 2 ? fill_loss<2, 2> : p.d.terms == 2 ? fill_loss<1, 2> : fill_loss<1, 1>;
        f(p, in, w, wp, d, row0, rows, n, targets, lse, dloss, s);
    }, [] {});
}

void launch_head_kl_grad(int32_t dtype, RowsArg dx, RowsArg base, RowsArg trial, int64_t n, const TileView &w,
                         const float *lse_base, const float *lse_trial, const float *dkl, void *ws, hipStream_t s) {
    const HeadGradPlan p = head_grad_plan(w, n, dtype, true, ws);
    const RowsIn in = rows_in(dtype, n, w.cols, base, &trial, p.x, s);
    int64_t strip = 0;
    head_grad(p, dtype, dx, RowsArg{}, n, w, s, [&](const Planes &wp, const Planes &d, const Planes &q, int64_t row0, int64_t rows) {
        auto f = p.x[0].terms == 3 ? fill_kl<3, 3> : p.x[0].terms == 2 ? fill_kl<2, 2> : p.d.terms == 2 ? fill_kl<1, 2> : fill_kl<1, 1>;
        f(p, in, w, wp, d, q, strip, row0, rows, n, lse_base, lse_trial, dkl, s);
        strip += grad_strips(p, w, rows);
    }, [&] {
        with_join_rows(n, [&](auto rows) {
            constexpr int TOK = decltype(rows)::value;
            hipLaunchKernelGGL(kl_times_kernel<TOK>, dim3((unsigned)ceil_div(n, TOK)), dim3(512), 0, s, p.times, p.sums,
                               lse_base, lse_trial, dkl, n, p.npad, p.strips);
        });
        DITCH_TRY_HIP(hipGetLastError());
    });
}

}  // namespace ditch
