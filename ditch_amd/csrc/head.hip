// head.hip — losses of rows against the head, and their gradients, without the
// logits: x W^T is formed in tiles whose epilogues keep what the result needs.
//
// Cross entropy: loss = lse - l_t with lse = log sum_v e^(l_v). Each wave's strip
// of the vocabulary leaves, for a row, its maximum m and sum of e^(l - m), and
// whichever holds the target its logit; a second kernel joins the strips in
// 64 bits. Gradient: d_v = g (e^(l_v - lse) - [v = t]), dx = d W, dW = d^T x; the
// logits are formed again, piece after piece of the vocabulary, and d is held
// for one piece only, as bf16 terms.
//
// Divergence of trial rows from base rows, KL = sum p (log p - log q): the two
// rows' blocks are interleaved in one product, so that a lane holds both logits
// of a word. With D = l_base - l_trial, c = lse_trial - lse_base and phi(u) = u +
// e^-u - 1 >= 0,
//   KL = sum p phi(D + c),
// term by term at least 0 (sum p D + c would lose what a small divergence is made
// of). c is known when all words have been seen: a strip sums phi(D - a) of a
// shift of its own, and the join moves it by delta = -c - a,
//   sum p phi(u - delta) = sum p (e^delta phi(u) - (e^delta - 1) u + e^delta - 1 - delta),
// in 64 bits. (sum p phi(D) - phi(-c), without shifts, lost divergences to rows whose logits
// moved alike: by 4, a divergence of 3e-5 was off by 2e-4 of itself, one of 5e-7 by 1e-2.)
// d = g (q - p).
#include "head.h"

namespace ditch {

// ---------------------------------------------------------------------------
// cross entropy

// Few rows a block where there are few, so that their strips are read side by
// side (1 row x 2376 strips by 8 threads took 220 us).
template <int TOK>
__global__ __launch_bounds__(512) void loss_join_kernel(float *loss, float *lse, const float2 *part,
                                                        const float *picked, const int32_t *targets, int64_t n,
                                                        int64_t npad, int64_t strips, int64_t vocab) {
    constexpr int SL = 512 / TOK;
    __shared__ float fl[8 * TOK];
    __shared__ double dl[8 * TOK];
    const int c = threadIdx.x % TOK, sl = threadIdx.x / TOK;
    const int64_t tok = (int64_t)blockIdx.x * TOK + c;
    float m = LOWEST, pick = 0.f;
    double sum = 0;
    int32_t t = -1;
    if (tok < n) {
        t = targets[tok];
        pick = picked[tok];  // (read ahead: whatever is there for rows without a target)
#pragma unroll 4
        for (int64_t k = sl; k < strips; k += SL) {
            const float2 v = part[k * npad + tok];
            const float to = fmaxf(m, v.x);
            sum = sum * (double)expf(m - to) + (double)v.y * (double)expf(v.x - to);
            m = to;
        }
    }
    const float top = block_max<TOK>(m, fl);
    sum = block_sum<TOK>(sum * exp((double)m - (double)top), dl);
    if (sl != 0 || tok >= n) return;
    const double l = (double)top + log(sum);
    lse[tok] = (float)l;
    loss[tok] = t < 0 ? 0.f : t >= vocab ? __builtin_nanf("") : (float)(l - (double)pick);
}

// ---------------------------------------------------------------------------
// divergence

template <int TOK>
__global__ __launch_bounds__(512) void kl_join_kernel(float *kl, float *lse_base, float *lse_trial, const float *part,
                                                      int64_t n, int64_t npad, int64_t strips) {
    constexpr int SL = 512 / TOK;
    __shared__ float fl[8 * TOK];
    __shared__ double dl[8 * TOK];
    const int c = threadIdx.x % TOK, sl = threadIdx.x / TOK;
    const int64_t tok = (int64_t)blockIdx.x * TOK + c;
    float m[2] = {LOWEST, LOWEST};
    double s[2] = {0, 0};
    if (tok < n) {
#pragma unroll 2
        for (int64_t k = sl; k < strips; k += SL) {
            const float2 *p = (const float2 *)(part + (k * npad + tok) * KL_STATS);
            const float2 v[2] = {p[0], p[1]};
            for (int h = 0; h < 2; h++) {
                const float to = fmaxf(m[h], v[h].x);
                s[h] = s[h] * (double)expf(m[h] - to) + (double)v[h].y * (double)expf(v[h].x - to);
                m[h] = to;
            }
        }
    }
    double lse[2];
    for (int h = 0; h < 2; h++) {
        const float top = block_max<TOK>(m[h], fl);
        lse[h] = (double)top + log(block_sum<TOK>(s[h] * exp((double)m[h] - (double)top), dl));
    }
    const double shift = lse[0] - lse[1];
    double sum = 0;
    if (tok < n) {
#pragma unroll 2
        for (int64_t k = sl; k < strips; k += SL) {
            const float2 *v = (const float2 *)(part + (k * npad + tok) * KL_STATS);
            const float2 base = v[0], trial = v[1], sums = v[2];
            const double delta = shift - (double)(base.x - trial.x);
            // what the strip's sums weigh in p, and that times e^delta: neither overflows
            const double p = exp((double)base.x - lse[0]);
            const double more = fabs(delta) < 1 ? p * expm1(delta) : exp((double)trial.x - lse[1]) - p;
            sum += (p + more) * sums.x - more * sums.y + (more - p * delta) * base.y;
        }
    }
    sum = block_sum<TOK>(sum, dl);
    if (sl != 0 || tok >= n) return;
    lse_base[tok] = (float)lse[0];
    lse_trial[tok] = (float)lse[1];
    kl[tok] = (float)sum;
}

// ---------------------------------------------------------------------------
// pieces of the vocabulary

// The forward of either loss: stats(g, piece's epilogue arguments).
struct HeadPlan {
    Planes x[2];
    int64_t piece = 0, strips = 0, npad = 0, nblocks = 0;
    int tile = 0, coded = 0;  // coded: the tile of rows_coded.h's product, 0: planes
    char *room = nullptr;
    char *part = nullptr;
    float *picked = nullptr;
    size_t bytes = 0;
};
static HeadPlan head_plan(const TileView &w, int64_t n, int32_t dtype, bool kl, void *ws) {
    HeadPlan p;
    Carver c(ws);
    for (int i = 0; i < (kl ? 2 : 1); i++) {
        p.x[i] = row_planes(n, w.cols, row_terms(dtype));
        p.x[i].p = c.take(p.x[i].bytes());
    }
    p.npad = n < 32 ? n : ceil_div(n, 32) * 32;  // (one row's strips follow each other)
    p.nblocks = row_blocks(n) * (kl ? 2 : 1);
    p.coded = rows_coded_tile(w, ceil_div(w.rows, 16), p.nblocks, false);
    const int64_t per = p.coded ? 0 : weight_row_bytes(w, ROWS_MAX_TERMS);
    p.piece = per ? piece_rows(w.rows, per) : w.rows;
    p.tile = p.coded ? p.coded : logits_tile(w, p.piece < w.rows ? p.piece : w.rows, p.x[0], p.nblocks, true);
    for (int64_t r = 0; r < w.rows; r += p.piece)
        p.strips += strips_of(w.rows - r < p.piece ? w.rows - r : p.piece, p.tile);
    p.part = c.take((size_t)p.strips * p.npad * (kl ? KL_STATS * sizeof(float) : sizeof(float2)));
    p.picked = c.take<float>(n);
    if (per) p.room = c.take(weight_planes_shape(w, p.piece, ROWS_MAX_TERMS).bytes());
    p.bytes = c.at;
    return p;
}

size_t head_loss_workspace(const TileView &w, int64_t n, int32_t dtype) {
    return head_plan(w, n, dtype, false, nullptr).bytes;
}
size_t head_kl_workspace(const TileView &w, int64_t n, int32_t dtype) {
    return head_plan(w, n, dtype, true, nullptr).bytes;
}

void launch_head_loss(float *loss, float *lse, int32_t dtype, RowsArg x, int64_t n, const TileView &w,
                      const int32_t *targets, void *ws, hipStream_t s) {
    const HeadPlan p = head_plan(w, n, dtype, false, ws);
    const RowsIn in = rows_in(dtype, n, w.cols, x, nullptr, p.x, s);
    int64_t strip = 0;
    for (int64_t r = 0; r < w.rows; r += p.piece) {
        const int64_t rows = w.rows - r < p.piece ? w.rows - r : p.piece;
        const EpiLossStats epi{(float2 *)p.part, p.picked, targets, p.npad, n, rows, r, strip};
        if (p.coded) {
            launch_loss_coded(p.tile, coded_product(w, in), p.x[0].terms, ceil_div(w.rows, 16), p.nblocks, epi, s);
            break;
        }
        const Planes wp = weight_planes(w, r, rows, ROWS_MAX_TERMS, p.room, s);
        with_terms(p.x[0].terms, [&](auto terms) {
            launch_rows_gemm<false, false, decltype(terms)::value>(p.tile, logits_gemm(wp, in), wp.groups,
                                                                   p.nblocks, epi, s);
        });
        strip += strips_of(rows, p.tile);
    }
    with_join_rows(n, [&](auto rows) {
        constexpr int TOK = decltype(rows)::value;
        hipLaunchKernelGGL(loss_join_kernel<TOK>, dim3((unsigned)ceil_div(n, TOK)), dim3(512), 0, s, loss, lse,
                           (const float2 *)p.part, p.picked, targets, n, p.npad, p.strips, w.rows);
    });
    DITCH_TRY_HIP(hipGetLastError());
}

void launch_head_kl(float *kl, float *lse_base, float *lse_trial, int32_t dtype, RowsArg base, RowsArg trial,
                    int64_t n, const TileView &w, void *ws, hipStream_t s) {
    const HeadPlan p = head_plan(w, n, dtype, true, ws);
    const RowsIn in = rows_in(dtype, n, w.cols, base, &trial, p.x, s);
    int64_t strip = 0;
    for (int64_t r = 0; r < w.rows; r += p.piece) {
        const int64_t rows = w.rows - r < p.piece ? w.rows - r : p.piece;
        const EpiKlStats epi{(float *)p.part, p.npad, n, rows, strip};
        if (p.coded) {
            launch_kl_coded(p.tile, coded_product(w, in), p.x[0].terms, ceil_div(w.rows, 16), p.nblocks, epi, s);
            break;
        }
        const Planes wp = weight_planes(w, r, rows, ROWS_MAX_TERMS, p.room, s);
        with_terms(p.x[0].terms, [&](auto terms) {
            launch_rows_gemm<false, false, decltype(terms)::value>(p.tile, logits_gemm(wp, in), wp.groups,
                                                                   p.nblocks, epi, s);
        });
        strip += strips_of(rows, p.tile);
    }
    with_join_rows(n, [&](auto rows) {
        constexpr int TOK = decltype(rows)::value;
        hipLaunchKernelGGL(kl_join_kernel<TOK>, dim3((unsigned)ceil_div(n, TOK)), dim3(512), 0, s, kl, lse_base,
                           lse_trial, (const float *)p.part, n, p.npad, p.strips);
    });
    DITCH_TRY_HIP(hipGetLastError());
}

}  // namespace ditch
