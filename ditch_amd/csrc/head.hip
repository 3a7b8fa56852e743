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
// of a word. With D = l_base - l_trial and phi(u) = u + e^-u - 1 >= 0,
//   KL = sum p phi(D) - (e^c - 1 - c),  c = lse_trial - lse_base,
// where nothing cancels for rows near each other (sum p D + c would lose what a
// small divergence is made of); for far ones, |c| > 1, sum p D + c is used.
// d = g (q - p).
#include "rows_gemm.h"

namespace ditch {

__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(__fmul_rn(x, 1.4426950408889634f)); }

constexpr float LOWEST = -3.0e38f;  // in place of words that are not there

// ---------------------------------------------------------------------------
// cross entropy

struct EpiLossStats {
    float2 *part;  // [strip][npad]: maximum, sum
    float *picked;  // [n]
    const int32_t *targets;
    int64_t npad, n;
    int64_t rows, row0, strip0;  // rows of this piece, its first word, its first strip
    template <int MI, int NJ>
    __device__ __forceinline__ void operator()(floatx4 (&acc)[MI][NJ], int mb, int nb, int lane) const {
        const int64_t strip = strip0 + mb / MI;
        const int64_t v0 = (int64_t)mb * 16 + 4 * (lane >> 4);
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int64_t tok = (int64_t)(nb + j) * 16 + (lane & 15);
            float m = LOWEST;
#pragma unroll
            for (int i = 0; i < MI; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if (v0 + i * 16 + r >= rows) acc[i][j][r] = -__builtin_inff();
                    m = fmaxf(m, acc[i][j][r]);
                }
            m = fmaxf(m, __shfl_xor(m, 16));
            m = fmaxf(m, __shfl_xor(m, 32));
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < MI; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) sum += fast_exp(acc[i][j][r] - m);
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (tok >= n) continue;
            if (lane < 16) part[strip * npad + tok] = make_float2(m, sum);
            const int64_t t = (int64_t)targets[tok] - row0 - v0;  // in this lane's words?
#pragma unroll
            for (int i = 0; i < MI; i++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (t == i * 16 + r && v0 + t < rows) picked[tok] = acc[i][j][r];
        }
    }
};

// A block 32 rows, 8 slices of the strips each.
__global__ __launch_bounds__(256) void loss_join_kernel(float *loss, float *lse, const float2 *part,
                                                        const float *picked, const int32_t *targets, int64_t n,
                                                        int64_t npad, int64_t strips, int64_t vocab) {
    __shared__ float mx[8][32];
    __shared__ double sx[8][32];
    const int c = threadIdx.x & 31, sl = threadIdx.x >> 5;
    const int64_t tok = (int64_t)blockIdx.x * 32 + c;
    float m = LOWEST;
    double sum = 0;
    if (tok < n) {
        for (int64_t k = sl; k < strips; k += 8) m = fmaxf(m, part[k * npad + tok].x);
        for (int64_t k = sl; k < strips; k += 8) {
            const float2 v = part[k * npad + tok];
            sum += (double)v.y * (double)expf(v.x - m);
        }
    }
    mx[sl][c] = m;
    sx[sl][c] = sum;
    __syncthreads();
    if (sl != 0 || tok >= n) return;
    for (int k = 1; k < 8; k++) m = fmaxf(m, mx[k][c]);
    sum = 0;
    for (int k = 0; k < 8; k++) sum += sx[k][c] * exp((double)mx[k][c] - (double)m);
    const double l = (double)m + log(sum);
    lse[tok] = (float)l;
    const int32_t t = targets[tok];
    loss[tok] = t < 0 ? 0.f : t >= vocab ? __builtin_nanf("") : (float)(l - (double)picked[tok]);
}

// d of a piece as terms. Rows without a target give zeros, targets past the
// vocabulary NaN.
template <int T>
struct EpiLossGrad {
    Planes d;
    const int32_t *targets;
    const float *lse, *dloss;
    int64_t n, rows, row0, vocab;
    template <int MI, int NJ>
    __device__ __forceinline__ void operator()(floatx4 (&acc)[MI][NJ], int mb, int nb, int lane) const {
        const int64_t v0 = (int64_t)mb * 16 + 4 * (lane >> 4);
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            if (nb + j >= d.groups) continue;
            const int64_t tok = (int64_t)(nb + j) * 16 + (lane & 15);
            float g = 0.f, l = 0.f;
            int64_t t = -1;
            bool live = false;
            if (tok < n) {
                const int32_t tt = targets[tok];
                live = tt >= 0;
                l = lse[tok];
                g = tt >= vocab ? __builtin_nanf("") : dloss[tok];
                t = (int64_t)tt - row0 - v0;
            }
#pragma unroll
            for (int i = 0; i < MI; i++) {
                if (((mb + i) >> 1) >= d.units) continue;
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float p = fast_exp(acc[i][j][r] - l) - (t == i * 16 + r ? 1.f : 0.f);
                    v[r] = live && v0 + i * 16 + r < rows ? __fmul_rn(g, p) : 0.f;
                }
                put_grad_terms<T>(d, mb + i, nb + j, lane, v);
            }
        }
    }
};

// ---------------------------------------------------------------------------
// divergence

// phi(u) = u + e^-u - 1 for |u| <= 1: its series to u^12 / 12!, 2^-30 of it
__device__ __forceinline__ float phi_near(float u) {
    float s = 1.f / 479001600.f;
    s = __builtin_fmaf(s, -u, 1.f / 39916800.f);
    s = __builtin_fmaf(s, -u, 1.f / 3628800.f);
    s = __builtin_fmaf(s, -u, 1.f / 362880.f);
    s = __builtin_fmaf(s, -u, 1.f / 40320.f);
    s = __builtin_fmaf(s, -u, 1.f / 5040.f);
    s = __builtin_fmaf(s, -u, 1.f / 720.f);
    s = __builtin_fmaf(s, -u, 1.f / 120.f);
    s = __builtin_fmaf(s, -u, 1.f / 24.f);
    s = __builtin_fmaf(s, -u, 1.f / 6.f);
    s = __builtin_fmaf(s, -u, 0.5f);
    return s * u * u;
}

constexpr int KL_STATS = 6;  // of a strip: base maximum, sum; trial maximum, sum; sums of w phi(D) and of w D
// The blocks 2i of n are base rows, 2i + 1 the same trial rows.
struct EpiKlStats {
    float *part;  // [strip][KL_STATS][npad]
    int64_t npad, n;
    int64_t rows, strip0;
    template <int MI, int NJ>
    __device__ __forceinline__ void operator()(floatx4 (&acc)[MI][NJ], int mb, int nb, int lane) const {
        const int64_t strip = strip0 + mb / MI;
        const int64_t v0 = (int64_t)mb * 16 + 4 * (lane >> 4);
#pragma unroll
        for (int j = 0; j < NJ; j += 2) {
            const int64_t tok = (int64_t)(nb + j) / 2 * 16 + (lane & 15);
            float mx[2] = {LOWEST, LOWEST}, sum[2] = {0.f, 0.f}, far = 0.f, near = 0.f;
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int i = 0; i < MI; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        if (v0 + i * 16 + r >= rows) acc[i][j + h][r] = LOWEST;
                        mx[h] = fmaxf(mx[h], acc[i][j + h][r]);
                    }
                mx[h] = fmaxf(mx[h], __shfl_xor(mx[h], 16));
                mx[h] = fmaxf(mx[h], __shfl_xor(mx[h], 32));
            }
#pragma unroll
            for (int i = 0; i < MI; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if (v0 + i * 16 + r >= rows) continue;
                    const float b = acc[i][j][r], t = acc[i][j + 1][r], u = b - t;
                    const float w = fast_exp(b - mx[0]);
                    sum[0] += w;
                    sum[1] += fast_exp(t - mx[1]);
                    far = __builtin_fmaf(w, u, far);
                    near += fabsf(u) <= 1.f ? w * phi_near(u) : w * (u - 1.f) + fast_exp(t - mx[0]);
                }
            float v[KL_STATS] = {mx[0], sum[0], mx[1], sum[1], near, far};
#pragma unroll
            for (int k = 0; k < KL_STATS; k++) {
                if (k != 0 && k != 2) {
                    v[k] += __shfl_xor(v[k], 16);
                    v[k] += __shfl_xor(v[k], 32);
                }
                if (tok < n && lane < 16) part[(strip * KL_STATS + k) * npad + tok] = v[k];
            }
        }
    }
};

__global__ __launch_bounds__(256) void kl_join_kernel(float *kl, float *lse_base, float *lse_trial, const float *part,
                                                      int64_t n, int64_t npad, int64_t strips) {
    __shared__ float ms[8][2][32];
    __shared__ double ss[8][4][32];
    const int c = threadIdx.x & 31, sl = threadIdx.x >> 5;
    const int64_t tok = (int64_t)blockIdx.x * 32 + c;
    float m[2] = {LOWEST, LOWEST};
    double s[4] = {0, 0, 0, 0};  // base sum, trial sum, near, far
    if (tok < n) {
        for (int64_t k = sl; k < strips; k += 8)
            for (int h = 0; h < 2; h++) m[h] = fmaxf(m[h], part[(k * KL_STATS + 2 * h) * npad + tok]);
        for (int64_t k = sl; k < strips; k += 8) {
            const float *p = part + k * KL_STATS * npad + tok;
            const double e = expf(p[0] - m[0]), f = expf(p[2 * npad] - m[1]);
            s[0] += e * p[npad];
            s[1] += f * p[3 * npad];
            s[2] += e * p[4 * npad];
            s[3] += e * p[5 * npad];
        }
    }
    for (int h = 0; h < 2; h++) ms[sl][h][c] = m[h];
    for (int k = 0; k < 4; k++) ss[sl][k][c] = s[k];
    __syncthreads();
    if (sl != 0 || tok >= n) return;
    for (int k = 1; k < 8; k++)
        for (int h = 0; h < 2; h++) m[h] = fmaxf(m[h], ms[k][h][c]);
    for (int k = 0; k < 4; k++) s[k] = 0;
    for (int k = 0; k < 8; k++) {
        const double e = exp((double)ms[k][0][c] - (double)m[0]), f = exp((double)ms[k][1][c] - (double)m[1]);
        s[0] += e * ss[k][0][c];
        s[1] += f * ss[k][1][c];
        s[2] += e * ss[k][2][c];
        s[3] += e * ss[k][3][c];
    }
    const double lb = (double)m[0] + log(s[0]), lt = (double)m[1] + log(s[1]), d = lt - lb;
    lse_base[tok] = (float)lb;
    lse_trial[tok] = (float)lt;
    kl[tok] = (float)(fabs(d) <= 1 ? s[2] / s[0] - (expm1(d) - d) : s[3] / s[0] + d);
}

template <int T>
struct EpiKlGrad {
    Planes d;
    const float *lse_base, *lse_trial, *dkl;
    int64_t n, rows;
    template <int MI, int NJ>
    __device__ __forceinline__ void operator()(floatx4 (&acc)[MI][NJ], int mb, int nb, int lane) const {
        const int64_t v0 = (int64_t)mb * 16 + 4 * (lane >> 4);
#pragma unroll
        for (int j = 0; j < NJ; j += 2) {
            const int tb = (nb + j) / 2;
            if (tb >= d.groups) continue;
            const int64_t tok = (int64_t)tb * 16 + (lane & 15);
            float g = 0.f, lb = 0.f, lt = 0.f;
            if (tok < n) {
                g = dkl[tok];
                lb = lse_base[tok];
                lt = lse_trial[tok];
            }
#pragma unroll
            for (int i = 0; i < MI; i++) {
                if (((mb + i) >> 1) >= d.units) continue;
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float q = fast_exp(acc[i][j + 1][r] - lt) - fast_exp(acc[i][j][r] - lb);
                    v[r] = tok < n && v0 + i * 16 + r < rows ? __fmul_rn(g, q) : 0.f;
                }
                put_grad_terms<T>(d, mb + i, tb, lane, v);
            }
        }
    }
};

// ---------------------------------------------------------------------------
// pieces of the vocabulary

// Words of a piece: what is held for one (d, and the weight's planes where they
// are decoded) stays within about 256 MB, the size of the last cache; pieces of
// whole 256-row tiles, alike in size.
static int64_t piece_rows(int64_t vocab, int64_t per_row) {
    const int64_t most = ((int64_t)256 << 20) / (per_row > 0 ? per_row : 1);
    int64_t pieces = most >= vocab ? 1 : ceil_div(vocab, most < 256 ? 256 : most);
    return ceil_div(ceil_div(vocab, pieces), 256) * 256;
}

static int64_t weight_row_bytes(const TileView &w) {
    return weight_is_planes(w) ? 0 : weight_planes_shape(w, 16).plane_bytes() * weight_terms(w) / 16;
}
static int order_of(int a, int b) { return a > b ? a : b; }
// strips of the vocabulary in a piece: one for each wave's rows of a tile
static int64_t strips_of(int64_t rows, int64_t nblocks) {
    return ceil_div(rows, 256) * (rows_tall(nblocks) ? 4 : 2);
}

// The forward of either loss: stats(g, piece's epilogue arguments).
struct HeadPlan {
    Planes x[2];
    int64_t piece = 0, strips = 0, npad = 0, nblocks = 0;
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
    p.npad = ceil_div(n, 32) * 32;
    p.nblocks = p.x[0].groups * (kl ? 2 : 1);
    const int64_t per = weight_row_bytes(w);
    p.piece = per ? piece_rows(w.rows, per) : w.rows;
    for (int64_t r = 0; r < w.rows; r += p.piece)
        p.strips += strips_of(w.rows - r < p.piece ? w.rows - r : p.piece, p.nblocks);
    p.part = c.take((size_t)p.strips * p.npad * (kl ? KL_STATS * sizeof(float) : sizeof(float2)));
    p.picked = c.take<float>(p.npad);
    if (per) p.room = c.take(weight_planes_shape(w, p.piece).bytes());
    p.bytes = c.at;
    return p;
}

size_t head_loss_workspace(const TileView &w, int64_t n, int32_t dtype) {
    return head_plan(w, n, dtype, false, nullptr).bytes;
}
size_t head_kl_workspace(const TileView &w, int64_t n, int32_t dtype) {
    return head_plan(w, n, dtype, true, nullptr).bytes;
}

static RowsGemm logits_gemm(const Planes &wp, const Planes &x, const Planes *second) {
    RowsGemm g;
    g.a = rows_inner(wp);
    g.b = rows_inner(x);
    if (second) {
        g.b.paired = 1;
        g.b.pair = second->p - x.p;
    }
    g.stages = (int32_t)(x.units / 2);
    rows_pairs(g, wp, x, order_of(wp.terms, x.terms));
    return g;
}

void launch_head_loss(float *loss, float *lse, int32_t dtype, RowsArg x, int64_t n, const TileView &w,
                      const int32_t *targets, void *ws, hipStream_t s) {
    const HeadPlan p = head_plan(w, n, dtype, false, ws);
    launch_pack_rows(p.x[0], x.p, dtype, n, w.cols, x.stride, s);
    int64_t strip = 0;
    for (int64_t r = 0; r < w.rows; r += p.piece) {
        const int64_t rows = w.rows - r < p.piece ? w.rows - r : p.piece;
        const Planes wp = weight_planes(w, r, rows, p.room, s);
        const EpiLossStats epi{(float2 *)p.part, p.picked, targets, p.npad, n, rows, r, strip};
        launch_rows_gemm<false, false>(logits_gemm(wp, p.x[0], nullptr), wp.groups, p.nblocks, epi, s);
        strip += strips_of(rows, p.nblocks);
    }
    hipLaunchKernelGGL(loss_join_kernel, dim3((unsigned)ceil_div(n, 32)), dim3(256), 0, s, loss, lse,
                       (const float2 *)p.part, p.picked, targets, n, p.npad, p.strips, w.rows);
    DITCH_TRY_HIP(hipGetLastError());
}

void launch_head_kl(float *kl, float *lse_base, float *lse_trial, int32_t dtype, RowsArg base, RowsArg trial,
                    int64_t n, const TileView &w, void *ws, hipStream_t s) {
    const HeadPlan p = head_plan(w, n, dtype, true, ws);
    launch_pack_rows(p.x[0], base.p, dtype, n, w.cols, base.stride, s);
    launch_pack_rows(p.x[1], trial.p, dtype, n, w.cols, trial.stride, s);
    int64_t strip = 0;
    for (int64_t r = 0; r < w.rows; r += p.piece) {
        const int64_t rows = w.rows - r < p.piece ? w.rows - r : p.piece;
        const Planes wp = weight_planes(w, r, rows, p.room, s);
        const EpiKlStats epi{(float *)p.part, p.npad, n, rows, strip};
        launch_rows_gemm<false, false>(logits_gemm(wp, p.x[0], &p.x[1]), wp.groups, p.nblocks, epi, s);
        strip += strips_of(rows, p.nblocks);
    }
    hipLaunchKernelGGL(kl_join_kernel, dim3((unsigned)ceil_div(n, 32)), dim3(256), 0, s, kl, lse_base, lse_trial,
                       (const float *)p.part, n, p.npad, p.strips);
    DITCH_TRY_HIP(hipGetLastError());
}

// ---------------------------------------------------------------------------
// gradients

struct HeadGradPlan {
    Planes x[2], d;
    int64_t piece = 0, nblocks = 0, ld = 0;
    int parts = 1;
    int order = 1;  // of the products with d
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
    p.nblocks = p.x[0].groups;
    p.piece = piece_rows(w.rows, p.nblocks * 32 * terms + weight_row_bytes(w));
    if (p.piece > ceil_div(w.rows, 64) * 64) p.piece = ceil_div(w.rows, 64) * 64;
    p.d = Planes{nullptr, p.nblocks, p.piece / 32, terms};
    p.d.p = c.take(p.d.bytes());
    p.ld = ceil_div(w.cols, 4) * 4;
    p.parts = rows_parts(ceil_div(w.cols, 16), p.nblocks, p.piece / 64);
    p.part = c.take<float>((size_t)p.parts * n * p.ld);
    p.order = terms > 1 || weight_terms(w) == 1 ? terms : 2;
    if (weight_row_bytes(w)) p.room = c.take(weight_planes_shape(w, p.piece).bytes());
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
        const Planes wp = weight_planes(w, r, rows, p.room, s);
        Planes d = p.d;
        d.units = ceil_div(rows, 64) * 2;
        fill(wp, d, r, rows);
        if (dx.p) {
            RowsGemm g;
            g.a = rows_outer(wp);
            g.b = rows_inner(d);
            g.stages = (int32_t)(d.units / 2);
            g.parts = p.parts;
            rows_pairs(g, wp, d, p.order);
            const EpiParts epi{p.part, n * p.ld, p.ld, n, p.ld, r > 0};
            launch_rows_gemm<true, false>(g, ceil_div(w.cols, 16), p.nblocks, epi, s);
        }
        if (dw.p) {
            RowsGemm g;
            g.a = rows_outer(p.x[0]);
            g.b = rows_outer(d);
            g.stages = (int32_t)(d.groups / 4);
            rows_pairs(g, p.x[0], d, d.terms);
            char *out = (char *)dw.p + r * dw.stride * row_size(dtype);
            const EpiRows epi{out, dw.stride, rows, w.cols, dtype, rows_wide(out, dw.stride, dtype)};
            launch_rows_gemm<true, true>(g, ceil_div(w.cols, 16), ceil_div(rows, 16), epi, s);
        }
    }
    if (dx.p) launch_join_parts(dx.p, dtype, dx.stride, p.part, p.parts, n * p.ld, p.ld, n, w.cols, s);
}

template <int T>
static void fill_loss(const HeadGradPlan &p, const Planes &wp, const Planes &d, int64_t row0, int64_t rows, int64_t n,
                      int64_t vocab, const int32_t *targets, const float *lse, const float *dloss, hipStream_t s) {
    const EpiLossGrad<T> epi{d, targets, lse, dloss, n, rows, row0, vocab};
    launch_rows_gemm<false, false>(logits_gemm(wp, p.x[0], nullptr), d.units * 2, p.nblocks, epi, s);
}
template <int T>
static void fill_kl(const HeadGradPlan &p, const Planes &wp, const Planes &d, int64_t rows, int64_t n,
                    const float *lse_base, const float *lse_trial, const float *dkl, hipStream_t s) {
    const EpiKlGrad<T> epi{d, lse_base, lse_trial, dkl, n, rows};
    launch_rows_gemm<false, false>(logits_gemm(wp, p.x[0], &p.x[1]), d.units * 2, 2 * p.nblocks, epi, s);
}

void launch_head_loss_grad(int32_t dtype, RowsArg dx, RowsArg dw, RowsArg x, int64_t n, const TileView &w,
                           const int32_t *targets, const float *lse, const float *dloss, void *ws, hipStream_t s) {
    const HeadGradPlan p = head_grad_plan(w, n, dtype, false, ws);
    launch_pack_rows(p.x[0], x.p, dtype, n, w.cols, x.stride, s);
    head_grad(p, dtype, dx, dw, n, w, s, [&](const Planes &wp, const Planes &d, int64_t row0, int64_t rows) {
        auto f = p.d.terms == 1 ? fill_loss<1> : p.d.terms == 2 ? fill_loss<2> : fill_loss<3>;
        f(p, wp, d, row0, rows, n, w.rows, targets, lse, dloss, s);
    });
}

void launch_head_kl_grad(int32_t dtype, RowsArg dx, RowsArg base, RowsArg trial, int64_t n, const TileView &w,
                         const float *lse_base, const float *lse_trial, const float *dkl, void *ws, hipStream_t s) {
    const HeadGradPlan p = head_grad_plan(w, n, dtype, true, ws);
    launch_pack_rows(p.x[0], base.p, dtype, n, w.cols, base.stride, s);
    launch_pack_rows(p.x[1], trial.p, dtype, n, w.cols, trial.stride, s);
    head_grad(p, dtype, dx, RowsArg{}, n, w, s, [&](const Planes &wp, const Planes &d, int64_t, int64_t rows) {
        auto f = p.d.terms == 1 ? fill_kl<1> : p.d.terms == 2 ? fill_kl<2> : fill_kl<3>;
        f(p, wp, d, rows, n, lse_base, lse_trial, dkl, s);
    });
}

}  // namespace ditch
