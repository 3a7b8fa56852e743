// head.h — what the head's losses (head.hip) and their gradients
// (head_grad.hip) share: pieces of the vocabulary, the logits' product.
#pragma once
#include "rows_coded.h"

namespace ditch {

__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(__fmul_rn(x, 1.4426950408889634f)); }


constexpr float LOWEST = -3.0e38f;  // in place of words that are not there

// ---------------------------------------------------------------------------
// joins of what the strips leave

// Sums of strips, each relative to its own reference (a maximum), over a block of
// 512: TOK rows, 512 / TOK slices of the strips each; row tid % TOK. The largest
// reference first, then every thread's sums once rescaled to it.
template <int TOK>
__device__ __forceinline__ float block_max(float m, float *lds) {  // lds[8][TOK]
#pragma unroll
    for (int o = TOK; o < 64; o *= 2) m = fmaxf(m, __shfl_xor(m, o));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane < TOK) lds[wave * TOK + lane] = m;
    __syncthreads();
    m = lds[threadIdx.x % TOK];
#pragma unroll
    for (int w = 1; w < 8; w++) m = fmaxf(m, lds[w * TOK + threadIdx.x % TOK]);
    __syncthreads();
    return m;
}
template <int TOK>
__device__ __forceinline__ double block_sum(double s, double *lds) {
#pragma unroll
    for (int o = TOK; o < 64; o *= 2) s += __shfl_xor(s, o);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane < TOK) lds[wave * TOK + lane] = s;
    __syncthreads();
    s = lds[threadIdx.x % TOK];
#pragma unroll
    for (int w = 1; w < 8; w++) s += lds[w * TOK + threadIdx.x % TOK];
    __syncthreads();
    return s;
}

// Rows of a join's block.
template <typename F>
void with_join_rows(int64_t n, F &&f) {
    if (n >= 4096) f(std::integral_constant<int, 32>{});
    else if (n >= 256) f(std::integral_constant<int, 8>{});
    else f(std::integral_constant<int, 1>{});
}

// ---------------------------------------------------------------------------
// what the forward products keep of their tiles (head.hip joins it)

struct EpiLossStats {
    static constexpr bool PAIRS = false;
    static constexpr bool F32_RESULT = true, ALL_PAIRS = true;
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

// phi(u) = u + e^-u - 1 for |u| <= 1/4: its series to u^7, off by 2^-27 of it
__device__ __forceinline__ float phi_near(float u) {
    float s = -1.f / 5040.f;
    s = __builtin_fmaf(s, u, 1.f / 720.f);
    s = __builtin_fmaf(s, u, -1.f / 120.f);
    s = __builtin_fmaf(s, u, 1.f / 24.f);
    s = __builtin_fmaf(s, u, -1.f / 6.f);
    s = __builtin_fmaf(s, u, 0.5f);
    return s * u * u;
}

// Of a strip: the base's maximum and sum, the trial's maximum and sum, and with w =
// e^(l_base - its maximum) and u = D less the maxima's difference (words that moved
// alike have small u, whatever they moved by) the sums of w phi(u) and of w u.
constexpr int KL_STATS = 6;
// The blocks 2i of n are base rows, 2i + 1 the same trial rows.
struct EpiKlStats {
    static constexpr bool PAIRS = true;  // of n's blocks
    static constexpr bool F32_RESULT = true, ALL_PAIRS = true;
    float *part;  // [strip][npad][KL_STATS]
    int64_t npad, n;
    int64_t rows, strip0;
    template <int MI, int NJ>
    __device__ __forceinline__ void operator()(floatx4 (&acc)[MI][NJ], int mb, int nb, int lane) const {
        const int64_t strip = strip0 + mb / MI;
        const int64_t v0 = (int64_t)mb * 16 + 4 * (lane >> 4);
        const bool whole = (int64_t)(mb + MI) * 16 <= rows;
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
                        // (both at LOWEST: no weight)
                        if (!whole && v0 + i * 16 + r >= rows) acc[i][j + h][r] = LOWEST;
                        mx[h] = fmaxf(mx[h], acc[i][j + h][r]);
                    }
                mx[h] = fmaxf(mx[h], __shfl_xor(mx[h], 16));
                mx[h] = fmaxf(mx[h], __shfl_xor(mx[h], 32));
            }
            const float moved = mx[0] - mx[1];
#pragma unroll
            for (int i = 0; i < MI; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float b = acc[i][j][r], t = acc[i][j + 1][r], u = (b - t) - moved;
                    const float w = fast_exp(b - mx[0]), x = fast_exp(t - mx[1]);  // x = w e^-u
                    sum[0] += w;
                    sum[1] += x;
                    far = __builtin_fmaf(w, u, far);
                    near += fabsf(u) <= 0.25f ? w * phi_near(u) : __builtin_fmaf(w, u - 1.f, x);
                }
            float v[KL_STATS] = {mx[0], sum[0], mx[1], sum[1], near, far};
#pragma unroll
            for (int k = 0; k < KL_STATS; k++) {
                if (k != 0 && k != 2) {
                    v[k] += __shfl_xor(v[k], 16);
                    v[k] += __shfl_xor(v[k], 32);
                }
            }
            if (tok < n && lane < 16) {
                float2 *o = (float2 *)(part + (strip * npad + tok) * KL_STATS);
                o[0] = make_float2(v[0], v[1]);
                o[1] = make_float2(v[2], v[3]);
                o[2] = make_float2(v[4], v[5]);
            }
        }
    }
};

// ---------------------------------------------------------------------------
// what the gradients' products leave of theirs (head_grad.hip)

// d of a piece as terms. Rows without a target give zeros, targets past the
// vocabulary NaN.
template <int T>
struct EpiLossGrad {
    static constexpr bool PAIRS = false;
    static constexpr bool F32_RESULT = false, ALL_PAIRS = true;  // (lse is of all of them)
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

// e^z - 1 for |z| <= 1/4: its series to z^8, off by 2^-34 of it
__device__ __forceinline__ float expm1_near(float z) {
    float s = 1.f / 40320.f;
    s = __builtin_fmaf(s, z, 1.f / 5040.f);
    s = __builtin_fmaf(s, z, 1.f / 720.f);
    s = __builtin_fmaf(s, z, 1.f / 120.f);
    s = __builtin_fmaf(s, z, 1.f / 24.f);
    s = __builtin_fmaf(s, z, 1.f / 6.f);
    s = __builtin_fmaf(s, z, 0.5f);
    return __builtin_fmaf(s * z, z, z);
}

// d = g (q - p) = g p (e^z - 1), z = (l_trial - l_base) - (lse_trial - lse_base), the
// latter form where z is small: what is left is as exact as z (d of one term, 2^-8 of
// itself, does not show it: 2 % of 1500 bf16 rows' time for nothing). And what mends
// the log sums' rounding (head_grad.hip): p as one term, the strips' sums of q - p.
template <int T>
struct EpiKlGrad {
    static constexpr bool PAIRS = true;  // of n's blocks
    static constexpr bool F32_RESULT = true, ALL_PAIRS = true;  // (of near rows' logits a difference is left)
    static constexpr bool NEAR = T > 1;
    Planes d;
    Planes p;     // (none: p.p NULL)
    float *sums;  // [strip][npad]
    const float *lse_base, *lse_trial, *dkl;
    int64_t n, rows, npad, strip0;
    template <int MI, int NJ>
    __device__ __forceinline__ void operator()(floatx4 (&acc)[MI][NJ], int mb, int nb, int lane) const {
        const int64_t v0 = (int64_t)mb * 16 + 4 * (lane >> 4);
#pragma unroll
        for (int j = 0; j < NJ; j += 2) {
            const int tb = (nb + j) / 2;
            if (tb >= d.groups) continue;
            const int64_t tok = (int64_t)tb * 16 + (lane & 15);
            float g = 0.f, lb = 0.f, c = 0.f, lt = 0.f, sum = 0.f;
            if (tok < n) {
                g = dkl[tok];
                lb = lse_base[tok];
                lt = lse_trial[tok];
                c = lt - lb;
            }
#pragma unroll
            for (int i = 0; i < MI; i++) {
                if (((mb + i) >> 1) >= d.units) continue;
                float v[4], w[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const bool in = tok < n && v0 + i * 16 + r < rows;
                    const float b = acc[i][j][r], t = acc[i][j + 1][r], e = fast_exp(b - lb);
                    float q = fast_exp(t - lt) - e;
                    if constexpr (NEAR) {
                        const float z = (t - b) - c;
                        if (fabsf(z) <= 0.25f) q = e * expm1_near(z);
                    }
                    v[r] = in ? __fmul_rn(g, q) : 0.f;
                    w[r] = in ? e : 0.f;
                    sum += in ? q : 0.f;
                }
                put_grad_terms<T>(d, mb + i, tb, lane, v);
                if constexpr (NEAR)
                    if (p.p) put_grad_terms<1>(p, mb + i, tb, lane, w);
            }
            if (!NEAR || !p.p) continue;
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (tok < n && lane < 16) sums[(strip0 + mb / MI) * npad + tok] = sum;
        }
    }
};

// ---------------------------------------------------------------------------
// products

// head_coded.hip: the same on weights that are not planes (rows_coded.h)
void launch_loss_coded(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks, const EpiLossStats &epi,
                       hipStream_t s);
void launch_kl_coded(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks, const EpiKlStats &epi,
                     hipStream_t s);
template <int T>
void launch_loss_grad_coded(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks,
                            const EpiLossGrad<T> &epi, hipStream_t s);
template <int T>
void launch_kl_grad_coded(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks,
                          const EpiKlGrad<T> &epi, hipStream_t s);

// Words of a piece: what is held for one (d, and the weight's planes where they
// are decoded) stays within about 256 MB, the size of the last cache; pieces of
// whole 256-row tiles, alike in size.
inline int64_t piece_rows(int64_t vocab, int64_t per_row) {
    const int64_t most = ((int64_t)256 << 20) / (per_row > 0 ? per_row : 1);
    int64_t pieces = most >= vocab ? 1 : ceil_div(vocab, most < 256 ? 256 : most);
    return ceil_div(ceil_div(vocab, pieces), 256) * 256;
}

// strips of the vocabulary in a piece: one for each wave's rows of a tile
inline int64_t strips_of(int64_t rows, int tile) {
    return ceil_div(ceil_div(rows, 16), rows_tile_blocks(tile)) * rows_tile_blocks(tile) / rows_strip_blocks(tile);
}

inline int64_t weight_row_bytes(const TileView &w, int x_terms) {
    return weight_is_planes(w) ? 0 : (int64_t)weight_planes_shape(w, 16, x_terms).bytes() / 16;
}
inline RowsGemm logits_gemm(const Planes &wp, const RowsIn &in) {
    RowsGemm g;
    g.a = rows_inner(wp);
    g.b = in.op;
    g.k32 = (int32_t)ceil_div(wp.units, 2) * 2;
    rows_pairs(g, wp, in.x, rows_order_of(wp.terms, in.x.terms, true));
    return g;
}

inline int logits_tile(const TileView &w, int64_t rows, const Planes &x, int64_t nblocks, bool f32_result) {
    const int a = rows_weight_terms(w, f32_result ? ROWS_MAX_TERMS : x.terms), order = rows_order_of(a, x.terms, true);
    return rows_tiling(ceil_div(rows, 16), nblocks, ceil_div(w.cols, 64) * 2, a, x.terms, order, 1, false, true).tile;
}

inline RowsCoded coded_product(const TileView &w, const RowsIn &in) {
    RowsCoded p;
    p.w[0] = p.w[1] = w;
    p.b = in.op;
    p.x = in.x.p;
    p.x_plane = in.x.plane_bytes();
    p.blocks = (int32_t)ceil_div(w.rows, 16);
    p.stages = (int32_t)w.units_k;
    return p;
}

}  // namespace ditch
