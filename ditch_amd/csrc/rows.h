// rows.h — products between rows of activations and registered weights in both
// directions, for the operators that hand back gradients (head.hip, glu.hip).
//
// Every operand is brought to one form, planes of bf16 terms in 1 KiB units of
// 16 rows x 32 columns, the layout in which bf16 tensors are registered:
// element (row, k) at 16 * (row % 16 + 16 * (k % 32 / 8)) + 2 * (k % 8) of unit
// [row / 16][k / 32]. A product contracts over the columns of such an operand
// ("inner") or over its rows ("outer", read through the transposing LDS load),
// so the same planes serve x W^T, d W and d^T x. bf16 values are one term, f16
// values exactly two, f32 values exactly three (each term the next 8 bits), FP8,
// MXFP4 and INT4 weights one (what they decode to), f16 weights two, Q8_0 and
// f32 weights three, or two beside 16-bit rows. A product of several terms adds the pairs i + j < order.
#pragma once
#include "gemm_common.h"
#include "internal.h"

namespace ditch {

constexpr int ROWS_MAX_TERMS = 3;

// Planes of terms: plane e at p + e * plane_bytes().
struct Planes {
    char *p = nullptr;
    int64_t groups = 0, units = 0;  // of 16 rows, of 32 columns
    int terms = 0;
    __host__ __device__ int64_t plane_bytes() const { return groups * units * 1024; }
    size_t bytes() const { return (size_t)terms * plane_bytes(); }
};

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline int row_terms(int32_t dtype) { return dtype == DITCH_BF16 ? 1 : dtype == DITCH_F16 ? 2 : 3; }
inline size_t row_size(int32_t dtype) { return dtype == DITCH_F32 ? 4 : 2; }
// The terms of a weight that results of x_terms take: all of them f32 ones, at
// most two (16 bits, rounded) 16-bit ones, whose own rounding is far above what is
// left out.
int rows_weight_terms(const TileView &w, int x_terms);
// The terms that d, what a gradient's two products hand over, is held in: those of
// the rows' type; bf16 rows up to 64 get a second one, which costs nothing while
// the products wait for the weight (one value of d makes most of such a gradient,
// and its rounding would be the gradient's).
inline int grad_term_count(int x_terms, int64_t n) { return x_terms == 1 && n <= 64 ? 2 : x_terms; }
// and the pairs of terms that are multiplied: i + j < order; logits take all that count
// in 24 bits (off by 2^-17 of their terms they left divergences of f16 rows 2^-6 apart
// off by 3e-4; and terms are cut, of their value's sign, so that what a pair left out
// takes away is 7e-6 of every logit alike: at logits of 40 the loss' gradient, whose
// log sum has it all, was off by 2e-3).
constexpr int rows_order_of(int w_terms, int x_terms, bool logits = false) {
    const int all = w_terms + x_terms - 1, most = w_terms > x_terms ? w_terms : x_terms;
    return logits ? (all < ROWS_MAX_TERMS ? all : ROWS_MAX_TERMS) : most;
}

// Rows of activations: 64 rows and 128 columns (a unit of 4-bit codes), zeros
// behind the last row and column.
inline Planes row_planes(int64_t n, int64_t cols, int terms) {
    return Planes{nullptr, ceil_div(n, 64) * 4, ceil_div(cols, 128) * 4, terms};
}
// Of which a product needs those with rows in them; d, read transposed too, 32 rows at a time.
inline int64_t row_blocks(int64_t n) { return ceil_div(n, 16); }
inline int64_t grad_blocks(int64_t n) { return ceil_div(n, 32) * 2; }
// (live: rows where it is negative are zeros, whatever they hold)
void launch_pack_rows(const Planes &out, const void *x, int32_t dtype, int64_t n, int64_t cols, int64_t stride,
                      hipStream_t s, const int32_t *live = nullptr);
// The weight's rows [row0, row0 + rows) as planes: its own tiles where they are
// that already (nothing launched), else decoded to `room` (row0 a multiple of 16).
bool weight_is_planes(const TileView &w);
Planes weight_planes_shape(const TileView &w, int64_t rows, int x_terms);
Planes weight_planes(const TileView &w, int64_t row0, int64_t rows, int x_terms, char *room, hipStream_t s);

// The grid of `blocks` workgroups, in rows of less than 2^32 threads, which is what a
// launch takes along x (2^24 rows on 40000 words are 2^32.3 in the largest tiles); a
// multiple of 8, so that rows_block() and the hardware number the XCDs alike. The
// last row may have blocks behind the last.
inline dim3 rows_grid(int64_t blocks, int threads, int64_t parts = 1) {
    const int64_t most = (((int64_t)1 << 32) - 1) / threads / 8 * 8, x = blocks < 1 ? 1 : blocks < most ? blocks : most;
    return dim3((unsigned)x, (unsigned)parts, (unsigned)ceil_div(blocks, x));
}
__device__ __forceinline__ int64_t rows_block() { return (int64_t)blockIdx.z * gridDim.x + blockIdx.x; }

// Scratch as one run of the caller's workspace.
struct Carver {
    char *base;
    size_t at = 0;
    explicit Carver(void *p) : base((char *)p) {}
    template <typename T = char>
    T *take(size_t count) {
        at = (at + 255) & ~(size_t)255;
        T *r = (T *)(base + at);
        at += count * sizeof(T);
        return base ? r : nullptr;
    }
};

// out[i][c] = the sum over parts of part[p][i][c], in f32, rounded to dtype; with
// `times`, and times[i] of the same of `more`.
struct MoreParts {
    const float *part = nullptr, *times = nullptr;
    int parts = 0;
};
void launch_join_parts(void *out, int32_t dtype, int64_t stride, const float *part, int parts, int64_t part_stride,
                       int64_t ld, int64_t n, int64_t cols, hipStream_t s, MoreParts more = {});

// The tile and the parts (of k) of a product of mblocks x nblocks 16-row blocks
// over k32 steps of 32 k of the pairs of terms i + j < order, `sets` times
// (rows.hip). Parts are tried only where `split`; inner: neither operand is read
// transposed.
constexpr int ROWS_FEW = 6;  // rows_gemm.h: no tile, k shared by the waves
struct RowsTiling {
    int tile = 0, parts = 1;
};
RowsTiling rows_tiling(int64_t mblocks, int64_t nblocks, int64_t k32, int a_terms, int b_terms, int order, int sets,
                       bool split, bool inner);
// 16-row blocks of a wave's strip and of a tile along m
inline int rows_strip_blocks(int tile) { return tile == 0 ? 8 : tile == 3 || tile == ROWS_FEW ? 2 : 4; }
inline int rows_tile_blocks(int tile) { return tile == 1 ? 8 : tile == 3 ? 4 : tile == ROWS_FEW ? 2 : 16; }
inline int rows_pair_count(int a, int b, int order) {
    int n = 0;
    for (int i = 0; i < a; i++) n += order - i < 0 ? 0 : order - i < b ? order - i : b;
    return n;
}

// rows_products.hip: c as parts of sums [part][n][ld] (added where `add`), a outer
// and b inner; and as rows of `dtype`, both outer (b paired: of two outputs)
struct RowsArg {
    void *p = nullptr;
    int64_t stride = 0;
};
struct RowsGemm;
void launch_rows_parts(int tile, const RowsGemm &g, float *part, int64_t ld, int64_t n, int64_t m, bool add, hipStream_t s);
void launch_rows_out(const RowsGemm &g, RowsArg out, RowsArg second, int32_t dtype, int64_t n, int64_t m, hipStream_t s);

// head.hip, head_grad.hip
size_t head_loss_workspace(const TileView &w, int64_t n, int32_t dtype);
void launch_head_loss(float *loss, float *lse, int32_t dtype, RowsArg x, int64_t n, const TileView &w,
                      const int32_t *targets, void *ws, hipStream_t s);
size_t head_loss_grad_workspace(const TileView &w, int64_t n, int32_t dtype, bool dw);
void launch_head_loss_grad(int32_t dtype, RowsArg dx, RowsArg dw, RowsArg x, int64_t n, const TileView &w,
                           const int32_t *targets, const float *lse, const float *dloss, void *ws, hipStream_t s);
size_t head_kl_workspace(const TileView &w, int64_t n, int32_t dtype);
void launch_head_kl(float *kl, float *lse_base, float *lse_trial, int32_t dtype, RowsArg base, RowsArg trial,
                    int64_t n, const TileView &w, void *ws, hipStream_t s);
size_t head_kl_grad_workspace(const TileView &w, int64_t n, int32_t dtype);
void launch_head_kl_grad(int32_t dtype, RowsArg dx, RowsArg base, RowsArg trial, int64_t n, const TileView &w,
                         const float *lse_base, const float *lse_trial, const float *dkl, void *ws, hipStream_t s);

// glu.hip
size_t glu_rows_workspace(const TileView &gate, const TileView &up, int64_t n, int32_t dtype);
void launch_glu_rows(int32_t dtype, RowsArg out, RowsArg x, int64_t n, const TileView &gate, const TileView &up,
                     uint32_t act, void *ws, hipStream_t s);
size_t glu_rows_grad_workspace(const TileView &gate, const TileView &up, int64_t n, int32_t dtype, bool dw);
void launch_glu_rows_grad(int32_t dtype, RowsArg dx, RowsArg dgate, RowsArg dup, RowsArg dout, RowsArg x, int64_t n,
                          const TileView &gate, const TileView &up, uint32_t act, void *ws, hipStream_t s);

}  // namespace ditch
