// rows.hip — operands of the products in rows_gemm.h: activations and weights
// as planes of bf16 terms, and the joining of partial sums.
#include "rows.h"

#include "tile_decode.h"
#include "tiled.h"

namespace ditch {

int rows_weight_terms(const TileView &w, int x_terms) {
    const int most = x_terms == 3 ? 3 : 2;
    const int own = w.tf == TF_F16 ? 2 : w.tf == TF_F32 || w.tf == TF_Q8 ? 3 : 1;
    return own < most ? own : most;
}

// v as terms: each but the last the next 8 bits of the remainder (cut, so that
// no finite value becomes infinite), the last one rounded to nearest even. With
// as many terms as the type's mantissa has bytes nothing is rounded. Infinities
// and NaN are all in the first term.
template <int T>
__device__ __forceinline__ void to_terms(float v, uint16_t (&t)[T]) {
    if ((f2u(v) & 0x7f800000u) == 0x7f800000u) {
        t[0] = (uint16_t)(f2u(v) >> 16) | ((f2u(v) & 0x7fffffu) ? 0x40 : 0);
#pragma unroll
        for (int e = 1; e < T; e++) t[e] = 0;
        return;
    }
#pragma unroll
    for (int e = 0; e < T; e++) {
        const uint32_t b = e + 1 < T ? f2u(v) & 0xffff0000u : rne_bits(v);
        t[e] = (uint16_t)(b >> 16);
        v = __fsub_rn(v, u2f(b));
    }
}

template <int DT>
__device__ __forceinline__ float row_value(const void *x, int64_t i) {
    if constexpr (DT == DITCH_F32) return ((const float *)x)[i];
    else if constexpr (DT == DITCH_F16) return f16_to_f32_hw(((const uint16_t *)x)[i]);
    else return bf16_to_f32(((const uint16_t *)x)[i]);
}

// A wave a unit: each lane 8 columns of a row, as whole 16-byte words where the
// rows are aligned to them.
template <int DT, int T>
__global__ __launch_bounds__(256) void pack_rows_kernel(Planes out, const void *x, int64_t n, int64_t cols,
                                                        int64_t stride, int wide, const int32_t *live) {
    const int lane = threadIdx.x & 63;
    const int64_t unit = rows_block() * 4 + (threadIdx.x >> 6);
    if (unit >= out.groups * out.units) return;
    const int64_t g = unit / out.units, u = unit % out.units;
    const int64_t row = g * 16 + (lane & 15), k = u * 32 + (lane >> 4) * 8;
    const bool there = row < n && (!live || live[row] >= 0);
    float v[8];
    uint16_t t[8][T];
    if (there && k + 8 <= cols && wide) {
        const int64_t at = row * stride + k;
        if constexpr (DT == DITCH_F32) {
            const float4 a = *(const float4 *)((const float *)x + at), b = *(const float4 *)((const float *)x + at + 4);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            const u32x4 a = *(const u32x4 *)((const uint16_t *)x + at);
            if constexpr (DT == DITCH_BF16) {
                *(u32x4 *)(out.p + unit * 1024 + lane * 16) = a;
                return;
            }
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = f16_to_f32_hw((uint16_t)(a[j / 2] >> (16 * (j & 1))));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = there && k + j < cols ? row_value<DT>(x, row * stride + k + j) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) to_terms<T>(v[j], t[j]);
#pragma unroll
    for (int e = 0; e < T; e++) {
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = (uint32_t)t[2 * j][e] | (uint32_t)t[2 * j + 1][e] << 16;
        *(u32x4 *)(out.p + e * out.plane_bytes() + unit * 1024 + lane * 16) = w;
    }
}

void launch_pack_rows(const Planes &out, const void *x, int32_t dtype, int64_t n, int64_t cols, int64_t stride,
                      hipStream_t s, const int32_t *live) {
    const int64_t units = out.groups * out.units;
    if (units == 0) return;
    const int wide = ((uintptr_t)x | (uintptr_t)(stride * (int64_t)row_size(dtype))) % 16 == 0;
    const dim3 grid = rows_grid(ceil_div(units, 4), 256);
    if (dtype == DITCH_F32)
        hipLaunchKernelGGL((pack_rows_kernel<DITCH_F32, 3>), grid, dim3(256), 0, s, out, x, n, cols, stride, wide, live);
    else if (dtype == DITCH_F16)
        hipLaunchKernelGGL((pack_rows_kernel<DITCH_F16, 2>), grid, dim3(256), 0, s, out, x, n, cols, stride, wide, live);
    else
        hipLaunchKernelGGL((pack_rows_kernel<DITCH_BF16, 1>), grid, dim3(256), 0, s, out, x, n, cols, stride, wide, live);
    DITCH_TRY_HIP(hipGetLastError());
}

// Tiles of 256 x 256, 128 x 128, 256 x 64, 64 x 64, and 256 x 64 with the whole LDS as
// its ring (three terms only: two stages of them fill half of it, and 224
// workgroups on as many CUs then wait for memory, 147 us against 109; where there
// are more than CUs two on each are better, 184 against 207). For each: how many workgroups fit a CU (by their LDS), and what 32 k of one, two or three terms of
// b take (us) where a workgroup is alone on its CU and where as many as fit share it,
// and what a round of workgroups takes to begin and end; measured over products of
// 4864 to 151936 rows, 1 to 3000 columns, 896 to 4096 k, and within a fifth of them.
// The cheapest by rounds over the chip's 256 CUs: large products take large tiles,
// where the LDS feeds the matrix cores best (872 us for 128256 x 1000 x 4096 in 256 x
// 256, 996 in 128 x 128, 1624 in 64 x 64), few columns the narrow ones (64 f32 columns:
// 179 us for 256 x 64, 546 for 256 x 256), small ones whichever spreads over the chip.
RowsTiling rows_tiling(int64_t mblocks, int64_t nblocks, int64_t k32, int a_terms, int b_terms, int order, int sets,
                       bool split, bool inner) {
    static const struct {
        int bm, bn, fit[3];
        double one[3], all[3], ends;
    } tiles[5] = {{16, 16, {1, 1, 1}, {0.67, 1.25, 1.72}, {0.78, 1.50, 2.13}, 8},
                  {8, 8, {2, 2, 2}, {0.34, 0.59, 0.85}, {0.46, 0.77, 1.13}, 4},
                  {16, 4, {2, 2, 2}, {0.35, 0.55, 0.85}, {0.54, 0.79, 1.08}, 4},
                  {4, 4, {4, 3, 2}, {0.19, 0.27, 0.31}, {0.40, 0.45, 0.47}, 4},
                  {16, 4, {1, 1, 1}, {9, 9, 0.70}, {9, 9, 0.72}, 4}};
    const int b = b_terms - 1;
    const double terms = (double)rows_pair_count(a_terms, b_terms, order) / b_terms * sets;  // stages a step
    // a is read once at least, 5.5 TB/s
    const double memory = (double)mblocks * k32 * a_terms * sets * 1024 / 5.5e6;
    RowsTiling best;
    double least = 1e30;
    for (int t = inner && b_terms == 3 ? 1 : 0; t < 5; t++) {  // (three terms: sums in two levels)
        const int64_t tiles_mn = ceil_div(mblocks, tiles[t].bm) * ceil_div(nblocks, tiles[t].bn);
        const int fit = tiles[t].fit[b];
        for (int64_t parts = 1; parts <= (split ? 64 : 1) && (parts == 1 || k32 / parts >= 8); parts++) {
            const int64_t wgs = tiles_mn * parts, full = 256 * fit, rest = wgs % full;
            const double stages = (double)ceil_div(k32, parts) * terms, share = tiles[t].all[b] / fit * ceil_div(rest, 256);
            double us = (wgs / full) * (stages * tiles[t].all[b] + tiles[t].ends);
            if (rest) us += stages * (share > tiles[t].one[b] ? share : tiles[t].one[b]) + tiles[t].ends;
            // (256 workgroups, each with a stage or two on its way, reach three quarters of that, 512 nine tenths)
            const double read = memory * (1 + 90.0 / (wgs < 90 ? 90 : wgs));
            if (us < read) us = read + us / 100;
            // parts are written, read and added: 4 bytes twice at 4 TB/s
            us += parts * (double)mblocks * nblocks * 256 * 8 / 4e6;
            if (us < least) {
                least = us;
                best.tile = t;
                best.parts = (int)parts;
            }
        }
    }
    // up to 64 16-bit rows on up to 1024 blocks (rows_gemm.h; the block of 2048 x 2048 and
    // one bf16 row 5.1 us, by tiles 13.6, of 4864 x 896 4.9 and 8.0; the loss of 16000 x 896 9.0
    // and 11.6; of 30000 x 2048 and 30 rows 36 and 29)
    if (inner && a_terms == 1 && b_terms < 3 && nblocks <= 4 && mblocks <= 1024) best.tile = ROWS_FEW;
    return best;
}

bool weight_is_planes(const TileView &w) { return w.tf == TF_BF16; }

Planes weight_planes_shape(const TileView &w, int64_t rows, int x_terms) {
    if (weight_is_planes(w)) return Planes{nullptr, ceil_div(rows, 16), w.units_k, 1};
    return Planes{nullptr, ceil_div(rows, 16), ceil_div(w.cols, 32), rows_weight_terms(w, x_terms)};
}

// The tiles' own words: a wave a unit of the weight (32 to 128 columns), each
// lane the 8 columns that it holds of each 32 as one word a term. FP8, MXFP4 and
// INT4 by the conversions of the tiled products (tensors that these decode
// exactly), f16, f32 and Q8_0 value by value. (An element at a time through
// decode_any_kernel took 199 us for 14336 x 4096 in FP8.)
template <int TF, int T>
__global__ __launch_bounds__(256) void decode_planes_kernel(Planes out, TileView w, int64_t group0) {
    constexpr int TILES = TF == TF_FP8 || TF == TF_Q8 ? 2 : TF == TF_MX4 || TF == TF_INT4 ? 4 : 1;
    const int lane = threadIdx.x & 63;
    const int64_t unit = rows_block() * 4 + (threadIdx.x >> 6);
    if (unit >= out.groups * w.units_k) return;
    const int64_t g = unit / w.units_k, u = unit % w.units_k, src = (group0 + g) * w.units_k + u;
    u32x4 words[TF == TF_F32 ? 2 : 1];
    if constexpr (TF == TF_F32) {
        words[0] = *(const u32x4 *)(w.codes + src * 2048 + lane * 16);
        words[1] = *(const u32x4 *)(w.codes + src * 2048 + 1024 + lane * 16);
    } else words[0] = *(const u32x4 *)(w.codes + src * 1024 + lane * 16);
    uint32_t sd[2] = {0, 0};
    if constexpr (T == 1) {
        const SideStep st = side_step<TF>(w);
        const uint32_t *side = w.side + side_row(w, group0 + g, lane);
        for (int j = 0; j < TileCfg<TF>::NS; j++) sd[j] = *side_word<TF>(st, side, u, j);
    }
#pragma unroll
    for (int t = 0; t < TILES; t++) {
        const int64_t ou = u * TILES + t;
        if (ou >= out.units) return;
        char *at = out.p + (g * out.units + ou) * 1024 + lane * 16;
        if constexpr (T == 1) {
            *(u32x4 *)at = decode_tile_lds<TF>(w, words, sd, t, true);
        } else {
            float v[8];
            if constexpr (TF == TF_F32) {
                for (int j = 0; j < 8; j++) v[j] = u2f(words[j / 4][j % 4]);
            } else if constexpr (TF == TF_F16) {
                for (int j = 0; j < 8; j++) v[j] = f16_to_f32_hw((uint16_t)(words[0][j / 2] >> (16 * (j & 1))));
            } else {
                int64_t row = (group0 + g) * 16 + (lane & 15);
                row = row < w.rows ? row : w.rows - 1;
                const float d = f16_to_f32(((const uint16_t *)w.scale)[row * w.scale_cols + (ou < w.scale_cols ? ou : 0)]);
                for (int j = 0; j < 8; j++)
                    v[j] = __fmul_rn((float)(int8_t)(words[0][2 * t + j / 4] >> (8 * (j % 4))), d);
            }
            uint16_t e[8][T];
#pragma unroll
            for (int j = 0; j < 8; j++) to_terms<T>(v[j], e[j]);
#pragma unroll
            for (int k = 0; k < T; k++) {
                u32x4 o;
#pragma unroll
                for (int j = 0; j < 4; j++) o[j] = (uint32_t)e[2 * j][k] | (uint32_t)e[2 * j + 1][k] << 16;
                *(u32x4 *)(at + k * out.plane_bytes()) = o;
            }
        }
    }
}

// Tensors that the conversions do not decode exactly (codes or scales that are
// not finite, odd blocks): a wave a unit, each lane 8 columns of a row.
__global__ __launch_bounds__(256) void decode_any_kernel(Planes out, TileView w, int64_t row0) {
    const int lane = threadIdx.x & 63;
    const int64_t unit = rows_block() * 4 + (threadIdx.x >> 6);
    if (unit >= out.groups * out.units) return;
    const int64_t g = unit / out.units, u = unit % out.units;
    const int64_t row = row0 + g * 16 + (lane & 15), k = u * 32 + (lane >> 4) * 8;
    uint16_t t[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int j = 0; j < 8; j++)
        if (row < w.rows && k + j < w.cols) (void)tiled_element_f32(w, row, k + j, &t[j]);
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = (uint32_t)t[2 * j] | (uint32_t)t[2 * j + 1] << 16;
    *(u32x4 *)(out.p + unit * 1024 + lane * 16) = o;
}

Planes weight_planes(const TileView &w, int64_t row0, int64_t rows, int x_terms, char *room, hipStream_t s) {
    Planes out = weight_planes_shape(w, rows, x_terms);
    if (weight_is_planes(w)) {
        out.p = (char *)w.codes + row0 / 16 * w.units_k * 1024;
        return out;
    }
    out.p = room;
    const dim3 grid = rows_grid(ceil_div(out.groups * w.units_k, 4), 256), each = rows_grid(ceil_div(out.groups * out.units, 4), 256);
    auto go = [&](auto tf, auto terms) {
        hipLaunchKernelGGL((decode_planes_kernel<decltype(tf)::value, decltype(terms)::value>), grid, dim3(256), 0, s, out,
                           w, row0 / 16);
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    using Three = std::integral_constant<int, 3>;
    if (w.tf == TF_F16) go(std::integral_constant<int, TF_F16>{}, Two{});
    else if (w.tf == TF_F32 && out.terms == 2) go(std::integral_constant<int, TF_F32>{}, Two{});
    else if (w.tf == TF_F32) go(std::integral_constant<int, TF_F32>{}, Three{});
    else if (w.tf == TF_Q8 && out.terms == 2) go(std::integral_constant<int, TF_Q8>{}, Two{});
    else if (w.tf == TF_Q8) go(std::integral_constant<int, TF_Q8>{}, Three{});
    else if (!w.fast) hipLaunchKernelGGL(decode_any_kernel, each, dim3(256), 0, s, out, w, row0);
    else if (w.tf == TF_FP8) go(std::integral_constant<int, TF_FP8>{}, One{});
    else if (w.tf == TF_MX4) go(std::integral_constant<int, TF_MX4>{}, One{});
    else go(std::integral_constant<int, TF_INT4>{}, One{});
    DITCH_TRY_HIP(hipGetLastError());
    return out;
}

__device__ __forceinline__ void put_row_value(void *out, int32_t dtype, int64_t i, float v) {
    if (dtype == DITCH_F32) ((float *)out)[i] = v;
    else if (dtype == DITCH_F16) ((_Float16 *)out)[i] = (_Float16)v;
    else ((__bf16 *)out)[i] = (__bf16)v;
}

__global__ __launch_bounds__(256) void join_parts_kernel(void *out, int32_t dtype, int64_t stride, const float *part,
                                                         int parts, int64_t part_stride, int64_t ld, int64_t n,
                                                         int64_t cols, MoreParts more) {
    const int64_t per = (cols + 3) / 4, i = rows_block() * 256 + threadIdx.x;
    if (i >= n * per) return;
    const int64_t row = i / per, c = i % per * 4;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int p = 0; p < parts; p++) {
        const float4 v = *(const float4 *)(part + p * part_stride + row * ld + c);
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    if (more.times) {
        const float times = more.times[row];
        float4 m = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int p = 0; p < more.parts; p++) {
            const float4 v = *(const float4 *)(more.part + p * part_stride + row * ld + c);
            m.x += v.x, m.y += v.y, m.z += v.z, m.w += v.w;
        }
        sum.x += times * m.x, sum.y += times * m.y, sum.z += times * m.z, sum.w += times * m.w;
    }
    const float v[4] = {sum.x, sum.y, sum.z, sum.w};
    for (int j = 0; j < 4; j++)
        if (c + j < cols) put_row_value(out, dtype, row * stride + c + j, v[j]);
}

void launch_join_parts(void *out, int32_t dtype, int64_t stride, const float *part, int parts, int64_t part_stride,
                       int64_t ld, int64_t n, int64_t cols, hipStream_t s, MoreParts more) {
    const int64_t total = n * ceil_div(cols, 4);
    hipLaunchKernelGGL(join_parts_kernel, rows_grid(ceil_div(total, 256), 256), dim3(256), 0, s, out, dtype, stride,
                       part, parts, part_stride, ld, n, cols, more);
    DITCH_TRY_HIP(hipGetLastError());
}

}  // namespace ditch
