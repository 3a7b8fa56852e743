// glu.h — the gated block's epilogue, shared by its products on planes (glu.hip)
// and on coded weights (glu_coded.hip).
#pragma once
#include "rows_coded.h"

namespace ditch {

// act(g) and its derivative; the activations of ditch_hip_gatedActivation. Towards
// the ends of f32, where they have long been flat, 1.702 g and g^2 are held finite:
// infinity times the 0 that is left of the slope would be NaN.
template <int A>
__device__ __forceinline__ void act_both(float g, float &y, float &dy) {
    if constexpr (A == 0 || A == 5) {
        constexpr float c = A == 0 ? 1.f : 1.702f;
        const float s = __fdiv_rn(1.f, 1.f + expf(-c * g));
        y = g * s;
        dy = s * __builtin_fmaf(__builtin_amdgcn_fmed3f(c * g, -1e30f, 1e30f), 1.f - s, 1.f);
    } else if constexpr (A == 1) {
        const float k = 0.7978845608028654f, g2 = fminf(g * g, 1e30f);
        const float t = tanhf(k * __builtin_fmaf(0.044715f * g2, g, g));
        y = 0.5f * g * (1.f + t);
        dy = 0.5f * (1.f + t) + 0.5f * g * (1.f - t * t) * k * __builtin_fmaf(3.f * 0.044715f, g2, 1.f);
    } else if constexpr (A == 2) {
        const float c = 0.5f * (1.f + erff(g * 0.7071067811865476f));
        y = g * c;
        dy = __builtin_fmaf(g * 0.3989422804014327f, expf(-0.5f * g * g), c);
    } else {
        const float r = fmaxf(g, 0.f);
        y = A == 3 ? r : r * r;
        dy = A == 3 ? (g > 0.f ? 1.f : 0.f) : 2.f * r;
        if (g != g) y = dy = g;
    }
}

// Blocks 2i of m are gate rows, 2i + 1 the same up rows.
struct EpiGlu {
    static constexpr bool PAIRS = false;
    static constexpr bool F32_RESULT = false, ALL_PAIRS = false;
    void *out;
    int64_t stride, n, rows;
    int32_t dtype, wide;
    uint32_t act;
    template <int A, int MI, int NJ>
    __device__ __forceinline__ void store(floatx4 (&acc)[MI][NJ], int mb, int nb, int lane) const {
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int64_t tok = (int64_t)(nb + j) * 16 + (lane & 15);
            if (tok >= n) continue;
#pragma unroll
            for (int i = 0; i < MI; i += 2) {
                const int64_t c = (int64_t)(mb + i) / 2 * 16 + 4 * (lane >> 4);
                if (c >= rows) continue;
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float y, dy;
                    act_both<A>(acc[i][j][r], y, dy);
                    v[r] = y * acc[i + 1][j][r];
                }
                put_row4(out, dtype, tok * stride + c, rows - c, wide, v);
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

// dg and du of the block as terms.
template <int T>
struct EpiGluGrad {
    static constexpr bool PAIRS = false;
    static constexpr bool F32_RESULT = false, ALL_PAIRS = false;
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

void launch_glu_coded(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks, const EpiGlu &epi,
                      hipStream_t s);
template <int T>
void launch_glu_grad_coded(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks,
                           const EpiGluGrad<T> &epi, hipStream_t s);

}  // namespace ditch
