// rows_coded_parts.hip — d W for few rows of d on weights that are not planes: like
// rows_coded.h the weight's own words are read once, here contracted over its rows.
//
// A workgroup computes a run of 64 or 128 columns for up to 64 rows of d; its four
// waves share the part's 32-row steps and add their sums at the end. What a wave
// reads is its own, so no barrier stands between a load and its use: the words of
// a step go to registers while the one before is multiplied, their bf16 terms to
// the wave's part of the LDS as units, and the transposing reads (rows_gemm.h)
// take the fragments from there. The LDS takes and gives a wave's accesses in
// their order.
#include "rows_coded.h"

namespace ditch {

template <int TF>
struct CodedCfg {
    static constexpr int OWN = TF == TF_F16 ? 2 : TF == TF_F32 || TF == TF_Q8 ? 3 : 1;
    static constexpr int KT = TF == TF_FP8 || TF == TF_Q8 ? 2 : TF == TF_MX4 || TF == TF_INT4 ? 4 : 1;
    static constexpr int HALVES = TF == TF_F32 ? 2 : 1;
    static constexpr int NS = TF == TF_INT4 ? 2 : TF == TF_F16 || TF == TF_F32 ? 0 : 1;
    static constexpr int UNITS = TF == TF_FP8 || KT == 1 ? 2 : 1;  // of a wave
    static constexpr int TILES = UNITS * KT;                       // 32 columns each
};

template <int TF, int TB, int NJ>
__global__ __launch_bounds__(256) void rows_coded_parts_kernel(CodedParts p, EpiParts epi) {
    using C = CodedCfg<TF>;
    constexpr int TA = TB == 3 || C::OWN < 2 ? C::OWN : 2;  // rows_weight_terms
    constexpr int ORDER = TA > TB ? TA : TB, MB = 2 * C::TILES;
    constexpr int WAVE = C::TILES * 2 * TA * 64;  // 16-byte words of a wave's units
    constexpr int SUMS = MB * NJ * 64;
    __shared__ u32x4 S[4 * WAVE > 2 * SUMS ? 4 * WAVE : 2 * SUMS];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int mt, nt;
    rows_map_tile(blockIdx.x, gridDim.x, p.tiles_m, p.tiles_n, mt, nt);
    const int all = p.steps * p.sets;
    const int first = (int)((int64_t)all * blockIdx.y / p.parts), last = (int)((int64_t)all * (blockIdx.y + 1) / p.parts);
    const int64_t units = p.w[0].units_k;
    int64_t unit[C::UNITS];
#pragma unroll
    for (int u = 0; u < C::UNITS; u++) {
        const int64_t at = (int64_t)mt * C::UNITS + u;
        unit[u] = at < units ? at : units - 1;
    }
    const SideStep st = side_step<TF>(p.w[0]);
    u32x4 *own = S + wave * WAVE;

    struct Step {
        u32x4 c[2][C::UNITS][C::HALVES];
        uint32_t sd[2][C::UNITS][C::NS ? C::NS : 1];
        u32x4 b[TB][NJ];
        bool second;  // the step's second 16 rows are there
    };
    auto load = [&](int t, Step &q) {
        const int set = t >= p.steps, s = set ? t - p.steps : t;
        const TileView &w = p.w[set];
        q.second = 2 * s + 1 < p.blocks;
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int64_t g = p.first + 2 * s + (r && q.second);
            const uint32_t *side = C::NS ? w.side + side_row(w, g, lane) : nullptr;
#pragma unroll
            for (int u = 0; u < C::UNITS; u++) {
                const char *src = (const char *)w.codes + (g * units + unit[u]) * (1024 * C::HALVES);
#pragma unroll
                for (int h = 0; h < C::HALVES; h++) q.c[r][u][h] = *(const u32x4 *)(src + h * 1024 + lane * 16);
#pragma unroll
                for (int k = 0; k < C::NS; k++) q.sd[r][u][k] = *side_word<TF>(st, side, unit[u], k);
            }
        }
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int g = nt * NJ + j < p.d_groups ? nt * NJ + j : p.d_groups - 1;  // (those behind are not stored)
#pragma unroll
            for (int e = 0; e < TB; e++)
                q.b[e][j] = *(const u32x4 *)(p.d[set] + e * p.d_plane + ((int64_t)g * p.d_units + s) * 1024 + lane * 16);
        }
    };
    floatx4 acc[MB][NJ];
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

    auto multiply = [&](const Step &q) {
#pragma unroll
        for (int u = 0; u < C::UNITS; u++)
#pragma unroll
            for (int kt = 0; kt < C::KT; kt++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const u32x4(&c)[C::HALVES] = q.c[r][u];
                    float v[8];
                    if constexpr (TA > 1) {
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            if constexpr (TF == TF_F32) v[j] = u2f(c[(j / 4) % C::HALVES][j % 4]);
                            else if constexpr (TF == TF_F16) v[j] = f16_to_f32_hw((uint16_t)(c[0][j / 2] >> (16 * (j & 1))));
                            else
                                v[j] = __fmul_rn((float)(int8_t)(c[0][(2 * kt + j / 4) % 4] >> (8 * (j % 4))),
                                                 f16_to_f32_hw((uint16_t)(q.sd[r][u][0] >> (16 * (kt & 1)))));
                        }
                    }
#pragma unroll
                    for (int ta = 0; ta < TA; ta++) {
                        u32x4 a;
                        if constexpr (TA > 1) {
                            if (ta + 1 == TA && TA < C::OWN) a = coded_term<true>(v);
                            else a = coded_term<false>(v);
                        } else a = decode_tile_lds<TF>(p.w[0], c, q.sd[r][u], kt, true);
                        // (d is zero there, which an infinity would not leave so)
                        if (r && !q.second) a = u32x4{0, 0, 0, 0};
                        own[((ta * C::TILES + u * C::KT + kt) * 2 + r) * 64 + lane] = a;
                    }
                }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int ta = 0; ta < TA; ta++)
#pragma unroll
            for (int i = 0; i < MB; i++) {
                const u32x4 a = rows_fragment<true>(own + ta * C::TILES * 128, i, lane);
#pragma unroll
                for (int e = 0; e < TB; e++) {
                    if (ta + e >= ORDER) continue;
#pragma unroll
                    for (int j = 0; j < NJ; j++) acc[i][j] = mfma_bf16(a, q.b[e][j], acc[i][j]);
                }
            }
        asm volatile("" ::: "memory");
    };
    int t = first + wave;
    if (t < last) {
        Step one, two;
        load(t, one);
        while (true) {
            if (t + 4 < last) load(t + 4, two);
            multiply(one);
            if ((t += 4) >= last) break;
            if (t + 4 < last) load(t + 4, one);
            multiply(two);
            if ((t += 4) >= last) break;
        }
    }
    // the waves' sums, in the same order always: 0 + 2, 1 + 3, both
    floatx4 *sums = (floatx4 *)S;
    auto give = [&](int slot) {
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int j = 0; j < NJ; j++) sums[slot * SUMS + (i * NJ + j) * 64 + lane] = acc[i][j];
    };
    auto take = [&](int slot) {
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int j = 0; j < NJ; j++) acc[i][j] += sums[slot * SUMS + (i * NJ + j) * 64 + lane];
    };
    __syncthreads();
    if (wave >= 2) give(wave - 2);
    __syncthreads();
    if (wave < 2) take(wave);
    __syncthreads();
    if (wave == 1) give(0);
    __syncthreads();
    if (wave == 0) {
        take(0);
        epi(acc, mt * MB, nt * NJ, lane);
    }
}

// Two workgroups a CU (14336 x 4096 f16 of 1 bf16 row 71 us of loss gradient, one 78,
// four 72), one where its sums are of 128 columns and 64 rows (FP8 of 60 rows: 67, 74,
// 89); steps of 32 rows enough for each wave to make up for its sums' joining.
int coded_parts_count(const TileView &w, int64_t rows, int64_t n, int sets) {
    const bool one = rows_weight_terms(w, 3) == 1;
    const int64_t tiles = ceil_div(w.cols, one ? 128 : 64) * ceil_div(n, 64), steps = ceil_div(rows, 32) * sets;
    const int64_t least = one && n <= 64 ? 8 : 16;
    int64_t parts = ceil_div(one && n > 16 ? 256 : 512, tiles);
    if (parts > steps / least) parts = steps / least;
    return parts < 1 ? 1 : parts > 64 ? 64 : (int)parts;
}

void launch_coded_parts(CodedParts p, int terms, float *part, int64_t ld, int64_t n, bool add, hipStream_t s) {
    const EpiParts epi{part, n * ld, ld, n, p.w[0].cols, add};
    auto go = [&](auto tf, auto tb, auto nj) {
        constexpr int TF = decltype(tf)::value, TB = decltype(tb)::value, NJ = decltype(nj)::value;
        p.tiles_m = (int32_t)ceil_div(p.w[0].cols, 32 * CodedCfg<TF>::TILES);
        p.tiles_n = (int32_t)ceil_div(n, 16 * NJ);
        hipLaunchKernelGGL((rows_coded_parts_kernel<TF, TB, NJ>), dim3((unsigned)(p.tiles_m * p.tiles_n), (unsigned)p.parts),
                           dim3(256), 0, s, p, epi);
    };
    with_terms(terms, [&](auto tb) {
        auto width = [&](auto tf) {
            if (n <= 16) go(tf, tb, std::integral_constant<int, 1>{});
            else go(tf, tb, std::integral_constant<int, 4>{});
        };
        switch (p.w[0].tf) {
        case TF_F16: width(std::integral_constant<int, TF_F16>{}); break;
        case TF_F32: width(std::integral_constant<int, TF_F32>{}); break;
        case TF_Q8: width(std::integral_constant<int, TF_Q8>{}); break;
        case TF_FP8: width(std::integral_constant<int, TF_FP8>{}); break;
        case TF_MX4: width(std::integral_constant<int, TF_MX4>{}); break;
        default: width(std::integral_constant<int, TF_INT4>{}); break;
        }
    });
    DITCH_TRY_HIP(hipGetLastError());
}

}  // namespace ditch
