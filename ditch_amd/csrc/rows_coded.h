// rows_coded.h — rows_gemm.h's product x W^T for few rows, on weights that are not
// planes: their own words go to the LDS and each wave makes the bf16 terms of its
// fragments from them, so that the weight is read once and nothing is written
// (planes of a weight take a pass of their own and 2 bytes a term and value, which
// many rows make up for and few do not).
//
// Tiles of 256 x 64 or 64 x 64. A stage is a unit of the weight, 32 (f16, f32), 64
// (FP8, Q8_0) or 128 columns (MXFP4, INT4), its side words (scales), and as many
// units of every term of x. The ring, the copies and the waits are rows_gemm.h's.
#pragma once
#include "rows_gemm.h"
#include "tile_decode.h"

namespace ditch {

// Whether the kernel takes a weight's format as it stands.
inline bool rows_coded_takes(const TileView &w) {
    return w.tf == TF_F16 || w.tf == TF_F32 ||
           (w.fast && (w.tf == TF_Q8 || w.tf == TF_FP8 || w.tf == TF_MX4 || w.tf == TF_INT4));
}

// Two weights side by side: one decode for both.
inline bool rows_coded_pair(const TileView &a, const TileView &b) {
    return rows_coded_takes(a) && rows_coded_takes(b) && a.scale_type == b.scale_type && a.group == b.group &&
           a.block_cols == b.block_cols;
}

// The tile of such a product, 0 where the weight's planes serve better: where x
// has many 16-row blocks, each of which has the weight decoded again. The planes
// cost the more the wider their words are to the weight's own. Measured over 4864 x
// 896, 14336 x 4096 and 64000 x 2048: f32 weights and 800 f32 rows 52, 543 and 1230 us,
// by planes 65, 692 and 1545, from 1000 rows on alike; f16 and 640 bf16 rows 34, 250 and
// 407, and 43, 232 and 523; MXFP4 and 800 bf16 rows 19, 101 and 208, and 27, 122 and
// 268; FP8 and 300 bf16 rows 18, 99 and 130, and 26, 85 and 196, more rows worse.
// A gradient reads the weight once more, transposed: f32 weights and 512 f32 rows
// 89, 675 and 1535 (107, 868 and 1889); f16 and 300 bf16 rows 37, 263 and 426 (50, 283
// and 635), 400 up to a fifth worse; MXFP4 and 200 bf16 rows 30, 111 and 211 (34, 123
// and 244); FP8 and 128 31, 86 and 156 (31, 94 and 219), 200 worse.
inline int rows_coded_tile(const TileView &w, int64_t mblocks, int64_t nblocks, bool grad) {
    const int most = w.tf == TF_F16 ? (grad ? 24 : 40) : w.tf == TF_FP8 ? (grad ? 8 : 16)
                     : w.tf == TF_F32 || w.tf == TF_Q8 ? (grad ? 32 : 56) : grad ? 16 : 56;
    if (!rows_coded_takes(w) || nblocks > most) return 0;
    return ceil_div(mblocks, 16) * ceil_div(nblocks, 4) < 160 ? 3 : 2;
}

struct RowsCoded {
    TileView w[2];   // paired: row blocks 2i and 2i + 1 of a are block i of the first and of the second
    int32_t paired = 0;
    RowsOperand b;
    const char *x = nullptr;
    int64_t x_plane = 0;
    int32_t blocks = 0;  // 16-row blocks of one weight, from `first` on
    int32_t first = 0;
    int32_t stages = 0;
    int32_t tiles_m = 0, tiles_n = 0;
};

// 4 bytes a lane to the LDS at `to`
__device__ __forceinline__ void rows_copy_words(const uint32_t *src, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(src) : "memory");
}

// The next term of eight values as a fragment's words, and what it leaves: their
// high halves, cut (three of them hold all bits of f32 values, two of f16 ones), or
// rounded to nearest where it is the last and more is left. An infinite or NaN
// value leaves NaN.
template <bool ROUND>
__device__ __forceinline__ u32x4 coded_term(float (&v)[8]) {
    u32x4 w;
    if constexpr (ROUND) {
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = cvt_pk_bf16(v[2 * j], v[2 * j + 1]);
        return w;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = pack_hi(v[2 * j], v[2 * j + 1]);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = __fsub_rn(v[j], u2f(f2u(v[j]) & 0xffff0000u));
    return w;
}

template <int WGM, int WGN, int MI, int NJ, int TF, int TB, typename Epi>
__global__ __launch_bounds__(WGM * WGN * 64) void rows_coded_kernel(RowsCoded p, Epi epi) {
    constexpr int OWN = TF == TF_F16 ? 2 : TF == TF_F32 || TF == TF_Q8 ? 3 : 1;
    constexpr int TA = TB == 3 || OWN < 2 || Epi::F32_RESULT ? OWN : 2;  // rows_weight_terms
    constexpr int KT = TF == TF_FP8 || TF == TF_Q8 ? 2 : TF == TF_MX4 || TF == TF_INT4 ? 4 : 1;
    constexpr int HALVES = TF == TF_F32 ? 2 : 1;
    constexpr int NS = TF == TF_INT4 ? 2 : TF == TF_F16 || TF == TF_F32 ? 0 : 1;
    constexpr int ORDER = rows_order_of(TA, TB, Epi::ALL_PAIRS);
    constexpr int WAVES = WGM * WGN, UA = WGM * MI, UB = WGN * NJ;
    constexpr int NA = UA * HALVES, PA = NA / WAVES, NBP = UB * KT;
    constexpr bool HALF = NBP * 2 == WAVES;
    constexpr int PB = HALF ? 1 : NBP / WAVES;
    static_assert(NA % WAVES == 0 && (HALF || NBP % WAVES == 0) && UA % 4 == 0, "copies split evenly");
    constexpr int SIDE = UA / 4 * NS;  // copies of 64 side words
    static_assert(SIDE <= WAVES, "a side copy a wave");
    constexpr int STAGE = NA + TB * NBP;                   // KB
    constexpr int WORDS = STAGE * 64 + SIDE * 16;           // 16-byte words
    constexpr int FIT = (WORDS * 16 * 2 <= 81920 ? 81920 : 159744) / (WORDS * 16);
    constexpr int NB = FIT > 4 ? 4 : FIT;
    static_assert(NB >= 2, "two stages");
    __shared__ u32x4 S0[WORDS], S1[WORDS], S2[NB > 2 ? WORDS : 1], S3[NB > 3 ? WORDS : 1];

    const int lane = threadIdx.x & 63;
    const uint32_t lane16 = lane * 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WGN, wn = wave % WGN;
    int mt, nt;
    if (!rows_tile_of_block(p.tiles_m, p.tiles_n, mt, nt)) return;

    const int64_t units = p.w[0].units_k;
    auto group = [&](int block, int &which) {
        int g = mt * UA + block;
        which = 0;
        if (p.paired) {
            which = g & 1;
            g >>= 1;
        }
        return p.first + (g < p.blocks ? g : p.blocks - 1);
    };
    // this wave's copies: of the weight's units, of its side words, of x
    const char *pa[PA];
#pragma unroll
    for (int j = 0; j < PA; j++) {
        const int q = wave * PA + j;
        int which;
        const int64_t g = group(q / HALVES, which);
        pa[j] = (const char *)p.w[which].codes + g * units * (1024 * HALVES) + q % HALVES * 1024;
    }
    const uint32_t *side = nullptr;
    int entry = 0;
    SideStep st{};
    if (NS > 0 && wave < SIDE) {
        int which;
        entry = wave % (NS ? NS : 1);
        const int64_t g = group(wave / (NS ? NS : 1) * 4 + (lane >> 4), which);
        const TileView &w = p.w[which];
        side = w.side + side_row(w, g, lane);
        st = side_step<TF>(p.w[0]);
    }
    const bool copies_b = !HALF || wave < NBP;
    int64_t ob[PB];
    int kb[PB];
#pragma unroll
    for (int j = 0; j < PB; j++) {
        const int q = (copies_b ? wave : 0) * PB + j;
        int g = nt * UB + q / KT, second = 0;
        if (p.b.paired) {
            second = g & 1;
            g >>= 1;
        }
        g = g < p.b.blocks ? g : p.b.blocks - 1;
        ob[j] = (int64_t)g * p.b.ldu * 1024 + (second ? p.b.pair : 0);
        kb[j] = q % KT;
    }
    const uint32_t lane_b = TB == 1 ? p.b.lane_at(lane) : lane16;
    int next = 0;
    const int stages = p.stages;
    auto copy = [&](u32x4 *S) {
        if (next >= stages) return;
        const uint32_t to = rows_lds_at(S);
#pragma unroll
        for (int j = 0; j < PA; j++)
            rows_copy_unit(pa[j] + (int64_t)next * (1024 * HALVES), lane16, to + (wave * PA + j) * 1024);
        if constexpr (NS > 0) {
            if (wave < SIDE) rows_copy_words(side_word<TF>(st, side, next, entry), to + STAGE * 1024 + wave * 256);
        }
        if (copies_b) {
#pragma unroll
            for (int e = 0; e < TB; e++)
#pragma unroll
                for (int j = 0; j < PB; j++) {
                    const int k = next * KT + kb[j] < p.b.ks ? next * KT + kb[j] : p.b.ks - 1;
                    rows_copy_unit(p.x + ob[j] + e * p.x_plane + (int64_t)k * p.b.unit, lane_b,
                                   to + (NA + e * NBP + wave * PB + j) * 1024);
                }
        }
        next++;
    };
    floatx4 acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

    // f32 rows' sums in two levels, as in rows_gemm.h
    constexpr bool LEVELS = TB == 3;
    floatx4 whole[LEVELS ? MI : 1][LEVELS ? NJ : 1];
#pragma unroll
    for (int i = 0; i < (LEVELS ? MI : 1); i++)
#pragma unroll
        for (int j = 0; j < (LEVELS ? NJ : 1); j++) whole[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    auto lift = [&] {
        if constexpr (LEVELS) {
#pragma unroll
            for (int i = 0; i < MI; i++)
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    whole[i][j] += acc[i][j];
                    acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
                }
        }
    };
    int rounds = 0;

    constexpr int FLIGHT = PA + (HALF ? 0 : TB * PB);  // copies of a stage that every wave makes at least
    // stage t from its buffer; the stage NB - 1 ahead copied to the buffer of the one before
    auto step = [&](int t, const u32x4 *S, u32x4 *before) {
        __builtin_amdgcn_sched_barrier(0);
        if (t + NB - 1 > stages || NB == 2) __builtin_amdgcn_s_waitcnt(rows_vmcnt(0) & ~0x0f00);
        else __builtin_amdgcn_s_waitcnt(rows_vmcnt((NB - 2) * FLIGHT) & ~0x0f00);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        copy(before);
        __builtin_amdgcn_sched_barrier(0);
        u32x4 c[MI][HALVES];
        uint32_t sd[MI][NS ? NS : 1];
#pragma unroll
        for (int i = 0; i < MI; i++) {
            const int block = wm * MI + i;
#pragma unroll
            for (int h = 0; h < HALVES; h++) c[i][h] = S[(block * HALVES + h) * 64 + lane];
#pragma unroll
            for (int s = 0; s < NS; s++)
                sd[i][s] = ((const uint32_t *)(S + STAGE * 64))[(block / 4 * NS + s) * 64 + block % 4 * 16 + (lane & 15)];
        }
#pragma unroll
        for (int kt = 0; kt < KT; kt++) {
            float v[TA > 1 ? MI : 1][8];
            if constexpr (TA > 1) {
#pragma unroll
                for (int i = 0; i < MI; i++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        if constexpr (TF == TF_F32) v[i][j] = u2f(c[i][(j / 4) % HALVES][j % 4]);
                        else if constexpr (TF == TF_F16) v[i][j] = f16_to_f32_hw((uint16_t)(c[i][0][j / 2] >> (16 * (j & 1))));
                        else
                            v[i][j] = __fmul_rn((float)(int8_t)(c[i][0][(2 * kt + j / 4) % 4] >> (8 * (j % 4))),
                                                f16_to_f32_hw((uint16_t)(sd[i][0] >> (16 * (kt & 1)))));
                    }
            }
#pragma unroll
            for (int ta = 0; ta < TA; ta++) {
                u32x4 a[MI];
#pragma unroll
                for (int i = 0; i < MI; i++) {
                    if constexpr (TA > 1) {
                        if (ta + 1 == TA && TA < OWN) a[i] = coded_term<true>(v[TA > 1 ? i : 0]);
                        else a[i] = coded_term<false>(v[TA > 1 ? i : 0]);
                    } else a[i] = decode_tile_lds<TF>(p.w[0], c[i], sd[i], kt, true);
                }
#pragma unroll
                for (int e = 0; e < TB; e++) {
                    if (ta + e >= ORDER) continue;
                    u32x4 b[NJ];
#pragma unroll
                    for (int j = 0; j < NJ; j++) b[j] = S[(NA + e * NBP + (wn * NJ + j) * KT + kt) * 64 + lane];
#pragma unroll
                    for (int i = 0; i < MI; i++)
#pragma unroll
                        for (int j = 0; j < NJ; j++) acc[i][j] = mfma_bf16(a[i], b[j], acc[i][j]);
                }
            }
        }
    };
    copy(S0);
    if (NB > 2) copy(S1);
    if (NB > 3) copy(S2);
    for (int t = 0; t < stages; t += NB) {
        if constexpr (NB == 2) {
            step(t, S0, S1);
            if (t + 1 < stages) step(t + 1, S1, S0);
        } else if constexpr (NB == 3) {
            step(t, S0, S2);
            if (t + 1 < stages) step(t + 1, S1, S0);
            if (t + 2 < stages) step(t + 2, S2, S1);
        } else {
            step(t, S0, S3);
            if (t + 1 < stages) step(t + 1, S1, S0);
            if (t + 2 < stages) step(t + 2, S2, S1);
            if (t + 3 < stages) step(t + 3, S3, S2);
        }
        if (LEVELS && (KT > 1 || (++rounds & 1) == 0)) lift();
    }
    lift();
    if constexpr (LEVELS) epi(whole, mt * UA + wm * MI, nt * UB + wn * NJ, lane);
    else epi(acc, mt * UA + wm * MI, nt * UB + wn * NJ, lane);
}

template <int WGM, int WGN, int MI, int NJ, int TF, int TB, typename Epi>
void launch_rows_coded_tile(RowsCoded p, int64_t mblocks, int64_t nblocks, const Epi &epi, hipStream_t s) {
    const int64_t tm = ceil_div(mblocks, WGM * MI), tn = ceil_div(nblocks, WGN * NJ);
    DITCH_CHECK(tm * tn < (int64_t)1 << 31, DITCH_INVALID_ARGUMENT, "rows product: more tiles than one launch holds");
    p.tiles_m = (int32_t)tm;
    p.tiles_n = (int32_t)tn;
    hipLaunchKernelGGL((rows_coded_kernel<WGM, WGN, MI, NJ, TF, TB, Epi>), rows_grid(tm * tn, WGM * WGN * 64),
                       dim3(WGM * WGN * 64), 0, s, p, epi);
    DITCH_TRY_HIP(hipGetLastError());
}

// tile: 2 (256 x 64) or 3 (64 x 64), rows_gemm.h's numbers
template <int TB, typename Epi>
void launch_rows_coded(int tile, const RowsCoded &p, int64_t mblocks, int64_t nblocks, const Epi &epi, hipStream_t s) {
    auto go = [&](auto tf) {
        constexpr int TF = decltype(tf)::value;
        if (tile == 3) launch_rows_coded_tile<2, 2, 2, 2, TF, TB>(p, mblocks, nblocks, epi, s);
        else launch_rows_coded_tile<4, 2, 4, 2, TF, TB>(p, mblocks, nblocks, epi, s);
    };
    switch (p.w[0].tf) {
    case TF_F16: go(std::integral_constant<int, TF_F16>{}); break;
    case TF_F32: go(std::integral_constant<int, TF_F32>{}); break;
    case TF_Q8: go(std::integral_constant<int, TF_Q8>{}); break;
    case TF_FP8: go(std::integral_constant<int, TF_FP8>{}); break;
    case TF_MX4: go(std::integral_constant<int, TF_MX4>{}); break;
    default: go(std::integral_constant<int, TF_INT4>{}); break;
    }
}

// A gradient's epilogue, which leaves T terms: those of x, or two of one (grad_term_count).
template <int T, typename Epi>
void launch_rows_coded_grad(int tile, const RowsCoded &p, int terms, int64_t mblocks, int64_t nblocks, const Epi &epi,
                            hipStream_t s) {
    if constexpr (T == 2) {
        if (terms == 1) {
            launch_rows_coded<1>(tile, p, mblocks, nblocks, epi, s);
            return;
        }
    }
    launch_rows_coded<T>(tile, p, mblocks, nblocks, epi, s);
}

// rows_coded_parts.hip: d W of weights that are not planes, as parts of sums
// [part][n][ld]; d inner planes, of each weight.
struct CodedParts {
    TileView w[2];
    const char *d[2] = {nullptr, nullptr};
    int64_t d_units = 0, d_plane = 0;
    int32_t d_groups = 0;
    int32_t first = 0, blocks = 0;  // the weights' 16-row groups
    int32_t steps = 0, sets = 1;    // of 32 rows; weights
    int32_t parts = 1;
    int32_t tiles_m = 0, tiles_n = 0;
};
int coded_parts_count(const TileView &w, int64_t rows, int64_t n, int sets);
void launch_coded_parts(CodedParts p, int terms, float *part, int64_t ld, int64_t n, bool add, hipStream_t s);

}  // namespace ditch
