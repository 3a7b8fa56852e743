// rows_gemm.h — the product over planes of bf16 terms (rows.h) and what is done
// with its tiles. Included by the operators that instantiate it.
//
// c[m][n] = sum over the pairs of terms and k of a[m][k] b[n][k]. Each operand
// is inner (its columns are k) or outer (its rows are k). A workgroup computes
// BM x BN; a stage is one term of a and all TB terms of b over 32 k: whole units are
// copied global -> LDS into a ring of buffers, some stages ahead. (A fragment of a
// then serves every term of b: with a stage a pair, f32 rows read a three times
// and the LDS was what they waited for.) Fragments are read while the ones
// before them are multiplied, across stages too.
// Fragments of inner operands are one 16-byte LDS read a lane, those of outer ones
// two transposing reads (ds_read_b64_tr_b16: lane t of 16 gets column t of four
// 16-column rows whose quarters the 16 lanes address).
// v_mfma_f32_16x16x32_bf16 leaves lane l with c[4 (l / 16) + r][l % 16], r =
// 0..3: four neighbours along m, one n. Every use has what must be contiguous
// in memory along m.
//
// Stages past an operand's end read its last unit again: the other operand's
// planes hold zeros there. Tiles past an operand's end repeat its last rows and
// are not stored.
#pragma once
#include <type_traits>

#include "rows.h"

namespace ditch {

typedef __attribute__((address_space(3))) void rows_lds_void;
typedef short rows_short4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) rows_short4 rows_lds_short4;

struct RowsOperand {
    int64_t ldu = 0;      // units of a 16-row group
    int64_t pair = 0;     // interleaved: bytes from the first planes to the second's
    int32_t blocks = 0;   // along the output: 16-row groups (inner), 32-column units (outer); of one of a pair
    int32_t ks = 0;       // along k: units (inner), groups (outer)
    int32_t paired = 0;   // blocks (units) 2i and 2i + 1 are block i of the first and of the second planes
    // up to 16 bf16 rows as the caller has them (rows_in): bytes from a 16 x 32
    // unit to the next, from a row to the next (0: units of planes), rows
    int32_t unit = 1024;
    uint32_t row_bytes = 0;
    int32_t rows = 0;
    // where a lane's 16 bytes of a unit are: row lane % 16, 8 columns at 8 (lane / 16)
    __device__ __forceinline__ uint32_t lane_at(int lane) const {
        if (!row_bytes) return lane * 16;
        const int row = (lane & 15) < rows ? lane & 15 : rows - 1;
        return row * row_bytes + (lane >> 4) * 16;
    }
};

struct RowsGemm {
    RowsOperand a, b;
    // a term of a and the first count of b's that it meets
    const char *sa[2 * ROWS_MAX_TERMS], *sb[2 * ROWS_MAX_TERMS];
    int32_t count[2 * ROWS_MAX_TERMS];
    int64_t b_plane = 0;  // bytes from one of b's planes to the next
    int32_t terms = 1;    // of b
    int32_t nseg = 0;
    int32_t k32 = 0;      // 32 k each
    int32_t parts = 1;    // the stages are split over blockIdx.y
    int32_t tiles_m = 0, tiles_n = 0;
};

// The pairs of terms i + j < order of two operands' planes.
inline void rows_pairs(RowsGemm &g, const Planes &a, const Planes &b, int order) {
    for (int i = 0; i < a.terms && i < order; i++) {
        g.sa[g.nseg] = a.p + i * a.plane_bytes();
        g.sb[g.nseg] = b.p;
        g.count[g.nseg++] = order - i < b.terms ? order - i : b.terms;
    }
    g.b_plane = b.plane_bytes();
    g.terms = b.terms;
}
inline RowsOperand rows_inner(const Planes &p) {
    RowsOperand o;
    o.ldu = p.units;
    o.blocks = (int32_t)p.groups;
    o.ks = (int32_t)p.units;
    return o;
}
inline RowsOperand rows_outer(const Planes &p) {
    RowsOperand o;
    o.ldu = p.units;
    o.blocks = (int32_t)p.units;
    o.ks = (int32_t)p.groups;
    return o;
}

// The rows of x (and second ones beside them) as the operand of x W^T.
struct RowsIn {
    Planes x;  // its terms; p: the first plane, or the caller's rows
    RowsOperand op;
};
// Packed to `planes`, unless they need no planes: up to 16 bf16 rows, of whose
// units each lane copies 16 bytes of its row, where the rows are aligned and
// whole units of any weight (128 columns). A pass and a launch less: the block of 4864
// x 896 and 1 row 8.0 us by tiles, packed 10.7.
inline RowsIn rows_in(int32_t dtype, int64_t n, int64_t cols, RowsArg x, const RowsArg *second, const Planes *planes,
                      hipStream_t s, const int32_t *live = nullptr) {
    RowsIn in{planes[0], rows_inner(planes[0])};
    in.op.paired = second ? 1 : 0;
    const bool direct = dtype == DITCH_BF16 && n <= 16 && cols % 128 == 0 && (uintptr_t)x.p % 16 == 0 &&
                        x.stride % 8 == 0 && x.stride < (int64_t)1 << 26 &&
                        (!second || ((uintptr_t)second->p % 16 == 0 && second->stride == x.stride));
    if (!direct) {
        launch_pack_rows(planes[0], x.p, dtype, n, cols, x.stride, s, live);
        if (second) {
            launch_pack_rows(planes[1], second->p, dtype, n, cols, second->stride, s);
            in.op.pair = planes[1].p - planes[0].p;
        }
        return in;
    }
    in.x.p = (char *)x.p;
    if (second) in.op.pair = (char *)second->p - (char *)x.p;
    in.op.blocks = 1;
    in.op.ks = (int32_t)(cols / 32);
    in.op.unit = 64;
    in.op.row_bytes = (uint32_t)x.stride * 2;
    in.op.rows = (int32_t)n;
    return in;
}

// Workgroups an XCD runs at one time (every eighth block) cover a patch of
// 8 tiles of m and a few of n, so that they share operands in its L2.
__device__ __forceinline__ void rows_map_tile(int g, int total, int tm, int tn, int &mt, int &nt) {
    const int xcd = g & 7, j = g >> 3, per = total >> 3, rem = total & 7;
    const int t = (xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per) + j;
    constexpr int GM = 8;
    const int width = GM * tn, grp = t / width, first = grp * GM;
    const int gs = tm - first < GM ? tm - first : GM, r = t - grp * width;
    mt = first + r % gs;
    nt = r / gs;
}

// This workgroup's tile, if it has one.
__device__ __forceinline__ bool rows_tile_of_block(int tm, int tn, int &mt, int &nt) {
    const int64_t block = rows_block();
    if (block >= tm * tn) return false;
    rows_map_tile((int)block, tm * tn, tm, tn, mt, nt);
    return true;
}

template <bool OUTER>
__device__ __forceinline__ u32x4 rows_fragment(const u32x4 *S, int block, int lane) {
    if constexpr (!OUTER) {
        return S[block * 64 + lane];
    } else {
        // k 8 g .. +8 of the step for lane group g: unit g / 2, rows 8 (g % 2) .. +8, four a read
        const int t = lane & 15, g = lane >> 4;
        const char *p = (const char *)S + (g >> 1) * 1024 + (8 * (g & 1) + (t >> 2) + 16 * ((t & 3) >> 1)) * 16 +
                        (t & 1) * 8;
        p += (block >> 1) * 2048 + (block & 1) * 512;
        const rows_short4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((rows_lds_short4 *)p);
        const rows_short4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((rows_lds_short4 *)(p + 64));
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        const u32x2 l = __builtin_bit_cast(u32x2, lo), h = __builtin_bit_cast(u32x2, hi);
        return u32x4{l[0], l[1], h[0], h[1]};
    }
}

// 1 KiB of `src` (16 bytes a lane at lane16) to the LDS at `to`. As an instruction
// of its own text: the compiler makes the transposing LDS reads wait for every
// copy in flight, whichever buffer it fills. It writes no register; the kernel
// below waits for it (rows_vmcnt). M0 needs a wait state before its use; nothing
// else in these kernels uses it.
__device__ __forceinline__ void rows_copy_unit(const char *src, uint32_t lane16, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(lane16), "s"(src)
                 : "memory");
}
__device__ __forceinline__ uint32_t rows_lds_at(const u32x4 *p) { return (uint32_t)(uintptr_t)(rows_lds_void *)p; }

// A wave's copies of one operand's planes: PER units of each of TERMS planes. Of
// an inner operand a stage is a unit of each 16-row block, of an outer one two
// 16-row groups of each 32-column unit.
template <bool OUTER, int PER, int TERMS>
struct RowsCopies {
    int64_t off[PER];      // where each begins
    int64_t step, plane;   // bytes from a unit along k to the next, from a plane to the next
    int32_t ks;
    int odd;               // outer, one unit a wave: which of the two groups
    __device__ __forceinline__ RowsCopies(const RowsOperand &o, int wave, int first, int64_t plane_bytes) {
        step = OUTER ? o.ldu * 1024 : o.unit;
        plane = plane_bytes;
        ks = o.ks;
        odd = OUTER && PER == 1 ? wave & 1 : 0;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int l = wave * PER + j;
            if (OUTER) {
                int u = first / 2 + l / 2, second = 0;
                if (o.paired) {
                    second = u & 1;
                    u >>= 1;
                }
                u = u < o.blocks ? u : o.blocks - 1;
                off[j] = (int64_t)u * 1024 + (second ? o.pair : 0);
            } else {
                int g = first + l, second = 0;
                if (o.paired) {
                    second = g & 1;
                    g >>= 1;
                }
                g = g < o.blocks ? g : o.blocks - 1;
                off[j] = (int64_t)g * o.ldu * 1024 + (second ? o.pair : 0);
            }
        }
    }
    // stage cs of the planes at `base` to S, this wave's first unit at unit wave * PER of every plane of `units`
    __device__ __forceinline__ void copy(const char *base, int cs, uint32_t S, int wave, int units, uint32_t lane16) const {
        static_assert(!OUTER || PER == 1 || PER % 2 == 0, "whole pairs of groups, or one unit");
        const int k0 = OUTER ? 2 * cs + odd : cs;
        const int64_t at0 = (k0 < ks ? k0 : ks - 1) * step;
        const int64_t at1 = OUTER ? (k0 + 1 < ks ? k0 + 1 : ks - 1) * step : 0;
#pragma unroll
        for (int e = 0; e < TERMS; e++)
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const char *src = base + (off[j] + (OUTER && (j & 1) ? at1 : at0) + e * plane);
                rows_copy_unit(src, lane16, S + (e * units + wave * PER + j) * 1024);
            }
    }
};

// s_waitcnt's operand for at most n vector memory operations in flight
constexpr int rows_vmcnt(int n) { return (n & 15) | (n >> 4) << 14 | 0x0f70; }

// The order of a region's instructions: after each product a read, or two, while there are any.
template <int PRODUCTS, int READS>
__device__ __forceinline__ void rows_order() {
    constexpr int EACH = (READS + PRODUCTS - 1) / PRODUCTS;
#pragma unroll
    for (int i = 0; i < PRODUCTS; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (i * EACH < READS) __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);
    }
}

// WGM x WGN waves of MI x NJ blocks of 16 x 16; WHOLE: one workgroup a CU.
template <int WGM, int WGN, int MI, int NJ, bool WHOLE, bool AO, bool BO, int TB, typename Epi>
__global__ __launch_bounds__(WGM * WGN * 64) void rows_gemm_kernel(RowsGemm p, Epi epi) {
    constexpr int WAVES = WGM * WGN, UA = WGM * MI, UB = WGN * NJ;  // tile in 16-row blocks: units of a stage
    static_assert(UA % 2 == 0 && UB % 2 == 0, "whole 32-column units");
    static_assert(UA % WAVES == 0 && (UB % WAVES == 0 || UB * 2 == WAVES), "copies split evenly");
    constexpr bool HALF = UB * 2 == WAVES;  // every other wave copies of b
    constexpr int PA = UA / WAVES, PB = HALF ? 1 : UB / WAVES;
    constexpr int STAGE = UA + TB * UB;  // units
    // a ring within half of the 160 KB of LDS (two workgroups a CU), or within all of it
    constexpr int ROOM = WHOLE ? 156 : 80, FIT = ROOM / STAGE;
    constexpr int NB = FIT > 4 ? 4 : FIT < 2 ? 2 : FIT;
    // distinct objects: the compiler sees that the copies into one do not touch what is read from the others
    __shared__ u32x4 S0[STAGE * 64], S1[STAGE * 64], S2[NB > 2 ? STAGE * 64 : 1], S3[NB > 3 ? STAGE * 64 : 1];

    const int lane = threadIdx.x & 63;
    const uint32_t lane16 = lane * 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WGN, wn = wave % WGN;
    int mt, nt;
    if (!rows_tile_of_block(p.tiles_m, p.tiles_n, mt, nt)) return;
    const bool copies_b = !HALF || wave < UB;
    const RowsCopies<AO, PA, 1> ca(p.a, wave, mt * UA, 0);
    const RowsCopies<BO, PB, TB> cb(p.b, copies_b ? wave : 0, nt * UB, p.b_plane);
    const uint32_t lane_b = TB == 1 && !BO ? p.b.lane_at(lane) : lane16;

    // a linear stage is (32 k, term of a): the terms of a step follow each
    // other, so that what they share is read from near
    const int nseg = p.nseg;
    const int first_t = (int)((int64_t)p.k32 * blockIdx.y / p.parts) * nseg;
    const int last_t = (int)((int64_t)p.k32 * (blockIdx.y + 1) / p.parts) * nseg;
    int cs = first_t / nseg, seg = 0, cur = 0;  // of the next copy; of the product
    const char *ba = p.sa[0], *bb = p.sb[0];
    int copied = first_t;
    auto copy = [&](u32x4 *S) {
        if (copied >= last_t) return;
        copied++;
        const uint32_t to = rows_lds_at(S);
        ca.copy(ba, cs, to, wave, UA, lane16);
        if (copies_b) cb.copy(bb, cs, to + UA * 1024, wave, UB, lane_b);
        if (nseg == 1) cs++;
        else {
            if (++seg == nseg) {
                seg = 0;
                cs++;
            }
            ba = p.sa[seg];
            bb = p.sb[seg];
        }
    };
    floatx4 acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    // f32 rows' logits in two levels: a sum of some stages from zero, then one
    // rounding of the whole. A logit of 10 over 896 k, 84 roundings of which each is
    // of the size of the sum, is off by 3e-6 in one level (over 4096 k by 6e-6): more
    // than the gradient of a divergence between near rows can have.
    constexpr bool LEVELS = TB == 3 && !AO && !BO;
    static_assert(!LEVELS || MI * NJ < 32, "no room for two sums in the largest tile");
    floatx4 whole[LEVELS ? MI : 1][LEVELS ? NJ : 1];
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
    if constexpr (LEVELS) {
#pragma unroll
        for (int i = 0; i < MI; i++)
#pragma unroll
            for (int j = 0; j < NJ; j++) whole[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    int rounds = 0;

    // the next stage's fragments in registers, where they fit beside the sums (the
    // largest tile holds 128 of these, and with several terms more fragments)
    constexpr bool AHEAD = TB == 1 || MI * NJ < 32;
    constexpr int FLIGHT = PA + (HALF ? 0 : TB * PB);  // copies of a stage that every wave makes at least
    u32x4 fa[AHEAD ? 2 : 1][MI], fb[2][NJ];
    auto read_a = [&](const u32x4 *S, u32x4 (&a)[MI]) {
#pragma unroll
        for (int i = 0; i < MI; i++) a[i] = rows_fragment<AO>(S, wm * MI + i, lane);
    };
    auto read_b = [&](const u32x4 *S, int e, u32x4 (&b)[NJ]) {
#pragma unroll
        for (int j = 0; j < NJ; j++) b[j] = rows_fragment<BO>(S + (UA + e * UB) * 64, wn * NJ + j, lane);
    };
    auto products = [&](const u32x4 (&a)[MI], const u32x4 (&b)[NJ]) {
#pragma unroll
        for (int i = 0; i < MI; i++)
#pragma unroll
            for (int j = 0; j < NJ; j++) acc[i][j] = mfma_bf16(a[i], b[j], acc[i][j]);
    };
    // every wave's copies but those of the last `later` stages have landed, and
    // every wave has the fragments that it asked for
    auto meet = [&](bool all) {
        __builtin_amdgcn_sched_barrier(0);
        constexpr int later = NB - 2;
        if (all || later == 0) __builtin_amdgcn_s_waitcnt(rows_vmcnt(0) & ~0x0f00);  // and lgkmcnt(0)
        else __builtin_amdgcn_s_waitcnt(rows_vmcnt(later * FLIGHT) & ~0x0f00);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    constexpr int READS_A = (AO ? 2 : 1) * MI, READS_B = (BO ? 2 : 1) * NJ;
    if constexpr (AHEAD) {
        // stage t, its fragments of a and of b's first term in set t % 2: each
        // further term of b is read while the one before is multiplied, and with the
        // last product the next stage's first fragments, from its buffer, while the
        // stage NB ahead is copied to this one's.
        auto last = [&](int t, u32x4 *S, const u32x4 *N, const u32x4 (&a)[MI], const u32x4 (&b)[NJ], u32x4 (&an)[MI],
                        u32x4 (&bn)[NJ]) {
            meet(t + NB > last_t);
            copy(S);
            __builtin_amdgcn_sched_barrier(0);
            read_a(N, an);  // (behind the last stage: whatever lies there, not used)
            read_b(N, 0, bn);
            products(a, b);
            rows_order<MI * NJ, READS_A + READS_B>();
        };
        auto step = [&](int t, u32x4 *S, const u32x4 *N, auto set) {
            constexpr int c = decltype(set)::value;
            if constexpr (TB == 1) {
                last(t, S, N, fa[c], fb[c], fa[c ^ 1], fb[c ^ 1]);
            } else {
                const int count = p.count[cur];
                cur = cur + 1 == nseg ? 0 : cur + 1;
                if (count > 1) {
                    u32x4 more[NJ];
                    __builtin_amdgcn_sched_barrier(0);
                    read_b(S, 1, more);
                    products(fa[c], fb[c]);
                    rows_order<MI * NJ, READS_B>();
                    __builtin_amdgcn_sched_barrier(0);
                    if (TB == 3 && count == 3) {
                        read_b(S, TB - 1, fb[c]);
                        products(fa[c], more);
                        rows_order<MI * NJ, READS_B>();
                        __builtin_amdgcn_sched_barrier(0);
                    } else {
#pragma unroll
                        for (int j = 0; j < NJ; j++) fb[c][j] = more[j];
                    }
                }
                last(t, S, N, fa[c], fb[c], fa[c ^ 1], fb[c ^ 1]);
            }
        };
        if (first_t < last_t) {
            copy(S0);
            copy(S1);
            if (NB > 2) copy(S2);
            if (NB > 3) copy(S3);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(rows_vmcnt(0));
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            read_a(S0, fa[0]);
            read_b(S0, 0, fb[0]);
            using Zero = std::integral_constant<int, 0>;
            using One = std::integral_constant<int, 1>;
            for (int t = first_t; t < last_t; t += NB == 3 ? 6 : NB) {
                if constexpr (NB == 2) {
                    step(t, S0, S1, Zero{});
                    if (t + 1 < last_t) step(t + 1, S1, S0, One{});
                } else if constexpr (NB == 3) {
                    step(t, S0, S1, Zero{});
                    if (t + 1 < last_t) step(t + 1, S1, S2, One{});
                    if (t + 2 < last_t) step(t + 2, S2, S0, Zero{});
                    if (t + 3 < last_t) step(t + 3, S0, S1, One{});
                    if (t + 4 < last_t) step(t + 4, S1, S2, Zero{});
                    if (t + 5 < last_t) step(t + 5, S2, S0, One{});
                } else {
                    step(t, S0, S1, Zero{});
                    if (t + 1 < last_t) step(t + 1, S1, S2, One{});
                    if (t + 2 < last_t) step(t + 2, S2, S3, Zero{});
                    if (t + 3 < last_t) step(t + 3, S3, S0, One{});
                }
                if (LEVELS && (++rounds & (NB == 2 ? 3 : 1)) == 0) lift();
            }
        }
    } else {
        // stage t from its buffer, a further term of b read while the one before
        // is multiplied; the stage NB - 1 ahead copied to the buffer of the one before
        auto step = [&](int t, const u32x4 *S, u32x4 *before) {
            meet(t + NB - 1 > last_t);
            copy(before);
            const int count = p.count[cur];
            cur = cur + 1 == nseg ? 0 : cur + 1;
            __builtin_amdgcn_sched_barrier(0);
            read_b(S, 0, fb[0]);
            read_a(S, fa[0]);
            read_b(S, 1, fb[1]);
            products(fa[0], fb[0]);
            if (count > 1) {
                __builtin_amdgcn_sched_barrier(0);
                if (TB == 3) read_b(S, TB - 1, fb[0]);
                products(fa[0], fb[1]);
                rows_order<MI * NJ, TB == 3 ? READS_B : 0>();
                __builtin_amdgcn_sched_barrier(0);
            }
            if (TB == 3 && count == 3) products(fa[0], fb[0]);
        };
        copy(S0);
        if (NB > 2) copy(S1);
        for (int t = first_t; t < last_t; t += NB) {
            if constexpr (NB == 2) {
                step(t, S0, S1);
                if (t + 1 < last_t) step(t + 1, S1, S0);
            } else {
                static_assert(NB <= 3, "no ring of four here");
                step(t, S0, S2);
                if (t + 1 < last_t) step(t + 1, S1, S0);
                if (t + 2 < last_t) step(t + 2, S2, S1);
            }
        }
    }
    lift();
    if constexpr (LEVELS) epi(whole, mt * UA + wm * MI, nt * UB + wn * NJ, lane);
    else epi(acc, mt * UA + wm * MI, nt * UB + wn * NJ, lane);
}

// ---------------------------------------------------------------------------
// what is done with the tiles: (mb, nb) = the wave's first blocks

// v as terms of a plane (rows.hip: to_terms; rounded to nearest where one is not enough)
template <int T>
__device__ __forceinline__ void grad_terms(float v, uint16_t (&t)[T]) {
#pragma unroll
    for (int e = 0; e < T; e++) {
        const bool cut = e + 1 < T && (f2u(v) & 0x7f800000u) != 0x7f800000u;
        const uint32_t b = cut ? f2u(v) & 0xffff0000u : is_nan(v) ? 0x7fc00000u : rne_bits(v);
        t[e] = (uint16_t)(b >> 16);
        v = cut ? __fsub_rn(v, u2f(b)) : 0.f;
    }
}

// Four values along m of block mb (rows of a weight) at token `tok`, to planes
// [token][weight row]: 8 bytes a lane and term.
template <int T>
__device__ __forceinline__ void put_grad_terms(const Planes &d, int64_t mb, int64_t nb, int lane, const float (&v)[4]) {
    uint16_t t[4][T];
#pragma unroll
    for (int r = 0; r < 4; r++) grad_terms<T>(v[r], t[r]);
    const int q = lane >> 4;
    char *at = d.p + (nb * d.units + (mb >> 1)) * 1024 + ((lane & 15) + 16 * (2 * (mb & 1) + (q >> 1))) * 16 + (q & 1) * 8;
#pragma unroll
    for (int e = 0; e < T; e++) {
        uint2 w;
        w.x = (uint32_t)t[0][e] | (uint32_t)t[1][e] << 16;
        w.y = (uint32_t)t[2][e] | (uint32_t)t[3][e] << 16;
        *(uint2 *)(at + e * d.plane_bytes()) = w;
    }
}

// Partial sums: part[blockIdx.y][n][m], added to where `add`.
struct EpiParts {
    float *part;
    int64_t part_stride, ld;
    int64_t n, m;
    int add;
    template <int MI, int NJ>
    __device__ __forceinline__ void operator()(floatx4 (&acc)[MI][NJ], int mb, int nb, int lane) const {
        float *base = part + blockIdx.y * part_stride;
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int64_t row = (int64_t)(nb + j) * 16 + (lane & 15);
            if (row >= n) continue;
#pragma unroll
            for (int i = 0; i < MI; i++) {
                const int64_t c = (int64_t)(mb + i) * 16 + 4 * (lane >> 4);
                if (c >= m) continue;
                float4 *o = (float4 *)(base + row * ld + c);
                float4 v = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
                if (add) {
                    const float4 w = *o;
                    v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
                }
                *o = v;
            }
        }
    }
};

// Four neighbours of a row as the caller's type.
__device__ __forceinline__ void put_row4(void *out, int32_t dtype, int64_t at, int64_t left, bool wide,
                                         const float (&v)[4]) {
    if (dtype == DITCH_F32) {
        float *o = (float *)out + at;
        if (wide && left >= 4) *(float4 *)o = make_float4(v[0], v[1], v[2], v[3]);
        else
            for (int r = 0; r < 4; r++)
                if (r < left) o[r] = v[r];
        return;
    }
    uint16_t h[4];
#pragma unroll
    for (int r = 0; r < 4; r++)
        h[r] = dtype == DITCH_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[r]) : __builtin_bit_cast(uint16_t, (__bf16)v[r]);
    uint16_t *o = (uint16_t *)out + at;
    if (wide && left >= 4) {
        uint2 w;
        w.x = (uint32_t)h[0] | (uint32_t)h[1] << 16;
        w.y = (uint32_t)h[2] | (uint32_t)h[3] << 16;
        *(uint2 *)o = w;
    } else
        for (int r = 0; r < 4; r++)
            if (r < left) o[r] = h[r];
}
// four values fit one store at every row
inline bool rows_wide(const void *p, int64_t stride, int32_t dtype) {
    const int64_t size = 4 * (int64_t)row_size(dtype);
    return ((uintptr_t)p | (uintptr_t)(stride * (int64_t)row_size(dtype))) % size == 0;
}

// out[n][m] as the caller's rows; with a second output, the 32-row units 2i of n
// are the first's unit i and 2i + 1 the second's.
struct EpiRows {
    void *out, *second;
    int64_t stride, second_stride;
    int64_t n, m;
    int32_t dtype, wide;
    template <int MI, int NJ>
    __device__ __forceinline__ void operator()(floatx4 (&acc)[MI][NJ], int mb, int nb, int lane) const {
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int block = nb + j;
            const bool other = second && (block & 2);
            const int64_t row = (int64_t)(second ? block >> 2 << 1 | (block & 1) : block) * 16 + (lane & 15);
            if (row >= n) continue;
            void *to = other ? second : out;
            const int64_t at = row * (other ? second_stride : stride);
#pragma unroll
            for (int i = 0; i < MI; i++) {
                const int64_t c = (int64_t)(mb + i) * 16 + 4 * (lane >> 4);
                if (c >= m) continue;
                const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                put_row4(to, dtype, at + c, m - c, wide, v);
            }
        }
    }
};

// ---------------------------------------------------------------------------
// x W^T for few 16-bit rows on weights of one term, where the grid of 64 x 64 tiles
// does not fill the chip (rows_tiling). What those tiles take is then not memory but steps, each a
// barrier and the LDS' latency (350 cycles, eight stages ahead as with four): here a
// workgroup computes 32 words and its four waves share k, each with loads straight
// to registers, which hold fragments as they lie in memory, and no barrier until
// the sums are added.
template <int NJ, int TB, typename Epi>
__global__ __launch_bounds__(256) void rows_few_kernel(RowsGemm p, Epi epi) {
    constexpr int MI = 2, AHEAD = NJ * TB <= 2 ? 8 : 4, SUMS = MI * NJ * 64;
    __shared__ floatx4 sums[2 * SUMS];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int mt = blockIdx.x;
    const char *pa[MI], *pb[NJ];
    auto at = [](const RowsOperand &o, int q) {
        int second = 0;
        if (o.paired) {
            second = q & 1;
            q >>= 1;
        }
        return (int64_t)(q < o.blocks ? q : o.blocks - 1) * o.ldu * 1024 + (second ? o.pair : 0);
    };
#pragma unroll
    for (int i = 0; i < MI; i++) pa[i] = p.sa[0] + at(p.a, mt * MI + i) + lane * 16;
    const uint32_t lane_b = p.b.lane_at(lane);
#pragma unroll
    for (int j = 0; j < NJ; j++) pb[j] = p.sb[0] + at(p.b, j) + lane_b;
    struct Chunk {
        u32x4 a[AHEAD][MI], b[AHEAD][TB][NJ];
    };
    const int first = (int)((int64_t)p.k32 * wave / 4), last = (int)((int64_t)p.k32 * (wave + 1) / 4);
    auto load = [&](int t, Chunk &c) {
#pragma unroll
        for (int s = 0; s < AHEAD; s++) {
            if (t + s >= last) break;
            const int64_t ka = t + s < p.a.ks ? t + s : p.a.ks - 1, kb = t + s < p.b.ks ? t + s : p.b.ks - 1;
#pragma unroll
            for (int i = 0; i < MI; i++) c.a[s][i] = *(const u32x4 *)(pa[i] + ka * 1024);
#pragma unroll
            for (int e = 0; e < TB; e++)
#pragma unroll
                for (int j = 0; j < NJ; j++) c.b[s][e][j] = *(const u32x4 *)(pb[j] + e * p.b_plane + kb * p.b.unit);
        }
    };
    floatx4 acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](int t, const Chunk &c) {
#pragma unroll
        for (int s = 0; s < AHEAD; s++) {
            if (t + s >= last) break;
#pragma unroll
            for (int e = 0; e < TB; e++)
#pragma unroll
                for (int i = 0; i < MI; i++)
#pragma unroll
                    for (int j = 0; j < NJ; j++) acc[i][j] = mfma_bf16(c.a[s][i], c.b[s][e][j], acc[i][j]);
        }
    };
    Chunk one, two;
    load(first, one);
    for (int t = first; t < last; t += 2 * AHEAD) {
        load(t + AHEAD, two);
        multiply(t, one);
        load(t + 2 * AHEAD, one);
        multiply(t + AHEAD, two);
    }
    // the waves' sums, in the same order always: 0 + 2, 1 + 3, both
    auto give = [&](int slot) {
#pragma unroll
        for (int i = 0; i < MI; i++)
#pragma unroll
            for (int j = 0; j < NJ; j++) sums[slot * SUMS + (i * NJ + j) * 64 + lane] = acc[i][j];
    };
    auto take = [&](int slot) {
#pragma unroll
        for (int i = 0; i < MI; i++)
#pragma unroll
            for (int j = 0; j < NJ; j++) acc[i][j] += sums[slot * SUMS + (i * NJ + j) * 64 + lane];
    };
    if (wave >= 2) give(wave - 2);
    __syncthreads();
    if (wave < 2) take(wave);
    __syncthreads();
    if (wave == 1) give(0);
    __syncthreads();
    if (wave == 0) {
        take(0);
        epi(acc, mt * MI, 0, lane);
    }
}

// ---------------------------------------------------------------------------
// launches

template <int TB, typename Epi>
void launch_rows_few(const RowsGemm &g, int64_t mblocks, int64_t nblocks, const Epi &epi, hipStream_t s) {
    auto go = [&](auto nj) {
        hipLaunchKernelGGL((rows_few_kernel<decltype(nj)::value, TB, Epi>), dim3((unsigned)ceil_div(mblocks, 2)), dim3(256), 0, s,
                           g, epi);
        DITCH_TRY_HIP(hipGetLastError());
    };
    if constexpr (!Epi::PAIRS)
        if (nblocks == 1) return go(std::integral_constant<int, 1>{});
    if (nblocks <= 2) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 4>{});
}

template <int WGM, int WGN, int MI, int NJ, bool WHOLE, bool AO, bool BO, int TB, typename Epi>
void launch_rows_gemm_tile(RowsGemm g, int64_t mblocks, int64_t nblocks, const Epi &epi, hipStream_t s) {
    const int64_t tm = ceil_div(mblocks, WGM * MI), tn = ceil_div(nblocks, WGN * NJ);
    // (what such a product leaves is more than a TB)
    DITCH_CHECK(tm * tn < (int64_t)1 << 31 && g.parts < 65536, DITCH_INVALID_ARGUMENT, "rows product: more tiles than one launch holds");
    g.tiles_m = (int32_t)tm;
    g.tiles_n = (int32_t)tn;
    hipLaunchKernelGGL((rows_gemm_kernel<WGM, WGN, MI, NJ, WHOLE, AO, BO, TB, Epi>), rows_grid(tm * tn, WGM * WGN * 64, g.parts),
                       dim3(WGM * WGN * 64), 0, s, g, epi);
    DITCH_TRY_HIP(hipGetLastError());
}

// `tile`: rows_tiling's choice, or rows_out_tile's.
template <bool AO, bool BO, int TB, typename Epi>
void launch_rows_gemm(int tile, const RowsGemm &g, int64_t mblocks, int64_t nblocks, const Epi &epi, hipStream_t s) {
    // (sums in two levels do not fit the largest tile)
    if constexpr (TB != 3 || AO || BO)
        if (tile == 0) return launch_rows_gemm_tile<2, 4, 8, 4, true, AO, BO, TB>(g, mblocks, nblocks, epi, s);
    if (tile == 1) return launch_rows_gemm_tile<2, 2, 4, 4, false, AO, BO, TB>(g, mblocks, nblocks, epi, s);
    if constexpr (AO && BO) {  // rows_out_tile
        if constexpr (TB == 1) launch_rows_gemm_tile<2, 2, 8, 4, false, AO, BO, TB>(g, mblocks, nblocks, epi, s);
    } else {
        if (tile == 2) return launch_rows_gemm_tile<4, 2, 4, 2, false, AO, BO, TB>(g, mblocks, nblocks, epi, s);
        if (tile == 3) return launch_rows_gemm_tile<2, 2, 2, 2, false, AO, BO, TB>(g, mblocks, nblocks, epi, s);
        if constexpr (TB < 3 && !AO) return launch_rows_few<TB>(g, mblocks, nblocks, epi, s);
        if constexpr (TB == 3) launch_rows_gemm_tile<4, 2, 4, 2, true, AO, BO, TB>(g, mblocks, nblocks, epi, s);
    }
}

template <typename F>
void with_terms(int terms, F &&f) {
    if (terms == 1) f(std::integral_constant<int, 1>{});
    else if (terms == 2) f(std::integral_constant<int, 2>{});
    else f(std::integral_constant<int, 3>{});
}

}  // namespace ditch
