// pages_attention.h — what the attention kernels over pages of 8-bit keys and
// values share (pages_attention.hip, pages_chunk.hip).
//
// Mathematics. For a query q, keys k_j = ks c_j (ks: the scale of the key's
// page and head, c: codes) and values v_j = vs e_j:
//   out = sum_j exp(s_j) vs_j e_j / sum_j exp(s_j),  s_j = scale ks_j (q . c_j)
// in one pass with a running maximum. The value scale goes into the
// exponent, w_j = 2^(s_j log2(e) + log2(vs_j) - m), so the accumulator sums
// w_j e_j with plain codes, and the denominator adds a granule's w times
// 1 / vs: one multiplication for a granule's eight weights a lane. The maximum
// is that of the weights, scale included, so the denominator relative to it
// spans what the scales do, 2^-126 to 2^127: it is held in 64 bits (32 would
// end at infinity where the first pages' values are below about 2^-113, and
// stay there when the maximum moves on).
//
// Codes of both kinds are exact in f16 (int8: 8 bits of 11; e4m3: 4 bits, the
// least 2^-9), so both products run on v_mfma_f32_16x16x32_f16 with exact
// cache operands. A query is scaled by a power of two that takes its largest
// coordinate to [2^14, 2^15): what f16's smallest steps drop is below
// 2^-39 of it. 16-bit queries enter as one f16 term (exact for f16, and for
// bf16's 8 bits), f32 ones as two (22 bits). Weights enter as one RNE f16
// (2^-12 of their value, below the output's own rounding of at least 2^-12)
// or, for f32 rows, as two terms.
#pragma once
#include "pages.h"

namespace ditch {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Weights are held relative to the running maximum, times 2^W_UP, and the
// maximum moves only when one would pass 2^W_MOST: f16 ends at 2^16, and
// its steps below 2^-14 are then 2^-36 of the largest weight.
constexpr float W_UP = 12.f, W_MOST = 15.f;
constexpr float M_NONE = -3e38f;  // the maximum over no keys
// From here on the steps of a maximum (1/2 and more) are no longer small beside
// W_MOST - W_UP: exponents are then formed as the maximum was, rounded
// before it is taken off, so that none is above it.
constexpr float M_FAR = 4194304.f;

// A value scale with log2 outside of this, or this far below that of the
// largest scale walked before it, goes its own way (see granule_scales). Of
// one-term weights the denominator sums what f16 leaves, off by 2^-25 a key,
// so that n keys of a scale 2^-NEAR of the one that the maximum holds to 2^12
// are off by n 2^(NEAR - 37) of the whole: 2^-13 at 2^18 keys. Two terms sum
// the weights in f32: they end at 2^-126.
constexpr float BIAS_PLAIN = 40.f;
template <int TERMS>
constexpr float BIAS_NEAR = TERMS == 1 ? 6.f : 60.f;

__device__ __forceinline__ floatx4 mfma_f16(half8 a, half8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The f16 values of 8 codes.
template <int KIND>
__device__ __forceinline__ half8 codes_f16(uint32_t lo, uint32_t hi) {
    u32x4 r;
    if constexpr (KIND == DITCH_KV_INT8) {
        // 0x64uu is 1024 + uu in f16; uu = code + 128
        lo ^= 0x80808080u;
        hi ^= 0x80808080u;
        r[0] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u);
        r[1] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u);
        r[2] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u);
        r[3] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u);
        return __builtin_bit_cast(half8, r) - (_Float16)1152.f;
    } else {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true));
        return __builtin_bit_cast(half8, r);
    }
}

// The largest over the four lanes (l, l ^ 16, l ^ 32, l ^ 48), the sum.
__device__ __forceinline__ float max_groups(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ double sum_groups(double x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}
// 2^t past f32's range.
__device__ __forceinline__ double exp2_wide(float t) {
    const double h = (double)__builtin_amdgcn_exp2f(0.5f * t);
    return h * h;
}

// A query tile's operands: lane (g, c) holds query c's dims 64 p + 16 g + 0..7
// (step 0) and + 8..15 (step 1) of every 64-dim unit p, in TERMS f16 terms,
// and the power of two that undoes the query's scaling.
template <int KP, int TERMS>
struct QueryTile {
    half8 f[KP][2][TERMS];
    float down;
};

// The lane's coordinates of a query as loaded. x: the query's head (NULL: zeros), hd its dims.
template <int KP>
struct RawQuery {
    float v[KP][16];
};
template <typename T, int KP>
__device__ __forceinline__ void load_query(RawQuery<KP> &q, const T *x, int hd, int g) {
#pragma unroll
    for (int p = 0; p < KP; p++) {
        const int d0 = 64 * p + 16 * g;
        if (x && d0 + 16 <= hd) {
#pragma unroll
            for (int j = 0; j < 16; j++) q.v[p][j] = (float)x[d0 + j];
        } else {
#pragma unroll
            for (int j = 0; j < 16; j++) q.v[p][j] = x && d0 + j < hd ? (float)x[d0 + j] : 0.f;
        }
    }
}
template <int KP, int TERMS>
__device__ __forceinline__ void query_terms(QueryTile<KP, TERMS> &q, const RawQuery<KP> &raw) {
    float most = 0.f;
#pragma unroll
    for (int p = 0; p < KP; p++)
#pragma unroll
        for (int j = 0; j < 16; j++) most = fmaxf(most, fabsf(raw.v[p][j]));
    most = max_groups(most);
    // 2^up takes the largest to [2^14, 2^15) (from a subnormal: as far as f32 goes)
    const int up = most > 0.f && most <= 3.4028234663852886e38f ? 14 - (int)((__float_as_uint(most) >> 23) - 127) : 0;
#pragma unroll
    for (int p = 0; p < KP; p++)
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float y = ldexpf(raw.v[p][8 * s + j], up);
                const _Float16 hi = (_Float16)y;
                q.f[p][s][0][j] = hi;
                if constexpr (TERMS == 2) q.f[p][s][1][j] = (_Float16)(y - (float)hi);
            }
    q.down = ldexpf(1.f, -up);
}

// The keys of a 16-token tile (kb: its KP 16-byte units a lane) times the queries.
template <int KIND, int KP, int TERMS>
__device__ __forceinline__ floatx4 scores(const u32x4 *kb, const QueryTile<KP, TERMS> &q) {
    floatx4 s{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < KP; p++) {
        const half8 k0 = codes_f16<KIND>(kb[p][0], kb[p][1]), k1 = codes_f16<KIND>(kb[p][2], kb[p][3]);
#pragma unroll
        for (int t = 0; t < TERMS; t++) {
            s = mfma_f16(k0, q.f[p][0][t], s);
            s = mfma_f16(k1, q.f[p][1][t], s);
        }
    }
    return s;
}

// 8 weights as the operand of the values' product, and their sum: of one
// term what the product really uses, so that a weight's rounding is the same
// above and below.
template <int TERMS>
struct Weights {
    half8 f[TERMS];
};
template <int TERMS>
__device__ __forceinline__ float weight_terms(Weights<TERMS> &w, const float (&x)[8]) {
    u32x4 hi;
    float sum = 0.f;
    if constexpr (TERMS == 1) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const half2_t h = __builtin_convertvector(floatx2{x[2 * j], x[2 * j + 1]}, half2_t);
            hi[j] = __builtin_bit_cast(uint32_t, h);
            sum = __builtin_amdgcn_fdot2(h, half2_t{(_Float16)1.f, (_Float16)1.f}, sum, false);
        }
        w.f[0] = __builtin_bit_cast(half8, hi);
    } else {
        u32x4 lo;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            // toward zero: the second term holds what is left
            const half2_t h = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(x[2 * j], x[2 * j + 1]));
            hi[j] = __builtin_bit_cast(uint32_t, h);
            lo[j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x[2 * j] - (float)h[0], x[2 * j + 1] - (float)h[1]));
            sum += x[2 * j] + x[2 * j + 1];
        }
        w.f[0] = __builtin_bit_cast(half8, hi);
        w.f[1] = __builtin_bit_cast(half8, lo);
    }
    return sum;
}

// A granule's scales as the loops use them. A value scale far from 1 would
// take the denominator's part out of the weights' range, and so would one far
// below the others; a NaN would reach rows that see none of the granule, and
// zero has no logarithm: such a granule is `odd` (see odd_granule), by itself
// with an inverse of 0. Zero goes below the least scale there is, so that it
// moves the maximum past no other's weights.
constexpr float BIAS_ZERO = -127.f;
struct GranuleScales {
    float key, bias, inverse;
};
__device__ __forceinline__ GranuleScales granule_scales(float ks, float vs) {
    const bool zero = fabsf(vs) < 1.17549435e-38f;  // (subnormal: the logarithm takes it for zero)
    const float bias = zero ? BIAS_ZERO : __builtin_amdgcn_logf(vs);
    const bool plain = fabsf(bias) <= BIAS_PLAIN && fabsf(ks) <= 3.4028234663852886e38f;
    return {ks, bias, plain ? 1.f / vs : 0.f};
}
// (top: the largest bias so far, this granule's included)
template <int TERMS>
__device__ __forceinline__ bool granule_odd(const GranuleScales &sc, float &top) {
    top = fmaxf(top, sc.bias);
    return sc.inverse == 0.f || sc.bias < top - BIAS_NEAR<TERMS>;
}

// The rows of a query tile: 16 consecutive (row, head of the KV head's
// group) pairs of one sequence and KV head; lane column c holds pair 16 tile + c.
struct TileRows {
    int t_lo, t_hi;  // positions of its first and last live row
    int granules;    // granules that any of them sees
    int sink_end;    // the first granules: 0 .. sink_end
    int skip;        // added to the index of the further ones
};
__device__ __forceinline__ TileRows tile_rows(const SeqRows &r, int first_row, int last_row, int window, int sinks) {
    TileRows t;
    t.t_lo = r.pos + first_row;
    t.t_hi = r.pos + (last_row < r.live ? last_row : r.live - 1);
    const int end = t.t_hi / GRANULE + 1;
    const int first = window && t.t_lo - window + 1 > 0 ? (t.t_lo - window + 1) / GRANULE : 0;
    const int sg = sinks > 0 && first > 0 ? (sinks - 1) / GRANULE + 1 : 0;
    t.sink_end = sg < first ? sg : first;
    t.skip = first - t.sink_end;
    t.granules = t.sink_end + end - first;
    return t;
}
__device__ __forceinline__ int granule_index(const TileRows &t, int k) { return k < t.sink_end ? k : k + t.skip; }
// Every token of granule gi is visible to every live row of the tile.
__device__ __forceinline__ bool granule_full(const TileRows &t, int gi, int window, int sinks) {
    const int a = gi * GRANULE, z = a + GRANULE - 1;
    return z <= t.t_lo && (!window || a > t.t_hi - window || z < sinks);
}
// What a column sees: the tokens first .. first + span (its own position) and
// those of the first `sinks` that lie before them.
struct Seen {
    int first;
    uint32_t span;
    int sinks;
};
__device__ __forceinline__ Seen seen_from(int t, int window, int sinks) {
    const int first = window && t - window + 1 > 0 ? t - window + 1 : 0;
    return {first, (uint32_t)(t - first), sinks < first ? sinks : first};
}
__device__ __forceinline__ bool token_seen(int j, const Seen &s) { return (uint32_t)(j - s.first) <= s.span || j < s.sinks; }

// The exponents of a granule's weights for one query tile, less the running
// maximum: s0, s1 the scores' products (tokens 4 g + i and 16 + 4 g + i of the
// granule), ck and add what takes them there.
__device__ __forceinline__ void granule_exponents(float (&w)[8], floatx4 s0, floatx4 s1, float ck, float add) {
#pragma unroll
    for (int j = 0; j < 8; j++) w[j] = __builtin_fmaf(j < 4 ? s0[j & 3] : s1[j & 3], ck, add);
}
// The same relative to a maximum past M_FAR.
__device__ __forceinline__ void far_exponents(float (&w)[8], floatx4 s0, floatx4 s1, float ck, float bias, float m) {
    granule_exponents(w, s0, s1, ck, bias);
#pragma unroll
    for (int j = 0; j < 8; j++) w[j] = (w[j] - m) + W_UP;
}
// A column of the wave has such a maximum.
__device__ __forceinline__ bool maximum_far(float m) { return __any(fabsf(m) > M_FAR && m != M_NONE); }
// Tokens that the column does not see; j0 the lane's first token.
__device__ __forceinline__ void granule_mask(float (&w)[8], int j0, const Seen &seen) {
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (!token_seen(j0 + (j < 4 ? j : 12 + j), seen)) w[j] = -INFINITY;
}
// (v_max3 itself: fmaxf would quiet each operand first. A NaN is passed over.)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}
__device__ __forceinline__ float most_of(const float (&w)[8]) {
    return max3(max3(w[0], w[1], w[2]), max3(w[3], w[4], w[5]), max3(w[6], w[7], w[7]));
}
// Moves the running maximum m to the exponents' largest where that passes
// W_MOST; returns the root of the factor of what was added up under the old one.
__device__ __forceinline__ float move_maximum(float (&w)[8], floatx4 s0, floatx4 s1, float ck, float bias, bool full, int j0,
                                              const Seen &seen, float &m) {
    granule_exponents(w, s0, s1, ck, bias);
    if (!full) granule_mask(w, j0, seen);
    const float next = fmaxf(m, max_groups(most_of(w))), root = __builtin_amdgcn_exp2f(0.5f * (m - next));
    m = next;
    far_exponents(w, s0, s1, ck, bias, m);
    if (!full) granule_mask(w, j0, seen);
    return root;
}
// An odd granule's part of the denominator, from the scores alone: the
// product's weights then add nothing to it (inverse 0), and under a value
// scale of zero there are none.
__device__ __forceinline__ double odd_granule(float (&w)[8], const GranuleScales &sc) {
    double sum = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        sum += w[j] == -INFINITY ? 0.0 : exp2_wide(w[j] - sc.bias);
        if (sc.bias == BIAS_ZERO) w[j] = -INFINITY;
    }
    return sum;
}
// The weights, and their sum.
template <int TERMS>
__device__ __forceinline__ float granule_weights(Weights<TERMS> &wt, const float (&w)[8]) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = __builtin_amdgcn_exp2f(w[j]);
    return weight_terms<TERMS>(wt, x);
}

// pages_chunk.hip: many rows a sequence
bool pages_chunk_takes(const PoolView &p, const BatchView &b, int heads, int32_t dtype);
void launch_pages_chunk(const PagesAttention &a, hipStream_t s);

}  // namespace ditch
