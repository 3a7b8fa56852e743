// pages_attention.hip — attention over pages of 8-bit keys and values for few
// rows a sequence (decode steps, short chunks).
//
// A workgroup takes 16 queries of one (sequence, KV head), the group's heads
// of as many rows as that is, and a part of the keys; its waves take granules
// of 32 tokens in turn, each with its own running maximum and accumulator,
// and join them through LDS at the end. Where sequences, heads and tiles give
// too few workgroups for the chip, the keys are split further over `splits`
// workgroups, whose unnormalised sums go to the workspace and are joined by a
// second kernel. Scores are formed transposed (keys x queries): the lanes
// that hold a query's scores then hold, in the operand order of the page
// format, the very tokens that the values' product takes from them, so the
// weights never leave the registers; and no operand passes through LDS, as
// each is used once.
//
// Bound by the read of the codes where they are many: 64 sequences of up to
// 8192 tokens (8 heads of 128, int8, 32 bf16 query heads, 714 MB) take 139 us,
// 5.1 TB/s, as a large copy does; one sequence of 130 001 (4 heads of 128,
// 133 MB) 26 us and 5 us for the join. Bound by latency where they are few
// (500 tokens: 9.7 us): page id, then scales and codes, then two products and
// the exponentials between them, a granule after the other.
#include <algorithm>

#include "pages_attention.h"

namespace ditch {

constexpr int MOST_SPLITS = 256;

struct RowsPlan {
    int tiles, splits, cols;  // query tiles of a (sequence, KV head); workgroups a tile; queries a tile
    int by_rows;              // tiles are those that can start in a row, and rows go in place of sequences
    int waves;                // of a workgroup: 4 or 8
    float *sums;              // [item][cols][DV]: splits > 1
    double *stats;            // [item][cols][2]: the maximum, the denominator relative to it
};

// Whose tile workgroup `blk` of a split has; false for none.
__device__ __forceinline__ bool place_tile(const PagesAttention &a, const RowsPlan &plan, int64_t blk, int &tile, int &h, int &seq,
                                           SeqRows &r) {
    const int u = (int)(blk % plan.tiles);
    blk /= plan.tiles;
    h = (int)(blk % a.p.kv_heads);
    const int at = (int)(blk / a.p.kv_heads), group = a.heads / a.p.kv_heads;
    if (!plan.by_rows) {
        tile = u;
        seq = at;
        r = seq_rows(a.b, seq);
        return tile * 16 / group < r.n;
    }
    const int i = row_place(a.b, at, seq, r);
    tile = (i * group + 15) / 16 + u;
    return i >= 0 && tile * 16 < (i + 1) * group;
}

template <typename T, int KIND, int DK, int DV, int NW>
__global__ __launch_bounds__(NW * 64) void pages_rows_kernel(PagesAttention a, RowsPlan plan) {
    constexpr int KP = DK / 64, VU = DV / 32, TERMS = sizeof(T) == 4 ? 2 : 1;
    constexpr int OS = DV + 4;
    extern __shared__ __attribute__((aligned(16))) float o_s[];  // [NW][cols][OS]
    __shared__ float m_s[NW][16];
    __shared__ double l_s[NW][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
    const int split = (int)(blockIdx.x % plan.splits);
    int tile, h, seq;
    SeqRows r;
    if (!place_tile(a, plan, blockIdx.x / plan.splits, tile, h, seq, r)) return;
    const int group = a.heads / a.p.kv_heads;
    const int first_row = tile * 16 / group, last_row = (tile * 16 + 15) / group;
    // rows past max_len
    if (split == 0 && last_row >= r.live) {
        for (int e = tid; e < 16 * a.p.vd; e += NW * 64) {
            const int qi = tile * 16 + e / a.p.vd, i = qi / group;
            if (i >= r.live && i < r.n)
                ((T *)a.out.data)[(int64_t)(r.row + i) * a.out.stride + (int64_t)(h * group + qi % group) * a.p.vd +
                                  e % a.p.vd] = (T)NAN;
        }
    }
    if (first_row >= r.live) return;
    const TileRows tr = tile_rows(r, first_row, last_row, a.window, a.sinks);
    const int qi = tile * 16 + c, row = qi / group;
    const bool mine = row < r.live;
    const Seen seen = seen_from(mine ? r.pos + row : tr.t_hi, a.window, a.sinks);

    RawQuery<KP> raw;
    load_query(raw, mine ? (const T *)a.q.data + (int64_t)(r.row + row) * a.q.stride +
                             (int64_t)(h * group + qi % group) * a.p.hd
                       : (const T *)nullptr,
               a.p.hd, g);
    QueryTile<KP, TERMS> q;
    float cq = 0.f;

    floatx4 o[DV / 16];
#pragma unroll
    for (int d = 0; d < DV / 16; d++) o[d] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = M_NONE, top = -INFINITY;
    double l = 0;
    bool far = false;

    const int k0 = (int)((int64_t)tr.granules * split / plan.splits), k1 = (int)((int64_t)tr.granules * (split + 1) / plan.splits);
    const int per = a.p.page / GRANULE;
    const int64_t head_stride = (int64_t)a.p.kv_heads * a.p.page_bytes;
    const uint8_t *base = a.p.codes + (int64_t)h * a.p.page_bytes + lane * 16;

    auto load = [&](u32x4 (&kb)[2 * KP], u32x4 (&vb)[VU], int id, int gi) {
        const int64_t in = gi & (per - 1);
        const uint8_t *kp = base + id * head_stride + in * (GRANULE * DK);
        const uint8_t *vp = base + id * head_stride + (int64_t)a.p.page * DK + in * (GRANULE * DV);
#pragma unroll
        for (int u = 0; u < 2 * KP; u++) kb[u] = *(const u32x4 *)(kp + u * 1024);
#pragma unroll
        for (int u = 0; u < VU; u++) vb[u] = *(const u32x4 *)(vp + u * 1024);
    };
    auto compute = [&](const u32x4 (&kb)[2 * KP], const u32x4 (&vb)[VU], int gi, const GranuleScales &sc) {
        const floatx4 s0 = scores<KIND, KP, TERMS>(kb, q), s1 = scores<KIND, KP, TERMS>(kb + KP, q);
        const float ck = cq * sc.key;
        const bool full = granule_full(tr, gi, a.window, a.sinks);
        const int j0 = gi * GRANULE + 4 * g;
        float w[8];
        granule_exponents(w, s0, s1, ck, sc.bias + (W_UP - m));
        if (!full || far) {
            if (far) far_exponents(w, s0, s1, ck, sc.bias, m);
            if (!full) granule_mask(w, j0, seen);
        }
        if (__any(most_of(w) > W_MOST)) {
            const float f = move_maximum(w, s0, s1, ck, sc.bias, full, j0, seen, m);
            far = maximum_far(m);
            l *= (double)f * f;
#pragma unroll
            for (int d = 0; d < DV / 16; d++) o[d] *= f * f;
        }
        float inverse = sc.inverse;
        if (granule_odd<TERMS>(sc, top)) {
            l += odd_granule(w, sc);
            inverse = 0.f;
        }
        Weights<TERMS> wt;
        l += (double)(granule_weights<TERMS>(wt, w) * inverse);
#pragma unroll
        for (int d = 0; d < DV / 16; d++) {
            const half8 v = codes_f16<KIND>(vb[d / 2][d % 2 * 2], vb[d / 2][d % 2 * 2 + 1]);
#pragma unroll
            for (int e = 0; e < TERMS; e++) o[d] = mfma_f16(v, wt.f[e], o[d]);
        }
    };

    // the wave's granules k0 + wave, + NW, ...: the pages and scales of 64 of
    // them at a time, one a lane, the codes one granule ahead. The first
    // codes are asked for before anything waits for the queries and scales.
    const int mine_n = k1 - k0 > wave ? (k1 - k0 - wave + NW - 1) / NW : 0;
    if (mine_n == 0) query_terms(q, raw);
    for (int b = 0; b < mine_n; b += 64) {
        const int n = mine_n - b < 64 ? mine_n - b : 64;
        const int gi_l = granule_index(tr, k0 + wave + NW * (b + (lane < n ? lane : 0)));
        const int id_l = page_of(a.b, a.p, seq, gi_l / per), in_l = id_l < 0 ? 0 : id_l;
        u32x4 ka[2 * KP], va[VU], kb[2 * KP], vb[VU];
        auto at = [&](float x, int i) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), i)); };
        auto id_at = [&](int i) { return __builtin_amdgcn_readlane(in_l, i); };
        auto gi_at = [&](int i) { return __builtin_amdgcn_readlane(gi_l, i); };
        load(ka, va, id_at(0), gi_at(0));
        const float2 sc = *(const float2 *)(a.p.scales + ((int64_t)in_l * a.p.kv_heads + h) * 2);
        if (b == 0) {
            query_terms(q, raw);
            cq = a.scale * 1.4426950408889634f * q.down;
        }
        // a page outside the pool: page 0's codes under scales of NaN
        const GranuleScales sc_l = granule_scales(id_l < 0 ? NAN : sc.x, id_l < 0 ? NAN : sc.y);
        for (int i = 0; i < n; i += 2) {
            if (i + 1 < n) load(kb, vb, id_at(i + 1), gi_at(i + 1));
            compute(ka, va, gi_at(i), GranuleScales{at(sc_l.key, i), at(sc_l.bias, i), at(sc_l.inverse, i)});
            if (i + 1 < n) {
                if (i + 2 < n) load(ka, va, id_at(i + 2), gi_at(i + 2));
                compute(kb, vb, gi_at(i + 1), GranuleScales{at(sc_l.key, i + 1), at(sc_l.bias, i + 1), at(sc_l.inverse, i + 1)});
            }
        }
    }

    // join the waves
    l = sum_groups(l);
    if (g == 0) {
        m_s[wave][c] = m;
        l_s[wave][c] = l;
    }
#pragma unroll
    for (int d = 0; d < DV / 16; d++)
        if (c < plan.cols) *(floatx4 *)&o_s[(wave * plan.cols + c) * OS + 16 * d + 4 * g] = o[d];
    __syncthreads();
    const int64_t item = (int64_t)blockIdx.x * plan.cols;
    for (int e = tid; e < plan.cols * (DV / 4); e += NW * 64) {
        const int cc = e / (DV / 4), d = e % (DV / 4) * 4, qq = tile * 16 + cc, i = qq / group;
        if (i >= r.live) continue;
        float mm = M_NONE;
#pragma unroll
        for (int w = 0; w < NW; w++) mm = fmaxf(mm, m_s[w][cc]);
        floatx4 sum{0.f, 0.f, 0.f, 0.f};
        double den = 0;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = __builtin_amdgcn_exp2f(0.5f * (m_s[w][cc] - mm));
            sum += *(const floatx4 *)&o_s[(w * plan.cols + cc) * OS + d] * (f * f);
            den += l_s[w][cc] * ((double)f * f);
        }
        if (plan.splits > 1) {
            *(floatx4 *)(plan.sums + (item + cc) * DV + d) = sum;
            if (d == 0) *(double2 *)(plan.stats + (item + cc) * 2) = make_double2((double)mm, den);
        } else {
            const double norm = 1.0 / den;
            T *out = (T *)a.out.data + (int64_t)(r.row + i) * a.out.stride + (int64_t)(h * group + qq % group) * a.p.vd;
            for (int j = 0; j < 4; j++)
                if (d + j < a.p.vd) out[d + j] = (T)(float)((double)sum[j] * norm);
        }
    }
}

// The splits of a query joined: a workgroup a query of a tile. Each group of
// dv / 4 threads (4 dims a thread) adds every 256 / (dv / 4)-th split, eight
// in flight; the groups' sums meet in LDS.
template <typename T>
__global__ __launch_bounds__(256) void pages_join_kernel(PagesAttention a, RowsPlan plan) {
    __shared__ float f_s[MOST_SPLITS], most_s[4];
    __shared__ double l_s[4];
    __shared__ __attribute__((aligned(16))) float o_s[256 * 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t blk = blockIdx.x / plan.cols;
    const int cc = (int)(blockIdx.x % plan.cols);
    const int64_t item = blk * plan.splits * plan.cols + cc;
    // the splits' maxima, factors and denominators
    const bool has = tid < plan.splits;
    const double2 st = has ? *(const double2 *)(plan.stats + (item + (int64_t)tid * plan.cols) * 2) : make_double2(M_NONE, 0);
    int tile, h, seq;
    SeqRows r;
    if (!place_tile(a, plan, blk, tile, h, seq, r)) return;
    const int group = a.heads / a.p.kv_heads, qq = tile * 16 + cc, i = qq / group;
    if (i >= r.live) return;
    float m = (float)st.x;
    for (int w = 32; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor(m, w, 64));
    if (lane == 0) most_s[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(most_s[0], most_s[1]), fmaxf(most_s[2], most_s[3]));
    const float f = __builtin_amdgcn_exp2f(0.5f * ((float)st.x - m));
    if (has) f_s[tid] = f * f;
    double l = has ? st.y * ((double)f * f) : 0;
    for (int w = 32; w > 0; w >>= 1) l += __shfl_xor(l, w, 64);
    if (lane == 0) l_s[wave] = l;
    __syncthreads();
    const int quads = a.p.dv / 4, groups = 256 / quads, mine = tid / quads, d = tid % quads * 4;
    floatx4 o{0.f, 0.f, 0.f, 0.f};
    if (mine < groups) {
        const float *p = plan.sums + item * a.p.dv + d;
        const int64_t step = (int64_t)plan.cols * a.p.dv;
#pragma unroll 8
        for (int s = mine; s < plan.splits; s += groups) o += *(const floatx4 *)(p + s * step) * f_s[s];
        *(floatx4 *)&o_s[mine * a.p.dv + d] = o;
    }
    __syncthreads();
    if (tid >= a.p.vd) return;
    float num = 0.f;
    for (int w = 0; w < groups; w++) num += o_s[w * a.p.dv + tid];
    ((T *)a.out.data)[(int64_t)(r.row + i) * a.out.stride + (int64_t)(h * group + qq % group) * a.p.vd + tid] =
        (T)(float)((double)num / ((l_s[0] + l_s[1]) + (l_s[2] + l_s[3])));
}

// ---------------------------------------------------------------------------
// the plan

static int64_t plan_items(const PoolView &p, const BatchView &b, const RowsPlan &plan) {
    return (int64_t)(plan.by_rows ? b.n_rows : b.n_seqs) * p.kv_heads * plan.tiles;
}

static RowsPlan rows_plan(const PoolView &p, const BatchView &b, int heads, uint32_t window, uint32_t sinks) {
    const int group = heads / p.kv_heads;
    RowsPlan plan{};
    const int64_t queries = (int64_t)b.max_rows * group;
    plan.tiles = (int)((queries + 15) / 16);
    plan.cols = (int)std::min<int64_t>(queries, 16);
    // granules that a tile can see
    int64_t keys = b.max_len;
    if (window) keys = std::min<int64_t>(keys, (int64_t)window + 16 + sinks + 2 * GRANULE);
    const int64_t granules = (keys + GRANULE - 1) / GRANULE;
    if (b.by_rows && (int64_t)b.n_rows * ((group + 15) / 16) < (int64_t)b.n_seqs * plan.tiles) {
        plan.by_rows = 1;
        plan.tiles = (group + 15) / 16;
    }
    const int64_t items = plan_items(p, b, plan);
    // Waves. 2048 (two a SIMD) saturate the memory: 64 sequences of up to 8192
    // tokens of 8 heads of 128 take 137 us with 512 tiles of 4 waves, 139 us
    // with twice the waves. A tile's first 8 waves share a workgroup, more go
    // to further workgroups and need the join, about 4 us; a granule takes a
    // wave about 0.4 us where latency counts, so up to 12 granules a wave one
    // workgroup is ahead (36 granules of a window, 96 tiles: 10.9 us against
    // 13.7 split; 4063 granules, 4 tiles: 34 us split). Four waves where the
    // registers of larger heads allow no more.
    const int64_t waves = std::min((2048 + items - 1) / items, granules);
    plan.waves = waves <= 4 || p.dk > 128 ? 4 : 8;
    plan.splits = 1;
    if (waves > plan.waves && granules > 12 * plan.waves)
        plan.splits = (int)std::min<int64_t>((waves + plan.waves - 1) / plan.waves, MOST_SPLITS);
    return plan;
}

size_t pages_attention_workspace(const PoolView &p, const BatchView &b, int heads, int32_t dtype, uint32_t window,
                                 uint32_t sinks, int few) {
    if (b.n_seqs == 0 || (!few && pages_chunk_takes(p, b, heads, dtype))) return 0;
    const RowsPlan plan = rows_plan(p, b, heads, window, sinks);
    if (plan.splits == 1) return 0;
    return (size_t)plan_items(p, b, plan) * plan.splits * plan.cols * (p.dv + 4) * 4;
}

template <typename T, int KIND, int DK, int DV, int NW>
static void rows_waves(const PagesAttention &a, const RowsPlan &plan, unsigned blocks, hipStream_t s) {
    hipLaunchKernelGGL((pages_rows_kernel<T, KIND, DK, DV, NW>), dim3(blocks), dim3(NW * 64),
                       (unsigned)(NW * plan.cols * (DV + 4) * 4), s, a, plan);
    DITCH_TRY_HIP(hipGetLastError());
}

template <typename T, int KIND, int DK, int DV>
static void rows_dims(const PagesAttention &a, const RowsPlan &plan, unsigned blocks, hipStream_t s) {
    if (plan.waves == 4) rows_waves<T, KIND, DK, DV, 4>(a, plan, blocks, s);
    else if constexpr (DK <= 128) rows_waves<T, KIND, DK, DV, 8>(a, plan, blocks, s);
}

template <typename T, int KIND>
static void rows_kind(const PagesAttention &a, const RowsPlan &plan, unsigned blocks, hipStream_t s) {
    if (a.p.dv == 256) rows_dims<T, KIND, 256, 256>(a, plan, blocks, s);
    else if (a.p.dv == 192) rows_dims<T, KIND, 192, 192>(a, plan, blocks, s);
    else if (a.p.dk == 192) rows_dims<T, KIND, 192, 128>(a, plan, blocks, s);
    else if (a.p.dv == 128) rows_dims<T, KIND, 128, 128>(a, plan, blocks, s);
    else rows_dims<T, KIND, 64, 64>(a, plan, blocks, s);
}

template <typename T>
static void rows_typed(const PagesAttention &a, const RowsPlan &plan, hipStream_t s) {
    const int64_t tiles = plan_items(a.p, a.b, plan);
    DITCH_CHECK(tiles * (plan.splits > 1 ? std::max(plan.splits, plan.cols) : 1) < ((int64_t)1 << 24), DITCH_INVALID_ARGUMENT,
                "kv attention: more work than one launch holds");
    if (a.p.kind == DITCH_KV_INT8) rows_kind<T, DITCH_KV_INT8>(a, plan, (unsigned)(tiles * plan.splits), s);
    else rows_kind<T, DITCH_KV_E4M3>(a, plan, (unsigned)(tiles * plan.splits), s);
    if (plan.splits > 1) {
        hipLaunchKernelGGL((pages_join_kernel<T>), dim3((unsigned)(tiles * plan.cols)), dim3(256), 0, s, a, plan);
        DITCH_TRY_HIP(hipGetLastError());
    }
}

void launch_pages_attention(const PagesAttention &a, void *ws, size_t ws_bytes, hipStream_t s) {
    if (a.b.n_seqs == 0) return;
    if (!a.few && pages_chunk_takes(a.p, a.b, a.heads, a.dtype)) return launch_pages_chunk(a, s);
    RowsPlan plan = rows_plan(a.p, a.b, a.heads, (uint32_t)a.window, (uint32_t)a.sinks);
    if (plan.splits > 1) {
        plan.sums = (float *)ws;
        plan.stats = (double *)(plan.sums + plan_items(a.p, a.b, plan) * plan.splits * plan.cols * a.p.dv);
    }
    if (a.dtype == DITCH_F32) rows_typed<float>(a, plan, s);
    else if (a.dtype == DITCH_F16) rows_typed<_Float16>(a, plan, s);
    else rows_typed<__bf16>(a, plan, s);
}

}  // namespace ditch
