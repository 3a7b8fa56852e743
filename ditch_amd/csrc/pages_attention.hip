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
#include <algorithm>

#include "pages_attention.h"

namespace ditch {

struct RowsPlan {
    int tiles, splits, cols;  // query tiles of a (sequence, KV head); workgroups a tile; queries a tile
    float *sums, *stats;      // [item][cols][DV], [item][cols][2]: splits > 1
};

template <typename T, int KIND, int DK, int DV, int NW>
__global__ __launch_bounds__(NW * 64) void pages_rows_kernel(PagesAttention a, RowsPlan plan) {
    constexpr int KP = DK / 64, VU = DV / 32, TERMS = sizeof(T) == 4 ? 2 : 1;
    constexpr int OS = DV + 4;
    __shared__ __attribute__((aligned(16))) float o_s[NW][16][OS];
    __shared__ float m_s[NW][16], l_s[NW][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
    int64_t blk = blockIdx.x;
    const int split = (int)(blk % plan.splits);
    blk /= plan.splits;
    const int tile = (int)(blk % plan.tiles);
    blk /= plan.tiles;
    const int h = (int)(blk % a.p.kv_heads), seq = (int)(blk / a.p.kv_heads);
    const SeqRows r = seq_rows(a.b, seq);
    const int group = a.heads / a.p.kv_heads;
    const int first_row = tile * 16 / group, last_row = (tile * 16 + 15) / group;
    if (first_row >= r.n) return;
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
    const int t = mine ? r.pos + row : tr.t_hi;  // the column's position

    QueryTile<KP, TERMS> q;
    load_query(q, mine ? (const T *)a.q.data + (int64_t)(r.row + row) * a.q.stride +
                             (int64_t)(h * group + qi % group) * a.p.hd
                       : (const T *)nullptr,
               a.p.hd, g);
    const float cq = a.scale * 1.4426950408889634f * q.down;

    floatx4 o[DV / 16];
#pragma unroll
    for (int d = 0; d < DV / 16; d++) o[d] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = M_NONE, l = 0.f;

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
        float x[8], w[8];
        const bool full = granule_full(tr, gi, a.window, a.sinks);
        const int j0 = gi * GRANULE + 4 * g;
        auto weigh = [&](float add) {
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = __builtin_fmaf(j < 4 ? s0[j & 3] : s1[j & 3], ck, add);
            if (!full)
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (!token_seen(j0 + (j < 4 ? j : 12 + j), t, a.window, a.sinks)) w[j] = -INFINITY;
        };
        weigh(sc.bias + (W_UP - m));
        float most = fmaxf(fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3])), fmaxf(fmaxf(w[4], w[5]), fmaxf(w[6], w[7])));
        if (__any(most > W_MOST)) {
            weigh(sc.bias);
            most = max_groups(fmaxf(fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3])), fmaxf(fmaxf(w[4], w[5]), fmaxf(w[6], w[7]))));
            const float next = fmaxf(m, most), f = __builtin_amdgcn_exp2f(m - next);
            m = next;
            l *= f;
#pragma unroll
            for (int d = 0; d < DV / 16; d++) o[d] *= f;
            weigh(sc.bias + (W_UP - m));
        }
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[j] = __builtin_amdgcn_exp2f(w[j]);
            sum += x[j];
        }
        if (fabsf(sc.bias) > BIAS_PLAIN) {
            // a value scale far from 1: the denominator from the scores alone
            sum = 0.f;
#pragma unroll
            for (int j = 0; j < 8; j++) sum += __builtin_amdgcn_exp2f(w[j] - sc.bias);
        } else if (sc.inverse != 0.f) {
            sum = sum == 0.f ? 0.f : sum * sc.inverse;
        }
        l += sum;
        if (sc.inverse == 0.f) return;  // values of scale zero
        Weights<TERMS> wt;
        weight_terms(wt, x);
#pragma unroll
        for (int d = 0; d < DV / 16; d++) {
            const half8 v = codes_f16<KIND>(vb[d / 2][d % 2 * 2], vb[d / 2][d % 2 * 2 + 1]);
#pragma unroll
            for (int e = 0; e < TERMS; e++) o[d] = mfma_f16(v, wt.f[e], o[d]);
        }
    };

    // the wave's granules k0 + wave, + NW, ...: the pages and scales of 64 of
    // them at a time, one a lane, the codes one granule ahead
    const int mine_n = k1 - k0 > wave ? (k1 - k0 - wave + NW - 1) / NW : 0;
    for (int b = 0; b < mine_n; b += 64) {
        const int n = mine_n - b < 64 ? mine_n - b : 64;
        int gi_l = 0, id_l = 0;
        GranuleScales sc_l{0.f, 0.f, 1.f};
        if (lane < n) {
            gi_l = granule_index(tr, k0 + wave + NW * (b + lane));
            id_l = page_of(a.b, a.p, seq, gi_l / per);
            float2 sc = make_float2(NAN, NAN);
            if (id_l >= 0) sc = *(const float2 *)(a.p.scales + ((int64_t)id_l * a.p.kv_heads + h) * 2);
            else id_l = 0;  // page 0's codes under scales of NaN
            sc_l = granule_scales(sc.x, sc.y);
        }
        u32x4 ka[2 * KP], va[VU], kb[2 * KP], vb[VU];
        auto at = [&](float x, int i) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), i)); };
        auto id_at = [&](int i) { return __builtin_amdgcn_readlane(id_l, i); };
        auto gi_at = [&](int i) { return __builtin_amdgcn_readlane(gi_l, i); };
        load(ka, va, id_at(0), gi_at(0));
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
    for (int d = 0; d < DV / 16; d++) *(floatx4 *)&o_s[wave][c][16 * d + 4 * g] = o[d];
    __syncthreads();
    const int64_t item = ((((int64_t)seq * a.p.kv_heads + h) * plan.tiles + tile) * plan.splits + split) * plan.cols;
    for (int e = tid; e < plan.cols * (DV / 4); e += NW * 64) {
        const int cc = e / (DV / 4), d = e % (DV / 4) * 4, qq = tile * 16 + cc, i = qq / group;
        if (i >= r.live) continue;
        float mm = M_NONE;
#pragma unroll
        for (int w = 0; w < NW; w++) mm = fmaxf(mm, m_s[w][cc]);
        floatx4 sum{0.f, 0.f, 0.f, 0.f};
        float den = 0.f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = __builtin_amdgcn_exp2f(m_s[w][cc] - mm);
            sum += *(const floatx4 *)&o_s[w][cc][d] * f;
            den += l_s[w][cc] * f;
        }
        if (plan.splits > 1) {
            *(floatx4 *)(plan.sums + (item + cc) * DV + d) = sum;
            if (d == 0) *(float2 *)(plan.stats + (item + cc) * 2) = make_float2(mm, den);
        } else {
            T *out = (T *)a.out.data + (int64_t)(r.row + i) * a.out.stride + (int64_t)(h * group + qq % group) * a.p.vd;
            for (int j = 0; j < 4; j++)
                if (d + j < a.p.vd) out[d + j] = (T)(sum[j] / den);
        }
    }
}

// The splits of a tile joined: a workgroup a tile.
template <typename T>
__global__ __launch_bounds__(256) void pages_join_kernel(PagesAttention a, RowsPlan plan) {
    const int64_t blk = blockIdx.x;
    const int tile = (int)(blk % plan.tiles), h = (int)(blk / plan.tiles % a.p.kv_heads),
              seq = (int)(blk / plan.tiles / a.p.kv_heads);
    const SeqRows r = seq_rows(a.b, seq);
    const int group = a.heads / a.p.kv_heads;
    const int64_t item = blk * plan.splits * plan.cols;
    for (int e = threadIdx.x; e < plan.cols * a.p.vd; e += 256) {
        const int cc = e / a.p.vd, d = e % a.p.vd, qq = tile * 16 + cc, i = qq / group;
        if (i >= r.live) break;
        float mm = M_NONE, num = 0.f, den = 0.f;
        for (int s = 0; s < plan.splits; s++) mm = fmaxf(mm, plan.stats[(item + (int64_t)s * plan.cols + cc) * 2]);
        for (int s = 0; s < plan.splits; s++) {
            const int64_t at = item + (int64_t)s * plan.cols + cc;
            const float f = __builtin_amdgcn_exp2f(plan.stats[at * 2] - mm);
            num += plan.sums[at * a.p.dv + d] * f;
            den += plan.stats[at * 2 + 1] * f;
        }
        ((T *)a.out.data)[(int64_t)(r.row + i) * a.out.stride + (int64_t)(h * group + qq % group) * a.p.vd + d] =
            (T)(num / den);
    }
}

// ---------------------------------------------------------------------------
// the plan

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
    const int64_t blocks = (int64_t)b.n_seqs * p.kv_heads * plan.tiles;
    int64_t splits = (1024 + blocks - 1) / blocks;
    splits = std::min(splits, (granules + 7) / 8);
    plan.splits = (int)std::max<int64_t>(splits, 1);
    return plan;
}

size_t pages_attention_workspace(const PoolView &p, const BatchView &b, int heads, int32_t dtype, uint32_t window,
                                 uint32_t sinks) {
    if (b.n_seqs == 0) return 0;
    const RowsPlan plan = rows_plan(p, b, heads, window, sinks);
    if (plan.splits == 1) return 0;
    return (size_t)b.n_seqs * p.kv_heads * plan.tiles * plan.splits * plan.cols * (p.dv + 2) * 4;
}

template <typename T, int KIND, int DK, int DV>
static void rows_dims(const PagesAttention &a, const RowsPlan &plan, unsigned blocks, hipStream_t s) {
    hipLaunchKernelGGL((pages_rows_kernel<T, KIND, DK, DV, 4>), dim3(blocks), dim3(256), 0, s, a, plan);
    DITCH_TRY_HIP(hipGetLastError());
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
    const int64_t tiles = (int64_t)a.b.n_seqs * a.p.kv_heads * plan.tiles;
    DITCH_CHECK(tiles * plan.splits < ((int64_t)1 << 24), DITCH_INVALID_ARGUMENT,
                "kv attention: more work than one launch holds");
    if (a.p.kind == DITCH_KV_INT8) rows_kind<T, DITCH_KV_INT8>(a, plan, (unsigned)(tiles * plan.splits), s);
    else rows_kind<T, DITCH_KV_E4M3>(a, plan, (unsigned)(tiles * plan.splits), s);
    if (plan.splits > 1) {
        hipLaunchKernelGGL((pages_join_kernel<T>), dim3((unsigned)tiles), dim3(256), 0, s, a, plan);
        DITCH_TRY_HIP(hipGetLastError());
    }
}

void launch_pages_attention(const PagesAttention &a, void *ws, size_t ws_bytes, hipStream_t s) {
    if (a.b.n_seqs == 0) return;
    RowsPlan plan = rows_plan(a.p, a.b, a.heads, (uint32_t)a.window, (uint32_t)a.sinks);
    if (plan.splits > 1) {
        plan.stats = (float *)ws;
        plan.sums = plan.stats + (int64_t)a.b.n_seqs * a.p.kv_heads * plan.tiles * plan.splits * plan.cols * 2;
    }
    if (a.dtype == DITCH_F32) rows_typed<float>(a, plan, s);
    else if (a.dtype == DITCH_F16) rows_typed<_Float16>(a, plan, s);
    else rows_typed<__bf16>(a, plan, s);
}

}  // namespace ditch
