// pages_chunk.hip — attention over pages of 8-bit keys and values for many
// rows a sequence (chunks of prompts).
//
// A workgroup takes 16 QT NW consecutive queries (rows x heads of the group)
// of one (sequence, KV head), QT tiles of 16 a wave, and walks the keys that
// any of them sees granule by granule. A granule's codes are converted to f16
// once, into LDS in operand order (each lane's 16 codes become two 16-byte
// operand entries of the same lane: no bank conflicts either way), two
// granules ahead of their use (and asked for three ahead), and every wave
// reads each operand once for its QT tiles. The scores of the next granule are
// formed in one straight run of code with the weights and values of this one,
// so that the matrix cores work while the vector units exponentiate.
//
// 2 x 2048 bf16 rows over 2048 cached tokens (32 heads of 128 over 8, e4m3):
// 206 GF in 228 to 239 us, 862 to 904 TFLOP/s, where a large f16 product
// reaches 1109. No unit is full (matrix cores 38 % of the cycles, vector issue
// 53 %, LDS 31 %): what bounds it is the order within a wave, products, then
// maxima and exponentials, then products, with two waves a SIMD to fill each
// other's gaps. f32 rows take two terms on both products: 5 x up to 1500 rows
// of 14 heads of 64 under a window of 512 take 45 us.
#include "pages_attention.h"

namespace ditch {

constexpr int RING = 3;    // granules in LDS
constexpr int META = 256;  // granules whose pages and scales are held in LDS

template <typename T, int KIND, int DK, int DV, int QT, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(DK <= 128 ? 2 : 1))) void pages_chunk_kernel(PagesAttention a, int tiles) {
    constexpr int KP = DK / 64, VU = DV / 32, TERMS = sizeof(T) == 4 ? 2 : 1;
    constexpr int UNITS = 2 * KP + VU;              // of a granule's codes, 1 KB each
    constexpr int PER = (UNITS + NW - 1) / NW;      // of a granule, a wave
    constexpr bool EVEN = UNITS % NW == 0;
    extern __shared__ __attribute__((aligned(16))) u32x4 ops[];  // [RING][2 UNITS][64]
    __shared__ int32_t id_s[META];
    __shared__ float key_s[META], bias_s[META], inverse_s[META];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    // Workgroups go to the 8 XCDs in turn. Each XCD takes whole heads, four at
    // a time (their keys and values share its L2), and the tiles with the most
    // keys first, so that the short ones fill the end.
    // (tiles 0: workgroups for the rows, the longest sequences' ends first)
    constexpr int QUERIES = 16 * QT * NW;
    const int heads = a.b.n_seqs * a.p.kv_heads, group = a.heads / a.p.kv_heads;
    int h, seq, tile;
    SeqRows r;
    if (tiles == 0) {
        const int per = (group + QUERIES - 1) / QUERIES;
        h = (int)(blockIdx.x % a.p.kv_heads);
        const int at = (int)(blockIdx.x / a.p.kv_heads), i = row_place(a.b, a.b.n_rows - 1 - at / per, seq, r);
        tile = (i * group + QUERIES - 1) / QUERIES + at % per;
        if (i < 0 || tile * QUERIES >= (i + 1) * group) return;
    } else {
        int head, rank;
        if (heads >= 8) {
            const int x = (int)(blockIdx.x % 8), j = (int)(blockIdx.x / 8);
            const int h0 = (int)((int64_t)heads * x / 8), h1 = (int)((int64_t)heads * (x + 1) / 8);
            const int set = j / (4 * tiles), first = h0 + 4 * set, many = h1 - first < 4 ? h1 - first : 4;
            if (many <= 0 || j - 4 * set * tiles >= many * tiles) return;
            head = first + (j - 4 * set * tiles) % many;
            rank = (j - 4 * set * tiles) / many;
        } else {
            head = (int)(blockIdx.x % heads);
            rank = (int)(blockIdx.x / heads);
        }
        h = head % a.p.kv_heads;
        seq = head / a.p.kv_heads;
        tile = tiles - 1 - rank;
        r = seq_rows(a.b, seq);
    }
    const int q0 = tile * QUERIES;  // the workgroup's first query
    if (q0 / group >= r.n) return;
    const int first_row = q0 / group, last_row = (q0 + QUERIES - 1) / group;
    if (last_row >= r.live) {  // rows past max_len
        for (int e = tid; e < QUERIES * a.p.vd; e += NW * 64) {
            const int qi = q0 + e / a.p.vd, i = qi / group;
            if (i >= r.live && i < r.n)
                ((T *)a.out.data)[(int64_t)(r.row + i) * a.out.stride + (int64_t)(h * group + qi % group) * a.p.vd +
                                  e % a.p.vd] = (T)NAN;
        }
    }
    if (first_row >= r.live) return;
    const TileRows tr = tile_rows(r, first_row, last_row, a.window, a.sinks);

    // the wave's tiles
    QueryTile<KP, TERMS> q[QT];
    float cq[QT], m[QT];
    float top = -INFINITY;
    bool far = false;
    double l[QT];
    Seen seen[QT];
    int lo[QT], hi[QT];  // positions of each tile's first and last live row
    floatx4 o[QT][DV / 16];
#pragma unroll
    for (int i = 0; i < QT; i++) {
        const int w0 = q0 + (wave * QT + i) * 16, qi = w0 + c;
        const int row = qi / group, ra = w0 / group, rz = (w0 + 15) / group;
        const bool mine = row < r.live;
        lo[i] = r.pos + ra;
        hi[i] = ra < r.live ? r.pos + (rz < r.live ? rz : r.live - 1) : -1;
        seen[i] = seen_from(mine ? r.pos + row : hi[i], a.window, a.sinks);
        RawQuery<KP> raw;
        load_query(raw, mine ? (const T *)a.q.data + (int64_t)(r.row + row) * a.q.stride +
                                   (int64_t)(h * group + qi % group) * a.p.hd
                             : (const T *)nullptr,
                   a.p.hd, g);
        query_terms(q[i], raw);
        cq[i] = a.scale * 1.4426950408889634f * q[i].down;
        m[i] = M_NONE;
        l[i] = 0;
#pragma unroll
        for (int d = 0; d < DV / 16; d++) o[i][d] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    const int per = a.p.page / GRANULE;
    const int64_t head_stride = (int64_t)a.p.kv_heads * a.p.page_bytes;
    const uint8_t *base = a.p.codes + (int64_t)h * a.p.page_bytes + lane * 16;
    u32x4 raw[PER];  // the wave's share of a granule's codes on their way
    auto fetch = [&](int b, int k) {
        const int64_t at = granule_index(tr, b + k) & (per - 1);
        const uint8_t *p = base + __builtin_amdgcn_readfirstlane(id_s[k]) * head_stride;
        const uint8_t *kp = p + at * (GRANULE * DK), *vp = p + (int64_t)a.p.page * DK + at * (GRANULE * DV);
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int u = wave + i * NW;
            // (known when compiled where the waves share the units evenly: no branch in the loop)
            const bool keys = 2 * KP % NW == 0 ? i < 2 * KP / NW : u < 2 * KP;
            if (EVEN || u < UNITS) raw[i] = *(const u32x4 *)(keys ? kp + u * 1024 : vp + (u - 2 * KP) * 1024);
        }
    };
    auto store = [&](int slot) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int u = wave + i * NW;
            if (EVEN || u < UNITS) {
                u32x4 *to = ops + ((slot * UNITS + u) * 2) * 64 + lane;
                to[0] = __builtin_bit_cast(u32x4, codes_f16<KIND>(raw[i][0], raw[i][1]));
                to[64] = __builtin_bit_cast(u32x4, codes_f16<KIND>(raw[i][2], raw[i][3]));
            }
        }
    };
    floatx4 s[QT][2];  // the coming granule's scores
    auto form_scores = [&](int slot) {
        const half8 *k = (const half8 *)(ops + slot * UNITS * 2 * 64) + lane;
#pragma unroll
        for (int i = 0; i < QT; i++) s[i][0] = s[i][1] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = 0; p < 2 * KP; p++) {
            const half8 k0 = k[p * 64], k1 = k[(2 * KP + p) * 64];
#pragma unroll
            for (int i = 0; i < QT; i++)
#pragma unroll
                for (int x = 0; x < TERMS; x++) {
                    s[i][0] = mfma_f16(k0, q[i].f[p / 2][p % 2][x], s[i][0]);
                    s[i][1] = mfma_f16(k1, q[i].f[p / 2][p % 2][x], s[i][1]);
                }
        }
    };
    // (w: this granule's exponents)
    auto add_values = [&](int slot, const float (&w)[QT][8], float inverse) {
        const half8 *v = (const half8 *)(ops + (slot * UNITS + 2 * KP) * 2 * 64) + lane;
        Weights<TERMS> wt[QT];
#pragma unroll
        for (int i = 0; i < QT; i++) l[i] += (double)(granule_weights<TERMS>(wt[i], w[i]) * inverse);
#pragma unroll
        for (int d = 0; d < DV / 16; d++) {
            const half8 x = v[d * 64];
#pragma unroll
            for (int i = 0; i < QT; i++)
#pragma unroll
                for (int e = 0; e < TERMS; e++) o[i][d] = mfma_f16(x, wt[i].f[e], o[i][d]);
        }
    };

    for (int b = 0; b < tr.granules; b += META) {
        const int n = tr.granules - b < META ? tr.granules - b : META;
        __syncthreads();
        for (int e = tid; e < n; e += NW * 64) {
            const int id = page_of(a.b, a.p, seq, granule_index(tr, b + e) / per), in = id < 0 ? 0 : id;
            float2 sc = *(const float2 *)(a.p.scales + ((int64_t)in * a.p.kv_heads + h) * 2);
            if (id < 0) sc = make_float2(NAN, NAN);  // a page outside the pool: page 0's codes under scales of NaN
            const GranuleScales gs = granule_scales(sc.x, sc.y);
            id_s[e] = in;
            key_s[e] = gs.key;
            bias_s[e] = gs.bias;
            inverse_s[e] = gs.inverse;
        }
        __syncthreads();
        fetch(b, 0);
        store(0);
        fetch(b, n > 1 ? 1 : 0);
        store(1);
        fetch(b, n > 2 ? 2 : 0);
        __syncthreads();
        form_scores(0);
        int slot = 0;
        // granule k: granule k + 2 to LDS, k + 3 on its way
#pragma unroll 1
        for (int k = 0; k < n; k++) {
            const int next = slot == RING - 1 ? 0 : slot + 1, after = next == RING - 1 ? 0 : next + 1;
            const int gi = granule_index(tr, b + k), a0 = gi * GRANULE, z0 = a0 + GRANULE - 1;
            auto uniform = [](float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x))); };
            const GranuleScales sc{uniform(key_s[k]), uniform(bias_s[k]), uniform(inverse_s[k])};
            float w[QT][8];
            bool full = true, more = false;
#pragma unroll
            for (int i = 0; i < QT; i++) {
                full &= z0 <= lo[i] && (!a.window || a0 > hi[i] - a.window || z0 < a.sinks);
                granule_exponents(w[i], s[i][0], s[i][1], cq[i] * sc.key, sc.bias + (W_UP - m[i]));
            }
            if (!full || far)
#pragma unroll
                for (int i = 0; i < QT; i++) {
                    if (far) far_exponents(w[i], s[i][0], s[i][1], cq[i] * sc.key, sc.bias, m[i]);
                    if (!full) granule_mask(w[i], a0 + 4 * g, seen[i]);
                }
#pragma unroll
            for (int i = 0; i < QT; i++) more |= most_of(w[i]) > W_MOST;
            if (__any(more)) {
                far = false;
#pragma unroll
                for (int i = 0; i < QT; i++) {
                    const float f = move_maximum(w[i], s[i][0], s[i][1], cq[i] * sc.key, sc.bias, full, a0 + 4 * g, seen[i], m[i]);
                    far |= maximum_far(m[i]);
                    l[i] *= (double)f * f;
#pragma unroll
                    for (int d = 0; d < DV / 16; d++) o[i][d] *= f * f;
                }
            }
            float inverse = sc.inverse;
            if (granule_odd<TERMS>(sc, top)) {
#pragma unroll
                for (int i = 0; i < QT; i++) l[i] += odd_granule(w[i], sc);
                inverse = 0.f;
            }
            // one straight run: behind the batch's last granules the scores and
            // the copies are of whatever is there, and not used. The wave that
            // feeds the matrix cores goes first: 235 -> 232 us and, of two
            // terms, 49 -> 46 us (the calls above)
            __builtin_amdgcn_s_setprio(1);
            form_scores(next);
            store(after);
            fetch(b, k + 3 < n ? k + 3 : n - 1);
            add_values(slot, w, inverse);
            __builtin_amdgcn_s_setprio(0);
            __syncthreads();
            slot = next;
        }
    }

#pragma unroll
    for (int i = 0; i < QT; i++) {
        const double norm = 1.0 / sum_groups(l[i]);
        const int qi = q0 + (wave * QT + i) * 16 + c, row = qi / group;
        if (row >= r.live) continue;
        T *out = (T *)a.out.data + (int64_t)(r.row + row) * a.out.stride + (int64_t)(h * group + qi % group) * a.p.vd;
#pragma unroll
        for (int d = 0; d < DV / 16; d++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (16 * d + 4 * g + j < a.p.vd) out[16 * d + 4 * g + j] = (T)(float)((double)o[i][d][j] * norm);
    }
}

// ---------------------------------------------------------------------------

// Two tiles a wave, four waves: with 2 x 2048 rows over 2048 cached tokens (32
// heads of 128 over 8, bf16, e4m3) 228 to 239 us; three tiles a wave 316 us, with one
// wave a SIMD left; eight waves 242 us there, but 78 us against 46 us with
// 5 x 1500 rows under a window; registers for three waves a SIMD (19 of them
// spilled) 323 us.
constexpr int CHUNK_TILES = 2, CHUNK_WAVES = 4;

// A workgroup here walks all of its keys by itself, so it takes enough of them
// to fill the chip; the few-row kernel, in tiles of 16 queries, splits the keys
// instead and is ahead below that. Both measured (int8, 32 heads of 128 over 8,
// bf16, us few-row / chunk): 1024 tiles of 16 (512 rows, 4000 cached) 102 / 135,
// 2048 (1024 rows, 2000 cached) 124 / 98, 2048 (8 x 128 rows, 1000 cached)
// 63 / 50, 4096 (32 x 64 rows, 200 cached) 69 / 36; 14 heads of 64 over 2: 896
// tiles 41 / 75, 1792 tiles 18 / 20 (past the border by so little that the
// rule, which knows neither the heads' size nor the keys, is 2 us behind).
// Under 64 queries a head half of a
// workgroup's lanes hold none.
bool pages_chunk_takes(const PoolView &p, const BatchView &b, int heads, int32_t dtype) {
    const int64_t queries = (int64_t)b.max_rows * (heads / p.kv_heads);
    return queries >= 64 && (int64_t)b.n_seqs * p.kv_heads * ((queries + 15) / 16) >= 1536;
}

template <typename T, int KIND, int DK, int DV>
static void chunk_dims(const PagesAttention &a, hipStream_t s) {
    constexpr int LDS = RING * (2 * (DK / 64) + DV / 32) * 2048;
    const int per = 16 * CHUNK_TILES * CHUNK_WAVES;
    const int64_t group = a.heads / a.p.kv_heads, queries = a.b.max_rows * group, heads = (int64_t)a.b.n_seqs * a.p.kv_heads;
    int64_t tiles = (queries + per - 1) / per, blocks = heads >= 8 ? (heads + 7) / 8 * 8 * tiles : heads * tiles;
    const int64_t by_rows = a.b.n_rows * ((group + per - 1) / per) * a.p.kv_heads;
    if (a.b.by_rows && by_rows < blocks) {
        tiles = 0;
        blocks = by_rows;
    }
    DITCH_CHECK(blocks < ((int64_t)1 << 24) && queries < ((int64_t)1 << 30), DITCH_INVALID_ARGUMENT, "kv attention: more work than one launch holds");
    auto *kernel = pages_chunk_kernel<T, KIND, DK, DV, CHUNK_TILES, CHUNK_WAVES>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(CHUNK_WAVES * 64), LDS, s, a, (int)tiles);
    DITCH_TRY_HIP(hipGetLastError());
}

template <typename T, int KIND>
static void chunk_kind(const PagesAttention &a, hipStream_t s) {
    if (a.p.dv == 256) chunk_dims<T, KIND, 256, 256>(a, s);
    else if (a.p.dv == 192) chunk_dims<T, KIND, 192, 192>(a, s);
    else if (a.p.dk == 192) chunk_dims<T, KIND, 192, 128>(a, s);
    else if (a.p.dv == 128) chunk_dims<T, KIND, 128, 128>(a, s);
    else chunk_dims<T, KIND, 64, 64>(a, s);
}

template <typename T>
static void chunk_typed(const PagesAttention &a, hipStream_t s) {
    if (a.p.kind == DITCH_KV_INT8) chunk_kind<T, DITCH_KV_INT8>(a, s);
    else chunk_kind<T, DITCH_KV_E4M3>(a, s);
}

void launch_pages_chunk(const PagesAttention &a, hipStream_t s) {
    if (a.dtype == DITCH_F32) chunk_typed<float>(a, s);
    else if (a.dtype == DITCH_F16) chunk_typed<_Float16>(a, s);
    else chunk_typed<__bf16>(a, s);
}

}  // namespace ditch
