// pages.hip — pages of 8-bit keys and values: appending rows (with the
// position rotation), reading them back, and reordering the beams' states.
#include <string>

#include "pages.h"

namespace ditch {

// ---------------------------------------------------------------------------
// checks

static int padded_dim(uint32_t d) { return (int)((d + 63) / 64 * 64); }

static bool shape_ok(const ditch_kv_pages *p) {
    if (!p || (p->kind != DITCH_KV_INT8 && p->kind != DITCH_KV_E4M3)) return false;
    if (p->layers == 0 || p->n_pages == 0 || p->n_pages > (uint32_t)INT32_MAX || p->kv_heads == 0 || p->kv_heads > 65535)
        return false;
    if (p->page_tokens != 32 && p->page_tokens != 64 && p->page_tokens != 128 && p->page_tokens != 256) return false;
    return p->head_dim > 0 && p->v_head_dim > 0 && p->head_dim <= 256 && p->v_head_dim <= 256;
}

// (layers, n_pages < 2^32 and 2^31, kv_heads <= 65535, page_bytes <= 2^17: checked against 2^63)
uint64_t pool_scales_bytes(const ditch_kv_pages *p) {
    if (!shape_ok(p)) return 0;
    const unsigned __int128 n = (unsigned __int128)p->layers * p->n_pages * p->kv_heads * 8;
    return n >> 62 ? 0 : (uint64_t)n;
}

uint64_t pool_codes_bytes(const ditch_kv_pages *p) {
    if (!shape_ok(p)) return 0;
    const unsigned __int128 n = (unsigned __int128)p->layers * p->n_pages * p->kv_heads * p->page_tokens *
                                (uint32_t)(padded_dim(p->head_dim) + padded_dim(p->v_head_dim));
    return n >> 62 ? 0 : (uint64_t)n;
}

PoolView pool_view(const ditch_kv_pages *p, uint32_t layer) {
    DITCH_CHECK(p, DITCH_INVALID_ARGUMENT, "kv pages: NULL pool");
    DITCH_CHECK(shape_ok(p) && pool_codes_bytes(p) > 0, DITCH_INVALID_ARGUMENT,
                "kv pages: the pool's kind or shape (pages of 32, 64, 128 or 256 tokens, head dims 1..256)");
    PoolView v{};
    v.dk = padded_dim(p->head_dim);
    v.dv = padded_dim(p->v_head_dim);
    DITCH_CHECK(v.dk == v.dv || (v.dk == 192 && v.dv == 128), DITCH_UNSUPPORTED,
                "kv pages: head_dim and v_head_dim of different size (other than 192 and 128)");
    DITCH_CHECK(p->codes && p->scales, DITCH_INVALID_ARGUMENT, "kv pages: NULL codes or scales");
    DITCH_CHECK((uintptr_t)p->codes % 16 == 0 && (uintptr_t)p->scales % 8 == 0, DITCH_INVALID_ARGUMENT,
                "kv pages: codes not aligned to 16 bytes or scales not to 8");
    DITCH_CHECK(p->codes_bytes >= pool_codes_bytes(p) && p->scales_bytes >= pool_scales_bytes(p),
                DITCH_INVALID_ARGUMENT, "kv pages: codes or scales shorter than the pool's shape");
    DITCH_CHECK(layer < p->layers, DITCH_INVALID_ARGUMENT, "kv pages: layer outside the pool");
    v.page = (int32_t)p->page_tokens;
    v.page_shift = __builtin_ctz(p->page_tokens);
    v.page_bytes = (int64_t)v.page * (v.dk + v.dv);
    v.kind = p->kind;
    v.n_pages = (int32_t)p->n_pages;
    v.kv_heads = (int32_t)p->kv_heads;
    v.hd = (int32_t)p->head_dim;
    v.vd = (int32_t)p->v_head_dim;
    v.codes = (uint8_t *)p->codes + (int64_t)layer * v.n_pages * v.kv_heads * v.page_bytes;
    v.scales = p->scales + (int64_t)layer * v.n_pages * v.kv_heads * 2;
    return v;
}

BatchView batch_view(const ditch_kv_batch *b, const PoolView &p) {
    DITCH_CHECK(b, DITCH_INVALID_ARGUMENT, "kv pages: NULL batch");
    DITCH_CHECK(b->n_rows <= (uint64_t)INT32_MAX && b->n_seqs <= (uint32_t)INT32_MAX &&
                    b->max_rows <= (uint32_t)INT32_MAX && b->max_len <= (uint32_t)INT32_MAX - 256,
                DITCH_INVALID_ARGUMENT, "kv pages: more rows, sequences or positions than 2^31");
    BatchView v{b->table, b->starts, b->pos, (int64_t)b->table_stride, (int32_t)b->n_seqs, (int32_t)b->n_rows,
                (int32_t)b->max_rows, (int32_t)b->max_len};
    if (v.n_seqs == 0 || v.n_rows == 0 || v.max_rows == 0 || v.max_len == 0) {
        v.n_seqs = 0;
        return v;
    }
    DITCH_CHECK(b->table && b->starts && b->pos, DITCH_INVALID_ARGUMENT, "kv pages: NULL table, starts or pos");
    DITCH_CHECK((uint64_t)b->table_stride * p.page >= (uint64_t)b->max_len, DITCH_INVALID_ARGUMENT,
                "kv pages: max_len beyond the page table's row");
    return v;
}

RowsView rows_view(const ditch_kv_rows *r, uint64_t n_rows, uint64_t width, int32_t dtype, const char *what) {
    const std::string name(what);
    DITCH_CHECK(dtype == DITCH_F32 || dtype == DITCH_F16 || dtype == DITCH_BF16, DITCH_INVALID_ARGUMENT,
                "kv pages: rows of f32, f16 or bf16");
    DITCH_CHECK(r, DITCH_INVALID_ARGUMENT, name + ": NULL rows");
    const uint64_t e = dtype == DITCH_F32 ? 4 : 2;
    if (n_rows == 0) return RowsView{r->data, (int64_t)r->stride};
    DITCH_CHECK(r->data && (uintptr_t)r->data % e == 0, DITCH_INVALID_ARGUMENT, name + ": NULL or misaligned rows");
    DITCH_CHECK(r->stride >= width && r->stride <= (uint64_t)1 << 40, DITCH_INVALID_ARGUMENT,
                name + ": row stride below the row's width");
    DITCH_CHECK((unsigned __int128)(n_rows - 1) * r->stride + width <= r->bytes / e, DITCH_INVALID_ARGUMENT,
                name + ": buffer shorter than its rows");
    return RowsView{r->data, (int64_t)r->stride};
}

static unsigned grid_blocks(int64_t n, const char *what) {
    // (a launch holds fewer than 2^32 threads, 256 a workgroup)
    DITCH_CHECK(n < ((int64_t)1 << 24), DITCH_INVALID_ARGUMENT, std::string(what) + ": more work than one launch holds");
    return (unsigned)n;
}

// ---------------------------------------------------------------------------
// device helpers

template <typename T>
__device__ __forceinline__ double row_value(const T *p) {
    if constexpr (sizeof(T) == 4) return (double)*p;
    else return (double)(float)*p;
}

// Coordinate d of a head rotated to its position (c, s: the position's row
// of the tables; half 0: as it is), in 64 bits: the codes are rounded once.
template <typename T>
__device__ __forceinline__ double rotated(const T *x, int d, int half, int style, const float *c, const float *s) {
    if (d >= 2 * half) return row_value(x + d);
    int i, a, b;
    bool second;
    if (style == DITCH_ROPE_NEOX) {
        second = d >= half;
        i = second ? d - half : d;
        a = i;
        b = i + half;
    } else {
        second = d & 1;
        i = d >> 1;
        a = 2 * i;
        b = a + 1;
    }
    const double xa = row_value(x + a), xb = row_value(x + b), cc = c[i], ss = s[i];
    return second ? xb * cc + xa * ss : xa * cc - xb * ss;
}

// The code nearest to y (ties to even), y within the code's range after the clamp.
template <int KIND>
__device__ __forceinline__ uint8_t nearest_code(double y) {
    constexpr double most = KIND == DITCH_KV_INT8 ? 127.0 : 448.0;
    y = fmin(fmax(y, -most), most);
    if constexpr (KIND == DITCH_KV_INT8) return (uint8_t)(int8_t)(int)rint(y);
    // e4m3: 3 bits behind the leading one, the least step 2^-9
    int e = (int)((__double_as_longlong(y) >> 52) & 0x7ff) - 1023;
    e = e < -6 ? -6 : e;
    const double up = __longlong_as_double((int64_t)(1023 + 3 - e) << 52);
    const double down = __longlong_as_double((int64_t)(1023 - 3 + e) << 52);
    const float v = (float)(rint(y * up) * down);  // a code's value: the conversion is exact
    return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xff);
}

template <int KIND>
__device__ __forceinline__ float code_value(uint8_t c) {
    if constexpr (KIND == DITCH_KV_INT8) return (float)(int8_t)c;
    return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
}

// ---------------------------------------------------------------------------
// append

struct AppendArgs {
    PoolView p;
    BatchView b;
    RowsView k, v, q, q_out;
    RopeView rope;
    int32_t slots;   // pages that a sequence's rows can touch
    int32_t heads;   // query heads (0: no queries)
    int64_t kv_blocks;
};

// A workgroup per (sequence, touched page, head, keys or values), then one
// per query row.
template <typename T, int KIND>
__global__ __launch_bounds__(256) void pages_append_kernel(AppendArgs a) {
    __shared__ double part[4];
    const int tid = threadIdx.x;
    int64_t blk = blockIdx.x;
    if (blk >= a.kv_blocks) {
        blk -= a.kv_blocks;
        const int seq = (int)(blk / a.b.max_rows), i = (int)(blk % a.b.max_rows);
        const SeqRows r = seq_rows(a.b, seq);
        if (i >= r.live) return;
        const T *src = (const T *)a.q.data + (r.row + i) * a.q.stride;
        T *dst = (T *)a.q_out.data + (r.row + i) * a.q_out.stride;
        const int half = a.rope.half, hd = a.p.hd;
        const float *c = a.rope.cos_t + (int64_t)(r.pos + i) * half, *s = a.rope.sin_t + (int64_t)(r.pos + i) * half;
        // a pair a thread: the rows may be the same
        const int pairs = half, rest = hd - 2 * half, per = pairs + rest;
        for (int e = tid; e < a.heads * per; e += 256) {
            const int h = e / per, j = e % per;
            const T *x = src + (int64_t)h * hd;
            T *y = dst + (int64_t)h * hd;
            if (j >= pairs) {
                y[pairs + j] = x[pairs + j];
                continue;
            }
            const int d0 = a.rope.style == DITCH_ROPE_NEOX ? j : 2 * j;
            const int d1 = a.rope.style == DITCH_ROPE_NEOX ? j + half : 2 * j + 1;
            const double y0 = rotated(x, d0, half, a.rope.style, c, s), y1 = rotated(x, d1, half, a.rope.style, c, s);
            y[d0] = (T)(float)y0;
            y[d1] = (T)(float)y1;
        }
        return;
    }
    const int which = (int)(blk & 1);
    blk >>= 1;
    const int h = (int)(blk % a.p.kv_heads);
    blk /= a.p.kv_heads;
    const int slot = (int)(blk % a.slots), seq = (int)(blk / a.slots);
    const SeqRows r = seq_rows(a.b, seq);
    const int page_index = (r.pos >> a.p.page_shift) + slot, t0 = page_index << a.p.page_shift;
    const int end = r.pos + r.live;
    if (r.live == 0 || t0 >= end) return;
    const int id = page_of(a.b, a.p, seq, page_index);
    if (id < 0) return;
    const int lo = r.pos > t0 ? r.pos - t0 : 0, hi = end - t0 < a.p.page ? end - t0 : a.p.page;  // new tokens [lo, hi)
    const int D = which ? a.p.vd : a.p.hd, DP = which ? a.p.dv : a.p.dk, half = which ? 0 : a.rope.half;
    const RowsView &rv = which ? a.v : a.k;
    const T *rows = (const T *)rv.data + (int64_t)(r.row + t0 + lo - r.pos) * rv.stride + (int64_t)h * D;
    const float *ct = a.rope.cos_t, *st = a.rope.sin_t;
    auto value = [&](int t, int d) -> double {  // new token lo + t
        const int64_t at = (int64_t)(t0 + lo + t) * half;
        return rotated(rows + t * rv.stride, d, half, a.rope.style, ct + at, st + at);
    };
    double most = 0;
    bool bad = false;
    for (int e = tid; e < (hi - lo) * D; e += 256) {
        const double y = fabs(value(e / D, e % D));
        bad |= !(y <= 3.4028234663852886e38);
        most = fmax(most, y);
    }
    if (bad) most = INFINITY;
    for (int o = 32; o > 0; o >>= 1) most = fmax(most, __shfl_xor(most, o, 64));
    if ((tid & 63) == 0) part[tid >> 6] = most;
    __syncthreads();
    most = fmax(fmax(part[0], part[1]), fmax(part[2], part[3]));
    float *sp = a.p.scales + ((int64_t)id * a.p.kv_heads + h) * 2 + which;
    const float before = lo > 0 ? *sp : 0.f;
    __syncthreads();  // every thread has read it
    float after = __fmul_rn((float)most, 1.f / code_most(KIND));
    after = before > after ? before : after;
    const bool poison = !(before <= 3.4028234663852886e38f) || !(after <= 3.4028234663852886e38f);
    if (poison) after = NAN;
    if (tid == 0) *sp = after;
    const double inverse = after > 0.f ? 1.0 / (double)after : 0.0;
    uint8_t *codes = a.p.codes + ((int64_t)id * a.p.kv_heads + h) * a.p.page_bytes + (which ? (int64_t)a.p.page * a.p.dk : 0);
    // the tokens that stay, to the new scale
    if (lo > 0 && after > before) {
        const double f = (double)before * inverse;
        for (int e = tid; e < lo * DP; e += 256) {
            const int o = which ? value_offset(e / DP, e % DP, DP) : key_offset(e / DP, e % DP, DP);
            codes[o] = nearest_code<KIND>((double)code_value<KIND>(codes[o]) * f);
        }
    }
    // the new ones, and zeros up to the end of a granule that they start
    const int fill = hi % GRANULE && hi / GRANULE * GRANULE >= lo ? (hi / GRANULE + 1) * GRANULE : hi;
    for (int e = tid; e < (fill - lo) * DP; e += 256) {
        const int t = e / DP, d = e % DP;
        const int o = which ? value_offset(lo + t, d, DP) : key_offset(lo + t, d, DP);
        codes[o] = t < hi - lo && d < D && !poison ? nearest_code<KIND>(value(t, d) * inverse) : 0;
    }
}

template <typename T>
static void append_typed(const AppendArgs &a, unsigned blocks, hipStream_t s) {
    if (a.p.kind == DITCH_KV_INT8)
        hipLaunchKernelGGL((pages_append_kernel<T, DITCH_KV_INT8>), dim3(blocks), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((pages_append_kernel<T, DITCH_KV_E4M3>), dim3(blocks), dim3(256), 0, s, a);
    DITCH_TRY_HIP(hipGetLastError());
}

void launch_pages_append(const PoolView &p, const BatchView &b, int32_t dtype, const RowsView &k, const RowsView &v,
                         const RopeView &rope, const RowsView *q, const RowsView *q_out, int heads, hipStream_t s) {
    if (b.n_seqs == 0) return;
    AppendArgs a{p, b, k, v, q ? *q : RowsView{}, q ? *q_out : RowsView{}, rope, 0, q ? heads : 0, 0};
    a.slots = (b.max_rows + p.page - 2) / p.page + 1;
    a.kv_blocks = (int64_t)b.n_seqs * a.slots * p.kv_heads * 2;
    const unsigned blocks = grid_blocks(a.kv_blocks + (q ? (int64_t)b.n_seqs * b.max_rows : 0), "kv append");
    if (dtype == DITCH_F32) append_typed<float>(a, blocks, s);
    else if (dtype == DITCH_F16) append_typed<_Float16>(a, blocks, s);
    else append_typed<__bf16>(a, blocks, s);
}

// ---------------------------------------------------------------------------
// read

struct ReadArgs {
    PoolView p;
    BatchView b;
    RowsView k, v;
};

template <typename T, int KIND>
__global__ __launch_bounds__(256) void pages_read_kernel(ReadArgs a) {
    int64_t blk = blockIdx.x;
    const int seq = (int)(blk / a.b.max_rows), i = (int)(blk % a.b.max_rows);
    const SeqRows r = seq_rows(a.b, seq);
    if (i >= r.live) return;
    const int pos = r.pos + i, id = page_of(a.b, a.p, seq, pos >> a.p.page_shift), t = pos & (a.p.page - 1);
    for (int which = 0; which < 2; which++) {
        const int D = which ? a.p.vd : a.p.hd, DP = which ? a.p.dv : a.p.dk;
        const RowsView &rv = which ? a.v : a.k;
        T *row = (T *)rv.data + (int64_t)(r.row + i) * rv.stride;
        for (int e = threadIdx.x; e < a.p.kv_heads * D; e += 256) {
            const int h = e / D, d = e % D;
            float x = NAN;
            if (id >= 0) {
                const int64_t ph = (int64_t)id * a.p.kv_heads + h;
                const uint8_t *codes = a.p.codes + ph * a.p.page_bytes + (which ? (int64_t)a.p.page * a.p.dk : 0);
                x = code_value<KIND>(codes[which ? value_offset(t, d, DP) : key_offset(t, d, DP)]) *
                    a.p.scales[ph * 2 + which];
            }
            row[e] = (T)x;
        }
    }
}

template <typename T>
static void read_typed(const ReadArgs &a, unsigned blocks, hipStream_t s) {
    if (a.p.kind == DITCH_KV_INT8)
        hipLaunchKernelGGL((pages_read_kernel<T, DITCH_KV_INT8>), dim3(blocks), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((pages_read_kernel<T, DITCH_KV_E4M3>), dim3(blocks), dim3(256), 0, s, a);
    DITCH_TRY_HIP(hipGetLastError());
}

void launch_pages_read(const PoolView &p, const BatchView &b, int32_t dtype, const RowsView &k, const RowsView &v,
                       hipStream_t s) {
    if (b.n_seqs == 0) return;
    const ReadArgs a{p, b, k, v};
    const unsigned blocks = grid_blocks((int64_t)b.n_seqs * b.max_rows, "kv read");
    if (dtype == DITCH_F32) read_typed<float>(a, blocks, s);
    else if (dtype == DITCH_F16) read_typed<_Float16>(a, blocks, s);
    else read_typed<__bf16>(a, blocks, s);
}

// ---------------------------------------------------------------------------
// fork

struct ForkArgs {
    uint8_t *codes;
    float *scales;
    int64_t layer_pages, head_bytes;  // pages a layer; bytes of one head's page
    int32_t page, n_pages, kv_heads;
    int32_t *table_out, *spare_out;
    const int32_t *table, *parents, *spare;
    const uint32_t *lens;
    int64_t table_stride;
    int32_t beams;
};

// The parent of the group's sequence c.
__device__ __forceinline__ int parent_of(const int32_t *parents, int64_t first, int c, int beams) {
    const int32_t p = parents[first + c];
    return (uint32_t)p < (uint32_t)beams ? p : c;
}

// A workgroup per (sequence, layer and head); those of the first layer and
// head write the sequence's table row and spare page too.
__global__ __launch_bounds__(256) void pages_fork_kernel(ForkArgs a) {
    const int64_t seq = blockIdx.x, g = seq / a.beams, first = g * a.beams;
    const int c = (int)(seq % a.beams);
    const int64_t len = a.lens[g], full = len / a.page, part = len % a.page;
    const int p = parent_of(a.parents, first, c, a.beams);
    const bool has = part && full < a.table_stride;
    // a child before this one has taken the parent's last page over
    bool copies = false;
    for (int e = 0; e < c && has; e++) copies |= parent_of(a.parents, first, e, a.beams) == p;
    const int32_t src = has ? a.table[(first + p) * a.table_stride + full] : -1, mine = a.spare[seq];
    if (blockIdx.y == 0) {
        for (int64_t j = threadIdx.x; j < a.table_stride; j += 256) {
            int32_t v = a.table[(j < full ? first + p : seq) * a.table_stride + j];
            if (has && j == full) v = copies ? mine : src;
            a.table_out[seq * a.table_stride + j] = v;
        }
        if (threadIdx.x == 0) {
            int32_t left = mine;
            if (copies) {
                // the n-th copying sequence of the group gets the page of the n-th childless one
                int nth = 0;
                for (int e = 0; e < c; e++) {
                    const int q = parent_of(a.parents, first, e, a.beams);
                    bool before = false;
                    for (int f = 0; f < e; f++) before |= parent_of(a.parents, first, f, a.beams) == q;
                    nth += before;
                }
                for (int e = 0; e < a.beams; e++) {
                    bool child = false;
                    for (int f = 0; f < a.beams; f++) child |= parent_of(a.parents, first, f, a.beams) == e;
                    if (!child && nth-- == 0) left = a.table[(first + e) * a.table_stride + full];
                }
            }
            a.spare_out[seq] = left;
        }
    }
    if (!copies || (uint32_t)src >= (uint32_t)a.n_pages || (uint32_t)mine >= (uint32_t)a.n_pages || src == mine) return;
    const int64_t layer = blockIdx.y / a.kv_heads, h = blockIdx.y % a.kv_heads;
    const int64_t from = (layer * a.layer_pages + src) * a.kv_heads + h, to = (layer * a.layer_pages + mine) * a.kv_heads + h;
    const int n = (int)(a.head_bytes / 16);
    const uint4 *cs = (const uint4 *)(a.codes + from * a.head_bytes);
    uint4 *cd = (uint4 *)(a.codes + to * a.head_bytes);
    for (int i = threadIdx.x; i < n; i += 256) cd[i] = cs[i];
    if (threadIdx.x < 2) a.scales[to * 2 + threadIdx.x] = a.scales[from * 2 + threadIdx.x];
}

void launch_pages_fork(const ditch_kv_pages *p, int32_t *table_out, int32_t *spare_out, const int32_t *table,
                       int64_t table_stride, const int32_t *parents, const int32_t *spare, const uint32_t *lens,
                       int64_t groups, int64_t beams, hipStream_t s) {
    const PoolView v = pool_view(p, 0);
    const int64_t lh = (int64_t)p->layers * v.kv_heads;
    DITCH_CHECK(lh <= 65535, DITCH_INVALID_ARGUMENT, "kv fork: more than 65535 layers x heads");
    const ForkArgs a{v.codes, v.scales, v.n_pages, v.page_bytes, v.page, v.n_pages, v.kv_heads, table_out, spare_out,
                     table, parents, spare, lens, table_stride, (int32_t)beams};
    hipLaunchKernelGGL(pages_fork_kernel, dim3(grid_blocks(groups * beams, "kv fork"), (unsigned)lh), dim3(256), 0, s, a);
    DITCH_TRY_HIP(hipGetLastError());
}

}  // namespace ditch
