// pages.hip — pages of 8-bit keys and values: appending rows (with the
// position rotation), reading them back, and reordering the beams' states.
#include <algorithm>
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
    BatchView v{b->table, b->starts, b->starts ? b->starts + 1 : nullptr, b->pos, nullptr, (int64_t)b->table_stride,
                (int32_t)b->n_seqs, (int32_t)b->n_rows, (int32_t)b->max_rows, (int32_t)b->max_len, 0};
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

// The most rows of a sequence that can have a place in the cache.
static int32_t most_rows(const BatchView &b) { return std::min(b.max_rows, std::min(b.max_len, b.n_rows)); }

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

// The codes nearest to y (ties to even; a scale below f32's normal range can
// leave a y past the largest code: that one). Four at a time: the conversions
// and their checks are what an append computes.
template <int KIND>
__device__ __forceinline__ uint32_t nearest_codes(const double (&y)[4]) {
    if constexpr (KIND == DITCH_KV_INT8) {
        int c[4];
#pragma unroll
        for (int j = 0; j < 4; j++) c[j] = min(max((int)rint(y[j]), -127), 127);
        return (c[0] & 0xff) | (c[1] & 0xff) << 8 | (c[2] & 0xff) << 16 | (uint32_t)c[3] << 24;
    } else {
        // e4m3: 3 bits behind the leading one, the least step 2^-9. Through f32
        // and the conversion instruction the value is rounded twice, which differs
        // from once only where the f32 value is half way between two codes (its
        // low 20 bits say so above 2^-6): there, and below, in 64 bits.
        float v[4];
        bool odd = false;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[j] = __builtin_amdgcn_fmed3f((float)y[j], -448.f, 448.f);
            odd |= (__float_as_uint(v[j]) & 0xfffffu) == 0x80000u || fabsf(v[j]) < 0.015625f;
        }
        if (odd) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const double z = fmin(fmax(y[j], -448.0), 448.0);
                int e = (int)((__double_as_longlong(z) >> 52) & 0x7ff) - 1023;
                e = e < -6 ? -6 : e;
                const double up = __longlong_as_double((int64_t)(1023 + 3 - e) << 52);
                const double down = __longlong_as_double((int64_t)(1023 - 3 + e) << 52);
                v[j] = (float)(rint(z * up) * down);  // a code's value: the conversion is exact
            }
        }
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], r, true);
        return (uint32_t)r;
    }
}

template <int KIND>
__device__ __forceinline__ float code_value(uint8_t c) {
    if constexpr (KIND == DITCH_KV_INT8) return (float)(int8_t)c;
    return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
}

// ---------------------------------------------------------------------------
// append
//
// The new tokens of a (page, head), keys or values, belong to one workgroup.
// It forms every value in 64 bits twice: for the largest, which gives the
// scale, and, the rows by then in the caches, for the codes, which it puts in
// the page's order in LDS; whole granules go out, and the one that holds
// tokens of before came in first. (Staging the values themselves needs four to
// eight times the LDS and took 233 us where this takes 85: 24 sequences
// of up to 500 f32 rows of 8 heads of 128 and 32 query heads.) That call moves
// 314 MB, 239 of them the queries: 79 us, 4.0 TB/s; the keys and values alone
// take half of that, bound by the operations of the conversions in 64 bits. One
// row for each of 64 sequences takes 7 us, the latency of a chain of table,
// scale, the page's codes of before (rounded again where the scale grows) and
// the stores.

constexpr int TILE = 16384;  // codes staged (the page in parts where it has more)

struct AppendArgs {
    PoolView p;
    BatchView b;
    RowsView k, v, q, q_out;
    RopeView rope;
    int32_t slots;   // pages that a sequence's rows can touch (0: workgroups for the rows)
    int32_t heads;   // query heads (0: no queries)
    int32_t q_parts; // workgroups a query row
    int64_t kv_blocks;
};

// Four consecutive elements, or as many as `n` of them.
template <typename T>
__device__ __forceinline__ void load4(float (&v)[4], const T *p, bool whole, int n) {
    if (whole) {
        typedef T vec __attribute__((ext_vector_type(4)));
        const vec x = *(const vec *)p;
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = (float)x[j];
    } else
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = j < n ? (float)p[j] : 0.f;
}
template <typename T>
__device__ __forceinline__ void store4(T *p, const float (&v)[4], bool whole, int n) {
    if (whole) {
        typedef T vec __attribute__((ext_vector_type(4)));
        vec x;
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = (T)v[j];
        *(vec *)p = x;
    } else
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (j < n) p[j] = (T)v[j];
}
// Rows of quads of T that may be moved whole.
template <typename T>
__device__ __forceinline__ bool quads_ok(const RowsView &r, int dim) {
    return dim % 4 == 0 && r.stride % 4 == 0 && (uintptr_t)r.data % (4 * sizeof(T)) == 0;
}

// One query row's heads [part, + q_parts, ...) rotated; four pairs a thread.
template <typename T>
__device__ __forceinline__ void rotate_queries(const AppendArgs &a, const SeqRows &r, int i, int part) {
    const T *src = (const T *)a.q.data + (int64_t)(r.row + i) * a.q.stride;
    T *dst = (T *)a.q_out.data + (int64_t)(r.row + i) * a.q_out.stride;
    const int half = a.rope.half, hd = a.p.hd;
    const float *c = a.rope.cos_t + (int64_t)(r.pos + i) * half, *s = a.rope.sin_t + (int64_t)(r.pos + i) * half;
    const bool fours = half % 4 == 0 && quads_ok<T>(a.q, hd) && quads_ok<T>(a.q_out, hd);
    const int n_pairs = (half + 3) / 4, n_rest = (hd - 2 * half + 3) / 4, per = n_pairs + n_rest;
    const bool table = half % 4 == 0 && ((uintptr_t)a.rope.cos_t | (uintptr_t)a.rope.sin_t) % 16 == 0;
#pragma unroll 2
    for (int e = part * 256 + threadIdx.x; e < a.heads * per; e += a.q_parts * 256) {
        const int h = e / per, j = e % per;
        const T *x = src + (int64_t)h * hd;
        T *y = dst + (int64_t)h * hd;
        float u[4], w[4];
        if (j >= n_pairs) {
            const int d = 2 * half + (j - n_pairs) * 4;
            load4(u, x + d, fours, hd - d);
            store4(y + d, u, fours, hd - d);
            continue;
        }
        const int i0 = 4 * j, n = half - i0;
        float cc[4], ss[4];
        load4(cc, c + i0, table, n);
        load4(ss, s + i0, table, n);
        if (a.rope.style == DITCH_ROPE_NEOX) {
            load4(u, x + i0, fours, n);
            load4(w, x + half + i0, fours, n);
            float yu[4], yw[4];
#pragma unroll
            for (int z = 0; z < 4; z++) {
                const double p = u[z], q = w[z], co = cc[z], si = ss[z];
                yu[z] = (float)(p * co - q * si);
                yw[z] = (float)(q * co + p * si);
            }
            store4(y + i0, yu, fours, n);
            store4(y + half + i0, yw, fours, n);
        } else {
            load4(u, x + 2 * i0, fours, 2 * n);
            load4(w, x + 2 * i0 + 4, fours, 2 * n - 4);
            float yu[4], yw[4];
#pragma unroll
            for (int z = 0; z < 2; z++) {
                const double p = u[2 * z], q = u[2 * z + 1], co = cc[z], si = ss[z];
                yu[2 * z] = (float)(p * co - q * si);
                yu[2 * z + 1] = (float)(q * co + p * si);
                const double p2 = w[2 * z], q2 = w[2 * z + 1], co2 = cc[2 + z], si2 = ss[2 + z];
                yw[2 * z] = (float)(p2 * co2 - q2 * si2);
                yw[2 * z + 1] = (float)(q2 * co2 + p2 * si2);
            }
            store4(y + 2 * i0, yu, fours, 2 * n);
            store4(y + 2 * i0 + 4, yw, fours, 2 * n - 4);
        }
    }
}

// Calls f(t, d, n, y) for the values y[0..n) of every new token t in [z0, z1)
// and dims d, d + 1, ..: keys, rotated. x: the rows (token 0's), at: token 0's
// position.
template <typename T, typename F>
__device__ __forceinline__ void each_key(const T *x, int64_t stride, bool quads, int z0, int z1, int D, const RopeView &rope,
                                         int64_t at, F &&f) {
    const int half = rope.half;
    if (half % 4 == 0 && quads) {
        const int pairs = half / 4, per = pairs + (D - 2 * half) / 4;
        const bool table = ((uintptr_t)rope.cos_t | (uintptr_t)rope.sin_t) % 16 == 0, neox = rope.style == DITCH_ROPE_NEOX;
        for (int e = threadIdx.x; e < (z1 - z0) * per; e += 256) {
            const int t = z0 + e / per, j = e % per;
            const T *row = x + (int64_t)t * stride;
            float u[4], w[4];
            if (j >= pairs) {
                const int d = 2 * half + (j - pairs) * 4;
                load4(u, row + d, true, 4);
                const double y[4] = {u[0], u[1], u[2], u[3]};
                f(t, d, 4, y);
                continue;
            }
            const int i0 = 4 * j, du = neox ? i0 : 2 * i0, dw = neox ? half + i0 : 2 * i0 + 4;
            float cc[4], ss[4];
            load4(u, row + du, true, 4);
            load4(w, row + dw, true, 4);
            load4(cc, rope.cos_t + (at + t) * half + i0, table, 4);
            load4(ss, rope.sin_t + (at + t) * half + i0, table, 4);
            double yu[4], yw[4];
            if (neox) {
#pragma unroll
                for (int z = 0; z < 4; z++) {
                    const double p = u[z], q = w[z], co = cc[z], si = ss[z];
                    yu[z] = p * co - q * si;
                    yw[z] = q * co + p * si;
                }
            } else {
#pragma unroll
                for (int z = 0; z < 4; z++) {
                    const float *v = z < 2 ? u : w;
                    double *y = z < 2 ? yu : yw;
                    const double p = v[z % 2 * 2], q = v[z % 2 * 2 + 1], co = cc[z], si = ss[z];
                    y[z % 2 * 2] = p * co - q * si;
                    y[z % 2 * 2 + 1] = q * co + p * si;
                }
            }
            f(t, du, 4, yu);
            f(t, dw, 4, yw);
        }
    } else {
        for (int e = threadIdx.x; e < (z1 - z0) * D; e += 256) {
            const int t = z0 + e / D, d = e % D;
            const int64_t row = (at + t) * half;
            const double y[4] = {rotated(x + (int64_t)t * stride, d, half, rope.style, rope.cos_t + row, rope.sin_t + row)};
            f(t, d, 1, y);
        }
    }
}

// A workgroup per (sequence, touched page, head, keys or values), then those
// of the query rows.
// Five waves a SIMD: four, with two registers more, took 7 us longer for the
// 24 sequences above; six and eight, which spill, 2 and 14 us.
template <typename T, int KIND>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(5))) void pages_append_kernel(AppendArgs a) {
    __shared__ double part[4];
    __shared__ __attribute__((aligned(16))) uint8_t tile[TILE];
    const int tid = threadIdx.x;
    int64_t blk = blockIdx.x;
    if (blk >= a.kv_blocks) {
        blk -= a.kv_blocks;
        const int q_part = (int)(blk % a.q_parts), row = (int)(blk / a.q_parts);
        // the row's sequence: the last whose rows start at or before it, 64 candidates at a time
        int seq = 0, span = a.b.n_seqs;
        if (a.b.rows) {
            const uint32_t of = a.b.rows[row].b;
            if (of >= (uint32_t)a.b.n_seqs) return;
            seq = (int)of;
            span = 1;
        }
        while (span > 1) {
            const int step = (span + 63) / 64, at = seq + (tid & 63) * step;
            const uint64_t before = __ballot(at < seq + span && a.b.starts[at < seq + span ? at : seq] <= (uint32_t)row);
            if (!before) return;
            const int last = 63 - __builtin_clzll(before), end = seq + span;
            seq += last * step;
            span = end - seq < step ? end - seq : step;
        }
        const SeqRows r = seq_rows(a.b, seq);
        const int i = row - r.row;
        if (i < 0) return;
        if (i < r.live) rotate_queries<T>(a, r, i, q_part);
        return;
    }
    const int which = (int)(blk & 1);
    blk >>= 1;
    const int h = (int)(blk % a.p.kv_heads);
    blk /= a.p.kv_heads;
    int seq, page_index;
    SeqRows r;
    if (a.slots) {
        seq = (int)(blk / a.slots);
        r = seq_rows(a.b, seq);
        page_index = (r.pos >> a.p.page_shift) + (int)(blk % a.slots);
    } else {
        const int i = row_place(a.b, (int)blk, seq, r);
        // (the page's first new row)
        if (i < 0 || i >= r.live || (i > 0 && ((r.pos + i) & (a.p.page - 1)))) return;
        page_index = (r.pos + i) >> a.p.page_shift;
    }
    const int end = r.pos + r.live;
    // (by the page: its first position may lie past 2^31)
    if (r.live == 0 || page_index > (end - 1) >> a.p.page_shift) return;
    const int t0 = page_index << a.p.page_shift;
    const int id = page_of(a.b, a.p, seq, page_index);
    if (id < 0) return;
    const int lo = r.pos > t0 ? r.pos - t0 : 0, hi = end - t0 < a.p.page ? end - t0 : a.p.page;  // new tokens [lo, hi)
    const int D = which ? a.p.vd : a.p.hd, DP = which ? a.p.dv : a.p.dk;
    const RowsView &rv = which ? a.v : a.k;
    const T *rows = (const T *)rv.data + (int64_t)(r.row + (t0 - r.pos)) * rv.stride + (int64_t)h * D;  // token 0's
    float *sp = a.p.scales + ((int64_t)id * a.p.kv_heads + h) * 2 + which;
    const float before = lo > 0 ? *sp : 0.f;
    const bool quads = quads_ok<T>(rv, D);

    double most = 0;
    bool bad = false;
    auto largest = [&](double y) {
        bad |= !(fabs(y) <= 3.4028234663852886e38);
        most = fmax(most, fabs(y));
    };
    float most_value = 0;  // (a value is an f32: no rotation)
    auto largest_value = [&](float y) {
        bad |= !(fabsf(y) <= 3.4028234663852886e38f);
        most_value = fmaxf(most_value, fabsf(y));
    };
    if (which == 0) {
        each_key(rows, rv.stride, quads, lo, hi, D, a.rope, t0, [&](int t, int d, int n, const double *y) {
            for (int j = 0; j < n; j++) largest(y[j]);
        });
    } else if (quads) {
        const int per = D / 4;
#pragma unroll 2
        for (int e = tid; e < (hi - lo) * per; e += 256) {
            float v[4];
            load4(v, rows + (int64_t)(lo + e / per) * rv.stride + e % per * 4, true, 4);
#pragma unroll
            for (int j = 0; j < 4; j++) largest_value(v[j]);
        }
    } else {
        for (int e = tid; e < (hi - lo) * D; e += 256) largest_value((float)rows[(int64_t)(lo + e / D) * rv.stride + e % D]);
    }
    if (which) most = (double)most_value;
    if (bad) most = INFINITY;
    for (int o = 32; o > 0; o >>= 1) most = fmax(most, __shfl_xor(most, o, 64));
    if ((tid & 63) == 0) part[tid >> 6] = most;
    __syncthreads();
    most = fmax(fmax(part[0], part[1]), fmax(part[2], part[3]));
    float after = __fmul_rn((float)most, 1.f / code_most(KIND));
    after = before > after ? before : after;
    const bool poison = !(before <= 3.4028234663852886e38f) || !(after <= 3.4028234663852886e38f);
    if (poison) after = NAN;
    if (tid == 0) *sp = after;  // (every thread has read it: the barrier above)
    const double inverse = after > 0.f ? 1.0 / (double)after : 0.0;
    const bool grown = lo > 0 && after > before;
    const double f = grown ? (double)before * inverse : 0.0;
    uint8_t *codes = a.p.codes + ((int64_t)id * a.p.kv_heads + h) * a.p.page_bytes + (which ? (int64_t)a.p.page * a.p.dk : 0);

    // the granules to write: from the first that changes to the end of the one
    // that holds the last new token (what it has behind that, zeros where the
    // new tokens start it, is dead)
    const int room = DP <= 64 ? 256 : DP <= 128 ? 128 : 64, CT = room < a.p.page ? room : a.p.page;
    const int z_first = grown ? 0 : lo / GRANULE * GRANULE, z_last = (hi + GRANULE - 1) / GRANULE * GRANULE;
    for (int c0 = z_first; c0 < z_last; c0 += CT) {
        const int c1 = c0 + CT < z_last ? c0 + CT : z_last, n0 = c0 > lo ? c0 : lo, n1 = c1 < hi ? c1 : hi;
        uint4 *page = (uint4 *)(codes + (int64_t)c0 * DP);
        for (int u = tid; u < (c1 - c0) * DP / 16; u += 256) {
            union {
                uint4 q;
                uint8_t b[16];
                uint32_t d[4];
            } w;
            w.q = make_uint4(0, 0, 0, 0);
            if (c0 + u * 16 / (GRANULE * DP) * GRANULE < lo) {  // the granule holds tokens of before
                w.q = page[u];
                if (grown) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        double y[4];
#pragma unroll
                        for (int z = 0; z < 4; z++) y[z] = (double)code_value<KIND>(w.b[4 * j + z]) * f;
                        w.d[j] = nearest_codes<KIND>(y);
                    }
                }
            }
            ((uint4 *)tile)[u] = w.q;
        }
        __syncthreads();
        auto code = [&](const double (&y)[4]) {
            const double z[4] = {y[0] * inverse, y[1] * inverse, y[2] * inverse, y[3] * inverse};
            return poison ? 0u : nearest_codes<KIND>(z);
        };
        if (which == 0) {
            each_key(rows, rv.stride, quads, n0, n1, D, a.rope, t0, [&](int t, int d, int n, const double *y) {
                uint8_t *at = tile + key_offset(t - c0, d, DP);
                if (n == 4) *(uint32_t *)at = code({y[0], y[1], y[2], y[3]});
                else *at = (uint8_t)code({y[0], 0.0, 0.0, 0.0});
            });
        } else {
            // a dim of four tokens that lie next to each other in the page
            const int q0 = n0 / 4, q1 = (n1 + 3) / 4;
#pragma unroll 2
            for (int e = tid; e < (q1 - q0) * D; e += 256) {
                const int t = (q0 + e / D) * 4, d = e % D;
                double y[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const bool in = t + j >= n0 && t + j < n1;
                    y[j] = in ? (double)(float)rows[(int64_t)(t + j) * rv.stride + d] : 0.0;
                }
                const uint32_t c = code(y);
                uint8_t *at = tile + value_offset(t - c0, d, DP);
                if (t >= n0 && t + 4 <= n1) *(uint32_t *)at = c;
                else
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (t + j >= n0 && t + j < n1) at[j] = (uint8_t)(c >> 8 * j);
            }
        }
        __syncthreads();
        for (int u = tid; u < (c1 - c0) * DP / 16; u += 256) page[u] = ((const uint4 *)tile)[u];
        __syncthreads();
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
    AppendArgs a{p, b, k, v, q ? *q : RowsView{}, q ? *q_out : RowsView{}, rope, 0, q ? heads : 0, 1, 0};
    a.b.max_rows = most_rows(b);
    a.slots = (a.b.max_rows + p.page - 2) / p.page + 1;
    if (b.by_rows && b.n_rows < (int64_t)b.n_seqs * a.slots) a.slots = 0;
    a.kv_blocks = (a.slots ? (int64_t)b.n_seqs * a.slots : b.n_rows) * p.kv_heads * 2;
    // a row's heads over several workgroups until the rows fill the chip, a
    // thread a pair of quads or a quad that stays as it is (see rotate_queries)
    const int64_t rows = b.n_rows, quads = (rope.half + 3) / 4 + (p.hd - 2 * rope.half + 3) / 4;
    if (q && rows < 1024) a.q_parts = (int)std::min<int64_t>((heads * quads + 255) / 256, 1024 / rows + 1);
    const unsigned blocks = grid_blocks(a.kv_blocks + (q ? rows * a.q_parts : 0), "kv append");
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
    int32_t granules;  // that a sequence's rows can touch
};

// A workgroup per (sequence, granule, head, keys or values): its units
// decoded into LDS rows, which go out as rows: both sides of the transposition
// in 16-byte accesses. 7291 f32 rows of 8 heads of 128, 75 MB, in 20 us, 3.8 TB/s;
// up to 64 of 64 sequences 9 us: a workgroup's 4 KB are loaded, transposed and
// stored one after the other, and what the others do meanwhile does not fill
// the memory.
template <typename T, int KIND>
__global__ __launch_bounds__(256) void pages_read_kernel(ReadArgs a) {
    extern __shared__ __attribute__((aligned(16))) float tile[];  // [GRANULE][DP + 4]
    const int tid = threadIdx.x;
    int64_t blk = blockIdx.x;
    const int which = (int)(blk & 1);
    blk >>= 1;
    const int h = (int)(blk % a.p.kv_heads);
    blk /= a.p.kv_heads;
    const int slot = (int)(blk % a.granules), seq = (int)(blk / a.granules);
    const SeqRows r = seq_rows(a.b, seq);
    const int gi = r.pos / GRANULE + slot, end = r.pos + r.live;
    if (r.live == 0 || gi > (end - 1) / GRANULE) return;
    const int t0 = gi * GRANULE;
    const int id = page_of(a.b, a.p, seq, t0 >> a.p.page_shift);
    const int D = which ? a.p.vd : a.p.hd, DP = which ? a.p.dv : a.p.dk, S = DP + 4;
    const float scale = id < 0 ? NAN : a.p.scales[((int64_t)id * a.p.kv_heads + h) * 2 + which];
    const int lo = r.pos > t0 ? r.pos - t0 : 0, hi = end - t0 < GRANULE ? end - t0 : GRANULE;
    const uint8_t *codes = a.p.codes + ((int64_t)(id < 0 ? 0 : id) * a.p.kv_heads + h) * a.p.page_bytes +
                           (which ? (int64_t)a.p.page * a.p.dk : 0) + (int64_t)(t0 & (a.p.page - 1)) * DP;
    for (int u = tid; u < 2 * DP; u += 256) {  // GRANULE * DP / 16 units
        union {
            uint4 q;
            uint8_t b[16];
        } w;
        w.q = *(const uint4 *)(codes + u * 16);
        float x[16];
#pragma unroll
        for (int j = 0; j < 16; j++) x[j] = id < 0 ? NAN : code_value<KIND>(w.b[j]) * scale;
        if (which == 0) {
            const int t = u / (DP / 64 * 64) * 16 + u % 16, d = u / 64 % (DP / 64) * 64 + u / 16 % 4 * 16;
#pragma unroll
            for (int j = 0; j < 16; j += 4) *(float4 *)&tile[t * S + d + j] = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
        } else {
            const int d = u / 64 * 32 + u % 16, t = u / 16 % 4 * 4;
#pragma unroll
            for (int j = 0; j < 16; j++) tile[(t + (j & 4 ? 16 : 0) + (j & 3)) * S + d + (j & 8 ? 16 : 0)] = x[j];
        }
    }
    __syncthreads();
    const RowsView &rv = which ? a.v : a.k;
    T *rows = (T *)rv.data + (int64_t)(r.row + (t0 - r.pos)) * rv.stride + (int64_t)h * D;
    const bool quads = quads_ok<T>(rv, D);
    const int per = (D + 3) / 4;
    for (int e = tid; e < (hi - lo) * per; e += 256) {
        const int t = lo + e / per, d = e % per * 4;
        const float4 f = *(const float4 *)&tile[t * S + d];
        const float v[4] = {f.x, f.y, f.z, f.w};
        store4(rows + (int64_t)t * rv.stride + d, v, quads, D - d);
    }
}

template <typename T>
static void read_typed(const ReadArgs &a, unsigned blocks, hipStream_t s) {
    const unsigned lds = GRANULE * (std::max(a.p.dk, a.p.dv) + 4) * 4;
    if (a.p.kind == DITCH_KV_INT8)
        hipLaunchKernelGGL((pages_read_kernel<T, DITCH_KV_INT8>), dim3(blocks), dim3(256), lds, s, a);
    else
        hipLaunchKernelGGL((pages_read_kernel<T, DITCH_KV_E4M3>), dim3(blocks), dim3(256), lds, s, a);
    DITCH_TRY_HIP(hipGetLastError());
}

void launch_pages_read(const PoolView &p, const BatchView &b, int32_t dtype, const RowsView &k, const RowsView &v,
                       hipStream_t s) {
    if (b.n_seqs == 0) return;
    ReadArgs a{p, b, k, v, 0};
    a.b.max_rows = most_rows(b);
    a.granules = (a.b.max_rows + GRANULE - 2) / GRANULE + 1;
    const unsigned blocks = grid_blocks((int64_t)b.n_seqs * a.granules * p.kv_heads * 2, "kv read");
    if (dtype == DITCH_F32) read_typed<float>(a, blocks, s);
    else if (dtype == DITCH_F16) read_typed<_Float16>(a, blocks, s);
    else read_typed<__bf16>(a, blocks, s);
}

// ---------------------------------------------------------------------------
// fork

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
// 16-byte words that a workgroup copies: 32 a thread in flight. The last pages
// of 16 x 8 beams (32 layers of 8 heads of 128, 368 MB moved): 76 us the
// kernel; measured in one sitting, 92 us a call, with 16 a thread 102, with 8
// or fewer 105 to 112.
constexpr int FORK_PART = 8192;

struct ForkArgs {
    uint8_t *codes;
    float *scales;
    int64_t layer_pages, head_bytes;  // pages a layer; bytes of one head's page
    int32_t page, n_pages, kv_heads, parts;  // parts: workgroups a page of a layer
    int32_t *table_out, *spare_out;
    const int32_t *table, *parents, *spare;
    const uint32_t *lens;
    int64_t table_stride;
    int32_t beams;
};

// A workgroup per (sequence, layer, part of the page's heads); the first of a
// sequence writes its table row and spare page too. Lane e of every wave holds
// the parent of the group's sequence e, so the group's state is a few ballots.
__global__ __launch_bounds__(256) void pages_fork_kernel(ForkArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t seq = blockIdx.x, g = seq / a.beams, first = g * a.beams;
    const int c = (int)(seq % a.beams);
    const int32_t named = lane < a.beams ? a.parents[first + lane] : -1;
    const int64_t len = a.lens[g], full = len / a.page, part = len % a.page;
    const int parent = lane >= a.beams ? -1 : (uint32_t)named < (uint32_t)a.beams ? named : lane;
    const int p = __builtin_amdgcn_readlane(parent, c);
    const bool has = part && full < a.table_stride;
    // a child before this one has taken the parent's last page over
    const uint64_t before = ((uint64_t)1 << c) - 1;
    const bool copies = has && (__ballot(parent == p) & before);
    if (!copies && blockIdx.y) return;
    const int32_t src = has ? a.table[(first + p) * a.table_stride + full] : -1, mine = a.spare[seq];
    if (blockIdx.y == 0) {
#pragma unroll 1
        for (int64_t j = threadIdx.x; j < a.table_stride; j += 256) {
            int32_t v = a.table[(j < full ? first + p : seq) * a.table_stride + j];
            if (has && j == full) v = copies ? mine : src;
            a.table_out[seq * a.table_stride + j] = v;
        }
        // the n-th copying sequence of the group gets the page of the n-th childless one
        bool again = false, child = false;  // lane e: copies too; is a parent
#pragma unroll 1
        for (int e = 0; e < a.beams; e++) {
            const int q = __builtin_amdgcn_readlane(parent, e);
            again |= e < lane && q == parent;
            child |= q == lane;
        }
        const int nth = __popcll(__ballot(again && lane < a.beams) & before);
        uint64_t free = __ballot(!child && lane < a.beams);
#pragma unroll 1
        for (int e = 0; e < nth; e++) free &= free - 1;
        if (threadIdx.x == 0)
            a.spare_out[seq] = copies ? a.table[(first + __ffsll((unsigned long long)free) - 1) * a.table_stride + full] : mine;
    }
    if (!copies || (uint32_t)mine >= (uint32_t)a.n_pages || src == mine) return;
    // a page's heads lie next to each other: the workgroup's part of them
    const int64_t layer = blockIdx.y / a.parts, piece = blockIdx.y % a.parts;
    if ((uint32_t)src >= (uint32_t)a.n_pages) {  // no page to copy: NaN, as where it is looked for
        if (piece == 0)
            for (int i = threadIdx.x; i < 2 * a.kv_heads; i += 256)
                a.scales[(layer * a.layer_pages + mine) * a.kv_heads * 2 + i] = NAN;
        return;
    }
    const int64_t from = (layer * a.layer_pages + src) * a.kv_heads, to = (layer * a.layer_pages + mine) * a.kv_heads;
    const int64_t n = a.kv_heads * a.head_bytes / 16, p0 = piece * FORK_PART, left = n - p0 < FORK_PART ? n - p0 : FORK_PART;
    const u32x4_t *cs = (const u32x4_t *)(a.codes + from * a.head_bytes) + p0;
    u32x4_t *cd = (u32x4_t *)(a.codes + to * a.head_bytes) + p0;
    const int tid = threadIdx.x;
    if (left == FORK_PART) {
        u32x4_t v[FORK_PART / 256];
#pragma unroll
        for (int j = 0; j < FORK_PART / 256; j++) v[j] = cs[tid + 256 * j];
#pragma unroll
        for (int j = 0; j < FORK_PART / 256; j++) cd[tid + 256 * j] = v[j];
    } else {
#pragma unroll 4
        for (int i = tid; i < left; i += 256) cd[i] = cs[i];
    }
    if (piece == 0)
#pragma unroll 1
        for (int i = threadIdx.x; i < 2 * a.kv_heads; i += 256) a.scales[to * 2 + i] = a.scales[from * 2 + i];
}

void launch_pages_fork(const ditch_kv_pages *p, int32_t *table_out, int32_t *spare_out, const int32_t *table,
                       int64_t table_stride, const int32_t *parents, const int32_t *spare, const uint32_t *lens,
                       int64_t groups, int64_t beams, hipStream_t s) {
    const PoolView v = pool_view(p, 0);
    const int64_t parts = (v.kv_heads * v.page_bytes / 16 + FORK_PART - 1) / FORK_PART, lh = p->layers * parts;
    DITCH_CHECK(lh <= 65535, DITCH_INVALID_ARGUMENT, "kv fork: more than 65535 x 128 KB of layers a page");
    const ForkArgs a{v.codes, v.scales, v.n_pages, v.page_bytes, v.page, v.n_pages, v.kv_heads, (int32_t)parts, table_out, spare_out,
                     table, parents, spare, lens, table_stride, (int32_t)beams};
    hipLaunchKernelGGL(pages_fork_kernel, dim3(grid_blocks(groups * beams, "kv fork"), (unsigned)lh), dim3(256), 0, s, a);
    DITCH_TRY_HIP(hipGetLastError());
}

// ---------------------------------------------------------------------------
// a model's own cache in pages

// A workgroup a prompt, one more for the rows of no prompt: it looks all rows
// over once. A prompt's rows follow each other if they are as many as lie
// between its first and its last, and all as far from their indexes.
constexpr int ROWS_BATCH = 1024;
__global__ __launch_bounds__(ROWS_BATCH) void rows_batch_kernel(const ditch_row *rows, uint32_t n, uint32_t B, uint32_t max_len,
                                                                uint32_t *starts, uint32_t *ends, uint32_t *pos, float *x,
                                                                int64_t hidden) {
    __shared__ uint32_t part[5][ROWS_BATCH / 64];
    const uint32_t b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    auto mine = [&](uint32_t of) { return b < B ? of == b : of >= B; };
    // its first and last row, their number, the least and largest distance of a position from its index
    uint32_t lo = ~0u, hi = 0, many = 0, near = ~0u, far = 0;
#pragma unroll 4
    for (uint32_t i = tid; i < n; i += ROWS_BATCH) {
        const ditch_row r = rows[i];
        if (!mine(r.b)) continue;
        const uint32_t d = r.pos - i;
        lo = i < lo ? i : lo;
        hi = i;
        many++;
        near = d < near ? d : near;
        far = d > far ? d : far;
    }
    for (int o = 32; o > 0; o >>= 1) {
        lo = min(lo, (uint32_t)__shfl_xor(lo, o, 64));
        hi = max(hi, (uint32_t)__shfl_xor(hi, o, 64));
        many += __shfl_xor(many, o, 64);
        near = min(near, (uint32_t)__shfl_xor(near, o, 64));
        far = max(far, (uint32_t)__shfl_xor(far, o, 64));
    }
    if (lane == 0) {
        part[0][wave] = lo;
        part[1][wave] = hi;
        part[2][wave] = many;
        part[3][wave] = near;
        part[4][wave] = far;
    }
    __syncthreads();
    lo = near = ~0u;
    hi = many = far = 0;
    for (int w = 0; w < ROWS_BATCH / 64; w++) {
        lo = min(lo, part[0][w]);
        hi = max(hi, part[1][w]);
        many += part[2][w];
        near = min(near, part[3][w]);
        far = max(far, part[4][w]);
    }
    const bool ok = b < B && many && hi - lo + 1 == many && near == far;
    if (tid == 0 && b < B) {
        starts[b] = many ? lo : 0;
        ends[b] = ok ? hi + 1 : 0;
        pos[b] = ok ? near + lo : max_len;
    }
    // (the last: of one that ends within the cache every row has a place)
    if (!many || (ok && near + hi < max_len && near + lo <= near + hi)) return;
    for (uint32_t i = wave; i < n; i += ROWS_BATCH / 64)
        if (mine(rows[i].b) && !(ok && rows[i].pos < max_len))
            for (int64_t d = lane; d < hidden; d += 64) x[i * hidden + d] = NAN;
}

__global__ __launch_bounds__(256) void own_pages_kernel(int32_t *table, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) table[i] = (int32_t)i;
}

void launch_rows_batch(const ditch_row *rows, int64_t n, int64_t B, int64_t max_len, uint32_t *starts, uint32_t *ends,
                       uint32_t *pos, float *x, int64_t hidden, hipStream_t s) {
    hipLaunchKernelGGL(rows_batch_kernel, dim3((unsigned)(B + 1)), dim3(ROWS_BATCH), 0, s, rows, (uint32_t)n, (uint32_t)B,
                       (uint32_t)max_len, starts, ends, pos, x, hidden);
    DITCH_TRY_HIP(hipGetLastError());
}

void launch_own_pages(int32_t *table, int64_t n, hipStream_t s) {
    hipLaunchKernelGGL(own_pages_kernel, dim3(grid_blocks((n + 255) / 256, "kv cache")), dim3(256), 0, s, table, n);
    DITCH_TRY_HIP(hipGetLastError());
}

}  // namespace ditch
