// pages.h — paged 8-bit keys and values: the pool's layout and the batch's
// rows as the kernels see them (pages.hip, pages_attention.hip).
#pragma once
#include "internal.h"

namespace ditch {

// One layer of a pool (ditch_kv_pages), checked on the host.
struct PoolView {
    uint8_t *codes;      // [n_pages][kv_heads][page_bytes]
    float *scales;       // [n_pages][kv_heads][2]
    int64_t page_bytes;  // of one head: page * (dk + dv)
    int32_t kind;
    int32_t n_pages, page, page_shift, kv_heads;
    int32_t hd, vd;      // head dims
    int32_t dk, dv;      // as stored: rounded up to multiples of 64
};

// The batch (ditch_kv_batch), checked on the host as far as it can be; or a
// forward's, whose sequences lie in any order: `ends` are then its own, and
// `rows` (else NULL) say whose a row is. Where max_rows is no more than the
// number of rows (by_rows), a grid of sequences x max_rows grows with its
// square; launches may then have workgroups for the rows instead, of which
// the first row of a tile or page finds work.
struct BatchView {
    const int32_t *table;
    const uint32_t *starts, *ends, *pos;
    const ditch_row *rows;
    int64_t table_stride;
    int32_t n_seqs, n_rows, max_rows, max_len, by_rows;
};

struct RowsView {
    void *data;
    int64_t stride;  // elements
};

struct RopeView {
    const float *cos_t, *sin_t;
    int32_t half, style;
};

// A sequence's rows: `n` of them from row `row` on, the first at position
// `pos`; the first `live` lie below max_len.
struct SeqRows {
    int32_t row, n, live, pos;
};

__device__ __forceinline__ SeqRows seq_rows(const BatchView &b, int s) {
    const uint32_t lo = b.starts[s], hi = b.ends[s], pos = b.pos[s];
    SeqRows r{0, 0, 0, 0};
    if (lo >= (uint32_t)b.n_rows || hi <= lo) return r;
    uint32_t n = hi - lo;
    n = n < (uint32_t)b.max_rows ? n : (uint32_t)b.max_rows;
    n = n < (uint32_t)b.n_rows - lo ? n : (uint32_t)b.n_rows - lo;
    r.row = (int32_t)lo;
    r.n = (int32_t)n;
    if (pos < (uint32_t)b.max_len) {
        const uint32_t room = (uint32_t)b.max_len - pos;
        r.live = (int32_t)(n < room ? n : room);
        r.pos = (int32_t)pos;
    }
    return r;
}

// The sequence of row `row` of a batch with `rows`, and the row's place in it;
// -1 for none.
__device__ __forceinline__ int32_t row_place(const BatchView &b, int row, int &seq, SeqRows &r) {
    const uint32_t of = b.rows[row].b;
    if (of >= (uint32_t)b.n_seqs) return -1;
    seq = (int)of;
    r = seq_rows(b, seq);
    const int i = row - r.row;
    return i >= 0 && i < r.n ? i : -1;
}

// The page that holds position page_index * page .. of sequence s; -1 when
// the table names none of the pool.
__device__ __forceinline__ int32_t page_of(const BatchView &b, const PoolView &p, int s, int page_index) {
    const int32_t id = b.table[(int64_t)s * b.table_stride + page_index];
    return (uint32_t)id < (uint32_t)p.n_pages ? id : -1;
}

// Where a head's page holds the code of (token t of the page, dim d): the
// operand order of v_mfma_f32_16x16x32_f16 with 16 bytes a lane. Keys: lane
// (g, c) of a 16-token, 64-dim unit holds token c's dims 16 g .. + 16.
// Values: lane (g, c) of a 32-token, 32-dim unit holds dims c and 16 + c at
// the tokens 4 g + {0..3} and 16 + 4 g + {0..3}, which are those whose scores
// the lanes of group g hold.
__host__ __device__ inline int key_offset(int t, int d, int dk) {
    return (t / 16 * (dk / 64) + d / 64) * 1024 + d % 64 / 16 * 256 + t % 16 * 16 + d % 16;
}
__host__ __device__ inline int value_offset(int t, int d, int dv) {
    return (t / 32 * (dv / 32) + d / 32) * 1024 + t % 16 / 4 * 256 + d % 16 * 16 + d % 32 / 16 * 8 + t % 32 / 16 * 4 +
           t % 4;
}

__host__ __device__ inline float code_most(int kind) { return kind == DITCH_KV_INT8 ? 127.f : 448.f; }

// The tokens of a granule (32) share the values' units.
constexpr int GRANULE = 32;

// pages.hip
PoolView pool_view(const ditch_kv_pages *p, uint32_t layer);  // throws where the pool is refused
uint64_t pool_codes_bytes(const ditch_kv_pages *p);
uint64_t pool_scales_bytes(const ditch_kv_pages *p);
BatchView batch_view(const ditch_kv_batch *b, const PoolView &p);
RowsView rows_view(const ditch_kv_rows *r, uint64_t n_rows, uint64_t width, int32_t dtype, const char *what);
void launch_pages_append(const PoolView &p, const BatchView &b, int32_t dtype, const RowsView &k, const RowsView &v,
                         const RopeView &rope, const RowsView *q, const RowsView *q_out, int heads, hipStream_t s);
void launch_pages_read(const PoolView &p, const BatchView &b, int32_t dtype, const RowsView &k, const RowsView &v,
                       hipStream_t s);
void launch_pages_fork(const ditch_kv_pages *p, int32_t *table_out, int32_t *spare_out, const int32_t *table,
                       int64_t table_stride, const int32_t *parents, const int32_t *spare, const uint32_t *lens,
                       int64_t groups, int64_t beams, hipStream_t s);

// The batch of a forward's rows {b, pos}, each prompt's one after the other, the
// prompts in any order: starts, ends and pos [B]. A prompt whose rows do not
// lie so gets the position max_len, past which nothing is appended; its rows,
// those at such positions and those of prompts from B on become NaN in x
// [n][hidden].
void launch_rows_batch(const ditch_row *rows, int64_t n, int64_t B, int64_t max_len, uint32_t *starts, uint32_t *ends,
                       uint32_t *pos, float *x, int64_t hidden, hipStream_t s);
// table [B][cols] = b cols + j
void launch_own_pages(int32_t *table, int64_t n, hipStream_t s);

// pages_attention.hip
struct PagesAttention {
    PoolView p;
    BatchView b;
    RowsView q, out;
    int32_t dtype, heads;
    float scale;
    int32_t window, sinks;
    int32_t few;  // one row a sequence, as far as can be told: the few-row kernel
};
size_t pages_attention_workspace(const PoolView &p, const BatchView &b, int heads, int32_t dtype, uint32_t window,
                                 uint32_t sinks, int few = 0);
void launch_pages_attention(const PagesAttention &a, void *ws, size_t ws_bytes, hipStream_t s);

// beam.hip
size_t beam_select_workspace(int64_t prompts, int64_t beams, int64_t vocab, int64_t k);
void launch_beam_select(float *scores, int32_t *parents, uint32_t *tokens, const float *logits, const float *prev,
                        int64_t prompts, int64_t beams, int64_t vocab, int64_t k, void *ws, size_t ws_bytes,
                        hipStream_t s);

}  // namespace ditch
