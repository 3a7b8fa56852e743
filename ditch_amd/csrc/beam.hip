// beam.hip — the beam step: the k best continuations over beams and vocabulary.
//
// score(beam, token) = prev[beam] + x[beam][token] - log sum exp x[beam]. Within
// a beam the order is that of the logits, so one pass over them is enough: a
// workgroup takes a chunk of a row into registers, forms its maximum, the sum
// of exponentials relative to it, and its k best logits; a second kernel joins
// the chunks of a prompt's beams, forms the scores in 64 bits and takes the k
// best of beams x chunks x k. A row is cut by its tokens, whatever its address,
// and summed in units of 2048 whatever the chunks: equal rows have equal sums,
// to the bit, in every beam and every batch, so that equal scores stay ties.
//
// The k best of a wave's part: with the maxima of its 128 half lanes, any
// threshold that k of them reach is reached by the k best, and by few
// others; it is found by bisection with ballots. What reaches it goes to a
// list, or, should that be more than the list holds (many equal logits, the
// best in few lanes, a mask that leaves fewer than k), exactly the k best do, by
// bisection over the elements, some 33 passes: 59 us with 60 000 finite logits
// a row of the call below, 760 with 1000, 2800 with 32.
//
// 64 prompts of 8 beams over 128 256 tokens (263 MB), 16 best: 45 us, 5.8 TB/s
// (a large copy: 5.1; some of it is still cached), and 8 us for the join; 1 prompt of 4 beams over 151 936
// tokens 14 us for both kernels. Vector issue comes next: a candidate's place
// in the list and its rank are few operations each (with twice as many the
// kernel took 62 us). Loads past the caches and half the chunk changed nothing.
#include "pages.h"

namespace ditch {

constexpr int BEAM_MOST_K = 128, BEAM_MOST_BEAMS = 64;
constexpr int LIST = 256;          // candidates of a wave
constexpr uint32_t NO_TOKEN = ~0u;  // an unused candidate

// An order of logits as unsigned keys: larger key = larger logit, NaN last
// (0), both zeros the same.
__device__ __forceinline__ uint32_t logit_key(float x) {
    if (!(x == x)) return 0;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t key) {
    return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}
// A candidate as one number: the larger goes first, among equal logits the
// lower token.
__device__ __forceinline__ uint64_t candidate_rank(float x, uint32_t token) {
    return (uint64_t)logit_key(x) << 32 | ~token;
}
__device__ __forceinline__ uint64_t score_key(double x) {
    if (!(x == x)) return 0;
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return b >> 63 ? ~b : b | ((uint64_t)1 << 63);
}

struct Candidate {
    float x;
    uint32_t token;
};

struct BeamArgs {
    float *scores;
    int32_t *parents;
    uint32_t *tokens;
    const float *logits, *prev;
    Candidate *list;  // [rows][chunks][k]
    double *stats;    // [rows][units][2]: maximum, sum of exponentials relative to it
    int32_t beams, k, chunks, units;  // units: of 2048 tokens, those of a row's chunks
    int64_t vocab;
};

// (rows start at any multiple of 4 bytes)
typedef float quad_t __attribute__((ext_vector_type(4), aligned(4)));
constexpr int UNIT = 8;  // quads a lane of a unit

// A workgroup of 4 waves a chunk of 256 R quads of a row.
template <int R>
__global__ __launch_bounds__(256) void beam_chunk_kernel(BeamArgs a) {
    __shared__ uint64_t list[4][LIST];
    __shared__ int count_s[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / a.chunks;
    const int chunk = (int)(blockIdx.x % a.chunks), k = a.k;
    const float *x = a.logits + row * a.vocab;
    // (vocab <= 2^30: 32 bits hold the last chunk's end)
    const int V = (int)a.vocab;
    const int first = (chunk * 4 + wave) * R * 256, t0 = first + 4 * lane;  // the lane's quad r: from t0 + 256 r
    float v[R][4];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int t = t0 + 256 * r;
        if (t + 4 <= V) {
            const quad_t f = *(const quad_t *)(x + t);
#pragma unroll
            for (int j = 0; j < 4; j++) v[r][j] = f[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) v[r][j] = t + j < V ? x[t + j] : -INFINITY;
        }
    }
    // the half lanes' maxima, and each unit's maximum and sum
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < 4; j++) top[r >= R / 2] = fmaxf(top[r >= R / 2], v[r][j]);
    double *st = a.stats + (row * a.units + (chunk * 4 + wave) * (R / UNIT)) * 2;
#pragma unroll
    for (int u = 0; u < R / UNIT; u++) {
        float m = R == UNIT ? fmaxf(top[0], top[1]) : top[u];
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        double sum = 0;
#pragma unroll
        for (int r = UNIT * u; r < UNIT * (u + 1); r++) {
            float s[4];
#pragma unroll
            for (int j = 0; j < 4; j++) s[j] = __builtin_amdgcn_exp2f((v[r][j] - m) * 1.44269504f);
            sum += (double)((s[0] + s[1]) + (s[2] + s[3]));
        }
        // (a unit of -infinities or past the row has no sum; a NaN shows in it)
        if (m == -INFINITY) {
            bool nan = false;
#pragma unroll
            for (int r = UNIT * u; r < UNIT * (u + 1); r++)
#pragma unroll
                for (int j = 0; j < 4; j++) nan |= v[r][j] != v[r][j];
            sum = nan ? NAN : 0;
        }
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if (lane == 0) {
            st[2 * u] = m;
            st[2 * u + 1] = sum;
        }
    }

    // the wave's tokens, and how many of them the list needs
    const int hi = first + R * 256 < V ? first + R * 256 : V;
    const int have = hi > first ? hi - first : 0, need = have < k ? have : k;
    int count = 0;
    bool done = need == 0;
    if (!done && need == k) {
        const uint32_t k0 = logit_key(top[0]), k1 = logit_key(top[1]);
        uint32_t a0 = k0 < k1 ? k0 : k1, b0 = k0 < k1 ? k1 : k0;
        for (int o = 32; o > 0; o >>= 1) {
            const uint32_t u = __shfl_xor(a0, o, 64), w = __shfl_xor(b0, o, 64);
            a0 = u < a0 ? u : a0;
            b0 = w > b0 ? w : b0;
        }
        // at `low` all 128 half lanes reach the threshold; `high` is the largest
        uint32_t low = a0, high = b0;
        while (low < high) {
            const uint32_t mid = low + (high - low + 1) / 2;
            const int c = __popcll(__ballot(k0 >= mid)) + __popcll(__ballot(k1 >= mid));
            if (c >= k) {
                low = mid;
                if (c <= k + k / 4 + 2) break;
            } else high = mid - 1;
        }
        // (low's logit; the key of a half lane without one is that of -infinity)
        const float tau = key_logit(low);
        // (a threshold of -infinity would take what pads the row, too)
        if (tau > -INFINITY) {
#pragma unroll
            for (int r = 0; r < R; r++) {
                uint64_t in[4];
#pragma unroll
                for (int j = 0; j < 4; j++) in[j] = __ballot(v[r][j] >= tau);
                if (in[0] | in[1] | in[2] | in[3]) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (in[j]) {
                            const int at = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(in[j] >> 32),
                                                                          __builtin_amdgcn_mbcnt_lo((uint32_t)in[j], count));
                            if (v[r][j] >= tau && at < LIST)
                                list[wave][at] = candidate_rank(v[r][j], (uint32_t)(t0 + 256 * r + j));
                            count += __popcll(in[j]);
                        }
                }
            }
        }
        done = count >= k && count <= LIST;
    }
    if (!done) {
        // exactly the `need` best: the largest key that as many reach, those
        // above it, and the first equal ones (read again: the registers are
        // not indexed at run time)
        uint32_t low = 0, high = ~0u;
        auto logit = [&](int r, int j, bool &in) {
            const int t = t0 + 256 * r + j;
            in = t < V;
            return in ? x[t] : 0.f;
        };
        auto reach = [&](uint32_t key) {
            int c = 0;
#pragma unroll 1
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    bool in;
                    const float f = logit(r, j, in);
                    c += __popcll(__ballot(in && logit_key(f) >= key));
                }
            return c;
        };
        while (low < high) {
            const uint32_t mid = low + (high - low) / 2 + 1;
            if (reach(mid) >= need) low = mid;
            else high = mid - 1;
        }
        const int above = low == ~0u ? 0 : reach(low + 1);
        int equal = need - above, put = 0;
#pragma unroll 1
        for (int r = 0; r < R; r++) {
            // index order: lane after lane, each lane's four
            uint64_t bg[4], be[4];
            float f[4];
            int eq = 0, gt = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                bool in;
                f[j] = logit(r, j, in);
                const uint32_t key = logit_key(f[j]);
                bg[j] = __ballot(in && key > low);
                be[j] = __ballot(in && key == low);
                eq += __popcll(be[j]);
                gt += __popcll(bg[j]);
            }
            const uint64_t bit = (uint64_t)1 << lane, before = bit - 1;
            int e = 0, g = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                e += __popcll(be[j] & before);
                g += __popcll(bg[j] & before);
            }
            const int take = eq < equal ? eq : equal;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const bool is_e = be[j] & bit, is_g = bg[j] & bit;
                const uint64_t c = candidate_rank(f[j], (uint32_t)(t0 + 256 * r + j));
                if (is_g) list[wave][put + g] = c;
                if (is_e && e < take) list[wave][put + gt + e] = c;
                g += is_g;
                e += is_e;
            }
            put += gt + take;
            equal -= take;
        }
        count = need;
    }
    if (lane == 0) count_s[wave] = count;
    __syncthreads();
    // the workgroup's k best by their ranks among its waves' candidates
    const int n0 = count_s[0], n1 = count_s[1], n2 = count_s[2], n3 = count_s[3], n = n0 + n1 + n2 + n3;
    Candidate *out = a.list + (int64_t)blockIdx.x * k;
    for (int e = tid; e < n; e += 256) {
        const int w = e < n0 ? 0 : e < n0 + n1 ? 1 : e < n0 + n1 + n2 ? 2 : 3;
        const uint64_t c = list[w][e - (w > 0 ? n0 : 0) - (w > 1 ? n1 : 0) - (w > 2 ? n2 : 0)];
        int rank = 0;
        for (int u = 0; u < 4; u++)
#pragma unroll 8
            for (int i = 0; i < count_s[u]; i++) rank += list[u][i] > c;
        if (rank < k) out[rank] = Candidate{key_logit((uint32_t)(c >> 32)), ~(uint32_t)c};
    }
    for (int e = n + tid; e < k; e += 256) out[e] = Candidate{0.f, NO_TOKEN};
}

// A workgroup a prompt: 8 us, bound by its chain: the beams' statistics, the
// candidates' scores, the search for the k-th of them (five turns of some 900
// cycles), the ranking. Every wave of a SIMD repeats the steps between, so 1024
// threads took 1.4 us more; with 256 the beams' statistics queue up (2 us more).
constexpr uint32_t JOIN = 512, HELD = 8;  // threads; candidates a thread holds in registers
constexpr int NEAR = 256;             // candidates that are ranked against each other
__global__ __launch_bounds__(JOIN) void beam_join_kernel(BeamArgs a) {
    __shared__ double lse_s[BEAM_MOST_BEAMS], prev_s[BEAM_MOST_BEAMS];
    __shared__ uint64_t lo_s[16], hi_s[16];
    __shared__ int count_s[2][16];
    __shared__ int put;
    __shared__ uint64_t key_s[NEAR], tie_s[NEAR];
    __shared__ uint32_t token_s[NEAR];
    __shared__ float score_s[NEAR];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = a.k;
    const int64_t row0 = (int64_t)blockIdx.x * a.beams;
    const uint32_t per = (uint32_t)a.chunks * k, n = a.beams * per;  // (2^30 and a few at most)
    const Candidate *list = a.list + (size_t)row0 * per;
    Candidate held_c[HELD];  // (asked for before the sums)
#pragma unroll
    for (int j = 0; j < HELD; j++) {
        held_c[j] = Candidate{0.f, NO_TOKEN};
        if (tid + JOIN * j < n) held_c[j] = list[tid + JOIN * j];
    }
    for (int b = wave; b < a.beams; b += JOIN / 64) {
        double sum = 0;
        float most;  // (the maxima are f32)
        const double *st = a.stats + (row0 + b) * a.units * 2;
        // (a lane's first part stays in registers, as few have a second)
        const double2 one = lane < a.units ? *(const double2 *)(st + 2 * lane) : make_double2(-INFINITY, 0);
        const float prev = a.prev[row0 + b];
        most = (float)one.x;
        for (int c = lane + 64; c < a.units; c += 64) most = fmaxf(most, (float)st[2 * c]);
        for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
        const double m = most;
        auto add = [&](double cm, double cs) { sum += cm == -INFINITY ? cs : cs * exp(cm - m); };
        add(one.x, one.y);
        for (int c = lane + 64; c < a.units; c += 64) add(st[2 * c], st[2 * c + 1]);
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if (lane == 0) {
            lse_s[b] = m == -INFINITY || m == INFINITY ? NAN : m + log(sum);
            prev_s[b] = (double)prev;
        }
    }
    if (tid == 0) put = 0;
    __syncthreads();

    struct Item {
        uint64_t key, tie;  // tie: beam, then the logit, inverted: smaller first
        uint32_t token;
        float score;
    };
    auto item = [&](uint32_t e, Candidate c) {
        const int b = (int)(e / per);
        const double s = prev_s[b] + ((double)c.x - lse_s[b]);
        return Item{score_key(s), (uint64_t)b << 32 | (uint32_t)~logit_key(c.x), c.token, (float)s};
    };
    Item held[HELD];
#pragma unroll
    for (int j = 0; j < HELD; j++) {
        held[j] = Item{0, 0, NO_TOKEN, 0.f};
        if (JOIN * j < n && held_c[j].token != NO_TOKEN) held[j] = item(tid + JOIN * j, held_c[j]);
    }
    auto each = [&](auto &&f) {
#pragma unroll
        for (int j = 0; j < HELD; j++)
            if (JOIN * j < n && held[j].token != NO_TOKEN) f(held[j]);
        for (uint32_t e = tid + JOIN * HELD; e < n; e += JOIN) {
            const Item it = item(e, list[e]);
            if (it.token != NO_TOKEN) f(it);
        }
    };
    int turn = 0;
    // how many candidates the predicate takes, over the workgroup
    auto count = [&](auto &&takes) {
        int c = 0;
#pragma unroll
        for (int j = 0; j < HELD; j++)  // (the waves' time is their number of operations: none for empty places)
            if (JOIN * j < n) c += __popcll(__ballot(held[j].token != NO_TOKEN && takes(held[j])));
        for (uint32_t e = JOIN * HELD; e < n; e += JOIN) {
            Item it{0, 0, NO_TOKEN, 0.f};
            if (e + tid < n) it = item(e + tid, list[e + tid]);
            c += __popcll(__ballot(it.token != NO_TOKEN && takes(it)));
        }
        if (lane == 0) count_s[turn][wave] = c;
        __syncthreads();
        c = 0;
#pragma unroll
        for (int w = 0; w < JOIN / 64; w++) c += count_s[turn][w];
        turn ^= 1;
        return c;
    };
    // the k-th largest score: between the least of the threads' largest (as
    // many threads as have candidates, or k, reach it) and the largest
    uint64_t low = ~(uint64_t)0, high = 0;
    {
        uint64_t mine = 0;
        bool any = false;
        each([&](const Item &it) {
            mine = it.key > mine ? it.key : mine;
            any = true;
        });
        low = any ? mine : low;
        high = mine;
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t u = __shfl_xor(low, o, 64), w = __shfl_xor(high, o, 64);
            low = u < low ? u : low;
            high = w > high ? w : high;
        }
        if (lane == 0) {
            lo_s[wave] = low;
            hi_s[wave] = high;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < JOIN / 64; w++) {
            low = lo_s[w] < low ? lo_s[w] : low;
            high = hi_s[w] > high ? hi_s[w] : high;
        }
    }
    if (count([&](const Item &it) { return it.key >= low; }) < k) low = 0;
    int reach = 0;
    while (low < high) {
        const uint64_t mid = low + (high - low) / 2 + 1;
        const int c = count([&](const Item &it) { return it.key >= mid; });
        if (c >= k) {
            low = mid;
            reach = c;
            if (c <= k + k / 2 + 8) break;  // few enough to rank
        } else high = mid - 1;
    }
    // should more than can be ranked reach it: exactly k; among equal scores the lowest beams, in a beam the largest logits, among equal logits the lowest tokens
    uint64_t tie = ~(uint64_t)0;
    uint32_t token = ~0u;
    if (reach < k || reach > NEAR) {
        int need = k - count([&](const Item &it) { return it.key > low; });
        uint64_t l = 0, h = ((uint64_t)BEAM_MOST_BEAMS << 32) - 1;
        while (l < h) {
            const uint64_t mid = l + (h - l) / 2;
            if (count([&](const Item &it) { return it.key == low && it.tie <= mid; }) >= need) h = mid;
            else l = mid + 1;
        }
        tie = l;
        need -= count([&](const Item &it) { return it.key == low && it.tie < tie; });
        uint32_t tl = 0, th = (uint32_t)a.vocab - 1;
        while (tl < th) {
            const uint32_t mid = tl + (th - tl) / 2;
            if (count([&](const Item &it) { return it.key == low && it.tie == tie && it.token <= mid; }) >= need) th = mid;
            else tl = mid + 1;
        }
        token = tl;
    }
    each([&](const Item &it) {
        if (it.key > low || (it.key == low && (it.tie < tie || (it.tie == tie && it.token <= token)))) {
            const int at = atomicAdd(&put, 1);
            if (at < NEAR) {
                key_s[at] = it.key;
                tie_s[at] = it.tie;
                token_s[at] = it.token;
                score_s[at] = it.score;
            }
        }
    });
    __syncthreads();
    // k or a few more, in any order: each goes to its rank
    const int n_near = put < NEAR ? put : NEAR;
    if (tid < n_near) {
        const uint64_t key = key_s[tid], t = tie_s[tid];
        const uint32_t tok = token_s[tid];
        int rank = 0, same = 0;
#pragma unroll 8
        for (int i = 0; i < n_near; i++) {
            rank += key_s[i] > key;
            same += key_s[i] == key;
        }
        if (same > 1)
            for (int i = 0; i < n_near; i++)
                rank += key_s[i] == key && (tie_s[i] < t || (tie_s[i] == t && token_s[i] < tok));
        if (rank < k) {
            const int64_t o = (int64_t)blockIdx.x * k + rank;
            a.scores[o] = score_s[tid];
            a.parents[o] = (int32_t)(t >> 32);
            a.tokens[o] = tok;
        }
    }
}

// Chunks of 8192 logits; of 16384 once they fill the chip (their lists are
// half as many, and so is the bisection's share).
static int beam_quads(int64_t rows, int64_t vocab) { return rows * vocab >= (int64_t)1024 * 16384 ? 16 : 8; }
static int64_t beam_chunks(int64_t rows, int64_t vocab) {
    const int64_t per = beam_quads(rows, vocab) * 1024;
    return (vocab + per - 1) / per;
}
static int64_t beam_units(int64_t rows, int64_t vocab) { return beam_chunks(rows, vocab) * 4 * beam_quads(rows, vocab) / UNIT; }

size_t beam_select_workspace(int64_t prompts, int64_t beams, int64_t vocab, int64_t k) {
    const int64_t rows = prompts * beams;
    return (size_t)rows * (beam_chunks(rows, vocab) * k * sizeof(Candidate) + beam_units(rows, vocab) * 2 * sizeof(double));
}

void launch_beam_select(float *scores, int32_t *parents, uint32_t *tokens, const float *logits, const float *prev,
                        int64_t prompts, int64_t beams, int64_t vocab, int64_t k, void *ws, size_t ws_bytes,
                        hipStream_t s) {
    const int64_t rows = prompts * beams, chunks = beam_chunks(rows, vocab), units = beam_units(rows, vocab);
    DITCH_CHECK(rows * chunks < (int64_t)1 << 24, DITCH_INVALID_ARGUMENT, "beam select: more logits than one launch holds");
    double *stats = (double *)ws;
    const BeamArgs a{scores, parents, tokens, logits, prev, (Candidate *)(stats + rows * units * 2), stats,
                     (int32_t)beams, (int32_t)k, (int32_t)chunks, (int32_t)units, vocab};
    if (beam_quads(rows, vocab) == 16)
        hipLaunchKernelGGL(beam_chunk_kernel<16>, dim3((unsigned)(rows * chunks)), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(beam_chunk_kernel<8>, dim3((unsigned)(rows * chunks)), dim3(256), 0, s, a);
    DITCH_TRY_HIP(hipGetLastError());
    hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)prompts), dim3(JOIN), 0, s, a);
    DITCH_TRY_HIP(hipGetLastError());
}

}  // namespace ditch
