// beam.hip — the beam step: the k best continuations over beams and vocabulary.
#include "pages.h"

namespace ditch {

// An order of f64 scores as unsigned keys: larger key = better, NaN last.
__device__ __forceinline__ uint64_t score_key(double x) {
    if (!(x == x)) return 0;
    const uint64_t b = (uint64_t)__double_as_longlong(x);
    return b >> 63 ? ~b : b | ((uint64_t)1 << 63);
}

struct BeamArgs {
    float *scores;
    int32_t *parents;
    uint32_t *tokens;
    const float *logits, *prev;
    double *lse;  // [prompts][beams]
    int32_t beams, k;
    int64_t vocab;
};

// log sum exp of a row: the f32 maximum, f64 sum
__global__ __launch_bounds__(1024) void beam_lse_kernel(BeamArgs a) {
    __shared__ double part[16];
    const float *x = a.logits + (int64_t)blockIdx.x * a.vocab;
    const int tid = threadIdx.x;
    float m = -INFINITY;
    for (int64_t i = tid; i < a.vocab; i += 1024) m = fmaxf(m, x[i]);
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if ((tid & 63) == 0) part[tid >> 6] = m;
    __syncthreads();
    for (int w = 0; w < 16; w++) m = fmaxf(m, (float)part[w]);
    __syncthreads();
    double sum = 0;
    for (int64_t i = tid; i < a.vocab; i += 1024) sum += (double)expf(x[i] - m);
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if ((tid & 63) == 0) part[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) {
        sum = 0;
        for (int w = 0; w < 16; w++) sum += part[w];
        a.lse[blockIdx.x] = (double)m + log(sum);
    }
}

// k times the best continuation behind the last one
__global__ __launch_bounds__(1024) void beam_pick_kernel(BeamArgs a) {
    __shared__ uint64_t key_s[16];
    __shared__ int64_t at_s[16];
    const int tid = threadIdx.x;
    const int64_t prompt = blockIdx.x, n = a.beams * a.vocab;
    uint64_t last = ~(uint64_t)0;
    int64_t last_at = -1;
    for (int j = 0; j < a.k; j++) {
        uint64_t best = 0;
        int64_t at = n;
        for (int64_t i = tid; i < n; i += 1024) {
            const int b = (int)(i / a.vocab);
            const double s = (double)a.prev[prompt * a.beams + b] +
                             ((double)a.logits[prompt * n + i] - a.lse[prompt * a.beams + b]);
            const uint64_t key = score_key(s);
            if ((key < last || (key == last && i > last_at)) && (at == n || key > best)) {
                best = key;
                at = i;
            }
        }
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t ok = __shfl_xor(best, o, 64);
            const int64_t oa = __shfl_xor(at, o, 64);
            if (oa < n && (at == n || ok > best || (ok == best && oa < at))) {
                best = ok;
                at = oa;
            }
        }
        if ((tid & 63) == 0) {
            key_s[tid >> 6] = best;
            at_s[tid >> 6] = at;
        }
        __syncthreads();
        best = key_s[0];
        at = at_s[0];
        for (int w = 1; w < 16; w++)
            if (at_s[w] < n && (at == n || key_s[w] > best || (key_s[w] == best && at_s[w] < at))) {
                best = key_s[w];
                at = at_s[w];
            }
        __syncthreads();
        last = best;
        last_at = at;
        if (tid == 0) {
            const int b = (int)(at / a.vocab);
            a.parents[prompt * a.k + j] = b;
            a.tokens[prompt * a.k + j] = (uint32_t)(at % a.vocab);
            a.scores[prompt * a.k + j] = (float)((double)a.prev[prompt * a.beams + b] +
                                                 ((double)a.logits[prompt * n + at] - a.lse[prompt * a.beams + b]));
        }
    }
}

size_t beam_select_workspace(int64_t prompts, int64_t beams, int64_t vocab, int64_t k) {
    return (size_t)(prompts * beams) * sizeof(double);
}

void launch_beam_select(float *scores, int32_t *parents, uint32_t *tokens, const float *logits, const float *prev,
                        int64_t prompts, int64_t beams, int64_t vocab, int64_t k, void *ws, size_t ws_bytes,
                        hipStream_t s) {
    const BeamArgs a{scores, parents, tokens, logits, prev, (double *)ws, (int32_t)beams, (int32_t)k, vocab};
    hipLaunchKernelGGL(beam_lse_kernel, dim3((unsigned)(prompts * beams)), dim3(1024), 0, s, a);
    DITCH_TRY_HIP(hipGetLastError());
    hipLaunchKernelGGL(beam_pick_kernel, dim3((unsigned)prompts), dim3(1024), 0, s, a);
    DITCH_TRY_HIP(hipGetLastError());
}

}  // namespace ditch
