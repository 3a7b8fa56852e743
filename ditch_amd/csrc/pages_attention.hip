// pages_attention.hip — attention over pages of 8-bit keys and values.
#include "pages.h"

namespace ditch {

template <typename T, int KIND>
__global__ __launch_bounds__(256) void pages_attention_kernel(PagesAttention a) {
    __shared__ float qs[256], wm[4], wl[4], wo[4][256], pw[4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int64_t blk = blockIdx.x;
    const int h = (int)(blk % a.heads);
    blk /= a.heads;
    const int i = (int)(blk % a.b.max_rows), seq = (int)(blk / a.b.max_rows);
    const SeqRows r = seq_rows(a.b, seq);
    if (i >= r.n) return;
    T *out = (T *)a.out.data + (int64_t)(r.row + i) * a.out.stride + (int64_t)h * a.p.vd;
    if (i >= r.live) {
        for (int d = tid; d < a.p.vd; d += 256) out[d] = (T)NAN;
        return;
    }
    const T *q = (const T *)a.q.data + (int64_t)(r.row + i) * a.q.stride + (int64_t)h * a.p.hd;
    for (int d = tid; d < a.p.dk; d += 256) qs[d] = d < a.p.hd ? (float)q[d] : 0.f;
    __syncthreads();
    const int hk = h / (a.heads / a.p.kv_heads), t = r.pos + i;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = wave * 64; k0 <= t; k0 += 256) {
        const int j = k0 + lane;
        float s = -INFINITY, sv = 0.f;
        const bool seen = j <= t && (a.window == 0 || t - j < a.window || j < a.sinks);
        if (!__any(seen)) continue;
        if (seen) {
            const int id = page_of(a.b, a.p, seq, j >> a.p.page_shift);
            if (id < 0) s = sv = NAN;
            else {
                const int64_t ph = (int64_t)id * a.p.kv_heads + hk;
                const uint8_t *codes = a.p.codes + ph * a.p.page_bytes;
                float acc = 0.f;
                for (int d = 0; d < a.p.hd; d++) {
                    const uint8_t c = codes[key_offset(j & (a.p.page - 1), d, a.p.dk)];
                    acc += qs[d] * (KIND == DITCH_KV_INT8 ? (float)(int8_t)c : __builtin_amdgcn_cvt_f32_fp8((int)c, 0));
                }
                s = acc * a.p.scales[ph * 2] * a.scale;
                sv = a.p.scales[ph * 2 + 1];
            }
        }
        float mx = s;
        for (int w = 32; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor(mx, w, 64));
        const float mn = fmaxf(m, mx);
        const float p = seen ? expf(s - mn) : 0.f, f = m == -INFINITY ? 0.f : expf(m - mn);
        float sum = p;
        for (int w = 32; w > 0; w >>= 1) sum += __shfl_xor(sum, w, 64);
        l = l * f + sum;
        m = mn;
        pw[wave][lane] = seen ? p * sv : 0.f;
        __builtin_amdgcn_wave_barrier();
        for (int c = 0; c < 4; c++) o[c] *= f;
        for (int jj = 0; jj < 64 && k0 + jj <= t; jj++) {
            const int id = page_of(a.b, a.p, seq, (k0 + jj) >> a.p.page_shift);
            if (id < 0) continue;
            const uint8_t *codes = a.p.codes + ((int64_t)id * a.p.kv_heads + hk) * a.p.page_bytes + (int64_t)a.p.page * a.p.dk;
            const float w = pw[wave][jj];
            if (w == 0.f) continue;
            for (int c = 0; c < a.p.dv / 64; c++) {
                const uint8_t x = codes[value_offset((k0 + jj) & (a.p.page - 1), c * 64 + lane, a.p.dv)];
                o[c] += w * (KIND == DITCH_KV_INT8 ? (float)(int8_t)x : __builtin_amdgcn_cvt_f32_fp8((int)x, 0));
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    if (lane == 0) {
        wm[wave] = m;
        wl[wave] = l;
    }
    for (int c = 0; c < 4; c++) wo[wave][c * 64 + lane] = o[c];
    __syncthreads();
    const float mm = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
    for (int d = tid; d < a.p.vd; d += 256) {
        float num = 0.f, den = 0.f;
        for (int w = 0; w < 4; w++) {
            const float f = wm[w] == -INFINITY && wl[w] == 0.f ? 0.f : expf(wm[w] - mm);
            num += wo[w][d] * f;
            den += wl[w] * f;
        }
        out[d] = (T)(num / den);
    }
}

size_t pages_attention_workspace(const PoolView &p, const BatchView &b, int heads, int32_t dtype, uint32_t window,
                                 uint32_t sinks) {
    return 0;
}

template <typename T>
static void attention_typed(const PagesAttention &a, unsigned blocks, hipStream_t s) {
    if (a.p.kind == DITCH_KV_INT8)
        hipLaunchKernelGGL((pages_attention_kernel<T, DITCH_KV_INT8>), dim3(blocks), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((pages_attention_kernel<T, DITCH_KV_E4M3>), dim3(blocks), dim3(256), 0, s, a);
    DITCH_TRY_HIP(hipGetLastError());
}

void launch_pages_attention(const PagesAttention &a, void *ws, size_t ws_bytes, hipStream_t s) {
    if (a.b.n_seqs == 0) return;
    const int64_t n = (int64_t)a.b.n_seqs * a.b.max_rows * a.heads;
    DITCH_CHECK(n < ((int64_t)1 << 24), DITCH_INVALID_ARGUMENT, "kv attention: more work than one launch holds");
    if (a.dtype == DITCH_F32) attention_typed<float>(a, (unsigned)n, s);
    else if (a.dtype == DITCH_F16) attention_typed<_Float16>(a, (unsigned)n, s);
    else attention_typed<__bf16>(a, (unsigned)n, s);
}

}  // namespace ditch
