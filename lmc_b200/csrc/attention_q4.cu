// attention_q4.cu - decode attention over 4-bit K/V rows (LMC_KV_Q4).
//
// One CTA per (query head, row): the new K/V row is quantized into shared
// memory (and, by the first head of the group, into the cache), each warp
// walks every fourth cached position with its own running maximum, sum and
// accumulator, and the warps' results are merged at the end.
#include "attention.cuh"
#include "kv_q4.cuh"
#include "lmc_common.cuh"
#include "lmc_internal.h"

namespace {

__device__ int g_attn_q4_err;  // a page id outside the pool was met (lmc_device_status)

__device__ __forceinline__ const uint8_t *q4_row(const AttnArgs &a, const void *cache, size_t cs, int kh, int t, int RB,
                                                 bool *ok) {
    const uint8_t *c = (const uint8_t *)cache;
    if (!a.pages) return c + (((long long)cs * a.Hkv + kh) * a.S + t) * RB;
    int pg = __ldg(a.pages + cs * a.max_pages + (t >> a.page_shift));
    *ok = pg >= 0 && pg < a.n_pages;
    if (!*ok) {
        atomicExch(&g_attn_q4_err, 1);
        pg = 0;
    }
    return c + ((((long long)pg * a.Hkv + kh) << a.page_shift) + (t & ((1 << a.page_shift) - 1))) * RB;
}

__global__ void __launch_bounds__(128) k_attn_q4(AttnArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ uint32_t newrow[2][40];
    __shared__ float red[4][256], stat[4][2];
    const int h = blockIdx.x, b = blockIdx.y, G = a.H / a.Hkv, kh = h / G, Dh = a.Dh, RB = kv_q4_row_bytes(Dh);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, NW = Dh / 8;
    const int pos = a.pos[b];
    if (pos < 0 || pos >= a.S) return;
    const size_t cs = a.seq ? (size_t)a.seq[b] : (size_t)b;
    const float *rc = a.rope_cos ? a.rope_cos + (size_t)pos * (Dh / 2) : nullptr;
    const float *rs = a.rope_sin ? a.rope_sin + (size_t)pos * (Dh / 2) : nullptr;
    if (a.append && warp < 2) {
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (lane < NW) {
            const float *src = (warp ? a.v_new : a.k_new) + (size_t)b * a.ldkv + (size_t)kh * Dh + 8 * lane;
            for (int i = 0; i < 4; i++) {
                x[2 * i] = src[2 * i];
                x[2 * i + 1] = src[2 * i + 1];
                if (!warp && rc) {
                    const float c = rc[4 * lane + i], s = rs[4 * lane + i], x0 = x[2 * i], x1 = x[2 * i + 1];
                    x[2 * i] = x0 * c - x1 * s;
                    x[2 * i + 1] = x0 * s + x1 * c;
                }
            }
        }
        uint32_t codes, dm;
        kv_q4_quantize<32>(x, lane < NW, codes, dm);
        if (lane < NW) {
            newrow[warp][lane] = codes;
            if (lane % 8 == 0) newrow[warp][NW + lane / 8] = dm;
        }
        bool ok = true;
        uint32_t *dst = (uint32_t *)q4_row(a, warp ? a.v_cache : a.k_cache, cs, kh, pos, RB, &ok);
        if (lane < NW && h % G == 0 && ok) {
            dst[lane] = codes;
            if (lane % 8 == 0) dst[NW + lane / 8] = dm;
        }
    }
    float q[8];
    for (int i = 0; i < 8; i++) q[i] = 0.0f;
    if (lane < NW) {
        const float *qp = a.q + (size_t)b * a.ldq + (size_t)h * Dh + 8 * lane;
        for (int i = 0; i < 4; i++) {
            q[2 * i] = qp[2 * i];
            q[2 * i + 1] = qp[2 * i + 1];
            if (rc) {
                const float c = rc[4 * lane + i], s = rs[4 * lane + i], x0 = q[2 * i], x1 = q[2 * i + 1];
                q[2 * i] = x0 * c - x1 * s;
                q[2 * i + 1] = x0 * s + x1 * c;
            }
        }
    }
    __syncthreads();
    const float scale = 1.0f / sqrtf((float)Dh);
    float m = -INFINITY, l = 0.0f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int t = warp; t <= pos; t += 4) {
        bool ok;
        const uint32_t *kr = (const uint32_t *)q4_row(a, a.k_cache, cs, kh, t, RB, &ok);
        const uint32_t *vr = (const uint32_t *)q4_row(a, a.v_cache, cs, kh, t, RB, &ok);
        if (a.append && t == pos) { kr = newrow[0]; vr = newrow[1]; }
        float s = 0.0f;
        if (lane < NW) {
            const uint32_t w = kr[lane], dm = kr[NW + lane / 8];
            const float d = __half2float(__ushort_as_half((unsigned short)(dm & 0xffff)));
            const float mm = __half2float(__ushort_as_half((unsigned short)(dm >> 16)));
            for (int i = 0; i < 8; i++) s = fmaf(q[i], fmaf(d, (float)((w >> (4 * i)) & 15u), mm), s);
        }
        s = warp_sum(s) * scale;
        const float mn = fmaxf(m, s), f = expf(m - mn), p = expf(s - mn);
        m = mn;
        l = l * f + p;
        if (lane < NW) {
            const uint32_t w = vr[lane], dm = vr[NW + lane / 8];
            const float d = __half2float(__ushort_as_half((unsigned short)(dm & 0xffff)));
            const float mm = __half2float(__ushort_as_half((unsigned short)(dm >> 16)));
            for (int i = 0; i < 8; i++) acc[i] = fmaf(p, fmaf(d, (float)((w >> (4 * i)) & 15u), mm), acc[i] * f);
        }
    }
    if (lane == 0) { stat[warp][0] = m; stat[warp][1] = l; }
    if (lane < NW)
        for (int i = 0; i < 8; i++) red[warp][8 * lane + i] = acc[i];
    __syncthreads();
    float M = -INFINITY, L = 0.0f;
    for (int w = 0; w < 4; w++) M = fmaxf(M, stat[w][0]);
    for (int w = 0; w < 4; w++) if (stat[w][0] != -INFINITY) L += stat[w][1] * expf(stat[w][0] - M);
    for (int d = threadIdx.x; d < Dh; d += 128) {
        float o = 0.0f;
        for (int w = 0; w < 4; w++) if (stat[w][0] != -INFINITY) o += red[w][d] * expf(stat[w][0] - M);
        a.out[(size_t)b * a.ldo + (size_t)h * Dh + d] = o / L;
    }
}

}  // namespace

extern "C" int lmc_attention_q4_launch(const AttnArgs *a, int batch, size_t ws_bytes, cudaStream_t s) {
    (void)ws_bytes;
    LMC_LAUNCH("attention (4-bit rows)", k_attn_q4, dim3(a->H, batch), 128, 0, s, *a);
    return LMC_OK;
}

extern "C" int lmc_attn_q4_status(void) {
    int v = 0;
    LMC_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_attn_q4_err, sizeof(int)));
    if (!v) return LMC_OK;
    const int zero = 0;
    LMC_CUDA_TRY(cudaMemcpyToSymbol(g_attn_q4_err, &zero, sizeof(int)));
    return lmc_set_error(LMC_ERR_INVALID, "paged attention: a page id outside the pool (page 0 read instead)");
}
