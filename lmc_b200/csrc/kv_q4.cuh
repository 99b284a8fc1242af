// kv_q4.cuh - 4-bit K/V rows (LMC_KV_Q4): the row format and its quantizer.
//
// A row of Dh values (Dh a multiple of 32, at most 256) is Dh / 8 words of
// eight codes (nibble j of word w = dim 8 w + j, so dim 2 i is the low half
// of byte i), then one word (fp16 d, fp16 m) for each group of 64 dims, the
// last group having 32 when Dh % 64 is 32; value = d * code + m.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

constexpr int KV_Q4_GROUP = 64;  // dims that share one (d, m)

__host__ __device__ constexpr int kv_q4_groups(int Dh) { return (Dh + KV_Q4_GROUP - 1) / KV_Q4_GROUP; }
__host__ __device__ constexpr int kv_q4_row_bytes(int Dh) { return Dh / 2 + 4 * kv_q4_groups(Dh); }

// Code of x in a group with scale d > 0 and offset m: the whole number
// nearest to (x - m) / d, ties to even, clamped to 0..15.  inv = 1 / d in
// fp32.  The fp32 quotient is off by less than 2^-20 for results up to 16
// (three roundings), so it decides unless it lies within 2e-5 of a tie; only
// then (one value in 25,000) is the quotient taken in 64 bits, where x - m
// is exact (or d is too small for the last bit to matter) and the division
// cannot round across a tie of two fp16 numbers.
__device__ __forceinline__ uint32_t kv_q4_code(float x, float m, float d, float inv) {
    const float t = (x - m) * inv;
    float k = rintf(t);
    if (fabsf(t - k) > 0.49998f && t > -1.0f && t < 16.0f) k = (float)rint(((double)x - (double)m) / (double)d);
    return (uint32_t)fminf(fmaxf(k, 0.0f), 15.0f);
}

// LPR lanes (4, 8, 16 or 32; the power of two >= Dh / 8) quantize one row:
// lane w < Dh / 8 holds dims 8 w .. 8 w + 7 in x and gets its word of codes
// and its group's (d, m) word.  Every lane of the warp calls this.
template <int LPR>
__device__ __forceinline__ void kv_q4_quantize(const float (&x)[8], bool active, uint32_t &codes, uint32_t &dm) {
    float lo = INFINITY, hi = -INFINITY, fin = 0.0f;
    if (active) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            lo = fminf(lo, x[i]);
            hi = fmaxf(hi, x[i]);
            fin += x[i] * 0.0f;  // NaN as soon as one value is not finite
        }
    }
#pragma unroll
    for (int o = 1; o < (LPR < 8 ? LPR : 8); o <<= 1) {  // the group's lanes: 8, or the row's last 4
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        fin += __shfl_xor_sync(0xffffffffu, fin, o);
    }
    codes = 0u;
    if (fin != 0.0f) {  // NaN: the group reads back as NaN
        dm = 0x7e00u;
        return;
    }
    const __half mh = __float2half_rn(fminf(fmaxf(lo, -65504.0f), 65504.0f));
    const float m = __half2float(mh);
    const __half dh = __float2half_rn(fminf(__fdiv_rn(fmaxf(hi - m, 0.0f), 15.0f), 65504.0f));
    const float d = __half2float(dh);
    dm = (uint32_t)__half_as_ushort(dh) | (uint32_t)__half_as_ushort(mh) << 16;
    if (d > 0.0f) {
        const float inv = 1.0f / d;
#pragma unroll
        for (int i = 0; i < 8; i++) codes |= kv_q4_code(x[i], m, d, inv) << (4 * i);
    }
}
