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

// min / max that keep a NaN.
__device__ __forceinline__ float kv_min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// x / 15 rounded to nearest, x in [0, 2^127): the product with the rounded
// reciprocal is off by at most one step, the FMA's remainder is exact, and
// adding its share rounds correctly (Markstein's theorem; 15's reciprocal is
// rounded correctly).  Below 2^-80, where the remainder would underflow, the
// quotient may be off by a step; as fp16 it is 0 there.
__device__ __forceinline__ float kv_div15(float x) {
    const float r = 1.0f / 15.0f, q = x * r;
    return fmaf(fmaf(-15.0f, q, x), r, q);
}

// A group's (d, m) word from its minimum (NaN when the group has one) and
// maximum; d = m = 0 and `bad` when a value is not finite.
__device__ __forceinline__ uint32_t kv_q4_scale(float lo, float hi, float &d, float &m, bool &bad) {
    bad = !(fabsf(lo) < INFINITY && fabsf(hi) < INFINITY);
    const __half mh = __float2half_rn(fminf(fmaxf(lo, -65504.0f), 65504.0f));
    m = __half2float(mh);
    const __half dh = __float2half_rn(fminf(kv_div15(fmaxf(hi - m, 0.0f)), 65504.0f));
    d = __half2float(dh);
    return bad ? 0x7e00u : (uint32_t)__half_as_ushort(dh) | (uint32_t)__half_as_ushort(mh) << 16;
}

// The word of codes of x (code i in bits 4 i .. 4 i + 3): the whole number
// nearest to (x - m) / d, ties to even, clamped to 0..15; 0 when d is 0 or the
// group is bad.  t is that quotient over 15, clamped to 0..1; 15 t is off by
// less than 2^-17 (x - m, the reciprocal, the product), so it decides unless
// it lies within 2e-5 of a tie; only then (one value in 25,000) is the word
// taken again in 64 bits, where x - m is exact (or d is too small for its last
// bit to matter) and the division cannot round across a tie of two fp16
// numbers.  Adding 1.5 * 2^23 rounds 15 t to a whole number, which then is the
// low bits of the sum.
__device__ __forceinline__ uint32_t kv_q4_codes(const float (&x)[8], float d, float m, bool bad) {
    const float inv = d > 0.0f && !bad ? __fdividef(1.0f, 15.0f * d) : 0.0f;
    uint32_t codes = 0u;
    float far = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float t = __saturatef((x[i] - m) * inv), k = fmaf(t, 15.0f, 12582912.0f);
        far = fmaxf(far, fabsf(fmaf(t, 15.0f, -(k - 12582912.0f))));
        codes += __float_as_uint(k) << (4 * i);
    }
    codes -= (uint32_t)(0x4b400000ull * 0x11111111ull);  // the eight sums' 1.5 * 2^23
    if (__builtin_expect(far > 0.49998f, 0)) {
        codes = 0u;
#pragma unroll 1
        for (int i = 0; i < 8; i++) {
            float xi = x[0];
#pragma unroll
            for (int e = 1; e < 8; e++) xi = i == e ? x[e] : xi;
            codes |= (uint32_t)fmin(fmax(rint(((double)xi - (double)m) / (double)d), 0.0), 15.0) << (4 * i);
        }
    }
    return codes;
}

// LPR lanes (4, 8, 16 or 32) quantize one row: lane w < Dh / 8 of them holds
// dims 8 w .. 8 w + 7 in x and gets its word of codes and its group's (d, m)
// word.  Every lane of the warp calls this.
template <int LPR>
__device__ __forceinline__ void kv_q4_quantize(const float (&x)[8], bool active, uint32_t &codes, uint32_t &dm) {
    float lo = INFINITY, hi = -INFINITY;
    if (active) {
        lo = kv_min_nan(kv_min_nan(kv_min_nan(x[0], x[1]), kv_min_nan(x[2], x[3])), kv_min_nan(kv_min_nan(x[4], x[5]), kv_min_nan(x[6], x[7])));
        hi = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    }
#pragma unroll
    for (int o = 1; o < (LPR < 8 ? LPR : 8); o <<= 1) {  // the group's lanes: 8, or the row's last 4
        lo = kv_min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    float d, m;
    bool bad;
    dm = kv_q4_scale(lo, hi, d, m, bad);
    codes = kv_q4_codes(x, d, m, bad);
}
