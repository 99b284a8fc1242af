// kv_rows.cu - K/V rows into a cache and back (lmc_kv_append, lmc_kv_read),
// any row form, contiguous or paged.
//
// Both stream: append reads 4 Dh bytes per row and side and writes the row's
// form, read the reverse, so HBM bounds them, and close behind it the
// instructions per value (4-bit append issues in 74 of 100 cycles); a thread
// therefore has the K and the V side of its rows, whose place in the cache it
// works out once, and starts all loads before it uses the first.  LPR = 4 ..
// 32 lanes per row, eight dims a lane: append takes neighbouring dims (a word
// of codes, three shuffles for a group's minimum and maximum; 16 bytes of
// fp16), read two runs of four (stores without gaps).
// 32000 rows of 8 x 128, append / read: 4-bit 61 / 50 us (4.9 / 5.9 TB/s),
// int8 60 / 54 us, fp16 59 / 61 us (6.7 / 6.4 TB/s), fp32 80 / 79 us (6.6 TB/s); 509 rows of 4 x 64 take
// 2.9 / 1.8 us in 4 bits, most of it latency.
#include <type_traits>

#include "attention.cuh"
#include "kv_q4.cuh"
#include "lmc_common.cuh"
#include "lmc_internal.h"

namespace {

__device__ int g_kv_rows_err;  // an index outside its range was met (lmc_device_status)

struct RowArgs {
    float *k, *v;  // fp32 rows (read by append, written by read); NULL: that side is left out
    uint8_t *kc, *vc;
    const int *seq, *pos, *pages;
    const float *rope_cos, *rope_sin;  // append: K rotated when given
    int ldk, ldv, rows, n_seqs, Hkv, Dh, S, page_shift, max_pages, n_pages;
    int RB;   // row bytes
    int vec;  // fp32 rows can be moved 16 bytes at a time
};

// Byte offset of (row r, kv head kh) in its cache, or -1: padding, or an
// index outside its range (flagged).
__device__ __forceinline__ long long row_offset(const RowArgs &a, int r, int kh) {
    const int pos = a.pos[r], seq = a.seq ? a.seq[r] : r;
    if (pos < 0) return -1;
    bool ok = pos < a.S && seq >= 0 && (a.n_seqs == 0 || seq < a.n_seqs);
    long long base = 0;
    if (ok && a.pages) {
        const int pg = __ldg(a.pages + (size_t)seq * a.max_pages + (pos >> a.page_shift));
        ok = pg >= 0 && pg < a.n_pages;
        base = ((((long long)pg * a.Hkv + kh) << a.page_shift) + (pos & ((1 << a.page_shift) - 1))) * a.RB;
    } else if (ok) {
        base = (((long long)seq * a.Hkv + kh) * a.S + pos) * a.RB;
    }
    if (!ok) {
        atomicExch(&g_kv_rows_err, 1);
        return -1;
    }
    return base;
}

__device__ __forceinline__ void load8(const float *p, bool vec, float (&x)[8]) {
    if (vec) {
        const float4 u = *reinterpret_cast<const float4 *>(p), w = *reinterpret_cast<const float4 *>(p + 4);
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
        x[4] = w.x; x[5] = w.y; x[6] = w.z; x[7] = w.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = p[i];
    }
}

struct KvQ4 {};  // the form's tag

// Dims 8 w .. 8 w + 7 of a row into the cache (`active`: this lane has them);
// the LPR lanes of a row call this together.
template <typename KV, int LPR> __device__ __forceinline__ void store8(uint8_t *row, bool active, int w, int Dh, const float (&x)[8]) {
    if constexpr (std::is_same_v<KV, KvQ4>) {
        uint32_t codes, dm;
        kv_q4_quantize<LPR>(x, active, codes, dm);
        if (!active) return;
        reinterpret_cast<uint32_t *>(row)[w] = codes;
        if (w % 8 == 0) reinterpret_cast<uint32_t *>(row)[Dh / 8 + w / 8] = dm;
    } else if constexpr (KvT<KV>::Q8) {  // (as kv_q8_store_row)
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(x[i]));  // (0 in lanes without dims)
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (!active) return;
        const float inv = m > 0.0f ? 127.0f / m : 0.0f;
        uint32_t c[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; i++)
            c[i / 4] |= (uint32_t)(max(-127, min(127, __float2int_rn(__fmul_rn(x[i], inv)))) & 0xff) << (8 * (i % 4));
        reinterpret_cast<uint2 *>(row)[w] = make_uint2(c[0], c[1]);
        if (w == 0) *reinterpret_cast<float *>(row + Dh) = m / 127.0f;
    } else if (active) {
        KV y[8];
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = kv_cvt<KV>(x[i]);
#pragma unroll
        for (int i = 0; i < (int)sizeof y / 16; i++) reinterpret_cast<uint4 *>(row)[w * (sizeof y / 16) + i] = reinterpret_cast<const uint4 *>(y)[i];
    }
}

// Item = (row, kv head), heads innermost; a CTA has U x 128 / LPR neighbouring
// items, a thread items 128 / LPR apart.
template <typename KV, int LPR, int U> __global__ void __launch_bounds__(128) k_append(RowArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const int w = threadIdx.x % LPR;
    const unsigned first = blockIdx.x * (U * 128u / LPR) + threadIdx.x / LPR;
    float x[U][2][8];
    long long off[U];
    unsigned row[U], head[U];
    bool in[U];
    // the values first, padding's too: they do not wait for the place they go to
    // (after the position 32000 rows take 68 us, 509 rows of 4 x 64 3.9)
#pragma unroll
    for (int u = 0; u < U; u++) {
        const unsigned item = first + u * (128 / LPR);
        row[u] = item / a.Hkv;
        head[u] = item - row[u] * a.Hkv;
        in[u] = row[u] < (unsigned)a.rows && w < a.Dh / 8;
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int i = 0; i < 8; i++) x[u][0][i] = x[u][1][i] = 0.0f;
    if (a.k)
#pragma unroll
        for (int u = 0; u < U; u++)
            if (in[u]) load8(a.k + (size_t)row[u] * a.ldk + (size_t)head[u] * a.Dh + 8 * w, a.vec, x[u][0]);
    if (a.v)
#pragma unroll
        for (int u = 0; u < U; u++)
            if (in[u]) load8(a.v + (size_t)row[u] * a.ldv + (size_t)head[u] * a.Dh + 8 * w, a.vec, x[u][1]);
#pragma unroll
    for (int u = 0; u < U; u++) off[u] = in[u] ? row_offset(a, row[u], head[u]) : -1;
    if (a.k && a.rope_cos)  // pairs (2 d, 2 d + 1) (src/ops_llama.c:39-48)
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (off[u] < 0) continue;
            const size_t t = (size_t)a.pos[row[u]] * (a.Dh / 2) + 4 * w;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float c = a.rope_cos[t + i], s = a.rope_sin[t + i], x0 = x[u][0][2 * i], x1 = x[u][0][2 * i + 1];
                x[u][0][2 * i] = x0 * c - x1 * s;
                x[u][0][2 * i + 1] = x0 * s + x1 * c;
            }
        }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int side = 0; side < 2; side++) {
            if (!(side ? a.v : a.k)) continue;
            store8<KV, LPR>((side ? a.vc : a.kc) + off[u], off[u] >= 0, w, a.Dh, x[u][side]);
        }
}

// Two runs of four dims a lane, so a warp's stores leave no gaps.
template <typename KV, int LPR> __global__ void __launch_bounds__(128) k_read(RowArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const int w = threadIdx.x % LPR, half = a.Dh / 8;  // quads w and w + half
    if (w >= half) return;
    const unsigned item = blockIdx.x * (128u / LPR) + threadIdx.x / LPR, r = item / a.Hkv, kh = item - r * a.Hkv;
    const long long off = r < (unsigned)a.rows ? row_offset(a, r, kh) : -1;
    if (off < 0) return;
    using Raw = std::conditional_t<std::is_same_v<KV, float>, uint4, uint2>;
    Raw raw[2][2];  // every load before the first use
#pragma unroll
    for (int side = 0; side < 2; side++) {
        if (!(side ? a.v : a.k)) continue;
        const uint8_t *p = (side ? a.vc : a.kc) + off;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int quad = w + i * half;
            if constexpr (std::is_same_v<KV, KvQ4>)
                raw[side][i] = make_uint2(reinterpret_cast<const uint16_t *>(p)[quad], reinterpret_cast<const uint32_t *>(p)[half + quad / 16]);
            else if constexpr (KvT<KV>::Q8)
                raw[side][i] = make_uint2(reinterpret_cast<const uint32_t *>(p)[quad], *reinterpret_cast<const uint32_t *>(p + a.Dh));
            else
                raw[side][i] = reinterpret_cast<const Raw *>(p)[quad];
        }
    }
#pragma unroll
    for (int side = 0; side < 2; side++) {
        if (!(side ? a.v : a.k)) continue;
        float *to = (side ? a.v + (size_t)r * a.ldv : a.k + (size_t)r * a.ldk) + (size_t)kh * a.Dh + 4 * w;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const Raw u = raw[side][i];
            float y[4];
            if constexpr (std::is_same_v<KV, KvQ4>) {
                const float2 dm = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
#pragma unroll
                for (int e = 0; e < 4; e++)  // 2^23 | code is the number 2^23 + code
                    y[e] = fmaf(dm.x, __uint_as_float(0x4b000000u | ((u.x >> (4 * e)) & 15u)) - 8388608.0f, dm.y);
            } else if constexpr (KvT<KV>::Q8) {
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = (float)(int8_t)(u.x >> (8 * e)) * __uint_as_float(u.y);
            } else if constexpr (std::is_same_v<KV, float>) {
                y[0] = __uint_as_float(u.x); y[1] = __uint_as_float(u.y); y[2] = __uint_as_float(u.z); y[3] = __uint_as_float(u.w);
            } else {
                const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&u.x)), hi = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
                y[0] = lo.x; y[1] = lo.y; y[2] = hi.x; y[3] = hi.y;
            }
            float *p = to + 4 * half * i;
            if (a.vec) *reinterpret_cast<float4 *>(p) = make_float4(y[0], y[1], y[2], y[3]);
            else { p[0] = y[0]; p[1] = y[1]; p[2] = y[2]; p[3] = y[3]; }
        }
    }
}

// Appending, two items a thread from 32 CTAs (of one item) per SM on: 32000
// rows of 8 x 128 66 us with one, 63 with two; 2048 rows 6.4 and 6.8.  Reading
// gains nothing from a second (50 and 52 us).
template <typename KV, int LPR> int launch(const char *name, const RowArgs &a, bool read, cudaStream_t s) {
    const size_t items = (size_t)a.rows * a.Hkv;
    if (read) LMC_LAUNCH(name, (k_read<KV, LPR>), lmc_cdiv(items, 128 / LPR), 128, 0, s, a);
    else if (items * LPR >= 128ull * 32 * lmc_sm_count()) LMC_LAUNCH(name, (k_append<KV, LPR, 2>), lmc_cdiv(items, 2 * 128 / LPR), 128, 0, s, a);
    else LMC_LAUNCH(name, (k_append<KV, LPR, 1>), lmc_cdiv(items, 128 / LPR), 128, 0, s, a);
    return LMC_OK;
}
template <typename KV> int launch_form(const char *name, const RowArgs &a, bool read, cudaStream_t s) {
    const int lanes = a.Dh / 8;
    return lanes <= 4    ? launch<KV, 4>(name, a, read, s)
           : lanes <= 8  ? launch<KV, 8>(name, a, read, s)
           : lanes <= 16 ? launch<KV, 16>(name, a, read, s)
                         : launch<KV, 32>(name, a, read, s);
}
int rows_launch(const char *name, const RowArgs &a, int kv_dtype, bool read, cudaStream_t s) {
    return kv_dtype == LMC_KV_Q4    ? launch_form<KvQ4>(name, a, read, s)
           : kv_dtype == LMC_KV_Q8  ? launch_form<KvQ8>(name, a, read, s)
           : kv_dtype == LMC_KV_F16 ? launch_form<__half>(name, a, read, s)
                                    : launch_form<float>(name, a, read, s);
}

// The checks that lmc_kv_append and lmc_kv_read share; fills `a`.
int rows_args(const char *name, RowArgs *a, const float *k, const float *v, int ld, const void *kc, const void *vc,
              int kv_dtype, const int *d_seq, const int *d_pos, int rows, int n_seqs, int Hkv, int Dh, int S,
              const int *d_pages, int page_size, int n_pages) {
    if ((!k && !v) || (k && !kc) || (v && !vc) || !d_pos)
        return lmc_set_error(LMC_ERR_INVALID, "%s: null pointer", name);
    if (kv_dtype != LMC_KV_F32 && kv_dtype != LMC_KV_F16 && kv_dtype != LMC_KV_Q8 && kv_dtype != LMC_KV_Q4)
        return lmc_set_error(LMC_ERR_UNSUPPORTED, "%s: kv dtype %d", name, kv_dtype);
    if (rows < 0 || n_seqs <= 0 || Hkv <= 0 || Dh <= 0 || Dh % 32 || Dh > 256 || S <= 0 || (long long)Hkv * Dh > ld)
        return lmc_set_error(LMC_ERR_INVALID, "%s: rows=%d n_seqs=%d Hkv=%d Dh=%d S=%d ld=%d (need Dh%%32==0, "
                             "Dh<=256, ld>=Hkv*Dh)", name, rows, n_seqs, Hkv, Dh, S, ld);
    if ((long long)rows * Hkv > (1ll << 30))
        return lmc_set_error(LMC_ERR_INVALID, "%s: %d rows of %d heads in one call", name, rows, Hkv);
    if (((uintptr_t)(k ? kc : nullptr) | (uintptr_t)(v ? vc : nullptr)) & 15)
        return lmc_set_error(LMC_ERR_INVALID, "%s: the cache must start on a 16-byte boundary", name);
    int shift = 0;
    if (d_pages) {
        if (n_pages <= 0 || page_size < 16 || (page_size & (page_size - 1)) || S % page_size || S > (1 << 24))
            return lmc_set_error(LMC_ERR_INVALID, "%s: pages %d of %d positions, context %d", name, n_pages, page_size, S);
        while ((1 << shift) < page_size) shift++;
    }
    *a = RowArgs{const_cast<float *>(k), const_cast<float *>(v), (uint8_t *)const_cast<void *>(kc),
                 (uint8_t *)const_cast<void *>(vc), d_seq, d_pos, d_pages, nullptr, nullptr, ld, ld, rows, n_seqs, Hkv, Dh, S,
                 shift, d_pages ? S / page_size : 0, n_pages, (int)LMC_KV_ROW_BYTES(kv_dtype, Dh),
                 (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && ld % 4 == 0};
    return LMC_OK;
}

}  // namespace

extern "C" int lmc_kv_append(const float *k, const float *v, int ld, void *kc, void *vc, int kv_dtype, const int *d_seq,
                             const int *d_pos, int rows, int n_seqs, int Hkv, int Dh, int S, const int *d_pages,
                             int page_size, int n_pages, void *stream) {
    RowArgs a;
    const int rc = rows_args("kv_append", &a, k, v, ld, kc, vc, kv_dtype, d_seq, d_pos, rows, n_seqs, Hkv, Dh, S,
                             d_pages, page_size, n_pages);
    if (rc != LMC_OK || rows == 0) return rc;
    return rows_launch("kv append", a, kv_dtype, false, lmc_stream(stream));
}

extern "C" int lmc_kv_read(float *k, float *v, int ld, const void *kc, const void *vc, int kv_dtype, const int *d_seq,
                           const int *d_pos, int rows, int n_seqs, int Hkv, int Dh, int S, const int *d_pages,
                           int page_size, int n_pages, void *stream) {
    RowArgs a;
    const int rc = rows_args("kv_read", &a, k, v, ld, kc, vc, kv_dtype, d_seq, d_pos, rows, n_seqs, Hkv, Dh, S, d_pages,
                             page_size, n_pages);
    if (rc != LMC_OK || rows == 0) return rc;
    return rows_launch("kv read", a, kv_dtype, true, lmc_stream(stream));
}

extern "C" int lmc_kv_append_launch(const float *k, const float *v, int ldk, int ldv, void *kc, void *vc, int kv_dtype,
                                    const int *d_seq, const int *d_pos, int rows, int n_seqs, int Hkv, int Dh, int S,
                                    const int *d_pages, int page_shift, int max_pages, int n_pages,
                                    const float *rope_cos, const float *rope_sin, cudaStream_t s) {
    const RowArgs a = {const_cast<float *>(k), const_cast<float *>(v), (uint8_t *)kc, (uint8_t *)vc, d_seq, d_pos,
                       d_pages, rope_cos, rope_sin, ldk, ldv, rows, n_seqs, Hkv, Dh, S, page_shift, max_pages, n_pages,
                       (int)LMC_KV_ROW_BYTES(kv_dtype, Dh),
                       (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && ldk % 4 == 0 && ldv % 4 == 0};
    return rows_launch("kv append", a, kv_dtype, false, s);
}

extern "C" int lmc_kv_rows_status(void) {
    int v = 0;
    LMC_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_kv_rows_err, sizeof(int)));
    if (!v) return LMC_OK;
    const int zero = 0;
    LMC_CUDA_TRY(cudaMemcpyToSymbol(g_kv_rows_err, &zero, sizeof(int)));
    return lmc_set_error(LMC_ERR_INVALID, "kv rows: a position, sequence or page outside the cache (row left out)");
}
