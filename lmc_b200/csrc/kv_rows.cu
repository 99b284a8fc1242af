// kv_rows.cu - K/V rows into a cache and back (lmc_kv_append, lmc_kv_read),
// any row form, contiguous or paged.
//
// Both stream: append reads 4 Dh bytes per row and side and writes the row's
// form, read the reverse, so HBM bounds them, and close behind it the
// instructions per value; a thread therefore has the K and the V side of its
// rows, whose place in the cache it works out once, and starts all loads
// before it uses the first.  4-bit rows: LPR = 4 .. 32 lanes per row, eight
// dims a lane; append takes neighbouring dims (a word of codes, three shuffles
// for a group's minimum and maximum), read two runs of four (stores without
// gaps).  The other forms take a warp per row and side.
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

// Item = (row, kv head), heads innermost; a CTA has U x 128 / LPR neighbouring
// items, a thread items 128 / LPR apart.
template <int LPR, int U> __global__ void __launch_bounds__(128) k_append_q4(RowArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const int w = threadIdx.x % LPR;
    const unsigned first = blockIdx.x * (U * 128u / LPR) + threadIdx.x / LPR;
    float x[U][2][8];
    long long off[U];
    unsigned row[U], head[U];
    bool in[U];
    // the values first, for every item: they do not wait for the place they go to
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
            uint32_t codes, dm;
            kv_q4_quantize<LPR>(x[u][side], off[u] >= 0, codes, dm);
            if (off[u] < 0) continue;
            uint32_t *to = reinterpret_cast<uint32_t *>((side ? a.vc : a.kc) + off[u]);
            to[w] = codes;
            if (w % 8 == 0) to[a.Dh / 8 + w / 8] = dm;
        }
}

template <int LPR, int U> __global__ void __launch_bounds__(128) k_read_q4(RowArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const int w = threadIdx.x % LPR, half = a.Dh / 8;  // quads w and w + half
    if (w >= half) return;
    const unsigned first = blockIdx.x * (U * 128u / LPR) + threadIdx.x / LPR;
    uint32_t codes[U][2][2], dm[U][2][2];
    long long off[U];
    unsigned row[U], head[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const unsigned item = first + u * (128 / LPR), r = item / a.Hkv, kh = item - r * a.Hkv;
        off[u] = r < (unsigned)a.rows ? row_offset(a, r, kh) : -1;
        row[u] = r;
        head[u] = kh;
#pragma unroll
        for (int side = 0; side < 2; side++) {
            if (off[u] < 0 || !(side ? a.v : a.k)) continue;
            const uint8_t *p = (side ? a.vc : a.kc) + off[u];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                codes[u][side][i] = reinterpret_cast<const uint16_t *>(p)[w + i * half];
                dm[u][side][i] = reinterpret_cast<const uint32_t *>(p)[half + (w + i * half) / 16];
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int side = 0; side < 2; side++) {
            if (off[u] < 0 || !(side ? a.v : a.k)) continue;
            float *to = (side ? a.v + (size_t)row[u] * a.ldv : a.k + (size_t)row[u] * a.ldk) + (size_t)head[u] * a.Dh + 4 * w;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float d = __half2float(__ushort_as_half((unsigned short)(dm[u][side][i] & 0xffff)));
                const float m = __half2float(__ushort_as_half((unsigned short)(dm[u][side][i] >> 16)));
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; e++)  // 2^23 | code is the number 2^23 + code
                    x[e] = fmaf(d, __uint_as_float(0x4b000000u | ((codes[u][side][i] >> (4 * e)) & 15u)) - 8388608.0f, m);
                float *p = to + 4 * half * i;
                if (a.vec) *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
                else
#pragma unroll
                    for (int e = 0; e < 4; e++) p[e] = x[e];
            }
        }
}

template <int LPR, int U> int launch_q4(const char *name, const RowArgs &a, bool read, cudaStream_t s) {
    LMC_LAUNCH(name, (read ? k_read_q4<LPR, U> : k_append_q4<LPR, U>), lmc_cdiv((size_t)a.rows * a.Hkv, U * 128 / LPR), 128, 0, s, a);
    return LMC_OK;
}
// Two items a thread when that still gives every SM eight CTAs, else one.
template <int LPR> int launch_q4(const char *name, const RowArgs &a, bool read, cudaStream_t s) {
    const bool many = (long long)a.rows * a.Hkv * LPR >= 2ll * 128 * 8 * lmc_sm_count();
    return many ? launch_q4<LPR, 2>(name, a, read, s) : launch_q4<LPR, 1>(name, a, read, s);
}

// One warp per (row, kv head, side) for the other row forms.
template <typename KV, bool READ>
__global__ void __launch_bounds__(128) k_rows(RowArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const bool is_v = blockIdx.y;
    float *f = is_v ? a.v : a.k;
    if (!f) return;
    const unsigned item = blockIdx.x * 4u + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, r = (int)((unsigned)item / a.Hkv), kh = (int)((unsigned)item % a.Hkv);
    if (r >= a.rows) return;
    const long long off = row_offset(a, r, kh);
    if (off < 0) return;
    f += (size_t)r * (is_v ? a.ldv : a.ldk) + (size_t)kh * a.Dh;
    KV *row = reinterpret_cast<KV *>((is_v ? a.vc : a.kc) + off);
    if constexpr (KvT<KV>::Q8) {
        if constexpr (READ) {
            const float sc = kv_q8_scale(row, a.Dh);
            for (int d = lane; d < a.Dh; d += 32) f[d] = kv_ld<KV>(row + d) * sc;
        } else {
            kv_q8_store_row(row, f, nullptr, nullptr, a.Dh, lane);
        }
    } else {
        for (int d = lane; d < a.Dh; d += 32) {
            if constexpr (READ) f[d] = kv_ld<KV>(row + d);
            else row[d] = kv_cvt<KV>(f[d]);
        }
    }
}

int rows_launch(const char *name, const RowArgs &a, int kv_dtype, bool read, cudaStream_t s) {
    const long long items = (long long)a.rows * a.Hkv;
    if (kv_dtype == LMC_KV_Q4) {
        const int words = a.Dh / 8;
        return words <= 4    ? launch_q4<4>(name, a, read, s)
               : words <= 8  ? launch_q4<8>(name, a, read, s)
               : words <= 16 ? launch_q4<16>(name, a, read, s)
                             : launch_q4<32>(name, a, read, s);
    }
    const dim3 grid(lmc_cdiv(items, 4), 2);
    void (*fn)(RowArgs) = kv_dtype == LMC_KV_F32   ? (read ? k_rows<float, true> : k_rows<float, false>)
                          : kv_dtype == LMC_KV_F16 ? (read ? k_rows<__half, true> : k_rows<__half, false>)
                                                   : (read ? k_rows<KvQ8, true> : k_rows<KvQ8, false>);
    LMC_LAUNCH(name, fn, grid, 128, 0, s, a);
    return LMC_OK;
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
