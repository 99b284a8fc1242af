// attention_q4.cu - decode attention over 4-bit K/V rows (LMC_KV_Q4).
//
// With codes c and (d, m) of group j (64 dims) of row t:
//   s_t = sum_j [ d_tj (q_j . c_tj) + m_tj sum(q_j) ] / sqrt(Dh)
//   o_j = sum_t p_t d_tj (2 c_tj - 15) / 2 + sum_t p_t (m_tj + 7.5 d_tj),   p_t = 2^(s_t log2 e - max)
// so the matrix units only ever see whole numbers and fp32 factors; the scales
// are applied per group outside (keys) or folded into the probabilities
// (values).  Keys: integer products, q as whole numbers in four signed bytes,
// the largest |q| of a group of 64 dims in [2^29, 2^30): a channel down to 1/64
// of it keeps all of fp32's bits, a smaller one is off by at most 2^-30 of it.
// The products and sum(q) are exact, and the two terms, which can be large
// against their sum, are added with the rounding of the first one's product kept,
// so a group's score is rounded relative to itself.  The values' codes are
// centred, because sums over positive codes would be large against the result of
// a long, flat softmax and take their rounding with them.
//
// A value's code as fp16: a nibble ORed into bits 1 to 4 of 1024.0 is 1024 +
// 2 c, exactly, and 1039 less is 2 c - 15 (two instructions for two operands);
// the nibble above it gives 16 (2 c - 15), and the 16 goes into the final
// factor.  p d becomes an fp16 pair hi + lo (22 bits), scaled by a power of two
// that keeps it just below 2^15: its largest exponent so far is tracked like the
// running maximum, for each head and group of 64 dims, so that neither a group of
// larger values nor a row of large values without weight takes bits from it (a p d
// below 2^-18 of the largest is off by at most 2^-40 of that).  The matrix unit
// truncates its sums, so a tile's products (and its sums of p and of p with the
// minima) go to fresh accumulators that are added to the running ones in rounded
// fp32.
//
// Work: tiles of 64 positions (32 from head size 160 on) of one (sequence, kv
// head, 8 query heads).  All tiles of the batch, in order, are divided evenly
// over the CTAs and within a CTA over its four warps, so ragged batches and
// single long sequences load every SM alike.  A warp streams its tiles through
// its own ring in shared memory (bulk copies of the runs of rows that lie
// together, one lane each; 16-byte asynchronous copies where a contiguous
// cache's context is no multiple of 4 positions, which puts rows off the
// 16-byte boundaries) with a running softmax; parts of one item that lie in
// one CTA are merged in shared memory, parts in several CTAs through the
// workspace by k_q4_combine.
//
// Whole calls: 1 x 131072 positions of 8 kv heads of 128 dims 45 us, 128 ragged
// sequences of them 85 us (3.4 and 3.6 TB/s), 64 ragged ones of 4 heads of 64
// dims 19.0 us, one of 12 heads with 700 positions 7.7 us.  Instructions bound
// the first two (matrix, integer and half instructions share the issue), the
// latency of a warp's chain (its share, the copies, q, a tile, the merge) the
// others.
#include <algorithm>
#include <type_traits>
#include <vector>

#include "attention.cuh"
#include "kv_q4.cuh"
#include "lmc_common.cuh"
#include "lmc_internal.h"

namespace {

__device__ int g_attn_q4_err;  // bit 0: a page id outside the pool, bit 1: a wait ran out (lmc_device_status)

constexpr int Q4_WARPS = 4;
constexpr int Q4_STAGES = 2;  // tiles in a warp's ring
// What beginning and ending an item costs, in tiles (q, the new row, the
// result): 128 ragged sequences of 8 kv heads 91.8, 85.3, 87.0 us with 1, 2, 3;
// 64 of 4 kv heads, eight query heads each, 19.5, 19.0, 19.7.
constexpr int Q4_ITEM = 2;
constexpr float LOG2E = 1.4426950408889634f;
// Limit of a wait for bulk copies (nanoseconds of %globaltimer).
__device__ long long g_attn_q4_wait_ns = 1000000000ll;

constexpr int q4_tile(int NB) { return NB <= 4 ? 64 : 32; }  // positions per tile (registers and shared memory)

struct Q4Args {
    AttnArgs a;
    int G, HG;      // query heads per kv head, groups of 8 of them
    int rmin;       // tiles per CTA at least (workspace slots per head: a.nsplit)
    int items_only; // 1: an item is never divided (a.nsplit is 1)
    int batch, vec; // vec: q, new rows and out can be moved 16 bytes at a time
    int bulk;       // every run of rows starts on a 16-byte boundary, four rows are whole 16-byte pieces
    int run;        // rows that lie together: a page's, at most a tile's
    long long page_bytes; // of one kv head's rows of a page
    int lose_j, lose_tile; // self-test: warps with this tile of a sequence's item j wait for bytes that never come (-1: none)
};

template <int NB> struct Q4 {
    static constexpr int T = q4_tile(NB), DH = 32 * NB, NG = kv_q4_groups(DH), RB = kv_q4_row_bytes(DH);
    static constexpr int SIDE = T * RB + 16;              // a tile's K or V rows, from any 4-byte phase
    static constexpr int STAGE = 2 * SIDE;
    static constexpr int FRESH = (2 * RB + 15) / 16 * 16; // the new K and V rows
    static constexpr int WARP_BYTES = Q4_STAGES * STAGE + FRESH;
    static constexpr int SLOT = DH + 4;                   // floats of a head's partial result (accumulator, maximum, sum)
    static_assert(Q4_STAGES * STAGE >= 8 * SLOT * 4, "a partial result fits the ring that it is kept in");
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void hmma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void hmma0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// Two fp32 numbers, one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long &>(r))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)),
          "l"(reinterpret_cast<unsigned long long &>(c)));
    return r;
}
// Exponent field of p d, as far as a scale is made for it: 2^(141 - field) is a
// normal number, and p d is at most 65504.
__device__ __forceinline__ int pd_exponent(float x) { return min(max((int)(__float_as_uint(x) >> 23), 15), 142); }
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// x, y as fp16 pairs hi + lo
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    float rx, ry;  // hi - x, hi - y
    asm("sub.f32.f16 %0, %1, %2;" : "=f"(rx) : "h"(__half_as_ushort(__low2half(h))), "f"(x));
    asm("sub.f32.f16 %0, %1, %2;" : "=f"(ry) : "h"(__half_as_ushort(__high2half(h))), "f"(y));
    const __half2 l = __floats2half2_rn(-rx, -ry);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

// Barrier of a stage's bulk copies.
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
// Bounded: false (and the time-out is recorded) when the copies have not landed within the limit.
__device__ __noinline__ bool bar_wait_long(uint32_t bar, uint32_t parity) {
    long long t0, t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
    do {
        if (bar_try(bar, parity)) return true;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    } while (t - t0 < g_attn_q4_wait_ns);
    atomicOr(&g_attn_q4_err, 2);
    return false;
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const uint8_t *src, int bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// Eight codes of a word as fp16 pairs 2 c - 15: nibbles (0, 4), 16 x (1, 5), (2, 6), 16 x (3, 7).
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t h2sub(uint32_t x, uint32_t y) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&x), *reinterpret_cast<const __half2 *>(&y));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ void codes8(uint32_t w, uint32_t (&c)[4]) {
    const uint32_t w1 = w << 1, w8 = w >> 7;  // nibbles one bit up: 1024 + 2 c, 1024 + 32 c
    c[0] = h2sub(and_or(w1, 0x001e001eu, 0x64006400u), 0x640f640fu);
    c[1] = h2sub(and_or(w1, 0x01e001e0u, 0x64006400u), 0x64f064f0u);
    c[2] = h2sub(and_or(w8, 0x001e001eu, 0x64006400u), 0x640f640fu);
    c[3] = h2sub(and_or(w8, 0x01e001e0u, 0x64006400u), 0x64f064f0u);
}

// A place in the batch's order of tiles: sequences, their (kv head, head
// group) items, the item's tiles.  Work is divided in units: an item of nt
// tiles has Q4_ITEM + nt of them, the first ones for what its beginning and
// end cost, so that shares with many short items are not the last to finish
// (with items_only one unit, an item being one CTA's then).
struct Item {
    int b, j, kh, nt, pos;
    int tile, end;   // this warp's tiles of the item
    int unit, left;  // the item's first unit; units of this warp's share from there on
    long long off;   // contiguous: byte offset of the item's row 0 in a cache
    const int *row;  // paged: the sequence's table row
};
struct Part {  // of an item, left in shared memory by a warp: its first unit, sequence, heads, tiles [first, end) of nt
    int unit, b, head, heads, first, end, nt;
    int lost;  // a wait ran out: there is no result
};
__device__ __forceinline__ int seq_pos(const Q4Args &g, int b) {  // position, or -1 when the row has nothing to do
    const int p = __ldg(g.a.pos + b);
    return p < 0 || p >= g.a.S ? -1 : p;
}
__device__ __forceinline__ int item_units(const Q4Args &g, int nt) { return g.items_only ? 1 : nt + Q4_ITEM; }
// The item at (p.b, p.j), p.nt and p.pos known; its tiles up to the share's end.
template <int NB> __device__ __forceinline__ void set_item(const Q4Args &g, Item &p) {
    p.kh = g.HG == 1 ? p.j : p.j / g.HG;
    p.end = g.items_only ? (p.left > 0 ? p.nt : 0) : min(p.nt, p.left - Q4_ITEM);
    const long long cs = g.a.seq ? __ldg(g.a.seq + p.b) : p.b;
    p.row = g.a.pages + cs * g.a.max_pages;
    p.off = (cs * g.a.Hkv + p.kh) * g.a.S * Q4<NB>::RB;
}
template <int NB> __device__ __forceinline__ void set_seq(const Q4Args &g, Item &p) {  // first sequence >= p.b with work
    p.pos = -1;
    while (p.b < g.batch && (p.pos = seq_pos(g, p.b)) < 0) p.b++;
    p.nt = p.pos / Q4<NB>::T + 1;
}
// The share goes on behind the item.
__device__ __forceinline__ bool more_items(const Q4Args &g, const Item *at) { return at->left > item_units(g, at->nt); }
// The share's next item, in place (tile == end: of it there are no tiles).  The
// items of the copies and of the computation lie in shared memory: only what
// each tile needs is kept in registers.
template <int NB> __device__ __noinline__ void next_item(const Q4Args &g, Item *at) {
    Item p = *at;
    const int units = item_units(g, p.nt);
    p.unit += units;
    p.left -= units;
    p.tile = 0;
    if (++p.j == g.a.Hkv * g.HG) {
        p.j = 0;
        p.b++;
        set_seq<NB>(g, p);
    }
    set_item<NB>(g, p);
    p.end = max(p.end, 0);
    __syncwarp();
    *at = p;  // (every lane the same)
    __syncwarp();
}

__device__ __forceinline__ int checked_page(const AttnArgs &a, int pg, bool *ok) {  // page 0 for one outside the pool
    if ((unsigned)pg < (unsigned)a.n_pages) return pg;
    atomicOr(&g_attn_q4_err, 1);
    *ok = false;
    return 0;
}
// Byte offset of row t of an item in its cache; *ok: its page is in the pool.
template <int NB> __device__ __forceinline__ long long row_offset(const Q4Args &g, const Item &it, int t, bool *ok) {
    const AttnArgs &a = g.a;
    if (!a.pages) return it.off + (long long)t * Q4<NB>::RB;
    const int pg = checked_page(a, __ldg(it.row + (t >> a.page_shift)), ok);
    return ((long long)pg * a.Hkv + it.kh) * g.page_bytes + (long long)(t & ((1 << a.page_shift) - 1)) * Q4<NB>::RB;
}
// Starts the copies of a tile's rows, from any 4-byte phase: from the 16-byte
// boundary at or before the first row; the last copy reads no byte past the run.
template <int NB> __device__ __noinline__ void fetch_unaligned(const Q4Args &g, const Item *it, int tile, int rows, uint32_t stage) {
    bool ok;
    const long long off = row_offset<NB>(g, *it, tile * Q4<NB>::T, &ok);
    const int phase = (int)(off & 15), bytes = rows * Q4<NB>::RB + phase;  // (the caches themselves are aligned)
    const uint8_t *k = (const uint8_t *)g.a.k_cache + off - phase, *v = (const uint8_t *)g.a.v_cache + off - phase;
    for (int i = 16 * (threadIdx.x & 31); i < bytes; i += 512) {
        const int n = min(16, bytes - i);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(stage + i), "l"(k + i), "r"(n) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(stage + Q4<NB>::SIDE + i), "l"(v + i), "r"(n) : "memory");
    }
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
// Pairs (2 d, 2 d + 1) of dims d0 .. d0 + 7 rotated (src/ops_llama.c:39-48).
__device__ __forceinline__ void rope8(const AttnArgs &a, int pos, int Dh, int d0, float (&x)[8]) {
    if (!a.rope_cos) return;
    const size_t t = (size_t)pos * (Dh / 2) + d0 / 2;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float c = a.rope_cos[t + i], s = a.rope_sin[t + i], x0 = x[2 * i], x1 = x[2 * i + 1];
        x[2 * i] = x0 * c - x1 * s;
        x[2 * i + 1] = x0 * s + x1 * c;
    }
}

// ---------------------------------------------------------------------------
// A tile.  The positions are the rows of both products: of each 16 rows lane
// (g, t) holds the scores of rows 2 g and 2 g + 1, and the eight columns are
//   FEW    (at most four query heads per kv head) two parts of each head, so
//          columns 2 t, 2 t + 1 belong to head t and none is idle;
//   else   eight heads, columns 2 t, 2 t + 1 being heads 2 t, 2 t + 1.
// Scores: codes as bytes (nibbles of a word are two ANDs and a shift), q as
// 31-bit whole numbers in four signed bytes: integer products, exact.  FEW: two
// products, columns (byte 0, byte 1) and (byte 2, byte 3); else four, one for each byte.
// Output: p d as fp16 hi, lo, turned to the operand's order with movmatrix.
// FEW: hi and lo are a head's two columns; else two products.
// On this chip a warp-level MMA keeps the integer and half pipes from issuing
// (8 cycles each, measured in one loop with them), so their number counts: FEW
// has 32 for 32 rows of 128 dims, the other form 64.  4 heads per kv head of
// 128 dims, the other form against FEW: one sequence of 131072 positions 58.0
// -> 44.7 us, 128 ragged ones 115.1 -> 85.3; one head (GPT-2, 700 positions) 8.2
// -> 7.7.  Eight heads would take FEW twice, at 0.74 of the other's time each.
struct QGroup {  // of a head's q
    float w;       // factor of the group's whole numbers (a power of two; 1 for the head's largest)
    float hi, lo;  // the sums of their upper two bytes, times 2^16, and of the lower two: exact
};
template <int NB, bool FEW> struct State {
    static constexpr int HL = FEW ? 1 : 2;  // heads of a lane
    static constexpr int LP = FEW ? 2 : 4;  // products of q's bytes
    uint32_t q[LP][NB][2];                  // q as matrix operands
    QGroup qg[Q4<NB>::NG][HL];
    float qfac[HL];                         // the factor of the scores
    float2 o[2 * NB][2];                    // dims x this lane's two columns
    float om[Q4<NB>::NG][HL], l[HL];        // this lane's positions: sum p (m + 7.5 d), sum p
    float mx[HL];                           // maximum of s over qfac; p is 2^(s - max)
    float pd[Q4<NB>::NG][HL];               // largest p d so far; o is times 2^(141 - pd_exponent(pd))
};

__device__ __forceinline__ void imma(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turned(uint32_t x) {  // 8 x 8 halves of the warp, transposed
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// This lane's values of query `head` of the item's kv head (0 for heads past the last one).
template <int NB> __device__ __forceinline__ void fetch_q(const Q4Args &g, const Item &p, int lane, int head, float (&x)[NB][8]) {
#pragma unroll
    for (int i = 0; i < NB; i++) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[i][e] = 0.0f;
        if (head < g.G) load8(g.a.q + (size_t)p.b * g.a.ldq + ((size_t)p.kh * g.G + head) * Q4<NB>::DH + 32 * i + 8 * (lane & 3), g.vec, x[i]);
    }
}
// Lane (n, t) makes column n's operand: FEW: head n / 2, n odd: the middle byte (and 0), even: the top (and low) one.
template <int NB, bool FEW> __device__ __forceinline__ int q_head(const Q4Args &g, const Item &p, int lane) {
    return FEW ? lane >> 3 : (p.j - p.kh * g.HG) * 8 + (lane >> 2);
}
template <int NB, bool FEW>
__device__ __forceinline__ void load_q(const Q4Args &g, const Item &p, int lane, float (&x)[NB][8], State<NB, FEW> &st) {
    using S = State<NB, FEW>;
    const AttnArgs &a = g.a;
    constexpr int DH = Q4<NB>::DH, NG = Q4<NB>::NG;
    const int t = lane & 3;
    const bool odd = lane & 4;
    // a power of two that brings the group's largest |q| into [2^29, 2^30): four signed bytes hold it
    float big[NG] = {}, bad = 0.0f;  // (NaN when a value is)
    int ex[NG], top = -97;
#pragma unroll
    for (int i = 0; i < NB; i++) {
        rope8(a, p.pos, DH, 32 * i + 8 * t, x[i]);
#pragma unroll
        for (int e = 0; e < 8; e++) big[i / 2] = max_nan(big[i / 2], fabsf(x[i][e]));
    }
#pragma unroll
    for (int j = 0; j < NG; j++) {
        big[j] = max_nan(big[j], __shfl_xor_sync(0xffffffffu, big[j], 1));
        big[j] = max_nan(big[j], __shfl_xor_sync(0xffffffffu, big[j], 2));
        bad += big[j] - big[j];  // NaN, and with it every score, when a value is not finite; else 0
        ex[j] = min(max((int)(__float_as_uint(big[j]) >> 23) - 127, -97), 127);
        top = max(top, ex[j]);
    }
    int sum[NG][2] = {};  // of the upper two bytes (as one number) and of the lower two: exact
#pragma unroll
    for (int i = 0; i < NB; i++) {
        const float up = __uint_as_float((uint32_t)(127 + 29 - ex[i / 2]) << 23);
        uint32_t byte[4][2] = {};  // the highest first; each 128 more
#pragma unroll
        for (int e = 0; e < 8; e++) {  // dims 0, 2, 4, 6 of the word: its low nibbles; 1, 3, 5, 7: its high ones
            const uint32_t b = (uint32_t)__float2int_rn(x[i][e] * up) + 0x80808080u;
#pragma unroll
            for (int k = 0; k < 4; k++) byte[k][e & 1] |= (b >> (24 - 8 * k) & 0xffu) << (8 * (e >> 1));
        }
        int n[4] = {};
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int b = 0; b < 4; b++) {
                byte[b][k] ^= 0x80808080u;
                n[b] = __dp4a((int)byte[b][k], 0x01010101, n[b]);
            }
        sum[i / 2][0] += n[0] * 256 + n[1];
        sum[i / 2][1] += n[2] * 256 + n[3];
#pragma unroll
        for (int k = 0; k < 2; k++) {
#pragma unroll
            for (int b = 0; b < S::LP; b++) st.q[b][i][k] = FEW ? (odd ? byte[2 * b + 1][k] : byte[2 * b][k]) : byte[b][k];
        }
    }
    // lane (g, t) goes on with the heads of columns 2 t (and 2 t + 1)
#pragma unroll
    for (int j = 0; j < NG; j++)
#pragma unroll
        for (int k = 0; k < 2; k++) {
            sum[j][k] += __shfl_xor_sync(0xffffffffu, sum[j][k], 1);
            sum[j][k] += __shfl_xor_sync(0xffffffffu, sum[j][k], 2);
        }
    const float fac = LOG2E / sqrtf((float)DH) * __uint_as_float((uint32_t)(127 - 29 + top) << 23);
#pragma unroll
    for (int hl = 0; hl < S::HL; hl++) {
        st.qfac[hl] = __shfl_sync(0xffffffffu, fac, 8 * t + 4 * hl);
#pragma unroll
        for (int j = 0; j < NG; j++) {
            const int hi = __shfl_sync(0xffffffffu, sum[j][0], 8 * t + 4 * hl), lo = __shfl_sync(0xffffffffu, sum[j][1], 8 * t + 4 * hl);
            // (2^-126 for less: below what a score can show)
            const float w = __uint_as_float((uint32_t)max(127 + __shfl_sync(0xffffffffu, ex[j] - top, 8 * t + 4 * hl), 1) << 23);
            st.qg[j][hl] = {w, 65536.0f * (float)hi + __shfl_sync(0xffffffffu, bad, 8 * t + 4 * hl), (float)lo};
            st.om[j][hl] = 0.0f;
            st.pd[j][hl] = 0.0f;
        }
        st.l[hl] = 0.0f;
        st.mx[hl] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) st.o[i][0] = st.o[i][1] = make_float2(0.0f, 0.0f);
}

// The new K and V rows quantized into `fresh` (two rows) and, by the first
// head group, into the cache.
template <int NB> __device__ __forceinline__ void append(const Q4Args &g, const Item &p, uint32_t *fresh, int lane) {
    const AttnArgs &a = g.a;
    constexpr int DH = Q4<NB>::DH, NW = DH / 8, RB = Q4<NB>::RB;
    constexpr int SIDES = NW <= 16 ? 2 : 1;  // K in lanes 0-15, V in lanes 16-31 when they fit
    bool ok = true;
    const long long off = row_offset<NB>(g, p, p.pos, &ok);
    ok &= p.j == p.kh * g.HG;
#pragma unroll 1
    for (int side0 = 0; side0 < 2; side0 += SIDES) {
        const int side = SIDES == 2 ? lane >> 4 : side0, w = SIDES == 2 ? lane & 15 : lane;
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (w < NW) {
            load8((side ? a.v_new : a.k_new) + (size_t)p.b * a.ldkv + (size_t)p.kh * DH + 8 * w, g.vec, x);
            if (!side) rope8(a, p.pos, DH, 8 * w, x);
        }
        uint32_t codes, dm;
        kv_q4_quantize<32 / SIDES>(x, w < NW, codes, dm);
        uint32_t *dst = reinterpret_cast<uint32_t *>((uint8_t *)(side ? a.v_cache : a.k_cache) + off);
        if (w < NW) {
            fresh[side * (RB / 4) + w] = codes;
            if (ok) dst[w] = codes;
            if (w % 8 == 0) {
                fresh[side * (RB / 4) + NW + w / 8] = dm;
                if (ok) dst[NW + w / 8] = dm;
            }
        }
    }
}

// The (d, m) words of row r.
template <int NB> __device__ __forceinline__ void row_factors(const uint8_t *rows, int r, uint32_t (&w)[Q4<NB>::NG]) {
    constexpr int RB = Q4<NB>::RB, NG = Q4<NB>::NG, DH = Q4<NB>::DH;
    const uint8_t *at = rows + r * RB + DH / 2;
    if constexpr (NG % 2 == 0 && RB % 8 == 0) {
#pragma unroll
        for (int j = 0; j < NG; j += 2) {
            const uint2 v = *reinterpret_cast<const uint2 *>(at + 4 * j);
            w[j] = v.x;
            w[j + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NG; j++) w[j] = *reinterpret_cast<const uint32_t *>(at + 4 * j);
    }
}

// One tile: n valid rows at kt / vt (row r at r * RB).
template <int NB, bool FEW>
__device__ __forceinline__ void attend_tile(State<NB, FEW> &st, const uint8_t *kt, const uint8_t *vt, int n, int lane) {
    using S = State<NB, FEW>;
    constexpr int RB = Q4<NB>::RB, NG = Q4<NB>::NG, T = Q4<NB>::T, NH = T / 16, HL = S::HL;
    const int gq = lane >> 2, t = lane & 3;
    float s[NH][2][HL];  // scores over qfac of rows 16 h + 2 g, + 1
#pragma unroll
    for (int h = 0; h < NH; h++) {
        const uint32_t *const k0 = reinterpret_cast<const uint32_t *>(kt + (16 * h + 2 * gq) * RB) + t, *const k1 = k0 + RB / 4;
        uint32_t f[2][NG];
        row_factors<NB>(kt, 16 * h + 2 * gq, f[0]);
        row_factors<NB>(kt, 16 * h + 2 * gq + 1, f[1]);
#pragma unroll
        for (int j = 0; j < NG; j++) {
            int c[S::LP][4] = {};
#pragma unroll
            for (int i = 2 * j; i < 2 * j + 2 && i < NB; i++) {
                const uint32_t w0 = k0[4 * i], w1 = k1[4 * i];
                const uint32_t a0 = w0 & 0x0f0f0f0fu, a1 = w1 & 0x0f0f0f0fu, a2 = w0 >> 4 & 0x0f0f0f0fu, a3 = w1 >> 4 & 0x0f0f0f0fu;
#pragma unroll
                for (int b = 0; b < S::LP; b++) imma(c[b], a0, a1, a2, a3, st.q[b][i][0], st.q[b][i][1]);
            }
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const float2 d = __half22float2(*reinterpret_cast<const __half2 *>(&f[r][j]));
                const float d16 = 65536.0f * d.x;
#pragma unroll
                for (int hl = 0; hl < HL; hl++) {
                    // the sums of the upper and of the lower two bytes: below 2^24, exact in fp32, and below
                    // 2^25, off by 1 at most
                    const int hi = FEW ? c[0][2 * r] * 256 + c[0][2 * r + 1] : c[0][2 * r + hl] * 256 + c[1][2 * r + hl];
                    const int lo = FEW ? c[1][2 * r] * 256 + c[1][2 * r + 1] : c[S::LP - 2][2 * r + hl] * 256 + c[S::LP - 1][2 * r + hl];
                    // d (q . c) and m sum(q) may cancel: the first one's rounding goes into the low part
                    const float t = d16 * (float)hi, low = fmaf(d.x, (float)lo, fmaf(d.y, st.qg[j][hl].lo, fmaf(d16, (float)hi, -t)));
                    const float x = fmaf(d.y, st.qg[j][hl].hi, t) + low;
                    s[h][r][hl] = NG == 1 ? x : j ? fmaf(x, st.qg[j][hl].w, s[h][r][hl]) : x * st.qg[j][hl].w;
                }
            }
        }
    }
    uint32_t vf[NH][2][NG];  // (d, m) words of the values' rows
#pragma unroll
    for (int h = 0; h < NH; h++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
            row_factors<NB>(vt, 16 * h + 2 * gq + r, vf[h][r]);
            if (16 * h + 2 * gq + r >= n) {  // past the end
#pragma unroll
                for (int hl = 0; hl < HL; hl++) s[h][r][hl] = -INFINITY;
#pragma unroll
                for (int j = 0; j < NG; j++) vf[h][r][j] = 0u;
            }
        }
    float f[HL];
#pragma unroll
    for (int hl = 0; hl < HL; hl++) {  // running maximum
        float m = fmaxf(s[0][0][hl], s[0][1][hl]);
#pragma unroll
        for (int h = 1; h < NH; h++) m = fmaxf(m, fmaxf(s[h][0][hl], s[h][1][hl]));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        m = fmaxf(m, st.mx[hl]);
        f[hl] = ex2((st.mx[hl] - m) * st.qfac[hl]);  // (2^-inf = 0 the first time)
        st.mx[hl] = m;
        float l = 0.0f;  // (a tile's sums by themselves: small terms would be lost one by one beside a large one)
#pragma unroll
        for (int h = 0; h < NH; h++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                s[h][r][hl] = ex2((s[h][r][hl] - m) * st.qfac[hl]);
                l += s[h][r][hl];
            }
        st.l[hl] = fmaf(st.l[hl], f[hl], l);
    }
    // largest p d of each group and head: the upper halves of two of them in a word
    uint32_t top[(NG * HL + 1) / 2] = {};
#pragma unroll
    for (int j = 0; j < NG; j++)
#pragma unroll
        for (int hl = 0; hl < HL; hl++) {
            float x = 0.0f;
#pragma unroll
            for (int h = 0; h < NH; h++)
#pragma unroll
                for (int r = 0; r < 2; r++) x = fmaxf(x, s[h][r][hl] * __low2float(*reinterpret_cast<const __half2 *>(&vf[h][r][j])));
            const int i = j * HL + hl;
            top[i / 2] = __byte_perm(top[i / 2], __float_as_uint(x), i % 2 ? 0x7610 : 0x3276);
        }
#pragma unroll
    for (int i = 0; i < (NG * HL + 1) / 2; i++)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top[i] = max_u16x2(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
#pragma unroll
    for (int j = 0; j < NG; j++) {
        constexpr int PB = FEW ? 1 : 2;  // products of p d
        uint32_t b[NH][PB][2];           // p d of the 16 rows of each set: rows 2 g, 2 g + 1
        float om[HL] = {}, up[HL], ff[HL];
#pragma unroll
        for (int hl = 0; hl < HL; hl++) {
            const int i = j * HL + hl, was = pd_exponent(st.pd[j][hl]);
            // the largest so far goes down with its weight
            st.pd[j][hl] = fmaxf(__uint_as_float(i % 2 ? top[i / 2] & 0xffff0000u : top[i / 2] << 16), st.pd[j][hl] * f[hl]);
            const int e = pd_exponent(st.pd[j][hl]);
            up[hl] = __uint_as_float((uint32_t)(127 + 141 - e) << 23);
            ff[hl] = f[hl] * __uint_as_float((uint32_t)(127 + was - e) << 23);
        }
        const float2 ff2 = make_float2(ff[0], ff[HL - 1]);
#pragma unroll
        for (int h = 0; h < NH; h++) {
            const float2 d0 = __half22float2(*reinterpret_cast<const __half2 *>(&vf[h][0][j])), d1 = __half22float2(*reinterpret_cast<const __half2 *>(&vf[h][1][j]));
            const float m0 = fmaf(7.5f, d0.x, d0.y), m1 = fmaf(7.5f, d1.x, d1.y);
            float x0[HL], x1[HL];
#pragma unroll
            for (int hl = 0; hl < HL; hl++) {
                om[hl] = fmaf(s[h][0][hl], m0, fmaf(s[h][1][hl], m1, om[hl]));
                x0[hl] = s[h][0][hl] * d0.x * up[hl];
                x1[hl] = s[h][1][hl] * d1.x * up[hl];
            }
            uint32_t hi, lo;
            if (FEW) {
                split2(x0[0], x1[0], hi, lo);
                b[h][0][0] = turned(__byte_perm(hi, lo, 0x5410));  // row 2 g: (hi, lo)
                b[h][0][1] = turned(__byte_perm(hi, lo, 0x7632));
            } else {
                split2(x0[0], x0[HL - 1], hi, lo);  // row 2 g: both heads
                b[h][0][0] = turned(hi);
                b[h][PB - 1][0] = turned(lo);
                split2(x1[0], x1[HL - 1], hi, lo);
                b[h][0][1] = turned(hi);
                b[h][PB - 1][1] = turned(lo);
            }
        }
#pragma unroll
        for (int hl = 0; hl < HL; hl++) st.om[j][hl] = fmaf(st.om[j][hl], f[hl], om[hl]);
        // this lane's dims: word g of the group, or half a word of a group of 32
        const bool half = NB % 2 && j == NG - 1;
        const uint8_t *vr = vt + 4 * t * RB + 32 * j + (half ? 4 * (gq >> 1) : 4 * gq);
#pragma unroll
        for (int k = 0; k < (half ? 1 : 2); k++) {  // nibbles 0-3, 4-7 of the words (or the half word's four)
            const uint32_t sel = half ? ((gq & 1) ? 0x7632u : 0x5410u) : (k ? 0x7632u : 0x5410u);
            const int i = 4 * j + 2 * k;
            float c[2][4];
#pragma unroll
            for (int h = 0; h < NH; h++) {
                uint32_t cw[4], x[4], y[4];  // rows 4 t + (0, 2) and (1, 3)
#pragma unroll
                for (int r = 0; r < 4; r++) cw[r] = *reinterpret_cast<const uint32_t *>(vr + (16 * h + r) * RB);
                codes8(__byte_perm(cw[0], cw[2], sel), x);
                codes8(__byte_perm(cw[1], cw[3], sel), y);
#pragma unroll
                for (int b_ = 0; b_ < PB; b_++) {
                    if (h || b_) {
                        hmma(c[0], x[0], x[1], y[0], y[1], b[h][b_][0], b[h][b_][1]);
                        hmma(c[1], x[2], x[3], y[2], y[3], b[h][b_][0], b[h][b_][1]);
                    } else {
                        hmma0(c[0], x[0], x[1], y[0], y[1], b[h][b_][0], b[h][b_][1]);
                        hmma0(c[1], x[2], x[3], y[2], y[3], b[h][b_][0], b[h][b_][1]);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                st.o[i + e][0] = fma2(st.o[i + e][0], ff2, make_float2(c[e][0], c[e][1]));
                st.o[i + e][1] = fma2(st.o[i + e][1], ff2, make_float2(c[e][2], c[e][3]));
            }
        }
    }
}

// The item's result over its tiles so far, to dst + h * ld (heads h < heads
// of the group of 8): with fin divided by the sum; else the sums themselves,
// with the maximum of s and the sum of p behind them.  Lane (g, t) holds its
// heads' dims 8 g .. 8 g + 7 of each group of 64 (4 g .. 4 g + 3 of one of 32).
template <int NB, bool FEW>
__device__ __forceinline__ void result(const State<NB, FEW> &st, int lane, float *dst, int ld, int heads, bool fin, bool vec) {
    using S = State<NB, FEW>;
    const int gq = lane >> 2, t = lane & 3;
#pragma unroll
    for (int hl = 0; hl < S::HL; hl++) {
        const int h = S::HL * t + hl;
        float l = st.l[hl];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (!fin && gq == 0 && h < heads) {
            dst[h * ld + Q4<NB>::DH] = st.mx[hl] * st.qfac[hl];
            dst[h * ld + Q4<NB>::DH + 1] = l;
        }
        const float iv = fin ? 1.0f / l : 1.0f;
#pragma unroll
        for (int j = 0; j < Q4<NB>::NG; j++) {
            float m = st.om[j][hl];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
            // 2^(e - 142), 0 for 2^-127, and a 16th of it for the nibbles whose codes are times 16
            const float low = __uint_as_float((uint32_t)(pd_exponent(st.pd[j][hl]) - 15) << 23), high = low * 0.0625f;
            const bool half = NB % 2 && j == Q4<NB>::NG - 1;
#pragma unroll
            for (int k = 0; k < (half ? 1 : 2); k++) {
                const float2 *a = st.o[4 * j + 2 * k], *b = st.o[4 * j + 2 * k + 1];
                auto col = [&](const float2 &v) { return FEW ? v.x + v.y : hl ? v.y : v.x; };  // (hi and lo, or the head's)
                const float4 v = make_float4(fmaf(col(a[0]), low, m) * iv, fmaf(col(a[1]), high, m) * iv, fmaf(col(b[0]), low, m) * iv,
                                             fmaf(col(b[1]), high, m) * iv);
                float *o = dst + h * ld + 64 * j + (half ? 4 * gq : 8 * gq + 4 * k);
                if (h >= heads) continue;
                if (vec) *reinterpret_cast<float4 *>(o) = v;
                else { o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w; }
            }
        }
    }
}

// After a wait that ran out: the rest of the warp's share, from the item `at` on,
// has no result.  Its heads' outputs become NaN, here or where parts are merged.
template <int NB> __device__ __noinline__ void lose_items(const Q4Args &g, Item *at, Part *desc, int part, int lane) {
    const AttnArgs &a = g.a;
    constexpr int DH = Q4<NB>::DH;
    while (at->tile < at->end) {
        const int h0 = (at->j - at->kh * g.HG) * 8, heads = min(8, g.G - h0), head = at->kh * g.G + h0;
        if (at->tile == 0 && at->end == at->nt) {
            float *o = a.out + (size_t)at->b * a.ldo + (size_t)head * DH;
            for (int i = lane; i < heads * DH; i += 32) o[i] = NAN;
            if (lane < heads && a.nsplit > 1)
                a.ws[((size_t)at->b * a.H + head + lane) * ((size_t)a.nsplit * (DH + 2)) + DH + 1] = 0.0f;
        } else if (lane == 0) {
            desc[part] = Part{at->unit, at->b, head, heads, at->tile, at->end, at->nt, 1};
        }
        part = 1;
        if (!more_items(g, at)) break;
        next_item<NB>(g, at);
    }
}

template <int NB, bool FEW>
__global__ void __launch_bounds__(32 * Q4_WARPS, 2) k_attn_q4(const __grid_constant__ Q4Args g) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Item sh_item[Q4_WARPS][2];  // of the copies, of the computation
    __shared__ __align__(8) uint64_t sh_bar[Q4_WARPS][Q4_STAGES];
    __shared__ int sh_total[Q4_WARPS];
    __shared__ Part desc[Q4_WARPS][2];
    constexpr int DH = Q4<NB>::DH, SLOT = Q4<NB>::SLOT, RB = Q4<NB>::RB, T = Q4<NB>::T;
    const AttnArgs &a = g.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int G = g.G, items = a.Hkv * g.HG, GH = min(G, 8);
    if (lane == 0) {
        desc[warp][0].unit = desc[warp][1].unit = -1;
        for (int i = 0; i < Q4_STAGES; i++)
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"((uint32_t)__cvta_generic_to_shared(&sh_bar[warp][i])));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    pdl_wait();
    pdl_launch_dependents();
    // units (tiles) of the whole batch, and this CTA's and this warp's share
    auto units_at = [&](int pos) -> int { return pos < 0 ? 0 : item_units(g, pos / T + 1) * items; };
    // up to 32 sequences: each warp sums them by itself
    auto scan = [&](int mine) {  // inclusive sum over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, mine, o);
            if (lane >= o) mine += y;
        }
        return mine;
    };
    const bool small = g.batch <= 32;
    int pos = -1, mine = 0, inc = 0, total;  // lane's sequence
    if (small) {
        if (lane < g.batch) pos = seq_pos(g, lane);
        mine = units_at(pos);
        inc = scan(mine);
        total = __shfl_sync(0xffffffffu, inc, 31);
    } else {
        int sum = 0;
        for (int b = threadIdx.x; b < g.batch; b += 32 * Q4_WARPS) sum += units_at(seq_pos(g, b));
        sum = __reduce_add_sync(0xffffffffu, sum);
        if (lane == 0) sh_total[warp] = sum;
        __syncthreads();
        total = sh_total[0] + sh_total[1] + sh_total[2] + sh_total[3];
    }
    const int nC = min((int)gridDim.x, max(1, total / g.rmin));
    if ((int)blockIdx.x >= nC || total == 0) return;
    // CTA i has per or (the first `more`) per + 1 units, a warp the like of them
    const int per = total / nC, more = total - per * nC;
    auto cta_of = [&](int unit) { return unit < more * (per + 1) ? unit / (per + 1) : more + (unit - more * (per + 1)) / per; };
    const int cta = blockIdx.x, c0 = cta * per + min(cta, more), cn = per + (cta < more);
    const int wn = cn / Q4_WARPS, wm = cn % Q4_WARPS, u0 = c0 + warp * wn + min(warp, wm), u1 = u0 + wn + (warp < wm);
    uint8_t *const ring = smem + warp * Q4<NB>::WARP_BYTES;
    uint32_t *const fresh = reinterpret_cast<uint32_t *>(ring + Q4_STAGES * Q4<NB>::STAGE);
    float *const slots = reinterpret_cast<float *>(smem + Q4_WARPS * Q4<NB>::WARP_BYTES);  // [warp][GH][SLOT]
    const size_t hstride = (size_t)a.nsplit * (DH + 2);

    if (u0 < u1) {
        // where unit u0 lies
        Item p;
        p.b = p.pos = 0;
        int before = 0;
        for (int b0 = 0; b0 < g.batch; b0 += 32) {
            if (!small) {
                pos = b0 + lane < g.batch ? seq_pos(g, b0 + lane) : -1;
                mine = units_at(pos);
                inc = scan(mine);
            }
            const unsigned hit = __ballot_sync(0xffffffffu, before + inc > u0);
            if (hit) {
                const int w = __ffs(hit) - 1;
                p.b = b0 + w;
                p.pos = __shfl_sync(0xffffffffu, pos, w);
                before += __shfl_sync(0xffffffffu, inc - mine, w);
                break;
            }
            before += __shfl_sync(0xffffffffu, inc, 31);
        }
        p.nt = p.pos / T + 1;
        const int at = u0 - before, units = item_units(g, p.nt);
        p.j = at / units;
        const int within = at - p.j * units;
        p.unit = u0 - within;
        p.left = u1 - p.unit;
        p.tile = g.items_only ? 0 : max(0, within - Q4_ITEM);
        set_item<NB>(g, p);
        Item *const ia = &sh_item[warp][0], *const ii = &sh_item[warp][1];
        *ia = p;
        *ii = p;
        __syncwarp();
        // The copies' place: tiles [a_tile, a_end) of an item of which a_rows
        // rows are copied.  Lanes 0-3 copy the K rows' runs, lanes 4-7 the V
        // rows'; a lane looks its page up one tile ahead.
        const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring), bar = (uint32_t)__cvta_generic_to_shared(&sh_bar[warp][0]);
        const uint8_t *const cache = (const uint8_t *)(lane & 4 ? a.v_cache : a.k_cache);
        const int r0 = (lane & 3) * g.run;  // first row of this lane's run; T or more: it has none
        const uint32_t to = (lane & 4 ? Q4<NB>::SIDE : 0) + r0 * RB;
        int a_tile, a_end, a_rows, a_pg = 0;
        auto look_up = [&]() {
            if (a.pages && a_tile * T + r0 < a_rows && r0 < T) a_pg = __ldg(ia->row + ((a_tile * T + r0) >> a.page_shift));
        };
        auto item_ahead = [&](int i) {  // its first tile goes into stage i
            a_tile = ia->tile;
            a_end = ia->end;
            if (ia->j == g.lose_j && a_tile <= g.lose_tile && g.lose_tile < a_end && lane == 0)
                asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], 16;" ::"r"(bar + 8 * i) : "memory");
            a_rows = a.append ? ia->pos : ia->pos + 1;
            look_up();
        };
        auto fetch = [&](int i) {  // tile a_tile into stage i
            const int rows = min(T, a_rows - a_tile * T);
            const uint32_t stage = ring_s + i * Q4<NB>::STAGE;
            if (!g.bulk) {
                if (rows > 0) fetch_unaligned<NB>(g, ia, a_tile, rows, stage);
                return;
            }
            const int some = rows > 0 ? (rows + 3) & ~3 : 0;  // (at most three rows more, of the same page or cache)
            if (lane == 0) bar_expect(bar + 8 * i, 2 * some * RB);
            __syncwarp();
            if (lane < 8 && r0 < some) {
                long long off;
                if (a.pages) {
                    bool ok;
                    off = ((long long)checked_page(a, a_pg, &ok) * a.Hkv + ia->kh) * g.page_bytes +
                          (long long)((a_tile * T + r0) & ((1 << a.page_shift) - 1)) * RB;
                } else {
                    off = ia->off + (long long)a_tile * (T * RB);
                }
                bulk_copy(stage + to, cache + off, min(g.run, some - r0) * RB, bar + 8 * i);
            }
        };
        item_ahead(0);
        int tile = p.tile, end = p.end, nt = p.nt, phase = 0, part = 0, stage = 0, fill = 0;
        uint32_t parity = 0, flying = 0;  // phase bits of the stages' barriers; stages whose copies are not waited for
        bool begin = true;
        State<NB, FEW> st;
#pragma unroll 1
        for (int skip = Q4_STAGES - 1; tile < end; skip--) {  // the first turns only start copies
            if (a_tile < a_end) {
                fetch(fill);
                flying |= 1u << fill;
                if (++a_tile == a_end) {
                    if (more_items(g, ia)) {
                        next_item<NB>(g, ia);
                        item_ahead(fill + 1 == Q4_STAGES ? 0 : fill + 1);
                    } else {
                        a_tile = a_end = 0;
                    }
                } else {
                    look_up();
                }
            }
            if (!g.bulk) asm volatile("cp.async.commit_group;" ::: "memory");
            fill = fill + 1 == Q4_STAGES ? 0 : fill + 1;
            if (skip > 0) continue;
            if (begin) {
                phase = g.bulk ? 0 : (int)(ii->off & 15);  // rows lie in the ring at the phase that they have in the cache
                float x[NB][8];
                fetch_q<NB>(g, *ii, lane, q_head<NB, FEW>(g, *ii, lane), x);
                if (a.append && end == nt) append<NB>(g, *ii, fresh, lane);  // (while q is on its way)
                load_q<NB, FEW>(g, *ii, lane, x, st);
                begin = false;
            }
            if (!g.bulk) {
                asm volatile("cp.async.wait_group %0;" ::"n"(Q4_STAGES - 1) : "memory");
                __syncwarp();
            } else {
                bool here = bar_try(bar + 8 * stage, parity >> stage & 1);
                if (!here) here = bar_wait_long(bar + 8 * stage, parity >> stage & 1);
                if (!__all_sync(0xffffffffu, here)) break;  // gave up, tile < end (lmc_device_status)
                parity ^= 1u << stage;
            }
            flying &= ~(1u << stage);
            uint8_t *kt = ring + stage * Q4<NB>::STAGE + phase;
            stage = stage + 1 == Q4_STAGES ? 0 : stage + 1;
            int n = T;
            if (tile == nt - 1) {  // the item's last tile: fewer rows, the new row among them
                n = ii->pos + 1 - tile * T;
                if (a.append) {
                    for (int i = lane; i < RB / 4; i += 32) {
                        reinterpret_cast<uint32_t *>(kt + (n - 1) * RB)[i] = fresh[i];
                        reinterpret_cast<uint32_t *>(kt + Q4<NB>::SIDE + (n - 1) * RB)[i] = fresh[RB / 4 + i];
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the stage's next bulk copy
                    __syncwarp();
                }
            }
            attend_tile<NB, FEW>(st, kt, kt + Q4<NB>::SIDE, n, lane);
            __syncwarp();  // the stage is read; it may be written again
            if (++tile == end) {  // the item, or this warp's part of it, ends
                const int b = ii->b, kh = ii->kh, first = ii->tile;
                const int h0 = (ii->j - kh * g.HG) * 8, heads = min(8, G - h0), head = kh * G + h0;
                const bool whole = first == 0 && end == nt;
                float *slot = part ? reinterpret_cast<float *>(ring) : slots + warp * GH * SLOT;
                result<NB, FEW>(st, lane, whole ? a.out + (size_t)b * a.ldo + (size_t)head * DH : slot, whole ? DH : SLOT, heads, whole, !whole || g.vec);
                if (whole) {
                    if (lane < heads && a.nsplit > 1)  // nothing for the combine kernel to do
                        a.ws[((size_t)b * a.H + head + lane) * hstride + DH + 1] = 0.0f;
                } else if (lane == 0) {
                    desc[warp][part] = Part{ii->unit, b, head, heads, first, end, nt, 0};
                }
                part = 1;
                if (!more_items(g, ii)) break;
                next_item<NB>(g, ii);
                tile = ii->tile;
                end = ii->end;
                nt = ii->nt;
                begin = true;
            }
        }
        // (after a wait that ran out) the copies still in flight, bounded again
        for (int i = 0; g.bulk && i < Q4_STAGES; i++)
            if (flying >> i & 1) bar_wait_long(bar + 8 * i, parity >> i & 1);
        if (tile < end) lose_items<NB>(g, ii, desc[warp], part, lane);
    }
    __syncthreads();
    // merge this CTA's parts of each item: neighbours in (warp, part) order
    constexpr int PARTS = 2 * Q4_WARPS;
    const int id = lane < PARTS ? desc[lane >> 1][lane & 1].unit : -1;
    unsigned todo = __ballot_sync(0xffffffffu, id >= 0);
    while (todo) {
        const int k = __ffs(todo) - 1, unit = __shfl_sync(0xffffffffu, id, k);
        const unsigned parts = __ballot_sync(0xffffffffu, id == unit);
        todo &= ~parts;
        const int e = 31 - __clz(parts);
        const Part d = desc[k >> 1][k & 1];
        const bool whole = d.first == 0 && desc[e >> 1][e & 1].end == d.nt;
        // the slot is this CTA's place among those that hold the item's tiles
        const int slot = whole ? 0 : cta - cta_of(unit + Q4_ITEM);
        const bool last = !whole && cta_of(unit + Q4_ITEM + d.nt - 1) == cta;
        const bool lost = __ballot_sync(0xffffffffu, lane < PARTS && (parts >> lane & 1) && desc[lane >> 1][lane & 1].lost);
        for (int i = threadIdx.x; i < d.heads * (DH / 4); i += 32 * Q4_WARPS) {
            const int h = i / (DH / 4), x = 4 * (i % (DH / 4));
            float M = -INFINITY, L = 0.0f, m[PARTS], l[PARTS];
            float4 v[PARTS], acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int q = 0; q < PARTS; q++) {
                const float *s = (q % 2 ? reinterpret_cast<const float *>(smem + (q / 2) * Q4<NB>::WARP_BYTES) : slots + (q / 2) * GH * SLOT) + h * SLOT;
                m[q] = -INFINITY;
                if ((parts >> q & 1) && !lost) {
                    m[q] = s[DH];
                    l[q] = s[DH + 1];
                    v[q] = *reinterpret_cast<const float4 *>(s + x);
                }
                M = fmaxf(M, m[q]);
            }
#pragma unroll
            for (int q = 0; q < PARTS; q++)
                if ((parts >> q & 1) && !lost) {
                    const float f = ex2(m[q] - M);
                    L = fmaf(l[q], f, L);
                    acc.x = fmaf(v[q].x, f, acc.x);
                    acc.y = fmaf(v[q].y, f, acc.y);
                    acc.z = fmaf(v[q].z, f, acc.z);
                    acc.w = fmaf(v[q].w, f, acc.w);
                }
            if (lost) L = NAN;  // (and with it the item's output)
            float *w = a.ws + ((size_t)d.b * a.H + d.head + h) * hstride;
            if (whole) {
                const float iv = 1.0f / L;
                acc = make_float4(acc.x * iv, acc.y * iv, acc.z * iv, acc.w * iv);
                float *o = a.out + (size_t)d.b * a.ldo + (size_t)(d.head + h) * DH + x;
                if (g.vec) *reinterpret_cast<float4 *>(o) = acc;
                else { o[0] = acc.x; o[1] = acc.y; o[2] = acc.z; o[3] = acc.w; }
                if (x == 0 && a.nsplit > 1) w[DH + 1] = 0.0f;
            } else {
                w += (size_t)slot * (DH + 2);
                w[x] = acc.x; w[x + 1] = acc.y; w[x + 2] = acc.z; w[x + 3] = acc.w;
                if (x == 0) {
                    w[DH] = M;
                    // the sum; its sign bit marks the item's last part
                    w[DH + 1] = __uint_as_float((__float_as_uint(L) & 0x7fffffffu) | (last ? 0x80000000u : 0u));
                }
            }
        }
    }
}

// Merges the parts of each (row, query head) that several CTAs left in the
// workspace; nothing to do when slot 0's sum is zero.  W warps (1 or 4) share
// a head's parts: four when there are few heads, whose parts are then many
// (131072 positions of one sequence, 56 parts for each of 32 heads, the whole
// call: 49.8 us with one, 44.7 with four; 128 sequences of 32 heads 85.3 and 89.2).
template <int W> __global__ void __launch_bounds__(128) k_q4_combine(AttnArgs a, int batch) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float sh[W == 1 ? 1 : 4][256];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned id = W == 1 ? blockIdx.x * 4 + warp : blockIdx.x;  // (batch x H is an int)
    const int b = (int)(id / (unsigned)a.H), h = (int)(id - (unsigned)b * a.H), Dh = a.Dh;
    if (b >= batch) return;
    const int pos = a.pos[b], first = W == 1 ? 0 : warp;
    const float *w = a.ws + ((size_t)b * a.H + h) * a.nsplit * (Dh + 2);
    float v[4][8];
    auto load = [&](int k0, int n) {  // four parts' accumulators, one in W from k0 on
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int k = k0 + u * W;
                v[u][e] = k < n && lane + 32 * e < Dh ? w[(size_t)k * (Dh + 2) + lane + 32 * e] : 0.0f;
            }
    };
    // Few heads: beside the slots' maxima and sums, before those tell what is in them
    // (700 positions of 12 heads 8.0 -> 7.7 us); for many heads that reads too much.
    if (W > 1) load(first, a.nsplit);
    // offsets and sums of all slots (at most 64); slots past the last part hold anything
    float m[2], l[2];
    int n = a.nsplit;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int k = lane + 32 * i;
        m[i] = k < a.nsplit ? w[(size_t)k * (Dh + 2) + Dh] : 0.0f;
        l[i] = k < a.nsplit ? w[(size_t)k * (Dh + 2) + Dh + 1] : 0.0f;
    }
    if (pos < 0 || pos >= a.S || __shfl_sync(0xffffffffu, l[0], 0) == 0.0f) return;
#pragma unroll
    for (int i = 1; i >= 0; i--) {
        const unsigned last = __ballot_sync(0xffffffffu, __float_as_uint(l[i]) >> 31);
        if (last) n = min(n, 32 * i + __ffs(last));
    }
    float M = fmaxf(lane < n ? m[0] : -INFINITY, lane + 32 < n ? m[1] : -INFINITY);
    M = warp_max(M);
    float f[2];
#pragma unroll
    for (int i = 0; i < 2; i++) f[i] = lane + 32 * i < n ? ex2(m[i] - M) : 0.0f;
    const float L = warp_sum((lane < n ? fabsf(l[0]) * f[0] : 0.0f) + (lane + 32 < n ? fabsf(l[1]) * f[1] : 0.0f));
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int k0 = first; k0 < n; k0 += 4 * W) {
        if (W == 1 || k0 > first) load(k0, n);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int k = k0 + u * W;
            const float fk = __shfl_sync(0xffffffffu, (k & 32) ? f[1] : f[0], k & 31);
            if (k < n)
#pragma unroll
                for (int e = 0; e < 8; e++) acc[e] = fmaf(v[u][e], fk, acc[e]);
        }
    }
    float *out = a.out + (size_t)b * a.ldo + (size_t)h * Dh;
    if constexpr (W == 1) {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (lane + 32 * e < Dh) out[lane + 32 * e] = acc[e] / L;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (lane + 32 * e < Dh) sh[warp][lane + 32 * e] = acc[e];
        __syncthreads();
        for (int d = threadIdx.x; d < Dh; d += 128) out[d] = (sh[0][d] + sh[1][d] + sh[2][d] + sh[3][d]) / L;
    }
}

template <int NB, bool FEW> int launch(const Q4Args &g, int max_units, cudaStream_t s) {
    const int GH = g.a.H / g.a.Hkv < 8 ? g.a.H / g.a.Hkv : 8;
    const size_t smem = (size_t)Q4_WARPS * Q4<NB>::WARP_BYTES + (size_t)Q4_WARPS * GH * Q4<NB>::SLOT * sizeof(float);
    // the most that any G takes: threads that call with different ones set the same value
    constexpr int MOST = Q4_WARPS * Q4<NB>::WARP_BYTES + Q4_WARPS * (FEW ? 4 : 8) * Q4<NB>::SLOT * (int)sizeof(float);
    LMC_CUDA_TRY(cudaFuncSetAttribute((k_attn_q4<NB, FEW>), cudaFuncAttributeMaxDynamicSharedMemorySize, MOST));
    const int most = lmc_sm_count() * (smem + 2048 <= 114 * 1024 ? 2 : 1), want = max_units / g.rmin;
    LMC_LAUNCH("attention (4-bit rows)", (k_attn_q4<NB, FEW>), want < 1 ? 1 : want < most ? want : most, 32 * Q4_WARPS, smem, s, g);
    return LMC_OK;
}

}  // namespace

static int q4_launch(const AttnArgs *args, int batch, size_t ws_bytes, int lose_j, int lose_tile, cudaStream_t s) {
    Q4Args g;
    g.a = *args;
    g.lose_j = lose_j;
    g.lose_tile = lose_tile;
    AttnArgs &a = g.a;
    if (a.S > 1 << 30) return lmc_set_error(LMC_ERR_UNSUPPORTED, "attention: 4-bit rows take contexts of at most 2^30 positions (%d)", a.S);
    // one part per head and workspace slot: the most slots that fit, up to the plan's
    int CH;
    lmc_attn_plan(a.S, batch * a.H, 1, &CH, &a.nsplit);
    const size_t slot = (size_t)batch * a.H * (a.Dh + 2) * sizeof(float);
    if ((size_t)a.nsplit * slot > ws_bytes) a.nsplit = (int)(ws_bytes / slot);
    if (a.nsplit < 2 || !a.ws) a.nsplit = 1;
    const int G = a.H / a.Hkv, T = q4_tile(a.Dh / 32), NT = (a.S - 1) / T + 1;
    g.G = G;
    g.HG = (G + 7) / 8;
    g.batch = batch;
    g.items_only = a.nsplit == 1;
    // an item of NT tiles then lies in at most (NT - 2) / rmin + 2 <= nsplit CTAs;
    // and a CTA has at least an item of one tile (GPT-2, 700 positions, with 1, 3, 6
    // units a CTA: 8.5, 7.7, 9.3 us; 8 kv heads, 4000 positions: 13.5, 10.8, 11.1)
    g.rmin = g.items_only ? 1 : NT < 2 ? Q4_ITEM + 1 : std::max((NT - 2) / (a.nsplit - 1) + 1, Q4_ITEM + 1);
    g.vec = (((uintptr_t)a.q | (uintptr_t)a.k_new | (uintptr_t)a.v_new | (uintptr_t)a.out) & 15) == 0 && a.ldq % 4 == 0 &&
            a.ldkv % 4 == 0 && a.ldo % 4 == 0;
    g.page_bytes = (long long)kv_q4_row_bytes(a.Dh) << a.page_shift;
    g.bulk = a.pages || a.S % 4 == 0;
    g.run = a.pages && (1 << a.page_shift) < T ? 1 << a.page_shift : T;
    const long long units = (long long)batch * a.Hkv * g.HG * (g.items_only ? 1 : NT + Q4_ITEM);
    if (units > 0x7fffffffLL) return lmc_set_error(LMC_ERR_UNSUPPORTED, "attention: batch %d x context %d is too large", batch, a.S);
    int (*const fn[8][2])(const Q4Args &, int, cudaStream_t) = {
        {launch<1, false>, launch<1, true>}, {launch<2, false>, launch<2, true>}, {launch<3, false>, launch<3, true>}, {launch<4, false>, launch<4, true>},
        {launch<5, false>, launch<5, true>}, {launch<6, false>, launch<6, true>}, {launch<7, false>, launch<7, true>}, {launch<8, false>, launch<8, true>}};
    const int rc = fn[a.Dh / 32 - 1][G <= 4](g, (int)units, s);
    if (rc != LMC_OK || a.nsplit == 1) return rc;
    const size_t heads = (size_t)batch * a.H;
    if (heads <= 1024) LMC_LAUNCH("attention combine (4-bit rows)", k_q4_combine<4>, heads, 128, 0, s, a, batch);
    else LMC_LAUNCH("attention combine (4-bit rows)", k_q4_combine<1>, lmc_cdiv(heads, 4), 128, 0, s, a, batch);
    return LMC_OK;
}

extern "C" int lmc_attention_q4_launch(const AttnArgs *args, int batch, size_t ws_bytes, cudaStream_t s) {
    return q4_launch(args, batch, ws_bytes, -1, -1, s);
}

extern "C" int lmc_attn_q4_set_wait_limit(long long ns) {
    const long long v = ns > 0 ? ns : 1000000000ll;
    LMC_CUDA_TRY(cudaMemcpyToSymbol(g_attn_q4_wait_ns, &v, sizeof v));
    return LMC_OK;
}

// Failure-path self-test: a wait for bulk copies that nobody issued runs out,
// is recorded, and the kernel returns.
__global__ void k_attn_q4_wait_selftest(int *gave_up) {
    __shared__ __align__(8) uint64_t sh_bar;
    if (threadIdx.x) return;
    const uint32_t bar = (uint32_t)__cvta_generic_to_shared(&sh_bar);
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *gave_up = bar_wait_long(bar, 0u) ? 0 : 1;
}
extern "C" int lmc_attn_q4_wait_selftest(int *d_flag, cudaStream_t s) {
    k_attn_q4_wait_selftest<<<1, 32, 0, s>>>(d_flag);
    LMC_LAUNCH_CHECK("wait self-test");
    return LMC_OK;
}

// Failure-path self-test: attention over rows of zeros where the copies of one
// tile of kv head 1 never land, the workspace full of an earlier call's finite
// numbers.  Head 1 has to be NaN wherever that tile is one of its own, and no
// other output may be wrong (NaN, where the same warp has it behind the lost one, or 0).
extern "C" int lmc_attn_q4_lost_selftest(cudaStream_t s) {
    constexpr int Hkv = 2, Dh = 64, MOST = 400;
    // sequences, positions, query heads per kv head, lost tile: an item of one warp, of one CTA, of several
    // CTAs, items one after the other in a warp's share, rows of several workspaces' length
    static const int cases[][4] = {{2, 40, 1, 0}, {1, 128, 4, 1}, {1, 128, 8, 0}, {1, 4096, 1, 20}, {3, 4000, 8, 61}, {MOST, 200, 1, 2}};
    float *out = nullptr;
    uint8_t *cache = nullptr;
    int rc = LMC_OK;
    for (const auto &c : cases) {
        const int B = c[0], S = (c[1] + 3) & ~3, H = Hkv * c[2];
        const size_t rows = (size_t)B * Hkv * S * kv_q4_row_bytes(Dh), ws = lmc_attention_workspace_bytes(B, H, Dh, S);
        const size_t q = (size_t)B * H * Dh, kv = (size_t)B * Hkv * Dh;
        std::vector<float> got(q);
        std::vector<int> pos(B, c[1] - 1);
        AttnArgs a = {};
        cudaError_t e = cudaMalloc((void **)&cache, 2 * rows);
        if (e == cudaSuccess) e = cudaMalloc((void **)&out, (2 * q + kv) * sizeof(float) + (size_t)B * sizeof(int) + ws);
        float *const dq = out + q, *const dkv = dq + q;
        int *const dpos = reinterpret_cast<int *>(dkv + kv);
        if (e == cudaSuccess) e = cudaMemsetAsync(cache, 0, 2 * rows, s);
        if (e == cudaSuccess) e = cudaMemsetAsync(out, 0, (2 * q + kv) * sizeof(float), s);
        if (e == cudaSuccess) e = cudaMemcpyAsync(dpos, pos.data(), (size_t)B * sizeof(int), cudaMemcpyHostToDevice, s);
        if (e == cudaSuccess) e = cudaMemsetAsync(dpos + B, 0x3f, ws, s);
        if (e == cudaSuccess) {
            a.out = out;
            a.q = dq;
            a.k_new = a.v_new = dkv;
            a.k_cache = cache;
            a.v_cache = cache + rows;
            a.pos = dpos;
            a.H = H;
            a.Hkv = Hkv;
            a.Dh = Dh;
            a.S = S;
            a.ldo = a.ldq = H * Dh;
            a.ldkv = Hkv * Dh;
            a.append = 1;
            a.ws = reinterpret_cast<float *>(dpos + B);
            rc = q4_launch(&a, B, ws, 1, c[3], s);
            e = cudaMemcpyAsync(got.data(), out, q * sizeof(float), cudaMemcpyDeviceToHost, s);
            if (e == cudaSuccess) e = cudaStreamSynchronize(s);
        }
        cudaFree(cache);
        cudaFree(out);
        cache = nullptr;
        out = nullptr;
        if (rc != LMC_OK) return rc;
        if (e != cudaSuccess) return lmc_set_error(LMC_ERR_CUDA, "wait self-test: %s", cudaGetErrorString(e));
        for (size_t i = 0; i < q; i++) {
            const bool mine = (int)(i / Dh % H) / c[2] == 1;
            if (mine ? got[i] == got[i] : got[i] != 0.0f && got[i] == got[i])
                return lmc_set_error(LMC_ERR_CUDA, "wait self-test: %d sequences of %d positions: output %zu is %g", B, c[1], i, got[i]);
        }
    }
    return LMC_OK;
}

extern "C" int lmc_attn_q4_status(void) {
    int v = 0;
    LMC_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_attn_q4_err, sizeof(int)));
    if (!v) return LMC_OK;
    const int left = v & 2 ? v & ~2 : 0;  // one error a call: what is not reported now stays for the next
    LMC_CUDA_TRY(cudaMemcpyToSymbol(g_attn_q4_err, &left, sizeof(int)));
    if (v & 2) return lmc_set_error(LMC_ERR_TIMEOUT, "4-bit attention: a bounded wait ran out (bulk copy not completed)");
    return lmc_set_error(LMC_ERR_INVALID, "paged attention: a page id outside the pool (page 0 read instead)");
}
