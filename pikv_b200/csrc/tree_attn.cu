// Attention for a tree of drafted tokens over the paged cache, and the acceptance of one path of it.
//
// Node i of a stream is the cache row at position ctx + i.  Its query sees the ctx rows before the tree and the nodes its
// mask row names: out = sum_t w_t V_t, w = softmax(q . K_t / sqrt(128)) over the seen rows t.
#include "stream_list.cuh"
#include "tc_common.cuh"

#include <type_traits>
#include <utility>

namespace pikv {

struct TreeDev {
    CacheDev c;
    const __nv_bfloat16* q;              // [B][N][n_q][128]
    __nv_bfloat16* out;
    float* lse;                          // [B][N][n_q] or null
    int B, N, n_q, G;
    const int* seq_ids;
    const int* ctx_len;
    const int* nodes;                    // or null
    const uint8_t* mask;                 // [N][N], or [B][N][N]
    int mask_stride;                     // bytes from stream to stream
};

// rows in front of the tree, and drafted rows, of stream i (both 0 for an id outside the cache)
__device__ __forceinline__ int tree_lengths(const TreeDev& d, int i, int& row, int& nodes) {
    row = stream_row(d.c, d.seq_ids, i);
    nodes = row < 0 ? 0 : d.nodes ? max(0, min(__ldg(d.nodes + i), d.N)) : d.N;
    const int most = d.c.max_pages * PIKV_PAGE_TOKENS;
    const int ctx = row < 0 ? 0 : max(0, min(__ldg(d.ctx_len + i), most));
    if (nodes > most - ctx) {                                   // the tree does not fit behind its context (whose end may be next to 2^31)
        nodes = most - ctx;
        if (d.c.status) atomicOr(d.c.status, PIKV_ST_BAD_INDEX);
    }
    return ctx;
}

// ---- attention --------------------------------------------------------------------------------------------------
// The nodes of a stream times the query heads of one KV head are the rows of one product: S = Q K^T for 128 rows and 64 keys
// at a time, O += P V, both by tcgen05 with the accumulators in tensor memory.  The keys of all (stream, head, 128 rows)
// units form one list of tiles that a persistent grid cuts into equal runs, two CTAs per SM (or one of two halves, which have 128
// rows each of one head and share the converted tiles, so that these are made once: H = 2); a unit that one CTA holds
// whole is finished there, the pieces of others go to the workspace and a second kernel joins them.
//
// A half's warps (the second half has no copies to make and no scales to prepare):
//   0-3  softmax: thread = row.  S comes out of tensor memory, the weights go back into it as the A operand of the second
//        product; a row's maximum, denominator and the rescaling of its O live in its thread
//   4-5, 6-7  two pages (one where there are two halves) of every tile each: codes of K, of V, to f16, into the swizzled layout that both products read
//   8    issues the MMAs: Q K^T of tile n + 1 before P V of tile n, so that the products of one tile run while the softmax
//        of another does
//   9, 10  bulk copies of pages into two rings, K three tiles ahead, V two (one warp for both is late: 130 cycles a copy)
//   11   the rows' scales in the forms that the converting warps and the softmax use
// The query enters exactly: bf16 times a power of two per row that brings its largest entry to 2^14 is f16 down to 2^-38 of
// that entry.  Keys and values enter as f16 of code * scale, in units of a power of two per tile (2^(e + 9), 2^e above the tile's
// largest scale): one rounding, 2^-11 of the entry, the size of the weights' own (decode_attention keeps the codes of K exact), and
// 2^-25 of a unit where the entry is below f16's normal range; in return the softmax neither loads nor multiplies by the scales
// (shared-memory reads of the scales by every row were the busiest pipe of the kernel that applied them to exact integer products:
// 16 x 16384 x 32 nodes, 248 -> 221 us).
//   logit = 2^(e_k + 9) / sqrt(128) q . K16
//   O     = sum w V16,  w = f16(2^(logit - R + e_v + 9))
// Where a row's scale lies more than 2^8 (4 bit: 2^4) below the tile's largest, every row has an e of its own, and the softmax applies
// it to scores and weights: what a row holds, seen or not, takes no more than 2^-13 of another's largest entry from it.  (The few tiles
// of a prompt that have such rows, at padding and at its first tokens, take six times as long: one in each of 16 x 16384's, 182 -> 948 us.
// The rest paid 2 us for it, and 2 of 75 over the 4-bit cache, where the scales' warp first pushed its neighbours' loops out of the
// instruction cache.)
// A 4-bit code has its zero point taken off first, exactly where that is a whole number below 2048 (with the zero points' parts
// as products of their own in the softmax, it had to reload registers as well: 24 ragged streams to 6001, 103 -> 78 us, now 77).
// R is a row's reference: 2^TR_HEAD below the largest logit (log2 domain) plus e_v + 9 of the tile it was seen in, so that the weights sit
// at the top of f16's range whatever the size of V; it moves only when a tile exceeds it by 2^TR_SLACK.  The denominator is
// the fp32 sum of 2^(logit - R).  A row of V that is not finite enters as zeros and makes the result of the rows that see it
// not a number; one that a row does not see does not reach it.
//
// 16 streams x 16384 rows x 8 heads, 32 nodes x 4 query heads, int8: 213 us with the merge = 2.6 TB/s and 0.65 PFLOP/s in long
// runs under the power cap (226 on another GPU), 182 us in a burst (the bytes alone take 85 us, the products 82); 8 x 32768,
// 64 nodes: 350 and 303.  Bound by power and by the latency between the warps: the SM clock is at 1.6-1.75 GHz, and leaving out the conversion,
// either product, the copies or the weights shortens it by 20, 9 and 5, 6 and 8 %, none by what it costs alone.
constexpr int TR_THREADS = 384;          // of a half: three warpgroups
constexpr int TR_K = 4, TR_V = 6, TR_MMA = 8, TR_COPY = 9, TR_SCALES = 11;      // first warps of each kind
constexpr int TR_ROWS = 128;             // rows of a unit
constexpr int TR_KEYS = 64;              // keys of a tile
constexpr int TR_PAGES = TR_KEYS / PIKV_PAGE_TOKENS;
constexpr float TR_HEAD = 7.f, TR_SLACK = 15.f;       // log2 of the largest weight where a reference is set, and where it is left
template <int BITS> constexpr int TR_SPAN = BITS == 8 ? 8 : 4;      // binary orders that the scales of a tile with one unit may span
constexpr uint32_t TR_ODD_V = 1, TR_OWN_V = 2, TR_OWN_K = 1u << 31;        // a row of V is not finite; the rows of K, of V have exponents of their own
constexpr unsigned TR_WAIT_LIMIT = 1u << 24;
constexpr uint32_t TR_COL_O = 0, TR_COL_S = 128, TR_COLS = 256;      // of a half: S of even and odd tiles, the weights in its first columns

constexpr int TR_TILE = 2 * TR_KEYS * 128;                                     // bytes of a tile of f16: [2 halves of the channels][64 keys][128 bytes]
constexpr int TR_K_AHEAD = 3, TR_V_AHEAD = 2;                                   // tiles whose copies are on their way
constexpr int TR_SETS = 8;                                                      // tiles whose scales are kept as the warps want them

// shared memory behind a 1024-byte boundary, of a CTA of H halves
template <int BITS, int H> struct TRSmem {
    static constexpr int FACTOR = BITS == 8 ? 2 : 8;                            // bytes of a row's factors
    static constexpr int PAGE = 256 * BITS, META = BITS == 8 ? 32 : 96;        // codes of a page of one head; its scales (and zero points)
    static constexpr int QTILE = 2 * TR_ROWS * 128;
    static constexpr int Q = 0, K = Q + H * QTILE, V = K + H * TR_TILE,        // [H] each
                         KRING = V + H * TR_TILE,                              // [ahead][page of the tile] codes of K
                         VRING = KRING + TR_K_AHEAD * TR_PAGES * PAGE,
                         KMETA = VRING + TR_V_AHEAD * TR_PAGES * PAGE,         // [ahead][page] scales, zero points of K, of V
                         VMETA = KMETA + TR_K_AHEAD * TR_PAGES * META,
                         FACT = VMETA + TR_V_AHEAD * TR_PAGES * META,          // [sets][2][64] factors of the rows of K, of V
                         VEXP = FACT + TR_SETS * 2 * TR_KEYS * FACTOR,         // [sets] 2^(e_k + 9), with the sign TR_OWN_K, e_v + 9, 2^-(e_v + 9) as floats, TR_ODD_V | TR_OWN_V
                         ODD = VEXP + TR_SETS * 16,                            // [sets][2] even and odd rows of V that are not finite, a bit each
                         EXPS = ODD + TR_SETS * 8,                             // [sets][2][64] exponents of the rows of K, of V that have their own
                         BARS = EXPS + TR_SETS * 2 * TR_KEYS, NBARS = 4 + 7 * H + 2 * TR_SETS + 2 * (TR_K_AHEAD + TR_V_AHEAD),
                         PRE = BARS + NBARS * 8, MISC = PRE + (PIKV_STREAMS_PER_LAUNCH + 1) * 4, END = MISC + 16;
    static constexpr int BYTES = END + 1024;
};
__device__ __forceinline__ uint32_t tr_set(int n) { return (uint32_t)n % TR_SETS; }
__device__ __forceinline__ uint32_t tr_set_phase(int n) { return (uint32_t)n / TR_SETS & 1u; }

// what hardly ever happens goes behind the loops: a jump over it costs the instruction cache
#define TR_RARE(x) __builtin_expect(!!(x), 0)

struct TreeParts {
    float* o;                            // [C][2][halves][rows][128]
    float2* ml;                          // [C][2][halves][rows] reference and denominator
    int* plan;                           // [0] tiles per CTA, [1 ..] prefix of the streams' tiles
    int rows;                            // rows of a slot
    int halves;                          // of a CTA
};

// (the rows are below 2^31, not so with the rounding up)
__device__ __forceinline__ int tree_tiles(int ctx, int nodes) { return (int)(((uint32_t)(ctx + nodes) + TR_KEYS - 1) / TR_KEYS); }
// units of a head: TR_ROWS rows for each half of a CTA
__device__ __forceinline__ int tree_row_tiles(int nodes, int G, int halves) { return (nodes * G + halves * TR_ROWS - 1) / (halves * TR_ROWS); }

// a place in the list of tiles: stream b, unit (head, H x 128 rows) of it, tile of the unit
template <int H> struct TreeCursor {
    int b, head, row_tile, tile;
    int tiles, row_tiles;                // of the stream
    int row, ctx, nodes;
    __device__ __forceinline__ void load(const TreeDev& d) {
        ctx = tree_lengths(d, b, row, nodes);
        tiles = tree_tiles(ctx, nodes);
        row_tiles = tree_row_tiles(nodes, d.G, H);
    }
    __device__ __forceinline__ void start(const TreeDev& d, const int* pre, int f) {
        b = stream_of(pre, d.B, f);
        load(d);
        const int unit = (f - pre[b]) / tiles;
        tile = (f - pre[b]) % tiles;
        head = unit / row_tiles;
        row_tile = unit % row_tiles;
    }
    __device__ __forceinline__ void next(const TreeDev& d, const int* pre, int f) {      // f: the place after this one
        if (!TR_RARE(++tile >= tiles)) return;
        tile = 0;
        if (++row_tile < row_tiles) return;
        row_tile = 0;
        if (++head < d.c.n_kv) return;
        head = 0;
        do ++b; while (pre[b + 1] <= f);
        load(d);
    }
    __device__ __forceinline__ int end() const { return ctx + nodes; }
    __device__ __forceinline__ int pages() const { return min(TR_PAGES, (end() + PIKV_PAGE_TOKENS - 1) / PIKV_PAGE_TOKENS - tile * TR_PAGES); }
};

__device__ __forceinline__ bool tr_wait(uint32_t bar, uint32_t parity) {
#pragma unroll 1
    for (unsigned i = 0; i < TR_WAIT_LIMIT; ++i) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
    }
    return false;
}
// A from tensor memory (f16, two to a column), B from shared memory
__device__ __forceinline__ void tr_mma_ta(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accum) : "memory");
}
__device__ __forceinline__ void tr_tmem_ld32(uint32_t taddr, float* v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// loads done; ties their 32 registers to the wait, so that nothing of theirs is used before it
__device__ __forceinline__ void tr_tmem_ld_wait(float* v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]),
                   "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]),
                   "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
                 :: "memory");
}
__device__ __forceinline__ void tr_tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                 "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tr_tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tr_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tr_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tr_fence_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float tr_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two fp32 operations per instruction
__device__ __forceinline__ float2 tr_fma2(float2 a, float2 b, float2 c) {
    float2 e;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 z, x, y, z;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(e.x), "=f"(e.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return e;
}
__device__ __forceinline__ float2 tr_add2(float2 a, float2 b) {
    float2 c;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(c.x), "=f"(c.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return c;
}
__device__ __forceinline__ uint32_t tr_pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// exponent of a scale, for the reference; what is not finite has no say in it.  2^(e + 9) and 2^-(e + 9) are finite up to TR_MOST
constexpr int TR_MOST = 117;
constexpr float TR_HUGE = 1.661534995e35f;              // 2^117: a row whose scale is not below it counts as not finite
__device__ __forceinline__ int tr_exponent(uint32_t bits) {
    const int e = (int)((bits >> 23) & 0xffu);
    return e == 255 ? -100 : min(TR_MOST, max(-100, e - 126));
}
// position of a channel inside its group of eight in the 4-bit tiles: nibbles leave a word as (0, 4), (1, 5), (2, 6), (3, 7)
template <int BITS> __device__ __forceinline__ constexpr int tr_channel(int at) { return BITS == 8 ? at : (at & ~7) | ((at & 7) >> 1) | ((at & 1) << 2); }

// A page of codes on its way into the 16 rows of a [2 halves][64 keys][128 bytes] tile of f16, in the registers of a warp.
// Lane l holds, of rows base and base + 8 (base = 2 (l >> 3), with 5 added exclusively for l & 4), the logical chunks l & 3 and
// (l & 3) + 4 of 16 codes: eight neighbouring lanes then touch eight different 16-byte columns both where the cache's swizzle has
// put the codes and where the products' swizzle wants them.
__device__ __forceinline__ int tr_row(int lane) { return (2 * (lane >> 3)) ^ (lane & 4 ? 5 : 0); }
// byte of a lane's first piece in a page
template <int BITS>
__device__ __forceinline__ int tr_place(int lane) {
    const int r = tr_row(lane);
    return BITS == 8 ? r * 128 + 16 * ((lane & 3) ^ (r & 7)) : r * 64 + 8 * ((lane & 3) ^ (r & 4));
}
// two phases of which both are wanted: their polls overlap
__device__ __forceinline__ bool tr_wait2(uint32_t bar0, uint32_t parity0, uint32_t bar1, uint32_t parity1) {
#pragma unroll 1
    for (unsigned i = 0; i < TR_WAIT_LIMIT; ++i) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p, q;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tmbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
                     "and.pred p, p, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(bar0), "r"(parity0), "r"(bar1), "r"(parity1) : "memory");
        if (ok) return true;
    }
    return false;
}
__device__ __forceinline__ void tr_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// What makes an entry of a row's codes: 8 bit a n 2^-24 + b, 4 bit a (n 2^-24 + c) + b (b 0 where c and a are exact, otherwise what
// their roundings left out)
template <int BITS> struct TRFactor {
    __half2 a, b, c;
    __device__ __forceinline__ void load(const unsigned char* f) {
        if constexpr (BITS == 8) {
            a = __half2half2(*reinterpret_cast<const __half*>(f));
            b = __hmul2(a, __float2half2_rn(-128.f / 16777216.f));
        } else {
            const uint2 x = *reinterpret_cast<const uint2*>(f);
            const __half2 ac = *reinterpret_cast<const __half2*>(&x.x), b0 = *reinterpret_cast<const __half2*>(&x.y);
            a = __low2half2(ac);
            c = __high2half2(ac);
            b = b0;
        }
    }
};
template <int BITS> struct TRPage {
    uint32_t w[4][BITS / 2];
    __device__ __forceinline__ void load(const unsigned char* page, int at) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // the chunk of the upper half: 4 chunks on, exclusively
            const unsigned char* p = page + ((i & 1) ? at ^ (8 * BITS) : at) + (i >> 1) * 8 * (16 * BITS);
            if constexpr (BITS == 8) {
                const uint4 x = *reinterpret_cast<const uint4*>(p);
                w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2*>(p);
                w[i][0] = x.x; w[i][1] = x.y;
            }
        }
    }
    // A byte or nibble n in the low bits of an f16 is n 2^-24, exactly (a subnormal).  With a = scale 2^(15 - e), the fused
    // a n 2^-24 + b is (n - 128) scale 2^(-9 - e), rounded once, b the offset's part.
    static __device__ __forceinline__ uint32_t fma2(uint32_t x, __half2 a, __half2 b) {
        const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&x), a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    // f0, f1: factors of rows base and base + 8
    __device__ __forceinline__ void store(unsigned char* tile, int page, int lane, const TRFactor<BITS>& f0, const TRFactor<BITS>& f1) const {
        const int r = tr_row(lane), c = lane & 3;
        unsigned char* row = tile + (page * PIKV_PAGE_TOKENS + r) * 128;
        const int d0 = 16 * ((2 * c) ^ (r & 7)), d1 = 16 * ((2 * c + 1) ^ (r & 7));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            unsigned char* to = row + (i & 1) * TR_KEYS * 128 + (i >> 1) * 8 * 128;
            const TRFactor<BITS>& f = i >> 1 ? f1 : f0;
            if constexpr (BITS == 8) {
                uint32_t x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = w[i][k] ^ 0x80808080u;             // code + 128
                auto pair = [&](int k, uint32_t sel) { return fma2(__byte_perm(x[k], 0u, sel), f.a, f.b); };
                *reinterpret_cast<uint4*>(to + d0) = make_uint4(pair(0, 0x4140), pair(0, 0x4342), pair(1, 0x4140), pair(1, 0x4342));
                *reinterpret_cast<uint4*>(to + d1) = make_uint4(pair(2, 0x4140), pair(2, 0x4342), pair(3, 0x4140), pair(3, 0x4342));
            } else {
                auto low = [&](uint32_t x) {
                    x &= 0x000f000fu;
                    const __half2 t = __hadd2(*reinterpret_cast<const __half2*>(&x), f.c);
                    return fma2(*reinterpret_cast<const uint32_t*>(&t), f.a, f.b);
                };
                auto high = [&](uint32_t x) {                                          // n 2^-20
                    return fma2(fma2(x & 0x00f000f0u, __float2half2_rn(0.0625f), f.c), f.a, f.b);
                };
                const uint32_t x = w[i][0], y = w[i][1];
                *reinterpret_cast<uint4*>(to + d0) = make_uint4(low(x), high(x), low(x >> 8), high(x >> 8));
                *reinterpret_cast<uint4*>(to + d1) = make_uint4(low(y), high(y), low(y >> 8), high(y >> 8));
            }
        }
    }
};

// the largest of 32 products of a row; what `open` has no bit for becomes -infinity
template <bool EDGE>
__device__ __forceinline__ float tr_scores(float (&x)[32], uint32_t open) {
    float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
        if (EDGE) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!((open >> (j + i)) & 1u)) x[j + i] = -INFINITY;
        }
        m0 = fmaxf(m0, fmaxf(x[j], x[j + 1]));
        m1 = fmaxf(m1, fmaxf(x[j + 2], x[j + 3]));
    }
    return fmaxf(m0, m1);
}
// 32 scores to weights f16(2^(score mul + off)), and their sum
__device__ __forceinline__ void tr_weights(const float (&x)[32], uint32_t (&wgt)[16], float mul, float off, float& total) {
    float2 s0 = make_float2(0.f, 0.f), s1 = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
        float2 a = tr_fma2(make_float2(x[j], x[j + 1]), make_float2(mul, mul), make_float2(off, off));
        float2 c = tr_fma2(make_float2(x[j + 2], x[j + 3]), make_float2(mul, mul), make_float2(off, off));
        a = make_float2(tr_ex2(a.x), tr_ex2(a.y));
        c = make_float2(tr_ex2(c.x), tr_ex2(c.y));
        s0 = tr_add2(s0, a);
        s1 = tr_add2(s1, c);
        wgt[j / 2] = tr_pack(a.x, a.y);
        wgt[j / 2 + 1] = tr_pack(c.x, c.y);
    }
    s0 = tr_add2(s0, s1);
    total += s0.x + s0.y;
}

// A tile whose rows have exponents of their own, sixteen scores of a row of S at a time: hardly ever met, and small so that the loops
// around it keep their registers
struct TROwn {
    const unsigned char* at;              // bytes e of the 64 rows of K, of V
    uint32_t all_k, all_v;                // or the tile's e four times
    int ek;                               // the largest of K
    bool k, v;
    __device__ __forceinline__ TROwn(const unsigned char* exps, uint32_t flags, float of_k, float of_v) {
        at = exps;
        k = flags & TR_OWN_K;
        v = flags & TR_OWN_V;
        ek = (int)((__float_as_uint(of_k) >> 23) & 0xffu) - 136;
        all_k = (uint32_t)(ek & 0xff) * 0x01010101u;
        all_v = (uint32_t)(((int)of_v - 9) & 0xff) * 0x01010101u;
    }
    static __device__ __forceinline__ int byte(uint32_t w, int i) { return (int)(w << (24 - 8 * i)) >> 24; }
    __device__ __forceinline__ uint32_t of_k(int j) const { return k ? *reinterpret_cast<const uint32_t*>(at + j) : all_k; }
    __device__ __forceinline__ uint32_t of_v(int j) const { return v ? *reinterpret_cast<const uint32_t*>(at + TR_KEYS + j) : all_v; }
    // returns the largest of the rows seen
    __device__ __forceinline__ float scores(uint32_t taddr, uint64_t seen, float mul) const {
        float top = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < TR_KEYS; c += 16) {
            float x[16];
            uint32_t r[16];
            lr_tmem_ld16(taddr + c, x);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int up = max(byte(of_k(c + (j & ~3)), j & 3) - ek, -126);
                const float t = fmaf(x[j] * exp2_int(up), mul, (float)(byte(of_v(c + (j & ~3)), j & 3) + 9));
                if ((seen >> (c + j)) & 1u) top = fmaxf(top, t);
                r[j] = __float_as_uint(t);
            }
            tr_tmem_st16(taddr + c, r);
        }
        tr_tmem_st_wait();
        return top;
    }
    // sum of 2^(logit + off) over the rows seen
    __device__ __forceinline__ float total(uint32_t taddr, uint64_t seen, float off) const {
        float sum = 0.f;
#pragma unroll 1
        for (int c = 0; c < TR_KEYS; c += 16) {
            float x[16];
            lr_tmem_ld16(taddr + c, x);
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if ((seen >> (c + j)) & 1u) sum += tr_ex2(x[j] + off - (float)(byte(of_v(c + (j & ~3)), j & 3) + 9));
        }
        return sum;
    }
};

template <int BITS, int H>
__global__ void __launch_bounds__(H * TR_THREADS, 2 / H) tree_attn_kernel(TreeDev d, TreeParts parts) {
    using SM = TRSmem<BITS, H>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (lr_smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = lr_smem_u32(smem);
    const int half = H == 2 && threadIdx.x >= TR_THREADS, tid = threadIdx.x - half * TR_THREADS, lane = tid & 31, warp = tid >> 5;
    int* pre = reinterpret_cast<int*>(smem + SM::PRE);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + SM::MISC);
    const uint32_t bars = sbase + SM::BARS;
    const uint32_t k_full = bars, v_full = k_full + 16, k_side = v_full + 16, v_side = k_side + 8 * TR_SETS, kr_full = v_side + 8 * TR_SETS,
                   kr_empty = kr_full + 8 * TR_K_AHEAD, vr_full = kr_empty + 8 * TR_K_AHEAD, vr_empty = vr_full + 8 * TR_V_AHEAD,
                   own = vr_empty + 8 * TR_V_AHEAD;                      // the others are a half's own
    const uint32_t q_full = own + 56 * half, s_full = q_full + 8, p_full = s_full + 16, pv_done = p_full + 16;
    if (tid == 0) {
        lr_mbar_init(q_full, 4);
        for (int i = 0; i < 2; ++i) lr_mbar_init(s_full + 8 * i, 1), lr_mbar_init(p_full + 8 * i, 4), lr_mbar_init(pv_done + 8 * i, 1);
        if (half == 0) {
            for (int i = 0; i < H; ++i) lr_mbar_init(k_full + 8 * i, 2 * H), lr_mbar_init(v_full + 8 * i, 2 * H);
            for (int i = 0; i < TR_SETS; ++i) lr_mbar_init(k_side + 8 * i, 1), lr_mbar_init(v_side + 8 * i, 1);
            for (int i = 0; i < TR_K_AHEAD; ++i) lr_mbar_init(kr_full + 8 * i, 1), lr_mbar_init(kr_empty + 8 * i, 2 * H + 1);
            for (int i = 0; i < TR_V_AHEAD; ++i) lr_mbar_init(vr_full + 8 * i, 1), lr_mbar_init(vr_empty + 8 * i, 2 * H + 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Tensor memory is taken when the kernels before have given theirs back, and nothing behind this one starts until it is taken:
    // a kernel that waits for its predecessors with tensor memory in hand could keep it from one of them
    dependency_wait();
    if (half == 0 && warp == TR_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(lr_smem_u32(tmem_slot)), "r"(H * TR_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const int total = stream_prefix<H * TR_THREADS>(d.B, pre, [&](int i) {
        int row, nodes;
        const int ctx = tree_lengths(d, i, row, nodes);
        if (row < 0 && blockIdx.x == 0 && d.c.status) atomicOr(d.c.status, PIKV_ST_BAD_SEQ);
        return nodes > 0 ? d.c.n_kv * tree_row_tiles(nodes, d.G, H) * tree_tiles(ctx, nodes) : 0;
    });
    const int per = (max(total, 1) - 1) / (int)gridDim.x + 1;
    if (blockIdx.x == 0) {
        if (tid == 0) parts.plan[0] = per;
        for (int i = tid; i <= d.B; i += TR_THREADS) parts.plan[1 + i] = pre[i];       // (by either half)
    }
    tr_fence_before();
    __syncthreads();
    tr_fence_after();
    dependency_release();
    const uint32_t tmem = *tmem_slot + half * TR_COLS;
    const int f0 = (int)min((long long)total, (long long)blockIdx.x * per), f1 = (int)min((long long)total, (long long)f0 + per);
    bool failed = false;
    if (f0 < f1) {
        // registers go where the scores are: 120 + 72 + 48 of the 3 x 80 a thread that the block was launched with
        TreeCursor<H> cur;
        if (warp >= TR_MMA) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
            if (warp == TR_MMA) {
            cur.start(d, pre, f0);
            // ---- the products ----
            const uint32_t idesc_qk = (1u << 4) | ((uint32_t)(TR_KEYS >> 3) << 17) | ((uint32_t)(TR_ROWS >> 4) << 24);
            const uint32_t idesc_pv = (1u << 4) | (1u << 16) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(TR_ROWS >> 4) << 24);
            const uint32_t q_lo = lr_desc_lo(sbase + SM::Q + half * SM::QTILE), k_lo = lr_desc_lo(sbase + SM::K);
            // V: [64 channels][keys], channels contiguous: 64-channel halves 8192 bytes apart (leading), 8-key groups 1024 (stride)
            const uint32_t v_lo = (((sbase + SM::V) & 0x3FFFFu) >> 4) | ((uint32_t)(TR_KEYS * 128 >> 4) << 16);
            const int count = f1 - f0;
            uint32_t seg = 0;
            bool first_before = true;                                // whether tile n - 1 opened its unit here
            auto pv = [&](int m, bool first) {
                const uint32_t b = m & 1, ph = (uint32_t)(m >> 1) & 1u;
                const uint32_t buf = (uint32_t)m % H;
                if (TR_RARE(!tr_wait2(v_full + 8 * buf, (uint32_t)m / H & 1u, p_full + 8 * b, ph))) return false;
                tr_fence_after();
                if (lr_elect()) {
#pragma unroll
                    for (int k = 0; k < TR_KEYS / 16; ++k)
                        tr_mma_ta(tmem + TR_COL_O, tmem + TR_COL_S + TR_KEYS * b + 8 * k, lr_desc(v_lo + buf * (TR_TILE >> 4) + 128 * k), idesc_pv, !first || k ? 1u : 0u);
                    lr_commit(pv_done + 8 * b);
                }
                __syncwarp();
                return true;
            };
            for (int n = 0; n < count; ++n) {
                const bool first = n == 0 || cur.tile == 0;
                const uint32_t b = n & 1;
                if (TR_RARE(first)) {
                    // the next unit's Q takes the place of this one's after its last product
                    if (n > 0 && !pv(n - 1, first_before)) { failed = true; break; }
                    if (TR_RARE(!tr_wait(q_full, seg & 1u))) { failed = true; break; }
                    ++seg;
                }
                // (S of tile n lies where the weights of tile n - 2 were: their product has been issued before this one)
                const uint32_t buf = (uint32_t)n % H;
                if (TR_RARE(!tr_wait(k_full + 8 * buf, (uint32_t)n / H & 1u))) { failed = true; break; }
                tr_fence_after();
                if (lr_elect()) {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        lr_mma(tmem + TR_COL_S + TR_KEYS * b, lr_desc(q_lo + (k >> 2) * (TR_ROWS * 128 >> 4) + 2 * (k & 3)),
                               lr_desc(k_lo + buf * (TR_TILE >> 4) + (k >> 2) * (TR_KEYS * 128 >> 4) + 2 * (k & 3)), idesc_qk, k ? 1u : 0u);
                    lr_commit(s_full + 8 * b);
                }
                __syncwarp();
                if (!first && TR_RARE(!pv(n - 1, first_before))) { failed = true; break; }
                first_before = first;
                if (n + 1 < count) cur.next(d, pre, f0 + n + 1);
            }
            if (!failed) failed = !pv(count - 1, first_before);
            // nothing of this CTA's is in flight when its tensor memory goes back
            if (!failed) failed = !tr_wait(pv_done + 8 * ((count - 1) & 1), (uint32_t)((count - 1) >> 1) & 1u);
            } else if (half == 1) {                                  // the copies and the scales are the first half's
            } else if (warp < TR_SCALES) {
                // ---- pages into the rings, with their scales: a warp for K, one for V; lane = page of the tile ----
                cur.start(d, pre, f0);
                const bool of_v = warp > TR_COPY;
                const int count = f1 - f0, i = lane & 3, ahead = of_v ? TR_V_AHEAD : TR_K_AHEAD;
                const uint8_t* codes = of_v ? d.c.v_codes : d.c.k_codes;
                const uint16_t* scale = of_v ? d.c.v_scale : d.c.k_scale;
                const float* zp = of_v ? d.c.v_zp : d.c.k_zp;
                const uint32_t ring = sbase + (of_v ? SM::VRING : SM::KRING), metas = sbase + (of_v ? SM::VMETA : SM::KMETA);
                const uint32_t full = of_v ? vr_full : kr_full, empty = of_v ? vr_empty : kr_empty;
                int ids = -1, ids_row = -2, ids_at = 0;              // page numbers of this stream, 32 at a time: eight tiles
                int s = 0;
                uint32_t ph = 1;
                for (int n = 0; n < count; ++n) {
                    const int p = cur.tile * TR_PAGES, np = cur.pages();
                    if (TR_RARE(cur.row != ids_row || p < ids_at || p >= ids_at + 32)) {
                        ids_row = cur.row;
                        ids_at = p;
                        ids = p + lane < d.c.max_pages ? __ldg(d.c.page_table + (size_t)cur.row * d.c.max_pages + p + lane) : -1;
                    }
                    int page = __shfl_sync(0xffffffffu, ids, (p + i - ids_at) & 31);
                    if (TR_RARE(i < np && (page < 0 || page >= d.c.num_pages))) {
                        if (lane < 4 && d.c.status) atomicOr(d.c.status, PIKV_ST_BAD_PAGE);
                        page = 0;
                    }
                    const uint32_t unit = (uint32_t)page * (uint32_t)d.c.n_kv + (uint32_t)cur.head;
                    if (TR_RARE(!tr_wait(empty + 8 * s, ph))) { failed = true; break; }
                    const uint32_t bar = full + 8 * s;
                    if (lane == 0) lr_mbar_expect_tx(bar, (uint32_t)np * (SM::PAGE + SM::META));
                    __syncwarp();
                    if (lane < np) {
                        const uint32_t dst = metas + (s * TR_PAGES + i) * SM::META;
                        tr_bulk(ring + (s * TR_PAGES + i) * SM::PAGE, codes + (size_t)unit * SM::PAGE, SM::PAGE, bar);
                        tr_bulk(dst, scale + (size_t)unit * 16, 32, bar);
                        if (BITS == 4) tr_bulk(dst + 32, zp + (size_t)unit * 16, 64, bar);
                    }
                    if (++s == ahead) s = 0, ph ^= 1u;
                    if (n + 1 < count) cur.next(d, pre, f0 + n + 1);
                }
                // copies that a warp which gave up no longer waits for land before this CTA's shared memory goes to another
                for (int k = 0; k < ahead; ++k) (void)tr_wait(full + 8 * k, k < s ? ph ^ 1u : ph);
            } else {
                // ---- scales as the other warps want them, K of tile n + 1 before V of tile n; lane = rows 2 lane and 2 lane + 1 ----
                // The sets need no wait of their own: when K of tile n + 1 takes that of tile n - 7, V of tile n - 1 has come, into a
                // place that V of tile n - 3 left, behind the second product of tile n - 3 - H
                cur.start(d, pre, f0);
                const int count = f1 - f0;
                // One piece of code for K and V: what this warp runs through pushes the loops of its neighbours out of the instruction cache
                int ks = 0, vs = 0, left = 0, v_left = 0;
                uint32_t kph = 0, vph = 0;
#pragma unroll 1
                for (int i = 0; i <= 2 * count; ++i) {                // K of 0; K of 1, V of 0; K of 2, V of 1; ..; V of count - 1
                    const bool of_v = i > 0 && !(i & 1);
                    const int n = of_v ? i / 2 - 1 : (i + 1) / 2, s = of_v ? vs : ks;
                    if (!of_v) {
                        v_left = left;
                        if (n == count) continue;
                        left = cur.end() - cur.tile * TR_KEYS;
                    }
                    if (TR_RARE(!tr_wait((of_v ? vr_full : kr_full) + 8 * s, of_v ? vph : kph))) { failed = true; break; }
                    const int rows = of_v ? v_left : left;            // (none behind the end)
                    const unsigned char* own = smem + (of_v ? SM::VMETA : SM::KMETA) + (s * TR_PAGES + (lane >> 3)) * SM::META;
                    uint32_t two = 2 * lane < rows ? *reinterpret_cast<const uint32_t*>(own + (lane & 7) * 4) : 0u;
                    if (2 * lane + 1 == rows) two &= 0xffffu;
                    const float s0 = __uint_as_float(two << 16), s1 = __uint_as_float(two & 0xffff0000u);
                    float z0 = 0.f, z1 = 0.f, top0 = s0, top1 = s1;               // top: a sixteenth of a row's largest entry, 4 bit
                    if (BITS == 4) {
                        if (2 * lane < rows) {
                            const float2 zp = *reinterpret_cast<const float2*>(own + 32 + (lane & 7) * 8);
                            z0 = zp.x;
                            if (2 * lane + 1 < rows) z1 = zp.y;
                        }
                        if (!(fabsf(z0) <= 16.f)) top0 = s0 * (fabsf(z0) * 0.0625f);
                        if (!(fabsf(z1) <= 16.f)) top1 = s1 * (fabsf(z1) * 0.0625f);
                    }
                    const int e0 = tr_exponent(__float_as_uint(top0)), e1 = tr_exponent(__float_as_uint(top1));
                    const int e = __reduce_max_sync(0xffffffffu, max(e0, e1));
                    // a K that is not finite makes its logit so; a V enters as zeros
                    const bool odd0 = of_v && !(fabsf(top0) < TR_HUGE), odd1 = of_v && !(fabsf(top1) < TR_HUGE);
                    // a row too far below the largest; what is 0 or below 2^-100, -100 here, has no say
                    const bool far = __any_sync(0xffffffffu, min((uint32_t)(e0 + 99), (uint32_t)(e1 + 99)) < (uint32_t)max(e + 99 - TR_SPAN<BITS>, 0));
                    const bool odd = __any_sync(0xffffffffu, odd0 || odd1);
                    const int set = 2 * tr_set(n) + of_v;
                    if (TR_RARE(far)) *reinterpret_cast<uint16_t*>(smem + SM::EXPS + set * TR_KEYS + 2 * lane) = (uint16_t)((e0 & 0xff) | (e1 & 0xff) << 8);
                    const float a0 = odd0 ? 0.f : s0 * exp2_int(15 - (far ? e0 : e)), a1 = odd1 ? 0.f : s1 * exp2_int(15 - (far ? e1 : e));
                    unsigned char* fact = smem + SM::FACT + (set * TR_KEYS + 2 * lane) * SM::FACTOR;
                    if constexpr (BITS == 8) {
                        *reinterpret_cast<uint32_t*>(fact) = tr_pack(a0, a1);
                    } else {
                        constexpr float UNIT = 1.f / 16777216.f;
                        auto factors = [&](float a, float z) {
                            const uint32_t ac = tr_pack(a, -z * UNIT);
                            const float2 got = __half22float2(*reinterpret_cast<const __half2*>(&ac));
                            const float b = -z * UNIT * a - got.x * got.y;
                            return make_uint2(ac, tr_pack(b, b));
                        };
                        const uint2 f0 = factors(a0, odd0 ? 0.f : z0), f1 = factors(a1, odd1 ? 0.f : z1);
                        *reinterpret_cast<uint4*>(fact) = make_uint4(f0.x, f0.y, f1.x, f1.y);
                    }
                    if (TR_RARE(odd)) {
                        const uint32_t m0 = __ballot_sync(0xffffffffu, odd0), m1 = __ballot_sync(0xffffffffu, odd1);
                        if (lane == 0) *reinterpret_cast<uint2*>(smem + SM::ODD + tr_set(n) * 8) = make_uint2(m0, m1);
                    }
                    if (lane == 0) {
                        float* of = reinterpret_cast<float*>(smem + SM::VEXP + tr_set(n) * 16);
                        if (of_v) {
                            of[1] = (float)(e + 9);
                            *reinterpret_cast<float2*>(of + 2) = make_float2(exp2_int(-9 - e), __uint_as_float((odd ? TR_ODD_V : 0u) | (far ? TR_OWN_V : 0u)));
                        } else {
                            of[0] = __uint_as_float((uint32_t)(e + 136) << 23 | (far ? TR_OWN_K : 0u));
                        }
                    }
                    tr_fence_smem();                                 // before the ring's place is given back
                    __syncwarp();
                    if (lane == 0) {
                        lr_mbar_arrive((of_v ? v_side : k_side) + 8 * tr_set(n));
                        lr_mbar_arrive((of_v ? vr_empty : kr_empty) + 8 * s);
                    }
                    if (of_v) {
                        if (++vs == TR_V_AHEAD) vs = 0, vph ^= 1u;
                    } else {
                        if (++ks == TR_K_AHEAD) ks = 0, kph ^= 1u;
                        if (n + 1 < count) cur.next(d, pre, f0 + n + 1);
                    }
                }
            }
        } else if (warp >= TR_K) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
            // ---- codes to f16: warp w of the two or four of K, of V, takes pages 2 w and 2 w + 1, or page w, of every tile ----
            constexpr int MINE = TR_PAGES / (2 * H);
            const bool of_v = warp >= TR_V;
            const int page = (((warp - TR_K) & 1) + 2 * half) * MINE, count = f1 - f0, ahead = of_v ? TR_V_AHEAD : TR_K_AHEAD;
            const int at = tr_place<BITS>(lane);
            const unsigned char* ring = smem + (of_v ? SM::VRING : SM::KRING) + page * SM::PAGE;
            const unsigned char* facts = smem + SM::FACT + (of_v * TR_KEYS + page * PIKV_PAGE_TOKENS + tr_row(lane)) * SM::FACTOR;
            unsigned char* tile = smem + (of_v ? SM::V : SM::K);
            const uint32_t full = of_v ? vr_full : kr_full, empty = of_v ? vr_empty : kr_empty, read = own + (of_v ? 40 : 8), ready = of_v ? v_full : k_full,
                           sides = of_v ? v_side : k_side;
            int s = 0;
            uint32_t ph = 0;
            for (int n = 0; n < count; ++n) {
                if (TR_RARE(!tr_wait2(full + 8 * s, ph, sides + 8 * tr_set(n), tr_set_phase(n)))) { failed = true; break; }
                TRPage<BITS> x[MINE];
                TRFactor<BITS> f[MINE][2];
                const unsigned char* fact = facts + tr_set(n) * 2 * TR_KEYS * SM::FACTOR;
#pragma unroll
                for (int i = 0; i < MINE; ++i) {
                    x[i].load(ring + (s * TR_PAGES + i) * SM::PAGE, at);           // (what a page behind the end left there is finite)
                    f[i][0].load(fact + 16 * i * SM::FACTOR);
                    f[i][1].load(fact + (16 * i + 8) * SM::FACTOR);
                }
                // the products of the tile before in this buffer have read it
                const int m = n - H;
                if (m >= 0) {
                    const uint32_t bar = read + 8 * (m & 1), was = (uint32_t)(m >> 1) & 1u;
                    if (TR_RARE(H == 2 ? !tr_wait2(bar, was, bar + 56, was) : !tr_wait(bar, was))) { failed = true; break; }
                }
                unsigned char* to = tile + (uint32_t)n % H * TR_TILE;
#pragma unroll
                for (int i = 0; i < MINE; ++i) x[i].store(to, page + i, lane, f[i][0], f[i][1]);
                // also before the ring's place is given back: without the fence, a bulk copy may land under these warps' own reads
                tr_fence_smem();
                __syncwarp();
                if (lane == 0) {
                    lr_mbar_arrive(ready + 8 * ((uint32_t)n % H));
                    lr_mbar_arrive(empty + 8 * s);
                }
                if (++s == ahead) s = 0, ph ^= 1u;
            }
        } else {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 120;");
            cur.start(d, pre, f0);
            // ---- softmax: thread = row ----
            const uint32_t lanes = (uint32_t)(warp * 32) << 16;
            float qmul = 0.f, ref = -INFINITY, den = 0.f;
            float odd_v = 0.f;                                        // not a number once the row has seen a V that is not finite
            uint64_t tree = 0;
            int node = 0;
            bool live = false, warp_live = false;
            size_t out_row = 0;
            // One tile: scores out, weights in.  EDGE: some of its positions lie behind the context, or its rows have flags; a tile with
            // flags is left to that form
            enum { DONE, FAILED, FLAGGED };
            auto step = [&](auto edge_c, int n, int tile, bool first) {
                constexpr bool EDGE = decltype(edge_c)::value;
                if (TR_RARE(!tr_wait2(s_full + 8 * (n & 1), (uint32_t)(n >> 1) & 1u, v_side + 8 * tr_set(n), tr_set_phase(n)))) return FAILED;
                if (!warp_live) {
                    if (lane == 0) lr_mbar_arrive(p_full + 8 * (n & 1));
                    return DONE;
                }
                tr_fence_after();
                const uint32_t scores = tmem + lanes + TR_COL_S + TR_KEYS * (n & 1);
                float x0[32], x1[32];
                tr_tmem_ld32(scores, x0);
                tr_tmem_ld32(scores + 32, x1);
                float4 of = *reinterpret_cast<const float4*>(smem + SM::VEXP + tr_set(n) * 16);
                float mul = qmul * fabsf(of.x);
                if (mul == 0.f) mul = 1.17549435e-38f;                   // (masked scores are -infinity: times 0 they would not be a number)
                uint64_t seen = ~0ull;
                if (EDGE) {
                    // the positions behind the context show only where the mask opens them
                    const int sh = cur.ctx - tile * TR_KEYS;             // the tree's first bit
                    seen = sh >= 0 ? (sh < 64 ? tree << sh : 0ull) | (sh < 64 ? (1ull << sh) - 1 : ~0ull) : (sh > -64 ? tree >> -sh : 0ull);
                }
                // the reference moves to `want` where `move`
                auto refer = [&](float want, bool move) {
                    const float next = move ? want - TR_HEAD : ref;
                    const float fac = move ? tr_ex2(ref - next) : 1.f;     // 0 from -inf
                    ref = next;
                    den *= fac;
                    if (!first) {
                        if (TR_RARE(!tr_wait(pv_done + 8 * ((n - 1) & 1), (uint32_t)((n - 1) >> 1) & 1u))) return false;
                        tr_fence_after();
#pragma unroll 1
                        for (int c = 0; c < 128; c += 16) {             // few registers: the scores are in the others
                            float o[16];
                            lr_tmem_ld16(tmem + lanes + TR_COL_O + c, o);
                            uint32_t r[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(o[i] * fac);
                            tr_tmem_st16(tmem + lanes + TR_COL_O + c, r);
                        }
                        tr_tmem_st_wait();
                    }
                    return true;
                };
                const uint32_t flags = __float_as_uint(of.w) | (__float_as_uint(of.x) & TR_OWN_K);
                if (TR_RARE(flags != 0u)) {
                    tr_tmem_ld_wait(x0);                                 // (the loads above land before their registers are taken again)
                    tr_tmem_ld_wait(x1);
                    if constexpr (!EDGE) return FLAGGED;
                    if (flags & TR_ODD_V) {
                        const uint2 odd = *reinterpret_cast<const uint2*>(smem + SM::ODD + tr_set(n) * 8);
                        for (int j = 0; j < TR_KEYS; ++j)
                            if (((j & 1 ? odd.y : odd.x) >> (j >> 1)) & (uint32_t)(seen >> j) & 1u) odd_v = __uint_as_float(0x7fffffffu);
                    }
                    if (flags & (TR_OWN_K | TR_OWN_V)) {
                        // scores in the reference's units, where they lie: logit + e_v + 9 of each row; the denominator's part as well
                        const TROwn own_e(smem + SM::EXPS + tr_set(n) * 2 * TR_KEYS, flags, of.x, of.y);
                        const float want = own_e.scores(scores, seen, mul);
                        const bool move = want > ref + TR_SLACK;
                        if (__any_sync(0xffffffffu, move) && !refer(want, move)) return FAILED;
                        den += own_e.total(scores, seen, ref == -INFINITY ? 0.f : -ref);
                        tr_tmem_ld32(scores, x0);
                        tr_tmem_ld32(scores + 32, x1);
                        mul = 1.f;
                        of.y = of.z = 0.f;
                    }
                }
                tr_tmem_ld_wait(x0);
                tr_tmem_ld_wait(x1);
                const float mx = fmaxf(tr_scores<EDGE>(x0, (uint32_t)seen), tr_scores<EDGE>(x1, (uint32_t)(seen >> 32)));
                // does the reference hold?  (-inf while nothing has been seen)
                const float want = mx * mul + of.y;
                const bool move = mx > -INFINITY && want > ref + TR_SLACK;
                if (TR_RARE(__any_sync(0xffffffffu, move)) && !refer(want, move)) return FAILED;
                const float off = of.y - (ref == -INFINITY ? 0.f : ref);
                float total = 0.f;
                // the weights take the place of the scores that they come from, two to a column
                uint32_t wgt[16];
                tr_weights(x0, wgt, mul, off, total);
                tr_tmem_st16(scores, wgt);
                tr_weights(x1, wgt, mul, off, total);
                tr_tmem_st16(scores + 16, wgt);
                den += total * of.z;
                tr_tmem_st_wait();
                tr_fence_before();
                __syncwarp();
                if (lane == 0) lr_mbar_arrive(p_full + 8 * (n & 1));
                return DONE;
            };
            for (int n = 0, f = f0; f < f1;) {
                // ---- a unit, or the part of it that this CTA has: tiles t0 .. t1 - 1 ----
                const int t0 = cur.tile, t1 = min(cur.tiles, t0 + f1 - f), edge = max(t0, min(t1, cur.ctx / TR_KEYS));
                // ---- this row's query ----
                const int row = (cur.row_tile * H + half) * TR_ROWS + tid, h = cur.head;
                node = row / d.G;
                live = node < cur.nodes;
                warp_live = __any_sync(0xffffffffu, live);
                ref = -INFINITY;
                den = odd_v = 0.f;
                if (warp_live) {
                    out_row = ((size_t)cur.b * d.N + (live ? node : 0)) * d.n_q + (size_t)h * d.G + row % d.G;
                    const uint4* src = reinterpret_cast<const uint4*>(d.q + out_row * 128);
                    uint4 q4[16];                                     // (one trip: shared memory leaves next to no L1)
#pragma unroll
                    for (int i = 0; i < 16; ++i) q4[i] = live ? __ldg(src + i) : make_uint4(0u, 0u, 0u, 0u);
                    // largest entry by its bits, two to a word; what is not finite is above all that is
                    uint32_t top2 = 0;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint32_t a = __vmaxu2(q4[i].x & 0x7fff7fffu, q4[i].y & 0x7fff7fffu), b = __vmaxu2(q4[i].z & 0x7fff7fffu, q4[i].w & 0x7fff7fffu);
                        top2 = __vmaxu2(top2, __vmaxu2(a, b));
                    }
                    const uint32_t top = max(top2 & 0xffffu, top2 >> 16) << 16;
                    const float amax = __uint_as_float(top), odd = top >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : 0.f;
                    const int sh = amax > 0.f && amax < INFINITY ? min(126, 14 - ((int)(__float_as_uint(amax) >> 23) - 127)) : 0;
                    const float up = exp2_int(max(sh, -126));
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float x[8];
                        bf16x2_to_f32(q4[i].x, x[0], x[1]);
                        bf16x2_to_f32(q4[i].y, x[2], x[3]);
                        bf16x2_to_f32(q4[i].z, x[4], x[5]);
                        bf16x2_to_f32(q4[i].w, x[6], x[7]);
#pragma unroll
                        for (int k = 0; k < 8; ++k) x[k] *= up;
                        uint4 y;
                        y.x = tr_pack(x[tr_channel<BITS>(0)], x[tr_channel<BITS>(1)]);
                        y.y = tr_pack(x[tr_channel<BITS>(2)], x[tr_channel<BITS>(3)]);
                        y.z = tr_pack(x[tr_channel<BITS>(4)], x[tr_channel<BITS>(5)]);
                        y.w = tr_pack(x[tr_channel<BITS>(6)], x[tr_channel<BITS>(7)]);
                        *reinterpret_cast<uint4*>(smem + SM::Q + half * SM::QTILE + (i >> 3) * TR_ROWS * 128 + tid * 128 + 16 * ((i & 7) ^ (tid & 7))) = y;
                    }
                    qmul = exp2_int(-max(sh, -126)) * (0.08838834764831845f * 1.4426950408889634f) + odd;
                    tr_fence_smem();
                }
                __syncwarp();
                if (lane == 0) lr_mbar_arrive(q_full);
                if (warp_live) {
                    // what a node sees of the tree, a bit per node: the warp reads the mask rows of its nodes together
                    const int node0 = __shfl_sync(0xffffffffu, node, 0), node1 = min(__shfl_sync(0xffffffffu, node, 31), cur.nodes - 1);
                    const uint8_t* masks = d.mask + (size_t)cur.b * d.mask_stride;
                    tree = 0;
#pragma unroll 4
                    for (int i = node0; i <= node1; ++i) {
                        const bool lo = lane < cur.nodes && __ldg(masks + (size_t)i * d.N + lane) != 0;
                        const bool hi = lane + 32 < cur.nodes && __ldg(masks + (size_t)i * d.N + lane + 32) != 0;
                        const uint32_t m0 = __ballot_sync(0xffffffffu, lo), m1 = __ballot_sync(0xffffffffu, hi);
                        if (node == i) tree = (uint64_t)m1 << 32 | m0;
                    }
                }
                for (int t = t0; t < t1; ++t, ++n) {
                    int did = DONE;
                    for (; t < edge; ++t, ++n)
                        if ((did = step(std::false_type{}, n, t, t == t0)) != DONE) break;
                    if (did == FAILED || (t < t1 && step(std::true_type{}, n, t, t == t0) == FAILED)) { failed = true; break; }
                    if (t >= t1) break;
                }
                if (failed) break;
                // ---- this CTA's share of the unit is done ----
                if (TR_RARE(!tr_wait(pv_done + 8 * ((n - 1) & 1), (uint32_t)((n - 1) >> 1) & 1u))) { failed = true; break; }
                if (warp_live) {
                    tr_fence_after();
                    const bool begun = t0 == 0;                          // here, and not by the CTA before
                    const bool whole = begun && t1 == cur.tiles;
                    const float inv = den == 0.f ? 0.f : 1.f / den;
                    const size_t slot = (size_t)((2 * blockIdx.x + (begun ? 1 : 0)) * H + half) * parts.rows + tid;
#pragma unroll 1
                    for (int c = 0; c < 128; c += 32) {
                        float o[32];
                        tr_tmem_ld32(tmem + lanes + TR_COL_O + c, o);
                        tr_tmem_ld_wait(o);
                        if (BITS == 4) {
                            float t[32];
#pragma unroll
                            for (int i = 0; i < 32; ++i) t[tr_channel<BITS>(i)] = o[i];
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = t[i];
                        }
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] += odd_v;
                        if (live && whole) {
                            uint4* to = reinterpret_cast<uint4*>(d.out + out_row * 128 + c);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                uint32_t r[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    const __nv_bfloat162 h2 = __floats2bfloat162_rn(den == 0.f ? 0.f : o[8 * i + 2 * k] * inv, den == 0.f ? 0.f : o[8 * i + 2 * k + 1] * inv);
                                    r[k] = *reinterpret_cast<const uint32_t*>(&h2);
                                }
                                to[i] = make_uint4(r[0], r[1], r[2], r[3]);
                            }
                        } else if (live) {
                            float4* to = reinterpret_cast<float4*>(parts.o + slot * 128 + c);
#pragma unroll
                            for (int i = 0; i < 8; ++i) to[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        }
                        __syncwarp();
                    }
                    if (live && whole && d.lse) d.lse[out_row] = den == 0.f ? -INFINITY : ref * 0.6931471805599453f + logf(den);
                    if (live && !whole) parts.ml[slot] = make_float2(ref, den);
                    tr_fence_before();
                }
                f += t1 - t0;
                cur.tile = t1 - 1;
                if (f < f1) cur.next(d, pre, f);
            }
        }
        if (failed && lane == 0 && d.c.status) atomicOr(d.c.status, PIKV_ST_WAIT_TIMEOUT);
    }
    tr_fence_before();
    __syncthreads();
    if (half == 0 && warp == TR_MMA) {
        tr_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(H * TR_COLS) : "memory");
    }
}

constexpr int TM_THREADS = 128;
constexpr int TM_RESIDENT = 5;                                          // blocks of tree_merge_kernel<8> on an SM

// Joins the pieces of units that were cut, and answers for the rows that no unit has.  One warp per (stream, node, query head),
// lane = 4 channels: O = sum_i O_i 2^(R_i - R), the denominator likewise.
// Bound by the trips to the pieces (in L2): BATCH of them are on their way at once, and where BATCH is 8 the next ones while they are
// joined.  That takes 96 registers and is right while all rows' warps are resident with them (few rows have many pieces each: 1
// stream x 8 nodes 6.7 us against 8.5 with 4); more rows have fewer pieces and want the warps (47 registers, 16 streams x 32 nodes:
// 11.8 us against 16.0, and 14.8 with the next batch ahead).
template <int BATCH>
__global__ void __launch_bounds__(TM_THREADS) tree_merge_kernel(TreeDev d, TreeParts parts) {
    dependency_release();
    dependency_wait();
    const int lane = threadIdx.x & 31;
    const uint32_t at = blockIdx.x * (TM_THREADS / 32) + (threadIdx.x >> 5), rows = (uint32_t)d.N * (uint32_t)d.n_q;
    if (at >= (uint32_t)d.B * rows) return;
    const int b = (int)(at / rows), node = (int)(at % rows) / d.n_q, qh = (int)(at % rows) % d.n_q;
    const int per = parts.plan[0], pre0 = parts.plan[1 + b];
    int row, nodes;
    const int ctx = tree_lengths(d, b, row, nodes);
    uint2* out = reinterpret_cast<uint2*>(d.out + (size_t)at * 128) + lane;
    if (node >= nodes) {
        *out = make_uint2(0u, 0u);
        if (lane == 0 && d.lse) d.lse[at] = -INFINITY;
        return;
    }
    const int H = parts.halves, tiles = tree_tiles(ctx, nodes), row_tiles = tree_row_tiles(nodes, d.G, H);
    const int r = node * d.G + qh % d.G;
    const int f0 = pre0 + ((qh / d.G) * row_tiles + r / TR_ROWS / H) * tiles, f1 = f0 + tiles;
    const int c0 = f0 / per, c1 = (f1 - 1) / per;
    if (c0 == c1) return;                                               // whole: written by its CTA
    // piece i lies in the first slot of CTA c0 + i, the first piece in the second
    const size_t slot0 = (size_t)(2 * c0 * H + r / TR_ROWS % H) * parts.rows + r % TR_ROWS;
    const float4* o0 = reinterpret_cast<const float4*>(parts.o + slot0 * 128) + lane;
    const float2* ml0 = parts.ml + slot0;
    const int pieces = c1 - c0 + 1, stride = 2 * H * parts.rows;
    float M = -INFINITY, den = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    // pieces in batches
    constexpr bool AHEAD = BATCH == 8;
    float4 o[BATCH], next[AHEAD ? BATCH : 1];
    float2 ml, next_ml;
    auto fetch = [&](int g, float4 (&to)[BATCH], float2& to_ml) {
        to_ml = g + lane < pieces && lane < BATCH ? ml0[(size_t)(g + lane) * stride + (g + lane ? 0 : H * parts.rows)] : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int u = 0; u < BATCH; ++u)
            if (g + u < pieces) to[u] = o0[((size_t)(g + u) * stride + (g + u ? 0 : H * parts.rows)) * 32];
    };
    fetch(0, o, ml);
    for (int g = 0; g < pieces; g += BATCH) {
        if constexpr (AHEAD) {
            if (g + BATCH < pieces) fetch(g + BATCH, next, next_ml);
        }
        const float top = fmaxf(M, warp_max(ml.x)), base = top == -INFINITY ? 0.f : top;
        const float keep = M == -INFINITY ? (den == 0.f ? 0.f : 1.f) : exp2f(M - base);
        // a piece that saw nothing has no weight; one that is not a number keeps it
        const float w_l = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2f(ml.x - base);
        acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
        den *= keep;
        M = top;
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            if (g + u >= pieces) break;
            const float w = __shfl_sync(0xffffffffu, w_l, u), l = __shfl_sync(0xffffffffu, ml.y, u);
            acc.x += o[u].x * w; acc.y += o[u].y * w; acc.z += o[u].z * w; acc.w += o[u].w * w;
            den += l * w;
        }
        if constexpr (AHEAD) {
#pragma unroll
            for (int u = 0; u < BATCH; ++u) o[u] = next[u];
            ml = next_ml;
        } else if (g + BATCH < pieces) {
            fetch(g + BATCH, o, ml);
        }
    }
    const bool any = den != 0.f;
    const float inv = any ? 1.f / den : 0.f;
    const __nv_bfloat162 lo = __floats2bfloat162_rn(any ? acc.x * inv : 0.f, any ? acc.y * inv : 0.f);
    const __nv_bfloat162 hi = __floats2bfloat162_rn(any ? acc.z * inv : 0.f, any ? acc.w * inv : 0.f);
    *out = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    if (lane == 0 && d.lse) d.lse[at] = any ? (M == -INFINITY ? 0.f : M) * 0.6931471805599453f + logf(den) : -INFINITY;
}

static int tree_slot_rows(int N, int G) { return std::min(TR_ROWS, N * G); }
struct TreeLayout {
    size_t ml, o, total;
};
static TreeLayout tree_layout(int N, int G) {
    const size_t slots = (size_t)2 * sm_count() * 2, rows = tree_slot_rows(N, G);
    TreeLayout l;
    l.ml = ((size_t)(PIKV_STREAMS_PER_LAUNCH + 2) * sizeof(int) + 255) & ~(size_t)255;
    l.o = l.ml + slots * rows * sizeof(float2);
    l.total = l.o + slots * rows * 128 * sizeof(float);
    return l;
}

// ---- acceptance -------------------------------------------------------------------------------------------------
constexpr int TA_THREADS = 256;
constexpr int TA_BATCH = 4;              // rows a group of eight lanes has in flight

struct AcceptDev {
    CacheDev c;
    const int* path;                     // [B][depth]
    const int* path_len;                 // or null
    const int* seq_ids;
    const int* ctx_len;                  // may be `length`
    int B, depth;
    int* length;                         // [num_seqs] or null
    int* new_len;                        // [B]
    const int* all_ids;                  // the whole call's ids, for the search of an earlier one that names the same stream
    int b0;
};

// One CTA per stream, one warp per (head, K or V): eight lanes move a row, one chunk each.  A path ascends, so row i comes
// from position path[i] >= i: what a later row is read from lies behind everything written before it, and a batch of rows is
// read whole before it is written.  The chunk at physical place c of a row with swizzle key w goes to c ^ w ^ w'.
template <int BITS>
__global__ void __launch_bounds__(TA_THREADS) tree_accept_kernel(AcceptDev d) {
    constexpr int ROW = 128 * BITS / 8, CHUNK = ROW / 8, TURN = BITS == 8 ? 7 : 4;
    using Unit = typename std::conditional<BITS == 8, uint4, uint2>::type;
    dependency_release();
    dependency_wait();
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = stream_row(d.c, d.seq_ids, b);
    const int most = d.c.max_pages * PIKV_PAGE_TOKENS;
    const int ctx = row < 0 ? 0 : d.ctx_len[b];
    const int count = d.path_len ? d.path_len[b] : d.depth;
    const int* path = d.path + (size_t)b * d.depth;
    const int* table = d.c.page_table + (size_t)max(row, 0) * d.c.max_pages;
    unsigned wrong = row < 0 ? PIKV_ST_BAD_SEQ : 0u;
    if (d.all_ids)
        for (int i = tid; i < d.b0 + b; i += TA_THREADS)
            if (d.all_ids[i] == row) wrong |= PIKV_ST_BAD_SEQ;
    const bool sized = count >= 0 && count <= d.depth && ctx >= 0 && ctx <= most;
    if (row >= 0 && !sized) wrong |= PIKV_ST_BAD_INDEX;
    if (row >= 0 && sized)
        for (int i = tid; i < count; i += TA_THREADS) {
            const int at = path[i], prev = i ? path[i - 1] : -1;
            if (at <= prev || at >= most - ctx) {
                wrong |= PIKV_ST_BAD_INDEX;
                continue;
            }
            const int ps = table[(ctx + at) / PIKV_PAGE_TOKENS], pd = i < most - ctx ? table[(ctx + i) / PIKV_PAGE_TOKENS] : -1;
            if (ps < 0 || ps >= d.c.num_pages || pd < 0 || pd >= d.c.num_pages) wrong |= PIKV_ST_BAD_PAGE;
        }
    const int seq_bad = __syncthreads_or(wrong & PIKV_ST_BAD_SEQ);
    const int index_bad = __syncthreads_or(wrong & PIKV_ST_BAD_INDEX), page_bad = __syncthreads_or(wrong & PIKV_ST_BAD_PAGE);
    if (seq_bad || index_bad || page_bad) {
        if (tid == 0) {
            if (d.c.status)
                atomicOr(d.c.status, seq_bad ? PIKV_ST_BAD_SEQ : (index_bad ? PIKV_ST_BAD_INDEX : 0u) | (page_bad ? PIKV_ST_BAD_PAGE : 0u));
            d.new_len[b] = seq_bad ? 0 : ctx;
        }
        return;
    }
    const int g = lane >> 3, c = lane & 7;
    for (int unit = warp; unit < 2 * d.c.n_kv; unit += TA_THREADS / 32) {
        const int h = unit >> 1;
        uint8_t* codes = unit & 1 ? d.c.v_codes : d.c.k_codes;
        uint16_t* scale = unit & 1 ? d.c.v_scale : d.c.k_scale;
        float* zp = unit & 1 ? d.c.v_zp : d.c.k_zp;
        for (int i0 = 0; i0 < count; i0 += 4 * TA_BATCH) {
            Unit x[TA_BATCH];
            uint16_t s[TA_BATCH];
            float z[TA_BATCH];
            size_t to[TA_BATCH];
            int place[TA_BATCH];
#pragma unroll
            for (int u = 0; u < TA_BATCH; ++u) {
                const int i = i0 + 4 * u + g;
                place[u] = -1;
                if (i >= count) continue;
                const int from = ctx + path[i], dst = ctx + i;
                const int rs = from % PIKV_PAGE_TOKENS, rd = dst % PIKV_PAGE_TOKENS;
                const size_t src = ((size_t)table[from / PIKV_PAGE_TOKENS] * d.c.n_kv + h) * PIKV_PAGE_TOKENS + rs;
                to[u] = ((size_t)table[dst / PIKV_PAGE_TOKENS] * d.c.n_kv + h) * PIKV_PAGE_TOKENS + rd;
                place[u] = c ^ (rs & TURN) ^ (rd & TURN);
                x[u] = *reinterpret_cast<const Unit*>(codes + src * ROW + c * CHUNK);
                if (c == 0) s[u] = scale[src];
                if (c == 1 && zp) z[u] = zp[src];
            }
            __syncwarp();
#pragma unroll
            for (int u = 0; u < TA_BATCH; ++u) {
                if (place[u] < 0) continue;
                *reinterpret_cast<Unit*>(codes + to[u] * ROW + place[u] * CHUNK) = x[u];
                if (c == 0) scale[to[u]] = s[u];
                if (c == 1 && zp) zp[to[u]] = z[u];
            }
            __syncwarp();
        }
    }
    if (tid == 0) {                       // (every thread read ctx before the barriers above)
        d.new_len[b] = ctx + count;
        if (d.length) d.length[row] = ctx + count;
    }
}

}  // namespace pikv

using namespace pikv;

extern "C" size_t pikv_tree_attn_workspace_bytes(int32_t B, int32_t N, int32_t n_q, int32_t n_kv) {
    if (B <= 0 || N <= 0 || n_q <= 0 || n_kv <= 0 || n_q % n_kv != 0) return 0;
    return tree_layout(N, n_q / n_kv).total;
}

template <int BITS, int H>
static bool tree_launch(int grid, cudaStream_t st, const TreeDev& d, const TreeParts& parts) {
    if (!allow_smem<tree_attn_kernel<BITS, H>>(TRSmem<BITS, H>::BYTES)) return false;
    launch_dependent(tree_attn_kernel<BITS, H>, grid, H * TR_THREADS, TRSmem<BITS, H>::BYTES, st, d, parts);
    return true;
}

extern "C" int pikv_tree_attn(const pikv_paged_cache* c, const pikv_tree_params* p, pikv_stream_t stream) {
    TreeDev d;
    const int rc = cache_dev(c, d.c, "tree_attn", true);
    if (rc != PIKV_OK) return rc;
    PIKV_REQUIRE(p != nullptr && p->q && p->out && p->ctx_len && p->mask && p->workspace, PIKV_EINVAL, "tree_attn: null pointer");
    PIKV_REQUIRE(p->B > 0 && p->N > 0 && p->n_q > 0 && p->n_q % c->n_kv == 0, PIKV_EINVAL, "tree_attn: bad sizes");
    PIKV_REQUIRE(p->seq_ids || p->B <= c->num_seqs, PIKV_EINVAL, "tree_attn: %d streams, the cache has %d", p->B, c->num_seqs);
    PIKV_REQUIRE(p->N <= PIKV_TREE_NODES, PIKV_ELIMIT, "tree_attn: %d nodes per stream (max %d)", p->N, PIKV_TREE_NODES);
    PIKV_REQUIRE(p->n_q / c->n_kv <= 64, PIKV_EUNSUPPORTED, "tree_attn: %d query heads per KV head (max 64)", p->n_q / c->n_kv);
    PIKV_REQUIRE(((reinterpret_cast<uintptr_t>(p->workspace) | reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->out)) & 15) == 0, PIKV_EINVAL,
                 "tree_attn: q, out and workspace must be 16-byte aligned");
    d.N = p->N; d.n_q = p->n_q; d.G = p->n_q / c->n_kv;
    const TreeLayout lay = tree_layout(d.N, d.G);
    PIKV_REQUIRE(p->workspace_bytes >= lay.total, PIKV_EINVAL, "tree_attn: workspace too small (%zu bytes, %zu needed)", p->workspace_bytes, lay.total);
    const int64_t most = (int64_t)std::min(p->B, PIKV_STREAMS_PER_LAUNCH) * c->n_kv * ceil_div(d.N * d.G, TR_ROWS) * ceil_div(c->max_pages, TR_PAGES);
    PIKV_REQUIRE(most < (1ll << 31), PIKV_ELIMIT, "tree_attn: streams * heads * pages must stay below 2^33");
    unsigned char* ws = static_cast<unsigned char*>(p->workspace);
    TreeParts parts;
    parts.plan = reinterpret_cast<int*>(ws);
    parts.ml = reinterpret_cast<float2*>(ws + lay.ml);
    parts.o = reinterpret_cast<float*>(ws + lay.o);
    parts.rows = tree_slot_rows(d.N, d.G);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    d.mask_stride = p->mask_per_stream ? p->N * p->N : 0;
    const size_t rows = (size_t)p->N * p->n_q;
    for (int b0 = 0; b0 < p->B; b0 += PIKV_STREAMS_PER_LAUNCH) {
        d.B = std::min(p->B - b0, PIKV_STREAMS_PER_LAUNCH);
        d.c.page_table = c->page_table + (p->seq_ids ? 0 : (size_t)b0 * c->max_pages);
        d.c.num_seqs = p->seq_ids ? c->num_seqs : c->num_seqs - b0;
        d.seq_ids = p->seq_ids ? p->seq_ids + b0 : nullptr;
        d.ctx_len = p->ctx_len + b0;
        d.nodes = p->nodes ? p->nodes + b0 : nullptr;
        d.mask = p->mask + (size_t)b0 * d.mask_stride;
        d.q = static_cast<const __nv_bfloat16*>(p->q) + b0 * rows * 128;
        d.out = static_cast<__nv_bfloat16*>(p->out) + b0 * rows * 128;
        d.lse = p->lse ? p->lse + b0 * rows : nullptr;
        // Two CTAs per SM, or one whose halves share the tiles of K and V, where at least three quarters of its rows are used: 8 x 32768
        // with 256 rows 348 us against 308, with 208 rows 335 against 299; 8 x 8192 with 416 of 512 rows 106 against 102, with 336 86
        // against 97; 128 rows, a half idle, 187 against 272.  (Streams may have fewer nodes than N: with half as many 190 against 277.)
        const bool wide = 4 * d.N * d.G > 3 * 2 * TR_ROWS * ceil_div(d.N * d.G, 2 * TR_ROWS);
        parts.halves = wide ? 2 : 1;
        const int64_t units = (int64_t)d.B * c->n_kv * ceil_div(d.N * d.G, parts.halves * TR_ROWS);
        const int grid = (int)std::min<int64_t>(sm_count() * 2 / parts.halves, units * ceil_div(c->max_pages, TR_PAGES));
        const bool sent = c->bits == 8 ? (wide ? tree_launch<8, 2>(grid, st, d, parts) : tree_launch<8, 1>(grid, st, d, parts))
                                       : (wide ? tree_launch<4, 2>(grid, st, d, parts) : tree_launch<4, 1>(grid, st, d, parts));
        if (!sent) return check_launch("tree_attn smem attribute");
        const int blocks = (int)((d.B * rows + TM_THREADS / 32 - 1) / (TM_THREADS / 32));
        if (blocks <= sm_count() * TM_RESIDENT) launch_dependent(tree_merge_kernel<8>, blocks, TM_THREADS, 0, st, d, parts);
        else launch_dependent(tree_merge_kernel<4>, blocks, TM_THREADS, 0, st, d, parts);
        count_launch(2);
    }
    return check_launch("tree_attn_kernel");
}

static bool apart(const int32_t* a, int64_t n, const int32_t* b, int64_t m) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return !a || !b || x + (uintptr_t)n * 4 <= y || y + (uintptr_t)m * 4 <= x;
}

extern "C" int pikv_tree_accept(const pikv_paged_cache* c, const int32_t* path, const int32_t* path_len, const int32_t* seq_ids,
                                const int32_t* ctx_len, int32_t B, int32_t depth, int32_t* length, int32_t* new_len, pikv_stream_t stream) {
    AcceptDev d;
    const int rc = cache_dev(c, d.c, "tree_accept", false);
    if (rc != PIKV_OK) return rc;
    PIKV_REQUIRE((path || depth == 0) && ctx_len && new_len, PIKV_EINVAL, "tree_accept: null pointer");
    PIKV_REQUIRE(B > 0 && depth >= 0 && (seq_ids || B <= c->num_seqs), PIKV_EINVAL, "tree_accept: bad sizes");
    PIKV_REQUIRE(!(seq_ids && ctx_len == length), PIKV_EINVAL, "tree_accept: with seq_ids, ctx_len has an entry per stream of the call");
    // a stream's CTA writes its lengths while others still read theirs
    for (const auto& out : {std::make_pair((const int32_t*)length, (int64_t)c->num_seqs), std::make_pair((const int32_t*)new_len, (int64_t)B)}) {
        auto lies_apart = [&](const int32_t* in, int64_t n) { return apart(out.first, out.second, in, n); };
        PIKV_REQUIRE((out.first == ctx_len || lies_apart(ctx_len, B)) && lies_apart(path_len, B) && lies_apart(seq_ids, B) && lies_apart(path, (int64_t)B * depth),
                     PIKV_EINVAL, "tree_accept: length and new_len overlap an input (only ctx_len itself may be either)");
    }
    PIKV_REQUIRE(apart(length, c->num_seqs, new_len, B), PIKV_EINVAL, "tree_accept: length and new_len overlap");
    d.depth = depth;
    d.all_ids = seq_ids;
    for (int b0 = 0; b0 < B; b0 += PIKV_STREAMS_PER_LAUNCH) {
        d.B = std::min(B - b0, PIKV_STREAMS_PER_LAUNCH);
        d.b0 = b0;
        d.c.page_table = c->page_table + (seq_ids ? 0 : (size_t)b0 * c->max_pages);
        d.c.num_seqs = seq_ids ? c->num_seqs : c->num_seqs - b0;
        d.seq_ids = seq_ids ? seq_ids + b0 : nullptr;
        d.path = path + (size_t)b0 * depth;
        d.path_len = path_len ? path_len + b0 : nullptr;
        d.ctx_len = ctx_len + b0;
        d.length = length ? length + (seq_ids ? 0 : b0) : nullptr;
        d.new_len = new_len + b0;
        if (c->bits == 8) launch_dependent(tree_accept_kernel<8>, d.B, TA_THREADS, 0, static_cast<cudaStream_t>(stream), d);
        else launch_dependent(tree_accept_kernel<4>, d.B, TA_THREADS, 0, static_cast<cudaStream_t>(stream), d);
        count_launch(1);
    }
    return check_launch("tree_accept_kernel");
}
