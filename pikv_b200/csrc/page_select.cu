// Sparse decode attention: bounds of every page's keys, the pages that those bounds select for a query, and attention over
// them (decode_attn.cu, with a page list per stream and KV head).
//
// A page is 16 rows.  For channel c let hi_c and lo_c be the largest and smallest key on it: no key of the page gives a
// query q a logit above sum_c max(q_c hi_c, q_c lo_c) = sum_c (max(q_c, 0) hi_c + min(q_c, 0) lo_c).  (Ranking pages by the
// largest and smallest key of every channel is the method of QUEST.)  Bounds are kept as int8 in whole steps of a power of two,
// rounded outwards (256 bytes for the 2 KB of a page's keys), the query is brought to int8 steps too, rounded to the nearest:
// a score is the bound for that rounded query, and ONE product of a page's 256 bytes with 256 bytes of query on the integer tensor
// cores, an exact whole number times exact powers of two: the choice of pages depends neither on the order of a sum nor on the
// type it is held in.  (Of 59 pages of 2048 chosen for a query over topical keys, 99 % are those of the unrounded query, 93 %
// those of unrounded bounds as well.)
#include "stream_list.cuh"
#include "shard_decode.cuh"
#include "tc_common.cuh"

namespace pikv {

// ---- bounds ---------------------------------------------------------------------------------------------------
constexpr int PB_THREADS = 256;
constexpr int PB_CTAS = 4;               // per SM
constexpr int PB_STAGES = 3;             // pages that a warp has on their way or at hand

// a stage of a warp's ring: codes of a page of one head, scales (and zero points), and what the warp needs to know of it
template <int BITS> struct PBGeom {
    static constexpr int CODES = 256 * BITS, COPY = CODES + 32 + (BITS == 4 ? 64 : 0), STAGE = COPY + 16;
    static constexpr int SMEM = (PB_THREADS / 32) * PB_STAGES * (STAGE + 8);
};
constexpr float PB_HUGE = 5.192296858534828e33f;       // 2^112: 2^15 + 128 times a scale below it is finite
constexpr uint32_t PB_HUGE_BITS = 0x7780u;            // the same as bf16

struct BoundsDev {
    CacheDev c;
    uint8_t* codes;                      // [num_pages][n_kv][2][128]
    float* scale;                        // [num_pages][n_kv]
    const int* seq_ids;
    const int* start;
    const int* seq_len;
    int B;
};


__device__ __forceinline__ void pb_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// One warp per (page, head); a lane has CH channels of ROWS rows (8 bit: 4 channels of all sixteen, 4 bit: 8 channels of every
// second row, joined by one exchange), so that a load of the warp is whole rows, wherever the cache's swizzle has put their
// chunks, and next to nothing crosses lanes.  Pages come by bulk copies into a ring of the warp's own (with plain loads a warp
// had nothing on its way while it computed).
// Bound by the integer pipes.  Keys are compared as whole numbers: a scale is m 2^E with m below 2^8, so code m 2^(E - least E of the
// page) fits 32 bits where the exponents span at most 15; one byte-dot-product takes a code out of its word (and the zero point
// off), one multiplication does the rest, and two rows go into a three-operand maximum and minimum.  (As floats, a byte-permute, half
// a fused operation, a minimum and a maximum a key: 88 us for 8 x 32768 rows x 8 heads, now 74 = 4.1 TB/s.)  Pages that this does not fit,
// a stream's unfilled last one among them, take floats: a byte becomes 2^15 + u exactly by one byte-permute (u = code + 128 in
// the second byte of 0x47000000) and a key by (2^15 + u) s - (2^15 + 128) s, whose second factor has 17 bits and is exact.
template <int BITS>
__global__ void __launch_bounds__(PB_THREADS, PB_CTAS) page_bounds_kernel(BoundsDev d) {
    constexpr int ROWS = BITS == 8 ? 16 : 8, CH = BITS == 8 ? 4 : 8;
    __shared__ int pre[PIKV_STREAMS_PER_LAUNCH + 1];
    const int lane = threadIdx.x & 31;
    const int n_kv = d.c.n_kv, max_len = d.c.max_pages * PIKV_PAGE_TOKENS;
    dependency_release();
    dependency_wait();
    auto range = [&](int i, int& first, int& len) {
        const int row = stream_row(d.c, d.seq_ids, i);
        len = row < 0 ? 0 : max(0, min(__ldg(d.seq_len + i), max_len));
        first = d.start ? max(0, __ldg(d.start + i)) / PIKV_PAGE_TOKENS : 0;
        return row;
    };
    const int total = stream_prefix<PB_THREADS>(d.B, pre, [&](int i) {
        int first, len;
        if (range(i, first, len) < 0 && blockIdx.x == 0 && d.c.status) atomicOr(d.c.status, PIKV_ST_BAD_SEQ);
        // nothing is new where start is at or behind the end
        if (d.start && __ldg(d.start + i) >= len) return 0;
        return max(0, (len + PIKV_PAGE_TOKENS - 1) / PIKV_PAGE_TOKENS - first);
    });
    // runs of (page, head) items, heads innermost: they lie side by side in the pool
    const long long items = (long long)total * n_kv;
    const int warps = gridDim.x * (PB_THREADS / 32);
    const int self = (threadIdx.x >> 5) * gridDim.x + blockIdx.x;
    const long long run = (items + warps - 1) / warps, it0 = min(items, self * run);
    int left = (int)(min(items, it0 + run) - it0);
    if (left <= 0) return;
    extern __shared__ __align__(16) unsigned char pb_smem[];
    using GEO = PBGeom<BITS>;
    unsigned char* ring = pb_smem + (threadIdx.x >> 5) * PB_STAGES * GEO::STAGE;
    const uint32_t bar0 = lr_smem_u32(pb_smem + (PB_THREADS / 32) * PB_STAGES * GEO::STAGE) + (threadIdx.x >> 5) * PB_STAGES * 8;
    if (lane == 0) {
        for (int i = 0; i < PB_STAGES; ++i) lr_mbar_init(bar0 + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    // the item that is copied next
    int f = (int)(it0 / n_kv), h = (int)(it0 % n_kv);
    int b = stream_of(pre, d.B, f), first, len;
    int row = range(b, first, len);
    int lp = first + f - pre[b], page = stream_page(d.c, row, lp, -1);
    int to_copy = left;
    auto copy = [&](int stage) {
        if (to_copy == 0) return;
        // an entry that is no page has no bounds to write either: page 0 stands in for it in the ring, with no rows
        const size_t unit = (size_t)max(page, 0) * n_kv + h;
        const int rows = page < 0 ? 0 : min(PIKV_PAGE_TOKENS, len - lp * PIKV_PAGE_TOKENS);
        unsigned char* to = ring + stage * GEO::STAGE;
        if (lane == 0) {
            const uint32_t dst = lr_smem_u32(to), bar = bar0 + 8 * stage;
            *reinterpret_cast<int4*>(to + GEO::COPY) = make_int4((int)(uint32_t)unit, (int)(uint32_t)(unit >> 32), rows, 0);
            lr_mbar_expect_tx(bar, GEO::COPY);
            pb_bulk(dst, d.c.k_codes + unit * GEO::CODES, GEO::CODES, bar);
            pb_bulk(dst + GEO::CODES, d.c.k_scale + unit * 16, 32, bar);
            if (BITS == 4) pb_bulk(dst + GEO::CODES + 32, d.c.k_zp + unit * 16, 64, bar);
        }
        __syncwarp();
        if (--to_copy == 0) return;
        if (++h < n_kv) return;
        h = 0;
        if (++f == pre[b + 1]) {
            do ++b; while (pre[b + 1] <= f);
            row = range(b, first, len);
        }
        lp = first + f - pre[b];
        page = stream_page(d.c, row, lp, -1);
    };
    for (int i = 0; i < PB_STAGES - 1; ++i) copy(i);
    int stage = 0;
    uint32_t phase = 0;
    bool late = false;
    for (; left > 0; --left) {
        copy(stage == 0 ? PB_STAGES - 1 : stage - 1);            // the stage of the item before this one
        late |= !lr_mbar_wait(bar0 + 8 * stage, phase);
        if (late) break;
        const unsigned char* from = ring + stage * GEO::STAGE;
        const int4 what = *reinterpret_cast<const int4*>(from + GEO::COPY);
        const size_t unit = (size_t)(uint32_t)what.y << 32 | (uint32_t)what.x;
        const int rows = what.z;
        uint32_t w[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            // 8 bit: chunk lane / 4 of row i; 4 bit: unit (lane % 16) / 2 of row 2 i + lane / 16
            const int r = BITS == 8 ? i : 2 * i + (lane >> 4);
            const int at = BITS == 8 ? i * 128 + 16 * ((lane >> 2) ^ (i & 7)) + 4 * (lane & 3) : r * 64 + 8 * (((lane & 15) >> 1) ^ (r & 4)) + 4 * (lane & 1);
            w[i] = *reinterpret_cast<const uint32_t*>(from + at);
        }
        // this lane's row, lane % 16: scale as m 2^(E - 134)
        const uint32_t mine = reinterpret_cast<const uint16_t*>(from + GEO::CODES)[lane & 15];
        const bool inside = (lane & 15) < rows;
        const int E = max(1, (int)((mine >> 7) & 0xffu));
        const uint32_t m = (mine & 0x7fu) | (mine & 0x7f80u ? 0x80u : 0u);
        float zmine = 0.f;
        if (BITS == 4) zmine = reinterpret_cast<const float*>(from + GEO::CODES + 32)[lane & 15];
        // a row that bounds cannot hold
        const bool bad = __any_sync(0xffffffffu, inside && ((mine & 0x7fffu) >= PB_HUGE_BITS || !(fabsf(zmine) < PB_HUGE)));
        const int least = __reduce_min_sync(0xffffffffu, m ? E : 255), most = __reduce_max_sync(0xffffffffu, m ? E : 0);
        const bool whole = rows == PIKV_PAGE_TOKENS && least >= 8 && most - least <= 15 &&
                           __all_sync(0xffffffffu, mine < 0x8000u && (BITS == 8 || (fabsf(zmine) <= 127.f && zmine == rintf(zmine))));
        float hi[CH], lo[CH];
        if (whole) {
            // m 2^(E - least) of the rows, as the lanes of their rows have it, and (4 bit) the zero point
            const int factor = (int)(m << (m ? E - least : 0)), off = BITS == 4 ? -(int)zmine : 0;
            int ihi[CH], ilo[CH];
#pragma unroll
            for (int k = 0; k < CH; ++k) ihi[k] = -0x7fffffff, ilo[k] = 0x7fffffff;
            auto keys = [&](int i, int (&x)[CH]) {
                const int r = BITS == 8 ? i : 2 * i + (lane >> 4);
                const int mr = __shfl_sync(0xffffffffu, factor, r);
                if constexpr (BITS == 8) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        int p;                                               // byte k, with its sign
                        asm("dp4a.s32.u32 %0, %1, %2, 0;" : "=r"(p) : "r"(w[i]), "r"(1u << (8 * k)));
                        x[k] = p * mr;
                    }
                } else {
                    const int c = __shfl_sync(0xffffffffu, off, r);
                    const uint32_t n0 = w[i] & 0x0f0f0f0fu, n1 = (w[i] >> 4) & 0x0f0f0f0fu;       // even and odd channels
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        int p, q;                                            // code less zero point
                        asm("dp4a.s32.u32 %0, %1, %2, %3;" : "=r"(p) : "r"(n0), "r"(1u << (8 * k)), "r"(c));
                        asm("dp4a.s32.u32 %0, %1, %2, %3;" : "=r"(q) : "r"(n1), "r"(1u << (8 * k)), "r"(c));
                        x[2 * k] = p * mr;
                        x[2 * k + 1] = q * mr;
                    }
                }
            };
#pragma unroll
            for (int i = 0; i < ROWS; i += 2) {
                int x[CH], y[CH];
                keys(i, x);
                keys(i + 1, y);
#pragma unroll
                for (int k = 0; k < CH; ++k) {
                    ihi[k] = __vimax3_s32(ihi[k], x[k], y[k]);
                    ilo[k] = __vimin3_s32(ilo[k], x[k], y[k]);
                }
            }
            // (16 bits and a shift: exact)
            const float unit_of = exp2_int(least - 134);
#pragma unroll
            for (int k = 0; k < CH; ++k) hi[k] = (float)ihi[k] * unit_of, lo[k] = (float)ilo[k] * unit_of;
        } else {
            const uint4 s_lo = *reinterpret_cast<const uint4*>(from + GEO::CODES), s_hi = *reinterpret_cast<const uint4*>(from + GEO::CODES + 16);
            const uint32_t sw[8] = {s_lo.x, s_lo.y, s_lo.z, s_lo.w, s_hi.x, s_hi.y, s_hi.z, s_hi.w};
#pragma unroll
            for (int i = 0; i < CH; ++i) hi[i] = -INFINITY, lo[i] = INFINITY;
            auto scale = [&](int r) { return __uint_as_float(r & 1 ? sw[r >> 1] & 0xffff0000u : sw[r >> 1] << 16); };
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                float x[CH];
                if constexpr (BITS == 8) {
                    const float s = scale(i), c = -32896.f * s;
                    const uint32_t u = w[i] ^ 0x80808080u;                   // code + 128
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[k] = fmaf(__uint_as_float(__byte_perm(u, 0x47000000u, 0x7504u + 16u * k)), s, c);
                } else {
                    const float s = lane >> 4 ? scale(2 * i + 1) : scale(2 * i), z = reinterpret_cast<const float*>(from + GEO::CODES + 32)[2 * i + (lane >> 4)];
                    // even channels in the low nibbles; less the zero point, times the scale, each rounded as the cache's reader does
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = __fmul_rn(__fsub_rn((float)((w[i] >> (4 * k)) & 15u), z), s);
                }
                if ((BITS == 8 ? i : 2 * i + (lane >> 4)) < rows) {
#pragma unroll
                    for (int k = 0; k < CH; ++k) {
                        hi[k] = fmaxf(hi[k], x[k]);
                        lo[k] = fminf(lo[k], x[k]);
                    }
                }
            }
            // a bound too small for its quotient by the step to be a float is a step all the same: 2^-40 of the largest stands for it
            float a = 0.f;
#pragma unroll
            for (int k = 0; k < CH; ++k) a = fmaxf(a, fmaxf(hi[k], -lo[k]));
            const float some = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(a))) * 9.094947e-13f;
#pragma unroll
            for (int k = 0; k < CH; ++k) {
                if (hi[k] > 0.f) hi[k] = fmaxf(hi[k], some);
                if (lo[k] < 0.f) lo[k] = fminf(lo[k], -some);
            }
        }
        int at = 4 * lane;
        if (BITS == 4) {
            // lanes l and l + 16 have the same channels: each keeps four of the eight
            const bool up = lane >> 4;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float gh = __shfl_xor_sync(0xffffffffu, up ? hi[k] : hi[CH - 4 + k], 16), gl = __shfl_xor_sync(0xffffffffu, up ? lo[k] : lo[CH - 4 + k], 16);
                hi[k] = fmaxf(up ? hi[CH - 4 + k] : hi[k], gh);
                lo[k] = fminf(up ? lo[CH - 4 + k] : lo[k], gl);
            }
            at = 8 * (lane & 15) + (up ? 4 : 0);
        }
        float a = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) a = fmaxf(a, fmaxf(fabsf(hi[k]), fabsf(lo[k])));
        // (bits of a float that is not negative order as it does)
        const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(a));
        const bool odd = bad || top >= 0x7f800000u;
        const int e = odd ? 0 : step_exponent(__uint_as_float(top));
        const float inv = exp2_int(-e);
        uint32_t ph = 0, pl = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int ih = odd ? 0 : __float2int_ru(hi[k] * inv), il = odd ? 0 : __float2int_rd(lo[k] * inv);
            ph |= (uint32_t)(ih & 0xff) << (8 * k);
            pl |= (uint32_t)(il & 0xff) << (8 * k);
        }
        if (rows > 0) {
            *reinterpret_cast<uint32_t*>(d.codes + unit * 256 + at) = ph;
            *reinterpret_cast<uint32_t*>(d.codes + unit * 256 + 128 + at) = pl;
            if (lane == 0) d.scale[unit] = odd ? INFINITY : exp2_int(e);
        }
        // The stage is copied into again: this warp's reads come before the proxy that copies.  (Every word read has been used by here,
        // but nothing else would keep a read that the compiler moves down from a copy that lands under it.)
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (++stage == PB_STAGES) stage = 0, phase ^= 1u;
    }
    if (late) {
        if (lane == 0 && d.c.status) atomicOr(d.c.status, PIKV_ST_WAIT_TIMEOUT);
        // what is on its way lands before the block leaves
        for (int i = 0; i < PB_STAGES; ++i) (void)lr_mbar_wait(bar0 + 8 * i, i < stage ? phase ^ 1u : phase);
    }
}

// ---- scores ---------------------------------------------------------------------------------------------------
constexpr int PS_THREADS = 256;
constexpr int PS_CTAS = 3;               // per SM
constexpr int PS_GROUP = 8;              // query heads per KV head, at most

struct SelectDev {
    CacheDev c;
    const __nv_bfloat16* q;              // [B][n_q][128]
    int B, n_q, G;
    const int* seq_ids;
    const int* seq_len;
    const uint8_t* bound_codes;
    const float* bound_scale;
    int pages, first, recent;
    uint32_t* keys;                      // [B][n_kv][max_pages] ascending with the score; candidates from 0
    int* list;                           // [B][n_kv][pages] physical pages
    int* chosen;                         // the same as page numbers, or null
    int* eff_len;                        // [B] rows of the listed pages
};

__device__ __forceinline__ void ps_mma(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// rows of a stream that the call sees
__device__ __forceinline__ int select_len(const SelectDev& d, int i) {
    if (stream_row(d.c, d.seq_ids, i) < 0) return 0;
    return max(0, min(__ldg(d.seq_len + i), d.c.max_pages * PIKV_PAGE_TOKENS));
}

// A warp scores 16 pages of one KV head at a time: m16n8k32 with the pages' bounds as A (a row of 256 bytes per page, its 16
// chunks dealt to the four lanes of a row so that every load is 16 bytes) and the group's query heads as the 8 columns of B.
// Bound by the bytes: 260 a page and head, of the next 16 pages while these are scored; 64 streams x 8 heads x 2048 pages:
// 53 us = 5.2 TB/s.
__global__ void __launch_bounds__(PS_THREADS, PS_CTAS) page_score_kernel(SelectDev d) {
    __shared__ int pre[PIKV_STREAMS_PER_LAUNCH + 1];
    const int lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3;
    const int n_kv = d.c.n_kv;
    dependency_release();
    dependency_wait();
    auto candidates = [&](int i) {
        const int n = (select_len(d, i) + PIKV_PAGE_TOKENS - 1) / PIKV_PAGE_TOKENS;
        return n > d.pages ? n - d.first - d.recent : 0;
    };
    const int total = stream_prefix<PS_THREADS>(d.B, pre, [&](int i) { return (candidates(i) + 15) / 16; });
    const long long items = (long long)total * n_kv;                       // per stream: head by head, 16 pages each
    const int warps = gridDim.x * (PS_THREADS / 32);
    const int self = (threadIdx.x >> 5) * gridDim.x + blockIdx.x;
    const long long run = (items + warps - 1) / warps, it0 = min(items, self * run);
    int left = (int)(min(items, it0 + run) - it0);
    if (left <= 0) return;
    int b = stream_of(pre, d.B, (int)(it0 / n_kv)), h, g, groups, cand, row;
    auto enter = [&]() {
        groups = pre[b + 1] - pre[b];
        cand = candidates(b);
        row = stream_row(d.c, d.seq_ids, b);
    };
    enter();
    {
        const int in_b = (int)(it0 - (long long)pre[b] * n_kv);
        h = in_b / groups;
        g = in_b % groups;
    }
    // physical pages of candidates g * 16 + r and 8 on, of the next item while this one is scored
    auto pages = [&](int& lo, int& hi) {
        const int p = g * 16 + r;
        lo = p < cand ? stream_page(d.c, row, d.first + p) : 0;
        hi = p + 8 < cand ? stream_page(d.c, row, d.first + p + 8) : 0;
    };
    int page_lo, page_hi;
    pages(page_lo, page_hi);
    int have_b = -1, have_h = -1;
    uint32_t qf[16];
    float sq0 = 0.f, sq1 = 0.f;                                            // scale of query heads 2j, 2j+1; 0: no say
    for (;; --left) {
        if (b != have_b || h != have_h) {
            have_b = b;
            have_h = h;
            // column r = query head r: channels of chunks j and j + 4, twice: the positive part against the largest
            // keys, the negative part against the smallest
            float x[32];
            float a = 0.f;
            bool fin = true;
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] = 0.f;
            if (r < d.G) {
                const uint4* qp = reinterpret_cast<const uint4*>(d.q + ((size_t)b * d.n_q + (size_t)h * d.G + r) * 128);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint4 w = __ldg(qp + 2 * (j + 4 * (i >> 1)) + (i & 1));
                    bf16x2_to_f32(w.x, x[8 * i], x[8 * i + 1]);
                    bf16x2_to_f32(w.y, x[8 * i + 2], x[8 * i + 3]);
                    bf16x2_to_f32(w.z, x[8 * i + 4], x[8 * i + 5]);
                    bf16x2_to_f32(w.w, x[8 * i + 6], x[8 * i + 7]);
                }
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                a = fmaxf(a, fabsf(x[i]));
                fin &= fabsf(x[i]) < INFINITY;
            }
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
            fin = !(__ballot_sync(0xffffffffu, !fin) & (0xfu << (lane & ~3)));
            const int e = fin ? step_exponent(a) : 0;
            const float inv = exp2_int(-e);
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                uint32_t pos = 0, neg = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int u = fin ? __float2int_rn(x[4 * w + i] * inv) : 0;
                    pos |= (uint32_t)(max(u, 0) & 0xff) << (8 * i);
                    neg |= (uint32_t)(min(u, 0) & 0xff) << (8 * i);
                }
                qf[w] = pos;
                qf[8 + w] = neg;
            }
            // only ratios matter: relative to the group's largest step, and so small that products with a page's step stay in fp32's range
            const int e_most = __reduce_max_sync(0xffffffffu, fin && r < d.G ? e : -126);
            const float sq = fin && r < d.G ? exp2_int(max(-126, e - e_most - 23)) : 0.f;
            sq0 = __shfl_sync(0xffffffffu, sq, 8 * j);
            sq1 = __shfl_sync(0xffffffffu, sq, 8 * j + 4);
        }
        const uint4* lo = reinterpret_cast<const uint4*>(d.bound_codes + ((size_t)page_lo * n_kv + h) * 256);
        const uint4* hi = reinterpret_cast<const uint4*>(d.bound_codes + ((size_t)page_hi * n_kv + h) * 256);
        uint4 wl[4], wh[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            wl[i] = ld_stream_16(lo + j + 4 * i);
            wh[i] = ld_stream_16(hi + j + 4 * i);
        }
        const float s_lo = __ldg(d.bound_scale + (size_t)page_lo * n_kv + h), s_hi = __ldg(d.bound_scale + (size_t)page_hi * n_kv + h);
        const int p_lo = g * 16 + r, p_hi = p_lo + 8;                       // candidates behind the first pages
        uint32_t* to = d.keys + ((size_t)b * n_kv + h) * d.c.max_pages;
        const int cand_now = cand;
        if (left > 1) {
            if (++g == groups) {
                g = 0;
                if (++h == n_kv) {
                    h = 0;
                    do ++b; while (pre[b + 1] == pre[b]);
                    enter();
                }
            }
            pages(page_lo, page_hi);
        }
        int acc[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ps_mma(acc, wl[i].x, wh[i].x, wl[i].y, wh[i].y, qf[4 * i], qf[4 * i + 1]);
            ps_mma(acc, wl[i].z, wh[i].z, wl[i].w, wh[i].w, qf[4 * i + 2], qf[4 * i + 3]);
        }
        // (whole number below 2^23 * query step) * page step, and the best of the group's heads
        auto score = [&](int dot, float sp, float sq) { return sq > 0.f ? ((float)dot * sq) * sp : -INFINITY; };
        float t_lo = fmaxf(score(acc[0], s_lo, sq0), score(acc[1], s_lo, sq1));
        float t_hi = fmaxf(score(acc[2], s_hi, sq0), score(acc[3], s_hi, sq1));
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            t_lo = fmaxf(t_lo, __shfl_xor_sync(0xffffffffu, t_lo, o));
            t_hi = fmaxf(t_hi, __shfl_xor_sync(0xffffffffu, t_hi, o));
        }
        if (!(s_lo < INFINITY)) t_lo = INFINITY;
        if (!(s_hi < INFINITY)) t_hi = INFINITY;
        auto key = [](float t) {
            const uint32_t u = __float_as_uint(t + 0.f);                    // -0 is 0
            return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
        };
        if (j == 0) {
            if (p_lo < cand_now) to[p_lo] = key(t_lo);
            if (p_hi < cand_now) to[p_hi] = key(t_hi);
        }
        if (left == 1) return;
    }
}

// ---- selection ------------------------------------------------------------------------------------------------
constexpr int SL_THREADS = 512;
constexpr int SL_LOG_BINS = 10, SL_BINS = 1 << SL_LOG_BINS;

// One CTA per (stream, KV head): the want-th largest key, then the kept pages in ascending order.  Keys are read once into
// shared memory.  The threshold: bins of equal width over the range that the keys really have (bins over the bits of the
// key would put neighbouring exponents' keys on a few counters, one after the other), then the few keys of the bin that it
// falls into are ranked against one another; a bin that holds too many is cut into bins again.  A chain of block-wide steps:
// 17 us for 64 streams x 8 heads x 2048 keys, 8 us for one stream's.
__global__ void __launch_bounds__(SL_THREADS) page_select_kernel(SelectDev d) {
    extern __shared__ uint32_t keys[];
    __shared__ int hist[SL_BINS];
    __shared__ uint32_t few[SL_THREADS];
    __shared__ uint32_t warp_lo[SL_THREADS / 32], warp_hi[SL_THREADS / 32];
    __shared__ int warp_tot[2][SL_THREADS / 32];
    __shared__ int pick[3];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n_kv = d.c.n_kv, b = blockIdx.x / n_kv, h = blockIdx.x % n_kv;
    dependency_release();
    dependency_wait();
    const int row = stream_row(d.c, d.seq_ids, b);
    const int len = select_len(d, b);
    const int n = (len + PIKV_PAGE_TOKENS - 1) / PIKV_PAGE_TOKENS;
    const int count = min(n, d.pages);
    if (h == 0 && tid == 0) {
        d.eff_len[b] = count > 0 ? len - (n - count) * PIKV_PAGE_TOKENS : 0;
        if (row < 0 && d.c.status) atomicOr(d.c.status, PIKV_ST_BAD_SEQ);
    }
    int* list = d.list + (size_t)blockIdx.x * d.pages;
    int* chosen = d.chosen ? d.chosen + (size_t)blockIdx.x * d.pages : nullptr;
    const int* table = d.c.page_table + (size_t)max(row, 0) * d.c.max_pages;
    auto put = [&](int at, int page) {
        list[at] = __ldg(table + page);
        if (chosen) chosen[at] = page;
    };
    for (int i = count + tid; i < d.pages; i += SL_THREADS) {
        list[i] = -1;
        if (chosen) chosen[i] = -1;
    }
    if (n <= d.pages) {
        for (int i = tid; i < n; i += SL_THREADS) put(i, i);
        return;
    }
    const int cand = n - d.first - d.recent, want = d.pages - d.first - d.recent;
    for (int i = tid; i < d.first; i += SL_THREADS) put(i, i);
    for (int i = tid; i < d.recent; i += SL_THREADS) put(d.first + want + i, n - d.recent + i);
    if (want == 0) return;
    const uint32_t* from = d.keys + (size_t)blockIdx.x * d.c.max_pages;
    uint32_t lo = 0xffffffffu, hi = 0u;
    for (int i = tid; i < cand; i += SL_THREADS) {
        const uint32_t k = __ldcg(from + i);
        keys[i] = k;
        lo = min(lo, k);
        hi = max(hi, k);
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) warp_lo[warp] = lo, warp_hi[warp] = hi;
    for (int i = tid; i < SL_BINS; i += SL_THREADS) hist[i] = 0;
    __syncthreads();
    lo = __reduce_min_sync(0xffffffffu, warp_lo[lane % (SL_THREADS / 32)]);
    hi = __reduce_max_sync(0xffffffffu, warp_hi[lane % (SL_THREADS / 32)]);
    int left = want;                        // of the keys in [lo, hi], from the top
    uint32_t threshold;
    for (;;) {
        // bins of 2^shift keys over [lo, hi], the last one from the top
        const int shift = max(0, 32 - __clz((int)((hi - lo) | 1u)) - SL_LOG_BINS);
        for (int i = tid; i < cand; i += SL_THREADS) {
            const uint32_t k = keys[i];
            if (k >= lo && k <= hi) atomicAdd(&hist[(k - lo) >> shift], 1);
        }
        __syncthreads();
        // thread t owns bins per (t + 1) - 1 .. per t below the top
        constexpr int per = SL_BINS / SL_THREADS;
        const int top = SL_BINS - 1 - per * tid;
        int c[per], sum = 0;
#pragma unroll
        for (int i = 0; i < per; ++i) {
            c[i] = hist[top - i];
            sum += c[i];
        }
        int inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += x;
        }
        if (lane == 31) warp_tot[0][warp] = inc;
        if (tid == 0) pick[2] = 0;
        __syncthreads();
        int before = inc - sum;
        for (int w = 0; w < warp; ++w) before += warp_tot[0][w];
        if (before < left && before + sum >= left) {
            int i = 0, run = before;
#pragma unroll
            for (int k = 0; k < per - 1; ++k)
                if (i == k && run + c[k] < left) run += c[k], ++i;
            pick[0] = top - i;
            pick[1] = left - run;
        }
#pragma unroll
        for (int i = 0; i < per; ++i) hist[top - i] = 0;
        __syncthreads();
        left = pick[1];
        lo += (uint32_t)pick[0] << shift;
        if (shift == 0) {
            threshold = lo;                 // a bin is one key
            break;
        }
        hi = min(hi, lo + ((1u << shift) - 1u));
        for (int i = tid; i < cand; i += SL_THREADS) {
            const uint32_t k = keys[i];
            if (k >= lo && k <= hi) {
                const int at = atomicAdd(&pick[2], 1);
                if (at < SL_THREADS) few[at] = k;
            }
        }
        __syncthreads();
        const int m = pick[2];
        if (m <= SL_THREADS) {
            if (tid < m) {
                const uint32_t mine = few[tid];
                int above = 0, same = 0;
                for (int i = 0; i < m; ++i) {
                    above += few[i] > mine;
                    same += few[i] == mine;
                }
                // (threads with equal keys write the same)
                if (above < left && above + same >= left) pick[0] = (int)mine, pick[1] = left - above;
            }
            __syncthreads();
            threshold = (uint32_t)pick[0];
            left = pick[1];
            break;
        }
        __syncthreads();
    }
    // thread t owns a run of candidates: those above the threshold, and the first `left` equal to it
    const int per = (cand + SL_THREADS - 1) / SL_THREADS, c0 = min(cand, tid * per), c1 = min(cand, c0 + per);
    int above = 0, equal = 0;
    for (int i = c0; i < c1; ++i) {
        above += keys[i] > threshold;
        equal += keys[i] == threshold;
    }
    int ia = above, ie = equal;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int xa = __shfl_up_sync(0xffffffffu, ia, o), xe = __shfl_up_sync(0xffffffffu, ie, o);
        if (lane >= o) ia += xa, ie += xe;
    }
    if (lane == 31) warp_tot[0][warp] = ia, warp_tot[1][warp] = ie;
    __syncthreads();
    int at = ia - above, eq = ie - equal;
    for (int w = 0; w < warp; ++w) at += warp_tot[0][w], eq += warp_tot[1][w];
    at += min(eq, left);
    for (int i = c0; i < c1; ++i) {
        const uint32_t k = keys[i];
        if (k < threshold || (k == threshold && eq++ >= left)) continue;
        put(d.first + at++, d.first + i);
    }
}

// workspace: effective lengths, page lists, keys, then the decode kernels' own
struct SparseLayout {
    size_t list, keys, decode, total;
};
static SparseLayout sparse_layout(int64_t B, int n_q, int n_kv, int64_t max_pages, int64_t pages) {
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    SparseLayout l;
    l.list = up((size_t)B * sizeof(int));
    l.keys = l.list + up((size_t)(B * n_kv * pages) * sizeof(int));
    l.decode = l.keys + up((size_t)(B * n_kv * max_pages) * sizeof(uint32_t));
    l.total = l.decode + pikv_decode_attn_workspace_bytes((int32_t)B, n_q, n_kv, 0, 0);
    return l;
}

}  // namespace pikv

using namespace pikv;

extern "C" int pikv_page_bounds_update(const pikv_paged_cache* c, void* bound_codes, float* bound_scale, const int32_t* seq_ids,
                                       const int32_t* start, const int32_t* seq_len, int32_t B, pikv_stream_t stream) {
    BoundsDev d;
    const int rc = cache_dev(c, d.c, "page_bounds_update", true);
    if (rc != PIKV_OK) return rc;
    PIKV_REQUIRE(bound_codes && bound_scale && seq_len, PIKV_EINVAL, "page_bounds_update: null pointer");
    PIKV_REQUIRE(B > 0 && (seq_ids || B <= c->num_seqs), PIKV_EINVAL, "page_bounds_update: %d streams, the cache has %d", B, c->num_seqs);
    PIKV_REQUIRE((reinterpret_cast<uintptr_t>(bound_codes) & 15) == 0, PIKV_EINVAL, "page_bounds_update: bound_codes must be 16-byte aligned");
    PIKV_REQUIRE((long long)std::min(B, PIKV_STREAMS_PER_LAUNCH) * c->max_pages < (1ll << 31), PIKV_ELIMIT, "page_bounds_update: streams * max_pages must stay below 2^31");
    d.codes = static_cast<uint8_t*>(bound_codes);
    d.scale = bound_scale;
    for (int b0 = 0; b0 < B; b0 += PIKV_STREAMS_PER_LAUNCH) {
        d.B = std::min(B - b0, PIKV_STREAMS_PER_LAUNCH);
        // without ids stream b is row b: a chunk behind the first starts further down the table
        d.c.page_table = c->page_table + (seq_ids ? 0 : (size_t)b0 * c->max_pages);
        d.c.num_seqs = seq_ids ? c->num_seqs : c->num_seqs - b0;
        d.seq_ids = seq_ids ? seq_ids + b0 : nullptr;
        d.start = start ? start + b0 : nullptr;
        d.seq_len = seq_len + b0;
        const long long most = (long long)d.B * c->max_pages * c->n_kv;
        const int grid = (int)std::min<long long>((long long)sm_count() * PB_CTAS, (most + PB_THREADS / 32 - 1) / (PB_THREADS / 32));
        if (c->bits == 8) {
            if (!allow_smem<page_bounds_kernel<8>>(PBGeom<8>::SMEM)) return check_launch("page_bounds smem attribute");
            launch_dependent(page_bounds_kernel<8>, grid, PB_THREADS, PBGeom<8>::SMEM, static_cast<cudaStream_t>(stream), d);
        } else {
            if (!allow_smem<page_bounds_kernel<4>>(PBGeom<4>::SMEM)) return check_launch("page_bounds smem attribute");
            launch_dependent(page_bounds_kernel<4>, grid, PB_THREADS, PBGeom<4>::SMEM, static_cast<cudaStream_t>(stream), d);
        }
        count_launch(1);
    }
    return check_launch("page_bounds_kernel");
}

extern "C" size_t pikv_sparse_attn_workspace_bytes(int32_t B, int32_t n_q, int32_t n_kv, int32_t max_pages, int32_t pages) {
    if (B <= 0 || n_q <= 0 || n_kv <= 0 || n_q % n_kv != 0 || max_pages <= 0 || pages <= 0) return 0;
    return sparse_layout(std::min(B, PIKV_STREAMS_PER_LAUNCH), n_q, n_kv, max_pages, pages).total;
}

extern "C" int pikv_sparse_attn(const pikv_paged_cache* c, const pikv_sparse_params* p, pikv_stream_t stream) {
    SelectDev d;
    const int rc = cache_dev(c, d.c, "sparse_attn", true);
    if (rc != PIKV_OK) return rc;
    PIKV_REQUIRE(p != nullptr && p->q && p->out && p->seq_len && p->bound_codes && p->bound_scale && p->workspace, PIKV_EINVAL, "sparse_attn: null pointer");
    PIKV_REQUIRE(p->B > 0 && p->n_q > 0 && p->n_q % c->n_kv == 0, PIKV_EINVAL, "sparse_attn: bad head counts");
    PIKV_REQUIRE(p->seq_ids || p->B <= c->num_seqs, PIKV_EINVAL, "sparse_attn: %d streams, the cache has %d", p->B, c->num_seqs);
    PIKV_REQUIRE(p->n_q / c->n_kv <= PS_GROUP, PIKV_EUNSUPPORTED, "sparse_attn: %d query heads per KV head (max %d)", p->n_q / c->n_kv, PS_GROUP);
    PIKV_REQUIRE(p->first >= 0 && p->recent >= 1 && p->pages >= 1 && (long long)p->first + p->recent <= p->pages, PIKV_EINVAL,
                 "sparse_attn: first %d + recent %d (at least 1) must fit in %d pages", p->first, p->recent, p->pages);
    PIKV_REQUIRE(c->max_pages <= PIKV_SPARSE_MAX_PAGES, PIKV_ELIMIT, "sparse_attn: a stream has %d pages at most (got %d)", PIKV_SPARSE_MAX_PAGES, c->max_pages);
    PIKV_REQUIRE(((reinterpret_cast<uintptr_t>(p->workspace) | reinterpret_cast<uintptr_t>(p->bound_codes) | reinterpret_cast<uintptr_t>(p->q) |
                   reinterpret_cast<uintptr_t>(p->out)) & 15) == 0, PIKV_EINVAL, "sparse_attn: q, out, bound_codes and workspace must be 16-byte aligned");
    // a list longer than any stream's table holds nothing in its tail
    const int pages = p->pages;
    const SparseLayout lay = sparse_layout(std::min(p->B, PIKV_STREAMS_PER_LAUNCH), p->n_q, c->n_kv, c->max_pages, pages);
    PIKV_REQUIRE(p->workspace_bytes >= lay.total, PIKV_EINVAL, "sparse_attn: workspace too small (%zu bytes, %zu needed)", p->workspace_bytes, lay.total);
    PIKV_REQUIRE((long long)std::min(p->B, PIKV_STREAMS_PER_LAUNCH) * std::max(pages, c->max_pages) * c->n_kv < (1ll << 31), PIKV_ELIMIT,
                 "sparse_attn: streams * pages * heads must stay below 2^31");
    unsigned char* ws = static_cast<unsigned char*>(p->workspace);
    d.eff_len = reinterpret_cast<int*>(ws);
    d.list = reinterpret_cast<int*>(ws + lay.list);
    d.keys = reinterpret_cast<uint32_t*>(ws + lay.keys);
    d.n_q = p->n_q; d.G = p->n_q / c->n_kv;
    d.bound_codes = static_cast<const uint8_t*>(p->bound_codes);
    d.bound_scale = p->bound_scale;
    d.pages = pages; d.first = p->first; d.recent = p->recent;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int most = std::max(0, c->max_pages - p->first - p->recent);      // candidates of a stream
    for (int b0 = 0; b0 < p->B; b0 += PIKV_STREAMS_PER_LAUNCH) {
        d.B = std::min(p->B - b0, PIKV_STREAMS_PER_LAUNCH);
        d.c.page_table = c->page_table + (p->seq_ids ? 0 : (size_t)b0 * c->max_pages);
        d.c.num_seqs = p->seq_ids ? c->num_seqs : c->num_seqs - b0;
        d.seq_ids = p->seq_ids ? p->seq_ids + b0 : nullptr;
        d.seq_len = p->seq_len + b0;
        d.q = static_cast<const __nv_bfloat16*>(p->q) + (size_t)b0 * p->n_q * 128;
        d.chosen = p->chosen ? p->chosen + (size_t)b0 * c->n_kv * pages : nullptr;
        if (c->max_pages > pages) {                                          // else nothing can need a choice
            const long long items = (long long)d.B * c->n_kv * ((most + 15) / 16);
            const int grid = (int)std::min<long long>((long long)sm_count() * PS_CTAS, (items + PS_THREADS / 32 - 1) / (PS_THREADS / 32));
            // A plain launch: CTAs of a dependent one come to the SMs that the kernel before leaves first, several to one, and
            // each has its share of the list already (64 x 32768: 191 us a step against 125)
            page_score_kernel<<<grid, PS_THREADS, 0, st>>>(d);
            count_launch(1);
        }
        const size_t smem = c->max_pages > pages ? (size_t)most * sizeof(uint32_t) : 0;
        if (!allow_smem<page_select_kernel>(PIKV_SPARSE_MAX_PAGES * (int)sizeof(uint32_t))) return check_launch("page_select smem attribute");
        launch_dependent(page_select_kernel, d.B * c->n_kv, SL_THREADS, smem, st, d);
        count_launch(1);
        int err = check_launch("page_select_kernel");
        if (err != PIKV_OK) return err;
        pikv_decode_params a = {};
        a.q = d.q; a.out = static_cast<__nv_bfloat16*>(p->out) + (size_t)b0 * p->n_q * 128;
        a.lse = p->lse ? p->lse + (size_t)b0 * p->n_q : nullptr;
        a.B = d.B; a.n_q = p->n_q; a.n_kv = c->n_kv;
        a.seq_len = d.eff_len; a.page_table = d.list;
        a.num_seqs = d.B; a.max_pages = pages; a.num_pages = c->num_pages;
        a.k_codes = c->k_codes; a.v_codes = c->v_codes; a.k_scale = c->k_scale; a.v_scale = c->v_scale; a.k_zp = c->k_zp; a.v_zp = c->v_zp;
        a.workspace = ws + lay.decode; a.workspace_bytes = p->workspace_bytes - lay.decode; a.status = c->status;
        err = decode_attn_run(&a, st, c->bits, nullptr, nullptr, nullptr, true);
        if (err != PIKV_OK) return err;
    }
    return PIKV_OK;
}
