// Sparse decode attention: bounds of every page's keys, the pages that those bounds select for a query, and attention over
// them (decode_attn.cu, with a page list per stream and KV head).
//
// A page is 16 rows.  For channel c let hi_c and lo_c be the largest and smallest key on it: no key of the page gives a
// query q a logit above sum_c max(q_c hi_c, q_c lo_c) = sum_c (max(q_c, 0) hi_c + min(q_c, 0) lo_c).  Bounds are kept as
// int8 in whole steps of a power of two (256 bytes for the 4 KB of a page and head), the query is brought to int8 the same
// way, so a score is ONE product of a page's 256 bytes with 256 bytes of query on the integer tensor cores, an exact whole
// number times exact powers of two: the choice of pages depends neither on the order of a sum nor on the type it is held in.
#include "stream_list.cuh"
#include "shard_decode.cuh"

namespace pikv {

// ---- bounds ---------------------------------------------------------------------------------------------------
constexpr int PB_THREADS = 256;
constexpr int PB_CTAS = 4;               // per SM

struct BoundsDev {
    CacheDev c;
    uint8_t* codes;                      // [num_pages][n_kv][2][128]
    float* scale;                        // [num_pages][n_kv]
    const int* seq_ids;
    const int* start;
    const int* seq_len;
    int B;
};

__device__ __forceinline__ float unit_code(uint32_t w, int i) { return (float)(int8_t)(w >> (8 * i)); }

// One warp per (page, head).  Lane l holds channels 16 (l & 7) .. + 15 of rows (l >> 3) + 4 i: one 16-byte chunk (8 bit) or
// one 8-byte unit (4 bit) of four rows, read where the cache's swizzle has put them, so that eight lanes read a whole row.
// The four row groups are joined by two exchanges in which a lane gives away half of its channels each time.
template <int BITS>
__global__ void __launch_bounds__(PB_THREADS, PB_CTAS) page_bounds_kernel(BoundsDev d) {
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
    const long long items = (long long)total * n_kv;
    const int warps = gridDim.x * (PB_THREADS / 32);
    const int self = (threadIdx.x >> 5) * gridDim.x + blockIdx.x;
    const int ch = lane & 7, rg = lane >> 3;
    for (long long it = self; it < items; it += warps) {
        const int f = (int)(it / n_kv), h = (int)(it % n_kv);
        const int b = stream_of(pre, d.B, f);
        int first, len;
        const int row = range(b, first, len);
        const int lp = first + f - pre[b];
        const int page = stream_page(d.c, row, lp);
        const int rows = min(PIKV_PAGE_TOKENS, len - lp * PIKV_PAGE_TOKENS);
        const size_t base = ((size_t)page * n_kv + h) * PIKV_PAGE_TOKENS;
        float hi[16], lo[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) hi[i] = -INFINITY, lo[i] = INFINITY;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = rg + 4 * i;
            if (r >= rows) continue;
            const float s = bf16_bits_to_f32(__ldg(d.c.k_scale + base + r));
            bad |= !(fabsf(s) < INFINITY);
            if (BITS == 8) {
                const uint4 w = __ldg(reinterpret_cast<const uint4*>(d.c.k_codes + (base + r) * 128) + (ch ^ (r & 7)));
                const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float x = unit_code(ww[j >> 2], j & 3) * s;
                    hi[j] = fmaxf(hi[j], x);
                    lo[j] = fminf(lo[j], x);
                }
            } else {
                const float z = __ldg(d.c.k_zp + base + r);
                bad |= !(fabsf(z) < INFINITY);
                const uint2 w = __ldg(reinterpret_cast<const uint2*>(d.c.k_codes + (base + r) * 64) + (ch ^ (r & 4)));
                const uint32_t ww[2] = {w.x, w.y};
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float x = __fmul_rn(__fsub_rn((float)((ww[j >> 3] >> (4 * (j & 7))) & 15u), z), s);
                    hi[j] = fmaxf(hi[j], x);
                    lo[j] = fminf(lo[j], x);
                }
            }
        }
        // lanes l and l ^ 16 keep channels 0..7 / 8..15 of their chunk, then l and l ^ 8 four of those
        const bool up16 = lane & 16, up8 = lane & 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float gh = __shfl_xor_sync(0xffffffffu, up16 ? hi[j] : hi[j + 8], 16);
            const float gl = __shfl_xor_sync(0xffffffffu, up16 ? lo[j] : lo[j + 8], 16);
            hi[j] = fmaxf(up16 ? hi[j + 8] : hi[j], gh);
            lo[j] = fminf(up16 ? lo[j + 8] : lo[j], gl);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float gh = __shfl_xor_sync(0xffffffffu, up8 ? hi[j] : hi[j + 4], 8);
            const float gl = __shfl_xor_sync(0xffffffffu, up8 ? lo[j] : lo[j + 4], 8);
            hi[j] = fmaxf(up8 ? hi[j + 4] : hi[j], gh);
            lo[j] = fminf(up8 ? lo[j + 4] : lo[j], gl);
        }
        float a = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) a = fmaxf(a, fmaxf(fabsf(hi[j]), fabsf(lo[j])));
        a = warp_max(a);
        bad = __any_sync(0xffffffffu, bad || !(a < INFINITY));
        const int e = bad ? 0 : step_exponent(a);
        const float inv = exp2_int(-e);
        uint32_t ph = 0, pl = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int ih = bad ? 0 : __float2int_ru(hi[j] * inv), il = bad ? 0 : __float2int_rd(lo[j] * inv);
            ph |= (uint32_t)(ih & 0xff) << (8 * j);
            pl |= (uint32_t)(il & 0xff) << (8 * j);
        }
        const size_t out = ((size_t)page * n_kv + h) * 256;
        const int at = 16 * ch + (up16 ? 8 : 0) + (up8 ? 4 : 0);
        *reinterpret_cast<uint32_t*>(d.codes + out + at) = ph;
        *reinterpret_cast<uint32_t*>(d.codes + out + 128 + at) = pl;
        if (lane == 0) d.scale[(size_t)page * n_kv + h] = bad ? INFINITY : exp2_int(e);
    }
}

// ---- scores ---------------------------------------------------------------------------------------------------
constexpr int PS_THREADS = 256;
constexpr int PS_CTAS = 4;               // per SM
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
    const long long per = (items + warps - 1) / warps, end = min(items, (self + 1ll) * per);
    int have_b = -1, have_h = -1;
    uint32_t qf[16];
    float sq0 = 0.f, sq1 = 0.f;                                            // scale of query heads 2j, 2j+1; 0: no say
    for (long long it = self * per; it < end; ++it) {
        const int b = stream_of(pre, d.B, (int)(it / n_kv));
        const int groups = pre[b + 1] - pre[b];
        const long long in_b = it - (long long)pre[b] * n_kv;
        const int h = (int)(in_b / groups), g = (int)(in_b % groups);
        const int cand = candidates(b);
        const int row = stream_row(d.c, d.seq_ids, b);
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
            const float sq = fin && r < d.G ? exp2_int(e) : 0.f;
            sq0 = __shfl_sync(0xffffffffu, sq, 8 * j);
            sq1 = __shfl_sync(0xffffffffu, sq, 8 * j + 4);
        }
        const int p_lo = g * 16 + r, p_hi = p_lo + 8;                       // candidates behind the first pages
        const int page_lo = p_lo < cand ? stream_page(d.c, row, d.first + p_lo) : 0;
        const int page_hi = p_hi < cand ? stream_page(d.c, row, d.first + p_hi) : 0;
        const uint4* lo = reinterpret_cast<const uint4*>(d.bound_codes + ((size_t)page_lo * n_kv + h) * 256);
        const uint4* hi = reinterpret_cast<const uint4*>(d.bound_codes + ((size_t)page_hi * n_kv + h) * 256);
        uint4 wl[4], wh[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            wl[i] = ld_stream_16(lo + j + 4 * i);
            wh[i] = ld_stream_16(hi + j + 4 * i);
        }
        const float s_lo = __ldg(d.bound_scale + (size_t)page_lo * n_kv + h), s_hi = __ldg(d.bound_scale + (size_t)page_hi * n_kv + h);
        int acc[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ps_mma(acc, wl[i].x, wh[i].x, wl[i].y, wh[i].y, qf[4 * i], qf[4 * i + 1]);
            ps_mma(acc, wl[i].z, wh[i].z, wl[i].w, wh[i].w, qf[4 * i + 2], qf[4 * i + 3]);
        }
        // (whole number * page step) * query step, and the best of the group's heads
        auto score = [&](int dot, float sp, float sq) { return sq > 0.f ? ((float)dot * sp) * sq : -INFINITY; };
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
            uint32_t* to = d.keys + ((size_t)b * n_kv + h) * d.c.max_pages;
            if (p_lo < cand) to[p_lo] = key(t_lo);
            if (p_hi < cand) to[p_hi] = key(t_hi);
        }
    }
}

// ---- selection ------------------------------------------------------------------------------------------------
constexpr int SL_THREADS = 512;

// One CTA per (stream, KV head): the want-th largest key by three rounds of counting (11, 11 and 10 bits), then the kept
// pages in ascending order.  Keys are read once into shared memory.
__global__ void __launch_bounds__(SL_THREADS) page_select_kernel(SelectDev d) {
    extern __shared__ uint32_t keys[];
    __shared__ int hist[2048];
    __shared__ int warp_tot[2][SL_THREADS / 32];
    __shared__ int pick[2];
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
    for (int i = tid; i < cand; i += SL_THREADS) keys[i] = __ldcg(from + i);
    uint32_t prefix = 0, known = 0;
    int left = want;                                                        // of the keys that agree with prefix on known
#pragma unroll 1
    for (int round = 0; round < 3; ++round) {
        const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, bins = round == 2 ? 1024 : 2048;
        for (int i = tid; i < bins; i += SL_THREADS) hist[i] = 0;
        __syncthreads();
        for (int i = tid; i < cand; i += SL_THREADS) {
            const uint32_t k = keys[i];
            if ((k & known) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
        }
        __syncthreads();
        // bins from the top: thread t owns bins - 1 - per t downwards
        const int per = bins / SL_THREADS, top = bins - 1 - per * tid;
        int sum = 0;
        for (int i = 0; i < per; ++i) sum += hist[top - i];
        int inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += x;
        }
        if (lane == 31) warp_tot[0][warp] = inc;
        __syncthreads();
        int before = inc - sum;
        for (int w = 0; w < warp; ++w) before += warp_tot[0][w];
        if (before < left && before + sum >= left) {
            int i = 0, run = before;
            while (run + hist[top - i] < left) run += hist[top - i++];
            pick[0] = top - i;
            pick[1] = left - run;
        }
        __syncthreads();
        prefix |= (uint32_t)pick[0] << shift;
        known |= (uint32_t)(bins - 1) << shift;
        left = pick[1];
    }
    // thread t owns a run of candidates: those above the threshold, and the first `left` equal to it
    const int per = (cand + SL_THREADS - 1) / SL_THREADS, lo = min(cand, tid * per), hi = min(cand, lo + per);
    int above = 0, equal = 0;
    for (int i = lo; i < hi; ++i) {
        above += keys[i] > prefix;
        equal += keys[i] == prefix;
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
    for (int i = lo; i < hi; ++i) {
        const uint32_t k = keys[i];
        if (k < prefix || (k == prefix && eq++ >= left)) continue;
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
        if (c->bits == 8) launch_dependent(page_bounds_kernel<8>, grid, PB_THREADS, 0, static_cast<cudaStream_t>(stream), d);
        else launch_dependent(page_bounds_kernel<4>, grid, PB_THREADS, 0, static_cast<cudaStream_t>(stream), d);
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
            launch_dependent(page_score_kernel, grid, PS_THREADS, 0, st, d);
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
