// Ragged work lists over the streams of a call: every CTA scans the streams' lengths itself, so that no kernel has to plan
// for the next one and nothing about the lengths is needed on the host.
#pragma once
#include "common.cuh"

namespace pikv {

// the cache of one call, as the kernels read it
struct CacheDev {
    const int* page_table;
    int num_seqs, max_pages, num_pages, n_kv, bits;
    uint8_t* k_codes;
    uint8_t* v_codes;
    uint16_t* k_scale;
    uint16_t* v_scale;
    float* k_zp;
    float* v_zp;
    unsigned* status;
};

static inline int cache_dev(const pikv_paged_cache* c, CacheDev& d, const char* what, bool decodable) {
    PIKV_REQUIRE(c != nullptr, PIKV_EINVAL, "%s: null cache", what);
    PIKV_REQUIRE(c->page_table && c->k_codes && c->v_codes && c->k_scale && c->v_scale, PIKV_EINVAL, "%s: null cache pointer", what);
    PIKV_REQUIRE(c->num_seqs > 0 && c->max_pages > 0 && c->num_pages > 0 && c->n_kv > 0, PIKV_EINVAL, "%s: bad cache geometry", what);
    PIKV_REQUIRE(c->bits == 8 || c->bits == 4, PIKV_EINVAL, "%s: bits must be 4 or 8", what);
    PIKV_REQUIRE((long long)c->max_pages * PIKV_PAGE_TOKENS < (1ll << 31), PIKV_ELIMIT, "%s: positions must stay below 2^31", what);
    PIKV_REQUIRE((long long)c->num_pages * c->n_kv < (1ll << 32), PIKV_ELIMIT, "%s: num_pages * n_kv must stay below 2^32", what);
    for (const void* pool : {(const void*)c->k_codes, (const void*)c->v_codes, (const void*)c->k_scale, (const void*)c->v_scale, (const void*)c->k_zp, (const void*)c->v_zp})
        PIKV_REQUIRE((reinterpret_cast<uintptr_t>(pool) & 15) == 0, PIKV_EINVAL, "%s: the cache's pools must be 16-byte aligned", what);
    if (decodable) {
        PIKV_REQUIRE((c->bits == 8) == (c->symmetric != 0), PIKV_EUNSUPPORTED, "%s reads int8 symmetric and 4-bit asymmetric caches", what);
        PIKV_REQUIRE(c->bits == 8 || (c->k_zp && c->v_zp), PIKV_EINVAL, "%s: the 4-bit cache needs k_zp and v_zp", what);
    }
    d.page_table = c->page_table;
    d.num_seqs = c->num_seqs; d.max_pages = c->max_pages; d.num_pages = c->num_pages; d.n_kv = c->n_kv; d.bits = c->bits;
    d.k_codes = static_cast<uint8_t*>(c->k_codes); d.v_codes = static_cast<uint8_t*>(c->v_codes);
    d.k_scale = static_cast<uint16_t*>(c->k_scale); d.v_scale = static_cast<uint16_t*>(c->v_scale);
    d.k_zp = static_cast<float*>(c->k_zp); d.v_zp = static_cast<float*>(c->v_zp);
    d.status = c->status;
    return PIKV_OK;
}

#ifdef __CUDACC__
// pre[i] = count(0) + .. + count(i - 1) for i <= n, by one CTA; returns pre[n].  pre holds n + 1 words of shared memory.
template <int THREADS, typename F>
__device__ __forceinline__ int stream_prefix(int n, int* pre, F count) {
    __shared__ int totals[THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (n + THREADS - 1) / THREADS, lo = min(n, tid * per), hi = min(n, lo + per);
    int sum = 0;
    for (int i = lo; i < hi; ++i) {
        const int c = count(i);
        pre[i + 1] = c;
        sum += c;
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
    }
    if (lane == 31) totals[warp] = inc;
    if (tid == 0) pre[0] = 0;
    __syncthreads();
    int run = inc - sum;
    for (int w = 0; w < warp; ++w) run += totals[w];
    for (int i = lo; i < hi; ++i) {
        run += pre[i + 1];
        pre[i + 1] = run;
    }
    __syncthreads();
    return pre[n];
}
// the stream that item f of the list belongs to: pre[i] <= f < pre[i + 1]
__device__ __forceinline__ int stream_of(const int* pre, int n, int f) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pre[mid] <= f) lo = mid; else hi = mid - 1;
    }
    return lo;
}
// page-table row of stream i of the call, or -1 for an id outside the cache
__device__ __forceinline__ int stream_row(const CacheDev& c, const int* seq_ids, int i) {
    const int seq = seq_ids ? __ldg(seq_ids + i) : i;
    return seq >= 0 && seq < c.num_seqs ? seq : -1;
}
// physical page of a logical one; `none` and a status bit where the table holds none
__device__ __forceinline__ int stream_page(const CacheDev& c, int row, int page, int none = 0) {
    const int p = page < c.max_pages ? __ldg(c.page_table + (size_t)row * c.max_pages + page) : -1;
    if (p >= 0 && p < c.num_pages) return p;
    if (c.status) atomicOr(c.status, PIKV_ST_BAD_PAGE);
    return none;
}

// The smallest power of two p >= 2^-126 with a <= 127 p, as its exponent; a finite and >= 0.  127 / 128 = 0x7e0000 of the
// mantissa: a = f 2^x with f in [0.5, 1) fits 127 steps of 2^(x - 7) when f <= 127 / 128.
__device__ __forceinline__ int step_exponent(float a) {
    const uint32_t u = __float_as_uint(a);
    const int x = (int)(u >> 23) - 126;
    return max(-126, x - 7 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0));
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 <= e <= 127
#endif

}  // namespace pikv
