// Attention for a tree of drafted tokens over the paged cache, and the acceptance of one path of it.
//
// Node i of a stream is the cache row at position ctx + i.  Its query sees the ctx rows before the tree and the nodes its
// mask row names: out = sum_t w_t V_t, w = softmax(q . K_t / sqrt(128)) over the seen rows t.
#include "stream_list.cuh"

#include <type_traits>

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
    if (ctx + nodes > most) {                                   // the tree does not fit behind its context
        nodes = most - ctx;
        if (d.c.status) atomicOr(d.c.status, PIKV_ST_BAD_INDEX);
    }
    return ctx;
}

constexpr int TS_THREADS = 128;

// One warp per (stream, node, query head).  Scores: lane = (row of the page, half of the channels); output: lane = 4 channels.
template <int BITS>
__global__ void __launch_bounds__(TS_THREADS) tree_attn_simple_kernel(TreeDev d) {
    __shared__ float qs[TS_THREADS / 32][128];
    dependency_release();
    dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long unit = (long long)blockIdx.x * (TS_THREADS / 32) + warp;
    if (unit >= (long long)d.B * d.N * d.n_q) return;
    const int qh = (int)(unit % d.n_q), node = (int)(unit / d.n_q % d.N), b = (int)(unit / d.n_q / d.N);
    const int h = qh / d.G;
    int row, nodes;
    const int ctx = tree_lengths(d, b, row, nodes);
    if (row < 0 && lane == 0 && d.c.status) atomicOr(d.c.status, PIKV_ST_BAD_SEQ);
    const int total = node < nodes ? ctx + nodes : 0;
    for (int i = lane; i < 128; i += 32) qs[warp][i] = __bfloat162float(d.q[unit * 128 + i]);
    __syncwarp();
    const uint8_t* mask = d.mask + (size_t)b * d.mask_stride + (size_t)node * d.N;
    const int r = lane & 15, half = lane >> 4;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < total; p0 += PIKV_PAGE_TOKENS) {
        const int page = stream_page(d.c, row, p0 / PIKV_PAGE_TOKENS);
        const size_t base = ((size_t)page * d.c.n_kv + h) * PIKV_PAGE_TOKENS;
        const int pos = p0 + r;
        const bool open = pos < ctx || (pos < total && mask[pos - ctx] != 0);
        float s = 0.f;
        if (open) {
            const float ks = bf16_bits_to_f32(d.c.k_scale[base + r]), kz = BITS == 4 ? d.c.k_zp[base + r] : 0.f;
            for (int i = 0; i < 64; ++i) {
                const int c = 64 * half + i;
                float code;
                if (BITS == 8) code = (float)(int8_t)d.c.k_codes[(base + r) * 128 + 16 * ((c >> 4) ^ (r & 7)) + (c & 15)];
                else code = (float)((d.c.k_codes[(base + r) * 64 + 8 * ((c >> 4) ^ (r & 4)) + ((c & 15) >> 1)] >> (4 * (c & 1))) & 15) - kz;
                s += qs[warp][c] * code;
            }
            s *= ks * 0.08838834764831845f;
        }
        s += __shfl_xor_sync(0xffffffffu, s, 16);
        if (!open) s = -INFINITY;
        const float mn = fmaxf(m, warp_max(s)), mu = mn == -INFINITY ? 0.f : mn;
        const float p = expf(s - mu), al = expf(m - mu);
        l = l * al + warp_sum(half ? 0.f : p);
        m = mn;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= al;
        for (int t = 0; t < PIKV_PAGE_TOKENS; ++t) {
            const float w = __shfl_sync(0xffffffffu, p, t);
            if (!__shfl_sync(0xffffffffu, (int)open, t)) continue;
            const float vs = bf16_bits_to_f32(d.c.v_scale[base + t]), vz = BITS == 4 ? d.c.v_zp[base + t] : 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = 4 * lane + i;
                float code;
                if (BITS == 8) code = (float)(int8_t)d.c.v_codes[(base + t) * 128 + 16 * ((c >> 4) ^ (t & 7)) + (c & 15)];
                else code = (float)((d.c.v_codes[(base + t) * 64 + 8 * ((c >> 4) ^ (t & 4)) + ((c & 15) >> 1)] >> (4 * (c & 1))) & 15) - vz;
                o[i] += w * (code * vs);
            }
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;                 // nothing seen: zero; NaN stays NaN
#pragma unroll
    for (int i = 0; i < 4; ++i) d.out[unit * 128 + 4 * lane + i] = __float2bfloat16_rn(o[i] * inv);
    if (lane == 0 && d.lse) d.lse[unit] = l == 0.f ? -INFINITY : m + logf(l);
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
            const int ps = table[(ctx + at) / PIKV_PAGE_TOKENS], pd = ctx + i < most ? table[(ctx + i) / PIKV_PAGE_TOKENS] : -1;
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
    return 16;
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
        const int grid = (int)((d.B * rows + TS_THREADS / 32 - 1) / (TS_THREADS / 32));
        if (c->bits == 8) launch_dependent(tree_attn_simple_kernel<8>, grid, TS_THREADS, 0, static_cast<cudaStream_t>(stream), d);
        else launch_dependent(tree_attn_simple_kernel<4>, grid, TS_THREADS, 0, static_cast<cudaStream_t>(stream), d);
        count_launch(1);
    }
    return check_launch("tree_attn_kernel");
}

extern "C" int pikv_tree_accept(const pikv_paged_cache* c, const int32_t* path, const int32_t* path_len, const int32_t* seq_ids,
                                const int32_t* ctx_len, int32_t B, int32_t depth, int32_t* length, int32_t* new_len, pikv_stream_t stream) {
    AcceptDev d;
    const int rc = cache_dev(c, d.c, "tree_accept", false);
    if (rc != PIKV_OK) return rc;
    PIKV_REQUIRE(path && ctx_len && new_len, PIKV_EINVAL, "tree_accept: null pointer");
    PIKV_REQUIRE(B > 0 && depth > 0 && (seq_ids || B <= c->num_seqs), PIKV_EINVAL, "tree_accept: bad sizes");
    PIKV_REQUIRE(!(seq_ids && ctx_len == length), PIKV_EINVAL, "tree_accept: with seq_ids, ctx_len has an entry per stream of the call");
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
