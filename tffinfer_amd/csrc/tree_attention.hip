// Attention of trees of drafted tokens over the paged cache.  A request brings n nodes, whose keys and values lie in its pages behind
// its start_pos cached tokens, node j at place start_pos + j.  Node i sees the cached places and the nodes whose bit its row of
// `ancestors` has:
//   o_i = sum_j e^(s_ij - m) v_j / (sum_j e^(s_ij - m) [+ e^(sink - m)]),   s_ij = (q_i . k_j) scale  [s <- c tanh(s / c)]
// over the visible places j; under a window of w only the last w of them in the order of their places.  A node that sees nothing gets zeros.
// The reference has one row of a causal mask per token (src/kernel/cuda/mask_op.cu:37-43) and no trees.
#include "common.h"
#include "tffinfer_kernels.h"

#define TREE_WORDS 8                 // words of 32 bits a row of ancestors has at most: 256 nodes
#define TREE_MAX_D 512

// The request that row t belongs to, the same in every lane: as many of cu[1 .. n] as are not behind t (n: to none).
__device__ __forceinline__ int tree_row_request(const int32_t* __restrict__ cu, int n, int t) {
    int upto = 0;
    for (int r0 = 0; r0 < n; r0 += 64) {
        const int r = r0 + (int)(threadIdx.x & 63);
        upto += __popcll(__ballot(r < n && cu[min(r, n - 1) + 1] <= t));
    }
    return upto;
}

// What a node sees of its tree (bits of nodes that the request has not are dropped, and under a window the first ones), and the first cached place.
struct TreeRow {
    uint32_t bits[TREE_WORDS];
    int lo;
};
__device__ __forceinline__ TreeRow tree_row(const int32_t* __restrict__ row, int words, int nodes, int start, int window) {
    TreeRow t;
    int count = 0;
#pragma unroll
    for (int w = 0; w < TREE_WORDS; ++w) {
        const int left = nodes - 32 * w;
        t.bits[w] = w < words && left > 0 ? (uint32_t)row[w] & (left >= 32 ? ~0u : (1u << left) - 1) : 0u;
        count += __popc(t.bits[w]);
    }
    t.lo = 0;
    if (window > 0) {
        t.lo = max(0, min(start, start + count - window));
        int drop = count - window;           // the window ends among the nodes
#pragma unroll
        for (int w = 0; w < TREE_WORDS; ++w)
            while (drop > 0 && t.bits[w]) {
                t.bits[w] &= t.bits[w] - 1;
                --drop;
            }
    }
    return t;
}

// ---- any head size, page size and type: a wave per (node, q head), keys 64 at a time, one a lane ----
// The yardstick, and what sizes run on that the matrix cores' kernel does not take.
template <typename T>
__global__ __launch_bounds__(64) void tree_attention_generic_kernel(
    const T* __restrict__ q, int q_stride, T* __restrict__ out, const T* __restrict__ k_cache, const T* __restrict__ v_cache,
    const int32_t* __restrict__ block_tables, int bt_stride, const int32_t* __restrict__ cu_nodes, const int32_t* __restrict__ start_pos,
    const int32_t* __restrict__ ancestors, int words, int R, int rows, int nq, int nkv, int d, int page_size, int num_pages, int window,
    float scale, const float* __restrict__ sinks, float softcap) {
    __shared__ float qs[TREE_MAX_D];
    __shared__ long long voff[64];
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, g = h / (nq / nkv);
    const int r = tree_row_request(cu_nodes, R, t);
    if (r >= R) return;                          // (a row behind the last node is left as it is)
    const int nodes = min(cu_nodes[r + 1], rows) - max(cu_nodes[r], 0);
    const long long room = (long long)bt_stride * page_size;
    const int start = (int)min((long long)max(start_pos[r], 0), room), end = (int)min((long long)start + min(nodes, 32 * words), room);
    const TreeRow see = tree_row(ancestors + (size_t)t * words, words, end - start, start, window);
    const T* qp = q + (size_t)t * q_stride + (size_t)h * d;
    for (int e = lane; e < d; e += 64) qs[e] = to_f32(qp[e]);
    __syncthreads();

    float m = -INFINITY, l = 0.f;
    float acc[TREE_MAX_D / 64];
#pragma unroll
    for (int i = 0; i < TREE_MAX_D / 64; ++i) acc[i] = 0.f;
    const int32_t* bt = block_tables + (size_t)r * bt_stride;
    for (int base = see.lo; base < end; base += 64) {
        const int j = base + lane;
        bool valid = j < start;
        if (!valid && j < end) {
#pragma unroll
            for (int w = 0; w < TREE_WORDS; ++w)
                if (w == (j - start) >> 5) valid = (see.bits[w] >> ((j - start) & 31)) & 1;
        }
        float s = -INFINITY;
        long long off = 0;
        if (valid) {
            int page = bt[j / page_size];
            if (page < 0 || page >= num_pages) page = 0;
            const long long head_base = ((long long)page * nkv + g) * page_size * d;
            off = head_base + (j % page_size);   // values: [element][slot]
            const T* kp = k_cache + head_base + (long long)(j % page_size) * d;
            float dot = 0.f;
            for (int e = 0; e < d; ++e) dot = fmaf(qs[e], to_f32(kp[e]), dot);
            s = dot * scale;
            if (softcap > 0.f) s = softcap * tanhf(s / softcap);
        }
        __syncthreads();                         // earlier readers of voff are done
        voff[lane] = off;
        const unsigned long long live = __ballot(valid);
        const float m_new = fmaxf(m, wave_max(s));
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        const float p = valid ? expf(s - ref) : 0.f;
        const float corr = expf(m - ref);        // 0 before the first key
        l = l * corr + wave_sum(p);
        m = m_new;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TREE_MAX_D / 64; ++i) acc[i] *= corr;
        for (unsigned long long left = live; left; left &= left - 1) {
            const int jj = __ffsll((long long)left) - 1;
            const float pj = __shfl(p, jj, 64);
            const T* vp = v_cache + voff[jj];
#pragma unroll
            for (int i = 0; i < TREE_MAX_D / 64; ++i) {
                const int e = lane + 64 * i;
                if (e < d) acc[i] = fmaf(pj, to_f32(vp[(long long)e * page_size]), acc[i]);
            }
        }
    }
    T* op = out + ((size_t)t * nq + h) * d;
    if (sinks) {                                 // one more term in the denominator, with no key and no value
        const float ref = m == -INFINITY ? sinks[h] : m;
        l += expf(sinks[h] - ref);
    }
    const float inv = l > 0.f ? 1.0f / l : l != l ? l : 0.f;
#pragma unroll
    for (int i = 0; i < TREE_MAX_D / 64; ++i) {
        const int e = lane + 64 * i;
        if (e < d) op[e] = from_f32<T>(acc[i] * inv);
    }
}

TFF_API int tff_tree_attention(const void* q, int q_stride, void* out, const void* k_cache, const void* v_cache, const int32_t* block_tables,
                               int bt_stride, const int32_t* cu_nodes, const int32_t* start_pos, const int32_t* ancestors, int words, int R,
                               int rows, int nq, int nkv, int d, int page_size, int num_pages, int window, float scale, const float* sinks,
                               float softcap, int dtype, tff_stream_t stream) {
    TFF_REQUIRE(rows >= 0 && R >= 0, "tree_attention: bad sizes rows=%d requests=%d", rows, R);
    TFF_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "tree_attention: %d query heads are not a multiple of %d key heads", nq, nkv);
    TFF_REQUIRE(nq <= 65535, "tree_attention: too many heads");
    TFF_REQUIRE(d > 0 && d <= TREE_MAX_D, "tree_attention: head size %d not supported (1..%d)", d, TREE_MAX_D);
    TFF_REQUIRE(page_size > 0 && num_pages > 0 && bt_stride > 0 && window >= 0 && softcap >= 0.f,
                "tree_attention: bad cache geometry page_size=%d pages=%d table stride=%d window=%d", page_size, num_pages, bt_stride, window);
    TFF_REQUIRE(words > 0 && words <= TREE_WORDS, "tree_attention: ancestors of %d words (1..%d)", words, TREE_WORDS);
    TFF_REQUIRE(q_stride >= nq * d, "tree_attention: query row stride %d below %d", q_stride, nq * d);
    TFF_REQUIRE(dtype == TFF_F32 || dtype == TFF_BF16, "tree_attention: unknown dtype %d", dtype);
    if (rows == 0 || R == 0) return 0;
    TFF_REQUIRE(q && out && k_cache && v_cache && block_tables && cu_nodes && start_pos && ancestors, "tree_attention: null pointer");
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid(rows, nq);
#define TFF_TREE(TT)                                                                                                                       \
    tree_attention_generic_kernel<TT><<<grid, 64, 0, s>>>((const TT*)q, q_stride, (TT*)out, (const TT*)k_cache, (const TT*)v_cache,       \
                                                          block_tables, bt_stride, cu_nodes, start_pos, ancestors, words, R, rows, nq, nkv, d, \
                                                          page_size, num_pages, window, scale, sinks, softcap)
    if (dtype == TFF_F32) TFF_TREE(float);
    else TFF_TREE(bf16_t);
#undef TFF_TREE
    return tff_check_launch("tree_attention");
}
