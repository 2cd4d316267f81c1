// After a step over trees of drafted tokens: which of them the model agrees with, and their keys and values to the places they have
// from then on.  The reference generates token by token and has neither (src/core/runtime/InferRuntime.cu:415-429).
#include "common.h"
#include "tffinfer_kernels.h"

// ---- the walk ----
// From node 0 (the token the request already had) on: to the first child whose token is what the model chose after the node, until no
// child is or `max_path` nodes are kept.  A node's parent is the last node that it sees before itself.  A wave a request: a lane
// has the nodes lane, lane + 64, ..., and a level is a comparison and a ballot.  Bound by latency: two loads after each other, then
// registers.
#define TREE_WORDS 8                 // words of 32 bits a row of ancestors has at most: 256 nodes

__global__ __launch_bounds__(64) void tree_accept_kernel(const int32_t* __restrict__ choices, const int32_t* __restrict__ tokens,
                                                         const int32_t* __restrict__ cu_nodes, const int32_t* __restrict__ ancestors,
                                                         int words, int T, int max_path, int32_t* __restrict__ path,
                                                         int32_t* __restrict__ counts, int32_t* __restrict__ next) {
    constexpr int PER = TREE_WORDS / 2;
    const int r = blockIdx.x, lane = threadIdx.x;
    const int n0 = max(cu_nodes[r], 0), n = min(min(cu_nodes[r + 1], T) - n0, 32 * words);
    int token[PER], choice[PER], parent[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = lane + 64 * k;
        parent[k] = -1;
        token[k] = choice[k] = 0;
        if (i < n) {
            token[k] = tokens[n0 + i];
            choice[k] = choices[n0 + i];
            for (int w = 0; w <= (i >> 5); ++w) {
                uint32_t bits = (uint32_t)ancestors[(size_t)(n0 + i) * words + w];
                if (w == (i >> 5)) bits &= (1u << (i & 31)) - 1;
                if (bits) parent[k] = 32 * w + 31 - __clz((int)bits);
            }
        }
    }
    int at = n > 0 ? 0 : -1, kept = 0, want = -1;
    while (at >= 0) {
        if (lane == 0) path[(size_t)r * max_path + kept] = at;
        ++kept;
        int found = -1;
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (k == at >> 6) want = __shfl(choice[k], at & 63, 64);
        if (kept < max_path) {
#pragma unroll
            for (int k = PER - 1; k >= 0; --k) {
                const unsigned long long hit = __ballot(parent[k] == at && token[k] == want);
                if (hit) found = 64 * k + __ffsll((long long)hit) - 1;
            }
        }
        at = found;                  // (a child lies behind its parent, so the walk ends)
    }
    for (int i = kept + lane; i < max_path; i += 64) path[(size_t)r * max_path + i] = -1;
    if (lane == 0) {
        counts[r] = kept;
        next[r] = want;
    }
}

TFF_API int tff_tree_accept(const int32_t* choices, const int32_t* tokens, const int32_t* cu_nodes, const int32_t* ancestors, int words, int T,
                            int R, int max_path, int32_t* path, int32_t* counts, int32_t* next, tff_stream_t stream) {
    TFF_REQUIRE(T >= 0 && R >= 0 && max_path > 0, "tree_accept: bad sizes nodes=%d requests=%d path=%d", T, R, max_path);
    TFF_REQUIRE(words > 0 && words <= TREE_WORDS, "tree_accept: ancestors of %d words (1..%d)", words, TREE_WORDS);
    if (R == 0) return 0;
    TFF_REQUIRE(cu_nodes && path && counts && next && (T == 0 || (choices && tokens && ancestors)), "tree_accept: null pointer");
    tree_accept_kernel<<<R, 64, 0, (hipStream_t)stream>>>(choices, tokens, cu_nodes, ancestors, words, T, max_path, path, counts, next);
    return tff_check_launch("tree_accept");
}

// ---- the move ----
// For request r and i < counts[r]: the key and value at place start_pos[r] + path[r, i] of its pages to place start_pos[r] + i, in all
// caches of the call.  A block has one head's keys, or values, of one request and cache: it loads all that moves into LDS before it stores
// any of it, so a place may be both a source and a target, whatever the path.  Values lie transposed ([element][place]): their
// moves are elements, not rows.
#define KEEP_CACHES 64               // caches a launch takes: their pointers are its arguments
#define KEEP_PATH 256                // kept places of a request, at most
#define KEEP_LDS 32768               // bytes a block stages

struct KeepCaches {
    void *k[KEEP_CACHES], *v[KEEP_CACHES];
};

template <typename E>
__global__ __launch_bounds__(256) void cache_keep_kernel(const KeepCaches caches, const int32_t* __restrict__ block_tables, int bt_stride,
                                                         const int32_t* __restrict__ start_pos, const int32_t* __restrict__ path,
                                                         const int32_t* __restrict__ counts, int max_path, int nkv, int d, int page_size,
                                                         int num_pages) {
    __shared__ long long src[KEEP_PATH], dst[KEEP_PATH];       // places: page * nkv * d * page_size + offset within it
    __shared__ E stage[KEEP_LDS / sizeof(E)];
    __shared__ int moves_n;
    const int r = blockIdx.x, g = blockIdx.y, which = blockIdx.z >> 1, values = blockIdx.z & 1, tid = threadIdx.x;
    const int n = min(max(counts[r], 0), max_path);
    if (tid == 0) moves_n = 0;
    __syncthreads();
    const int s0 = max(start_pos[r], 0);
    const long long room = (long long)bt_stride * page_size;
    for (int i = tid; i < n; i += 256) {
        const int p = path[(size_t)r * max_path + i];
        const long long a = (long long)s0 + p, b = (long long)s0 + i;
        if (p >= 0 && p != i && a < room && b < room) {
            const int pa = block_tables[(size_t)r * bt_stride + a / page_size], pb = block_tables[(size_t)r * bt_stride + b / page_size];
            if (pa >= 0 && pa < num_pages && pb >= 0 && pb < num_pages) {
                const int at = atomicAdd(&moves_n, 1);
                const long long ha = ((long long)pa * nkv + g) * d * page_size, hb = ((long long)pb * nkv + g) * d * page_size;
                const int step = values ? 1 : d;
                src[at] = ha + (a % page_size) * step;
                dst[at] = hb + (b % page_size) * step;
            }
        }
    }
    __syncthreads();
    const int m = moves_n;
    if (m == 0) return;
    E* __restrict__ c = (E*)(values ? caches.v[which] : caches.k[which]);
    const int step = values ? page_size : 1;                   // between a place's elements
    const int slice = min(d, KEEP_LDS / (int)sizeof(E) / m);   // elements of every place that fit
    for (int e0 = 0; e0 < d; e0 += slice) {
        const int w = min(slice, d - e0), total = w * m;
        for (int x = tid; x < total; x += 256) {
            // neighbours: elements of a key, places of a value's element
            const int i = values ? x % m : x / w, e = e0 + (values ? x / m : x - (x / w) * w);
            stage[x] = c[src[i] + (long long)e * step];
        }
        __syncthreads();
        for (int x = tid; x < total; x += 256) {
            const int i = values ? x % m : x / w, e = e0 + (values ? x / m : x - (x / w) * w);
            c[dst[i] + (long long)e * step] = stage[x];
        }
        __syncthreads();
    }
}

TFF_API int tff_cache_keep(void* const* k_caches, void* const* v_caches, int num_caches, const int32_t* block_tables, int bt_stride,
                           const int32_t* start_pos, const int32_t* path, const int32_t* counts, int R, int max_path, int nkv, int d,
                           int page_size, int num_pages, int dtype, tff_stream_t stream) {
    TFF_REQUIRE(R >= 0 && num_caches >= 0 && max_path > 0, "cache_keep: bad sizes requests=%d caches=%d path=%d", R, num_caches, max_path);
    TFF_REQUIRE(max_path <= KEEP_PATH, "cache_keep: paths of %d places (at most %d)", max_path, KEEP_PATH);
    TFF_REQUIRE(nkv > 0 && nkv <= 65535 && d > 0 && page_size > 0 && num_pages > 0 && bt_stride > 0,
                "cache_keep: bad cache geometry heads=%d d=%d page_size=%d pages=%d table stride=%d", nkv, d, page_size, num_pages, bt_stride);
    TFF_REQUIRE(dtype == TFF_F32 || dtype == TFF_BF16, "cache_keep: unknown dtype %d", dtype);
    if (R == 0 || num_caches == 0) return 0;
    TFF_REQUIRE(k_caches && v_caches && block_tables && start_pos && path && counts, "cache_keep: null pointer");
    for (int i = 0; i < num_caches; ++i) TFF_REQUIRE(k_caches[i] && v_caches[i], "cache_keep: null pointer (cache %d)", i);
    for (int c0 = 0; c0 < num_caches; c0 += KEEP_CACHES) {
        const int nc = num_caches - c0 < KEEP_CACHES ? num_caches - c0 : KEEP_CACHES;
        KeepCaches a;
        for (int i = 0; i < KEEP_CACHES; ++i) {
            a.k[i] = i < nc ? k_caches[c0 + i] : nullptr;
            a.v[i] = i < nc ? v_caches[c0 + i] : nullptr;
        }
        const dim3 grid(R, nkv, 2 * nc);
        if (dtype == TFF_F32)
            cache_keep_kernel<uint32_t><<<grid, 256, 0, (hipStream_t)stream>>>(a, block_tables, bt_stride, start_pos, path, counts, max_path, nkv, d,
                                                                               page_size, num_pages);
        else
            cache_keep_kernel<uint16_t><<<grid, 256, 0, (hipStream_t)stream>>>(a, block_tables, bt_stride, start_pos, path, counts, max_path, nkv, d,
                                                                               page_size, num_pages);
        if (int rc = tff_check_launch("cache_keep")) return rc;
    }
    return 0;
}
