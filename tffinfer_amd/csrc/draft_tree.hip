// After a step over trees of drafted tokens: which of them the model agrees with, and their keys and values to the places they have
// from then on.  The reference generates token by token and has neither (src/core/runtime/InferRuntime.cu:415-429).
#include "common.h"
#include "tffinfer_kernels.h"
#include "tree_attention.h"

// ---- the walk ----
// From node 0 (the token the request already had) on: to the first child whose token is what the model chose after the node, until no
// child is or `max_path` nodes are kept.  A node's parent is the last node that it sees before itself.  A wave a request: a lane
// has the nodes lane, lane + 64, ..., and a level is a comparison and a ballot.  Bound by latency: two loads after each other, then
// registers (2.2 us for one request of 8 nodes, 3.9 for 64 of up to 64).
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
// caches of the call.  Whoever has an element of a head (eight of them, of a key) has it of all moves, and loads them all before it stores
// any, so a place may be both a source and a target, whatever the path: up to KEEP_FEW moves in a thread's registers, more through LDS.
// Values lie transposed ([element][place]): their moves are elements, 2 bytes of a line of memory each.  Bound by latency (the path, the pages, the
// data: 2.1 us for one request and 28 layers), and for many requests by the values' lines: 32 requests with paths of up to 8 and 8 layers of 8 heads
// of 128 move 4 MB of keys and values and touch some 40; 14 us with all moves through LDS and a block a head, 10.4 so.
#define KEEP_CACHES 64               // caches a launch takes: their pointers are its arguments
#define KEEP_PATH 256                // kept places of a request, at most
#define KEEP_FEW 8
#define KEEP_LDS 32768               // bytes a block stages

struct KeepCaches {
    void* p[2 * KEEP_CACHES];        // keys and values in turn
};
struct KeepArgs {
    const int32_t *block_tables, *start_pos, *path, *counts;
    int bt_stride, max_path, nkv, d, page_size, num_pages;
};

// A request's moves into LDS: offsets within a cache of the places, without head and element.  Returns how many.  `step`: between places.
__device__ __forceinline__ int keep_moves(const KeepArgs& a, int r, int step, long long* src, long long* dst, int* count) {
    const int tid = threadIdx.x;
    if (tid == 0) *count = 0;
    // (the path is asked for before it is known how much of it counts)
    const int n = min(max(a.counts[r], 0), a.max_path), p = tid < a.max_path ? a.path[(size_t)r * a.max_path + tid] : -1;
    const long long s0 = max(a.start_pos[r], 0), from = s0 + p, to = s0 + tid, room = (long long)a.bt_stride * a.page_size;
    __syncthreads();
    if (tid < n && p >= 0 && p != tid && from < room && to < room) {
        const int pf = (int)from / a.page_size, pt = (int)to / a.page_size;
        const int32_t* bt = a.block_tables + (size_t)r * a.bt_stride;
        const int page_from = bt[pf], page_to = bt[pt];
        if (((unsigned)page_from < (unsigned)a.num_pages) & ((unsigned)page_to < (unsigned)a.num_pages)) {      // (both are asked for at once)
            const int at = atomicAdd(count, 1);
            const long long page = (long long)a.nkv * a.d * a.page_size;
            src[at] = page_from * page + ((int)from - pf * a.page_size) * step;
            dst[at] = page_to * page + ((int)to - pt * a.page_size) * step;
        }
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(*count);
}

// `PIECE` of a head for every thread: for keys d / (sizeof PIECE / sizeof E) pieces that lie side by side, for values one element each.
typedef __attribute__((__vector_size__(4 * sizeof(uint32_t)))) uint32_t keep_16;
// (N moves, of which the last is repeated past the m-th: it stores the same once more)
template <int N, typename PIECE, typename E>
__device__ __forceinline__ void keep_few(E* c, const long long* src, const long long* dst, int m, long long at) {
    PIECE x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = *reinterpret_cast<const PIECE*>(c + src[min(i, m - 1)] + at);
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<PIECE*>(c + dst[min(i, m - 1)] + at) = x[i];
}

// A block: 256 pieces of a request's heads in one cache's keys (z even) or values (z odd).
template <typename E>
__global__ __launch_bounds__(256) void cache_keep_kernel(const KeepCaches caches, const KeepArgs a, const int key_piece) {
    __shared__ long long src[KEEP_PATH], dst[KEEP_PATH];
    __shared__ int count;
    extern __shared__ __attribute__((aligned(16))) char room_[];
    E* stage = (E*)room_;
    const int r = blockIdx.x, values = blockIdx.z & 1, tid = threadIdx.x;
    const int piece = values ? 1 : key_piece, pieces = a.nkv * a.d / piece;
    if ((int)blockIdx.y * 256 >= pieces) return;
    const int step = values ? 1 : a.d, m = keep_moves(a, r, step, src, dst, &count);
    if (m == 0) return;
    E* c = (E*)caches.p[blockIdx.z];
    const int p = blockIdx.y * 256 + tid, per_head = a.d / piece;
    const int g = p / per_head, e = (p - g * per_head) * piece;
    const long long head = (long long)g * a.d * a.page_size + (long long)e * (values ? a.page_size : 1);
    if (m <= KEEP_FEW) {
        if (p < pieces) {
            if (piece > 1) {
                if (m <= 2) keep_few<2, keep_16>(c, src, dst, m, head);
                else if (m <= 4) keep_few<4, keep_16>(c, src, dst, m, head);
                else keep_few<KEEP_FEW, keep_16>(c, src, dst, m, head);
            } else {
                if (m <= 2) keep_few<2, E>(c, src, dst, m, head);
                else if (m <= 4) keep_few<4, E>(c, src, dst, m, head);
                else keep_few<KEEP_FEW, E>(c, src, dst, m, head);
            }
        }
        return;
    }
    // many moves: this block's pieces, as many at a time as LDS holds of all moves
    const int mine = min(256, pieces - (int)blockIdx.y * 256) * piece, first = blockIdx.y * 256 * piece;      // elements (head, e) in a row
    const int slice = min(mine, KEEP_LDS / (int)sizeof(E) / m);
    for (int f0 = 0; f0 < mine; f0 += slice) {
        const int w = min(slice, mine - f0), total = w * m;
        auto at = [&](int x, const long long* place) {
            const int i = x % m, f = first + f0 + x / m, h = f / a.d;      // (a value's places are neighbours, and one thread's)
            return place[i] + (long long)h * a.d * a.page_size + (long long)(f - h * a.d) * (values ? a.page_size : 1);
        };
#pragma unroll 1
        for (int x = tid; x < total; x += 256) stage[x] = c[at(x, src)];
        __syncthreads();
#pragma unroll 1
        for (int x = tid; x < total; x += 256) c[at(x, dst)] = stage[x];
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
    TFF_REQUIRE((int64_t)nkv * d <= 65535 * 256, "cache_keep: %d heads of %d are more than a launch takes", nkv, d);
    TFF_REQUIRE((int64_t)bt_stride * page_size <= 0x7fffffff, "cache_keep: tables of %d pages of %d tokens", bt_stride, page_size);
    const KeepArgs args{block_tables, start_pos, path, counts, bt_stride, max_path, nkv, d, page_size, num_pages};
    const int esz = dtype == TFF_F32 ? 4 : 2;
    for (int i = 0; i < num_caches; ++i) TFF_REQUIRE(k_caches[i] && v_caches[i], "cache_keep: null pointer (cache %d)", i);
    for (int c0 = 0; c0 < num_caches; c0 += KEEP_CACHES) {
        const int nc = num_caches - c0 < KEEP_CACHES ? num_caches - c0 : KEEP_CACHES;
        KeepCaches a;
        for (int i = 0; i < KEEP_CACHES; ++i) {
            a.p[2 * i] = i < nc ? k_caches[c0 + i] : nullptr;
            a.p[2 * i + 1] = i < nc ? v_caches[c0 + i] : nullptr;
        }
        bool wide = ((size_t)d * esz) % 16 == 0;      // keys in pieces of 16 bytes
        for (int i = 0; i < nc; ++i) wide = wide && ((uintptr_t)a.p[2 * i] & 15) == 0;
        const int piece = wide ? 16 / esz : 1;
        const dim3 grid(R, (nkv * d + 255) / 256, 2 * nc);
        const int lds = max_path > KEEP_FEW ? KEEP_LDS : 0;
        if (dtype == TFF_F32) cache_keep_kernel<uint32_t><<<grid, 256, lds, (hipStream_t)stream>>>(a, args, piece);
        else cache_keep_kernel<uint16_t><<<grid, 256, lds, (hipStream_t)stream>>>(a, args, piece);
        if (int rc = tff_check_launch("cache_keep")) return rc;
    }
    return 0;
}
