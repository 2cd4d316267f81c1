// What the kernels of drafted trees' attention share: what a node sees, and how blocks deal the work among themselves.
#pragma once
#include "common.h"

#define TREE_WORDS 8                 // words of 32 bits a row of ancestors has at most: 256 nodes

// The request that row t belongs to, the same in every lane: as many of cu[1 .. n] as are not behind t (n: to none).
__device__ __forceinline__ int tree_row_request(const int32_t* __restrict__ cu, int n, int t) {
    int upto = t < cu[0] ? n : 0;
    for (int r0 = 0; r0 < n; r0 += 64) {
        const int r = r0 + (int)(threadIdx.x & 63);
        upto += __popcll(__ballot(r < n && cu[min(r, n - 1) + 1] <= t));
    }
    return min(upto, n);
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
        const int left = w < words ? nodes - 32 * w : 0;
        t.bits[w] = (uint32_t)row[min(w, words - 1)] & (left >= 32 ? ~0u : left > 0 ? (1u << left) - 1 : 0u);
        count += __popc(t.bits[w]);
    }
    t.lo = 0;
    if (window > 0) {
        t.lo = max(0, min(start, start + count - window));
        for (int drop = count - window; drop > 0; --drop) {      // (the window ends among the nodes)
            bool done = false;
#pragma unroll
            for (int w = 0; w < TREE_WORDS; ++w) {
                const uint32_t x = t.bits[w];
                if (!done && x) {
                    t.bits[w] = x & (x - 1);
                    done = true;
                }
            }
        }
    }
    return t;
}

struct TreeArgs {
    const void *q, *k_cache, *v_cache;
    void* out;
    const int32_t *block_tables, *cu_nodes, *start_pos, *ancestors;
    const float* sinks;
    float *part_o, *part_ml;         // [kv head][block][2][columns][D], [..][columns][2]
    int q_stride, bt_stride, words, R, rows, nq, nkv, page_size, page_shift, num_pages, window, blocks, least;
    float scale, softcap;
};

// What work is dealt by: the weight of a slice of a group of so many columns (wide: a step by its tiles of 64 columns, in ninths of a microsecond;
// narrow: one, whatever the columns), and of what a run takes beside its slices: a pipeline that fills, a partial result.
// (24 requests of 256 to 8,192 places and 24 to 48 nodes of 5 heads: 122 us with all slices and nothing else alike, 112.5 with a begin of 44, 110 with
// 70; 8 requests of 2,048, whose groups are alike: 38.1, 37.1, 36.9, and 42 with 100.)
template <int COLS>
__host__ __device__ constexpr int tree_weight(int columns) { return COLS >= 128 ? 3 + 2 * ((columns + 63) / 64) : 1; }
template <int SLICE, int COLS>
__host__ __device__ constexpr int tree_begin() { return COLS >= 128 ? 70 : 0; }

// One request's share of the work.
struct TreeRequest {
    int n0, nodes, start, end, first;    // its first row, nodes, cached places, places, and the first place that a slice begins with
    int slices, groups, last;            // (the weight of the last group's slices)
};
template <int SLICE, int COLS>
__device__ __forceinline__ TreeRequest tree_request(const TreeArgs& a, int r) {
    TreeRequest t;
    t.n0 = max(a.cu_nodes[r], 0);
    t.nodes = max(0, min(min(a.cu_nodes[r + 1], a.rows) - t.n0, 32 * a.words));
    const long long room = (long long)a.bt_stride * a.page_size;
    t.start = (int)min((long long)max(a.start_pos[r], 0), room);
    t.end = (int)min((long long)t.start + t.nodes, room);
    t.first = a.window > 0 ? max(0, t.start - a.window) / 32 * 32 : 0;
    const int columns = t.nodes * (a.nq / a.nkv);
    t.groups = (columns + COLS - 1) / COLS;
    t.last = tree_weight<COLS>(columns - max(t.groups - 1, 0) * COLS);
    // (a request with nodes has a slice even where its table has no room for them: its rows are written)
    t.slices = t.nodes > 0 ? max(1, (t.end - t.first + SLICE - 1) / SLICE) : 0;
    return t;
}
template <int SLICE, int COLS>
__device__ __forceinline__ int tree_cost(const TreeRequest& t) {
    return t.slices > 0 ? t.groups * tree_begin<SLICE, COLS>() + t.slices * ((t.groups - 1) * tree_weight<COLS>(COLS) + t.last) : 0;
}
// A group of a request: its weight's begin, the weight of a slice, and the first slice of the block whose share begins at x.  A share that would
// begin near the group's begin begins there, and one near its end behind it: what a block takes on for that is less than beginning once more and a
// partial result (float32's slices are too slow for that).  us before / so: 8 requests of 300 places and 20 columns 27.7 / 15.9, 3 of 90 and 80
// columns 29.0 / 17.7, 8 of 2,048 and 104 columns 37.1 / 33.6, 24 ragged ones 111 / 109.
template <int SLICE, int COLS>
struct TreeGroup {
    static constexpr int BEGIN = tree_begin<SLICE, COLS>(), NEAR = COLS >= 128 ? 44 : SLICE == 16 ? 1 : 8;
    int at, weight, slices;
    __device__ __forceinline__ TreeGroup(const TreeRequest& t, int before, int group) {
        at = before + group * (BEGIN + t.slices * tree_weight<COLS>(COLS));
        weight = group == t.groups - 1 ? t.last : tree_weight<COLS>(COLS);
        slices = t.slices;
    }
    __device__ __forceinline__ int end() const { return at + BEGIN + slices * weight; }
    __device__ __forceinline__ int slice(int x) const {
        if (x < at + NEAR) return 0;
        if (x > end() - NEAR) return slices;
        return max(1, (x - at - BEGIN + weight - 1) / weight);
    }
    // the blocks of its first slice and of its last
    __device__ __forceinline__ int first_block(int share) const {
        int b = at / share;
        while ((b + 1) * share < min(end(), at + NEAR)) ++b;
        return b;
    }
    __device__ __forceinline__ int last_block(int share) const {
        int b = (end() - 1) / share;
        while (b * share >= at + NEAR && b * share > end() - NEAR) --b;
        return b;
    }
};
__device__ __forceinline__ int tree_wave_scan(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(v, o, 64);
        if (lane >= o) v += up;
    }
    return v;
}

// The weight of all requests; the same in every lane.
template <int SLICE, int COLS>
__device__ __forceinline__ int tree_total(const TreeArgs& a) {
    int total = 0;
    for (int r0 = 0; r0 < a.R; r0 += 64) {
        const int r = r0 + (int)(threadIdx.x & 63);
        const int u = r < a.R ? tree_cost<SLICE, COLS>(tree_request<SLICE, COLS>(a, r)) : 0;
        total += __builtin_amdgcn_readlane(tree_wave_scan(u), 63);
    }
    return total;
}
// What a block takes: an equal share, and no less than `least` (a block has its loads to wait for before the first slice).
__device__ __forceinline__ int tree_share(int total, int blocks, int least) { return max((total + blocks - 1) / blocks, least); }

// Which run and kv head a block of the launch has: eight runs by eight, within them the kv heads, within a kv head the eight runs.  Blocks go
// to the XCDs in turn, so a run's kv heads are on one XCD and a page of keys is read through one L2 and one address translation.
__device__ __forceinline__ void tree_place(int nkv, int& b, int& g) {
    const int eight = blockIdx.x / (8 * nkv), within = blockIdx.x - eight * (8 * nkv);
    b = eight * 8 + (within & 7);
    g = within >> 3;
}
static inline int tree_grid(int nkv, int blocks) { return nkv * ((blocks + 7) / 8 * 8); }

// Block b's share x0 .. x1 - 1 (it has the slices that begin there), the request that x0 is in and the weight before it; the same in every lane.
struct TreeRun {
    int x0, x1, r, before;
    TreeRequest t;
};
template <int SLICE, int COLS>
__device__ __forceinline__ TreeRun tree_run(const TreeArgs& a, int b) {
    const int lane = threadIdx.x & 63;
    TreeRun run;
    int total = a.R > 64 ? tree_total<SLICE, COLS>(a) : 0;
    run.r = run.before = 0;
    for (int r0 = 0; r0 < a.R; r0 += 64) {
        TreeRequest t = tree_request<SLICE, COLS>(a, min(r0 + lane, a.R - 1));
        const int u = r0 + lane < a.R ? tree_cost<SLICE, COLS>(t) : 0, incl = tree_wave_scan(u), all = __builtin_amdgcn_readlane(incl, 63);
        if (r0 == 0) {
            if (a.R <= 64) total = all;
            const int share = tree_share(total, a.blocks, a.least);
            run.x0 = min(total, b * share);
            run.x1 = min(total, run.x0 + share);
        }
        if (run.before + all <= run.x0) {
            run.before += all;
            continue;
        }
        const int at = __ffsll((long long)__ballot(run.before + incl > run.x0)) - 1;
        run.r = r0 + at;
        run.before += __builtin_amdgcn_readlane(incl - u, at);
        run.t.n0 = __builtin_amdgcn_readlane(t.n0, at);
        run.t.nodes = __builtin_amdgcn_readlane(t.nodes, at);
        run.t.start = __builtin_amdgcn_readlane(t.start, at);
        run.t.end = __builtin_amdgcn_readlane(t.end, at);
        run.t.first = __builtin_amdgcn_readlane(t.first, at);
        run.t.slices = __builtin_amdgcn_readlane(t.slices, at);
        run.t.groups = __builtin_amdgcn_readlane(t.groups, at);
        run.t.last = __builtin_amdgcn_readlane(t.last, at);
        break;
    }
    return run;
}

// tree_attention_wide.hip: column tiles that a wave of it has at most for requests of so many columns (0: it is not for them), and its launch
int tree_wide_tiles(int columns, int d);
int tree_wide_launch(const TreeArgs& a, int d, hipStream_t stream);
