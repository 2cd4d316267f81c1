// Attention of trees of drafted tokens over the paged cache.  A request brings n nodes, whose keys and values lie in its pages behind
// its start_pos cached tokens, node j at place start_pos + j.  Node i sees the cached places and the nodes whose bit its row of
// `ancestors` has:
//   o_i = sum_j e^(s_ij - m) v_j / (sum_j e^(s_ij - m) [+ e^(sink - m)]),   s_ij = (q_i . k_j) scale  [s <- c tanh(s / c)]
// over the visible places j; under a window of w only the last w of them in the order of their places.  A node that sees nothing gets zeros.
// The reference has one row of a causal mask per token (src/kernel/cuda/mask_op.cu:37-43) and no trees.
#include "common.h"
#include "mfma_tiles.h"
#include "tffinfer_kernels.h"
#include "tree_attention.h"

#define TREE_MAX_D 512

// ---- any head size, page size and type: a wave per (node, q head), keys 64 at a time, one a lane ----
// The yardstick, and what sizes run on that the matrix cores' kernel does not take.  It reads a kv head's keys and values once per node and q head of
// the group, each lane a key of its own: one request of 300 places and 16 columns 105 us with a head of 80, 152 with one of 192; 8 of 2,048 and 104 columns
// 2,250 (heads of 64 and 128 on the matrix cores: 9.2; 30 and 36).
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
    if (r >= R || t - max(cu_nodes[r], 0) >= 32 * words) return;      // (a row that no request has is left as it is)
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
    if (sinks) l += m == -INFINITY ? 1.f : expf(sinks[h] - m);      // one more term, with no key and no value (nothing seen: zeros, whatever the sink)
    const float inv = l > 0.f ? 1.0f / l : l != l ? l : 0.f;
#pragma unroll
    for (int i = 0; i < TREE_MAX_D / 64; ++i) {
        const int e = lane + 64 * i;
        if (e < d) op[e] = from_f32<T>(acc[i] * inv);
    }
}

// ---- on the matrix cores: bfloat16 and float32, head sizes 64, 128 and 256, pages of a power of two of tokens, at least 8 ----
// The columns of a request and kv head are its (node, q head of the group) pairs, node * G + head, in groups of 16 CT.  The work
// is cut into slices of keys (32 in bfloat16, 16 in float32) of one group of columns; every block finds out by itself, from the
// requests' tables, which run of them is its own (an equal share of their weights, consecutive: the slices of a group of columns, then the next
// group's, then the next request's), so that blocks end together whatever the requests' lengths, nothing is planned on the host and a
// captured launch serves any lengths.  The four waves of a block take every fourth slice, with all the block's columns in
// registers: a key or value goes from memory into the registers of one wave and into no other, no LDS and no barrier in the loop.  S^T = K Q^T
// and O^T = V^T P^T: a lane's scores, weights and outputs all belong to column lane % 16, and with the keys in the order below the
// scores' registers are the second product's operand as they lie.  The maximum that the exponentials are taken against follows the true one
// when that is more than 2^8 ahead: the outputs are rescaled some times a run, not at every slice.  At a run's end the four waves meet in LDS; a
// group of columns whose slices went to several blocks leaves a partial result with each, merged by a second kernel.
// What bounds it: a few slices are latency, some 4.5 us until a run's first keys are there (tables, pages, keys) and 1.5 for every slice that a wave has
// (one request and 16 columns: 40 places, a slice a wave, 6.0 us, 150 7.4, 300 9.2, 480 10.8); many are the memory (4 requests of 32,000 places and 32
// columns, 524 MB: 102 us and a merge of 7, 4.8 TB/s).  float32 runs at its own MFMAs' rate, 2 us a slice and wave.
typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 tree_bf16x8;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float tree_f32x4;
typedef __attribute__((__vector_size__(4 * sizeof(uint32_t)))) uint32_t tree_u32x4;

#define TREE_LAG 8.0f                // log2 of what the running maximum may be behind

template <typename T, int D>
struct TreeMath;
template <int D>
struct TreeMath<bf16_t, D> {
    static constexpr int SLICE = 32, TILES = 2, PER = 8;     // keys of a slice, score tiles, elements of a 16-byte load
    static constexpr int QF = D / 32, KF = 2 * QF, VF = D / 16;
    typedef tree_bf16x8 frag;
    // scores of tile t (rows 4 kg + e: keys 8 kg + 4 t + e of the slice)
    static __device__ __forceinline__ tree_f32x4 scores(const frag (&k)[KF], const frag (&q)[QF], int t) {
        tree_f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int f = 0; f < QF; ++f) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[t * QF + f], q[f], s, 0, 0, 0);
        return s;
    }
    // c tanh(x / c) = c (1 - e) / (1 + e), e = e^(-2 |x| / c): off by about half a step of c, whatever the score; for caps of some ten to a hundred less
    // than a weight's rounding by far, as the attention of decoding has it in bfloat16
    static __device__ __forceinline__ float capped(float x, float cap) {
        const float e = __builtin_amdgcn_exp2f(-fabsf(x) * (2.f * 1.4426950408889634f / cap));
        return copysignf(cap * (1.f - e) / (1.f + e), x);
    }
    // A weight as the product takes it: rounded to bfloat16, half a step of 2^-8.  The sum of the weights is that of the rounded ones, so that a dominant
    // weight's rounding cancels.
    static __device__ __forceinline__ float weight(float x) { return (float)(bf16_t)x; }
    static __device__ __forceinline__ void add(tree_f32x4 (&o)[D / 16], const frag (&v)[VF], const float (&p)[4 * TILES]) {
        frag w;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = (bf16_t)p[i];       // (they are bfloat16 numbers)
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[dt], w, o[dt], 0, 0, 0);
    }
    // where a lane's row of key fragment f lies: (key of the slice, element)
    static __device__ __forceinline__ int key_row(int f, int qc) { return 8 * (qc >> 2) + 4 * (f / QF) + (qc & 3); }
    static __device__ __forceinline__ int key_elem(int f, int kg) { return (f % QF) * 32 + kg * 8; }
    static __device__ __forceinline__ int key_block(int qc) { return qc >> 2; }      // the eight keys it is among
    static __device__ __forceinline__ int value_key(int kg) { return 8 * kg; }       // first key of a lane's values
    // Zeros in the elements whose bit `live` has not; the bits of those left that are not finite come back.
    static __device__ __forceinline__ uint32_t clean(frag (&v)[VF], uint32_t live) {
        uint32_t keep[4], bad[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            keep[w] = ((live >> (2 * w)) & 1 ? 0xffffu : 0u) | ((live >> (2 * w + 1)) & 1 ? 0xffff0000u : 0u);
            bad[w] = 0;
        }
#pragma unroll
        for (int dt = 0; dt < VF; ++dt) {
            tree_u32x4 x = __builtin_bit_cast(tree_u32x4, v[dt]);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                x[w] &= keep[w];
                bad[w] |= (x[w] & 0x7f807f80u) + 0x00800080u;        // (bit 15 of a half: its exponent is all ones)
            }
            v[dt] = __builtin_bit_cast(frag, x);
        }
        uint32_t odd = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) odd |= (((bad[w] >> 15) & 1) | ((bad[w] >> 30) & 2)) << (2 * w);
        return odd;
    }
    static __device__ __forceinline__ void only_finite(frag (&v)[VF]) {
#pragma unroll
        for (int dt = 0; dt < VF; ++dt) {
            tree_u32x4 x = __builtin_bit_cast(tree_u32x4, v[dt]);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                if ((x[w] & 0x7f80u) == 0x7f80u) x[w] &= 0xffff0000u;
                if ((x[w] & 0x7f800000u) == 0x7f800000u) x[w] &= 0xffffu;
            }
            v[dt] = __builtin_bit_cast(frag, x);
            __builtin_amdgcn_sched_barrier(0);                       // (one after the other: no registers for all of them)
        }
    }
};
template <int D>
struct TreeMath<float, D> {
    static constexpr int SLICE = 16, TILES = 1, PER = 4;
    static constexpr int QF = D / 16, KF = QF, VF = D / 16;
    typedef tree_f32x4 frag;
    static __device__ __forceinline__ tree_f32x4 scores(const frag (&k)[KF], const frag (&q)[QF], int) {
        tree_f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int f = 0; f < QF; ++f)
#pragma unroll
            for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[f][e], q[f][e], s, 0, 0, 0);
        return s;
    }
    static __device__ __forceinline__ float capped(float x, float cap) { return cap * tanhf(x / cap); }      // (a few steps of the score)
    static __device__ __forceinline__ float weight(float x) { return x; }
    static __device__ __forceinline__ void add(tree_f32x4 (&o)[D / 16], const frag (&v)[VF], const float (&p)[4 * TILES]) {
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[dt][e], p[e], o[dt], 0, 0, 0);
    }
    static __device__ __forceinline__ int key_row(int, int qc) { return qc; }
    static __device__ __forceinline__ int key_elem(int f, int kg) { return f * 16 + kg * 4; }
    static __device__ __forceinline__ int key_block(int qc) { return qc >> 3; }
    static __device__ __forceinline__ int value_key(int kg) { return 4 * kg; }
    static __device__ __forceinline__ uint32_t clean(frag (&v)[VF], uint32_t live) {
        bool bad[4] = {false, false, false, false};
#pragma unroll
        for (int dt = 0; dt < VF; ++dt)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                if (!((live >> w) & 1)) v[dt][w] = 0.f;
                bad[w] |= !(fabsf(v[dt][w]) < INFINITY);
            }
        return (bad[0] ? 1u : 0u) | (bad[1] ? 2u : 0u) | (bad[2] ? 4u : 0u) | (bad[3] ? 8u : 0u);
    }
    static __device__ __forceinline__ void only_finite(frag (&v)[VF]) {
#pragma unroll
        for (int dt = 0; dt < VF; ++dt)
#pragma unroll
            for (int w = 0; w < 4; ++w) v[dt][w] = fabsf(v[dt][w]) < INFINITY ? v[dt][w] : 0.f;
    }
};

template <typename T, int D, int CT, int OCC>
__global__ __launch_bounds__(256, OCC) void tree_attention_kernel(const TreeArgs a) {
    typedef TreeMath<T, D> M;
    typedef typename M::frag frag;
    constexpr int COLS = 16 * CT, SLICE = M::SLICE, KEYS = 4 * M::TILES, LD = D + 4;
    __shared__ __attribute__((aligned(16))) float merge_o[4 * COLS * LD];    // a wave's outputs, [column][D] (4 more: banks)
    __shared__ float merge_m[4 * COLS], merge_l[4 * COLS];
    __shared__ uint32_t see[COLS * (TREE_WORDS + 1)];                        // the columns' bits, and a word of zeros
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), qc = lane & 15, kg = lane >> 4;
    const int G = a.nq / a.nkv;
    int b, g;
    tree_place(a.nkv, b, g);
    if (b >= a.blocks) return;
    const size_t page_stride = (size_t)a.nkv * a.page_size * D;
    const T* __restrict__ kc = (const T*)a.k_cache + (size_t)g * a.page_size * D;
    const T* __restrict__ vc = (const T*)a.v_cache + (size_t)g * a.page_size * D;
    const float log2e = 1.4426950408889634f;

    // the block's run of units, and the request that it begins in
    const TreeRun run = tree_run<SLICE, COLS>(a, b);
    const int x1 = run.x1;
    if (run.x0 >= x1) return;
    int r = run.r, before = run.before;
    TreeRequest t = run.t;

    for (int x = run.x0; x < x1;) {
        if (x >= before + tree_cost<SLICE, COLS>(t)) {
            before += tree_cost<SLICE, COLS>(t);
            t = tree_request<SLICE, COLS>(a, ++r);
            continue;
        }
        const int group = (x - before) / (tree_begin<SLICE, COLS>() + t.slices * tree_weight<COLS>(COLS));
        const TreeGroup<SLICE, COLS> span(t, before, group);
        const int s0 = span.slice(x), s1 = x1 < span.end() ? span.slice(x1) : t.slices;
        x = span.end();
        if (s0 >= s1) continue;          // (another block has it)
        const int ncols = min(COLS, t.nodes * G - group * COLS);
        const int32_t* __restrict__ bt = a.block_tables + (size_t)r * a.bt_stride;

        // places of slice s that a lane loads from: pages two slices ahead, so that no load of a page number waits behind keys and values
        const int last_block = (max(t.end, 1) - 1) >> 3;         // blocks of eight places lie in one page
        auto place = [&](int s, int block) { return min(((t.first + s * SLICE) >> 3) + block, last_block) << 3; };
        auto page_of = [&](int at) {
            const int p = bt[at >> a.page_shift];
            return (unsigned)p < (unsigned)a.num_pages ? p : 0;
        };
        auto slot_of = [&](int at) { return at & (a.page_size - 1); };
        const int kb = M::key_block(qc), vb = M::value_key(kg) >> 3;
        frag k[M::KF], v[M::VF];
        auto load_k = [&](int s, int page) {
            const int at = place(s, kb);
            const T* p = kc + (size_t)page * page_stride + (size_t)slot_of(at) * D;
#pragma unroll
            for (int f = 0; f < M::KF; ++f) k[f] = *reinterpret_cast<const frag*>(p + (M::key_row(f, qc) & 7) * D + M::key_elem(f, kg));
        };
        auto load_v = [&](int s, int page) {
            const int at = place(s, vb) + (M::value_key(kg) & 7);
            const T* p = vc + (size_t)page * page_stride + slot_of(at) + (size_t)qc * a.page_size;
#pragma unroll
            for (int dt = 0; dt < M::VF; ++dt) {
                v[dt] = *reinterpret_cast<const frag*>(p);
                p += 16 * a.page_size;
            }
        };

        // The first slice's page numbers, the queries and the columns' bits are asked for together, then the keys and values; the rest of what a run
        // begins with is done while they travel.
        int s = s0 + wv;
        const int pk0 = page_of(place(s, kb)), pv0 = page_of(place(s, vb));
        int pk = page_of(place(s + 4, kb)), pv = page_of(place(s + 4, vb));
        frag q[CT][M::QF];
        int lo[CT], lo_least = t.end, lo_most = 0;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            const int c = min(ct * 16 + qc, ncols - 1) + group * COLS, node = c / G, head = g * G + (c - node * G);
            const T* qp = (const T*)a.q + (size_t)(t.n0 + node) * a.q_stride + (size_t)head * D;
#pragma unroll
            for (int f = 0; f < M::QF; ++f) q[ct][f] = *reinterpret_cast<const frag*>(qp + M::key_elem(f, kg));
            lo[ct] = 0;
        }
        static_assert(COLS <= 64, "a lane a column");
        const TreeRow row = tree_row(a.ancestors + (size_t)(t.n0 + (min(lane, ncols - 1) + group * COLS) / G) * a.words, a.words, t.end - t.start,
                                     t.start, a.window);
        if (s < s1) {
            load_k(s, pk0);
            load_v(s, pv0);
        }
        __syncthreads();                 // (the run before is merged)
        if (tid < COLS) {
#pragma unroll
            for (int w = 0; w < TREE_WORDS; ++w) see[tid * (TREE_WORDS + 1) + w] = row.bits[w];
            see[tid * (TREE_WORDS + 1) + TREE_WORDS] = 0;
        }
        __syncthreads();
        if (a.window > 0) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                lo[ct] = __shfl(row.lo, ct * 16 + qc, 64);
                lo_least = min(lo_least, lo[ct]);
                lo_most = max(lo_most, lo[ct]);
            }
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) {
                lo_least = min(lo_least, __shfl_xor(lo_least, o, 64));
                lo_most = max(lo_most, __shfl_xor(lo_most, o, 64));
            }
            lo_least = __builtin_amdgcn_readfirstlane(lo_least);
            lo_most = __builtin_amdgcn_readfirstlane(lo_most);
        } else {
            lo_least = 0;
        }

        tree_f32x4 o[CT][D / 16];
        float m[CT], l[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            m[ct] = -INFINITY;
            l[ct] = 0.f;
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt) o[ct][dt] = tree_f32x4{0.f, 0.f, 0.f, 0.f};
        }

        // which of the places key, key + 1, ... column ct * 16 + qc sees: a bit each (the next 8 of them hold)
        auto visible = [&](int ct, int key) {
            const int j = key - t.start;
            const uint32_t* row = see + (ct * 16 + qc) * (TREE_WORDS + 1);
            if (j >= 0) {
                const int w = min(j >> 5, TREE_WORDS - 1);
                return j < 32 * TREE_WORDS ? __funnelshift_r(row[w], row[w + 1], j & 31) : 0u;
            }
            const int cached = min(-j, 31), below = min(max(lo[ct] - key, 0), 31);
            return (((1u << cached) - 1) & (~0u << below)) | (-j < 32 ? row[0] << -j : 0u);
        };

        // A slice's keys are asked for as soon as the slice before is multiplied, its values as soon as that one's are: either is on its way while
        // the wave works on the other, in one set of registers.
        for (; s < s1; s += 4) {
            const int k0 = t.first + s * SLICE;
            const bool masked = k0 + SLICE > t.start || k0 < lo_most;
            const int pk2 = page_of(place(s + 8, kb)), pv2 = page_of(place(s + 8, vb));
            float p[CT][KEYS];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int tile = 0; tile < M::TILES; ++tile) {
                    const tree_f32x4 sc = M::scores(k, q[ct], tile);
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[ct][4 * tile + e] = sc[e];
                }
            if (s + 4 < s1) load_k(s + 4, pk);
            if (a.softcap > 0.f) {
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                    for (int i = 0; i < KEYS; ++i) p[ct][i] = M::capped(p[ct][i] * a.scale, a.softcap) * log2e;
            } else {
                const float f = a.scale * log2e;
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                    for (int i = 0; i < KEYS; ++i) p[ct][i] *= f;
            }
            if (masked) {
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    const uint32_t sees = visible(ct, k0 + M::value_key(kg));
#pragma unroll
                    for (int i = 0; i < KEYS; ++i)
                        if (!((sees >> i) & 1)) p[ct][i] = -INFINITY;
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                float top = p[ct][0];
#pragma unroll
                for (int i = 1; i < KEYS; ++i) top = fmaxf(top, p[ct][i]);
                top = rows_max(top);
                const bool ahead = top > m[ct] + TREE_LAG;
                if (__any(ahead)) {
                    const float now = ahead ? top : m[ct], f = ahead ? __builtin_amdgcn_exp2f(m[ct] - now) : 1.f;
                    m[ct] = now;
                    l[ct] *= f;
#pragma unroll
                    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[ct][dt][e] *= f;
                }
                const float ref = m[ct] == -INFINITY ? 0.f : m[ct];
#pragma unroll
                for (int i = 0; i < KEYS; ++i) {
                    p[ct][i] = M::weight(__builtin_amdgcn_exp2f(p[ct][i] - ref));
                    l[ct] += p[ct][i];
                }
            }
            if (masked) {
                // Values of places that no column sees: what lies there is anything.  And a value that is not finite may only reach the columns that
                // see it: zero times it would not be zero.  The product takes zeros in their places, and who sees one has it added.
                uint32_t live = 0;
#pragma unroll
                for (int i = 0; i < KEYS; ++i) {
                    const int key = k0 + M::value_key(kg) + i;
                    if (key < t.end && key >= lo_least) live |= 1u << i;
                }
                uint32_t odd = M::clean(v, live) << M::value_key(kg);
                if (__any(odd != 0)) {
                    M::only_finite(v);
#pragma unroll
                    for (int x = 1; x < 64; x <<= 1) odd |= (uint32_t)__shfl_xor((int)odd, x, 64);
                    for (uint32_t left = __builtin_amdgcn_readfirstlane(odd); left; left &= left - 1) {
                        const int key = k0 + __ffs((int)left) - 1;
                        const T* vp = vc + (size_t)page_of(key) * page_stride + slot_of(key) + (size_t)(4 * kg) * a.page_size;
                        uint32_t sees[CT];
#pragma unroll
                        for (int ct = 0; ct < CT; ++ct) sees[ct] = visible(ct, key);
#pragma unroll
                        for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float x = to_f32(*vp);
                                vp += e < 3 ? a.page_size : 13 * a.page_size;
#pragma unroll
                                for (int ct = 0; ct < CT; ++ct)
                                    if ((sees[ct] & 1) && !(fabsf(x) < INFINITY)) o[ct][dt][e] += x;
                                asm volatile("" ::: "memory");       // (one element after the other: no registers for all of them)
                            }
                    }
                }
            }
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) M::add(o[ct], v, p[ct]);
            if (s + 4 < s1) load_v(s + 4, pv);
            pk = pk2;
            pv = pv2;
        }

        // the four waves' results together (addresses from a lane number taken here: not kept in registers through the loop)
        const int lane2 = w4_lane(), qc2 = lane2 & 15, kg2 = lane2 >> 4, tid2 = wv * 64 + lane2;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            const float sum = rows_sum(l[ct]);
            if (kg2 == 0) {
                merge_m[wv * COLS + ct * 16 + qc2] = m[ct];
                merge_l[wv * COLS + ct * 16 + qc2] = sum;
            }
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt)
                *reinterpret_cast<tree_f32x4*>(&merge_o[(wv * COLS + ct * 16 + qc2) * LD + dt * 16 + 4 * kg2]) = o[ct][dt];
        }
        __syncthreads();
        const bool whole = s0 == 0 && s1 == t.slices;
        const size_t part = (((size_t)g * a.blocks + b) * 2 + (s0 == 0 ? 1 : 0)) * COLS;
        for (int i = tid2; i < ncols * (D / 4); i += 256) {
            const int c = i / (D / 4), e = (i - c * (D / 4)) * 4;
            float top = merge_m[c];
#pragma unroll
            for (int w = 1; w < 4; ++w) top = fmaxf(top, merge_m[w * COLS + c]);
            const float ref = top == -INFINITY ? 0.f : top;
            float sum = 0.f;
            tree_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = __builtin_amdgcn_exp2f(merge_m[w * COLS + c] - ref);
                const tree_f32x4 ow = *reinterpret_cast<const tree_f32x4*>(&merge_o[(w * COLS + c) * LD + e]);
                sum += merge_l[w * COLS + c] * f;
#pragma unroll
                for (int z = 0; z < 4; ++z) acc[z] += ow[z] * f;
            }
            if (whole) {
                const int cc = c + group * COLS, node = cc / G, head = g * G + (cc - node * G);
                if (a.sinks) {
                    const float sink = a.sinks[head] * log2e;
                    if (top == -INFINITY) sum = 1.f;         // (nothing seen: zeros)
                    else sum += __builtin_amdgcn_exp2f(sink - top);
                }
                const float inv = sum > 0.f ? 1.0f / sum : sum != sum ? sum : 0.f;
                T* op = (T*)a.out + ((size_t)(t.n0 + node) * a.nq + head) * D + e;
#pragma unroll
                for (int z = 0; z < 4; ++z) op[z] = from_f32<T>(acc[z] * inv);
            } else {
                *reinterpret_cast<tree_f32x4*>(a.part_o + (part + c) * D + e) = acc;
                if (e == 0) {
                    a.part_ml[(part + c) * 2] = top;
                    a.part_ml[(part + c) * 2 + 1] = sum;
                }
            }
        }
    }
}

// The partial results of a group of columns, in the order of the keys: a wave has H q heads of a node, and 8 / H partial results of each on their way
// together.  A wave waits for memory four times one after the other, whatever it merges, so H is 4 where single heads would be more waves than the
// GPU holds twice (874 nodes of 40 heads: 23.6 us with single heads, 18.3 so; 35 nodes of 16: 4.0, and 8).
#define MERGE_HEADS 4
template <typename T, int SLICE, int D, int COLS, int H>
__global__ __launch_bounds__(256) void tree_merge_kernel(const TreeArgs a) {
    constexpr int N = D / 64, J = 8 / H;
    const int row = blockIdx.x, lane = threadIdx.x & 63, G = a.nq / a.nkv;
    const int head0 = (blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * H;
    if (head0 >= a.nq) return;
    // the row's request, the units before it and all of them, in one pass over the tables
    int r = 0, total = 0, before = 0;
    for (int r0 = 0; r0 < a.R; r0 += 64) {
        const TreeRequest t = tree_request<SLICE, COLS>(a, min(r0 + lane, a.R - 1));
        const bool in = r0 + lane < a.R;
        const int u = in ? tree_cost<SLICE, COLS>(t) : 0, incl = tree_wave_scan(u);
        const int behind = __popcll(__ballot(in && a.cu_nodes[min(r0 + lane, a.R - 1) + 1] <= row));
        if (r == r0) {
            if (behind > 0) before += __builtin_amdgcn_readlane(incl, behind - 1);
            r += behind;
        }
        total += __builtin_amdgcn_readlane(incl, 63);
    }
    if (r >= a.R) return;
    const TreeRequest t = tree_request<SLICE, COLS>(a, r);
    const int node = row - t.n0;
    if (node < 0 || node >= t.nodes) return;
    const int share = tree_share(total, a.blocks, a.least);
    const float log2e = 1.4426950408889634f;
    // per head: its first partial result (elements of part_o in units of D), how many, from which on they follow each other
    long long first[H], rest[H];
    int n[H], most = 0, which = -1, b0 = 0, b1 = 0;
#pragma unroll
    for (int k = 0; k < H; ++k) {
        const int head = min(head0 + k, a.nq - 1), g = head / G, col = node * G + head - g * G, group = col / COLS, c = col - group * COLS;
        if (group != which) {
            const TreeGroup<SLICE, COLS> from(t, before, group);
            b0 = from.first_block(share);
            b1 = from.last_block(share);
            which = group;
        }
        const long long base = (long long)g * a.blocks * 2 * COLS + c;
        first[k] = base + ((long long)b0 * 2 + 1) * COLS;
        rest[k] = base + (long long)b0 * 2 * COLS;
        n[k] = head0 + k < a.nq && b0 < b1 ? b1 - b0 + 1 : 0;         // (one block had all of it, and wrote the result)
        most = max(most, n[k]);
    }
    if (most == 0) return;
    auto part_of = [&](int k, int i) { return i == 0 ? first[k] : rest[k] + (long long)i * 2 * COLS; };
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml);
    float top[H], sum[H], acc[H][N];
#pragma unroll
    for (int k = 0; k < H; ++k) {
        top[k] = -INFINITY;
        sum[k] = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[k][i] = 0.f;
    }
    for (int c0 = 0; c0 < most; c0 += 64) {
        // (64 partial results at a time, against the largest reference so far)
        float2 v[H];
        float f[H];
#pragma unroll
        for (int k = 0; k < H; ++k) v[k] = c0 + lane < n[k] ? ml[part_of(k, c0 + lane)] : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int k = 0; k < H; ++k) {
            const float now = fmaxf(top[k], wave_max(v[k].x)), ref = now == -INFINITY ? 0.f : now, old = __builtin_amdgcn_exp2f(top[k] - ref);
            f[k] = __builtin_amdgcn_exp2f(v[k].x - ref);
            sum[k] = sum[k] * old + wave_sum(v[k].y * f[k]);
#pragma unroll
            for (int i = 0; i < N; ++i) acc[k][i] *= old;
            top[k] = now;
        }
        const int m = min(64, most - c0);
        for (int i0 = 0; i0 < m; i0 += J) {
            float o[J][H][N];
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int k = 0; k < H; ++k) {
                    // (past a head's last: the last once more, with a weight of zero)
                    const float* p = a.part_o + part_of(k, min(c0 + i0 + j, max(n[k] - 1, 0))) * D + lane;
#pragma unroll
                    for (int i = 0; i < N; ++i) o[j][k][i] = n[k] > 0 ? p[i * 64] : 0.f;
                }
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int k = 0; k < H; ++k) {
                    const float w = __shfl(f[k], min(i0 + j, 63), 64);
#pragma unroll
                    for (int i = 0; i < N; ++i) acc[k][i] += c0 + i0 + j < n[k] ? o[j][k][i] * w : 0.f;
                }
        }
    }
#pragma unroll
    for (int k = 0; k < H; ++k) {
        if (n[k] == 0) continue;
        if (a.sinks) {
            const float sink = a.sinks[head0 + k] * log2e;
            if (top[k] == -INFINITY) sum[k] = 1.f;
            else sum[k] += __builtin_amdgcn_exp2f(sink - top[k]);
        }
        const float inv = sum[k] > 0.f ? 1.0f / sum[k] : sum[k] != sum[k] ? sum[k] : 0.f;
        T* op = (T*)a.out + ((size_t)row * a.nq + head0 + k) * D;
#pragma unroll
        for (int i = 0; i < N; ++i) op[i * 64 + lane] = from_f32<T>(acc[k][i] * inv);
    }
}

// The launch's shape: column tiles of a block (narrow: all of them in every wave; wide: of each wave), blocks a kv head, units a block
// takes at least; 0 tiles: the general kernel.
struct TreePlan {
    int wide, tiles, blocks, least, columns, weight, begin;
};
static TreePlan tree_plan(int rows, int R, int nq, int nkv, int d, int page_size, int bt_stride, int dtype) {
    TreePlan p{0, 0, 0, 0, 0, 0, 0};
    if (!(d == 64 || d == 128 || d == 256) || page_size < 8 || page_size > 65536 || (page_size & (page_size - 1)) || nkv <= 0 || nq % nkv || R <= 0 || rows <= 0) return p;
    const int cols = (int)(((long long)rows * (nq / nkv) + R - 1) / R);      // a request's columns, on average
    int per_cu = 1;
    if (dtype == TFF_BF16 && tree_wide_tiles(cols, d) > 0) {
        p.wide = 1;
        p.tiles = tree_wide_tiles(cols, d);
        p.columns = 64 * p.tiles;
        p.weight = d == 256 ? tree_weight<128>(128) : tree_weight<256>(256);
        p.begin = tree_begin<32, 256>();
        p.least = 4 * p.weight + p.begin;
    } else {
        p.weight = 1;
        p.tiles = cols <= 16 || d == 256 ? 1 : 2;      // (two tiles of a head of 256 are more than the registers hold)
        p.columns = 16 * p.tiles;
        if (d < 256) per_cu = 2;
        // slices a wave, at least: two where they are quick, one where float32's are not (2 us each).  us with 16 slices a block / 8, one request of 1,500
        // places and 20 columns 19.0 / 15.6, 8 of 1,000 18.4 / 16.0
        p.least = dtype == TFF_F32 ? 4 : 8;
    }
    const int slice = dtype == TFF_F32 ? 16 : 32;
    const long long all = (long long)rows * (nq / nkv), most = (all > R ? all - R : 0) / p.columns + R;      // groups of columns, at most
    const long long units = most * (((long long)bt_stride * page_size + slice - 1) / slice * p.weight + p.begin);
    if (units > 0x3fffffff) return TreePlan{0, 0, 0, 0, 0, 0, 0};                  // (they are counted in 32 bits)
    long long blocks = (long long)tff_device_cus() * per_cu / nkv;
    if (blocks < 1) blocks = 1;
    if (blocks > (units + p.least - 1) / p.least) blocks = (units + p.least - 1) / p.least;
    // Tables of up to 512 places: what one block has whole needs no merge.  us of the kernels, one request and 16 columns, so / on several blocks: 40 places
    // 6.0 / 6.2 + 3.1, 150 7.4 / 7.6 + 3.0, 300 9.1 / 9.1 + 3.2, 480 10.8 / 8.1 + 5.0.  The lengths are the device's, so a wider table has the second
    // form whatever they are: 300 places under a table of 2,560 pages 9.3 + 3.1.
    p.blocks = !p.wide && dtype == TFF_BF16 && units <= 16 ? 1 : (int)blocks;
    return p;
}
TFF_API size_t tff_tree_attention_workspace_bytes(int rows, int R, int nq, int nkv, int d, int page_size, int bt_stride, int dtype) {
    const TreePlan p = tree_plan(rows, R, nq, nkv, d, page_size, bt_stride, dtype);
    return p.tiles ? (size_t)nkv * p.blocks * 2 * p.columns * (d + 2) * 4 : 0;
}

TFF_API int tff_tree_attention(const void* q, int q_stride, void* out, const void* k_cache, const void* v_cache, const int32_t* block_tables,
                               int bt_stride, const int32_t* cu_nodes, const int32_t* start_pos, const int32_t* ancestors, int words, int R,
                               int rows, int nq, int nkv, int d, int page_size, int num_pages, int window, float scale, const float* sinks,
                               float softcap, void* workspace, size_t workspace_bytes, int dtype, tff_stream_t stream) {
    TFF_REQUIRE(rows >= 0 && R >= 0, "tree_attention: bad sizes rows=%d requests=%d", rows, R);
    TFF_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "tree_attention: %d query heads are not a multiple of %d key heads", nq, nkv);
    TFF_REQUIRE(nq <= 65535, "tree_attention: too many heads");
    TFF_REQUIRE(d > 0 && d <= TREE_MAX_D, "tree_attention: head size %d not supported (1..%d)", d, TREE_MAX_D);
    TFF_REQUIRE(page_size > 0 && num_pages > 0 && bt_stride > 0 && window >= 0 && softcap >= 0.f,
                "tree_attention: bad cache geometry page_size=%d pages=%d table stride=%d window=%d", page_size, num_pages, bt_stride, window);
    TFF_REQUIRE(softcap < INFINITY, "tree_attention: a cap of %g (0: none)", (double)softcap);      // (times tanh(0), which is not a number)
    TFF_REQUIRE(words > 0 && words <= TREE_WORDS, "tree_attention: ancestors of %d words (1..%d)", words, TREE_WORDS);
    TFF_REQUIRE(q_stride >= nq * d, "tree_attention: query row stride %d below %d", q_stride, nq * d);
    TFF_REQUIRE(dtype == TFF_F32 || dtype == TFF_BF16, "tree_attention: unknown dtype %d", dtype);
    if (rows == 0 || R == 0) return 0;
    TFF_REQUIRE(q && out && k_cache && v_cache && block_tables && cu_nodes && start_pos && ancestors, "tree_attention: null pointer");
    TFF_REQUIRE((int64_t)bt_stride * page_size < 0x40000000, "tree_attention: tables of %d pages of %d tokens", bt_stride, page_size);
    hipStream_t s = (hipStream_t)stream;
    const int esz = dtype == TFF_F32 ? 4 : 2;
    const uintptr_t q0 = (uintptr_t)q, q1 = q0 + (size_t)rows * q_stride * esz, o0 = (uintptr_t)out, o1 = o0 + (size_t)rows * nq * d * esz;
    TFF_REQUIRE(o1 <= q0 || q1 <= o0, "tree_attention: the output overlaps the queries");      // (a block reads queries after others have written)
    const TreePlan p = tree_plan(rows, R, nq, nkv, d, page_size, bt_stride, dtype);
    const size_t need = tff_tree_attention_workspace_bytes(rows, R, nq, nkv, d, page_size, bt_stride, dtype);
    if (need > 0 && workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0 && ((uintptr_t)q & 15) == 0 &&
        ((size_t)q_stride * esz) % 16 == 0 && ((uintptr_t)k_cache & 15) == 0 && ((uintptr_t)v_cache & 15) == 0 &&
        (!p.wide || ((uintptr_t)out & 7) == 0)) {      // (the kernel of many columns stores 8 bytes at a time)
        int shift = 3;
        for (int i = 3; i < 31; ++i)
            if (page_size == 1 << i) shift = i;
        float* part_o = (float*)workspace;
        const TreeArgs a{q, k_cache, v_cache, out, block_tables, cu_nodes, start_pos, ancestors, sinks, part_o,
                         part_o + (size_t)nkv * p.blocks * 2 * p.columns * d, q_stride, bt_stride, words, R, rows, nq, nkv, page_size, shift,
                         num_pages, window, p.blocks, p.least, scale, softcap};
        const int heads = (int64_t)rows * nq > 2 * 32 * (int64_t)tff_device_cus() ? MERGE_HEADS : 1;      // (a CU holds 32 waves)
        const dim3 merge(rows, (nq + 4 * heads - 1) / (4 * heads));
        // (a block a kv head has every run whole)
#define TFF_TREE_MERGE(TT, SL, D, COLS)                                       \
    do {                                                                      \
        if (p.blocks == 1) return 0;                                          \
        if (heads == 1) tree_merge_kernel<TT, SL, D, COLS, 1><<<merge, 256, 0, s>>>(a); \
        else tree_merge_kernel<TT, SL, D, COLS, MERGE_HEADS><<<merge, 256, 0, s>>>(a);  \
        return tff_check_launch("tree_merge");                                \
    } while (0)
#define TFF_TREE_MM(TT, SL, D, CT, OCC)                                              \
    do {                                                                             \
        tree_attention_kernel<TT, D, CT, OCC><<<tree_grid(nkv, p.blocks), 256, 0, s>>>(a); \
        if (int rc = tff_check_launch("tree_attention")) return rc;                  \
        TFF_TREE_MERGE(TT, SL, D, 16 * CT);                                          \
    } while (0)
        if (p.wide) {
            if (int rc = tree_wide_launch(a, d, s)) return rc;
            if (d == 64) TFF_TREE_MERGE(bf16_t, 32, 64, 256);
            if (d == 128) TFF_TREE_MERGE(bf16_t, 32, 128, 256);
            TFF_TREE_MERGE(bf16_t, 32, 256, 128);
        }
#define TFF_TREE_TILES(TT, SL)                                   \
    do {                                                         \
        if (d == 64 && p.tiles == 1) TFF_TREE_MM(TT, SL, 64, 1, 2);   \
        if (d == 64) TFF_TREE_MM(TT, SL, 64, 2, 2);              \
        if (d == 128 && p.tiles == 1) TFF_TREE_MM(TT, SL, 128, 1, 2); \
        if (d == 128) TFF_TREE_MM(TT, SL, 128, 2, 2);            \
        TFF_TREE_MM(TT, SL, 256, 1, 1);                          \
    } while (0)
        if (dtype == TFF_BF16) TFF_TREE_TILES(bf16_t, 32);
        TFF_TREE_TILES(float, 16);
#undef TFF_TREE_TILES
#undef TFF_TREE_MM
#undef TFF_TREE_MERGE
    }
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
