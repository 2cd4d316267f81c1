// bfloat16 attention of drafted trees for requests of many columns (node, q head of the group): the four waves of a block take every fourth
// tile of 16 columns, up to CT each, and share the keys and values, which travel into a ring of slices in LDS while earlier slices are worked on.  What
// the columns are, how the work is dealt to blocks and what a partial result is: tree_attention.hip, whose kernel has every column in every
// wave and so wants few of them.
//
// A step's MFMAs, V(s-1)^T P(s-1)^T and then K(s+1) Q^T, wait for nothing that the softmax of slice s, which stands between them, has to
// say; they are issued with it in between, the fragments of K(s+1) read behind the first half and those of V(s) behind the second.  The
// exponentials' reference follows the largest score when that is more than 2^8 ahead, tested by the lanes on their own: most steps neither
// reduce a maximum nor rescale.  The sum of a column's weights is one more row of the second product (values of one): it is the sum of the
// weights as they are rounded, so that a dominant weight's rounding cancels.
// What bounds it: with 256 columns and a head of 128 the issue of a wave's 68 MFMAs, 32 exponentials and some 130 other instructions a
// slice, one wave a SIMD (the MFMAs are busy for two fifths of the time); with fewer columns the keys and values from memory.  us of the kernel for 4
// requests of 32,000 places (524 MB): 64 columns 101 (5.2 TB/s), 128 116, 192 136, 256 158 (847 TFLOP/s); the merges take 6 to 11 more.
#include <type_traits>
#include <utility>

#include "common.h"
#include "mfma_tiles.h"
#include "tree_attention.h"

#define TREE_PAGES 1024              // page numbers of a run's slices that LDS holds at a time

#define INLINE __attribute__((always_inline))      // a lambda that is not inlined has its accumulators in memory

namespace {

__device__ __forceinline__ void score_first(floatx4& s, const bf16x8& k, const bf16x8& q) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=&v"(s) : "v"(k), "a"(q));
}
__device__ __forceinline__ void score_next(floatx4& s, const bf16x8& k, const bf16x8& q) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(s) : "v"(k), "a"(q));
}
// 16 bytes a lane into LDS at lds + PLUS, from OFF bytes behind g (the instruction adds them to both addresses)
template <int OFF, int PLUS>
__device__ __forceinline__ void copy16_off(unsigned long long g, unsigned lds) {
    asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off offset:%2"
                 : : "s"(lds), "v"(g), "i"(OFF), "i"(PLUS - OFF) : "memory", "m0", "scc");
}
// an accumulator stays in its register class, and what follows reads it here
__device__ __forceinline__ void pin(floatx4& x) { asm volatile("" : "+a"(x)); }
// (as an instruction: the compiler would quiet every operand first)
__device__ __forceinline__ float largest3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ void to_acc(bf16x8& x) { asm volatile("" : "+a"(x)); }
__device__ __forceinline__ void hold(bf16x8& x) { asm volatile("" : "+v"(x)); }
// two values of bfloat16, zeros in the place of those that are not finite
__device__ __forceinline__ uint32_t only_finite(uint32_t x) {
    if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
    if ((x & 0x7f800000u) == 0x7f800000u) x &= 0xffffu;
    return x;
}
template <typename F, int... I>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F&& f) {
    each_of(f, std::make_integer_sequence<int, N>{});
}
// slices of keys and values that LDS holds
constexpr int ring_of(int d) { return d == 256 ? 4 : 8; }

template <int D, int CT, bool CAP>
__global__ __launch_bounds__(256, 1) void tree_wide_kernel(const TreeArgs a) {
    constexpr int COLS = 64 * CT, KS = D / 32, DT = D / 16, NR = ring_of(D);
    constexpr int KFR = 2 * KS, KC = KFR / 4, VC = DT / 4, CPI = KC + VC;      // fragments of a slice's keys, a wave's copies a step
    constexpr unsigned K_SLOT = KFR * 1024u, V_SLOT = DT * 1024u, V_BASE = NR * K_SLOT;
    constexpr float LAG = 8.f;
    __shared__ __attribute__((aligned(1024))) char smem[V_BASE + NR * V_SLOT];
    __shared__ int32_t pages[TREE_PAGES];
    __shared__ uint32_t see[COLS * (TREE_WORDS + 1)];                          // the columns' bits, and a word of zeros
    __shared__ int first_seen[COLS];                                           // the first cached place of each
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), qc = lane & 15, kg = lane >> 4;
    const int G = a.nq / a.nkv;
    int b, g;
    tree_place(a.nkv, b, g);
    if (b >= a.blocks) return;
    const bf16_t* __restrict__ kc = (const bf16_t*)a.k_cache + (size_t)g * a.page_size * D;
    const bf16_t* __restrict__ vc = (const bf16_t*)a.v_cache + (size_t)g * a.page_size * D;
    const size_t page_bytes = (size_t)a.nkv * a.page_size * D * 2;
    const float log2e = 1.4426950408889634f;
    // scores in the exponent's units: sl2 times the product, of queries whose sign is the scale's (with a cap the scores are in these units already)
    const float sl2 = CAP ? 1.f : fmaxf(fabsf(a.scale) * log2e, 1e-30f), lag = LAG / sl2;
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
    // what this wave copies: K fragments (tile c_kt, steps c_ks ..) and value tiles wave * VC ..
    const int c_kt = wave >> 1, c_ks = (wave & 1) * KC;
    const int c_key = (qc >> 2) * 8 + c_kt * 4 + (qc & 3);
    const unsigned lds0 = (unsigned)(size_t)(lds_ptr_t)smem;
    const unsigned k_to = lds0 + (unsigned)(wave * KC) * 1024u, v_to = lds0 + V_BASE + (unsigned)(wave * VC) * 1024u;
    const unsigned long long k_base = (unsigned long long)kc + (unsigned)((c_ks * 32 + kg * 8) * 2);
    const unsigned long long v_base = (unsigned long long)vc + (unsigned)((wave * VC * 16 + qc) * a.page_size * 2);
    const unsigned v_step = (unsigned)a.page_size * 32u;                       // bytes from a value tile to the next

    const TreeRun run = tree_run<32, COLS>(a, b);
    const int x1 = run.x1;
    if (run.x0 >= x1) return;
    int r = run.r, before = run.before;
    TreeRequest t = run.t;

    for (int x = run.x0; x < x1;) {
        if (x >= before + tree_cost<32, COLS>(t)) {
            before += tree_cost<32, COLS>(t);
            t = tree_request<32, COLS>(a, ++r);
            continue;
        }
        const int group = (x - before) / (tree_begin<32, COLS>() + t.slices * tree_weight<COLS>(COLS));
        const TreeGroup<32, COLS> span(t, before, group);
        const int s0 = span.slice(x), s1 = x1 < span.end() ? span.slice(x1) : t.slices;
        x = span.end();
        if (s0 >= s1) continue;          // (another block has it)
        const int ncols = min(COLS, t.nodes * G - group * COLS);
        const int32_t* __restrict__ bt = a.block_tables + (size_t)r * a.bt_stride;

        // The first chunk's page numbers, the columns' bits and the queries are asked for together.  (A chunk: slices whose page numbers fit,
        // beginning anywhere in a page.)
        const int last_block = (max(t.end, 1) - 1) & ~7;     // blocks of eight places lie in one page
        const int chunk = max(1, ((TREE_PAGES - 2) << a.page_shift) >> 5);
        auto chunk_page = [&](int c0) INLINE { return (t.first + c0 * 32) >> a.page_shift; };
        auto chunk_pages = [&](int c0) INLINE {
            return (min(last_block, t.first + min(c0 + chunk, s1) * 32 - 8) >> a.page_shift) - chunk_page(c0) + 1;
        };
        const int first_page = bt[chunk_page(s0) + min(tid, chunk_pages(s0) - 1)];
        static_assert(COLS <= 256, "a thread a column");
        const TreeRow row = tree_row(a.ancestors + (size_t)(t.n0 + (min(tid & (COLS - 1), ncols - 1) + group * COLS) / G) * a.words, a.words,
                                     t.end - t.start, t.start, a.window);
        // A wave's column tiles are every fourth: waves have as much to do whatever the columns, and a step is as long as the tiles there are.
        auto run_of = [&](auto TILES) INLINE {
        constexpr int NT = decltype(TILES)::value;
        constexpr int NPV = (DT + 1) * NT, NQK = KFR * NT, NS = NPV + NQK;         // a step's MFMAs (the sums' among them)
        constexpr int NP = 4 * NT, ITEMS = 3 * NP;                                 // pairs of scores a lane, three instructions' worth each
        bf16x8 q[NT][KS];
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) {
            const int c = min((ct * 4 + wave) * 16 + qc, ncols - 1) + group * COLS, node = c / G, head = g * G + (c - node * G);
            const bf16_t* qp = (const bf16_t*)a.q + (size_t)(t.n0 + node) * a.q_stride + (size_t)head * D + kg * 8;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) q[ct][ks] = *reinterpret_cast<const bf16x8*>(qp + ks * 32);
        }
        __syncthreads();                 // (the run before is done with LDS)
        if (tid < COLS) {
#pragma unroll
            for (int w = 0; w < TREE_WORDS; ++w) see[tid * (TREE_WORDS + 1) + w] = row.bits[w];
            see[tid * (TREE_WORDS + 1) + TREE_WORDS] = 0;
            first_seen[tid] = row.lo;
        }

        floatx4 o[NT][DT + 1], sc[2][NT][2];         // (the last of o: the sums, four times the same)
        bf16x8 pf[2][NT], kf[KFR], vf[DT], ones;
        float top_ref[NT], limit[NT], neg_ref[NT], factor[NT];  // a column's reference, what a score may be, minus the reference in the exponent's units, what the outputs still want
        bool rescale = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) ones[i] = (bf16_t)1.f;
        hold(ones);                      // (in registers from here on: made anew right before an MFMA, which the compiler does not know for one, they came too late)
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) {
            top_ref[ct] = limit[ct] = -INFINITY;
            neg_ref[ct] = 0.f;
            factor[ct] = 1.f;
        }
        each<NT * (DT + 1)>([&](auto I) INLINE {
            floatx4& x = o[decltype(I)::value % NT][decltype(I)::value / NT];
            x = floatx4{0.f, 0.f, 0.f, 0.f};
            pin(x);
        });
        int lo_most = 0, lo_least = 0;

        // which of the places key, key + 1, ... a column sees: a bit each (the next 8 of them hold)
        auto visible = [&](int ct, int key) INLINE {
            const int c = (ct * 4 + wave) * 16 + qc, j = key - t.start;
            const uint32_t* row = see + c * (TREE_WORDS + 1);
            if (j >= 0) {
                const int w = min(j >> 5, TREE_WORDS - 1);
                return j < 32 * TREE_WORDS ? __funnelshift_r(row[w], row[w + 1], j & 31) : 0u;
            }
            const int cached = min(-j, 31), below = min(max(first_seen[c] - key, 0), 31);
            return (((1u << cached) - 1) & (~0u << below)) | (-j < 32 ? row[0] << -j : 0u);
        };
        auto settle = [&](floatx4 (&x)[NT][2]) INLINE {
#pragma unroll
            for (int ct = 0; ct < NT; ++ct) asm volatile("" : "+v"(x[ct][0]), "+v"(x[ct][1]));
        };
        // the first place of slice s; behind the run's last slice one that nobody sees
        auto place_of = [&](int s) INLINE { return s < s1 ? t.first + s * 32 : 0x40000000; };
        auto is_masked = [&](int k0) INLINE { return k0 + 32 > t.start || k0 < lo_most; };
        auto mask = [&](floatx4 (&x)[NT][2], int k0) INLINE {
#pragma unroll
            for (int ct = 0; ct < NT; ++ct) {
                const uint32_t sees = visible(ct, k0 + kg * 8);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[ct][e >> 2][e & 3] = (sees >> e) & 1 ? x[ct][e >> 2][e & 3] : -INFINITY;
                asm volatile("" : "+v"(x[ct][0]), "+v"(x[ct][1]));      // (here, in the branch)
            }
        };
        auto cap = [&](floatx4 (&x)[NT][2]) INLINE {
            // c tanh(x / c) = c (1 - e) / (1 + e), e = e^(-2 |x| / c): off by about half a step of c, whatever the score; for caps of some ten to a
            // hundred less than a weight's rounding by far
            const float in = -2.f * fabsf(a.scale) / a.softcap * log2e, outer = a.softcap * log2e;
#pragma unroll
            for (int ct = 0; ct < NT; ++ct) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float s = x[ct][e >> 2][e & 3], z = __builtin_amdgcn_exp2f(-fabsf(s * in));
                    x[ct][e >> 2][e & 3] = copysignf(outer * (1.f - z) / (1.f + z), s);
                }
                asm volatile("" : "+v"(x[ct][0]), "+v"(x[ct][1]));
            }
        };
        // Values of places of slice k0 that no column sees: what lies there is anything, and becomes zeros.  A value that is not finite may only reach
        // the columns that see it (zero times it would not be zero): the product takes a zero, and who sees it has it added.
        auto clean = [&](int k0) INLINE {
            uint32_t live = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k0 + kg * 8 + i < t.end && k0 + kg * 8 + i >= lo_least) live |= 1u << i;
            uint32_t keep[4], bad[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                keep[w] = ((live >> (2 * w)) & 1 ? 0xffffu : 0u) | ((live >> (2 * w + 1)) & 1 ? 0xffff0000u : 0u);
                bad[w] = 0;
            }
            each<DT>([&](auto F) INLINE {
                constexpr int dt = decltype(F)::value;
                uint4 x = __builtin_bit_cast(uint4, vf[dt]);
                x.x &= keep[0]; x.y &= keep[1]; x.z &= keep[2]; x.w &= keep[3];
                // (bit 15 of a half of the sum: its exponent is all ones)
                bad[0] |= (x.x & 0x7f807f80u) + 0x00800080u;
                bad[1] |= (x.y & 0x7f807f80u) + 0x00800080u;
                bad[2] |= (x.z & 0x7f807f80u) + 0x00800080u;
                bad[3] |= (x.w & 0x7f807f80u) + 0x00800080u;
                vf[dt] = __builtin_bit_cast(bf16x8, x);
                hold(vf[dt]);
            });
            uint32_t odd = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) odd |= (((bad[w] >> 15) & 1) | ((bad[w] >> 30) & 2)) << (2 * w);
            odd <<= 8 * kg;
            if (__any(odd != 0)) {
#pragma unroll
                for (int x = 1; x < 64; x <<= 1) odd |= (uint32_t)__shfl_xor((int)odd, x, 64);
                each<DT>([&](auto F) INLINE {
                    constexpr int dt = decltype(F)::value;
                    uint4 x = __builtin_bit_cast(uint4, vf[dt]);
                    x = make_uint4(only_finite(x.x), only_finite(x.y), only_finite(x.z), only_finite(x.w));
                    vf[dt] = __builtin_bit_cast(bf16x8, x);
                    hold(vf[dt]);
                });
                asm volatile("s_nop 15\n\ts_nop 15");        // (the outputs' MFMAs have written)
                for (uint32_t left = __builtin_amdgcn_readfirstlane(odd); left; left &= left - 1) {
                    const int key = k0 + __ffs((int)left) - 1;
                    int page = bt[key >> a.page_shift];
                    if ((unsigned)page >= (unsigned)a.num_pages) page = 0;
                    const bf16_t* vp = vc + (size_t)page * (page_bytes / 2) + (key & (a.page_size - 1)) + (size_t)(4 * kg) * a.page_size;
                    uint32_t sees[NT];
#pragma unroll
                    for (int ct = 0; ct < NT; ++ct) sees[ct] = visible(ct, key);
                    each<DT>([&](auto F) INLINE {
                        constexpr int dt = decltype(F)::value;
                        each<4>([&](auto E) INLINE {
                            constexpr int e = decltype(E)::value;
                            const float x = to_f32(*vp);
                            vp += e < 3 ? a.page_size : 13 * a.page_size;
                            each<NT>([&](auto C) INLINE {
                                constexpr int ct = decltype(C)::value;
                                if ((sees[ct] & 1) && !(fabsf(x) < INFINITY)) o[ct][dt][e] += x;
                            });
                        });
                        each<NT>([&](auto C) INLINE { pin(o[decltype(C)::value][dt]); });
                    });
                }
            }
            asm volatile("s_nop 3");      // (what a vector instruction has written an MFMA may read some instructions later: the compiler does not know these for MFMAs)
        };

        // the copies: keys and values of slices, counted within a chunk that begins at slice c0
        int c0 = s0, page0 = 0;
        auto k_at = [&](int x) INLINE {
            const int key = t.first + (c0 + x) * 32 + c_key, at = (key & ~7) <= last_block ? key : last_block + (key & 7);
            return k_base + (unsigned long long)((unsigned)pages[(at >> a.page_shift) - page0]) * page_bytes +
                   (unsigned)((at & (a.page_size - 1)) * D * 2);
        };
        auto v_at = [&](int x) INLINE {
            const int at = min(t.first + (c0 + x) * 32 + kg * 8, last_block);
            return v_base + (unsigned long long)((unsigned)pages[(at >> a.page_shift) - page0]) * page_bytes + (unsigned)((at & (a.page_size - 1)) * 2);
        };
        auto copy_k = [&](auto C, unsigned long long at, unsigned to) INLINE {
            constexpr int c = decltype(C)::value;
            copy16_off<c * 64, c * 1024>(at, to);
        };
        auto copy_v = [&](auto C, unsigned long long& at, unsigned to) INLINE {
            constexpr int c = decltype(C)::value;
            copy16_off<0, c * 1024>(at, to);
            if constexpr (c + 1 < VC) at += v_step;
        };

        for (; c0 < s1; c0 += chunk) {
            const int n = min(chunk, s1 - c0);
            if (c0 > s0) {
                __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(0));      // the chunk before: its copies have landed, its slices and pages are read
                __syncthreads();
            }
            // (slices past the chunk's end are copied ahead in vain: their places are held to its pages)
            page0 = chunk_page(c0);
            const int pages_n = chunk_pages(c0);
            for (int i = tid; i < pages_n; i += 256) {
                const int p = c0 == s0 && i == tid ? first_page : bt[page0 + i];
                pages[i] = (unsigned)p < (unsigned)a.num_pages ? p : 0;
            }
            __syncthreads();
            if (c0 == s0 && a.window > 0) {
                lo_most = 0;
                lo_least = 0x7fffffff;
                for (int c = lane; c < COLS; c += 64) {
                    lo_most = max(lo_most, first_seen[c]);
                    lo_least = min(lo_least, first_seen[c]);
                }
#pragma unroll
                for (int x = 1; x < 64; x <<= 1) {
                    lo_most = max(lo_most, __shfl_xor(lo_most, x, 64));
                    lo_least = min(lo_least, __shfl_xor(lo_least, x, 64));
                }
                lo_most = __builtin_amdgcn_readfirstlane(lo_most);
                lo_least = __builtin_amdgcn_readfirstlane(lo_least);
            }
            auto held = [&](int x) INLINE { return min(x, n - 1); };
            // step x issues K(x + NR) and V(x + NR - 1): the steps -NR .. -1
#pragma unroll
            for (int x = 0; x < NR; ++x) {
                const unsigned long long ka = k_at(held(x));
                each<KC>([&](auto C) INLINE { copy_k(C, ka, k_to + x * K_SLOT); });
                if (x > 0) {
                    unsigned long long va = v_at(held(x - 1));
                    each<VC>([&](auto C) INLINE { copy_v(C, va, v_to + (x - 1) * V_SLOT); });
                }
            }
            if (c0 == s0) {
#pragma unroll
                for (int ct = 0; ct < NT; ++ct)
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        uint4 x = __builtin_bit_cast(uint4, q[ct][ks]);
                        x.x ^= flip; x.y ^= flip; x.z ^= flip; x.w ^= flip;
                        q[ct][ks] = __builtin_bit_cast(bf16x8, x);
                        to_acc(q[ct][ks]);
                    }
            }
            __builtin_amdgcn_s_waitcnt(vmcnt_imm((NR - 1) * CPI));
            __syncthreads();
            {
                const char* src = smem + lane * 16;
                each<KFR>([&](auto F) INLINE { kf[decltype(F)::value] = *reinterpret_cast<const bf16x8*>(src + decltype(F)::value * 1024); });
                each<NQK>([&](auto I) INLINE {
                    constexpr int f = decltype(I)::value / NT, ct = decltype(I)::value % NT, kt = f & 1, ks = f >> 1;
                    if constexpr (ks == 0) score_first(sc[0][ct][kt], kf[kt * KS + ks], q[ct][ks]);
                    else score_next(sc[0][ct][kt], kf[kt * KS + ks], q[ct][ks]);
                });
                const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int ct = 0; ct < NT; ++ct) pf[1][ct] = __builtin_bit_cast(bf16x8, zero);
                each<DT>([&](auto F) INLINE { vf[decltype(F)::value] = __builtin_bit_cast(bf16x8, zero); });
                asm volatile("s_nop 3");
            }
            unsigned k_rd = NR > 1 ? K_SLOT : 0, v_rd = 0;                // K(s + 1), V(s)
            unsigned k_wr = k_to, v_wr = v_to + (NR - 1) * V_SLOT;        // where K(s + NR), V(s + NR - 1) go
            int x_next = NR;                                              // and the first of these slices
            auto slice_place = [&](int s) INLINE { return s < n ? place_of(c0 + s) : 0x40000000; };
            auto step = [&](auto H, int s) INLINE {
                constexpr int h = decltype(H)::value;
                __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm((NR - 2) * CPI));
                asm volatile("s_barrier\n\ts_nop 7" ::: "memory");        // (the scores' last MFMAs have written before a vector instruction reads them)
                settle(sc[h]);
                const char* ksrc = smem + k_rd + lane * 16;
                const char* vsrc = smem + V_BASE + v_rd + lane * 16;
                const int k0 = slice_place(s), prev = s > 0 ? slice_place(s - 1) : 0;
                if (s > 0 && is_masked(prev)) clean(prev);
                float tmp0 = 0.f, tmp1 = 0.f, top[NT];
                bool ahead = false;
                constexpr bool SPREAD = NS >= 16;                     // the maxima go between the MFMAs, too, where there are enough of these
                constexpr int CHECK = SPREAD ? 5 + 4 * NT : 4;
                unsigned long long ka = 0, va = 0;
                each<NS>([&](auto slot) INLINE {
                    constexpr int n_ = decltype(slot)::value;
                    if constexpr (n_ < NPV) {
                        constexpr int ct = n_ % NT, dt = n_ / NT;
                        if constexpr (dt < DT) mfma_acc(o[ct][dt], vf[dt], pf[h ^ 1][ct]);
                        else mfma_acc(o[ct][DT], ones, pf[h ^ 1][ct]);
                    } else {
                        constexpr int f = (n_ - NPV) / NT, ct = (n_ - NPV) % NT, kt = f & 1, ks = f >> 1;
                        if constexpr (ks == 0) score_first(sc[h ^ 1][ct][kt], kf[kt * KS + ks], q[ct][ks]);
                        else score_next(sc[h ^ 1][ct][kt], kf[kt * KS + ks], q[ct][ks]);
                    }
                    // fragments: K(s + 1) in the order of their use behind the first half, then V(s)
                    each<KFR>([&](auto F) INLINE {
                        constexpr int f = decltype(F)::value, fr = (f & 1) * KS + (f >> 1);
                        if constexpr (f * NPV / KFR == n_) kf[fr] = *reinterpret_cast<const bf16x8*>(ksrc + fr * 1024);
                    });
                    each<DT>([&](auto F) INLINE {
                        constexpr int dt = decltype(F)::value;
                        if constexpr (NPV + dt * NQK / DT == n_) vf[dt] = *reinterpret_cast<const bf16x8*>(vsrc + dt * 1024);
                    });
                    // the softmax of slice s
                    if constexpr (n_ == 4) {
                        if constexpr (CAP) cap(sc[h]);
                        if (is_masked(k0)) mask(sc[h], k0);
                    }
                    each<4 * NT>([&](auto I) INLINE {
                        constexpr int ct = decltype(I)::value / 4, j = decltype(I)::value % 4;
                        if constexpr (n_ == (SPREAD ? 5 + decltype(I)::value : 4)) {
                            const floatx4 &x = sc[h][ct][0], &y = sc[h][ct][1];
                            if constexpr (j == 0) top[ct] = largest3(x[0], x[1], x[2]);
                            else if constexpr (j == 1) top[ct] = largest3(top[ct], x[3], y[0]);
                            else if constexpr (j == 2) top[ct] = largest3(top[ct], y[1], y[2]);
                            else {
                                top[ct] = largest3(top[ct], y[3], y[3]);
                                ahead |= top[ct] > limit[ct];
                            }
                        }
                    });
                    if constexpr (n_ == CHECK) {
                        if (__any(ahead)) {
                            rescale = true;
#pragma unroll
                            for (int ct = 0; ct < NT; ++ct) {
                                const float m = rows_max(top[ct]);
                                const bool up = m > limit[ct];
                                factor[ct] = up ? __builtin_amdgcn_exp2f((top_ref[ct] - m) * sl2) : 1.f;
                                top_ref[ct] = up ? m : top_ref[ct];
                                limit[ct] = up ? m + lag : limit[ct];
                                neg_ref[ct] = top_ref[ct] == -INFINITY ? 0.f : -top_ref[ct] * sl2;
                                asm volatile("" : "+v"(factor[ct]), "+v"(top_ref[ct]), "+v"(neg_ref[ct]), "+v"(limit[ct]));
                            }
                        }
                    }
                    if constexpr (n_ > CHECK) {
                        constexpr int i0 = (n_ - CHECK - 1) * ITEMS / (NS - CHECK - 1), i1 = (n_ - CHECK) * ITEMS / (NS - CHECK - 1);
                        each<i1 - i0>([&](auto I) INLINE {
                            constexpr int i = i0 + decltype(I)::value, p = i / 3, ct = p / 4, e = (p % 4) * 2;
                            if constexpr (i % 3 == 0) {
                                tmp0 = fmaf(sc[h][ct][e >> 2][e & 3], sl2, neg_ref[ct]);
                                tmp1 = fmaf(sc[h][ct][e >> 2][(e & 3) + 1], sl2, neg_ref[ct]);
                                tmp0 = __builtin_amdgcn_exp2f(tmp0);
                            } else if constexpr (i % 3 == 1) {
                                tmp1 = __builtin_amdgcn_exp2f(tmp1);
                            } else {
                                // (a weight rounds to bfloat16, half a step of 2^-8, as the product takes it)
                                pf[h][ct][e] = (bf16_t)tmp0;
                                pf[h][ct][e + 1] = (bf16_t)tmp1;
                            }
                        });
                    }
                    // the copies of later slices
                    if constexpr (n_ == NPV / 2) ka = k_at(held(x_next));
                    if constexpr (n_ == NPV - 1) va = v_at(held(x_next - 1));
                    if constexpr (n_ >= NPV) {
                        constexpr int j0 = (n_ - NPV) * CPI / NQK, j1 = (n_ - NPV + 1) * CPI / NQK;
                        each<j1 - j0>([&](auto J) INLINE {
                            constexpr int c = j0 + decltype(J)::value;
                            if constexpr (c < KC) copy_k(std::integral_constant<int, c < KC ? c : 0>{}, ka, k_wr);
                            else copy_v(std::integral_constant<int, c < KC ? 0 : c - KC>{}, va, v_wr);
                        });
                    }
                    __builtin_amdgcn_sched_barrier(0);
                });
                // (worked out here: the compiler would move the softmax out of the MFMAs, behind the next step's branch)
#pragma unroll
                for (int ct = 0; ct < NT; ++ct) asm volatile("" : "+v"(pf[h][ct]));
                if (rescale) {
                    // the outputs hold the slices before s - 1 and s - 1 itself, all against the reference before
                    asm volatile("s_nop 15\n\ts_nop 15");
                    each<NT*(DT + 1)>([&](auto I) INLINE {
                        constexpr int ct = decltype(I)::value % NT, dt = decltype(I)::value / NT;
                        pin(o[ct][dt]);
                        o[ct][dt] *= factor[ct];
                        pin(o[ct][dt]);
                    });
                    rescale = false;
                    asm volatile("s_nop 3");
                }
                ++x_next;
                k_wr = k_to + k_rd;
                v_wr = v_to + v_rd;
                k_rd = ring_next<K_SLOT, NR * K_SLOT>(k_rd);
                v_rd = ring_next<V_SLOT, NR * V_SLOT>(v_rd);
            };
            // (in pairs, whose second step may have nothing: with an end in between the compiler carries the accumulators from one set of registers to
            // another in every step)
            for (int s = 0; s < n; s += 2) {
                step(std::integral_constant<int, 0>{}, s);
                step(std::integral_constant<int, 1>{}, s + 1);
            }
            // the values of the chunk's last slice
            const int last = slice_place((n + 1) / 2 * 2 - 1);
            if (is_masked(last)) clean(last);
            asm volatile("s_nop 3");
            each<NPV>([&](auto I) INLINE {
                constexpr int ct = decltype(I)::value % NT, dt = decltype(I)::value / NT;
                if constexpr (dt < DT) mfma_acc(o[ct][dt], vf[dt], pf[1][ct]);
                else mfma_acc(o[ct][DT], ones, pf[1][ct]);
            });
        }
        __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(0));      // (the copies past the end must not outlive the block)
        asm volatile("s_nop 15\n\ts_nop 15");                // (the outputs' last MFMAs have written)
        each<NT*(DT + 1)>([&](auto I) INLINE { pin(o[decltype(I)::value % NT][decltype(I)::value / NT]); });

        const bool whole = s0 == 0 && s1 == t.slices;
        const size_t part = (((size_t)g * a.blocks + b) * 2 + (s0 == 0 ? 1 : 0)) * COLS;
        const int lane2 = w4_lane(), qc2 = lane2 & 15, kg2 = lane2 >> 4;
        each<NT>([&](auto C) INLINE {
            constexpr int ct = decltype(C)::value;
            const int c = (ct * 4 + wave) * 16 + qc2;
            if (c < ncols) {
                float sum = o[ct][DT][0];
                const float top = top_ref[ct] == -INFINITY ? -INFINITY : -neg_ref[ct];
                if (whole) {
                    const int cc = c + group * COLS, node = cc / G, head = g * G + (cc - node * G);
                    if (a.sinks) {
                        if (top == -INFINITY) sum = 1.f;         // (nothing seen: zeros)
                        else sum += __builtin_amdgcn_exp2f(a.sinks[head] * log2e - top);
                    }
                    const float inv = sum > 0.f ? 1.0f / sum : sum != sum ? sum : 0.f;
                    bf16_t* op = (bf16_t*)a.out + ((size_t)(t.n0 + node) * a.nq + head) * D + 4 * kg2;
                    each<DT>([&](auto F) INLINE {
                        constexpr int dt = decltype(F)::value;
                        typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 bf16x4;
                        bf16x4 x;
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = (bf16_t)(o[ct][dt][e] * inv);
                        *reinterpret_cast<bf16x4*>(op + dt * 16) = x;
                    });
                } else {
                    float* po = a.part_o + (part + c) * D + 4 * kg2;
                    each<DT>([&](auto F) INLINE { *reinterpret_cast<floatx4*>(po + decltype(F)::value * 16) = o[ct][decltype(F)::value]; });
                    if (kg2 == 0) *reinterpret_cast<float2*>(a.part_ml + (part + c) * 2) = make_float2(top, sum);
                }
            }
        });
        };
        const int nt = (ncols + 63) / 64;
        if constexpr (CT >= 4) {
            if (nt == 4) run_of(std::integral_constant<int, 4>{});
            else if (nt == 3) run_of(std::integral_constant<int, 3>{});
        }
        if constexpr (CT >= 2) {
            if (nt == 2) run_of(std::integral_constant<int, 2>{});
        }
        if (nt == 1) run_of(std::integral_constant<int, 1>{});
    }
}

}  // namespace

// Up to 32 columns all waves have all of them (tree_attention.hip): us of the kernels, merge included, here / there, pages of 64: one request of 200
// places, 32 columns 17.4 / 10.8, 36 columns 17.5 / 17.8; 8 of 2,000 33.6 / 30.9 and 34.5 / 35.9; 4 of 32,000 105 / 111 and 104 / 150.  A head of 256
// leaves registers for half as many tiles.
int tree_wide_tiles(int columns, int d) { return columns <= 32 ? 0 : d == 256 ? 2 : 4; }

int tree_wide_launch(const TreeArgs& a, int d, hipStream_t stream) {
    const int grid = tree_grid(a.nkv, a.blocks);
#define TFF_TREE_W(D, CT)                                                                       \
    do {                                                                                        \
        if (a.softcap > 0.f) tree_wide_kernel<D, CT, true><<<grid, 256, 0, stream>>>(a);        \
        else tree_wide_kernel<D, CT, false><<<grid, 256, 0, stream>>>(a);                       \
        return tff_check_launch("tree_attention");                                              \
    } while (0)
    if (d == 64) TFF_TREE_W(64, 4);
    if (d == 128) TFF_TREE_W(128, 4);
    if (d == 256) TFF_TREE_W(256, 2);
#undef TFF_TREE_W
    return tff_fail("tree_attention: no kernel for head size %d", d);
}
