// What the requests' options do to rows of logits before a token is chosen: penalties for tokens that the request has seen, biases of
// single tokens, a mask of the tokens that a grammar allows.  For token v of a row,
//   x <- x > 0 ? x / rep : x * rep            if v stands in the request's prompt or output (what tff_repetition_penalty does)
//   x <- x - freq n_v - pres [n_v > 0]        n_v: how often v stands in its output
//   x <- x + bias_v                           if v is listed
//   x <- -inf                                 where the row's mask has no bit
// The rows of drafted trees' nodes belong to the tree's request and have the tokens on their path (`ancestors`) as output besides: the history
// ends before node 0, which is the request's last token and on every path (the prompt's, where the prompt is longer than the history).
// The reference has the first of these, on the host (src/core/sampler/LLMSampler.cpp:21-34).
//
// A block takes a run of the vocabulary of one row and counts the tokens of the request's whole history that fall into it in LDS: the
// history comes as it is, with repetitions, no table of counts by token has to be kept or cleared, counts are integers and so
// do not depend on the order of the atomics.  Then it goes over its run once: what is masked is written and not read, and in place what no
// option touches is neither.  The bound is memory: 4 bytes a logit in and out, of what a mask forbids only out.
// us of the kernel, 151,936 logits a row: one row 4.2, 48 rows under grammars that allow one in fifty 13.8 (29 MB; a fill of as much takes 6.9, the
// rest is the histories), 150 rows of trees, nine in ten allowed, 38 (4.6 TB/s).  In place, where the counts say which logits are read and those so
// wait for them: 4.2, 13.8 and 46.
#include "common.h"
#include "tffinfer_kernels.h"
#include "tree_attention.h"

#define ADJUST_SEEN 0x80000000u      // in the prompt; the bits below count the output

struct AdjustArgs {
    const float* logits;
    float* out;
    int rows, V, runs;
    const int32_t *history, *cu_history, *prompt_lens;
    int history_len, requests;
    const float *repetition, *presence, *frequency;
    const int32_t* bias_ids;
    const float* bias_values;
    const int32_t* cu_bias;
    int bias_len;
    const int32_t* masks;
    int num_masks, mask_words;
    const int32_t* mask_rows;
    const int32_t *draft_tokens, *cu_nodes, *ancestors;
    int words;
};

// Four bits of a mask from token v on (the words behind the last are not read).
__device__ __forceinline__ uint32_t mask_bits4(const int32_t* __restrict__ mask, int words, int v) {
    const int w = v >> 5;
    return __funnelshift_r((uint32_t)mask[w], (uint32_t)mask[min(w + 1, words - 1)], v & 31);
}

// RUN tokens of one row for a block of 256 threads, RUN / 1024 groups of four a thread.  A row need not begin at a multiple of 16 bytes: the groups
// do, and up to three tokens before the first and behind the last are the first threads' besides.
template <int RUN>
__global__ __launch_bounds__(256) void adjust_logits_kernel(const AdjustArgs a, const int vec) {
    constexpr int PER = RUN / 1024;
    __shared__ __attribute__((aligned(16))) uint32_t cnt[RUN];
    const int t = blockIdx.x / a.runs, v0 = (blockIdx.x - t * a.runs) * RUN, n = min(RUN, a.V - v0), tid = threadIdx.x;
    const size_t base = (size_t)t * a.V + v0;
    const float* x = a.logits + base;
    float* y = a.out + base;                     // (may be x)
    const bool in_place = a.logits == a.out;
    const int mask_row = a.mask_rows ? a.mask_rows[t] : -1;
    int r = t;
    if (a.cu_nodes) r = tree_row_request(a.cu_nodes, a.requests, t);
    r = __builtin_amdgcn_readfirstlane(r);
    const bool has_request = r < a.requests;      // (a row that no request has is left as it is)
    const int32_t* __restrict__ mask = has_request && mask_row >= 0 && mask_row < a.num_masks ? a.masks + (size_t)mask_row * a.mask_words : nullptr;
    // (all that the rest hangs on, asked for at once)
    float rep = 1.f, pres = 0.f, freq = 0.f;
    int h0 = 0, h1 = 0, out0 = 0, b0 = 0, b1 = 0;
    if (has_request) {
        rep = a.repetition[r];
        pres = a.presence[r];
        freq = a.frequency[r];
        h0 = a.cu_history[r];
        h1 = a.cu_history[r + 1];
        out0 = a.prompt_lens[r];
        if (a.cu_bias) {
            b0 = a.cu_bias[r];
            b1 = a.cu_bias[r + 1];
        }
    }
    h0 = min(max(h0, 0), a.history_len);
    h1 = min(max(h1, h0), a.history_len);
    const bool prompt_root = out0 > h1 - h0;      // (node 0 is the prompt's last token)
    out0 = h0 + min(max(out0, 0), h1 - h0);
    b0 = min(max(b0, 0), a.bias_len);
    b1 = min(max(b1, b0), a.bias_len);
    const bool counts = h0 < h1 || a.cu_nodes ? rep != 1.f || pres != 0.f || freq != 0.f : false;
    const int q0 = min(h1, (h0 + 3) & ~3), q1 = max(q0, h1 & ~3);      // (the part of the history that int4 loads can take)
    const bool hvec = ((uintptr_t)a.history & 15) == 0;
    // the thread's first bias and the history's first tokens (a thread's share of the others is asked for three steps ahead)
    int bias_id = -1;
    float bias = 0.f;
    if (b0 + tid < b1) {
        bias_id = a.bias_ids[b0 + tid];
        bias = a.bias_values[b0 + tid];
    }
    constexpr int AHEAD = 4;
    int4 next[AHEAD];
    if (counts && hvec) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int i = q0 / 4 + tid + 256 * k;
            if (i < q1 / 4) next[k] = reinterpret_cast<const int4*>(a.history)[i];
        }
    }
    const int head = vec ? min(n, (int)(-base & 3)) : n, groups = (n - head) / 4;      // (without `vec` all are the first threads' besides)

    // the logits and their bits are on their way while the history is counted
    float4 v[PER];
    uint32_t allowed[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int j = tid + 256 * k;
        allowed[k] = 15u;
        if (mask && j < groups) allowed[k] = mask_bits4(mask, a.mask_words, v0 + head + 4 * j) & 15u;
    }
    if (!in_place) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int j = tid + 256 * k;
            if (j < groups && allowed[k]) v[k] = *reinterpret_cast<const float4*>(x + head + 4 * j);
        }
    }
    if (counts) {
        for (int i = tid; i < RUN / 4; i += 256) reinterpret_cast<uint4*>(cnt)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        auto count = [&](int token, bool output) {
            const unsigned at = (unsigned)token - (unsigned)v0;
            if (at < (unsigned)n) {
                if (output) atomicAdd(&cnt[at], 1u);
                else atomicOr(&cnt[at], ADJUST_SEEN);
            }
        };
        if (hvec) {
            for (int i0 = q0 / 4; i0 < q1 / 4; i0 += 256 * AHEAD) {
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    const int i = i0 + tid + 256 * k, later = i + 256 * AHEAD;
                    const int4 h = next[k];
                    if (later < q1 / 4) next[k] = reinterpret_cast<const int4*>(a.history)[later];
                    if (i < q1 / 4) {
                        count(h.x, 4 * i >= out0);
                        count(h.y, 4 * i + 1 >= out0);
                        count(h.z, 4 * i + 2 >= out0);
                        count(h.w, 4 * i + 3 >= out0);
                    }
                }
            }
            if (tid < 8) {
                const int i = tid < 4 ? h0 + tid : q1 + tid - 4;
                if (tid < 4 ? i < q0 : i < h1) count(a.history[i], i >= out0);
            }
        } else {
            for (int i = h0 + tid; i < h1; i += 256) count(a.history[i], i >= out0);
        }
        if (a.cu_nodes) {
            const int n0 = max(a.cu_nodes[r], 0), nodes = min(min(a.cu_nodes[r + 1], a.rows) - n0, 32 * a.words);
            for (int j = tid; j < nodes; j += 256)
                if ((a.ancestors[(size_t)t * a.words + (j >> 5)] >> (j & 31)) & 1) count(a.draft_tokens[n0 + j], j > 0 || !prompt_root);
        }
        __syncthreads();
    }
    auto adjusted = [&](float z, uint32_t c) {
        if (c) {
            z = z > 0.f ? z / rep : z * rep;
            const uint32_t k = c & ~ADJUST_SEEN;
            if (k) z = z - freq * (float)k - pres;
        }
        return z;
    };
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int j = tid + 256 * k, i = head + 4 * j;
        if (j >= groups) continue;
        uint4 c = make_uint4(0, 0, 0, 0);
        if (counts) c = head ? make_uint4(cnt[i], cnt[i + 1], cnt[i + 2], cnt[i + 3]) : *reinterpret_cast<const uint4*>(&cnt[i]);
        const bool some = (c.x | c.y) | (c.z | c.w);
        if (in_place && allowed[k] == 15u && !some) continue;
        float4 z = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (allowed[k]) {
            z = v[k];
            if (in_place) z = *reinterpret_cast<const float4*>(x + i);
            if (some) {
                z.x = adjusted(z.x, c.x);
                z.y = adjusted(z.y, c.y);
                z.z = adjusted(z.z, c.z);
                z.w = adjusted(z.w, c.w);
            }
            if (!(allowed[k] & 1)) z.x = -INFINITY;
            if (!(allowed[k] & 2)) z.y = -INFINITY;
            if (!(allowed[k] & 4)) z.z = -INFINITY;
            if (!(allowed[k] & 8)) z.w = -INFINITY;
        }
        *reinterpret_cast<float4*>(y + i) = z;
    }
    auto one = [&](int i) {
        const bool may = !mask || ((mask[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1);
        const uint32_t c = counts ? cnt[i] : 0u;
        if (!may) y[i] = -INFINITY;
        else if (c || !in_place) y[i] = adjusted(x[i], c);
    };
    for (int i = tid; i < head; i += 256) one(i);
    for (int i = head + 4 * groups + tid; i < n; i += 256) one(i);
    if (b0 < b1) {
        // of equal tokens the last one listed counts: the largest place among them wins, by an integer maximum
        auto each_bias = [&](auto f) {
            int at = bias_id - v0;
            if (b0 + tid < b1 && at >= 0 && at < n) f(at, tid, bias_id, bias);
            for (int i = b0 + 256 + tid; i < b1; i += 256) {
                const int z = a.bias_ids[i];
                at = z - v0;
                if (at >= 0 && at < n) f(at, i - b0, z, a.bias_values[i]);
            }
        };
        __syncthreads();
        each_bias([&](int at, int, int, float) { cnt[at] = 0; });
        __syncthreads();
        each_bias([&](int at, int i, int, float) { atomicMax(&cnt[at], (uint32_t)(i + 1)); });
        __syncthreads();
        each_bias([&](int at, int i, int z, float value) {
            if (cnt[at] == (uint32_t)(i + 1) && (!mask || ((mask[z >> 5] >> (z & 31)) & 1))) y[at] += value;
        });
    }
}

TFF_API int tff_adjust_logits(const float* logits, float* out, int rows, int V, int requests, const int32_t* history, int history_len,
                              const int32_t* cu_history, const int32_t* prompt_lens, const float* repetition, const float* presence,
                              const float* frequency, const int32_t* bias_ids, const float* bias_values, int bias_len, const int32_t* cu_bias,
                              const int32_t* masks, int num_masks, const int32_t* mask_rows, const int32_t* draft_tokens,
                              const int32_t* cu_nodes, const int32_t* ancestors, int words, tff_stream_t stream) {
    TFF_REQUIRE(rows >= 0 && V > 0 && requests >= 0, "adjust_logits: bad sizes rows=%d V=%d requests=%d", rows, V, requests);
    if (rows == 0) return 0;
    TFF_REQUIRE(logits && out && cu_history && prompt_lens && repetition && presence && frequency, "adjust_logits: null pointer");
    TFF_REQUIRE(history_len >= 0 && (history || history_len == 0), "adjust_logits: a history of %d tokens without its tokens", history_len);
    TFF_REQUIRE(bias_len >= 0 && (!cu_bias || bias_len == 0 || (bias_ids && bias_values)), "adjust_logits: %d biases without tokens and values",
                bias_len);
    TFF_REQUIRE(!mask_rows || num_masks == 0 || masks, "adjust_logits: rows with masks, and no masks");
    TFF_REQUIRE(!cu_nodes || (draft_tokens && ancestors && words > 0), "adjust_logits: nodes without their tokens and ancestors");
    TFF_REQUIRE(cu_nodes || rows == requests, "adjust_logits: %d rows of %d requests", rows, requests);
    // Runs of 4,096 tokens, or of 2,048 where those would leave CUs with less than two blocks: every run goes through the request's whole history, so
    // few and long ones are better as soon as they fill the chip, and of the longer ones fewer are on a CU at a time.  us a call of 2,048 / 4,096 / 8,192:
    // 48 rows of 151,936 logits, histories of up to 8,192 tokens 15.5 / 14.1 / 16.0, 150 rows of trees 44.2 / 38.2 / 45.3.
    const int run = (int64_t)rows * ((V + 4095) / 4096) >= 2 * tff_device_cus() ? 4096 : 2048, runs = (V + run - 1) / run;
    TFF_REQUIRE((int64_t)rows * runs <= 0x7fffffff, "adjust_logits: %d rows of %d logits are more than a launch takes", rows, V);
    const AdjustArgs a{logits, out, rows, V, runs, history, cu_history, prompt_lens, history_len, requests, repetition, presence, frequency,
                       bias_ids, bias_values, cu_bias, bias_len, masks, masks ? num_masks : 0, (V + 31) / 32, mask_rows, draft_tokens, cu_nodes, ancestors, words};
    const int vec = (((uintptr_t)logits | (uintptr_t)out) & 15) == 0;      // (rows of both then begin alike)
    if (run == 4096) adjust_logits_kernel<4096><<<rows * runs, 256, 0, (hipStream_t)stream>>>(a, vec);
    else adjust_logits_kernel<2048><<<rows * runs, 256, 0, (hipStream_t)stream>>>(a, vec);
    return tff_check_launch("adjust_logits");
}
