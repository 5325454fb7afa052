// Logits of a batch of rows before a token is taken from each: penalties for
// repeated tokens, biases, and masks of the tokens that a grammar allows; with
// `tokens`, each row's best token of the result.
//
// Row r, token t, logit x; count = occurrences of t in the generated part of the
// row's history and on its draft-tree path, seen = t occurs anywhere in them:
//   y = seen ? (x > 0 ? x / rep : x * rep) : x
//   y = count > 0 ? (y - freq * count) - pres : y
//   y = y + bias[t], and -inf where the mask's bit is not set.
// Every product and sum is rounded to f32 by itself, in this order.  The best
// token is the largest y, the lowest index on ties; NaN and -inf are never taken
// (-1 where nothing else is left: a mask that allows no token).
#include <math.h>

#include <algorithm>

#include "logits.hpp"
#include "tb_common.hpp"

namespace tb {

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kSeen = 0x80000000u;   // counts: occurs in the prompt part

// Tokens of one block: its counts (and biases) are kept in LDS.
int chunk_tokens(int rows, int vocab) {
    (void)rows;
    (void)vocab;
    return 4096;
}

// Orders as the values do, ties to the lower index; 0: nothing to take.
__device__ __forceinline__ uint64_t best_item(float y, int t) {
    if (!(y > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(y == 0.f ? 0.f : y);   // -0 ties with 0
    const uint32_t key = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ((uint64_t)key << 32) | (uint32_t)~t;
}

__device__ __forceinline__ uint64_t max_over_wave(uint64_t v) {
    for (int off = 32; off; off >>= 1) {
        const uint32_t lo = __shfl_xor((uint32_t)v, off), hi = __shfl_xor((uint32_t)(v >> 32), off);
        const uint64_t o = ((uint64_t)hi << 32) | lo;
        v = o > v ? o : v;
    }
    return v;
}

// Grid (token chunks, rows).
__global__ __launch_bounds__(kThreads) void k_logits(LogitsParams p, int chunk, uint64_t *part) {
    extern __shared__ uint32_t lds[];
    __shared__ uint64_t red[kThreads / 64];
    uint32_t *cnt = lds;
    float *bias = reinterpret_cast<float *>(lds + (p.hist || p.nodes ? chunk : 0));
    const int tid = threadIdx.x, r = blockIdx.y;
    const int t0 = blockIdx.x * chunk, nt = min(chunk, p.vocab - t0);
    const bool counted = p.hist || p.nodes;
    for (int i = tid; i < nt; i += kThreads) {
        if (counted) cnt[i] = 0;
        if (p.n_bias) bias[i] = 0.f;
    }
    __syncthreads();
    if (p.hist) {
        const int g = r / (p.rows / p.groups);
        const int len = p.history_len ? min(max(p.history_len[g], 0), p.hist) : p.hist;
        const int prompt = p.prompt_len ? p.prompt_len[g] : p.prompt;
        const int64_t *h = p.history + (size_t)g * p.hist;
        for (int i = tid; i < len; i += kThreads) {
            const int64_t t = h[i] - t0;
            if (t < 0 || t >= nt) continue;
            if (i < prompt) atomicOr(&cnt[t], kSeen);
            else atomicAdd(&cnt[t], 1u);
        }
    }
    if (p.nodes) {
        const int node = r % p.nodes, words = (p.nodes + 31) / 32;
        const int64_t *d = p.draft + (size_t)(r / p.nodes) * p.nodes;
        const int32_t *m = p.tree_mask + ((size_t)(r / p.nodes) * p.nodes + node) * words;
        for (int j = tid; j < p.nodes; j += kThreads) {
            if (!((uint32_t)m[j >> 5] >> (j & 31) & 1)) continue;
            const int64_t t = d[j] - t0;
            if (t >= 0 && t < nt) atomicAdd(&cnt[t], 1u);
        }
    }
    if (p.n_bias) {
        // a token named several times gets the sum, taken in order by the thread
        // of its first entry
        const size_t g = r / (p.rows / p.bias_groups);
        const int64_t *ids = p.bias_ids + g * p.n_bias;
        const float *val = p.bias + g * p.n_bias;
        for (int i = tid; i < p.n_bias; i += kThreads) {
            const int64_t id = ids[i];
            if (id < t0 || id >= t0 + nt) continue;
            bool first = true;
            for (int j = 0; j < i && first; ++j) first = ids[j] != id;
            if (!first) continue;
            float s = val[i];
            for (int j = i + 1; j < p.n_bias; ++j)
                if (ids[j] == id) s = __fadd_rn(s, val[j]);
            bias[id - t0] = s;
        }
    }
    __syncthreads();
    const float rep = p.rep_rows ? p.rep_rows[r] : p.rep;
    const float pres = p.pres_rows ? p.pres_rows[r] : p.pres;
    const float freq = p.freq_rows ? p.freq_rows[r] : p.freq;
    const float *x = p.x + (size_t)r * p.vocab + t0;
    uint64_t best = 0;
    for (int i = tid; i < nt; i += kThreads) {
        float y = x[i];
        if (counted && cnt[i]) {
            const uint32_t c = cnt[i] & ~kSeen;
            y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
            if (c) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, (float)c)), pres);
        }
        if (p.n_bias) y = __fadd_rn(y, bias[i]);
        const int t = t0 + i;
        if (p.allowed && !((uint32_t)p.allowed[r * p.allowed_stride + (t >> 5)] >> (t & 31) & 1))
            y = -INFINITY;
        if (p.y) p.y[(size_t)r * p.vocab + t] = y;
        const uint64_t it = best_item(y, t);
        best = it > best ? it : best;
    }
    if (!part) return;
    best = max_over_wave(best);
    if ((tid & 63) == 0) red[tid >> 6] = best;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kThreads / 64; ++w) best = red[w] > best ? red[w] : best;
        part[(size_t)r * gridDim.x + blockIdx.x] = best;
    }
}

// One wave per row: the best of its chunks.
__global__ __launch_bounds__(64) void k_best_token(const uint64_t *__restrict__ part, int chunks,
                                                   int64_t *__restrict__ tokens) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < chunks; i += 64) {
        const uint64_t v = part[(size_t)blockIdx.x * chunks + i];
        best = v > best ? v : best;
    }
    best = max_over_wave(best);
    if (threadIdx.x == 0) tokens[blockIdx.x] = best ? (int64_t)(uint32_t)~(uint32_t)best : -1;
}

}  // namespace

size_t logits_scratch(int rows, int vocab, bool tokens) {
    if (!tokens) return 0;
    const int chunk = chunk_tokens(rows, vocab);
    return (size_t)rows * ((vocab + chunk - 1) / chunk) * sizeof(uint64_t);
}

int launch_logits(const LogitsParams &p, void *scratch, hipStream_t s) {
    const int chunk = chunk_tokens(p.rows, p.vocab), chunks = (p.vocab + chunk - 1) / chunk;
    uint64_t *part = p.tokens ? static_cast<uint64_t *>(scratch) : nullptr;
    const size_t lds = ((p.hist || p.nodes ? 1 : 0) + (p.n_bias ? 1 : 0)) * (size_t)chunk * 4;
    hipLaunchKernelGGL(k_logits, dim3(chunks, p.rows), dim3(kThreads), lds, s, p, chunk, part);
    TB_LAUNCHED();
    if (part) {
        hipLaunchKernelGGL(k_best_token, dim3(p.rows), dim3(64), 0, s, part, chunks, p.tokens);
        TB_LAUNCHED();
    }
    return TB_OK;
}

}  // namespace tb
