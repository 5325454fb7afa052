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

constexpr int kThreads = 512;
constexpr uint32_t kSeen = 1u << 31;   // of a token's LDS word: occurs in the history
constexpr uint32_t kBias = 1u << 30;   // has a bias; the rest: its count
constexpr uint32_t kCount = kBias - 1;
constexpr int kBiasList = kThreads;    // biases of one block kept in LDS
constexpr int kSums = 2048;            // tokens whose biases are added up at once, past that many

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

// What this wave wrote to LDS before is there for what it reads after.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

struct Biases {
    int at[kBiasList], token[kBiasList];   // the entries of the block's tokens
    int count;                             // how many there are (past kBiasList: not all listed)
};

// One block per row and chunk of the vocabulary.  Bound by the logits' bytes: they
// pass through once, 16 bytes a lane, four loads in flight (a lane whose four
// tokens the mask excludes reads none).  A word of LDS per token holds what the
// history, the tree path and the biases say of it; the block reads those lists whole,
// which is why chunks are as large as the row count lets them be.  64 rows of 128256
// tokens with one history of 2048 take 17.6 us (67 MB, 3.8 TB/s), 192 with one of 1500
// and 64 biases each 53 (202 MB, 3.8 TB/s), where a large copy reaches 5.1; chunks half
// as large change neither.
// Tokens with a bias are left to a second pass, a thread for each from a list in LDS:
// 200 biases of one block of 1500 tokens take 26 us, 180 where the threads that meet
// such tokens look them up.  MANY, where a call has more biases than that list holds:
// blocks with too many of them keep a sum for each of their tokens (500 in the list
// take 53 us, 520 as sums 17, 4000 for 300 tokens 91, all 151936 of a vocabulary 214).
// It is a kernel of its own: in one with it, 64 rows of 128256 took 21 us instead of 17.
// Vectors start where the row's address is a multiple of 16 bytes, `lead` tokens
// into it; LDS word 4 is the chunk's first vector, the words before it are chunk
// 0's tokens ahead of that.  The last vector may be cut.
template <bool VEC, bool MANY>
__global__ __launch_bounds__(kThreads) void k_logits(LogitsParams p, int chunk, uint64_t *part) {
    extern __shared__ uint32_t word[];
    __shared__ uint64_t red[kThreads / 64];
    __shared__ Biases bias;
    const int tid = threadIdx.x, r = blockIdx.y, V = p.vocab;
    const bool marked = p.hist || p.nodes || p.n_bias;
    const float *x = p.x + (size_t)r * V;
    float *y = p.y ? p.y + (size_t)r * V : nullptr;
    const int lead = VEC ? (int)((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / 4) : 0;
    const int v0 = lead + blockIdx.x * chunk;                     // the first vector's token
    const int t0 = blockIdx.x ? v0 : 0, t1 = min(V, v0 + chunk);   // the block's tokens
    if (marked) {
        for (int i = tid; i < chunk + 4; i += kThreads) word[i] = 0;
        if (tid == 0) bias.count = 0;
        __syncthreads();
    }
    uint32_t *at = word + 4 - v0;   // token t's word
    if (p.hist) {
        const int g = r / (p.rows / p.groups);
        const int len = p.history_len ? min(max(p.history_len[g], 0), p.hist) : p.hist;
        const int prompt = p.prompt_len ? p.prompt_len[g] : p.prompt;
        const int64_t *h = p.history + (size_t)g * p.hist;
        for (int i = tid; i < len; i += kThreads) {
            const int64_t t = h[i];
            if (t < t0 || t >= t1) continue;
            if (i < prompt) atomicOr(&at[t], kSeen);
            else atomicAdd(&at[t], 1u);
        }
    }
    if (p.nodes) {
        const int node = r % p.nodes, words = (p.nodes + 31) / 32;
        const int64_t *d = p.draft + (size_t)(r / p.nodes) * p.nodes;
        const int32_t *m = p.tree_mask + ((size_t)(r / p.nodes) * p.nodes + node) * words;
        for (int j = tid; j < p.nodes; j += kThreads) {
            const int64_t t = d[j];
            if (t >= t0 && t < t1 && ((uint32_t)m[j >> 5] >> (j & 31) & 1)) atomicAdd(&at[t], 1u);
        }
    }
    if (p.n_bias) {
        const size_t g = r / (p.rows / p.bias_groups);
        const int64_t *ids = p.bias_ids + g * p.n_bias;
        for (int i = tid; i < p.n_bias; i += kThreads) {
            const int64_t t = ids[i];
            if (t < t0 || t >= t1) continue;
            atomicOr(&at[t], kBias);
            const int j = atomicAdd(&bias.count, 1);
            if (j < kBiasList) {
                bias.at[j] = i;
                bias.token[j] = (int)t;
            }
        }
    }
    if (marked) __syncthreads();
    const float rep = p.rep_rows ? p.rep_rows[r] : p.rep;
    const float pres = p.pres_rows ? p.pres_rows[r] : p.pres;
    const float freq = p.freq_rows ? p.freq_rows[r] : p.freq;
    const uint32_t *allow =
        p.allowed ? reinterpret_cast<const uint32_t *>(p.allowed) + r * p.allowed_stride : nullptr;
    uint64_t best = 0;
    auto penalised = [&](float v, uint32_t w) {
        if (w & ~kBias) v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
        const uint32_t n = w & kCount;
        return n ? __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)n)), pres) : v;
    };
    auto candidate = [&](float v, int t) {
        if (!part) return;
        const uint64_t it = best_item(v, t);
        best = it > best ? it : best;
    };
    auto one = [&](float v, int t, uint32_t w, bool ok) {
        if (ok && (w & kBias)) return v;   // as it is, for the second pass
        if (w) v = penalised(v, w);
        v = ok ? v : -INFINITY;
        candidate(v, t);
        return v;
    };
    auto scalar = [&](int t) {
        const bool ok = !allow || (allow[t >> 5] >> (t & 31) & 1);
        const float v = one(ok ? x[t] : 0.f, t, marked ? at[t] : 0u, ok);
        if (y) y[t] = v;
    };
    if (VEC) {
        const int nv = t1 > v0 ? (t1 - v0) / 4 : 0;   // whole vectors
        constexpr int U = 4;
        for (int v = tid; v < nv; v += U * kThreads) {
            uint32_t ok[U];
            float4 f[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = v + u * kThreads, t = v0 + 4 * i, sh = t & 31;
                ok[u] = 0;
                if (i < nv) {
                    ok[u] = 15u;
                    if (allow) {
                        ok[u] = allow[t >> 5] >> sh;
                        if (sh > 28) ok[u] |= allow[(t >> 5) + 1] << (32 - sh);
                        ok[u] &= 15u;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                f[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (ok[u])
                    f[u] = *reinterpret_cast<const float4 *>(x + v0 + 4 * (v + u * kThreads));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = v + u * kThreads, t = v0 + 4 * i;
                if (i >= nv || (!ok[u] && !y)) continue;
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (marked) w = *reinterpret_cast<const uint4 *>(word + 4 + 4 * i);
                const float4 was = f[u];
                float4 z;
                z.x = one(was.x, t, w.x, ok[u] & 1);
                z.y = one(was.y, t + 1, w.y, ok[u] & 2);
                z.z = one(was.z, t + 2, w.z, ok[u] & 4);
                z.w = one(was.w, t + 3, w.w, ok[u] & 8);
                // in place, what stays is not written
                if (y && !(y == x && ok[u] == 15u && (w.x | w.y | w.z | w.w) == 0))
                    *reinterpret_cast<float4 *>(y + t) = z;
            }
        }
        if (t0 + tid < min(v0, t1)) scalar(t0 + tid);
        const int rest = v0 + 4 * nv;
        if (rest + tid < t1) scalar(rest + tid);
    } else {
        for (int t = t0 + tid; t < t1; t += kThreads) scalar(t);
    }
    if (p.n_bias) {
        __syncthreads();
        // The entries of a token are added up in the order of the list.
        auto biased = [&](int t, float s) {
            if (allow && !(allow[t >> 5] >> (t & 31) & 1)) return;
            const float v = __fadd_rn(penalised(x[t], at[t]), s);
            if (y) y[t] = v;
            candidate(v, t);
        };
        const size_t g = r / (p.rows / p.bias_groups);
        const int64_t *ids = p.bias_ids + g * p.n_bias;
        const float *val = p.bias + g * p.n_bias;
        const int n = bias.count;
        if (!MANY || n <= kBiasList) {   // one entry a thread: into the list's order, then added up
            int mine = 0, token = 0, rank = 0;
            if (tid < n) {
                mine = bias.at[tid];
                token = bias.token[tid];
                for (int k = 0; k < n; ++k) rank += bias.at[k] < mine;
            }
            __syncthreads();
            if (tid < n) {
                bias.at[rank] = mine;
                bias.token[rank] = token;
            }
            __syncthreads();
            bool first = tid < n;
            if (first) token = bias.token[tid];
            for (int k = 0; first && k < tid; ++k) first = bias.token[k] != token;
            if (first) {
                float v = val[bias.at[tid]];
                for (int k = tid + 1; k < n; ++k)
                    if (bias.token[k] == token) v = __fadd_rn(v, val[bias.at[k]]);
                biased(token, v);
            }
        } else if (MANY) {
            // kSums tokens at a time: each one's sum of biases, and whose turn it is to add to
            // it.  The list goes by in windows of an entry a thread; the entries of one token
            // take turns by their place in it, wave by wave and then lane by lane.
            float *sum = reinterpret_cast<float *>(word + chunk + 4);
            uint32_t *next = word + chunk + 4 + kSums;
            const uint32_t wave = tid >> 6, lane = tid & 63;
            for (int s0 = t0; s0 < t1; s0 += kSums) {
                const int s1 = min(t1, s0 + kSums);
                __syncthreads();
                for (int i = tid; i < kSums; i += kThreads) {
                    sum[i] = -0.f;   // -0 + v is v
                    next[i] = ~0u;
                }
                for (int i0 = 0; i0 < p.n_bias; i0 += kThreads) {
                    const int64_t id = i0 + tid < p.n_bias ? ids[i0 + tid] : -1;
                    bool waits = id >= s0 && id < s1;
                    const int i = waits ? (int)id - s0 : 0;
                    const float v = waits ? val[i0 + tid] : 0.f;
                    while (__syncthreads_or(waits)) {
                        if (waits) atomicMin(&next[i], wave);
                        __syncthreads();
                        const bool mine = waits && next[i] == wave;
                        __syncthreads();
                        waits = waits && !mine;
                        if (mine) next[i] = ~0u;
                        // lane by lane, the loop's end known to all of them: one that each lane
                        // left after its own turn could be compiled into a wait for itself
                        for (uint64_t todo = __ballot(mine); todo; todo &= todo - 1) {
                            wave_fence();
                            if (lane == (uint32_t)__builtin_ctzll(todo))
                                sum[i] = __fadd_rn(sum[i], v);
                        }
                    }
                }
                for (int t = s0 + tid; t < s1; t += kThreads)
                    if (at[t] & kBias) biased(t, sum[t - s0]);
            }
        }
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

// Tokens of one block: large enough that the lists are read few times, small
// enough that the rows fill the GPU (four blocks a CU).
int chunk_tokens(int rows, int vocab) {
    int chunk = 2048;
    while (chunk < 8192 && (int64_t)rows * ((vocab + 2 * chunk - 1) / (2 * chunk)) >= 512) chunk *= 2;
    return chunk;
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
    size_t lds = p.hist || p.nodes || p.n_bias ? (size_t)(chunk + 4) * 4 : 0;
    // Rows of x and y are equally far from a 16-byte boundary, or go word by word.
    const bool vec = !p.y || (reinterpret_cast<uintptr_t>(p.x) - reinterpret_cast<uintptr_t>(p.y)) % 16 == 0;
    const bool many = p.n_bias > kBiasList;   // a block may have more than its list holds
    if (many) lds += 2 * kSums * 4;
    auto *k = vec ? (many ? k_logits<true, true> : k_logits<true, false>)
                  : (many ? k_logits<false, true> : k_logits<false, false>);
    hipLaunchKernelGGL(k, dim3(chunks, p.rows), dim3(kThreads), lds, s, p, chunk, part);
    TB_LAUNCHED();
    if (part) {
        hipLaunchKernelGGL(k_best_token, dim3(p.rows), dim3(64), 0, s, part, chunks, p.tokens);
        TB_LAUNCHED();
    }
    return TB_OK;
}

}  // namespace tb
