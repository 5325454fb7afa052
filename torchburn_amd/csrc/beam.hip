// Beam search: the best continuations of a group of beams, and the beams' caches
// after them.
//
// Candidate (b, t) of a group has the value  score[b] + x[b][t] - log sum_u exp x[b][u];
// a finished beam has the single one (eos, score[b]).  The k largest are taken, of equal
// ones the lowest beam's and then the lowest token.  Values are kept in 64 bits, so that
// only what is equal ties: sums of exponentials, their logarithm and the values.
#include <math.h>

#include <algorithm>

#include "beam.hpp"
#include "tb_common.hpp"

namespace tb {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;

// A logit and its token as one number that orders as the logits do, equal ones by the
// lower token; 0 for what is never taken, -inf and NaN.
__device__ __forceinline__ uint32_t order_key(float y) {
    if (!(y > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(y == 0.f ? 0.f : y);   // -0 ties with 0
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// e^d of d <= 0 in 64 bits (2^-52 and the sum's own roundings): 2^t as a Taylor sum of
// degree 10 on t's fraction, 2e-13 past it.
__device__ __forceinline__ double exp64(double d) {
    const double t = d * 1.44269504088896340736, n = rint(t), f = t - n;
    constexpr double c[11] = {1.0, 0.69314718055994530942, 0.24022650695910071233,
                              0.055504108664821579953, 0.0096181291076284771619,
                              0.0013333558146428443423, 0.00015403530393381609954,
                              1.5252733804059840280e-05, 1.3215486790144309489e-06,
                              1.0178086009239699728e-07, 7.0549116208011233299e-09};
    double p = c[10];
#pragma unroll
    for (int i = 9; i >= 0; --i) p = fma(p, f, c[i]);
    return d < -700.0 ? 0.0 : ldexp(p, (int)n);   // NaN stays NaN
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
    const uint32_t lo = __shfl_xor((uint32_t)v, o), hi = __shfl_xor((uint32_t)(v >> 32), o);
    return ((uint64_t)hi << 32) | lo;
}

// The k-th largest of a wave's N numbers a lane (0: none), which differ unless 0; 1 when
// there are fewer than k.  Bit by bit, the count of those not below by ballots: first the
// keys, then, only where several are equal at the border, the rest.
template <int N>
__device__ __forceinline__ uint64_t kth_largest(const uint64_t (&v)[N], int k) {
    auto count = [&](uint64_t least) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) n += __popcll(__ballot(v[i] >= least));
        return n;
    };
    if (count(1) < k) return 1;
    uint64_t at = 0;
    for (int bit = 63; bit >= 0; --bit) {
        const uint64_t to = at | (1ull << bit);
        const int n = count(to);
        if (n < k) continue;
        at = to;
        if (n == k) break;
    }
    return at ? at : 1;
}

// What this wave wrote to LDS before is there for what it reads after.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A chunk's exponentials, at most 1 each and 2^13 of them, are multiples of 2^-kGrid: their
// sum takes 53 bits.  (e + kRound) - kRound is e so rounded.
constexpr int kGrid = 40;
constexpr double kRound = 1.5 * (double)(1ull << (52 - kGrid));

// A chunk's sum of exponentials: that of e^(x - top).
struct Part {
    double sum, top;
};

// One block per row and chunk of 1024 U tokens, whose logits stay in registers: the
// largest, the sum of exponentials from it, and the k largest logits in order.  The k-th
// largest of the threads' own largest bounds the k-th largest of all from below, so that
// few logits are collected in LDS, at most the 4 U + 1 of each of k threads; they are
// ranked there.  Exponentials are rounded to multiples of 2^-kGrid, whose sums are exact,
// so that rows that are alike have sums that are alike, however they lie in memory:
// vectors start where the row's address is a multiple of 16 bytes, `lead` tokens ahead of
// the chunk's first, and its last `lead` tokens are left to a thread each.
//
// Bound by the logits' bytes.
template <int U>
__global__ __launch_bounds__(kThreads) void k_beam_chunk(BeamSelect p, Part *__restrict__ parts,
                                                         uint64_t *__restrict__ best) {
    extern __shared__ uint64_t items[];   // [(4 U + 1) k]
    __shared__ uint64_t top_of[kThreads];
    __shared__ double sums[kThreads / 64];
    __shared__ int found;
    const int tid = threadIdx.x, row = blockIdx.y, V = p.vocab;
    if (p.finished && p.finished[row]) return;
    const float *x = p.logits + (size_t)row * V;
    const int lead = (int)(reinterpret_cast<uintptr_t>(x) % 16 / 4);
    const int c0 = blockIdx.x * 1024 * U, c1 = min(V, c0 + 1024 * U);
    const int t0 = c0 - lead + 4 * tid;   // of vector 0
    float v[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int t = t0 + 1024 * u;
        if (t >= c0 && t + 3 < c1) {
            const float4 y = *reinterpret_cast<const float4 *>(x + t);
            v[u][0] = y.x; v[u][1] = y.y; v[u][2] = y.z; v[u][3] = y.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[u][i] = t + i >= c0 && t + i < c1 ? x[t + i] : -INFINITY;
        }
    }
    const int t_rest = c0 + 1024 * U - lead + tid;
    const float rest = tid < lead && t_rest < c1 ? x[t_rest] : -INFINITY;
    auto item = [](float y, int t) { return ((uint64_t)order_key(y) << 32) | (uint32_t)~t; };
    uint64_t mine = 0;
    auto larger = [&](float y, int t) {
        const uint64_t it = item(y, t);
        if (it >> 32 && it > mine) mine = it;
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) larger(v[u][i], t0 + 1024 * u + i);
    if (lead) larger(rest, t_rest);
    top_of[tid] = mine;
    if (tid == 0) found = 0;
    __syncthreads();
    // ---- each wave for itself: the chunk's largest, and the border
    uint64_t tops[4], top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        tops[i] = top_of[(tid & 63) + 64 * i];
        top = max(top, tops[i]);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) top = max(top, shfl_xor64(top, o));
    const uint64_t least = kth_largest<4>(tops, p.k);
    const float least_logit = least == 1 ? -INFINITY : key_logit((uint32_t)(least >> 32));
    auto collect = [&](float y, int t) {
        if (y >= least_logit) {
            const uint64_t it = item(y, t);
            if (it >> 32 && it >= least) items[atomicAdd(&found, 1)] = it;
        }
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) collect(v[u][i], t0 + 1024 * u + i);
    if (lead) collect(rest, t_rest);
    // ---- the sum; nothing to take: 0 from 0, or NaN (a NaN or an infinity makes one)
    const double ref = top ? (double)key_logit((uint32_t)(top >> 32)) : 0.0;
    double sum = 0.0;
    auto add = [&](float y) { sum += (exp64((double)y - ref) + kRound) - kRound; };
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) add(v[u][i]);
    if (lead) add(rest);
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if ((tid & 63) == 0) sums[tid >> 6] = sum;
    __syncthreads();
    const size_t at = (size_t)row * gridDim.x + blockIdx.x;
    if (tid == 0) parts[at] = {(sums[0] + sums[1]) + (sums[2] + sums[3]), ref};
    const int n = found;
    uint64_t *to = best + at * p.k;
    for (int i = tid; i < n; i += kThreads) {
        const uint64_t it = items[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += items[j] > it;
        if (rank < p.k) to[rank] = it;
    }
    for (int i = n + tid; i < p.k; i += kThreads) to[i] = 0;
}

// A row's k largest of a group, ready to be ranked among the other rows'.
struct Pick {
    double value;
    uint64_t item;
};

// One block per group.  A wave takes its rows in turn: the row's sum of exponentials from its
// chunks', and its k largest logits from theirs (again by a border, and ranked in LDS).
// Then each of them is ranked among the group's, by a search in every row's list.
// Bound by the launch and the waits of these steps.
__global__ __launch_bounds__(1024) void k_beam_pick(BeamSelect p, const Part *__restrict__ parts,
                                                    const uint64_t *__restrict__ best, int chunks,
                                                    int cap) {
    extern __shared__ uint64_t lds[];   // picks [beams][k], then items [waves][cap]
    __shared__ int counts[16], lengths[kMaxBeams];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    const int k = p.k, group = blockIdx.x;
    Pick *pick = reinterpret_cast<Pick *>(lds);
    uint64_t *items = lds + 2 * (size_t)p.beams * k + (size_t)wave * cap;
    for (int b = wave; b < p.beams; b += waves) {
        const int row = group * p.beams + b;
        const float score = p.scores[row];
        Pick *out = pick + b * k;
        const bool fin = score - score == 0.f;   // an infinite or NaN score: no candidates
        if (!fin || (p.finished && p.finished[row])) {
            if (lane == 0) {
                out[0] = {(double)score, (uint32_t)~(uint32_t)p.eos};
                lengths[b] = fin ? 1 : 0;
            }
            continue;
        }
        // ---- the row's log of its sum of exponentials
        const Part *pt = parts + (size_t)row * chunks;
        double top = -INFINITY, sum = 0.0;
        for (int c = lane; c < chunks; c += 64) {
            const Part x = pt[c];
            if (x.sum != 0.0) top = fmax(top, x.top);
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) top = fmax(top, __shfl_xor(top, o));
        for (int c = lane; c < chunks; c += 64) {
            const Part x = pt[c];
            if (x.sum != 0.0) sum += x.sum * exp64(x.top - top);
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
        const double lse = top + log(sum);
        // ---- its k largest logits
        const uint64_t *src = best + (size_t)row * chunks * k;
        const int total = chunks * k;
        uint64_t mine[1] = {0};
        for (int i = lane; i < total; i += 64) mine[0] = max(mine[0], src[i]);
        const uint64_t least = kth_largest<1>(mine, k);
        if (lane == 0) counts[wave] = 0;
        wave_fence();
        for (int i = lane; i < total; i += 64) {
            const uint64_t it = src[i];
            if (it >= least) items[atomicAdd(&counts[wave], 1)] = it;
        }
        wave_fence();
        const int n = counts[wave];
        int length = 0;
        for (int i = lane; i < n; i += 64) {
            const uint64_t it = items[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += items[j] > it;
            const double value = (double)key_logit((uint32_t)(it >> 32)) - lse + (double)score;
            if (rank < k && value > -INFINITY) {   // not NaN
                out[rank] = {value, it};
                ++length;
            }
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) length += __shfl_xor(length, o);
        if (lane == 0) lengths[b] = length;
        wave_fence();   // the items are the next row's
    }
    __syncthreads();
    int total = 0;
    for (int b = 0; b < p.beams; ++b) total += lengths[b];
    float *scores = p.out_scores + (size_t)group * k;
    int64_t *tokens = p.tokens + (size_t)group * k, *parents = p.parents + (size_t)group * k;
    for (int i = tid; i < p.beams * k; i += blockDim.x) {
        const int b = i / k, j = i - b * k;
        if (j >= lengths[b]) continue;
        const Pick mine = pick[i];
        int rank = j;
        for (int r = 0; r < p.beams; ++r) {
            if (r == b) continue;
            // how many of row r come before: those of larger values, in lower rows equal ones too
            int lo = 0, hi = lengths[r];
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                const double v = pick[r * k + mid].value;
                if (v > mine.value || (v == mine.value && r < b)) lo = mid + 1;
                else hi = mid;
            }
            rank += lo;
        }
        if (rank >= k) continue;
        scores[rank] = (float)mine.value;
        tokens[rank] = (uint32_t)~(uint32_t)mine.item;
        parents[rank] = b;
    }
    for (int i = total + tid; i < k; i += blockDim.x) {
        scores[i] = -INFINITY;
        tokens[i] = parents[i] = -1;
    }
}

// Vectors a thread: as few as leave at most 2048 blocks, and at most 32 a row (128 of the largest
// vocabulary).
int vectors(int rows, int vocab) {
    for (int u = 1; u < 8; u *= 2) {
        const int64_t chunks = (vocab + 1024 * u - 1) / (1024 * u);
        if (chunks <= 32 && rows * chunks <= 2048) return u;
    }
    return 8;
}
int chunks_of(int vocab, int u) { return (vocab + 1024 * u - 1) / (1024 * u); }

// ---- the caches ---------------------------------------------------------------

struct LayerCaches {
    float *k[kBeamLayersPerLaunch], *v[kBeamLayersPerLaunch];
};

// A thread has the same 16 bytes of every beam: it reads what any beam takes over, then
// writes, so that the rows change places without a copy beside them.  Blocks go along a
// group's positions and heads, whose number only the device may know.  A beam that goes on
// from itself, or from none, is neither read nor written.
// Bound by the bytes moved.
// Grid (units side by side, 2 * layers, groups).
template <int NB>
__global__ __launch_bounds__(256) void k_beam_reorder(BeamReorder p, LayerCaches lc) {
    __shared__ int from[NB], until[NB];
    const int t = threadIdx.x, group = blockIdx.z, layer = blockIdx.y >> 1;
    if (t < NB) {
        int src = -1, n = 0;
        if (t < p.beams) {
            const int64_t b = p.parents[(size_t)group * p.beams + t];
            if (b >= 0 && b < p.beams && b != t) {
                src = (int)b;
                n = p.lens ? p.lens[(size_t)group * p.beams + src] : p.len;
            }
        }
        from[t] = src;
        until[t] = min(max(n, 0), p.max_seq);
    }
    __syncthreads();
    int src[NB], len[NB], most = 0;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        src[j] = __builtin_amdgcn_readfirstlane(from[j]);
        len[j] = __builtin_amdgcn_readfirstlane(until[j]);
        most = max(most, len[j]);
    }
    const bool is_v = blockIdx.y & 1;
    const int64_t sb = is_v ? p.vsb : p.ksb, sh = is_v ? p.vsh : p.ksh, ss = is_v ? p.vss : p.kss;
    float *base = (is_v ? lc.v[layer] : lc.k[layer]) + group * (is_v ? p.vsg : p.ksg);
    const int cols = p.hd / 4, each = 256 / cols, pos = t / cols, col = t - pos * cols;
    const int steps = (most + each - 1) / each;      // of a head
    for (int64_t unit = blockIdx.x; unit < (int64_t)steps * p.hkv; unit += gridDim.x) {
        const int head = (int)(unit / steps), at = (int)(unit - (int64_t)head * steps) * each + pos;
        if (pos >= each) continue;
        float *here = base + head * sh + at * ss + 4 * col;
        f32x4 v[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            v[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (at < len[j]) v[j] = *reinterpret_cast<const f32x4 *>(here + src[j] * sb);
        }
#pragma unroll
        for (int j = 0; j < NB; ++j)
            if (at < len[j]) *reinterpret_cast<f32x4 *>(here + j * sb) = v[j];
    }
}

}  // namespace

size_t beam_select_scratch(int groups, int beams, int vocab, int k) {
    const size_t chunks = chunks_of(vocab, vectors(groups * beams, vocab));
    return (size_t)groups * beams * chunks * (sizeof(Part) + k * sizeof(uint64_t));
}

int launch_beam_select(const BeamSelect &p, void *scratch, hipStream_t s) {
    const int rows = p.groups * p.beams, u = vectors(rows, p.vocab), chunks = chunks_of(p.vocab, u);
    Part *parts = static_cast<Part *>(scratch);
    uint64_t *best = reinterpret_cast<uint64_t *>(parts + (size_t)rows * chunks);
    const size_t lds = (size_t)(4 * u + 1) * p.k * sizeof(uint64_t);
    auto *k = u == 1 ? k_beam_chunk<1> : u == 2 ? k_beam_chunk<2> : u == 4 ? k_beam_chunk<4> : k_beam_chunk<8>;
    hipLaunchKernelGGL(k, dim3(chunks, rows), dim3(kThreads), lds, s, p, parts, best);
    TB_LAUNCHED();
    // A lane's items are each its largest at most: so many pass the border.
    const int cap = p.k * ((chunks * p.k + 63) / 64);
    const size_t picks = (size_t)p.beams * p.k * sizeof(Pick);
    int waves = std::min(16, p.beams);
    while (waves > 1 && picks + (size_t)waves * cap * sizeof(uint64_t) > (64 << 10)) --waves;
    const size_t need = picks + (size_t)waves * cap * sizeof(uint64_t);
    if (need > (64 << 10))
        TB_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(k_beam_pick),
                                   hipFuncAttributeMaxDynamicSharedMemorySize, (int)need));
    hipLaunchKernelGGL(k_beam_pick, dim3(p.groups), dim3(64 * waves), need, s, p, parts, best,
                       chunks, cap);
    TB_LAUNCHED();
    return TB_OK;
}

int launch_beam_reorder(const BeamReorder &p, float *const *kc, float *const *vc, hipStream_t s) {
    for (int l0 = 0; l0 < p.layers; l0 += kBeamLayersPerLaunch) {
        LayerCaches lc{};
        const int layers = std::min(kBeamLayersPerLaunch, p.layers - l0);
        for (int l = 0; l < layers; ++l) {
            lc.k[l] = kc[l0 + l];
            lc.v[l] = vc[l0 + l];
        }
        const int each = 256 / (p.hd / 4), most = p.lens ? p.max_seq : p.len;
        const int64_t units = (int64_t)p.hkv * ((most + each - 1) / each);
        const int64_t want = std::max<int64_t>(1, 8192 / ((int64_t)2 * layers * p.groups));
        const dim3 grid((uint32_t)std::max<int64_t>(1, std::min(units, want)), 2 * layers, p.groups);
        auto *k = p.beams <= 4    ? k_beam_reorder<4>
                  : p.beams <= 8  ? k_beam_reorder<8>
                  : p.beams <= 16 ? k_beam_reorder<16>
                  : p.beams <= 32 ? k_beam_reorder<32>
                                  : k_beam_reorder<64>;
        hipLaunchKernelGGL(k, grid, dim3(256), 0, s, p, lc);
        TB_LAUNCHED();
    }
    return TB_OK;
}

}  // namespace tb
