// Beam search: the best continuations of a group of beams, and the beams' caches
// after them.
//
// Candidate (b, t) of a group has the value  score[b] + x[b][t] - log sum_u exp x[b][u];
// a finished beam has the single one (eos, score[b]).  The k largest are taken, of equal
// ones the lowest beam's and then the lowest token.  Sums of exponentials, their logarithm and
// the values are kept in 64 bits; the exponentials are a fit to 5.5e-11, which with the
// argument's rounding, 3.4e-16 of the logit, is a row's error.  So the order is exact among a
// row's tokens, that of 64 bits among rows that are alike, whose errors are equal, and good to
// 2e-10 between others.
#include <float.h>
#include <math.h>

#include <algorithm>

#include "beam.hpp"
#include "tb_common.hpp"

namespace tb {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kThreads = 256;
constexpr double kLog2e = 1.44269504088896340736, kLn2 = 0.69314718055994530942;

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
    const double t = d * kLog2e, n = rint(t), f = t - n;
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

// A chunk's sum of exponentials: that of e^(x - top).
struct Part {
    double sum, top;
};

// A fit of degree 7 to 2^f on +-1/2, 5.5e-11 of it off at most.
constexpr double kMagic = 1.5 * (double)(1ull << 52);   // y + kMagic has rint(y) in its low word
__device__ __forceinline__ double exp2_fit(double f) {
    constexpr double c[8] = {0.9999999999595618,    0.6931471805568324,   0.24022651213498092,
                             0.055504109063258665,  0.009618025613318034, 0.0013333478473685416,
                             0.00015469729214118296, 1.5303700711365693e-05};
    double p = c[7];
#pragma unroll
    for (int i = 6; i >= 0; --i) p = fma(p, f, c[i]);
    return p;
}

// One block per row and chunk of 1024 U tokens, whose logits stay in registers: the
// largest, the sum of exponentials from it, and the k largest logits in order.  The k-th
// largest of the threads' own largest bounds the k-th largest of all from below, so that
// few logits are collected in LDS, at most the 4 U of each of k threads; they are ranked
// there.  Where logits that are equal at this border make them more, the border is found
// anew with the tokens, which differ.  Threads take tokens by their number, not by their
// address (rows of an odd vocabulary are read in vectors that are not aligned), so that rows
// that are alike have sums that are alike to the last bit.
//
// Bound by the logits' bytes, 27 us of 131 MB, and the exponentials, 14 instructions in 64
// bits each: 256 rows of 128256 take 32.7 us with seven blocks a CU, for which U = 8 spills 8
// registers, 37.8 with the five that they would have without, 59.6 where blocks ask for their
// next chunk ahead and three fit, 56.8 with a Taylor sum of degree 10 and the border by every
// wave from logits and tokens.
template <int U>
__global__ __launch_bounds__(kThreads, 7) void k_beam_chunk(BeamSelect p, Part *__restrict__ parts,
                                                         uint64_t *__restrict__ best) {
    extern __shared__ uint64_t items[];   // [4 U k]
    __shared__ uint64_t top_of[kThreads];
    __shared__ uint32_t keys[kThreads];
    __shared__ double sums[kThreads / 64];
    __shared__ float tops[kThreads / 64], border;
    __shared__ int found, bad;
    const int tid = threadIdx.x, row = blockIdx.y, V = p.vocab;
    if (p.finished && p.finished[row]) return;
    const float *x = p.logits + (size_t)row * V;
    const int c0 = blockIdx.x * 1024 * U, t0 = c0 + 4 * tid;
    float v[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int t = t0 + 1024 * u;
        if (t + 3 < V) {
            const f32x4_any y = *reinterpret_cast<const f32x4_any *>(x + t);
            v[u][0] = y.x; v[u][1] = y.y; v[u][2] = y.z; v[u][3] = y.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[u][i] = t + i < V ? x[t + i] : -INFINITY;
        }
    }
    if (tid == 0) found = bad = 0;
    // ---- the largest
    float mine = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            mine = fmaxf(mine, v[u][i]);
            nan |= v[u][i] != v[u][i];
        }
    keys[tid] = order_key(mine);
    float top = mine;
#pragma unroll
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
    if (__any(nan) && (tid & 63) == 0) bad = 1;
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    // ---- one wave: the border
    if (tid < 64) {
        const uint32_t k4[4] = {keys[tid], keys[tid + 64], keys[tid + 128], keys[tid + 192]};
        uint32_t at = 0;
        for (int bit = 31; bit >= 0; --bit) {   // the k-th largest, or 0 where there are fewer
            const uint32_t to = at | (1u << bit);
            int n = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) n += __popcll(__ballot(k4[i] >= to));
            if (n < p.k) continue;
            at = to;
            if (n == p.k) break;
        }
        // keys up to that of -inf stand for nothing that is taken
        if (tid == 0) border = at <= 0x007FFFFFu ? -FLT_MAX : fmaxf(key_logit(at), -FLT_MAX);
    }
    // ---- the sum from 2^-n, n the largest one's exponent
    double sum = 0.0, ref = 0.0;
    if (fabsf(top) < 524288.f) {
        const double n = rint((double)top * kLog2e), low = n - kMagic;
        const float least = top - 80.f;   // e^-80 for -inf, which is no part of the sum
        ref = n * kLn2;
        auto add = [&](float y) {
            const double t = (double)fmaxf(y, least) * kLog2e, r = t - low;   // rint(t) - n
            const double e = exp2_fit(t - (r + low));
            const int up = (int)__double2loint(r);
            sum += __hiloint2double(__double2hiint(e) + (up << 20), __double2loint(e));
        };
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) add(v[u][i]);
    } else if (top > -INFINITY) {   // far out, or infinite, which makes it NaN
        ref = top;
        auto add = [&](float y) { sum += exp64((double)y - ref); };
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) add(v[u][i]);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if ((tid & 63) == 0) sums[tid >> 6] = sum;
    __syncthreads();
    const size_t at = (size_t)row * gridDim.x + blockIdx.x;
    if (tid == 0) {
        sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        parts[at] = {bad ? (double)NAN : sum, ref};
    }
    // ---- what is not below the border
    const int cap = 4 * U * p.k;
    const float least = border;
    auto item = [](float y, int t) { return ((uint64_t)order_key(y) << 32) | (uint32_t)~t; };
    auto collect = [&](float y, int t) {
        if (y >= least) {
            const int i = atomicAdd(&found, 1);
            if (i < cap) items[i] = item(y, t);
        }
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) collect(v[u][i], t0 + 1024 * u + i);
    __syncthreads();
    int n = found;
    if (n > cap) {   // many equal ones: the border among the threads' best tokens of them
        uint64_t most = 0;
        auto larger = [&](float y, int t) {
            const uint64_t it = item(y, t);
            if (it >> 32 && it > most) most = it;
        };
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) larger(v[u][i], t0 + 1024 * u + i);
        top_of[tid] = most;
        __syncthreads();
        if (tid == 0) found = 0;
        uint64_t all[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) all[i] = top_of[(tid & 63) + 64 * i];
        const uint64_t bound = kth_largest<4>(all, p.k);
        __syncthreads();
        auto again = [&](float y, int t) {
            const uint64_t it = item(y, t);
            if (it >> 32 && it >= bound) items[atomicAdd(&found, 1)] = it;
        };
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) again(v[u][i], t0 + 1024 * u + i);
        __syncthreads();
        n = found;
    }
    uint64_t *to = best + at * p.k;
    for (int i = tid; i < n; i += kThreads) {
        const uint64_t it = items[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += items[j] > it;
        if (rank < p.k) to[rank] = it;
    }
    for (int i = n + tid; i < p.k; i += kThreads) to[i] = 0;
}

constexpr int kAhead = 8;   // a lane's items of a row that are requested at once
constexpr int kPickWaves = 16;
// LDS of k_beam_pick: what every block has, and what the launch adds.  A launch may have 64 KiB in
// all by itself; for more the kernel's limit is set to the most that any call takes, with 64
// beams, 64 results and 128 chunks: it is one for all threads of the process, so that a limit of
// the call's own size could be another's between its set and its launch.
constexpr size_t kPickStatic = (kPickWaves + kMaxBeams) * sizeof(int);
constexpr size_t kPickPlain = (64 << 10) - kPickStatic;
constexpr size_t kPickMost = 128 << 10;

// A row's k largest of a group, ready to be ranked among the other rows'.
struct Pick {
    double value;
    uint64_t item;
};

// One block per group.  A wave takes its rows in turn: the row's sum of exponentials from its
// chunks', and its k largest logits from theirs (again by a border, and ranked in LDS).
// Then each of them is ranked among the group's, by a search in every row's list.
// Bound by the launch and the waits of these steps: 9.1 us for 32 groups of 8 beams, 16 chunks
// and k = 16, 6.0 for one of 4 beams, 32 chunks and k = 8.
__global__ __launch_bounds__(64 * kPickWaves) void k_beam_pick(
    BeamSelect p, const Part *__restrict__ parts, const uint64_t *__restrict__ best, int chunks,
    int cap) {
    extern __shared__ uint64_t lds[];   // picks [beams][k], then items [waves][cap]
    __shared__ int counts[kPickWaves], lengths[kMaxBeams];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    const int k = p.k, group = blockIdx.x;
    Pick *pick = reinterpret_cast<Pick *>(lds);
    uint64_t *items = lds + 2 * (size_t)p.beams * k + (size_t)wave * cap;
    for (int b = wave; b < p.beams; b += waves) {
        const int row = group * p.beams + b;
        // What will be read is requested at once.
        const float score = p.scores[row];
        const bool done = p.finished && p.finished[row];
        const Part *pt = parts + (size_t)row * chunks;
        const uint64_t *src = best + (size_t)row * chunks * k;
        const int total = chunks * k;
        const Part first = pt[min(lane, chunks - 1)];
        uint64_t ahead[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ahead[i] = src[min(lane + 64 * i, total - 1)];
        Pick *out = pick + b * k;
        const bool fin = score - score == 0.f;   // an infinite or NaN score: no candidates
        if (!fin || done) {
            if (lane == 0) {
                out[0] = {(double)score, (uint32_t)~(uint32_t)p.eos};
                lengths[b] = fin ? 1 : 0;
            }
            continue;
        }
        // ---- the row's log of its sum of exponentials
        double top = -INFINITY, sum = 0.0;
        auto each = [&](auto f) {
            if (lane < chunks) f(first);
            for (int c = lane + 64; c < chunks; c += 64) f(pt[c]);
        };
        each([&](const Part &x) {
            if (x.sum != 0.0) top = fmax(top, x.top);
        });
#pragma unroll
        for (int o = 32; o; o >>= 1) top = fmax(top, __shfl_xor(top, o));
        each([&](const Part &x) {
            if (x.sum != 0.0) sum += x.sum * exp64(x.top - top);
        });
#pragma unroll
        for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
        const double lse = top + log(sum);
        // ---- its k largest logits
        uint64_t mine[1] = {0};
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (lane + 64 * i < total) mine[0] = max(mine[0], ahead[i]);
        for (int i = lane + 64 * kAhead; i < total; i += 64) mine[0] = max(mine[0], src[i]);
        const uint64_t least = kth_largest<1>(mine, k);
        if (lane == 0) counts[wave] = 0;
        wave_fence();
        auto collect = [&](uint64_t it) {
            if (it >= least) items[atomicAdd(&counts[wave], 1)] = it;
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (lane + 64 * i < total) collect(ahead[i]);
        for (int i = lane + 64 * kAhead; i < total; i += 64) collect(src[i]);
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
    // Several lanes share an item where the block has them.
    int share = 1;
    while (share < 8 && 2 * share * p.beams * k <= (int)blockDim.x) share *= 2;
    for (int i0 = 0; i0 < p.beams * k; i0 += blockDim.x / share) {
        const int i = i0 + tid / share, b = i / k, j = i - b * k;
        const bool real = b < p.beams && j < lengths[min(b, p.beams - 1)];
        const Pick mine = pick[real ? i : 0];
        int rank = 0;
        for (int r = tid % share; r < p.beams && real; r += share) {
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
        for (int o = 1; o < share; o <<= 1) rank += __shfl_xor(rank, o);
        rank += j;
        if (!real || tid % share || rank >= k) continue;
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
// Bound by the bytes moved: 32 layers of four groups of eight beams, 93 positions of 8 heads of
// 128, 631 MB, 151 us and 4.2 TB/s, where a large copy reaches 4.9; 157 with ordinary stores.
// Two groups of 16 beams, one of 32 and one of 64 (32, 32 and 16 layers of that) move at 4.4, 5.1
// and 4.9 TB/s, although 34, 146 and 372 scalar registers spill and the last has a wave a SIMD.
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
            if (at < len[j])
                __builtin_nontemporal_store(v[j], reinterpret_cast<f32x4 *>(here + j * sb));
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
    const size_t lds = (size_t)4 * u * p.k * sizeof(uint64_t);
    auto *k = u == 1   ? k_beam_chunk<1>
              : u == 2 ? k_beam_chunk<2>
              : u == 4 ? k_beam_chunk<4>
                       : k_beam_chunk<8>;
    hipLaunchKernelGGL(k, dim3(chunks, rows), dim3(kThreads), lds, s, p, parts, best);
    TB_LAUNCHED();
    // A lane's items are each its largest at most: so many pass the border.
    const int cap = p.k * ((chunks * p.k + 63) / 64);
    const size_t picks = (size_t)p.beams * p.k * sizeof(Pick);
    int waves = std::min(kPickWaves, p.beams);
    while (waves > 1 && picks + (size_t)waves * cap * sizeof(uint64_t) > kPickPlain) --waves;
    const size_t need = picks + (size_t)waves * cap * sizeof(uint64_t);
    if (need > kPickPlain)
        TB_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(k_beam_pick),
                                   hipFuncAttributeMaxDynamicSharedMemorySize, (int)kPickMost));
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
        // us at 512 / 1024 / 2048 / 4096 blocks in all: 160 / 155 / 151 / 152 (k_beam_reorder)
        const int64_t want = std::max<int64_t>(1, 2048 / ((int64_t)2 * layers * p.groups));
        const dim3 grid((uint32_t)std::max<int64_t>(1, std::min(units, want)), 2 * layers,
                        p.groups);
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
