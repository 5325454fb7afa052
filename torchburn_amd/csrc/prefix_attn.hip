// Attention of sequences that share a prefix: each query row over its group's
// prefix, whose K and V are read once for all of the group's rows, and over its
// own cache, for GQA and f32 caches.
//
//   o = sum_p w_p v_p / sum_p w_p,  w_p = exp(scale q.k_p - m)
//
// over the prefix's positions and the row's own ones.  One pass over K and V with a
// running reference m and sum; the positions are split over blocks, whose
// results are merged in the order of the splits.
#include <math.h>

#include <algorithm>

#include "prefix.hpp"
#include "tb_common.hpp"

namespace tb {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMaxSplits = 64;   // of the prefix, and of a row's own cache
// A row's reference is set this far (in powers of two) above a score that passes it, so
// that the outputs' rescale runs in few tiles; weights stay below 1.
constexpr float kLead = 8.f;

// f over the lanes c, c + 16, c + 32, c + 48: a swap of 16- or 32-lane halves of a
// register with itself leaves both halves' values in every lane.
template <class F>
__device__ __forceinline__ float over_groups(float v, F f) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_over_groups(float v) {
    return over_groups(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float sum_over_groups(float v) {
    return over_groups(v, [](float a, float b) { return a + b; });
}

__device__ __forceinline__ int length(const int32_t *lens, int len, int i, int most) {
    return min(max(lens ? lens[i] : len, 0), most);
}

// What one block works on: query rows i0 .. i1 - 1 of one KV head of one group (row i is
// sequence i / G's query head i % G of the KV head's G) over the positions of one cache.
struct Job {
    const float *k, *v;   // the KV head's rows
    int64_t ks, vs;
    int group, kvh, i0, i1;
    int slot;             // its place among the partial results
    int t0, t1, len;      // tiles of the positions below len
    bool none;            // this split is not among the cache's
};

// The plan of a launch; the blocks' order: the prefix's, then the sequences' own.
struct Plan {
    int rb;               // 16 * rb rows a block
    int ptiles, gtiles;   // row tiles of a group's rows, of a sequence's
    int pcap, ocap;       // splits at most
    int pblocks, oblocks;
    int slots;            // partial results a row; 1: none, the output itself
};

// Split `split` of a cache of len positions where at most cap are wanted: only the length
// counts, so that within one plan a result is the same whatever the bound.
constexpr int kTile = 16, kMinTiles = 4;
struct Range {
    int t0, t1, splits;
};
__device__ __forceinline__ Range split_range(int len, int cap, int split) {
    const int tiles = (len + kTile - 1) / kTile;
    const int each = max((tiles + cap - 1) / cap, kMinTiles);
    return {min(split * each, tiles), min((split + 1) * each, tiles), (tiles + each - 1) / each};
}

// KV heads first: the row tiles that read the same K and V are a multiple of the KV
// heads apart, on one of the eight dies (block i goes to die i % 8) where those are 8.
__device__ __forceinline__ Job job_of(const PrefixAttn &a, const Plan &p, int block) {
    Job j;
    const int G = a.hq / a.hkv, rows = 16 * p.rb;
    if (block < p.pblocks) {
        j.kvh = block % a.hkv;
        block /= a.hkv;
        const int rt = block % p.ptiles;
        block /= p.ptiles;
        const int split = block % p.pcap;
        j.group = block / p.pcap;
        j.i0 = rt * rows;
        j.i1 = min(j.i0 + rows, a.rows * G);
        j.k = a.kp.p + j.group * a.kp.sb + j.kvh * a.kp.sh;
        j.v = a.vp.p + j.group * a.vp.sb + j.kvh * a.vp.sh;
        j.ks = a.kp.ss;
        j.vs = a.vp.ss;
        j.len = length(a.prefix_lens, a.prefix_len, j.group, a.max_prefix);
        const Range r = split_range(j.len, p.pcap, split);
        j.t0 = r.t0;
        j.t1 = r.t1;
        j.none = split >= r.splits;
        j.slot = split;
    } else {
        block -= p.pblocks;
        j.kvh = block % a.hkv;
        block /= a.hkv;
        const int gt = block % p.gtiles;
        block /= p.gtiles;
        const int split = block % p.ocap, seq = block / p.ocap;
        j.group = seq / a.rows;
        const int i = (seq - j.group * a.rows) * G;
        j.i0 = i + gt * rows;
        j.i1 = min(j.i0 + rows, i + G);
        j.k = a.k.p + seq * a.k.sb + j.kvh * a.k.sh;
        j.v = a.v.p + seq * a.v.sb + j.kvh * a.v.sh;
        j.ks = a.k.ss;
        j.vs = a.v.ss;
        j.len = length(a.own_lens, a.own_len, seq, a.max_own);
        const Range r = split_range(j.len, p.ocap, split);
        j.t0 = r.t0;
        j.t1 = r.t1;
        j.none = split >= r.splits;
        j.slot = p.pcap + split;
    }
    return j;
}

__device__ __forceinline__ size_t row_of(const PrefixAttn &a, const Job &j, int i) {
    const int G = a.hq / a.hkv;
    return ((size_t)j.group * a.rows + i / G) * a.hq + j.kvh * G + i % G;
}

// A block's four waves take tiles of 16 positions in turn, each with the block's 16 * RB
// rows and references, sums and outputs of its own, and meet in LDS once at the end.
// Both products run on f32 MFMA (v_mfma_f32_16x16x4_f32), whose factors are as they are
// in memory.  Lane (g, c) = (lane / 16, lane % 16) has A[c][g] and B[g][c] of a product
// of depth 4, and gets D[4g + r][c] in register r:
//   S^T = K Q^T: A = position c's dimension 16 x + 4g + j, B = row c's, so that a lane
//     has 16-byte pieces of K and Q and the products j = 0 .. 3 take them apart;
//   O^T = V^T P^T: product j's depth g is position 4g + j, whose score the lane holds in
//     register j for row c, and A's row c of block (q, i) is dimension 64 q + 4 c + i.
template <int DP, int RB>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void k_prefix_attn(PrefixAttn a, Plan plan,
                                                                        float *__restrict__ part,
                                                                        float *__restrict__ pml) {
    constexpr int NX = DP / 16, NB = DP / 64, ROWS = 16 * RB;
    __shared__ __attribute__((aligned(16))) float lo[ROWS][DP + 4];
    __shared__ float lm[4][ROWS], ls[4][ROWS];
    const Job job = job_of(a, plan, blockIdx.x);
    if (job.none && part) return;   // the merge skips this split
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, c = lane & 15, g = lane >> 4;
    const int D = a.hd;
    float4 kr[NX], vr[4][NB];
    auto load_k = [&](int tile) {
        const float *r = job.k + min(tile * kTile + c, job.len - 1) * job.ks + 4 * g;
#pragma unroll
        for (int x = 0; x < NX; ++x)
            if (16 * x < D) kr[x] = *reinterpret_cast<const float4 *>(r + 16 * x);
    };
    auto load_v = [&](int tile) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = tile * kTile + 4 * g + j;
            const float *r = job.v + min(at, job.len - 1) * job.vs;
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                vr[j][q] = *reinterpret_cast<const float4 *>(r + min(64 * q + 4 * c, D - 4));
                // weight 0 must meet no infinity or NaN
                if (at >= job.len) vr[j][q] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
    };
    const int first = job.t0 + wave;
    if (first < job.t1) {
        load_k(first);
        load_v(first);
    }
    float4 qr[RB][NX];
    float m[RB], l[RB];
    f32x4 o[RB][NB][4];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int i = min(job.i0 + 16 * rb + c, job.i1 - 1);   // rows past the last repeat it
        const float *q = a.q + row_of(a, job, i) * D + 4 * g;
#pragma unroll
        for (int x = 0; x < NX; ++x)
            if (16 * x < D) qr[rb][x] = *reinterpret_cast<const float4 *>(q + 16 * x);
        m[rb] = -INFINITY;
        l[rb] = 0.f;
#pragma unroll
        for (int q2 = 0; q2 < NB; ++q2)
#pragma unroll
            for (int i2 = 0; i2 < 4; ++i2) o[rb][q2][i2] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float f = a.scale * kLog2e;

    for (int tile = first; tile < job.t1; tile += 4) {
        // ---- scores, in powers of two
        f32x4 s[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) s[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < NX; ++x)
            if (16 * x < D) {
                const float k4[4] = {kr[x].x, kr[x].y, kr[x].z, kr[x].w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        const float4 &q = qr[rb][x];
                        const float q1 = j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w;
                        s[rb] = __builtin_amdgcn_mfma_f32_16x16x4f32(k4[j], q1, s[rb], 0, 0, 0);
                    }
            }
        if (tile + 4 < job.t1) load_k(tile + 4);
        // ---- the rows' references
        bool moved = false;
        float was[RB];
        const int left = job.len - tile * kTile - 4 * g;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[rb][r] = r < left ? s[rb][r] * f : -INFINITY;
            const float top = max_over_groups(
                fmaxf(fmaxf(s[rb][0], s[rb][1]), fmaxf(s[rb][2], s[rb][3])));
            was[rb] = m[rb];
            if (top > m[rb]) m[rb] = top + kLead;
            moved |= m[rb] != was[rb];
        }
        if (__any(moved)) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const float alpha =
                    was[rb] == m[rb] ? 1.f : __builtin_amdgcn_exp2f(was[rb] - m[rb]);
                l[rb] *= alpha;
#pragma unroll
                for (int q = 0; q < NB; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[rb][q][i] *= alpha;
            }
        }
        // ---- weights and outputs
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const float base = m[rb] == -INFINITY ? 0.f : m[rb];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[rb][r] = __builtin_amdgcn_exp2f(s[rb][r] - base);
                l[rb] += s[rb][r];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                const float v4[4] = {vr[j][q].x, vr[j][q].y, vr[j][q].z, vr[j][q].w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb)
                        o[rb][q][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(v4[i], s[rb][j],
                                                                          o[rb][q][i], 0, 0, 0);
            }
        if (tile + 4 < job.t1) load_v(tile + 4);
    }

    // ---- the four waves' outputs, normalised, in the shares of their sums, in wave order
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        l[rb] = sum_over_groups(l[rb]);
        if (l[rb] != l[rb] && m[rb] == -INFINITY) m[rb] = INFINITY;   // only NaN seen: NaN
        if (g == 0) {
            lm[wave][16 * rb + c] = m[rb];
            ls[wave][16 * rb + c] = l[rb];
        }
    }
    __syncthreads();
    // Row r's reference, sum and share of wave w.
    auto shares = [&](int r, int w, float &top, float &sum) {
        top = fmaxf(fmaxf(lm[0][r], lm[1][r]), fmaxf(lm[2][r], lm[3][r]));
        sum = 0.f;
        float mine = 0.f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const float y =
                lm[x][r] == -INFINITY ? 0.f : ls[x][r] * __builtin_amdgcn_exp2f(lm[x][r] - top);
            sum += y;
            mine = x == w ? y : mine;
        }
        return sum == 0.f ? 0.f : mine / sum;
    };
    float top, sum;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const float x = shares(16 * rb + c, wave, top, sum);
        l[rb] = l[rb] == 0.f ? 0.f : x / l[rb];
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (wave == w) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const int r = 16 * rb + c;
                const float x = l[rb];
#pragma unroll
                for (int q = 0; q < NB; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {   // dimensions 64 q + 16 g + 4 i .. + 3
                        float4 *d = reinterpret_cast<float4 *>(&lo[r][64 * q + 16 * g]) + i;
                        float4 y = w ? *d : make_float4(0.f, 0.f, 0.f, 0.f);
                        if (x != 0.f) {
                            y.x = fmaf(o[rb][q][0][i], x, y.x);
                            y.y = fmaf(o[rb][q][1][i], x, y.y);
                            y.z = fmaf(o[rb][q][2][i], x, y.z);
                            y.w = fmaf(o[rb][q][3][i], x, y.w);
                        }
                        *d = y;
                    }
            }
        }
        __syncthreads();
    }
    const int cols = D / 4, n = job.i1 - job.i0, R = a.rows * (a.hq / a.hkv);
    for (int x = t; x < n * cols; x += 256) {
        const int r = x / cols, d = x - r * cols;
        const float4 y = *reinterpret_cast<const float4 *>(&lo[r][4 * d]);
        if (part) {
            const size_t at =
                (((size_t)job.group * a.hkv + job.kvh) * plan.slots + job.slot) * R + job.i0 + r;
            reinterpret_cast<float4 *>(part + at * D)[d] = y;
            if (d == 0) {
                shares(r, 0, top, sum);
                pml[2 * at] = top;
                pml[2 * at + 1] = sum;
            }
        } else {
            reinterpret_cast<float4 *>(a.out + row_of(a, job, job.i0 + r) * D)[d] = y;
        }
    }
}

// A row's partial results, normalised, in the shares of their sums, a wave per row: lanes of
// LC columns of four dimensions, 64 / LC slots side by side.
template <int LC>
__global__ __launch_bounds__(256) void k_prefix_merge(PrefixAttn a, Plan plan,
                                                      const float *__restrict__ part,
                                                      const float *__restrict__ pml) {
    constexpr int NG = 64 / LC;
    __shared__ float w[4][2 * kMaxSplits];
    const int G = a.hq / a.hkv, R = a.rows * G, cols = a.hd / 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i = blockIdx.x * 4 + wave, kvh = blockIdx.y, group = blockIdx.z;
    if (i >= R) return;
    const int pu = split_range(length(a.prefix_lens, a.prefix_len, group, a.max_prefix), plan.pcap, 0)
                       .splits;
    const int ou = split_range(length(a.own_lens, a.own_len, group * a.rows + i / G, a.max_own),
                               plan.ocap, 0)
                       .splits;
    const int used = pu + ou;
    auto slot = [&](int x) { return x < pu ? x : plan.pcap + x - pu; };
    const size_t at = ((size_t)group * a.hkv + kvh) * plan.slots * R + i;
    float m[2], l[2], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        m[x] = -INFINITY;
        l[x] = 0.f;
        if (lane + 64 * x < used) {
            const float *p = pml + 2 * (at + (size_t)slot(lane + 64 * x) * R);
            m[x] = p[0];
            l[x] = p[1];
        }
        top = fmaxf(top, m[x]);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        m[x] = m[x] == -INFINITY ? 0.f : l[x] * __builtin_amdgcn_exp2f(m[x] - top);
        sum += m[x];
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
    for (int x = 0; x < 2; ++x) w[wave][lane + 64 * x] = m[x] * inv;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int d = min(lane % LC, cols - 1), grp = lane / LC;
    const float4 *src = reinterpret_cast<const float4 *>(part + at * a.hd) + d;
    const size_t step = (size_t)R * cols;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = grp; s < used; s += NG) {
        const float x = w[wave][s];
        const float4 v = src[slot(s) * step];
        if (x != 0.f) {   // a split that sees nothing of the row counts for nothing
            y.x = fmaf(v.x, x, y.x);
            y.y = fmaf(v.y, x, y.y);
            y.z = fmaf(v.z, x, y.z);
            y.w = fmaf(v.w, x, y.w);
        }
    }
#pragma unroll
    for (int o = LC; o < 64; o <<= 1) {
        y.x += __shfl_xor(y.x, o);
        y.y += __shfl_xor(y.y, o);
        y.z += __shfl_xor(y.z, o);
        y.w += __shfl_xor(y.w, o);
    }
    if (lane >= cols) return;
    float *out = a.out + (((size_t)group * a.rows + i / G) * a.hq + kvh * G + i % G) * a.hd;
    reinterpret_cast<float4 *>(out)[d] = y;
}

// prefix, own: the positions that the caches hold, or the lengths where the host knows them.
Plan plan_of(int groups, int rows, int hq, int hkv, int hd, int prefix, int own) {
    Plan p{};
    const int G = hq / hkv, R = rows * G;
    p.rb = R <= 16 || hd > 128 ? 1 : 2;
    p.ptiles = (R + 16 * p.rb - 1) / (16 * p.rb);
    p.gtiles = (G + 16 * p.rb - 1) / (16 * p.rb);
    auto cap = [](int64_t blocks, int len) {
        const int tiles = (len + kTile - 1) / kTile;
        const int64_t most = std::min<int64_t>((tiles + kMinTiles - 1) / kMinTiles, kMaxSplits);
        return (int)std::max<int64_t>(1, std::min<int64_t>(512 / blocks, most));
    };
    const int64_t pb = (int64_t)groups * hkv * p.ptiles, ob = (int64_t)groups * rows * hkv * p.gtiles;
    p.pcap = prefix || !own ? cap(pb, prefix) : 0;   // without positions: the zeros
    p.ocap = own ? cap(ob, own) : 0;
    p.pblocks = (int)(pb * p.pcap);
    p.oblocks = (int)(ob * p.ocap);
    p.slots = p.pcap + p.ocap;
    return p;
}

}  // namespace

size_t prefix_attention_scratch(int groups, int rows, int hq, int hkv, int hd, int prefix, int own) {
    const int slots = plan_of(groups, rows, hq, hkv, hd, prefix, own).slots;
    return slots > 1 ? (size_t)groups * rows * hq * slots * (hd + 2) * sizeof(float) : 0;
}

int launch_prefix_attention(const PrefixAttn &a, float *scratch, hipStream_t s) {
    const Plan p = plan_of(a.groups, a.rows, a.hq, a.hkv, a.hd, a.prefix_lens ? a.max_prefix : a.prefix_len,
                           a.own_lens ? a.max_own : a.own_len);
    float *part = p.slots > 1 ? scratch : nullptr;
    const size_t rows = (size_t)a.groups * a.rows * a.hq;
    float *pml = part ? part + rows * p.slots * a.hd : nullptr;
    const dim3 grid(p.pblocks + p.oblocks);
#define TB_PA(DP, RB)                                                                       \
    hipLaunchKernelGGL((k_prefix_attn<DP, RB>), grid, dim3(256), 0, s, a, p, part, pml)
    if (a.hd <= 64) {
        if (p.rb == 1) TB_PA(64, 1);
        else TB_PA(64, 2);
    } else if (a.hd <= 128) {
        if (p.rb == 1) TB_PA(128, 1);
        else TB_PA(128, 2);
    } else {
        TB_PA(256, 1);
    }
#undef TB_PA
    TB_LAUNCHED();
    if (part) {
        const dim3 blocks((a.rows * (a.hq / a.hkv) + 3) / 4, a.hkv, a.groups);
        if (a.hd <= 32)
            hipLaunchKernelGGL(k_prefix_merge<8>, blocks, dim3(256), 0, s, a, p, part, pml);
        else if (a.hd <= 64)
            hipLaunchKernelGGL(k_prefix_merge<16>, blocks, dim3(256), 0, s, a, p, part, pml);
        else if (a.hd <= 128)
            hipLaunchKernelGGL(k_prefix_merge<32>, blocks, dim3(256), 0, s, a, p, part, pml);
        else
            hipLaunchKernelGGL(k_prefix_merge<64>, blocks, dim3(256), 0, s, a, p, part, pml);
        TB_LAUNCHED();
    }
    return TB_OK;
}

}  // namespace tb
