// Attention of sequences that share a prefix: each query row over its group's
// prefix and over its own cache, for GQA and f32 caches.  A prefix's K and V are read
// once for a block's 16 to 128 of the group's rows; where caches are short and
// sequences few, by each sequence for itself.
//
//   o = sum_p w_p v_p / sum_p w_p,  w_p = exp(scale q.k_p - m)
//
// over the prefix's positions and the row's own ones.  One pass over K and V with a
// running reference m and sum; the positions are split over blocks, whose
// results are merged in the order of the splits.  Few rows go through f32 MFMA,
// whose factors are as they are in memory (k_prefix_stream), many through bf16 MFMA with
// three limbs a factor (k_prefix_dense); the sequences' own caches always through the first.
#include <math.h>

#include <algorithm>

#include "prefix.hpp"
#include "tb_common.hpp"

namespace tb {

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896340736f;
// Splits of the prefix, and of a row's own cache, at most: a wave of the merge has both in two
// passes over its lanes.  With eight KV heads the blocks wanted are fewer; with one or two, on
// prefixes past some thousand positions, it leaves CUs without a block: 32768 positions of two KV
// heads of 64, in cache, are read at 2.1 TB/s for 2 sequences and 1.1 for 5, those of eight heads
// of 128 at 5.8 for 2.
constexpr int kMaxSplits = 64;
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

// One cache's rows of a KV head, of which the first len positions count.
struct Rows {
    const float *k, *v;
    int64_t ks, vs;
    int len;
};

__device__ __forceinline__ Rows prefix_rows(const PrefixAttn &a, int group, int kvh) {
    return {a.kp.p + group * a.kp.sb + kvh * a.kp.sh, a.vp.p + group * a.vp.sb + kvh * a.vp.sh,
            a.kp.ss, a.vp.ss, length(a.prefix_lens, a.prefix_len, group, a.max_prefix)};
}
__device__ __forceinline__ Rows own_rows(const PrefixAttn &a, int seq, int kvh) {
    return {a.k.p + seq * a.k.sb + kvh * a.k.sh, a.v.p + seq * a.v.sb + kvh * a.v.sh, a.k.ss,
            a.v.ss, length(a.own_lens, a.own_len, seq, a.max_own)};
}

// What one block works on: query rows i0 .. i1 - 1 of one KV head of one group (row i is
// sequence i / G's query head i % G of the KV head's G) over tiles t0 .. t1 - 1 of the positions
// of x, followed by all of y's.
struct Job {
    Rows x, y;
    int group, kvh, i0, i1;
    int slot;   // its place among the partial results
    int t0, t1;
    bool none;  // nothing to do: this split is not among the cache's, and the merge skips it
};

// The plan of a launch; the blocks' order: the prefix's, then the sequences' own.
struct Plan {
    int nw;               // waves a block
    int rb, prows;        // 16 * rb rows of a group a block (16 of a sequence), dense ones prows
    int ptiles, gtiles;   // row tiles of a group's rows, of a sequence's
    int pcap, ocap;       // splits at most
    int pblocks, oblocks;
    int slots;            // partial results a row; 1: none, the output itself
    bool joined;          // the sequences' blocks take the prefix too
    bool dense;           // the prefix's blocks share limbs in LDS
};

// Split `split` of a cache of len positions where at most cap are wanted: only the length
// counts, so that within one plan a result is the same whatever the bound.
constexpr int kTile = 16, kMinTiles = 4;
struct Range {
    int t0, t1, splits;
};
__device__ __forceinline__ Range split_range(int len, int cap, int split) {
    const int tiles = (len + kTile - 1) / kTile;
    cap = max(cap, 1);   // 0 for a cache without positions
    const int each = max(((tiles + cap - 1) / cap + 3) & ~3, kMinTiles);   // the waves' alike
    return {min(split * each, tiles), min((split + 1) * each, tiles), (tiles + each - 1) / each};
}

// The row tiles that read the same K and V are eight blocks apart, so that they run on the
// same of the eight dies (block i goes to die i % 8) and share its cache.
__device__ __forceinline__ Job job_of(const PrefixAttn &a, const Plan &p, int block, bool part) {
    Job j;
    const int G = a.hq / a.hkv;
    if (block < p.pblocks) {
        const int rt = block / 8 % p.ptiles, unit = block / (8 * p.ptiles) * 8 + block % 8;
        j.kvh = unit % a.hkv;
        const int split = unit / a.hkv % p.pcap;
        j.group = unit / (a.hkv * p.pcap);
        j.i0 = rt * p.prows;
        j.i1 = min(j.i0 + p.prows, a.rows * G);
        j.slot = split;
        j.none = true;
        j.t0 = j.t1 = 0;
        if (j.group >= a.groups) return j;   // the last units make eight
        j.x = prefix_rows(a, j.group, j.kvh);
        j.y = j.x;
        j.y.len = 0;
        const Range r = split_range(j.x.len, p.pcap, split);
        j.t0 = r.t0;
        j.t1 = r.t1;
        j.none = split >= r.splits && part;
    } else {
        block -= p.pblocks;
        j.kvh = block % a.hkv;
        block /= a.hkv;
        const int gt = block % p.gtiles;
        block /= p.gtiles;
        const int split = block % p.ocap, seq = block / p.ocap;
        j.group = seq / a.rows;
        const int i = (seq - j.group * a.rows) * G;
        j.i0 = i + 16 * gt;
        j.i1 = min(j.i0 + 16, i + G);
        j.y = own_rows(a, seq, j.kvh);
        if (p.joined) {
            j.x = prefix_rows(a, j.group, j.kvh);
            j.t0 = 0;
            j.t1 = (j.x.len + kTile - 1) / kTile;
            j.none = false;
        } else {
            j.x = j.y;
            j.y.len = 0;
            const Range r = split_range(j.x.len, p.ocap, split);
            j.t0 = r.t0;
            j.t1 = r.t1;
            j.none = split >= r.splits && part;
        }
        j.slot = p.pcap + split;
    }
    return j;
}

__device__ __forceinline__ size_t row_of(const PrefixAttn &a, const Job &j, int i) {
    const int G = a.hq / a.hkv;
    return ((size_t)j.group * a.rows + i / G) * a.hq + j.kvh * G + i % G;
}

// What 16 * RB query rows have seen so far: their references, sums, and outputs of lane
// (g, c): dimensions 64 q + 16 g + 4 r + i of row 16 b + c in register r of o[b][q][i].
template <int D, int RB>
struct State {
    float m[RB], l[RB];
    f32x4 o[RB][(D + 63) / 64][4];
};

// A wave's pass over the tiles first, first + step .. of a job, for its rows i0 + 16 b + c
// (those from i1 on repeat the last).  Both products run on f32 MFMA (v_mfma_f32_16x16x4_f32),
// whose factors are as they are in memory.  Lane (g, c) = (lane / 16, lane % 16) has A[c][g]
// and B[g][c] of a product of depth 4, and gets D[4g + r][c] in register r:
//   S^T = K Q^T: A = position c's dimension 16 x + 4g + j, B = row c's, so that a lane
//     has 16-byte pieces of K and Q and the products j = 0 .. 3 take them apart;
//   O^T = V^T P^T: product j's depth g is position 4g + j, whose score the lane holds in
//     register j for row c, and A's row c of block (q, i) is dimension 64 q + 4 c + i.
// The next tile's K is requested when this one's scores are on their way, its V when
// this one's outputs are.
//
// Bound by memory, on short prefixes by the launch and the blocks' first and last
// steps (6.4 us of the second): 8 KV heads of 128, 16 rows on 32767 positions 50 us (5.4 TB/s
// of K and V), 32 rows on 4096 17.4.  The f32 MFMA (154 TFLOP/s in a large product) would
// bound 64 rows: 104 us on 32767 positions, k_prefix_dense 76.
template <int D, int RB>
__device__ __forceinline__ void stream(const PrefixAttn &a, const Job &job, int i0, int i1,
                                       int first, int step, State<D, RB> &st) {
    constexpr int NX = D / 16, NB = (D + 63) / 64;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int xt = job.t1 - job.t0, end = xt + (job.y.len + kTile - 1) / kTile;
    float4 kr[NX], vr[4][NB];
    // Tile t of the job: its cache and first position.
    auto rows = [&](int t) { return t < xt ? job.x : job.y; };
    auto place = [&](int t) { return kTile * (t < xt ? job.t0 + t : t - xt); };
    auto load_k = [&](int t) {
        const Rows x = rows(t);
        const int p0 = place(t);
        const float *r = x.k + p0 * x.ks + (c * x.ks + 4 * g);
        if (p0 + kTile > x.len) r -= max(p0 + c - (x.len - 1), 0) * x.ks;   // repeats the last
#pragma unroll
        for (int i = 0; i < NX; ++i) kr[i] = *reinterpret_cast<const float4 *>(r + 16 * i);
    };
    auto load_v = [&](int t) {
        const Rows x = rows(t);
        const int p0 = place(t);
        const float *r = x.v + p0 * x.vs + 4 * g * x.vs;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float *v = r + j * x.vs;
            if (p0 + kTile > x.len) v -= max(p0 + 4 * g + j - (x.len - 1), 0) * x.vs;
#pragma unroll
            for (int q = 0; q < NB; ++q)
                vr[j][q] = *reinterpret_cast<const float4 *>(v + min(64 * q + 4 * c, D - 4));
        }
    };
    if (first < end) {
        load_k(first);
        load_v(first);
    }
    float4 qr[RB][NX];
    float m[RB], l[RB];
    f32x4(&o)[RB][NB][4] = st.o;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const float *q = a.q + row_of(a, job, min(i0 + 16 * b + c, i1 - 1)) * D + 4 * g;
#pragma unroll
        for (int x = 0; x < NX; ++x) qr[b][x] = *reinterpret_cast<const float4 *>(q + 16 * x);
        m[b] = -INFINITY;
        l[b] = 0.f;
#pragma unroll
        for (int y = 0; y < NB; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[b][y][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float f = a.scale * kLog2e;

    for (int t = first; t < end; t += step) {
        // ---- scores, in powers of two; two sums a row block, where there are few
        f32x4 s[RB], s2[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b) s[b] = s2[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < NX; ++x) {
            const float k4[4] = {kr[x].x, kr[x].y, kr[x].z, kr[x].w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int b = 0; b < RB; ++b) {
                    const float4 &q = qr[b][x];
                    f32x4 &d = RB <= 2 && j & 1 ? s2[b] : s[b];
                    d = __builtin_amdgcn_mfma_f32_16x16x4f32(
                        k4[j], j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w, d, 0, 0, 0);
                }
        }
        if (t + step < end) load_k(t + step);
        const int left = rows(t).len - place(t);
#pragma unroll
        for (int b = 0; b < RB; ++b) s[b] = (RB <= 2 ? s[b] + s2[b] : s[b]) * f;
        if (left < kTile) {   // a cache's last tile: weight 0, which must meet no infinity or NaN
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool in = 4 * g + r < left;
#pragma unroll
                for (int b = 0; b < RB; ++b) s[b][r] = in ? s[b][r] : -INFINITY;
#pragma unroll
                for (int q = 0; q < NB; ++q)
                    vr[r][q] = in ? vr[r][q] : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
        // ---- the rows' references
        float top[RB];
        bool moves = false;
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            top[b] = max_over_groups(fmaxf(fmaxf(s[b][0], s[b][1]), fmaxf(s[b][2], s[b][3])));
            moves |= top[b] > m[b];
        }
        if (__any(moves)) {
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                const float was = m[b];
                if (top[b] > m[b]) m[b] = top[b] + kLead;
                const float alpha = was == m[b] ? 1.f : __builtin_amdgcn_exp2f(was - m[b]);
                l[b] *= alpha;
#pragma unroll
                for (int q = 0; q < NB; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[b][q][i] *= alpha;
            }
        }
        // ---- weights and outputs
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const float base = m[b] == -INFINITY ? 0.f : m[b];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[b][r] = __builtin_amdgcn_exp2f(s[b][r] - base);
                l[b] += s[b][r];
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
                    for (int b = 0; b < RB; ++b)
                        o[b][q][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                            v4[i], s[b][j], o[b][q][i], 0, 0, 0);
            }
        if (t + step < end) load_v(t + step);
    }
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        st.l[b] = sum_over_groups(l[b]);
        // NaN and nothing else: the reference of a row that is NaN
        st.m[b] = st.l[b] != st.l[b] && m[b] == -INFINITY ? INFINITY : m[b];
    }
}

// LDS of a block of NW waves that meet: their outputs, references, sums and shares.
template <int D, int RB, int NW>
struct Meeting {
    float o[NW][16 * RB][(D + 63) / 64 * 64 + 4];
    float m[NW][16 * RB], l[NW][16 * RB], share[NW][16 * RB], top[16 * RB], sum[16 * RB];
};

// A block's NW waves take tiles of 16 positions in turn, each with the block's rows and a
// state of its own, and meet in LDS once at the end.
template <int D, int RB, int NW>
__device__ __forceinline__ void stream_block(const PrefixAttn &a, const Plan &plan, const Job &job,
                                             Meeting<D, RB, NW> &lds, float *part, float *pml) {
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int c = lane & 15, g = lane >> 4;
    State<D, RB> st;
    stream<D, RB>(a, job, job.i0, job.i1, wave, NW, st);
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const int r = 16 * b + c;
        if (g == 0) {
            lds.m[wave][r] = st.m[b];
            lds.l[wave][r] = st.l[b];
        }
#pragma unroll
        for (int q = 0; q < (D + 63) / 64; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i)   // dimensions 64 q + 16 g + 4 i .. + 3
                *reinterpret_cast<float4 *>(&lds.o[wave][r][64 * q + 16 * g + 4 * i]) =
                    make_float4(st.o[b][q][0][i], st.o[b][q][1][i], st.o[b][q][2][i],
                                st.o[b][q][3][i]);
    }
    __syncthreads();
    // ---- each row's reference, sum and the waves' factors: e^(m - top) over the sum
    if (t < 16 * RB) {
        float top = -INFINITY, sum = 0.f, e[NW];
#pragma unroll
        for (int w = 0; w < NW; ++w) top = fmaxf(top, lds.m[w][t]);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float m = lds.m[w][t];
            e[w] = m == -INFINITY ? -1.f : __builtin_amdgcn_exp2f(m - top);
            if (m != -INFINITY) sum = fmaf(lds.l[w][t], e[w], sum);
        }
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        // A share of 0 counts too: NaN times 0 is NaN.  -1: the wave saw nothing of the row.
#pragma unroll
        for (int w = 0; w < NW; ++w) lds.share[w][t] = e[w] == -1.f ? -1.f : e[w] * inv;
        lds.top[t] = top;
        lds.sum[t] = sum;
    }
    __syncthreads();
    constexpr int cols = D / 4;
    const int n = job.i1 - job.i0, R = a.rows * (a.hq / a.hkv);
    for (int x = t; x < n * cols; x += 64 * NW) {
        const int r = x / cols, d = x % cols;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float4 z = *reinterpret_cast<const float4 *>(&lds.o[w][r][4 * d]);
            const float k = lds.share[w][r];
            if (!(k < 0.f)) {
                y.x = fmaf(z.x, k, y.x);
                y.y = fmaf(z.y, k, y.y);
                y.z = fmaf(z.z, k, y.z);
                y.w = fmaf(z.w, k, y.w);
            }
        }
        if (part) {
            const size_t at =
                (((size_t)job.group * a.hkv + job.kvh) * plan.slots + job.slot) * R + job.i0 + r;
            reinterpret_cast<float4 *>(part + at * D)[d] = y;
            if (d == 0) {
                pml[2 * at] = lds.top[r];
                pml[2 * at + 1] = lds.sum[r];
            }
        } else {
            reinterpret_cast<float4 *>(a.out + row_of(a, job, job.i0 + r) * D)[d] = y;
        }
    }
}

template <int D, int RB, int NW>
__global__ __launch_bounds__(64 * NW, D <= 192 ? 2 : 1) void k_prefix_stream(
    PrefixAttn a, Plan plan, float *__restrict__ part, float *__restrict__ pml) {
    __shared__ __attribute__((aligned(16))) union {
        Meeting<D, RB, NW> prefix;
        Meeting<D, 1, NW> own;
    } lds;
    const Job job = job_of(a, plan, blockIdx.x, part != nullptr);
    if (job.none) return;
    if (RB > 1 && (int)blockIdx.x < plan.pblocks)
        stream_block<D, RB, NW>(a, plan, job, lds.prefix, part, pml);
    else
        stream_block<D, 1, NW>(a, plan, job, lds.own, part, pml);
}

// ---- many rows: bf16 MFMA -------------------------------------------------------

// 8 values as three bf16 limbs, x = hi + mid + lo but for 2^-27 of x (and 2^-134, the half of
// bf16's smallest step): each is the rounded rest of those before.  bf16 has f32's
// exponents, so that nothing is scaled.
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 &hi, bf16x8 &mid, bf16x8 &lo) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const f32x2 y = {x[j], x[j + 1]};
        const bf16x2 h = __builtin_convertvector(y, bf16x2);
        const f32x2 r = {y.x - (float)h.x, y.y - (float)h.y};
        const bf16x2 m = __builtin_convertvector(r, bf16x2);
        const f32x2 e = {r.x - (float)m.x, r.y - (float)m.y};
        const bf16x2 l = __builtin_convertvector(e, bf16x2);
        hi[j] = h.x; hi[j + 1] = h.y;
        mid[j] = m.x; mid[j + 1] = m.y;
        lo[j] = l.x; lo[j + 1] = l.y;
    }
}

// d += a b of two factors of three limbs: all products but those below 2^-25 of it.
__device__ __forceinline__ f32x4 mfma6(const bf16x8 (&a)[3], const bf16x8 (&b)[3], f32x4 d) {
    d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[2], b[0], d, 0, 0, 0);
    d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[2], d, 0, 0, 0);
    d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[1], b[1], d, 0, 0, 0);
    d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[1], b[0], d, 0, 0, 0);
    d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[1], d, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[0], d, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma6(const bf16x8 (&a)[3], const bf16x8 (&b)[3], f32x16 d) {
    d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[2], b[0], d, 0, 0, 0);
    d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[2], d, 0, 0, 0);
    d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[1], d, 0, 0, 0);
    d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[0], d, 0, 0, 0);
    d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[1], d, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], d, 0, 0, 0);
}

// Over the lanes that share a row, two of 32 rows or four of 16.
template <int W, class F>
__device__ __forceinline__ float over_row(float v, F f) {
    if constexpr (W == 16) {
        return over_groups(v, f);
    } else {
        const auto r =
            __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
}

// LDS of a dense block: a tile's limbs of 32 positions in operand order, [limb][lane].
template <int D>
struct Limbs {
    bf16x8 k[D / 16][3][64], v[D / 16][3][64];
};

// A block of four waves takes 4 W rows of a group, W = 32 or 16 a wave, and a split of the
// prefix in tiles of 32 positions.  Per tile its waves build the limbs of K and V, a
// quarter each, in LDS, and then every wave multiplies all of them with its rows, so that
// each f32 of the prefix is read and split once a block; the next tile is requested before.
// Products are of depth P = 512 / W (v_mfma_f32_32x32x16_bf16, v_mfma_f32_16x16x32_bf16): lane
// (h, c) = (lane / W, lane % W) has A[c][8h ..] and B[8h ..][c], and gets D[4h + r % 4 +
// 8 (r / 4)][c] in register r (W = 16: r < 4):
//   S^T = K Q^T: A = W positions, position c's dimensions P x + 8h .., B = row c's, in registers;
//   O^T = V^T P^T: A = W dimensions, dimension c's eight positions whose scores the lane
//     holds for row c: 16 u + 4h + (0 .. 3, 8 .. 11), or 4h + (0 .. 3, 16 .. 19).
// Every product of f32 factors is six of limbs (mfma6): 22 bits and more of it, at a sixth
// of the bf16 rate, where the f32 MFMA has a sixteenth.  An infinity or NaN among K, V or
// the queries makes NaN of the limbs' products: a wave that has one in its results
// works its rows out anew in f32 (stream()).
//
// Bound by the matrix unit at the clock it leaves itself, and by what shares the SIMDs
// with it: 256 rows of 128 on 32767 positions of 8 KV heads 205 us (168 TFLOP/s of f32
// products, six bf16 ones each; a large bf16 product reaches 1219), of which the MFMAs
// alone take 131, with their operands' reads 160, with the limbs 182.  Operands read an
// MFMA group ahead by force spill and gain nothing (218).  Registers spill in this form too, 91
// and 9 with 16 and 32 rows of 128 a wave, 57 and 104 with 32 of 224 and 256; the first has three
// blocks a CU for it (64 rows on 4096 positions 20 us, with two 25).
template <int D, int W>
__device__ __forceinline__ void dense_block(const PrefixAttn &a, const Plan &plan, const Job &job,
                                            Limbs<D> &lds, float *part, float *pml) {
    constexpr int P = 512 / W, H = 64 / W;          // depth of a product; lanes that share a row
    constexpr int NX = D / P, NY = D / W;           // products of a score, blocks of dimensions
    constexpr int NS = 32 / W, SR = W * W / 64;     // blocks of positions, their registers
    constexpr int KD = D / 8, KU = (KD + 7) / 8, VU = (D + 63) / 64;
    constexpr int kSwap = KD > 8 ? 1 : 16 / KD;
    typedef float acc __attribute__((ext_vector_type(SR)));
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int c = lane & (W - 1), h = lane / W;
    const int G = a.hq / a.hkv, R = a.rows * G;
    const int t0 = job.t0 / 2, t1 = (job.t1 + 1) / 2, len = job.x.len;

    // ---- this thread's parts of a tile: 8 dimensions of position kunit / KD, and of dimension
    // lane + 64 u the positions vpos(0) .. vpos(7)
    float kr[KU][8], vr[VU][8];
    auto kunit = [&](int u) { return min(t + 256 * u, 32 * KD - 1); };
    auto vpos = [&](int i) {
        return W == 32 ? 16 * (wave >> 1) + 4 * (wave & 1) + 8 * (i >> 2) + (i & 3)
                       : 4 * wave + 16 * (i >> 2) + (i & 3);
    };
    auto load = [&](int tile) {
        const bool whole = 32 * tile + 32 <= len;
        const float *kt = job.x.k + (int64_t)32 * tile * job.x.ks;
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            const int kp = kunit(u) / KD;
            const float *k = kt + (kp * job.x.ks + 8 * (kunit(u) % KD));
            if (!whole)   // the last tile repeats the last position
                k -= max(32 * tile + kp - (len - 1), 0) * job.x.ks;
            const float4 x = reinterpret_cast<const float4 *>(k)[0];
            const float4 y = reinterpret_cast<const float4 *>(k)[1];
            kr[u][0] = x.x; kr[u][1] = x.y; kr[u][2] = x.z; kr[u][3] = x.w;
            kr[u][4] = y.x; kr[u][5] = y.y; kr[u][6] = y.z; kr[u][7] = y.w;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float *v = job.x.v + min(32 * tile + vpos(i), len - 1) * job.x.vs;
#pragma unroll
            for (int u = 0; u < VU; ++u) vr[u][i] = v[(uint32_t)min(lane + 64 * u, D - 1)];
        }
    };
    // Lanes are swapped within 16 by the dimensions, or a wave's stores of K would meet in a
    // part of the banks.
    auto klane = [](int p, int kd) { return (p + W * (kd % H)) ^ (kd * kSwap); };
    auto store = [&](int tile) {
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            const int kp = kunit(u) / KD, kd = kunit(u) % KD;
            bf16x8 x[3];
            split8(kr[u], x[0], x[1], x[2]);
            if (32 * KD % 256 == 0 || t + 256 * u < 32 * KD)
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    lds.k[kd / H * NS + kp / W][i][klane(kp & (W - 1), kd)] = x[i];
        }
        if (32 * tile + 32 > len) {   // weight 0 must meet no infinity or NaN
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (32 * tile + vpos(i) >= len)
#pragma unroll
                    for (int u = 0; u < VU; ++u) vr[u][i] = 0.f;
        }
#pragma unroll
        for (int u = 0; u < VU; ++u) {
            const int vd = lane + 64 * u;
            bf16x8 x[3];
            split8(vr[u], x[0], x[1], x[2]);
            if (D % 64 == 0 || vd < D)
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    lds.v[W == 32 ? (wave >> 1) * NY + vd / W : vd / W][i]
                         [vd % W + W * (wave & (H - 1))] = x[i];
        }
    };
    if (t0 < t1) load(t0);

    // ---- the wave's query rows, row c in this lane; with the sign of the score's factor
    const int w0 = job.i0 + W * wave;
    const bool busy = w0 < job.i1;
    const float f = fabsf(a.scale) * kLog2e;
    bf16x8 q[NX][3];
    {
        const float *x = a.q + row_of(a, job, min(w0 + c, R - 1)) * D + 8 * h;
#pragma unroll
        for (int i = 0; i < NX; ++i) {
            const float4 u = reinterpret_cast<const float4 *>(x + P * i)[0];
            const float4 v = reinterpret_cast<const float4 *>(x + P * i)[1];
            float y[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = a.scale < 0.f ? -y[j] : y[j];
            split8(y, q[i][0], q[i][1], q[i][2]);
        }
    }
    float m = -INFINITY, l = 0.f;
    acc o[NY];
#pragma unroll
    for (int y = 0; y < NY; ++y)
#pragma unroll
        for (int r = 0; r < SR; ++r) o[y][r] = 0.f;

    for (int tile = t0; tile < t1; ++tile) {
        __syncthreads();
        store(tile);
        if (tile + 1 < t1) load(tile + 1);
        __syncthreads();
        if (!busy) continue;
        // ---- scores: the lane's positions in its registers' order
        acc sa[NS];
#pragma unroll
        for (int y = 0; y < NS; ++y)
#pragma unroll
            for (int r = 0; r < SR; ++r) sa[y][r] = 0.f;
#pragma unroll
        for (int x = 0; x < NX; ++x)
#pragma unroll
            for (int y = 0; y < NS; ++y) {
                bf16x8 k[3];
#pragma unroll
                for (int i = 0; i < 3; ++i) k[i] = lds.k[x * NS + y][i][klane(c, H * x + h)];
                sa[y] = mfma6(k, q[x], sa[y]);
            }
        float s[NS * SR];
#pragma unroll
        for (int i = 0; i < NS * SR; ++i) s[i] = sa[i / SR][i % SR];
        // ---- the rows' references, in powers of two
        if (32 * tile + 32 > len) {
            const int left = len - 32 * tile - 4 * h;
#pragma unroll
            for (int i = 0; i < NS * SR; ++i)
                if ((W == 32 ? 8 : 16) * (i >> 2) + (i & 3) >= left) s[i] = -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int i = 1; i < NS * SR; ++i) top = fmaxf(top, s[i]);
        top = over_row<W>(top, [](float x, float y) { return fmaxf(x, y); }) * f;
        if (__any(top > m)) {
            const float was = m;
            if (top > m) m = top + kLead;
            const float alpha = was == m ? 1.f : __builtin_amdgcn_exp2f(was - m);
            l *= alpha;
#pragma unroll
            for (int y = 0; y < NY; ++y)
#pragma unroll
                for (int r = 0; r < SR; ++r) o[y][r] *= alpha;
        }
        // ---- weights and outputs
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int u = 0; u < NS * SR / 8; ++u) {
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w[i] = __builtin_amdgcn_exp2f(fmaf(s[8 * u + i], f, -base));
                l += w[i];
            }
            bf16x8 p[3];
            split8(w, p[0], p[1], p[2]);
#pragma unroll
            for (int y = 0; y < NY; ++y) {
                bf16x8 v[3];
#pragma unroll
                for (int i = 0; i < 3; ++i) v[i] = lds.v[u * NY + y][i][lane];
                o[y] = mfma6(v, p, o[y]);
            }
        }
    }
    if (!busy) return;
    l = over_row<W>(l, [](float x, float y) { return x + y; });
    const bool row = w0 + c < job.i1;
    bool bad = !(l <= 3.4e38f);
#pragma unroll
    for (int y = 0; y < NY; ++y)
#pragma unroll
        for (int r = 0; r < SR; ++r) bad |= !(fabsf(o[y][r]) <= 3.4e38f);
    const size_t slot = (((size_t)job.group * a.hkv + job.kvh) * plan.slots + job.slot) * R;
    if (__builtin_expect(__any(bad && row), 0)) {
        const int c16 = lane & 15, g16 = lane >> 4, i1 = min(w0 + W, job.i1);
#pragma unroll 1
        for (int i0 = w0; i0 < i1; i0 += 16) {
            State<D, 1> st;
            stream<D, 1>(a, job, i0, i1, 0, 1, st);
            const int i = i0 + c16;
            if (i >= i1) continue;
            const float inv = st.l[0] == 0.f ? 0.f : 1.0f / st.l[0];
            float *to = part ? part + (slot + i) * D : a.out + row_of(a, job, i) * D;
            if (part && g16 == 0) {
                pml[2 * (slot + i)] = st.m[0];
                pml[2 * (slot + i) + 1] = st.l[0];
            }
#pragma unroll
            for (int y = 0; y < (D + 63) / 64; ++y)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (64 * y + 16 * g16 < D)
                        *reinterpret_cast<float4 *>(to + 64 * y + 16 * g16 + 4 * r) =
                            make_float4(st.o[0][y][0][r] * inv, st.o[0][y][1][r] * inv,
                                        st.o[0][y][2][r] * inv, st.o[0][y][3][r] * inv);
        }
        return;
    }
    if (!row) return;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    const int i = w0 + c;
    float *to = part ? part + (slot + i) * D : a.out + row_of(a, job, i) * D;
    if (part && h == 0) {
        pml[2 * (slot + i)] = m;
        pml[2 * (slot + i) + 1] = l;
    }
#pragma unroll
    for (int y = 0; y < NY; ++y)
#pragma unroll
        for (int r = 0; r < SR; r += 4)
            *reinterpret_cast<float4 *>(to + W * y + 2 * r + 4 * h) =
                make_float4(o[y][r] * inv, o[y][r + 1] * inv, o[y][r + 2] * inv, o[y][r + 3] * inv);
}

template <int D, int W>
__global__ __launch_bounds__(256, D > 128 ? 1 : W == 32 ? 2 : 3) void k_prefix_dense(
    PrefixAttn a, Plan plan, float *__restrict__ part, float *__restrict__ pml) {
    __shared__ __attribute__((aligned(16))) union {
        Limbs<D> limbs;
        Meeting<D, 1, 4> meeting;
    } lds;
    const Job job = job_of(a, plan, blockIdx.x, part != nullptr);
    if (job.none) return;
    if ((int)blockIdx.x < plan.pblocks)
        dense_block<D, W>(a, plan, job, lds.limbs, part, pml);
    else
        stream_block<D, 1, 4>(a, plan, job, lds.meeting, part, pml);
}

// A row's partial results, normalised, in the shares of their sums, in the order of the slots, by
// WR waves: groups of LC lanes of four dimensions each take every 64 WR / LC-th slot, the
// first of them requested before the shares are known (every slot's place in the scratch
// can be read, and what was not written is left out).  Bound by the launch and the way
// of those reads: 4.0 us for 256 rows of 33 slots, 9.5 for 2048 (34.6 MB).
template <int LC, int WR>
__global__ __launch_bounds__(256) void k_prefix_merge(PrefixAttn a, Plan plan,
                                                      const float *__restrict__ part,
                                                      const float *__restrict__ pml) {
    constexpr int NG = 64 * WR / LC, AHEAD = 8;
    __shared__ float w[4][2 * kMaxSplits];
    __shared__ float4 col[4][LC];
    const int G = a.hq / a.hkv, R = a.rows * G, cols = a.hd / 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i = blockIdx.x * (4 / WR) + wave / WR, kvh = blockIdx.y, group = blockIdx.z;
    if (WR == 1 && i >= R) return;
    const size_t at = ((size_t)group * a.hkv + kvh) * plan.slots * R + i;
    const int d = min(lane % LC, cols - 1), grp = (threadIdx.x % (64 * WR)) / LC;
    const float4 *src = reinterpret_cast<const float4 *>(part + at * a.hd) + d;
    const size_t step = (size_t)R * cols;
    float4 z[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) z[k] = src[min(grp + NG * k, plan.slots - 1) * step];
    float m[2], l[2], top = -INFINITY, sum = 0.f;
    bool seen[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const float *p = pml + 2 * (at + (size_t)min(lane + 64 * x, plan.slots - 1) * R);
        m[x] = p[0];
        l[x] = p[1];
    }
    const int plen = length(a.prefix_lens, a.prefix_len, group, a.max_prefix);
    const int olen = length(a.own_lens, a.own_len, group * a.rows + i / G, a.max_own);
    const int pu = split_range(plen, plan.pcap, 0).splits;
    const int ou = split_range(olen, plan.ocap, 0).splits;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int s = lane + 64 * x;
        if (!(s < pu || (s >= plan.pcap && s < plan.pcap + ou))) m[x] = -INFINITY;
        top = fmaxf(top, m[x]);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        seen[x] = m[x] != -INFINITY;
        m[x] = seen[x] ? l[x] * __builtin_amdgcn_exp2f(m[x] - top) : 0.f;
        sum += m[x];
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
    for (int x = 0; x < 2; ++x) w[wave][lane + 64 * x] = seen[x] ? m[x] * inv : -1.f;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](int s, const float4 &v) {
        const float x = w[wave][s];
        if (!(x < 0.f)) {   // a split that sees nothing of the row counts for nothing
            y.x = fmaf(v.x, x, y.x);
            y.y = fmaf(v.y, x, y.y);
            y.z = fmaf(v.z, x, y.z);
            y.w = fmaf(v.w, x, y.w);
        }
    };
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
        if (grp + NG * k < plan.slots) add(grp + NG * k, z[k]);
    for (int s = grp + NG * AHEAD; s < plan.slots; s += NG) add(s, src[s * step]);
#pragma unroll
    for (int o = LC; o < 64; o <<= 1) {
        y.x += __shfl_xor(y.x, o);
        y.y += __shfl_xor(y.y, o);
        y.z += __shfl_xor(y.z, o);
        y.w += __shfl_xor(y.w, o);
    }
    if (WR == 4) {
        if (lane < LC) col[wave][lane] = y;
        __syncthreads();
        if ((int)threadIdx.x >= cols) return;
        const float4 y0 = col[0][d], y1 = col[1][d], y2 = col[2][d], y3 = col[3][d];
        y = make_float4((y0.x + y1.x) + (y2.x + y3.x), (y0.y + y1.y) + (y2.y + y3.y),
                        (y0.z + y1.z) + (y2.z + y3.z), (y0.w + y1.w) + (y2.w + y3.w));
    }
    if (lane >= cols) return;
    float *out = a.out + (((size_t)group * a.rows + i / G) * a.hq + kvh * G + i % G) * a.hd;
    reinterpret_cast<float4 *>(out)[d] = y;
}

// prefix, own: the positions that the caches hold, or the lengths where the host knows them.
Plan plan_of(int groups, int rows, int hq, int hkv, int hd, int prefix, int own) {
    Plan p{};
    const int G = hq / hkv, R = rows * G;
    const int pt = (prefix + kTile - 1) / kTile, ot = (own + kTile - 1) / kTile;
    const int64_t seqs = (int64_t)groups * rows;
    p.gtiles = (G + 15) / 16;
    const int64_t units = (int64_t)groups * hkv, ob = seqs * hkv * p.gtiles;
    // Short caches and few sequences: a sequence's block reads the prefix for itself, and nothing
    // is merged.  That reads the prefix once a sequence, so it pays for a block a CU, or more
    // blocks of few tiles.  us in one launch / in two, 8 KV heads of 128, 4 query heads each:
    //   sequences        4        16        32        64       128       256
    //    6 tiles    9 /  9   10 / 15   10 / 19   16 / 20   28 / 24   50 / 33
    //   20 tiles   15 / 11   15 / 15   16 / 20   27 / 22   48 / 29   91 / 43
    // Over 1512 shapes of 1, 4 and 8 query heads of 32 to 256 for each of 2 and 8 KV heads, 1 to
    // 256 sequences and 3 to 20 tiles this is 3% slower than the faster one each time (always
    // one: 7%, two: 28%), at worst 1.65 times (one sequence, 20 tiles of 256: 21 / 13), where
    // one launch for all is 3.3.  29 tiles, 4 sequences in groups of 7 heads of 64: 17 / 11.
    const int tiles = std::max(pt + ot, 1);
    p.joined = tiles <= 20 && (ob <= 256 || ob * tiles <= 6144);
    // f32 MFMA for up to 32 rows, or limbs for 64 or 128 of them: us of 32 rows of 128 on 32767
    // positions 57 / 62, of 64 rows 104 / 76.
    p.dense = !p.joined && R > 32;
    p.rb = p.joined || p.dense ? 1 : std::min((R + 15) / 16, hd <= 128 ? 2 : 1);
    p.prows = p.dense ? (R <= 64 ? 64 : 128) : 16 * p.rb;
    p.nw = p.joined && hd <= 128 ? 8 : 4;
    p.ptiles = (R + p.prows - 1) / p.prows;
    if (p.joined) {
        p.ocap = p.slots = 1;
        p.oblocks = (int)ob;
        return p;
    }
    auto cap = [](int64_t want, int64_t blocks, int tiles) {
        const int64_t most = std::min<int64_t>((tiles + kMinTiles - 1) / kMinTiles, kMaxSplits);
        return (int)std::max<int64_t>(1, std::min<int64_t>(want / blocks, most));
    };
    // Blocks wanted, us with them / with half as many or half as many again: 256 for one pass of
    // few rows (32 rows on 4096 positions 17.4, 512: 20.2; 16 rows 12.8, 13.9), but 512 past
    // 128 dimensions (28 rows of 256, 7 groups of up to 13296: 169, 256: 186); 768 dense ones of
    // 64 rows, three a CU (64 rows on 4096 positions 20.2, 512: 25.3), 512 of 128 (32767
    // positions 119, 256: 148), and 256 past 128 dimensions, one a CU (256 rows of 256 on 8192
    // positions 199, 512: 219, on f32 MFMA 257; of 160 dimensions 95, on f32 MFMA 160).
    const int want = hd > 128 ? (p.dense ? 256 : 512) : !p.dense ? 256 : p.prows == 64 ? 768 : 512;
    p.pcap = pt ? cap(want, units * p.ptiles, pt) : 0;
    p.ocap = ot ? cap(256, ob, ot) : 0;
    p.pblocks = (int)((units * p.pcap + 7) / 8 * 8 * p.ptiles);
    p.oblocks = (int)(ob * p.ocap);
    p.slots = p.pcap + p.ocap;
    return p;
}

template <int LC>
void merge(const PrefixAttn &a, const Plan &p, const float *part, const float *pml, hipStream_t s) {
    const int R = a.rows * (a.hq / a.hkv);
    if (p.slots > 8)
        hipLaunchKernelGGL((k_prefix_merge<LC, 4>), dim3(R, a.hkv, a.groups), dim3(256), 0, s, a, p,
                           part, pml);
    else
        hipLaunchKernelGGL((k_prefix_merge<LC, 1>), dim3((R + 3) / 4, a.hkv, a.groups), dim3(256),
                           0, s, a, p, part, pml);
}

}  // namespace

bool prefix_attention_fits(int groups, int rows, int hq, int hkv, int hd, int prefix, int own) {
    const Plan p = plan_of(groups, rows, hq, hkv, hd, prefix, own);
    return ((int64_t)p.pblocks + p.oblocks) * 64 * p.nw <= kMaxThreads;
}

size_t prefix_attention_scratch(int groups, int rows, int hq, int hkv, int hd, int prefix,
                                int own) {
    const int slots = plan_of(groups, rows, hq, hkv, hd, prefix, own).slots;
    return slots > 1 ? (size_t)groups * rows * hq * slots * (hd + 2) * sizeof(float) : 0;
}

int launch_prefix_attention(const PrefixAttn &a, float *scratch, hipStream_t s) {
    const Plan p = plan_of(a.groups, a.rows, a.hq, a.hkv, a.hd,
                           a.prefix_lens ? a.max_prefix : a.prefix_len,
                           a.own_lens ? a.max_own : a.own_len);
    float *part = p.slots > 1 ? scratch : nullptr;
    const size_t rows = (size_t)a.groups * a.rows * a.hq;
    float *pml = part ? part + rows * p.slots * a.hd : nullptr;
    const dim3 grid(p.pblocks + p.oblocks);
#define TB_PREFIX(D)                                                                          \
    case D:                                                                                   \
        if (p.dense) k = p.prows == 64 ? k_prefix_dense<D, 16> : k_prefix_dense<D, 32>;       \
        if constexpr (D <= 128) {                                                             \
            if (!k && p.nw == 8) k = k_prefix_stream<D, 1, 8>;                                \
            if (!k && p.rb == 2) k = k_prefix_stream<D, 2, 4>;                                \
        }                                                                                     \
        if (!k) k = k_prefix_stream<D, 1, 4>;                                                 \
        break
    void (*k)(PrefixAttn, Plan, float *, float *) = nullptr;
    switch (a.hd) {
        TB_PREFIX(32);
        TB_PREFIX(64);
        TB_PREFIX(96);
        TB_PREFIX(128);
        TB_PREFIX(160);
        TB_PREFIX(192);
        TB_PREFIX(224);
        TB_PREFIX(256);
    }
#undef TB_PREFIX
    hipLaunchKernelGGL(k, grid, dim3(64 * p.nw), 0, s, a, p, part, pml);
    TB_LAUNCHED();
    if (part) {
        if (a.hd <= 32) merge<8>(a, p, part, pml, s);
        else if (a.hd <= 64) merge<16>(a, p, part, pml, s);
        else if (a.hd <= 128) merge<32>(a, p, part, pml, s);
        else merge<64>(a, p, part, pml, s);
        TB_LAUNCHED();
    }
    return TB_OK;
}

}  // namespace tb
