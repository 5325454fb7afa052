// Attention of a drafted tree's nodes over the cached prefix and their own
// ancestors, for GQA and an f32 cache.
//
//   o = sum_p w_p v_p / sum_p w_p,  w_p = exp(scale q.k_p - m), m the row's largest score
//
// over the positions p < len of the prefix and len + j for the bits j of the
// node's mask row.  One pass over K and V with a running maximum and sum.
//
// Both products run on f16 MFMA (v_mfma_f32_16x16x32_f16) with every f32 factor
// as two f16 limbs, x 2^s = hi + lo, and three products, hi hi + hi lo + lo hi:
// 22 bits and more of each factor, so that an error against exact arithmetic
// stays that of an f32 product, at a third of the f16 rate (the f32 MFMA has a
// sixteenth of it).  s puts the largest factor of a tile (K, V) or row (Q) at
// 2^14, so factors down to 2^-25 of it keep both limbs whole and smaller ones an
// error of 2^-39 of it.  Weights are taken as w 2^14 for the same reason.  Scores,
// running maxima, sums and outputs are f32.
#include <math.h>

#include <algorithm>

#include "gemv_common.hpp"
#include "tb_common.hpp"
#include "tree.hpp"

namespace tb {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;        // positions per tile of one wave
constexpr int kMaxSplits = 128;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kTop = 14;         // factors are scaled to below 2^(kTop + 1)

// Exponent of the largest magnitude given its bits, such that 2^(kTop - e) is a
// normal f32 (values below 2^-113 keep an error below the smallest f32).
__device__ __forceinline__ int exponent(uint32_t bits) {
    return min(max((int)(bits >> 23) - 127, kTop - 127), 127);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// The two f16 limbs of 8 values times sc, as MFMA operands.  x * sc is exact, so
// lo is the rounded rest of hi.
__device__ __forceinline__ void split8(const float (&x)[8], float sc, f16x8 &hi, f16x8 &lo) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        hi[j] = (_Float16)__builtin_fmaf(x[j], sc, 0.f);
        lo[j] = (_Float16)__builtin_fmaf(x[j], sc, -(float)hi[j]);
    }
}

// max(m, |a|, |b|) without the canonicalising moves of fmaxf.
__device__ __forceinline__ void max3_abs(float &m, float a, float b) {
    asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(m) : "v"(a), "v"(b));
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
constexpr uint32_t kInf = 0x7F800000u;

__device__ __forceinline__ float max_over_groups(float v) {   // lanes c, c + 16, c + 32, c + 48
    v = fmaxf(v, gemv::shfl_xor_u(v, 16));
    return fmaxf(v, gemv::shfl_xor_u(v, 32));
}
__device__ __forceinline__ float sum_over_groups(float v) {
    v += gemv::shfl_xor_u(v, 16);
    return v + gemv::shfl_xor_u(v, 32);
}
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1)
        v = max(v, __float_as_uint(gemv::shfl_xor_u(__uint_as_float(v), m)));
    return __builtin_amdgcn_readfirstlane(v);
}

// Tiles of one split: whole rounds of the block's four waves.
__host__ __device__ inline int tiles_per_split(int tiles, int nsplit) {
    return ((tiles + nsplit - 1) / nsplit + 3) / 4 * 4;
}

// A block takes 16 * RB query rows of one KV head, a row being a (node, head of
// the group) pair i = node * G + head, and a range of the positions.  Its four
// waves take tiles of 32 positions in turn, each with its own running maximum,
// sum and output; they meet in LDS once at the end.  So nothing in the loop
// waits for another wave, and K and V go from memory to MFMA operands in
// registers:
//   lane (g, c) = (lane / 16, lane % 16) has A[c][8g ..] and B[8g ..][c] of a
//   product of depth 32, and gets D[4g + r][c] in register r;
//   S^T = K Q^T: A = 16 positions, position c with the 8 dimensions 4g.. and
//     16 + 4g.. of each 32 (a K row is read in whole 64-byte pieces); B = the
//     query rows, from LDS in operand order;
//   O^T = V^T P^T: A's row c of block (b, j) is dimension 64 b + 4 c + j and its
//     depth 8g + i is position 4g + i (i < 4) or 16 + 4g + i - 4, the positions
//     whose scores the lane holds for row c, so P^T needs no exchange and a V
//     row is read in 256-byte pieces.
// The next tile's K is requested when this one's limbs are built, V likewise.
//
// A tile with infinities (or NaN, behind the prefix) takes its sums one by one
// in f32, so that positions that a row does not see stay out of its result.
template <int DP, int RB>
__global__ __launch_bounds__(256, RB * DP <= 64 ? 2 : 1) void k_tree_attn(TreeAttn a, int nsplit,
                                                                         float *__restrict__ part,
                                                                         float *__restrict__ pml) {
    constexpr int NS = DP / 32, NB = DP / 64, ROWS = 16 * RB;
    __shared__ __attribute__((aligned(16))) float lds[ROWS * DP];   // Q limbs; then the outputs
    __shared__ float sm[4][ROWS], sl[4][ROWS];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, c = lane & 15, g = lane >> 4;
    const int G = a.hq / a.hkv, R = a.n * G, D = a.hd, words = (a.n + 31) / 32;
    const int split = blockIdx.x, kvh = blockIdx.y % a.hkv, i0 = blockIdx.y / a.hkv * ROWS;
    const int b = blockIdx.z;
    const int len = prefix_len(a.kv_lens, a.kv_len, b, a.max_seq), end = min(len + a.n, a.max_seq);
    const int tiles = (end + kTile - 1) / kTile, tps = tiles_per_split(tiles, nsplit);
    const int t0 = split * tps, t1 = min(tiles, t0 + tps);
    if (split > 0 && t0 >= t1) return;   // the merge skips this split
    const float *kb = a.k.p + b * a.k.sb + kvh * a.k.sh + 4 * g;
    const float *vb = a.v.p + b * a.v.sb + kvh * a.v.sh + 4 * c;

    float kr[2][NS][8], vr[8][NB][4];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) kr[0][s][j] = kr[1][s][j] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int q = 0; q < NB; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j) vr[i][q][j] = 0.f;
    auto load_k = [&](int tile) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float *r = kb + min(tile * kTile + 16 * h + c, end - 1) * a.k.ss;
#pragma unroll
            for (int s = 0; s < NS; ++s)
                if (32 * s < D) {
                    const float4 x = *reinterpret_cast<const float4 *>(r + 32 * s);
                    const float4 y = *reinterpret_cast<const float4 *>(r + 32 * s + 16);
                    float *k = kr[h][s];
                    k[0] = x.x; k[1] = x.y; k[2] = x.z; k[3] = x.w;
                    k[4] = y.x; k[5] = y.y; k[6] = y.z; k[7] = y.w;
                }
        }
    };
    auto load_v = [&](int tile) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int p = min(tile * kTile + (i < 4 ? 4 * g + i : 12 + 4 * g + i), end - 1);
            const float *r = vb + p * a.v.ss;
#pragma unroll
            for (int q = 0; q < NB; ++q)
                if (64 * q + 4 * c < D) {
                    const float4 x = *reinterpret_cast<const float4 *>(r + 64 * q);
                    vr[i][q][0] = x.x; vr[i][q][1] = x.y; vr[i][q][2] = x.z; vr[i][q][3] = x.w;
                }
        }
    };
    const int first = t0 + wave;
    if (first < t1) {
        load_k(first);
        load_v(first);
    }

    // The query rows' limbs, in B-operand order: [row block][32 dimensions][limb][lane].
    f16x8 *qs = reinterpret_cast<f16x8 *>(lds);
    for (int rb = wave; rb < RB; rb += 4) {
        const int i = i0 + 16 * rb + c, iq = i < R ? i : 0;
        const float *q = a.q + (((size_t)b * a.n + iq / G) * a.hq + kvh * G + iq % G) * D + 4 * g;
        float x[NS][8];
        float top = 0.f;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            float4 u = make_float4(0.f, 0.f, 0.f, 0.f), v = u;
            if (32 * s < D) {
                u = *reinterpret_cast<const float4 *>(q + 32 * s);
                v = *reinterpret_cast<const float4 *>(q + 32 * s + 16);
            }
            x[s][0] = u.x; x[s][1] = u.y; x[s][2] = u.z; x[s][3] = u.w;
            x[s][4] = v.x; x[s][5] = v.y; x[s][6] = v.z; x[s][7] = v.w;
#pragma unroll
            for (int j = 0; j < 8; j += 2) max3_abs(top, x[s][j], x[s][j + 1]);
        }
        const int e = exponent(__float_as_uint(max_over_groups(top)));
        if (g == 0) sm[0][16 * rb + c] = __int_as_float(e);
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            f16x8 hi, lo;
            split8(x[s], pow2(kTop - e), hi, lo);
            qs[((rb * NS + s) * 2 + 0) * 64 + lane] = hi;
            qs[((rb * NS + s) * 2 + 1) * 64 + lane] = lo;
        }
    }
    // Per row block: the lane's row c.
    const int32_t *mrow[RB];
    bool live[RB];
    float m[RB], l[RB];
    int qe[RB];
    f32x4 o[RB][NB][4];
    const uint32_t last_bits = a.n % 32 ? (1u << (a.n % 32)) - 1 : ~0u;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int i = i0 + 16 * rb + c;
        mrow[rb] = a.mask + b * a.mask_sb + (int64_t)((i < R ? i : 0) / G) * words;
        uint32_t any = 0;
        for (int w = g; w < words; w += 4)
            any |= (uint32_t)mrow[rb][w] & (w == words - 1 ? last_bits : ~0u);
        live[rb] = i < R && max_over_groups(any ? 1.f : 0.f) > 0.f;
        m[rb] = -INFINITY;
        l[rb] = 0.f;
#pragma unroll
        for (int q = 0; q < NB; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[rb][q][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __syncthreads();
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) qe[rb] = __float_as_int(sm[0][16 * rb + c]);
    int ve = 0, ve_top = -1000;   // exponent of the outputs' scale; the largest one so far
    const float f = a.scale * kLog2e;

    for (int tile = first; tile < t1; tile += 4) {
        const int p0 = tile * kTile;
        const bool open = p0 + kTile <= len;   // every live row sees every position
        // ---- K: the tile's scale, its limbs, the next tile's request
        uint32_t top;
        {
            float mx = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int s = 0; s < NS; ++s)
#pragma unroll
                    for (int j = 0; j < 8; j += 2) max3_abs(mx, kr[h][s][j], kr[h][s][j + 1]);
            top = wave_max_bits(__float_as_uint(mx) & 0x7FFFFFFFu);
        }
        const bool slow_k = top >= kInf;
        const int ke = exponent(top);
        f16x8 kh[2][NS], kl[2][NS];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int s = 0; s < NS; ++s) split8(kr[h][s], pow2(kTop - ke), kh[h][s], kl[h][s]);
        if (tile + 4 < t1) load_k(tile + 4);
        // ---- scores, running maxima, weights
        f16x8 ph[RB], pl[RB];
        float alpha[RB];
        bool moved = false;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
            float s8[8];
            if (!slow_k) {
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    const f16x8 qh = qs[((rb * NS + s) * 2 + 0) * 64 + lane];
                    const f16x8 ql = qs[((rb * NS + s) * 2 + 1) * 64 + lane];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl[h][s], qh, acc[h], 0, 0, 0);
                        acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[h][s], ql, acc[h], 0, 0, 0);
                        acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[h][s], qh, acc[h], 0, 0, 0);
                    }
                }
                const float fx = ldexpf(f, qe[rb] + ke - 2 * kTop);
#pragma unroll
                for (int j = 0; j < 8; ++j) s8[j] = acc[j >> 2][j & 3] * fx;
            } else {
                const int i = min(i0 + 16 * rb + c, R - 1);
                const float *q = a.q + (((size_t)b * a.n + i / G) * a.hq + kvh * G + i % G) * D;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int p = min(p0 + (j < 4 ? 4 * g + j : 12 + 4 * g + j), end - 1);
                    const float *k = a.k.p + b * a.k.sb + kvh * a.k.sh + p * a.k.ss;
                    float s = 0.f;
                    for (int d = 0; d < D; ++d) s = fmaf(q[d], k[d], s);
                    s8[j] = s * f;
                }
            }
            if (!open) {
                // 32 bits: which of the tile's positions row c sees
                uint32_t see = 0;
                const int at = p0 - len;   // the tree's bit of the tile's first position
                if (live[rb]) {
                    if (at < 0) {
                        see = (1u << -at) - 1;
                        see |= (uint32_t)mrow[rb][0] << -at;
                    } else {
                        const int w = at >> 5, sh = at & 31;
                        see = (uint32_t)mrow[rb][w] >> sh;
                        if (sh && w + 1 < words) see |= (uint32_t)mrow[rb][w + 1] << (32 - sh);
                    }
                    if (end - p0 < 32) see &= (1u << (end - p0)) - 1;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!(see >> (j < 4 ? 4 * g + j : 12 + 4 * g + j) & 1)) s8[j] = -INFINITY;
            }
            float mt = s8[0];
#pragma unroll
            for (int j = 1; j < 8; ++j) mt = fmaxf(mt, s8[j]);
            const float mn = fmaxf(m[rb], max_over_groups(mt));
            const float base = mn == -INFINITY ? 0.f : mn;   // nothing seen so far: every weight 0
            alpha[rb] = __builtin_amdgcn_exp2f(m[rb] - base);
            moved |= m[rb] != mn;
            m[rb] = mn;
            float sum = 0.f;
            float p8[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p8[j] = __builtin_amdgcn_exp2f(s8[j] - base);
                sum += p8[j];
            }
            l[rb] = fmaf(l[rb], alpha[rb], sum);
            split8(p8, pow2(kTop), ph[rb], pl[rb]);
        }
        // ---- V: the tile's scale, the outputs' rescale, the limbs, the next request
        if (open) {
            float mx = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int q = 0; q < NB; ++q) {
                    max3_abs(mx, vr[i][q][0], vr[i][q][1]);
                    max3_abs(mx, vr[i][q][2], vr[i][q][3]);
                }
            top = __float_as_uint(mx) & 0x7FFFFFFFu;
        } else {   // NaN too: a row that does not see its position must not get it
            top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int q = 0; q < NB; ++q)
#pragma unroll
                    for (int j = 0; j < 4; ++j) top = max(top, abs_bits(vr[i][q][j]));
        }
        top = wave_max_bits(top);
        const bool slow_v = top >= kInf;
        if (slow_v) {   // the finite values' scale
            top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int q = 0; q < NB; ++q)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t x = abs_bits(vr[i][q][j]);
                        top = max(top, x < kInf ? x : 0u);
                    }
            top = wave_max_bits(top);
        }
        // The outputs keep their scale while the tile fits it and loses at most 6
        // bits of range to it; 64 bits below the largest scale it stays (their f32
        // must not overflow).
        const int e = exponent(top);
        ve_top = max(ve_top, e);
        int down = 0;
        if (e > ve || e < ve - 6) {
            const int to = max(e, ve_top - 64);
            down = ve - to;
            ve = to;
        }
        if (__any(moved) || down != 0) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const float x = ldexpf(alpha[rb], min(down, 120));
#pragma unroll
                for (int q = 0; q < NB; ++q)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[rb][q][j] *= x;
            }
        }
        if (!slow_v) {
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                f16x8 vh[4], vl[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = vr[i][q][j];
                    split8(x, pow2(kTop - ve), vh[j], vl[j]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        f32x4 &x = o[rb][q][j];
                        x = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl[j], ph[rb], x, 0, 0, 0);
                        x = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh[j], pl[rb], x, 0, 0, 0);
                        x = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh[j], ph[rb], x, 0, 0, 0);
                    }
            }
        } else {
            const float *v = a.v.p + b * a.v.sb + kvh * a.v.sh + 16 * g;
            for (int i = 0; i < 32; ++i) {
                const int from = i >> 3, j = i & 7;
                const int p = min(p0 + (j < 4 ? 4 * from + j : 12 + 4 * from + j), end - 1);
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    float w = 0.f;
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (k == j) w = (float)ph[rb][k] + (float)pl[rb][k];
                    w = __shfl(w, c + 16 * from);
                    if (w == 0.f) continue;
#pragma unroll
                    for (int q = 0; q < NB; ++q)
#pragma unroll
                        for (int y = 0; y < 16; ++y)
                            if (64 * q + 16 * g < D)
                                o[rb][q][y & 3][y >> 2] =
                                    fmaf(w, ldexpf(v[p * a.v.ss + 64 * q + y], kTop - ve),
                                         o[rb][q][y & 3][y >> 2]);
                }
            }
        }
        if (tile + 4 < t1) load_v(tile + 4);
    }

    // ---- the four waves' outputs, brought to one maximum and summed in wave order
    __syncthreads();   // every wave is done with the query rows and sm
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        if (!live[rb]) m[rb] = -INFINITY;
        l[rb] = live[rb] ? sum_over_groups(l[rb]) : 0.f;
        if (g == 0) {
            sm[wave][16 * rb + c] = m[rb];
            sl[wave][16 * rb + c] = l[rb];
        }
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (wave == w) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const int r = 16 * rb + c;
                const float top = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
                const float x = m[rb] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[rb] - top);
#pragma unroll
                for (int q = 0; q < NB; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float4 *d = reinterpret_cast<float4 *>(lds + r * DP + 64 * q + 16 * g) + i;
                        float4 y = w ? *d : make_float4(0.f, 0.f, 0.f, 0.f);
                        if (x != 0.f) {
                            y.x = fmaf(ldexpf(o[rb][q][0][i], ve - 2 * kTop), x, y.x);
                            y.y = fmaf(ldexpf(o[rb][q][1][i], ve - 2 * kTop), x, y.y);
                            y.z = fmaf(ldexpf(o[rb][q][2][i], ve - 2 * kTop), x, y.z);
                            y.w = fmaf(ldexpf(o[rb][q][3][i], ve - 2 * kTop), x, y.w);
                        }
                        *d = y;
                    }
            }
        }
        __syncthreads();
    }
    const int cols = D / 4;
    for (int x = t; x < ROWS * cols; x += 256) {
        const int r = x / cols, d = x % cols, i = i0 + r;
        if (i >= R) break;
        const float top = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w)
            if (sm[w][r] != -INFINITY) sum = fmaf(sl[w][r], __builtin_amdgcn_exp2f(sm[w][r] - top), sum);
        float4 y = *reinterpret_cast<const float4 *>(lds + r * DP + 4 * d);
        if (part) {
            const size_t at = (((size_t)b * a.hkv + kvh) * nsplit + split) * R + i;
            reinterpret_cast<float4 *>(part + at * D)[d] = y;
            if (d == 0) {
                pml[2 * at] = top;
                pml[2 * at + 1] = sum;
            }
        } else {
            const float inv = sum == 0.f ? 0.f : 1.0f / sum;
            float *out = a.out + (((size_t)b * a.n + i / G) * a.hq + kvh * G + i % G) * D;
            reinterpret_cast<float4 *>(out)[d] =
                make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
        }
    }
}

// The splits' outputs brought to one maximum: a thread per four columns of a row.
__global__ __launch_bounds__(256) void k_tree_merge(TreeAttn a, int nsplit,
                                                    const float *__restrict__ part,
                                                    const float *__restrict__ pml) {
    const int G = a.hq / a.hkv, R = a.n * G, cols = a.hd / 4, per = 256 / cols;
    const int r = threadIdx.x / cols, d = threadIdx.x % cols;
    const int i = blockIdx.x * per + r, kvh = blockIdx.y, b = blockIdx.z;
    if (r >= per || i >= R) return;
    const int len = prefix_len(a.kv_lens, a.kv_len, b, a.max_seq), end = min(len + a.n, a.max_seq);
    const int tiles = (end + kTile - 1) / kTile, tps = tiles_per_split(tiles, nsplit);
    const int used = tps ? (tiles + tps - 1) / tps : 0;
    const size_t at = ((size_t)b * a.hkv + kvh) * nsplit * R + i;
    float top = -INFINITY;
    for (int s = 0; s < used; ++s) top = fmaxf(top, pml[2 * (at + (size_t)s * R)]);
    float sum = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < used; ++s) {
        const size_t p = at + (size_t)s * R;
        const float m = pml[2 * p];
        if (m == -INFINITY) continue;
        const float x = __builtin_amdgcn_exp2f(m - top);
        const float4 z = reinterpret_cast<const float4 *>(part + p * a.hd)[d];
        sum = fmaf(pml[2 * p + 1], x, sum);
        y.x = fmaf(z.x, x, y.x);
        y.y = fmaf(z.y, x, y.y);
        y.z = fmaf(z.z, x, y.z);
        y.w = fmaf(z.w, x, y.w);
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    float *out = a.out + (((size_t)b * a.n + i / G) * a.hq + kvh * G + i % G) * a.hd;
    reinterpret_cast<float4 *>(out)[d] = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
}

struct Plan {
    int dp, rb, nsplit;
};

Plan plan(int batch, int n, int hq, int hkv, int hd, int max_len) {
    Plan p;
    p.dp = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    const int R = n * (hq / hkv);
    p.rb = R <= 16 ? 1 : R <= 32 || p.dp == 256 ? 2 : 4;
    const int rtiles = (R + 16 * p.rb - 1) / (16 * p.rb), tiles = (max_len + kTile - 1) / kTile;
    const int64_t blocks = (int64_t)rtiles * hkv * batch;
    const int64_t want = std::max<int64_t>(1, 512 / blocks);
    p.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({want, (tiles + 3) / 4, kMaxSplits}));
    return p;
}

}  // namespace

size_t tree_attention_scratch(int batch, int n, int hq, int hkv, int hd, int max_len) {
    const int ns = plan(batch, n, hq, hkv, hd, max_len).nsplit;
    return ns > 1 ? (size_t)batch * hq * n * ns * (hd + 2) * sizeof(float) : 0;
}

int launch_tree_attention(const TreeAttn &a, int max_len, float *scratch, hipStream_t s) {
    const Plan p = plan(a.batch, a.n, a.hq, a.hkv, a.hd, max_len);
    const int R = a.n * (a.hq / a.hkv), rtiles = (R + 16 * p.rb - 1) / (16 * p.rb);
    float *part = p.nsplit > 1 ? scratch : nullptr;
    float *pml = part ? part + (size_t)a.batch * a.hq * a.n * p.nsplit * a.hd : nullptr;
    const dim3 grid(p.nsplit, a.hkv * rtiles, a.batch);
#define TB_TA(DP, RB)                                                                        \
    if (p.dp == DP && p.rb == RB)                                                            \
    hipLaunchKernelGGL((k_tree_attn<DP, RB>), grid, dim3(256), 0, s, a, p.nsplit, part, pml)
    TB_TA(64, 1);
    TB_TA(64, 2);
    TB_TA(64, 4);
    TB_TA(128, 1);
    TB_TA(128, 2);
    TB_TA(128, 4);
    TB_TA(256, 1);
    TB_TA(256, 2);
#undef TB_TA
    TB_LAUNCHED();
    if (part) {
        const int per = 256 / (a.hd / 4);
        hipLaunchKernelGGL(k_tree_merge, dim3((R + per - 1) / per, a.hkv, a.batch), dim3(256), 0, s,
                           a, p.nsplit, part, pml);
        TB_LAUNCHED();
    }
    return TB_OK;
}

}  // namespace tb
