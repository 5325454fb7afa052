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
// sixteenth of it).  s puts the largest factor of a few positions (K, V) or a row
// (Q) at 2^14, so factors down to 2^-17 of it keep both limbs whole and smaller ones
// an error of 2^-39 of it.  Weights are taken as w 2^7 for the same reason, less
// where the positions' V is smaller than others', with low limbs times 2^11: 22 bits
// down to 2^-21 of the row's reference score's weight, and an error of 2^-43 of that one
// times the largest V for every position below, which add up.  The reference falls with
// the scores (kDrop), so that only the tile of a large weight whose V is zero shows it.
// Behind the prefix, where rows see different positions, a tile whose K or V
// spread wider than that is worked in f32 (as one with infinities is), so that
// nothing that a row does not see costs it bits.  Scores, running maxima, sums and
// outputs are f32.
#include <math.h>

#include <algorithm>

#include "gemv_common.hpp"
#include "tb_common.hpp"
#include "tree.hpp"

namespace tb {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// For lambdas that are called more than once, which would become functions with their
// captures in memory.
#define TB_INLINE __attribute__((always_inline))

constexpr int kMaxSplits = 128;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kTop = 14;         // factors are scaled to below 2^(kTop + 1)
// A row's reference maximum follows its scores only when they pass it by more than
// 2^kLag: the outputs' rescale (a third of a tile's vector work where one of 32
// rows needs it in most tiles) then runs in few of them.  Weights reach 2^kLag and
// are scaled by 2^kWeight, so that they stay below 2^(kTop + 2), the f16 range.
constexpr float kLag = 8.f;
constexpr int kWeight = 7;
// The low limb of a weight is kept times 2^kLow, as f16's smallest steps would take what
// is below 2^-32 of the reference; V's high limb is divided by it for that product.
// (32767 positions 21.1 below a score whose V is zero: 1.53e-5 without, the result is
// 2.27e-5.)  It costs 40 vector instructions a tile: 40.0 / 139 us without, 41.2 / 144.
constexpr int kLow = 11;
// The reference also follows down, to a tile's largest score that is more than 2^kDrop
// below it: where the largest weights meet a V of zero, the small ones are the result.
// As far down as the sum of weights stays below 2^kRoom and the outputs within f32.
// Scores whose standard deviation is 11 powers of two take 148 us with 24, 150 with 20
// and 136 without, ordinary ones the same.
constexpr float kDrop = 24.f;
constexpr int kRoom = 36;

constexpr int kBias = 1 << 10, kSlow = 1 << 20;
constexpr int kNoV = -1000;          // in place of an exponent: none yet
constexpr int kLeast = kTop - 127;   // the smallest exponent()

// Exponent of the largest magnitude given its bits, such that 2^(kTop - e) is a
// normal f32 (values below 2^-113 keep an error below the smallest f32).
__device__ __forceinline__ int exponent(uint32_t bits) {
    return min(max((int)(bits >> 23) - 127, kLeast), 127);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// The two f16 limbs of 8 values times sc, x sc being exact: hi the rounded
// product, lo its rounded rest.  (`one` keeps a v_fma_mix of the f16 and f32
// factors where a constant would make it a conversion and a difference.)
__device__ __forceinline__ void split8(const float (&x)[8], float sc, f16x8 &hi, f16x8 &lo) {
    float one = 1.f;
    asm("" : "+s"(one));
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const f32x2 y = {x[j] * sc, x[j + 1] * sc};
        const f16x2 h = __builtin_convertvector(y, f16x2);
        const f32x2 r = {__builtin_fmaf(y.x, one, -(float)h.x), __builtin_fmaf(y.y, one, -(float)h.y)};
        const f16x2 e = __builtin_convertvector(r, f16x2);
        hi[j] = h.x; hi[j + 1] = h.y;
        lo[j] = e.x; lo[j + 1] = e.y;
    }
}

// The same of N loaded values on their way to LDS, an instruction per limb:
// v_fma_mix takes f32 and f16 factors side by side and writes either half of a
// register.  Only for results that no MFMA reads: the compiler does not count the
// wait states from inline assembly to one.
template <int N>
using f16v = _Float16 __attribute__((ext_vector_type(N)));
template <int N>
__device__ __forceinline__ void split_to_lds(const float (&x)[N], float sc, f16v<N> &hi,
                                             f16v<N> &lo) {
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        f16x2 h, r;
        asm("v_fma_mixlo_f16 %0, %1, %2, 0" : "=v"(h) : "v"(x[j]), "v"(sc));
        asm("v_fma_mixhi_f16 %0, %1, %2, 0" : "+v"(h) : "v"(x[j + 1]), "v"(sc));
        asm("v_fma_mixlo_f16 %0, %1, %2, -%3 op_sel_hi:[0,0,1]"
            : "=v"(r)
            : "v"(x[j]), "v"(sc), "v"(h));
        asm("v_fma_mixhi_f16 %0, %1, %2, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]"
            : "+v"(r)
            : "v"(x[j + 1]), "v"(sc), "v"(h));
        hi[j] = h.x; hi[j + 1] = h.y;
        lo[j] = r.x; lo[j + 1] = r.y;
    }
}

// The limbs of 8 weights given times 2^kLow, the low one times 2^kLow.
__device__ __forceinline__ void split_weights(const float (&y)[8], f16x8 &hi, f16x8 &lo) {
    float up = (float)(1 << kLow), down = 1.f / (1 << kLow);
    asm("" : "+s"(up));
    asm("" : "+s"(down));
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        f16x2 h = {(_Float16)__builtin_fmaf(y[j], down, 0.f),
                   (_Float16)__builtin_fmaf(y[j + 1], down, 0.f)};
        asm("" : "+v"(h));
        hi[j] = h.x; hi[j + 1] = h.y;
        lo[j] = (_Float16)__builtin_fmaf(-(float)h.x, up, y[j]);
        lo[j + 1] = (_Float16)__builtin_fmaf(-(float)h.y, up, y[j + 1]);
    }
}

// V's high limbs for the weights' low ones.
__device__ __forceinline__ f16x8 low(const f16x8 &v) { return v * (_Float16)(1.f / (1 << kLow)); }

// max(m, |a|, |b|) of loaded values without the canonicalising moves of fmaxf.
__device__ __forceinline__ void max3_abs(float &m, float a, float b) {
    asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(m) : "v"(a), "v"(b));
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
constexpr uint32_t kInf = 0x7F800000u;
template <int N>
__device__ __forceinline__ uint32_t top_bits(const float (&x)[N]) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) top = max(top, abs_bits(x[j]));
    return top;
}
// low takes the bits of the smallest magnitude but 0, turned over.
__device__ __forceinline__ void low_bits(uint32_t &low, uint32_t bits) {
    low = max(low, bits ? ~bits : 0u);
}
// Whether the smallest of some positions' magnitudes is so far below 2^top that limbs in
// one scale would not keep it whole (they do down to 2^-17), with a margin: 6 bits of
// the outputs' scale, and that the smallest is one over a few dimensions.
__device__ __forceinline__ bool spread(int top, uint32_t low) {
    return low && top - exponent(~low) > 10;
}

// Over the lanes c, c + 16, c + 32, c + 48: a swap of 16- or 32-lane halves of a
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
// Two maxima over the wave side by side: rotations within 16 lanes, then as above.
__device__ __forceinline__ void wave_max_bits(uint32_t &a, uint32_t &b) {
#define TB_ROR(n)                                                                       \
    {                                                                                   \
        const uint32_t x = (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0x120 + n, 0xF, 0xF, true); \
        const uint32_t y = (uint32_t)__builtin_amdgcn_mov_dpp((int)b, 0x120 + n, 0xF, 0xF, true); \
        a = max(a, x);                                                                  \
        b = max(b, y);                                                                  \
    }
    TB_ROR(8) TB_ROR(4) TB_ROR(2) TB_ROR(1)
#undef TB_ROR
    auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    auto s = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    a = max(r[0], r[1]);
    b = max(s[0], s[1]);
    r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    s = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    a = __builtin_amdgcn_readfirstlane(max(r[0], r[1]));
    b = __builtin_amdgcn_readfirstlane(max(s[0], s[1]));
}

// What this wave wrote to LDS before is there for what it reads after.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// x, which the compiler must take as new: what follows from it is worked out where
// it is used instead of waiting in registers across the loop.
__device__ __forceinline__ int fresh(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// The lane, counted anew.
__device__ __forceinline__ int fresh_lane() {
    int x;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
    return x;
}

// Position j of lane group g's scores among a tile's.
__device__ __forceinline__ int position(int j, int g) {
    return 32 * (j >> 3) + 16 * (j >> 2 & 1) + 4 * g + (j & 3);
}

// Which of the positions p0 .. p0 + 31 a row sees, as bits.
__device__ __forceinline__ uint32_t seen(const int32_t *mrow, int words, int p0, int len, int end) {
    const int at = p0 - len;   // the tree's bit of the first one
    uint32_t see = 0;
    if (at <= -32) {
        see = ~0u;
    } else if (at < 0) {
        see = ((1u << -at) - 1) | (uint32_t)mrow[0] << -at;
    } else if (at >> 5 < words) {
        const int w = at >> 5, sh = at & 31;
        see = (uint32_t)mrow[w] >> sh;
        if (sh && w + 1 < words) see |= (uint32_t)mrow[w + 1] << (32 - sh);
    }
    if (end - p0 < 32) see = end > p0 ? see & ((1u << (end - p0)) - 1) : 0;
    return see;
}

// Query row i's limbs for lane group g, and its scale's exponent; with the sign of
// the score's factor, which is then positive.  Rows past the last one repeat row 0.
template <int NS>
__device__ __forceinline__ void query_row(const TreeAttn &a, int b, int kvh, int i, int g,
                                          f16x8 (&qh)[NS], f16x8 (&ql)[NS], int &qe) {
    const int G = a.hq / a.hkv, D = a.hd;
    i = i < a.n * G ? i : 0;
    const float *q = a.q + (((size_t)b * a.n + i / G) * a.hq + kvh * G + i % G) * D + 4 * g;
    float x[NS][8];
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int d = 64 * (s >> 1);
        float4 u = *reinterpret_cast<const float4 *>(q + 16 * (s & 1) + (d < D ? d : 0));
        float4 v = *reinterpret_cast<const float4 *>(q + 16 * (s & 1) + (d + 32 < D ? d + 32 : 0));
        if (d >= D) u = make_float4(0.f, 0.f, 0.f, 0.f);
        if (d + 32 >= D) v = make_float4(0.f, 0.f, 0.f, 0.f);
        x[s][0] = u.x; x[s][1] = u.y; x[s][2] = u.z; x[s][3] = u.w;
        x[s][4] = v.x; x[s][5] = v.y; x[s][6] = v.z; x[s][7] = v.w;
#pragma unroll
        for (int j = 0; j < 8; j += 2) max3_abs(top, x[s][j], x[s][j + 1]);
    }
    qe = exponent(abs_bits(max_over_groups(top)));
#pragma unroll
    for (int s = 0; s < NS; ++s)
        split8(x[s], a.scale < 0.f ? -pow2(kTop - qe) : pow2(kTop - qe), qh[s], ql[s]);
}

// Whether a mask row has a bit among the tree's n, its words shared by the lane groups.
__device__ __forceinline__ bool any_bit(const int32_t *row, int words, int n, int g) {
    const uint32_t last = n % 32 ? (1u << (n % 32)) - 1 : ~0u;
    uint32_t any = 0;
    for (int w = g; w < words; w += 4) any |= (uint32_t)row[w] & (w == words - 1 ? last : ~0u);
    return max_over_groups(any ? 1.f : 0.f) > 0.f;
}

// Row i's scores with the lane's positions of a tile whose K is not finite.
template <int N>
__device__ __forceinline__ void scores_in_f32(const TreeAttn &a, int b, int kvh, int i, int p0,
                                              int end, int g, float (&s8)[N]) {
    const int G = a.hq / a.hkv, D = a.hd;
    i = fresh(i);
    const float *q = a.q + (((size_t)b * a.n + i / G) * a.hq + kvh * G + i % G) * D;
    const float *kb = a.k.p + b * a.k.sb + kvh * a.k.sh;
    uint32_t off[N];   // in 16-byte units from the tile's first row
#pragma unroll
    for (int j = 0; j < N; ++j) {
        off[j] = min(position(j, g), end - 1 - p0) * (uint32_t)(a.k.ss / 4);
        s8[j] = 0.f;
    }
    const float4 *k = reinterpret_cast<const float4 *>(kb + p0 * a.k.ss);
    for (int d = 0; d < D / 4; ++d) {
        const float4 x = reinterpret_cast<const float4 *>(q)[d];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float4 y = k[off[j] + d];
            s8[j] = fmaf(x.w, y.w, fmaf(x.z, y.z, fmaf(x.y, y.y, fmaf(x.x, y.x, s8[j]))));
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) s8[j] *= a.scale * kLog2e;
}

// The least exponent of a weight's scale.  Where V is that small against the outputs'
// scale 2^(kTop - oe), the limbs (below 2^(kTop + 1)) come out too large, by less than
// 2^(oe - 60), and the sum still gets every weight down to 2^-66.
constexpr int kWeightLow = -60;

// Adds a tile's V, taken in f32, with its weights (row c's in lane group `from` for its
// positions) to the outputs of row c, whose scale is `by`.  The scale is such that no V
// passes 2^90 in it (raise()).
template <int NB, int N>
__device__ __forceinline__ void add_in_f32(const TreeAttn &a, const float *vb, int p0, int end,
                                           int g, int c, const float (&p)[N], float by,
                                           f32x4 (&o)[NB][4]) {
    for (int i = 0; i < 4 * N; ++i) {
        const int sub = i >> 5, from = i >> 3 & 3, j = i & 7;
        const float *v = vb + min(p0 + 32 * sub + position(j, from), end - 1) * a.v.ss;
        float w = 0.f;
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k == j + 8 * sub) w = p[k];
        w = __shfl(w, c + 16 * from);
        if (w == 0.f) continue;   // not seen, NaN or not
#pragma unroll
        for (int q = 0; q < NB; ++q)
#pragma unroll
            for (int y = 0; y < 16; ++y)
                if (64 * q + 16 * g < a.hd)
                    o[q][y & 3][y >> 2] = fmaf(w, v[64 * q + 16 * g + y] * by, o[q][y & 3][y >> 2]);
    }
}

// What a partial result's maximum is merged as: -inf when it saw nothing, infinity
// when its sum is NaN without a score to refer to (a NaN among the queries), which
// makes the row NaN.
__device__ __forceinline__ float reference(bool live, float m, float sum) {
    return !live ? -INFINITY : sum != sum && m == -INFINITY ? INFINITY : m;
}

// A row's reference m, of sum `sum` so far, for a tile whose largest score is `top`: down
// to that where it is more than 2^kDrop below, but the outputs, at most sum 2^(kWeight +
// kTop + 1 + oe_top - oe) and through rescale() 2^64 times as much, stay below 2^127.
__device__ __forceinline__ float drop(float m, float top, float sum, int oe, int oe_top) {
    const int least = (int)(__float_as_uint(sum) >> 23) - 127;
    const int room = min(kRoom, 96 - (oe_top - oe)) - least;
    const float to = fmaxf(top, m - (float)min(room, kRoom));
    return top < m - kDrop && top > -INFINITY && room > 0 ? to : m;
}

// The outputs' scale 2^(kTop - oe) for a tile of V's exponent ve: how far it moves
// down.  It stays while the tile fits it and loses at most 6 bits of range to it, and
// stays 64 bits below the largest one so far (the outputs' f32 must not overflow).
__device__ __forceinline__ int rescale(int ve, int &oe, int &oe_top) {
    oe_top = max(oe_top, ve);
    if (ve <= oe && ve >= oe - 6) return 0;
    const int to = max(ve, oe_top - 64), down = oe - to;
    oe = to;
    return down;
}

// The same before add_in_f32, of V up to 2^ve: it may stay up to 90 below, so that the
// largest V of one row and the ordinary ones of another both fit f32.
__device__ __forceinline__ int raise(int ve, int &oe, int &oe_top) {
    oe_top = max(oe_top, ve);
    const int to = max(oe, ve - 90), down = oe - to;
    oe = to;
    return down;
}

// Positions per tile: the same bytes for every head_dim up to 128.
__host__ __device__ constexpr int tile_of(int dp) { return dp == 64 ? 64 : 32; }
// A split's tiles t0 .. t1 - 1 of a sequence, and how many splits it has where at most
// `cap` are wanted.  Tiles behind the prefix, whose masks are read and applied, count
// twice: they take 6 us where others take 3, and the splits that have them would end
// last (49 nodes on 4096 positions: at 36 us, the others at 28; a call 40.9 us, so
// 39.6).  Only the sequence's own lengths count, so that within one plan a result is
// the same whatever the bound and the batch.  us with 2 / 4 / 8 tiles at least, groups
// of 4 heads of 128: 60 nodes on 512 positions 25 / 26 / 34, 32 on 4096 38 / 34 / 36;
// groups of 7 heads of 64, 16 on 1000 21 / 21 / 31.
constexpr int kMinTiles = 4;
struct Range {
    int t0, t1, splits;
};
__device__ __forceinline__ Range split_range(int len, int end, int tk, int cap, int split) {
    const int tiles = (end + tk - 1) / tk, open = min(len / tk, tiles), units = 2 * tiles - open;
    const int each = max((units + cap - 1) / cap, kMinTiles);
    auto tile = [&](int unit) { return unit <= open ? unit : open + (unit - open) / 2; };
    return {tile(split * each), tile(min(units, (split + 1) * each)), (units + each - 1) / each};
}

// A block of NW waves takes 16 * RB * NW query rows of one KV head, a row being a
// (node, head of the group) pair i = node * G + head, 16 * RB of them a wave, and a
// range of the positions in tiles of TK.  Per tile the waves build the limbs of an
// NW-th of K and of V each, in LDS and in MFMA operand order, and then every wave
// multiplies all of them with its rows: so each f32 of the cache is read and split
// once a block.  Two buffers, one barrier a tile: while tile i is multiplied, tile
// i + 1 goes from registers to the other buffer and tile i + 2 is requested.  Where
// one block has a CU to itself (NW = 8) half of its waves multiply first and half
// build first, so that a SIMD's two waves want its matrix and its vector unit in turn.
//   Lane (g, c) = (lane / 16, lane % 16) has A[c][8g ..] and B[8g ..][c] of a
//   product of depth 32, and gets D[4g + r][c] in register r:
//   S^T = K Q^T: A = 16 positions, position c with the 8 dimensions 16 x + 4g ..
//     and 32 + 16 x + 4g .. of each 64, x = 0, 1 (so that the lanes read K rows in
//     whole 128-byte pieces); B = the wave's query rows, in registers;
//   O^T = V^T P^T: A's row c of block (q, j) is dimension 64 q + 4 c + j and its
//     depth 8g + i is position 4g + i (i < 4) or 16 + 4g + i - 4 of 32: the
//     positions whose scores the lane holds for row c, so P^T needs no exchange
//     and V rows are read in whole 256-byte pieces.
// What a wave builds has a scale of its own: of every 32 positions, K's 32 / NW from
// w * 32 / NW on, and V's of lane group g = w (NW = 4), or of half h and group g,
// w = 4 h + g (NW = 8).
//
// A tile with infinities, and one behind the prefix with NaN in V or with K or V too
// far apart for limbs in common scales, goes in f32, as do those after such a one
// behind the prefix: its scores come from f32 sums, its weights leave the MFMAs as 0,
// and then V is added in f32.  (Positions behind the prefix are few, and this is rare:
// 49 nodes on 4096 positions take 146 us with such a node and 44 without.)
//
// Bound by what a SIMD can issue: a wave has 96 MFMAs and 450 to 510 vector
// instructions (limbs, exponentials, maxima, sums; eight waves, four) a tile of 32
// positions of 128 and 32 rows, and the two overlap in part only: loops of MFMAs for
// 36.8 ns and vector instructions for 46 take 60.7 together on one SIMD.  8 KV heads
// of 128 in groups of 4: 49 nodes on 4096 positions 41 us, 64 on 32767 143 us (1.9 TB/s
// of K and V, 242 TFLOP/s of f32 products on three times that of f16 ones, of 1186 that
// a large product reaches); VALU sums in f32, one wave a row, took 1344 and 14693 us.
template <int DP, int RB, int NW>
__global__ __launch_bounds__(64 * NW, DP <= 128 || NW == 8 ? 2 : 1) void k_tree_attn(
    TreeAttn a, int cap, float *__restrict__ part, float *__restrict__ pml) {
    constexpr int NS = DP / 32, NB = DP / 64, TK = tile_of(DP), KT = TK / 32;
    constexpr int PW = 32 / NW, LX = 16 / PW;   // K positions a wave, operands of one side by side
    constexpr int KU = KT * NS / LX;            // K operands (8 values) a lane
    constexpr int VU = KT * NB / 2, VP = 16 / NW;   // V: columns of 4 a lane, positions of each
    // Operands read at a time.  (32 rows of 128 dimensions have all 256 registers: 3 to 5 spill.
    // With 1 of V the four-wave block spills none, and is no faster: 41.1 us both, 137 / 132.)
    constexpr int KG = RB == 1 ? 2 : 1, VG = RB == 1 ? 4 : 2;
    __shared__ f16x8 sk[2][KT * 2 * NS * 2 * 64];       // [32 positions][16][32 dims][limb][lane]
    __shared__ f16x8 sv[2][KT * NB * 4 * 2 * 64];       // [32 positions][64 dims][j][limb][lane]
    // The shares' exponents, K's and V's; V's + kBias again with kSlow where K or V is for f32.
    __shared__ int se[2][2][NW], sw[2][NW];
    // A share's largest and least exponent of V in the tiles behind the prefix so far.
    __shared__ int behind[2][2][NW];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, c = lane & 15, g = lane >> 4;
    const int G = a.hq / a.hkv, R = a.n * G, D = a.hd, words = (a.n + 31) / 32;
    const int split = blockIdx.y, kvh = blockIdx.x % a.hkv, b = blockIdx.z;
    // The row tile: the last one, which may be mostly empty, is another block's in every split,
    // or some dies would have nothing else (12 sequences, 147 rows 147 us instead of 137).
    const int rtiles = gridDim.x / a.hkv, rtile = ((int)blockIdx.x / a.hkv + split + b) % rtiles;
    const int w0 = (rtile * NW + wave) * 16 * RB;   // the wave's first row
    const int len = prefix_len(a.kv_lens, a.kv_len, b, a.max_seq), end = min(len + a.n, a.max_seq);
    const Range range = split_range(len, end, TK, cap, split);
    const int t0 = range.t0, t1 = range.t1;
    if (split > 0 && split >= range.splits) return;   // the merge skips this split
    const float *kb = a.k.p + b * a.k.sb + kvh * a.k.sh, *vb = a.v.p + b * a.v.sb + kvh * a.v.sh;

    // ---- this thread's part of a tile: operand (sub, s) of K position kpos, column (sub, q)
    // of V positions vpos ..
    auto kpos = [&](int ln) { return wave * PW + (ln & (PW - 1)); };
    auto kgrp = [](int ln) { return ln / PW & 3; };
    auto kop = [](int ln, int u) { return u * LX + ln / (4 * PW); };   // sub * NS + s
    auto vpos = [&](int ln) {
        return NW == 4 ? 16 * (ln & 1) + 4 * wave : 4 * wave + 2 * (ln & 1);
    };
    auto vcol = [](int ln) { return ln >> 1 & 15; };
    auto vsub = [](int ln) { return KT == 2 ? ln >> 5 : 0; };
    auto vq = [](int ln, int u) { return KT == 2 ? 0 : (ln >> 5) + 2 * u; };
    float kr[KU][8], vr[VU][VP][4];
    // Its addresses, in 16-byte units from the tile's first row.  Dimensions past head_dim
    // repeat others: the query limbs are zero there, and those outputs are not kept.
    const uint32_t ks4 = (uint32_t)(a.k.ss / 4), vs4 = (uint32_t)(a.v.ss / 4);
    uint32_t koff[KU], koff2[KU], voff[VU];
#pragma unroll
    for (int u = 0; u < KU; ++u) {
        const int s = kop(lane, u) % NS, d = 64 * (s >> 1);
        koff[u] = (32 * (kop(lane, u) / NS) + kpos(lane)) * ks4 + 4 * (s & 1) + kgrp(lane) +
                  (d < D ? d / 4 : 0);
        koff2[u] = d + 32 < D ? 8 : 0;
    }
#pragma unroll
    for (int u = 0; u < VU; ++u)
        voff[u] = (32 * vsub(lane) + vpos(lane)) * vs4 +
                  min(16 * vq(lane, u) + vcol(lane), D / 4 - 1);
    auto load_k = [&](int tile) {
        const float4 *kt = reinterpret_cast<const float4 *>(kb + (int64_t)tile * TK * a.k.ss);
        const int last = end - 1 - tile * TK;   // the last tile repeats the last position
        const bool whole = last >= TK - 1;
        const int ln = fresh_lane();
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            uint32_t at = (uint32_t)fresh((int)koff[u]);
            if (!whole) at -= max(32 * (kop(ln, u) / NS) + kpos(ln) - last, 0) * ks4;
            const float4 x = kt[at], y = kt[at + koff2[u]];
            kr[u][0] = x.x; kr[u][1] = x.y; kr[u][2] = x.z; kr[u][3] = x.w;
            kr[u][4] = y.x; kr[u][5] = y.y; kr[u][6] = y.z; kr[u][7] = y.w;
        }
    };
    auto load_v = [&](int tile) {
        const float4 *vt = reinterpret_cast<const float4 *>(vb + (int64_t)tile * TK * a.v.ss);
        const int last = end - 1 - tile * TK;
        const bool whole = last >= TK - 1;
        const int ln = fresh_lane();
#pragma unroll
        for (int u = 0; u < VU; ++u)
#pragma unroll
            for (int i = 0; i < VP; ++i) {
                uint32_t at = (uint32_t)fresh((int)voff[u]) + i * vs4;
                if (!whole) at -= max(32 * vsub(ln) + vpos(ln) + i - last, 0) * vs4;
                const float4 x = vt[at];
                vr[u][i][0] = x.x; vr[u][i][1] = x.y; vr[u][i][2] = x.z; vr[u][i][3] = x.w;
            }
    };
    // The tile's limbs to a buffer; the registers then take the next tile's values.
    auto store = [&](int tile, int buf) {
        const int ln = fresh_lane();
        const bool open = (tile + 1) * TK <= len;
        float km = 0.f, vm = 0.f, kn = 0.f, vn = 0.f;
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                max3_abs(km, kr[u][j], kr[u][j + 1]);
                max3_abs(kn, kr[u][j + 2], kr[u][j + 3]);
            }
#pragma unroll
        for (int u = 0; u < VU; ++u)
#pragma unroll
            for (int i = 0; i < VP; ++i) {
                max3_abs(vm, vr[u][i][0], vr[u][i][1]);
                max3_abs(vn, vr[u][i][2], vr[u][i][3]);
            }
        uint32_t kt = max(abs_bits(km), abs_bits(kn)), vt = max(abs_bits(vm), abs_bits(vn));
        bool slow = false;
        if (!open) {   // NaN in V too: a row that does not see its position must not get it
            uint32_t k_low = 0, v_low = 0;
#pragma unroll
            for (int u = 0; u < KU; ++u) low_bits(k_low, top_bits(kr[u]));
#pragma unroll
            for (int i = 0; i < VP; ++i) {
                uint32_t top = 0;
#pragma unroll
                for (int u = 0; u < VU; ++u) top = max(top, top_bits(vr[u][i]));
                vt = max(vt, top);
                low_bits(v_low, top);
            }
            wave_max_bits(kt, vt);
            wave_max_bits(k_low, v_low);
            slow = spread(exponent(kt), k_low) || spread(exponent(vt), v_low);
        } else {
            wave_max_bits(kt, vt);
        }
        slow |= kt >= kInf || vt >= kInf;
        if (__builtin_expect(vt >= kInf, 0)) {   // the largest finite one
            vt = 0;
#pragma unroll
            for (int u = 0; u < VU; ++u)
#pragma unroll
                for (int i = 0; i < 4 * VP; ++i) {
                    float &x = vr[u][i >> 2][i & 3];
                    x = abs_bits(x) < kInf ? x : 0.f;
                    vt = max(vt, abs_bits(x));
                }
            uint32_t v2 = vt;
            wave_max_bits(vt, v2);
        }
        const int ke = exponent(kt), ve = exponent(vt);
        int high = kNoV, low = -kNoV;
        if (!open) {
            if (tile > t0) {   // what those before it were, it is
                high = behind[buf ^ 1][0][wave];
                low = behind[buf ^ 1][1][wave];
                slow |= (tile * TK > len && sw[buf ^ 1][wave] >= kSlow) ||
                        ve - se[buf ^ 1][1][wave] > 20;
            }
            high = max(high, ve);
            low = min(low, ve == kLeast ? -kNoV : ve);
        }
        if (ln == 0) {
            behind[buf][0][wave] = high;
            behind[buf][1][wave] = low;
            se[buf][0][wave] = ke;
            se[buf][1][wave] = ve;
            sw[buf][wave] = ve + kBias + (slow ? kSlow : 0);
        }
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            const int sub = kop(ln, u) / NS, s = kop(ln, u) % NS, p = kpos(ln);
            f16x8 hi, lo;
            split_to_lds<8>(kr[u], pow2(kTop - ke), hi, lo);
            f16x8 *d = sk[buf] + (((sub * 2 + (p >> 4)) * NS + s) * 2) * 64 + 16 * kgrp(ln) + (p & 15);
            d[0] = hi;
            d[64] = lo;
        }
        if (tile + 1 < t1) load_k(tile + 1);
#pragma unroll
        for (int u = 0; u < VU; ++u) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float x[VP];
#pragma unroll
                for (int i = 0; i < VP; ++i) x[i] = vr[u][i][j];
                f16v<VP> hi, lo;
                split_to_lds<VP>(x, pow2(kTop - ve), hi, lo);
                const int p = vpos(ln);   // half p / 16, group p % 16 / 4, first of it p % 4
                f16v<VP> *d = reinterpret_cast<f16v<VP> *>(
                    reinterpret_cast<_Float16 *>(
                        sv[buf] + (((vsub(ln) * NB + vq(ln, u)) * 4 + j) * 2) * 64 +
                        16 * (p >> 2 & 3) + vcol(ln)) +
                    4 * (p >> 4) + (p & 3));
                d[0] = hi;
                d[64 * 8 / VP] = lo;
            }
        }
        if (tile + 1 < t1) load_v(tile + 1);
    };
    if (t0 < t1) {
        load_k(t0);
        load_v(t0);
    }

    const int32_t *mask = a.mask + b * a.mask_sb;
    // ---- the wave's query rows, row c of each block in this lane
    f16x8 qh[RB][NS], ql[RB][NS];
    int mrow[RB], qe[RB];
    bool live[RB];
    float m[RB], l[RB];
    f32x4 o[RB][NB][4];
    const bool busy = w0 < R;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int i = w0 + 16 * rb + c;
        query_row<NS>(a, b, kvh, i, g, qh[rb], ql[rb], qe[rb]);
        mrow[rb] = (i < R ? i : 0) / G * words;
        live[rb] = i < R && any_bit(mask + mrow[rb], words, a.n, g);
        m[rb] = -INFINITY;
        l[rb] = 0.f;
#pragma unroll
        for (int q = 0; q < NB; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[rb][q][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    int oe = 0, oe_top = kNoV;   // exponent of the outputs' scale; the largest V's so far
    const float f = fabsf(a.scale) * kLog2e;

    if (t0 < t1) {
        store(t0, 0);
        __syncthreads();
    }
    // Without the positions that the row does not see.
    auto mask_scores = [&](int rb, int p0, int g, float (&s)[8 * KT]) TB_INLINE {
#pragma unroll
        for (int sub = 0; sub < KT; ++sub) {
            const uint32_t see =
                live[rb] ? seen(mask + mrow[rb], words, p0 + 32 * sub, len, end) : 0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!(see >> position(j, g) & 1)) s[8 * sub + j] = -INFINITY;
        }
    };
    auto multiply = [&](int tile, int buf) {
        const int p0 = tile * TK;
        if (busy) {
            const bool open = p0 + TK <= len;   // every live row sees every position
            const int ln = fresh_lane(), g = ln >> 4;
            // ---- scores, in powers of two.  A group's operands are read while the
            // MFMAs of the one before run.
            float s8[RB][8 * KT];
            f32x4 acc[RB][KT][2];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int sub = 0; sub < KT; ++sub)
                    acc[rb][sub][0] = acc[rb][sub][1] = f32x4{0.f, 0.f, 0.f, 0.f};
            f16x8 kf[2][KG][2][2];   // [group parity][32 dimensions][16 positions][limb]
            auto read_k = [&](int grp) {
#pragma unroll
                for (int x = 0; x < KG; ++x)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const int sub = grp / (NS / KG), s = grp % (NS / KG) * KG + x;
                            kf[grp & 1][x][h][y] =
                                sk[buf][(((sub * 2 + h) * NS + s) * 2 + y) * 64 + ln];
                        }
            };
            read_k(0);
#pragma unroll
            for (int grp = 0; grp < KT * NS / KG; ++grp) {
                if (grp + 1 < KT * NS / KG) read_k(grp + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int x = 0; x < KG; ++x)
#pragma unroll
                    for (int y = 0; y < 3; ++y)
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int sub = grp / (NS / KG), s = grp % (NS / KG) * KG + x;
                                f32x4 &d = acc[rb][sub][h];
                                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                    kf[grp & 1][x][h][y == 0], y == 1 ? ql[rb][s] : qh[rb][s], d,
                                    0, 0, 0);
                            }
                __builtin_amdgcn_sched_barrier(0);
            }
            // The first operands of the outputs, read during the softmax.
            f16x8 vf[2][VG][2];   // [group parity][block of 16 dimensions][limb]
            auto read_v = [&](int grp) {
#pragma unroll
                for (int j = 0; j < VG; ++j)
#pragma unroll
                    for (int y = 0; y < 2; ++y)
                        vf[grp & 1][j][y] = sv[buf][((grp * VG + j) * 2 + y) * 64 + ln];
            };
            read_v(0);
            const int ke[2] = {se[buf][0][4 * g / PW], se[buf][0][(16 + 4 * g) / PW]};
            const int ve[2] = {se[buf][1][g], se[buf][1][NW == 4 ? g : 4 + g]};
            int word = sw[buf][0];
#pragma unroll
            for (int w = 1; w < NW; ++w) word = max(word, sw[buf][w]);
            word = __builtin_amdgcn_readfirstlane(word);
            bool slow = word >= kSlow;
            int vtop = se[buf][1][0];
#pragma unroll
            for (int w = 1; w < NW; ++w) vtop = max(vtop, se[buf][1][w]);
            vtop = __builtin_amdgcn_readfirstlane(vtop);
            if (NW == 4 || !open) {   // (a branch has four waves of 32 rows spill 160 registers)
                int high = behind[buf][0][0], low = behind[buf][1][0];
#pragma unroll
                for (int w = 1; w < NW; ++w) {
                    high = max(high, behind[buf][0][w]);
                    low = min(low, behind[buf][1][w]);
                }
                slow |= __builtin_amdgcn_readfirstlane(high - low) > 8;
            }
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const float sx[2] = {ldexpf(f, qe[rb] + ke[0] - 2 * kTop),
                                     ldexpf(f, qe[rb] + ke[1] - 2 * kTop)};
#pragma unroll
                for (int j = 0; j < 8 * KT; ++j)
                    s8[rb][j] = acc[rb][j >> 3][j >> 2 & 1][j & 3] * sx[j >> 2 & 1];
            }
            if (__builtin_expect(slow, 0)) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
                    scores_in_f32<8 * KT>(a, b, kvh, min(w0 + 16 * rb + c, R - 1), p0, end, g,
                                          s8[rb]);
            }
            // ---- running maxima
            float was[RB];
            bool moved = false, below = false;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                if (!open) mask_scores(rb, p0, g, s8[rb]);
                float t = s8[rb][0];
#pragma unroll
                for (int j = 1; j < 8 * KT; ++j) t = fmaxf(t, s8[rb][j]);
                was[rb] = m[rb];
                t = max_over_groups(t);
                below |= t < m[rb] - kDrop;
                m[rb] = t > m[rb] + kLag ? t : m[rb];
                moved |= m[rb] != was[rb];
            }
            if (__builtin_expect(__any(below), 0)) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    float t = s8[rb][0];
#pragma unroll
                    for (int j = 1; j < 8 * KT; ++j) t = fmaxf(t, s8[rb][j]);
                    m[rb] = drop(m[rb], max_over_groups(t), sum_over_groups(l[rb]), oe, oe_top);
                    moved |= m[rb] != was[rb];
                }
            }
            const int down = slow ? raise(vtop, oe, oe_top) : rescale(vtop, oe, oe_top);
            if (__any(moved) || down != 0) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    const float alpha =
                        was[rb] == m[rb] ? 1.f : __builtin_amdgcn_exp2f(was[rb] - m[rb]);
                    l[rb] *= alpha;
                    const float x = ldexpf(alpha, min(down, 120));
#pragma unroll
                    for (int q = 0; q < NB; ++q)
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[rb][q][j] *= x;
                }
            }
            // ---- weights, in the scale of the positions' V: 2^pe w
            f16x8 ph[RB][KT], pl[RB][KT];
            const int pe[2] = {max(kWeight + ve[0] - oe, kWeightLow),
                               max(kWeight + ve[1] - oe, kWeightLow)};
            const float back[2] = {pow2(-pe[0] - kLow), pow2(-pe[1] - kLow)};
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                float top = m[rb] == -INFINITY ? 0.f : m[rb];   // nothing seen: weights 0
                if (slow) top = INFINITY;   // V in f32 below: weights 0 here
                const float base[2] = {(float)(pe[0] + kLow) - top, (float)(pe[1] + kLow) - top};
#pragma unroll
                for (int sub = 0; sub < KT; ++sub) {
                    float p8[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        p8[j] = __builtin_amdgcn_exp2f(s8[rb][8 * sub + j] + base[j >> 2]);
                        l[rb] = fmaf(p8[j], back[j >> 2], l[rb]);
                    }
                    split_weights(p8, ph[rb][sub], pl[rb][sub]);
                }
            }
            // ---- outputs
#pragma unroll
            for (int grp = 0; grp < KT * NB * 4 / VG; ++grp) {
                if (grp + 1 < KT * NB * 4 / VG) read_v(grp + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int y = 0; y < 3; ++y)
#pragma unroll
                    for (int j = 0; j < VG; ++j)
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) {
                            const int at = grp * VG + j;   // [32 positions][64 dims][j]
                            f32x4 &d = o[rb][at / 4 % NB][at % 4];
                            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                y == 1 ? low(vf[grp & 1][j][0]) : vf[grp & 1][j][y == 0],
                                y == 1 ? pl[rb][at / (4 * NB)] : ph[rb][at / (4 * NB)], d, 0, 0, 0);
                        }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (__builtin_expect(slow, 0)) {   // weights anew: nothing waits for this in registers
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    float p[8 * KT];
                    scores_in_f32<8 * KT>(a, b, kvh, min(w0 + 16 * rb + c, R - 1), p0, end, g, p);
                    if (!open) mask_scores(rb, p0, g, p);
                    const float base = (float)kWeight - (m[rb] == -INFINITY ? 0.f : m[rb]);
#pragma unroll
                    for (int j = 0; j < 8 * KT; ++j) {
                        p[j] = __builtin_amdgcn_exp2f(p[j] + base);
                        l[rb] = fmaf(p[j], pow2(-kWeight), l[rb]);
                    }
                    add_in_f32<NB, 8 * KT>(a, vb, p0, end, g, c, p, pow2(kTop - oe), o[rb]);
                }
            }
        }
    };
    if constexpr (NW == 4) {
        for (int tile = t0; tile < t1; ++tile) {
            const int buf = (tile - t0) & 1;
            multiply(tile, buf);
            if (tile + 1 < t1) store(tile + 1, buf ^ 1);
            __syncthreads();
        }
    } else {
        for (int step = 0; step < 2 * (t1 - t0); ++step) {
            const int tile = t0 + (step >> 1), buf = step >> 1 & 1;
            if ((step ^ wave >> 2) & 1) {
                if (tile + 1 < t1) store(tile + 1, buf ^ 1);
            } else {
                multiply(tile, buf);
            }
            if (step & 1) __syncthreads();
        }
    }
    if (!busy) return;

    // ---- results: lane (g, c) holds dimensions 64 q + 16 g .. + 15 of row c
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int i = w0 + 16 * rb + c;
        const float sum = live[rb] ? sum_over_groups(l[rb]) : 0.f;
        if (i >= R) continue;
        const size_t at = (((size_t)b * a.hkv + kvh) * gridDim.y + split) * R + i;
        float *to = part ? part + at * D   // normalised, so that the largest V do not overflow
                         : a.out + (((size_t)b * a.n + i / G) * a.hq + kvh * G + i % G) * D;
        const float x = sum == 0.f ? 0.f : 1.0f / sum;
        if (part && g == 0) {
            pml[2 * at] = reference(live[rb], m[rb], sum);
            pml[2 * at + 1] = sum;
        }
#pragma unroll
        for (int q = 0; q < NB; ++q)
            if (64 * q + 16 * g < D)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float4 y;
                    y.x = ldexpf(o[rb][q][0][r] * x, oe - kTop - kWeight);
                    y.y = ldexpf(o[rb][q][1][r] * x, oe - kTop - kWeight);
                    y.z = ldexpf(o[rb][q][2][r] * x, oe - kTop - kWeight);
                    y.w = ldexpf(o[rb][q][3][r] * x, oe - kTop - kWeight);
                    if (!live[rb]) y = make_float4(0.f, 0.f, 0.f, 0.f);
                    reinterpret_cast<float4 *>(to + 64 * q + 16 * g)[r] = y;
                }
    }
}

// The same for few rows (up to 32 of a KV head), where K and V have to stream: a
// block's waves take tiles of 32 positions in turn, each with the block's 16 * RB
// rows and maxima, sums and outputs of its own, and meet in LDS once at the end.
// K and V go from memory to MFMA operands in the wave's own registers, and nothing
// in the loop waits for another wave.  The next tile's K is requested when this
// one's scores are on their way, its V when this one's limbs are built.  Every K and
// V row is read once: non-temporal loads (8 rows of each KV head over 32775 positions of
// 8 heads of 128: 62 us and 4.3 TB/s, 67 with ordinary ones).  Bound by the loads that
// its waves keep on their way, and on short caches by the two launches: 8 nodes on
// 4096 positions take 27 us, 1 node 21.
template <int DP, int RB>
__global__ __launch_bounds__(256, 1) void k_tree_attn_few(TreeAttn a, int cap,
                                                          float *__restrict__ part,
                                                          float *__restrict__ pml) {
    constexpr int NS = DP / 32, NB = DP / 64, ROWS = 16 * RB, TK = 32;
    __shared__ __attribute__((aligned(16))) float lo[ROWS][DP + 4];
    __shared__ float lm[4][ROWS], ls[4][ROWS];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, c = lane & 15, g = lane >> 4;
    const int G = a.hq / a.hkv, R = a.n * G, D = a.hd, words = (a.n + 31) / 32;
    const int split = blockIdx.y, kvh = blockIdx.x, b = blockIdx.z;
    const int len = prefix_len(a.kv_lens, a.kv_len, b, a.max_seq), end = min(len + a.n, a.max_seq);
    const Range range = split_range(len, end, TK, cap, split);
    const int t0 = range.t0, t1 = range.t1;
    if (split > 0 && split >= range.splits) return;   // the merge skips this split
    const float *kb = a.k.p + b * a.k.sb + kvh * a.k.sh, *vb = a.v.p + b * a.v.sb + kvh * a.v.sh;
    const int32_t *mask = a.mask + b * a.mask_sb;

    float kr[2][NS][8], vr[8][NB][4];
    auto load_k = [&](int tile) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float *r = kb + min(tile * TK + 16 * h + c, end - 1) * a.k.ss + 4 * g;
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const int d = 64 * (s >> 1);
                const float4 x = gemv::load_nt_f4(r + 16 * (s & 1) + (d < D ? d : 0));
                const float4 y = gemv::load_nt_f4(r + 16 * (s & 1) + (d + 32 < D ? d + 32 : 0));
                float *k = kr[h][s];
                k[0] = x.x; k[1] = x.y; k[2] = x.z; k[3] = x.w;
                k[4] = y.x; k[5] = y.y; k[6] = y.z; k[7] = y.w;
            }
        }
    };
    auto load_v = [&](int tile) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float *r = vb + min(tile * TK + position(i, g), end - 1) * a.v.ss;
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                const float4 x = gemv::load_nt_f4(r + min(64 * q + 4 * c, D - 4));
                vr[i][q][0] = x.x; vr[i][q][1] = x.y; vr[i][q][2] = x.z; vr[i][q][3] = x.w;
            }
        }
    };
    const int first = t0 + wave;
    if (first < t1) {
        load_k(first);
        load_v(first);
    }
    f16x8 qh[RB][NS], ql[RB][NS];
    int mrow[RB], qe[RB];
    bool live[RB];
    float m[RB], l[RB];
    f32x4 o[RB][NB][4];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int i = 16 * rb + c;
        query_row<NS>(a, b, kvh, i, g, qh[rb], ql[rb], qe[rb]);
        mrow[rb] = (i < R ? i : 0) / G * words;
        live[rb] = i < R && any_bit(mask + mrow[rb], words, a.n, g);
        m[rb] = -INFINITY;
        l[rb] = 0.f;
#pragma unroll
        for (int q = 0; q < NB; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[rb][q][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    int oe = 0, oe_top = kNoV;   // exponent of the outputs' scale; the largest V's so far
    // The largest V's behind the prefix so far; the first tile there whose V went in f32.
    int behind = kNoV, f32_since = t1;
    const float f = fabsf(a.scale) * kLog2e;

    for (int tile = first; tile < t1; tile += 4) {
        const int p0 = tile * TK;
        const bool open = p0 + TK <= len;   // every live row sees every position
        // ---- the tile's scales
        float km = 0.f, kn = 0.f, vm = 0.f, vn = 0.f;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                max3_abs(km, kr[0][s][j], kr[0][s][j + 1]);
                max3_abs(kn, kr[1][s][j], kr[1][s][j + 1]);
            }
        uint32_t kt = max(abs_bits(km), abs_bits(kn)), k_low = 0;
        if (!open) {
            low_bits(k_low, abs_bits(km));
            low_bits(k_low, abs_bits(kn));
        }
        wave_max_bits(kt, k_low);
        const int ke = exponent(kt);
        const bool slow_k = kt >= kInf || spread(ke, k_low);
        // ---- scores, in powers of two
        f32x4 acc[RB][2];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) acc[rb][0] = acc[rb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            f16x8 kh[2], kl[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) split8(kr[h][s], pow2(kTop - ke), kh[h], kl[h]);
#pragma unroll
            for (int x = 0; x < 3; ++x)
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        acc[rb][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            x == 0 ? kl[h] : kh[h], x == 1 ? ql[rb][s] : qh[rb][s], acc[rb][h], 0,
                            0, 0);
        }
        if (tile + 4 < t1) load_k(tile + 4);
        float s8[RB][8];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const float sx = ldexpf(f, qe[rb] + ke - 2 * kTop);
#pragma unroll
            for (int j = 0; j < 8; ++j) s8[rb][j] = acc[rb][j >> 2][j & 3] * sx;
        }
        if (__builtin_expect(slow_k, 0)) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
                scores_in_f32<8>(a, b, kvh, min(16 * rb + c, R - 1), p0, end, g, s8[rb]);
        }
        // ---- running maxima
        float was[RB];
        bool moved = false, below = false;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            if (!open) {
                const uint32_t see = live[rb] ? seen(mask + mrow[rb], words, p0, len, end) : 0;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!(see >> position(j, g) & 1)) s8[rb][j] = -INFINITY;
            }
            float t = s8[rb][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) t = fmaxf(t, s8[rb][j]);
            was[rb] = m[rb];
            t = max_over_groups(t);
            below |= t < m[rb] - kDrop;
            m[rb] = t > m[rb] + kLag ? t : m[rb];
            moved |= m[rb] != was[rb];
        }
        if (__builtin_expect(__any(below), 0)) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                float t = s8[rb][0];
#pragma unroll
                for (int j = 1; j < 8; ++j) t = fmaxf(t, s8[rb][j]);
                m[rb] = drop(m[rb], max_over_groups(t), sum_over_groups(l[rb]), oe, oe_top);
                moved |= m[rb] != was[rb];
            }
        }
        // ---- V's scale and the outputs'
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                max3_abs(vm, vr[i][q][0], vr[i][q][1]);
                max3_abs(vn, vr[i][q][2], vr[i][q][3]);
            }
        uint32_t vt = max(abs_bits(vm), abs_bits(vn)), v_low = 0;
        if (!open) {   // NaN too: a row that does not see its position must not get it
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t top = 0;
#pragma unroll
                for (int q = 0; q < NB; ++q) top = max(top, top_bits(vr[i][q]));
                vt = max(vt, top);
                low_bits(v_low, top);
            }
        }
        wave_max_bits(vt, v_low);
        bool slow_v = vt >= kInf;
        if (__builtin_expect(slow_v, 0)) {   // the largest finite one
            vt = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int q = 0; q < NB; ++q)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t x = abs_bits(vr[i][q][j]);
                        vt = max(vt, x < kInf ? x : 0);
                    }
            uint32_t v2 = vt;
            wave_max_bits(vt, v2);
        }
        const int ve = exponent(vt);
        if (!open) {
            behind = max(behind, ve);
            slow_v |= f32_since < tile || spread(behind, v_low) || (oe_top != kNoV && ve - oe > 20);
            if (slow_v) f32_since = min(f32_since, tile);
        }
        const int down = slow_v ? raise(ve, oe, oe_top) : rescale(ve, oe, oe_top);
        if (__any(moved) || down != 0) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const float alpha = was[rb] == m[rb] ? 1.f : __builtin_amdgcn_exp2f(was[rb] - m[rb]);
                l[rb] *= alpha;
                const float x = ldexpf(alpha, min(down, 120));
#pragma unroll
                for (int q = 0; q < NB; ++q)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[rb][q][j] *= x;
            }
        }
        // ---- weights 2^(kWeight + kLow) w, their sums of 2^kWeight w
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const float base = (float)(kWeight + kLow) - (m[rb] == -INFINITY ? 0.f : m[rb]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                s8[rb][j] = __builtin_amdgcn_exp2f(s8[rb][j] + base);
                l[rb] = fmaf(s8[rb][j], 1.f / (1 << kLow), l[rb]);
            }
        }
        // ---- outputs; V takes the outputs' scale
        if (__builtin_expect(slow_v, 0)) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
                add_in_f32<NB, 8>(a, vb, p0, end, g, c, s8[rb], pow2(kTop - kLow - oe), o[rb]);
            if (tile + 4 < t1) load_v(tile + 4);
            continue;
        }
        f16x8 ph[RB], pl[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) split_weights(s8[rb], ph[rb], pl[rb]);
#pragma unroll
        for (int q = 0; q < NB; ++q) {
            f16x8 vh[4], vl[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x[8] = {vr[0][q][j], vr[1][q][j], vr[2][q][j], vr[3][q][j],
                                    vr[4][q][j], vr[5][q][j], vr[6][q][j], vr[7][q][j]};
                split8(x, pow2(kTop - oe), vh[j], vl[j]);
            }
#pragma unroll
            for (int x = 0; x < 3; ++x)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb)
                        o[rb][q][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            x == 0 ? vl[j] : x == 1 ? low(vh[j]) : vh[j],
                            x == 1 ? pl[rb] : ph[rb], o[rb][q][j], 0, 0, 0);
        }
        if (tile + 4 < t1) load_v(tile + 4);
    }

    // ---- the four waves' outputs, normalised, in the shares of their sums, in wave order
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const float sum = sum_over_groups(l[rb]);
        l[rb] = live[rb] ? sum : 0.f;
        m[rb] = reference(live[rb], m[rb], sum);
        if (g == 0) {
            lm[wave][16 * rb + c] = m[rb];
            ls[wave][16 * rb + c] = l[rb];
        }
    }
    __syncthreads();
    // Row r's maximum, sum and share of wave w.
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
                    for (int i = 0; i < 4; ++i) {
                        float4 *d = reinterpret_cast<float4 *>(&lo[r][64 * q + 16 * g]) + i;
                        float4 y = w ? *d : make_float4(0.f, 0.f, 0.f, 0.f);
                        if (x != 0.f) {
                            y.x += ldexpf(o[rb][q][0][i] * x, oe - kTop);
                            y.y += ldexpf(o[rb][q][1][i] * x, oe - kTop);
                            y.z += ldexpf(o[rb][q][2][i] * x, oe - kTop);
                            y.w += ldexpf(o[rb][q][3][i] * x, oe - kTop);
                        }
                        *d = y;
                    }
            }
        }
        __syncthreads();
    }
    const int cols = D / 4;
    for (int x = t; x < ROWS * cols; x += 256) {
        const int r = x / cols, d = x % cols;
        if (r >= R) break;
        const float4 y = *reinterpret_cast<const float4 *>(&lo[r][4 * d]);
        if (part) {
            const size_t at = (((size_t)b * a.hkv + kvh) * gridDim.y + split) * R + r;
            reinterpret_cast<float4 *>(part + at * D)[d] = y;
            if (d == 0) {
                shares(r, 0, top, sum);
                pml[2 * at] = top;
                pml[2 * at + 1] = sum;
            }
        } else {
            float *out = a.out + (((size_t)b * a.n + r / G) * a.hq + kvh * G + r % G) * D;
            reinterpret_cast<float4 *>(out)[d] = y;
        }
    }
}

// The splits' outputs, normalised, in the shares of their sums, a block per row.  Each
// wave works out every split's share (lane s: splits s and s + 64); the columns are taken by
// 256 / LC groups of LC lanes, group i with the splits i, i + 256 / LC, ...  The first
// of those are requested before the weights are known: every split's place in the
// scratch can be read, and what was not written has weight 0.  Bound by the launch and
// the way of those reads: 7.1 us for 1568 rows of 27 splits, 8.6 for 2048 of 32.
template <int LC>
__global__ __launch_bounds__(256) void k_tree_merge(TreeAttn a, int tk, int cap, int nsplit,
                                                    const float *__restrict__ part,
                                                    const float *__restrict__ pml) {
    constexpr int NG = 256 / LC, AHEAD = 8;
    __shared__ float w[4][kMaxSplits];
    __shared__ float4 col[4][LC];
    const int G = a.hq / a.hkv, R = a.n * G, cols = a.hd / 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    const size_t at = ((size_t)b * a.hkv + kvh) * nsplit * R + i;
    const int d = min((int)threadIdx.x % LC, cols - 1), grp = threadIdx.x / LC;
    const float4 *src = reinterpret_cast<const float4 *>(part + at * a.hd) + d;
    const size_t step = (size_t)R * cols;
    float4 z[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) z[k] = src[min(grp + NG * k, nsplit - 1) * step];
    float m[2], l[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const float *p = pml + 2 * (at + (size_t)min(lane + 64 * x, nsplit - 1) * R);
        m[x] = p[0];
        l[x] = p[1];
    }
    const int len = prefix_len(a.kv_lens, a.kv_len, b, a.max_seq), end = min(len + a.n, a.max_seq);
    const int used = split_range(len, end, tk, cap, 0).splits;
#pragma unroll
    for (int x = 0; x < 2; ++x)
        if (lane + 64 * x >= used) m[x] = -INFINITY;
    float top = fmaxf(m[0], m[1]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, gemv::shfl_xor_u(top, o));
    float sum = 0.f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        m[x] = m[x] == -INFINITY ? 0.f : l[x] * __builtin_amdgcn_exp2f(m[x] - top);
        sum += m[x];
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) sum += gemv::shfl_xor_u(sum, o);
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
    for (int x = 0; x < 2; ++x) w[wave][lane + 64 * x] = m[x] * inv;
    wave_fence();
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](int s, const float4 &v) {
        const float x = w[wave][s];
        if (x != 0.f) {   // a split that sees nothing of the row counts for nothing
            y.x = fmaf(v.x, x, y.x);
            y.y = fmaf(v.y, x, y.y);
            y.z = fmaf(v.z, x, y.z);
            y.w = fmaf(v.w, x, y.w);
        }
    };
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
        if (grp + NG * k < used) add(grp + NG * k, z[k]);
    for (int s = grp + NG * AHEAD; s < used; s += NG) add(s, src[s * step]);
#pragma unroll
    for (int o = LC; o < 64; o <<= 1) {
        y.x += gemv::shfl_xor_u(y.x, o);
        y.y += gemv::shfl_xor_u(y.y, o);
        y.z += gemv::shfl_xor_u(y.z, o);
        y.w += gemv::shfl_xor_u(y.w, o);
    }
    if (lane < LC) col[wave][lane] = y;
    __syncthreads();
    if ((int)threadIdx.x >= cols) return;
    const float4 y0 = col[0][d], y1 = col[1][d], y2 = col[2][d], y3 = col[3][d];
    float *out = a.out + (((size_t)b * a.n + i / G) * a.hq + kvh * G + i % G) * a.hd;
    reinterpret_cast<float4 *>(out)[d] =
        make_float4((y0.x + y1.x) + (y2.x + y3.x), (y0.y + y1.y) + (y2.y + y3.y),
                    (y0.z + y1.z) + (y2.z + y3.z), (y0.w + y1.w) + (y2.w + y3.w));
}

struct Plan {
    bool few;
    int dp, rb, nw, tk, rtiles, cap, nsplit;
};

Plan plan(int batch, int n, int hq, int hkv, int hd, int max_len, bool ragged) {
    Plan p;
    p.dp = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    const int R = n * (hq / hkv);
    p.few = R <= 32 && p.dp <= 128;
    p.rb = p.few ? (R <= 16 ? 1 : 2) : R <= 64 || p.dp == 256 ? 1 : 2;
    p.tk = p.few ? 32 : tile_of(p.dp);
    const int tiles = (max_len + p.tk - 1) / p.tk;
    // Eight waves build a tile's limbs for 256 rows, half as much a row, where that leaves
    // each of 256 blocks 16 tiles and few of the rows empty.  us with four / eight, 8 heads of
    // 128 and groups of 4: 64 nodes on 32767 positions 180 / 164, 60 on 16384 94 / 92, on
    // 4096 45.4 / 45.9, on 1024 28 / 33; groups of 7, 12 sequences of 21 nodes (147 rows) on
    // up to 6000 142 / 147.
    p.nw = p.rb == 2 && (R + 63) / 64 % 4 == 0 && (int64_t)tiles * hkv * batch >= 16 * 256 ? 8 : 4;
    const int rows = 16 * p.rb * p.nw;
    p.rtiles = p.few ? 1 : (R + rows - 1) / rows;
    // As many blocks as run at once: two per CU, or one where registers or LDS allow one
    // (few rows, eight waves, head_dim past 128).  us at half as many / this / half as many
    // again, 8 heads of 128: 4096 + 49 nodes 41.7 / 43.4 / 51.5, 32767 + 64 198 / 178 / 201, 8
    // sequences of up to 6000 + 16 100 / 73 / 78; head_dim 256, 8192 + 16: - / 37.1 / 43.9.
    const int64_t want = (p.few || p.nw == 8 || p.dp == 256 ? 256 : 512) /
                         ((int64_t)p.rtiles * hkv * batch);
    p.cap = (int)std::max<int64_t>(1, std::min<int64_t>(want, kMaxSplits));
    // Twice as many for sequences of different lengths where the longest's splits would still
    // have 16 tiles: the call ends with them.  us without / with: 12 sequences of up to 6000
    // positions, 147 rows (38 tiles) 148 / 136, 28 rows of up to 3000 (47) 72 / 70; 8 of up to
    // 6000, 64 rows (23) 76 / 78, 4 of them, 128 rows (12) 61 / 74; equal lengths gain nothing
    // (12 of 6123, 147 rows 174 / 202) and are better given as a number.
    if (ragged && batch > 1 && tiles >= 32 * p.cap) p.cap = std::min(2 * p.cap, kMaxSplits);
    const int units = tiles + (n + p.tk - 1) / p.tk + 1;   // of a sequence at most (split_range)
    if (tiles <= kMinTiles) p.cap = 1;
    p.nsplit = std::max(1, std::min(p.cap, (units + kMinTiles - 1) / kMinTiles));
    return p;
}

}  // namespace

size_t tree_attention_scratch(int batch, int n, int hq, int hkv, int hd, int max_len) {
    const int ns = plan(batch, n, hq, hkv, hd, max_len, true).nsplit;   // the more of the two
    return ns > 1 ? (size_t)batch * hq * n * ns * (hd + 2) * sizeof(float) : 0;
}

int launch_tree_attention(const TreeAttn &a, int max_len, float *scratch, hipStream_t s) {
    const Plan p = plan(a.batch, a.n, a.hq, a.hkv, a.hd, max_len, a.kv_lens != nullptr);
    float *part = p.nsplit > 1 ? scratch : nullptr;
    float *pml = part ? part + (size_t)a.batch * a.hq * a.n * p.nsplit * a.hd : nullptr;
    // Heads first: the row tiles of a KV head, which read the same K and V, on one of the
    // eight dies (block i goes to die i % 8), and the splits that a sequence has not on all of
    // them.  Splits first, 24 nodes on 4096 positions of 8 heads take 31.7 us instead of 28.3.
    const dim3 grid(a.hkv * p.rtiles, p.nsplit, a.batch);
#define TB_TF(DP, RB)                                                                        \
    if (p.few && p.dp == DP && p.rb == RB)                                                   \
    hipLaunchKernelGGL((k_tree_attn_few<DP, RB>), grid, dim3(256), 0, s, a, p.cap, part, pml)
#define TB_TA(DP, RB, NW)                                                                    \
    if (!p.few && p.dp == DP && p.rb == RB && p.nw == NW)                                    \
    hipLaunchKernelGGL((k_tree_attn<DP, RB, NW>), grid, dim3(64 * NW), 0, s, a, p.cap, part, pml)
    TB_TF(64, 1);
    TB_TF(64, 2);
    TB_TF(128, 1);
    TB_TF(128, 2);
    TB_TA(64, 1, 4);
    TB_TA(64, 2, 4);
    TB_TA(64, 2, 8);
    TB_TA(128, 1, 4);
    TB_TA(128, 2, 4);
    TB_TA(128, 2, 8);
    TB_TA(256, 1, 4);
#undef TB_TA
#undef TB_TF
    TB_LAUNCHED();
    if (part) {
        const int R = a.n * (a.hq / a.hkv);
        const dim3 rows(R, a.hkv, a.batch);
        if (a.hd <= 32)
            hipLaunchKernelGGL(k_tree_merge<8>, rows, dim3(256), 0, s, a, p.tk, p.cap,
                               p.nsplit, part, pml);
        else if (a.hd <= 64)
            hipLaunchKernelGGL(k_tree_merge<16>, rows, dim3(256), 0, s, a, p.tk, p.cap,
                               p.nsplit, part, pml);
        else if (a.hd <= 128)
            hipLaunchKernelGGL(k_tree_merge<32>, rows, dim3(256), 0, s, a, p.tk, p.cap,
                               p.nsplit, part, pml);
        else
            hipLaunchKernelGGL(k_tree_merge<64>, rows, dim3(256), 0, s, a, p.tk, p.cap,
                               p.nsplit, part, pml);
        TB_LAUNCHED();
    }
    return TB_OK;
}

}  // namespace tb
