// Norms of the query and key heads and their position rotation in one pass; in a
// decode step the key and value rows go straight to their caches.
//
//   y = x w / sqrt(mean(x^2) + eps) over a head (y = x without weights)
//   (a, b) -> c (a cos t - b sin t, b cos t + a sin t),  t = position * inv_freq[i]
//
// for the pair i of the head's first `rotary` dimensions: (i, i + rotary / 2), or
// (2i, 2i + 1) interleaved; the other dimensions stay y.  c is the attention
// factor of scaled positions.
#include <math.h>

#include <algorithm>

#include "rope.hpp"
#include "tb_common.hpp"

namespace tb {

namespace {

// cos t and sin t times c, t = turns whole turns.  In 64 bits: a position of 10^6 times
// a frequency leaves 1e-10 of a turn, and the MI355X issues an f64 multiply-add as
// often as an f32 one.  Octants by quarter turns, then the Taylor sums on +-pi/4
// (2e-9 past x^9 of the sine, 1e-10 past x^10 of the cosine).
__device__ __forceinline__ void turn(double turns, double c, float &co, float &si) {
    const double f = turns - rint(turns), q = rint(4.0 * f);
    const double x = (f - 0.25 * q) * 6.283185307179586477, z = x * x;
    const double s =
        x * fma(z, fma(z, fma(z, fma(z, 1.0 / 362880, -1.0 / 5040), 1.0 / 120), -1.0 / 6), 1.0);
    const double k = fma(
        z, fma(z, fma(z, fma(z, fma(z, -1.0 / 3628800, 1.0 / 40320), -1.0 / 720), 1.0 / 24), -0.5),
        1.0);
    const int n = (int)q & 3;
    const double a = n & 1 ? s : k, b = n & 1 ? k : s;
    co = (float)(n == 1 || n == 2 ? -c * a : c * a);
    si = (float)(n >= 2 ? -c * b : c * b);
}

// The sum over the L lanes of a head.
template <int L>
__device__ __forceinline__ double head_sum(double v) {
#pragma unroll
    for (int o = 1; o < L; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

template <int W>
struct Piece {
    float a[W], b[W];   // the two pieces of W dimensions that a unit has
};

// A group of L lanes takes a token's heads h0 .. h0 + per - 1 (queries, then keys, then
// values), a lane NU units of 2 W dimensions of each: W pairs of the rotation, whose
// angles it works out once for all of them (180 instructions in 64 bits, against 60 a head:
// 4096 tokens of 40 heads take 68, 45, 36 and 42 us with 1, 2, 4 and 8 heads a group), or 2 W
// dimensions behind it.  W = 4: 16-byte loads, and both pieces of a pair of the half layout in
// one lane; W = 1 where sizes, strides or addresses do not allow it, bound by its 4-byte loads: 40
// heads of 80 that turn in 20 dimensions, 4096 tokens in cache, 54 us; all 80 turning, W = 4, 27.
//
// Bound by the heads' bytes, on few tokens by the launch: 4096 tokens of 32 + 8 heads of 128,
// 168 MB, take 37 us a call (4.5 TB/s, a large copy 4.9; the kernel 32 where part of its input
// is in cache); four tokens 5.2.
template <int L, int NU, int W, bool INTERLEAVED>
__global__ __launch_bounds__(256) void k_norm_rope(RopeParams p, int per, int parts) {
    const int lane = threadIdx.x % L;
    const uint32_t item = blockIdx.x * (256 / L) + threadIdx.x / L;
    const bool on = item < (uint32_t)p.n * parts;   // all lanes take part in the sums
    const int token = on ? (int)(item / parts) : 0;
    const int D = p.hd, heads = p.hq + (p.append ? 2 : 1) * p.hkv;
    const int h0 = (int)(item - token * parts) * per, h1 = on ? min(heads, h0 + per) : 0;
    const int units = D / (2 * W), turning = p.rotary / (2 * W);

    // ---- the units' places and angles
    int ia[NU], ib[NU];
    bool has[NU];
    float co[NU][W], si[NU][W];
    Piece<W> qw[NU], kw[NU];
    const double pos = (double)p.positions[token];
#pragma unroll
    for (int n = 0; n < NU; ++n) {
        const int u = lane + n * L;
        has[n] = u < units;
        const bool turns = u < turning;
        if (INTERLEAVED || !turns) {
            ia[n] = 2 * W * u;
            ib[n] = 2 * W * u + W;
        } else {
            ia[n] = W * u;
            ib[n] = p.rotary / 2 + W * u;
        }
#pragma unroll
        for (int i = 0; i < W; ++i) {
            co[n][i] = 1.f;
            si[n][i] = 0.f;
            if (turns)
                turn(pos * (p.inv_freq[W * u + i] * 0.15915494309189533577), p.attention_factor,
                     co[n][i], si[n][i]);
        }
    }
    auto load = [&](const float *from, int n) {
        Piece<W> x;
        if constexpr (W == 4) {
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
            if (has[n]) {
                a = *reinterpret_cast<const float4 *>(from + ia[n]);
                b = *reinterpret_cast<const float4 *>(from + ib[n]);
            }
            x.a[0] = a.x; x.a[1] = a.y; x.a[2] = a.z; x.a[3] = a.w;
            x.b[0] = b.x; x.b[1] = b.y; x.b[2] = b.z; x.b[3] = b.w;
        } else {
            x.a[0] = has[n] ? from[ia[n]] : 0.f;
            x.b[0] = has[n] ? from[ib[n]] : 0.f;
        }
        return x;
    };
    auto store = [&](float *to, int n, const Piece<W> &x) {
        if (!has[n]) return;
        if constexpr (W == 4) {
            *reinterpret_cast<float4 *>(to + ia[n]) = make_float4(x.a[0], x.a[1], x.a[2], x.a[3]);
            *reinterpret_cast<float4 *>(to + ib[n]) = make_float4(x.b[0], x.b[1], x.b[2], x.b[3]);
        } else {
            to[ia[n]] = x.a[0];
            to[ib[n]] = x.b[0];
        }
    };
#pragma unroll
    for (int n = 0; n < NU; ++n) {
        if (p.qw) qw[n] = load(p.qw, n);
        if (p.kw) kw[n] = load(p.kw, n);
    }
    const int at = p.at ? p.at[token] : p.at_all;
    const bool fits = at >= 0 && at < p.max_seq;

    // ---- the heads, B at a time; every lane of a wave makes the same rounds
    constexpr int B = NU == 1 ? 4 : 1;
    for (int d = 0; d < per; d += B) {
        Piece<W> x[B][NU];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int h = min(h0 + d + i, heads - 1);
            const float *from =
                h < p.hq ? p.q.p + token * p.q.st + h * p.q.sh
                : h < p.hq + p.hkv ? p.k.p + token * p.k.st + (h - p.hq) * p.k.sh
                                   : p.v.p + token * p.v.st + (h - p.hq - p.hkv) * p.v.sh;
#pragma unroll
            for (int n = 0; n < NU; ++n) x[i][n] = load(from, n);
        }
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int h = h0 + d + i;
            const bool is_q = h < p.hq, is_v = h >= p.hq + p.hkv;
            const bool norm = is_q ? p.qw != nullptr : p.kw != nullptr && !is_v;
            float scale = 1.f;   // times 2^up: of a head at f32's ends it is no f32 itself
            int up = 0;
            if (p.qw || p.kw) {   // squares and their sum in 64 bits: none is out of range
                double sum = 0.0;
#pragma unroll
                for (int n = 0; n < NU; ++n)
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        sum = fma((double)x[i][n].a[j], (double)x[i][n].a[j], sum);
                        sum = fma((double)x[i][n].b[j], (double)x[i][n].b[j], sum);
                    }
                if (norm) scale = (float)frexp(1.0 / sqrt(head_sum<L>(sum) / D + p.eps), &up);
            }
            if (d + i >= per || h >= h1) continue;
#pragma unroll
            for (int n = 0; n < NU; ++n) {
                Piece<W> &y = x[i][n];
                if (norm) {
                    const Piece<W> &w = is_q ? qw[n] : kw[n];
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        y.a[j] = ldexpf(y.a[j], up) * scale * w.a[j];
                        y.b[j] = ldexpf(y.b[j], up) * scale * w.b[j];
                    }
                }
                if (!is_v && lane + n * L < turning) {
                    float z[2 * W];
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        z[j] = y.a[j];
                        z[W + j] = y.b[j];
                    }
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        // pair j: elements j and W + j of the unit, or 2j and 2j + 1
                        const int ea = INTERLEAVED ? 2 * j : j;
                        const int eb = INTERLEAVED ? 2 * j + 1 : W + j;
                        const float a = z[ea], b = z[eb];
                        z[ea] = fmaf(a, co[n][j], -(b * si[n][j]));
                        z[eb] = fmaf(b, co[n][j], a * si[n][j]);
                    }
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        y.a[j] = z[j];
                        y.b[j] = z[W + j];
                    }
                }
                if (is_q) {
                    store(p.q_out + ((int64_t)token * p.hq + h) * D, n, y);
                } else if (!p.append) {
                    store(p.k_out + ((int64_t)token * p.hkv + h - p.hq) * D, n, y);
                } else if (fits) {
                    const RopeCache &c = is_v ? p.vc : p.kc;
                    const int hh = h - p.hq - (is_v ? p.hkv : 0);
                    store(c.p + token * c.sb + hh * c.sh + at * c.ss, n, y);
                }
            }
        }
    }
}

bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <int L, int NU, int W>
int launch(const RopeParams &p, hipStream_t s) {
    const int heads = p.hq + (p.append ? 2 : 1) * p.hkv;
    // Heads a group: up to four share the angles, but groups for every CU first.
    const int64_t groups = (int64_t)p.n * heads;
    int per = 1;
    while (per < 4 && groups / (2 * per) * L >= 256 * 512) per *= 2;
    const int parts = (heads + per - 1) / per;
    const int64_t blocks = ((int64_t)p.n * parts + 256 / L - 1) / (256 / L);
    TB_REQUIRE(blocks * 256 <= kMaxThreads, TB_ERR_UNSUPPORTED,
               "TB_UNSUPPORTED: norm_rope: more threads than one launch has, 2^32 - 1");
    if (p.interleaved)
        hipLaunchKernelGGL((k_norm_rope<L, NU, W, true>), dim3((uint32_t)blocks), dim3(256), 0, s,
                           p, per, parts);
    else
        hipLaunchKernelGGL((k_norm_rope<L, NU, W, false>), dim3((uint32_t)blocks), dim3(256), 0, s,
                           p, per, parts);
    TB_LAUNCHED();
    return TB_OK;
}

}  // namespace

int launch_norm_rope(const RopeParams &p, hipStream_t s) {
    auto rows4 = [](const void *q, int64_t a, int64_t b, int64_t c) {
        return aligned16(q) && a % 4 == 0 && b % 4 == 0 && c % 4 == 0;
    };
    const bool wide = p.hd % 8 == 0 && p.rotary % 8 == 0 && rows4(p.q.p, p.q.st, p.q.sh, 0) &&
                      rows4(p.k.p, p.k.st, p.k.sh, 0) && rows4(p.v.p, p.v.st, p.v.sh, 0) &&
                      rows4(p.kc.p, p.kc.sb, p.kc.sh, p.kc.ss) &&
                      rows4(p.vc.p, p.vc.sb, p.vc.sh, p.vc.ss) && aligned16(p.qw) &&
                      aligned16(p.kw) && aligned16(p.q_out) && aligned16(p.k_out);
    const int units = wide ? p.hd / 8 : p.hd / 2;
    if (wide)
        return units <= 4    ? launch<4, 1, 4>(p, s)
               : units <= 8  ? launch<8, 1, 4>(p, s)
               : units <= 16 ? launch<16, 1, 4>(p, s)
               : units <= 32 ? launch<32, 1, 4>(p, s)
                             : launch<64, 1, 4>(p, s);
    return units <= 16   ? launch<16, 1, 1>(p, s)
           : units <= 64 ? launch<64, 1, 1>(p, s)
                         : launch<64, 4, 1>(p, s);
}

}  // namespace tb
