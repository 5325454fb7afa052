// Launcher of the head norms with the position rotation (rope.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tb {

constexpr int kMaxRopeHeadDim = 512;

// Strides are in elements; the innermost dimension is contiguous.
struct RopeHeads {
    const float *p;
    int64_t st, sh;   // token, head
};
struct RopeCache {
    float *p;
    int64_t sb, sh, ss;   // token's cache, head, position
};

struct RopeParams {
    RopeHeads q, k, v;            // v: with the caches only
    const int64_t *positions;     // [n]
    const double *inv_freq;       // [rotary / 2], in radians a position
    const float *qw, *kw;         // [head_dim] each, or null: no norm
    float *q_out, *k_out;         // [n][heads][head_dim]; k_out null with the caches
    RopeCache kc, vc;
    const int32_t *at;            // [n] where in its cache a token goes, or null: at_all
    int at_all, max_seq;
    int n, hq, hkv, hd, rotary;
    bool interleaved;
    bool append;                  // key and value rows go to the caches
    float attention_factor;
    double eps;
};

int launch_norm_rope(const RopeParams &p, hipStream_t s);

}  // namespace tb
