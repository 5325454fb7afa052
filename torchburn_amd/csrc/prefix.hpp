// Launcher of attention over a shared prefix and sequences' own caches (prefix_attn.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace tb {

constexpr int kMaxPrefixHeads = 1024;          // query heads
constexpr int kMaxPrefixRows = 1 << 23;        // groups times rows times query heads

// Strides are in elements; the innermost dimension is contiguous.
struct PrefixCache {
    const float *p;
    int64_t sb, sh, ss;   // group (sequence of its own caches), KV head, position
};

struct PrefixAttn {
    const float *q;               // [groups][rows][hq][hd]
    PrefixCache kp, vp;           // shared by a group's rows
    PrefixCache k, v;             // a row's own, sb between rows
    const int32_t *prefix_lens;   // [groups] on the device, or null: prefix_len
    const int32_t *own_lens;      // [groups * rows] on the device, or null: own_len
    int prefix_len, own_len;
    int max_prefix, max_own;      // positions that the caches hold
    float *out;                   // [groups][rows][hq][hd]
    int groups, rows, hq, hkv, hd;
    float scale;
};

// Whether one launch can have the threads of a call with lengths up to prefix and own.
bool prefix_attention_fits(int groups, int rows, int hq, int hkv, int hd, int prefix, int own);
// Scratch for lengths up to prefix and own; 0 where a single block sees a row's all.
size_t prefix_attention_scratch(int groups, int rows, int hq, int hkv, int hd, int prefix, int own);
int launch_prefix_attention(const PrefixAttn &a, float *scratch, hipStream_t s);

}  // namespace tb
