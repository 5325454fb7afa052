// Launchers of the draft-tree operators (tree.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace tb {

constexpr int kMaxTreeNodes = 1024;      // nodes of one draft tree
constexpr int kMaxTreeHeads = 1024;      // query heads: rows of a KV head stay below 2^20
constexpr int kTreeLayersPerLaunch = 64; // caches that one accept launch moves rows in

// parents [batch][n] -> ancestor-or-self bit masks [batch][n][ceil(n / 32)] and
// depths [batch][n].
int launch_tree_masks(const int32_t *parents, int32_t *mask, int32_t *depth, int batch, int n,
                      hipStream_t s);

// Strides are in elements; the innermost dimension is contiguous.
struct TreeCache {
    const float *p;
    int64_t sb, sh, ss;   // sequence, KV head, position
};

struct TreeAttn {
    const float *q;          // [batch][n][hq][hd]
    TreeCache k, v;
    const int32_t *mask;     // [batch][n][ceil(n / 32)], mask_sb words between sequences
    int64_t mask_sb;
    const int32_t *kv_lens;  // [batch] on the device, or null: kv_len for every sequence
    int kv_len;
    float *out;              // [batch][n][hq][hd]
    int batch, n, hq, hkv, hd, max_seq;
    float scale;
};

// Scratch for keys up to position max_len (kv_len + n, or max_seq where the
// lengths are on the device); 0 where one block walks all of them.
size_t tree_attention_scratch(int batch, int n, int hq, int hkv, int hd, int max_len);
int launch_tree_attention(const TreeAttn &a, int max_len, float *scratch, hipStream_t s);

// The length of sequence b's prefix, inside the cache whatever the device holds.
__device__ __forceinline__ int prefix_len(const int32_t *lens, int len, int b, int max_seq) {
    const int l = lens ? lens[b] : len;
    return min(max(l, 0), max_seq);
}

struct TreeAccept {
    const int32_t *parents;          // [batch][n]
    const int64_t *draft, *next;     // [batch][n]
    const int32_t *kv_lens;          // [batch] or null: kv_len
    int kv_len;
    int32_t *path, *n_path;          // [batch][n], [batch]
    int64_t *token;                  // [batch]
    int batch, n, hkv, hd, max_seq, layers;
    TreeCache k, v;                  // strides of every layer's caches; p unused
};

// The accepted path of every tree, and its rows' move to the prefix's end in
// the `layers` caches at kc / vc (host arrays of device pointers).
int launch_tree_accept(const TreeAccept &a, float *const *kc, float *const *vc, hipStream_t s);

}  // namespace tb
