// Speculative decoding over a drafted tree: ancestor masks from the parent list,
// and acceptance, which keeps one path of the tree in the cache (the attention
// between them is tree_attn.hip).
//
// A tree's n nodes are in topological order: parents[i] is -1 (a root: a child
// of the prefix's last token) or an earlier node.  Anything else marks node i
// as padding, and its descendants with it.  Node i's K / V row sits in the cache
// at position len + i, behind the prefix of len positions.
#include <math.h>

#include <algorithm>
#include <string>

#include "tb_common.hpp"
#include "tree.hpp"

namespace tb {

namespace {

// ---- ancestor masks -------------------------------------------------------
//
// mask(i) = {i} u mask(parent(i)), depth(i) = |mask(i)| - 1; a padding node has
// no bits and depth 0.  One block per tree, a thread per node.  Indices fall along
// a chain, so a row's words come one after the other: a thread first walks its
// chain to the end of its own 32 nodes (at most 31 steps), and then takes whole
// words from the nodes where the chain enters them (at most 31 more, where a walk
// by single nodes takes 1023 twice).  A drafter's tree of 26 takes 1.9 us, the launch alone,
// a chain of 64 nodes 3.2 (8.3 node by node).  Large trees are bound by the LDS reads
// of the chains, each waiting for the one before, and then by the rows' words, which
// leave one by one, a row apart from lane to lane: 64 trees of 512 take 7.7 us (5.2
// without those stores), a chain of 1024 19.2 (8.8; 117 node by node).
__global__ void k_tree_masks(const int32_t *__restrict__ parents, int32_t *__restrict__ mask,
                             int32_t *__restrict__ depth, int n) {
    __shared__ int par[kMaxTreeNodes], up[kMaxTreeNodes];
    __shared__ uint32_t in[kMaxTreeNodes];
    const size_t b = blockIdx.x;
    const int words = (n + 31) / 32;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int p = parents[b * n + i];
        par[i] = p < -1 || p >= i ? -2 : p;   // -1: a root, -2: padding
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        uint32_t bits = 0;
        int at = i;
        while (at >= (i & ~31)) {
            bits |= 1u << (at & 31);
            at = par[at];
        }
        in[i] = bits;
        up[i] = at;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        int d = -1, at = i;
        while (at >= 0) {
            d += __popc(in[at]);
            at = up[at];
        }
        const bool live = at == -1;
        int32_t *row = mask + (b * n + i) * words;
        at = live ? i : -1;
        for (int w = words - 1; w >= 0; --w) {
            const bool on = at >= 32 * w;   // at < 32 * (w + 1) here
            row[w] = on ? (int32_t)in[at] : 0;
            if (on) at = up[at];
        }
        depth[b * n + i] = live ? d : 0;
    }
}

// ---- acceptance -------------------------------------------------------------

struct LayerCaches {
    float *k[kTreeLayersPerLaunch], *v[kTreeLayersPerLaunch];
};

// The walk: node 0 is the root; from a node the path goes on to its lowest child
// whose drafted token (a negative one is none) is the node's next token.  Whether a
// node is such a child does not depend on the walk, so every node is tested at once
// (child[p] = the lowest one of node p), and one thread then follows child[].
//
// The move: K / V row len + path[j] to len + j.  path[j] >= j and path rises, so
// row j's source is past every row written for j' < j: each thread copies its
// columns in path order, and blocks share no columns.  Every block does the walk
// for itself (a few LDS steps against a second launch); block (0, 0) writes it.
// Bound by the launch and that walk: 5.0 us for 64 caches of 8 heads of 128.
// Grid (max(1, 2 * layers), column blocks, batch).
__global__ __launch_bounds__(256) void k_tree_accept(TreeAccept a, LayerCaches lc, bool report) {
    __shared__ int child[kMaxTreeNodes], path[kMaxTreeNodes];
    __shared__ int count;
    const int t = threadIdx.x, b = blockIdx.z, n = a.n;
    const int32_t *par = a.parents + (size_t)b * n;
    const int64_t *draft = a.draft + (size_t)b * n, *next = a.next + (size_t)b * n;
    for (int i = t; i < n; i += 256) child[i] = n;
    __syncthreads();
    for (int i = t; i < n; i += 256) {
        const int p = par[i];
        if (p >= 0 && p < i && draft[i] >= 0 && draft[i] == next[p]) atomicMin(&child[p], i);
    }
    __syncthreads();
    if (t == 0) {
        int c = 0;
        for (int at = par[0] == -1 ? 0 : n; at < n; at = child[at]) path[c++] = at;
        count = c;
    }
    __syncthreads();
    const int c = count;
    if (report && blockIdx.x == 0 && blockIdx.y == 0) {
        for (int i = t; i < n; i += 256) a.path[(size_t)b * n + i] = i < c ? path[i] : -1;
        if (t == 0) {
            a.n_path[b] = c;
            a.token[b] = c ? next[path[c - 1]] : -1;
        }
    }
    const int layer = blockIdx.x >> 1, col = blockIdx.y * 256 + t, per = a.hd / 4;
    if (layer >= a.layers || col >= a.hkv * per) return;
    const bool is_v = blockIdx.x & 1;
    const TreeCache &ca = is_v ? a.v : a.k;
    const int len = prefix_len(a.kv_lens, a.kv_len, b, a.max_seq);
    float *base = (is_v ? lc.v[layer] : lc.k[layer]) + b * ca.sb + (col / per) * ca.sh + 4 * (col % per);
    for (int j = 0; j < c; ++j) {
        const int from = path[j];
        if (from == j || len + from >= a.max_seq) continue;
        *reinterpret_cast<float4 *>(base + (len + j) * ca.ss) =
            *reinterpret_cast<const float4 *>(base + (len + from) * ca.ss);
    }
}

}  // namespace

int launch_tree_masks(const int32_t *parents, int32_t *mask, int32_t *depth, int batch, int n,
                      hipStream_t s) {
    const int threads = std::min(1024, (n + 63) / 64 * 64);
    hipLaunchKernelGGL(k_tree_masks, dim3(batch), dim3(threads), 0, s, parents, mask, depth, n);
    TB_LAUNCHED();
    return TB_OK;
}

int launch_tree_accept(const TreeAccept &a, float *const *kc, float *const *vc, hipStream_t s) {
    for (int l0 = 0; l0 == 0 || l0 < a.layers; l0 += kTreeLayersPerLaunch) {
        TreeAccept p = a;
        LayerCaches lc{};
        p.layers = std::min(kTreeLayersPerLaunch, a.layers - l0);
        for (int l = 0; l < p.layers; ++l) {
            lc.k[l] = kc[l0 + l];
            lc.v[l] = vc[l0 + l];
        }
        const dim3 grid(std::max(1, 2 * p.layers),
                        p.layers ? (p.hkv * (p.hd / 4) + 255) / 256 : 1, p.batch);
        hipLaunchKernelGGL(k_tree_accept, grid, dim3(256), 0, s, p, lc, l0 == 0);
        TB_LAUNCHED();
    }
    return TB_OK;
}

}  // namespace tb
