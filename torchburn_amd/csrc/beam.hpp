// Launchers of beam search's selection and its caches' reordering (beam.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace tb {

constexpr int kMaxBeams = 64;            // beams of a group
constexpr int kMaxBeamResults = 64;      // continuations taken of a group
constexpr int kMaxBeamVocab = 1 << 20;
constexpr int kBeamLayersPerLaunch = 64;   // layers that one reorder launch moves

struct BeamSelect {
    const float *logits;       // [groups][beams][vocab]
    const float *scores;       // [groups][beams]
    const uint8_t *finished;   // [groups][beams] or null
    int64_t eos;               // the one continuation of a finished beam
    float *out_scores;         // [groups][k]
    int64_t *tokens, *parents; // [groups][k]
    int groups, beams, vocab, k;
};

size_t beam_select_scratch(int groups, int beams, int vocab, int k);
int launch_beam_select(const BeamSelect &p, void *scratch, hipStream_t s);

struct BeamReorder {
    const int64_t *parents;    // [groups][beams]
    const int32_t *lens;       // [groups][beams] on the device, or null: len
    int len;
    int groups, beams, layers, hkv, hd, max_seq;
    int64_t ksg, ksb, ksh, kss;   // strides of every layer's caches in elements: group, beam,
    int64_t vsg, vsb, vsh, vss;   // KV head, position
};

// Beam j of a group takes over the first positions of beam parents[j]'s rows, in the `layers`
// caches at kc / vc (host arrays of device pointers).
int launch_beam_reorder(const BeamReorder &p, float *const *kc, float *const *vc, hipStream_t s);

}  // namespace tb
