// Launcher of the logits processor (logits.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace tb {

struct LogitsParams {
    const float *x;          // [rows][vocab]
    float *y;                // processed logits [rows][vocab] (may be x), or null
    int64_t *tokens;         // each row's best token [rows], or null
    int rows, vocab;
    // Tokens so far, [groups][hist]; row r has group r / (rows / groups).
    const int64_t *history;
    const int32_t *history_len, *prompt_len;   // [groups], or null: hist, prompt
    int groups, hist, prompt;
    // The penalties: one value, or one a row.
    float rep, pres, freq;
    const float *rep_rows, *pres_rows, *freq_rows;
    // Biases [bias_groups][n_bias]; row r has group r / (rows / bias_groups).
    const int64_t *bias_ids;
    const float *bias;
    int bias_groups, n_bias;
    const int32_t *allowed;   // bit masks [rows][ceil(vocab / 32)], allowed_stride words a row
    int64_t allowed_stride;
    // Draft trees: row r is node r % nodes of tree r / nodes.
    const int64_t *draft;         // [rows / nodes][nodes]
    const int32_t *tree_mask;     // [rows / nodes][nodes][ceil(nodes / 32)]
    int nodes;
};

// Scratch of a call with tokens; 0 without.
size_t logits_scratch(int rows, int vocab, bool tokens);
int launch_logits(const LogitsParams &p, void *scratch, hipStream_t s);

}  // namespace tb
