// Descriptor of the step from logits to the next token, as plain C++, for the kernel and the compiled wrappers.
#pragma once

struct CmeToken {
    int rows, vocab, dtype;              // CME_BF16 or CME_F32, of logits and processed
    const void* logits; long long logits_ld;
    void* processed;                     // [rows, vocab] or null
    const int* history; long long history_ld; int history_len;    // [rows, history_len] or null
    const int* lengths;                  // [rows]: entries of a history that count
    const int* prompts;                  // [rows] or null: entries before this one were given, not generated
    const float* repetition; const float* presence; const float* frequency; const float* temperature;    // [rows] or null
    const int* bias_ids; const float* bias_values; int biases;    // [rows, biases] or null
    const int* allowed; long long allowed_ld;                     // [rows, ceil(vocab / 32)], 0 between rows: one for all; or null
    const float* noise;                  // [rows, vocab] or null
    int* token; float* logprob;          // [rows]
};
