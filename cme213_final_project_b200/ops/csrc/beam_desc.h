// Descriptors of the steps of a search with several beams, as plain C++, for the kernels and the compiled wrappers.
#pragma once

struct CmeBeams {
    int groups, beams, width, vocab, dtype;    // CME_BF16 or CME_F32, of logits
    const void* logits; long long logits_ld;   // [groups x beams, vocab]
    const float* scores;                 // [groups, beams]; others than finite ones: the beam does not take part
    const unsigned char* finished;       // [groups, beams] or null
    const int* allowed; long long allowed_ld;  // [groups x beams, ceil(vocab / 32)], 0 between rows: one for all; or null
    int* parents; int* tokens; float* out;     // [groups, width]
    void* ws; long long ws_bytes;        // scratch of cme_beam_step_ws_bytes() bytes
};

// One tensor whose pages are copied: [layers, pages, heads, rows, row_bytes], strides in bytes; rows of a page: one for each `per` slots.
struct CmePages {
    char* base;
    int heads, row_bytes, per;
    long long layer, page, head, row;
};
struct CmeReorder {
    int groups, beams, width, slots, layers, num_pages, tensors;      // width: columns of the tables
    CmePages t[4];
    const int* pages; long long pages_ld;      // [groups x beams, width]
    const int* spare;                    // [groups x beams]
    const int* parents;                  // [groups, beams], numbers within the group
    const int* lengths;                  // [groups]
    int* new_pages; int* new_spare;      // as pages (contiguous) and spare
};
