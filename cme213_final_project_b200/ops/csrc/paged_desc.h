// Descriptor of a call over a paged cache of keys and values, as plain C++, for the kernels' side (paged.h) and the compiled
// wrappers.
#pragma once

// Position p of a sequence lies in slot p % page of the cache's page pages[sequence, p / page]; a table entry outside [0, num_pages)
// stands for a page that is not there.  Strides count elements; the columns of a head are contiguous.
struct CmePaged {
    int seqs, heads, kv_heads, head_dim;
    int page, width, num_pages;          // slots of a page, columns of the table, pages of the cache
    int dtype;                           // CME_BF16 or CME_F32, of everything but lse
    int rows;                            // new tokens of all sequences
    int max_len;                         // keys from this position on do not take part, as those beyond the table
    float scale;                         // of the scores
    long long q_token, q_head;           // strides of q (attention) or of the new keys (append)
    long long v_token, v_head;           // strides of the new values (append)
    long long k_page_stride, k_head_stride, k_slot_stride;
    long long v_page_stride, v_head_stride, v_slot_stride;
    const void* q;                       // attention: [rows, heads, head_dim];  append: the new keys [rows, kv_heads, head_dim]
    const void* nv;                      // append: the new values
    void* k; void* v;                    // the cache, [num_pages, kv_heads, page, head_dim]
    const int* pages; long long pages_ld;    // [seqs, width]
    const int* offsets;                  // [seqs + 1]: rows of sequence b are [offsets[b], offsets[b + 1])
    const int* lengths;                  // [seqs]: tokens of a sequence, the new ones among them
    void* o; float* lse;                 // [rows, heads, head_dim] and [rows, heads]
    float* ws; long long ws_bytes;       // scratch of cme_paged_attention_ws_bytes() bytes
};

// Scales of a cache of 8-bit integers (whose CmePaged has the type of the new rows, and strides of the cache in bytes): slot s of a page and
// head stands for its integers times [page, head, s / block].
struct CmePagedScales {
    float* k; float* v;
    int block;                           // slots of a scale: a multiple of 8 that divides a page
    long long k_page, k_head, v_page, v_head;    // strides, in elements
};
