// The arguments of attention over an 8-bit cache as one structure (attention_cache8.cu, attention_cache8_tc.cu).
#pragma once

struct Cache8Call {
    const void *q, *k, *v;
    const float *k_scale, *v_scale;
    void* out;
    const int *block_table, *seq_start, *seq_past, *seq_len;
    float *part_acc, *part_ml;
    int* status;
    void* stream;
    double scale;
    int dtype, max_blocks, n_pages, n_seqs, n_tokens, max_q_len, nq, nkv, d, ranges, range_pages, clusters;
};
static_assert(sizeof(Cache8Call) == 15 * 8 + 12 * 4, "14 addresses, a number of 64 bits and 12 of 32, without gaps");
