// Arguments shared by the attention kernels over the 8-bit paged cache.
#pragma once

#include "q8.cuh"

namespace dkv {

constexpr int kQ8MaxRows = 64;         // query rows (token x GQA head) of a decode / verify call
constexpr size_t kQ8Tickets = 16384;   // fixed ticket region at the start of the work buffer

struct Q8AttnArgs {
    Q8View v;
    int group, T, batch;
    const float* q;              // [batch * T][n_kv * group][d]
    const int32_t* entry0;       // [batch]
    const int32_t* n_rows;       // [batch] or null: tokens of the call a sequence has
    void* out;                   // [batch * T][n_kv * group * d]
    int out_dtype;
    int split, n_splits, n_rb;   // keys per split, splits, row blocks per (sequence, head)
    float scale;                 // log2 e / sqrt(d)
    float* part;                 // [batch][n_kv][n_rb][n_splits][rows a block][d + 2]
    unsigned* tickets;           // [batch][n_kv][n_rb]
    float* scores;               // [batch][n_kv][capacity][s_ld] (log2 units) or null
    float2* stats;               // [batch][n_kv][T * group] (max in log2 units, 1 / sum)
    int s_ld;
    uint32_t* err;

    // entries the T tokens of sequence b may see at most (its own included)
    DKV_DEV int n_keys(int b) const {
        const int n = n_rows ? min(n_rows[b], T) : T;
        if (n <= 0) return 0;
        const long long e = (long long)entry0[b] + n;
        return (int)min(max(e, 0ll), (long long)v.capacity());
    }
    DKV_DEV bool beyond(int b) const {
        const int n = n_rows ? min(n_rows[b], T) : T;
        return n > 0 && (long long)entry0[b] + n > (long long)v.capacity();
    }
};

int attn_q8_prefill(Q8AttnArgs& a, dkv_dims dims, void* work, size_t work_bytes, cudaStream_t st);
size_t attn_q8_prefill_work(dkv_dims dims, int group, int T, int capacity, int split_keys);

}  // namespace dkv
