// Arguments shared by the attention kernels over the 8-bit paged cache.
#pragma once

#include "q8.cuh"

namespace dkv {

constexpr int kQ8MaxRows = 64;         // query rows (token x GQA head) of a decode / verify call
constexpr size_t kQ8Tickets = 16384;   // fixed ticket region at the start of the work buffer
static_assert(kQ8Tickets * sizeof(unsigned) == 65536, "the 64 KB that callers clear");

struct Q8AttnArgs {
    Q8View v;
    int group, T, batch;
    const float* q;              // [batch * T][n_kv * group][d]
    const int32_t* entry0;       // [batch]
    const int32_t* n_rows;       // [batch] or null: tokens of the call a sequence has
    void* out;                   // [batch * T][n_kv * group * d]
    int out_dtype;
    int split, n_splits, n_rb;   // keys per split (prompt chunks), splits, row blocks per (sequence, head)
    float scale;                 // log2 e / sqrt(d)
    float* part;                 // [batch][n_kv][n_rb][n_splits][rows a block][d + 4]: max, sum, -, -, O
    unsigned* tickets;           // [batch][n_kv][n_rb]
    float* scores;               // [batch][n_kv][capacity][s_ld] (log2 units) or null
    float2* stats;               // [batch][n_kv][T * group] (max in log2 units, 1 / sum)
    int s_ld;
    uint32_t* err;

    // token 0's entry, held to the capacity (entries behind it are recorded by beyond())
    DKV_DEV int first(int b) const { return min(entry0[b], v.capacity()); }
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

DKV_DEV float q8_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// Two outputs of query row gr (elements e, e + 1); rows of tokens a sequence
// does not have stay as they were.
template <int D>
DKV_DEV void q8_store2(const Q8AttnArgs& a, int b, int h, int gr, int n_tok, int e, float x0, float x1) {
    const int t = gr / a.group;
    if (t >= n_tok) return;
    const size_t at = (((size_t)b * a.T + t) * a.v.n_kv * a.group + h * a.group + gr % a.group) * D + e;
    if (a.out_dtype == DKV_F32)
        *reinterpret_cast<float2*>(reinterpret_cast<float*>(a.out) + at) = make_float2(x0, x1);
    else
        *reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<uint16_t*>(a.out) + at) = __floats2bfloat162_rn(x0, x1);
}

// After a CTA has stored its split's partial rows (max in log2 units, sum,
// unnormalised O; an empty split has max -infinity and no O) of row block
// `bhr`, the last CTA to arrive merges all splits and writes the outputs (and
// the rows' stats).  A thread merges an element pair on its own, online in
// split order with kMergeQ splits' loads in flight: no barrier, one round of
// loads up to kMergeQ splits.
template <int D, int RB>
DKV_DEV void q8_merge_splits(const Q8AttnArgs& a, size_t bhr, int b, int h, int rbase, int R, int n_tok) {
    constexpr int PS = D + 4, kMergeQ = 16;
    __shared__ int is_last;
    __syncthreads();                     // the CTA's partials are stored
    if (threadIdx.x == 0) {
        // release and acquire on the device, cumulative over the barriers: the
        // CTA's stores before, the other CTAs' partials after
        unsigned* tk = a.tickets + bhr;
        unsigned before;
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;\n" : "=r"(before) : "l"(tk) : "memory");
        is_last = before == (unsigned)(a.n_splits - 1);
        if (is_last) *tk = 0u;
    }
    __syncthreads();
    if (!is_last) return;
    const int ns = a.n_splits;
    const float* parts = a.part + bhr * ns * (size_t)RB * PS;
    for (int i = threadIdx.x; i < R * (D / 2); i += blockDim.x) {
        const int r = i / (D / 2), e = i % (D / 2) * 2;
        float M = -INFINITY, L = 0.f, x0 = 0.f, x1 = 0.f;
        for (int q0 = 0; q0 < ns; q0 += kMergeQ) {
            float2 ml[kMergeQ], y[kMergeQ];
#pragma unroll
            for (int k = 0; k < kMergeQ; ++k) {
                ml[k] = make_float2(-INFINITY, 0.f);
                y[k] = make_float2(0.f, 0.f);
                if (q0 + k < ns) {
                    const float* at = parts + ((size_t)(q0 + k) * RB + r) * PS;
                    ml[k] = __ldcg(reinterpret_cast<const float2*>(at));
                    y[k] = __ldcg(reinterpret_cast<const float2*>(at + 4 + e));
                }
            }
            float m = M;
#pragma unroll
            for (int k = 0; k < kMergeQ; ++k) m = fmaxf(m, ml[k].x);
            if (m == -INFINITY) continue;
            const float al = M == -INFINITY ? 0.f : q8_ex2(M - m);
            M = m;
            L *= al;
            x0 *= al;
            x1 *= al;
#pragma unroll
            for (int k = 0; k < kMergeQ; ++k) {
                if (ml[k].x == -INFINITY) continue;        // (its O was never written)
                const float w = q8_ex2(ml[k].x - m);
                L += ml[k].y * w;
                x0 += y[k].x * w;
                x1 += y[k].y * w;
            }
        }
        q8_store2<D>(a, b, h, rbase + r, n_tok, e, L == 0.f ? 0.f : x0 / L, L == 0.f ? 0.f : x1 / L);
        if (e == 0 && a.stats)
            a.stats[((size_t)b * a.v.n_kv + h) * (a.T * a.group) + rbase + r] =
                make_float2(M, L == 0.f || (rbase + r) / a.group >= n_tok ? 0.f : 1.f / L);
    }
}

int attn_q8_prefill(Q8AttnArgs& a, dkv_dims dims, void* work, size_t work_bytes, cudaStream_t st);
size_t attn_q8_prefill_work(dkv_dims dims, int group, int T, int capacity);
// Scratch for every T up to max_T (a shorter prompt chunk may take more splits).
size_t attn_q8_work_upto(dkv_dims dims, int group, int max_T, int capacity, bool mass);

}  // namespace dkv
