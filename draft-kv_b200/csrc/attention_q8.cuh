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
    float* part;                 // [batch][n_kv][n_rb][n_splits][rows a block][d + 4]: max, sum, -, -, O / sum
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
// Rows r = i / (D / E), E elements from E (i % (D / E)) on, for items i = i0 + u *
// stride (u < U): online over the splits in order, Q of them at a time, the loads
// of all U items of a step in flight together.  What is carried is the average so
// far (sums of V near fp32's largest would overflow).
template <int D, int RB, int E, int U, int Q>
DKV_DEV void q8_merge_items(const Q8AttnArgs& a, const float* parts, int b, int h, int rbase, int R, int n_tok, int i0,
                            int stride) {
    constexpr int PS = D + 4;
    float M[U], L[U], x[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        M[u] = -INFINITY, L[u] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) x[u][e] = 0.f;
    }
    for (int q0 = 0; q0 < a.n_splits; q0 += Q) {
        float2 ml[U][Q];
        float y[U][Q][E];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < Q; ++k) {
                const int i = i0 + u * stride;
                ml[u][k] = make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int e = 0; e < E; ++e) y[u][k][e] = 0.f;
                if (i < R * (D / E) && q0 + k < a.n_splits) {
                    const float* at = parts + ((size_t)(q0 + k) * RB + i / (D / E)) * PS;
                    ml[u][k] = __ldcg(reinterpret_cast<const float2*>(at));
#pragma unroll
                    for (int e = 0; e < E; e += 2) {
                        const float2 t = __ldcg(reinterpret_cast<const float2*>(at + 4 + i % (D / E) * E + e));
                        y[u][k][e] = t.x, y[u][k][e + 1] = t.y;
                    }
                }
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float m = M[u];
#pragma unroll
            for (int k = 0; k < Q; ++k) m = fmaxf(m, ml[u][k].x);
            if (m == -INFINITY) continue;
            float w[Q];
            const float before = M[u] == -INFINITY ? 0.f : L[u] * q8_ex2(M[u] - m);
            M[u] = m;
            L[u] = before;
#pragma unroll
            for (int k = 0; k < Q; ++k) {
                w[k] = ml[u][k].x == -INFINITY ? 0.f : ml[u][k].y * q8_ex2(ml[u][k].x - m);
                L[u] += w[k];
            }
            const float inv = 1.f / L[u];                  // (a split with a key has a sum of 1 or more, or NaN)
#pragma unroll
            for (int e = 0; e < E; ++e) x[u][e] *= before * inv;
#pragma unroll
            for (int k = 0; k < Q; ++k) {
                if (ml[u][k].x == -INFINITY) continue;     // (its O was never written)
#pragma unroll
                for (int e = 0; e < E; ++e) x[u][e] += y[u][k][e] * (w[k] * inv);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = i0 + u * stride, r = i / (D / E), at = i % (D / E) * E;
        if (i >= R * (D / E)) continue;
        const bool none = L[u] == 0.f;
#pragma unroll
        for (int e = 0; e < E; e += 2)
            q8_store2<D>(a, b, h, rbase + r, n_tok, at + e, x[u][e], x[u][e + 1]);
        if (at == 0 && a.stats)
            a.stats[((size_t)b * a.v.n_kv + h) * (a.T * a.group) + rbase + r] =
                make_float2(M[u], none || (rbase + r) / a.group >= n_tok ? 0.f : 1.f / L[u]);
    }
}

// After a CTA has stored its split's partial rows (max in log2 units, sum, O over
// the sum; an empty split has max -infinity and no O) of row block
// `bhr`, the last CTA to arrive merges all splits and writes the outputs (and
// the rows' stats).  A thread merges an element pair on its own, 16 loads of
// partials in flight: several splits of one item, or with few splits several
// items.
template <int D, int RB>
DKV_DEV void q8_merge_splits(const Q8AttnArgs& a, size_t bhr, int b, int h, int rbase, int R, int n_tok) {
    constexpr int PS = D + 4;
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
    const float* parts = a.part + bhr * a.n_splits * (size_t)RB * PS;
    const int nt = blockDim.x, i0 = threadIdx.x;
    if (a.n_splits <= 4) {
        for (int i = i0; i < R * (D / 2); i += 4 * nt) q8_merge_items<D, RB, 2, 4, 4>(a, parts, b, h, rbase, R, n_tok, i, nt);
    } else {
        for (int i = i0; i < R * (D / 2); i += nt) q8_merge_items<D, RB, 2, 1, 16>(a, parts, b, h, rbase, R, n_tok, i, nt);
    }
}

int attn_q8_prefill(Q8AttnArgs& a, dkv_dims dims, void* work, size_t work_bytes, cudaStream_t st);
size_t attn_q8_prefill_work(dkv_dims dims, int group, int T, int capacity);
// Scratch for every T up to max_T (a shorter prompt chunk may take more splits).
size_t attn_q8_work_upto(dkv_dims dims, int group, int max_T, int capacity, bool mass);

}  // namespace dkv
