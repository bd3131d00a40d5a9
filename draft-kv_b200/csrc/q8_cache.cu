// The 8-bit paged KV cache: append, read-back and eviction by attention mass.
//
// Stands beside dkv_full_write / dkv_full_read (draftkv/compress.py:59-73,
// draftkv/paged.py:120-138) and the drafter's eviction (draftkv/compress.py:
// 154-179); the reference has no 8-bit paged cache.
#include <algorithm>

#include "q8.cuh"

namespace dkv {

int q8_view(const char* who, const dkv_q8_cache* c, dkv_dims dims, int layer, Q8View* out) {
    DKV_REQUIRE(c && c->codes && c->scale && c->page_table, "%s: cache arrays required", who);
    DKV_REQUIRE(((uintptr_t)c->codes & 15) == 0 && ((uintptr_t)c->scale & 7) == 0, "%s: cache arrays misaligned", who);
    DKV_REQUIRE(dims.batch >= 1 && dims.n_kv >= 1 && dims.n_layers >= 1 && layer >= 0 && layer < dims.n_layers,
                "%s: dims/layer", who);
    DKV_UNSUPPORTED(dims.d == 64 || dims.d == 128, "%s: head size %d (64 or 128)", who, dims.d);
    DKV_UNSUPPORTED(c->page_size == 16 || c->page_size == 32 || c->page_size == 64 || c->page_size == 128,
                    "%s: page size %d (16, 32, 64 or 128)", who, c->page_size);
    DKV_REQUIRE(c->n_pages >= 1 && c->max_pages >= 1 && c->max_pages <= (1 << 30) / c->page_size,
                "%s: page counts", who);
    DKV_REQUIRE(dims.n_kv <= 65535 && dims.batch <= 32767, "%s: batch %d or heads %d too large", who, dims.batch,
                dims.n_kv);
    out->codes = c->codes;
    out->scale = c->scale;
    out->table = c->page_table;
    out->n_pages = c->n_pages;
    out->page = c->page_size;
    out->page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
    out->max_pages = c->max_pages;
    out->n_layers = dims.n_layers;
    out->n_kv = dims.n_kv;
    out->d = dims.d;
    out->layer = layer;
    return DKV_OK;
}

namespace {

constexpr int kQ8Threads = 128;

// Staged rows: fp32 [page][d + 8] (the 8 spreads a fragment's rows over the
// banks).
DKV_DEV int stage_ld(int d) { return d + 8; }

// Rows [lo, hi) of `stage` become codes of one side of a page under exponent
// e; rows below lo are re-rounded from exponent e_old to e when they differ;
// rows from hi on keep their bytes.  One 16-byte fragment a thread and step;
// a tile that gets no new byte is not touched, one that gets only new bytes
// is not read.
DKV_DEV void encode_side(uint8_t* side, const float* stage, int d, int page, bool is_v, int lo, int hi, int e,
                         int e_old) {
    const float up = q8_pow2(-e), again = q8_pow2(max(e_old - e, -126));
    const bool rescale = lo > 0 && e != e_old;
    const int ld = stage_ld(d), frags = d;                  // 16-byte fragments per 16-token tile
    const int t_first = rescale ? 0 : lo >> 4, t_last = (hi + 15) >> 4;
    for (int i = threadIdx.x; i < (t_last - t_first) * frags; i += blockDim.x) {
        const int tile = t_first + i / frags, f = i % frags;
        const int blk = f >> 5, lane = f & 31, g = lane >> 2, t = lane & 3;
        uint4* at = reinterpret_cast<uint4*>(side + (size_t)tile * 16 * d + (size_t)f * 16);
        const int k0 = tile * 16;
        const bool whole = lo <= k0 && hi >= k0 + 16;
        uint4 cur = whole ? make_uint4(0u, 0u, 0u, 0u) : *at;
        uint32_t w[4] = {cur.x, cur.y, cur.z, cur.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t out = 0;
#pragma unroll
            for (int c2 = 0; c2 < 2; ++c2) {               // byte pairs: columns 2t + 8 c2, + 1
                const uint32_t was = (w[q] >> (16 * c2)) & 0xffffu;
                const int col = 2 * t + 8 * c2;
                int tok0, tok1, x0, x1;
                if (is_v) {
                    tok0 = k0 + col;
                    tok1 = tok0 + 1;
                    x0 = x1 = blk * 32 + (q >> 1) * 16 + (q & 1) * 8 + g;
                } else {
                    tok0 = tok1 = k0 + g + 8 * (q & 1);
                    x0 = blk * 32 + (q >> 1) * 16 + col;
                    x1 = x0 + 1;
                }
                const bool n0 = tok0 >= lo && tok0 < hi, n1 = tok1 >= lo && tok1 < hi;
                const float a = n0 ? stage[tok0 * ld + x0] * up : q8_decode(was) * again;
                const float b = n1 ? stage[tok1 * ld + x1] * up : q8_decode(was >> 8) * again;
                uint32_t enc = q8_encode2(a, b);
                if (!n0 && !(rescale && tok0 < lo)) enc = (enc & 0xff00u) | (was & 0xffu);
                if (!n1 && !(rescale && tok1 < lo)) enc = (enc & 0x00ffu) | (was & 0xff00u);
                out |= enc << (16 * c2);
            }
            w[q] = out;
        }
        *at = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// A finite stand-in for what was given: NaN -> 0, infinities -> the largest.
DKV_DEV float finite(float x, bool& bad) {
    if ((__float_as_uint(x) & 0x7f800000u) != 0x7f800000u) return x;
    bad = true;
    return x != x ? 0.f : copysignf(3.402823466e38f, x);
}

struct Q8AppendArgs {
    Q8View v;
    const void* k;
    const void* vv;
    int src_dtype, rows;
    int64_t sb, st, sh;          // source strides (elements) of sequence, token, head
    const int32_t* entry0;
    const int32_t* n_rows;
    const int32_t* pos0;
    float* mass;                 // [batch][n_kv][capacity] or null
    int32_t* pos;
    uint32_t* err;
};

// One CTA per (page a run of rows reaches, head, sequence x {K, V}).  The
// page's new rows are staged in shared memory in fp32 (bf16 and fp32 sources
// are exact there) while their largest magnitude is taken, so each source
// element is read once; the scale is a power of two, so scaling is exact and
// a code is rounded once.  Memory-bound: rows * 2 d * (source bytes + 1) per
// head and, for a page begun earlier, that page's codes.
template <bool VEC>
__global__ void __launch_bounds__(kQ8Threads) q8_append_kernel(Q8AppendArgs a) {
    extern __shared__ __align__(16) float stage[];
    __shared__ float red[32];
    pdl_trigger();
    pdl_wait();
    const Q8View& v = a.v;
    const int b = blockIdx.z >> 1, i = blockIdx.z & 1, h = blockIdx.y;
    const int n = a.n_rows ? min(a.n_rows[b], a.rows) : a.rows;
    const int e0 = a.entry0[b];
    if (n <= 0) return;
    if (e0 < 0 || e0 > v.capacity() - n) {                  // rows outside the table: nothing of this run is written
        if (threadIdx.x == 0) atomicOr(a.err, kErrQ8Page);
        return;
    }
    const int pg = (e0 >> v.page_shift) + blockIdx.x;
    const int base = pg << v.page_shift;
    const int lo = max(e0 - base, 0), hi = min(e0 + n - base, v.page);
    if (hi <= lo) return;
    const int pid = v.row(b)[pg];
    if (!v.ok(pid)) {
        if (threadIdx.x == 0) atomicOr(a.err, kErrQ8Page);
        return;
    }
    const int d = v.d, ld = stage_ld(d), r0 = base + lo - e0;     // first source row of this page
    const int64_t off = (int64_t)b * a.sb + (int64_t)h * a.sh + (int64_t)r0 * a.st;
    const void* src = i ? a.vv : a.k;
    float amax = 0.f;
    bool bad = false;
    if (VEC) {
        const int cpr = d / 8;                                    // chunks of 8 elements a row
        for (int c = threadIdx.x; c < (hi - lo) * cpr; c += kQ8Threads) {
            const int r = c / cpr, x = (c % cpr) * 8;
            const int64_t o = off + r * a.st + x;
            float e[8];
            if (a.src_dtype == DKV_F32) {
                const float4 p = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(src) + o));
                const float4 q = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(src) + o + 4));
                e[0] = p.x, e[1] = p.y, e[2] = p.z, e[3] = p.w, e[4] = q.x, e[5] = q.y, e[6] = q.z, e[7] = q.w;
            } else {
                const uint4 p = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(src) + o));
                const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    e[2 * q] = __uint_as_float(w[q] << 16);
                    e[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
                }
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                e[q] = finite(e[q], bad);
                amax = fmaxf(amax, fabsf(e[q]));
            }
            float* to = stage + (lo + r) * ld + x;
            *reinterpret_cast<float4*>(to) = make_float4(e[0], e[1], e[2], e[3]);
            *reinterpret_cast<float4*>(to + 4) = make_float4(e[4], e[5], e[6], e[7]);
        }
    } else {
        for (int c = threadIdx.x; c < (hi - lo) * d; c += kQ8Threads) {
            const int r = c / d, x = c % d;
            const float e = finite(load_as_f32(src, a.src_dtype, (size_t)(off + r * a.st + x)), bad);
            amax = fmaxf(amax, fabsf(e));
            stage[(lo + r) * ld + x] = e;
        }
    }
    if (bad) atomicOr(a.err, kErrQ8NonFinite);
    if (i == 0 && a.mass) {
        const size_t m0 = ((size_t)b * v.n_kv + h) * v.capacity() + base;
        for (int r = lo + threadIdx.x; r < hi; r += kQ8Threads) a.mass[m0 + r] = 0.f;
    }
    if (i == 0 && a.pos) {
        const size_t m0 = ((size_t)b * v.n_kv + h) * v.capacity() + base;
        const int p0 = a.pos0 ? a.pos0[b] : e0;
        for (int r = lo + threadIdx.x; r < hi; r += kQ8Threads) a.pos[m0 + r] = p0 + base + r - e0;
    }
    amax = block_max(amax, red);
    float* sc = v.scale + v.scale_at(pid, h, i);
    const int e_old = lo > 0 ? min(max(q8_scale_exp(*sc), kQ8ExpMin), kQ8ExpMax) : kQ8ExpMin;
    const int e = max(q8_exp_of(amax), e_old);
    __syncthreads();                                              // every thread has read the old scale
    if (threadIdx.x == 0) *sc = q8_pow2(e);
    encode_side(v.side(pid, h, i), stage, d, v.page, i != 0, lo, hi, e, e_old);
}

// [n][n_kv][2][d] fp32 of entries [0, n) of one sequence: one CTA per
// (16-token tile, head), a thread per 16-byte fragment of K and V.
__global__ void q8_read_kernel(Q8View v, int b, int n, float* dst, uint32_t* err) {
    const int tile = blockIdx.x, h = blockIdx.y, d = v.d;
    const int pid = v.row(b)[(tile * 16) >> v.page_shift];
    const bool ok = v.ok(pid);
    if (!ok && threadIdx.x == 0) atomicOr(err, kErrQ8Page);
    const int in_page = (tile * 16) & (v.page - 1);
    for (int f = threadIdx.x; f < 16 * d * 2; f += blockDim.x) {
        const int x = f % d, i = (f / d) & 1, k = f / (2 * d);
        const int key = tile * 16 + k;
        if (key >= n) continue;
        float val = 0.f;
        if (ok) {
            const int byte = i ? q8_v_byte(d, in_page + k, x) : q8_k_byte(d, in_page + k, x);
            val = q8_decode(v.side(pid, h, i)[byte]) * v.scale[v.scale_at(pid, h, i)];
        }
        dst[(((size_t)key * v.n_kv + h) * 2 + i) * d + x] = val;
    }
}

// ---------------------------------------------------------------- eviction
// Order-preserving integer of a mass: equal masses compare equal (-0 = +0),
// NaN above everything.
DKV_DEV uint32_t mass_key(float m) {
    if (m != m) return 0xffffffffu;
    const uint32_t u = __float_as_uint(m + 0.f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

struct Q8EvictArgs {
    Q8View v;
    const int32_t* out_table;    // [batch][out_pages]
    int out_pages;
    const float* mass;           // [batch][n_kv][capacity]
    const int32_t* pos;
    float* mass_out;
    int32_t* pos_out;
    const int32_t* n;
    const int32_t* budget;
    int sink, recent;
    int32_t* kept;               // [batch][n_kv][out_pages * page], -1 behind the last
    uint32_t* err;
};

// Entries a sequence keeps: min(n, max(budget, sink + recent)), bounded by the
// output table (recorded as an error when that is smaller).
DKV_DEV int evict_keep(const Q8EvictArgs& a, int b, int* n_out) {
    const int n = min(max(a.n[b], 0), a.v.capacity());
    const int want = min(n, max(a.budget[b], a.sink + a.recent));
    *n_out = n;
    return min(max(want, 0), a.out_pages << a.v.page_shift);
}

constexpr int kSelThreads = 1024;

// Which entries stay: per (sequence, head) the `drop` lowest (mass, index)
// of the unprotected entries go.  The drop-th smallest mass is found by a
// radix select (four passes of 8 bits over the masses), then one ordered pass
// counts the entries that stay and writes their indices, masses and positions.
__global__ void __launch_bounds__(kSelThreads) q8_select_kernel(Q8EvictArgs a) {
    __shared__ unsigned hist[256];
    __shared__ unsigned s_prefix, s_need;
    __shared__ int wsum_lt[32], wsum_eq[32];
    const int h = blockIdx.x, b = blockIdx.y;
    int n;
    const int keep = evict_keep(a, b, &n);
    if (threadIdx.x == 0 && (a.n[b] > a.v.capacity() || a.n[b] < 0 ||
                             keep < min(n, max(a.budget[b], a.sink + a.recent))))
        atomicOr(a.err, kErrQ8Page);
    const size_t cap = a.v.capacity(), row = ((size_t)b * a.v.n_kv + h);
    const float* mass = a.mass + row * cap;
    const int out_cap = a.out_pages << a.v.page_shift;
    int32_t* kept = a.kept + row * out_cap;
    const int f0 = min(a.sink, n), f1 = max(n - a.recent, f0);     // unprotected entries [f0, f1)
    const int drop = min(n - keep, f1 - f0);
    // radix select of the drop-th smallest key
    unsigned prefix = 0, need = (unsigned)drop;
    if (drop > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = threadIdx.x; i < 256; i += kSelThreads) hist[i] = 0;
            __syncthreads();
            const unsigned hi_mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
            for (int i = f0 + threadIdx.x; i < f1; i += kSelThreads) {
                const unsigned key = mass_key(mass[i]);
                if ((key & hi_mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
            }
            __syncthreads();
            if (threadIdx.x == 0) {
                unsigned left = need;
                int bin = 0;
                while (bin < 255 && hist[bin] < left) left -= hist[bin++];
                s_prefix = prefix | ((unsigned)bin << shift);
                s_need = left;
            }
            __syncthreads();
            prefix = s_prefix;
            need = s_need;                 // how many entries equal to the key found so far go
            __syncthreads();
        }
    }
    // ordered pass: an unprotected entry goes if its key is below `prefix`, or
    // equal with fewer than `need` equal ones before it
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int done_gone = 0, done_eq = 0;
    for (int c0 = 0; c0 < n; c0 += kSelThreads) {
        const int i = c0 + threadIdx.x;
        const bool in = i < n, open = in && i >= f0 && i < f1 && drop > 0;
        const float mval = in ? mass[i] : 0.f;
        const unsigned key = open ? mass_key(mval) : 0xffffffffu;
        const bool eq = open && key == prefix;
        const unsigned beq = __ballot_sync(0xffffffffu, eq);
        if (lane == 0) wsum_eq[warp] = __popc(beq);
        __syncthreads();
        int eq_before = done_eq + __popc(beq & ((1u << lane) - 1u)), eq_all = 0;
        for (int w = 0; w < kSelThreads / 32; ++w) {
            if (w < warp) eq_before += wsum_eq[w];
            eq_all += wsum_eq[w];
        }
        const bool gone = open && (key < prefix || (eq && eq_before < (int)need));
        const unsigned bg = __ballot_sync(0xffffffffu, gone);
        if (lane == 0) wsum_lt[warp] = __popc(bg);
        __syncthreads();
        int gone_before = done_gone + __popc(bg & ((1u << lane) - 1u)), gone_all = 0;
        for (int w = 0; w < kSelThreads / 32; ++w) {
            if (w < warp) gone_before += wsum_lt[w];
            gone_all += wsum_lt[w];
        }
        if (in && !gone) {
            const int o = i - gone_before;
            if (o < out_cap) {
                kept[o] = i;
                a.mass_out[row * cap + o] = mval;
                if (a.pos_out) a.pos_out[row * cap + o] = a.pos[row * cap + i];
            }
        }
        done_eq += eq_all;
        done_gone += gone_all;
        __syncthreads();
    }
    const int left = min(n - drop, out_cap);
    for (int i = left + threadIdx.x; i < out_cap; i += kSelThreads) kept[i] = -1;
    for (size_t i = left + threadIdx.x; i < cap; i += kSelThreads) {
        a.mass_out[row * cap + i] = 0.f;
        if (a.pos_out) a.pos_out[row * cap + i] = -1;
    }
}

// The kept rows of one output page, head and side: gathered as fp32 values
// (exact: an e4m3 code times a power of two), then written under the smallest
// scale that holds them, as an append of those values to an empty page would.
__global__ void __launch_bounds__(kQ8Threads) q8_gather_kernel(Q8EvictArgs a) {
    extern __shared__ __align__(16) float stage[];
    __shared__ float red[32];
    const Q8View& v = a.v;
    const int b = blockIdx.z >> 1, i = blockIdx.z & 1, h = blockIdx.y, pg = blockIdx.x;
    int n;
    const int keep = evict_keep(a, b, &n);
    const int cnt = min(keep - (pg << v.page_shift), v.page);
    if (cnt <= 0) return;
    const int pid = a.out_table[(size_t)b * a.out_pages + pg];
    const int32_t* kept = a.kept + (((size_t)b * v.n_kv + h) * a.out_pages + pg) * v.page;
    if (!v.ok(pid)) {
        if (threadIdx.x == 0) atomicOr(a.err, kErrQ8Page);
        return;
    }
    const int d = v.d, ld = stage_ld(d);
    const int32_t* tab = v.row(b);
    float amax = 0.f;
    for (int c = threadIdx.x; c < cnt * d; c += kQ8Threads) {
        const int r = c / d, x = c % d;
        const int src = kept[r];
        const int sp = src >= 0 ? tab[src >> v.page_shift] : -1;
        float val = 0.f;
        if (v.ok(sp)) {
            const int k = src & (v.page - 1);
            const int byte = i ? q8_v_byte(d, k, x) : q8_k_byte(d, k, x);
            val = q8_decode(v.side(sp, h, i)[byte]) * v.scale[v.scale_at(sp, h, i)];
        } else {
            atomicOr(a.err, kErrQ8Page);
        }
        amax = fmaxf(amax, fabsf(val));
        stage[r * ld + x] = val;
    }
    amax = block_max(amax, red);
    const int e = q8_exp_of(amax);
    if (threadIdx.x == 0) v.scale[v.scale_at(pid, h, i)] = q8_pow2(e);
    encode_side(v.side(pid, h, i), stage, d, v.page, i != 0, 0, cnt, e, e);
}

size_t stage_bytes(int page, int d) { return (size_t)page * (d + 8) * sizeof(float); }

}  // namespace
}  // namespace dkv

using namespace dkv;

extern "C" int dkv_q8_append(const dkv_q8_cache* cache, dkv_dims dims, int layer, const void* k, const void* vsrc,
                             int src_dtype, int rows, int64_t seq_stride, int64_t token_stride, int64_t head_stride,
                             const int32_t* entry0, const int32_t* n_rows, const int32_t* pos0, float* mass, int32_t* pos,
                             void* stream) {
    Q8AppendArgs a{};
    DKV_TRY(q8_view("dkv_q8_append", cache, dims, layer, &a.v));
    DKV_REQUIRE(rows >= 0 && (rows == 0 || (k && vsrc && entry0)), "dkv_q8_append: rows/sources");
    DKV_REQUIRE(src_dtype == DKV_F32 || src_dtype == DKV_BF16, "dkv_q8_append: source dtype %d", src_dtype);
    DKV_REQUIRE(rows <= a.v.capacity(), "dkv_q8_append: %d rows > capacity %d", rows, a.v.capacity());
    if (rows == 0) return DKV_OK;
    a.k = k;
    a.vv = vsrc;
    a.src_dtype = src_dtype;
    a.rows = rows;
    a.sb = seq_stride;
    a.st = token_stride;
    a.sh = head_stride;
    a.entry0 = entry0;
    a.n_rows = n_rows;
    a.pos0 = pos0;
    a.mass = mass;
    a.pos = pos;
    a.err = device_error_word();
    DKV_REQUIRE(a.err, "dkv_q8_append: device error word unavailable");
    const int page = a.v.page, touched = (rows + page - 2) / page + 1;
    const int64_t align = src_dtype == DKV_F32 ? 4 : 8;      // elements in 16 bytes
    const bool vec = (((uintptr_t)k | (uintptr_t)vsrc) & 15) == 0 && seq_stride % align == 0 &&
                     token_stride % align == 0 && head_stride % align == 0;
    const dim3 grid((unsigned)touched, (unsigned)dims.n_kv, (unsigned)dims.batch * 2);
    const size_t smem = stage_bytes(page, dims.d);
    ProfScope ps(DKV_PROF_APPEND, 0.0, (cudaStream_t)stream);
    if (vec) {
        DKV_CUDA(allow_smem_max_once<q8_append_kernel<true>>());
        DKV_CUDA(launch_pdl(q8_append_kernel<true>, grid, dim3(kQ8Threads), smem, (cudaStream_t)stream, a));
    } else {
        DKV_CUDA(allow_smem_max_once<q8_append_kernel<false>>());
        DKV_CUDA(launch_pdl(q8_append_kernel<false>, grid, dim3(kQ8Threads), smem, (cudaStream_t)stream, a));
    }
    return DKV_OK;
}

extern "C" int dkv_q8_read(const dkv_q8_cache* cache, dkv_dims dims, int b, int layer, int n, float* dst, void* stream) {
    Q8View v;
    DKV_TRY(q8_view("dkv_q8_read", cache, dims, layer, &v));
    DKV_REQUIRE(b >= 0 && b < dims.batch && n >= 0 && n <= v.capacity() && (n == 0 || dst), "dkv_q8_read args");
    if (n == 0) return DKV_OK;
    uint32_t* err = device_error_word();
    DKV_REQUIRE(err, "dkv_q8_read: device error word unavailable");
    q8_read_kernel<<<dim3((n + 15) / 16, dims.n_kv), 256, 0, (cudaStream_t)stream>>>(v, b, n, dst, err);
    DKV_LAUNCHED();
    return DKV_OK;
}

extern "C" int dkv_q8_evict(const dkv_q8_cache* cache, dkv_dims dims, int layer, const int32_t* n, const int32_t* budget,
                            int sink, int recent, const float* mass, const int32_t* pos, const int32_t* out_table,
                            int out_pages, float* mass_out, int32_t* pos_out, int32_t* kept, void* stream) {
    Q8EvictArgs a{};
    DKV_TRY(q8_view("dkv_q8_evict", cache, dims, layer, &a.v));
    DKV_REQUIRE(n && budget && mass && mass_out && out_table && kept, "dkv_q8_evict: arrays required");
    DKV_REQUIRE(mass != mass_out && (!pos || pos != pos_out), "dkv_q8_evict: mass and pos are written out of place");
    DKV_REQUIRE((pos == nullptr) == (pos_out == nullptr), "dkv_q8_evict: pos and pos_out go together");
    DKV_REQUIRE(sink >= 0 && recent >= 0 && sink <= (1 << 30) - recent, "dkv_q8_evict: sink %d, recent %d", sink, recent);
    DKV_REQUIRE(out_pages >= 1 && out_pages <= a.v.max_pages, "dkv_q8_evict: out_pages %d", out_pages);
    a.out_table = out_table;
    a.out_pages = out_pages;
    a.mass = mass;
    a.pos = pos;
    a.mass_out = mass_out;
    a.pos_out = pos_out;
    a.n = n;
    a.budget = budget;
    a.sink = sink;
    a.recent = recent;
    a.kept = kept;
    a.err = device_error_word();
    DKV_REQUIRE(a.err, "dkv_q8_evict: device error word unavailable");
    cudaStream_t st = (cudaStream_t)stream;
    q8_select_kernel<<<dim3(dims.n_kv, dims.batch), kSelThreads, 0, st>>>(a);
    DKV_LAUNCHED();
    DKV_CUDA(allow_smem_max_once<q8_gather_kernel>());
    q8_gather_kernel<<<dim3(out_pages, dims.n_kv, dims.batch * 2), kQ8Threads, stage_bytes(a.v.page, dims.d), st>>>(a);
    DKV_LAUNCHED();
    return DKV_OK;
}
