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
// head and, for a page begun earlier, that page's codes.  4 x 512 tokens of 8
// heads, d 128 (8.4 MB read, 4.2 MB written): 10.8 us from a cold start, of which
// 8 are one token's.
template <bool VEC>
__global__ void __launch_bounds__(kQ8Threads) q8_append_kernel(Q8AppendArgs a) {
    extern __shared__ __align__(16) float stage[];
    __shared__ float red[32];
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
                const float4 p = q8_ld(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(src) + o));
                const float4 q = q8_ld(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(src) + o + 4));
                e[0] = p.x, e[1] = p.y, e[2] = p.z, e[3] = p.w, e[4] = q.x, e[5] = q.y, e[6] = q.z, e[7] = q.w;
            } else {
                const uint4 p = q8_ld(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(src) + o));
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
    pdl_trigger();
    amax = block_max(amax, red);
    float* sc = v.scale + v.scale_at(pid, h, i);
    const int e_old = lo > 0 ? min(max(q8_scale_exp(*sc), kQ8ExpMin), kQ8ExpMax) : kQ8ExpMin;
    const int e = max(q8_exp_of(amax), e_old);
    __syncthreads();                                              // every thread has read the old scale
    if (threadIdx.x == 0) *sc = q8_pow2(e);
    encode_side(v.side(pid, h, i), stage, d, v.page, i != 0, lo, hi, e, e_old);
}

// [n][n_kv][2][d] fp32 of entries [0, n) of one sequence: one CTA per
// (16-token tile, head), a thread an element at a time (byte loads: for reading
// back and tests, no path of a forward).
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
constexpr int kSelBits = 11, kSelBins = 1 << kSelBits;
constexpr int kSelMaxCluster = 8;
constexpr int kSelSmemKeys = 48 * 1024;         // keys of a CTA's slice that shared memory holds
constexpr size_t kSelSmem = 3 * kSelBins * sizeof(unsigned);      // its histograms, one a pass

DKV_DEV uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
    return r;
}
DKV_DEV void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
DKV_DEV void cluster_arrive_all() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
DKV_DEV void cluster_wait_all() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
// Two words of the CTA `rank`'s shared memory at this CTA's address p
DKV_DEV uint2 dsmem_ld2(const void* p, uint32_t rank) {
    uint2 v;
    asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %2, %3;\n ld.shared::cluster.v2.u32 {%0, %1}, [a];\n}\n"
        : "=r"(v.x), "=r"(v.y)
        : "r"(smem_u32(p)), "r"(rank));
    return v;
}
DKV_DEV unsigned dsmem_ld(const void* p, uint32_t rank) {
    unsigned v;
    asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.u32 %0, [a];\n}\n"
                 : "=r"(v)
                 : "r"(smem_u32(p)), "r"(rank));
    return v;
}
DKV_DEV unsigned warp_scan(unsigned v) {      // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    return v;
}
// Inclusive sums over the block's threads in order (all 32 warps; a barrier inside).
DKV_DEV unsigned block_scan(unsigned v, unsigned* wsum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned run = warp_scan(v);
    if (lane == 31) wsum[warp] = run;
    __syncthreads();
    const unsigned w = wsum[lane], upto = warp_scan(w);
    return run + __shfl_sync(0xffffffffu, upto - w, warp);
}

// Which entries stay: per (sequence, head) the `drop` lowest (mass, index) of
// the unprotected entries go.  A cluster of CTAs takes a (sequence, head), each
// CTA a contiguous slice of the entries whose order-preserving keys it keeps in
// shared memory (slices that do not fit are read from global memory again).
// Radix select of the drop-th smallest key in three passes (11, 11, 10 bits):
// the CTAs' histograms are summed over the cluster through distributed shared
// memory, a part of the bins a CTA (every pass has a histogram of its own), and
// every CTA finds the same bin.  Plain shared-memory atomics: grouping a warp's
// equal bins first (match) took 200 cycles a warp, more than 32 atomics to one
// address.  The counts below and at the key give each slice its place, and an
// ordered pass over it (a warp a contiguous part) writes the kept indices: order
// and result are fixed.  Their masses and positions follow, spread over all
// threads (loaded where the indices are made, 256 entries took a warp 6700
// cycles).  One sequence of 262144 entries, 8 heads: 46 us before, 40 us so;
// what is left are the cluster barriers and scans of three passes, 9 us of them.
__global__ void __launch_bounds__(kSelThreads) q8_select_kernel(Q8EvictArgs a, int cluster, int smem_keys) {
    extern __shared__ __align__(16) unsigned sel_sm[];
    unsigned* keys_s = sel_sm + 3 * kSelBins;      // (histograms [3][kSelBins] first)
    __shared__ unsigned part_s[kSelThreads], wsum[32], wbelow[32], wcnt[64], s_bin, s_below, s_from, s_upto;
    __shared__ __align__(8) uint2 counts;
    const uint32_t rank = cluster > 1 ? cluster_rank() : 0u;
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int i = tid; i < 3 * kSelBins; i += kSelThreads) sel_sm[i] = 0u;
    pdl_wait();
    int n;
    const int keep = evict_keep(a, b, &n);
    if (rank == 0 && tid == 0 && (a.n[b] > a.v.capacity() || a.n[b] < 0 ||
                                  keep < min(n, max(a.budget[b], a.sink + a.recent))))
        atomicOr(a.err, kErrQ8Page);
    const size_t cap = a.v.capacity(), row = (size_t)b * a.v.n_kv + h;
    const float* mass = a.mass + row * cap;
    const int out_cap = a.out_pages << a.v.page_shift;
    const int f0 = min(a.sink, n), f1 = max(n - a.recent, f0);     // unprotected entries [f0, f1)
    const int drop = min(n - keep, f1 - f0);
    // this CTA's slice [i0, i1): a multiple of 32 entries a warp
    const int slice = ((n + cluster - 1) / cluster + kSelThreads - 1) / kSelThreads * kSelThreads;
    const int i0 = min((int)rank * slice, n), i1 = min(i0 + slice, n);
    const bool staged = slice <= smem_keys;
    // key of entry i, 0xffffffff for protected ones (which never go)
    auto key_of = [&](int i, float m) { return i >= f0 && i < f1 ? mass_key(m) : 0xffffffffu; };
    if (staged && drop > 0) {
        constexpr int U = 16;                      // loads in flight a thread
        for (int c0 = i0 + tid; c0 < i1; c0 += U * kSelThreads) {
            float m[U];
#pragma unroll
            for (int u = 0; u < U; ++u) m[u] = c0 + u * kSelThreads < i1 ? q8_ld(mass + c0 + u * kSelThreads) : 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c0 + u * kSelThreads < i1) keys_s[c0 + u * kSelThreads - i0] = key_of(c0 + u * kSelThreads, m[u]);
        }
    }
    int32_t* kept = a.kept + row * out_cap;
    {
        // behind the kept entries (early: these stores drain while the keys are searched)
        const int left = min(n - drop, out_cap), stride = kSelThreads * cluster;
        for (int i = left + (int)rank * kSelThreads + tid; i < out_cap; i += stride) kept[i] = -1;
        for (size_t i = left + (size_t)rank * kSelThreads + tid; i < cap; i += stride) {
            a.mass_out[row * cap + i] = 0.f;
            if (a.pos_out) a.pos_out[row * cap + i] = -1;
        }
    }
    auto key_at = [&](int i) { return staged ? keys_s[i - i0] : key_of(i, q8_ld(mass + i)); };
    __syncthreads();

    unsigned prefix = 0, need = (unsigned)drop, below = 0, equal = 0;      // below, equal: this slice's counts
    if (drop > 0) {
        for (int pass = 0; pass < 3; ++pass) {
            unsigned* hist = sel_sm + pass * kSelBins;
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : kSelBits;
            const unsigned mask = pass == 0 ? 0u : 0xffffffffu << (shift + bits);
            const int from = max(i0, f0), to = min(i1, f1);
#pragma unroll 8
            for (int i = from + tid; i < to; i += kSelThreads) {
                const unsigned key = key_at(i);
                if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1u)], 1u);
            }
            if (cluster > 1)
                cluster_sync_all();
            else
                __syncthreads();
            const uint2 own = *reinterpret_cast<const uint2*>(hist + 2 * tid);
            if (cluster == 1) {
                // thread i's bins 2 i and 2 i + 1, and the prefix sums over all
                const unsigned before = block_scan(own.x + own.y, wsum) - own.x - own.y;
                const unsigned e1 = before + own.x;                           // entries in bins below
                if (before < need && need <= e1) s_bin = 2 * tid, s_below = before;
                if (e1 < need && need <= e1 + own.y) s_bin = 2 * tid + 1, s_below = e1;
            } else {
                // a CTA sums a part of the bins over the cluster and scans it; every
                // CTA then finds the part that holds the bin, and the bin in it
                const int part = kSelBins / cluster;
                unsigned c = 0;
                if (tid < part) {
                    unsigned x[kSelMaxCluster];
#pragma unroll
                    for (int r = 0; r < kSelMaxCluster; ++r)
                        x[r] = r < cluster ? dsmem_ld(hist + (int)rank * part + tid, r) : 0u;
#pragma unroll
                    for (int r = 0; r < kSelMaxCluster; ++r) c += x[r];
                }
                const unsigned upto = block_scan(c, wsum);
                part_s[tid] = upto;
                cluster_sync_all();
                const unsigned tot = lane < cluster ? dsmem_ld(part_s + part - 1, lane) : 0u;
                const unsigned end = warp_scan(tot);
                const unsigned hit = __ballot_sync(0xffffffffu, end - tot < need && need <= end);
                const int owner = __ffs(hit) - 1;
                const unsigned start = __shfl_sync(0xffffffffu, end - tot, owner);
                if (tid < part) {
                    const unsigned hi = start + dsmem_ld(part_s + tid, owner);
                    const unsigned lo = tid ? start + dsmem_ld(part_s + tid - 1, owner) : start;
                    if (lo < need && need <= hi) s_bin = owner * part + tid, s_below = lo;
                }
            }
            __syncthreads();
            // this slice's entries in bins below the one found
            const unsigned bin = s_bin;
            unsigned mine = (2u * tid < bin ? own.x : 0u) + (2u * tid + 1u < bin ? own.y : 0u);
            prefix |= bin << shift;
            need -= s_below;
            equal = hist[bin];
            mine = (unsigned)warp_sum_i((int)mine);
            if (lane == 0) wbelow[warp] = mine;
            __syncthreads();
            below += (unsigned)warp_sum_i((int)wbelow[lane]);
        }
    }
    // entries that go before this slice: all below the key, and the first `need` equal ones
    unsigned gone_before = 0, eq_before = 0;
    if (cluster > 1) {
        if (tid == 0) counts = make_uint2(below, equal);
        cluster_sync_all();
        for (uint32_t r = 0; r < rank; ++r) {
            const uint2 c = dsmem_ld2(&counts, r);
            gone_before += c.x;
            eq_before += c.y;
        }
        gone_before += min(eq_before, need);
        cluster_arrive_all();                      // (waited for at the end: shared memory outlives its readers)
    }

    pdl_trigger();
    if (i0 < i1) {
        // A warp a contiguous part of the slice, 32 groups of 32 entries at a time:
        // lane g holds, as bits, which entries of group g lie below the key and at
        // it; from the counts of both come the part's place, the groups' places and
        // with them the kept indices
        const int part = slice / 32, p0 = min(i0 + warp * part, i1), p1 = min(p0 + part, i1);
        unsigned lt = 0, at = 0;
        auto look = [&](int c0) {
            lt = at = 0;
#pragma unroll 8
            for (int g = 0; g < 32; ++g) {
                const int i = c0 + 32 * g + lane;
                const bool open = drop > 0 && i < p1 && i >= f0 && i < f1;
                const unsigned k = open ? key_at(i) : 0xffffffffu;
                const unsigned l = __ballot_sync(0xffffffffu, open && k < prefix);
                const unsigned e = __ballot_sync(0xffffffffu, open && k == prefix);
                if (lane == g) lt = l, at = e;
            }
        };
        unsigned my_eq = 0, my_lt = 0;
        for (int c0 = p0; c0 < p1; c0 += 1024) {
            look(c0);
            my_eq += __popc(at);
            my_lt += __popc(lt);
        }
        my_eq = (unsigned)warp_sum_i((int)my_eq);
        my_lt = (unsigned)warp_sum_i((int)my_lt);
        if (lane == 0) wcnt[warp] = my_eq, wcnt[32 + warp] = my_lt;
        __syncthreads();
        const unsigned we = wcnt[lane], wl = wcnt[32 + lane];
        const unsigned se = warp_scan(we) - we, sl = warp_scan(wl) - wl;
        // equal entries before the part, and where its first kept entry goes
        unsigned eq = eq_before + __shfl_sync(0xffffffffu, se, warp);
        unsigned to = p0 - (gone_before + __shfl_sync(0xffffffffu, sl, warp) + (min(eq, need) - min(eq_before, need)));
        if (tid == 0) s_from = to;
        for (int c0 = p0; c0 < p1; c0 += 1024) {
            if (part > 1024) look(c0);             // (else the masks are the ones just made)
            const unsigned n_eq = __popc(at), eq_at = eq + warp_scan(n_eq) - n_eq;
            const unsigned go = min(need - min(need, eq_at), n_eq);
            unsigned gone = at;                    // of the equal ones the first `go` go
            for (unsigned k = n_eq; k > go; --k) gone &= ~(0x80000000u >> __clz(gone));
            const int there = min(max(p1 - (c0 + 32 * lane), 0), 32);
            const unsigned stay = (there == 32 ? 0xffffffffu : (1u << there) - 1u) & ~(lt | gone), n_stay = __popc(stay);
            const unsigned first = to + warp_scan(n_stay) - n_stay;
#pragma unroll 8
            for (int g = 0; g < 32; ++g) {
                const unsigned m = __shfl_sync(0xffffffffu, stay, g);
                const unsigned o = __shfl_sync(0xffffffffu, first, g) + __popc(m & ((1u << lane) - 1u));
                if (((m >> lane) & 1u) && o < (unsigned)out_cap) kept[o] = c0 + 32 * g + lane;
            }
            eq += (unsigned)warp_sum_i((int)n_eq);
            to += (unsigned)warp_sum_i((int)n_stay);
        }
        if (tid == kSelThreads - 1) s_upto = to;
        __syncthreads();                           // the slice's kept indices are written
        constexpr int U = 4;
        const int upto = min((int)s_upto, out_cap);
        for (int o0 = (int)s_from + tid; o0 < upto; o0 += U * kSelThreads) {
            int src[U];
            float m[U];
            int32_t p[U];
#pragma unroll
            for (int u = 0; u < U; ++u) src[u] = o0 + u * kSelThreads < upto ? q8_ld(kept + o0 + u * kSelThreads) : i0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                m[u] = q8_ld(mass + src[u]);
                p[u] = a.pos_out ? q8_ld(a.pos + row * cap + src[u]) : 0;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int o = o0 + u * kSelThreads;
                if (o >= upto) continue;
                a.mass_out[row * cap + o] = m[u];
                if (a.pos_out) a.pos_out[row * cap + o] = p[u];
            }
        }
    }
    if (cluster > 1) cluster_wait_all();
}

// The kept rows of one output page and head, K or V: a thread makes 16-byte
// fragments of the output.  A K fragment holds two rows (words 0, 2 and 1, 3), a
// V fragment a byte of four rows in each word; the sources are the fragments of
// those rows' tiles at the same dims, loaded whole and picked apart in
// registers.  The page's scale is the smallest that holds the values (as an
// append of them to an empty page gives), so the fragments wait in registers for
// the largest magnitude, and codes whose scale changes are rounded once.  What
// bounds it: the sectors the kept rows touch (half of a tile's K sectors for 4
// kept rows of 16, nearly all of V's, whose rows are the bytes of every word):
// 4 x 8 heads, 8192 of 32768 rows of d 128: 215 MB read and 45 MB written in 55 us;
// 8 heads, 32768 of 262144 rows: 350 MB and 54 MB in 74 us.
struct __align__(16) GatherRow {
    const uint4* at;      // its first fragment (null: bad page or not there)
    uint32_t pick;        // which byte (V, as a byte selector of two words) or word (K) of a fragment is its own
};

DKV_DEV __half2 as_h2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }
DKV_DEV uint32_t as_u32(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
// Largest magnitude of four codes (exact).
DKV_DEV float largest4(uint32_t w) {
    uint32_t lo, hi;
    q8_decode4(w, lo, hi);
    const __half2 m = __hmax2(__habs2(as_h2(lo)), __habs2(as_h2(hi)));
    return __half2float(__hmax(__low2half(m), __high2half(m)));
}
// 2^(e_src - e_dst) as two f16 factors (each twice): codes that are not zero fit
// below 2^18, and below 2^-28 every product rounds to zero.  What ends as a code
// other than zero (2^-10 and more) is exact after each factor.
DKV_DEV uint2 shift_of(int e_src, int e_dst) {
    const int d = min(max(e_src - e_dst, -28), 18), x = d / 2;
    return make_uint2(as_u32(__float2half2_rn(q8_pow2(x))), as_u32(__float2half2_rn(q8_pow2(d - x))));
}
// Four codes times such a factor, rounded to codes again.
DKV_DEV uint32_t times4(uint32_t w, uint2 f) {
    uint32_t lo, hi;
    q8_decode4(w, lo, hi);
    lo = as_u32(__hmul2(__hmul2(as_h2(lo), as_h2(f.x)), as_h2(f.y)));
    hi = as_u32(__hmul2(__hmul2(as_h2(hi), as_h2(f.x)), as_h2(f.y)));
    uint32_t r;
    asm("{\n .reg .b16 a, b;\n cvt.rn.satfinite.e4m3x2.f16x2 a, %1;\n cvt.rn.satfinite.e4m3x2.f16x2 b, %2;\n mov.b32 %0, {a, b};\n}\n"
        : "=r"(r)
        : "r"(lo), "r"(hi));
    return r;
}
// Bytes i of word q <-> bytes q of word i.
DKV_DEV void transpose4(uint32_t (&w)[4]) {
    const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);      // 0: w0.0 w1.0 w0.1 w1.1
    const uint32_t c = __byte_perm(w[0], w[1], 0x7362), d = __byte_perm(w[2], w[3], 0x7362);
    w[0] = __byte_perm(a, b, 0x5410);
    w[1] = __byte_perm(a, b, 0x7632);
    w[2] = __byte_perm(c, d, 0x5410);
    w[3] = __byte_perm(c, d, 0x7632);
}

// A CTA makes one side of a page, a thread a fragment (two or more for the
// largest pages).  Loads go out in three rounds: kept indices, page ids, then
// data and scales together (the largest magnitude needs the scales only at the
// end).
constexpr int gather_threads(int d, int tiles) { return d * tiles < 512 ? d * tiles : 512; }

template <int D, int TILES>              // tiles a page
__global__ void __launch_bounds__(gather_threads(D, TILES)) q8_gather_kernel(Q8EvictArgs a) {
    constexpr int NT = gather_threads(D, TILES), WS = NT / 32, NJ = D / 32, FR = TILES * NJ / WS;
    static_assert(NT >= TILES * 16, "a thread for every row");
    // per row: where its bytes are, its scale, the factors that bring its codes to
    // the new scale
    __shared__ GatherRow rows[TILES * 16];
    __shared__ uint2 factors[TILES * 16];
    __shared__ float scales[TILES * 16];
    __shared__ int emax;
    const Q8View& v = a.v;
    const int b = blockIdx.z >> 1, side = blockIdx.z & 1, h = blockIdx.y, pg = blockIdx.x, tid = threadIdx.x;
    const int wi = tid >> 5, lane = tid & 31;
    pdl_wait();
    const int src = tid < TILES * 16 ? a.kept[(((size_t)b * v.n_kv + h) * a.out_pages + pg) * v.page + tid] : -1;
    const int pid = q8_ld(a.out_table + (size_t)b * a.out_pages + pg);
    int n;
    const int keep = evict_keep(a, b, &n);
    const int cnt = min(keep - (pg << v.page_shift), v.page);
    if (cnt <= 0) return;
    if (!v.ok(pid)) {
        if (tid == 0) atomicOr(a.err, kErrQ8Page);
        return;
    }
    if (tid == 0) emax = kQ8ExpMin;
    int sp = -1;
    if (tid < TILES * 16) {
        GatherRow r{nullptr, 0x40u};
        if (tid < cnt) {
            if (src >= 0 && src < n) sp = q8_ld(v.row(b) + (src >> v.page_shift));
            if (v.ok(sp)) {
                const int k = src & 15;
                r.at = reinterpret_cast<const uint4*>(v.side(sp, h, side)) + ((src & (v.page - 1)) >> 4) * D +
                       (side ? (k & 7) >> 1 : (k & 7) * 4);
                r.pick = side ? 0x40u + 0x11u * (uint32_t)((k >> 3) * 2 + (k & 1)) : (uint32_t)(k >> 3);
            } else {
                sp = -1;
                atomicOr(a.err, kErrQ8Page);              // (its values count as zeros)
            }
        }
        rows[tid] = r;
    }
    __syncthreads();
    const int g = lane >> 2, t = lane & 3;
    auto row_of = [&](int tile, int i) {                  // K: rows g, g + 8; V: tokens 2t, 2t + 1, 2t + 8, 2t + 9
        return tile * 16 + (side ? 2 * t + (i & 1) + 8 * (i >> 1) : g + 8 * i);
    };
    float sc = 1.f;
    if (sp >= 0) sc = q8_ld(v.scale + v.scale_at(sp, h, side));
    // fragment x of this warp: block x * WS + wi of the side = tile block / NJ, dims
    // block block % NJ, as words of one row each (K: rows g, g + 8, g, g + 8; V: a
    // word a row, turned at the end)
    uint32_t w[FR][4];
#pragma unroll
    for (int x = 0; x < FR; ++x) {
        const int blk = x * WS + wi, tile = blk / NJ, j = blk % NJ;
#pragma unroll
        for (int q = 0; q < 4; ++q) w[x][q] = 0u;
        if (tile * 16 >= cnt) continue;
        if (side == 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const GatherRow r = rows[row_of(tile, i)];
                if (r.at == nullptr) continue;
                const uint4 s = q8_ld(r.at + j * 32 + t);
                w[x][i] = r.pick ? s.y : s.x;
                w[x][2 + i] = r.pick ? s.w : s.z;
            }
        } else {
            uint4 s[4];
            uint32_t pick[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const GatherRow r = rows[row_of(tile, i)];
                pick[i] = r.pick;
                s[i] = r.at == nullptr ? make_uint4(0u, 0u, 0u, 0u) : q8_ld(r.at + j * 32 + g * 4);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[x][i] = __byte_perm(__byte_perm(s[i].x, s[i].y, pick[i]), __byte_perm(s[i].z, s[i].w, pick[i]), 0x5410);
        }
    }
    int er = 0;
    if (tid < TILES * 16) {
        er = min(max(q8_scale_exp(sc), kQ8ExpMin), kQ8ExpMax);
        scales[tid] = q8_pow2(er);
    }
    __syncthreads();
    float amax = 0.f;
#pragma unroll
    for (int x = 0; x < FR; ++x) {
        const int tile = (x * WS + wi) / NJ;
        if (side == 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                amax = fmaxf(amax, fmaxf(largest4(w[x][i]), largest4(w[x][2 + i])) * scales[row_of(tile, i)]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) amax = fmaxf(amax, largest4(w[x][i]) * scales[row_of(tile, i)]);
        }
    }
    amax = warp_max(amax);
    if (lane == 0) atomicMax(&emax, q8_exp_of(amax));
    __syncthreads();
    const int e = emax;
    if (tid < TILES * 16) factors[tid] = shift_of(er, e);
    if (tid == 0) v.scale[v.scale_at(pid, h, side)] = q8_pow2(e);
    __syncthreads();
    pdl_trigger();
    uint8_t* out = v.side(pid, h, side);
#pragma unroll
    for (int x = 0; x < FR; ++x) {
        const int blk = x * WS + wi, tile = blk / NJ;
        if (tile * 16 >= cnt) continue;
        uint4* at = reinterpret_cast<uint4*>(out + (size_t)blk * 512 + lane * 16);
        if (side == 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint2 f = factors[row_of(tile, i)];
                w[x][i] = times4(w[x][i], f), w[x][2 + i] = times4(w[x][2 + i], f);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[x][i] = times4(w[x][i], factors[row_of(tile, i)]);
        }
        if (tile * 16 + 16 > cnt) {                       // rows that are not there keep their bytes
            const uint4 was = *at;
            uint32_t old[4] = {was.x, was.y, was.z, was.w};
            if (side) transpose4(old);
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (row_of(tile, side ? q : q & 1) >= cnt) w[x][q] = old[q];
        }
        if (side) transpose4(w[x]);
        *at = make_uint4(w[x][0], w[x][1], w[x][2], w[x][3]);
    }
}

// CTAs a (sequence, head)'s selection is spread over: one wave of the GPU's SMs,
// each CTA with 2048 entries at least, and its keys in shared memory.
int select_cluster(int batch, int n_kv, int capacity) {
    int c = 1;
    while (c < kSelMaxCluster && ((capacity / (2 * c) >= 2048 && (long long)batch * n_kv * 2 * c <= 148) ||
                                  capacity / c > kSelSmemKeys))
        c *= 2;
    return c;
}

template <int D, int TILES>
cudaError_t launch_gather(const Q8EvictArgs& a, int batch, cudaStream_t st) {
    const dim3 grid((unsigned)a.out_pages, (unsigned)a.v.n_kv, (unsigned)batch * 2);
    return launch_pdl(q8_gather_kernel<D, TILES>, grid, dim3((unsigned)gather_threads(D, TILES)), 0, st, a);
}
template <int D>
cudaError_t launch_gather_page(const Q8EvictArgs& a, int batch, cudaStream_t st) {
    switch (a.v.page) {
        case 16: return launch_gather<D, 1>(a, batch, st);
        case 32: return launch_gather<D, 2>(a, batch, st);
        case 64: return launch_gather<D, 4>(a, batch, st);
        default: return launch_gather<D, 8>(a, batch, st);
    }
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
    const int cap = a.v.capacity(), cl = select_cluster(dims.batch, dims.n_kv, cap);
    const int per = ((cap + cl - 1) / cl + kSelThreads - 1) / kSelThreads * kSelThreads;
    const int smem_keys = per <= kSelSmemKeys ? per : 0;
    DKV_CUDA(allow_smem_max_once<q8_select_kernel>());
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)cl, (unsigned)dims.n_kv, (unsigned)dims.batch);
    cfg.blockDim = dim3(kSelThreads);
    cfg.dynamicSmemBytes = kSelSmem + (size_t)smem_keys * sizeof(unsigned);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cl;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    DKV_CUDA(cudaLaunchKernelEx(&cfg, q8_select_kernel, a, cl, smem_keys));
    DKV_CUDA(dims.d == 128 ? launch_gather_page<128>(a, dims.batch, st) : launch_gather_page<64>(a, dims.batch, st));
    return DKV_OK;
}
