// Prompt attention over the 8-bit paged cache on the fifth-generation tensor
// cores: more than 64 query rows (token x GQA head) a KV head.
//
// Flash attention as in the bf16 prefill kernel (two 128-row query tiles a CTA
// alternate on the tensor core; Q and K in shared memory, S, P and O in tensor
// memory), with the cache's codes turned into f16 operands on the way:
//   warps 8-11 -- converters: a 128-key tile's codes come from global memory
//     straight into registers, one tile ahead (16-byte fragments, 512 B a warp
//     and load), are widened e4m3 -> f16 (exact) and stored with 16-byte stores
//     in the swizzled K-major layout the MMA reads.  2 x 32 KB K and V rings;
//   warp 12 -- tensor memory, and lane 0 issues the MMAs: per key tile j and
//     query tile t, O_t += P_t(j-1) V(j-1), then S_t(j) = Q_t K_j^T;
//   warps 0-3 / 4-7 -- softmax of query tiles A / B, one row a thread.
// The order of a contraction is free, so both operands of each product take the
// order in which a lane's bytes lie: dims are permuted alike in Q and K, keys
// alike in S, P and V (qp_key: a tile's column c belongs to the 16-token group
// (c >> 6) * 4 + ((c >> 2) & 3)).
// Block scales never touch the operands: K's multiplies the fp32 score, V's is added
// to the exponent of the probability that enters the product (over the largest of
// the key tiles so far, to which O is brought when it grows; in a row's last tiles
// over the largest that the row itself sees, so that no row's precision depends on
// keys it does not see), and divided out of the row sum again.  Weights of blocks
// more than 2^40 below that are zeros in f16 whatever they are.
// Rounding, bf16 outputs: queries are one f16 number each (2^-11 of the row's
// largest), probabilities too, biased by 2^6 so that f16 keeps 2^-30 of the max;
// max, sum and O are fp32.  fp32 outputs (WIDE): both are two f16 numbers, as in
// calls of up to 64 rows; products double, and one query tile a CTA does not
// overlap with another (512 tokens over 2 x 8192 entries 420 us).
// Bound by the softmax warps: a key tile takes 4100 cycles at d = 128, of which
// the tensor cores work half and the exp2 units half (each 2050 for both query
// tiles), and a CTA 12000 more for its start and its end.  512 tokens of 2
// sequences of up to 8192 entries, 8 heads, group 4: 161 us (98.7 GFLOP, 58 us at
// the measured matrix rate; the shorter sequence's SMs idle at the end); 4096
// tokens from the start: 184 us.
// Every mbarrier wait is bounded (error word 0x80).
#include <algorithm>
#include <type_traits>

#include "attention_q8.cuh"
#include "prefill_common.cuh"

namespace dkv {

namespace {

constexpr int kQpTile = 128, kQpKeys = 128;
// Query rows a CTA: two tiles, or one whose queries' lower parts take the second's place
constexpr int qp_rows(bool wide) { return wide ? kQpTile : 2 * kQpTile; }
constexpr int kQpSoft = 256, kQpConv = 128;
constexpr int kQpThreads = kQpSoft + kQpConv + 32;
constexpr int kQpNst = 2;               // K and V ring depth
constexpr int kQpTmemCols = 512;        // per query tile t: S at 256 t (P over it), O at 256 t + 128
constexpr int kQpSplit = 16384;         // most keys a split has (page ids staged in shared memory)
constexpr int kQpMinSplit = 512;
constexpr float kQpLazy = 8.f;
constexpr int kQpBias = 6;
constexpr int kQpDown = -40;            // V block exponents below the largest that probabilities carry

// Element i (0..7) of a row's 16-byte unit u (of the d / 8) is dim
// 32 (2 (u >> 3) + (u & 1)) + 16 (i >> 2) + 8 ((i >> 1) & 1) + 2 ((u & 7) >> 1) + (i & 1):
// what lane t = (u & 7) >> 1 of a fragment of that 32-dim block holds.
// Key (0..127) of a tile's column c: 16-byte unit 2 t + pair of a 64-key half,
// 4 tokens of each of the pair's groups.
__host__ __device__ constexpr int qp_key(int c) {
    return (c >> 6) * 64 + ((c >> 3) & 1) * 32 + ((c >> 2) & 1) * 16 + ((c >> 1) & 1) * 8 + 2 * ((c >> 4) & 3) + (c & 1);
}

template <int D>
struct QpGeo {
    static constexpr int CH = D / 64;
    static constexpr int QT = CH * 16384;        // one query tile
    static constexpr int KVB = kQpKeys * D * 2;  // one K (or V) tile
    static constexpr int K0 = 2 * QT, V0 = K0 + kQpNst * KVB;
    static constexpr size_t SMEM = (size_t)V0 + kQpNst * KVB + 1024;
};

// kind::f16 instruction descriptor: f16 A and B, f32 D, K-major both, M 128.
__host__ __device__ constexpr uint32_t qp_idesc(int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

DKV_DEV uint32_t h2(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
// What h = h2(lo, hi) leaves of its numbers.
DKV_DEV uint32_t h2_rest(float lo, float hi, uint32_t h) {
    const float2 x = __half22float2(*reinterpret_cast<__half2*>(&h));
    return h2(lo - x.x, hi - x.y);
}
DKV_DEV uint32_t pack_bf2(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
// V exponent of a group below a row's unit, as probabilities carry it (all whole
// numbers; a group that the row does not see may lie above: its probabilities are 0).
DKV_DEV float qp_below(float ev, float unit) { return fmaxf(fminf(ev, unit) - unit, (float)kQpDown); }

// A score's factor: the row's times the K scale, and not zero (a row of zeros against
// a block of zeros), which would make NaN of the -infinity of what is not seen.
DKV_DEV float qp_factor(float row, float kscale) { return fmaxf(row * kscale, 1.175494351e-38f); }

// The second softmax pass (below) a group at a time, under the row's own unit: tiles
// in which a row of the warp sees less than what the tile's V exponents are counted
// from, and WIDE's, whose probabilities' lower parts go 256 columns further.  A call
// of its own, since the loop around it fills the instruction cache (inlined but not
// taken, it cost 512 tokens over 8192 entries 6 us of 161 at d 128, 14 of 141 at d 64).
// Returns the tile's row sum.
template <bool WIDE>
__device__ __noinline__ float qp_weigh_groups(uint32_t sb, const float* kf, const float* ev, float c, float off, float unit) {
    float l = 0.f;
#pragma unroll 1
    for (int cc = 0; cc < 4; ++cc) {
        uint32_t x[32], pk[16], lo[16];
        tmem_ld32(sb + 32 * cc, x);
        tmem_wait_ld();
#pragma unroll
        for (int gi = 0; gi < 4; ++gi) {
            const int g = (cc >> 1) * 4 + gi;
            const float below = qp_below(ev[g], unit), f = qp_factor(c, kf[g]);
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
                if (((e >> 2) & 3) != gi) continue;
                const float p0 = pf_ex2(fmaf(__uint_as_float(x[e]), f, off + below));
                const float p1 = pf_ex2(fmaf(__uint_as_float(x[e + 1]), f, off + below));
                sum += p0 + p1;
                pk[e / 2] = h2(p0, p1);
                if (WIDE) lo[e / 2] = h2_rest(p0, p1, pk[e / 2]);
            }
            l += sum * q8_pow2(-(int)below);
        }
        tmem_st16(sb + 16 * cc, pk);
        if (WIDE) tmem_st16(sb + 256 + 16 * cc, lo);
    }
    return l;
}

// WIDE (fp32 outputs): queries and probabilities are two f16 numbers each; the CTA
// has one query tile, the lower parts take the other's shared and tensor memory.
template <int D, bool WIDE>
__global__ void __launch_bounds__(kQpThreads, 1) q8_prefill_kernel(const __grid_constant__ Q8AttnArgs a) {
    using Geo = QpGeo<D>;
    constexpr int PS = D + 4, ROWS = qp_rows(WIDE), TILES = ROWS / kQpTile;
    extern __shared__ uint8_t qp_raw[];
    uint8_t* sm = qp_raw + ((1024u - (smem_u32(qp_raw) & 1023u)) & 1023u);
    __shared__ __align__(8) uint64_t k_full[kQpNst], k_empty[kQpNst], v_full[kQpNst], v_empty[kQpNst];
    __shared__ __align__(8) uint64_t s_full[2], p_full[2], o_done, drain;
    __shared__ uint32_t tmem_slot;
    __shared__ int32_t page_s[kQpSplit / 16];
    // per 16-key group: K scale, V exponent, that below the largest of the tiles so far, 2^-that
    __shared__ __align__(16) float kf_s[kQpSplit / 16], ev_s[kQpSplit / 16], dv_s[kQpSplit / 16], iv_s[kQpSplit / 16];
    __shared__ float top_s[kQpSplit / kQpKeys];                      // largest V exponent of the tiles so far
    __shared__ uint32_t bad_s[kQpSplit / kQpKeys / 4];               // 8 bits a key tile: 16-key groups not to be seen

    const Q8View& v = a.v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // a sequence's last row blocks, which see the most keys, start first, all
    // heads together (a prompt of 4096 tokens, 8 KV heads, group 4: 298 us with
    // the row blocks in order, head by head, 255 us so); sequence by sequence, for
    // long and short ones side by side in the last wave
    const int h = (int)(blockIdx.x % v.n_kv);
    const int s = (int)(blockIdx.x / v.n_kv % a.n_splits);
    const int rb = a.n_rb - 1 - (int)(blockIdx.x / v.n_kv / a.n_splits % a.n_rb);
    const int b = (int)(blockIdx.x / v.n_kv / a.n_splits / a.n_rb);
    const int G = a.group;
    const int r0 = rb * ROWS, R = min(ROWS, a.T * G - r0);
    const size_t bhr = ((size_t)b * v.n_kv + h) * a.n_rb + rb;
    const bool alone = a.n_splits == 1;

    pdl_wait();
    const int e0 = a.first(b);
    const int n_tok = a.n_rows ? min(a.n_rows[b], a.T) : a.T;
    const int t_last = min((r0 + R - 1) / G, n_tok - 1);
    const int n_keys = t_last >= r0 / G ? max(0, min(a.n_keys(b), e0 + t_last + 1)) : 0;
    const int k0 = s * a.split;                               // a multiple of 128
    const int kend = min(n_keys, k0 + a.split);
    const int ntiles = kend > k0 ? (kend - k0 + kQpKeys - 1) / kQpKeys : 0;
    if (s == 0 && h == 0 && rb == 0 && threadIdx.x == 0 && a.beyond(b)) atomicOr(a.err, kErrQ8Page);
    if (ntiles == 0) {
        if (alone) {
            for (int i = threadIdx.x; i < R * (D / 2); i += kQpThreads)
                q8_store2<D>(a, b, h, r0 + i / (D / 2), n_tok, i % (D / 2) * 2, 0.f, 0.f);
            return;
        }
        for (int r = threadIdx.x; r < R; r += kQpThreads)
            *reinterpret_cast<float2*>(a.part + ((bhr * a.n_splits + s) * ROWS + r) * PS) = make_float2(-INFINITY, 0.f);
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < kQpNst; ++i) {
            mbar_init(&k_full[i], kQpConv);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], kQpConv);
            mbar_init(&v_empty[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t], 128);
        }
        mbar_init(&o_done, 1);
        mbar_init(&drain, 1);
        fence_barrier_init();
        fence_async_shared();
    }
    for (int i = threadIdx.x; i < (ntiles + 3) / 4; i += kQpThreads) bad_s[i] = 0u;
    if (warp == 12) tmem_alloc(&tmem_slot, kQpTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    // Converters and the MMA warp, while the others load Q: per 16-key group of the
    // key range, page id and scales (all of a thread's loads in two rounds); keys of
    // a bad page are not seen.  The MMA warp meets the softmax warps after this.
    if (warp >= 8) {
        constexpr int NS = kQpThreads - kQpSoft, PER = (kQpSplit / 16 + NS - 1) / NS;
        const int first = threadIdx.x - kQpSoft, n_grp = (kend - k0 + 15) / 16;
        int pid[PER];
        float2 sc[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int i = first + k * NS;
            pid[k] = i < n_grp ? q8_ld(v.row(b) + ((k0 + i * 16) >> v.page_shift)) : -1;
        }
#pragma unroll
        for (int k = 0; k < PER; ++k)
            sc[k] = v.ok(pid[k]) ? q8_ld(reinterpret_cast<const float2*>(v.scale + v.scale_at(pid[k], h, 0))) : make_float2(1.f, 1.f);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int i = first + k * NS;
            if (i >= ntiles * 8) break;
            const bool there = v.ok(pid[k]);
            const int ev = there ? min(max(q8_scale_exp(sc[k].y), kQ8ExpMin), kQ8ExpMax) : kQ8ExpMin;
            if (!there && i < n_grp) {
                atomicOr(a.err, kErrQ8Page);
                atomicOr(&bad_s[i >> 5], 1u << (i & 31));
            }
            page_s[i] = there ? pid[k] : -1;
            kf_s[i] = sc[k].x;
            ev_s[i] = (float)ev;
        }
        named_sync(2, NS);
        if (warp == 8) {
            constexpr int PL = kQpSplit / kQpKeys / 32;           // tiles a lane, in order
            float top[PL], run = (float)kQ8ExpMin;
#pragma unroll
            for (int k = 0; k < PL; ++k) {
                const int j = lane * PL + k;
                for (int i = 0; i < 8 && j < ntiles; ++i) run = fmaxf(run, ev_s[j * 8 + i]);
                top[k] = run;
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const float y = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run = fmaxf(run, y);
            }
            float before = __shfl_up_sync(0xffffffffu, run, 1);
            if (lane == 0) before = (float)kQ8ExpMin;
#pragma unroll
            for (int k = 0; k < PL; ++k)
                if (lane * PL + k < ntiles) top_s[lane * PL + k] = fmaxf(top[k], before);
        }
        named_sync(2, NS);
        for (int i = first; i < ntiles * 8; i += NS) {
            const float dv = qp_below(ev_s[i], top_s[i >> 3]);
            dv_s[i] = dv;
            iv_s[i] = q8_pow2(-(int)dv);
        }
        named_sync(2, NS);
    }

    bool ok = true;
    if (warp >= 8 && warp < 12) {
        // ---------------- converters: warp w takes groups 2 w and 2 w + 1 of a tile
        constexpr int NJ = D / 32;                                // 512-byte blocks a group and side
        const int w = warp - 8, g = lane >> 2, t = lane & 3;
        uint4 kr[2][NJ], vr[2][NJ];
        auto load = [&](int j, int i, uint4 (&r)[2][NJ]) {
#pragma unroll
            for (int gb = 0; gb < 2; ++gb) {
                const int grp = j * 8 + 2 * w + gb;               // from k0
                const int pid = j < ntiles ? page_s[grp] : -1;
                const uint8_t* at = v.side(max(pid, 0), h, i) + (size_t)((k0 + grp * 16) & (v.page - 1)) * D + lane * 16;
#pragma unroll
                for (int x = 0; x < NJ; ++x)
                    r[gb][x] = pid >= 0 ? q8_ld(reinterpret_cast<const uint4*>(at + x * 512)) : make_uint4(0u, 0u, 0u, 0u);
            }
        };
        // row of key g (+8: row + 2) of group 2 w + gb, see qp_key; unit 2 t + (x & 1) of the 64-dim half x >> 1
        auto put_k = [&](uint8_t* dst) {
#pragma unroll
            for (int gb = 0; gb < 2; ++gb) {
                const int row = (w >> 1) * 64 + (2 * (g >> 1) + (w & 1)) * 8 + gb * 4 + (g & 1);
#pragma unroll
                for (int x = 0; x < NJ; ++x) {
                    const uint4 f = kr[gb][x];
                    uint4 a0, a1;
                    q8_decode4(f.x, a0.x, a0.y);
                    q8_decode4(f.z, a0.z, a0.w);
                    q8_decode4(f.y, a1.x, a1.y);
                    q8_decode4(f.w, a1.z, a1.w);
                    uint8_t* at = dst + (x >> 1) * 16384 + row * 128;
                    const int unit = 2 * t + (x & 1);
                    *reinterpret_cast<uint4*>(at + ((unit ^ (row & 7)) << 4)) = a0;
                    *reinterpret_cast<uint4*>(at + 256 + ((unit ^ ((row + 2) & 7)) << 4)) = a1;
                }
            }
        };
        // V: rows are dims 32 x + 8 q' + g; unit 2 t + (w & 1) of key half w >> 1 holds 4 tokens of each group
        auto put_v = [&](int j, uint8_t* dst) {
            // rare: bytes of tokens that are not there become zeros (their weight is
            // 0, but 0 x NaN would not be)
#pragma unroll
            for (int gb = 0; gb < 2; ++gb) {
                const int left = kend - k0 - (j * 8 + 2 * w + gb) * 16;
                if (left < 16) {
                    const uint32_t vm = (2 * t < left ? 0xffu : 0u) | (2 * t + 1 < left ? 0xff00u : 0u) |
                                        (2 * t + 8 < left ? 0xff0000u : 0u) | (2 * t + 9 < left ? 0xff000000u : 0u);
#pragma unroll
                    for (int x = 0; x < NJ; ++x) {
                        uint4& r = vr[gb][x];
                        r.x &= vm, r.y &= vm, r.z &= vm, r.w &= vm;
                    }
                }
            }
            auto word = [&](const uint4& r, int q) { return q == 0 ? r.x : q == 1 ? r.y : q == 2 ? r.z : r.w; };
#pragma unroll
            for (int x = 0; x < NJ; ++x)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint4 o;
                    q8_decode4(word(vr[0][x], q), o.x, o.y);
                    q8_decode4(word(vr[1][x], q), o.z, o.w);
                    const int row = x * 32 + (q >> 1) * 16 + (q & 1) * 8 + g, unit = 2 * t + (w & 1);
                    *reinterpret_cast<uint4*>(dst + (w >> 1) * (D * 128) + row * 128 + ((unit ^ (row & 7)) << 4)) = o;
                }
        };
        load(0, 0, kr);
        load(0, 1, vr);
        for (int j = 0; j < ntiles; ++j) {
            const int slot = j % kQpNst;
            const uint32_t ph = (uint32_t)((j / kQpNst - 1) & 1);
            // the slot's K was read by S_A(j-2), S_B(j-2); its V by the P V products of tile j - 2
            if (j >= kQpNst && !__all_sync(0xffffffffu, mbar_wait(&k_empty[slot], ph, a.err))) {
                ok = false;
                break;
            }
            put_k(sm + Geo::K0 + slot * Geo::KVB);
            fence_async_shared();
            mbar_arrive(&k_full[slot]);
            load(j + 1, 0, kr);
            if (j >= kQpNst && !__all_sync(0xffffffffu, mbar_wait(&v_empty[slot], ph, a.err))) {
                ok = false;
                break;
            }
            put_v(j, sm + Geo::V0 + slot * Geo::KVB);
            fence_async_shared();
            mbar_arrive(&v_full[slot]);
            load(j + 1, 1, vr);
        }
    } else if (warp == 12) {
        // ---------------- MMA issuer (the warp waits together, lane 0 issues)
        const uint32_t q_s = smem_u32(sm), k_s0 = smem_u32(sm + Geo::K0), v_s0 = smem_u32(sm + Geo::V0);
        constexpr uint32_t idS = qp_idesc(kQpKeys), idO = qp_idesc(D);
        auto wait_all = [&](uint64_t* bar, uint32_t parity) {
            return __all_sync(0xffffffffu, mbar_wait(bar, parity, a.err));
        };
        auto issue_pv = [&](int t, int i) {
            const uint32_t v_s = v_s0 + (i % kQpNst) * Geo::KVB;
            const uint32_t base = tmem + (uint32_t)(t * 256);
#pragma unroll
            for (int ks = 0; ks < kQpKeys / 16; ++ks)
                tc_mma_ts(base + 128, base + ks * 8, sw128_desc(v_s + (ks >> 2) * (D * 128) + (ks & 3) * 32), idO,
                          (i | ks) != 0 ? 1u : 0u);
            if (WIDE) {
#pragma unroll
                for (int ks = 0; ks < kQpKeys / 16; ++ks)
                    tc_mma_ts(base + 128, base + 256 + ks * 8, sw128_desc(v_s + (ks >> 2) * (D * 128) + (ks & 3) * 32), idO, 1u);
            }
        };
        auto issue_s = [&](int t, int j) {
            const uint32_t k_s = k_s0 + (j % kQpNst) * Geo::KVB;
            const uint32_t qt = q_s + t * Geo::QT;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
                tc_mma_i(tmem + (uint32_t)(t * 256), sw128_desc(qt + (kk >> 2) * 16384 + (kk & 3) * 32),
                         sw128_desc(k_s + (kk >> 2) * 16384 + (kk & 3) * 32), idS, kk != 0 ? 1u : 0u);
            if (WIDE) {
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    tc_mma_i(tmem, sw128_desc(q_s + Geo::QT + (kk >> 2) * 16384 + (kk & 3) * 32),
                             sw128_desc(k_s + (kk >> 2) * 16384 + (kk & 3) * 32), idS, 1u);
            }
            tc_commit(&s_full[t]);
        };
        named_sync(1, kQpSoft + 32);      // Q is in shared memory, and the softmax warps may read the scales
        for (int j = 0; j < ntiles && ok; ++j) {
            if (!wait_all(&k_full[j % kQpNst], (uint32_t)((j / kQpNst) & 1)) ||
                (j >= 1 && !wait_all(&v_full[(j - 1) % kQpNst], (uint32_t)(((j - 1) / kQpNst) & 1)))) {
                ok = false;
                break;
            }
            for (int t = 0; t < TILES; ++t) {
                if (j >= 1 && !wait_all(&p_full[t], (uint32_t)((j - 1) & 1))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (lane == 0) {
                    if (j >= 1) issue_pv(t, j - 1);
                    issue_s(t, j);
                }
                __syncwarp();
            }
            if (!ok) break;
            if (lane == 0) {
                tc_commit(&k_empty[j % kQpNst]);
                if (j >= 1) tc_commit(&v_empty[(j - 1) % kQpNst]);
            }
            __syncwarp();
        }
        if (ok) {
            const int i = ntiles - 1;
            ok = wait_all(&v_full[i % kQpNst], (uint32_t)((i / kQpNst) & 1));
            for (int t = 0; t < TILES && ok; ++t) {
                if (!wait_all(&p_full[t], (uint32_t)(i & 1))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (lane == 0) issue_pv(t, i);
                __syncwarp();
            }
            if (ok && lane == 0) tc_commit(&o_done);
            __syncwarp();
        }
    } else {
        // ---------------- softmax: row rt of query tile t = TMEM lane rt; CTA row cr.
        // (WIDE: tile 0 alone; warps 4-7 load the queries' lower parts and are done)
        const int half = warp >> 2, t = WIDE ? 0 : half, rt = threadIdx.x & 127, cr = t * kQpTile + rt, gr = r0 + cr;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t sb = lanes + (uint32_t)(t * 256), ob = sb + 128;
        const bool mine = cr < R && gr / G < n_tok;
        float c = 1.f;                                            // scores = S * c * (K scale), log2 units
        {
            // the warp's 32 rows of Q as f16 of q * log2 e / sqrt(d) * 2^-x, x the
            // row's exponent.  8 lanes a row: of each 64-dim half a lane makes one
            // 16-byte unit, li, from the four pairs it consists of.  The loads of 16
            // rows go out together
            constexpr int B = 4, CH = Geo::CH;                    // 4-row steps a round, 64-dim halves
            const int li = lane & 7, from = 32 * (li & 1) + 2 * (li >> 1);
            uint8_t* qt = sm + half * Geo::QT;
#pragma unroll 1
            for (int i0 = 0; i0 < 8; i0 += B) {
                float2 x[B][CH][4];
#pragma unroll
                for (int k = 0; k < B; ++k) {
                    const int row = (warp & 3) * 32 + (i0 + k) * 4 + (lane >> 3), qr = r0 + t * kQpTile + row;
                    const bool there = t * kQpTile + row < R && qr / G < n_tok;
                    const float* at = a.q + (((size_t)b * a.T + qr / G) * v.n_kv * G + h * G + qr % G) * D + from;
#pragma unroll
                    for (int ch = 0; ch < CH; ++ch)
#pragma unroll
                        for (int p = 0; p < 4; ++p)
                            x[k][ch][p] = there ? q8_ld(reinterpret_cast<const float2*>(at + ch * 64 + p * 8)) : make_float2(0.f, 0.f);
                }
#pragma unroll
                for (int k = 0; k < B; ++k) {
                    const int row = (warp & 3) * 32 + (i0 + k) * 4 + (lane >> 3);
                    float am = 0.f;
#pragma unroll
                    for (int ch = 0; ch < CH; ++ch)
#pragma unroll
                        for (int p = 0; p < 4; ++p) am = pf_max3(am, fabsf(x[k][ch][p].x), fabsf(x[k][ch][p].y));
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, o));
                    const int ex = min(max((int)(__float_as_uint(am * a.scale) >> 23) - 127, -126), 126);
                    const float f = a.scale * q8_pow2(-ex);
                    const int mx = __shfl_sync(0xffffffffu, ex, (lane & 3) * 8);
                    if ((lane >> 2) == i0 + k) c = q8_pow2(mx);   // (this thread's own row)
#pragma unroll
                    for (int ch = 0; ch < CH; ++ch) {
                        uint32_t u[4];
#pragma unroll
                        for (int p = 0; p < 4; ++p) {
                            const float y0 = x[k][ch][p].x * f, y1 = x[k][ch][p].y * f;
                            u[p] = h2(y0, y1);
                            if (WIDE && half) u[p] = h2_rest(y0, y1, u[p]);
                        }
                        *reinterpret_cast<uint4*>(qt + ch * 16384 + row * 128 + ((li ^ (row & 7)) << 4)) =
                            make_uint4(u[0], u[1], u[2], u[3]);
                    }
                }
            }
            fence_async_shared();
            named_sync(1, kQpSoft + 32);
        }
        // this row's last key; rows that are not there see every key
        const int lim = mine ? min(e0 + gr / G, kend - 1) : kend - 1;
        float m = -INFINITY, l = 0.f, unit = (float)kQ8ExpMin;
        auto factor = [&](float kscale) { return qp_factor(c, kscale); };
        const bool idle = WIDE && half;
        for (int j = 0; j < ntiles && !idle; ++j) {
            if (!__all_sync(0xffffffffu, mbar_wait(&s_full[t], (uint32_t)(j & 1), a.err))) {
                ok = false;
                break;
            }
            tc_fence_after();
            const int lc = lim - (k0 + j * kQpKeys);              // last live column
            const uint32_t bad = (bad_s[j >> 2] >> ((j & 3) * 8)) & 0xffu;
            float to = top_s[j];                                  // O's unit with this tile
            bool apart = false;                                   // a row has a smaller one
            if (__any_sync(0xffffffffu, lc < kQpKeys - 1 || bad != 0u)) {
                // a row's last tiles, or a bad page: -infinity over what is not seen
                // (kept out of the loops below: their code has to stay small)
#pragma unroll 1
                for (int cc = 0; cc < 4; ++cc) {
                    uint32_t x[32];
                    tmem_ld32(sb + 32 * cc, x);
                    tmem_wait_ld();
                    const int last = lc - (cc >> 1) * 64 - (cc & 1) * 4;      // qp_key(32 cc + e) = qp_key(e) + that
                    const uint32_t groups = bad >> ((cc >> 1) * 4);
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (qp_key(e) > last || ((groups >> ((e >> 2) & 3)) & 1u)) x[e] = __float_as_uint(-INFINITY);
                    tmem_st32(sb + 32 * cc, x);
                }
                tmem_wait_st();
                to = unit;                                        // the groups this row sees count
#pragma unroll 1
                for (int i = 0; i < 8; ++i)
                    if (16 * i <= lc) to = fmaxf(to, ev_s[j * 8 + i]);
                apart = __any_sync(0xffffffffu, to != top_s[j]) != 0;
            }
            // pass 1: the largest score, group by group (one factor a group)
            float mn = -INFINITY;
            const float4* kf = reinterpret_cast<const float4*>(kf_s + j * 8);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float mx[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) mx[k] = -INFINITY;
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                    uint32_t sr[32];
                    tmem_ld32(sb + half * 64 + cc * 32, sr);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const int k = 2 * ((e >> 2) & 3) + ((e >> 1) & 1);
                        mx[k] = pf_max3(mx[k], __uint_as_float(sr[e]), __uint_as_float(sr[e + 1]));
                    }
                }
                const float4 f = kf[half];
                mn = pf_max3(mn, fmaxf(mx[0], mx[1]) * factor(f.x), fmaxf(mx[2], mx[3]) * factor(f.y));
                mn = pf_max3(mn, fmaxf(mx[4], mx[5]) * factor(f.z), fmaxf(mx[6], mx[7]) * factor(f.w));
            }
            float alpha = 1.f;
            if (mn > m + kQpLazy) {
                alpha = pf_ex2(m - mn);                           // 0 from -infinity
                m = mn;
            }
            float shrink = alpha;                                 // O's factor: in units of 2^(unit - bias)
            if (to > unit) {
                shrink *= q8_pow2((int)fmaxf(unit - to, -126.f));
                unit = to;
            }
            if (j >= 1 && __any_sync(0xffffffffu, shrink != 1.f)) {
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 32) {
                    uint32_t o[32];
                    tmem_ld32(ob + c0, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink);
                    tmem_st32(ob + c0, o);
                }
            }
            // pass 2: probabilities 2^(s - m + bias + dv), as f16 pairs into columns read before
            const float off = m == -INFINITY ? 0.f : (float)kQpBias - m;
            l *= alpha;
            if (WIDE || apart) {
                l += qp_weigh_groups<WIDE>(sb, kf_s + j * 8, ev_s + j * 8, c, off, unit);
            } else {
                uint32_t sr[2][32];
#pragma unroll 1
                for (int k = 0; k < 2; ++k) {
                    tmem_ld32(sb + 64 * k, sr[0]);
                    tmem_ld32(sb + 64 * k + 32, sr[1]);
                    const float4 f = kf[k];
                    const float4 dv = *reinterpret_cast<const float4*>(dv_s + j * 8 + 4 * k);
                    const float4 iv = *reinterpret_cast<const float4*>(iv_s + j * 8 + 4 * k);
                    uint64_t cg[4], og[4], sum2[4] = {0ull, 0ull, 0ull, 0ull};
                    const float fx = factor(f.x), fy = factor(f.y), fz = factor(f.z), fw = factor(f.w);
                    cg[0] = pf_pack2(fx, fx), cg[1] = pf_pack2(fy, fy), cg[2] = pf_pack2(fz, fz), cg[3] = pf_pack2(fw, fw);
                    og[0] = pf_pack2(off + dv.x, off + dv.x), og[1] = pf_pack2(off + dv.y, off + dv.y);
                    og[2] = pf_pack2(off + dv.z, off + dv.z), og[3] = pf_pack2(off + dv.w, off + dv.w);
                    tmem_wait_ld();
                    uint32_t pk[32];
#pragma unroll
                    for (int h3 = 0; h3 < 2; ++h3) {
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const int gi = (e >> 2) & 3;
                            float d0, d1;
                            pf_unpack2(pf_fma2(pf_pack2(__uint_as_float(sr[h3][e]), __uint_as_float(sr[h3][e + 1])), cg[gi], og[gi]),
                                       d0, d1);
                            const float p0 = pf_ex2(d0), p1 = pf_ex2(d1);
                            sum2[gi] = pf_add2(sum2[gi], pf_pack2(p0, p1));
                            pk[h3 * 16 + e / 2] = h2(p0, p1);
                        }
                    }
                    tmem_st32(sb + 32 * k, pk);
                    const float ivs[4] = {iv.x, iv.y, iv.z, iv.w};
#pragma unroll
                    for (int gi = 0; gi < 4; ++gi) {
                        float a0, a1;
                        pf_unpack2(sum2[gi], a0, a1);
                        l += (a0 + a1) * ivs[gi];
                    }
                }
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&p_full[t]);
        }
        if (ok && !idle) {
            ok = __all_sync(0xffffffffu, mbar_wait(&o_done, 0u, a.err));
            tc_fence_after();
        }
        // ---- the row's output (one split) or its partial (max, sum, O over the sum)
        float* mypart = alone ? nullptr : a.part + ((bhr * a.n_splits + s) * ROWS + cr) * PS;
        if (l != l && m == -INFINITY) m = 0.f;     // NaN scores have no max: give the row one, so that its NaN comes out
        const bool live = ok && m != -INFINITY;
        // O is in units of 2^(unit - bias), l in units of 2^-bias.  (Apart from the
        // sum: 2^unit / l may be too small for fp32 where their result is not.)
        const float un = q8_pow2((int)unit);
        const float f = live ? 1.f / l : 1.f;
        const size_t out_at = (((size_t)b * a.T + gr / G) * v.n_kv * G + h * G + gr % G) * D;
        if (__all_sync(0xffffffffu, ok) && !idle) {
            // through the drained K and V rings (a part of each warp's own), so that
            // whole rows are stored: a lane's 16-byte chunk ch of row r at ch ^ r
            const bool wide = WIDE || !alone;
            uint8_t* stg = sm + Geo::K0 + warp * (32 * D * 4);
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
                uint32_t o[32];
                tmem_ld32(ob + c0, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = live ? __float_as_uint(__uint_as_float(o[e]) * f * un) : 0u;
                if (wide) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<uint4*>(stg + lane * D * 4 + ((((c0 + e) / 4) ^ (lane & (D / 4 - 1))) << 4)) =
                            make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                } else {
                    auto bf2 = [&](int e) { return pack_bf2(__uint_as_float(o[e]), __uint_as_float(o[e + 1])); };
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        *reinterpret_cast<uint4*>(stg + lane * D * 2 + ((((c0 + e) / 8) ^ (lane & (D / 8 - 1))) << 4)) =
                            make_uint4(bf2(e), bf2(e + 2), bf2(e + 4), bf2(e + 6));
                }
            }
            __syncwarp();
            const unsigned rows = __ballot_sync(0xffffffffu, mine);
            auto copy_rows = [&](auto lanes_a_row, auto dest) {
                constexpr int LP = decltype(lanes_a_row)::value;      // 16-byte chunks a row
                const int ch = lane % LP;
#pragma unroll 4
                for (int i = 0; i < LP; ++i) {
                    const int r = i * (32 / LP) + lane / LP;
                    const size_t at = __shfl_sync(0xffffffffu, out_at, r);
                    if ((rows >> r) & 1u)
                        *reinterpret_cast<uint4*>(dest(r, at) + ch * 16) =
                            *reinterpret_cast<const uint4*>(stg + r * LP * 16 + ((ch ^ (r & (LP - 1))) << 4));
                }
            };
            if (!alone)
                copy_rows(std::integral_constant<int, D / 4>{}, [&](int r, size_t) { return reinterpret_cast<uint8_t*>(mypart + (r - lane) * PS + 4); });
            else if (wide)
                copy_rows(std::integral_constant<int, D / 4>{}, [&](int, size_t at) { return reinterpret_cast<uint8_t*>(a.out) + at * 4; });
            else
                copy_rows(std::integral_constant<int, D / 8>{}, [&](int, size_t at) { return reinterpret_cast<uint8_t*>(a.out) + at * 2; });
        }
        if (!alone && cr < R && !idle)
            *reinterpret_cast<float2*>(mypart) = make_float2(live ? m : -INFINITY, live ? l * q8_pow2(-kQpBias) : 0.f);
    }

    pdl_trigger();
    const bool all_ok = __syncthreads_and(ok) != 0;
    if (!all_ok && warp == 12 && lane == 0) {
        // a wait ran out: the MMAs still in flight end before the memory is let go
        tc_commit(&drain);
        mbar_wait(&drain, 0u, nullptr);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, kQpTmemCols);
    }
}

// The splits' partial rows merged into outputs, D / 4 threads a row (a launch of
// its own: 256 rows of a block, by the CTA that ends last, took 35 to 60 us).
constexpr int kQpMergeThreads = 256;
template <int D, int BLOCK>              // rows a block of the partials
__global__ void __launch_bounds__(kQpMergeThreads) q8_prefill_merge_kernel(Q8AttnArgs a) {
    constexpr int PS = D + 4, ROWS = kQpMergeThreads * 4 / D;          // rows a CTA
    pdl_wait();
    const int h = blockIdx.y, b = blockIdx.z, row0 = blockIdx.x * ROWS, rb = row0 / BLOCK, r0 = rb * BLOCK;
    const int n_tok = a.n_rows ? min(a.n_rows[b], a.T) : a.T;
    const size_t bhr = ((size_t)b * a.v.n_kv + h) * a.n_rb + rb;
    q8_merge_items<D, BLOCK, 4, 1, 8>(a, a.part + bhr * a.n_splits * (size_t)BLOCK * PS, b, h, r0,
                                      min(BLOCK, a.T * a.group - r0), n_tok, (row0 - r0) * (D / 4) + threadIdx.x, 0);
}

// Keys per split: the whole capacity up to 16384 keys; where the row blocks
// alone leave SMs idle, as many splits of at least 512 keys as fill them (333 rows
// of 2 heads over 4 x 2565 entries: 53 us at 2048, 44 at 1024, 38 at 512).
int prefill_split(dkv_dims dims, int n_rb, int capacity) {
    const long long ctas = (long long)dims.batch * dims.n_kv * n_rb;
    const int most = std::max(1, (capacity + kQpMinSplit - 1) / kQpMinSplit);
    const int want = std::max((capacity + kQpSplit - 1) / kQpSplit, (int)std::min<long long>(most, std::max(1ll, 148 / ctas)));
    const int keys = (capacity + want - 1) / want;
    return std::min((keys + kQpKeys - 1) / kQpKeys * kQpKeys, kQpSplit);
}

size_t prefill_layout(dkv_dims dims, int group, int T, int capacity, bool wide, Q8AttnArgs* a, Arena* ar) {
    const int R = T * group, rows = qp_rows(wide), n_rb = (R + rows - 1) / rows;
    const int split = prefill_split(dims, n_rb, capacity), ns = std::max(1, (capacity + split - 1) / split);
    const size_t part = ns == 1 ? 0 : (size_t)dims.batch * dims.n_kv * n_rb * ns * rows * (dims.d + 4);
    if (a) {
        a->split = split;
        a->n_splits = ns;
        a->n_rb = n_rb;
        ar->take<unsigned>(kQ8Tickets);                    // (zero for other calls over the same buffer)
        a->part = ar->take<float>(part);
    }
    return kQ8Tickets * sizeof(unsigned) + align_up(part * sizeof(float), 256) + 1024;
}

template <int D, bool WIDE>
int launch_prefill(const Q8AttnArgs& a, dkv_dims dims, cudaStream_t st) {
    const size_t ctas = (size_t)dims.batch * dims.n_kv * a.n_rb * a.n_splits;
    DKV_REQUIRE(ctas <= 0x7fffffffu, "dkv_q8_attn: batch x heads x row blocks too large");
    constexpr auto kernel = q8_prefill_kernel<D, WIDE>;
    DKV_CUDA(allow_smem_max_once<kernel>());
    DKV_CUDA(launch_pdl(kernel, dim3((unsigned)ctas), dim3(kQpThreads), QpGeo<D>::SMEM, st, a));
    if (a.n_splits > 1) {
        constexpr int rows = kQpMergeThreads * 4 / D;
        const dim3 mg((unsigned)((a.T * a.group + rows - 1) / rows), (unsigned)dims.n_kv, (unsigned)dims.batch);
        constexpr auto merge = q8_prefill_merge_kernel<D, qp_rows(WIDE)>;
        DKV_CUDA(launch_pdl(merge, mg, dim3(kQpMergeThreads), 0, st, a));
    }
    return DKV_OK;
}

}  // namespace

// (for either type of outputs)
size_t attn_q8_prefill_work(dkv_dims dims, int group, int T, int capacity) {
    return std::max(prefill_layout(dims, group, T, capacity, false, nullptr, nullptr),
                    prefill_layout(dims, group, T, capacity, true, nullptr, nullptr));
}

int attn_q8_prefill(Q8AttnArgs& a, dkv_dims dims, void* work, size_t work_bytes, cudaStream_t st) {
    const bool wide = a.out_dtype == DKV_F32;
    Arena ar(work, work_bytes);
    prefill_layout(dims, a.group, a.T, a.v.capacity(), wide, &a, &ar);
    DKV_REQUIRE(a.part, "dkv_q8_attn: work buffer");
    ProfScope ps(DKV_PROF_ATTN_FULL, 0.0, st);
    if (dims.d == 128) return wide ? launch_prefill<128, true>(a, dims, st) : launch_prefill<128, false>(a, dims, st);
    return wide ? launch_prefill<64, true>(a, dims, st) : launch_prefill<64, false>(a, dims, st);
}

}  // namespace dkv
