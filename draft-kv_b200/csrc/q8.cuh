// The 8-bit paged KV cache shared by its kernels (append, read, evict,
// attention): the storage view, the byte order of a page, and e4m3 helpers.
//
// A page of one KV head holds `page` tokens as e4m3 codes, K then V, and one
// power-of-two scale for each: value = code * scale.  Codes of 16 tokens form
// a tile of 16 * d bytes in the operand order of the m16n8k16 tensor-core
// product, so that a warp fetches an operand with one 16-byte load a lane: a
// tile is d / 32 blocks of 512 bytes, lane 4 g + t owns 16 bytes of a block,
// and its 32-bit word w holds columns 2t, 2t+1, 2t+8, 2t+9 of operand row
// g + 8 (w & 1).  K: rows are tokens, columns are dims 32 j + 16 (w >> 1) + c.
// V: rows are dims 32 j + 16 (w >> 1) + g + 8 (w & 1), columns are tokens.
//
// These kernels call pdl_trigger() in their last part, not first: while CTAs of
// a grid of several waves are still to come, the next kernel's early ones would
// take their SMs and wait there (60 verify rows with the mass over 11 x 5 heads of
// 3857 entries: 294 us triggering first, 172 so).
#pragma once

#include "common.cuh"

namespace dkv {

uint32_t* device_error_word();

constexpr uint32_t kErrQ8Page = 0x400u;       // page id or entry outside the cache
constexpr uint32_t kErrQ8NonFinite = 0x800u;  // infinity or NaN written to the cache

// Exponents a scale may take: 2^-e and 2^e stay normal fp32 numbers, and
// 448 * 2^119 < FLT_MAX (values above it, the top 1/8 of the last binade, are
// stored as 448 * 2^119; values below 2^-130 as zero).
constexpr int kQ8ExpMin = -120, kQ8ExpMax = 119;

struct Q8View {
    uint8_t* codes;             // [n_pages][n_kv][2][page * d]
    float* scale;               // [n_pages][n_kv][2]
    const int32_t* table;       // [batch][n_layers][max_pages]
    int n_pages, page, page_shift, max_pages;
    int n_layers, n_kv, d, layer;

    DKV_DEV const int32_t* row(int b) const { return table + ((size_t)b * n_layers + layer) * max_pages; }
    DKV_DEV bool ok(int pid) const { return (unsigned)pid < (unsigned)n_pages; }
    // K (i = 0) or V (i = 1) codes of one head in one page
    DKV_DEV uint8_t* side(int pid, int h, int i) const {
        return codes + (((size_t)pid * n_kv + h) * 2 + i) * ((size_t)page * d);
    }
    DKV_DEV size_t scale_at(int pid, int h, int i) const { return ((size_t)pid * n_kv + h) * 2 + i; }
    __host__ __device__ int capacity() const { return max_pages * page; }
};

// 2^e for e in [-126, 127]
DKV_DEV float q8_pow2(int e) { return __int_as_float((e + 127) << 23); }

// Exponent of a power-of-two scale.
DKV_DEV int q8_scale_exp(float s) { return (int)((__float_as_uint(s) >> 23) & 0xffu) - 127; }

// Smallest e with amax * 2^-e <= 448 (448 = 1.75 * 2^8), clamped; amax finite, >= 0.
DKV_DEV int q8_exp_of(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int k = (int)(u >> 23) - 127;                     // amax = 1.m * 2^k (k = -127: zero or subnormal)
    const int e = k - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, kQ8ExpMin), kQ8ExpMax);
}

// Loads of what an earlier kernel of the stream may write.  Not the read-only
// path: this kernel's start and the earlier one's end overlap (pdl_wait), so
// the memory is not read-only while it runs, and a load must not pass the wait.
DKV_DEV uint4 q8_ld(const uint4* p) {
    uint4 x;
    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(p));
    return x;
}
DKV_DEV float4 q8_ld(const float4* p) {
    float4 x;
    asm volatile("ld.global.v4.f32 {%0,%1,%2,%3}, [%4];\n" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "l"(p));
    return x;
}
DKV_DEV float2 q8_ld(const float2* p) {
    float2 x;
    asm volatile("ld.global.v2.f32 {%0,%1}, [%2];\n" : "=f"(x.x), "=f"(x.y) : "l"(p));
    return x;
}
DKV_DEV float q8_ld(const float* p) {
    float x;
    asm volatile("ld.global.f32 %0, [%1];\n" : "=f"(x) : "l"(p));
    return x;
}
DKV_DEV int32_t q8_ld(const int32_t* p) {
    int32_t x;
    asm volatile("ld.global.s32 %0, [%1];\n" : "=r"(x) : "l"(p));
    return x;
}

// Two fp32 values to two e4m3 codes (low byte = a), nearest even, saturating.
DKV_DEV uint32_t q8_encode2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
DKV_DEV uint8_t q8_encode(float a) { return (uint8_t)(q8_encode2(a, 0.f) & 0xffu); }

// Four e4m3 codes of a word as two f16 pairs (exact): bytes 0, 1 and 2, 3.
DKV_DEV void q8_decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}\n"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}
// One code as fp32.
DKV_DEV float q8_decode(uint32_t byte) {
    uint32_t lo, hi;
    q8_decode4(byte & 0xffu, lo, hi);
    return half_bits_to_f32((uint16_t)(lo & 0xffffu));
}

// Byte of element (token, dim) inside a page's K / V side.
DKV_DEV int q8_k_byte(int d, int tok, int x) {
    const int k = tok & 15, c = x & 15;
    return (tok >> 4) * 16 * d + (x >> 5) * 512 + ((k & 7) * 4 + ((c & 7) >> 1)) * 16 + (((x >> 4) & 1) * 2 + (k >> 3)) * 4 +
           (c >> 3) * 2 + (c & 1);
}
DKV_DEV int q8_v_byte(int d, int tok, int x) {
    const int k = tok & 15, c = x & 15;
    return (tok >> 4) * 16 * d + (x >> 5) * 512 + ((c & 7) * 4 + ((k & 7) >> 1)) * 16 + (((x >> 4) & 1) * 2 + (c >> 3)) * 4 +
           (k >> 3) * 2 + (k & 1);
}

// Host: checks a cache descriptor and builds the kernels' view of one layer.
int q8_view(const char* who, const dkv_q8_cache* c, dkv_dims dims, int layer, Q8View* out);

}  // namespace dkv
