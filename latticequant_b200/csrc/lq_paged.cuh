// lq_paged.cuh -- the paged E8 cache: pool layout and the block decode shared
// by its kernels.
//
// A pool layer is two arrays over pages of P tokens (P a power of two in
// 16..256):
//   codes   u32  [n_pages][2][n_heads][P][D/8]   (index 0 of the pair: K, 1: V)
//   scales  fp32 [n_pages][2][n_heads][P]
// A code word holds one block of 8 channels as the 4-bit compact code
// (core/compact_storage.py:87-222), read as a big-endian integer:
//   bit 31 coset | 27..30 u0 | 23..26 u1 | ... | 3..6 u6 | 0..2 u7 >> 1
// with u = floor coordinate + 8 and u7's low bit the parity of u0..u6; the
// channel's value is (u - 8 + coset/2) * scale.  Every word is a valid point,
// so a page's unwritten rows decode to finite values.
#pragma once

#include "lq_attn_common.cuh"

namespace lq {

// The word of a block of zeros (u = 8 throughout).  A vector of them has scale 1.
constexpr uint32_t kZeroWord = 0x44444444u;

__host__ __device__ constexpr bool paged_page_ok(int p) { return p >= 16 && p <= 256 && (p & (p - 1)) == 0; }
__host__ __device__ constexpr bool paged_dim_ok(int d) { return d == 64 || d == 128; }

// ---- block decode -----------------------------------------------------------
// A word's eight 4-bit fields become four fp16 pairs by one logic op and one
// exact fp16 op each: a field lands in the mantissa of 1024, either at bits
// 1-4 (value 1024 + 2u + coset, then -1040) or at bits 5-8 (1024 + 32u + 16
// coset, then /16 - 80), so that one right shift serves both pairs of half
// the word.  Every pair comes out as 2 * (u - 8) + coset, exact.  What bounds
// the kernels is the integer ALU pipe; left shifts, the coset's constants and
// the top bit are written as multiplications, which run on the FMA pipe.
constexpr float kCodeUnit = 0.5f;  // what one unit of the decoded pairs stands for

constexpr uint32_t kField1 = 0x001e001eu, kField5 = 0x01e001e0u;  // fields at bits 1-4 and 5-8 of each half

__device__ __forceinline__ uint32_t pair_at1(uint32_t x, uint32_t magic) {
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"((x & kField1) | magic), "r"(0xe410e410u));  // - (1024 + 16)
    return r;
}
__device__ __forceinline__ uint32_t pair_at5(uint32_t x, uint32_t magic) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;"
        : "=r"(r)
        : "r"((x & kField5) | magic), "r"(0x2c002c00u), "r"(0xd500d500u));  // * 1/16 - (64 + 16)
    return r;
}

// The low bit of u7, shifted out of the word: the parity of u0..u6.
__device__ __forceinline__ uint32_t odd_sum(uint32_t v) { return (uint32_t)__popc(v & 0x08888888u); }  // bit 0

// The pairs of one block: pair s holds channels 7 - s (low half) and 3 - s.
__device__ __forceinline__ void decode_block(uint32_t v, uint32_t (&pair)[4]) {
    const uint32_t a = ((odd_sum(v) * 2u) & 2u) | (v * 4u);  // u7, u6 | u3, u2 at bits 1-8 of the halves
    const uint32_t b = v >> 6;                               // u5, u4 | u1, u0
    const uint32_t half = __umulhi(v, 2u);                   // the coset
    const uint32_t m1 = half * 0x00010001u + 0x64006400u, m5 = half * 0x00100010u + 0x64006400u;
    pair[0] = pair_at1(a, m1);
    pair[1] = pair_at5(a, m5);
    pair[2] = pair_at1(b, m1);
    pair[3] = pair_at5(b, m5);
}

// The pairs of one block of two tokens: low[s] holds channel 7 - s of token x
// (low half) and of token y, high[s] channel 3 - s of both.
struct TokenPair {
    uint32_t la, lb, ha, hb, m1, m5;
};
__device__ __forceinline__ TokenPair pair_tokens(uint32_t x, uint32_t y) {
    const uint32_t tx = x * 2u, ty = y * 2u;
    const uint32_t l = __byte_perm(tx, ty, 0x5410), h = __byte_perm(tx, ty, 0x7632);
    const uint32_t odd = odd_sum(y) * 0x20000u + odd_sum(x) * 2u;
    const uint32_t half = __umulhi(y, 2u) * 0x10000u + __umulhi(x, 2u);
    TokenPair p;
    p.la = (odd & 0x00020002u) | (l * 2u);
    p.lb = l >> 7;
    p.ha = h * 2u;
    p.hb = h >> 7;
    p.m1 = half + 0x64006400u;
    p.m5 = half * 16u + 0x64006400u;
    return p;
}
template <int S>
__device__ __forceinline__ void decode_pair(const TokenPair &p, uint32_t &low, uint32_t &high) {
    if constexpr (S == 0) {
        low = pair_at1(p.la, p.m1);
        high = pair_at1(p.ha, p.m1);
    } else if constexpr (S == 1) {
        low = pair_at5(p.la, p.m5);
        high = pair_at5(p.ha, p.m5);
    } else if constexpr (S == 2) {
        low = pair_at1(p.lb, p.m1);
        high = pair_at1(p.hb, p.m1);
    } else {
        low = pair_at5(p.lb, p.m5);
        high = pair_at5(p.hb, p.m5);
    }
}

}  // namespace lq
