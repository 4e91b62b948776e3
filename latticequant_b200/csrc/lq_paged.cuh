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

__host__ __device__ constexpr bool paged_page_ok(int p) { return p >= 16 && p <= 256 && (p & (p - 1)) == 0; }
__host__ __device__ constexpr bool paged_dim_ok(int d) { return d == 64 || d == 128; }

// A code word ready for extraction: nibble 7 - i of `w` is u_i, `magic` the
// floating-point constant that carries the coset's half.
struct CodeWord {
    uint32_t w, magic;
};

// `w` regains u7's low bit: with the coset bit shifted out, the parity of
// u0..u6 is the population of their low bits (bits 4, 8, .. 28).
template <bool BF16>
__device__ __forceinline__ CodeWord code_word(uint32_t v) {
    CodeWord c;
    const uint32_t t = v << 1;
    c.w = t | (__popc(t & 0x11111110u) & 1);
    const uint32_t half = v >> 31;
    // fp16: 1024 + 16 u + 8 coset (unit 1 in the mantissa); bf16: 128 + 2 u + coset
    c.magic = BF16 ? half * 0x00010001u + 0x43004300u : half * 0x00080008u + 0x64006400u;
    return c;
}

// Channels (7 - S, 3 - S) of the block as a packed pair, in units of 1/16
// (fp16) or 1/2 (bf16): one shift, one three-input logic op and one exact
// subtraction for two channels.
template <bool BF16, int S>
__device__ __forceinline__ uint32_t code_pair(const CodeWord &c) {
    if constexpr (BF16) {
        const uint32_t x = S == 0 ? c.w << 1 : c.w >> (4 * S - 1);
        const uint32_t y = (x & 0x001e001eu) | c.magic;
        const uint32_t off = 0xc310c310u;  // -(128 + 16)
        uint32_t r;
        asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(y), "r"(off));
        return r;
    } else {
        const uint32_t x = S == 0 ? c.w << 4 : S == 1 ? c.w : c.w >> (4 * S - 4);
        const uint32_t y = (x & 0x00f000f0u) | c.magic;
        const uint32_t off = 0xe480e480u;  // -(1024 + 128)
        uint32_t r;
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(y), "r"(off));
        return r;
    }
}

template <bool BF16>
constexpr float kCodeUnit = BF16 ? 0.5f : 0.0625f;  // what one unit of code_pair's values stands for

}  // namespace lq
