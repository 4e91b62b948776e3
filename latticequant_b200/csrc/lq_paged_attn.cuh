// lq_paged_attn.cuh -- arguments and epilogue shared by the attention kernels
// over the paged E8 cache.
#pragma once

#include "lq_paged.cuh"

namespace lq {

struct PagedAttnArgs {
    const void *q;  // 16-bit elements, last dimension contiguous
    int64_t q_stride_b, q_stride_h, q_stride_t;
    const uint32_t *codes;
    const float *scales;
    int64_t n_pages;
    uint32_t page_log2;
    const int32_t *table;  // [batch][table_width], rows table_stride apart
    int64_t table_width, table_stride;
    const int32_t *lens;
    int64_t bound;        // tokens that a row of the table holds
    const uint8_t *mask;  // [batch or 1][T][T], or NULL: drafts <= t
    int64_t mask_stride_b;
    uint32_t n_heads, group, T, rows;  // rows = T * group, row = t * group + g
    FastDiv by_group;
    int64_t chunk;  // tokens of a split
    uint32_t splits;
    bool clustered;  // the splits of a row are a cluster and join in its shared memory
    float qk_log2;  // sm_scale * log2(e)
    void *out;      // [batch][n_heads * group][T][D] in q's type
    float *lse;     // [batch][n_heads * group][T] natural log, may be NULL
    float *part;    // [batch][n_heads][splits] of paged_part
    uint32_t *err;
};

// The reference M of the base-2 weights 2^(x - M): "none yet", how far an x
// may exceed it (fp16 holds 2^15), and how far below a maximum it is put: the
// 2^4 keep weights down to 2^-18 of the largest out of fp16's subnormals, and
// the 2^11 left let the maximum grow before M has to move again.
constexpr float kNoRef = -1e30f, kRefSlack = 15.f, kRefBelow = 4.f;

// A V vector of zeros is stored with scale 1, and where it holds most of the
// weight that scale would move M so far up that the others' weights leave
// fp16's range.  Its product with the point is zero whatever the scale is, so
// one that is about to move M counts as 2^-60 instead.
constexpr float kZeroLog2 = -60.f, kZeroInv = 0x1p60f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ int64_t paged_len(const PagedAttnArgs &a, uint32_t b) {
    return min(max((int64_t)a.lens[b], (int64_t)0), a.bound);
}

// Where this CTA's split of the tokens ends: the last one takes what lies beyond the length that was planned for.
__device__ __forceinline__ int paged_split_end(const PagedAttnArgs &a, int first, int len) {
    const int end = first + (int)a.chunk;
    return end < len && blockIdx.x + 1 < a.splits ? end : len;
}

// Whether position t of sequence b sees draft j.
__device__ __forceinline__ bool paged_sees(const PagedAttnArgs &a, uint32_t b, uint32_t t, int64_t j) {
    return a.mask ? a.mask[b * a.mask_stride_b + (int64_t)t * a.T + j] != 0 : j <= (int64_t)t;
}

// Partial results of one (sequence, head, split): o [rows][D], then [rows] of
// (reference, denominator), in rows * (D + 4) floats so that rows stay 16-byte aligned.
template <int D>
__device__ __forceinline__ float *paged_part(const PagedAttnArgs &a, uint32_t bh, uint32_t split) {
    return a.part + ((int64_t)bh * a.splits + split) * a.rows * (D + 4);
}

// Row r from its weighted sums (a warp: D / 32 channels a lane), denominator and reference.
template <bool BF16, int D>
__device__ __forceinline__ void paged_store_row(const PagedAttnArgs &a, uint32_t b, uint32_t h, uint32_t r,
                                                const float (&o)[D / 32], float l, float m) {
    const uint32_t lane = threadIdx.x & 31, t = a.by_group.div(r), qh = h * a.group + (r - t * a.group);
    const int64_t row = ((int64_t)b * a.n_heads * a.group + qh) * a.T + t;
    // a row that sees nothing has l = 0 (a NaN denominator stays NaN)
    const float inv = l == 0.f ? 0.f : kCodeUnit / l;
    uint32_t w[D / 64];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        if constexpr (BF16) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(o[2 * i] * inv, o[2 * i + 1] * inv);
            w[i] = *reinterpret_cast<const uint32_t *>(&p);
        } else {
            const __half2 p = __floats2half2_rn(o[2 * i] * inv, o[2 * i + 1] * inv);
            w[i] = *reinterpret_cast<const uint32_t *>(&p);
        }
    }
    uint32_t *out = static_cast<uint32_t *>(a.out) + (row * D + lane * (D / 32)) / 2;
    if constexpr (D == 128) *reinterpret_cast<uint2 *>(out) = make_uint2(w[0], w[1]);
    else *out = w[0];
    if (a.lse && lane == 0) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// paged_store_row, or the split's partial result.
template <bool BF16, int D>
__device__ __forceinline__ void paged_emit_row(const PagedAttnArgs &a, uint32_t b, uint32_t h, uint32_t r, uint32_t split,
                                               const float (&o)[D / 32], float l, float m) {
    if (a.splits == 1) {
        paged_store_row<BF16, D>(a, b, h, r, o, l, m);
        return;
    }
    const uint32_t lane = threadIdx.x & 31;
    float *p = paged_part<D>(a, b * a.n_heads + h, split), *po = p + (int64_t)r * D + lane * (D / 32);
    if constexpr (D == 128) *reinterpret_cast<float4 *>(po) = make_float4(o[0], o[1], o[2], o[3]);
    else *reinterpret_cast<float2 *>(po) = make_float2(o[0], o[1]);
    if (lane == 0) *reinterpret_cast<float2 *>(p + (int64_t)a.rows * D + 2 * r) = make_float2(m, l);
}

// A bf16 pair times the power of two f, as an fp16 pair.
__device__ __forceinline__ uint32_t bf16_to_f16(uint32_t x, float f) {
    const __half2 h = __floats2half2_rn(__uint_as_float(x << 16) * f, __uint_as_float(x & 0xffff0000u) * f);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// The tensor-core kernel for many rows (lq_paged_attn_tc.cu): `tile` rows a
// CTA, 16, 32 or 64; a.chunk a multiple of 128.
int launch_paged_tc(const PagedAttnArgs &a, bool bf16, int head_dim, int tile, uint32_t batch, cudaStream_t st);

}  // namespace lq
