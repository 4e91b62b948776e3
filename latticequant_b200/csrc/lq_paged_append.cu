// lq_paged_append.cu -- quantising new tokens into the pages of an E8 cache.
//
// The chunk codecs give a head the rate's scale and let an entropy coder (or
// fallback rows) take the points that fall out of range
// (llm/compressed_kv_cache.py:176-204).  A page has no room for either, so a
// token's K or V vector of one head gets the smallest scale that keeps its
// points in the 4-bit range:
//   s = amax / (7 - 1/64)        (1 where amax < 1e-6, the point is then 0)
//   q = nearest E8 point of x / s
// With |x / s| < 7 both D8 searches stay in [-8, 7]: rounding gives at most
// +-7 (the half coset -8..6), and a parity flip moves towards x, so it never
// leaves the range on the side where |x| is largest.  The lattice search is
// the framework's own (e8_nearest_symbols), bit for bit the torch form.
//
// One thread per block of 8 channels: a token-head is 8 or 16 neighbouring
// lanes, its amax a shuffle maximum.  What bounds it is instruction issue, most
// of it the search (480 instructions a thread, 76% of issue slots): 16,411
// tokens of 4 heads of 128 in fp16 with their values returned take 35 us, 2.2
// TB/s.
#include "lq_paged.cuh"

namespace lq {
namespace {

constexpr float kInvBound = 1.0f / (7.0f - 1.0f / 64.0f);

struct AppendArgs {
    const void *x[2];  // K, V
    int64_t stride_n[2], stride_h[2];
    void *out[2];  // dequantised [n][n_heads][D] in the input's dtype, or NULL
    const int64_t *slots;
    uint32_t *codes;
    float *scales;
    uint32_t *err;
    uint32_t n_vec, n_heads, page_log2;
    int64_t n_slots;
    FastDiv by_heads;
};

template <int DT, int D>
__global__ void __launch_bounds__(256) paged_append_kernel(AppendArgs a) {
    constexpr int BPT = D / 8;
    const uint32_t i = blockIdx.x * (256 / BPT) + threadIdx.x / BPT;  // token-head
    const uint32_t b = threadIdx.x % BPT;
    const int side = blockIdx.y;
    const bool live = i < a.n_vec;
    const uint32_t n = live ? a.by_heads.div(i) : 0, h = live ? i - n * a.n_heads : 0;
    float v[8];
    load_block8<DT>(static_cast<const typename Elem<DT>::T *>(a.x[side]) + n * a.stride_n[side] + h * a.stride_h[side],
                    b, v);
    const int64_t slot = __ldg(a.slots + n);

    float amax = 0.f;
    bool finite = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        amax = fmaxf(amax, fabsf(v[j]));
        finite = finite && isfinite(v[j]);
    }
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t group = (BPT == 32 ? 0xffffffffu : ((1u << BPT) - 1)) << (lane & ~(BPT - 1));
    finite = (__ballot_sync(0xffffffffu, !finite) & group) == 0;
#pragma unroll
    for (int o = BPT / 2; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (!live) return;

    // a vector with a NaN or an infinity is stored as zeros and reported
    const bool zero = !finite || amax < 1e-6f;
    const float s = zero ? 1.0f : __fmul_rn(amax, kInvBound);
    uint32_t word = kZeroWord;  // u = 8 in bits 27..30, 23..26, .., u7 >> 1 = 4
    float q[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (!zero) {
        float y[8];
        div_block_by_scale<false>(v, s, __frcp_rn(s), scale_ok_for_fast_div(s), y);
        int sym[8];
        bool ok;
        const int coset = e8_nearest_symbols<true>(y, q, sym, &ok);
        word = (uint32_t)coset << 31;
#pragma unroll
        for (int j = 0; j < 7; ++j) word |= (uint32_t)(sym[j] + 8) << (27 - 4 * j);
        word |= (uint32_t)(sym[7] + 4);
    } else if (!finite && b == 0) {
        raise_flag(a.err, LQ_EF_NONFINITE);
    }
    if (a.out[side]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = __fmul_rn(q[j], s);
        store_block8<DT>(a.out[side], (int64_t)i * BPT + b, q);
    }
    if (slot < 0) return;
    if (slot >= a.n_slots) {
        if (b == 0) raise_flag(a.err, LQ_EF_PAGE);
        return;
    }
    const int64_t page = slot >> a.page_log2;
    const int64_t row = (((page * 2 + side) * a.n_heads + h) << a.page_log2) + (slot & ((1 << a.page_log2) - 1));
    a.codes[row * BPT + b] = word;
    if (b == 0) a.scales[row] = s;
}

template <int DT>
int launch_append(const AppendArgs &a, int D, cudaStream_t st) {
    if (D == 128)
        paged_append_kernel<DT, 128><<<dim3((unsigned)ceil_div(a.n_vec, 16), 2), 256, 0, st>>>(a);
    else
        paged_append_kernel<DT, 64><<<dim3((unsigned)ceil_div(a.n_vec, 32), 2), 256, 0, st>>>(a);
    return check_launch();
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" int lq_paged_append(const void *k, const void *v, int dtype, int64_t n_tokens, int n_heads, int head_dim,
                               int64_t k_stride_n, int64_t k_stride_h, int64_t v_stride_n, int64_t v_stride_h,
                               const int64_t *slots, int64_t n_pages, int page_tokens, int32_t *codes, float *scales,
                               void *k_out, void *v_out, uint32_t *err, void *stream) {
    LQ_NVTX_RANGE();
    if (n_tokens < 0 || n_heads < 1 || !paged_dim_ok(head_dim) || !paged_page_ok(page_tokens) || n_pages < 0 ||
        n_tokens > 0x7fffffff / n_heads || n_pages > 0x7fffffff)
        return LQ_ERR_INVALID;
    if (n_tokens == 0) return LQ_OK;
    if (!k || !v || !slots || !codes || !scales) return LQ_ERR_INVALID;
    // 16-byte loads of 8 channels: rows start on a multiple of 8 elements
    const uintptr_t p = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                        reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out);
    if ((p & 15) != 0 || ((k_stride_n | k_stride_h | v_stride_n | v_stride_h) & 7) != 0) return LQ_ERR_INVALID;
    AppendArgs a{};
    a.x[0] = k;
    a.x[1] = v;
    a.stride_n[0] = k_stride_n;
    a.stride_n[1] = v_stride_n;
    a.stride_h[0] = k_stride_h;
    a.stride_h[1] = v_stride_h;
    a.out[0] = k_out;
    a.out[1] = v_out;
    a.slots = slots;
    a.codes = reinterpret_cast<uint32_t *>(codes);
    a.scales = scales;
    a.err = err;
    a.n_vec = (uint32_t)(n_tokens * n_heads);
    a.n_heads = (uint32_t)n_heads;
    a.page_log2 = (uint32_t)__builtin_ctz((unsigned)page_tokens);
    a.n_slots = n_pages * page_tokens;
    a.by_heads = FastDiv((uint32_t)n_heads);
    cudaStream_t st = as_stream(stream);
    if (dtype == LQ_BF16) return launch_append<LQ_BF16>(a, head_dim, st);
    if (dtype == LQ_F16) return launch_append<LQ_F16>(a, head_dim, st);
    if (dtype == LQ_F32) return launch_append<LQ_F32>(a, head_dim, st);
    return LQ_ERR_INVALID;
}
