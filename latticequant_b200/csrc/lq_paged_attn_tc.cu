// lq_paged_attn_tc.cu -- attention over the pages of an E8 cache on the
// 5th-generation tensor cores, for many query rows (trees, prompt chunks).
//
// The same mathematics as lq_paged_attn.cu, in the same transposed form: a
// CTA takes 128 tokens at a time and up to N query rows of one KV head,
//   S^T [128 tokens x N] = K [128 x D] Q^T      (tcgen05.mma, into TMEM)
//   x = S^T * ks * c + log2(vs),  w = 2^(x - M),  l += w / vs
//   O^T [D x N] += V^T [D x 128] W [128 x N]    (tcgen05.mma, stays in TMEM)
// Tokens are the MMA's 128 rows, so no row is padding however few queries
// there are; a softmax thread owns one token (a TMEM lane) and 16 of the N columns.
//
// The warps have four parts, which meet only at mbarriers:
//   the producer  bulk-copies a tile's code words and scales, page by page, into
//       a ring of stages
//   decoders   turn the words into the swizzled shared-memory layout that both
//       MMAs read (a decoded block of 8 channels is one 16-byte chunk; V^T is
//       read from the same token-major layout as an MN-major operand)
//   two issuers start the two MMAs of every tile
//   softmax    scores out of TMEM, weights to shared memory, a row of N per token
// so copying, decoding, the tensor cores and the exponentials overlap.  What a
// tile waits for in the last part, and with few rows in decoding, is latency: 16
// columns a thread keep enough warps there, with up to 32 rows two sets of
// softmax warps take the tiles in turn, each with references, denominators and
// an O of its own that are joined at the end, and with up to 16 two sets of
// decoders do.
//
// 64 positions over 4 sequences of 32,768 tokens (448 rows of 4 KV heads of 128):
// 303 us, 397 TFLOP/s, bound by issue (69% of the slots): 7,220 instructions and
// 2,630 cycles a tile of 128 tokens and 64 rows.  Earlier forms of the product took 749 us (mma.sync
// from registers) and 413 (tcgen05 with one barrier-synchronised part).
//
// M is a reference per row, moved only when an x exceeds it by kRefSlack,
// which a vote of the 128 threads finds; O is then rescaled in TMEM.
//
// Every wait is bounded (LQ_EF_TIMEOUT after about a second; the results are
// then wrong, the thread's later waits return at once, and nothing more is
// started).
#include "lq_paged_attn.cuh"

namespace lq {
namespace {

constexpr int kTok = 128;               // tokens of a tile
constexpr int kHalfBytes = kTok * 128;  // 64 channels (or weights) of a tile's tokens in fp16, 128-byte rows

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void store16(uint32_t addr, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                 : "memory");
}

// A contiguous copy from global to shared memory that completes on a barrier; all 16-byte aligned.
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void arrive_expecting(uint32_t bar, uint32_t bytes) {
    asm volatile("{\n.reg .b64 t;\nmbarrier.arrive.expect_tx.shared::cta.b64 t, [%0], %1;\n}" ::"r"(bar), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void load16(uint32_t addr, uint32_t (&v)[4]) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(addr)
                 : "memory");
}

// Matrix descriptor of a 128-byte-swizzled operand: lead and stride in bytes.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead, uint32_t stride) {
    return (uint64_t)(addr >> 4 & 0x3fffu) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | 1ull << 46 |
           2ull << 61;
}

// Instruction descriptor: fp16 operands, fp32 accumulator, M = 128.
template <int N>
constexpr uint32_t kShape = 1u << 4 | (uint32_t)(N >> 3) << 17 | (128u >> 4) << 24;
constexpr uint32_t kTransposeA = 1u << 15, kTransposeB = 1u << 16;

// One step of an MMA, ACC: added to d.  Called by a whole warp with warp-uniform
// arguments, which then stay in uniform registers; one lane issues.
template <bool ACC>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, uint32_t lane_ok) {
    asm volatile(
        "{\n.reg .pred p, q;\nsetp.ne.u32 q, %4, 0;\nsetp.eq.u32 p, %5, 1;\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(shape), "r"(lane_ok), "n"(ACC ? 1 : 0)
        : "memory");
}
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t r;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(r));
    return r;
}
__device__ __forceinline__ void mma_done(uint32_t bar, uint32_t lane_ok) {
    asm volatile(
        "{\n.reg .pred q;\nsetp.ne.u32 q, %1, 0;\n"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(bar),
        "r"(lane_ok)
        : "memory");
}

__device__ __forceinline__ bool passed(uint32_t bar, uint32_t phase) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok)
                 : "r"(bar), "r"(phase)
                 : "memory");
    return ok != 0;
}
// Waits for the barrier's phase, at most about a second; false then.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t phase) {
    if (passed(bar, phase)) return true;
    const long long start = clock64();
    while (!passed(bar, phase))
        if (clock64() - start > 2000000000ll) return false;
    return true;
}

// C consecutive TMEM columns of the warp's 32 lanes.
template <int C>
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[C]) {
    static_assert(C % 8 == 0);
    __syncwarp();  // a wait's loop may have left the lanes apart
#pragma unroll
    for (int i = 0; i < C; i += 8)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=f"(v[i]), "=f"(v[i + 1]), "=f"(v[i + 2]), "=f"(v[i + 3]), "=f"(v[i + 4]), "=f"(v[i + 5]),
                       "=f"(v[i + 6]), "=f"(v[i + 7])
                     : "r"(addr + i));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < C; ++i) asm volatile("" : "+f"(v[i]));  // no use of v moves above the wait
}
template <int C>
__device__ __forceinline__ void tmem_store(uint32_t addr, const float (&v)[C]) {
#pragma unroll
    for (int i = 0; i < C; i += 8)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr + i),
                     "f"(v[i]), "f"(v[i + 1]), "f"(v[i + 2]), "f"(v[i + 3]), "f"(v[i + 4]), "f"(v[i + 5]),
                     "f"(v[i + 6]), "f"(v[i + 7])
                     : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Generic writes to shared memory become visible to the tensor cores.
__device__ __forceinline__ void publish_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void arrive(uint32_t bar) {
    asm volatile("{\n.reg .b64 t;\nmbarrier.arrive.shared::cta.b64 t, [%0];\n}" ::"r"(bar) : "memory");
}
// One arrival for the warp, after all its lanes' writes.
__device__ __forceinline__ void arrive_warp(uint32_t bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) arrive(bar);
}
template <class X>
__device__ __forceinline__ void sync_softmax() {
    asm volatile("bar.sync 8, %0;" ::"n"(32 * X::kSoftmax) : "memory");
}
// Barrier of 128 threads, and its vote.
__device__ __forceinline__ void sync128(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool any128(int id, bool x) {
    uint32_t r;
    asm volatile(
        "{\n.reg .pred p, q;\nsetp.ne.u32 p, %2, 0;\nbar.red.or.pred q, %1, 128, p;\nselp.u32 %0, 1, 0, q;\n}"
        : "=r"(r)
        : "r"(id), "r"((uint32_t)x)
        : "memory");
    return r != 0;
}

// C values of every lane folded over the warp: lane i ends with value i / (32 / C).  Each step halves the
// values that a lane carries and sends the other half, so C shuffles do for C values.
template <int C, class Op>
__device__ __forceinline__ float fold(float (&v)[C], Op op) {
    const int lane = threadIdx.x & 31;
    int off = 16;
#pragma unroll
    for (int n = C / 2; n >= 1; n /= 2, off /= 2) {
        const bool up = lane & off;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float keep = up ? v[i + n] : v[i], send = up ? v[i] : v[i + n];
            v[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, off));
        }
    }
#pragma unroll
    for (; off >= 1; off /= 2) v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], off));
    return v[0];
}

// Whether the decoded row of a token at `at` is zero, once `full` has come to its phase; -1: it did not.  (Rarely
// called, and apart because its code within the softmax loop cost 2%: 308 for 302.6 us, 64 positions over 4 x 32,768.)
template <int D>
__device__ __noinline__ int zero_row(uint32_t full, uint32_t phase, uint32_t at) {
    if (!wait_for(full, phase)) return -1;
    uint32_t bits = 0;
#pragma unroll 1
    for (int i = 0; i < D / 8; ++i) {
        uint32_t w[4];
        load16(at + (i >> 3) * kHalfBytes + ((i & 7) << 4), w);
        bits |= w[0] | w[1] | w[2] | w[3];
    }
    return bits == 0;
}

// The kernel for D channels and up to COLS query rows a CTA.
template <int D, int COLS>
struct Shape {
    static constexpr int kN = COLS;                    // columns of the MMAs
    static constexpr int kC = 16;                      // columns of a softmax thread
    static constexpr int kGroups = COLS / kC;          // column groups of 4 warps
    static constexpr int kSets = COLS <= 32 ? 2 : 1;   // of softmax warps, which take the tiles in turn
    static constexpr int kSoftmax = 4 * kGroups * kSets;
    static constexpr int kDecodeSets = COLS <= 16 ? 2 : 1;
    static constexpr int kDecode = 8;                  // warps of a set
    static constexpr int kIssue = kSoftmax + kDecode * kDecodeSets;  // first of the two issuers and the producer
    static constexpr int kThreads = 32 * (kIssue + 4);
    static constexpr int kPerRow = D / 32;                  // decoder threads of a token's row, four words each
    static constexpr int kRowStep = 32 * kDecode / kPerRow; // token rows the decoders take at once
    static constexpr int kRows = kTok / kRowStep;           // of a thread
    static constexpr uint32_t kTmem = (2 + kSets) * kN <= 64 ? 64 : 4 * kN;  // S^T twice and the sets' O^T
    static_assert(kRows >= 1 && kRowStep % 8 == 0);
    static constexpr int kTileBytes = D / 64 * kHalfBytes;  // K or V of a tile; both are double-buffered
    static constexpr int kOperands = 4 * kTileBytes + kN * D * 2 + kSets * kHalfBytes;
    // a stage: the code words of K and V and the scales of K and V of 128 tokens
    static constexpr int kWordBytes = kTok * D / 2, kStageBytes = 2 * kWordBytes + 2 * kTok * 4;
    static constexpr int kStages = D == 128 ? 3 : 6;
};

// Shared memory after the 1024-byte aligned operands and the stages.
template <class X>
struct Small {
    uint64_t stage_full[X::kStages], stage_free[X::kStages], k_full[2], k_free[2], v_full[2], v_free[2];
    uint64_t s_full[2], s_free[2], p_full[X::kSets], p_free[X::kSets], q_full;
    alignas(16) float minus_m[X::kSets][X::kN];
    alignas(16) float f[X::kSets][X::kN];
    float red[X::kSets][4][X::kN];
    uint32_t bad[X::kStages];  // bit: a page of the stage's tokens lies outside the pool
    float back[X::kN];  // what a row's scores are multiplied by where `apart`
    uint32_t tmem, exponent, apart;
};

// The lane order of a decoded block: position p holds channel kChannel >> 4p & 15.
constexpr uint32_t kChannel = 0x04152637u;

// A wait that gives up once and for all after about a second.
struct Waiter {
    bool alive = true;
    __device__ __forceinline__ void operator()(const uint64_t &bar, uint32_t phase) {
        alive = alive && wait_for(smem_u32(&bar), phase & 1);
    }
};

template <bool BF16, int D, int COLS>
__global__ void __launch_bounds__(Shape<D, COLS>::kThreads, 1)
    paged_attn_tc_kernel(const __grid_constant__ PagedAttnArgs a) {
    using X = Shape<D, COLS>;
    constexpr int N = X::kN, C = X::kC, W = D / 8, kThreads = X::kThreads;
    extern __shared__ char raw[];
    char *buf = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    // V first: at D = 64 the O MMA's upper 64 rows read past it, into the next buffer (and are not used)
    const uint32_t sv = smem_u32(buf), sk = sv + 2 * X::kTileBytes, sq = sk + 2 * X::kTileBytes, sp = sq + N * D * 2;
    const uint32_t stages = sv + X::kOperands;
    Small<X> &sm = *reinterpret_cast<Small<X> *>(buf + X::kOperands + X::kStages * X::kStageBytes);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t b = blockIdx.z, rt = blockIdx.y / a.n_heads, h = blockIdx.y - rt * a.n_heads;
    const uint32_t row0 = rt * COLS;
    const int len = (int)paged_len(a, b);
    const int first = (int)(blockIdx.x * a.chunk), last = paged_split_end(a, first, len);
    const int drafts = len - (int)a.T;
    if (len < a.lens[b] && (blockIdx.x | blockIdx.y | tid) == 0) raise_flag(a.err, LQ_EF_PAGE);
    const int live = (int)min((uint32_t)COLS, a.rows - row0);
    if (first >= last) {  // nothing to read; without a split the rows are still written
        if (a.splits == 1)
            for (int n = warp; n < live; n += kThreads / 32) {
                const float zero[D / 32] = {};
                paged_emit_row<BF16, D>(a, b, h, row0 + n, 0, zero, 0.f, kNoRef);
            }
        return;
    }
    const int n_tiles = (last - first + kTok - 1) / kTok;

    if (warp == X::kIssue) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)),
                     "r"(X::kTmem)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (tid == 32 * (X::kIssue + 1)) {
        auto init = [](uint64_t &bar, uint32_t n) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&bar)), "r"(n) : "memory");
        };
        init(sm.q_full, X::kSoftmax);
        for (int i = 0; i < X::kStages; ++i) {
            init(sm.stage_full[i], 1);
            init(sm.stage_free[i], X::kDecode + 4 * X::kGroups);
        }
        for (int i = 0; i < X::kSets; ++i) {
            init(sm.p_full[i], 4 * X::kGroups);
            init(sm.p_free[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            init(sm.k_full[i], X::kDecode);
            init(sm.k_free[i], 1);
            init(sm.v_full[i], X::kDecode);
            init(sm.v_free[i], 1);
            init(sm.s_full[i], 1);
            init(sm.s_free[i], 4 * X::kGroups);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sm.exponent = sm.apart = 0;
    }
    for (int n = tid; n < X::kSets * N; n += kThreads) sm.minus_m[n / N][n % N] = -kNoRef;

    // Q's loads are on their way over the barrier, and the producer's first pages
    constexpr int kLoaders = 32 * X::kSoftmax, kChunks = N * W;  // 16-byte chunks of Q
    constexpr int kQ = (kChunks + kLoaders - 1) / kLoaders;
    uint4 q[kQ];
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
        const int e = tid + i * kLoaders, n = e / W, c = e % W;
        q[i] = make_uint4(0, 0, 0, 0);
        if (tid < kLoaders && e < kChunks && n < live) {
            const uint32_t r = row0 + n, qt = a.by_group.div(r), qh = h * a.group + (r - qt * a.group);
            q[i] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) + b * a.q_stride_b +
                                                         qh * a.q_stride_h + qt * a.q_stride_t) + c);
        }
    }
    const int seg_log2 = min((int)a.page_log2, 7), segs = kTok >> seg_log2;  // runs of a tile's rows in one page
    const int32_t *table = a.table + b * a.table_stride;
    auto entry_of = [&](int tok) { return lane < segs && tok < last ? __ldg(table + (tok >> a.page_log2)) : 0; };
    int tok_p = first + (lane << seg_log2), page = 0;
    if (warp == X::kIssue + 2) page = entry_of(tok_p);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t ts = sm.tmem, to = ts + 2 * N;
    Waiter wait, drain;

    if (warp < X::kSoftmax) {
        // ---- softmax: token tl (a TMEM lane), columns col0.., every kSets-th tile
        // Q: fp16 rows in the decoded blocks' channel order; rows past the last are zero
        float qk = a.qk_log2 * kCodeUnit;
        {
            // bf16: a power of two puts the rows' largest finite value in [2^10, 2^11).  Rows down to 2^-kNear of it share
            // the power, which goes into qk and leaves them every bit; a row further down has its own, and its scores
            // are multiplied back.
            if constexpr (BF16) {
                constexpr uint32_t kLeast = 27, kNear = 10;  // rows under 2^-100 count as 2^-100
                uint32_t e[kQ], top = kLeast;  // exponent of the chunk's row: the W chunks of a row are neighbouring lanes
    #pragma unroll
                for (int i = 0; i < kQ; ++i) {
                    const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
                    e[i] = 0;
    #pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t lo = w[k] >> 7 & 0xffu, hi = w[k] >> 23 & 0xffu;
                        e[i] = max(e[i], max(lo == 0xffu ? 0u : lo, hi == 0xffu ? 0u : hi));
                    }
    #pragma unroll
                    for (int o = W / 2; o >= 1; o >>= 1) e[i] = max(e[i], __shfl_xor_sync(0xffffffffu, e[i], o));
                    top = max(top, e[i]);
                }
                top = __reduce_max_sync(0xffffffffu, top);
                if (lane == 0) atomicMax(&sm.exponent, top);
                sync_softmax<X>();
                top = sm.exponent;
                qk *= __uint_as_float((top - 10u) << 23);
    #pragma unroll
                for (int i = 0; i < kQ; ++i) {
                    const int at = tid + i * kLoaders;
                    const uint32_t own = max(e[i], kLeast), down = top - own;
                    const bool far = e[i] != 0 && down > kNear;
                    const float f = __uint_as_float((264u - (far ? own : top)) << 23);
                    q[i] = make_uint4(bf16_to_f16(q[i].x, f), bf16_to_f16(q[i].y, f), bf16_to_f16(q[i].z, f),
                                      bf16_to_f16(q[i].w, f));
                    if (at < kChunks && at % W == 0) {  // 2^-down in two steps: down may reach 227
                        sm.back[at / W] = far ? __uint_as_float((127u - down / 2) << 23) *
                                                    __uint_as_float((127u - (down + 1) / 2) << 23)
                                              : 1.f;
                        if (far) sm.apart = 1;
                    }
                }
                sync_softmax<X>();
            }
    #pragma unroll
            for (int i = 0; i < kQ; ++i) {
                const int e = tid + i * kLoaders, n = e / W, c = e % W;
                if (e >= kChunks) break;
                // pairs (7, 3), (6, 2), (5, 1), (4, 0)
                const uint32_t v[4] = {__byte_perm(q[i].w, q[i].y, 0x7632), __byte_perm(q[i].w, q[i].y, 0x5410),
                                       __byte_perm(q[i].z, q[i].x, 0x7632), __byte_perm(q[i].z, q[i].x, 0x5410)};
                store16(sq + (c >> 3) * (N * 128) + n * 128 + (((c & 7) ^ (n & 7)) << 4), v);
            }
        }
        publish_smem();
        arrive_warp(smem_u32(&sm.q_full));
        const int tl = (warp & 3) * 32 + lane, group = (warp >> 2) % X::kGroups, set = (warp >> 2) / X::kGroups;
        const int col0 = group * C, vote = 1 + (warp >> 2);
        const uint32_t my_lanes = (uint32_t)((warp & 3) * 32) << 16, o_at = to + set * N + my_lanes + col0;
        float *const minus_m = sm.minus_m[set] + col0, *const f = sm.f[set] + col0;
        float(*const red)[N] = sm.red[set];
        const uint32_t my_p = sp + set * kHalfBytes + tl * 128;
        const bool apart = BF16 && sm.apart;
        unsigned long long l[C / 2];  // of two columns each, as packed fp32
#pragma unroll
        for (int c = 0; c < C / 2; ++c) l[c] = 0;
        int done = 0;  // tiles of this set
        for (int j = set; j < n_tiles; j += X::kSets, ++done) {
            const int s = j & 1, tok = first + j * kTok + tl, stage = j % X::kStages;
            wait(sm.stage_full[stage], j / X::kStages);
            float ks, vs;
            const uint32_t from = stages + stage * X::kStageBytes + 2 * X::kWordBytes + tl * 4;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(ks) : "r"(from) : "memory");
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(vs) : "r"(from + kTok * 4) : "memory");
            // tokens past the end, and those whose page is outside the pool, weigh nothing
            const bool none = tok >= last || (sm.bad[stage] >> (tl >> seg_log2) & 1);
            arrive_warp(smem_u32(&sm.stage_free[stage]));
            const float kx = none ? 0.f : ks * qk;
            float lv = none ? -INFINITY : lg2(vs), rvs = none ? 0.f : rcp(vs);
            uint32_t hidden = 0;  // columns that do not see the token
            if (tok >= drafts && tok < last)
#pragma unroll 1
                for (uint32_t c = 0; c < C && row0 + col0 + c < a.rows; ++c)
                    hidden |= (uint32_t)!paged_sees(a, b, a.by_group.div(row0 + col0 + c), tok - drafts) << c;
            wait(sm.s_full[s], j >> 1);
            tmem_fence_after();
            float x[C];
            auto scores = [&]() {
                tmem_load<C>(ts + s * N + my_lanes + col0, x);
                if (apart) {
#pragma unroll
                    for (int c = 0; c < C; ++c) x[c] *= sm.back[col0 + c];
                }
                const unsigned long long mul = f2_pack(kx, kx), add = f2_pack(lv, lv);
#pragma unroll
                for (int c = 0; c < C; c += 2) f2_unpack(f2_fma(f2_pack(x[c], x[c + 1]), mul, add), x[c], x[c + 1]);
                if (__any_sync(0xffffffffu, hidden != 0)) {
#pragma unroll
                    for (int c = 0; c < C; ++c) x[c] = hidden >> c & 1 ? -INFINITY : x[c];
                }
            };
            auto less_reference = [&]() {
                float top = -INFINITY;
#pragma unroll
                for (int c = 0; c < C; c += 4) {
                    const float4 m = *reinterpret_cast<const float4 *>(minus_m + c);
                    f2_unpack(f2_add(f2_pack(x[c], x[c + 1]), f2_pack(m.x, m.y)), x[c], x[c + 1]);
                    f2_unpack(f2_add(f2_pack(x[c + 2], x[c + 3]), f2_pack(m.z, m.w)), x[c + 2], x[c + 3]);
                    top = fmaxf(fmaxf(fmaxf(top, x[c]), fmaxf(x[c + 1], x[c + 2])), x[c + 3]);
                }
                return top > kRefSlack;
            };
            scores();
            const bool move = any128(vote, less_reference());
            if (done > 0) wait(sm.p_free[set], done - 1);  // O of the set's tile before is done: W's buffer is free
            if (move) {
                if (__any_sync(0xffffffffu, rvs == 1.f)) {  // V vectors of zeros, perhaps
                    const int zero = zero_row<D>(smem_u32(&sm.v_full[s]), (j >> 1) & 1, sv + s * X::kTileBytes + tl * 128);
                    wait.alive = wait.alive && zero >= 0;
                    if (zero > 0 && rvs == 1.f) {
                        lv = kZeroLog2;
                        rvs = kZeroInv;
                    }
                }
                // the tile's column maxima move the references; l and O follow
                scores();
                const float warp_top = fold(x, [](float p, float q) { return fmaxf(p, q); });
                if (lane % (32 / C) == 0) red[warp & 3][col0 + lane / (32 / C)] = warp_top;
                sync128(vote);
                if (tl < C) {
                    const int n = col0 + tl;
                    const float top = fmaxf(fmaxf(red[0][n], red[1][n]), fmaxf(red[2][n], red[3][n]));
                    const float m = -minus_m[tl], next = fmaxf(m, top - kRefBelow);
                    f[tl] = ex2(m - next);
                    minus_m[tl] = -next;
                }
                sync128(vote);
                scores();
                less_reference();
#pragma unroll
                for (int c = 0; c < C; c += 2) l[c / 2] = f2_mul(l[c / 2], f2_pack(f[c], f[c + 1]));
                if (done > 0) {  // this warp's lanes (channels) and columns of O
                    tmem_fence_after();
                    float o[C];
                    tmem_load<C>(o_at, o);
#pragma unroll
                    for (int c = 0; c < C; ++c) o[c] *= f[c];
                    tmem_store<C>(o_at, o);
                }
            }
            tmem_fence_before();
            arrive_warp(smem_u32(&sm.s_free[s]));
            // weights: this token's row of columns
            const unsigned long long rvs2 = f2_pack(rvs, rvs);
#pragma unroll
            for (int c = 0; c < C; c += 8) {
                uint32_t pair[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float w0 = ex2(x[c + 2 * i]), w1 = ex2(x[c + 2 * i + 1]);
                    l[c / 2 + i] = f2_fma(f2_pack(w0, w1), rvs2, l[c / 2 + i]);
                    const __half2 h2 = __floats2half2_rn(w0, w1);
                    pair[i] = *reinterpret_cast<const uint32_t *>(&h2);
                }
                const int n = col0 + c;
                store16(my_p + (((n >> 3 & 7) ^ (tl & 7)) << 4), pair);
            }
            publish_smem();
            arrive_warp(smem_u32(&sm.p_full[set]));
        }
        // denominators over the 128 tokens, then O: a lane is a channel
        if (done > 0) wait(sm.p_free[set], done - 1);
        tmem_fence_after();
        float sums[C];
#pragma unroll
        for (int c = 0; c < C; c += 2) f2_unpack(l[c / 2], sums[c], sums[c + 1]);
        const float sum = fold(sums, [](float p, float q) { return p + q; });
        if (lane % (32 / C) == 0) red[warp & 3][col0 + lane / (32 / C)] = sum;
        float o[C];
        tmem_load<C>(o_at, o);
        tmem_fence_before();
        // all sets are through (every operand has been read), then through shared memory to rows of channels
        sync_softmax<X>();
        float *rows = reinterpret_cast<float *>(buf);
        const int d = (tl & ~7) + (int)(kChannel >> (4 * (tl & 7)) & 15u);
        if (D == 128 || tl < 64)
#pragma unroll
            for (int c = 0; c < C; ++c) rows[(set * COLS + col0 + c) * D + d] = done > 0 ? o[c] : 0.f;
        sync_softmax<X>();
        for (int n = warp; n < live; n += X::kSoftmax) {
            float m = kNoRef, den = 0.f, w[X::kSets], od[D / 32];
#pragma unroll
            for (int i = 0; i < X::kSets; ++i) m = fmaxf(m, -sm.minus_m[i][n]);
#pragma unroll
            for (int i = 0; i < X::kSets; ++i) {
                w[i] = ex2(-sm.minus_m[i][n] - m);
                den = fmaf((sm.red[i][0][n] + sm.red[i][1][n]) + (sm.red[i][2][n] + sm.red[i][3][n]), w[i], den);
            }
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
                od[k] = 0.f;
#pragma unroll
                for (int i = 0; i < X::kSets; ++i)
                    od[k] = fmaf(rows[(i * COLS + n) * D + lane * (D / 32) + k], w[i], od[k]);
            }
            paged_emit_row<BF16, D>(a, b, h, row0 + n, blockIdx.x, od, den, m);
        }
    } else if (warp < X::kIssue) {
        // ---- decoders: kRows rows of four words each of K and V, every kDecodeSets-th tile
        const int set = (warp - X::kSoftmax) / X::kDecode, dt = tid - 32 * (X::kSoftmax + set * X::kDecode);
        const int part = dt % X::kPerRow, drow = dt / X::kPerRow;
        // At D = 128 the two 64-channel halves of an operand fall on the same banks, so the threads of the
        // upper one take their words in the order 2, 3, 0, 1.
        const bool upper = D == 128 && part >= 2;
        uint32_t chunk_at[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            chunk_at[i] = (D == 128 ? (part >> 1) * kHalfBytes : 0) + drow * 128 +
                          (((((part & 1) * 4 + i) ^ (upper ? 2 : 0)) ^ (drow & 7)) << 4);
        constexpr uint32_t kRowBytes = 32 * X::kDecode * 16;  // between a thread's rows in a stage
        auto put = [&](uint32_t dst, uint32_t src) {
#pragma unroll
            for (int r = 0; r < X::kRows; ++r) {
                uint32_t w[4];
                load16(src + r * kRowBytes, w);
                const uint32_t v[4] = {upper ? w[2] : w[0], upper ? w[3] : w[1], upper ? w[0] : w[2],
                                       upper ? w[1] : w[3]};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t pair[4];
                    decode_block(v[i], pair);
                    store16(dst + chunk_at[i] + r * (X::kRowStep * 128), pair);
                }
            }
        };
        for (int j = set; j < n_tiles; j += X::kDecodeSets) {
            const int s = j & 1, stage = j % X::kStages;
            const uint32_t from = stages + stage * X::kStageBytes + dt * 16;
            if (j >= 2) wait(sm.k_free[s], (j >> 1) - 1);
            wait(sm.stage_full[stage], j / X::kStages);
            put(sk + s * X::kTileBytes, from);
            publish_smem();
            arrive_warp(smem_u32(&sm.k_full[s]));
            if (j >= 2) wait(sm.v_free[s], (j >> 1) - 1);
            put(sv + s * X::kTileBytes, from + X::kWordBytes);
            publish_smem();
            __syncwarp();
            if (lane == 0) {
                arrive(smem_u32(&sm.v_full[s]));
                arrive(smem_u32(&sm.stage_free[stage]));
            }
        }
    } else {
        // ---- the issuers (the first warp starts S, the second O) and the producer
        const int issuer = __shfl_sync(0xffffffffu, warp - X::kIssue, 0);  // uniform
        const uint32_t one = elect_lane();
        // Nothing of this block's is under way when it ends: what an issuer or the producer has started arrives
        // first, also where a wait gave up (it starts nothing more then).
        if (issuer == 0) {
            const uint64_t dq = operand(sq, 16, 1024), dk = operand(sk, 16, 1024);
            wait(sm.q_full, 0);
            int j = 0;
            for (; j < n_tiles; ++j) {
                const int s = j & 1;
                wait(sm.k_full[s], j >> 1);
                if (j >= 2) wait(sm.s_free[s], (j >> 1) - 1);
                if (__any_sync(0xffffffffu, !wait.alive)) break;
                tmem_fence_after();
                const uint64_t dks = dk + (uint32_t)(s * (X::kTileBytes >> 4));
                mma<false>(ts + s * N, dks, dq, kShape<N>, one);
#pragma unroll
                for (int k = 1; k < D / 16; ++k) {
                    const uint32_t in = (k & 3) * 2;  // 32 bytes on within the swizzled rows
                    mma<true>(ts + s * N, dks + (k >> 2) * (kHalfBytes >> 4) + in, dq + (k >> 2) * (N * 128 >> 4) + in,
                              kShape<N>, one);
                }
                mma_done(smem_u32(&sm.s_full[s]), one);
                mma_done(smem_u32(&sm.k_free[s]), one);
            }
            for (int i = max(j - 2, 0); i < j; ++i) drain(sm.k_free[i & 1], i >> 1);
        } else if (issuer == 1) {
            constexpr uint32_t shape = kShape<N> | kTransposeA | kTransposeB;
            const uint64_t dp = operand(sp, kHalfBytes, 1024), dv = operand(sv, kHalfBytes, 1024);
            int j = 0;
            for (; j < n_tiles; ++j) {
                const int s = j & 1, set = j % X::kSets, turn = j / X::kSets;
                wait(sm.v_full[s], j >> 1);
                wait(sm.p_full[set], turn);
                if (__any_sync(0xffffffffu, !wait.alive)) break;
                tmem_fence_after();
                const uint64_t dvs = dv + (uint32_t)(s * (X::kTileBytes >> 4)), dps = dp + set * (kHalfBytes >> 4);
                const uint32_t d = to + set * N;
                if (turn == 0) mma<false>(d, dvs, dps, shape, one);
                else mma<true>(d, dvs, dps, shape, one);
#pragma unroll
                for (int k = 1; k < kTok / 16; ++k) mma<true>(d, dvs + k * (2048 >> 4), dps + k * (2048 >> 4), shape, one);
                mma_done(smem_u32(&sm.p_free[set]), one);
                mma_done(smem_u32(&sm.v_free[s]), one);
            }
            for (int i = max(j - 2, 0); i < j; ++i) drain(sm.v_free[i & 1], i >> 1);
        } else if (issuer == 2) {
            // lane i < segs copies the tile's i-th run of rows that lie in one page
            const int64_t side = (int64_t)a.n_heads << a.page_log2;
            const uint32_t *kbase = a.codes + ((int64_t)h << a.page_log2) * W;
            const float *sbase = a.scales + ((int64_t)h << a.page_log2);
            int stage = 0, j = 0;
            for (; j < n_tiles; ++j, tok_p += kTok) {
                const int tok = tok_p;
                const bool mine = lane < segs && tok < last, bad = mine && (uint32_t)page >= (uint32_t)a.n_pages;
                const int64_t row = 2 * side * (bad ? 0 : page) + (tok & ((1 << a.page_log2) - 1));
                page = entry_of(tok + kTok);
                if (j >= X::kStages) wait(sm.stage_free[stage], j / X::kStages - 1);
                if (__any_sync(0xffffffffu, !wait.alive)) break;
                const uint32_t runs = __popc(__ballot_sync(0xffffffffu, mine)), out = __ballot_sync(0xffffffffu, bad);
                const uint32_t bar = smem_u32(&sm.stage_full[stage]);
                if (lane == 0) {
                    sm.bad[stage] = out;
                    if (out) raise_flag(a.err, LQ_EF_PAGE);
                    arrive_expecting(bar, (runs << seg_log2) * (D + 8));  // a token: two rows of D / 2, two scales
                }
                __syncwarp();
                if (mine) {
                    const uint32_t to_stage = stages + stage * X::kStageBytes;
                    const uint32_t words = (uint32_t)(D / 2) << seg_log2, at = lane << seg_log2;
                    bulk_copy(to_stage + at * (D / 2), kbase + row * W, words, bar);
                    bulk_copy(to_stage + X::kWordBytes + at * (D / 2), kbase + (row + side) * W, words, bar);
                    bulk_copy(to_stage + 2 * X::kWordBytes + at * 4, sbase + row, 4u << seg_log2, bar);
                    bulk_copy(to_stage + 2 * X::kWordBytes + (kTok + at) * 4, sbase + row + side, 4u << seg_log2, bar);
                }
                stage = stage == X::kStages - 1 ? 0 : stage + 1;
            }
            for (int i = max(j - X::kStages, 0); i < j; ++i) drain(sm.stage_full[i % X::kStages], i / X::kStages);
        }
    }
    if (!wait.alive || !drain.alive) raise_flag(a.err, LQ_EF_TIMEOUT);
    __syncthreads();
    if (warp == X::kIssue)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(ts), "r"(X::kTmem) : "memory");
}

template <bool BF16, int D, int COLS>
int launch_n(const PagedAttnArgs &a, uint32_t batch, cudaStream_t st) {
    using X = Shape<D, COLS>;
    constexpr size_t smem = 1024 + X::kOperands + X::kStages * X::kStageBytes + sizeof(Small<X>);
    static_assert(smem <= 227 * 1024);
    if (cudaFuncSetAttribute(paged_attn_tc_kernel<BF16, D, COLS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)smem) != cudaSuccess)
        return LQ_ERR_CUDA;
    paged_attn_tc_kernel<BF16, D, COLS>
        <<<dim3(a.splits, a.n_heads * (uint32_t)ceil_div(a.rows, COLS), batch), X::kThreads, smem, st>>>(a);
    return check_launch();
}

template <bool BF16, int D>
int launch_d(const PagedAttnArgs &a, int tile, uint32_t batch, cudaStream_t st) {
    if constexpr (D == 128) {  // up to 16 rows of 64 channels go to the other kernel
        if (tile == 16) return launch_n<BF16, D, 16>(a, batch, st);
    }
    if (tile == 32) return launch_n<BF16, D, 32>(a, batch, st);
    return launch_n<BF16, D, 64>(a, batch, st);
}

}  // namespace

int launch_paged_tc(const PagedAttnArgs &a, bool bf16, int head_dim, int tile, uint32_t batch, cudaStream_t st) {
    if (bf16) return head_dim == 128 ? launch_d<true, 128>(a, tile, batch, st) : launch_d<true, 64>(a, tile, batch, st);
    return head_dim == 128 ? launch_d<false, 128>(a, tile, batch, st) : launch_d<false, 64>(a, tile, batch, st);
}

}  // namespace lq
