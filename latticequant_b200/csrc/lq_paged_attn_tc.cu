// lq_paged_attn_tc.cu -- attention over the pages of an E8 cache on the
// 5th-generation tensor cores, for many query rows (trees, prompt chunks).
//
// The same mathematics as lq_paged_attn.cu, in the same transposed form: a
// CTA takes 128 tokens at a time and up to N query rows of one KV head,
//   S^T [128 tokens x N] = K [128 x D] Q^T      (tcgen05.mma, into TMEM)
//   x = S^T * ks * c + log2(vs),  w = 2^(x - M),  l += w / vs
//   O^T [D x N] += V^T [D x 128] W [128 x N]    (tcgen05.mma, stays in TMEM)
// Tokens are the MMA's 128 rows, so no row is padding however few queries
// there are; a thread owns one token (a TMEM lane) and half of the N columns.
//
// The threads decode a tile's code words straight into the swizzled
// shared-memory layout that both MMAs read (a decoded block of 8 channels is
// one 16-byte chunk; V^T is read from the same token-major layout as an
// MN-major operand, and so are the weights, a row of N per token).  The tensor cores run beside them, one tile apart:
//   decode K of tile j+1 | decode V of tile j | scores of j, vote | S of j+1
//   starts | weights of j | O of j starts | ..
// with two barriers a tile.  What bounds it is instruction issue: the decode
// (about 20 instructions a block) and four a score.
//
// M is a reference per row, moved only when an x exceeds it by kRefSlack,
// which a block-wide vote finds; O is then rescaled in TMEM.
//
// Every wait is bounded (LQ_EF_TIMEOUT after about a second; the results are
// then wrong, and later waits return at once).
#include "lq_paged_attn.cuh"

namespace lq {
namespace {

constexpr int kTok = 128;       // tokens of a tile
constexpr int kHalfBytes = kTok * 128;  // 64 channels (or weights) of a tile's tokens in fp16, 128-byte rows

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void store16(uint32_t addr, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                 : "memory");
}

// Read-only global loads that stay where they are written (the compiler would
// sink them to their use, a tile later, to save registers).
__device__ __forceinline__ uint4 load_early(const uint4 *p) {
    uint4 v;
    asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ float load_early(const float *p) {
    float v;
    asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p));
    return v;
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

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(shape), "r"((uint32_t)accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_done(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// Waits for the barrier's phase, at most about a second; false then.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t phase) {
    const long long start = clock64();
    for (;;) {
        uint32_t ok;
        asm volatile(
            "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
            : "=r"(ok)
            : "r"(bar), "r"(phase)
            : "memory");
        if (ok) return true;
        if (clock64() - start > 2000000000ll) return false;
    }
}

// C consecutive TMEM columns of the warp's 32 lanes.
template <int C>
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[C]) {
    static_assert(C % 8 == 0);
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

// Shared memory after the 1024-byte aligned operands.
template <int N>
struct Small {
    uint64_t bar_s, bar_o;
    uint32_t tmem, exponent;
    alignas(16) float minus_m[N];
    float f[N], red[4][N];
    int pages[4][8];  // of four tiles; -1: outside the pool
};

template <int D, int N>
constexpr size_t smem_bytes() {
    return 1024 + 2 * (size_t)(D / 64) * kHalfBytes + (size_t)N * D * 2 + (size_t)(N + 63) / 64 * kHalfBytes + sizeof(Small<N>);
}

// The lane order of a decoded block: position p holds channel kChannel >> 4p & 15.
constexpr uint32_t kChannel = 0x04152637u;

template <int N>
constexpr int kThreads = N <= 64 ? 256 : 512;

template <bool BF16, int D, int N>
__global__ void __launch_bounds__(kThreads<N>, N <= 16 ? 3 : N <= 64 ? 2 : 1)
    paged_attn_tc_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr int kThreads = lq::kThreads<N>;
    constexpr int W = D / 8, H = D / 64;              // words of a row, 64-channel halves
    constexpr int C = N * 128 / kThreads;             // columns of a thread
    constexpr int RPT = kTok * (W / 4) / kThreads;    // token rows a thread decodes, four words of each
    constexpr uint32_t kCols = N <= 16 ? 64 : 4 * N;  // TMEM: S^T twice and O^T
    static_assert(RPT >= 1 && kCols <= 512);
    extern __shared__ char raw[];
    char *buf = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    // V first: at D = 64 the O MMA's upper 64 rows read past it, into K (and are not used)
    const uint32_t sv = smem_u32(buf), sk = sv + H * kHalfBytes, sq = sk + H * kHalfBytes, sp = sq + N * D * 2;
    Small<N> &sm = *reinterpret_cast<Small<N> *>(buf + 2 * H * kHalfBytes + N * D * 2 + (N + 63) / 64 * kHalfBytes);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t b = blockIdx.z, rt = blockIdx.y / a.n_heads, h = blockIdx.y - rt * a.n_heads;
    const uint32_t row0 = rt * N;
    const int len = (int)paged_len(a, b);
    const int first = (int)(blockIdx.x * a.chunk), last = (int)min(first + a.chunk, (int64_t)len);
    const int drafts = len - (int)a.T;
    if (len < a.lens[b] && (blockIdx.x | blockIdx.y | tid) == 0) raise_flag(a.err, LQ_EF_PAGE);
    const int live = (int)min((uint32_t)N, a.rows - row0);
    if (first >= last) {  // nothing to read; without a split the rows are still written
        if (a.splits == 1)
            for (int e = tid; e < live * D; e += kThreads)
                paged_store<BF16, D>(a, b, h, row0 + e / D, e % D, 0.f, 0.f, kNoRef);
        return;
    }

    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)),
                     "r"(kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (tid == 0) {
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&sm.bar_s)) : "memory");
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&sm.bar_o)) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sm.exponent = 27;
    }
    for (int n = tid; n < N; n += kThreads) sm.minus_m[n] = -kNoRef;

    // ---- Q: fp16 rows in the decoded blocks' channel order; rows past the last are zero
    constexpr int kChunks = N * W;  // 16-byte chunks
    constexpr int kQ = (kChunks + kThreads - 1) / kThreads;
    uint4 q[kQ];
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
        const int e = tid + i * kThreads, n = e / W, c = e % W;
        q[i] = make_uint4(0, 0, 0, 0);
        if (e < kChunks && n < live) {
            const uint32_t r = row0 + n, qt = a.by_group.div(r), qh = h * a.group + (r - qt * a.group);
            q[i] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) + b * a.q_stride_b +
                                                         qh * a.q_stride_h + qt * a.q_stride_t) + c);
        }
    }
    float qk = a.qk_log2 * kCodeUnit;
    if constexpr (BF16) {  // a power of two for all rows puts the largest finite value in [2^10, 2^11)
        uint32_t e = 27;   // (at least 2^-100)
#pragma unroll
        for (int i = 0; i < kQ; ++i) {
            const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t lo = w[k] >> 7 & 0xffu, hi = w[k] >> 23 & 0xffu;
                e = max(e, max(lo == 0xffu ? 0u : lo, hi == 0xffu ? 0u : hi));
            }
        }
        e = __reduce_max_sync(0xffffffffu, e);
        __syncthreads();
        if (lane == 0) atomicMax(&sm.exponent, e);
        __syncthreads();
        e = sm.exponent;
        const float f = __uint_as_float((264u - e) << 23);
        qk *= __uint_as_float((e - 10u) << 23);
#pragma unroll
        for (int i = 0; i < kQ; ++i)
            q[i] = make_uint4(bf16_to_f16(q[i].x, f), bf16_to_f16(q[i].y, f), bf16_to_f16(q[i].z, f),
                              bf16_to_f16(q[i].w, f));
    }
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
        const int e = tid + i * kThreads, n = e / W, c = e % W;
        if (e >= kChunks) break;
        // pairs (7, 3), (6, 2), (5, 1), (4, 0)
        const uint32_t v[4] = {__byte_perm(q[i].w, q[i].y, 0x7632), __byte_perm(q[i].w, q[i].y, 0x5410),
                               __byte_perm(q[i].z, q[i].x, 0x7632), __byte_perm(q[i].z, q[i].x, 0x5410)};
        store16(sq + (c >> 3) * (N * 128) + n * 128 + (((c & 7) ^ (n & 7)) << 4), v);
    }

    // ---- what this thread reads of a tile: RPT rows of four words each of K and V, the scales of its token
    constexpr int kPerRow = W / 4;  // threads of a row
    constexpr int kRowStep = kThreads / kPerRow;
    const int part = tid % kPerRow, drow = tid / kPerRow;
    const int tl = (warp & 3) * 32 + lane;  // the token (TMEM lane) whose scores it handles
    const int col0 = (warp >> 2) * C;
    const int32_t *table = a.table + b * a.table_stride;
    const int64_t side = (int64_t)a.n_heads << a.page_log2;
    const uint32_t *kbase = a.codes + ((int64_t)h << a.page_log2) * W + part * 4;
    const float *sbase = a.scales + ((int64_t)h << a.page_log2);
    const int page_mask = (1 << a.page_log2) - 1;
    // Entry i of a tile's pages (0 where it has none); kept in the ring as -1 where it lies outside the
    // pool: reported, read as page 0, its tokens masked.
    auto page_entry = [&](int t0, int i) {
        const int tok = ((t0 >> a.page_log2) + i) << a.page_log2;
        return max(tok, t0) < min(t0 + kTok, last) ? __ldg(table + (tok >> a.page_log2)) : 0;
    };
    auto keep_entry = [&](int t0, int i, int page) {
        if ((uint32_t)page >= (uint32_t)a.n_pages) {
            raise_flag(a.err, LQ_EF_PAGE);
            page = -1;
        }
        sm.pages[t0 >> 7 & 3][i] = page;
    };
    auto page_of = [&](int t0, int i) {  // of token i of the tile at t0
        return sm.pages[t0 >> 7 & 3][(((t0 & page_mask) + i) >> a.page_log2) & 7];
    };
    auto row_of = [&](int t0, int i) {
        return 2 * side * max(page_of(t0, i), 0) + ((t0 + i) & page_mask);
    };
    uint4 kw[RPT], vw[RPT];
    float ks, vs;
    bool bad;
    // K of the tile at tk, V and scales of the one at tv: all page lookups, then all loads (a lookup
    // behind a load in flight would wait for it)
    auto fetch = [&](int tk, int tv) {
        int64_t rk[RPT], rv[RPT];
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
            rk[r] = tk < last ? row_of(tk, drow + r * kRowStep) : 0;
            rv[r] = tv < last ? row_of(tv, drow + r * kRowStep) : 0;
        }
        const int64_t rs = tv < last ? row_of(tv, tl) : 0;
        bad = tv < last && page_of(tv, tl) < 0;
#pragma unroll
        for (int r = 0; r < RPT; ++r) kw[r] = load_early(reinterpret_cast<const uint4 *>(kbase + rk[r] * W));
#pragma unroll
        for (int r = 0; r < RPT; ++r) vw[r] = load_early(reinterpret_cast<const uint4 *>(kbase + (rv[r] + side) * W));
        ks = load_early(sbase + rs);
        vs = load_early(sbase + rs + side);
    };
    // Decoded rows into an operand.  At D = 128 the two 64-channel halves fall on the same banks, so the
    // threads of the upper one take their words in the order 2, 3, 0, 1.
    const bool upper = D == 128 && part >= 2;
    uint32_t chunk_at[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        chunk_at[j] = (D == 128 ? (part >> 1) * kHalfBytes : 0) + drow * 128 +
                      (((((part & 1) * 4 + j) ^ (upper ? 2 : 0)) ^ (drow & 7)) << 4);
    auto put = [&](uint32_t dst, const uint4 (&w)[RPT]) {
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
            const uint32_t v[4] = {upper ? w[r].z : w[r].x, upper ? w[r].w : w[r].y, upper ? w[r].x : w[r].z,
                                   upper ? w[r].y : w[r].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t pair[4];
                decode_block(v[j], pair);
                store16(dst + chunk_at[j] + r * (kRowStep * 128), pair);
            }
        }
    };
    static_assert(kRowStep % 8 == 0);  // the rows of a thread share their swizzle

    if (tid < 24) keep_entry(first + tid / 8 * kTok, tid % 8, page_entry(first + tid / 8 * kTok, tid % 8));
    int entry = tid < 8 ? page_entry(first + 3 * kTok, tid) : 0;  // on its way to the ring
    __syncthreads();
    fetch(first, first);
    put(sk, kw);
    fetch(first + kTok, first);
    publish_smem();
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t ts = sm.tmem, to = ts + 2 * N, my_lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t bar_s = smem_u32(&sm.bar_s), bar_o = smem_u32(&sm.bar_o);
    const uint64_t dk = operand(sk, 16, 1024), dq = operand(sq, 16, 1024), dp = operand(sp, kHalfBytes, 1024),
                   dv = operand(sv, kHalfBytes, 1024);
    auto start_scores = [&](uint32_t to_s) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            const uint32_t in = (k & 3) * 2;  // 32 bytes on within the swizzled rows
            mma(to_s, dk + (k >> 2) * (kHalfBytes >> 4) + in, dq + (k >> 2) * (N * 128 >> 4) + in, kShape<N>, k > 0);
        }
        mma_done(bar_s);
    };
    if (tid == 0) start_scores(ts);

    unsigned long long l[C / 2];  // of two columns each, as packed fp32
#pragma unroll
    for (int c = 0; c < C / 2; ++c) l[c] = 0;
    bool alive = true;
    uint32_t phase = 0;  // of both barriers, per tile; also the tile's S^T
    for (int t0 = first; t0 < last; t0 += kTok, phase ^= 1) {
        const bool more = t0 + kTok < last;
        const uint32_t s_now = ts + phase * N;
        alive = alive && wait_for(bar_s, phase);  // S is there, K's buffer free
        tmem_fence_after();
        if (more) put(sk, kw);
        if (t0 > first) alive = alive && wait_for(bar_o, phase ^ 1);  // V's and W's buffers are free
        put(sv, vw);
        const int tok = t0 + tl;
        const bool past = tok >= last || bad;
        const float kx = ks * qk, lv = lg2(vs), rvs = past ? 0.f : rcp(vs);
        fetch(t0 + 2 * kTok, t0 + kTok);
        if (tid < 8) {  // pages of the tile after the next two (read after this tile's barriers)
            keep_entry(t0 + 3 * kTok, tid, entry);
            entry = page_entry(t0 + 4 * kTok, tid);
        }

        uint32_t hidden = past ? 0xffffffffu : 0u;  // columns that do not see the token
        if (tok >= drafts && !past)
#pragma unroll 1
            for (uint32_t c = 0; c < C && row0 + col0 + c < a.rows; ++c)
                hidden |= (uint32_t)!paged_sees(a, b, a.by_group.div(row0 + col0 + c), tok - drafts) << c;
        float x[C];
        auto scores = [&]() {
            tmem_load<C>(s_now + my_lanes + col0, x);
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
                const float4 m = *reinterpret_cast<const float4 *>(sm.minus_m + col0 + c);
                f2_unpack(f2_add(f2_pack(x[c], x[c + 1]), f2_pack(m.x, m.y)), x[c], x[c + 1]);
                f2_unpack(f2_add(f2_pack(x[c + 2], x[c + 3]), f2_pack(m.z, m.w)), x[c + 2], x[c + 3]);
                top = fmaxf(fmaxf(fmaxf(top, x[c]), fmaxf(x[c + 1], x[c + 2])), x[c + 3]);
            }
            return top > kRefSlack;
        };
        scores();
        const bool grow = less_reference();
        publish_smem();
        tmem_fence_before();
        const bool move = __syncthreads_or(grow);
        if (tid == 0 && more) {
            tmem_fence_after();
            start_scores(ts + (phase ^ 1) * N);
        }
        if (move) {
            // the tile's column maxima move the references; l and O follow
            scores();
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float top = x[c];
#pragma unroll
                for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                if (lane == 0) sm.red[warp & 3][col0 + c] = top;
            }
            __syncthreads();
            for (int n = tid; n < N; n += kThreads) {
                const float top = fmaxf(fmaxf(sm.red[0][n], sm.red[1][n]), fmaxf(sm.red[2][n], sm.red[3][n]));
                const float m = -sm.minus_m[n], next = fmaxf(m, top);
                sm.f[n] = ex2(m - next);
                sm.minus_m[n] = -next;
            }
            __syncthreads();
            less_reference();
#pragma unroll
            for (int c = 0; c < C; c += 2) l[c / 2] = f2_mul(l[c / 2], f2_pack(sm.f[col0 + c], sm.f[col0 + c + 1]));
            if (t0 > first) {  // this warp's lanes (channels) and columns of O; its MMAs are done
                float o[C];
                tmem_load<C>(to + my_lanes + col0, o);
#pragma unroll
                for (int c = 0; c < C; ++c) o[c] *= sm.f[col0 + c];
                tmem_store<C>(to + my_lanes + col0, o);
            }
        }
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
            store16(sp + (n >> 6) * kHalfBytes + tl * 128 + (((n >> 3 & 7) ^ (tl & 7)) << 4), pair);
        }
        publish_smem();
        tmem_fence_before();
        __syncthreads();
        if (tid == 0) {
            tmem_fence_after();
#pragma unroll
            for (int k = 0; k < kTok / 16; ++k)
                mma(to, dv + k * (2048 >> 4), dp + k * (2048 >> 4), kShape<N> | kTransposeA | kTransposeB,
                    t0 > first || k > 0);
            mma_done(bar_o);
        }
    }
    alive = alive && wait_for(bar_o, phase ^ 1);
    tmem_fence_after();
    if (!alive) raise_flag(a.err, LQ_EF_TIMEOUT);

    // denominators over the 128 tokens, then O: a lane is a channel
#pragma unroll
    for (int c = 0; c < C; ++c) {
        float l0, l1;
        f2_unpack(l[c / 2], l0, l1);
        float sum = c & 1 ? l1 : l0;
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) sm.red[warp & 3][col0 + c] = sum;
    }
    float o[C];
    tmem_load<C>(to + my_lanes + col0, o);
    // through shared memory (the operands are done with) to rows of channels
    float *rows = reinterpret_cast<float *>(buf);
    const int d = (tl & ~7) + (int)(kChannel >> (4 * (tl & 7)) & 15u);
    if (D == 128 || tl < 64)
#pragma unroll
        for (int c = 0; c < C; ++c) rows[(col0 + c) * D + d] = o[c];
    __syncthreads();
    for (int e = tid; e < live * D; e += kThreads) {
        const int n = e / D;
        const float den = (sm.red[0][n] + sm.red[1][n]) + (sm.red[2][n] + sm.red[3][n]);
        paged_emit<BF16, D>(a, b, h, row0 + n, e % D, blockIdx.x, rows[e], den, -sm.minus_m[n]);
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == 0)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(ts), "r"(kCols) : "memory");
}

template <bool BF16, int D, int N>
int launch_n(const PagedAttnArgs &a, uint32_t batch, cudaStream_t st) {
    constexpr size_t smem = smem_bytes<D, N>();
    if (cudaFuncSetAttribute(paged_attn_tc_kernel<BF16, D, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
        cudaSuccess)
        return LQ_ERR_CUDA;
    paged_attn_tc_kernel<BF16, D, N>
        <<<dim3(a.splits, a.n_heads * (uint32_t)ceil_div(a.rows, N), batch), kThreads<N>, smem, st>>>(a);
    return check_launch();
}

template <bool BF16, int D>
int launch_d(const PagedAttnArgs &a, int tile, uint32_t batch, cudaStream_t st) {
    if (tile == 16) return launch_n<BF16, D, 16>(a, batch, st);
    if (tile == 32) return launch_n<BF16, D, 32>(a, batch, st);
    if constexpr (D == 128)
        if (tile == 128) return launch_n<BF16, D, 128>(a, batch, st);
    return launch_n<BF16, D, 64>(a, batch, st);
}

}  // namespace

int launch_paged_tc(const PagedAttnArgs &a, bool bf16, int head_dim, int tile, uint32_t batch, cudaStream_t st) {
    if (bf16) return head_dim == 128 ? launch_d<true, 128>(a, tile, batch, st) : launch_d<true, 64>(a, tile, batch, st);
    return head_dim == 128 ? launch_d<false, 128>(a, tile, batch, st) : launch_d<false, 64>(a, tile, batch, st);
}

}  // namespace lq
