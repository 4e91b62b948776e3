// lq_paged_attn.cu -- attention of a block of query positions over the pages
// of an E8 cache, on warp-level tensor-core instructions.
//
// For every sequence b, query head hq = h * G + g and position t < T:
//   o = softmax(q . K^T * sm_scale) V  over the tokens p < len[b] that t sees:
//   all of the context (p < len - T) and, of the last T tokens (the drafts),
//   those whose mask[t][p - (len - T)] is set (without a mask: drafts <= t).
// The reference has no counterpart: its decode attends one position over the
// dequantised buffer (llm/compressed_kv_cache.py:342-395).
//
// Mathematics.  A query row r = t * G + g; the tile of a warp is 16 tokens by
// 8 rows.  Scores S = K Q^T put tokens on the rows of the MMA, so a
// lane's A registers are whole code words of "its" two tokens, decoded in
// registers to fp16, which holds every point exactly.  A bf16 query becomes
// fp16 times a power of two of its row (its largest value then lies in
// [2^10, 2^11); what falls under fp16's smallest step is 2^-35 of that), and
// the token's and the row's factors multiply the fp32 score.  V's scale goes into the exponent:
//   x = s * log2(e) * sm_scale * ks + log2(vs),  w = 2^(x - M),
//   o += w * point,  l += w / vs
// so the fp16 weights w stay within 2^15 whatever the scales are.  M is a
// reference, not the running maximum: it moves (to the maximum less 4) only
// when an x exceeds it by 15, which a warp vote finds; the statistics are then
// rescaled.  (x is one fp32 number: beyond scores of about 1e4 its rounding
// reaches that of the fp16 weights, and beyond 1e7 log2(vs) is lost in it, which
// shows where keys are equal; a row whose scores all lie under -1e30 counts as
// seeing nothing.)  W^T reaches its B registers with one 8x8 transpose per 8
// tokens; V's A registers pair two tokens' decoded channels by byte permutes.
//
// Registers feed the MMAs, no shared memory: with 8 rows a tile's MMAs are few,
// and what bounds the kernel is issue, most of it the decode (489 instructions a
// warp and tile of 16 tokens; 66% of issue slots, the integer ALU over half).
// The next tile's words load into the registers that this tile's were decoded
// from.  32 sequences of 16,384 tokens, 8 KV heads of 128, 4 query heads each:
// 195 us, 2.9 TB/s; 1 sequence of 777 tokens: 6.3 us.
#include "lq_paged.cuh"
#include "lq_paged_attn.cuh"

namespace lq {
namespace {

constexpr int kWarps = 4;
constexpr int kTileRows = 8;  // query rows of a CTA

__device__ __forceinline__ void mma_16816(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <int N>
__device__ __forceinline__ void load_words(const uint32_t *p, uint32_t w[N]) {
    if constexpr (N == 4) {
        const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p));
        w[0] = u.x;
        w[1] = u.y;
        w[2] = u.z;
        w[3] = u.w;
    } else if constexpr (N == 2) {
        const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p));
        w[0] = u.x;
        w[1] = u.y;
    } else {
        w[0] = __ldg(p);
    }
}

// The CTAs of a cluster: a barrier that also orders their shared memory, and reads of another's.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_cta(const void *p, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}
template <int N>
__device__ __forceinline__ void load_cluster(uint32_t addr, float (&v)[N]) {
    if constexpr (N == 4)
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
                     : "r"(addr)
                     : "memory");
    else
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(addr) : "memory");
}

// What a lane (g = lane / 4, t = lane % 4) reads of a 16-token tile: K words
// t*KW.. of tokens g and g + 8, V words g*VW.. of tokens 2t, 2t+1, 2t+8,
// 2t+9, and the scales of tokens g and g + 8.
template <int D>
struct Tile {
    static constexpr int KW = D / 32, VW = D / 64;
    uint32_t k[2][KW], v[4][VW];
    float ks[2], vs[2];
};

// Where a tile's rows are: the K words, V words and scales of its first token.
struct TileAt {
    const uint32_t *k, *v;
    const float *ks, *vs;
};

template <int D>
__device__ __forceinline__ void load_k(const TileAt &at, uint32_t g, uint32_t t, Tile<D> &x) {
#pragma unroll
    for (int r = 0; r < 2; ++r) load_words<Tile<D>::KW>(at.k + (g + 8 * r) * (D / 8) + t * Tile<D>::KW, x.k[r]);
}
template <int D>
__device__ __forceinline__ void load_scales(const TileAt &at, uint32_t g, Tile<D> &x) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        x.ks[r] = __ldg(at.ks + g + 8 * r);
        x.vs[r] = __ldg(at.vs + g + 8 * r);
    }
}
template <int D>
__device__ __forceinline__ void load_v(const TileAt &at, uint32_t g, uint32_t t, Tile<D> &x) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        load_words<Tile<D>::VW>(at.v + (2 * t + (i & 1) + 8 * (i >> 1)) * (D / 8) + g * Tile<D>::VW, x.v[i]);
}

// v[block][half]: tokens 2t, 2t+1 (+ 8 half) of this lane's blocks
template <int D, int S>
__device__ __forceinline__ void pv_step(const TokenPair v[D / 64][2], const uint32_t (&p)[2], float (*o)[4]) {
    if constexpr (D == 128) {
        uint32_t a[4], b[4];  // [block + 2 half] of the pair's two channels
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int half = 0; half < 2; ++half) decode_pair<S>(v[blk][half], a[blk + 2 * half], b[blk + 2 * half]);
        mma_16816(o[S], a[0], a[1], a[2], a[3], p[0], p[1]);
        mma_16816(o[4 + S], b[0], b[1], b[2], b[3], p[0], p[1]);
    } else {
        uint32_t a[4];  // one block: its two channels are the MMA's two row groups
#pragma unroll
        for (int half = 0; half < 2; ++half) decode_pair<S>(v[0][half], a[2 * half], a[1 + 2 * half]);
        mma_16816(o[S], a[0], a[1], a[2], a[3], p[0], p[1]);
    }
}

// grid (splits, n_heads * row tiles, batch); a CTA's warps take the 16-token
// tiles of its chunk in turn.
template <bool BF16, int D>
__global__ void __launch_bounds__(32 * kWarps, 4) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr int KW = D / 32, VW = D / 64, W = D / 8, MT = D / 16;
    extern __shared__ __align__(16) float sm[];  // [warps][kTileRows][D + 4]
    const int warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t b = blockIdx.z, rt = blockIdx.y / a.n_heads, h = blockIdx.y - rt * a.n_heads;
    const uint32_t row0 = rt * kTileRows;
    // positions fit 32 bits: a table is at most 2^20 pages of 2^8 tokens
    const int len = (int)paged_len(a, b);
    const int first = (int)(blockIdx.x * a.chunk), last = paged_split_end(a, first, len);
    const int drafts = len - (int)a.T;  // position of draft 0
    if (len < a.lens[b] && (blockIdx.x | blockIdx.y | threadIdx.x) == 0) raise_flag(a.err, LQ_EF_PAGE);

    // Q's B registers: row lane / 4, this lane's blocks
    uint32_t qf[KW * 4];
    float qk[2];  // what a score of the lane's rows 2t, 2t + 1 is multiplied by
    const uint32_t r = row0 + g;
    const bool in = r < a.rows;
    const uint32_t qt = in ? a.by_group.div(r) : 0, qh = h * a.group + (in ? r - qt * a.group : 0);
    const uint4 *qp = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) + b * a.q_stride_b +
                                                      qh * a.q_stride_h + qt * a.q_stride_t);
    uint4 u[KW];
#pragma unroll
    for (int j = 0; j < KW; ++j) u[j] = in ? __ldg(qp + t * KW + j) : make_uint4(0, 0, 0, 0);
    float back = a.qk_log2 * kCodeUnit;
    if constexpr (BF16) {
        uint32_t e = 0;  // the row's largest finite exponent
#pragma unroll
        for (int j = 0; j < KW; ++j) {
            const uint32_t w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t lo = w[i] >> 7 & 0xffu, hi = w[i] >> 23 & 0xffu;
                e = max(e, max(lo == 0xffu ? 0u : lo, hi == 0xffu ? 0u : hi));
            }
        }
        e = max(e, __shfl_xor_sync(0xffffffffu, e, 1));
        e = max(e, __shfl_xor_sync(0xffffffffu, e, 2));
        e = max(e, 27u);  // rows under 2^-100 count as 2^-100
        const float f = __uint_as_float((264u - e) << 23);  // 2^(10 - (e - 127))
        back *= __uint_as_float((e - 10u) << 23);           // 1 / f
#pragma unroll
        for (int j = 0; j < KW; ++j)
            u[j] = make_uint4(bf16_to_f16(u[j].x, f), bf16_to_f16(u[j].y, f), bf16_to_f16(u[j].z, f),
                              bf16_to_f16(u[j].w, f));
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) qk[c] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + c));
#pragma unroll
    for (int j = 0; j < KW; ++j) {  // decode_block's pair s: channels 7 - s, 3 - s
        qf[4 * j + 0] = __byte_perm(u[j].w, u[j].y, 0x7632);
        qf[4 * j + 1] = __byte_perm(u[j].w, u[j].y, 0x5410);
        qf[4 * j + 2] = __byte_perm(u[j].z, u[j].x, 0x7632);
        qf[4 * j + 3] = __byte_perm(u[j].z, u[j].x, 0x5410);
    }

    float o[MT][4], l[2], m[2];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[i][c] = 0.f;
    l[0] = l[1] = 0.f;
    m[0] = m[1] = kNoRef;

    const int32_t *table = a.table + b * a.table_stride;
    const uint32_t *kbase = a.codes + ((int64_t)h << a.page_log2) * W;
    const float *sbase = a.scales + ((int64_t)h << a.page_log2);
    const int64_t side = (int64_t)a.n_heads << a.page_log2;
    const int page_mask = (1 << a.page_log2) - 1, n_pages = (int)a.n_pages;
    constexpr int kStep = 16 * kWarps;
    // a table entry outside the pool is reported, and read as page 0 with its tokens masked
    auto page_of = [&](int tok) { return tok < last ? __ldg(table + (tok >> a.page_log2)) : 0; };
    auto usable = [&](int page) { return (uint32_t)page < (uint32_t)n_pages; };
    auto locate = [&](int tok, int page) {
        const int64_t row = 2 * side * (usable(page) ? page : 0) + (tok & page_mask);
        const uint32_t *k = kbase + row * W;
        return TileAt{k, k + side * W, sbase + row, sbase + row + side};
    };

    int page = page_of(first + 16 * warp), page_nx = page_of(first + 16 * warp + kStep);
    Tile<D> x;
    if (first + 16 * warp < last) {
        const TileAt at = locate(first + 16 * warp, page);
        load_k<D>(at, g, t, x);
        load_scales<D>(at, g, x);
        load_v<D>(at, g, t, x);
    }
    for (int tok = first + 16 * warp; tok < last; tok += kStep) {
        // the next tile's words load into x as soon as this one's are decoded
        const bool bad = !usable(page), more = tok + kStep < last;
        const TileAt next = locate(tok + kStep, page_nx);
        page = page_nx;
        page_nx = page_of(tok + 2 * kStep);

        float s[4] = {};
#pragma unroll
        for (int j = 0; j < KW; ++j) {
            uint32_t k0[4], k1[4];
            decode_block(x.k[0][j], k0);
            decode_block(x.k[1][j], k1);
            mma_16816(s, k0[0], k1[0], k0[1], k1[1], qf[4 * j], qf[4 * j + 1]);
            mma_16816(s, k0[2], k1[2], k0[3], k1[3], qf[4 * j + 2], qf[4 * j + 3]);
        }

        if (more) load_k<D>(next, g, t, x);

        // x = s * ks + log2(vs), and 1 / vs for the denominator
        float rvs[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float lv = lg2(x.vs[r]);
            rvs[r] = rcp(x.vs[r]);
            s[2 * r] = fmaf(s[2 * r], x.ks[r] * qk[0], lv);
            s[2 * r + 1] = fmaf(s[2 * r + 1], x.ks[r] * qk[1], lv);
        }
        if (more) load_scales<D>(next, g, x);
        if (tok + 16 > drafts || bad) {  // drafts, tokens past the end: whole warp
            if (bad && lane == 0) raise_flag(a.err, LQ_EF_PAGE);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int p = tok + (int)g + 8 * r;
                const bool past = p >= last || bad;
                if (past) rvs[r] = 0.f;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t row = row0 + 2 * t + c;
                    if (past || (p >= drafts && row < a.rows && !paged_sees(a, b, a.by_group.div(row), p - drafts)))
                        s[2 * r + c] = -INFINITY;
                }
            }
        }

        bool grow = false;
#pragma unroll
        for (int c = 0; c < 2; ++c) grow |= fmaxf(s[c], s[2 + c]) > m[c] + kRefSlack;
        if (__any_sync(0xffffffffu, grow)) {
            // V vectors of zeros move no reference.  A lane holds blocks of four tokens, and the lanes of its t their others.
            uint32_t zero[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bool z = true;
#pragma unroll
                for (int j = 0; j < VW; ++j) z = z && x.v[i][j] == kZeroWord;
                zero[i] = __ballot_sync(0xffffffffu, z);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {  // token g + 8r is the (g & 1)-th of half r for the lanes with t = g / 2
                const uint32_t all = (g & 1 ? zero[2 * r + 1] : zero[2 * r]) >> (g >> 1) & 0x11111111u;
                if (all == 0x11111111u) {
                    rvs[r] *= kZeroInv;
                    s[2 * r] += kZeroLog2;
                    s[2 * r + 1] += kZeroLog2;
                }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float mx = fmaxf(s[c], s[2 + c]);
#pragma unroll
                for (int off = 4; off <= 16; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                const float mn = fmaxf(m[c], mx - kRefBelow);
                const float f = exp2f(m[c] - mn);
                m[c] = mn;
                l[c] *= f;
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    o[i][c] *= f;
                    o[i][2 + c] *= f;
                }
            }
        }

        uint32_t p[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float w0 = ex2(s[2 * r] - m[0]), w1 = ex2(s[2 * r + 1] - m[1]);
            l[0] = fmaf(w0, rvs[r], l[0]);
            l[1] = fmaf(w1, rvs[r], l[1]);
            const __half2 hw = __floats2half2_rn(w0, w1);
            p[r] = transpose_8x8(*reinterpret_cast<const uint32_t *>(&hw));
        }

        TokenPair v[VW][2];
#pragma unroll
        for (int j = 0; j < VW; ++j)
#pragma unroll
            for (int half = 0; half < 2; ++half) v[j][half] = pair_tokens(x.v[2 * half][j], x.v[2 * half + 1][j]);
        if (more) load_v<D>(next, g, t, x);
        pv_step<D, 0>(v, p, o);
        pv_step<D, 1>(v, p, o);
        pv_step<D, 2>(v, p, o);
        pv_step<D, 3>(v, p, o);
    }

    // the warps' statistics and outputs, merged in warp order
    constexpr int rs = D + 4;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) l[c] += __shfl_xor_sync(0xffffffffu, l[c], off);
        float *dst = sm + (warp * kTileRows + 2 * t + c) * rs;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if constexpr (D == 128) {  // tile i: channel 7 - i of blocks 2g and 2g + 1
                dst[16 * g + 7 - i] = o[i][c];
                dst[16 * g + 15 - i] = o[i][2 + c];
            } else {  // tile i: channels 7 - i and 3 - i of block g
                dst[8 * g + 7 - i] = o[i][c];
                dst[8 * g + 3 - i] = o[i][2 + c];
            }
        }
        if (g == 0) {
            dst[D] = m[c];
            dst[D + 1] = l[c];
        }
    }
    // rows in turn to the warps of the CTA, or of the cluster, whose CTAs are then the splits
    const uint32_t ranks = a.clustered ? a.splits : 1, rank = a.clustered ? blockIdx.x : 0;
    if (a.clustered) cluster_sync();
    else __syncthreads();
    for (uint32_t r = rank + ranks * warp; r < min((uint32_t)kTileRows, a.rows - row0); r += ranks * kWarps) {
        float mx = kNoRef, ld = 0.f, od[D / 32] = {};
        for (uint32_t p = lane; p < ranks * kWarps; p += 32) {
            float st[2];
            load_cluster(in_cta(sm + ((p % kWarps) * kTileRows + r) * rs + D, p / kWarps), st);
            mx = fmaxf(mx, st[0]);
        }
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        for (uint32_t q = 0; q < ranks; ++q) {
            const uint32_t base = in_cta(sm + r * rs, q);
            float st[kWarps][2], v[kWarps][D / 32];
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                load_cluster(base + (w * kTileRows * rs + D) * 4, st[w]);
                load_cluster(base + (w * kTileRows * rs + lane * (D / 32)) * 4, v[w]);
            }
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = ex2(st[w][0] - mx);
                ld = fmaf(st[w][1], f, ld);
#pragma unroll
                for (int k = 0; k < D / 32; ++k) od[k] = fmaf(v[w][k], f, od[k]);
            }
        }
        if (a.clustered) paged_store_row<BF16, D>(a, b, h, row0 + r, od, ld, mx);
        else paged_emit_row<BF16, D>(a, b, h, row0 + r, blockIdx.x, od, ld, mx);
    }
    if (a.clustered) cluster_sync();  // nobody leaves while its shared memory is read
}

// A warp per row: the splits' partial results joined in split order.
template <bool BF16, int D>
__global__ void __launch_bounds__(128) paged_combine_kernel(const __grid_constant__ PagedAttnArgs a, uint32_t n_rows) {
    const uint32_t i = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (i >= n_rows) return;
    after_previous();
    const uint32_t bh = i / a.rows, r = i - bh * a.rows;
    const uint32_t b = bh / a.n_heads, h = bh - b * a.n_heads;
    const float *p = paged_part<D>(a, bh, 0);
    const int64_t step = (int64_t)a.rows * (D + 4);
    const uint32_t used = min((uint32_t)ceil_div(paged_len(a, b), a.chunk), a.splits);
    float m = kNoRef;
    for (uint32_t s = lane; s < used; s += 32) m = fmaxf(m, p[s * step + (int64_t)a.rows * D + 2 * r]);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float l = 0.f, od[D / 32] = {};
#pragma unroll 4
    for (uint32_t s = 0; s < used; ++s) {
        const float *q = p + s * step;
        const float2 st = *reinterpret_cast<const float2 *>(q + (int64_t)a.rows * D + 2 * r);
        const float f = ex2(st.x - m);
        l = fmaf(st.y, f, l);
        float v[D / 32];
        if constexpr (D == 128) {
            const float4 x = *reinterpret_cast<const float4 *>(q + (int64_t)r * D + lane * 4);
            v[0] = x.x;
            v[1] = x.y;
            v[2] = x.z;
            v[3] = x.w;
        } else {
            const float2 x = *reinterpret_cast<const float2 *>(q + (int64_t)r * D + lane * 2);
            v[0] = x.x;
            v[1] = x.y;
        }
#pragma unroll
        for (int k = 0; k < D / 32; ++k) od[k] = fmaf(v[k], f, od[k]);
    }
    paged_store_row<BF16, D>(a, b, h, r, od, l, m);
}

template <bool BF16, int D>
int launch_dim(const PagedAttnArgs &a, int tile, uint32_t batch, cudaStream_t st) {
    int status;
    if (tile == kTileRows) {
        const dim3 grid(a.splits, a.n_heads * (uint32_t)ceil_div(a.rows, kTileRows), batch);
        status = launch_clustered(paged_attn_kernel<BF16, D>, grid, a.clustered ? a.splits : 1, 32 * kWarps,
                                  kWarps * kTileRows * (D + 4) * 4, st, a);
    } else {
        status = launch_paged_tc(a, BF16, D, tile, batch, st);
    }
    if (status != LQ_OK || a.splits == 1 || a.clustered) return status;
    const uint32_t n = batch * a.n_heads * a.rows;
    return launch_overlapped(paged_combine_kernel<BF16, D>, dim3((unsigned)ceil_div(n, 4)), 128, 0, st, a, n);
}

// The kernel, its rows a CTA and the tokens of a split.
//
// Few rows go to the kernel of this file, the others to tcgen05.  A row tile
// takes the decode again, so 16 rows of 128 channels are slower here (us, this
// kernel : tcgen05; 8 KV heads): 379 : 245 for 32 x 16,384 tokens and 25 : 22 for 8 x
// 2,048, where 8 rows are 197 : 241 for the first.  64 channels give a tile half the
// decode: 16 rows 244 : 296 (32 x 16,384), 39.1 : 56.6 (8 x 8,192) and 9.9 : 14.7
// (4 x 2,048); against a form of 16 columns, no longer here, 243 : 243, 38.8 : 46.0
// and 9.5 : 12.0.  24 rows are 340 : 250, 50.3 : 50.4 and 15.8 : 14.8.
//
// The CTAs of a call come in rounds of as many as the GPU holds, so the number
// of splits is the one whose rounds times a CTA's time (its tiles, and
// kStartTiles tiles' worth of start and end) is smallest, among those that fill
// two rounds where the tokens allow chunks of kShortest tiles, for lengths that
// differ from the bound.  (Tree of 13 over
// 16 sequences of up to 8,190 tokens, mean over eight draws of their lengths:
// no such floor 92.7 us, one round 83.1, two 75.2, three 74.9, five 83.4; tree
// of 64 over 4 x 32,768 tokens: 5 splits 303 us, 6 318, 4 365.)
// Up to kClusterMax splits of the few-rows kernel form a cluster and join over
// its shared memory, which spares the second launch and the workspace; short
// contexts take fewer splits for it than would fill the GPU.
struct Plan {
    int tile;
    int64_t chunk;
    uint32_t splits;
    bool clustered;
};
constexpr int64_t kClusterMax = 8, kClusterTokens = 256;  // splits, and the chunk up to which 8 of them are enough
constexpr int64_t kStartTiles = 3, kShortest = 4, kMostSplits = 512, kMostRounds = 16;

// What a plan starts from.
struct Work {
    bool few;
    int tile;
    int64_t tile_tokens, slots, units, tokens, tiles;  // units: CTAs without a split
    int64_t most;                                      // splits looked at: past this there are only more starts
    Work(int64_t batch, int n_heads, int64_t rows, int head_dim, int64_t max_len) {
        few = rows <= (head_dim == 64 ? 16 : 8);
        tile = few ? kTileRows : rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
        tile_tokens = few ? 64 : 128;
        slots = 148 * (few ? 4 : 1);
        units = batch * n_heads * ceil_div(rows, tile);
        tokens = max_len < 1 ? 1 : max_len;
        tiles = ceil_div(tokens, tile_tokens);
        most = kMostRounds * slots / units + 1;
        most = most < kMostSplits ? most : kMostSplits;
        most = most < tiles ? most : tiles;
    }
};

Plan plan(int64_t batch, int n_heads, int64_t rows, int head_dim, int64_t max_len) {
    const auto [few, tile, tile_tokens, slots, units, tokens, tiles, most] = Work(batch, n_heads, rows, head_dim, max_len);
    Plan p;
    p.tile = tile;
    int64_t best = 0, best_cost = INT64_MAX;
    for (int64_t s = 1; s <= most; ++s) {
        const int64_t each = ceil_div(tiles, s);
        if (ceil_div(tiles, each) != s) continue;  // no such split
        if (units * s < 2 * slots && each > kShortest && s < kMostSplits && s < tiles) continue;
        const int64_t cost = ceil_div(units * s, slots) * (each + kStartTiles);
        if (cost < best_cost) {
            best_cost = cost;
            best = each;
        }
    }
    if (best == 0) best = ceil_div(tiles, kMostSplits);
    p.chunk = best * tile_tokens;
    p.splits = (uint32_t)ceil_div(tokens, p.chunk);
    p.clustered = few && p.splits > 1 && (p.splits <= kClusterMax || tokens <= kClusterMax * kClusterTokens);
    if (p.clustered) {  // 2, 4 or 8 CTAs (the last may find nothing to do)
        p.splits = p.splits <= 2 ? 2 : p.splits <= 4 ? 4 : 8;
        p.chunk = ceil_div(ceil_div(tokens, p.splits), tile_tokens) * tile_tokens;
    }
    return p;
}

size_t workspace_of(const Plan &p, int64_t bh_rows, int head_dim) {
    return p.splits > 1 && !p.clustered ? (size_t)bh_rows * p.splits * (head_dim + 4) * 4 : 0;
}

// What no plan for these or fewer tokens goes beyond.  The splits that plan() takes are not monotone in the length, but
// the most that it looks at are.
size_t workspace_bound(int64_t batch, int n_heads, int64_t rows, int head_dim, int64_t max_len) {
    const Work w(batch, n_heads, rows, head_dim, max_len);
    const bool clustered = w.few && (w.most <= kClusterMax || w.tokens <= kClusterMax * kClusterTokens);
    return w.most > 1 && !clustered ? (size_t)(batch * n_heads * rows) * w.most * (head_dim + 4) * 4 : 0;
}

}  // namespace
}  // namespace lq

using namespace lq;

static bool paged_shape_ok(int64_t batch, int n_heads, int group, int64_t n_query, int head_dim) {
    return batch >= 0 && batch <= 65535 && n_heads >= 1 && n_heads <= 1024 && group >= 1 && group <= 64 && n_query >= 1 &&
           n_query <= 4096 && paged_dim_ok(head_dim) && n_heads * ceil_div(n_query * group, 8) <= 65535 &&
           batch * n_heads * n_query * group <= 0x7fffffff;
}

extern "C" size_t lq_paged_attention_workspace(int64_t batch, int n_heads, int group, int64_t n_query, int head_dim,
                                               int64_t max_len) {
    if (!paged_shape_ok(batch, n_heads, group, n_query, head_dim) || batch == 0 || max_len < 0) return 0;
    return workspace_bound(batch, n_heads, n_query * group, head_dim, max_len);
}

extern "C" int lq_paged_attention(const void *q, int q_dtype, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t,
                                  const int32_t *codes, const float *scales, int64_t n_pages, int page_tokens,
                                  const int32_t *table, int64_t table_width, int64_t table_stride, const int32_t *lens,
                                  int64_t max_len, const uint8_t *mask, int64_t mask_stride_b, int64_t batch,
                                  int n_heads, int group, int64_t n_query, int head_dim, float sm_scale, void *out,
                                  float *lse, void *workspace, size_t workspace_bytes, uint32_t *err, void *stream) {
    LQ_NVTX_RANGE();
    if (!paged_shape_ok(batch, n_heads, group, n_query, head_dim) || !paged_page_ok(page_tokens) || n_pages < 1 ||
        n_pages > 0x7fffffff || table_width < 0 || table_width > (1 << 20) || max_len < 0 ||
        (q_dtype != LQ_F16 && q_dtype != LQ_BF16))
        return LQ_ERR_INVALID;
    if (batch == 0) return LQ_OK;
    if (!q || !codes || !scales || (!table && table_width > 0) || !lens || !out) return LQ_ERR_INVALID;
    const uintptr_t al = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(codes) |
                         reinterpret_cast<uintptr_t>(scales);
    if ((al & 15) != 0 || ((q_stride_b | q_stride_h | q_stride_t) & 7) != 0) return LQ_ERR_INVALID;
    // a lane stores head_dim / 32 elements at once
    if ((reinterpret_cast<uintptr_t>(out) & (head_dim / 16 - 1)) != 0) return LQ_ERR_INVALID;
    const int64_t cap = table_width * page_tokens;
    const Plan p = plan(batch, n_heads, n_query * group, head_dim, max_len < cap ? max_len : cap);
    if (const size_t need = workspace_of(p, batch * n_heads * n_query * group, head_dim)) {
        if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return LQ_ERR_INVALID;
        if (workspace_bytes < need) return LQ_ERR_CAPACITY;
    }
    PagedAttnArgs a{};
    a.q = q;
    a.q_stride_b = q_stride_b;
    a.q_stride_h = q_stride_h;
    a.q_stride_t = q_stride_t;
    a.codes = reinterpret_cast<const uint32_t *>(codes);
    a.scales = scales;
    a.n_pages = n_pages;
    a.page_log2 = (uint32_t)__builtin_ctz((unsigned)page_tokens);
    a.table = table;
    a.table_width = table_width;
    a.table_stride = table_stride;
    a.lens = lens;
    a.bound = cap;
    a.mask = mask;
    a.mask_stride_b = mask_stride_b;
    a.n_heads = (uint32_t)n_heads;
    a.group = (uint32_t)group;
    a.T = (uint32_t)n_query;
    a.rows = (uint32_t)(n_query * group);
    a.by_group = FastDiv((uint32_t)group);
    a.chunk = p.chunk;
    a.splits = p.splits;
    a.clustered = p.clustered;
    a.qk_log2 = sm_scale * kLog2e;
    a.out = out;
    a.lse = lse;
    a.part = static_cast<float *>(workspace);
    a.err = err;
    cudaStream_t st = as_stream(stream);
    const uint32_t B = (uint32_t)batch;
    if (q_dtype == LQ_BF16)
        return head_dim == 128 ? launch_dim<true, 128>(a, p.tile, B, st) : launch_dim<true, 64>(a, p.tile, B, st);
    return head_dim == 128 ? launch_dim<false, 128>(a, p.tile, B, st) : launch_dim<false, 64>(a, p.tile, B, st);
}
