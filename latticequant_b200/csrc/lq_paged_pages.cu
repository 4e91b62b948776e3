// lq_paged_pages.cu -- operations on the pages of an E8 cache: fork, free and
// reserve (one table update with the copies it needs), compact, copy, accept.
//
// The tables of a cache are shared by its layers; the pool holds the layers'
// pages one layer after another.  A page is free when refs[page] == 0, so the
// reference counts are the only allocator state and allocation is
// deterministic: free pages are taken in ascending order, children in
// ascending order, columns in ascending order.
//
// All tables come out of place: the copies of a fork read pages that its
// input still owns and write pages that its input had free, so nothing is
// overwritten that a later copy reads, and no order between copies matters.
// Data moves at 16 bytes a thread.  Compacting 512 pages, half of them live, in
// 16 layers (285 MB) takes 47.5-52 us, 5.5-6.0 TB/s; forking 32 beams in 32 layers
// (23 MB) 11.5 us; accepting 5 drafts of 32 rows in 32 layers 7.1 us.  The plans
// are one CTA each, prefix sums over the pool's counts.  A plan's time grows with
// the pool: reserving a token for 32 rows takes 5.3 us with 632 pages, 6.9 with
// 8,192 and 12.3 with 32,768; forking them with the free pages at the end of the
// pool 10.4, 15.9 and 31.3.
#include "lq_paged.cuh"

namespace lq {
namespace {

constexpr int kPlanThreads = 1024;

// Exclusive prefix sum over the block of one int per thread; *total gets the sum.
__device__ __forceinline__ int block_scan(int v, int *warp_sums, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // the previous call's readers are done
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int w = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    *total = warp_sums[31];
    return x - v + (warp ? warp_sums[warp - 1] : 0);
}

// ---- fork ------------------------------------------------------------------
struct ForkArgs {
    const int32_t *table;  // [rows][width]
    const int32_t *lens, *refs;
    const int64_t *parents;  // [children], -1: an empty sequence
    int64_t rows, width, children, n_pages, reserve;
    uint32_t page_log2;
    int32_t *new_table, *new_lens, *new_refs;
    // workspace: a row's first child, a child's first free-list entry, the free list
    int32_t *owner, *base, *fresh;
    int64_t fresh_cap;
    uint32_t *codes;
    float *scales;
    int64_t n_layers, page_rows;  // page_rows = 2 * n_heads * P
    int W;
    uint32_t *err;
};

// A child's live length, and the columns of its table that it may write to: [full, need).
struct Child {
    int64_t parent, len, full, need;
    bool first;
};

__device__ __forceinline__ Child child_of(const ForkArgs &a, int64_t i) {
    Child c{a.parents[i], 0, 0, 0, false};
    if (c.parent < 0 || c.parent >= a.rows) {
        c.parent = -1;
        return c;
    }
    c.len = min(max((int64_t)a.lens[c.parent], (int64_t)0), a.width << a.page_log2);
    c.full = c.len >> a.page_log2;
    c.need = min((c.len + a.reserve + (1 << a.page_log2) - 1) >> a.page_log2, a.width);
    c.first = a.owner[c.parent] == (int32_t)i;
    return c;
}

// Whether child c keeps its parent's page of column col >= full: it will write
// there, so no other entry may name the page (rows that went back behind the
// point of a fork share pages that they had filled).
__device__ __forceinline__ bool keeps(const ForkArgs &a, const Child &c, int64_t col) {
    if (!c.first) return false;
    const int32_t p = a.table[c.parent * a.width + col];
    return p >= 0 && (p >= a.n_pages || a.refs[p] <= 1);
}

// One CTA: owners, fresh pages of each child, the free list, a copy of the counts.
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const __grid_constant__ ForkArgs a) {
    __shared__ int warp_sums[32];
    for (int64_t i = threadIdx.x; i < a.rows; i += kPlanThreads) a.owner[i] = INT32_MAX;
    __syncthreads();
    for (int64_t i = threadIdx.x; i < a.children; i += kPlanThreads) {
        const int64_t p = a.parents[i];
        if (p >= 0 && p < a.rows) {
            atomicMin(a.owner + p, (int32_t)i);
            const int64_t len = max(a.lens[p], 0);
            if (len > (a.width << a.page_log2) || len + a.reserve > (a.width << a.page_log2))
                raise_flag(a.err, LQ_EF_PAGE);
        } else if (p >= a.rows) {
            raise_flag(a.err, LQ_EF_PAGE);
        }
    }
    __syncthreads();
    int64_t wanted = 0;
    for (int64_t i0 = 0; i0 < a.children; i0 += kPlanThreads) {
        const int64_t i = i0 + threadIdx.x;
        int n = 0;
        if (i < a.children) {
            const Child c = child_of(a, i);
            a.new_lens[i] = (int32_t)c.len;
            for (int64_t col = c.full; col < c.need; ++col) n += !keeps(a, c, col);
        }
        int total;
        const int at = block_scan(n, warp_sums, &total);
        if (i < a.children) a.base[i] = (int32_t)min(wanted + at, (int64_t)INT32_MAX);
        wanted += total;
    }
    int found = 0;
    for (int64_t p0 = 0; p0 < a.n_pages; p0 += kPlanThreads) {
        const int64_t p = p0 + threadIdx.x;
        const int r = p < a.n_pages ? a.refs[p] : 1;
        if (p < a.n_pages) a.new_refs[p] = r;
        if (found >= wanted) continue;  // the same for the whole CTA
        int total;
        const int at = found + block_scan(r == 0, warp_sums, &total);
        if (r == 0 && at < wanted) a.fresh[at] = (int32_t)p;
        found += total;
    }
    for (int64_t i = found + threadIdx.x; i < min(wanted, a.fresh_cap); i += kPlanThreads) a.fresh[i] = -1;
    if (found < wanted && threadIdx.x == 0) raise_flag(a.err, LQ_EF_CAPACITY);
}

// The first `n` token rows of every (K or V, head) of page src to page dst in
// one layer; a row is W words, its scale one float.
__device__ __forceinline__ void copy_rows(uint32_t *codes, float *scales, int64_t src, int64_t dst, int64_t page_rows,
                                          uint32_t page_log2, int W, int n) {
    const int vecs = n * W / 4;  // of 16 bytes, per head
    const int heads = (int)(page_rows >> page_log2);
    const uint4 *cs = reinterpret_cast<const uint4 *>(codes + src * page_rows * W);
    uint4 *cd = reinterpret_cast<uint4 *>(codes + dst * page_rows * W);
    const int64_t hv = (int64_t)W / 4 << page_log2;
    for (int h = threadIdx.x >> 6; h < heads; h += blockDim.x >> 6)
        for (int i = threadIdx.x & 63; i < vecs; i += 64) cd[h * hv + i] = __ldg(cs + h * hv + i);
    for (int e = threadIdx.x; e < heads << page_log2; e += blockDim.x)
        if ((e & ((1 << page_log2) - 1)) < n) scales[dst * page_rows + e] = __ldg(scales + src * page_rows + e);
}

// grid (max(children, rows), 1 + n_layers): y = 0 writes the tables and the
// counts, y = 1 + layer copies the live rows of that child's open page.
__global__ void __launch_bounds__(256) fork_apply_kernel(const __grid_constant__ ForkArgs a) {
    const int64_t i = blockIdx.x;
    if (blockIdx.y == 0) {
        if (i < a.rows)
            for (int64_t col = threadIdx.x; col < a.width; col += blockDim.x) {
                const int32_t p = a.table[i * a.width + col];
                if (p >= 0 && p < a.n_pages) atomicSub(a.new_refs + p, 1);
            }
        if (i >= a.children) return;
        const Child c = child_of(a, i);
        for (int64_t col = threadIdx.x; col < a.width; col += blockDim.x) {
            int32_t p = -1;
            if (col < c.full) {
                p = a.table[c.parent * a.width + col];
            } else if (col < c.need) {
                if (keeps(a, c, col)) {
                    p = a.table[c.parent * a.width + col];
                } else {
                    int64_t at = a.base[i];
                    for (int64_t k = c.full; k < col; ++k) at += !keeps(a, c, k);
                    p = at < a.fresh_cap ? a.fresh[at] : -1;
                }
            }
            a.new_table[i * a.width + col] = p;
            if (p >= 0 && p < a.n_pages) atomicAdd(a.new_refs + p, 1);
        }
        return;
    }
    if (i >= a.children) return;
    const Child c = child_of(a, i);
    const int n = (int)(c.len & ((1 << a.page_log2) - 1));
    if (c.parent < 0 || n == 0 || c.full >= c.need || a.base[i] >= a.fresh_cap || keeps(a, c, c.full)) return;
    const int32_t src = a.table[c.parent * a.width + c.full], dst = a.fresh[a.base[i]];
    if (src < 0 || src >= a.n_pages || dst < 0) return;
    const int64_t layer = (int64_t)(blockIdx.y - 1) * a.n_pages;
    copy_rows(a.codes, a.scales, layer + src, layer + dst, a.page_rows, a.page_log2, a.W, n);
}

// ---- compact, copy -----------------------------------------------------------
struct MoveArgs {
    const int32_t *refs;
    const int32_t *table;
    int64_t entries, n_pages;
    int32_t *new_table, *new_refs, *n_live;
    int32_t *src, *dst, *count;  // the moves, at most `most`; `to`: a page's new place
    int64_t most;
    int32_t *to;
    uint32_t *codes;
    float *scales;
    int64_t n_layers, page_rows;
    int W;
    uint32_t *err;
};

// One CTA: the live pages at or above the live count go, in order, to the free pages below it.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const __grid_constant__ MoveArgs a) {
    __shared__ int warp_sums[32];
    int mine = 0, live, total;
    for (int64_t p = threadIdx.x; p < a.n_pages; p += kPlanThreads) mine += a.refs[p] > 0;
    block_scan(mine, warp_sums, &live);
    int holes = 0, moved = 0;
    for (int64_t p0 = 0; p0 < a.n_pages; p0 += kPlanThreads) {
        const int64_t p = p0 + threadIdx.x;
        const bool in = p < a.n_pages, used = in && a.refs[p] > 0;
        const bool hole = in && !used && p < live, move = used && p >= live;
        // both counts in one scan: at most 1024 of each per round
        const int at = block_scan((hole ? 1 : 0) | (move ? 1 << 16 : 0), warp_sums, &total);
        if (hole) a.dst[holes + (at & 0xffff)] = (int32_t)p;
        if (move) a.src[moved + (at >> 16)] = (int32_t)p;
        holes += total & 0xffff;
        moved += total >> 16;
    }
    __syncthreads();
    for (int64_t p = threadIdx.x; p < a.n_pages; p += kPlanThreads) {
        a.to[p] = (int32_t)p;
        a.new_refs[p] = p < live ? a.refs[p] : 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < moved; i += kPlanThreads) {
        a.to[a.src[i]] = a.dst[i];
        a.new_refs[a.dst[i]] = a.refs[a.src[i]];
    }
    if (threadIdx.x == 0) {
        *a.count = moved;
        *a.n_live = live;
    }
}

// Whole pages: block x strides over (move, layer) pairs; the table is renamed on the way.
__global__ void __launch_bounds__(256) move_pages_kernel(const __grid_constant__ MoveArgs a) {
    if (a.new_table)
        for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < a.entries; e += (int64_t)gridDim.x * 256) {
            const int32_t p = a.table[e];
            a.new_table[e] = p >= 0 && p < a.n_pages ? a.to[p] : -1;
            if (p >= a.n_pages) raise_flag(a.err, LQ_EF_PAGE);
        }
    const int64_t units = min((int64_t)*a.count, a.most) * a.n_layers;
    const int64_t cv = a.page_rows * a.W / 4, sv = a.page_rows / 4;  // 16-byte vectors (P is a multiple of 16)
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int64_t i = u / a.n_layers, layer = (u - i * a.n_layers) * a.n_pages;
        const int32_t src = a.src[i], dst = a.dst[i];
        if (src < 0 || src >= a.n_pages || dst < 0 || dst >= a.n_pages) {
            if (threadIdx.x == 0) raise_flag(a.err, LQ_EF_PAGE);
            continue;
        }
        const uint4 *cs = reinterpret_cast<const uint4 *>(a.codes) + (layer + src) * cv;
        uint4 *cd = reinterpret_cast<uint4 *>(a.codes) + (layer + dst) * cv;
        const uint4 *ss = reinterpret_cast<const uint4 *>(a.scales) + (layer + src) * sv;
        uint4 *sd = reinterpret_cast<uint4 *>(a.scales) + (layer + dst) * sv;
        for (int64_t k = threadIdx.x; k < cv; k += 256) cd[k] = __ldg(cs + k);
        for (int64_t k = threadIdx.x; k < sv; k += 256) sd[k] = __ldg(ss + k);
    }
}

// ---- accept ------------------------------------------------------------------
struct AcceptArgs {
    const int32_t *table, *lens, *accepted;
    const int32_t *refs;  // NULL: every page is its row's own
    int64_t width, n_pages, n_draft, most;
    uint32_t page_log2;
    int32_t *new_lens;
    uint32_t *codes;
    float *scales;
    int64_t page_rows;
    int W;
    uint32_t *err;
};

// grid (rows, n_layers).  A thread owns 16 bytes (or the scale) of one (K or
// V, head) across the accepted tokens.  The drafts are taken in ascending
// order and move down or stay, so a source is never a place already written;
// a thread reads eight ahead of its writes.
__global__ void __launch_bounds__(128) accept_kernel(const __grid_constant__ AcceptArgs a) {
    const int64_t b = blockIdx.x, layer = (int64_t)blockIdx.y * a.n_pages;
    const int32_t *acc = a.accepted + b * a.most;
    const int64_t base = a.lens[b] - a.n_draft;
    const int32_t *table = a.table + b * a.width;
    __shared__ int s_n;
    if (threadIdx.x < 32) {  // accepted drafts: up to the first negative, strictly ascending
        int n = 0;
        bool ok = true;
        for (int64_t j0 = 0; j0 < a.most; j0 += 32) {
            const int64_t j = j0 + threadIdx.x;
            const int v = j < a.most ? acc[j] : -1;
            const int prev = j == 0 ? -1 : j < a.most ? acc[j - 1] : -1;
            const uint32_t end = __ballot_sync(0xffffffffu, v < 0);
            const int here = end ? __ffs(end) - 1 : 32;
            const bool bad = (int)threadIdx.x < here && (v <= prev || v >= a.n_draft);
            ok = ok && !__any_sync(0xffffffffu, bad);
            n += here;
            if (end) break;
        }
        ok = ok && (n == 0 || (base >= 0 && a.lens[b] <= a.width << a.page_log2));
        if (ok && a.refs) {  // a row that moves moves nothing into a page that somebody else holds too
            bool shared = false;
            for (int64_t j = threadIdx.x; j < n; j += 32) {
                const int32_t p = table[(base + j) >> a.page_log2];
                shared |= acc[j] != j && p >= 0 && p < a.n_pages && a.refs[p] > 1;
            }
            ok = !__any_sync(0xffffffffu, shared);
        }
        if (threadIdx.x == 0) {
            s_n = ok ? n : 0;
            if (!ok && blockIdx.y == 0) raise_flag(a.err, LQ_EF_PAGE);
            if (blockIdx.y == 0) a.new_lens[b] = ok ? (int32_t)(max(base, (int64_t)0) + n) : a.lens[b];
        }
    }
    __syncthreads();
    const int n = s_n;
    const uint32_t mask = (1u << a.page_log2) - 1;
    auto row_of = [&](int64_t tok, int64_t head) -> int64_t {  // -1: no page there
        const int32_t p = table[tok >> a.page_log2];
        return p < 0 || p >= a.n_pages ? -1 : (layer + p) * a.page_rows + (head << a.page_log2) + (tok & mask);
    };
    const int vec = a.W / 4 + 1;  // 16-byte pieces of a row, then its scale
    const int heads = (int)(a.page_rows >> a.page_log2);
    for (int u = threadIdx.x; u < heads * vec; u += blockDim.x) {
        const int head = u / vec, piece = u - head * vec;
        uint4 *codes = reinterpret_cast<uint4 *>(a.codes) + piece;
        for (int j0 = 0; j0 < n; j0 += 8) {
            uint4 v[8];
            int64_t from[8], to[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                from[k] = to[k] = -1;
                if (j0 + k >= n) continue;
                const int src = acc[j0 + k];
                if (src == j0 + k) continue;
                from[k] = row_of(base + src, head);
                to[k] = row_of(base + j0 + k, head);
                if (from[k] < 0 || to[k] < 0) continue;
                if (piece < vec - 1) v[k] = codes[from[k] * (a.W / 4)];
                else v[k].x = __float_as_uint(a.scales[from[k]]);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (j0 + k >= n || acc[j0 + k] == j0 + k) continue;
                if (from[k] < 0 || to[k] < 0) {
                    raise_flag(a.err, LQ_EF_PAGE);
                    continue;
                }
                if (piece < vec - 1) codes[to[k] * (a.W / 4)] = v[k];
                else a.scales[to[k]] = __uint_as_float(v[k].x);
            }
        }
    }
}

bool pool_ok(const void *codes, const void *scales, int64_t n_layers, int64_t n_pages, int n_heads, int page_tokens,
             int head_dim) {
    return n_layers >= 1 && n_layers <= 65534 && n_pages >= 1 && n_pages <= 0x7fffffff && n_heads >= 1 &&
           n_heads <= 1024 && paged_page_ok(page_tokens) && paged_dim_ok(head_dim) && codes && scales &&
           ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) & 15) == 0;
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_pages_fork_workspace(int64_t rows, int64_t children, int64_t n_pages) {
    if (rows < 0 || children < 0 || n_pages < 0) return 0;
    return (size_t)(rows + children + n_pages) * 4;
}

extern "C" int lq_pages_fork(const int32_t *table, int64_t rows, int64_t width, const int32_t *lens,
                             const int32_t *refs, const int64_t *parents, int64_t children, int64_t reserve,
                             int32_t *new_table, int32_t *new_lens, int32_t *new_refs, int32_t *codes, float *scales,
                             int64_t n_layers, int64_t n_pages, int n_heads, int page_tokens, int head_dim,
                             void *workspace, size_t workspace_bytes, uint32_t *err, void *stream) {
    LQ_NVTX_RANGE();
    if (!pool_ok(codes, scales, n_layers, n_pages, n_heads, page_tokens, head_dim) || rows < 0 || width < 1 ||
        children < 0 || reserve < 0 || reserve > 0x7fffffff || rows > (1 << 24) || children > (1 << 24) ||
        width > (1 << 20))
        return LQ_ERR_INVALID;
    if (!refs || !new_refs || (rows > 0 && (!table || !lens)) || (children > 0 && (!parents || !new_table || !new_lens)) ||
        !workspace)
        return LQ_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(workspace) & 3) != 0) return LQ_ERR_INVALID;
    if (workspace_bytes < lq_pages_fork_workspace(rows, children, n_pages)) return LQ_ERR_CAPACITY;
    ForkArgs a{};
    a.table = table;
    a.lens = lens;
    a.refs = refs;
    a.parents = parents;
    a.rows = rows;
    a.width = width;
    a.children = children;
    a.n_pages = n_pages;
    a.reserve = reserve;
    a.page_log2 = (uint32_t)__builtin_ctz((unsigned)page_tokens);
    a.new_table = new_table;
    a.new_lens = new_lens;
    a.new_refs = new_refs;
    a.owner = static_cast<int32_t *>(workspace);
    a.base = a.owner + rows;
    a.fresh = a.base + children;
    a.fresh_cap = n_pages;
    a.codes = reinterpret_cast<uint32_t *>(codes);
    a.scales = scales;
    a.n_layers = n_layers;
    a.page_rows = (int64_t)2 * n_heads * page_tokens;
    a.W = head_dim / 8;
    a.err = err;
    cudaStream_t st = as_stream(stream);
    fork_plan_kernel<<<1, kPlanThreads, 0, st>>>(a);
    if (check_launch() != LQ_OK) return LQ_ERR_CUDA;
    const int64_t x = children > rows ? children : rows;
    if (x > 0) fork_apply_kernel<<<dim3((unsigned)x, (unsigned)(1 + n_layers)), 256, 0, st>>>(a);
    return check_launch();
}

extern "C" size_t lq_pages_compact_workspace(int64_t n_pages) {
    return n_pages < 0 ? 0 : (size_t)n_pages * 12 + 4;
}

extern "C" int lq_pages_compact(const int32_t *table, int64_t entries, const int32_t *refs, int32_t *new_table,
                                int32_t *new_refs, int32_t *n_live, int32_t *codes, float *scales, int64_t n_layers,
                                int64_t n_pages, int n_heads, int page_tokens, int head_dim, void *workspace,
                                size_t workspace_bytes, uint32_t *err, void *stream) {
    LQ_NVTX_RANGE();
    if (!pool_ok(codes, scales, n_layers, n_pages, n_heads, page_tokens, head_dim) || entries < 0) return LQ_ERR_INVALID;
    if (!refs || !new_refs || !n_live || (entries > 0 && (!table || !new_table)) || !workspace) return LQ_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(workspace) & 3) != 0) return LQ_ERR_INVALID;
    if (workspace_bytes < lq_pages_compact_workspace(n_pages)) return LQ_ERR_CAPACITY;
    MoveArgs a{};
    a.refs = refs;
    a.table = table;
    a.entries = entries;
    a.n_pages = n_pages;
    a.new_table = entries > 0 ? new_table : nullptr;
    a.new_refs = new_refs;
    a.n_live = n_live;
    a.count = static_cast<int32_t *>(workspace);
    a.most = n_pages;
    a.src = a.count + 1;
    a.dst = a.src + n_pages;
    a.to = a.dst + n_pages;
    a.codes = reinterpret_cast<uint32_t *>(codes);
    a.scales = scales;
    a.n_layers = n_layers;
    a.page_rows = (int64_t)2 * n_heads * page_tokens;
    a.W = head_dim / 8;
    a.err = err;
    cudaStream_t st = as_stream(stream);
    compact_plan_kernel<<<1, kPlanThreads, 0, st>>>(a);
    if (check_launch() != LQ_OK) return LQ_ERR_CUDA;
    move_pages_kernel<<<148 * 8, 256, 0, st>>>(a);
    return check_launch();
}

extern "C" int lq_pages_copy(const int32_t *src, const int32_t *dst, const int32_t *count, int64_t most, int32_t *codes,
                             float *scales, int64_t n_layers, int64_t n_pages, int n_heads, int page_tokens,
                             int head_dim, uint32_t *err, void *stream) {
    LQ_NVTX_RANGE();
    if (!pool_ok(codes, scales, n_layers, n_pages, n_heads, page_tokens, head_dim) || most < 0) return LQ_ERR_INVALID;
    if (most == 0) return LQ_OK;
    if (!src || !dst || !count) return LQ_ERR_INVALID;
    MoveArgs a{};
    a.n_pages = n_pages;
    a.src = const_cast<int32_t *>(src);
    a.dst = const_cast<int32_t *>(dst);
    a.count = const_cast<int32_t *>(count);
    a.most = most;
    a.codes = reinterpret_cast<uint32_t *>(codes);
    a.scales = scales;
    a.n_layers = n_layers;
    a.page_rows = (int64_t)2 * n_heads * page_tokens;
    a.W = head_dim / 8;
    a.err = err;
    const int64_t units = most * n_layers;
    move_pages_kernel<<<(unsigned)(units < 148 * 8 ? units : 148 * 8), 256, 0, as_stream(stream)>>>(a);
    return check_launch();
}

static int accept(const int32_t *table, int64_t rows, int64_t width, const int32_t *lens, const int32_t *refs,
                  int64_t n_draft, const int32_t *accepted, int64_t most, int32_t *new_lens, int32_t *codes,
                  float *scales, int64_t n_layers, int64_t n_pages, int n_heads, int page_tokens, int head_dim,
                  uint32_t *err, void *stream) {
    if (!pool_ok(codes, scales, n_layers, n_pages, n_heads, page_tokens, head_dim) || rows < 0 || rows > (1 << 24) ||
        width < 1 || width > (1 << 20) || n_draft < 1 || n_draft > 4096 || most < 0)
        return LQ_ERR_INVALID;
    if (rows == 0) return LQ_OK;
    if (!table || !lens || (most > 0 && !accepted) || !new_lens) return LQ_ERR_INVALID;
    AcceptArgs a{};
    a.table = table;
    a.lens = lens;
    a.accepted = accepted;
    a.refs = refs;
    a.width = width;
    a.n_pages = n_pages;
    a.n_draft = n_draft;
    a.most = most;
    a.page_log2 = (uint32_t)__builtin_ctz((unsigned)page_tokens);
    a.new_lens = new_lens;
    a.codes = reinterpret_cast<uint32_t *>(codes);
    a.scales = scales;
    a.page_rows = (int64_t)2 * n_heads * page_tokens;
    a.W = head_dim / 8;
    a.err = err;
    accept_kernel<<<dim3((unsigned)rows, (unsigned)n_layers), 128, 0, as_stream(stream)>>>(a);
    return check_launch();
}

extern "C" int lq_pages_accept(const int32_t *table, int64_t rows, int64_t width, const int32_t *lens, int64_t n_draft,
                               const int32_t *accepted, int64_t most, int32_t *new_lens, int32_t *codes, float *scales,
                               int64_t n_layers, int64_t n_pages, int n_heads, int page_tokens, int head_dim,
                               uint32_t *err, void *stream) {
    LQ_NVTX_RANGE();
    return accept(table, rows, width, lens, nullptr, n_draft, accepted, most, new_lens, codes, scales, n_layers, n_pages,
                  n_heads, page_tokens, head_dim, err, stream);
}

extern "C" int lq_pages_accept_shared(const int32_t *table, int64_t rows, int64_t width, const int32_t *lens,
                                      const int32_t *refs, int64_t n_draft, const int32_t *accepted, int64_t most,
                                      int32_t *new_lens, int32_t *codes, float *scales, int64_t n_layers,
                                      int64_t n_pages, int n_heads, int page_tokens, int head_dim, uint32_t *err,
                                      void *stream) {
    LQ_NVTX_RANGE();
    if (!refs) return LQ_ERR_INVALID;
    return accept(table, rows, width, lens, refs, n_draft, accepted, most, new_lens, codes, scales, n_layers, n_pages,
                  n_heads, page_tokens, head_dim, err, stream);
}
