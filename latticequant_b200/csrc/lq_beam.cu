// lq_beam.cu -- beam search's selection over beams and vocabulary.
//
// For every sequence with beams k and words v:
//   lp[k][v] = (x[k][v] - m[k]) - ln sum_v exp(x[k][v] - m[k]),   m[k] = max_v x[k][v]
//   total = scores[k] + lp
// the n largest totals, best first; equal totals go to the lower beam, then
// the larger logit, then the lower word.  A candidate needs a total above
// -inf (a banned word, a NaN logit or a dead beam gives none); places left
// without a candidate hold -inf and -1.  The reference has no counterpart
// (it decodes greedily, llm/e2e_eval.py:212).
//
// Each logit is read once.  Within a beam the order of the totals is the
// order of the logits, so a part of a row can give up all but its n best
// before the row's log-sum-exp is known:
//   beam_part_kernel  a CTA streams its part of a row through registers, 64
//       bytes a thread at a time with the next 64 in flight.  Every thread
//       keeps a maximum and a sum of exponentials of its own.  The n best
//       are kept by a bound: among the largest per-thread maxima of each warp
//       of the first tile the n-th largest is at most the n-th best of the
//       row.  A 16-byte load whose largest logit reaches the bound (few do) is
//       put aside whole, in its warp's list; a warp whose list grows long
//       raises the bound to the n-th largest of the list's maxima and drops
//       what no longer reaches it.  The warps never wait for one another; in
//       the end the bound is found again among the lists, and the logits that
//       reach it are ranked by counting.
//   beam_merge_kernel  a CTA per sequence joins the parts' statistics and
//       picks the n best totals the same way.
// 32 sequences of 8 beams over 128,256 words in bf16 take 27.2 us (2.4 TB/s):
// 256 rows give 148 SMs 1.7 CTAs each, and more parts a row (29 us with two, 32
// with four) cost more in their starts and rankings than they even out.
// 4 beams over 32,000 words take 8.6-9.1 us, most of it the two launches' latency.
// A part with so many equal logits that a list or the ranking overflows is ranked by
// n rounds of a block-wide maximum instead, over the logits in memory.
#include "lq_attn_common.cuh"

namespace lq {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kVecs = 4;  // 16-byte loads of a thread and tile
constexpr int kAside = 320, kAsideLong = kAside - 32 * kVecs;  // loads a warp's list holds; it is cut when this long
constexpr int kMaxPicked = 1024, kMaxN = 128, kMaxBeams = 256, kMaxVocab = 1 << 24;

// Order-preserving image of a float: larger x, larger value; 0 for no
// candidate (-inf, NaN), and one value for both zeros.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return x > -INFINITY ? o : 0u;
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// A candidate: hi its rank in value, lo what decides between equals.
struct Key {
    uint32_t hi;
    uint64_t lo;
    __device__ bool operator>(const Key &o) const { return hi != o.hi ? hi > o.hi : lo > o.lo; }
};

struct Picker {  // shared memory of a selection
    uint32_t top[kWarps * 32];
    uint32_t hi[kMaxPicked];
    uint64_t lo[kMaxPicked];
    uint32_t bound;
    int count;
};

// A value that at least n of the block's candidates reach (0: any), from each
// thread's best.  Every warp lists its r largest; the n-th largest of the
// lists is the bound.
__device__ __forceinline__ void find_bound(uint32_t best, int n, Picker &s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = min(32, 2 * ((n + kWarps - 1) / kWarps));
    for (int i = 0; i < r; ++i) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, best);
        if (lane == 0) s.top[warp * r + i] = m;
        const uint32_t at = __ballot_sync(0xffffffffu, best == m);
        if (lane == __ffs(at) - 1) best = 0;
    }
    if (threadIdx.x == 0) {
        s.bound = 0;
        s.count = 0;
    }
    __syncthreads();
    if (threadIdx.x < kWarps * r) {
        const uint32_t v = s.top[threadIdx.x];
        int above = 0;
        for (int j = 0; j < kWarps * r; ++j) above += s.top[j] > v || (s.top[j] == v && j < (int)threadIdx.x);
        if (above == n - 1) s.bound = v;
    }
    __syncthreads();
}

__device__ __forceinline__ void pick(Picker &s, uint32_t hi, uint64_t lo) {
    const int at = atomicAdd(&s.count, 1);
    if (at < kMaxPicked) {
        s.hi[at] = hi;
        s.lo[at] = lo;
    }
}

// emit(rank, key) for the n largest picked keys (all distinct); false: too many were picked.
template <class Emit>
__device__ __forceinline__ bool rank_picked(Picker &s, int n, Emit emit) {
    __syncthreads();
    const int c = s.count;
    if (c > kMaxPicked) return false;
    for (int i = threadIdx.x; i < c; i += kThreads) {
        const Key k{s.hi[i], s.lo[i]};
        int above = 0;
        for (int j = 0; j < c; ++j) above += Key{s.hi[j], s.lo[j]} > k;
        if (above < n) emit(above, k);
    }
    for (int i = c + threadIdx.x; i < n; i += kThreads) emit(i, Key{0u, 0ull});
    return true;
}

// emit(rank, key) by n rounds of a block-wide maximum over best_below(key), a thread's largest key under `key`.
template <class Best, class Emit>
__device__ void rank_by_rounds(Picker &s, int n, Best best_below, Emit emit) {
    Key last{0xffffffffu, ~0ull};
    for (int i = 0; i < n; ++i) {
        Key b = best_below(last);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
            const Key other{__shfl_xor_sync(0xffffffffu, b.hi, o), __shfl_xor_sync(0xffffffffu, b.lo, o)};
            if (other > b) b = other;
        }
        __syncthreads();
        if ((threadIdx.x & 31) == 0) {
            s.hi[threadIdx.x >> 5] = b.hi;
            s.lo[threadIdx.x >> 5] = b.lo;
        }
        __syncthreads();
        Key top{0u, 0ull};
        for (int w = 0; w < kWarps; ++w) {
            const Key k{s.hi[w], s.lo[w]};
            if (k > top) top = k;
        }
        if (threadIdx.x == 0) emit(i, top);
        if (top.hi == 0) {
            for (int j = i + 1 + threadIdx.x; j < n; j += kThreads) emit(j, Key{0u, 0ull});
            return;
        }
        last = top;
    }
}

// The loads that the warps put aside.
struct Aside {
    uint4 data[kWarps][kAside];
    int word[kWarps][kAside];  // of element 0
    int count[kWarps];
    int overflow;
};

struct BeamArgs {
    const void *logits;
    int64_t stride_b, stride_k;
    const float *scores;  // [batch][beams]
    int beams, vocab, n, parts, tiles;  // tiles: of a part
    FastDiv by_beams, by_keys;          // keys: parts * n
    float2 *stat;      // [batch * beams][parts]: maximum, sum of exp(x - maximum)
    uint64_t *keys;    // [batch * beams][parts][n]: ordered(x) << 24 | (2^24 - 1 - word), 0: none
    float *top_score;  // [batch][n]
    int64_t *top_beam, *top_word;
};

constexpr uint64_t kWordMask = (1u << 24) - 1;

__device__ __forceinline__ uint64_t key_of(uint32_t value, int word) {
    return (uint64_t)value << 24 | (kWordMask - (uint32_t)word);
}

// Element e of a 16-byte load.
template <int DT>
__device__ __forceinline__ float element(const uint32_t (&r)[4], int e) {
    if constexpr (DT == LQ_F32) return __uint_as_float(r[e]);
    else if constexpr (DT == LQ_F16) return __half2float(__ushort_as_half((uint16_t)(r[e / 2] >> (16 * (e & 1)))));
    else return __uint_as_float(e & 1 ? r[e / 2] & 0xffff0000u : r[e / 2] << 16);
}

// The largest element of a 16-byte load, NaNs aside (two at a time in 16 bits).
template <int DT>
__device__ __forceinline__ float largest(const uint4 &v) {
    if constexpr (DT == LQ_F32) {
        return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    } else {
        uint32_t r[3];
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const uint32_t p = i < 2 ? w[2 * i] : r[0], q = i < 2 ? w[2 * i + 1] : r[1];
            if constexpr (DT == LQ_F16) asm("max.f16x2 %0, %1, %2;" : "=r"(r[i]) : "r"(p), "r"(q));
            else asm("max.bf16x2 %0, %1, %2;" : "=r"(r[i]) : "r"(p), "r"(q));
        }
        const uint32_t pair[4] = {r[2], 0u, 0u, 0u};
        return fmaxf(element<DT>(pair, 0), element<DT>(pair, 1));
    }
}

__device__ __forceinline__ float exp_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A warp's list cut by the n-th largest of its loads' maxima, which becomes the bound for all.
template <int DT>
__device__ __noinline__ void cut_aside(Aside &x, int warp, int n, uint32_t *bound) {
    const int lane = threadIdx.x & 31, c = x.count[warp];
    uint32_t top[kAside / 32];
#pragma unroll
    for (int q = 0; q < kAside / 32; ++q) {
        const int i = lane + 32 * q;
        top[q] = i < c ? ordered(largest<DT>(x.data[warp][i])) : 0u;
    }
    uint32_t nth = 0;
    for (int r = 0; r < n; ++r) {  // n rounds of a maximum, one load leaving in each
        uint32_t mine = 0;
#pragma unroll
        for (int q = 0; q < kAside / 32; ++q) mine = max(mine, top[q]);
        nth = __reduce_max_sync(0xffffffffu, mine);
        const bool first = lane == __ffs(__ballot_sync(0xffffffffu, mine == nth)) - 1;
        bool gone = !first;
#pragma unroll
        for (int q = 0; q < kAside / 32; ++q)
            if (!gone && top[q] == nth) {
                top[q] = 0;
                gone = true;
            }
    }
    int kept = 0;
    for (int i0 = 0; i0 < c; i0 += 32) {
        const int i = i0 + lane;
        const uint4 d = x.data[warp][min(i, kAside - 1)];
        const int w = x.word[warp][min(i, kAside - 1)];
        const bool keep = i < c && ordered(largest<DT>(d)) >= max(nth, 1u);
        const uint32_t all = __ballot_sync(0xffffffffu, keep);
        if (keep) {  // at or before its old place
            const int at = kept + __popc(all & ((1u << lane) - 1));
            x.data[warp][at] = d;
            x.word[warp][at] = w;
        }
        kept += __popc(all);
        __syncwarp();
    }
    if (lane == 0) {
        x.count[warp] = kept;
        atomicMax(bound, nth);
        if (kept > kAsideLong) x.overflow = 1;  // as many equal maxima
    }
    __syncwarp();
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 3) beam_part_kernel(const __grid_constant__ BeamArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int V = 16 / sizeof(T);  // elements of a load
    constexpr int kTile = kThreads * kVecs * V;
    extern __shared__ __align__(16) char raw[];
    Aside &aside = *reinterpret_cast<Aside *>(raw);
    __shared__ Picker s;
    __shared__ float2 red[kWarps];
    const int warp = threadIdx.x >> 5;
    allow_next();
    const int row = blockIdx.y, part = blockIdx.x;
    const int b = (int)a.by_beams.div((uint32_t)row), k = row - b * a.beams;
    const T *x0 = static_cast<const T *>(a.logits) + b * a.stride_b + k * a.stride_k;
    // loads start on the 16-byte boundary at or before the row
    const int mis = (int)((reinterpret_cast<uintptr_t>(x0) & 15) / sizeof(T));
    const uint4 *base = reinterpret_cast<const uint4 *>(x0 - mis) + threadIdx.x;
    const int first = part * a.tiles, last = min(first + a.tiles, (a.vocab + mis + kTile - 1) / kTile);
    auto word_of = [&](int tile, int i) {  // of element 0 of load i
        return tile * kTile + (i * kThreads + (int)threadIdx.x) * V - mis;
    };
    uint32_t none;  // a pair (or one) of -inf
    if constexpr (DT == LQ_F32) none = 0xff800000u;
    else if constexpr (DT == LQ_F16) none = 0xfc00fc00u;
    else none = 0xff80ff80u;
    auto fetch = [&](int tile, uint4 (&r)[kVecs]) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int w = word_of(tile, i);
            r[i] = make_uint4(none, none, none, none);
            if (w < a.vocab && w + V > 0) r[i] = __ldcs(base + (int64_t)tile * (kThreads * kVecs) + i * kThreads);
        }
    };
    // words before the row's first and past its last become -inf
    auto trim = [&](int tile, uint4 (&r)[kVecs]) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int w = word_of(tile, i);
            uint32_t u[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (w + e < 0 || w + e >= a.vocab) {
                    if constexpr (DT == LQ_F32) u[e] = none;
                    else u[e / 2] = e & 1 ? (u[e / 2] & 0xffffu) | (none & 0xffff0000u)
                                          : (u[e / 2] & 0xffff0000u) | (none & 0xffffu);
                }
            r[i] = make_uint4(u[0], u[1], u[2], u[3]);
        }
    };

    float m = -INFINITY, sum = 0.f;
    uint4 nx[kVecs];
    if (threadIdx.x < kWarps) aside.count[threadIdx.x] = 0;
    if (threadIdx.x == 0) aside.overflow = 0;
    if (first < last) fetch(first, nx);
    volatile uint32_t *const bound = &s.bound;
    volatile int *const count = &aside.count[warp];
    for (int tile = first; tile < last; ++tile) {
        uint4 cur[kVecs];
#pragma unroll
        for (int i = 0; i < kVecs; ++i) cur[i] = nx[i];
        if (tile + 1 < last) fetch(tile + 1, nx);
        if (tile * kTile < mis || (tile + 1) * kTile - mis > a.vocab) trim(tile, cur);

        float top[kVecs], mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            top[i] = largest<DT>(cur[i]);
            mx = fmaxf(mx, top[i]);
        }
        if (tile == first) find_bound(ordered(mx), a.n, s);
        // (any finite logit while there are fewer than n)
        const uint32_t reach = *bound;
        const float low = reach ? from_ordered(reach) : -3.402823466e38f;
        if (__any_sync(0xffffffffu, mx >= low)) {
#pragma unroll
            for (int i = 0; i < kVecs; ++i)
                if (top[i] >= low) {
                    const int at = atomicAdd(&aside.count[warp], 1);
                    if (at < kAside) {
                        aside.data[warp][at] = cur[i];
                        aside.word[warp][at] = word_of(tile, i);
                    }
                }
            __syncwarp();
            // after an overflow the list no longer matters: it is kept short
            if (*count > kAsideLong) cut_aside<DT>(aside, warp, a.n, &s.bound);
            if (*count > kAsideLong) {
                __syncwarp();
                *count = 0;
                __syncwarp();
            }
        }
        // the thread's own maximum and sum; the maximum finite, so that -inf - m is -inf
        const float m1 = fmaxf(fmaxf(m, mx), -3.402823466e38f);
        sum *= exp2f((m - m1) * kLog2e);
        m = m1;
        const unsigned long long minus = f2_pack(-m, -m), scale = f2_pack(kLog2e, kLog2e);
        unsigned long long acc = 0;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const uint32_t u[4] = {cur[i].x, cur[i].y, cur[i].z, cur[i].w};
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                float y0, y1;
                f2_unpack(f2_mul(f2_add(f2_pack(element<DT>(u, e), element<DT>(u, e + 1)), minus), scale), y0, y1);
                acc = f2_add(acc, f2_pack(exp_of(y0), exp_of(y1)));
            }
        }
        float a0, a1;
        f2_unpack(acc, a0, a1);
        a0 += a1;
        if (a0 != a0) {  // a NaN logit (left out), or +inf (stays NaN)
            a0 = 0.f;
#pragma unroll 1
            for (int i = 0; i < kVecs; ++i) {
                const uint4 c = i == 0 ? cur[0] : i == 1 ? cur[1] : i == 2 ? cur[2] : cur[3];
                const uint32_t u[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                for (int e = 0; e < V; ++e) a0 += exp_of((fmaxf(element<DT>(u, e), -INFINITY) - m) * kLog2e);
            }
        }
        sum += a0;
    }

#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, sum, o);
        const float top = fmaxf(fmaxf(m, m2), -3.402823466e38f);
        sum = sum * exp2f((m - top) * kLog2e) + s2 * exp2f((m2 - top) * kLog2e);
        m = top;
    }
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(m, sum);
    __syncthreads();
    const int64_t at = (int64_t)row * a.parts + part;
    if (threadIdx.x == 0) {
        float top = red[0].x, all = 0.f;
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, red[w].x);
        for (int w = 0; w < kWarps; ++w) all += red[w].y * exp2f((red[w].x - top) * kLog2e);
        a.stat[at] = make_float2(top, all);
    }

    // the bound again, among what was put aside (the barrier above is past every warp's last load)
    uint32_t best = 0;
    for (int i = threadIdx.x & 31; i < aside.count[warp]; i += 32) best = max(best, ordered(largest<DT>(aside.data[warp][i])));
    find_bound(best, a.n, s);
    const uint32_t reach = max(s.bound, 1u);
    for (int i = threadIdx.x & 31; i < aside.count[warp]; i += 32) {
        const uint4 d = aside.data[warp][i];
        const int w = aside.word[warp][i];
        const uint32_t u[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const uint32_t o = ordered(element<DT>(u, e));
            if (o >= reach) pick(s, 0u, key_of(o, w + e));
        }
    }
    uint64_t *out = a.keys + at * a.n;
    auto emit = [&](int i, const Key &key) { out[i] = key.lo; };
    if (aside.overflow || !rank_picked(s, a.n, emit))
        rank_by_rounds(
            s, a.n,
            [&](const Key &under) {
                Key top{0u, 0ull};
                for (int tile = first; tile < last; ++tile) {
                    uint4 r[kVecs];
                    fetch(tile, r);
                    trim(tile, r);
                    for (int i = 0; i < kVecs; ++i) {
                        const uint32_t u[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const uint32_t o = ordered(element<DT>(u, e));
                            const uint64_t lo = o ? key_of(o, word_of(tile, i) + e) : 0ull;
                            if (lo < under.lo && lo > top.lo) top.lo = lo;
                        }
                    }
                }
                top.hi = top.lo ? 1u : 0u;
                return top;
            },
            emit);
}

__global__ void __launch_bounds__(kThreads) beam_merge_kernel(const __grid_constant__ BeamArgs a) {
    __shared__ Picker s;
    // a row's log-sum-exp in two parts: rounded to one, a large maximum would take the digits of the sum
    __shared__ float top[kMaxBeams], log_sum[kMaxBeams], score[kMaxBeams];
    const int b = blockIdx.x, lane = threadIdx.x & 31;
    after_previous();
    for (int k = threadIdx.x >> 5; k < a.beams; k += kWarps) {
        const float2 *st = a.stat + ((int64_t)b * a.beams + k) * a.parts;
        float m = -INFINITY;
        for (int i = lane; i < a.parts; i += 32) m = fmaxf(m, st[i].x);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        float sum = 0.f;
        for (int i = lane; i < a.parts; i += 32)
            if (st[i].x > -INFINITY) sum += st[i].y * exp2f((st[i].x - m) * kLog2e);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            top[k] = m;
            log_sum[k] = logf(sum);
            score[k] = a.scores[(int64_t)b * a.beams + k];
        }
    }
    __syncthreads();
    const int total = a.beams * a.parts * a.n;
    const uint64_t *keys = a.keys + (int64_t)b * total;
    auto key_at = [&](int i) {
        const uint64_t lo = keys[i];
        const int k = (int)a.by_keys.div((uint32_t)i);
        const float x = from_ordered((uint32_t)(lo >> 24));
        const float v = __fadd_rn(__fsub_rn(__fsub_rn(x, top[k]), log_sum[k]), score[k]);
        return lo ? Key{ordered(v), (uint64_t)(255 - k) << 56 | lo} : Key{0u, 0ull};
    };
    uint32_t best = 0;
    for (int i = threadIdx.x; i < total; i += kThreads) best = max(best, key_at(i).hi);
    find_bound(best, a.n, s);
    const uint32_t bound = max(s.bound, 1u);
    if (best >= bound)
        for (int i = threadIdx.x; i < total; i += kThreads) {
            const Key k = key_at(i);
            if (k.hi >= bound) pick(s, k.hi, k.lo);
        }
    auto emit = [&](int i, const Key &k) {
        const int64_t at = (int64_t)b * a.n + i;
        a.top_score[at] = k.hi ? from_ordered(k.hi) : -INFINITY;
        a.top_beam[at] = k.hi ? (int64_t)(255 - (k.lo >> 56)) : -1;
        a.top_word[at] = k.hi ? (int64_t)(kWordMask - (k.lo & kWordMask)) : -1;
    };
    if (!rank_picked(s, a.n, emit))
        rank_by_rounds(
            s, a.n,
            [&](const Key &under) {
                Key top{0u, 0ull};
                for (int i = threadIdx.x; i < total; i += kThreads) {
                    const Key k = key_at(i);
                    if (under > k && k > top) top = k;
                }
                return top;
            },
            emit);
}

// Parts of a row: as many as three resident CTAs a SM allow, a tile at least
// (larger batches stream whole rows).
struct Plan {
    int parts, tiles;
};

Plan plan(int64_t rows, int64_t vocab, int dtype) {
    const int64_t tile = (int64_t)kThreads * kVecs * (dtype == LQ_F32 ? 4 : 8);
    const int64_t all = ceil_div(vocab + 7, tile);  // a misaligned row starts up to 7 words in
    int64_t parts = 148 * 3 / (rows < 1 ? 1 : rows);
    parts = parts < 1 ? 1 : parts > all ? all : parts;
    const int64_t tiles = ceil_div(all, parts);
    return Plan{(int)ceil_div(all, tiles), (int)tiles};
}

template <int DT>
int launch_part(const BeamArgs &a, dim3 grid, cudaStream_t st) {
    if (cudaFuncSetAttribute(beam_part_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Aside)) !=
        cudaSuccess)
        return LQ_ERR_CUDA;
    beam_part_kernel<DT><<<grid, kThreads, sizeof(Aside), st>>>(a);
    return check_launch();
}

bool beam_ok(int64_t batch, int64_t beams, int64_t vocab, int64_t n, int dtype) {
    return batch >= 0 && beams >= 1 && beams <= kMaxBeams && vocab >= 1 && vocab <= kMaxVocab && n >= 1 && n <= kMaxN &&
           batch <= 65535 && batch * beams <= 65535 && (dtype == LQ_F32 || dtype == LQ_F16 || dtype == LQ_BF16);
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_beam_select_workspace(int dtype, int64_t batch, int64_t beams, int64_t vocab, int64_t n) {
    if (!beam_ok(batch, beams, vocab, n, dtype)) return 0;
    return (size_t)batch * beams * plan(batch * beams, vocab, dtype).parts * (sizeof(float2) + 8 * n);
}

extern "C" int lq_beam_select(const void *logits, int dtype, int64_t batch, int64_t beams, int64_t vocab,
                              int64_t stride_b, int64_t stride_k, const float *scores, int64_t n, float *top_score,
                              int64_t *top_beam, int64_t *top_word, void *workspace, size_t workspace_bytes,
                              void *stream) {
    LQ_NVTX_RANGE();
    if (!beam_ok(batch, beams, vocab, n, dtype)) return LQ_ERR_INVALID;
    if (batch == 0) return LQ_OK;
    if (!logits || !scores || !top_score || !top_beam || !top_word || !workspace) return LQ_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(workspace) & 7) != 0) return LQ_ERR_INVALID;
    if (workspace_bytes < lq_beam_select_workspace(dtype, batch, beams, vocab, n)) return LQ_ERR_CAPACITY;
    const Plan p = plan(batch * beams, vocab, dtype);
    BeamArgs a{};
    a.logits = logits;
    a.stride_b = stride_b;
    a.stride_k = stride_k;
    a.scores = scores;
    a.beams = (int)beams;
    a.vocab = (int)vocab;
    a.n = (int)n;
    a.parts = p.parts;
    a.tiles = p.tiles;
    a.by_beams = FastDiv((uint32_t)beams);
    a.by_keys = FastDiv((uint32_t)(p.parts * n));
    a.stat = static_cast<float2 *>(workspace);
    a.keys = reinterpret_cast<uint64_t *>(a.stat + batch * beams * p.parts);
    a.top_score = top_score;
    a.top_beam = top_beam;
    a.top_word = top_word;
    cudaStream_t st = as_stream(stream);
    const dim3 grid((unsigned)p.parts, (unsigned)(batch * beams));
    const int status = dtype == LQ_F32   ? launch_part<LQ_F32>(a, grid, st)
                       : dtype == LQ_F16 ? launch_part<LQ_F16>(a, grid, st)
                                         : launch_part<LQ_BF16>(a, grid, st);
    if (status != LQ_OK) return status;
    return launch_overlapped(beam_merge_kernel, dim3((unsigned)batch), kThreads, 0, st, a);
}
