// lq_beam.cu -- beam search's selection over beams and vocabulary.
//
// For every sequence with beams k and words v:
//   lp[k][v] = x[k][v] - ln sum_v exp(x[k][v]),   total = scores[k] + lp
// the n largest totals, best first; equal totals go to the lower beam, then
// the larger logit, then the lower word.  A candidate needs a total above
// -inf (a banned word, a NaN logit or a dead beam gives none); places left
// without a candidate hold -inf and -1.  The reference has no counterpart
// (it decodes greedily, llm/e2e_eval.py:212).
//
// Each logit is read once.  Within a beam the order of the totals is the
// order of the logits, so a slice of a row can give up all but its n best
// before the row's log-sum-exp is known:
//   beam_slice_kernel  a CTA holds 8192 logits in registers: their maximum
//       and sum of exponentials, and their n best as sorted keys.  The n
//       best are found from a bound: among the largest per-thread maxima of
//       each warp the n-th largest is at most the n-th largest logit, few
//       logits reach it, and those are ranked by counting.
//   beam_merge_kernel  a CTA per sequence joins the slices' statistics and
//       picks the n best totals the same way.
// A row with so many equal logits that more than kMaxPicked reach the bound
// is ranked by n rounds of a block-wide maximum instead.
#include "lq_attn_common.cuh"

namespace lq {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kPerThread = 32, kSlice = kThreads * kPerThread;
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

struct BeamArgs {
    const void *logits;
    int64_t stride_b, stride_k;
    const float *scores;  // [batch][beams]
    int beams, vocab, n, slices;
    float2 *stat;      // [batch * beams][slices]: maximum, sum of exp(x - maximum)
    uint64_t *keys;    // [batch * beams][slices][n]: ordered(x) << 24 | (2^24 - 1 - word), 0: none
    float *top_score;  // [batch][n]
    int64_t *top_beam, *top_word;
};

constexpr uint64_t kWordMask = (1u << 24) - 1;

template <int DT>
__global__ void __launch_bounds__(kThreads) beam_slice_kernel(const __grid_constant__ BeamArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int V = 16 / sizeof(T);  // elements of a 16-byte load
    __shared__ Picker s;
    __shared__ float red[2 * kWarps];
    const int row = blockIdx.y, slice = blockIdx.x;
    const int b = row / a.beams, k = row - b * a.beams;
    const T *x0 = static_cast<const T *>(a.logits) + b * a.stride_b + k * a.stride_k;
    // loads start on the 16-byte boundary at or before the row
    const int mis = (int)((reinterpret_cast<uintptr_t>(x0) & 15) / sizeof(T));
    const uint4 *base = reinterpret_cast<const uint4 *>(x0 - mis);
    float x[kPerThread];
    auto word_of = [&](int j) {  // of x[j]
        return slice * kSlice + ((j / V) * kThreads + (int)threadIdx.x) * V + j % V - mis;
    };
#pragma unroll
    for (int j = 0; j < kPerThread; j += V) {
        const int w = word_of(j);
        uint4 u = make_uint4(0, 0, 0, 0);
        if (w < a.vocab && w + V > 0) u = __ldg(base + (slice * kSlice / V + (j / V) * kThreads + threadIdx.x));
        const uint32_t r[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float f;
            if constexpr (DT == LQ_F32) f = __uint_as_float(r[e]);
            else if constexpr (DT == LQ_F16) f = __half2float(__ushort_as_half((uint16_t)(r[e / 2] >> (16 * (e & 1)))));
            else f = __uint_as_float(e & 1 ? r[e / 2] & 0xffff0000u : r[e / 2] << 16);
            x[j + e] = w + e >= 0 && w + e < a.vocab && f == f ? f : -INFINITY;
        }
    }
    float mx = x[0];
#pragma unroll
    for (int j = 1; j < kPerThread; ++j) mx = fmaxf(mx, x[j]);

    const uint32_t best = ordered(mx);
    find_bound(best, a.n, s);
    const uint32_t bound = max(s.bound, 1u);
    if (best >= bound) {
#pragma unroll
        for (int j = 0; j < kPerThread; ++j)
            if (ordered(x[j]) >= bound)
                pick(s, 0u, (uint64_t)ordered(x[j]) << 24 | (kWordMask - (uint32_t)word_of(j)));
    }

    // the slice's maximum and sum of exponentials
    float top = mx;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, red[w]);
    float sum = 0.f;
    if (top > -INFINITY) {
#pragma unroll
        for (int j = 0; j < kPerThread; ++j) sum += exp2f((x[j] - top) * kLog2e);
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) red[kWarps + (threadIdx.x >> 5)] = sum;
    __syncthreads();
    const int64_t at = (int64_t)row * a.slices + slice;
    if (threadIdx.x == 0) {
        float all = 0.f;
        for (int w = 0; w < kWarps; ++w) all += red[kWarps + w];
        a.stat[at] = make_float2(top, all);
    }

    uint64_t *out = a.keys + at * a.n;
    auto emit = [&](int i, const Key &key) { out[i] = key.lo; };
    if (!rank_picked(s, a.n, emit))
        rank_by_rounds(
            s, a.n,
            [&](const Key &under) {
                Key best{0u, 0ull};
#pragma unroll
                for (int j = 0; j < kPerThread; ++j) {
                    const uint32_t o = ordered(x[j]);
                    const uint64_t lo = o ? (uint64_t)o << 24 | (kWordMask - (uint32_t)word_of(j)) : 0ull;
                    if (lo < under.lo && lo > best.lo) best.lo = lo;
                }
                best.hi = best.lo ? 1u : 0u;
                return best;
            },
            emit);
}

__global__ void __launch_bounds__(kThreads) beam_merge_kernel(const __grid_constant__ BeamArgs a) {
    __shared__ Picker s;
    __shared__ float lse[kMaxBeams], score[kMaxBeams];
    const int b = blockIdx.x, lane = threadIdx.x & 31;
    for (int k = threadIdx.x >> 5; k < a.beams; k += kWarps) {
        const float2 *st = a.stat + ((int64_t)b * a.beams + k) * a.slices;
        float m = -INFINITY;
        for (int i = lane; i < a.slices; i += 32) m = fmaxf(m, st[i].x);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        float sum = 0.f;
        for (int i = lane; i < a.slices; i += 32)
            if (st[i].x > -INFINITY) sum += st[i].y * exp2f((st[i].x - m) * kLog2e);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            lse[k] = m + logf(sum);
            score[k] = a.scores[(int64_t)b * a.beams + k];
        }
    }
    __syncthreads();
    const int per_beam = a.slices * a.n, total = a.beams * per_beam;
    const uint64_t *keys = a.keys + (int64_t)b * total;
    auto key_of = [&](int i) {
        const uint64_t lo = keys[i];
        const int k = i / per_beam;
        const float v = __fadd_rn(__fsub_rn(from_ordered((uint32_t)(lo >> 24)), lse[k]), score[k]);
        return lo ? Key{ordered(v), (uint64_t)(255 - k) << 56 | lo} : Key{0u, 0ull};
    };
    uint32_t best = 0;
    for (int i = threadIdx.x; i < total; i += kThreads) best = max(best, key_of(i).hi);
    find_bound(best, a.n, s);
    const uint32_t bound = max(s.bound, 1u);
    if (best >= bound)
        for (int i = threadIdx.x; i < total; i += kThreads) {
            const Key k = key_of(i);
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
                    const Key k = key_of(i);
                    if (under > k && k > top) top = k;
                }
                return top;
            },
            emit);
}

int slices_of(int64_t vocab) { return (int)ceil_div(vocab + 7, kSlice); }  // a misaligned row starts up to 7 words in

bool beam_ok(int64_t batch, int64_t beams, int64_t vocab, int64_t n) {
    return batch >= 0 && beams >= 1 && beams <= kMaxBeams && vocab >= 1 && vocab <= kMaxVocab && n >= 1 && n <= kMaxN &&
           batch * beams <= 65535 && beams * slices_of(vocab) * n <= 0x7fffffff;
}

size_t stat_bytes(int64_t rows, int slices) { return (size_t)rows * slices * sizeof(float2); }

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_beam_select_workspace(int64_t batch, int64_t beams, int64_t vocab, int64_t n) {
    if (!beam_ok(batch, beams, vocab, n)) return 0;
    const int64_t rows = batch * beams;
    return stat_bytes(rows, slices_of(vocab)) + (size_t)rows * slices_of(vocab) * n * 8;
}

extern "C" int lq_beam_select(const void *logits, int dtype, int64_t batch, int64_t beams, int64_t vocab,
                              int64_t stride_b, int64_t stride_k, const float *scores, int64_t n, float *top_score,
                              int64_t *top_beam, int64_t *top_word, void *workspace, size_t workspace_bytes,
                              void *stream) {
    LQ_NVTX_RANGE();
    if (!beam_ok(batch, beams, vocab, n)) return LQ_ERR_INVALID;
    if (batch == 0) return LQ_OK;
    if (!logits || !scores || !top_score || !top_beam || !top_word || !workspace) return LQ_ERR_INVALID;
    if (workspace_bytes < lq_beam_select_workspace(batch, beams, vocab, n)) return LQ_ERR_CAPACITY;
    BeamArgs a{};
    a.logits = logits;
    a.stride_b = stride_b;
    a.stride_k = stride_k;
    a.scores = scores;
    a.beams = (int)beams;
    a.vocab = (int)vocab;
    a.n = (int)n;
    a.slices = slices_of(vocab);
    a.stat = static_cast<float2 *>(workspace);
    a.keys = reinterpret_cast<uint64_t *>(static_cast<char *>(workspace) + stat_bytes(batch * beams, a.slices));
    a.top_score = top_score;
    a.top_beam = top_beam;
    a.top_word = top_word;
    cudaStream_t st = as_stream(stream);
    const dim3 grid((unsigned)a.slices, (unsigned)(batch * beams));
    if (dtype == LQ_F32) beam_slice_kernel<LQ_F32><<<grid, kThreads, 0, st>>>(a);
    else if (dtype == LQ_F16) beam_slice_kernel<LQ_F16><<<grid, kThreads, 0, st>>>(a);
    else if (dtype == LQ_BF16) beam_slice_kernel<LQ_BF16><<<grid, kThreads, 0, st>>>(a);
    else return LQ_ERR_INVALID;
    if (check_launch() != LQ_OK) return LQ_ERR_CUDA;
    beam_merge_kernel<<<(unsigned)batch, kThreads, 0, st>>>(a);
    return check_launch();
}
