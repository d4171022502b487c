// token_logprobs.hip -- log probabilities of given tokens, entropy and the
// largest alternatives of rows of logits, and their gradient.
//
// No reference counterpart: Ember's CrossEntropyLoss (ember/loss/losses.py:
// 29-56) takes a dense target of rows * classes floats and keeps the
// probabilities.  Here a row is read once and nothing of its size is written:
//   m = max x,  s = sum e^(x - m),  w = sum (x - m) e^(x - m)
//   lse = m + ln s,  logp = (x_tok - m) - ln s,  entropy = ln s - w / s
// Sums over parts of a row join by
//   s = sum s_i f_i,  w = sum (w_i + (m_i - m) s_i) f_i,  f_i = e^(m_i - m).
//
// A workgroup takes a segment of a row into registers (32 floats a thread), so
// that the maximum is known before the sums without a second read; segments of
// a row are joined by token_logprobs_join.  HBM-bound: 4 bytes per logit.
//
// The `top` largest: floats are ordered as unsigned integers (all bits turned
// over where the sign is set, else the sign alone), with the complement of the
// index below them, so that one comparison of 64 bits has the order asked for.
// Each wave keeps its best in order, one per lane.  A first bound is the k-th
// largest of its lanes' largest, to 16 bits, found by halving on ballots; the
// few elements from it on are put in one by one.
#include <math.h>

#include <algorithm>

#include "common.h"

namespace ember {
namespace {

constexpr int kMostTop = 64;
constexpr int kThreads = 256;
constexpr int kPerThread = 32;
constexpr int kSegment = kThreads * kPerThread;

typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));  // rows start anywhere

struct ScoreArgs {
    const float *x;
    const int32_t *tokens;
    float *logp, *lse, *entropy;
    int32_t *top_tokens;
    float *top_logp;
    float *part;      // m, s, w of each (row, segment)
    uint64_t *lists;  // its best, `top` keys
    int64_t stride;
    int rows, classes, segments, top;
};

struct Sums {
    float m, s, w;
};

// One side's part of a sum whose maximum is m.  Nothing is added where it holds
// nothing but -infinity (no inf - inf) or is too far below (no 0 * inf).
__device__ __forceinline__ Sums moved(Sums a, float m)
{
    const float d = a.s == 0.0f ? 0.0f : a.m - m, f = expf(d);
    return f == 0.0f ? Sums{m, 0.0f, 0.0f} : Sums{m, a.s * f, (a.w + d * a.s) * f};
}

__device__ __forceinline__ Sums join(Sums a, Sums b)
{
    const float m = fmaxf(a.m, b.m);
    a = moved(a, m), b = moved(b, m);
    return {m, a.s + b.s, a.w + b.w};
}

__device__ __forceinline__ uint64_t key_of(float x, int i)
{
    const unsigned u = __builtin_bit_cast(unsigned, x + 0.0f);  // -0 as 0
    const unsigned v = u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
    return ((uint64_t)v << 32) | (0xffffffffu - (unsigned)i);
}
__device__ __forceinline__ float value_of(uint64_t key)
{
    const unsigned v = (unsigned)(key >> 32);
    return __builtin_bit_cast(float, v ^ (v & 0x80000000u ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int index_of(uint64_t key)
{
    return (int)(0xffffffffu - (unsigned)key);
}

__device__ __forceinline__ uint64_t lane_key(uint64_t k, int lane)
{
    return ((uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(k >> 32), lane) << 32) |
           (unsigned)__builtin_amdgcn_readlane((int)(unsigned)k, lane);
}

// A wave's `top` largest keys, the largest in lane 0.  Empty places hold 0,
// below every key of a float.
struct Best {
    uint64_t mine = 0, last = 0;  // last: the lowest that is kept
    __device__ __forceinline__ void put(uint64_t key, int top)  // the same in every lane
    {
        const int at = __popcll(__ballot(mine > key));
        const uint64_t up = ((uint64_t)(unsigned)__shfl_up((int)(mine >> 32), 1, 64) << 32) | (unsigned)__shfl_up((int)(unsigned)mine, 1, 64);
        const int lane = threadIdx.x & 63;
        mine = lane < at ? mine : lane == at ? key : up;
        last = lane_key(mine, top - 1);
    }
    // Takes in one key of each lane (0: none).
    __device__ __forceinline__ void take(uint64_t key, int top)
    {
        for (uint64_t left = __ballot(key > last); left; left &= left - 1) {
            const uint64_t k = lane_key(key, __builtin_ctzll(left));
            if (k > last) put(k, top);
        }
    }
};

__device__ __forceinline__ Sums wave_join(Sums a)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a = join(a, Sums{__shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64), __shfl_xor(a.w, o, 64)});
    return a;
}

// The row's results, from its sums; `best` is lane i's i-th key.  One wave.
__device__ __forceinline__ void finish(const ScoreArgs &a, int row, Sums t, uint64_t best)
{
    const int lane = threadIdx.x & 63;
    const float logs = logf(t.s);
    if (lane == 0) {
        const int tok = a.tokens[row];
        a.logp[row] = tok >= 0 && tok < a.classes ? (a.x[row * a.stride + tok] - t.m) - logs : 0.0f;
        if (a.lse) a.lse[row] = t.m + logs;
        if (a.entropy) a.entropy[row] = logs - t.w / t.s;
    }
    if (lane < a.top) {
        a.top_tokens[(int64_t)row * a.top + lane] = index_of(best);
        a.top_logp[(int64_t)row * a.top + lane] = (value_of(best) - t.m) - logs;
    }
}

template <bool TOP>
__global__ __launch_bounds__(kThreads) void token_logprobs_kernel(ScoreArgs a)
{
    __shared__ Sums sums[4];
    __shared__ uint64_t lists[4][kMostTop];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.x / a.segments, seg = blockIdx.x - row * a.segments;
    const int64_t first = (int64_t)seg * kSegment;
    const float *p = a.x + row * a.stride + first;
    const int n = (int)min((int64_t)kSegment, a.classes - first);

    f4 x[kPerThread / 4];
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPerThread / 4; ++j) {
        const int c = 4 * (kThreads * j + (int)threadIdx.x);
        if (c + 4 <= n) {
            x[j] = *(const f4 *)(p + c);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[j][i] = c + i < n ? p[c + i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) m = fmaxf(m, x[j][i]);
    }
    Sums t = {m, 0.0f, 0.0f};
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int j = 0; j < kPerThread / 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float d = x[j][i] - ref, e = expf(d);
            t.s += e;
            t.w += e == 0.0f ? 0.0f : d * e;
        }
    t = wave_join(t);
    if (lane == 0) sums[wave] = t;

    if (TOP) {
        // The lanes' largest, and the k-th of them from below.
        unsigned most = 0;
        auto key = [&](int j, int i) {
            const int c = 4 * (kThreads * j + (int)threadIdx.x) + i;
            return c < n ? key_of(x[j][i], (int)first + c) : 0;
        };
#pragma unroll
        for (int j = 0; j < kPerThread / 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = max(most, (unsigned)(key(j, i) >> 32));
        unsigned bound = 0;
        for (unsigned bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
            if (__popcll(__ballot(most >= (bound | bit))) >= a.top) bound |= bit;
        Best best;
        best.last = bound ? ((uint64_t)bound << 32) - 1 : 0;
#pragma unroll
        for (int j = 0; j < kPerThread / 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint64_t k = key(j, i);
                for (uint64_t left = __ballot(k > best.last); left; left &= left - 1) {
                    const uint64_t one = lane_key(k, __builtin_ctzll(left));
                    if (one <= best.last) continue;
                    best.put(one, a.top);
                    if (bound) best.last = max(best.last, ((uint64_t)bound << 32) - 1);
                }
            }
        if (lane < a.top) lists[wave][lane] = best.mine;
    }
    __syncthreads();
    if (wave) return;
    t = join(join(sums[0], sums[1]), join(sums[2], sums[3]));
    Best best;
    if (TOP) {
        if (lane < a.top) best.mine = lists[0][lane];
        best.last = lane_key(best.mine, a.top - 1);
#pragma unroll
        for (int w = 1; w < 4; ++w) best.take(lane < a.top ? lists[w][lane] : 0, a.top);
    }
    if (a.segments == 1) {
        finish(a, row, t, best.mine);
        return;
    }
    if (lane == 0) *(Sums *)(a.part + 3 * (int64_t)blockIdx.x) = t;
    if (TOP && lane < a.top) a.lists[(int64_t)blockIdx.x * a.top + lane] = best.mine;
}

// One wave per row.
__global__ __launch_bounds__(64) void token_logprobs_join(ScoreArgs a)
{
    const int row = blockIdx.x, lane = threadIdx.x;
    const int64_t first = (int64_t)row * a.segments;
    Sums t = {-INFINITY, 0.0f, 0.0f};
    for (int s = lane; s < a.segments; s += 64) t = join(t, *(const Sums *)(a.part + 3 * (first + s)));
    t = wave_join(t);
    Best best;
    if (a.top)
        for (int s = 0; s < a.segments; s += 64)
            for (int i = 0; i < a.top; ++i) {
                const uint64_t k = s + lane < a.segments ? a.lists[(first + s + lane) * a.top + i] : 0;
                if (!__any(k > best.last)) break;  // nor the lists' further ones
                best.take(k, a.top);
            }
    finish(a, row, t, best.mine);
}

struct GradArgs {
    const float *x;
    const int32_t *tokens;
    const float *lse, *entropy, *d_logp, *d_entropy;
    float *dx;
    int64_t stride, out_stride;
    int rows, classes, segments;
};

constexpr int kGradSegment = kThreads * 16;

__global__ __launch_bounds__(kThreads) void token_logprobs_bwd_kernel(GradArgs a)
{
    const int row = blockIdx.x / a.segments, seg = blockIdx.x - row * a.segments;
    const int64_t first = (int64_t)seg * kGradSegment;
    const float *p = a.x + row * a.stride + first;
    float *q = a.dx + row * a.out_stride + first;
    const int n = (int)min((int64_t)kGradSegment, a.classes - first);
    const int token = a.tokens[row];
    const bool known = token >= 0 && token < a.classes;
    const int at = known ? (int)max(min(token - first, (int64_t)kGradSegment), (int64_t)-1) : -1;
    const float lse = a.lse[row], dp = known && a.d_logp ? a.d_logp[row] : 0.0f;
    const float dh = a.d_entropy ? a.d_entropy[row] : 0.0f, h = dh != 0.0f ? a.entropy[row] : 0.0f;
    auto grad = [&](float x, int c) {
        const float logp = x - lse, pr = expf(logp);
        // p ln p is 0 where p is.
        const float g = -pr * (dp + (pr == 0.0f ? 0.0f : dh * (logp + h)));
        return c == at ? g + dp : g;
    };
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = 4 * (kThreads * j + (int)threadIdx.x);
        if (c + 4 <= n) {
            const f4 x = *(const f4 *)(p + c);
            f4 y;
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = grad(x[i], c + i);
            *(f4 *)(q + c) = y;
        } else {
            for (int i = 0; i < 4; ++i)
                if (c + i < n) q[c + i] = grad(p[c + i], c + i);
        }
    }
}

constexpr int64_t kMostClasses = 0x7fffffff - 65535;
constexpr int64_t kMostBlocks = (int64_t(1) << 32) / kThreads - 1;  // a grid's threads are counted in 32 bits

}  // namespace
}  // namespace ember

extern "C" int token_logprobs(const float *logits, int64_t row_stride, const int32_t *tokens, int64_t rows, int64_t classes,
                              float *logp, float *lse, float *entropy, int32_t *top_tokens, float *top_logp, int top)
{
    using namespace ember;
    const char *what = "token_logprobs";
    const int64_t segments = (classes + kSegment - 1) / kSegment;
    if (rows < 0 || classes < 1 || classes > kMostClasses || row_stride < classes || top < 0 || top > kMostTop || top > classes ||
        rows > kMostBlocks / segments)
        return record_error(EMBER_ERR_INVALID_ARGUMENT, what);
    if (rows == 0) return EMBER_OK;
    if (!logits || !tokens || !logp || (top && (!top_tokens || !top_logp)) ||
        (((uintptr_t)logits | (uintptr_t)tokens | (uintptr_t)logp | (uintptr_t)lse | (uintptr_t)entropy | (uintptr_t)top_tokens | (uintptr_t)top_logp) & 3))
        return record_error(EMBER_ERR_INVALID_ARGUMENT, what);
    ScoreArgs a = {logits, tokens, logp, lse, entropy, top_tokens, top_logp, nullptr, nullptr, row_stride, (int)rows, (int)classes, (int)segments, top};
    const int64_t blocks = rows * segments;
    if (segments > 1) {
        const size_t lists = ((size_t)blocks * 12 + 15) / 16 * 16;
        char *ws = (char *)scratch(kScratchLogprobs, lists + (size_t)blocks * top * 8);
        if (!ws) return EMBER_ERR_OUT_OF_MEMORY;
        a.part = (float *)ws, a.lists = (uint64_t *)(ws + lists);
    }
    if (top) hipLaunchKernelGGL(token_logprobs_kernel<true>, dim3((unsigned)blocks), dim3(kThreads), 0, 0, a);
    else hipLaunchKernelGGL(token_logprobs_kernel<false>, dim3((unsigned)blocks), dim3(kThreads), 0, 0, a);
    if (!launch_ok("token_logprobs")) return EMBER_ERR_DEVICE;
    if (segments > 1) {
        hipLaunchKernelGGL(token_logprobs_join, dim3((unsigned)rows), dim3(64), 0, 0, a);
        if (!launch_ok("token_logprobs_join")) return EMBER_ERR_DEVICE;
    }
    return EMBER_OK;
}

extern "C" int token_logprobs_bwd(const float *logits, int64_t row_stride, const int32_t *tokens, const float *lse,
                                  const float *entropy, const float *d_logp, const float *d_entropy, float *d_logits,
                                  int64_t out_stride, int64_t rows, int64_t classes)
{
    using namespace ember;
    const char *what = "token_logprobs_bwd";
    const int64_t segments = (classes + kGradSegment - 1) / kGradSegment;
    if (rows < 0 || classes < 1 || classes > kMostClasses || row_stride < classes || out_stride < classes || rows > kMostBlocks / segments)
        return record_error(EMBER_ERR_INVALID_ARGUMENT, what);
    if (rows == 0) return EMBER_OK;
    if (!logits || !tokens || !lse || !d_logits || (d_entropy && !entropy) || (logits == d_logits && row_stride != out_stride) ||
        (((uintptr_t)logits | (uintptr_t)tokens | (uintptr_t)lse | (uintptr_t)entropy | (uintptr_t)d_logp | (uintptr_t)d_entropy | (uintptr_t)d_logits) & 3))
        return record_error(EMBER_ERR_INVALID_ARGUMENT, what);
    const GradArgs a = {logits, tokens, lse, entropy, d_logp, d_entropy, d_logits, row_stride, out_stride, (int)rows, (int)classes, (int)segments};
    hipLaunchKernelGGL(token_logprobs_bwd_kernel, dim3((unsigned)(rows * segments)), dim3(kThreads), 0, 0, a);
    return launch_ok(what) ? EMBER_OK : EMBER_ERR_DEVICE;
}
