// token_logprobs.hip -- log probabilities of given tokens, entropy and the
// largest alternatives of rows of logits, and their gradient.
//
// No reference counterpart: Ember's CrossEntropyLoss (ember/loss/losses.py:
// 29-56) takes a dense target of rows * classes floats and keeps the
// probabilities.  Here a row is read once and nothing of its size is written:
//   m = max x,  s = sum e^(x - m),  w = sum (x - m) e^(x - m)
//   lse = m + ln s,  logp = (x_tok - m) - ln s,  entropy = ln s - w / s
// (and what rounding lse leaves out, for the gradient: where m is far from 0, ln s
// has few bits left in lse.)
// Sums over parts of a row join by
//   s = sum s_i f_i,  w = sum (w_i + (m_i - m) s_i) f_i,  f_i = e^(m_i - m).
//
// A thread takes 16 logits at a time into registers, so that their maximum is
// known before the sums, and the next 16 are on their way meanwhile; where rows
// are few, a row is cut over workgroups, and the last of them to be done (by a
// count that they add to) joins their sums.  HBM-bound: 4 bytes per logit, read
// past the caches (4096 x 32001: 88 us, 6.0 TB/s; through them 98).
//
// The `top` largest: floats are ordered as unsigned integers (all bits turned
// over where the sign is set, else the sign alone), with the complement of the
// index below them, so that one comparison of 64 bits has the order asked for.
// Each wave keeps its best in order, one per lane, and tests each logit against
// the last of them; before it has any, against the k-th largest of its lanes'
// largest (found to 16 bits, by halving on ballots), so that few are put in that
// do not stay.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "lds_dma.h"
#include "wave.h"

namespace ember {
namespace {

constexpr int kMostTop = 64;
constexpr int kThreads = 256;
constexpr int kPerThread = 16;
constexpr int kChunk = kThreads * kPerThread;
constexpr int kMostRows = 1 << 13;  // that are cut
constexpr int kKeys = 2048;         // of lists that are joined at a time,
constexpr int kNear = 8;            // the first ones of each
constexpr float kLog2e = 1.4426950408889634f;

typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));  // rows start anywhere

struct ScoreArgs {
    const float *x;
    const int32_t *tokens;
    float *logp, *lse, *rest, *entropy;
    int32_t *top_tokens;
    float *top_logp;
    char *part;  // of each workgroup: m, s, w, and its waves' best (`top` keys each); null: rows are not cut
    int64_t stride;
    int rows, classes, chunks, pieces, per, top;  // chunks of a row, pieces that it is cut into, chunks of a piece
    int row0;
};

// Rows that are cut: how many of their workgroups are done.  Zero between
// launches: the last one, which all the others have added to, clears its row's.
// All calls run on the null stream, so no two use it at once.
__device__ unsigned g_rows_done[kMostRows];

struct Sums {
    float m, s, w;
};

// One side's part of a sum whose maximum is m.  A side that holds nothing but
// -infinity stays 0 (no inf - inf); one that is too far below adds no w (no 0 *
// inf), but a NaN in its s stays.
__device__ __forceinline__ Sums moved(Sums a, float m)
{
    const float d = a.s == 0.0f ? 0.0f : a.m - m, f = expf(d);
    return {m, a.s * f, f == 0.0f ? 0.0f : (a.w + d * a.s) * f};
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
    const unsigned v = x == x ? u ^ ((unsigned)((int)u >> 31) | 0x80000000u) : 0xffffffffu;
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

// Appends the lanes' keys above `last` to `found`, which has c; returns how many
// there are then (those past kFound are not kept).
constexpr int kFound = 256;
__device__ __forceinline__ int gather(uint64_t *found, int c, uint64_t key, uint64_t last)
{
    const uint64_t some = __ballot(key > last);
    const int at = c + __builtin_amdgcn_mbcnt_hi((unsigned)(some >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)some, 0));
    if (key > last && at < kFound) found[at] = key;
    return c + __popcll(some);
}

// A wave's `top` largest keys, the largest in lane 0.  Empty places hold 0,
// below every key of a float.  Only keys above `last` are taken: the lowest that
// is kept, or a bound that at least `top` others are known to pass.
struct Best {
    uint64_t mine = 0, last = 0;
    __device__ __forceinline__ void put(uint64_t key, int top)  // the same in every lane
    {
        const int at = __popcll(__ballot(mine > key)), lane = threadIdx.x & 63;
        // From the lane below (a wave's shift by one, in registers).
        const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(mine >> 32), 0x138, 0xf, 0xf, false);
        const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)mine, 0x138, 0xf, 0xf, false);
        mine = lane < at ? mine : lane == at ? key : ((uint64_t)hi << 32) | lo;
        const uint64_t l = lane_key(mine, top - 1);
        last = l > last ? l : last;
    }
    // Takes in one key of each lane (0: none).
    __device__ __forceinline__ void take(uint64_t key, int top)
    {
        for (uint64_t left = __ballot(key > last); left; left &= left - 1) {
            const uint64_t k = lane_key(key, __builtin_ctzll(left));
            if (k > last) put(k, top);
        }
    }
    // Of two keys of each lane (their upper halves; 0: none): the k-th largest, cut
    // to 16 bits, is a bound (none if there are fewer).
    __device__ __forceinline__ void raise(unsigned u0, unsigned u1, int top)
    {
        unsigned bound = 0;
        for (unsigned bit = 0x80000000u; bit >= 0x10000u; bit >>= 1) {
            const unsigned to = bound | bit;
            if (__popcll(__ballot(u0 >= to)) + __popcll(__ballot(u1 >= to)) >= top) bound = to;
        }
        const uint64_t l = bound ? ((uint64_t)bound << 32) - 1 : 0;
        last = l > last ? l : last;
    }
    // The `top` largest of c keys in `found` (c <= 64 * N), each put where the
    // number of larger ones says; `found` is used up.
    template <int N>
    __device__ __forceinline__ void sort(uint64_t *found, int c, int top)
    {
        const int lane = threadIdx.x & 63;
        wave_sync();
        uint64_t k[N];
        int above[N];
#pragma unroll
        for (int j = 0; j < N; ++j) k[j] = lane + 64 * j < c ? found[lane + 64 * j] : 0, above[j] = 0;
#pragma unroll 8
        for (int i = 0; i < c; ++i) {
            const uint64_t other = found[i];
#pragma unroll
            for (int j = 0; j < N; ++j) above[j] += other > k[j];
        }
        wave_sync();
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (lane + 64 * j < c && above[j] < top) found[above[j]] = k[j];
        wave_sync();
        mine = lane < min(c, top) ? found[lane] : 0;
        const uint64_t l = lane_key(mine, top - 1);
        last = l > last ? l : last;
    }
    __device__ __forceinline__ void sort(uint64_t *found, int c, int top)
    {
        if (c <= 128) sort<2>(found, c, top);
        else sort<4>(found, c, top);
    }
    // Takes in n sorted lists of `top` keys: key(i, at) is list i's `at`-th, and the
    // first `near` of a list are at hand.
    template <class F>
    __device__ __forceinline__ void join(int n, int near, int top, uint64_t *found, F key)
    {
        const int lane = threadIdx.x & 63;
        // A bound from the lists' first keys: two places of a list (or lists) to a lane.
        unsigned head[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = lane + 64 * j, at = n < 128 ? i / n : 0;
            uint64_t k = at < near ? key(i - at * n, at) : 0;
            for (int more = i + 128; more < n; more += 128) k = max(k, key(more, 0));
            head[j] = (unsigned)(k >> 32);
        }
        raise(head[0], head[1], top);
        auto all = [&](auto f) {
            for (int i = lane; i - lane < n; i += 64)
                for (int at = 0; at < top; ++at) {
                    const uint64_t k = i < n ? key(i, at) : 0;
                    if (!__any(k > last)) break;  // nor the lists' further ones
                    f(k);
                }
        };
        int c = gather(found, 0, mine, 0);
        all([&](uint64_t k) { c = gather(found, c, k, last); });
        if (c <= kFound) sort(found, c, top);
        else all([&](uint64_t k) { take(k, top); });
    }
};

__device__ __forceinline__ Sums wave_join(Sums a)
{
    a = moved(a, wave_max(a.m));
    return {a.m, wave_sum(a.s), wave_sum(a.w)};
}

// The row's results, from its sums and its token's logit; `best` is lane i's i-th
// key.  One wave.
__device__ __forceinline__ void finish(const ScoreArgs &a, int row, Sums t, bool known, float of_token, uint64_t best)
{
    const int lane = threadIdx.x & 63;
    const float logs = logf(t.s);
    if (lane == 0) {
        a.logp[row] = known ? (of_token - t.m) - logs : 0.0f;
        const float lse = t.m + logs, moved = lse - t.m;
        if (a.lse) a.lse[row] = lse;
        if (a.rest) a.rest[row] = fabsf(lse) < INFINITY ? (t.m - (lse - moved)) + (logs - moved) : 0.0f;
        if (a.entropy) a.entropy[row] = logs - t.w / t.s;
    }
    if (lane < a.top) {
        a.top_tokens[(int64_t)row * a.top + lane] = index_of(best);
        a.top_logp[(int64_t)row * a.top + lane] = (value_of(best) - t.m) - logs;
    }
}

// Sums over 16 more logits; missing ones are -infinity.
__device__ __forceinline__ void add(Sums &t, const f4 *x, float most)
{
    const float m = fmaxf(t.m, most), ref = m == -INFINITY ? 0.0f : m;
    if (__any(t.m < m)) {
        t = moved(t, ref);
        t.m = m;
    }
    float s = t.s, w = t.w;
#pragma unroll
    for (int j = 0; j < kPerThread / 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float d = x[j][i] - ref, e = __builtin_amdgcn_exp2f(d * kLog2e);
            s += e;
            w = fmaf(d, e, w);
        }
    if (__any(w != w)) {  // -infinity among them: 0 there, and not 0 * inf
        w = t.w;
#pragma unroll
        for (int j = 0; j < kPerThread / 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float d = x[j][i] - ref, e = __builtin_amdgcn_exp2f(d * kLog2e);
                w += e == 0.0f ? 0.0f : d * e;
            }
    }
    t.s = s, t.w = w;
}

template <bool TOP>
__global__ __launch_bounds__(kThreads) void token_logprobs_kernel(ScoreArgs a)
{
    __shared__ Sums sums[4];
    __shared__ uint64_t lists[TOP ? kKeys : 1], found[TOP ? 4 : 1][kFound];
    __shared__ bool last;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int index = blockIdx.x / a.pieces, piece = blockIdx.x - index * a.pieces, row = a.row0 + index;
    const float *p = a.x + row * a.stride;
    const int end = min((piece + 1) * a.per, a.chunks);

    f4 x[kPerThread / 4], next[kPerThread / 4];
    auto load = [&](f4 *to, int chunk) {
        const int64_t first = (int64_t)chunk * kChunk + 4 * (int)threadIdx.x;
        if ((int64_t)(chunk + 1) * kChunk <= a.classes) {
#pragma unroll
            for (int j = 0; j < kPerThread / 4; ++j) to[j] = __builtin_nontemporal_load((const f4 *)(p + first + 4 * kThreads * j));
        } else {
#pragma unroll
            for (int j = 0; j < kPerThread / 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t c = first + 4 * kThreads * j + i;
                    to[j][i] = c < a.classes ? p[c] : -INFINITY;
                }
        }
    };
    Sums t = {-INFINITY, 0.0f, 0.0f};
    Best best;
    load(next, piece * a.per);
    // Beside the first chunk, not at the end, where nothing hides two loads in turn.
    const int token = a.tokens[row];
    const bool known = token >= 0 && token < a.classes;
    const float of_token = p[known ? token : 0];
    for (int chunk = piece * a.per; chunk < end; ++chunk) {
        float half[2] = {-INFINITY, -INFINITY};  // the largest of 8
#pragma unroll
        for (int j = 0; j < kPerThread / 4; ++j) {
            x[j] = next[j];
            half[j & 1] = fmaxf(half[j & 1], fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])));
        }
        if (chunk + 1 < end) load(next, chunk + 1);
        add(t, x, fmaxf(half[0], half[1]));
        if (TOP) {
            const int64_t first = (int64_t)chunk * kChunk + 4 * (int)threadIdx.x;
            auto all = [&](auto f) {
#pragma unroll
                for (int j = 0; j < kPerThread / 4; ++j) {
                    // Below the last that is kept?  (A NaN goes with the others of its
                    // four; its place in the order is not specified.)
                    const float least = value_of(best.last + 1);
                    if (!__any(!(fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])) < least))) continue;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int64_t c = first + 4 * kThreads * j + i;
                        f(c < a.classes ? key_of(x[j][i], (int)c) : 0);
                    }
                }
            };
            auto take = [&](uint64_t k) { best.take(k, a.top); };
            if (chunk == piece * a.per) {
                best.raise((unsigned)(key_of(half[0], 0) >> 32), (unsigned)(key_of(half[1], 0) >> 32), a.top);
                int c = 0;
                all([&](uint64_t k) { c = gather(found[wave], c, k, best.last); });
                if (c <= kFound) best.sort(found[wave], c, a.top);
                else all(take);
            } else {
                all(take);
            }
        }
    }
    t = wave_join(t);
    if (lane == 0) sums[wave] = t;
    if (a.pieces > 1) {
        const int64_t size = 16 + 32 * (int64_t)a.top;
        char *mine = a.part + blockIdx.x * size;
        if (TOP && lane < a.top) put8(mine + 16 + 8 * (wave * a.top + lane), best.mine);
        __syncthreads();
        if (threadIdx.x == 0) {
            t = join(join(sums[0], sums[1]), join(sums[2], sums[3]));
            put8(mine, (uint64_t)__builtin_bit_cast(unsigned, t.s) << 32 | __builtin_bit_cast(unsigned, t.m));
            put8(mine + 8, __builtin_bit_cast(unsigned, t.w));
        }
        wait_vmem();  // the stores have reached memory
        __syncthreads();
        if (threadIdx.x == 0) last = last_of(&g_rows_done[index], a.pieces);
        __syncthreads();
        if (!last) return;
        const char *from = a.part + (int64_t)index * a.pieces * size;
        constexpr int at_once = kKeys / (4 * kNear);  // pieces
        uint64_t k[kKeys / kThreads];
        auto place = [&](int i, int at) { return from + (i >> 2) * size + 16 + 8 * ((i & 3) * a.top + at); };
        // The first keys of the lists of pieces i0 .., a thread's loads on their way together.
        auto heads = [&](int i0) {
#pragma unroll
            for (int j = 0; j < kKeys / kThreads; ++j) {
                const int i = 4 * i0 + (j * kThreads + (int)threadIdx.x) / kNear, at = threadIdx.x % kNear;
                k[j] = i < 4 * a.pieces && at < a.top ? get8(place(i, at)) : 0;
            }
        };
        if (TOP) heads(0);
        t = {-INFINITY, 0.0f, 0.0f};
        for (int i = threadIdx.x; i < a.pieces; i += kThreads) {
            const uint64_t ms = get8(from + i * size), w = get8(from + i * size + 8);
            t = join(t, Sums{__builtin_bit_cast(float, (unsigned)ms), __builtin_bit_cast(float, (unsigned)(ms >> 32)),
                             __builtin_bit_cast(float, (unsigned)w)});
        }
        t = wave_join(t);
        if (lane == 0) sums[wave] = t;
        if (TOP) {
            best = Best();
            for (int i0 = 0; i0 < a.pieces; i0 += at_once) {
                if (i0) {
                    __syncthreads();
                    heads(i0);
                }
#pragma unroll
                for (int j = 0; j < kKeys / kThreads; ++j) lists[j * kThreads + threadIdx.x] = k[j];
                __syncthreads();
                if (wave == 0)
                    best.join(4 * min(at_once, a.pieces - i0), min(kNear, a.top), a.top, found[0],
                              [&](int i, int at) { return at < kNear ? lists[i * kNear + at] : get8(place(4 * i0 + i, at)); });
            }
        }
    } else if (TOP) {
        if (lane < a.top) lists[wave * a.top + lane] = best.mine;
    }
    __syncthreads();
    if (wave) return;
    t = join(join(sums[0], sums[1]), join(sums[2], sums[3]));
    if (TOP && a.pieces == 1) {
        best = Best();
        if (4 * a.top <= 128) best.sort<2>(lists, 4 * a.top, a.top);
        else best.join(4, a.top, a.top, found[0], [&](int i, int at) { return lists[i * a.top + at]; });
    }
    finish(a, row, t, known, of_token, best.mine);
}

// The gradient: each logit read once and each result written once, 8 bytes an element
// (4096 x 50021: 293 us, 5.6 TB/s, above the rate of a large copy).  A workgroup takes
// 4096 neighbours of a row, so that a row of any length has enough of them.  Past the
// caches as the forward: 295 and 293, so plain.
struct GradArgs {
    const float *x;
    const int32_t *tokens;
    const float *lse, *rest, *entropy, *d_logp, *d_entropy;
    float *dx;
    int64_t stride, out_stride;
    int classes, segments, row0;
};

constexpr int kGradSegment = kThreads * 16;

__global__ __launch_bounds__(kThreads) void token_logprobs_bwd_kernel(GradArgs a)
{
    const int index = blockIdx.x / a.segments, seg = blockIdx.x - index * a.segments, row = a.row0 + index;
    const int64_t first = (int64_t)seg * kGradSegment;
    const float *p = a.x + row * a.stride + first;
    float *q = a.dx + row * a.out_stride + first;
    const int n = (int)min((int64_t)kGradSegment, a.classes - first);
    const int token = a.tokens[row];
    const bool known = token >= 0 && token < a.classes;
    const int at = known ? (int)max(min(token - first, (int64_t)kGradSegment), (int64_t)-1) : -1;
    const float lse = a.lse[row], rest = a.rest ? a.rest[row] : 0.0f, dp = known && a.d_logp ? a.d_logp[row] : 0.0f;
    const float dh = a.d_entropy ? a.d_entropy[row] : 0.0f, h = dh != 0.0f ? a.entropy[row] : 0.0f;
    if (dp == 0.0f && dh == 0.0f) {  // a padded row: whatever it holds
        for (int c = threadIdx.x; c < n; c += kThreads) q[c] = 0.0f;
        return;
    }
    auto grad = [&](float x, int c) {
        const float logp = (x - lse) - rest, pr = expf(logp);
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

// Whether two arrays of `rows` rows of `classes` floats, both `stride` apart, have
// an element in common, the same rows aside.
bool rows_meet(const float *x, const float *y, int64_t stride, int64_t rows, int64_t classes)
{
    const uintptr_t a = (uintptr_t)x, b = (uintptr_t)y;
    const int64_t apart = (int64_t)((a < b ? b - a : a - b) / sizeof(float)), over = apart / stride, left = apart - over * stride;
    return apart && ((over < rows && left < classes) || (over + 1 < rows && stride - left < classes));
}

}  // namespace
}  // namespace ember

extern "C" int token_logprobs_ex(const float *logits, int64_t row_stride, const int32_t *tokens, int64_t rows, int64_t classes,
                                 float *logp, float *lse, float *lse_rest, float *entropy, int32_t *top_tokens, float *top_logp,
                                 int top)
{
    using namespace ember;
    const char *what = "token_logprobs";
    if (rows < 0 || rows > 0x7fffffff || classes < 1 || classes > kMostClasses || row_stride < classes || top < 0 || top > kMostTop ||
        top > classes)
        return record_error(EMBER_ERR_INVALID_ARGUMENT, what);
    if (rows == 0) return EMBER_OK;
    if (!logits || !tokens || !logp || (top && (!top_tokens || !top_logp)) ||
        (((uintptr_t)logits | (uintptr_t)tokens | (uintptr_t)logp | (uintptr_t)lse | (uintptr_t)lse_rest | (uintptr_t)entropy | (uintptr_t)top_tokens | (uintptr_t)top_logp) & 3))
        return record_error(EMBER_ERR_INVALID_ARGUMENT, what);
    ScoreArgs a = {logits, tokens, logp, lse, lse_rest, entropy, top_tokens, top_logp, nullptr, row_stride, (int)rows, (int)classes};
    a.chunks = (int)((classes + kChunk - 1) / kChunk), a.top = top;
    // A row to a workgroup, unless there are too few for the chip: then pieces, 8 to
    // a CU (which holds 8 at once without alternatives; with them 5, by their 86
    // registers and 24.6 KB), but of a chunk at least.
    const int64_t slots = std::min<int64_t>(8 * (int64_t)std::max(device_cu_count(), 1), kMostRows);
    a.pieces = (int)std::max<int64_t>(1, std::min<int64_t>(a.chunks, slots / rows));
    a.per = (a.chunks + a.pieces - 1) / a.pieces;
    a.pieces = (a.chunks + a.per - 1) / a.per;
    if (a.pieces > 1) {  // then there are no more rows than slots
        a.part = (char *)scratch(kScratchLogprobs, (size_t)rows * a.pieces * (16 + 32 * top));
        if (!a.part) return EMBER_ERR_OUT_OF_MEMORY;
    }
    const int64_t most = kMostBlocks / a.pieces;
    for (int64_t row = 0; row < rows; row += most) {
        a.row0 = (int)row;
        const unsigned blocks = (unsigned)(std::min(most, rows - row) * a.pieces);
        if (top) hipLaunchKernelGGL(token_logprobs_kernel<true>, dim3(blocks), dim3(kThreads), 0, 0, a);
        else hipLaunchKernelGGL(token_logprobs_kernel<false>, dim3(blocks), dim3(kThreads), 0, 0, a);
        if (!launch_ok("token_logprobs")) return EMBER_ERR_DEVICE;
    }
    return EMBER_OK;
}

extern "C" int token_logprobs(const float *logits, int64_t row_stride, const int32_t *tokens, int64_t rows, int64_t classes,
                              float *logp, float *lse, float *entropy, int32_t *top_tokens, float *top_logp, int top)
{
    return token_logprobs_ex(logits, row_stride, tokens, rows, classes, logp, lse, nullptr, entropy, top_tokens, top_logp, top);
}

extern "C" int token_logprobs_bwd_ex(const float *logits, int64_t row_stride, const int32_t *tokens, const float *lse,
                                     const float *lse_rest, const float *entropy, const float *d_logp, const float *d_entropy,
                                     float *d_logits, int64_t out_stride, int64_t rows, int64_t classes)
{
    using namespace ember;
    const char *what = "token_logprobs_bwd";
    const int64_t segments = (classes + kGradSegment - 1) / kGradSegment;
    if (rows < 0 || rows > 0x7fffffff || classes < 1 || classes > kMostClasses || row_stride < classes || out_stride < classes)
        return record_error(EMBER_ERR_INVALID_ARGUMENT, what);
    if (rows == 0) return EMBER_OK;
    if (!logits || !tokens || !lse || !d_logits || (d_entropy && !entropy) || (logits == d_logits && row_stride != out_stride) ||
        (row_stride == out_stride && rows_meet(logits, d_logits, row_stride, rows, classes)) ||
        (((uintptr_t)logits | (uintptr_t)tokens | (uintptr_t)lse | (uintptr_t)lse_rest | (uintptr_t)entropy | (uintptr_t)d_logp | (uintptr_t)d_entropy | (uintptr_t)d_logits) & 3))
        return record_error(EMBER_ERR_INVALID_ARGUMENT, what);
    GradArgs a = {logits, tokens, lse, lse_rest, entropy, d_logp, d_entropy, d_logits, row_stride, out_stride, (int)classes, (int)segments};
    const int64_t most = kMostBlocks / segments;
    for (int64_t row = 0; row < rows; row += most) {
        a.row0 = (int)row;
        hipLaunchKernelGGL(token_logprobs_bwd_kernel, dim3((unsigned)(std::min(most, rows - row) * segments)), dim3(kThreads), 0, 0, a);
        if (!launch_ok(what)) return EMBER_ERR_DEVICE;
    }
    return EMBER_OK;
}

extern "C" int token_logprobs_bwd(const float *logits, int64_t row_stride, const int32_t *tokens, const float *lse,
                                  const float *entropy, const float *d_logp, const float *d_entropy, float *d_logits,
                                  int64_t out_stride, int64_t rows, int64_t classes)
{
    return token_logprobs_bwd_ex(logits, row_stride, tokens, lse, nullptr, entropy, d_logp, d_entropy, d_logits, out_stride, rows, classes);
}
