// gated.hip -- gated feed-forward layers in fp32: h = act(x wg + bg) * (x wu + bu)
// and the gradient with respect to both sums.  No reference counterpart:
// pawel002/ember composes feed-forward layers from Linear and an activation.
//   forward:  pre = x [wg | wu] + bias;  h = act(gate) * up  (gate, up: pre's halves)
//   backward: dh = dy w_down^T;  dpre = [dh * up * act'(gate) | dh * act(gate)]
// Both are the split-bf16 product of gemm.hip, its tiles and its choice of them
// (choose_gemm), with the gate in the epilogue: the sums are gated where they stand
// in registers, and neither dh nor, without pre, the sums go to memory.  In the
// forward a tile has half its columns from each projection and a wave both sums of
// its elements.  Where choose_gemm splits k, the parts are added by a kernel that
// gates them.  The gradients of x, of both weights and of the bias are products and
// sums with dpre, which gemm_ex and col_sum form.
#include <algorithm>

#include "gemm_split.h"

namespace ember {
namespace {

// h (and pre) from the parts of both sums, (splits, n, 2 hidden), added in order.
__global__ __launch_bounds__(256) void gate_fwd_reduce(GemmArgs g, int splits, int64_t total)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / g.hidden, col = i - row * g.hidden, at = row * 2 * g.hidden + col;
        float x = g.part[at], u = g.part[at + g.hidden];
        for (int z = 1; z < splits; ++z) x += g.part[z * 2 * total + at], u += g.part[z * 2 * total + at + g.hidden];
        if (g.bias) x += g.bias[col], u += g.bias[g.hidden + col];
        if (g.pre) g.pre[at] = x, g.pre[at + g.hidden] = u;
        g.c[i] = gated(g.steep, x, u);
    }
}

// dsums from the parts of dh, (splits, n, hidden).
__global__ __launch_bounds__(256) void gate_bwd_reduce(GemmArgs g, int splits, int64_t total)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / g.hidden, col = i - row * g.hidden, at = row * 2 * g.hidden + col;
        float dh = g.part[i];
        for (int z = 1; z < splits; ++z) dh += g.part[z * total + i];
        const GateGrad d = gate_grad(g.steep, g.sums[at], g.sums[at + g.hidden], dh);
        g.dsums[at] = d.gate, g.dsums[at + g.hidden] = d.up;
    }
}

// The tiles of gemm.hip; the smallest, in which a wave has one block of columns, is
// twice as wide where a wave needs a pair (300 x 1000 x 3001: 41 us; two waves that
// have a pair each in 64 x 64: 54).
template <bool TB, Gate GATE>
void launch_shape(GemmArgs &g, int ksplit, int shape)
{
    if (shape == 0)
        launch_tiles<256, 256, 4, 2, 16, 1, false, false, TB, GATE>(g, 1, ksplit);
    else if (shape == 1)
        launch_tiles<128, 128, 4, 2, 32, 1, true, false, TB, GATE>(g, 1, ksplit);
    else
        launch_tiles<64, GATE == kGateForward ? 128 : 64, 2, 2, 32, GATE == kGateForward ? 2 : 3, true, false, TB, GATE>(g, 1, ksplit);
}

// g's product as choose_gemm has it: gated by its own kernel, or in parts that
// `reduce` adds and gates.
template <bool TB, Gate GATE, class R>
int gated_launch(GemmArgs &g, R reduce, const char *who, const char *joined)
{
    const GemmChoice choice = choose_gemm(g.n, g.m, g.k, 1, num_cus());
    if (choice.ksplit > 1) {
        const int64_t total = (int64_t)g.n * g.m;
        g.part = (float *)scratch(kScratchGated, (size_t)choice.ksplit * total * sizeof(float), true);
        if (g.part) {  // else there is no memory for the parts: one sum per element
            g.kchunk = (int)choice.kchunk;
            launch_shape<TB, kNoGate>(g, choice.ksplit, choice.shape);
            if (!launch_ok(who)) return EMBER_ERR_DEVICE;
            const int64_t elements = (int64_t)g.n * g.hidden;
            hipLaunchKernelGGL(reduce, dim3((unsigned)std::min<int64_t>((elements + 255) / 256, 8 * num_cus())), dim3(256), 0, 0, g, choice.ksplit, elements);
            return launch_ok(joined) ? EMBER_OK : EMBER_ERR_DEVICE;
        }
    }
    launch_shape<TB, GATE>(g, 1, choice.shape);
    return launch_ok(who) ? EMBER_OK : EMBER_ERR_DEVICE;
}

constexpr int kMostHidden = (1 << 29) - 1;  // byte offsets of both halves of a row fit 32 bits

bool gated_args(const void *const *ptrs, int count, int n, int hidden, int d, int act)
{
    if (n < 0 || hidden < 1 || hidden > kMostHidden || d < 1 || act < kActGelu || act > kActSilu) return false;
    for (int i = 0; i < count; ++i)
        if (!ptrs[i] || ((uintptr_t)ptrs[i] & 3)) return false;
    return true;
}

GemmArgs gated_product(const float *a, const float *b, int n, int m, int k, int ldb, int hidden, int act)
{
    GemmArgs g = {};
    g.a = a, g.b = b;
    g.n = n, g.m = m, g.k = k;
    g.lda = k, g.ldb = ldb;
    g.sc = (int64_t)n * m;
    g.kchunk = k;
    g.hidden = hidden;
    g.steep = act == kActGelu ? kSteepGelu : kSteepSilu;
    return g;
}

}  // namespace
}  // namespace ember

extern "C" int gated_fwd(const float *x, const float *w, const float *bias, float *h, float *pre, int n, int hidden, int d, int act)
{
    using namespace ember;
    const void *ptrs[] = {x, w, h};
    if (!gated_args(ptrs, 3, n, hidden, d, act) || (((uintptr_t)bias | (uintptr_t)pre) & 3))
        return record_error(EMBER_ERR_INVALID_ARGUMENT, "gated_fwd");
    if (n == 0) return EMBER_OK;
    GemmArgs g = gated_product(x, w, n, 2 * hidden, d, 2 * hidden, hidden, act);
    g.c = h, g.pre = pre, g.bias = bias;
    return gated_launch<false, kGateForward>(g, gate_fwd_reduce, "gated_fwd", "gate_fwd_reduce");
}

extern "C" int gated_bwd(const float *dy, const float *w_down, const float *pre, float *dpre, int n, int hidden, int d, int act)
{
    using namespace ember;
    const void *ptrs[] = {dy, w_down, pre, dpre};
    if (!gated_args(ptrs, 4, n, hidden, d, act)) return record_error(EMBER_ERR_INVALID_ARGUMENT, "gated_bwd");
    if (n == 0) return EMBER_OK;
    GemmArgs g = gated_product(dy, w_down, n, hidden, d, d, hidden, act);
    g.sums = pre, g.dsums = dpre;
    return gated_launch<true, kGateBackward>(g, gate_bwd_reduce, "gated_bwd", "gate_bwd_reduce");
}
