// gated.hip -- gated feed-forward layers in fp32: h = act(x wg + bg) * (x wu + bu)
// and the gradient with respect to both sums.  No reference counterpart:
// pawel002/ember composes feed-forward layers from Linear and an activation.
//   forward:  pre = x [wg | wu] + bias;  h = act(gate) * up  (gate, up: pre's halves)
//   backward: dh = dy w_down^T;  dpre = [dh * up * act'(gate) | dh * act(gate)]
// The gradients of x, of both weights and of the bias are products and sums with
// dpre, which gemm_ex and col_sum form.
#include <algorithm>

#include "activation.h"
#include "common.h"

namespace ember {
namespace {

__global__ __launch_bounds__(256) void gate_fwd_kernel(const float *__restrict__ pre, float *__restrict__ h, int64_t total, int hidden, int act)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t at = i + i / hidden * hidden;
        h[i] = gated(steepness(act), pre[at], pre[at + hidden]);
    }
}

__global__ __launch_bounds__(256) void gate_bwd_kernel(const float *__restrict__ dh, const float *__restrict__ pre, float *__restrict__ dpre,
                                                       int64_t total, int hidden, int act)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t at = i + i / hidden * hidden;
        const Activated a = activate(steepness(act), pre[at]);
        const float up = pre[at + hidden], g = dh[i];
        dpre[at] = g * up * a.slope;
        dpre[at + hidden] = g * a.value;
    }
}

unsigned gate_grid(int64_t total)
{
    return (unsigned)std::min<int64_t>((total + 255) / 256, 1 << 16);
}

bool gated_args(const void *const *ptrs, int count, int n, int hidden, int d, int act)
{
    if (n < 0 || hidden < 1 || hidden > (1 << 30) - 1 || d < 1 || act < kActGelu || act > kActSilu) return false;
    for (int i = 0; i < count; ++i)
        if (!ptrs[i] || ((uintptr_t)ptrs[i] & 3)) return false;
    return true;
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
    const int64_t total = (int64_t)n * hidden;
    if (!pre) pre = (float *)scratch(kScratchGated, 2 * (size_t)total * sizeof(float));
    if (!pre) return EMBER_ERR_OUT_OF_MEMORY;
    const int st = linear_fwd(x, w, bias, nullptr, pre, nullptr, n, 2 * hidden, d, 0);
    if (st) return st;
    hipLaunchKernelGGL(gate_fwd_kernel, dim3(gate_grid(total)), dim3(256), 0, 0, pre, h, total, hidden, act);
    return launch_ok("gated_fwd") ? EMBER_OK : EMBER_ERR_DEVICE;
}

extern "C" int gated_bwd(const float *dy, const float *w_down, const float *pre, float *dpre, int n, int hidden, int d, int act)
{
    using namespace ember;
    const void *ptrs[] = {dy, w_down, pre, dpre};
    if (!gated_args(ptrs, 4, n, hidden, d, act)) return record_error(EMBER_ERR_INVALID_ARGUMENT, "gated_bwd");
    if (n == 0) return EMBER_OK;
    const int64_t total = (int64_t)n * hidden;
    float *dh = (float *)scratch(kScratchGated, (size_t)total * sizeof(float));
    if (!dh) return EMBER_ERR_OUT_OF_MEMORY;
    const int st = gemm_ex(dy, w_down, dh, 1, n, hidden, d, 0, 1, nullptr, nullptr, nullptr, 0);
    if (st) return st;
    hipLaunchKernelGGL(gate_bwd_kernel, dim3(gate_grid(total)), dim3(256), 0, 0, dh, pre, dpre, total, hidden, act);
    return launch_ok("gated_bwd") ? EMBER_OK : EMBER_ERR_DEVICE;
}
