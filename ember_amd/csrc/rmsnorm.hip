// rmsnorm.hip -- RMS norm over the last dimension, the residual's addition
// before it, an output in fp32 or in 8 bits, and the gradient.  No reference
// counterpart: pawel002/ember has no norms.
//   s = x + residual;  rstd = 1/sqrt(sum(s^2)/d + eps);  y = s*rstd*gamma
//   backward (xhat = s*rstd, g = dy*gamma):
//   dx = rstd*(g - xhat*sum(g*xhat)/d)  (+ dres, the gradient that reaches s past
//        the norm, when given);  dgamma = sum_rows(dy*xhat)
//
// HBM-bound.  A row is held in registers, 16 bytes a lane and chunk in up to four
// chunks, by as few waves as that takes (1 to d = 1024, 4 to 4096, 16 to 16384),
// so x is read once and rows of any length have as much in flight.
//
// The forward's sum and its products with rstd and gamma are formed in 64 bits
// and y rounded once (the double rate is far above what the bytes need): the
// rounding of y to 8 bits must not turn on the order of a sum.  The gradient is
// formed in 32 bits, and dgamma's sum of many rows in 64.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "rows8.h"
#include "wave.h"

namespace ember {
namespace {

constexpr int kChunks = 4;  // of 16 bytes to a lane

// The sum over the W waves of a row, in each of their lanes; `red` has a place
// for each wave of the workgroup.
template <int W, class T>
__device__ __forceinline__ T row_sum(T v, T *red)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    if (W == 1) return v;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    T s = red[0];
#pragma unroll
    for (int w = 1; w < W; ++w) s += red[w];
    return s;
}

struct NormArgs {
    const float *x, *residual, *gamma;
    float *sum, *y, *rstd;  // each may be null
    Rows8 y8;
    int64_t rows;
    int d;
    float eps;
};

// W waves to a row, max(1, 4 / W) rows to a workgroup.  x and the residual may be
// sum or y: an element is read and written by the same lane.
template <int W, bool TO8>
__global__ __launch_bounds__(W < 4 ? 256 : 64 * W) void rms_fwd_kernel(NormArgs a)
{
    __shared__ double red[W];
    const int t = threadIdx.x % (64 * W);
    const int64_t row = (int64_t)blockIdx.x * (W < 4 ? 4 / W : 1) + threadIdx.x / (64 * W);
    if (row >= a.rows) return;  // whole waves; with W > 1 the grid is the rows
    const int64_t base = row * a.d;
    f32x4 s[kChunks], r[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int col = 4 * (64 * W * c + t);
        s[c] = col < a.d ? *(const f32x4 *)(a.x + base + col) : f32x4{0, 0, 0, 0};
        r[c] = a.residual && col < a.d ? *(const f32x4 *)(a.residual + base + col) : f32x4{0, 0, 0, 0};
    }
    double q = 0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        if (a.residual) s[c] += r[c];
#pragma unroll
        for (int j = 0; j < 4; ++j) q = fma((double)s[c][j], (double)s[c][j], q);
    }
    const double rstd = 1.0 / sqrt(row_sum<W>(q, red) / a.d + (double)a.eps);
    if (a.rstd && t == 0) a.rstd[row] = (float)rstd;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int col = 4 * (64 * W * c + t);
        if (a.sum && col < a.d) *(f32x4 *)(a.sum + base + col) = s[c];
        const f32x4 g = col < a.d ? *(const f32x4 *)(a.gamma + col) : f32x4{0, 0, 0, 0};
        f32x4 y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = col < a.d ? (float)((double)s[c][j] * rstd * (double)g[j]) : 0.0f;
        if (!TO8) {
            if (col < a.d) *(f32x4 *)(a.y + base + col) = y;
        } else if (col / kGroup8 < a.y8.scale_pitch) {  // a half wave has a group
            const unsigned mine = max(max(size_bits8(y[0]), size_bits8(y[1])), max(size_bits8(y[2]), size_bits8(y[3])));
            const unsigned byte = scale_byte8(max_of_32(mine));
            if (col / kGroup8 < a.y8.groups)
                *(unsigned *)(a.y8.codes + row * a.y8.pitch() + col) = byte == 255 ? 0 : codes8(y[0], y[1], y[2], y[3], inverse_scale8(byte));
            if (t % 32 == 0) a.y8.scales[row * a.y8.scale_pitch + col / kGroup8] = (uint8_t)byte;
        }
    }
}

// dx of a run of rows, and their sum of dy*xhat, which goes to part[blockIdx.x].  Runs
// grow with the rows: the sum is formed over kShort rows at a time in 32 bits, and over
// those in 64, in LDS (in registers fewer workgroups would share a CU), so that its
// error does not.
constexpr int kShort = 32;
template <int W>
__global__ __launch_bounds__(W < 4 ? 256 : 64 * W) void rms_bwd_kernel(const float *__restrict__ s, const float *__restrict__ gamma,
                                                                       const float *__restrict__ rstd_in, const float *__restrict__ dy,
                                                                       const float *dres, float *dx, float *__restrict__ part,
                                                                       int64_t rows, int d, int rows_per_block)
{
    constexpr int R = W < 4 ? 4 / W : 1;  // rows at a time
    __shared__ float red[2][W];
    const int t = threadIdx.x % (64 * W), which = threadIdx.x / (64 * W);
    __shared__ double all[4 * kChunks][64 * W * R];
    f32x4 pg[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) pg[c] = f32x4{0, 0, 0, 0};
    bool some = false;  // of this lane's sums are in `all`
    const auto put_by = [&] {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                double &to = all[4 * c + j][threadIdx.x];
                to = (some ? to : 0.0) + (double)pg[c][j];
                pg[c][j] = 0;
            }
        some = true;
    };
    const int64_t first = (int64_t)blockIdx.x * rows_per_block, end = min(first + rows_per_block, rows);
    int turn = 0, summed = 0;
    for (int64_t row = first + which; row < end; row += R, turn ^= 1) {
        if (summed++ == kShort) put_by(), summed = 1;
        const float rstd = rstd_in[row];
        f32x4 xh[kChunks], g[kChunks], more[kChunks];
        float m = 0;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int col = 4 * (64 * W * c + t);
            const bool in = col < d;
            xh[c] = in ? *(const f32x4 *)(s + row * d + col) : f32x4{0, 0, 0, 0};
            g[c] = in ? *(const f32x4 *)(dy + row * d + col) : f32x4{0, 0, 0, 0};
            more[c] = in && dres ? *(const f32x4 *)(dres + row * d + col) : f32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int col = 4 * (64 * W * c + t);
            if (col >= d) continue;
            xh[c] *= rstd;
            pg[c] += g[c] * xh[c];
            g[c] *= *(const f32x4 *)(gamma + col);
            m += (g[c][0] * xh[c][0] + g[c][1] * xh[c][1]) + (g[c][2] * xh[c][2] + g[c][3] * xh[c][3]);
        }
        m = row_sum<W>(m, red[turn]) / (float)d;  // two places: a wave may be a row ahead
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int col = 4 * (64 * W * c + t);
            if (col < d) *(f32x4 *)(dx + row * d + col) = rstd * (g[c] - xh[c] * m) + more[c];
        }
    }
    if (some) {
        put_by();
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) pg[c][j] = (float)all[4 * c + j][threadIdx.x];
    }
    if (R > 1) {  // the waves' sums in their order
        __shared__ f32x4 sums[R][64];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            __syncthreads();
            sums[which][t] = pg[c];
            __syncthreads();
            if (which == 0)
#pragma unroll
                for (int w = 1; w < R; ++w) pg[c] += sums[w][t];
        }
    }
    if (which == 0)
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int col = 4 * (64 * W * c + t);
            if (col < d) *(f32x4 *)(part + (int64_t)blockIdx.x * d + col) = pg[c];
        }
}

// dgamma = the sum of n rows of `part`: a workgroup owns 8 quads of columns, a line of
// memory of each row, and its 128 groups of threads every 128th row each; the groups'
// sums are added in order.  (The gradient of 8192 x 1024 31.1 us, with 16 quads and
// 64 groups 32.1; of 256 x 256 5.6 and 5.2.)
constexpr int kQuads = 8, kGroups = 128;
__global__ __launch_bounds__(kQuads *kGroups) void rms_param_grad_kernel(const float *__restrict__ part, float *__restrict__ dgamma, int n, int d)
{
    __shared__ f32x4 red[kGroups][kQuads];
    const int q = threadIdx.x % kQuads, g = threadIdx.x / kQuads, col = 4 * (blockIdx.x * kQuads + q);
    f32x4 s = {0, 0, 0, 0};
    if (col < d) {
        int b = g;
        for (; b + 7 * kGroups < n; b += 8 * kGroups) {  // eight loads in flight
            f32x4 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = *(const f32x4 *)(part + (int64_t)(b + kGroups * u) * d + col);
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
        for (; b < n; b += kGroups) s += *(const f32x4 *)(part + (int64_t)b * d + col);
    }
    red[g][q] = s;
    __syncthreads();
    // Sixteen groups' sums by eight groups of threads, then those by the first.
    if (g < 8) {
#pragma unroll
        for (int i = 1; i < kGroups / 8; ++i) s += red[g + 8 * i][q];
        red[g][q] = s;
    }
    __syncthreads();
    if (g == 0 && col < d) {
#pragma unroll
        for (int i = 1; i < 8; ++i) s += red[i][q];
        *(f32x4 *)(dgamma + col) = s;
    }
}

// Sizes and pointers (n of them, none null).
int norm_args(const void *const *ptrs, int n, const void *const *optional, int m, int64_t rows, int64_t d, const char *who)
{
    if (rows < 0 || rows > 0x7fffffff || d <= 0 || d % 4) return record_error(EMBER_ERR_INVALID_ARGUMENT, who);
    if (d > 64 * 4 * kChunks * 16) return record_error(EMBER_ERR_UNSUPPORTED, who);
    for (int i = 0; i < n; ++i)
        if (!ptrs[i] || ((uintptr_t)ptrs[i] & 15)) return record_error(EMBER_ERR_INVALID_ARGUMENT, who);
    for (int i = 0; i < m; ++i)
        if ((uintptr_t)optional[i] & 15) return record_error(EMBER_ERR_INVALID_ARGUMENT, who);
    return EMBER_OK;
}

template <bool TO8>
int norm_launch(const NormArgs &all, const char *who)
{
    if (!(all.eps >= 0.0f) || isinf(all.eps)) return record_error(EMBER_ERR_INVALID_ARGUMENT, who);
    // A grid holds fewer than 2^32 threads.
    constexpr int64_t kRowsPerLaunch = 1 << 21;
    for (int64_t row = 0; row < all.rows; row += kRowsPerLaunch) {
        NormArgs a = all;
        a.rows = std::min(all.rows - row, kRowsPerLaunch);
        a.x += row * a.d;
        if (a.residual) a.residual += row * a.d;
        if (a.sum) a.sum += row * a.d;
        if (a.y) a.y += row * a.d;
        if (a.rstd) a.rstd += row;
        if (TO8) a.y8.codes += row * a.y8.pitch(), a.y8.scales += row * a.y8.scale_pitch;
        const unsigned rows = (unsigned)a.rows;
        if (a.d <= 1024)
            hipLaunchKernelGGL((rms_fwd_kernel<1, TO8>), dim3((rows + 3) / 4), dim3(256), 0, 0, a);
        else if (a.d <= 4096)
            hipLaunchKernelGGL((rms_fwd_kernel<4, TO8>), dim3(rows), dim3(256), 0, 0, a);
        else
            hipLaunchKernelGGL((rms_fwd_kernel<16, TO8>), dim3(rows), dim3(1024), 0, 0, a);
    }
    return launch_ok(who) ? EMBER_OK : EMBER_ERR_DEVICE;
}

}  // namespace
}  // namespace ember

extern "C" int rmsnorm_fwd(const float *x, const float *residual, const float *gamma, float *sum, float *y, float *rstd, int64_t rows,
                           int64_t d, float eps)
{
    using namespace ember;
    const void *ptrs[] = {x, gamma, y}, *optional[] = {residual, sum};
    const int st = norm_args(ptrs, 3, optional, 2, rows, d, "rmsnorm_fwd");
    if (st) return st;
    if (((uintptr_t)rstd & 3) || sum == y) return record_error(EMBER_ERR_INVALID_ARGUMENT, "rmsnorm_fwd");
    return norm_launch<false>({x, residual, gamma, sum, y, rstd, {}, rows, (int)d, eps}, "rmsnorm_fwd");
}

extern "C" int rmsnorm_fwd8(const float *x, const float *residual, const float *gamma, float *sum, const ember_rows8 *y, float eps)
{
    using namespace ember;
    Rows8 y8;
    int st = rows8_view(y, &y8, "rmsnorm_fwd8");
    if (st) return st;
    const void *ptrs[] = {x, gamma}, *optional[] = {residual, sum};
    st = norm_args(ptrs, 2, optional, 2, y8.rows, y8.cols, "rmsnorm_fwd8");
    if (st) return st;
    return norm_launch<true>({x, residual, gamma, sum, nullptr, nullptr, y8, y8.rows, y8.cols, eps}, "rmsnorm_fwd8");
}

extern "C" int rmsnorm_bwd(const float *s, const float *gamma, const float *rstd, const float *dy, const float *dres, float *dx,
                           float *dgamma, int64_t rows, int64_t d)
{
    using namespace ember;
    const void *ptrs[] = {s, gamma, dy, dx, dgamma}, *optional[] = {dres};
    const int st = norm_args(ptrs, 5, optional, 1, rows, d, "rmsnorm_bwd");
    if (st) return st;
    if (!rstd || ((uintptr_t)rstd & 3)) return record_error(EMBER_ERR_INVALID_ARGUMENT, "rmsnorm_bwd");
    const dim3 quads((unsigned)((d / 4 + kQuads - 1) / kQuads));
    if (rows == 0) {  // a sum over no rows
        hipLaunchKernelGGL(rms_param_grad_kernel, quads, dim3(kQuads * kGroups), 0, 0, (const float *)nullptr, dgamma, 0, (int)d);
        return launch_ok("rmsnorm_bwd") ? EMBER_OK : EMBER_ERR_DEVICE;
    }
    // A run of rows to a workgroup: as many workgroups as fill the chip (four to a CU;
    // of sixteen waves one), and no more, for each writes a row of partial sums.
    // (8192 x 1024 in runs of 8: 31 us, of 32: 34; 64 x 4096 in runs of 1: 6.6, of 8: 19;
    // 1000 x 16384 in runs of 4: 64, of 1: 76.)
    const int64_t most = d <= 4096 ? 1024 : 256, at_once = d <= 1024 ? 4 : 1;
    const int64_t run = std::max<int64_t>(at_once, (rows + most - 1) / most + at_once - 1) / at_once * at_once;
    const int blocks = (int)((rows + run - 1) / run);
    float *part = (float *)scratch(kScratchRmsNorm, (size_t)blocks * d * sizeof(float));
    if (!part) return EMBER_ERR_OUT_OF_MEMORY;
    if (d <= 1024)
        hipLaunchKernelGGL(rms_bwd_kernel<1>, dim3(blocks), dim3(256), 0, 0, s, gamma, rstd, dy, dres, dx, part, rows, (int)d, (int)run);
    else if (d <= 4096)
        hipLaunchKernelGGL(rms_bwd_kernel<4>, dim3(blocks), dim3(256), 0, 0, s, gamma, rstd, dy, dres, dx, part, rows, (int)d, (int)run);
    else
        hipLaunchKernelGGL(rms_bwd_kernel<16>, dim3(blocks), dim3(1024), 0, 0, s, gamma, rstd, dy, dres, dx, part, rows, (int)d, (int)run);
    if (!launch_ok("rmsnorm_bwd")) return EMBER_ERR_DEVICE;
    hipLaunchKernelGGL(rms_param_grad_kernel, quads, dim3(kQuads * kGroups), 0, 0, part, dgamma, blocks, (int)d);
    return launch_ok("rms_param_grad_kernel") ? EMBER_OK : EMBER_ERR_DEVICE;
}
