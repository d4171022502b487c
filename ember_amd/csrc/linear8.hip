// linear8.hip -- products of two 8-bit matrices, out(n x m) = a(n x k) w(m x k)^T
// with the epilogue of linear_fwd, and gated layers of them, h = act(a wg^T + bg)
// * (a wu^T + bu).  No reference counterpart: pawel002/ember computes in fp32.
//
// The products run on the bf16 matrix instruction, codes turned into bf16 with
// their scales on the way (rows8.h; exact), so every product is exact and sums
// are fp32.  gfx950's 8-bit instruction would be twice as fast, but it loses what
// lies far below the largest product of a sum: measured against float64, relative
// 2-norm error at K = 4096 of N(0, 1) operands 1.5e-5, of all codes alike 5.2e-5,
// at one instruction (K = 64) the same; this one 0.9e-7 and 4.3e-7.
#include <algorithm>

#include "activation.h"
#include "linear8.h"

namespace ember {
namespace {

__device__ __forceinline__ f32x4 mfma_16x16x32(u32x4 a, u32x4 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Few rows: bound by w's bytes.  A workgroup has 16 columns of out (a gated layer:
// 16 of the gate and their 16 others) and 16*NT rows; its 8 waves take the groups
// of k in turn, each straight from memory into registers, and add their sums in
// wave order.  w's rows are the matrix instruction's rows, so that a lane ends up
// with 4 neighbouring columns of a row of out.  A lane holds 32 neighbours of a
// row's group, 8 to an instruction; which k those are only has to agree.
template <int NT, bool GATED>
__global__ __launch_bounds__(512) void linear8_few(Linear8Args g)
{
    constexpr int W = 8, NB = GATED ? 2 : 1;
    __shared__ f32x4 sums[W][NB][NT][64];
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col0 = 16 * blockIdx.x, row0 = 16 * NT * blockIdx.y;
    const int64_t pitch = g.w.pitch();
    const uint8_t *wc[NB], *ws[NB], *ac[NT], *as[NT];
#pragma unroll
    for (int b = 0; b < NB; ++b) {  // rows past the end re-read the last one; their results are not stored
        const int64_t row = min(col0 + r, g.m - 1) + (int64_t)b * g.m;
        wc[b] = g.w.codes + row * pitch + 32 * q;
        ws[b] = g.w.scales + row * g.w.scale_pitch;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t row = min(row0 + 16 * t + r, g.n - 1);
        ac[t] = g.a.codes + row * pitch + 32 * q;
        as[t] = g.a.scales + row * g.a.scale_pitch;
    }
    f32x4 acc[NB][NT];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[b][t] = f32x4{0, 0, 0, 0};
    for (int i = w; i < g.w.groups; i += W) {
        u32x4 x[NB][2], y[NT][2];
        float sx[NB], sy[NT];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            x[b][0] = *(const u32x4 *)(wc[b] + (int64_t)i * kGroup8);
            x[b][1] = *(const u32x4 *)(wc[b] + (int64_t)i * kGroup8 + 16);
            sx[b] = scale8(ws[b][i]);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            y[t][0] = *(const u32x4 *)(ac[t] + (int64_t)i * kGroup8);
            y[t][1] = *(const u32x4 *)(ac[t] + (int64_t)i * kGroup8 + 16);
            sy[t] = scale8(as[t][i]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const u32x4 v = bf16_of8(y[t][j / 2][j % 2 * 2], y[t][j / 2][j % 2 * 2 + 1], sy[t]);
#pragma unroll
                for (int b = 0; b < NB; ++b)
                    acc[b][t] = mfma_16x16x32(bf16_of8(x[b][j / 2][j % 2 * 2], x[b][j / 2][j % 2 * 2 + 1], sx[b]), v, acc[b][t]);
            }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < NT; ++t) sums[w][b][t][lane] = acc[b][t];
    __syncthreads();
    if (threadIdx.x >= 64 * NT) return;
    f32x4 v[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        v[b] = sums[0][b][w][lane];
#pragma unroll
        for (int i = 1; i < W; ++i) v[b] += sums[i][b][w][lane];
    }
    const int row = row0 + 16 * w + r;
    if (row >= g.n) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int col = col0 + 4 * q + i;
        if (col >= g.m) break;
        float o = v[0][i] + (g.bias ? g.bias[col] : 0.0f);
        if (GATED) {
            o = gated(g.act, o, v[1][i] + (g.bias ? g.bias[g.m + col] : 0.0f));
        } else {
            if (g.act == kActGelu) o = gelu08(o);
            if (g.residual) o += g.residual[(int64_t)row * g.m + col];
        }
        g.out[(int64_t)row * g.m + col] = o;
    }
}

template <bool GATED>
int linear8_launch(const Linear8Args &g, const char *who)
{
    const int nt = g.n <= 16 ? 1 : g.n <= 32 ? 2 : 4;
    // Rows beyond a grid's 65535 in y go in further launches.
    for (int64_t row = 0; row < g.n; row += int64_t(65535) * 64) {
        Linear8Args p = g;
        p.n = (int)std::min<int64_t>(g.n - row, int64_t(65535) * 64);
        p.a.codes += row * g.a.pitch();
        p.a.scales += row * g.a.scale_pitch;
        p.out += row * g.m;
        if (p.residual) p.residual += row * g.m;
        const dim3 grid((g.m + 15) / 16, (p.n + 16 * nt - 1) / (16 * nt));
        if (nt == 1)
            hipLaunchKernelGGL((linear8_few<1, GATED>), grid, dim3(512), 0, 0, p);
        else if (nt == 2)
            hipLaunchKernelGGL((linear8_few<2, GATED>), grid, dim3(512), 0, 0, p);
        else
            hipLaunchKernelGGL((linear8_few<4, GATED>), grid, dim3(512), 0, 0, p);
        if (!launch_ok(who)) return EMBER_ERR_DEVICE;
    }
    return EMBER_OK;
}

// Both operands, of as many columns.
int operands(const ember_rows8 *a, const ember_rows8 *w, Linear8Args *g, const char *who)
{
    int st = rows8_view(a, &g->a, who);
    if (!st) st = rows8_view(w, &g->w, who);
    if (st) return st;
    if (g->a.cols != g->w.cols) return record_error(EMBER_ERR_INVALID_ARGUMENT, who);
    return EMBER_OK;
}

}  // namespace
}  // namespace ember

extern "C" int linear8_fwd(const ember_rows8 *a, const ember_rows8 *w, const float *bias, const float *residual, float *out, int act)
{
    using namespace ember;
    Linear8Args g = {};
    const int st = operands(a, w, &g, "linear8_fwd");
    if (st) return st;
    if (!out || (((uintptr_t)out | (uintptr_t)bias | (uintptr_t)residual) & 3) || act < kActNone || act > kActGelu)
        return record_error(EMBER_ERR_INVALID_ARGUMENT, "linear8_fwd");
    g.bias = bias, g.residual = residual, g.out = out, g.n = g.a.rows, g.m = g.w.rows, g.act = act;
    return g.n && g.m ? linear8_launch<false>(g, "linear8_fwd") : EMBER_OK;
}

extern "C" int gated8_fwd(const ember_rows8 *a, const ember_rows8 *w, const float *bias, const ember_rows8 *h, int act)
{
    using namespace ember;
    Linear8Args g = {};
    Rows8 to;
    int st = operands(a, w, &g, "gated8_fwd");
    if (!st) st = rows8_view(h, &to, "gated8_fwd");
    if (st) return st;
    if (((uintptr_t)bias & 3) || act < kActGelu || act > kActSilu || g.w.rows != 2 * (int64_t)to.cols || g.a.rows != to.rows)
        return record_error(EMBER_ERR_INVALID_ARGUMENT, "gated8_fwd");
    if (to.rows == 0) return EMBER_OK;
    g.bias = bias, g.n = to.rows, g.m = to.cols, g.act = act;
    g.out = (float *)scratch(kScratchLinear8, (size_t)g.n * g.m * sizeof(float));
    if (!g.out) return EMBER_ERR_OUT_OF_MEMORY;
    st = linear8_launch<true>(g, "gated8_fwd");
    return st ? st : rows8_write_launch(to, g.out, g.m, 0, "gated8_fwd");
}
