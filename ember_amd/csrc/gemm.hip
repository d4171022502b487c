// gemm.hip -- fp32 GEMM on gfx950 matrix cores behind Ember's matmul ABI.
//
// Replaces the reference's cuBLAS calls (src/tensor/operators_gpu.cu:114-136):
//   matmul(a, b, out, n, m, k):          out(n x m) = a(n x k) @ b(k x m)
//   matmul_batched(..., batch, n, m, k): the same per batch with strides
//                                        n*k, k*m, n*m
// and adds gemm_ex, which also takes either operand transposed in place
// (a stored k x n, b stored m x k: the weight- and input-gradient products of
// a Linear layer, ember/nn/layers.py:50-56, without materialising T(x)) and
// the fused epilogue of linear_fwd, all row-major fp32.
//
// Products run on the bf16 matrix cores at fp32 precision: every operand is
// split exactly into three bf16 parts (split_bf16.h), and six of the nine
// part products are accumulated in fp32.  One kernel (gemm_split.h) covers every
// shape, orientation and alignment; choose_gemm (gemm_shape.h) picks its tile.
#include <algorithm>

#include "gemm_split.h"

namespace ember {
namespace {

__device__ __forceinline__ float epilogue(const GemmArgs &g, float v, int64_t off, int col)
{
    if (g.bias) v += g.bias[col];
    if (g.pre) g.pre[off] = v;
    if (g.act == 1) v = gelu08(v);
    if (g.residual) v += g.residual[off];
    return v;
}

// out = epilogue(sum over z of part[z]), z in order; VEC: m % 4 == 0 and
// 16-byte aligned operands.
template <int V>
__global__ __launch_bounds__(256) void gemm_splitk_reduce(GemmArgs g, int ksplit, int64_t total)
{
    typedef float vec __attribute__((ext_vector_type(V)));
    const int64_t nv = total / V;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < nv; q += (int64_t)gridDim.x * 256) {
        const int64_t off = V * q;
        vec s = *(const vec *)&g.part[off];
        for (int z = 1; z < ksplit; ++z) s += *(const vec *)&g.part[(int64_t)z * total + off];
        if (g.bias || g.pre || g.act || g.residual) {
            const int col = (int)(off % g.m);
#pragma unroll
            for (int c = 0; c < V; ++c) s[c] = epilogue(g, s[c], off + c, col + c);
        }
        *(vec *)&g.c[off] = s;
    }
}

template <bool TA, bool TB>
void launch_shape(GemmArgs &g, int batch, int ksplit, int shape)
{
    if (shape == 0)
        launch_tiles<256, 256, 4, 2, 16, 1, false, TA, TB>(g, batch, ksplit);
    else if (shape == 1)
        launch_tiles<128, 128, 4, 2, 32, 1, true, TA, TB>(g, batch, ksplit);
    else
        launch_tiles<64, 64, 2, 2, 32, 3, true, TA, TB>(g, batch, ksplit);
}

int gemm_launch(const float *a, const float *b, float *out, int batch, int n, int m, int k,
                const char *who, const float *bias = nullptr, const float *residual = nullptr,
                float *pre = nullptr, int act = 0, int ta = 0, int tb = 0)
{
    if (n < 0 || m < 0 || k < 0 || batch < 0) return record_error(EMBER_ERR_INVALID_ARGUMENT, who);
    if ((int64_t)n * m == 0 || batch == 0) return EMBER_OK;
    // k == 0: a and b are empty (null from alloc_memory(0)) and every output
    // is an empty sum, i.e. 0 before the epilogue, as in the reference's CPU
    // loop; the kernel never reads a or b then.
    if (!out || (k > 0 && (!a || !b))) return record_error(EMBER_ERR_INVALID_ARGUMENT, who);
    if (batch > 65535) return record_error(EMBER_ERR_UNSUPPORTED, who);
    GemmArgs g = {};
    g.a = a;
    g.b = b;
    g.c = out;
    g.n = n;
    g.m = m;
    g.k = k;
    g.lda = ta ? n : k;
    g.ldb = tb ? k : m;
    g.sa = (int64_t)n * k;
    g.sb = (int64_t)k * m;
    g.sc = (int64_t)n * m;
    g.kchunk = k;
    g.part = nullptr;
    g.bias = bias;
    g.residual = residual;
    g.pre = pre;
    g.act = act;

    const GemmChoice choice = choose_gemm(n, m, k, batch, num_cus());
    const int shape = choice.shape;
    int ksplit = choice.ksplit;
    const int64_t total = (int64_t)batch * n * m;
    if (ksplit > 1) {
        g.part = (float *)scratch(kScratchGemmSplit, (size_t)ksplit * total * sizeof(float), true);
        if (g.part)
            g.kchunk = (int)choice.kchunk;
        else
            ksplit = 1;  // no memory for the parts: one sum per element
    }
    if (ta)
        tb ? launch_shape<true, true>(g, batch, ksplit, shape) : launch_shape<true, false>(g, batch, ksplit, shape);
    else
        tb ? launch_shape<false, true>(g, batch, ksplit, shape) : launch_shape<false, false>(g, batch, ksplit, shape);
    if (!launch_ok(who)) return EMBER_ERR_DEVICE;
    if (ksplit > 1) {
        const bool vec = m % 4 == 0 && ((uintptr_t)out | (uintptr_t)pre | (uintptr_t)residual | (uintptr_t)bias) % 16 == 0;
        int64_t blocks = (total / (vec ? 4 : 1) + 255) / 256;
        if (blocks > 8 * num_cus()) blocks = 8 * num_cus();
        if (vec)
            hipLaunchKernelGGL(gemm_splitk_reduce<4>, dim3((unsigned)blocks), dim3(256), 0, 0, g, ksplit, total);
        else
            hipLaunchKernelGGL(gemm_splitk_reduce<1>, dim3((unsigned)blocks), dim3(256), 0, 0, g, ksplit, total);
        if (!launch_ok("gemm_splitk_reduce")) return EMBER_ERR_DEVICE;
    }
    return EMBER_OK;
}

}  // namespace
}  // namespace ember

extern "C" {

void matmul(const float *a, const float *b, float *out, int n, int m, int k)
{
    ember::gemm_launch(a, b, out, 1, n, m, k, "matmul");
}

void matmul_batched(const float *a, const float *b, float *out, int batch, int n, int m, int k)
{
    ember::gemm_launch(a, b, out, batch, n, m, k, "matmul_batched");
}

int linear_fwd(const float *a, const float *b, const float *bias, const float *residual,
               float *out, float *pre, int n, int m, int k, int act)
{
    if (act < 0 || act > 1) return ember::record_error(EMBER_ERR_INVALID_ARGUMENT, "linear_fwd");
    return ember::gemm_launch(a, b, out, 1, n, m, k, "linear_fwd", bias, residual, pre, act);
}

int gemm_ex(const float *a, const float *b, float *out, int batch, int n, int m, int k,
            int trans_a, int trans_b, const float *bias, const float *residual, float *pre, int act)
{
    if (act < 0 || act > 1 || (trans_a != 0 && trans_a != 1) || (trans_b != 0 && trans_b != 1))
        return ember::record_error(EMBER_ERR_INVALID_ARGUMENT, "gemm_ex");
    return ember::gemm_launch(a, b, out, batch, n, m, k, "gemm_ex", bias, residual, pre, act,
                              trans_a, trans_b);
}

}  // extern "C"
