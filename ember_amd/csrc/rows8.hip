// rows8.hip -- matrices rounded to 8 bits, row by row in groups of 128, and read
// back.  No reference counterpart: pawel002/ember computes in fp32 alone.
//
// HBM-bound: 4 bytes read and 129/128 written per element, and the other way
// round.  A half wave takes a group, 4 neighbours a lane, so that a wave reads 1
// KiB in a row; the largest size is found in register moves.  A matrix that is
// stored transposed (a Linear layer's weight, in x out) is read with the lanes
// along its rows: a lane holds a whole group and writes its 128 bytes, 16 at a time at
// a row's pitch, which holds it back.  21846 x 4096: written in 82 us, 5.4 TB/s (a copy
// of 4 GiB 4.75), transposed in 127, 3.5, read in 90, 5.0; 8 x 4096, a launch: 3.1, 5.6
// and 3.0.
#include <algorithm>

#include "rows8.h"
#include "wave.h"

namespace ember {

int rows8_view(const ember_rows8 *m, Rows8 *out, const char *what)
{
    if (!m || m->rows < 0 || m->rows > (1 << 26) || m->cols < 1 || m->cols > (1 << 23) || !m->codes || !m->scales ||
        (((uintptr_t)m->codes | (uintptr_t)m->scales) & 15))
        return record_error(EMBER_ERR_INVALID_ARGUMENT, what);
    const int groups = (int)((m->cols + kGroup8 - 1) / kGroup8);
    *out = {(uint8_t *)m->codes, (uint8_t *)m->scales, (int)m->rows, (int)m->cols, groups, (groups + 3) / 4 * 4};
    return EMBER_OK;
}

namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

__global__ __launch_bounds__(256) void rows8_write_kernel(Rows8 to, const float *__restrict__ x, int64_t ld, int64_t tasks)
{
    const int l32 = threadIdx.x & 31;
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < tasks; i += (int64_t)gridDim.x * 8) {
        const int64_t row = i / to.scale_pitch;
        const int g = (int)(i - row * to.scale_pitch), col = g * kGroup8 + 4 * l32;
        float v[4] = {0, 0, 0, 0};
        const float *const at = x + row * ld + col;
        if (col + 4 <= to.cols) {
            const f32x4u u = *(const f32x4u *)at;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = u[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < to.cols) v[j] = at[j];
        }
        const unsigned byte = scale_byte8(max_of_32(max(max(size_bits8(v[0]), size_bits8(v[1])), max(size_bits8(v[2]), size_bits8(v[3])))));
        const unsigned w = byte == 255 ? 0 : codes8(v[0], v[1], v[2], v[3], inverse_scale8(byte));
        if (g < to.groups) *(unsigned *)(to.codes + row * to.pitch() + col) = w;
        if (l32 == 0) to.scales[i] = (uint8_t)byte;
    }
}

// x is (cols, rows).  A lane per row and group.
__global__ __launch_bounds__(64) void rows8_write_transposed(Rows8 to, const float *__restrict__ x, int64_t ld)
{
    const int64_t row = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (row >= to.rows) return;
    for (int g = blockIdx.y; g < to.scale_pitch; g += gridDim.y) {
        float v[kGroup8];
        const int col = g * kGroup8, n = min(kGroup8, to.cols - col);
        const float *const at = x + col * ld + row;
        unsigned top = 0;
        if (n == kGroup8) {
#pragma unroll
            for (int j = 0; j < kGroup8; ++j) v[j] = at[j * ld];
        } else {
#pragma unroll
            for (int j = 0; j < kGroup8; ++j) v[j] = j < n ? at[j * ld] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < kGroup8; ++j) top = max(top, size_bits8(v[j]));
        const unsigned byte = scale_byte8(top);
        to.scales[row * to.scale_pitch + g] = (uint8_t)byte;
        if (g >= to.groups) continue;
        const float inverse = byte == 255 ? 0.0f : inverse_scale8(byte);
        u32x4 *const out = (u32x4 *)(to.codes + row * to.pitch() + col);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            u32x4 w;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float *const p = v + 16 * j + 4 * k;
                w[k] = byte == 255 ? 0 : codes8(p[0], p[1], p[2], p[3], inverse);
            }
            out[j] = w;
        }
    }
}

__global__ __launch_bounds__(256) void rows8_read_kernel(Rows8 from, float *__restrict__ out, int64_t ld, int64_t tasks)
{
    const int l32 = threadIdx.x & 31;
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < tasks; i += (int64_t)gridDim.x * 8) {
        const int64_t row = i / from.groups;
        const int g = (int)(i - row * from.groups), col = g * kGroup8 + 4 * l32;
        const unsigned w = *(const unsigned *)(from.codes + row * from.pitch() + col);
        const float scale = scale8(from.scales[row * from.scale_pitch + g]);
        const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true);
        const float v[4] = {(float)a[0], (float)a[1], (float)b[0], (float)b[1]};
        float *const at = out + row * ld + col;
        if (col + 4 <= from.cols) {
            *(f32x4u *)at = f32x4u{v[0], v[1], v[2], v[3]};
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < from.cols) at[j] = v[j];
        }
    }
}

}  // namespace

int rows8_write_launch(const Rows8 &to, const float *x, int64_t ld, int trans, const char *what)
{
    if (to.rows == 0) return EMBER_OK;
    if (trans) {
        hipLaunchKernelGGL(rows8_write_transposed, dim3((to.rows + 63u) / 64, std::min(to.scale_pitch, 65535)), dim3(64), 0, 0, to, x, ld);
    } else {
        const int64_t tasks = (int64_t)to.rows * to.scale_pitch;
        hipLaunchKernelGGL(rows8_write_kernel, dim3((unsigned)std::min<int64_t>((tasks + 7) / 8, 1 << 20)), dim3(256), 0, 0, to, x, ld, tasks);
    }
    return launch_ok(what) ? EMBER_OK : EMBER_ERR_DEVICE;
}

}  // namespace ember

extern "C" int rows8_write(const ember_rows8 *to, const float *x, int64_t ld, int trans)
{
    using namespace ember;
    Rows8 m;
    const int st = rows8_view(to, &m, "rows8_write");
    if (st) return st;
    if (!x || ((uintptr_t)x & 3) || (trans != 0 && trans != 1) || ld < (trans ? m.rows : m.cols) || ld > (int64_t(1) << 40))
        return record_error(EMBER_ERR_INVALID_ARGUMENT, "rows8_write");
    return rows8_write_launch(m, x, ld, trans, "rows8_write");
}

extern "C" int rows8_read(const ember_rows8 *from, float *out, int64_t ld)
{
    using namespace ember;
    Rows8 m;
    const int st = rows8_view(from, &m, "rows8_read");
    if (st) return st;
    if (!out || ((uintptr_t)out & 3) || ld < m.cols || ld > (int64_t(1) << 40)) return record_error(EMBER_ERR_INVALID_ARGUMENT, "rows8_read");
    if (m.rows == 0) return EMBER_OK;
    const int64_t tasks = (int64_t)m.rows * m.groups;
    hipLaunchKernelGGL(rows8_read_kernel, dim3((unsigned)std::min<int64_t>((tasks + 7) / 8, 1 << 20)), dim3(256), 0, 0, m, out, ld, tasks);
    return launch_ok("rows8_read") ? EMBER_OK : EMBER_ERR_DEVICE;
}
