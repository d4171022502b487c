// rows8.h -- a matrix in 8 bits as its kernels see it (not part of the public
// ABI; the format is described in include/ember_amd.h).
//
// gfx950 rounds floats to E4M3 in hardware, to nearest, ties to the even code
// (v_cvt_pk_fp8_f32), and gives codes back as bf16 times a scale of which only
// the exponent counts (v_cvt_scalef32_pk_bf16_fp8): 4 bits of significand, so
// every code times every scale that is written is a bf16 number.
#pragma once

#include "common.h"
#include "mfma.h"
#include "split_bf16.h"
#include "wave.h"

namespace ember {

constexpr int kGroup8 = 128;      // neighbours that share a scale
constexpr int kLeastScale8 = 8;   // the smallest scale byte that is written

struct Rows8 {
    uint8_t *codes, *scales;
    int rows, cols;
    int groups;       // of a row
    int scale_pitch;  // bytes from row to row of the scales: groups in whole fours
    __host__ __device__ int64_t pitch() const { return (int64_t)groups * kGroup8; }
};

// Checks `m` and fills `out`; records and returns a status.
int rows8_view(const ember_rows8 *m, Rows8 *out, const char *what);
// Rounds x into `to` on the null stream: element (r, c) is x[r*ld + c], or with
// trans x[c*ld + r].
int rows8_write_launch(const Rows8 &to, const float *x, int64_t ld, int trans, const char *what);

// (A bit cast of a vector's element in place gives element 0's bits; a float
// passed by value is safe.)
__device__ __forceinline__ unsigned size_bits8(float x)
{
    return __builtin_bit_cast(unsigned, x) & 0x7fffffffu;
}
// The largest of 32 neighbouring lanes, in each of them.
__device__ __forceinline__ unsigned max_of_32(unsigned v)
{
    const auto f = [](float a, float b) {
        return __builtin_bit_cast(float, max(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b)));
    };
    return __builtin_bit_cast(unsigned, across_16(row_all(__builtin_bit_cast(float, v), f), f));
}
// The scale byte of a group whose largest size has these bits (as integers the
// sizes of floats sort alike, infinities and NaNs above all).  With amax = f *
// 2^x, 1 <= f < 2: e = x - 8 if f <= 1.75, else x - 7; adding 0x1FFFFF to the bits
// carries into the exponent just when f > 1.75.
__device__ __forceinline__ unsigned scale_byte8(unsigned top)
{
    if (top >= 0x7f000000u) return 255;
    const int e = (int)((top + 0x1FFFFFu) >> 23) - 8;
    return top ? (unsigned)(e < kLeastScale8 ? kLeastScale8 : e) : 127u;
}
// 2^-e of a byte that is not 255.
__device__ __forceinline__ float inverse_scale8(unsigned byte)
{
    return __builtin_bit_cast(float, (254u - byte) << 23);
}
// Four elements as codes, the first in the low byte.
__device__ __forceinline__ unsigned codes8(float x0, float x1, float x2, float x3, float inverse)
{
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x0 * inverse, x1 * inverse, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(x2 * inverse, x3 * inverse, w, true);
    return (unsigned)w;
}
// The scale that a byte stands for; infinity (byte 255) makes every code a NaN.
__device__ __forceinline__ float scale8(unsigned byte)
{
    return __builtin_bit_cast(float, byte << 23);
}
// Two neighbouring codes, pair i of lo (0, 1) and hi (2, 3), as packed bf16.
__device__ __forceinline__ unsigned bf16_pair8(unsigned lo, unsigned hi, int i, float scale)
{
    const unsigned w = i < 2 ? lo : hi;
    return i & 1 ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))
                 : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
}
// Eight codes as one bf16 operand of a matrix instruction.
__device__ __forceinline__ u32x4 bf16_of8(unsigned lo, unsigned hi, float scale)
{
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = bf16_pair8(lo, hi, i, scale);
    return v;
}

}  // namespace ember
