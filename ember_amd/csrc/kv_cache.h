// kv_cache.h -- the 4-bit key/value cache as its kernels see it (not part of
// the public ABI; the format is described in include/ember_amd.h).
//
// gfx950 converts E2M1 codes in hardware, two to an instruction, with a scale
// of which only the exponent counts: v_cvt_scalef32_pk_f32_fp4 and
// v_cvt_scalef32_pk_bf16_fp4 (every code times every scale that is written is
// a bf16 number: 2 bits of significand, sizes from 2^-120 to 1.5 * 2^127), and
// v_cvt_scalef32_pk_fp4_f32 the other way, to nearest, ties to the even code.
// A scale whose bits are those of infinity (byte 255) makes every code a NaN.
// All 256 bytes and all multiples of 1/64 up to 6 were compared with the
// format's definition on the device.
#pragma once

#include "common.h"
#include "mfma.h"

namespace ember {

// The scale bytes that are written for numbers; 255 says that the group holds
// something else.
constexpr int kLeastScale = 8, kMostScale = 252;

struct KvCache {
    uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
    const int32_t *table;
    int pages, heads, page_shift, D;
    int sequences, max_pages;
};

// Checks `cache` and fills `out`; records and returns a status.
int kv_cache_view(const ember_kv_cache *cache, KvCache *out, const char *what);

// The strides of a (sequences, T, heads, D) operand.
struct RowStrides {
    int64_t sb, sh, ss;
};

// Whether rows of D floats with these strides can be read and written 16 bytes
// at a time.
inline bool row_strides_ok(const void *p, int64_t sb, int64_t sh, int64_t ss)
{
    return ((uintptr_t)p & 15) == 0 && sb % 4 == 0 && sh % 4 == 0 && ss % 4 == 0 && sb >= 0 && sh >= 0 && ss >= 0 &&
           ss < (int64_t(1) << 24);
}

// Where a sequence's rows of this call stand.
struct Span {
    int start, count;
};

__device__ __forceinline__ Span span_of(const int32_t *start, const int32_t *count, int b, int T)
{
    const int n = count ? count[b] : T;
    return {start ? start[b] : 0, min(max(n, 0), T)};
}

// The page that the table names for 16 tokens of a sequence (pos a multiple of 16:
// pages hold them whole; the table has a page at least, and the last one stands
// for those past it).  b and pos are the same in all lanes, so the table is read
// through the scalar cache.
__device__ __forceinline__ int page_of(const KvCache &c, int b, int pos)
{
    typedef const __attribute__((address_space(4))) int32_t *scalar;
    return ((scalar)(uintptr_t)c.table)[(int64_t)b * c.max_pages + min(pos >> c.page_shift, c.max_pages - 1)];
}
// Their first row of head h, or -1 where there is no such page.
__device__ __forceinline__ int64_t row_on(const KvCache &c, int page, int h, int pos)
{
    const int64_t row = (((int64_t)page * c.heads + h) << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
    return (unsigned)page < (unsigned)c.pages ? row : -1;
}
__device__ __forceinline__ int64_t row_of(const KvCache &c, int b, int h, int pos)
{
    return row_on(c, page_of(c, b, pos), h, pos);
}

// The scale that a byte stands for.
__device__ __forceinline__ float scale_of(unsigned byte)
{
    return __builtin_bit_cast(float, byte << 23);
}

// Two neighbouring codes, byte `s` of `w`, as floats.
template <int S>
__device__ __forceinline__ f32x2 fp4_pair(unsigned w, float scale)
{
    return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, S);
}

}  // namespace ember
