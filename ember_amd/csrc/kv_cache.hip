// kv_cache.hip -- keys and values rounded to 4 bits as they enter the cache,
// and read back.  No reference counterpart: pawel002/ember has no cache.
//
// Per group of 32 neighbours of a head row, with amax their largest size:
//   amax = f * 2^x, 1 <= f < 2:  e = x - 2 if f <= 1.5, else x - 1
//   code = nearest of {0, .5, 1, 1.5, 2, 3, 4, 6} to |v| * 2^-e (ties: even)
// e is found on the bits of amax: adding 0x3FFFFF to them carries into the
// exponent just when f > 1.5.  The largest size is taken on the bits too (as
// integers the sizes of floats sort alike, infinities and NaNs above all), so
// no NaN is lost in it.
//
// A lane holds 8 neighbours (two 16-byte loads, one 4-byte store of codes), so
// a group is 4 lanes and a row of D = 128 is 16.  HBM-bound: 4 bytes read and
// 17/32 written per element, and the other way round.
#include "kv_cache.h"

namespace ember {

int kv_cache_view(const ember_kv_cache *c, KvCache *out, const char *what)
{
    constexpr int64_t kMost = 0x7fffffff;
    if (!c || c->pages < 0 || c->pages > kMost || c->heads < 1 || c->heads > 65535 || c->sequences < 0 ||
        c->sequences > 65535 || c->max_pages < 0 || c->max_pages > kMost || c->page_size < 16 || c->page_size > 65536 ||
        (c->page_size & (c->page_size - 1)) || c->max_pages * c->page_size > kMost - 65535)
        return record_error(EMBER_ERR_INVALID_ARGUMENT, what);
    if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128) return record_error(EMBER_ERR_UNSUPPORTED, what);
    const uintptr_t all = (uintptr_t)c->k_codes | (uintptr_t)c->k_scales | (uintptr_t)c->v_codes | (uintptr_t)c->v_scales;
    if (c->pages && (!c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales || (all & 15)))
        return record_error(EMBER_ERR_INVALID_ARGUMENT, what);
    if (c->sequences && c->max_pages && (!c->page_table || ((uintptr_t)c->page_table & 3)))
        return record_error(EMBER_ERR_INVALID_ARGUMENT, what);
    *out = {(uint8_t *)c->k_codes, (uint8_t *)c->k_scales, (uint8_t *)c->v_codes, (uint8_t *)c->v_scales, c->page_table,
            (int)c->pages, (int)c->heads, __builtin_ctzll((unsigned long long)c->page_size), (int)c->head_dim,
            (int)c->sequences, (int)c->max_pages};
    return EMBER_OK;
}

namespace {

struct CopyArgs {
    KvCache c;
    const float *in[2];
    float *out[2];
    RowStrides st;
    const int32_t *start, *count;
    int32_t *next;
    int T;
};

// (A bit cast of a vector's element in place gives element 0's bits; a float
// passed by value is safe.)
__device__ __forceinline__ unsigned size_bits(float x)
{
    return __builtin_bit_cast(unsigned, x) & 0x7fffffffu;
}

// A lane's place in the call's rows: grid (blocks of rows, sequences, k or v).
template <int D>
struct Place {
    static constexpr int LPR = D / 8;        // lanes per row
    static constexpr int RPB = 256 / LPR;    // rows per workgroup
    unsigned rows;
    int lane;
    __device__ __forceinline__ Place(const CopyArgs &a) : rows((unsigned)a.T * a.c.heads), lane(threadIdx.x % LPR) {}
};

template <int D>
__global__ __launch_bounds__(256) void kv_write_kernel(CopyArgs a)
{
    const Place<D> pl(a);
    const int b = blockIdx.y;
    const Span sp = span_of(a.start, a.count, b, a.T);
    if (a.next && blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) a.next[b] = sp.start + sp.count;
    const float *in = a.in[blockIdx.z];
    uint8_t *codes = blockIdx.z ? a.c.v_codes : a.c.k_codes, *scales = blockIdx.z ? a.c.v_scales : a.c.k_scales;
    for (unsigned row = blockIdx.x * pl.RPB + threadIdx.x / pl.LPR; row < pl.rows; row += gridDim.x * pl.RPB) {
        const int t = (int)(row / (unsigned)a.c.heads), h = (int)(row - (unsigned)t * a.c.heads);
        const int64_t pos = (int64_t)sp.start + t;
        if (t >= sp.count || pos < 0) continue;
        const int64_t slot = pos <= 0x7fffffff ? slot_of(a.c, b, (int)pos) : -1;
        if (slot < 0) continue;
        const f32x4 *src = (const f32x4 *)(in + b * a.st.sb + h * a.st.sh + t * a.st.ss + 8 * pl.lane);
        const f32x4 x0 = src[0], x1 = src[1];
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            top = max(top, size_bits(x0[i]));
            top = max(top, size_bits(x1[i]));
        }
        top = max(top, (unsigned)__shfl_xor((int)top, 1, 64));
        top = max(top, (unsigned)__shfl_xor((int)top, 2, 64));
        const bool held = top < 0x7f000000u;
        unsigned byte = top ? max((int)((top + 0x3FFFFFu) >> 23) - 2, kLeastScale) : 127;
        byte = held ? byte : 255;
        const float scale = scale_of(byte);
        unsigned w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x0[0], x0[1], scale, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x0[2], x0[3], scale, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x1[0], x1[1], scale, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x1[2], x1[3], scale, 3);
        const int64_t at = slot + ((int64_t)h << a.c.page_shift);
        *(unsigned *)(codes + at * (D / 2) + 4 * pl.lane) = held ? w : 0u;
        if (pl.lane % 4 == 0) scales[at * (D / 32) + pl.lane / 4] = (uint8_t)byte;
    }
}

template <int D>
__global__ __launch_bounds__(256) void kv_read_kernel(CopyArgs a)
{
    const Place<D> pl(a);
    const int b = blockIdx.y;
    const Span sp = span_of(a.start, a.count, b, a.T);
    float *out = a.out[blockIdx.z];
    const uint8_t *codes = blockIdx.z ? a.c.v_codes : a.c.k_codes, *scales = blockIdx.z ? a.c.v_scales : a.c.k_scales;
    for (unsigned row = blockIdx.x * pl.RPB + threadIdx.x / pl.LPR; row < pl.rows; row += gridDim.x * pl.RPB) {
        const int t = (int)(row / (unsigned)a.c.heads), h = (int)(row - (unsigned)t * a.c.heads);
        const int64_t pos = (int64_t)sp.start + t;
        const int64_t slot = t < sp.count && pos >= 0 && pos <= 0x7fffffff ? slot_of(a.c, b, (int)pos) : -1;
        f32x4 x0 = {0, 0, 0, 0}, x1 = x0;
        if (slot >= 0) {
            const int64_t at = slot + ((int64_t)h << a.c.page_shift);
            const unsigned w = *(const unsigned *)(codes + at * (D / 2) + 4 * pl.lane);
            const float scale = scale_of(scales[at * (D / 32) + pl.lane / 4]);
            const f32x2 p0 = fp4_pair<0>(w, scale), p1 = fp4_pair<1>(w, scale);
            const f32x2 p2 = fp4_pair<2>(w, scale), p3 = fp4_pair<3>(w, scale);
            x0 = f32x4{p0[0], p0[1], p1[0], p1[1]};
            x1 = f32x4{p2[0], p2[1], p3[0], p3[1]};
        }
        f32x4 *dst = (f32x4 *)(out + b * a.st.sb + h * a.st.sh + t * a.st.ss + 8 * pl.lane);
        dst[0] = x0;
        dst[1] = x1;
    }
}

// Enough workgroups to fill the chip; each takes further rows in strides.
template <int D>
dim3 copy_grid(const CopyArgs &a)
{
    const int64_t blocks = ((int64_t)a.T * a.c.heads + Place<D>::RPB - 1) / Place<D>::RPB;
    const int64_t most = 8192 / (2 * a.c.sequences) + 1;
    return dim3((unsigned)(blocks < 1 ? 1 : blocks < most ? blocks : most), (unsigned)a.c.sequences, 2);
}

int check_copy(const ember_kv_cache *cache, const void *k, const void *v, int64_t T, int64_t sb, int64_t sh, int64_t ss,
               const int32_t *start, const int32_t *count, CopyArgs *a, const char *what)
{
    const int st = kv_cache_view(cache, &a->c, what);
    if (st) return st;
    if (T < 0 || T > (0x7fffffff - 65536) / a->c.heads || !row_strides_ok(k, sb, sh, ss) || !row_strides_ok(v, sb, sh, ss) ||
        (((uintptr_t)start | (uintptr_t)count) & 3) || (T && a->c.sequences && (!k || !v)))
        return record_error(EMBER_ERR_INVALID_ARGUMENT, what);
    a->st = {sb, sh, ss};
    a->start = start, a->count = count, a->T = (int)T;
    return EMBER_OK;
}

}  // namespace
}  // namespace ember

extern "C" int kv_cache_write(const ember_kv_cache *cache, const float *k, const float *v, int64_t T, int64_t in_sb,
                              int64_t in_sh, int64_t in_ss, const int32_t *start, const int32_t *count, int32_t *next)
{
    using namespace ember;
    CopyArgs a = {};
    const int st = check_copy(cache, k, v, T, in_sb, in_sh, in_ss, start, count, &a, "kv_cache_write");
    if (st) return st;
    if (((uintptr_t)next & 3) || (next && next == start)) return record_error(EMBER_ERR_INVALID_ARGUMENT, "kv_cache_write");
    if (a.c.sequences == 0 || (T == 0 && !next)) return EMBER_OK;
    a.in[0] = k, a.in[1] = v, a.next = next;
    if (a.c.D == 128) hipLaunchKernelGGL(kv_write_kernel<128>, copy_grid<128>(a), dim3(256), 0, 0, a);
    else if (a.c.D == 64) hipLaunchKernelGGL(kv_write_kernel<64>, copy_grid<64>(a), dim3(256), 0, 0, a);
    else hipLaunchKernelGGL(kv_write_kernel<32>, copy_grid<32>(a), dim3(256), 0, 0, a);
    return launch_ok("kv_cache_write") ? EMBER_OK : EMBER_ERR_DEVICE;
}

extern "C" int kv_cache_read(const ember_kv_cache *cache, float *k, float *v, int64_t T, int64_t out_sb, int64_t out_sh,
                             int64_t out_ss, const int32_t *start, const int32_t *count)
{
    using namespace ember;
    CopyArgs a = {};
    const int st = check_copy(cache, k, v, T, out_sb, out_sh, out_ss, start, count, &a, "kv_cache_read");
    if (st) return st;
    if (a.c.sequences == 0 || T == 0) return EMBER_OK;
    a.out[0] = k, a.out[1] = v;
    if (a.c.D == 128) hipLaunchKernelGGL(kv_read_kernel<128>, copy_grid<128>(a), dim3(256), 0, 0, a);
    else if (a.c.D == 64) hipLaunchKernelGGL(kv_read_kernel<64>, copy_grid<64>(a), dim3(256), 0, 0, a);
    else hipLaunchKernelGGL(kv_read_kernel<32>, copy_grid<32>(a), dim3(256), 0, 0, a);
    return launch_ok("kv_cache_read") ? EMBER_OK : EMBER_ERR_DEVICE;
}
