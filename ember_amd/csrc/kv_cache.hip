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
// A wave takes 16 tokens of a sequence that are on one page (the table is read
// once, through the scalar cache), of one head, keys or values.  A lane has 4
// neighbours at a time, so that a wave reads and writes 1 KiB of floats in a row;
// a group is 8 lanes, and its largest size found in register moves.  HBM-bound: 4
// bytes read and 17/32 written per element, and the other way round (8 x up to 4096
// rows of 16 heads of 64, padded: written in 36 us, read back in 43; 4 x up to 8191 of 8
// heads of 128 read back in 46, 5.9 TB/s).
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

template <int CTRL>
__device__ __forceinline__ unsigned max_with(unsigned x)
{
    return max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, false));
}
// The largest of 8 neighbouring lanes.
__device__ __forceinline__ unsigned max_of_8(unsigned x)
{
    x = max_with<0xB1>(x);    // the other of a pair
    x = max_with<0x4E>(x);    // the other pair of 4
    return max_with<0x141>(x);  // the other 4, mirrored
}

// What a wave does: 16 tokens from `pos` on (a multiple of 16) of a sequence.
struct Task {
    int b, h, which;  // sequence, head, keys (0) or values (1)
    Span sp;
    int64_t pos, at;  // the first token, and its row in the cache or -1
    bool first;       // of its sequence
};

// Pieces of 16 tokens that T rows of a sequence may touch, wherever they start.
__host__ __device__ inline unsigned pieces_of(int T)
{
    return ((unsigned)T + 30) >> 4;
}

// Task i of sequence blockIdx.y; neighbours are of neighbouring heads.
__device__ __forceinline__ Task task_of(const CopyArgs &a, unsigned i)
{
    Task k;
    k.b = blockIdx.y;
    const unsigned heads = a.c.heads, pair = i / heads, piece = pair >> 1;
    k.h = i - pair * heads;
    k.which = pair & 1;
    k.sp = span_of(a.start, a.count, k.b, a.T);
    k.pos = ((int64_t)(k.sp.start >> 4) + piece) << 4;
    k.at = k.pos >= 0 && k.pos >> a.c.page_shift < a.c.max_pages ? row_of(a.c, k.b, k.h, (int)k.pos) : -1;
    k.first = i == 0;
    return k;
}

template <int D>
__global__ __launch_bounds__(256) void kv_write_kernel(CopyArgs a, unsigned tasks)
{
    constexpr int LPR = D / 4, RPI = 64 / LPR, N = 16 / RPI;  // lanes of a row, rows at a time, times
    const int lane = threadIdx.x & 63, col = lane % LPR;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (unsigned i = blockIdx.x * 4 + wave; i < tasks; i += gridDim.x * 4) {
        const Task k = task_of(a, i);
        if (a.next && k.first && lane == 0) a.next[k.b] = (int)((unsigned)k.sp.start + k.sp.count);
        if (k.at < 0) continue;
        const float *in = a.in[k.which] + k.b * a.st.sb + k.h * a.st.sh + 4 * col;
        uint8_t *codes = (k.which ? a.c.v_codes : a.c.k_codes) + k.at * (D / 2);
        uint8_t *scales = (k.which ? a.c.v_scales : a.c.k_scales) + k.at * (D / 32);
        f32x4 x[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int64_t t = k.pos - k.sp.start + RPI * j + lane / LPR;
            x[j] = t >= 0 && t < k.sp.count ? *(const f32x4 *)(in + t * a.st.ss) : f32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int row = RPI * j + lane / LPR;
            const int64_t t = k.pos - k.sp.start + row;
            const unsigned top = max_of_8(max(max(size_bits(x[j][0]), size_bits(x[j][1])), max(size_bits(x[j][2]), size_bits(x[j][3]))));
            const bool held = top < 0x7f000000u;
            unsigned byte = top ? max((int)((top + 0x3FFFFFu) >> 23) - 2, kLeastScale) : 127;
            byte = held ? byte : 255;
            const float scale = scale_of(byte);
            unsigned w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[j][0], x[j][1], scale, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[j][2], x[j][3], scale, 1);
            if (t >= 0 && t < k.sp.count) {
                *(uint16_t *)(codes + row * (D / 2) + 2 * col) = held ? (uint16_t)w : 0;
                if (col % 8 == 0) scales[row * (D / 32) + col / 8] = (uint8_t)byte;
            }
        }
    }
}

// STREAM: past the caches.
template <int D, bool STREAM>
__global__ __launch_bounds__(256) void kv_read_kernel(CopyArgs a, unsigned tasks)
{
    constexpr int LPR = D / 4, RPI = 64 / LPR, N = 16 / RPI;
    const int lane = threadIdx.x & 63, col = lane % LPR;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (unsigned i = blockIdx.x * 4 + wave; i < tasks; i += gridDim.x * 4) {
        const Task k = task_of(a, i);
        float *out = a.out[k.which] + k.b * a.st.sb + k.h * a.st.sh + 4 * col;
        const uint8_t *codes = (k.which ? a.c.v_codes : a.c.k_codes) + k.at * (D / 2);
        const uint8_t *scales = (k.which ? a.c.v_scales : a.c.k_scales) + k.at * (D / 32);
        unsigned w[N], byte[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int row = RPI * j + lane / LPR;
            const int64_t t = k.pos - k.sp.start + row;
            const bool there = k.at >= 0 && t >= 0 && t < k.sp.count;
            w[j] = there ? *(const uint16_t *)(codes + row * (D / 2) + 2 * col) : 0;
            byte[j] = there ? scales[row * (D / 32) + col / 8] : 127;
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int64_t t = k.pos - k.sp.start + RPI * j + lane / LPR;
            const f32x2 p0 = fp4_pair<0>(w[j], scale_of(byte[j])), p1 = fp4_pair<1>(w[j], scale_of(byte[j]));
            const f32x4 x = {p0[0], p0[1], p1[0], p1[1]};
            if (t >= 0 && t < a.T) {
                f32x4 *to = (f32x4 *)(out + t * a.st.ss);
                if (STREAM) __builtin_nontemporal_store(x, to);
                else *to = x;
            }
        }
    }
}

// Of a sequence; T * heads is below 2^31 - 2^16.
unsigned tasks_of(const CopyArgs &a)
{
    return pieces_of(a.T) * a.c.heads * 2;
}
// Four tasks to a workgroup; beyond 2^18 of them, each takes further ones.
dim3 copy_grid(const CopyArgs &a)
{
    const unsigned n = tasks_of(a);
    return dim3((n < (1 << 20) ? n + 3 : 1 << 20) / 4, a.c.sequences);
}

// What the card's last cache (256 MB) cannot hold is better written past it: 268
// MB read back take 46 us so and 77 through it (with a kernel that reads it next,
// 148 and 163); 134 MB 25 and 27 (60 and 57), 33 MB 8.6 and 10.9 (24.7 and 24.1).
constexpr int64_t kStreamBytes = int64_t(192) << 20;

template <int D>
void launch_read(const CopyArgs &a, unsigned n)
{
    if ((int64_t)a.c.sequences * a.T * a.c.heads * D * 8 > kStreamBytes)
        hipLaunchKernelGGL((kv_read_kernel<D, true>), copy_grid(a), dim3(256), 0, 0, a, n);
    else
        hipLaunchKernelGGL((kv_read_kernel<D, false>), copy_grid(a), dim3(256), 0, 0, a, n);
}

// Whether arrays of nx and ny integers have one in common.
bool share(const int32_t *x, int64_t nx, const int32_t *y, int64_t ny)
{
    const uintptr_t a = (uintptr_t)x, b = (uintptr_t)y;
    return x && y && (a < b ? b - a < nx * sizeof(int32_t) : a - b < ny * sizeof(int32_t));
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
    // Some workgroups read start, count and the table when others have written next.
    const int64_t B = a.c.sequences;
    if (((uintptr_t)next & 3) || share(next, B, start, B) || share(next, B, count, B) || share(next, B, a.c.table, B * a.c.max_pages))
        return record_error(EMBER_ERR_INVALID_ARGUMENT, "kv_cache_write");
    if (a.c.sequences == 0 || (T == 0 && !next)) return EMBER_OK;
    a.in[0] = k, a.in[1] = v, a.next = next;
    const unsigned n = tasks_of(a);
    if (a.c.D == 128) hipLaunchKernelGGL(kv_write_kernel<128>, copy_grid(a), dim3(256), 0, 0, a, n);
    else if (a.c.D == 64) hipLaunchKernelGGL(kv_write_kernel<64>, copy_grid(a), dim3(256), 0, 0, a, n);
    else hipLaunchKernelGGL(kv_write_kernel<32>, copy_grid(a), dim3(256), 0, 0, a, n);
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
    const unsigned n = tasks_of(a);
    if (a.c.D == 128) launch_read<128>(a, n);
    else if (a.c.D == 64) launch_read<64>(a, n);
    else launch_read<32>(a, n);
    return launch_ok("kv_cache_read") ? EMBER_OK : EMBER_ERR_DEVICE;
}
