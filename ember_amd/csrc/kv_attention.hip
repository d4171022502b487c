// kv_attention.hip -- attention of a few query rows over the 4-bit cache.
//
// No reference counterpart.  For a cache head and its G query heads the rows
// are (t, g), t a token of the call; per row
//   s_j = scale * <q, k_j>,  o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m)
// over the keys it sees, in one pass with the running maximum m (base 2, raised
// only where a score passes it by more than 2^8, as the other attention
// kernels do).
//
// Products run on v_mfma_f32_16x16x32_bf16.  A cached value is a bf16 number,
// so only the fp32 operand is split (x = hi + mid + lo, 8 bits each, by cutting
// off: exact for all that is not denormal) and a product is three instructions
// where two fp32 operands take six.  Operands come straight from the cache:
//   S^T (16 keys x 16 columns) = K . Q^T.  Lane l holds key l % 16 and, of its
//     row, the D/4 elements from (l / 16) * D/4 on: one load of D/8 bytes and one
//     scale, 8 codes to an instruction.  Which 8 elements of D that are is free, as
//     long as Q's operand has the same.
//   O^T += V^T . P^T.  Lane l of S^T holds column l % 16 and keys 4*(l/16) .. +3.
//     P is used from those registers, so V's operand has to hold these four
//     tokens too, and for each of them a code conversion gives two neighbouring
//     elements of D.  They are taken as two contraction elements, (token, even)
//     and (token, odd), and P^T has a column for each: p or 0 for the even one, 0
//     or p for the odd one.  So a wave has 8 rows in 16 columns, and no value of V
//     is moved between lanes or within a register.
// A workgroup is 4 waves that take turns at tiles of 32 keys and join at the
// end; a sequence's keys are cut into `splits` parts, each with a workgroup of
// its own, and kv_attention_join adds the parts.
#include <math.h>

#include <algorithm>

#include "kv_cache.h"
#include "split_bf16.h"

namespace ember {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNone = -3.402823466e38f;  // the running maximum before any key
constexpr float kRaise = 8.0f;
constexpr int kWaves = 4;
constexpr int kTile = 32;  // keys
constexpr int kRows = 8;   // rows per workgroup

struct KvAttnArgs {
    KvCache c;
    const float *q;
    float *o, *lse;
    RowStrides qs, os;
    const int32_t *start, *count;
    float *part;  // O (rows, D) of each (unit, split), then m and l of each row
    int T, q_heads, group, tiles, splits, causal;
    float scale2;  // scale * log2(e)
};

__device__ __forceinline__ f32x4 mfma_16x16x32(u32x4 a, u32x4 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <int S>
__device__ __forceinline__ unsigned fp4_bf16(unsigned w, float scale)
{
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, S));
}

// N bytes (a power of two up to 16) as words; the pointer is aligned to N.
template <int N>
struct Words {
    unsigned w[N < 4 ? 1 : N / 4];
    __device__ __forceinline__ void load(const uint8_t *p)
    {
        if constexpr (N == 16) {
            const u32x4 x = *(const u32x4 *)p;
            w[0] = x[0], w[1] = x[1], w[2] = x[2], w[3] = x[3];
        } else if constexpr (N == 8) {
            const uint2 x = *(const uint2 *)p;
            w[0] = x.x, w[1] = x.y;
        } else if constexpr (N == 4) {
            w[0] = *(const unsigned *)p;
        } else if constexpr (N == 2) {
            w[0] = *(const uint16_t *)p;
        } else {
            w[0] = *p;
        }
    }
    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (unsigned &x : w) x = 0;
    }
    __device__ __forceinline__ unsigned byte(int i) const  // i known when compiled, or N <= 4
    {
        return (w[i >> 2] >> (8 * (i & 3))) & 0xff;
    }
};

// What a lane holds of 16 keys and values.
template <int D>
struct Piece {
    Words<D / 8> k;
    unsigned ks;
    Words<D / 32> v[4];
    Words<D / 8> vs;  // the scales of its 4 tokens
    bool there;

    // Key `pos` (a multiple of 16) is the first; pages hold whole pieces.
    __device__ __forceinline__ void load(const KvCache &c, int b, int h, int pos, int lane)
    {
        const int64_t slot = slot_of(c, b, pos);
        there = slot >= 0;
        if (!there) {
            k.zero(), vs.zero(), ks = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i].zero();
            return;
        }
        const int64_t at = slot + ((int64_t)h << c.page_shift);
        const int col = lane & 15, r = lane >> 4;
        k.load(c.k_codes + (at + col) * (D / 2) + r * (D / 8));
        ks = c.k_scales[(at + col) * (D / 32) + r * D / 128];
        const uint8_t *vp = c.v_codes + (at + 4 * r) * (D / 2) + col * (D / 32);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i].load(vp + i * (D / 2));
        vs.load(c.v_scales + (at + 4 * r) * (D / 32));
    }
};

// The upper halves of three floats' parts: hi, mid and lo of x.
__device__ __forceinline__ void cut3(float x, unsigned &hi, unsigned &mid, unsigned &lo)
{
    hi = float_bits(x) & 0xffff0000u;
    x -= __builtin_bit_cast(float, hi);
    mid = float_bits(x) & 0xffff0000u;
    x -= __builtin_bit_cast(float, mid);
    lo = float_bits(x) & 0xffff0000u;
}

template <int D>
__global__ __launch_bounds__(64 * kWaves) void kv_attention_kernel(KvAttnArgs a)
{
    constexpr int KS = D / 32;  // contraction steps of S, and pairs of elements of a lane of O
    constexpr int STR = D + 4;
    __shared__ float slab[kWaves][kRows * STR];
    __shared__ float stat[kWaves][kRows][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, r = lane >> 4, row8 = col >> 1;
    const bool odd = col & 1;
    const int split = blockIdx.x % a.splits;
    const int unit = blockIdx.x / a.splits, tile = unit % a.tiles, bh = unit / a.tiles;
    const int b = bh / a.c.heads, h = bh - b * a.c.heads;
    const Span sp = span_of(a.start, a.count, b, a.T);
    const int64_t room = (int64_t)a.c.max_pages << a.c.page_shift;
    const int len = (int)max(min((int64_t)sp.start + sp.count, room), (int64_t)0);

    // This lane's row, and the first key that it does not see.
    const int row = tile * kRows + row8, t = row / a.group, g = row - t * a.group;
    const bool valid = t < sp.count;
    const int last_t = min((tile * kRows + kRows - 1) / a.group, sp.count - 1);
    auto limit_of = [&](int t) { return a.causal ? (int)max(min((int64_t)sp.start + t + 1, (int64_t)len), (int64_t)0) : len; };
    const int keys = tile * kRows / a.group < sp.count ? limit_of(last_t) : 0;  // all that the workgroup's rows see
    const int limit = valid ? limit_of(t) : keys;
    const int sure = keys ? limit_of(tile * kRows / a.group) : 0;  // every row sees the keys before

    u32x4 q[KS][3];
    {
        const float *src = a.q + b * a.qs.sb + (int64_t)(h * a.group + g) * a.qs.sh + t * a.qs.ss + r * (D / 4);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x2 x = valid ? *(const f32x2 *)(src + 8 * s + 2 * i) : f32x2{0, 0};
                unsigned p0[3], p1[3];
                cut3(x[0], p0[0], p0[1], p0[2]);
                cut3(x[1], p1[0], p1[1], p1[2]);
#pragma unroll
                for (int j = 0; j < 3; ++j) q[s][j][i] = (p0[j] >> 16) | p1[j];
            }
    }

    f32x4 acc[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) acc[s] = f32x4{0, 0, 0, 0};
    float m = kNone, l = 0.0f;
    const int shift = odd ? 0 : 16;

    const int n = (keys + kTile - 1) / kTile, per = (n + a.splits - 1) / a.splits;
    const int end = min(n, (split + 1) * per);
    for (int tl = split * per + wave; tl < end; tl += kWaves) {
        Piece<D> pc[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) pc[j].load(a.c, b, h, tl * kTile + 16 * j, lane);
        float s[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            f32x4 sum = {0, 0, 0, 0};
            const float scale = scale_of(pc[j].ks);
            // The small parts first.
#pragma unroll
            for (int part = 2; part >= 0; --part)
#pragma unroll
                for (int x = 0; x < KS; ++x) {
                    const unsigned w = pc[j].k.w[x];
                    const u32x4 k = {fp4_bf16<0>(w, scale), fp4_bf16<1>(w, scale), fp4_bf16<2>(w, scale), fp4_bf16<3>(w, scale)};
                    sum = mfma_16x16x32(k, q[x][part], sum);
                }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[j][i] = sum[i] * a.scale2;
        }
        const bool partly = tl * kTile + kTile > sure || !pc[0].there || !pc[1].there;
        if (partly) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (tl * kTile + 16 * j + 4 * r + i >= limit || !pc[j].there) s[j][i] = -INFINITY;
        }
        float top = kNone;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, s[j][i]);
        if (__any(top > m + kRaise)) {
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float to = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int x = 0; x < KS; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[x][i] *= f;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            u32x4 p[3];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = __builtin_amdgcn_exp2f(s[j][i] - m);
                l += e;
                unsigned hi, mid, lo;
                cut3(e, hi, mid, lo);
                p[0][i] = hi >> shift, p[1][i] = mid >> shift, p[2][i] = lo >> shift;
            }
            float vscale[4];
            const int gv = col * D / 512;  // the lane's group of 32
            bool spoilt = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned word = pc[j].vs.w[i * D / 128];
                const unsigned byte = (word >> (8 * ((i * (D / 32) & 3) + gv))) & 0xff;
                vscale[i] = scale_of(byte);
                spoilt |= byte > kMostScale;
            }
            if (partly && __any(spoilt)) {
                // A value that is no number, in a place that some rows do not
                // see (or that was never written): zero in the product, and
                // NaN given to the rows that do see it.
                const int64_t slot = slot_of(a.c, b, tl * kTile + 16 * j);
                bool mine = false;
                for (int x = 0; x < 16; ++x) {
                    const int64_t at = slot + ((int64_t)h << a.c.page_shift) + x;
                    mine |= pc[j].there && tl * kTile + 16 * j + x < limit && a.c.v_scales[at * (D / 32) + r * D / 128] > kMostScale;
                }
#pragma unroll
                for (int x = 0; x < KS; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[x][i] = mine ? NAN : acc[x][i];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (vscale[i] >= scale_of(kMostScale + 1)) {
                        vscale[i] = 1.0f;
                        pc[j].v[i].zero();
                    }
            }
#pragma unroll
            for (int part = 2; part >= 0; --part) {
                auto step = [&](auto S) {
                    constexpr int x = decltype(S)::value;
                    const u32x4 v = {fp4_bf16<x>(pc[j].v[0].w[0], vscale[0]), fp4_bf16<x>(pc[j].v[1].w[0], vscale[1]),
                                     fp4_bf16<x>(pc[j].v[2].w[0], vscale[2]), fp4_bf16<x>(pc[j].v[3].w[0], vscale[3])};
                    acc[x] = mfma_16x16x32(v, p[part], acc[x]);
                };
                step(std::integral_constant<int, 0>{});
                if constexpr (KS > 1) step(std::integral_constant<int, 1>{});
                if constexpr (KS > 2) {
                    step(std::integral_constant<int, 2>{});
                    step(std::integral_constant<int, 3>{});
                }
            }
        }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    // Join the waves.
    if (!odd && r == 0) stat[wave][row8][0] = m, stat[wave][row8][1] = l;
#pragma unroll
    for (int x = 0; x < KS; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) slab[wave][row8 * STR + (4 * r + i) * (D / 16) + 2 * x + odd] = acc[x][i];
    __syncthreads();
    for (int at = threadIdx.x; at < kRows * D / 4; at += 64 * kWaves) {
        const int rw = at / (D / 4), d = at % (D / 4) * 4;
        float top = kNone, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stat[w][rw][0]);
        f32x4 o = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(stat[w][rw][0] - top);
            sum += f * stat[w][rw][1];
            o += f * *(const f32x4 *)&slab[w][rw * STR + d];
        }
        const int row = tile * kRows + rw, t = row / a.group, g = row - t * a.group;
        if (t >= a.T) continue;
        if (a.splits > 1) {
            const int64_t block = blockIdx.x;
            *(f32x4 *)(a.part + (block * kRows + rw) * D + d) = o;
            if (d == 0) {
                float *st = a.part + (int64_t)gridDim.x * kRows * D + (block * kRows + rw) * 2;
                st[0] = top, st[1] = sum;
            }
        } else {
            const int head = h * a.group + g;
            const bool empty = t >= sp.count || sum == 0.0f;
            *(f32x4 *)(a.o + b * a.os.sb + head * a.os.sh + t * a.os.ss + d) = empty ? f32x4{0, 0, 0, 0} : o / sum;
            if (a.lse && d == 0)
                a.lse[((int64_t)b * a.q_heads + head) * a.T + t] = empty ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
        }
    }
}

// Adds the parts of each row: D/4 lanes a row.
template <int D>
__global__ __launch_bounds__(256) void kv_attention_join(KvAttnArgs a, int units)
{
    constexpr int LPR = D / 4;
    const int64_t at = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;  // (unit, row of the tile)
    const int d = threadIdx.x % LPR * 4;
    const int64_t unit = at / kRows;
    if (unit >= units) return;
    const int rw = (int)(at % kRows), tile = (int)(unit % a.tiles), bh = (int)(unit / a.tiles);
    const int b = bh / a.c.heads, h = bh - b * a.c.heads;
    const int row = tile * kRows + rw, t = row / a.group, g = row - t * a.group;
    if (t >= a.T) return;
    const Span sp = span_of(a.start, a.count, b, a.T);
    const float *st = a.part + (int64_t)units * a.splits * kRows * D;
    float top = kNone;
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, st[((unit * a.splits + s) * kRows + rw) * 2]);
    float sum = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    for (int s = 0; s < a.splits; ++s) {
        const int64_t i = (unit * a.splits + s) * kRows + rw;
        const float f = __builtin_amdgcn_exp2f(st[2 * i] - top);
        sum += f * st[2 * i + 1];
        o += f * *(const f32x4 *)(a.part + i * D + d);
    }
    const int head = h * a.group + g;
    const bool empty = t >= sp.count || sum == 0.0f;
    *(f32x4 *)(a.o + b * a.os.sb + head * a.os.sh + t * a.os.ss + d) = empty ? f32x4{0, 0, 0, 0} : o / sum;
    if (a.lse && d == 0)
        a.lse[((int64_t)b * a.q_heads + head) * a.T + t] = empty ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

template <int D>
int launch(KvAttnArgs &a)
{
    const int64_t units = (int64_t)a.c.sequences * a.c.heads * a.tiles;
    // Enough workgroups for the chip, 4 of them to a CU, and at least 64 keys
    // each of the longest sequence that the table has room for.
    const int64_t room = (int64_t)a.c.max_pages << a.c.page_shift;
    const int cus = std::max(device_cu_count(), 1);
    const int64_t want = std::min((4 * cus + units - 1) / units, room / 64);
    a.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want, 256));
    if (units * a.splits * 64 * kWaves > 0xffffffff) return record_error(EMBER_ERR_INVALID_ARGUMENT, "kv_cache_attention");
    if (a.splits > 1) {
        a.part = (float *)scratch(kScratchKvAttention, (size_t)units * a.splits * kRows * (D + 2) * sizeof(float));
        if (!a.part) return EMBER_ERR_OUT_OF_MEMORY;
    }
    hipLaunchKernelGGL(kv_attention_kernel<D>, dim3((unsigned)(units * a.splits)), dim3(64 * kWaves), 0, 0, a);
    if (!launch_ok("kv_attention")) return EMBER_ERR_DEVICE;
    if (a.splits > 1) {
        constexpr int rpb = 256 / (D / 4);
        hipLaunchKernelGGL(kv_attention_join<D>, dim3((unsigned)((units * kRows + rpb - 1) / rpb)), dim3(256), 0, 0, a, (int)units);
        if (!launch_ok("kv_attention_join")) return EMBER_ERR_DEVICE;
    }
    return EMBER_OK;
}

}  // namespace
}  // namespace ember

extern "C" int kv_cache_attention(const ember_kv_cache *cache, const float *q, float *o, float *lse, int64_t T, int64_t q_heads,
                                  float scale, int causal, int64_t in_sb, int64_t in_sh, int64_t in_ss, int64_t out_sb,
                                  int64_t out_sh, int64_t out_ss, const int32_t *start, const int32_t *count)
{
    using namespace ember;
    const char *what = "kv_cache_attention";
    KvAttnArgs a = {};
    const int st = kv_cache_view(cache, &a.c, what);
    if (st) return st;
    if (T < 0 || q_heads < 1 || q_heads > 65535 || q_heads % a.c.heads || T > (1 << 30) / (q_heads / a.c.heads) || !(scale >= 0.0f) || scale == INFINITY ||
        !row_strides_ok(q, in_sb, in_sh, in_ss) || !row_strides_ok(o, out_sb, out_sh, out_ss) ||
        (((uintptr_t)start | (uintptr_t)count | (uintptr_t)lse) & 3))
        return record_error(EMBER_ERR_INVALID_ARGUMENT, what);
    if (T == 0 || a.c.sequences == 0) return EMBER_OK;
    if (!q || !o || q == o) return record_error(EMBER_ERR_INVALID_ARGUMENT, what);
    a.q = q, a.o = o, a.lse = lse;
    a.qs = {in_sb, in_sh, in_ss}, a.os = {out_sb, out_sh, out_ss};
    a.start = start, a.count = count;
    a.T = (int)T, a.q_heads = (int)q_heads, a.group = (int)(q_heads / a.c.heads);
    a.tiles = (int)((T * a.group + kRows - 1) / kRows);
    a.causal = causal != 0, a.scale2 = scale * kLog2e;
    return a.c.D == 128 ? launch<128>(a) : a.c.D == 64 ? launch<64>(a) : launch<32>(a);
}
