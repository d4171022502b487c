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
// end.  A unit's keys are cut into pieces, each with a workgroup of its own; the
// last of them to be done (by a count that they all add to) joins the pieces, in
// their order.
#include <algorithm>
#include <type_traits>

#include "kv_attention.h"
#include "lds_dma.h"

namespace ember {
namespace {

constexpr int kTile = 32;  // keys
constexpr int kRows = 8;   // rows per workgroup
constexpr int kPerCu = 3;  // workgroups that a CU holds at once
constexpr int kLeast = 8;  // tiles of a piece: two for each wave
constexpr int kFewRows = 40;

// Units that are cut: how many of their workgroups are done.  Zero between
// calls: the last one, which all the others have added to, clears its unit's.
// All calls run on the null stream, so no two use it at once.
__device__ unsigned g_done[kMostUnits];

// N bytes (a power of two up to 16) as words; the pointer is aligned to N.
template <int N>
struct Words {
    static constexpr int kWords = N < 4 ? 1 : N / 4;
    unsigned w[kWords];
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
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
};

// What a lane holds of 16 keys, and of 16 values.  Where there are none (at < 0)
// it takes the cache's first ones, which then count for nothing.
template <int D>
struct Keys {
    Words<D / 8> code;
    unsigned scale;
    __device__ __forceinline__ void load(const KvCache &c, int64_t at, int lane)
    {
        const int col = lane & 15, r = lane >> 4;
        at = max(at, (int64_t)0);
        code.load(c.k_codes + at * (D / 2) + (col * (D / 2) + r * (D / 8)));
        scale = (c.k_scales + at * (D / 32))[col * (D / 32) + r * D / 128];
    }
};

template <int D>
struct Values {
    Words<D / 32> code[4];
    Words<D / 8> scale;  // of its 4 tokens
    __device__ __forceinline__ void load(const KvCache &c, int64_t at, int lane)
    {
        const int col = lane & 15, r = lane >> 4;
        at = max(at, (int64_t)0);
        const uint8_t *p = c.v_codes + at * (D / 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) code[i].load(p + ((4 * r + i) * (D / 2) + col * (D / 32)));
        scale.load(c.v_scales + at * (D / 32) + 4 * r * (D / 32));
    }
};

template <int D>
__global__ __launch_bounds__(64 * kWaves, kPerCu) void kv_attention_kernel(KvAttnArgs a)
{
    constexpr int KS = D / 32;  // contraction steps of S, and pairs of elements of a lane of O
    constexpr int STR = D + 4;
    __shared__ float slab[kWaves][kRows * STR];
    __shared__ float stat[kWaves][kRows][2];
    __shared__ bool last;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, r = lane >> 4, row8 = col >> 1;
    const bool odd = col & 1;
    const int units = a.c.heads * a.tiles;
    Plan plan;
    const Place pl = start_block(a, plan);
    if (pl.b < 0) return;
    const int b = __builtin_amdgcn_readfirstlane(pl.b), unit = __builtin_amdgcn_readfirstlane(pl.unit);
    const int h = unit / a.tiles, tile = unit - h * a.tiles;
    const Span sp = span_of(a.start, a.count, b, a.T);
    const int len = length_of(a, sp);

    // This lane's row, and the first key that it does not see.
    const int row = tile * kRows + row8, t = row / a.group, g = row - t * a.group;
    const bool valid = t < sp.count;
    const int last_t = min((tile * kRows + kRows - 1) / a.group, sp.count - 1);
    const int keys = tile * kRows / a.group < sp.count && a.c.pages ? limit_of(a, sp, len, last_t) : 0;  // all that the workgroup's rows see
    const int limit = valid ? limit_of(a, sp, len, t) : keys;
    const int sure = keys ? limit_of(a, sp, len, tile * kRows / a.group) : 0;  // every row sees the keys before

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
    const unsigned half = odd ? 0x03020c0cu : 0x0c0c0302u;  // a float's upper half as the upper or the lower of two
    const unsigned turn = 8 * (col * D / 512) + 9;          // the byte of the lane's group of 32 to bits 23 .. 30

    const int n = (keys + kTile - 1) / kTile;
    const int end = pl.piece + 1 < pl.pieces ? min(n, (pl.piece + 1) * plan.per) : n;
    int tl = __builtin_amdgcn_readfirstlane(pl.piece * plan.per) + wave;
    int64_t at[2], ahead[2];
    Keys<D> kk[2];
    Values<D> vv[2];
    // One tile; the next one's keys are loaded as soon as this one's are used,
    // and its values after this one's.
    auto step = [&](auto more) {
        float s[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            f32x4 sum = {0, 0, 0, 0};
            const float scale = scale_of(kk[j].scale);
#pragma unroll
            for (int x = 0; x < KS; ++x) {
                const unsigned w = kk[j].code.w[x];
                const u32x4 k = {fp4_bf16<0>(w, scale), fp4_bf16<1>(w, scale), fp4_bf16<2>(w, scale), fp4_bf16<3>(w, scale)};
#pragma unroll
                for (int part = 2; part >= 0; --part) sum = mfma_16x16x32(k, q[x][part], sum);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[j][i] = sum[i];
        }
        if constexpr (more.value) {
#pragma unroll
            for (int j = 0; j < 2; ++j) kk[j].load(a.c, ahead[j], lane);
        }
        const bool partly = tl * kTile + kTile > sure || at[0] < 0 || at[1] < 0;
        if (partly) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (tl * kTile + 16 * j + 4 * r + i >= limit || at[j] < 0) s[j][i] = -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, s[j][i]);
        top *= a.scale2;
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
        auto values = [&](auto J) {
            constexpr int j = decltype(J)::value;
            u32x4 p[3];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[j][i], a.scale2, -m));
                l += e;
                unsigned hi, mid, lo;
                cut3(e, hi, mid, lo);
                p[0][i] = __builtin_amdgcn_perm(0, hi, half), p[1][i] = __builtin_amdgcn_perm(0, mid, half);
                p[2][i] = __builtin_amdgcn_perm(0, lo, half);
            }
            // The scale's byte turned to where a float has its exponent: no
            // other bit of it counts.
            float vscale[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned w = vv[j].scale.w[i * D / 128];
                vscale[i] = __builtin_bit_cast(float, __builtin_amdgcn_alignbit(w, w, turn + 8 * (i * (D / 32) & 3)));
            }
            if (partly) {
                // Is a value no number, in a place that some rows do not see
                // (or that was never written)?  Then zero in the product, and
                // NaN given to the rows that do see it.
                bool spoilt[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) spoilt[i] = ((float_bits(vscale[i]) >> 23) & 0xff) > kMostScale;
                if (__any(spoilt[0] || spoilt[1] || spoilt[2] || spoilt[3])) {
                    bool mine = false;
                    for (int x = 0; x < 16; ++x)
                        mine |= at[j] >= 0 && tl * kTile + 16 * j + x < limit &&
                                a.c.v_scales[(at[j] + x) * (D / 32) + r * D / 128] > kMostScale;
#pragma unroll
                    for (int x = 0; x < KS; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[x][i] = mine ? NAN : acc[x][i];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        vscale[i] = spoilt[i] ? 1.0f : vscale[i];
                        vv[j].code[i].w[0] = spoilt[i] ? 0 : vv[j].code[i].w[0];
                    }
                }
            }
            u32x4 v[KS];
            auto convert = [&](auto X) {
                constexpr int x = decltype(X)::value;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[x][i] = fp4_bf16<x>(vv[j].code[i].w[0], vscale[i]);
            };
            convert(std::integral_constant<int, 0>{});
            if constexpr (KS > 1) convert(std::integral_constant<int, 1>{});
            if constexpr (KS > 2) {
                convert(std::integral_constant<int, 2>{});
                convert(std::integral_constant<int, 3>{});
            }
#pragma unroll
            for (int part = 2; part >= 0; --part)  // the small parts first
#pragma unroll
                for (int x = 0; x < KS; ++x) acc[x] = mfma_16x16x32(v[x], p[part], acc[x]);
        };
        values(std::integral_constant<int, 0>{});
        values(std::integral_constant<int, 1>{});
        if constexpr (more.value) {
            tl += kWaves;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                vv[j].load(a.c, ahead[j], lane);
                at[j] = ahead[j];
                ahead[j] = tl + kWaves < end ? row_of(a.c, b, h, (tl + kWaves) * kTile + 16 * j) : -1;
            }
        }
    };
    if (tl < end) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            at[j] = row_of(a.c, b, h, tl * kTile + 16 * j);
            kk[j].load(a.c, at[j], lane);
            vv[j].load(a.c, at[j], lane);
            ahead[j] = tl + kWaves < end ? row_of(a.c, b, h, (tl + kWaves) * kTile + 16 * j) : -1;
        }
        while (tl + kWaves < end) step(std::true_type{});
        step(std::false_type{});
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
    const int rw = threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
    const bool works = rw < kRows;
    float top = kNone, sum = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    if (works) {
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stat[w][rw][0]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(stat[w][rw][0] - top);
            sum += f * stat[w][rw][1];
            o += f * *(const f32x4 *)&slab[w][rw * STR + d];
        }
    }
    if (pl.pieces > 1) {
        constexpr int PART = kRows * (D + 2);
        if (works) {
            float *mine = a.part + (int64_t)blockIdx.x * PART;
            put2(mine + rw * D + d, o[0], o[1]);
            put2(mine + rw * D + d + 2, o[2], o[3]);
            if (d == 0) put2(mine + kRows * D + 2 * rw, top, sum);
        }
        wait_vmem();  // the stores have reached memory
        __syncthreads();
        if (threadIdx.x == 0) last = last_of(&g_done[b * units + unit], pl.pieces);
        __syncthreads();
        if (!last) return;
        if (works) {
            const float *from = a.part + (int64_t)pl.first * PART;
            const int64_t step = (int64_t)units * PART;
            top = kNone, sum = 0.0f, o = f32x4{0, 0, 0, 0};
            constexpr int N = 6;  // pieces whose loads are in flight at once
            for (int i = 0; i < pl.pieces; i += N) {
                f32x2 st[N], o0[N], o1[N];
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float *one = from + min(i + j, pl.pieces - 1) * step;
                    st[j] = get2(one + kRows * D + 2 * rw), o0[j] = get2(one + rw * D + d), o1[j] = get2(one + rw * D + d + 2);
                }
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    if (i + j >= pl.pieces) break;
                    const float to = fmaxf(top, st[j][0]), f = __builtin_amdgcn_exp2f(top - to), g = __builtin_amdgcn_exp2f(st[j][0] - to);
                    top = to;
                    sum = sum * f + st[j][1] * g;
                    o = o * f + f32x4{o0[j][0], o0[j][1], o1[j][0], o1[j][1]} * g;
                }
            }
        }
    }
    if (works) {
        const int row = tile * kRows + rw, t = row / a.group, head = h * a.group + row - t * a.group;
        if (t >= a.T) return;
        const bool empty = t >= sp.count || sum == 0.0f;
        *(f32x4 *)(a.o + b * a.os.sb + head * a.os.sh + t * a.os.ss + d) = empty ? f32x4{0, 0, 0, 0} : o / sum;
        if (a.lse && d == 0)
            a.lse[((int64_t)b * a.q_heads + head) * a.T + t] = empty ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
    }
}

template <int D>
int launch(KvAttnArgs &a)
{
    const int st = cut_keys(a, kRows, kTile, kLeast, kPerCu);
    if (st) return st;
    hipLaunchKernelGGL(kv_attention_kernel<D>, dim3((unsigned)a.blocks), dim3(64 * kWaves), 0, 0, a);
    return launch_ok("kv_attention") ? EMBER_OK : EMBER_ERR_DEVICE;
}

}  // namespace

int cut_keys(KvAttnArgs &a, int rows, int keys, int least, int per_cu)
{
    a.tiles = (int)(((int64_t)a.T * a.group + rows - 1) / rows);
    a.keys = keys, a.least = least;
    const int64_t all = (int64_t)a.c.sequences * a.c.heads * a.tiles;  // units
    if (all * 64 * kWaves > 0xffffffff) return record_error(EMBER_ERR_INVALID_ARGUMENT, "kv_cache_attention");
    // One round of workgroups over the chip; where the units alone are about as
    // many, two pieces each, so that the longest sequence does not decide.  With
    // many units none is cut.
    const int64_t slots = (int64_t)per_cu * std::max(device_cu_count(), 1);
    const bool cut = a.c.sequences <= kMostPlan && all <= std::min<int64_t>(kMostUnits, 4 * slots);
    a.blocks = (int)(cut ? std::max(slots, 2 * all) : all);
    if (cut) {
        a.part = (float *)scratch(kScratchKvAttention, (size_t)a.blocks * rows * (a.c.D + 2) * sizeof(float));
        if (!a.part) return EMBER_ERR_OUT_OF_MEMORY;
    }
    return EMBER_OK;
}

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
    a.causal = causal != 0;
    // Above 0, so that a masked score stays -infinity under it; a scale of 0 then
    // gives scores that differ by nothing.
    a.scale2 = std::max(scale * kLog2e, 1e-37f);
    if (T * a.group > kFewRows) return launch_kv_attention_rows(a);
    return a.c.D == 128 ? launch<128>(a) : a.c.D == 64 ? launch<64>(a) : launch<32>(a);
}
