// kv_attention_rows.hip -- attention of many query rows over the 4-bit cache: a
// prompt read in pieces, on what is cached.
//
// The same sums as in kv_attention.hip, on v_mfma_f32_32x32x16_f16: a workgroup
// has 128 rows, 32 to a wave, and its waves share tiles of 64 keys and values
// that are converted once and laid out in LDS as the matrix core takes them, so
// that the conversion is a small part of the work:
//   S^T (32 keys x 32 rows) = K . Q^T, Q's parts in registers;
//   O^T (D x 32 rows) += V^T . P^T, P's parts from S^T's registers: lane l holds
//     column l % 32 and, of each 16 keys, those of its half h = l / 32: 4h .. 4h+3
//     and 8+4h .. 8+4h+3.  V^T lies in LDS with its keys in that order.
//
// Numbers.  In units of a power of two, u, of the workgroup's, each cached value whose
// scale is from 2^-13 to 2^13 of u is a normal fp16 number.  (Denormal ones, to 2^-23,
// would be exact too, but the matrix cores add their products as those of unnormalized
// numbers: off by up to 2^-16 of themselves.)  The fp32 operands are cut into two fp16
// parts, hi = fp16(x) and lo = fp16(x - hi), off by at most 2^-23 of x, or by 2^-25
// where x is below 1.  A row of Q is shifted so that its largest is
// in [2^14, 2^15): what is lost there is 2^-39 of it.  Weights are e^(s - m) * 2^7 (at
// most 2^15, as m lags by 2^8 at most): what is lost is 2^-32 of the largest weight,
// where the sums' own fp32 loses 2^-25 of theirs.  u is taken near the scales of the
// piece's first token; where a value that a row sees fits no fp16 (far larger or
// smaller than that, or no number), the workgroup walks its keys again with bf16
// values, which hold them all, and three parts.
//   2 x 1024 rows of 32 / 8 heads of 128 over up to 8192 (186 GFLOP): two fp16 parts 345
//   us, three bf16 ones 486, and both, where every piece has such a value, 2.1 times the
//   first's.
// Two tiles of LDS: while one is worked on, the next is converted into the other
// and the one after is loaded; one barrier a tile.
//
// LDS: K rows are D numbers of 16 bits long (fp16, or bf16 in the second walk), V^T
// rows 64, cut into pieces of 16 bytes whose place in the row is turned by the row's
// number (k_place, v_place), so that neither the 32 rows that a wave reads at once
// nor the ones that it writes lie in the same banks.
//
// Work: 8 * T * keys * D matrix operations a head where 4 are the definition's.
// Bound by power: 2 x 1024 rows of 32 / 8 heads of 128 over 8192 keys each, causal, take
// 490 us, 526 TFLOP/s of the definition's and 1.05 PFLOP/s of fp16 at about 1.9 GHz (a
// large bf16 library product reaches 1.23), the matrix cores busy 51 % of the time and
// the vector units 43 %, however the two are mixed; 4 x 512
// rows of 16 heads of 64 over 4096 61 us.
#include <type_traits>

#include "kv_attention.h"
#include "lds_dma.h"

namespace ember {
namespace {

constexpr int kTile = 64;    // keys
// Workgroups that a CU holds at once: as many as their registers allow.
constexpr int per_cu(int D)
{
    return D == 128 ? 2 : D == 64 ? 3 : 4;
}
// Tiles of a piece at least.  With 4, 6, 8 and 16 (us): 300 rows of 16 / 4 heads of 128
// over 2000 38.8, 39.3, 35.3, 50.2; 64 rows of 16 heads of 64 over 8192 30.3, 27.0, 25.4,
// 29.4; 64 rows of 8 x 8 heads of 128 over 4096 33.3, 32.7, 33.2, 37.3; 1000 rows of 4
// heads of 128 over 1000 24.7, 27.8, 31.0, 43.7.
constexpr int kLeast = 8;
// Every code but 0 times 2^kLeastUnit .. 2^kMostUnit is a normal fp16 number.
constexpr int kLeastUnit = -13, kMostUnit = 13;

// As in kv_attention.hip.
__device__ unsigned g_done[kMostUnits];

template <int D>
struct Lds {
    uint4 k[kTile * D / 8], v[kTile * D / 8];  // fp16, or bf16 in the second walk
    // Of the tile's 64 tokens and each group of 32, whether the values are no
    // numbers (bytes: token within the group of D); then, of each 16 tokens,
    // whether they are not there.
    unsigned flags[16 * (D / 32) + 4];
};

// The piece of 16 bytes where elements 8c .. 8c+7 of key `key` are, and where V^T
// has piece c (of 8) of its row d.
template <int D>
__device__ __forceinline__ int k_place(int key, int c)
{
    constexpr int N = D / 8;
    return key * N + (c ^ (D == 128 ? key & 15 : D == 64 ? key & 7 : (key >> 1) & 3));
}
template <int D>
__device__ __forceinline__ int v_place(int d, int c)
{
    return d * 8 + (c ^ ((d ^ (d / (D / 16))) & 7));
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// HALF: the exponent bytes of the scales that K and V are held in units of.
struct Units {
    int k, v;
};

// The scale that a group is converted with; fits = false if there is none that
// keeps its values.
template <bool HALF>
__device__ __forceinline__ float unit_scale(unsigned byte, int unit, bool &fits)
{
    if (!HALF) {
        fits = byte <= kMostScale;
        return scale_of(byte);
    }
    const int over = (int)byte - unit, to = min(max(over, kLeastUnit), kMostUnit);
    fits = to == over;
    return scale_of(to + 127);
}

// Two neighbouring codes as numbers of 16 bits.
template <bool HALF, int S>
__device__ __forceinline__ unsigned fp4_pair16(unsigned w, float scale)
{
    if constexpr (HALF) return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, S));
    else return fp4_bf16<S>(w, scale);
}

// What a thread loads of a tile: a quarter of a key's row, and of 4 tokens' values
// D/16 elements each.  A wave's keys and values are the tile's tokens 16w ..
// 16w+15, which are on one page.
template <int D>
struct Raw {
    static constexpr int KW = D / 32 == 1 ? 1 : D / 32;  // words of a quarter row
    unsigned k[KW], ks, v[4], vs[KW];
    bool there;

    __device__ __forceinline__ void load(const KvCache &c, int64_t at, int thread)
    {
        there = at >= 0;
        at = at < 0 ? 0 : at;
        const int key = (thread >> 2) & 15, r = thread & 3;
        const uint8_t *kp = c.k_codes + at * (D / 2) + (key * (D / 2) + r * (D / 8));
        words(kp, k);
        ks = (c.k_scales + at * (D / 32))[key * (D / 32) + r * D / 128];
        const int quad = (thread >> 4) & 3, col = thread & 15;
        const uint8_t *vp = c.v_codes + at * (D / 2) + (4 * quad * (D / 2) + col * (D / 32));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (D == 128) v[i] = *(const unsigned *)(vp + i * (D / 2));
            else if constexpr (D == 64) v[i] = *(const uint16_t *)(vp + i * (D / 2));
            else v[i] = vp[i * (D / 2)];
        }
        words(c.v_scales + at * (D / 32) + 4 * quad * (D / 32), vs);
    }
    __device__ __forceinline__ static void words(const uint8_t *p, unsigned *w)
    {
        if constexpr (D == 128) {
            const u32x4 x = *(const u32x4 *)p;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = x[i];
        } else if constexpr (D == 64) {
            const uint2 x = *(const uint2 *)p;
            w[0] = x.x, w[1] = x.y;
        } else {
            w[0] = *(const unsigned *)p;
        }
    }

    // Converts and writes them; false if what one of the first `keys` of the tile
    // holds (of those that are there) does not fit the number type.
    template <bool HALF>
    __device__ __forceinline__ bool put(Lds<D> &lds, int thread, Units at, int keys) const
    {
        const int key = thread >> 2, r = thread & 3;
        bool fits = true;
        const float kscale = unit_scale<HALF>(ks, at.k, fits);
        unsigned some = 0;  // not zero
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            some |= k[i];
            lds.k[k_place<D>(key, r * (D / 32) + i)] = uint4{fp4_pair16<HALF, 0>(k[i], kscale), fp4_pair16<HALF, 1>(k[i], kscale),
                                                            fp4_pair16<HALF, 2>(k[i], kscale), fp4_pair16<HALF, 3>(k[i], kscale)};
        }
        bool all = !HALF || fits || (!(some & 0x77777777) && ks <= kMostScale) || key >= keys;
        const int quad = thread >> 4, col = thread & 15;
        float scale[4];
        unsigned w[4], byte[4], bad = 0;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            byte[i] = (vs[i * D / 128] >> (8 * ((i * (D / 32) & 3) + col * D / 512))) & 0xff;
            w[i] = v[i];
            scale[i] = unit_scale<HALF>(byte[i], at.v, fits);
            odd |= !fits;
        }
        if (odd) {  // seldom
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                unit_scale<HALF>(byte[i], at.v, fits);
                if (byte[i] > kMostScale) w[i] = 0, scale[i] = 1.0f, bad |= 1u << (8 * i);  // zero in the products
                else all &= fits || !(w[i] & 0x77777777) || 4 * quad + i >= keys;
            }
        }
        if (col % (16 / (D / 32)) == 0) lds.flags[16 * (col * D / 512) + quad] = bad;
        if ((thread & 63) == 0) lds.flags[16 * (D / 32) + (thread >> 6)] = there ? 0 : 1;
        // Keys 16s .. +15 of a row of V^T: the 8 of half 0, then those of half 1;
        // a quad is 8 bytes.
        const int s = quad >> 2, piece = 2 * s + (quad & 1), half = (quad >> 1) & 1;
        uint2 *to = (uint2 *)lds.v;
        auto pair = [&](auto X) {
            constexpr int x = decltype(X)::value;
            const unsigned a = fp4_pair16<HALF, x>(w[0], scale[0]), b = fp4_pair16<HALF, x>(w[1], scale[1]);
            const unsigned e = fp4_pair16<HALF, x>(w[2], scale[2]), f = fp4_pair16<HALF, x>(w[3], scale[3]);
            const int d = col * (D / 16) + 2 * x;
            to[2 * v_place<D>(d, piece) + half] = uint2{__builtin_amdgcn_perm(b, a, 0x05040100), __builtin_amdgcn_perm(f, e, 0x05040100)};
            to[2 * v_place<D>(d + 1, piece) + half] = uint2{__builtin_amdgcn_perm(b, a, 0x07060302), __builtin_amdgcn_perm(f, e, 0x07060302)};
        };
        pair(std::integral_constant<int, 0>{});
        if constexpr (D > 32) pair(std::integral_constant<int, 1>{});
        if constexpr (D > 64) {
            pair(std::integral_constant<int, 2>{});
            pair(std::integral_constant<int, 3>{});
        }
        return all || !there;
    }
};

template <bool HALF>
__device__ __forceinline__ f32x16 mfma32(uint4 a, u32x4 b, f32x16 c)
{
    if constexpr (HALF) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return mfma_32x32x16(u32x4{a.x, a.y, a.z, a.w}, b, c);
}

// Two floats' upper halves as a packed pair.
__device__ __forceinline__ unsigned upper_halves(float x0, float x1)
{
    return __builtin_amdgcn_perm(float_bits(x1), float_bits(x0), 0x07060302);
}
__device__ __forceinline__ float lower_part(float x)
{
    return x - __builtin_bit_cast(float, float_bits(x) & 0xffff0000u);
}

// Parts of an fp32 operand, and a pair of its elements cut into them.
template <bool HALF>
constexpr int kParts = HALF ? 2 : 3;
template <bool HALF>
__device__ __forceinline__ void cut_pair(float x0, float x1, u32x4 (&to)[kParts<HALF>], int i)
{
    if constexpr (HALF) {
        const f16x2 hi = __builtin_convertvector((f32x2{x0, x1}), f16x2);
        float minus = -1.0f;
        asm("" : "+s"(minus));  // not seen to be -1: x - hi is one instruction (v_fma_mix), not two
        const f16x2 lo = __builtin_convertvector((f32x2{fmaf((float)hi[0], minus, x0), fmaf((float)hi[1], minus, x1)}), f16x2);
        to[0][i] = __builtin_bit_cast(unsigned, hi);
        to[1][i] = __builtin_bit_cast(unsigned, lo);
    } else {
        to[0][i] = upper_halves(x0, x1);
        x0 = lower_part(x0), x1 = lower_part(x1);
        to[1][i] = upper_halves(x0, x1);
        x0 = lower_part(x0), x1 = lower_part(x1);
        to[2][i] = upper_halves(x0, x1);
    }
}

// Two fp16 parts of x0 * f and x1 * f, the lower one from the exact products.
__device__ __forceinline__ void cut_scaled(float x0, float x1, float f, u32x4 (&to)[2], int i)
{
    const f16x2 hi = __builtin_convertvector((f32x2{product(x0, f), product(x1, f)}), f16x2);
    const f16x2 lo = __builtin_convertvector((f32x2{fmaf(x0, f, -(float)hi[0]), fmaf(x1, f, -(float)hi[1])}), f16x2);
    to[0][i] = __builtin_bit_cast(unsigned, hi);
    to[1][i] = __builtin_bit_cast(unsigned, lo);
}

// Units near the scales of a piece's first tokens; the bytes past kMostScale, of what
// is no number, fit none.
__device__ __forceinline__ Units units_at(const KvCache &c, int64_t at)
{
    typedef const __attribute__((address_space(4))) unsigned *scalar;
    auto most = [&](const uint8_t *p) {
        const unsigned w = *(scalar)(uintptr_t)(p + max(at, (int64_t)0) * c.D / 32);
        const unsigned top = max(max(w & 0xff, w >> 8 & 0xff), max(w >> 16 & 0xff, w >> 24));
        return (int)(at < 0 || top > kMostScale ? 127 : min(top, (unsigned)(kMostScale - kMostUnit)));
    };
    return {most(c.k_scales), most(c.v_scales)};
}

// KW = 1: 128 rows, every wave takes all keys of a tile.  KW = 2, up to 64 rows: a
// wave takes 32 keys of a tile, and pairs of waves join at the end (when both took
// three bf16 parts, 64 rows of 8 x 8 heads of 128 over 4096 keys 42 us, with KW = 1 61;
// 65 rows and more would convert every tile twice).
template <int D, int KW>
__global__ __launch_bounds__(64 * kWaves, per_cu(D)) void kv_attention_rows_kernel(KvAttnArgs a)
{
    constexpr int KS = D / 16, DB = D / 32;
    constexpr int kRows = 32 * kWaves / KW;  // rows per workgroup
    __shared__ Lds<D> lds[2];
    __shared__ bool last;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, half = lane >> 5, rows32 = wave / KW;
    const int units = a.c.heads * a.tiles;
    Plan plan;
    const Place pl = start_block(a, plan);
    if (pl.b < 0) return;
    const int b = __builtin_amdgcn_readfirstlane(pl.b), unit = __builtin_amdgcn_readfirstlane(pl.unit);
    // The last rows see most keys: they start first.
    const int h = a.by_tiles.of(unit), tile = a.tiles - 1 - (unit - h * a.tiles);
    const Span sp = pl.sp;
    const int len = pl.len;

    // This lane's row, and the first key that it does not see.
    const int row = tile * kRows + rows32 * 32 + l32, t = a.by_group.of(row), g = row - t * a.group;
    const bool valid = t < sp.count;
    const int first_t = a.by_group.of(tile * kRows), last_t = min(a.by_group.of(tile * kRows + kRows - 1), sp.count - 1);
    const int keys = first_t < sp.count && a.c.pages ? limit_of(a, sp, len, last_t) : 0;  // all that the workgroup's rows see
    const int limit = valid ? limit_of(a, sp, len, t) : keys;
    // All of the wave's rows see the keys before `sure`, none those from `seen` on.
    const int wave_row = tile * kRows + rows32 * 32;
    const int sure = min(keys, limit_of(a, sp, len, a.by_group.of(wave_row)));
    const int seen = a.by_group.of(wave_row) < sp.count ? min(keys, limit_of(a, sp, len, a.by_group.of(wave_row + 31))) : 0;

    const int n = (keys + kTile - 1) / kTile;
    const int first = __builtin_amdgcn_readfirstlane(pl.piece * plan.per);
    const int end = pl.piece + 1 < pl.pieces ? min(n, first + plan.per) : n;

    f32x16 acc[DB];
    float m, l;  // the weights' unit (their maximum, in the end), and their sum
    const auto larger = [](float x, float y) { return fmaxf(x, y); };
    auto piece_at = [&](int tl) { return tl < end ? row_of(a.c, b, h, tl * kTile + 16 * wave) : -1; };
    // The piece's tiles; false if a value does not fit (then the sums are worth nothing).
    auto walk = [&](auto H) -> bool {
        constexpr bool HALF = decltype(H)::value;
        constexpr int P = kParts<HALF>;
        Raw<D> raw;
        bool fits = true;
        Units units16 = {127, 127};
        if (first < end) {
            raw.load(a.c, piece_at(first), threadIdx.x);
            if (HALF) units16 = units_at(a.c, row_of(a.c, b, h, first * kTile));
        }
        u32x4 q[KS][P];
        float scale2 = 1.0f;
        {
            const float *src = a.q + b * a.qs.sb + (int64_t)(h * a.group + g) * a.qs.sh + t * a.qs.ss + 8 * half;
            f32x4 x[KS][2];
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) x[s][i] = valid ? *(const f32x4 *)(src + 16 * s + 4 * i) : f32x4{0, 0, 0, 0};
            int shift = 0;
            if (HALF) {
                float most = 0.0f;
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) most = fmaxf(most, fabsf(x[s][i][j]));
                most = across_32(most, larger) * fmaxf(a.q_scale, 0.5f);  // (0: any shift that Q can take)
                shift = 14 + 127 - (int)(float_bits(most) >> 23);
                scale2 = fminf(fmaxf(ldexpf(a.scale2, units16.k - 127 - shift), 0x1p-126f), 0x1p127f);
            }
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float x0 = x[s][i][2 * j], x1 = x[s][i][2 * j + 1];
                        if constexpr (HALF) cut_scaled(ldexpf(x0, shift), ldexpf(x1, shift), a.q_scale, q[s], 2 * i + j);
                        else cut_pair<false>(product(x0, a.scale), product(x1, a.scale), q[s], 2 * i + j);
                    }
        }
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] = zero16();
        // A weight is 2^(s + c), c = up - m: with the same c for all of a row's weights,
        // whatever m's size, and at most 2^(up + kRaise).
        constexpr float up = HALF ? 7.0f : 0.0f;
        float c = -kNone;
        l = 0.0f;
        auto block = [&](const Lds<D> &at, int key0, auto KB) {
            constexpr int kb = decltype(KB)::value;
            f32x16 s = zero16();
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int x = 0; x < KS; ++x) {
                const uint4 k = at.k[k_place<D>(32 * kb + l32, 2 * x + half)];
#pragma unroll
                for (int part = P - 1; part >= 0; --part) s = mfma32<HALF>(k, q[x][part], s);
            }
            // Vector work goes before other waves' products, which fill the time beside
            // it (D = 64: 66.7 -> 65.2 us at 512 rows of 4 x 16 heads over 4096; D = 128,
            // 2 x 1024 rows of 32 / 8 heads over 8192: 360.4 -> 357.9).  Both halves'
            // scores before the weights gave nothing (351 and 357).
            __builtin_amdgcn_s_setprio(1);
            bool partly = key0 + 32 > sure;  // (no branch: the flags are read early)
            partly |= at.flags[16 * DB + 2 * kb] != 0;
            partly |= at.flags[16 * DB + 2 * kb + 1] != 0;
            if (__builtin_amdgcn_readfirstlane(partly)) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (key0 + acc_row(i, half) >= limit || at.flags[16 * DB + 2 * kb + i / 8]) s[i] = -INFINITY;
            }
            float top = s[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
            top *= scale2;
            if (__any(top + c > up + kRaise)) {
                top = across_32(top, larger);
                const float to = fminf(c, up - top), f = __builtin_amdgcn_exp2f(to - c);
                c = to;
                l *= f;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[d][i] *= f;
            }
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                u32x4 p[P];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e0 = __builtin_amdgcn_exp2f(fmaf(s[8 * st + 2 * i], scale2, c));
                    const float e1 = __builtin_amdgcn_exp2f(fmaf(s[8 * st + 2 * i + 1], scale2, c));
                    l += e0;
                    l += e1;
                    cut_pair<HALF>(e0, e1, p, i);
                }
                constexpr int NP = DB < 2 ? 1 : 2;  // products in turn, so that none waits for the one before
#pragma unroll
                for (int d = 0; d < DB; d += NP) {
                    uint4 v[NP];
#pragma unroll
                    for (int j = 0; j < NP; ++j) v[j] = at.v[v_place<D>(32 * (d + j) + l32, 2 * (2 * kb + st) + half)];
#pragma unroll
                    for (int part = P - 1; part >= 0; --part)
#pragma unroll
                        for (int j = 0; j < NP; ++j) acc[d + j] = mfma32<HALF>(v[j], p[part], acc[d + j]);
                }
            }
        };

        auto put = [&](int tl, Lds<D> &to) {
            fits &= raw.template put<HALF>(to, threadIdx.x, units16, keys - tl * kTile);
        };
        if (first < end) {
            put(first, lds[0]);
            if (first + 1 < end) raw.load(a.c, piece_at(first + 1), threadIdx.x);
            __syncthreads();
        }
        auto step = [&](int tl, const Lds<D> &at, Lds<D> &other) {
            if (tl + 1 < end) {
                put(tl + 1, other);
                if (tl + 2 < end) raw.load(a.c, piece_at(tl + 2), threadIdx.x);
            }
            const int key0 = tl * kTile;
            if (key0 < seen) {
                const unsigned bad = lane < 16 * DB ? at.flags[lane] : 0;
                if (KW == 1 || wave % 2 == 0) block(at, key0, std::integral_constant<int, 0>{});
                if ((KW == 1 || wave % 2 == 1) && key0 + 32 < seen) block(at, key0 + 32, std::integral_constant<int, 1>{});
                // Values that are no numbers: NaN for the rows that see them.
                if (__any(bad)) {
#pragma unroll
                    for (int d = 0; d < DB; ++d)
                        for (int x = 0; x < kTile; ++x)
                            if ((at.flags[16 * d + x / 4] >> (8 * (x & 3)) & 1) && key0 + x < limit && !at.flags[16 * DB + x / 16])
#pragma unroll
                                for (int i = 0; i < 16; ++i) acc[d][i] = NAN;
                }
            }
            __syncthreads();
        };
        for (int tl = first; tl < end; tl += 2) {  // (so that places in LDS are the same each time)
            step(tl, lds[0], lds[1]);
            if (tl + 1 < end) step(tl + 1, lds[1], lds[0]);
        }
        m = -c;
        if (HALF) {
            const float unit = scale_of(units16.v);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[d][i] *= unit;
        }
        return !HALF || __syncthreads_and(fits);
    };
    if (!walk(std::true_type{})) walk(std::false_type{});
    l = across_32(l, [](float x, float y) { return x + y; });

    auto take_in = [&](float m1, float l1, auto value) {  // another part of this wave's rows
        const float to = fmaxf(m, m1), f = __builtin_amdgcn_exp2f(m - to), e = __builtin_amdgcn_exp2f(m1 - to);
        m = to;
        l = l * f + l1 * e;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const f32x2 x = value(8 * d + i);
                acc[d][2 * i] = acc[d][2 * i] * f + x[0] * e;
                acc[d][2 * i + 1] = acc[d][2 * i + 1] * f + x[1] * e;
            }
    };
    if (KW == 2) {
        // The tiles' LDS is free (a barrier ends the loop).
        f32x2 *part = (f32x2 *)lds + rows32 * (16 * D + 64) + lane;
        if (wave % 2 == 1) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 8; ++i) part[64 * (8 * d + i)] = f32x2{acc[d][2 * i], acc[d][2 * i + 1]};
            part[16 * D] = f32x2{m, l};
        }
        __syncthreads();
        if (wave % 2 == 0) {
            const f32x2 st = part[16 * D];
            take_in(st[0], st[1], [&](int i) { return part[64 * i]; });
        }
    }
    const bool keeps = wave % KW == 0 && a.by_group.of(wave_row) < a.T;  // has rows to write
    if (pl.pieces > 1) {
        constexpr int PART = kRows * (D + 2), SUMS = kRows * D;
        float *mine = a.part + (int64_t)blockIdx.x * PART;
        const int at = rows32 * 32 * D + 2 * lane;
        if (keeps) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 8; ++i) put2(mine + at + (8 * d + i) * 128, acc[d][2 * i], acc[d][2 * i + 1]);
            if (half == 0) put2(mine + SUMS + 2 * (rows32 * 32 + l32), m, l);
        }
        wait_vmem();  // the stores have reached memory
        __syncthreads();
        if (threadIdx.x == 0) last = last_of(&g_done[b * units + unit], pl.pieces);
        __syncthreads();
        if (!last || !keeps) return;
        const float *from = a.part + (int64_t)pl.first * PART;
        m = kNone, l = 0.0f;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] = zero16();
        for (int i = 0; i < pl.pieces; ++i, from += (int64_t)units * PART) {
            const f32x2 st = get2(from + SUMS + 2 * (rows32 * 32 + l32));
            take_in(st[0], st[1], [&](int i) { return get2(from + at + i * 128); });
        }
    }
    if (!keeps) return;
    if (t >= a.T) return;
    const int head = h * a.group + g;
    const bool empty = !valid || l == 0.0f;
    const float inv = 1.0f / l;
    float *o = a.o + b * a.os.sb + head * a.os.sh + t * a.os.ss + 4 * half;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f32x4 x;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = empty ? 0.0f : acc[d][4 * i + j] * inv;
            *(f32x4 *)(o + 32 * d + 8 * i) = x;
        }
    if (a.lse && half == 0)
        a.lse[((int64_t)b * a.q_heads + head) * a.T + t] = empty ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

template <int D, int KW>
int launch(KvAttnArgs &a)
{
    const int st = cut_keys(a, 32 * kWaves / KW, kTile, kLeast, per_cu(D), per_cu(D));
    if (st) return st;
    hipLaunchKernelGGL((kv_attention_rows_kernel<D, KW>), dim3((unsigned)a.blocks), dim3(64 * kWaves), 0, 0, a);
    return launch_ok("kv_attention_rows") ? EMBER_OK : EMBER_ERR_DEVICE;
}

}  // namespace

int launch_kv_attention_rows(KvAttnArgs &a)
{
    const bool few = a.T * a.group <= 64;
    if (a.c.D == 128) return few ? launch<128, 2>(a) : launch<128, 1>(a);
    if (a.c.D == 64) return few ? launch<64, 2>(a) : launch<64, 1>(a);
    return few ? launch<32, 2>(a) : launch<32, 1>(a);
}

}  // namespace ember
