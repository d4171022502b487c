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
// off: exact for all that is not denormal).  K and V come straight from the cache:
//   K's operand: lane l holds key l % 16 and the D/4 elements of its row from
//     (l / 16) * D/4 on: one load of D/8 bytes and one scale, 8 codes to an operand.
//     Which 8 elements of D that are is free, as long as Q's operand has the same.
//   O^T (D x 16) += V^T . P^T.  Of V, lane l holds tokens 4*(l/16) .. +3 of 16.  For
//     each a code conversion gives two neighbouring elements of D; they are taken
//     as two contraction elements, (token, even) and (token, odd), and P^T has a
//     column for each: p or 0 for the even one, 0 or p for the odd one.  So no
//     value of V is moved between lanes or within a register.
// Eight rows to a workgroup: S^T (16 keys x 16 columns) = K . Q^T, a column for a row's
//   even elements and one for its odd ones, and three instructions for a product.
//   Lane l has column l % 16 and keys 4*(l/16) .. +3, which is what P^T needs: P
//   stays in registers.
// Two or four rows: the parts share an instruction.  S (16 x 16 keys) = Q . K^T, and
//   row 4*a + i of Q's operand is part i of row a (i = 3: nothing), so that lane l
//   has the parts' products of row l / 16 and key l % 16, and adds them: one score
//   for 16 keys (for 32 with two rows, where the two tiles' are shared out), where
//   eight rows' lanes have four each.  P's parts go through LDS to the lanes of
//   their columns: (row, even or odd, part), three parts of two rows, or two of
//   four rows with the third in a second instruction.  A tile of 32 keys takes 16 to
//   24 matrix instructions in place of 48.
// Which is taken goes by a head's rows (2, 4 or more).  Measured (us), the eight-row
// scheme and these: 32 sequences of up to 8192, one token of 32 / 8 heads of 128: 41.1
// and 37.8; 32 x 2048, 16 heads of 64: 19.7 and 17.2.  With eight rows through LDS: 32
// x 16 heads of 64, 24 rows over 2048 46.4 and 50.4.
// A workgroup is 4 waves that take turns at tiles of 32 keys and join at the
// end.  A unit's keys are cut into pieces, each with a workgroup of its own; the
// last of them to be done (by a count that they all add to) joins the pieces, in
// their order.
//
// HBM-bound where contexts are long: 17/32 byte of K and V per element.  32 sequences
// of up to 8192, 32 / 8 heads of 128 (148 MB) take 36.5 us, 4 of up to 32768, 16 heads
// of 128 (178 MB) 42.6, of which about 8 are the launch, the plan, the first loads and
// the join; what is between runs at 5.2 to 5.5 TB/s.  16 x 5 rows over 3001, 16 heads of
// 64 (28 MB) 14.8.
//
// Compiled with blocks that are only jumped to at multiples of 64 bytes, a line of the
// instruction cache: how the loop's blocks fall on lines decides short calls, and any
// edit before them moved it.  One token of 2 x 5 heads of 64 over up to 20206 12.9 us
// so, 12.8 to 14.5 by the place of the loop without (with 32 bytes 12.8, and after an edit
// 14.7); of 32 / 8 heads of 128 over 131072 36.0, and to 39.2; other long calls alike.
#include <algorithm>
#include <type_traits>

#include "kv_attention.h"
#include "lds_dma.h"

namespace ember {
namespace {

constexpr int kTile = 32;  // keys
// Workgroups that a CU holds at once: as many as their registers allow.
constexpr int per_cu(int D, int rows)
{
    return D == 128 && rows == 8 ? 3 : 4;
}
// Workgroups that the keys are cut for, to a CU: fewer than fit, as every further piece
// of a unit is joined by one workgroup in the end, and more of them stream no faster.
// As many as fit and these (us): D = 128, 4 x 1 token, 16 heads over up to 32768 46.5
// and 42.8, 4 tokens of 16 / 4 heads over 16384 18.0 and 16.3, 8 rows of 8 x 8 heads over
// 4096 13.2 and 11.9; D = 64, 4 x 4 tokens of 16 heads over up to 16384 19.1 and 17.9; 16
// x 5 rows over 3001 14.8 and 14.8, with two 16.1.
constexpr int cut_for(int D, int rows)
{
    return D == 128 ? (rows == 8 ? 1 : 2) : 3;
}
// Tiles of a piece at least: five for each wave.  With 8, 16, 20 and 24: 32 / 8 heads of
// 128 over 8192 14.2, 12.8, 12.5, 12.5; 8 x 8 heads of 128 over 4096 10.9, 10.4, 10.6, 10.6;
// 16 x 5 rows over 3001, 16 heads of 64, 14.6, 14.8, 14.9, 15.4.
constexpr int kLeast = 20;

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

// The value of another lane of four: the other of a pair (0xB1), or of the other
// pair (0x4E).
template <int CTRL>
__device__ __forceinline__ float quad(float x)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
}

// ROWS (2, 4 or 8) rows to a workgroup.
template <int D, int ROWS>
__global__ __launch_bounds__(64 * kWaves, per_cu(D, ROWS)) void kv_attention_kernel(KvAttnArgs a)
{
    constexpr int KS = D / 32;  // contraction steps of S, and pairs of elements of a lane of O
    constexpr int STR = D + 4;
    constexpr bool SHARED = ROWS < 8;           // the parts share an instruction
    constexpr int SC = ROWS == 2 ? 1 : ROWS == 4 ? 2 : 8;  // scores of a lane in a tile
    constexpr int SLOTS = 8 / ROWS;             // columns of O for a row's parts
    constexpr int OPS = ROWS == 2 ? 1 : ROWS == 4 ? 2 : 3;
    __shared__ float slab[kWaves][ROWS * STR];
    __shared__ float stat[kWaves][ROWS][2];
    __shared__ uint16_t parts[SHARED ? kWaves : 1][3][ROWS][kTile];
    __shared__ bool last;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, r = lane >> 4;
    const int units = a.c.heads * a.tiles;
    Plan plan;
    const Place pl = start_block(a, plan);
    if (pl.b < 0) return;
    const int b = __builtin_amdgcn_readfirstlane(pl.b), unit = __builtin_amdgcn_readfirstlane(pl.unit);
    const int h = a.by_tiles.of(unit), row0 = (unit - h * a.tiles) * ROWS;
    const Span sp = pl.sp;
    const int len = pl.len;

    const int last_t = min(a.by_group.of(row0 + ROWS - 1), sp.count - 1);
    const int keys = a.by_group.of(row0) < sp.count && a.c.pages ? limit_of(a, sp, len, last_t) : 0;  // all that the rows see
    const int sure = keys ? limit_of(a, sp, len, a.by_group.of(row0)) : 0;  // every row sees the keys before
    auto row_limit = [&](int row) {  // the first key that a row does not see
        const int t = a.by_group.of(row0 + row);
        return t < sp.count ? limit_of(a, sp, len, t) : keys;
    };
    // This lane's row, half and parts of O, and its row and keys of S: score x is
    // of key s_key(x) of the tile.
    const int o_row = col / (2 * SLOTS), slot = col % SLOTS;
    const bool odd = col / SLOTS & 1;
    const int s_row = ROWS == 2 ? r & 1 : ROWS == 4 ? r : o_row;
    auto s_key = [&](int x) { return ROWS == 2 ? 16 * (r >> 1) + col : ROWS == 4 ? 16 * x + col : 16 * (x >> 2) + 4 * r + (x & 3); };
    const int s_limit = row_limit(s_row), o_limit = row_limit(o_row);

    f32x4 acc[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) acc[s] = f32x4{0, 0, 0, 0};
    float m = kNone, l = 0.0f;
    const int n = (keys + kTile - 1) / kTile;
    const int end = pl.piece + 1 < pl.pieces ? min(n, (pl.piece + 1) * plan.per) : n;
    int tl = __builtin_amdgcn_readfirstlane(pl.piece * plan.per) + wave;
    if (tl < end) {
        // Q, and the first tile's keys and values on its heels.
        f32x4 raw[KS][2];
        bool any;
        const int part = SHARED ? col & 3 : 0;  // SHARED: the operand's row is (row, part)
        {
            const int row = row0 + (ROWS == 2 ? col >> 2 & 1 : ROWS == 4 ? col >> 2 : o_row);
            // A row that is not there reads another, for nothing: without a branch,
            // so that waiting for Q is not waiting for what is loaded after it.
            any = a.by_group.of(row) < sp.count && part < 3;
            const int t = any ? a.by_group.of(row) : 0, g = any ? row - t * a.group : 0;
            const float *src = a.q + b * a.qs.sb + (int64_t)(h * a.group + g) * a.qs.sh + t * a.qs.ss + r * (D / 4);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) raw[s][i] = *(const f32x4 *)(src + 8 * s + 4 * i);
        }
        int64_t at[2], ahead[2];
        int page[2];  // of the next tile: both lookups are on their way together, beside the products
        Keys<D> kk[2];
        Values<D> vv[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            at[j] = row_of(a.c, b, h, tl * kTile + 16 * j);
            page[j] = page_of(a.c, b, (tl + kWaves) * kTile + 16 * j);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) kk[j].load(a.c, at[j], lane);
#pragma unroll
        for (int j = 0; j < 2; ++j) vv[j].load(a.c, at[j], lane);
        // No use of Q, and so no wait for it, between the loads, which the compiler mixes
        // (8 rows of 8 x 8 heads of 128 over 4096 13.1 -> 11.9 us; with four rows 12.7 ->
        // 13.3, and with heads of 64 12.5 -> 12.7).
        if (D == 128 && ROWS == 8) __builtin_amdgcn_sched_barrier(0);

        u32x4 q[SHARED ? 1 : 3][KS];
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                unsigned p0[3], p1[3];
                cut3(any ? product(raw[s][i >> 1][2 * (i & 1)], a.scale) : 0.0f, p0[0], p0[1], p0[2]);
                cut3(any ? product(raw[s][i >> 1][2 * (i & 1) + 1], a.scale) : 0.0f, p1[0], p1[1], p1[2]);
                if (SHARED) {
                    p0[0] = part == 0 ? p0[0] : part == 1 ? p0[1] : p0[2];
                    p1[0] = part == 0 ? p1[0] : part == 1 ? p1[1] : p1[2];
                }
#pragma unroll
                for (int j = 0; j < (SHARED ? 1 : 3); ++j) q[j][s][i] = (p0[j] >> 16) | p1[j];
            }

        // Where a half goes in a pair, by v_perm; nowhere for the part that a column
        // has none of.
        const unsigned low_half = odd ? 0x01000c0cu : 0x0c0c0100u, high_half = odd ? 0x03020c0cu : 0x0c0c0302u;
        unsigned low[2], high[2];
        int from[2];  // the column's part, row and tokens in `parts`
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool none = ROWS == 2 ? slot == 3 : i == 1 && slot == 1;
            low[i] = none ? 0x0c0c0c0cu : low_half;
            high[i] = none ? 0x0c0c0c0cu : high_half;
            const int part = ROWS == 2 ? min(slot, 2) : i == 1 ? 2 : slot;
            from[i] = (part * ROWS + o_row) * kTile + 4 * r;
        }
        const unsigned turn = 8 * (col * D / 512) + 9;  // the byte of the lane's group of 32 to bits 23 .. 30

        // One tile; the next one's keys are loaded as soon as this one's are used,
        // and its values after this one's.
        auto step = [&](auto more) {
            float s[8];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                f32x4 sum = {0, 0, 0, 0};
                const float scale = scale_of(kk[j].scale);
#pragma unroll
                for (int x = 0; x < KS; ++x) {
                    const unsigned w = kk[j].code.w[x];
                    const u32x4 k = {fp4_bf16<0>(w, scale), fp4_bf16<1>(w, scale), fp4_bf16<2>(w, scale), fp4_bf16<3>(w, scale)};
                    if constexpr (SHARED) {
                        sum = mfma_16x16x32(q[0][x], k, sum);
                    } else {
#pragma unroll
                        for (int part = 2; part >= 0; --part) sum = mfma_16x16x32(k, q[part][x], sum);
                    }
                }
                if constexpr (SHARED) {
                    s[j] = (sum[2] + sum[1]) + sum[0];
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[4 * j + i] = sum[i];
                }
            }
            if (ROWS == 2) s[0] = r >> 1 ? s[1] : s[0];
            if constexpr (more.value) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    ahead[j] = row_on(a.c, page[j], h, (tl + kWaves) * kTile + 16 * j);
                    kk[j].load(a.c, ahead[j], lane);
                }
            }
            const bool partly = tl * kTile + kTile > sure || at[0] < 0 || at[1] < 0;
            if (partly) {
#pragma unroll
                for (int x = 0; x < SC; ++x)
                    if (tl * kTile + s_key(x) >= s_limit || (s_key(x) < 16 ? at[0] : at[1]) < 0) s[x] = -INFINITY;
            }
            float top = s[0];
#pragma unroll
            for (int x = 1; x < SC; ++x) top = fmaxf(top, s[x]);
            if (__any(top > m + kRaise)) {
                // The lanes of a row: 16 neighbours (and as many 32 on), or those 16 apart.
                const auto most = [](float x, float y) { return fmaxf(x, y); };
                top = SHARED ? row_all(top, most) : across_16(top, most);
                if (ROWS != 4) top = across_32(top, most);
                const float to = fmaxf(m, top);
                float f = __builtin_amdgcn_exp2f(m - to);
                m = to;
                l *= f;
                if (SHARED) f = __shfl(f, 16 * o_row, 64);
#pragma unroll
                for (int x = 0; x < KS; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[x][i] *= f;
            }
            unsigned cut[SC][3];
#pragma unroll
            for (int x = 0; x < SC; ++x) {
                const float e = __builtin_amdgcn_exp2f(s[x] - m);
                l += e;
                cut3(e, cut[x][0], cut[x][1], cut[x][2]);
                if (SHARED)
#pragma unroll
                    for (int part = 0; part < 3; ++part) parts[wave][part][s_row][s_key(x)] = (uint16_t)(cut[x][part] >> 16);
            }
            if (SHARED) wave_sync();
            auto values = [&](auto J) {
                constexpr int j = decltype(J)::value;
                u32x4 p[OPS];
                if constexpr (SHARED) {
#pragma unroll
                    for (int i = 0; i < OPS; ++i) {
                        const uint2 w = *(const uint2 *)(&parts[wave][0][0][0] + from[i] + 16 * j);
                        p[i] = u32x4{__builtin_amdgcn_perm(0, w.x, low[i]), __builtin_amdgcn_perm(0, w.x, high[i]),
                                     __builtin_amdgcn_perm(0, w.y, low[i]), __builtin_amdgcn_perm(0, w.y, high[i])};
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < OPS; ++i)
#pragma unroll
                        for (int x = 0; x < 4; ++x) p[i][x] = __builtin_amdgcn_perm(0, cut[4 * j + x][i], high_half);
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
                            mine |= at[j] >= 0 && tl * kTile + 16 * j + x < o_limit &&
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
                for (int i = OPS - 1; i >= 0; --i)  // the small parts first
#pragma unroll
                    for (int x = 0; x < KS; ++x) acc[x] = mfma_16x16x32(v[x], p[i], acc[x]);
            };
            values(std::integral_constant<int, 0>{});
            values(std::integral_constant<int, 1>{});
            if (SHARED) wave_sync();
            if constexpr (more.value) {
                tl += kWaves;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    vv[j].load(a.c, ahead[j], lane);
                    at[j] = ahead[j];
                    page[j] = page_of(a.c, b, (tl + kWaves) * kTile + 16 * j);  // past the end: not used
                }
            }
        };
        while (tl + kWaves < end) step(std::true_type{});
        step(std::false_type{});
    }
    const auto sum2 = [](float x, float y) { return x + y; };
    l = SHARED ? row_all(l, sum2) : across_16(l, sum2);
    if (ROWS != 4) l = across_32(l, sum2);
    if (SHARED ? col == 0 && r < ROWS : !odd && r == 0) stat[wave][s_row][0] = m, stat[wave][s_row][1] = l;

    // Join the parts, and the waves.
#pragma unroll
    for (int x = 0; x < KS; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float o = acc[x][i];
#pragma unroll
            for (int k = 1; k < SLOTS; k <<= 1) o += k == 1 ? quad<0xB1>(o) : quad<0x4E>(o);
            if (slot == 0) slab[wave][o_row * STR + (4 * r + i) * (D / 16) + 2 * x + odd] = o;
        }
    __syncthreads();
    const int rw = threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
    const bool works = rw < ROWS;
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
        constexpr int PART = ROWS * (D + 2);
        if (works) {
            float *mine = a.part + (int64_t)blockIdx.x * PART;
            put2(mine + rw * D + d, o[0], o[1]);
            put2(mine + rw * D + d + 2, o[2], o[3]);
            if (d == 0) put2(mine + ROWS * D + 2 * rw, top, sum);
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
                    st[j] = get2(one + ROWS * D + 2 * rw), o0[j] = get2(one + rw * D + d), o1[j] = get2(one + rw * D + d + 2);
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
        const int row = row0 + rw, t = a.by_group.of(row), head = h * a.group + row - t * a.group;
        if (t >= a.T) return;
        const bool empty = t >= sp.count || sum == 0.0f;
        *(f32x4 *)(a.o + b * a.os.sb + head * a.os.sh + t * a.os.ss + d) = empty ? f32x4{0, 0, 0, 0} : o / sum;
        if (a.lse && d == 0)
            a.lse[((int64_t)b * a.q_heads + head) * a.T + t] = empty ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
    }
}

template <int D, int ROWS>
int launch(KvAttnArgs &a)
{
    const int st = cut_keys(a, ROWS, kTile, kLeast, per_cu(D, ROWS), cut_for(D, ROWS));
    if (st) return st;
    hipLaunchKernelGGL((kv_attention_kernel<D, ROWS>), dim3((unsigned)a.blocks), dim3(64 * kWaves), 0, 0, a);
    return launch_ok("kv_attention") ? EMBER_OK : EMBER_ERR_DEVICE;
}

template <int D>
int launch_rows(KvAttnArgs &a)
{
    const int rows = a.T * a.group;
    return rows <= 2 ? launch<D, 2>(a) : rows <= 4 ? launch<D, 4>(a) : launch<D, 8>(a);
}

// Rows of a cache head beyond which the kernel for many rows takes over: it walks
// the keys once for 64 rows, this one for 8, but its start is longer, which shows
// where the sequences' heads do not fill the chip by themselves.  This one and that
// one (us, over 2048 keys): 256 heads of 64, 24 rows 24.9 and 21.4, 32 rows 30.5 and
// 24.0; 512 of 64, 16 rows 28.6 and 38.2, 24 rows 39.0 and 38.7; 512 of 128, 24 rows 60
// and 64.  128 heads of 128, 28 rows 26.4 and 27.0, 40 rows 31.2 and 29.8; 16 of 64
// over 8192, 40 rows 17.6 and 26.0.
int few_rows(const KvCache &c)
{
    return (int64_t)c.sequences * c.heads >= device_cu_count() ? 24 : 40;
}

}  // namespace

int cut_keys(KvAttnArgs &a, int rows, int keys, int least, int per_cu, int cut_for)
{
    a.tiles = (int)(((int64_t)a.T * a.group + rows - 1) / rows);
    a.key_shift = __builtin_ctz(keys), a.least = least;
    const int64_t all = (int64_t)a.c.sequences * a.c.heads * a.tiles;  // units
    if (all * 64 * kWaves > 0xffffffff) return record_error(EMBER_ERR_INVALID_ARGUMENT, "kv_cache_attention");
    a.by_group = Divisor(a.group), a.by_tiles = Divisor(a.tiles), a.by_units = Divisor(a.c.heads * a.tiles);
    // cut_for workgroups to a CU; where the units alone are about as
    // many, two pieces each, so that the longest sequence does not decide; but no
    // more than the page table has room for.  With units of several rounds (beyond 4 *
    // slots) only what is longer than two sequences of the mean length is cut: one
    // token of 80 x 32 heads of 128, one sequence of 32768 and 79 of 500, 189 us uncut
    // and 63 so; all of 2000 119 uncut, 134 in two pieces each and 120 so.  With more units
    // yet, where the pieces' results were large, or where no sequence can be longer than
    // a piece, none is cut (and none plans: one token of 4 heads of 64 over 256 5.8 ->
    // 5.0 us).
    const int64_t cus = std::max(device_cu_count(), 1), slots = cut_for * cus;
    const int64_t longest = (((int64_t)a.c.max_pages << a.c.page_shift) + keys - 1) / keys, pieces = (longest + least - 1) / least;
    const bool rounds = all > 4 * slots;
    const int64_t blocks = std::min(rounds ? all + all / 2 : std::max(slots, 2 * all), all * pieces), bytes = blocks * rows * (a.c.D + 2) * (int64_t)sizeof(float);
    const bool cut = pieces > 1 && a.c.sequences <= kMostPlan && all <= std::min<int64_t>(kMostUnits, 4 * per_cu * cus) && bytes <= kMostScratch;
    a.blocks = (int)(cut ? blocks : all);
    a.most = a.blocks / (a.c.heads * a.tiles);
    a.shares = rounds ? 0.5f * a.c.sequences : (float)a.most;
    if (cut) {
        a.part = (float *)scratch(kScratchKvAttention, (size_t)bytes);
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
    a.scale = std::min(scale * kLog2e, 3.402823466e38f);
    int e;
    frexpf(a.scale, &e);
    e = std::min(std::max(e, -126), 127);  // scale2 is a normal number: a masked score stays -infinity under it
    a.q_scale = ldexpf(a.scale, -e), a.scale2 = ldexpf(1.0f, e);
    if (T * a.group > few_rows(a.c)) return launch_kv_attention_rows(a);
    return a.c.D == 128 ? launch_rows<128>(a) : a.c.D == 64 ? launch_rows<64>(a) : launch_rows<32>(a);
}
