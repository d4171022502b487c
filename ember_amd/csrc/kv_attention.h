// kv_attention.h -- what the kernels of attention over the 4-bit cache share (not
// part of the public ABI): arguments, how keys are cut into pieces, and the parts
// of an fp32 operand.
#pragma once

#include <math.h>

#include "kv_cache.h"
#include "split_bf16.h"
#include "wave.h"

namespace ember {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNone = -3.402823466e38f;  // the running maximum before any key
constexpr float kRaise = 8.0f;
constexpr int kWaves = 4;        // of a workgroup
constexpr int kMostPlan = 1024;  // sequences that are planned for; with more, a unit is not cut
constexpr int kMostUnits = 1 << 14;  // that are cut
constexpr int64_t kMostScratch = int64_t(160) << 20;  // bytes of their pieces

// Division by a number that the host knows: with inv = floor(2^32 / d) the
// product's upper half is the quotient or one below it, for every n below 2^32.
struct Divisor {
    unsigned d, inv;
    Divisor(unsigned d = 1) : d(d), inv(d > 1 ? (unsigned)((uint64_t(1) << 32) / d) : 0xffffffffu) {}
    __device__ __forceinline__ int of(int n) const
    {
        const unsigned q = __umulhi((unsigned)n, inv);
        return (int)(q + ((unsigned)n - q * d >= d));
    }
};

struct KvAttnArgs {
    KvCache c;
    const float *q;
    float *o, *lse;
    RowStrides qs, os;
    const int32_t *start, *count;
    float *part;  // of each workgroup: O (rows, D), then m and l of each row; null: units are not cut
    int T, q_heads, group, tiles, blocks, causal;  // tiles: of rows, of a head
    int key_shift, least;  // of the keys of a tile, tiles of a piece at least
    // scale * log2(e): Q is multiplied by it as it is read, and a score is the sum of
    // products.  (Scaled then and rounded, the largest of a row and the same score under an
    // fma would differ by half a step: 32 from 2^29 on, a factor of 2^32.)  Where Q is
    // shifted to its row's size, by q_scale (from 0.5 to 1, or 0), and what is left,
    // scale2, is a power of two.
    float scale, q_scale, scale2;
    Divisor by_group, by_tiles, by_units;  // units: of a sequence
    int most;      // pieces of a unit of each sequence, together
    float shares;  // a piece is not less than all sequences' tiles over this, either
};

// Tokens that a sequence has after the call, as far as its table has room.
__device__ __forceinline__ int length_of(const KvAttnArgs &a, Span sp)
{
    const int64_t room = (int64_t)a.c.max_pages << a.c.page_shift;
    return (int)max(min((int64_t)sp.start + sp.count, room), (int64_t)0);
}

// How the keys are cut: into pieces of `per` tiles, the same for every unit (a
// sequence's cache head and a tile of its rows), so that no workgroup has more than
// another however the sequences' lengths differ.  per is the smallest, in steps
// of an eighth, that needs no more workgroups than there are.  Each wave finds
// it for itself; sequences are taken 64 at a time.  Pieces are not made smaller than
// a join is worth.
struct Plan {
    int per;
    // Of sequence `lane`, of the first 64: its rows, length and tiles.
    Span sp;
    int len, tiles;
    __device__ __forceinline__ int pieces(int tiles) const { return max((tiles + per - 1) / per, 1); }
};

__device__ __forceinline__ int tiles_of(const KvAttnArgs &a, int len)
{
    return (len + (1 << a.key_shift) - 1) >> a.key_shift;
}
__device__ __forceinline__ int tiles_of_sequence(const KvAttnArgs &a, int b)
{
    return b < a.c.sequences ? tiles_of(a, length_of(a, span_of(a.start, a.count, b, a.T))) : 0;
}

__device__ __forceinline__ Plan make_plan(const KvAttnArgs &a)
{
    const int lane = threadIdx.x & 63, most = a.most;
    Plan p;
    p.sp = span_of(a.start, a.count, min(lane, a.c.sequences - 1), a.T);
    p.len = length_of(a, p.sp);
    p.tiles = tiles_of(a, p.len);
    auto sum = [&](auto f) {
        auto n = wave_sum(lane < a.c.sequences ? f(p.tiles) : decltype(f(0))(0));
        for (int b = 64; b < a.c.sequences; b += 64)
            n += wave_sum(b + lane < a.c.sequences ? f(tiles_of_sequence(a, b + lane)) : decltype(f(0))(0));
        return n;
    };
    // The sum of all tiles may pass 32 bits; as a float it is near enough.
    p.per = max((int)(sum([](int n) { return (float)n; }) / a.shares), a.least);
    while (sum([&](int n) { return p.pieces(n); }) > most) p.per += p.per / 8 + 1;
    return p;
}

__device__ __forceinline__ f32x4 mfma_16x16x32(u32x4 a, u32x4 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <int S>
__device__ __forceinline__ unsigned fp4_bf16(unsigned w, float scale)
{
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, S));
}

// x * f, rounded to 24 bits before its parts are taken (not kept in an fma).
__device__ __forceinline__ float product(float x, float f)
{
#pragma clang fp contract(off)
    return x * f;
}

// The upper halves of three floats' parts: hi, mid and lo of x.
__device__ __forceinline__ void cut3(float x, unsigned &hi, unsigned &mid, unsigned &lo)
{
    hi = float_bits(x) & 0xffff0000u;
    x -= __builtin_bit_cast(float, hi);
    mid = float_bits(x) & 0xffff0000u;
    x -= __builtin_bit_cast(float, mid);
    lo = float_bits(x) & 0xffff0000u;
}

// Where a workgroup stands: its sequence's rows and length, its unit, its piece of
// the unit's keys, and the unit's first workgroup (its further ones follow
// `units` apart).  The same in all lanes.
struct Place {
    int b, unit, piece, pieces, first;
    Span sp;
    int len;
};

// The place of workgroup `block`; b = -1 where the plan needs fewer.
__device__ __forceinline__ Place place_of(const KvAttnArgs &a, const Plan &p, int block)
{
    const int lane = threadIdx.x & 63, units = a.c.heads * a.tiles;
    int before = 0;
    for (int b0 = 0; b0 < a.c.sequences; b0 += 64) {
        const int tiles = b0 ? tiles_of_sequence(a, b0 + lane) : p.tiles;
        const int n = b0 + lane < a.c.sequences ? p.pieces(tiles) : 0;
        const int upto = wave_scan_sum(n);
        const int at = __popcll(__ballot(block >= before + upto * units));  // sequences that end before
        if (at < 64) {
            Place pl;
            pl.b = b0 + at;
            pl.pieces = __builtin_amdgcn_readlane(n, at);
            const int from = before + (__builtin_amdgcn_readlane(upto, at) - pl.pieces) * units;
            pl.piece = a.by_units.of(block - from), pl.unit = block - from - pl.piece * units;
            pl.first = from + pl.unit;
            if (b0) {
                pl.sp = span_of(a.start, a.count, pl.b, a.T);
                pl.len = length_of(a, pl.sp);
            } else {
                pl.sp = {__builtin_amdgcn_readlane(p.sp.start, at), __builtin_amdgcn_readlane(p.sp.count, at)};
                pl.len = __builtin_amdgcn_readlane(p.len, at);
            }
            return pl;
        }
        before += __builtin_amdgcn_readlane(upto, 63) * units;
    }
    return {-1, 0, 0, 0, 0, {0, 0}, 0};
}

__device__ __forceinline__ void put2(float *p, float x, float y)
{
    put8(p, (uint64_t)float_bits(y) << 32 | float_bits(x));
}
__device__ __forceinline__ f32x2 get2(const float *p)
{
    const uint64_t v = get8(p);
    return f32x2{__builtin_bit_cast(float, (unsigned)v), __builtin_bit_cast(float, (unsigned)(v >> 32))};
}

// The first key that row t of a sequence with `len` tokens does not see.
__device__ __forceinline__ int limit_of(const KvAttnArgs &a, Span sp, int len, int t)
{
    return a.causal ? (int)max(min((int64_t)sp.start + t + 1, (int64_t)len), (int64_t)0) : len;
}

// A unit's workgroup: its place, or b = -1.
__device__ __forceinline__ Place start_block(const KvAttnArgs &a, Plan &plan)
{
    const int units = a.c.heads * a.tiles;
    if (a.part) {
        plan = make_plan(a);
        return place_of(a, plan, blockIdx.x);
    }
    plan.per = 0x40000000;
    const int b = a.by_units.of(blockIdx.x);
    const Span sp = span_of(a.start, a.count, b, a.T);
    return {b, (int)blockIdx.x - b * units, 0, 1, 0, sp, length_of(a, sp)};
}

// Attention for many rows (kv_attention_rows.hip).
int launch_kv_attention_rows(KvAttnArgs &a);
// Fills in how the keys are cut, for workgroups of `rows` rows of which a CU
// holds per_cu and is to be given cut_for, and tiles of `keys` keys; records and
// returns a status.
int cut_keys(KvAttnArgs &a, int rows, int keys, int least, int per_cu, int cut_for);

}  // namespace ember
