// linear8.hip -- products of two 8-bit matrices, out(n x m) = a(n x k) w(m x k)^T
// with the epilogue of linear_fwd, and gated layers of them, h = act(a wg^T + bg)
// * (a wu^T + bu).  No reference counterpart: pawel002/ember computes in fp32.
//
// The products run on the bf16 matrix instruction, codes turned into bf16 with
// their scales on the way (rows8.h; exact), so every product is exact and sums
// are fp32.  gfx950's 8-bit instruction would be twice as fast, but it loses what
// lies far below the largest product of a sum: measured against float64, relative
// 2-norm error at K = 4096 of N(0, 1) operands 1.5e-5, of all codes alike 5.2e-5,
// at one instruction (K = 64) the same; this one 0.9e-7 and 4.3e-7.
#include <algorithm>

#include "activation.h"
#include "lds_dma.h"
#include "linear8.h"
#include "linear8_shape.h"
#include "wave.h"

namespace ember {
namespace {

__device__ __forceinline__ f32x4 mfma_16x16x32(u32x4 a, u32x4 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// 16 bytes per lane from base + offset + at (the same in all lanes) into LDS, lane
// l's at to + l.
__device__ __forceinline__ void dma16_at(__amdgpu_buffer_rsrc_t rsrc, unsigned offset, unsigned at, u32x4 *to)
{
    typedef __attribute__((address_space(3))) void lvoid;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lvoid *)to, 16, offset, at, 0, 0);
}

// The buffer of a tile whose first row is at p (linear8_shape.h).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t bytes_from(const uint8_t *p)
{
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, (short)0, (int)kBufferBytes, 0x00020000);
}

// 16 (4) bytes from base + offset + at (the same in all lanes).
__device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t rsrc, unsigned offset, unsigned at)
{
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, offset, at, 0));
}
__device__ __forceinline__ unsigned load4(__amdgpu_buffer_rsrc_t rsrc, unsigned offset, unsigned at)
{
    return __builtin_amdgcn_raw_buffer_load_b32(rsrc, offset, at, 0);
}

// Few rows: bound by w's bytes.  A workgroup has 16*MB columns of out (a gated
// layer: of the gate, and the same of the other projection) and 16*NT rows.  Its W
// waves share k, each a run of groups, read straight from memory into registers up
// to three groups ahead, and add their sums in wave order.  a comes out of the L2
// once for each workgroup, so columns are many where there are enough of them to
// have all CUs busy.  w's rows are the matrix instruction's rows, so that a lane
// ends up with 4 neighbouring columns of a row of out.  A lane holds a
// 16-byte unit of both halves of a row's group, 8 codes to an instruction; which k
// those are only has to agree.
template <int NT, int MB, int W, bool GATED>
__global__ __launch_bounds__(64 * W) void linear8_few(Linear8Args g)
{
    constexpr int NB = GATED ? 2 : 1, WB = NB * MB;
    constexpr int S = (WB + NT) * 32 <= 128 ? 4 : 2;  // groups in registers (37 x 4096 x 16384 with four: 20.2 us, with two 18.5)
    __shared__ f32x4 sums[W][WB][NT][64];
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col0 = 16 * MB * blockIdx.x, row0 = 16 * NT * blockIdx.y;
    const int64_t pitch = g.w.pitch();
    // Rows past the end re-read the last one; their results are not stored.  A row
    // has at most 2^23 bytes, so offsets fit 32 bits.
    __amdgpu_buffer_rsrc_t wc[NB], ws[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int64_t row = col0 + (int64_t)b * g.m;
        wc[b] = bytes_from(g.w.codes + row * pitch);
        ws[b] = bytes_from(g.w.scales + row * g.w.scale_pitch);
    }
    const auto ac = bytes_from(g.a.codes + row0 * pitch), as = bytes_from(g.a.scales + (int64_t)row0 * g.a.scale_pitch);
    unsigned wo[MB], wso[MB], ao[NT], aso[NT];
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const unsigned row = min(16 * m + r, g.m - 1 - col0);
        wo[m] = row * (unsigned)pitch + 16 * q, wso[m] = row * (unsigned)g.w.scale_pitch;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const unsigned row = min(16 * t + r, g.n - 1 - row0);
        ao[t] = row * (unsigned)pitch + 16 * q, aso[t] = row * (unsigned)g.a.scale_pitch;
    }
    // This wave's groups.  A run of more than two begins with a row's four scales,
    // a shorter one does not go on into the next four.
    const int begin = w * g.chunk, end = min(begin + g.chunk, g.w.groups);
    f32x4 acc[WB][NT];
#pragma unroll
    for (int b = 0; b < WB; ++b)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[b][t] = f32x4{0, 0, 0, 0};
    if (begin < end) {
        u32x4 x[S][WB][2], y[S][NT][2];
        unsigned sx[WB], sy[NT], nx[WB], ny[NT];
        // No branches around the loads, so that they stay ahead of their use: past
        // the run's end nothing is read.
        auto load = [&](int k, int i) {
            const unsigned at = i * kGroup8;
            const bool there = i < end;
#pragma unroll
            for (int b = 0; b < WB; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) x[k][b][h] = load16(wc[b / MB], lane_offset(wo[b % MB], there) + 64 * h, at);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) y[k][t][h] = load16(ac, lane_offset(ao[t], there) + 64 * h, at);
        };
        auto load_scales = [&](int i) {
            const unsigned at = i & ~3;
            const bool there = i < end;
#pragma unroll
            for (int b = 0; b < WB; ++b) nx[b] = load4(ws[b / MB], lane_offset(wso[b % MB], there), at);
#pragma unroll
            for (int t = 0; t < NT; ++t) ny[t] = load4(as, lane_offset(aso[t], there), at);
        };
        load_scales(begin);
#pragma unroll
        for (int k = 0; k < S - 1; ++k) load(k, begin + k);
        for (int i = begin; i < end;) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (k == 0) {
#pragma unroll
                    for (int b = 0; b < WB; ++b) sx[b] = nx[b];
#pragma unroll
                    for (int t = 0; t < NT; ++t) sy[t] = ny[t];
                    load_scales(i + 4);
                }
                load((k + S - 1) % S, i + S - 1);
                __builtin_amdgcn_sched_barrier(0);
                const int shift = 8 * (i & 3);
                float fx[WB], fy[NT];
#pragma unroll
                for (int b = 0; b < WB; ++b) fx[b] = scale8(sx[b] >> shift & 255);
#pragma unroll
                for (int t = 0; t < NT; ++t) fy[t] = scale8(sy[t] >> shift & 255);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    u32x4 v[NT];
#pragma unroll
                    for (int t = 0; t < NT; ++t) v[t] = bf16_of8(y[k % S][t][j / 2][j % 2 * 2], y[k % S][t][j / 2][j % 2 * 2 + 1], fy[t]);
#pragma unroll
                    for (int b = 0; b < WB; ++b) {
                        const u32x4 u = bf16_of8(x[k % S][b][j / 2][j % 2 * 2], x[k % S][b][j / 2][j % 2 * 2 + 1], fx[b]);
#pragma unroll
                        for (int t = 0; t < NT; ++t) acc[b][t] = mfma_16x16x32(u, v[t], acc[b][t]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                if (++i == end) break;
            }
        }
    }
#pragma unroll
    for (int b = 0; b < WB; ++b)
#pragma unroll
        for (int t = 0; t < NT; ++t) sums[w][b][t][lane] = acc[b][t];
    __syncthreads();
    for (int p = w; p < MB * NT; p += W) {
        const int m = p / NT, t = p % NT;
        f32x4 v[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            v[b] = sums[0][b * MB + m][t][lane];
#pragma unroll
            for (int i = 1; i < W; ++i) v[b] += sums[i][b * MB + m][t][lane];
        }
        const int row = row0 + 16 * t + r, col = col0 + 16 * m + 4 * q;
        if (row >= g.n || col >= g.m) continue;
        const int64_t off = (int64_t)row * g.m + col;
        const bool whole = g.aligned;
        f32x4 more = {0, 0, 0, 0};
        if (!GATED && g.residual) {
            if (whole) {
                more = *(const f32x4 *)(g.residual + off);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (col + i < g.m) more[i] = g.residual[off + i];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = col + i < g.m;
            float o = v[0][i] + (g.bias && in ? g.bias[col + i] : 0.0f);
            if (GATED)
                o = gated(steepness(g.act), o, v[NB - 1][i] + (g.bias && in ? g.bias[g.m + col + i] : 0.0f));
            else if (g.act == kActGelu)
                o = gelu08(o);
            v[0][i] = o + more[i];
        }
        if (whole) {
            *(f32x4 *)(g.out + off) = v[0];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (col + i < g.m) g.out[off + i] = v[0][i];
        }
    }
}

// A workgroup's barrier behind a wave's reads of LDS.  __syncthreads would wait for
// the wave's copies into LDS too, those of later stages as well.
__device__ __forceinline__ void meet()
{
    wait_lds();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Many rows: bound by the matrix cores.  A TM x TN block of out per workgroup of
// WR x WC waves (a gated layer: TN/2 columns of the gate and the same of the other
// projection, dealt alike to the waves, so that a lane has both sums of an
// element).
//   * A stage is a group of k, 128 bytes of each row, copied from memory to LDS
//     past the registers, NBUF buffers in turn.  Row r's 16-byte unit q lies at unit
//     q ^ (r/2)%8, so that 16 neighbouring rows of one unit, which a quarter wave
//     reads together, are on different banks; a row's 8 units are copied by
//     neighbouring lanes and stay one line of memory.
//   * Codes become bf16 when they have been read from LDS: LDS then moves and
//     holds half the bytes, and a code is converted by the WC (WR) waves that read
//     it.
//   * Three quarters through a stage all of it is in registers: there is the
//     barrier, behind which the next stage's first operands are read and its
//     buffer's next stage is requested, a copy at a time between products.  There are
//     no branches: past the last stage requests read nothing, and what is read of them
//     is not used.
//   * A product occupies the matrix cores for 32 cycles and a conversion the vector
//     unit for 4: each product is followed by three conversions for later ones, in this
//     order in the code (all conversions of a quarter before its products: 8192 x
//     8192 x 8192 798 us, in turn 772, copies too 761, the four stages that share a
//     load of scales in a row 748).  Then power bounds it: at 4096 x 4096 x 16384
//     1.90 GHz with 68 % of cycles busy, before 1.94 GHz and 65 %; four waves of 128 x
//     128 convert and read a third less and reach the same there.
template <int TM, int TN, int WR, int WC, int NBUF, bool GATED>
__global__ __launch_bounds__(64 * WR * WC, TM * TN == 128 * 128 && NBUF == 2 ? 2 : 1) void linear8_tiles(Linear8Args g)
{
    constexpr int NW = WR * WC, RB = TM / WR / 32, CB = TN / WC / 32, CBH = CB / 2;
    constexpr int CA = TM / 8 / NW, CW = TN / 8 / NW;  // copies of 8 rows to a wave
    static_assert(CA * NW * 8 == TM && CW * NW * 8 == TN && (!GATED || (CW % 2 == 0 && CB % 2 == 0 && TN == 256)), "whole copies");
    // A buffer each: the compiler then knows that a copy into one does not feed
    // reads of another.
    __shared__ u32x4 A0[TM * 8], A1[TM * 8], B0[TN * 8], B1[TN * 8];
    __shared__ u32x4 A2[NBUF > 2 ? TM * 8 : 1], A3[NBUF > 2 ? TM * 8 : 1], B2[NBUF > 2 ? TN * 8 : 1], B3[NBUF > 2 ? TN * 8 : 1];
    const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = w / WC, wc = w % WC;

    // Workgroups are dealt to the 8 XCDs in turn: each gets a run of tiles, grouped
    // 8 row tiles to a panel of columns, for its L2.
    constexpr int COLS = GATED ? TN / 2 : TN;
    const int tiles_n = (g.n + TM - 1) / TM, tiles_m = (g.m + COLS - 1) / COLS, ntiles = tiles_n * tiles_m;
    int tile = blockIdx.x;
    if (ntiles % 8 == 0) tile = tile % 8 * (ntiles / 8) + tile / 8;
    const int per_panel = 8 * tiles_m, panel = tile / per_panel, in_panel = tile - panel * per_panel;
    const int high = min(8, tiles_n - 8 * panel);
    const int row0 = __builtin_amdgcn_readfirstlane((8 * panel + in_panel % high) * TM);
    const int col0 = __builtin_amdgcn_readfirstlane(in_panel / high * COLS);
    const int first = blockIdx.y * g.chunk, stages = min(g.chunk, g.w.groups - first);

    // Rows past the end re-read the last one; their results are not stored.  A row
    // has at most 2^23 bytes, so offsets within a tile fit 32 bits.
    const int64_t pitch = g.w.pitch();
    const auto ra = bytes_from(g.a.codes + row0 * pitch + (int64_t)first * kGroup8);
    const auto rw = bytes_from(g.w.codes + col0 * pitch + (int64_t)first * kGroup8);
    const auto ru = GATED ? bytes_from(g.w.codes + ((int64_t)g.m + col0) * pitch + (int64_t)first * kGroup8) : rw;
    unsigned aoff[CA], woff[CW];
#pragma unroll
    for (int c = 0; c < CA; ++c) {
        const int r = (c * NW + w) * 8 + lane / 8;
        aoff[c] = (unsigned)min(r, g.n - 1 - row0) * (unsigned)pitch + 16 * (lane % 8 ^ r / 2 % 8);
    }
#pragma unroll
    for (int c = 0; c < CW; ++c) {
        const int r = (c * NW + w) * 8 + lane / 8;
        woff[c] = (unsigned)min(r % COLS, g.m - 1 - col0) * (unsigned)pitch + 16 * (lane % 8 ^ r / 2 % 8);
    }
    // Copies `from` to `to` (of CA + CW) of stage s.
    auto request = [&](int s, u32x4 *as, u32x4 *bs, int from, int to) {
        const unsigned at = (unsigned)s * kGroup8;
        const bool there = s < stages;
#pragma unroll
        for (int c = from; c < to; ++c)
            if (c < CA)
                dma16_at(ra, lane_offset(aoff[c], there), at, as + (c * NW + w) * 64);
            else
                dma16_at(c - CA < CW / 2 ? rw : ru, lane_offset(woff[c - CA], there), at, bs + ((c - CA) * NW + w) * 64);
    };

    // This lane's rows of both tiles, 32 apart, and their scales.
    const int arow = 32 * RB * wr + l32;
    auto brow = [&](int cb) { return l32 + (GATED ? (cb < CBH ? 32 * (CBH * wc + cb) : TN / 2 + 32 * (CBH * wc + cb - CBH)) : 32 * (CB * wc + cb)); };
    const uint8_t *const sa = g.a.scales + (int64_t)row0 * g.a.scale_pitch + first;
    const uint8_t *const sw = g.w.scales + (int64_t)col0 * g.w.scale_pitch + first;
    const uint8_t *const su = GATED ? sw + (int64_t)g.m * g.w.scale_pitch : sw;
    unsigned saoff[RB], swoff[CB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) saoff[rb] = (unsigned)min(arow + 32 * rb, g.n - 1 - row0) * (unsigned)g.a.scale_pitch;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) swoff[cb] = (unsigned)min(brow(cb) % COLS, g.m - 1 - col0) * (unsigned)g.w.scale_pitch;
    // A row's scales are read four at a time, in fours of the matrix' groups (first
    // is a multiple of 4).  With two buffers, whose copies are all waited for at every
    // stage, in the last stage of the four before; with more, where a wait for them
    // is one for the copies before them too, three stages ahead.
    constexpr bool AHEAD = NBUF > 2;
    unsigned xa[RB], xw[CB], na[AHEAD ? RB : 1], nw[AHEAD ? CB : 1];
    auto load_scales = [&](int s, unsigned *a, unsigned *w) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) a[rb] = *(const unsigned *)(sa + saoff[rb] + s);
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) w[cb] = *(const unsigned *)((GATED && cb >= CBH ? su : sw) + swoff[cb] + s);
    };

    f32x16 acc[RB][CB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) acc[rb][cb] = zero16();

    // Quarter j of a stage is 32 k: a lane reads unit 2j + half of its rows, of
    // which either 8 codes (t = 0, 1) go to one instruction.  Products and conversions
    // are issued in turn: beside a product run the conversions of the operands of the
    // next one (of w) and of the next t (of a).  What a conversion has read is
    // requested for the next quarter at once.
    u32x4 fa[2][RB], fb[CB], x[2][RB], y[2];
    float fsa[RB], fsw[CB];
    const int at0 = half ^ (l32 >> 1 & 7);
    auto read_a = [&](const u32x4 *as, int j, u32x4 (&to)[RB]) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) to[rb] = as[8 * (arow + 32 * rb) + (at0 ^ 2 * j)];
    };
    auto read_b = [&](const u32x4 *bs, int j, int cb) { fb[cb] = bs[8 * brow(cb) + (at0 ^ 2 * j)]; };
    auto scales_a = [&](int shift) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) fsa[rb] = scale8(xa[rb] >> shift & 255);
    };
    auto scales_w = [&](int shift) {
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) fsw[cb] = scale8(xw[cb] >> shift & 255);
    };
    // Stage s, s % 4 = U, in as, bs, the next one in an, bn.  Its first operands and its
    // scales are there already, and it leaves the next one's.
    auto stage = [&](auto unrolled, int s, u32x4 *as, u32x4 *bs, u32x4 *an, u32x4 *bn) {
        constexpr int U = decltype(unrolled)::value;
        if (AHEAD && U == 0) load_scales(min(s + 4, stages - 1) & ~3, na, nw);
        if (AHEAD && U == 3) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) xa[rb] = na[rb];
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) xw[cb] = nw[cb];
        }
        if (!AHEAD && U == 3) load_scales(min(s + 1, stages - 1) & ~3, xa, xw);
        const int shift = 8 * ((U + 1) % 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const u32x4 *const ar = j < 3 ? as : an, *const br = j < 3 ? bs : bn;
            const int next = (j + 1) % 4;
            if (j == 3) {
                wait_vmem_n<(NBUF - 2) * (CA + CW)>();  // this wave's copies of the next stage, not those of later ones
                meet();
            }
            read_a(ar, next, fa[next & 1]);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (j == 3 && t == 1) scales_a(shift);
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    if (j == 3 && t == 1 && cb == CB - 1) scales_w(shift);
                    const int u = t * CB + cb, ncb = (cb + 1) % CB, nt = cb + 1 == CB ? t ^ 1 : t;
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        acc[rb][cb] = mfma_32x32x16(x[t][rb], y[u & 1], acc[rb][cb]);
#pragma unroll
                        for (int i = 4 * rb / RB; i < 4 * (rb + 1) / RB; ++i)
                            y[(u + 1) & 1][i] = bf16_pair8(fb[ncb][2 * nt], fb[ncb][2 * nt + 1], i, fsw[ncb]);
                        constexpr int SLOTS = 2 * CB * RB;
                        if (j == 3) request(s + NBUF, as, bs, (u * RB + rb) * (CA + CW) / SLOTS, (u * RB + rb + 1) * (CA + CW) / SLOTS);
                        const auto &a = fa[(t ? next : j) & 1];
#pragma unroll
                        for (int q = (cb * RB + rb) * 4 / CB; q < (cb * RB + rb + 1) * 4 / CB; ++q)
                            x[t ^ 1][q / 4][q % 4] = bf16_pair8(a[q / 4][2 * (t ^ 1)], a[q / 4][2 * (t ^ 1) + 1], q % 4, fsa[q / 4]);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    if (nt == 1) read_b(br, next, ncb);
                }
            }
        }
    };
    load_scales(0, xa, xw);
    request(0, A0, B0, 0, CA + CW);
    request(1, A1, B1, 0, CA + CW);
    if constexpr (AHEAD) {
        request(2, A2, B2, 0, CA + CW);
        request(3, A3, B3, 0, CA + CW);
    }
    wait_vmem_n<(NBUF - 1) * (CA + CW)>();
    meet();
    read_a(A0, 0, fa[0]);
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) read_b(B0, 0, cb);
    scales_a(0);
    scales_w(0);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) x[0][rb] = bf16_of8(fa[0][rb][0], fa[0][rb][1], fsa[rb]);
    y[0] = bf16_of8(fb[0][0], fb[0][1], fsw[0]);
    std::integral_constant<int, 0> u0;
    std::integral_constant<int, 1> u1;
    std::integral_constant<int, 2> u2;
    std::integral_constant<int, 3> u3;
    int s = 0;
    constexpr bool FOUR = NBUF > 2;
    for (; s + 4 <= stages; s += 4) {
        stage(u0, s, A0, B0, A1, B1);
        stage(u1, s + 1, A1, B1, FOUR ? A2 : A0, FOUR ? B2 : B0);
        stage(u2, s + 2, FOUR ? A2 : A0, FOUR ? B2 : B0, FOUR ? A3 : A1, FOUR ? B3 : B1);
        stage(u3, s + 3, FOUR ? A3 : A1, FOUR ? B3 : B1, A0, B0);
    }
    if (s < stages) stage(u0, s, A0, B0, A1, B1);
    if (s + 1 < stages) stage(u1, s + 1, A1, B1, FOUR ? A2 : A0, FOUR ? B2 : B0);
    if (s + 2 < stages) stage(u2, s + 2, FOUR ? A2 : A0, FOUR ? B2 : B0, FOUR ? A3 : A1, FOUR ? B3 : B1);

    // The sums go through LDS, 32 rows of the waves that share rows at a time (each
    // such set has a buffer), and leave in rows: a loop of few instructions, where
    // one over registers would be unrolled to many times the main loop's code.  32
    // columns are swapped in every other four rows, so that the two halves of a
    // wave write to different banks.
    static_assert(WR <= 2 || (WR <= 4 && TM >= TN), "32 rows fit a buffer");
    float *const rows = (float *)(wr == 0 ? B0 : wr == 1 || WR <= 2 ? B1 : wr == 2 ? A0 : A1);
    auto at = [](int r, int col) { return r * TN + (col ^ (r & 4) << 3); };
    // at(acc_row(i, half), l32 + a block's column) of even and of odd blocks.
    float *const put[2] = {rows + 4 * half * TN + l32 + 32 * half, rows + 4 * half * TN + l32 - 32 * half};
    const int t = threadIdx.x % (64 * WC);
    wait_vmem();  // requests past the last stage still write to the buffers
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        __syncthreads();
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
            for (int i = 0; i < 16; ++i) put[(brow(cb) - l32) / 32 & 1][acc_row(i, 0) * TN + brow(cb) - l32] = acc[rb][cb][i];
        __syncthreads();
        const int row1 = row0 + 32 * (RB * wr + rb);
        if constexpr (!GATED) {
            const int q = t % (TN / 4), col = col0 + 4 * q;
            float *const out = g.part ? g.part + (int64_t)blockIdx.y * g.n * g.m : g.out;
            f32x4 bias = {0, 0, 0, 0};
            if (!g.part && g.bias)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (col + i < g.m) bias[i] = g.bias[col + i];
            const bool whole = g.aligned && col < g.m;
            constexpr int STEP = 64 * WC / (TN / 4), N = 4;  // rows at a time, and times whose loads are in flight together
            for (int r0 = t / (TN / 4); r0 < 32; r0 += N * STEP) {
                f32x4 v[N], more[N];
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const int r = r0 + k * STEP;
                    const int64_t off = (int64_t)(row1 + r) * g.m + col;
                    v[k] = *(const f32x4 *)&rows[at(r, 4 * q)] + bias;
                    more[k] = f32x4{0, 0, 0, 0};
                    if (g.part || !g.residual || row1 + r >= g.n) continue;
                    if (whole) {
                        more[k] = *(const f32x4 *)(g.residual + off);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (col + i < g.m) more[k][i] = g.residual[off + i];
                    }
                }
                if (!g.part && g.act == kActGelu)
#pragma unroll
                    for (int k = 0; k < N; ++k)
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[k][i] = gelu08(v[k][i]);
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const int r = r0 + k * STEP;
                    const int64_t off = (int64_t)(row1 + r) * g.m + col;
                    if (row1 + r >= g.n) continue;
                    v[k] += more[k];
                    if (whole) {
                        *(f32x4 *)(out + off) = v[k];
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (col + i < g.m) out[off + i] = v[k][i];
                    }
                }
            }
        } else {
            // The tile's 128 columns are a group of h: a half wave has a row.
            const int q = t % 32, col = col0 + 4 * q, group = col0 / kGroup8;
            f32x4 bg = {0, 0, 0, 0}, bu = bg;
            if (g.bias)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (col + i < g.m) bg[i] = g.bias[col + i], bu[i] = g.bias[g.m + col + i];
            const float c = steepness(g.act);
            constexpr int STEP = 2 * WC, N = 4;  // rows at a time, and times taken together
            for (int r0 = t / 32; r0 < 32; r0 += N * STEP) {
                f32x4 x[N], u[N];
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    x[k] = *(const f32x4 *)&rows[at(r0 + k * STEP, 4 * q)] + bg;
                    u[k] = *(const f32x4 *)&rows[at(r0 + k * STEP, TN / 2 + 4 * q)] + bu;
                }
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const int64_t row = row1 + r0 + k * STEP;
                    f32x4 v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = col + i < g.m ? gated(c, x[k][i], u[k][i]) : 0.0f;
                    const unsigned byte = scale_byte8(max_of_32(max(max(size_bits8(v[0]), size_bits8(v[1])), max(size_bits8(v[2]), size_bits8(v[3])))));
                    if (row >= g.n) continue;
                    *(unsigned *)(g.h.codes + row * g.h.pitch() + col) = byte == 255 ? 0 : codes8(v[0], v[1], v[2], v[3], inverse_scale8(byte));
                    uint8_t *const to = g.h.scales + row * g.h.scale_pitch;
                    if (q == 0) to[group] = (uint8_t)byte;
                    if (group == g.h.groups - 1 && q > 0 && group + q < g.h.scale_pitch) to[group + q] = 127;
                }
            }
        }
    }
}

// out = epilogue(sum over z of part[z]), z in order.
__global__ __launch_bounds__(256) void linear8_reduce(Linear8Args g, int splits, int64_t total)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        float v = g.part[i];
        for (int z = 1; z < splits; ++z) v += g.part[z * total + i];
        if (g.bias) v += g.bias[i % g.m];
        if (g.act == kActGelu) v = gelu08(v);
        if (g.residual) v += g.residual[i];
        g.out[i] = v;
    }
}

// The same for a gated layer, whose parts are (n, 2 hidden): a half wave has a
// group of h, a lane 4 neighbours.
__global__ __launch_bounds__(256) void gated8_reduce(Linear8Args g, int splits, int64_t tasks)
{
    const int l32 = threadIdx.x & 31, hidden = g.h.cols;
    const int64_t total = (int64_t)g.n * 2 * hidden;
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < tasks; i += (int64_t)gridDim.x * 8) {
        const int64_t row = i / g.h.scale_pitch;
        const int group = (int)(i - row * g.h.scale_pitch), col = group * kGroup8 + 4 * l32;
        float v[4];
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = 0;
            if (col + j < hidden) {
                const float *const p = g.part + row * 2 * hidden + col + j;
                float a = p[0], b = p[hidden];
                for (int z = 1; z < splits; ++z) a += p[z * total], b += p[z * total + hidden];
                if (g.bias) a += g.bias[col + j], b += g.bias[hidden + col + j];
                v[j] = gated(steepness(g.act), a, b);
            }
            top = max(top, size_bits8(v[j]));
        }
        const unsigned byte = scale_byte8(max_of_32(top));
        if (group < g.h.groups)
            *(unsigned *)(g.h.codes + row * g.h.pitch() + col) = byte == 255 ? 0 : codes8(v[0], v[1], v[2], v[3], inverse_scale8(byte));
        if (l32 == 0) g.h.scales[i] = (uint8_t)byte;
    }
}

template <int TM, int TN, int WR, int WC, int NBUF, bool GATED>
bool launch_tiles(const Linear8Args &g, int splits, const char *kernel)
{
    const int64_t tiles = (((int64_t)g.n + TM - 1) / TM) * (((int64_t)g.m + (GATED ? TN / 2 : TN) - 1) / (GATED ? TN / 2 : TN));
    hipLaunchKernelGGL((linear8_tiles<TM, TN, WR, WC, NBUF, GATED>), dim3((unsigned)tiles, splits), dim3(64 * WR * WC), 0, 0, g);
    return launch_ok(kernel);
}

// 128 x 128 tiles: four buffers, which leave room for one workgroup on a CU, where
// there are no more than CUs.
bool launch_small(const Linear8Args &g, int splits)
{
    const int64_t tiles = (((int64_t)g.n + 127) / 128) * (((int64_t)g.m + 127) / 128);
    return tiles * splits <= num_cus() ? launch_tiles<128, 128, 2, 2, 4, false>(g, splits, "linear8_tiles128_ahead")
                                       : launch_tiles<128, 128, 2, 2, 2, false>(g, splits, "linear8_tiles128");
}

template <int NT, int MB, int W, bool GATED>
void launch_few_as(Linear8Args g)
{
    // A wave's run of groups: one, two or fours.
    g.chunk = (g.w.groups + W - 1) / W;
    if (g.chunk > 2) g.chunk = (g.chunk + 3) / 4 * 4;
    const dim3 grid((g.m + 16 * MB - 1) / (16 * MB), (g.n + 16 * NT - 1) / (16 * NT));
    hipLaunchKernelGGL((linear8_few<NT, MB, W, GATED>), grid, dim3(64 * W), 0, 0, g);
}

template <int NT, bool GATED>
void launch_few_rows(const Linear8Args &g)
{
    const int cus = num_cus(), mb = few_columns(g.n, g.m, GATED, cus);
    if constexpr (GATED) {
        if (NT > 2 && mb == 2) launch_few_as<NT, (NT > 2 ? 2 : 1), 2, true>(g);
        else launch_few_as<NT, 1, 2, true>(g);
    } else {
        if (mb == 4) launch_few_as<NT, 4, 4, false>(g);
        else if (mb == 2) launch_few_as<NT, 2, 2, false>(g);
        else if (NT == 1 && four_waves(g.m, g.w.groups, cus)) launch_few_as<NT, 1, (NT == 1 ? 4 : 2), false>(g);
        else launch_few_as<NT, 1, 2, false>(g);
    }
}

template <bool GATED>
bool launch_few(const Linear8Args &g)
{
    switch (few_rows(g.n)) {
        case 1: launch_few_rows<1, GATED>(g); break;
        case 2: launch_few_rows<2, GATED>(g); break;
        case 3: launch_few_rows<3, GATED>(g); break;
        default: launch_few_rows<4, GATED>(g);
    }
    return launch_ok(GATED ? "gated8_few" : "linear8_few");
}

// Whether rows of out and residual can be moved 16 bytes at a time (a split's parts,
// which are the library's, then can too).
bool aligned_rows(const Linear8Args &g)
{
    return g.m % 4 == 0 && (((uintptr_t)g.out | (uintptr_t)g.residual) & 15) == 0;
}

// Rows of a call that go in one launch (grids, and products of tiles, stay small).
constexpr int64_t kRowsPerLaunch = 1 << 20;

Linear8Args rows_from(const Linear8Args &g, int64_t row)
{
    Linear8Args p = g;
    p.n = p.a.rows = p.h.rows = (int)std::min<int64_t>(g.n - row, kRowsPerLaunch);
    p.a.codes += row * g.a.pitch();
    p.a.scales += row * g.a.scale_pitch;
    if (p.out) p.out += row * g.m;
    if (p.residual) p.residual += row * g.m;
    if (p.h.codes) p.h.codes += row * g.h.pitch(), p.h.scales += row * g.h.scale_pitch;
    return p;
}

int linear8_launch(const Linear8Args &all)
{
    for (int64_t row = 0; row < all.n; row += kRowsPerLaunch) {
        Linear8Args g = rows_from(all, row);
        Choice c = choose(g.n, g.m, g.w.groups, false, num_cus());
        const int64_t total = (int64_t)g.n * g.m;
        g.aligned = aligned_rows(g);
        if (c.splits > 1) {
            g.part = (float *)scratch(kScratchLinear8, (size_t)c.splits * total * sizeof(float), true);
            if (!g.part) c = without_scratch(g.w.groups, false);
        }
        g.chunk = c.chunk;
        if (!(c.kernel == kFew ? launch_few<false>(g)
              : c.kernel == kLargeTiles ? launch_tiles<256, 256, 4, 2, 2, false>(g, 1, "linear8_tiles256")
                                        : launch_small(g, c.splits)))
            return EMBER_ERR_DEVICE;
        if (c.splits > 1) {
            hipLaunchKernelGGL(linear8_reduce, dim3((unsigned)std::min<int64_t>((total + 255) / 256, 1 << 13)), dim3(256), 0, 0, g, c.splits, total);
            if (!launch_ok("linear8_reduce")) return EMBER_ERR_DEVICE;
        }
    }
    return EMBER_OK;
}

int gated8_launch(const Linear8Args &all)
{
    for (int64_t row = 0; row < all.n; row += kRowsPerLaunch) {
        Linear8Args g = rows_from(all, row);
        Choice c = choose(g.n, g.m, g.w.groups, true, num_cus());
        if (c.kernel == kFew || c.kernel == kSmallTiles) {  // h, or the parts of both sums, in fp32
            const size_t sums = (size_t)g.n * g.m * (c.kernel == kFew ? 1 : 2 * c.splits);
            float *const p = (float *)scratch(kScratchLinear8, sums * sizeof(float), true);
            if (!p) c = without_scratch(g.w.groups, true);
            (c.kernel == kFew ? g.out : g.part) = p;
        }
        g.chunk = c.chunk;
        if (c.kernel == kLargeTiles || c.kernel == kMidTiles) {
            if (!(c.kernel == kMidTiles ? launch_tiles<128, 256, 2, 4, 2, true>(g, 1, "gated8_tiles128")
                                        : launch_tiles<256, 256, 4, 2, 2, true>(g, 1, "gated8_tiles256")))
                return EMBER_ERR_DEVICE;
        } else if (c.kernel == kFew) {
            g.aligned = aligned_rows(g);
            if (!launch_few<true>(g)) return EMBER_ERR_DEVICE;
            const int st = rows8_write_launch(g.h, g.out, g.m, 0, "rows8_write");
            if (st) return st;
        } else {
            const int64_t tasks = (int64_t)g.n * g.h.scale_pitch;
            g.m *= 2;
            g.aligned = g.m % 4 == 0;
            if (!launch_small(g, c.splits)) return EMBER_ERR_DEVICE;
            hipLaunchKernelGGL(gated8_reduce, dim3((unsigned)std::min<int64_t>((tasks + 7) / 8, 1 << 13)), dim3(256), 0, 0, g, c.splits, tasks);
            if (!launch_ok("gated8_reduce")) return EMBER_ERR_DEVICE;
        }
    }
    return EMBER_OK;
}

// Both operands, of as many columns.
int operands(const ember_rows8 *a, const ember_rows8 *w, Linear8Args *g, const char *who)
{
    int st = rows8_view(a, &g->a, who);
    if (!st) st = rows8_view(w, &g->w, who);
    if (st) return st;
    if (g->a.cols != g->w.cols) return record_error(EMBER_ERR_INVALID_ARGUMENT, who);
    return EMBER_OK;
}

}  // namespace
}  // namespace ember

extern "C" int linear8_fwd(const ember_rows8 *a, const ember_rows8 *w, const float *bias, const float *residual, float *out, int act)
{
    using namespace ember;
    Linear8Args g = {};
    const int st = operands(a, w, &g, "linear8_fwd");
    if (st) return st;
    if (!out || (((uintptr_t)out | (uintptr_t)bias | (uintptr_t)residual) & 3) || act < kActNone || act > kActGelu)
        return record_error(EMBER_ERR_INVALID_ARGUMENT, "linear8_fwd");
    g.bias = bias, g.residual = residual, g.out = out, g.n = g.a.rows, g.m = g.w.rows, g.act = act;
    return g.n && g.m ? linear8_launch(g) : EMBER_OK;
}

extern "C" int gated8_fwd(const ember_rows8 *a, const ember_rows8 *w, const float *bias, const ember_rows8 *h, int act)
{
    using namespace ember;
    Linear8Args g = {};
    Rows8 to;
    int st = operands(a, w, &g, "gated8_fwd");
    if (!st) st = rows8_view(h, &to, "gated8_fwd");
    if (st) return st;
    if (((uintptr_t)bias & 3) || act < kActGelu || act > kActSilu || g.w.rows != 2 * (int64_t)to.cols || g.a.rows != to.rows)
        return record_error(EMBER_ERR_INVALID_ARGUMENT, "gated8_fwd");
    if (to.rows == 0) return EMBER_OK;
    g.bias = bias, g.h = to, g.n = to.rows, g.m = to.cols, g.act = act;
    return gated8_launch(g);
}
