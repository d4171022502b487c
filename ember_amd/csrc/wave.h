// wave.h -- sums and maxima over a wave's 64 lanes in register moves (DPP), and
// values passed between workgroups of a launch (not part of the public ABI).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ember {

// The value of a lane further down; lanes that have none get `none`.
template <int CTRL, int ROWS, class V>
__device__ __forceinline__ V lane_below(V v, V none)
{
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}

// f over the lanes up to this one; `none` is f's neutral value.
template <class V, class F>
__device__ __forceinline__ V wave_scan(V v, V none, F f)
{
    v = f(v, lane_below<0x111, 0xf>(v, none));  // from 1, 2, 4 and 8 lanes below, within 16
    v = f(v, lane_below<0x112, 0xf>(v, none));
    v = f(v, lane_below<0x114, 0xf>(v, none));
    v = f(v, lane_below<0x118, 0xf>(v, none));
    v = f(v, lane_below<0x142, 0xa>(v, none));  // the last lane of the 16 below, and of the 32 below
    v = f(v, lane_below<0x143, 0xc>(v, none));
    return v;
}
template <class V, class F>
__device__ __forceinline__ V wave_all(V v, V none, F f)
{
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_scan(v, none, f)), 63));
}
template <class V>
__device__ __forceinline__ V wave_scan_sum(V v)
{
    return wave_scan(v, V(0), [](V a, V b) { return a + b; });
}
template <class V>
__device__ __forceinline__ V wave_sum(V v)
{
    return wave_all(v, V(0), [](V a, V b) { return a + b; });
}
__device__ __forceinline__ float wave_max(float v)
{
    return wave_all(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}

// f over the 16 neighbouring lanes that a lane is of, the same in each of them.
template <class F>
__device__ __forceinline__ float row_all(float v, F f)
{
    v = f(v, lane_below<0x121, 0xf>(v, v));  // from 1, 2, 4 and 8 lanes below, around the 16
    v = f(v, lane_below<0x122, 0xf>(v, v));
    v = f(v, lane_below<0x124, 0xf>(v, v));
    return f(v, lane_below<0x128, 0xf>(v, v));
}
// f of a lane's value and that of the lane 16 (32) from it, in both.
template <class F>
__device__ __forceinline__ float across_16(float v, F f)
{
    const auto x = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    return f(__builtin_bit_cast(float, (unsigned)x[0]), __builtin_bit_cast(float, (unsigned)x[1]));
}
template <class F>
__device__ __forceinline__ float across_32(float v, F f)
{
    const auto x = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    return f(__builtin_bit_cast(float, (unsigned)x[0]), __builtin_bit_cast(float, (unsigned)x[1]));
}

// What the lanes of a wave have written to LDS is there for all of them.
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
}

// Stores and loads at device scope pass the L2s by: the workgroups of a launch
// are on XCDs with an L2 each.  What a workgroup has put is there for others once
// its waves have waited for their stores (wait_vmem) and met at a barrier; a
// release fence would write a whole L2 back.
__device__ __forceinline__ void put8(void *p, uint64_t v)
{
    __hip_atomic_store((uint64_t *)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t get8(const void *p)
{
    return __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Adds one to *done, which `of` workgroups do; true for the last, which sets
// it back to 0.  One thread of a workgroup.
__device__ __forceinline__ bool last_of(unsigned *done, unsigned of)
{
    if (__hip_atomic_fetch_add(done, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != of - 1) return false;
    __hip_atomic_store(done, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}

}  // namespace ember
