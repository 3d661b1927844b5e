// lg_block.h — sums, running sums and extremes over a wavefront and a workgroup, of whole numbers: the same whatever the order.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

typedef unsigned long long lg_u64;

// A lane's neighbour by data-parallel primitives, 0 where there is none: 0x111.. row_shr 1.., 0x142 row_bcast 15 (into rows 1 and 3), 0x143 row_bcast 31 (into rows 2 and 3)
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lg_shift(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ lg_u64 lg_shift(lg_u64 v) { return (lg_u64)lg_shift<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | lg_shift<CTRL, ROWS>((uint32_t)v); }
// Inclusive running sum over the lanes; the last lane has the wavefront's sum
template <typename T>
__device__ __forceinline__ T lg_wave_run(T v) {
    v += lg_shift<0x111, 0xF>(v);
    v += lg_shift<0x112, 0xF>(v);
    v += lg_shift<0x114, 0xF>(v);
    v += lg_shift<0x118, 0xF>(v);
    v += lg_shift<0x142, 0xA>(v);
    v += lg_shift<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ uint32_t lg_last_lane(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, 63); }
__device__ __forceinline__ lg_u64 lg_last_lane(lg_u64 v) { return (lg_u64)lg_last_lane((uint32_t)(v >> 32)) << 32 | lg_last_lane((uint32_t)v); }
template <typename T>
__device__ __forceinline__ T lg_wave_total(T v) { return lg_last_lane(lg_wave_run(v)); }
// The largest of the lanes' numbers (0 and up)
__device__ __forceinline__ uint32_t lg_wave_max(uint32_t v) {
    auto top = [&](uint32_t u) { if (u > v) v = u; };
    top(lg_shift<0x111, 0xF>(v)); top(lg_shift<0x112, 0xF>(v)); top(lg_shift<0x114, 0xF>(v));
    top(lg_shift<0x118, 0xF>(v)); top(lg_shift<0x142, 0xA>(v)); top(lg_shift<0x143, 0xC>(v));
    return lg_last_lane(v);
}

// Over a workgroup of NT threads; `part` is LDS of NT / 64 words.  A barrier before its first use by the caller's earlier reads is in here.
template <int NT, typename T>
__device__ __forceinline__ T lg_block_run(T v, T *part, T *total) {           // inclusive
    const int wave = threadIdx.x >> 6;
    v = lg_wave_run(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) part[wave] = v;
    __syncthreads();
    T before = 0, all = 0;
    #pragma unroll
    for (int w = 0; w < NT / 64; ++w) { const T p = part[w]; if (w < wave) before += p; all += p; }
    *total = all;
    return v + before;
}
template <int NT, typename T>
__device__ __forceinline__ T lg_block_sum(T v, T *part) {
    T all;
    lg_block_run<NT>(v, part, &all);
    return all;
}
template <int NT>
__device__ __forceinline__ uint32_t lg_block_max(uint32_t v, uint32_t *part) {
    v = lg_wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    #pragma unroll
    for (int w = 0; w < NT / 64; ++w) if (part[w] > v) v = part[w];
    return v;
}
