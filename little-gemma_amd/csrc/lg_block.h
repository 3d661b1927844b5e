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
// The largest of the lanes' numbers (0 and up): of each sixteen in the last of them, and of all
template <typename T>
__device__ __forceinline__ T lg_row_max(T v) {
    auto top = [&](T u) { if (u > v) v = u; };
    top(lg_shift<0x111, 0xF>(v)); top(lg_shift<0x112, 0xF>(v)); top(lg_shift<0x114, 0xF>(v)); top(lg_shift<0x118, 0xF>(v));
    return v;
}
template <typename T>
__device__ __forceinline__ T lg_wave_max(T v) {
    auto top = [&](T u) { if (u > v) v = u; };
    v = lg_row_max(v);
    top(lg_shift<0x142, 0xA>(v)); top(lg_shift<0x143, 0xC>(v));
    return lg_last_lane(v);
}
// A lane's number, the same lane for the whole wavefront
__device__ __forceinline__ uint32_t lg_lane(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ lg_u64 lg_lane(lg_u64 v, int lane) { return (lg_u64)lg_lane((uint32_t)(v >> 32), lane) << 32 | lg_lane((uint32_t)v, lane); }

// Over a workgroup of NT <= 1024 threads; `part` is LDS of NT / 64 words.  A barrier before its first use, for the caller's earlier reads, is in here.
// A wavefront reads the others' parts with one load, a lane each, and runs over them by primitives: with a load per part from every wavefront the LDS is
// what 16 of them wait for.
template <int NT, typename T>
__device__ __forceinline__ T lg_block_run(T v, T *part, T *total) {           // inclusive
    constexpr int NW = NT / 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    v = lg_wave_run(v);
    __syncthreads();
    if (lane == 63) part[wave] = v;
    __syncthreads();
    T x = lane < NW ? part[lane] : 0;
    x += lg_shift<0x111, 0xF>(x);
    x += lg_shift<0x112, 0xF>(x);
    x += lg_shift<0x114, 0xF>(x);
    x += lg_shift<0x118, 0xF>(x);
    *total = lg_lane(x, NW - 1);
    return wave ? v + lg_lane(x, wave - 1) : v;
}
template <int NT, typename T>
__device__ __forceinline__ T lg_block_sum(T v, T *part) {
    T all;
    lg_block_run<NT>(v, part, &all);
    return all;
}
template <int NT, typename T>
__device__ __forceinline__ T lg_block_max(T v, T *part) {
    v = lg_wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return lg_wave_max((threadIdx.x & 63) < NT / 64 ? part[threadIdx.x & 63] : 0);
}
// Two at once
template <int NT, typename T>
__device__ __forceinline__ void lg_block_max2(T &u, T &v, T *part) {          // part: NT / 32 words
    constexpr int NW = NT / 64;
    const int lane = threadIdx.x & 63;
    u = lg_wave_max(u); v = lg_wave_max(v);
    __syncthreads();
    if (lane == 0) { part[threadIdx.x >> 6] = u; part[NW + (threadIdx.x >> 6)] = v; }
    __syncthreads();
    u = lg_wave_max(lane < NW ? part[lane] : 0);
    v = lg_wave_max(lane < NW ? part[NW + lane] : 0);
}
// Three running sums at once (exclusive), their totals in `all`; part: 3 NT / 64 words
template <int NT>
__device__ __forceinline__ void lg_block_run3(lg_u64 (&v)[3], lg_u64 (&all)[3], lg_u64 *part) {
    constexpr int NW = NT / 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    lg_u64 own[3];
    #pragma unroll
    for (int k = 0; k < 3; ++k) { own[k] = v[k]; v[k] = lg_wave_run(v[k]); }
    __syncthreads();
    if (lane == 63)
        #pragma unroll
        for (int k = 0; k < 3; ++k) part[k * NW + wave] = v[k];
    __syncthreads();
    #pragma unroll
    for (int k = 0; k < 3; ++k) {
        const lg_u64 x = lg_wave_run(lane < NW ? part[k * NW + lane] : 0);
        all[k] = lg_lane(x, NW - 1);
        v[k] += (wave ? lg_lane(x, wave - 1) : 0) - own[k];
    }
}
