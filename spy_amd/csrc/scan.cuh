// Inclusive sums over lanes without LDS: shifts by 1, 2, 4, 8 inside the rows of 16 lanes, then the last lanes of rows 0 and 2, and of row 1, to the rows behind.
#pragma once

#include "common.cuh"

template <int CTRL, int ROWS> static __device__ __forceinline__ uint32_t moved(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false); }
template <int CTRL, int ROWS> static __device__ __forceinline__ unsigned long long moved(unsigned long long v) {
    return (unsigned long long)moved<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | moved<CTRL, ROWS>((uint32_t)v);
}
template <class T> static __device__ __forceinline__ T row_scan(T v) {
    v += moved<0x111, 0xF>(v);
    v += moved<0x112, 0xF>(v);
    v += moved<0x114, 0xF>(v);
    v += moved<0x118, 0xF>(v);
    return v;
}
template <class T> static __device__ __forceinline__ T wave_scan(T v) {
    v = row_scan(v);
    v += moved<0x142, 0xA>(v);
    v += moved<0x143, 0xC>(v);
    return v;
}
