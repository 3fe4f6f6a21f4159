// vs_wave.h -- reductions over a wave in its vector registers.
#pragma once

#include "vs_internal.h"

namespace vs {

// Data-parallel primitives: a shuffle through LDS takes several times as long.
// Where the source lane is out of range `same` is taken, which changes nothing.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t dpp(uint32_t same, uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)same, (int)x, CTRL, ROWS, 0xf, false);
}
constexpr int kSwap1 = 0xB1, kSwap2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140;
constexpr int kBcast15 = 0x142, kBcast31 = 0x143;

// The largest x of the wave, in every lane (NaNs are passed over).
__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, float_of(dpp<kSwap1>(bits_of(x), bits_of(x))));
    x = fmaxf(x, float_of(dpp<kSwap2>(bits_of(x), bits_of(x))));
    x = fmaxf(x, float_of(dpp<kHalfMirror>(bits_of(x), bits_of(x))));
    x = fmaxf(x, float_of(dpp<kMirror>(bits_of(x), bits_of(x))));
    const float a = float_of(__builtin_amdgcn_readlane(bits_of(x), 0));
    const float b = float_of(__builtin_amdgcn_readlane(bits_of(x), 16));
    const float c = float_of(__builtin_amdgcn_readlane(bits_of(x), 32));
    const float d = float_of(__builtin_amdgcn_readlane(bits_of(x), 48));
    return fmaxf(fmaxf(a, b), fmaxf(c, d));
}

// Inclusive prefix sum over the lanes.
__device__ __forceinline__ int prefix_sum(int x) {
    x += (int)dpp<0x111>(0, x);            // one lane up within rows of 16, then 2, 4, 8
    x += (int)dpp<0x112>(0, x);
    x += (int)dpp<0x114>(0, x);
    x += (int)dpp<0x118>(0, x);
    x += (int)dpp<kBcast15, 0xa>(0, x);    // rows 1 and 3 take the sum of the one before
    x += (int)dpp<kBcast31, 0xc>(0, x);    // the upper half that of the lower
    return x;
}

// Of all lanes; the sum fits 32 bits.
__device__ __forceinline__ uint32_t wave_sum(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_readlane(prefix_sum((int)x), 63);
}

// The same, where a sum may pass 32 bits: it stays at the largest number then.
__device__ __forceinline__ uint32_t prefix_sum_sat(uint32_t x) {
    x = __builtin_elementwise_add_sat(x, dpp<0x111>(0, x));
    x = __builtin_elementwise_add_sat(x, dpp<0x112>(0, x));
    x = __builtin_elementwise_add_sat(x, dpp<0x114>(0, x));
    x = __builtin_elementwise_add_sat(x, dpp<0x118>(0, x));
    x = __builtin_elementwise_add_sat(x, dpp<kBcast15, 0xa>(0, x));
    x = __builtin_elementwise_add_sat(x, dpp<kBcast31, 0xc>(0, x));
    return x;
}

constexpr int kPlan = 1024;  // threads of plans that are made by one workgroup

// Exclusive prefix sum of x over the workgroup's kPlan threads; *total its sum.
__device__ __forceinline__ int block_scan(int x, int *total, int *lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int incl = prefix_sum(x);
    __syncthreads();
    if (lane == 63) lds[wave] = incl;
    __syncthreads();
    // every wave sums the waves' totals for itself
    const int w = prefix_sum(lane < kPlan / 64 ? lds[lane] : 0);
    *total = __builtin_amdgcn_readlane(w, 63);
    return incl - x + (wave ? __builtin_amdgcn_readlane(w, wave - 1) : 0);
}

// The same with sums that stay at the largest number; the prefixes hold where
// the total is below it.
__device__ __forceinline__ uint32_t block_scan_sat(uint32_t x, uint32_t *total, int *lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t incl = prefix_sum_sat(x);
    __syncthreads();
    if (lane == 63) lds[wave] = (int)incl;
    __syncthreads();
    const uint32_t w = prefix_sum_sat(lane < kPlan / 64 ? (uint32_t)lds[lane] : 0);
    *total = (uint32_t)__builtin_amdgcn_readlane((int)w, 63);
    return incl - x + (wave ? (uint32_t)__builtin_amdgcn_readlane((int)w, wave - 1) : 0);
}

}  // namespace vs
