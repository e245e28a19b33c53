// Reductions over a wave of 64 lanes without LDS: DPP within rows of sixteen, then the permlane swaps. Every lane must be active.
#pragma once
#include "norm_math.h"

namespace vk {

// over the four lanes of equal place in their rows of sixteen
__device__ __forceinline__ int across_max(int v) {
    auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(int(a[0]), int(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(int(b[0]), int(b[1]));
}
__device__ __forceinline__ int across_sum(int v) {
    auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = int(a[0] + a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return int(b[0] + b[1]);
}

// over a row of sixteen lanes
__device__ __forceinline__ unsigned row_max(unsigned v) {
    v = max(v, unsigned(dpp32<DPP_XOR1>(int(v))));
    v = max(v, unsigned(dpp32<DPP_XOR2>(int(v))));
    v = max(v, unsigned(dpp32<DPP_HALF_MIRROR>(int(v))));
    return max(v, unsigned(dpp32<DPP_MIRROR>(int(v))));
}
__device__ __forceinline__ int row_sum(int v) {
    v += dpp32<DPP_XOR1>(v);
    v += dpp32<DPP_XOR2>(v);
    v += dpp32<DPP_HALF_MIRROR>(v);
    return v + dpp32<DPP_MIRROR>(v);
}

__device__ __forceinline__ int wave_max(int v) {
    v = max(v, dpp32<DPP_XOR1>(v));
    v = max(v, dpp32<DPP_XOR2>(v));
    v = max(v, dpp32<DPP_HALF_MIRROR>(v));
    v = max(v, dpp32<DPP_MIRROR>(v));
    return across_max(v);
}
__device__ __forceinline__ int wave_sum(int v) { return across_sum(row_sum(v)); }

template <int CTRL>
__device__ __forceinline__ i64 dpp64(i64 v) { return i64(u64(unsigned(dpp32<CTRL>(int(v)))) | u64(unsigned(dpp32<CTRL>(int(v >> 32)))) << 32); }
template <class F>
__device__ __forceinline__ i64 wave_fold64(i64 v, F f) {
    v = f(v, dpp64<DPP_XOR1>(v));
    v = f(v, dpp64<DPP_XOR2>(v));
    v = f(v, dpp64<DPP_HALF_MIRROR>(v));
    v = f(v, dpp64<DPP_MIRROR>(v));
    const auto l16 = __builtin_amdgcn_permlane16_swap(int(v), int(v), false, false), h16 = __builtin_amdgcn_permlane16_swap(int(v >> 32), int(v >> 32), false, false);
    v = f(i64(u64(l16[0]) | u64(h16[0]) << 32), i64(u64(l16[1]) | u64(h16[1]) << 32));
    const auto l32 = __builtin_amdgcn_permlane32_swap(int(v), int(v), false, false), h32 = __builtin_amdgcn_permlane32_swap(int(v >> 32), int(v >> 32), false, false);
    return f(i64(u64(l32[0]) | u64(h32[0]) << 32), i64(u64(l32[1]) | u64(h32[1]) << 32));
}
__device__ __forceinline__ i64 wave_sum64(i64 v) {
    return wave_fold64(v, [](i64 a, i64 b) { return a + b; });
}
__device__ __forceinline__ i64 wave_max64(i64 v) {
    return wave_fold64(v, [](i64 a, i64 b) { return a > b ? a : b; });
}

// inclusive running sum over the wave: within rows, then the rows' totals handed on
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);   // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast 15 into rows 1 and 3, then 31 into 2 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

}  // namespace vk
