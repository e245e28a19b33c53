// Device arithmetic shared by the row normalisations (norms.hip, rmsnorm.hip): exact integer division and
// square root, wave reductions, and the normalised value in its double and integer forms.
#pragma once
#include <climits>

#include "vk_common.h"

namespace vk {

// floor(a / b) for b != 0 (src/intops.cuh:18)
__device__ __forceinline__ i64 floor_div64(i64 a, i64 b) {
    i64 q = a / b;
    if (a % b != 0 && ((a < 0) != (b < 0))) --q;
    return q;
}

// e = #{k in [15, 32): m >= 2^k} for a 64-bit m (src/intops.cuh:37-38)
__device__ __forceinline__ int row_exp64(i64 m) {
    if (m < (1LL << 15)) return 0;
    if (m >= (1LL << 32)) return 17;
    return 32 - __clz(unsigned(m)) - 15;
}

// floor(sqrt(v)) for v >= 0 (0 for v <= 0): a double estimate, then exact integer corrections
__device__ __forceinline__ i64 isqrt64(i64 v) {
    if (v <= 0) return 0;
    i64 s = i64(sqrt(double(v)));
    while (s > 0 && s * s > v) --s;
    while ((s + 1) * (s + 1) <= v) ++s;
    return s;
}

// (x - mean) rounded and shifted right by e, no saturation (src/kernels.cu:197)
__device__ __forceinline__ i64 dev_shift(i64 d, int e) { return e ? ((d >> e) + ((d >> (e - 1)) & 1)) : d; }

__device__ __forceinline__ double clamp32d(double v) { return fmin(fmax(v, -2147483648.0), 2147483647.0); }

// ---------------------------------------------------------------- wave reductions (DPP)
//
// Four in-row DPP steps (lane ^ 1, lane ^ 2, the half-row mirror, the row mirror) leave every lane
// of a 16-lane row with the row's total; the four row totals are then read into scalar registers.
// Every lane of the wave must be active.
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140;

template <int CTRL>
__device__ __forceinline__ int dpp32(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false); }
template <int CTRL>
__device__ __forceinline__ double dppf64(double v) {
    const u64 b = __builtin_bit_cast(u64, v);
    const unsigned lo = unsigned(dpp32<CTRL>(int(b))), hi = unsigned(dpp32<CTRL>(int(b >> 32)));
    return __builtin_bit_cast(double, (u64(hi) << 32) | lo);
}
__device__ __forceinline__ double readlanef64(double v, int l) {
    const u64 b = __builtin_bit_cast(u64, v);
    const unsigned lo = unsigned(__builtin_amdgcn_readlane(int(b), l)), hi = unsigned(__builtin_amdgcn_readlane(int(b >> 32), l));
    return __builtin_bit_cast(double, (u64(hi) << 32) | lo);
}

// sum of integer-valued doubles whose partial sums stay below 2^53 (exact in any order)
__device__ __forceinline__ double wave_sumf64(double v) {
    v += dppf64<DPP_XOR1>(v);
    v += dppf64<DPP_XOR2>(v);
    v += dppf64<DPP_HALF_MIRROR>(v);
    v += dppf64<DPP_MIRROR>(v);
    return (readlanef64(v, 0) + readlanef64(v, 16)) + (readlanef64(v, 32) + readlanef64(v, 48));
}
__device__ __forceinline__ uint32_t wave_umax32(uint32_t v) {
    v = max(v, uint32_t(dpp32<DPP_XOR1>(int(v))));
    v = max(v, uint32_t(dpp32<DPP_XOR2>(int(v))));
    v = max(v, uint32_t(dpp32<DPP_HALF_MIRROR>(int(v))));
    v = max(v, uint32_t(dpp32<DPP_MIRROR>(int(v))));
    const uint32_t a = uint32_t(__builtin_amdgcn_readlane(int(v), 0)), b = uint32_t(__builtin_amdgcn_readlane(int(v), 16));
    const uint32_t c = uint32_t(__builtin_amdgcn_readlane(int(v), 32)), d = uint32_t(__builtin_amdgcn_readlane(int(v), 48));
    return max(max(a, b), max(c, d));
}

// ---------------------------------------------------------------- the normalised value
//
// yy = floor((d 2^s + sd) / (2 sd)) with d = x - mean, s = 25 - e (src/kernels.cu:217,296,380) equals
// floor(d K + 1/2) for the exact K = 2^(s - 1) / sd. In double, with d exact (|mean| < 2^36) and K
// correctly rounded, t = fma(d, K, 1/2) differs from d K + 1/2 by at most 2^-52 (|t| + 1): below 2^-30
// for |t| < 2^21, so floor(t) is exact whenever t lies at least 2^-16 from an integer. Then with
// |yy| < 2^21 and an int32 g, yy g is below 2^52 and rshr(yy g, 16) = floor(yy g 2^-16 + 1/2) is one
// exact FMA, a scaling by 2^-16 and a floor, and the saturations and the add of beta are exact double
// operations. The other elements (about one in 2^15 on any data, and those with |yy| >= 2^21), and
// every group whose record is outside the double form's range, take the exact integer form.
struct NormK {
    double mean;   // NaN: every element takes the exact form
    double K;      // 0 for sd = 0 (yy = 0)
};

__device__ __forceinline__ NormK norm_const(i64 mean, int e, i64 sd) {
    const bool ok = mean > -(1LL << 36) && mean < (1LL << 36) && e >= 0 && e <= 25 && sd >= 0 && sd < (1LL << 52);
    NormK k;
    k.mean = ok ? double(mean) : __builtin_nan("");
    k.K = (ok && sd > 0) ? (e <= 24 ? double(1 << (24 - e)) : 0.5) / double(sd) : 0.0;
    return k;
}

// the exact integer form (0 for sd = 0); the shift and the additions wrap in 64 bits
__device__ __forceinline__ i64 norm_exact(int x, i64 mean, int e, i64 sd) {
    if (sd == 0) return 0;
    const i64 d = i64(u64(i64(x)) - u64(mean));
    return floor_div64(i64((u64(d) << (25 - e)) + u64(sd)), i64(2 * u64(sd)));
}

// the general form: yy g wraps in 64 bits (src/kernels.cu:218)
__device__ __forceinline__ int norm_affine64(i64 yy, i64 g, i64 beta) {
    return int(sat32(i64(u64(rshr(i64(u64(yy) * u64(g)), 16)) + u64(beta))));
}

// the normalised value's double form (see NormK): f = floor(t), exact when ok
__device__ __forceinline__ double norm_floor(int x, const NormK& k, bool& ok) {
    const double t = fma(double(x) - k.mean, k.K, 0.5);
    const double f = floor(t);
    ok = fabs(t) < 0x1p21 && fabs((t - f) - 0.5) <= 0.5 - 0x1p-16;   // false for NaN
    return f;
}
// sat32(sat32(rshr(yy g, 16)) + beta) in double: with |yy g| < 2^52, (yy 2^-16) g + 1/2 is exact in one FMA
__device__ __forceinline__ double affine_d(double yy, int g, int beta) {
    return clamp32d(clamp32d(floor(fma(yy * 0x1p-16, double(g), 0.5))) + double(beta));
}

}  // namespace vk
