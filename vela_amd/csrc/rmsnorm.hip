// Root-mean-square norm of rows with the residual's addition, in the row normalisations' integer arithmetic, and
// 8-bit rows (or the int16 view) of the result for the products that read it:
//   h = sat32(x + r), ex = max(0, row_exp(max |h|) - 5), ss = sum rshr(h, ex)^2, var = floor(ss / C),
//   sd = isqrt((var + eps) << 16) with eps = floor((2^(32 - 2 ex) + den / 2) / den),
//   yy = floor((h 2^(25 - ex) + sd) / 2 sd), y = sat32(rshr(yy g, 16)), m = max |y|,
//   e = #{k in [7, 32): m >= 2^k}, q = clamp(rshr(y, e), -127, 127)     (the int16 view: 15 and 32767)
//
// A value moves 13 bytes (x, r and h in 32 bits, q in 8) and takes about twenty double operations, so long inputs are
// bound by memory (4096 x 4096: 42.0 us, 5.2 TB/s) and few rows by the latency of the three reductions that follow one another (max |h|, ss, max |y|). A
// row stays in registers from its one read on. The arithmetic is exact in double as for LayerNorm (see NormK): a shifted
// value is at most 2^20 in magnitude, ss at most C 2^40 <= 2^53 for C <= 8192, and floor(ss / C) follows from the
// correctly rounded quotient, whose error (below 2^-13) is smaller than the 1 / C gap of a non-integer quotient to the next integer.
#include <climits>

#include "norm_math.h"
#include "vk_common.h"

namespace vk {

// eps for every shift ex (0..12), computed on the host from den
struct RmsEps {
    long long v[13];
};

struct RmsArgs {
    const int32_t *X, *R;
    int M, C;
    const int32_t* g;
    int32_t* H;
    int8_t *hi, *lo;
    int32_t* e;
    int Kp;
    RmsEps eps;
};

// TR threads per row (64: four rows in a block of four waves, else one row a block), NV channel quads per thread,
// VIEW: the int16 view instead of 8-bit rows
template <int TR, int NV, bool VIEW>
__global__ void __launch_bounds__(TR < 256 ? 256 : TR) rmsnorm_kernel(RmsArgs a) {
    touch_args<int(sizeof(RmsArgs))>();
    constexpr int NW = TR / 64;
    __shared__ uint32_t s_max[NW];
    __shared__ double s_sum[NW];
    __shared__ uint32_t s_ymax[NW];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int tr = TR == 64 ? lane : int(threadIdx.x);
    const int row = TR == 64 ? int(blockIdx.x) * 4 + wave : int(blockIdx.x);
    if (TR == 64 && row >= a.M) return;   // no barrier follows in this form
    const int Q = a.C >> 2;
    const int4* x = reinterpret_cast<const int4*>(a.X + size_t(row) * a.C);
    int h[NV][4];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int q4 = tr + TR * j;
        const int4 v = x[q4 < Q ? q4 : 0];
        h[j][0] = v.x; h[j][1] = v.y; h[j][2] = v.z; h[j][3] = v.w;
    }
    int4 g[NV];   // the gains, on their way during the reductions: 4096 x 4096 46.0 -> 42.0 us
#pragma unroll
    for (int j = 0; j < NV; ++j) g[j] = reinterpret_cast<const int4*>(a.g)[tr + TR * j < Q ? tr + TR * j : 0];
    if (a.R) {
        const int4* r = reinterpret_cast<const int4*>(a.R + size_t(row) * a.C);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int q4 = tr + TR * j;
            const int4 v = r[q4 < Q ? q4 : 0];
            h[j][0] = add_sat(h[j][0], v.x); h[j][1] = add_sat(h[j][1], v.y);
            h[j][2] = add_sat(h[j][2], v.z); h[j][3] = add_sat(h[j][3], v.w);
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int q4 = tr + TR * j;
        if (q4 < Q) m = max(m, max(max(uabs(h[j][0]), uabs(h[j][1])), max(uabs(h[j][2]), uabs(h[j][3]))));
    }
    m = wave_umax32(m);
    if constexpr (NW > 1) {
        if (lane == 0) s_max[wave] = m;
        __syncthreads();
        m = s_max[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) m = max(m, s_max[w]);
    }
    const int ex = max(0, row_exp64(i64(m)) - 5);
    const double sc = double(1 << (12 - ex)) * 0x1p-12;   // 2^-ex (ex <= 12)
    double ss = 0.0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const bool in = tr + TR * j < Q;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const double dd = floor(fma(double(h[j][k]), sc, 0.5));
            ss = in ? fma(dd, dd, ss) : ss;
        }
    }
    ss = wave_sumf64(ss);
    if constexpr (NW > 1) {
        if (lane == 0) s_sum[wave] = ss;
        __syncthreads();
        ss = s_sum[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) ss += s_sum[w];
    }
    const i64 sd = isqrt64(i64(u64(i64(floor(ss / double(a.C))) + a.eps.v[ex]) << 16));
    const NormK kk = norm_const(0, ex, sd);
    uint32_t ym = 0;
    int y[NV][4];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int q4 = tr + TR * j;
        const bool sl = q4 < Q;
        const int g4[4] = {g[j].x, g[j].y, g[j].z, g[j].w};
        unsigned slow = 0;   // bit k: element k needs the exact form
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            bool ok;
            const double f = norm_floor(h[j][k], kk, ok);
            y[j][k] = int(clamp32d(floor(fma(f * 0x1p-16, double(g4[k]), 0.5))));
            slow |= (sl && !ok) ? 1u << k : 0u;
        }
        if (__builtin_amdgcn_ballot_w64(slow != 0)) {
            while (slow) {
                const int k = __builtin_ctz(slow);
                slow &= slow - 1;
                int hk = 0, gk = 0;
#pragma unroll
                for (int k2 = 0; k2 < 4; ++k2) {
                    hk = k == k2 ? h[j][k2] : hk;
                    gk = k == k2 ? g4[k2] : gk;
                }
                const int r = norm_affine64(norm_exact(hk, 0, ex, sd), gk, 0);
#pragma unroll
                for (int k2 = 0; k2 < 4; ++k2) y[j][k2] = k == k2 ? r : y[j][k2];
            }
        }
        if (sl) ym = max(ym, max(max(uabs(y[j][0]), uabs(y[j][1])), max(uabs(y[j][2]), uabs(y[j][3]))));
    }
    ym = wave_umax32(ym);
    if constexpr (NW > 1) {
        if (lane == 0) s_ymax[wave] = ym;
        __syncthreads();
        ym = s_ymax[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) ym = max(ym, s_ymax[w]);
    }
    const int e = VIEW ? rowexp_u32(ym) : (ym ? max(0, 32 - __clz(ym) - 7) : 0);
    if (tr == 0) a.e[row] = e;
    unsigned* ph = reinterpret_cast<unsigned*>(a.hi + size_t(row) * a.Kp);
    unsigned* pl = VIEW ? reinterpret_cast<unsigned*>(a.lo + size_t(row) * a.Kp) : nullptr;
    int4* po = a.H ? reinterpret_cast<int4*>(a.H + size_t(row) * a.C) : nullptr;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int q4 = tr + TR * j;
        if (q4 >= Q) continue;
        int q[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (VIEW) q[k] = quant16_32(y[j][k], e);
            else q[k] = min(max(e ? ((y[j][k] >> e) + ((y[j][k] >> (e - 1)) & 1)) : y[j][k], -127), 127);
        }
        if constexpr (VIEW) {
            ph[q4] = __builtin_amdgcn_perm(unsigned(q[1]), unsigned(q[0]), 0x0c0c0501u) | __builtin_amdgcn_perm(unsigned(q[3]), unsigned(q[2]), 0x05010c0cu);
            pl[q4] = (__builtin_amdgcn_perm(unsigned(q[1]), unsigned(q[0]), 0x0c0c0400u) | __builtin_amdgcn_perm(unsigned(q[3]), unsigned(q[2]), 0x04000c0cu)) ^ 0x80808080u;
        } else {
            ph[q4] = __builtin_amdgcn_perm(unsigned(q[1]), unsigned(q[0]), 0x0c0c0400u) | __builtin_amdgcn_perm(unsigned(q[3]), unsigned(q[2]), 0x04000c0cu);
        }
        if (po) po[q4] = make_int4(h[j][0], h[j][1], h[j][2], h[j][3]);
    }
    for (int q4 = Q + tr; q4 < (a.Kp >> 2); q4 += TR) {   // pad columns hold the value 0
        ph[q4] = 0u;
        if constexpr (VIEW) pl[q4] = 0x80808080u;
    }
}

template <int TR, int NV>
static void rmsnorm_launch(hipStream_t st, const RmsArgs& a) {
    const dim3 grid(TR == 64 ? unsigned((a.M + 3) / 4) : unsigned(a.M)), block(TR < 256 ? 256 : TR);
    if (a.lo) hipLaunchKernelGGL((rmsnorm_kernel<TR, NV, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((rmsnorm_kernel<TR, NV, false>), grid, block, 0, st, a);
}

hipError_t launch_rmsnorm_q(hipStream_t st, const int32_t* X, const int32_t* R, int M, int C, const int32_t* g, i64 den, int32_t* H, int8_t* hi, int8_t* lo,
                            int32_t* e, int Kp) {
    RmsArgs a{X, R, M, C, g, H, hi, lo, e, Kp, {}};
    for (int ex = 0; ex < 13; ++ex) a.eps.v[ex] = ((1LL << (32 - 2 * ex)) + den / 2) / den;
    // Up to 1024 values a row is a wave's, up to 4096 a block's of 256 threads, wider ones of 512 (4096 x 8192: 83.8 us, 5.2 TB/s, 93.0 with 256
    // threads of eight quads; 37 x 5120: 6.3, 7.1 with 256, 6.4 with 1024)
    const int Q = C / 4;
    if (Q <= 64) rmsnorm_launch<64, 1>(st, a);
    else if (Q <= 128) rmsnorm_launch<64, 2>(st, a);
    else if (Q <= 256) rmsnorm_launch<64, 4>(st, a);
    else if (Q <= 512) rmsnorm_launch<256, 2>(st, a);
    else if (Q <= 1024) rmsnorm_launch<256, 4>(st, a);
    else rmsnorm_launch<512, 4>(st, a);
    return hipGetLastError();
}

}  // namespace vk
