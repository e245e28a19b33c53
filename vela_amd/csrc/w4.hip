// Products of few rows with 4-bit weights (vgemm_w4) and their layout (vgemm_w4_pack); the core is in w4_kernel.h.
#include <algorithm>

#include "dispatch_rules.h"
#include "w4.h"

namespace vk {

// ---------------------------------------------------------------- layout

// One thread per 16 bytes of a tile (a lane's share): grid.x over tiles of a matrix, grid.y over matrices.
__global__ void __launch_bounds__(256) w4_pack_kernel(int N, int K, int group, uint8_t* __restrict__ q, size_t stride, const uint8_t* __restrict__ nib, int ldn,
                                                      const uint16_t* __restrict__ scale, const uint8_t* __restrict__ zero, int lds) {
    const int KT = w4_kt(K), CT = w4_ct(N), NG = 128 / group;
    const int tile = int(blockIdx.x) * 4 + int(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (tile >= CT * KT) return;
    const int ct = tile / KT, kt = tile - ct * KT, n = ct * 16 + (lane & 15), j = lane >> 4;
    q += stride * blockIdx.y;
    const size_t row = size_t(blockIdx.y) * N + n;
    uint8_t b[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) b[i] = 0;
    if (n < N) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            unsigned v = 0;
            for (int h = 0; h < 2; ++h) {
                const int k = kt * 128 + 64 * h + (group == 32 ? 32 * (i >> 3) + 8 * j + (i & 7) : 16 * j + i);
                unsigned u = 8;
                if (k < K) u = (nib[row * ldn + (k >> 1)] >> (4 * (k & 1))) & 15u;
                else if (zero) u = zero[row * lds + min(k / group, (K - 1) / group)] & 15u;
                v |= u << (4 * h);
            }
            b[i] = uint8_t(v);
        }
    }
    uint4 w;
    w.x = b[0] | b[1] << 8 | b[2] << 16 | unsigned(b[3]) << 24;
    w.y = b[4] | b[5] << 8 | b[6] << 16 | unsigned(b[7]) << 24;
    w.z = b[8] | b[9] << 8 | b[10] << 16 | unsigned(b[11]) << 24;
    w.w = b[12] | b[13] << 8 | b[14] << 16 | unsigned(b[15]) << 24;
    reinterpret_cast<uint4*>(q + size_t(tile) * 1024)[lane] = w;
    uint16_t* s = reinterpret_cast<uint16_t*>(q + size_t(CT) * KT * 1024 + size_t(tile) * 32 * NG);
    for (int i = lane; i < 16 * NG; i += 64) {
        const int c = i / NG, g = kt * NG + i % NG, m = ct * 16 + c;
        unsigned word = 8u << 12;
        if (m < N && g * group < K) {
            const size_t at = (size_t(blockIdx.y) * N + m) * lds + g;
            word = (zero ? zero[at] & 15u : 8u) << 12 | min(unsigned(scale[at]), 4095u);
        }
        s[i] = uint16_t(word);
    }
}

// cst of column n: {m, s, b} as given and wsum = sum of (u - z) sc, |wsum| <= 32768 * 15 * 4095 < 2^31. One wave per column.
__global__ void __launch_bounds__(256) w4_cst_kernel(int N, int K, int group, int4* __restrict__ cst, const uint8_t* __restrict__ nib, int ldn,
                                                     const uint16_t* __restrict__ scale, const uint8_t* __restrict__ zero, int lds, const int32_t* __restrict__ msb) {
    const int n = int(blockIdx.x) * 4 + int(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int N16 = w4_ct(N) * 16;
    if (n >= N16) return;
    int4 c = make_int4(0, 0, 0, 0);
    if (n < N) {
        const size_t row = size_t(blockIdx.y) * N + n;
        int sum = 0;
        for (int k = lane; k < K; k += 64) {
            const int g = k / group, u = (nib[row * ldn + (k >> 1)] >> (4 * (k & 1))) & 15;
            sum += (u - (zero ? int(zero[row * lds + g] & 15) : 8)) * min(int(scale[row * lds + g]), 4095);
        }
        for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
        c = make_int4(msb[4 * row], msb[4 * row + 1], msb[4 * row + 2], sum);
    }
    if (lane == 0) cst[size_t(blockIdx.y) * N16 + n] = c;
}

hipError_t launch_w4_pack(hipStream_t st, int N, int K, int group, uint8_t* q, int4* cst, int n, const uint8_t* nib, int ldn, const uint16_t* scale,
                          const uint8_t* zero, int lds, const int32_t* msb) {
    const int tiles = w4_ct(N) * w4_kt(K);
    const size_t stride = w4_bytes(N, K, group);
    hipLaunchKernelGGL(w4_pack_kernel, dim3(cdiv(tiles, 4), n), dim3(256), 0, st, N, K, group, q, stride, nib, ldn, scale, zero, lds);
    hipLaunchKernelGGL(w4_cst_kernel, dim3(cdiv(w4_ct(N) * 16, 4), n), dim3(256), 0, st, N, K, group, cst, nib, ldn, scale, zero, lds, msb);
    return hipGetLastError();
}

// ---------------------------------------------------------------- products

// A block owns one column tile and 16 MT rows; its waves split K by tiles of 128 (wave w takes tiles w, w + waves, ...), each
// with DEPTH tiles of weights in flight, and join their sums in LDS. SRC: 0 8-bit rows, 1 planes, 2 int32 rows.
template <int MT, int SRC, int G>
__global__ void __launch_bounds__(MT == 1 ? 1024 : (MT == 2 ? 512 : 256)) w4_kernel(W4Args a) {
    constexpr int P = SRC == 0 ? 1 : 2, RT = 16 * MT, DEPTH = MT == 1 && SRC == 0 && G != 32 ? 4 : 2;
    constexpr int NG = 128 / G;
    extern __shared__ uint4 s_dyn[];
    __shared__ int s_e[SRC == 2 ? RT : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int ct = blockIdx.x, row0 = int(blockIdx.y) * RT, nrows = min(RT, a.M - row0), KT = a.w.KT;
    const uint8_t* q = a.w.q + size_t(ct) * KT * 1024;
    const uint8_t* s = a.w.s + size_t(ct) * KT * 32 * NG;

    W4Tile<G> t[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
        const int kt = wave + d * waves;
        if (kt < KT) t[d].load(q + size_t(kt) * 1024, s + size_t(kt) * 32 * NG, lane);
    }
    double acc[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[mt][r] = 0.0;

    if constexpr (SRC == 2) {
        if (int(threadIdx.x) < nrows) s_e[threadIdx.x] = rowexp_u32(a.xmax[row0 + threadIdx.x]);
        __syncthreads();
        uint8_t* lds = reinterpret_cast<uint8_t*>(s_dyn) + wave * (2 * RT * W4_LDR);
        W4Quads<RT> xq;
        const int32_t* x0 = a.x + size_t(row0) * a.ldx;
        const auto rowp = [&](int r) { return x0 + size_t(r) * a.ldx; };
        if (wave < KT) xq.load(rowp, nrows, wave * 128, a.w.K, lane);
        for (int kt = wave; kt < KT; kt += DEPTH * waves) {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                const int kd = kt + d * waves;
                if (kd < KT) {
                    wave_lds_fence();
                    xq.stage(lds, s_e, nrows, lane);
                    wave_lds_fence();
                    if (kd + waves < KT) xq.load(rowp, nrows, (kd + waves) * 128, a.w.K, lane);
                    W4Rows<2> rows[MT];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const int r = min(16 * mt + (lane & 15), nrows - 1);
                        rows[mt].template load<G>(reinterpret_cast<const int8_t*>(lds + r * W4_LDR), reinterpret_cast<const int8_t*>(lds + (RT + r) * W4_LDR), 0, 128, lane);
                    }
                    w4_tile<MT, 2, G>(t[d], rows, acc);
                    const int kn = kd + DEPTH * waves;
                    if (kn < KT) t[d].load(q + size_t(kn) * 1024, s + size_t(kn) * 32 * NG, lane);
                }
            }
        }
        __syncthreads();   // the staging area is used again below
    } else {
        const int8_t *hi[MT], *lo[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const size_t off = size_t(row0 + min(16 * mt + (lane & 15), nrows - 1)) * a.ld8;   // lanes of absent rows compute another row's sums, which nobody reads
            hi[mt] = a.hi + off;
            lo[mt] = a.lo + off;
        }
        W4Rows<P> rows[DEPTH][MT];
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int kt = wave + d * waves;
            if (kt < KT) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) rows[d][mt].template load<G>(hi[mt], lo[mt], kt * 128, a.Kp16, lane);
            }
        }
        for (int kt = wave; kt < KT; kt += DEPTH * waves) {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                const int kd = kt + d * waves;
                if (kd < KT) {
                    w4_tile<MT, P, G>(t[d], rows[d], acc);
                    const int kn = kd + DEPTH * waves;
                    if (kn < KT) {
                        t[d].load(q + size_t(kn) * 1024, s + size_t(kn) * 32 * NG, lane);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) rows[d][mt].template load<G>(hi[mt], lo[mt], kn * 128, a.Kp16, lane);
                    }
                }
            }
        }
    }

    // join the waves' sums: [wave][row tile][column pair][lane] pairs of doubles
    double2* red = reinterpret_cast<double2*>(s_dyn);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) red[((wave * MT + mt) * 2 + h) * 64 + lane] = make_double2(acc[mt][2 * h], acc[mt][2 * h + 1]);
    __syncthreads();
    for (int slot = wave; slot < 2 * MT; slot += waves) {
        const int mt = slot >> 1, h = slot & 1;
        double2 v = red[slot * 64 + lane];
        for (int w = 1; w < waves; ++w) {
            const double2 o = red[(w * MT * 2 + slot) * 64 + lane];
            v.x += o.x;
            v.y += o.y;
        }
        const int rr = 16 * mt + (lane & 15), n = ct * 16 + 4 * (lane >> 4) + 2 * h;
        const bool live = rr < nrows && n < a.w.N;
        const int r = row0 + min(rr, nrows - 1);
        const int e = SRC == 2 ? s_e[min(rr, nrows - 1)] : (a.e ? a.e[r] : 0);
        const int4 c0 = a.w.cst[n], c1 = a.w.cst[n + 1];
        int y0 = w4_requant(i64(v.x), P == 2, c0, e), y1 = w4_requant(i64(v.y), P == 2, c1, e);
        uint32_t m = 0;
        if (a.geglu) {
            y0 = geglu_exact(y0, y1, a.Lphi);
            if (live) {
                a.Y[size_t(r) * a.ldy + (n >> 1)] = y0;
                m = uabs(y0);
            }
        } else if (live) {
            const size_t at = size_t(r) * a.ldy + n;
            const bool two = n + 1 < a.w.N;
            if (a.R) {
                y0 = add_sat(y0, a.R[at]);
                if (two) y1 = add_sat(y1, a.R[at + 1]);
            }
            a.Y[at] = y0;
            if (two) a.Y[at + 1] = y1;
            m = max(uabs(y0), two ? uabs(y1) : 0u);
        }
        if (a.rowmax) {
            m = max(m, uint32_t(__shfl_xor(int(m), 16)));
            m = max(m, uint32_t(__shfl_xor(int(m), 32)));
            if (lane < 16 && live && m) atomicMax(a.rowmax + r, m);
        }
    }
}

template <int MT, int SRC, int G>
static void w4_launch(hipStream_t st, const W4Args& a, int waves) {
    constexpr int P = SRC == 0 ? 1 : 2;
    const size_t red = size_t(waves) * MT * 2 * 64 * 16, stage = SRC == 2 ? size_t(waves) * 2 * 16 * MT * W4_LDR : 0;
    hipLaunchKernelGGL((w4_kernel<MT, SRC, G>), dim3(a.w.CT, cdiv(a.M, 16 * MT)), dim3(64 * waves), std::max(red, stage), st, a);
}

template <int MT, int SRC>
static void w4_group(hipStream_t st, const W4Args& a, int waves) {
    if (a.group == 32) w4_launch<MT, SRC, 32>(st, a, waves);
    else if (a.group == 64) w4_launch<MT, SRC, 64>(st, a, waves);
    else w4_launch<MT, SRC, 128>(st, a, waves);
}

template <int MT>
static void w4_source(hipStream_t st, const W4Args& a, int waves) {
    if (a.x) w4_group<1, 2>(st, a, waves);
    else if (a.lo) w4_group<MT, 1>(st, a, waves);
    else w4_group<MT, 0>(st, a, waves);
}

hipError_t launch_w4(hipStream_t st, const W4Args& a) {
    const int MT = a.M <= 16 || a.x ? 1 : (a.M <= 32 ? 2 : 4);
    const long long blocks = (long long)a.w.CT * cdiv(a.M, 16 * MT);
    int waves = MT == 1 ? 16 : (MT == 2 ? 8 : 4);
    while (waves > 1 && (waves > a.w.KT || (waves > 4 && blocks * waves > 8192))) waves /= 2;
    if (MT == 1) w4_source<1>(st, a, waves);
    else if (MT == 2) w4_source<2>(st, a, waves);
    else w4_source<4>(st, a, waves);
    return hipGetLastError();
}

}  // namespace vk
