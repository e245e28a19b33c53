// Products of few rows with 4-bit weights (vgemm_w4) and their layout (vgemm_w4_pack); the core is in w4_kernel.h.
#include <algorithm>

#include "dispatch_rules.h"
#include "w4.h"

namespace vk {

// ---------------------------------------------------------------- layout

// A block per column tile, a wave every fourth of its tiles of K, a lane its 16 bytes of the tile: four pieces of eight nibbles, piece
// (h, i) half h of bytes 8 i and on. The column constants' wsum = sum of (u - z) sc goes along: |wsum| <= 32768 * 15 * 4095 < 2^31.
// 4096 x 22016 with groups of 128: 87 us (a thread a byte, the sums by a second kernel: 173 + 111 us).
template <int G>
__global__ void __launch_bounds__(256) w4_pack_kernel(int N, int K, uint8_t* __restrict__ q, size_t stride, int4* __restrict__ cst, const uint8_t* __restrict__ nib, int ldn,
                                                      const uint16_t* __restrict__ scale, const uint8_t* __restrict__ zero, int lds, const int32_t* __restrict__ msb) {
    constexpr int NG = 128 / G;
    __shared__ int s_sum[4][16];
    const int KT = w4_kt(K), CT = w4_ct(N), ct = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = ct * 16 + (lane & 15), j = lane >> 4;
    q += stride * blockIdx.y;
    const size_t row = size_t(blockIdx.y) * N + n;
    const auto zero_of = [&](int g) { return zero ? unsigned(zero[row * lds + g] & 15) : 8u; };
    const auto scale_of = [&](int g) { return min(unsigned(scale[row * lds + g]), 4095u); };
    int sum = 0;
    for (int kt = wave; kt < KT; kt += 4) {
        unsigned x[2][2] = {{0, 0}, {0, 0}};   // a piece's nibbles in order
        if (n < N) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int k = kt * 128 + 64 * h + (G == 32 ? 32 * i + 8 * j : 16 * j + 8 * i);
                    const int g = min(k, K - 1) / G;
                    const unsigned z = zero_of(g);
                    if (k + 8 <= K) {
                        __builtin_memcpy(&x[h][i], nib + row * ldn + (k >> 1), 4);   // at any address
                    } else {
                        for (int e = 0; e < 8; ++e) {   // past the row's end: the zero point
                            const unsigned u = k + e < K ? (nib[row * ldn + ((k + e) >> 1)] >> (4 * (e & 1))) & 15u : z;
                            x[h][i] |= u << (4 * e);
                        }
                    }
                    const int s = __builtin_amdgcn_udot4(x[h][i] & 0x0f0f0f0fu, 0x01010101u, __builtin_amdgcn_udot4(x[h][i] >> 4 & 0x0f0f0f0fu, 0x01010101u, 0u, false), false);
                    sum += (s - 8 * int(z)) * int(scale_of(g));
                }
            }
        }
        uint4 w;
        unsigned* wp = &w.x;
#pragma unroll
        for (int i = 0; i < 2; ++i) {   // byte b of a piece: nibble b of both halves
            const unsigned even = (x[0][i] & 0x0f0f0f0fu) | (x[1][i] << 4 & 0xf0f0f0f0u), odd = (x[0][i] >> 4 & 0x0f0f0f0fu) | (x[1][i] & 0xf0f0f0f0u);
            wp[2 * i] = __builtin_amdgcn_perm(odd, even, 0x05010400u);
            wp[2 * i + 1] = __builtin_amdgcn_perm(odd, even, 0x07030602u);
        }
        const size_t tile = size_t(ct) * KT + kt;
        reinterpret_cast<uint4*>(q + tile * 1024)[lane] = w;
        uint16_t* words = reinterpret_cast<uint16_t*>(q + size_t(CT) * KT * 1024 + tile * 32 * NG);
        if (j < NG) {   // column lane & 15, group j of the tile
            const int g = kt * NG + j;
            words[(lane & 15) * NG + j] = uint16_t(n < N && g * G < K ? zero_of(g) << 12 | scale_of(g) : 8u << 12);
        }
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (lane < 16) s_sum[wave][lane] = sum;
    __syncthreads();
    if (threadIdx.x < 16) {
        const int all = s_sum[0][lane] + s_sum[1][lane] + s_sum[2][lane] + s_sum[3][lane];
        cst[size_t(blockIdx.y) * CT * 16 + n] = n < N ? make_int4(msb[4 * row], msb[4 * row + 1], msb[4 * row + 2], all) : make_int4(0, 0, 0, 0);
    }
}

hipError_t launch_w4_pack(hipStream_t st, int N, int K, int group, uint8_t* q, int4* cst, int n, const uint8_t* nib, int ldn, const uint16_t* scale,
                          const uint8_t* zero, int lds, const int32_t* msb) {
    const auto kernel = group == 32 ? w4_pack_kernel<32> : (group == 64 ? w4_pack_kernel<64> : w4_pack_kernel<128>);
    hipLaunchKernelGGL(kernel, dim3(w4_ct(N), n), dim3(256), 0, st, N, K, q, w4_bytes(N, K, group), cst, nib, ldn, scale, zero, lds, msb);
    return hipGetLastError();
}

// ---------------------------------------------------------------- products

// What two columns' epilogue reads besides the sums
struct W4Epi {
    int4 c0, c1;
    int e, r0, r1;
};

// A block computes `js` column tiles for up to 4 RR MT rows (see w4_kernel.h). LDS: the rows' chunk, then the sums.
template <int MT, int RR, int P, int G>
__global__ void __launch_bounds__(1024) w4_kernel(W4Args a, int js, W4Chunks ch, int rows_lds) {
    // tiles in flight: 48 of a CU's sixteen waves; with 4 and 6 a wave, 5 x 11008 x 4096 took 11.6 and 12.3 against 11.4 us, 1 x 4096 x 22016 10.1
    // and 10.8 against 10.0, 1 x 8192 x 28672 23.7 and 24.1 against 24.1
    constexpr int TR = 4 * RR * MT, DEPTH = 3;
    touch_args<int(sizeof(W4Args) + sizeof(W4Chunks) + 8)>();
    extern __shared__ uint4 s_dyn[];
    __shared__ uint32_t s_rm[TR];
    __shared__ int s_e[TR];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = __builtin_amdgcn_readfirstlane(blockDim.x >> 6);
    const int ct0 = int(blockIdx.x) * js, tiles = min(js, a.w.CT - ct0), row0 = int(blockIdx.y) * TR, rows = min(TR, a.M - row0), KT = a.w.KT;
    const int prows = MT == 1 ? rows : TR;
    uint8_t* lds = reinterpret_cast<uint8_t*>(s_dyn);
    unsigned long long* sums = reinterpret_cast<unsigned long long*>(lds + rows_lds);
    int32_t* lut = reinterpret_cast<int32_t*>(sums + js * TR * 16);   // GEGLU
    const W4Columns from{a.w.q + size_t(ct0) * KT * 1024, a.w.s + size_t(ct0) * KT * (4096 / G), KT};
    const bool x32 = P == 2 && a.x;
    W4Ring<G, DEPTH> ring;
    int e = 0;   // of row threadIdx.x. Storing it to s_e waits for every load asked for until then (how many is not known at compile
                 // time), the first tiles and the gate's table among them, and the rows are asked for only after that
    if (int(threadIdx.x) < rows) e = x32 ? rowexp_u32(a.xmax[row0 + threadIdx.x]) : (a.e ? a.e[row0 + threadIdx.x] : 0);
    for (int i = threadIdx.x; i < tiles * TR * 16; i += blockDim.x) sums[i] = 0;
    ring.start(from, KT, tiles, 0, ch, lane, wave, waves);
    // two columns a thread; a thread's first two's constants and residual come from here on, where there are registers for them
    const int items = tiles * rows * 8;
    W4Epi ep;
    const auto fetch = [&](int i) {
        const int ctt = w4_div(i >> 3, rows), t = (i >> 3) - ctt * rows, n = (ct0 + ctt) * 16 + 2 * (i & 7);
        ep.c0 = a.w.cst[n];
        ep.c1 = a.w.cst[n + 1];
        ep.r0 = ep.r1 = 0;
        if (a.R) {
            const int32_t* R = a.R + size_t(row0 + t) * a.ldy + n;
            if (n < a.w.N) ep.r0 = R[0];
            if (n + 1 < a.w.N) ep.r1 = R[1];
        }
    };
    if (MT == 1 && int(threadIdx.x) < items) fetch(threadIdx.x);
    if (a.geglu) w4_load_lut(lut, a.Lphi, lane, wave, waves);
    if (int(threadIdx.x) < rows) {
        s_rm[threadIdx.x] = 0;
        s_e[threadIdx.x] = e;
    }
    for (int c = 0;;) {
        const int k0 = c * ch.kc, kc = min(ch.kc, KT - k0);
        if (x32)
            w4_stage_x32(lds, ch.ld(), prows, rows, k0, kc, a.w.K, a.x + size_t(row0) * a.ldx, [&](int r) { return unsigned(r) * unsigned(a.ldx); }, [&](int r) { return rowexp_u32(a.xmax[row0 + r]); }, lane, wave, waves);
        else
            w4_stage<P>(lds, ch.ld(), prows, rows, k0, kc, a.Kp16, a.hi + size_t(row0) * a.ld8, P == 2 ? a.lo + size_t(row0) * a.ld8 : nullptr,
                        [&](int r) { return unsigned(r) * unsigned(a.ld8); });
        __syncthreads();
        w4_share<MT, RR, P, G>(ring, lds, ch.ld(), prows, rows, [](int) { return 0; }, sums, lane);
        if (++c == ch.n) break;
        ring.start(from, KT, tiles, c, ch, lane, wave, waves);   // on its way while the rows are staged
        __syncthreads();
    }
    if (MT == 2 && int(threadIdx.x) < items) fetch(threadIdx.x);
    __syncthreads();
    for (int i = threadIdx.x; i < items; i += blockDim.x) {
        const int c = w4_div(i >> 3, rows), t = (i >> 3) - c * rows, n = (ct0 + c) * 16 + 2 * (i & 7), r = row0 + t;
        if (i != int(threadIdx.x)) fetch(i);
        if (n >= a.w.N) continue;
        const longlong2 v = *reinterpret_cast<const longlong2*>(&sums[(c * TR + t) * 16 + 2 * (i & 7)]);
        int y0 = w4_requant(v.x, P == 2, ep.c0, s_e[t]), y1 = w4_requant(v.y, P == 2, ep.c1, s_e[t]);
        uint32_t m;
        if (a.geglu) {
            y0 = geglu_exact(y0, y1, lut);
            a.Y[size_t(r) * a.ldy + (n >> 1)] = y0;
            m = uabs(y0);
        } else {
            const size_t at = size_t(r) * a.ldy + n;
            const bool two = n + 1 < a.w.N;
            y0 = add_sat(y0, ep.r0);
            y1 = add_sat(y1, ep.r1);
            a.Y[at] = y0;
            if (two) a.Y[at + 1] = y1;
            m = max(uabs(y0), two ? uabs(y1) : 0u);
        }
        if (a.rowmax) atomicMax(&s_rm[t], m);
    }
    if (a.rowmax) {
        __syncthreads();
        // a maximum only grows: a row whose value stands already, even read late, needs no atomic
        if (int(threadIdx.x) < rows) {
            uint32_t* to = a.rowmax + row0 + threadIdx.x;
            const uint32_t m = s_rm[threadIdx.x];
            if (m > __hip_atomic_load(to, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) atomicMax(to, m);
        }
    }
}

// Column tiles a block has, of up to TR rows: what one round of blocks, one a CU, takes; at most 64 KiB of sums
static int w4_js(const W4Args& a, int TR) { return std::min(512 / TR, cdiv(a.w.CT, std::max(1, NCU / cdiv(a.M, TR)))); }

template <int MT, int RR, int P, int G>
static void w4_launch(hipStream_t st, const W4Args& a) {
    constexpr int TR = 4 * RR * MT;
    // Sixteen waves a block, a block a CU: halves of that, two a CU, staged the rows twice as often and, with twice as many blocks adding to the row
    // maxima, took 18.1 against 16.0 us for 16 x 4096 x 22016 with GEGLU, 16.1 against 13.2 with 16-bit rows.
    const int rb = cdiv(a.M, TR), js = w4_js(a, TR);
    const int lut = a.geglu ? W4_LUT_LDS : 0, most = (156 << 10) - js * TR * 128 - lut, prows = MT == 1 ? std::min(TR, a.M) : TR;
    const W4Chunks ch = W4Chunks::of(prows, P, a.w.KT, most);   // whole rows where they fit
    const int rows_lds = prows * P * ch.ld();
    hipLaunchKernelGGL((w4_kernel<MT, RR, P, G>), dim3(cdiv(a.w.CT, js), rb), dim3(1024), rows_lds + size_t(js) * TR * 128 + lut, st, a, js, ch, rows_lds);
}

template <int MT, int RR, int P>
static void w4_group(hipStream_t st, const W4Args& a) {
    if (a.group == 32) w4_launch<MT, RR, P, 32>(st, a);
    else if (a.group == 64) w4_launch<MT, RR, P, 64>(st, a);
    else w4_launch<MT, RR, P, 128>(st, a);
}

template <int MT, int RR>
static void w4_planes(hipStream_t st, const W4Args& a) {
    if (a.x || a.lo) w4_group<MT, RR, 2>(st, a);
    else w4_group<MT, RR, 1>(st, a);
}

// More than sixteen rows go in blocks of 16 where a block then has few column tiles, so that staging (and quantising) the rows counts
// more than reading the weights again, else in blocks of 32; int32 rows by the same reason in blocks of 8:
//                                   16        32 rows a block
//   int32, 32 x 11008 x 4096        22.7      46.9 us    2 column tiles a block of 16 rows
//          64 x 4096 x 12288        20.6      23.0      12
//          64 x 4096 x 22016        37.4      40.3      22
//   16-bit, 32 x 11008 x 4096       15.1      21.9       2
//          128 x 4096 x 4096        14.5      14.3       8
//          64 x 4096 x 12288        17.8      17.4      12
//   8-bit, 32 x 11008 x 4096        11.3      12.8       2
//          20 x 4096 x 4096          6.0       5.9       2
//          128 x 4096 x 4096        11.9       9.3       8
//          32 x 4096 x 22016        18.0      12.8      11
//                                    8        16 rows a block
//   int32, 16 x 11008 x 4096        14.2      19.9 us    2 column tiles a block of 8 rows
//          32 x 11008 x 4096        19.4      22.7       4
//          64 x 11008 x 4096        28.2      28.1       8
//          16 x 4096 x 22016        19.3      14.8      11
// (Two medians differ by up to 5 %, so the line for int32 rows, between 12 and 22 tiles, could stand higher.)
hipError_t launch_w4(hipStream_t st, const W4Args& a) {
    if (a.M <= 4) w4_planes<1, 1>(st, a);
    else if (a.M <= 8 || (a.x && w4_js(a, 8) <= 8)) w4_planes<1, 2>(st, a);
    else if (a.M <= 16 || w4_js(a, 16) <= (a.x ? 16 : (a.lo ? 8 : 2))) w4_planes<1, 4>(st, a);
    else w4_planes<2, 4>(st, a);
    return hipGetLastError();
}

}  // namespace vk
