// Products of few rows with 4-bit weights in group scales: the device core of w4.hip and moe.hip.
//
//   acc[r, n] = sum over groups G of sc[n, G] * sum_{k in G} q[r, k] (u[n, k] - z[n, G])
//
// The inner sums run on int8 MFMA (16 columns x 64 values of K x 16 rows; 32 values of K where a group has 32): the
// nibbles are spread to bytes and shifted by their zero point in registers, 16-bit rows go through as two planes. A
// group's sum (below 2^27) is scaled and added in double, which is exact: |acc| <= 2^15 * 15 * 4095 * K < 2^46.
//
// Layout of a matrix: tiles of 16 columns x 128 values of K, [column tile][K tile], 1 KiB of nibbles each, so that a wave
// streams a tile with one 16-byte load a lane; lane l = 16 j + n holds column n, and nibble half h of its byte b is
//   groups of 64 and 128:  k = 64 h + 16 j + b
//   groups of 32:          k = 64 h + 32 (b / 8) + 8 j + b % 8
// behind all tiles the group words [column tile][K tile][16 columns][128 / group], zero << 12 | scale. Columns past N and
// values past K have scale 0 and u = z.
#pragma once
#include "vk_common.h"

namespace vk {

struct W4View {
    const uint8_t* q;      // nibbles
    const uint8_t* s;      // group words
    const int4* cst;       // {m, s, b, wsum}
    int N, K, KT, CT;      // columns, depth, tiles of 128 and of 16
};

__host__ __device__ constexpr int w4_kt(int K) { return (K + 127) / 128; }
__host__ __device__ constexpr int w4_ct(int N) { return (N + 15) / 16; }
__host__ __device__ constexpr size_t w4_bytes(int N, int K, int group) { return size_t(w4_ct(N)) * w4_kt(K) * (1024 + 32 * (128 / group)); }

typedef unsigned u2v __attribute__((ext_vector_type(2)));
typedef unsigned u4v __attribute__((ext_vector_type(4)));

// One tile's words as a lane holds them: its 32 nibbles, the group words of its own column n = lane & 15 (for the zero points)
// and those of the four columns 4 (lane >> 4) + r whose sums it receives.
template <int G>
struct W4Tile {
    static constexpr int NG = 128 / G;
    u4v w;
    unsigned own[(NG + 1) / 2];
    unsigned four[2 * NG];
    __device__ __forceinline__ void load(const uint8_t* q, const uint8_t* s, int lane) {
        w = *reinterpret_cast<const u4v*>(q + 16 * lane);
        const uint8_t* so = s + (lane & 15) * NG * 2;
        const uint8_t* sf = s + (lane >> 4) * NG * 8;
        if constexpr (NG == 1) {
            own[0] = *reinterpret_cast<const uint16_t*>(so);
            const u2v f = *reinterpret_cast<const u2v*>(sf);
            four[0] = f.x; four[1] = f.y;
        } else if constexpr (NG == 2) {
            own[0] = *reinterpret_cast<const unsigned*>(so);
            const u4v f = *reinterpret_cast<const u4v*>(sf);
            four[0] = f.x; four[1] = f.y; four[2] = f.z; four[3] = f.w;
        } else {
            const u2v o = *reinterpret_cast<const u2v*>(so);
            own[0] = o.x; own[1] = o.y;
            const u4v f = *reinterpret_cast<const u4v*>(sf), f2 = *reinterpret_cast<const u4v*>(sf + 16);
            four[0] = f.x; four[1] = f.y; four[2] = f.z; four[3] = f.w;
            four[4] = f2.x; four[5] = f2.y; four[6] = f2.z; four[7] = f2.w;
        }
    }
    // zero point of the lane's column in group g, in every byte
    __device__ __forceinline__ unsigned zero(int g) const {
        const unsigned z = (g & 1) ? own[g >> 1] >> 28 : (own[g >> 1] >> 12) & 15u;
        return z * 0x01010101u;
    }
    // scale of column 4 (lane >> 4) + r in group g
    __device__ __forceinline__ double scale(int g, int r) const {
        const int i = r * NG + g;
        const unsigned v = (i & 1) ? (four[i >> 1] >> 16) & 0xfffu : four[i >> 1] & 0xfffu;
        return double(int(v));
    }
};

// the low (h = 0) or high nibbles of a word as signed bytes u - z: the bytes 0x80 + u - z borrow nothing from one
// another, and flipping the top bit leaves u - z in two's complement
__device__ __forceinline__ int w4_spread(unsigned w, int h, unsigned zz) { return int((((h ? w >> 4 : w) & 0x0f0f0f0fu) | 0x80808080u) - zz) ^ int(0x80808080u); }

// One tile's rows: planes b[p][...] of a lane's row, as the tile's K order needs them (G = 128, 64: values 16 j .. 16 j + 15
// of each half; G = 32: values 8 j .. 8 j + 7 of each group), 32 bytes a plane.
template <int P>
struct W4Rows {
    v4i b[P][2];
    template <int G>
    __device__ __forceinline__ void load(const int8_t* hi, const int8_t* lo, int k0, int Kp16, int lane) {
        // values past the row's end meet zero weights: any address inside the row will do
        if constexpr (G == 32) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int k = k0 + 32 * g + 8 * (lane >> 4), kk = k < Kp16 ? k : 0;
                const u2v h = *reinterpret_cast<const u2v*>(hi + kk);
                b[0][g >> 1][2 * (g & 1)] = int(h.x); b[0][g >> 1][2 * (g & 1) + 1] = int(h.y);
                if constexpr (P == 2) {
                    const u2v l = *reinterpret_cast<const u2v*>(lo + kk);
                    b[P - 1][g >> 1][2 * (g & 1)] = int(l.x); b[P - 1][g >> 1][2 * (g & 1) + 1] = int(l.y);
                }
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = k0 + 64 * h + 16 * (lane >> 4), kk = k < Kp16 ? k : 0;
                b[0][h] = *reinterpret_cast<const v4i*>(hi + kk);
                if constexpr (P == 2) b[P - 1][h] = *reinterpret_cast<const v4i*>(lo + kk);
            }
        }
    }
};

__device__ __forceinline__ long w4_pair(int a, int b) { return long((u64(unsigned(b)) << 32) | unsigned(a)); }

// acc[r] += the tile's product for column 4 (lane >> 4) + r and row lane & 15, for MT row tiles
template <int MT, int P, int G>
__device__ __forceinline__ void w4_tile(const W4Tile<G>& t, const W4Rows<P> (&rows)[MT], double (&acc)[MT][4]) {
    constexpr int NG = 128 / G;
    const v4i zero4 = {0, 0, 0, 0};
    v4i c[MT][P];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        int a[4];
        if constexpr (G == 32) {
            const unsigned z0 = t.zero(2 * h), z1 = t.zero(2 * h + 1);
            a[0] = w4_spread(t.w.x, h, z0); a[1] = w4_spread(t.w.y, h, z0);
            a[2] = w4_spread(t.w.z, h, z1); a[3] = w4_spread(t.w.w, h, z1);
        } else {
            const unsigned z = t.zero(NG == 2 ? h : 0);
            a[0] = w4_spread(t.w.x, h, z); a[1] = w4_spread(t.w.y, h, z);
            a[2] = w4_spread(t.w.z, h, z); a[3] = w4_spread(t.w.w, h, z);
        }
        if constexpr (G == 32) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int g = 2 * h + i;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                    for (int p = 0; p < P; ++p)
                        c[mt][p] = __builtin_amdgcn_mfma_i32_16x16x32_i8(w4_pair(a[2 * i], a[2 * i + 1]), w4_pair(rows[mt].b[p][h][2 * i], rows[mt].b[p][h][2 * i + 1]), zero4, 0, 0, 0);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const double sc = t.scale(g, r);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const int v = P == 2 ? c[mt][0][r] * 256 + c[mt][P - 1][r] : c[mt][0][r];
                        acc[mt][r] = fma(double(v), sc, acc[mt][r]);
                    }
                }
            }
        } else {
            const v4i av = {a[0], a[1], a[2], a[3]};
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int p = 0; p < P; ++p)
                    c[mt][p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(av, rows[mt].b[p][h], (NG == 1 && h) ? c[mt][p] : zero4, 0, 0, 0);
            }
            if (NG == 2 || h == 1) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const double sc = t.scale(NG == 2 ? h : 0, r);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const int v = P == 2 ? c[mt][0][r] * 256 + c[mt][P - 1][r] : c[mt][0][r];
                        acc[mt][r] = fma(double(v), sc, acc[mt][r]);
                    }
                }
            }
        }
    }
}

// The quads of int32 rows of one tile, quantised to planes in a wave's own LDS: rows 2 i + (lane >> 5) of `nrows`, 32 lanes a
// row, [plane][row][W4_LDR]. Row shifts are in se[row].
constexpr int W4_LDR = 144;   // bytes between rows: 16-byte reads of 16 rows fall on distinct banks
template <int RT>
struct W4Quads {
    int4 v[RT / 2];
    // rowp(r): address of row r (r < nrows)
    template <class F>
    __device__ __forceinline__ void load(F rowp, int nrows, int k0, int K, int lane) {
        const int k = k0 + 4 * (lane & 31);
#pragma unroll
        for (int i = 0; i < RT / 2; ++i) {
            if (2 * i >= nrows) break;
            const int r = 2 * i + (lane >> 5);
            v[i] = make_int4(0, 0, 0, 0);
            if (r < nrows && k < K) v[i] = *reinterpret_cast<const int4*>(rowp(r) + k);
        }
    }
    __device__ __forceinline__ void stage(uint8_t* lds, const int* se, int nrows, int lane) const {
#pragma unroll
        for (int i = 0; i < RT / 2; ++i) {
            if (2 * i >= nrows) break;
            const int r = 2 * i + (lane >> 5);
            if (r < nrows) {
                const int e = se[r];
                const int q0 = quant16_32(v[i].x, e), q1 = quant16_32(v[i].y, e), q2 = quant16_32(v[i].z, e), q3 = quant16_32(v[i].w, e);
                unsigned* h = reinterpret_cast<unsigned*>(lds + r * W4_LDR + 4 * (lane & 31));
                unsigned* l = reinterpret_cast<unsigned*>(lds + (RT + r) * W4_LDR + 4 * (lane & 31));
                *h = __builtin_amdgcn_perm(unsigned(q1), unsigned(q0), 0x0c0c0501u) | __builtin_amdgcn_perm(unsigned(q3), unsigned(q2), 0x05010c0cu);
                *l = (__builtin_amdgcn_perm(unsigned(q1), unsigned(q0), 0x0c0c0400u) | __builtin_amdgcn_perm(unsigned(q3), unsigned(q2), 0x04000c0cu)) ^ 0x80808080u;
            }
        }
    }
};

// orders a wave's LDS writes before its other lanes' reads (and the reverse); LDS operations of a wave run in order
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The exact epilogue value of a column: acc the product, planes whether the rows carry the offset low plane
__device__ __forceinline__ int w4_requant(i64 acc, bool planes, const int4& c, int e) {
    const i64 a = acc + (planes ? 128LL * c.w : 0LL);
    return int(sat32(rshr(i64(u64(a) * u64(i64(c.x))), i64(c.y) - e) + c.z));
}

}  // namespace vk
