// Products of few rows with 4-bit weights in group scales: the device core of w4.hip and moe.hip.
//
//   acc[r, n] = sum over groups G of sc[n, G] * sum_{k in G} q[r, k] (u[n, k] - z[n, G])
//
// The inner sums run on int8 MFMA (16 rows x 64 values of K x 16 columns; 32 values of K where a group has 32): the
// nibbles are spread to bytes and shifted by their zero point in registers, 16-bit rows go through as two planes. A
// group's sum (below 2^27) is scaled and added in 64 bits, one v_mad_i64_i32 a value (6 cycles of a SIMD here; a
// conversion to double and an fma take 10): |acc| <= 2^15 * 15 * 4095 * K < 2^46.
//
// Layout of a matrix: tiles of 16 columns x 128 values of K, [column tile][K tile], 1 KiB of nibbles each, so that a wave
// streams a tile with one 16-byte load a lane; lane l = 16 j + n holds column n, and nibble half h of its byte b is
//   groups of 64 and 128:  k = 64 h + 16 j + b
//   groups of 32:          k = 64 h + 32 (b / 8) + 8 j + b % 8
// behind all tiles the group words [column tile][K tile][16 columns][128 / group], zero << 12 | scale. Columns past N and
// values past K have scale 0 and u = z.
//
// Work of a block: a segment of column tiles against up to 32 rows. The rows are staged in LDS, as much of K at a time as fits
// (a chunk): read from memory by every wave, 16 rows of 64 bytes would take 65 cycles of a CU's address unit a load, against
// 17 for a tile's nibbles and 6 for its words. The chunk's tiles, a column tile's one after the other, are split evenly over the
// waves, which stream them with DEPTH tiles in flight and add each column tile's sums to 64-bit integers in LDS; the epilogue
// reads those. Integer sums: their order does not matter.
//
// Bound by the weights' stream for a few rows (1 x 8192 x 28672, groups of 128: 24.0 us, 5.05 TB/s; 1 x 4096 x 22016 9.4-10.2 us), for tens
// of rows by their staging and the groups' scaling (64 x 4096 x 22016 21.3 us; 51 x 2600 x 9999 in 16 bits, groups of 32, 18 us).
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

// One tile as a lane holds it: its 32 nibbles and the group words of its column n = lane & 15. Loaded through buffer resources made
// from scalars, so that the lane offsets never change and no 64-bit address stands in vector registers.
template <int G>
struct W4Tile {
    static constexpr int NG = 128 / G;
    u4v w;
    unsigned own[(NG + 1) / 2];
    __device__ __forceinline__ void load(const uint8_t* q, const uint8_t* s, int lane) {
        const __amdgpu_buffer_rsrc_t rq = make_rsrc(q, 1024u), rs = make_rsrc(s, 32u * NG);
        w = __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(rq, 16 * lane, 0, 0));
        const int so = (lane & 15) * NG * 2;
        if constexpr (NG == 1) {   // both columns of a pair: a 16-bit load is widened where it ends, which would wait for the newest of them
            own[0] = __builtin_amdgcn_raw_buffer_load_b32(rs, so & ~3, 0, 0);
        } else if constexpr (NG == 2) {
            own[0] = __builtin_amdgcn_raw_buffer_load_b32(rs, so, 0, 0);
        } else {
            const u2v o = __builtin_bit_cast(u2v, __builtin_amdgcn_raw_buffer_load_b64(rs, so, 0, 0));
            own[0] = o.x; own[1] = o.y;
        }
    }
    // the word of group g begins at bit 0 or 16 of own[g / 2]
    __device__ __forceinline__ int half(int g, int lane) const { return NG == 1 ? lane & 1 : g & 1; }
    // 0x80 - zero point of group g, in every byte: both words' zero points, each shifted into the low half of its byte, at once (a
    // multiplication by 0x01010101 takes the time of four such instructions)
    __device__ __forceinline__ unsigned zero(int g, int lane) const {
        const unsigned both = 0x80808080u - (own[g >> 1] >> 4 & 0x0f000f00u);
        return __builtin_amdgcn_perm(both, both, half(g, lane) ? 0x03030303u : 0x01010101u);
    }
    __device__ __forceinline__ int scale(int g, int lane) const { return int(__builtin_amdgcn_ubfe(own[g >> 1], unsigned(16 * half(g, lane)), 12u)); }
};

// the low (h = 0) or high nibbles of a word as signed bytes u - z: no byte of u + (0x80 - z) carries into the next, and
// flipping the top bit leaves u - z in two's complement
__device__ __forceinline__ int w4_spread(unsigned w, int h, unsigned zz) { return int((((h ? w >> 4 : w) & 0x0f0f0f0fu) + zz) ^ 0x80808080u); }

__device__ __forceinline__ long w4_pair(int a, int b) { return long((u64(unsigned(b)) << 32) | unsigned(a)); }

// Rows in the sums' registers. A lane receives rows 4 (lane >> 4) + r of the 16 of a matrix instruction; with at most 4 RR of
// them in use they are put where r < RR, so that the others' scaling can be left out: row i of the instruction is row
// (i / 4) RR + i % RR of the tile.
template <int RR>
__device__ __forceinline__ int w4_row(int i) { return (i >> 2) * RR + (i & (RR - 1)); }

// acc[mt][r] += the tile's product for column lane & 15 and the rows above, rows from LDS: a[p] + mt_stride mt is the lane's row of
// plane p at the tile's first value and the lane's part of it
template <int MT, int RR, int P, int G>
__device__ __forceinline__ void w4_tile(const W4Tile<G>& t, const uint8_t* const (&a)[P], int mt_stride, i64 (&acc)[MT][RR], int lane) {
    constexpr int NG = 128 / G;
    const v4i zero4 = {0, 0, 0, 0};
    v4i c[MT][P];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        int b[4];
        if constexpr (G == 32) {
            const unsigned z0 = t.zero(2 * h, lane), z1 = t.zero(2 * h + 1, lane);
            b[0] = w4_spread(t.w.x, h, z0); b[1] = w4_spread(t.w.y, h, z0);
            b[2] = w4_spread(t.w.z, h, z1); b[3] = w4_spread(t.w.w, h, z1);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int g = 2 * h + i, sc = t.scale(g, lane);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        const u2v r = *reinterpret_cast<const u2v*>(a[p] + mt * mt_stride + 32 * g);
                        c[mt][p] = __builtin_amdgcn_mfma_i32_16x16x32_i8(w4_pair(int(r.x), int(r.y)), w4_pair(b[2 * i], b[2 * i + 1]), zero4, 0, 0, 0);
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int r = 0; r < RR; ++r) acc[mt][r] += i64(P == 2 ? c[mt][0][r] * 256 + c[mt][P - 1][r] : c[mt][0][r]) * sc;
            }
        } else {
            const unsigned z = t.zero(NG == 2 ? h : 0, lane);
            b[0] = w4_spread(t.w.x, h, z); b[1] = w4_spread(t.w.y, h, z);
            b[2] = w4_spread(t.w.z, h, z); b[3] = w4_spread(t.w.w, h, z);
            const v4i bv = {b[0], b[1], b[2], b[3]};
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int p = 0; p < P; ++p)
                    c[mt][p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const v4i*>(a[p] + mt * mt_stride + 64 * h), bv, (NG == 1 && h) ? c[mt][p] : zero4, 0, 0, 0);
            }
            if (NG == 2 || h == 1) {
                const int sc = t.scale(NG == 2 ? h : 0, lane);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int r = 0; r < RR; ++r) acc[mt][r] += i64(P == 2 ? c[mt][0][r] * 256 + c[mt][P - 1][r] : c[mt][0][r]) * sc;
            }
        }
    }
}

// a / b for 0 <= a < 2^22, 0 < b: a quotient of floats is off by less than one
__device__ __forceinline__ int w4_div(int a, int b) {
    int q = int(float(a) * __builtin_amdgcn_rcpf(float(b)));
    const int r = a - q * b;
    q += r >= b ? 1 : 0;
    return q - (r < 0 ? 1 : 0);
}

// The rows of a chunk in LDS, [plane][prows][ld]: ld = the chunk's bytes a row + 16, so that 16 rows' 16-byte reads fall on
// distinct banks. As many tiles of K a chunk as `lds` bytes hold, chunks of even size.
struct W4Chunks {
    int kc, n;   // tiles of K a chunk, chunks
    __host__ __device__ __forceinline__ int ld() const { return kc * 128 + 16; }
    static __host__ W4Chunks of(int prows, int P, int KT, int lds) {
        const int fit = (lds / (prows * P) - 16) / 128, most = fit < 1 ? 1 : fit;
        W4Chunks c;
        c.n = (KT + most - 1) / most;
        c.kc = (KT + c.n - 1) / c.n;
        c.n = (KT + c.kc - 1) / c.kc;
        return c;
    }
};

// i / per by a multiplication, for i * per < 2^32
struct W4Per {
    unsigned per, m;
    __device__ __forceinline__ explicit W4Per(int n) : per(n), m(0xffffffffu / unsigned(n) + 1u) {}
    __device__ __forceinline__ int of(int i) const { return per == 1 ? i : int(__umulhi(unsigned(i), m)); }
};

// int8 planes to LDS, 16 bytes a thread and step, four steps in flight. off(r): byte offset of row r in its plane (below 2^30); bytes
// past Kp16 are not written (they meet zero weights)
template <int P, class F>
__device__ __forceinline__ void w4_stage(uint8_t* lds, int ld, int prows, int rows, int k0, int kc, int Kp16, const int8_t* hi, const int8_t* lo, F off) {
    const int per = min(kc * 8, (Kp16 - k0 * 128) >> 4), items = rows * per, step = blockDim.x;
    const W4Per div(per);
    for (int i0 = threadIdx.x; i0 < items; i0 += 4 * step) {
        v4i v[4][P];
        int at[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int i = min(i0 + b * step, items - 1), r = div.of(i), c = 16 * (i - r * per);
            at[b] = r * ld + c;
            const unsigned from = off(r) + unsigned(k0 * 128 + c);
            v[b][0] = *reinterpret_cast<const v4i*>(hi + from);
            if constexpr (P == 2) v[b][P - 1] = *reinterpret_cast<const v4i*>(lo + from);
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {   // the last item may be written more than once
            *reinterpret_cast<v4i*>(lds + at[b]) = v[b][0];
            if constexpr (P == 2) *reinterpret_cast<v4i*>(lds + prows * ld + at[b]) = v[b][P - 1];
        }
    }
}

// int32 rows quantised to planes in LDS, a wave eight times 64 quads of one row at once, so that the row's address and shift are
// scalars: off(r) the row's offset in values, shift(r) its shift, asked for when the values are on their way. K % 4 == 0.
template <class F, class S>
__device__ __forceinline__ void w4_stage_x32(uint8_t* lds, int ld, int prows, int rows, int k0, int kc, int K, const int32_t* x, F off, S shift, int lane, int wave, int waves) {
    constexpr int B = 8;
    const int quads = min(kc * 32, (K - k0 * 128) >> 2), blocks = (quads + 63) >> 6, parts = (blocks + B - 1) / B, items = rows * parts;
    const s2 lim = {-32767, -32767};
    for (int i = wave; i < items; i += waves) {
        const int r = __builtin_amdgcn_readfirstlane(w4_div(i, parts)), b0 = (i - r * parts) * B, n = min(B, blocks - b0);
        const int from = k0 * 128 + b0 * 256;
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(x + __builtin_amdgcn_readfirstlane(off(r)) + from, unsigned(K - from) * 4u);
        v4i v[B];
#pragma unroll
        for (int b = 0; b < B; ++b)
            if (b < n) v[b] = bload16(rs, unsigned(b * 1024 + 16 * lane));
        __builtin_amdgcn_sched_barrier(0);
        const int e = __builtin_amdgcn_readfirstlane(shift(r)), one = e ? 1 : 0;
        // quant16_32 of a value: (v >> e) + bit e - 1 of v; the conversion of pairs to 16 bits clamps the upper end, and only -32768
        // is left to raise
        const auto q = [&](int w) { return (w >> e) + int(__builtin_amdgcn_ubfe(unsigned(w), unsigned(e - 1), unsigned(one))); };
        uint8_t* to = lds + r * ld + b0 * 256 + 4 * lane;
        const int left = quads - b0 * 64 - lane;   // the lane's quads from here on
#pragma unroll
        for (int b = 0; b < B; ++b) {
            if (b >= n) continue;
            const s2 q0 = __builtin_elementwise_max(__builtin_amdgcn_cvt_pk_i16(q(v[b][0]), q(v[b][1])), lim);
            const s2 q1 = __builtin_elementwise_max(__builtin_amdgcn_cvt_pk_i16(q(v[b][2]), q(v[b][3])), lim);
            const unsigned u0 = __builtin_bit_cast(unsigned, q0), u1 = __builtin_bit_cast(unsigned, q1);
            if (64 * b < left) {
                *reinterpret_cast<unsigned*>(to + 256 * b) = __builtin_amdgcn_perm(u1, u0, 0x07050301u);
                *reinterpret_cast<unsigned*>(to + 256 * b + prows * ld) = __builtin_amdgcn_perm(u1, u0, 0x06040200u) ^ 0x80808080u;
            }
        }
    }
}

// The gate's table in LDS, where two dependent reads an output are fast: 64 entries a wave and step straight from memory, with nobody
// waiting for them (through registers they held the rows' staging up). Zeros behind the last entry.
constexpr int W4_LUT = 2049, W4_LUT_STEPS = (W4_LUT + 63) / 64, W4_LUT_LDS = W4_LUT_STEPS * 256;
__device__ __forceinline__ void w4_load_lut(int32_t* to, const int32_t* L, int lane, int wave, int waves) {
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(L, W4_LUT * 4u);
    for (int i = wave; i < W4_LUT_STEPS; i += waves)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(to + 64 * i), 4, 4 * lane, 256 * i, 0, 0);
}

// Column tiles c = 0, 1, ... of a matrix, one behind the other
struct W4Columns {
    const uint8_t *q, *s;      // of the first
    int KT;
    template <int G>
    __device__ __forceinline__ void at(int c, int k, const uint8_t*& qc, const uint8_t*& sc) const {   // tile k of column tile c
        const size_t tile = size_t(c) * KT + k;
        qc = q + tile * 1024;
        sc = s + tile * (4096 / G);
    }
};

// A wave's share of a chunk: tiles u of the column tiles c = u / kc, in the order of their addresses
template <int G, int DEPTH, class Src = W4Columns>
struct W4Ring {
    W4Tile<G> t[DEPTH];
    Src src;
    int k0, kc;                // the chunk's tiles of K
    int u0, u1;                // the wave's tiles
    const uint8_t *qc, *sc;    // the column tile loaded from
    int c, k;                  // the tile loaded next
    __device__ __forceinline__ void fetch(int d, int lane) {
        t[d].load(qc + size_t(k) * 1024, sc + size_t(k) * (4096 / G), lane);
        if (++k == kc) {
            k = 0;
            src.template at<G>(++c, k0, qc, sc);
        }
    }
    __device__ __forceinline__ void start(const Src& from, int KT, int cols, int chunk, const W4Chunks& ch, int lane, int wave, int waves) {
        src = from;
        k0 = chunk * ch.kc;
        kc = min(ch.kc, KT - k0);
        const int units = cols * kc;
        u0 = __builtin_amdgcn_readfirstlane(w4_div(units * wave, waves));
        u1 = __builtin_amdgcn_readfirstlane(w4_div(units * (wave + 1), waves));
        c = __builtin_amdgcn_readfirstlane(w4_div(u0, kc));
        k = u0 - c * kc;
        src.template at<G>(c, k0, qc, sc);
#pragma unroll
        for (int d = 0; d < DEPTH; ++d)
            if (u0 + d < u1) fetch(d, lane);
    }
};

// The wave's share: sums of column tile c, row t and column n are added to sums[(c * TR + t) * 16 + n], TR = 4 RR MT. rows_of(c): the
// first of the rows column tile c meets
template <int MT, int RR, int P, int G, int DEPTH, class Src, class F>
__device__ __forceinline__ void w4_share(W4Ring<G, DEPTH, Src>& ring, const uint8_t* lds, int ld, int prows, int rows, F rows_of, unsigned long long* sums, int lane) {
    constexpr int TR = 4 * RR * MT;
    int u = ring.u0, c = __builtin_amdgcn_readfirstlane(w4_div(u, ring.kc)), k = u - c * ring.kc;
    if (u >= ring.u1) return;
    // rows of the instruction past the last one repeat it (in the last row tile of several: what stands there): nobody reads
    // their sums
    const uint8_t* base[P];
    static_assert(MT == 1 || RR == 4, "row tiles are whole");
    const int lane_off = G == 32 ? 8 * (lane >> 4) : 16 * (lane >> 4);
#pragma unroll
    for (int p = 0; p < P; ++p) base[p] = lds + (p * prows + min(w4_row<RR>(lane & 15), rows - 1)) * ld + lane_off;
    i64 acc[MT][RR];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < RR; ++r) acc[mt][r] = 0;
    int row = rows_of(c) * ld;
    const auto step = [&](int d, bool last) {
        const uint8_t* a[P];
#pragma unroll
        for (int p = 0; p < P; ++p) a[p] = base[p] + row + k * 128;
        w4_tile<MT, RR, P, G>(ring.t[d], a, 16 * ld, acc, lane);
        if (++k == ring.kc || last) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int r = 0; r < RR; ++r) {
                    atomicAdd(&sums[(c * TR + 16 * mt + (lane >> 4) * RR + r) * 16 + (lane & 15)], (unsigned long long)acc[mt][r]);
                    acc[mt][r] = 0;
                }
            k = 0;
            row = rows_of(++c) * ld;
        }
        __builtin_amdgcn_sched_barrier(0);   // one tile at a time: stages drawn into one another spill
    };
    // Rounds of the ring that use and refill every stage, so that the compiler counts the loads in flight and waits for one tile at
    // a time; then the rest, where a load may be left out and it waits for all of a round. (Refilling past the last tile instead, with loads
    // that fetch nothing, cost 1 us of 4.6 for 1 x 2048 x 2048.)
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): the first tiles are here, the rows' staging waited for younger loads
    for (; u + 2 * DEPTH <= ring.u1; u += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            step(d, false);
            ring.fetch(d, lane);
        }
    }
    for (; u < ring.u1; u += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (u + d < ring.u1) {
                step(d, u + d + 1 == ring.u1);
                if (u + d + DEPTH < ring.u1) ring.fetch(d, lane);
            }
        }
    }
}

// The exact epilogue value of a column: acc the product, planes whether the rows carry the offset low plane
__device__ __forceinline__ int w4_requant(i64 acc, bool planes, const int4& c, int e) {
    const i64 a = acc + (planes ? 128LL * c.w : 0LL);
    return int(sat32(rshr(i64(u64(a) * u64(i64(c.x))), i64(c.y) - e) + c.z));
}

}  // namespace vk
