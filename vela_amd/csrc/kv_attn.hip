// Attention of one new token over a paged cache (vgemm_kv_attention), exact in integers: include/vgemm_kv.h states the formulas.
//
// The weights of a softmax need the row's maximum before their sum, and a rounded weight cannot be rescaled exactly. The
// operator is therefore defined on spans of 256 positions: a span's weights are relative to its own maximum, its mean is rounded to 32 bits, and the means
// are joined with the spans' weights. A span needs one pass over its keys and values, any split of the sequence into spans gives the same
// numbers, and what goes from the first kernel to the join is 4 D bytes a span and query head beside 512 D planes of cache.
//
// A block of four waves takes a span of one sequence and key head with up to sixteen of its query heads, one a column of the 16x16x64 int8
// matrix instruction.
//   * Scores: wave w has the positions [64 w, 64 w + 64). The keys are the A operand; row i of subtile ks is position 16 (i / 4) + 4 ks + i % 4, so that
//     lane (fg, query) ends with the scores of the 16 positions from 16 fg on, in order. Quarters of four tokens
//     lie together in a page (vgemm_kv.h), so a load touches four runs of 256 bytes.
//   * Queries are quantised by every wave for itself while its keys are on their way, in signed digits q = 256 h + l (15 bits leave h in [-64, 64]),
//     so that keys of 8 bits need two products a piece and no correction.
//   * A score is floor(S m 2^(eq + ek - s) + 1/2) in double: |S m| <= 2^52, so the product is exact and so is the sum with 1/2.
//   * Weights with the values' shifts, x = -P 2^(ev - least ev of the span), go as signed digits of 8 bits through LDS: two digits where all shifts
//     are equal, three up to 8 apart, up to six in general. Negated, the top digit lies in [-128, 0].
//   * Values lie transposed in a page, D x 16 tokens: the A operand of 16 dimensions and 64 positions is one 16-byte load a lane. Wave w takes
//     the dimensions 16 (w + 4 i) of all 256 positions, so nothing is added across waves.
// Positions that do not count have weight 0; their keys and values are read from page 0 (which is there) or from the rest of a page.
#include <algorithm>
#include <climits>

#include "kv.h"
#include "norm_math.h"

namespace vk {

namespace {

constexpr int EXP_N = 1025;
constexpr int MAX_DIGITS = 6;         // 15 bits and shifts up to 25 apart
constexpr int P_LD = KV_SPAN + 16;    // bytes of a query's weights in LDS, one digit: rows 4 banks apart
constexpr int TOP_SHIFT = 25;         // of an int32 in 8 bits

// what a wave waits for before it meets the others: its own LDS traffic, not its loads
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ i64 shfl_xor64(i64 v, int d) { return i64(__shfl_xor((long long)v, d)); }

// floor(n / l) saturated to 32 bits, l > 0, inv = 1 / l: the quotient in double is off by less than one
__device__ __forceinline__ int div_sat(i64 n, i64 l, double inv) {
    double q = floor(double(n) * inv);
    const i64 r = n - i64(cvt_sat(q)) * l;
    if (r < 0) q -= 1.0;
    if (r >= l) q += 1.0;
    return cvt_sat(q);
}

struct Lds {
    uint2 table[EXP_N];                        // entry i: Lexp[i] + 2^14, Lexp[i + 1] - Lexp[i]; the last one stands for 0
    int8_t p[MAX_DIGITS][16][P_LD];
    int mx[4][16], sum[4][16], lo[4], hi[4];
    i64 x[4][16];
};

// rshr(lutexp(d), 15), at most 32767
__device__ __forceinline__ int weight(const Lds& s, unsigned d) {
    const uint2 t = s.table[min(d >> 10, unsigned(EXP_N - 1))];
    const i64 prod = i64(int(t.y)) * int(d & 1023);
    return min(int((t.x + unsigned(int(prod >> 10))) >> 15), 32767);
}

template <int NS, int PL>
__global__ void __launch_bounds__(256) kv_attn_kernel(KvAttnArgs a) {
    constexpr bool EARLY = NS * PL <= 4;       // values asked for with the keys: 32 NS PL registers for both
    __shared__ __attribute__((aligned(16))) Lds s;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fg = lane >> 4;
    const int head = blockIdx.x / a.qtiles, q0 = (blockIdx.x % a.qtiles) * 16, row = blockIdx.y;
    const KvView& c = a.c;
    const int D = c.D, P = 1 << c.lp;
    const int n = int(min(i64(max(min(a.len[row], a.max_len), 0)), i64(a.width) << c.lp)), first = a.window > 0 ? max(0, n - a.window) : 0;
    const int u0 = first / KV_SPAN, u1 = (n + KV_SPAN - 1) / KV_SPAN;
    const int nq = min(16, a.group - q0);      // query heads of this block
    const bool mine = fr < nq;
    const int qh = head * a.group + q0 + fr;
    if (n == 0) {
        if (blockIdx.z == 0)
            for (int i = tid; i < nq * D; i += 256) a.out[size_t(row) * a.ldo + (head * a.group + q0) * D + i] = 0;
        return;
    }
    if (u0 + int(blockIdx.z) >= u1) return;

    for (int i = tid; i < EXP_N; i += 256) {
        const i64 t = a.Lexp[i], t1 = a.Lexp[min(i + 1, EXP_N - 1)];
        s.table[i] = i < EXP_N - 1 ? make_uint2(unsigned(t) + (1u << 14), unsigned(t1 - t)) : make_uint2(0, 0);
    }

    // queries: lane (fg, fr) holds the values [64 c + 16 fg, + 16) of query fr
    v4i qd[NS][2];
    int qsum = 0;
    double scale;
    {
        int x[NS][16];
        unsigned m = 0;
        const int32_t* q = a.Q + size_t(row) * a.ldq + size_t(mine ? qh : head * a.group) * D;
#pragma unroll
        for (int b = 0; b < NS; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 64 * b + 16 * fg + 4 * i;
                const int4 v = mine && d < D ? *reinterpret_cast<const int4*>(q + d) : make_int4(0, 0, 0, 0);
                x[b][4 * i] = v.x; x[b][4 * i + 1] = v.y; x[b][4 * i + 2] = v.z; x[b][4 * i + 3] = v.w;
                m = max(max(m, max(uabs(v.x), uabs(v.y))), max(uabs(v.z), uabs(v.w)));
            }
        m = max(m, unsigned(__shfl_xor(int(m), 16)));
        m = max(m, unsigned(__shfl_xor(int(m), 32)));
        const int e = max(0, 32 - __clz(int(m)) - 14);
#pragma unroll
        for (int b = 0; b < NS; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                unsigned h = 0, l = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int v = x[b][4 * i + j], r = e ? (v >> e) + ((v >> (e - 1)) & 1) : v;
                    qsum += r;
                    h |= unsigned(((r + 128) >> 8) & 255) << (8 * j);
                    l |= unsigned(r & 255) << (8 * j);
                }
                qd[b][0][i] = int(h);
                qd[b][1][i] = int(l);
            }
        if (PL == 2) {
            qsum += __shfl_xor(qsum, 16);
            qsum += __shfl_xor(qsum, 32);
        }
        scale = ldexp(double(a.m), e - a.s);
    }
    __syncthreads();

    const int pieces = D >> 4;
    const int32_t* table = a.table + size_t(row) * a.ldt;
    for (int u = u0 + int(blockIdx.z); u < u1; u += int(gridDim.z)) {
        const int base = u * KV_SPAN;
        // pages of the span's sixteen groups, in lanes 0..15
        int page;
        {
            const int pos = base + 16 * fr;
            page = pos < n ? table[pos >> c.lp] : -1;
            if (unsigned(page) >= unsigned(c.pages)) page = -1;
        }
        // group g of the span: its bytes in a page of keys, and whether there is one
        auto group = [&](int g, bool& there) {
            const int p = __shfl(page, g);
            there = p >= 0;
            return c.keys(max(p, 0), head) + (((base + 16 * g) & (P - 1)) >> 4) * c.group_bytes();
        };
        bool there;
        const int8_t* kg = group(4 * wave + (fr >> 2), there) + (fr & 3) * 16 + fg * 64;
        v4i kv[4][NS][PL], vv[NS][4][PL];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int b = 0; b < NS; ++b)
#pragma unroll
                for (int p = 0; p < PL; ++p)
                    kv[ks][b][p] = 4 * b + fg < pieces ? *reinterpret_cast<const v4i*>(kg + p * 16 * D + ks * 4 * D + b * 256) : v4i{0, 0, 0, 0};
        const int8_t* vg[4];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            bool ok;
            vg[kt] = group(4 * kt + fg, ok) + c.half_bytes() + fr * 16;
        }
        auto load_values = [&]() {
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int p = 0; p < PL; ++p)
                        vv[i][kt][p] = wave + 4 * i < pieces ? *reinterpret_cast<const v4i*>(vg[kt] + p * 16 * D + (wave + 4 * i) * 256) : v4i{0, 0, 0, 0};
        };
        if (EARLY) load_values();

        // shifts of the lane's sixteen positions, and which of them count
        const int p0 = base + 64 * wave + 16 * fg;
        uint4 ek, ev;
        unsigned live;
        {
            const int pg = __shfl(page, 4 * wave + fg);
            const uint8_t* sh = c.shifts(max(pg, 0), head) + (p0 & (P - 1));
            ek = *reinterpret_cast<const uint4*>(sh);
            ev = *reinterpret_cast<const uint4*>(sh + P);
            const int from = min(max(first - p0, 0), 16), to = min(max(n - p0, 0), 16);
            live = pg >= 0 && to > from ? ((1u << to) - 1) & ~((1u << from) - 1) : 0;
        }
        const unsigned* ekw = reinterpret_cast<const unsigned*>(&ek);
        const unsigned* evw = reinterpret_cast<const unsigned*>(&ev);

        int sc[16];
        int mx = INT_MIN, lo = 255, hi = 0;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            v4i h = {0, 0, 0, 0}, mid = {0, 0, 0, 0}, l = {0, 0, 0, 0};
#pragma unroll
            for (int b = 0; b < NS; ++b) {
                h = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv[ks][b][0], qd[b][0], h, 0, 0, 0);
                if constexpr (PL == 1) {
                    l = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv[ks][b][0], qd[b][1], l, 0, 0, 0);
                } else {
                    mid = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv[ks][b][0], qd[b][1], mid, 0, 0, 0);
                    mid = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv[ks][b][1], qd[b][0], mid, 0, 0, 0);
                    l = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv[ks][b][1], qd[b][1], l, 0, 0, 0);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = 4 * ks + j;
                double S;
                if constexpr (PL == 1) S = double(256 * h[j] + l[j]);
                else S = fma(double(h[j]), 65536.0, fma(double(mid[j]), 256.0, double(l[j] + 128 * qsum)));
                const int e = int((ekw[ks] >> (8 * j)) & 255), f = min(int((evw[ks] >> (8 * j)) & 255), TOP_SHIFT);
                const double up = __builtin_bit_cast(double, u64(unsigned(1023 + e)) << 52);
                sc[i] = cvt_sat(floor(fma(S * scale, up, 0.5)));
                if (live >> i & 1) {
                    mx = max(mx, sc[i]);
                    lo = min(lo, f);
                    hi = max(hi, f);
                }
            }
        }
        mx = max(mx, __shfl_xor(mx, 16));
        mx = max(mx, __shfl_xor(mx, 32));
        lo = min(lo, __shfl_xor(lo, 16));
        lo = min(lo, __shfl_xor(lo, 32));
        hi = max(hi, __shfl_xor(hi, 16));
        hi = max(hi, __shfl_xor(hi, 32));
        if (fg == 0) s.mx[wave][fr] = mx;
        if (lane == 0) {
            s.lo[wave] = lo;
            s.hi[wave] = hi;
        }
        lds_barrier();
        mx = max(max(s.mx[0][fr], s.mx[1][fr]), max(s.mx[2][fr], s.mx[3][fr]));
        lo = min(min(s.lo[0], s.lo[1]), min(s.lo[2], s.lo[3]));
        hi = max(max(s.hi[0], s.hi[1]), max(s.hi[2], s.hi[3]));
        const int digits = __builtin_amdgcn_readfirstlane(hi <= lo ? 2 : 2 + (hi - lo + 7) / 8);   // a span where nothing counts has lo > hi

        int sum = 0;
        i64 xs = 0;
        unsigned pk[MAX_DIGITS][4];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            int w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = 4 * ks + j;
                w[j] = live >> i & 1 ? weight(s, unsigned(mx) - unsigned(sc[i])) : 0;
                sum += w[j];
            }
            if (digits <= 3) {
                unsigned y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int f = min(int((evw[ks] >> (8 * j)) & 255), TOP_SHIFT);
                    const int x = -int(unsigned(w[j]) << ((f - lo) & 31));
                    if (PL == 2) xs += x;
                    y[j] = unsigned(x) + 0x8080u;
                }
                pk[0][ks] = pk[1][ks] = pk[2][ks] = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    pk[0][ks] |= (y[j] & 255) << (8 * j);
                    pk[1][ks] |= (y[j] >> 8 & 255) << (8 * j);
                    pk[2][ks] |= (y[j] >> 16 & 255) << (8 * j);
                }
                pk[0][ks] ^= 0x80808080u;
                pk[1][ks] ^= 0x80808080u;
                // with two digits the third is the sign of the second: it is not used
            } else {
#pragma unroll
                for (int t = 0; t < MAX_DIGITS; ++t) pk[t][ks] = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int f = min(int((evw[ks] >> (8 * j)) & 255), TOP_SHIFT);
                    i64 x = -i64(u64(unsigned(w[j])) << ((f - lo) & 63));
                    if (PL == 2) xs += x;
#pragma unroll
                    for (int t = 0; t < MAX_DIGITS; ++t) {
                        const int b = int(int8_t(x));
                        pk[t][ks] |= unsigned(b & 255) << (8 * j);
                        x = (x - b) >> 8;
                    }
                }
            }
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (PL == 2) {
            xs += shfl_xor64(xs, 16);
            xs += shfl_xor64(xs, 32);
        }
        if (fg == 0) {
            s.sum[wave][fr] = sum;
            if (PL == 2) s.x[wave][fr] = xs;
        }
#pragma unroll
        for (int t = 0; t < MAX_DIGITS; ++t)
            if (t < digits) *reinterpret_cast<uint4*>(&s.p[t][fr][64 * wave + 16 * fg]) = make_uint4(pk[t][0], pk[t][1], pk[t][2], pk[t][3]);
        lds_barrier();
        sum = s.sum[0][fr] + s.sum[1][fr] + s.sum[2][fr] + s.sum[3][fr];
        if (PL == 2) xs = s.x[0][fr] + s.x[1][fr] + s.x[2][fr] + s.x[3][fr];
        if (!EARLY) load_values();

        i64 O[NS][4];
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) O[i][j] = 0;
        for (int t = digits - 1; t >= 0; --t) {
            v4i pb[4];
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) pb[kt] = *reinterpret_cast<const v4i*>(&s.p[t][fr][64 * kt + 16 * fg]);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                v4i h = {0, 0, 0, 0}, l = {0, 0, 0, 0};
#pragma unroll
                for (int kt = 0; kt < 4; ++kt) {
                    h = __builtin_amdgcn_mfma_i32_16x16x64_i8(vv[i][kt][0], pb[kt], h, 0, 0, 0);
                    if constexpr (PL == 2) l = __builtin_amdgcn_mfma_i32_16x16x64_i8(vv[i][kt][1], pb[kt], l, 0, 0, 0);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) O[i][j] = O[i][j] * 256 + (PL == 1 ? h[j] : 256 * h[j] + l[j]);
            }
        }
        if (!mine) {
            // fall through to the barrier-free end of the loop
        } else {
            const double inv = 1.0 / double(max(sum, 1));
            const bool only = u1 - u0 == 1;
            const size_t at = (size_t(row) * a.Hq + qh) * a.spans + u;
            unsigned big = 0;
            if (!only && wave == 0 && fg == 0) a.stat[at] = make_int2(mx, sum);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const int d = 16 * (wave + 4 * i) + 4 * fg;
                if (wave + 4 * i >= pieces) break;
                int r[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const i64 num = -(O[i][j] + (PL == 2 ? 128 * xs : 0));
                    r[j] = sum ? div_sat(i64(u64(num) << lo) + (sum >> 1), sum, inv) : 0;
                    big = max(big, uabs(r[j]));
                }
                int32_t* y = only ? a.out + size_t(row) * a.ldo + size_t(qh) * D + d : a.part + at * D + d;
                *reinterpret_cast<int4*>(y) = make_int4(r[0], r[1], r[2], r[3]);
            }
            if (only && a.rowmax) {
                big = max(big, unsigned(__shfl_xor(int(big), 16)));
                big = max(big, unsigned(__shfl_xor(int(big), 32)));
                if (fg == 0 && big) atomicMax(a.rowmax + row, big);
            }
        }
    }
}

// ---------------------------------------------------------------- the join

constexpr int JOIN_CHUNK = 1024;   // spans whose weights stand in LDS at a time
constexpr int JOIN_D = 32;         // dimensions of a block: eight lanes of four, 32 spans at a time

__device__ __forceinline__ i64 join_weight(const KvAttnArgs& a, int mx, int2 st) {
    const unsigned d = unsigned(mx) - unsigned(st.x);
    if (st.y == 0 || d >= (1u << 20)) return 0;
    const i64 t = a.Lexp[d >> 10], t1 = a.Lexp[(d >> 10) + 1];
    return ((t + (((t1 - t) * i64(d & 1023)) >> 10) + 64) >> 7) * st.y;
}

__global__ void __launch_bounds__(256) kv_join_kernel(KvAttnArgs a) {
    __shared__ int mxs[4];
    __shared__ i64 sums[4];
    __shared__ int g[JOIN_CHUNK];
    __shared__ i64 acc[4][8][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int D = a.c.D, parts = (D + JOIN_D - 1) / JOIN_D, qh = blockIdx.x / parts, d0 = (blockIdx.x % parts) * JOIN_D, row = blockIdx.y;
    const int n = int(min(i64(max(min(a.len[row], a.max_len), 0)), i64(a.width) << a.c.lp)), first = a.window > 0 ? max(0, n - a.window) : 0;
    const int u0 = first / KV_SPAN, u1 = (n + KV_SPAN - 1) / KV_SPAN;
    if (u1 - u0 <= 1) return;      // the first kernel has written the row
    const size_t at = (size_t(row) * a.Hq + qh) * a.spans;
    int mx = INT_MIN;
    for (int u = u0 + tid; u < u1; u += 256) {
        const int2 st = a.stat[at + u];
        if (st.y) mx = max(mx, st.x);
    }
    for (int d = 32; d; d >>= 1) mx = max(mx, __shfl_xor(mx, d));
    if (lane == 0) mxs[wave] = mx;
    __syncthreads();
    mx = max(max(mxs[0], mxs[1]), max(mxs[2], mxs[3]));
    i64 G = 0;
    for (int u = u0 + tid; u < u1; u += 256) G += join_weight(a, mx, a.stat[at + u]);
    for (int d = 32; d; d >>= 1) G += shfl_xor64(G, d);
    if (lane == 0) sums[wave] = G;
    __syncthreads();
    G = sums[0] + sums[1] + sums[2] + sums[3];
    const int h = max(0, 64 - __clzll((long long)G) - 30);
    const i64 half = (i64(1) << h) >> 1;
    const int dl = 4 * (tid & 7), k0 = tid >> 3;
    const bool in = d0 + dl < D;
    i64 x[4] = {0, 0, 0, 0}, T = 0;
    for (int c = u0; c < u1; c += JOIN_CHUNK) {
        const int m = min(JOIN_CHUNK, u1 - c);
        __syncthreads();
        for (int k = tid; k < m; k += 256) g[k] = int((join_weight(a, mx, a.stat[at + c + k]) + half) >> h);
        __syncthreads();
        for (int k = k0; k < m; k += 32) {
            const i64 w = g[k];
            if (in) {
                const int4 v = *reinterpret_cast<const int4*>(a.part + (at + c + k) * D + d0 + dl);
                x[0] += w * v.x;
                x[1] += w * v.y;
                x[2] += w * v.z;
                x[3] += w * v.w;
            }
            T += w;
        }
    }
#pragma unroll
    for (int d = 8; d < 64; d <<= 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] += shfl_xor64(x[j], d);
        T += shfl_xor64(T, d);
    }
    if (lane == 0) sums[wave] = T;   // its last readers are two barriers back
    if (lane < 8)
        for (int j = 0; j < 4; ++j) acc[wave][lane][j] = x[j];
    __syncthreads();
    if (tid >= 32) return;
    T = sums[0] + sums[1] + sums[2] + sums[3];
    const int d = d0 + tid;
    if (d >= D) return;
    const i64 X = acc[0][tid >> 2][tid & 3] + acc[1][tid >> 2][tid & 3] + acc[2][tid >> 2][tid & 3] + acc[3][tid >> 2][tid & 3];
    const int r = T ? div_sat(X + (T >> 1), T, 1.0 / double(T)) : 0;
    a.out[size_t(row) * a.ldo + size_t(qh) * D + d] = r;
    if (a.rowmax && r) atomicMax(a.rowmax + row, uabs(r));
}

template <int PL>
void launch_spans(hipStream_t st, const KvAttnArgs& a, dim3 g) {
    switch ((a.c.D + 63) / 64) {
        case 1: kv_attn_kernel<1, PL><<<g, 256, 0, st>>>(a); break;
        case 2: kv_attn_kernel<2, PL><<<g, 256, 0, st>>>(a); break;
        case 3: kv_attn_kernel<3, PL><<<g, 256, 0, st>>>(a); break;
        default: kv_attn_kernel<4, PL><<<g, 256, 0, st>>>(a);
    }
}

}  // namespace

hipError_t launch_kv_attention(hipStream_t st, const KvAttnArgs& a) {
    // blocks a sequence and head: every span one, while that is no more than KV_BLOCKS in all; a block then takes every z-th span
    constexpr int KV_BLOCKS = 8192;
    const int heads = a.c.heads * a.qtiles;
    const int split = std::max(1, std::min(a.spans, KV_BLOCKS / std::max(1, heads * a.rows)));
    const dim3 g(heads, a.rows, split);
    if (a.c.planes == 1) launch_spans<1>(st, a, g);
    else launch_spans<2>(st, a, g);
    if (hipError_t e = hipGetLastError()) return e;
    if (a.spans > 1) kv_join_kernel<<<dim3(a.Hq * ((a.c.D + JOIN_D - 1) / JOIN_D), a.rows), 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace vk
