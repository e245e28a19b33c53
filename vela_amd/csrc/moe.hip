// A mixture-of-experts layer for few tokens: the router (vgemm_moe_route, one or two kernels) and the chosen experts' feed-forward on
// 4-bit weights with its combination (vgemm_moe: up with GEGLU, down, and the sum over a token's choices).
#include <algorithm>
#include <cmath>

#include "dispatch_rules.h"
#include "moe.h"
#include "norm_math.h"

namespace vk {

// ---------------------------------------------------------------- router

// exp table lookup of the attention: 0 from 2^20 on, else linear between entries z >> 10 and (z >> 10) + 1
__device__ __forceinline__ i64 moe_lutexp(uint32_t z, const i64* L) {
    if (z >= (16u << 16)) return 0;
    const i64 a = L[z >> 10], b = L[(z >> 10) + 1];
    return a + (((b - a) * i64(z & 1023)) >> 10);
}

__device__ __forceinline__ int wave_sum32(int v) {
    v += dpp32<DPP_XOR1>(v);
    v += dpp32<DPP_XOR2>(v);
    v += dpp32<DPP_HALF_MIRROR>(v);
    v += dpp32<DPP_MIRROR>(v);
    return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) + __builtin_amdgcn_readlane(v, 48);
}

__device__ __forceinline__ int dot16(const v4i& a, const v4i& b, int c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_sdot4(a[i], b[i], c, false);
    return c;
}

constexpr int ROUTE_THREADS = 1024;
constexpr int EXP_N = 1025;
constexpr int ROUTE_RANK = ROUTE_THREADS / 8;   // experts whose places are counted by all threads: 512 took 12 us so, 16 choices 2
constexpr int ROUTE_ONE = 1 << 18;   // bytes of weights one block a token reads

// sum over the wave of values whose total stays below 2^63
__device__ __forceinline__ i64 wave_sum64(i64 v) {
    for (int d = 32; d; d >>= 1) v += i64(__shfl_xor((long long)v, d));
    return v;
}

// floor(2^62 / s): from a quotient of doubles, whose error is below one for s >= 2^20 (quotients below 2^42)
__device__ __forceinline__ u64 route_recip(u64 s) {
    const u64 one = u64(1) << 62;
    if (s < (1u << 20)) return s ? one / s : 0;
    u64 q = u64(0x1p62 / double(s));
    i64 r = i64(one - q * s);
    if (r < 0) {
        --q;
        r += i64(s);
    }
    return r >= i64(s) ? q + 1 : q;
}

// The router moves the layer's int8 weights once a token or four, which is little beside its latency: 3.5 us for 8 experts x 1024, 6.1 for 64 x
// 2048, 9.2 for 16 tokens of 128 x 2048 in one kernel.
//
// Logits of T tokens and eight experts a block, two a wave. Plane sums stay below 16384 * 2^14 = 2^28.
constexpr int LOGITS_X = 8;
template <int T>
__global__ void __launch_bounds__(256) moe_logits_kernel(RouteArgs a, int M) {
    touch_args<int(sizeof(RouteArgs) + 4)>();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), x0 = int(blockIdx.y) * LOGITS_X + 2 * wave, t0 = int(blockIdx.x) * T;
    if (x0 >= a.experts) return;
    int ch[T][2], cl[T][2];
#pragma unroll
    for (int t = 0; t < T; ++t) ch[t][0] = ch[t][1] = cl[t][0] = cl[t][1] = 0;
    const int8_t *w0 = a.W + size_t(x0) * a.ldw, *w1 = a.W + size_t(min(x0 + 1, a.experts - 1)) * a.ldw;
    const int x = x0 + (lane & 1), t = t0 + (lane >> 1);   // of the logit this lane writes
    const bool mine = lane < 2 * T && x < a.experts && t < M;
    const int4 cst = mine ? a.cst[x] : make_int4(0, 0, 0, 0);
    const int e = mine && a.e ? a.e[t] : 0;
#pragma unroll 4
    for (int k = lane * 16; k < a.K; k += 1024) {
        const v4i u0 = *reinterpret_cast<const v4i*>(w0 + k), u1 = *reinterpret_cast<const v4i*>(w1 + k);
#pragma unroll
        for (int i = 0; i < T; ++i) {
            const size_t row = size_t(min(t0 + i, M - 1)) * a.ld8 + k;
            const v4i h = *reinterpret_cast<const v4i*>(a.hi + row);
            ch[i][0] = dot16(h, u0, ch[i][0]);
            ch[i][1] = dot16(h, u1, ch[i][1]);
            if (a.lo) {
                const v4i l = *reinterpret_cast<const v4i*>(a.lo + row);
                cl[i][0] = dot16(l, u0, cl[i][0]);
                cl[i][1] = dot16(l, u1, cl[i][1]);
            }
        }
    }
    i64 acc = 0;
#pragma unroll
    for (int i = 0; i < 2 * T; ++i) {
        const int sh = wave_sum32(ch[i >> 1][i & 1]), sl = a.lo ? wave_sum32(cl[i >> 1][i & 1]) : 0;
        if (lane == i) acc = a.lo ? 256LL * sh + sl : i64(sh);
    }
    if (mine) a.logits[size_t(t) * a.experts + x] = w4_requant(acc, a.lo != nullptr, cst, e);
}

// A block per token, which computes the logits, a wave U experts at once, or (U = 0) finds them in a.logits
template <int U>
__global__ void __launch_bounds__(ROUTE_THREADS) moe_route_kernel(RouteArgs a) {
    touch_args<int(sizeof(RouteArgs))>();
    __shared__ __align__(16) int s_z[MOE_EXPERTS + 16];
    __shared__ int s_h[MOE_EXPERTS], s_l[MOE_EXPERTS];
    __shared__ int s_top[MOE_TOPK];
    __shared__ i64 s_exp[EXP_N];
    __shared__ u64 s_sum[ROUTE_THREADS / 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = blockIdx.x;
    const int8_t* hi = a.hi + size_t(t) * a.ld8;
    const int8_t* lo = a.lo ? a.lo + size_t(t) * a.ld8 : nullptr;
    const int e = a.e ? a.e[t] : 0, i = threadIdx.x;
    // on their way while the products run: the constants of expert i, entry i of the table
    const int4 cst = U && i < a.experts ? a.cst[i] : make_int4(0, 0, 0, 0);
    const int found = !U && i < a.experts ? a.logits[size_t(t) * a.experts + i] : 0;
    const long long ex = a.Lexp[i], ex_last = a.Lexp[EXP_N - 1];
    static_assert(EXP_N == ROUTE_THREADS + 1, "an entry a thread, and the last");
    if constexpr (U > 0) for (int x0 = wave * U; x0 < a.experts; x0 += ROUTE_THREADS / 64 * U) {
        int ch[U], cl[U];
#pragma unroll
        for (int u = 0; u < U; ++u) ch[u] = cl[u] = 0;
#pragma unroll 2
        for (int k = lane * 16; k < a.K; k += 1024) {
            const v4i h = *reinterpret_cast<const v4i*>(hi + k);
            const v4i l = lo ? *reinterpret_cast<const v4i*>(lo + k) : v4i{0, 0, 0, 0};
            v4i w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = *reinterpret_cast<const v4i*>(a.W + size_t(min(x0 + u, a.experts - 1)) * a.ldw + k);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                ch[u] = dot16(h, w[u], ch[u]);
                if (lo) cl[u] = dot16(l, w[u], cl[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int sh = wave_sum32(ch[u]), sl = lo ? wave_sum32(cl[u]) : 0;
            const int x = x0 + u;
            if (lane == 0 && x < a.experts) {
                s_h[x] = sh;
                s_l[x] = sl;
            }
        }
    }
    s_exp[i] = ex;
    if (i == 0) s_exp[EXP_N - 1] = ex_last;
    if (i < 16) s_z[a.experts + i] = INT_MIN;
    if constexpr (U > 0) __syncthreads();
    const int z = i >= a.experts ? 0 : (U ? w4_requant(lo ? 256LL * s_h[i] + s_l[i] : i64(s_h[i]), lo != nullptr, cst, e) : found);
    if (i < a.experts) {
        s_z[i] = z;
        if (U && a.logits) a.logits[size_t(t) * a.experts + i] = z;
    }
    __syncthreads();
    if (a.experts > ROUTE_RANK) {   // choice by choice: the first wave's largest, of equal ones the lowest index
        if (wave == 0) {
            uint32_t key[MOE_EXPERTS / 64];
            unsigned left = 0;          // bit s: expert 64 s + lane is there and not chosen yet
#pragma unroll
            for (int s = 0; s < MOE_EXPERTS / 64; ++s) {
                const int x = 64 * s + lane;
                key[s] = x < a.experts ? uint32_t(s_z[x]) ^ 0x80000000u : 0u;
                left |= x < a.experts ? 1u << s : 0u;
            }
            for (int r = 0; r < a.topk; ++r) {
                uint32_t best = 0;
                int at = -1;
#pragma unroll
                for (int s = MOE_EXPERTS / 64 - 1; s >= 0; --s) {
                    const bool take = (left >> s & 1) && key[s] >= best;
                    best = take ? key[s] : best;
                    at = take ? s : at;
                }
                const uint32_t m = wave_umax32(best);
                const int x = int(~wave_umax32(best == m && at >= 0 ? ~unsigned(64 * at + lane) : 0u));
                if (lane == (x & 63)) left &= ~(1u << (x >> 6));
                if (lane == 0) {
                    a.idx[size_t(t) * a.topk + r] = x;
                    s_top[r] = int(m ^ 0x80000000u);
                }
            }
        }
    } else {   // an expert's place: the logits before it in falling order; eight threads an expert, 16 logits a step (INT_MIN behind the
               // last expert counts for nobody)
        const int x = i >> 3;
        if (x < a.experts) {
            const int zx = s_z[x];
            int rank = 0;
            for (int j = 16 * (i & 7); j < a.experts; j += 128) {
#pragma unroll
                for (int k = 0; k < 16; k += 4) {
                    const int4 o = *reinterpret_cast<const int4*>(&s_z[j + k]);
                    rank += (o.x > zx || (o.x == zx && j + k < x)) ? 1 : 0;
                    rank += (o.y > zx || (o.y == zx && j + k + 1 < x)) ? 1 : 0;
                    rank += (o.z > zx || (o.z == zx && j + k + 2 < x)) ? 1 : 0;
                    rank += (o.w > zx || (o.w == zx && j + k + 3 < x)) ? 1 : 0;
                }
            }
            for (int d = 1; d < 8; d <<= 1) rank += __shfl_xor(rank, d);
            if ((i & 7) == 0 && rank < a.topk) {
                a.idx[size_t(t) * a.topk + rank] = x;
                s_top[rank] = zx;
            }
        }
    }
    __syncthreads();
    const uint32_t top = uint32_t(s_top[0]);
    const i64 mine = i < a.topk ? moe_lutexp(top - uint32_t(s_top[i]), s_exp) : 0;   // the i-th choice's
    const int members = a.renorm ? a.topk : a.experts;
    u64 sum = 0;   // of this wave's members; the chosen ones are all in the first wave, and each of its lanes has their sum
    if (64 * wave < members) {
        sum = u64(wave_sum64(a.renorm ? mine : (i < a.experts ? moe_lutexp(top - uint32_t(z), s_exp) : 0)));
        if (!a.renorm && lane == 0) s_sum[wave] = sum;
    }
    if (!a.renorm) __syncthreads();
    if (i < a.topk) {
        if (!a.renorm) {
            sum = 0;
            for (int w = 0; 64 * w < members; ++w) sum += s_sum[w];
        }
        const u64 p = (u64(mine) * route_recip(sum) + (u64(1) << 46)) >> 47;
        a.p[size_t(t) * a.topk + i] = int(min(p, u64(32767)));
    }
}

hipError_t launch_moe_route(hipStream_t st, const RouteArgs& a, int M) {
    const int waves = ROUTE_THREADS / 64;
    // One block reads 256 x 7168 in 26.0 us, 512 x 4096 in 29.2: with room for the logits a kernel before computes them on many CUs, 3.7 + 4.8
    // and 3.2 + 4.7 us. 128 x 2048 takes 6.8 us in one kernel and 3.1 + 3.1 in two for one token, 7.4 and 4.1 + 4.0 for sixteen, 129 x 2048 8.9
    // and 3.1 + 4.8: the tokens, each with a block of its own either way, change little of it.
    if (a.logits && (long long)a.experts * a.K > ROUTE_ONE) {
        if (M < 4) hipLaunchKernelGGL(moe_logits_kernel<1>, dim3(M, cdiv(a.experts, LOGITS_X)), dim3(256), 0, st, a, M);
        else hipLaunchKernelGGL(moe_logits_kernel<4>, dim3(cdiv(M, 4), cdiv(a.experts, LOGITS_X)), dim3(256), 0, st, a, M);
        if (hipError_t e = hipGetLastError()) return e;
        hipLaunchKernelGGL(moe_route_kernel<0>, dim3(M), dim3(ROUTE_THREADS), 0, st, a);
        return hipGetLastError();
    }
    if (a.experts <= waves) hipLaunchKernelGGL(moe_route_kernel<1>, dim3(M), dim3(ROUTE_THREADS), 0, st, a);
    else if (a.experts <= 4 * waves) hipLaunchKernelGGL(moe_route_kernel<4>, dim3(M), dim3(ROUTE_THREADS), 0, st, a);
    else hipLaunchKernelGGL(moe_route_kernel<8>, dim3(M), dim3(ROUTE_THREADS), 0, st, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------- experts
//
// Both products are cut into items (row tile of at most 16 of an expert's pairs, segment of `js` column tiles), a block each,
// which computes as w4_kernel.h says. Bound by the chosen experts' weights where there are many (16 tokens x 8 of 128, 2048 x 768, groups of
// 64: up 29.4 us for 135 MB, down 19.0 for 67) or they are large (2 tokens x 8 of 256, 7168 x 2048: up 47.7 us for 240 MB, down 26.8 for
// 120), else by a block's chain of latencies (one token x 2 of 8, 1024 x 2048: 5.7 and 5.6 us).

// Row tile `tile` of the pairs sorted by expert: its expert and rows; n = 0 past the last tile. pair[]: the tile's pairs, the same in every
// block (in the order of the pairs), written by the first wave. Every block finds its own: a kernel that did it once took 2 to 5 us.
struct MoeTile {
    int x, n;
};
struct MoeFind {
    int idx[MOE_PAIRS], cnt[MOE_EXPERTS];
};
__device__ __forceinline__ MoeTile moe_find(const MoeArgs& a, int tile, MoeFind& T, int* pair) {
    const int pairs = a.M * a.topk, lane = threadIdx.x & 63;
    if (a.M == 1) {   // one token: its choices are the tiles
        const int x = a.idx[tile];
        if (threadIdx.x == 0) pair[0] = tile;
        return {x, unsigned(x) < unsigned(a.experts) ? 1 : 0};
    }
    for (int i = threadIdx.x; i < a.experts; i += blockDim.x) T.cnt[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
        const int x = a.idx[i];
        T.idx[i] = x;
        if (unsigned(x) < unsigned(a.experts)) atomicAdd(&T.cnt[x], 1);
    }
    __syncthreads();
    const u64 before = (u64(1) << lane) - 1;
    for (int c = 0; c < a.experts; c += 64) {
        const int n = c + lane < a.experts ? T.cnt[c + lane] : 0, nt = (n + 15) >> 4;
        int first = 0, all = 0;   // tiles of the lanes before, of all: bit by bit of the counts
#pragma unroll
        for (int bit = 0; (1 << bit) <= MOE_PAIRS / 16; ++bit) {
            const u64 m = __builtin_amdgcn_ballot_w64((nt >> bit) & 1);
            first += __builtin_popcountll(m & before) << bit;
            all += __builtin_popcountll(m) << bit;
        }
        if (tile >= all) {
            tile -= all;
            continue;
        }
        const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(tile >= first && tile < first + nt));
        const int x = c + l, r0 = 16 * (tile - __builtin_amdgcn_readlane(first, l)), rows = min(16, __builtin_amdgcn_readlane(n, l) - r0);
        if (threadIdx.x < 64) {
            for (int i = 0, at = -r0; i < pairs; i += 64) {
                const bool hit = i + lane < pairs && T.idx[i + lane] == x;
                const u64 m = __builtin_amdgcn_ballot_w64(hit);
                const int r = at + __builtin_popcountll(m & before);
                if (hit && r >= 0 && r < rows) pair[r] = i + lane;
                at += __builtin_popcountll(m);
            }
        }
        return {x, rows};
    }
    return {-1, 0};
}

// the shift of pair pr's row v: of the largest of its segments' maxima
__device__ __forceinline__ int moe_shift(const MoeArgs& a, int pr, int lane) {
    const uint32_t* vm = a.vmax + size_t(pr) * a.up_segs;
    uint32_t m = 0;
    for (int k = lane; k < a.up_segs; k += 64) m = max(m, vm[k]);
    return rowexp_u32(wave_umax32(m));
}

constexpr int MOE_JS = 24;   // column tiles a segment has at most: 48 KiB of sums

// DOWN = false: rows of the tokens' planes, GEGLU to v [pairs x F], and max |v| of the segment. DOWN = true: rows v, quantised by the
// largest of their segments' maxima, y [pairs x MOE_COLS].
template <bool DOWN, int P, int G>
__global__ void __launch_bounds__(1024) moe_kernel(MoeArgs a, int js, int rows_lds) {
    constexpr int DEPTH = DOWN ? 6 : 4;   // 2 experts, 8 tokens, 4096 x 4480: up 13.3 us with 6, 12.6 with 4; down 27.6 against 28.5 for 43 tokens with 6
    touch_args<int(sizeof(MoeArgs) + 8)>();
    extern __shared__ uint4 s_dyn[];
    __shared__ uint32_t s_max[16];
    __shared__ int s_se[16], s_pair[16];
    __shared__ MoeFind s_find;
    const MoeTile mt = moe_find(a, blockIdx.y, s_find, s_pair);
    const int x = __builtin_amdgcn_readfirstlane(mt.x), n = __builtin_amdgcn_readfirstlane(mt.n);
    if (n == 0) return;
    const W4View& W = DOWN ? a.down : a.up;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = __builtin_amdgcn_readfirstlane(blockDim.x >> 6);
    const int ctb = DOWN ? a.col0 / 16 : 0, CT = DOWN ? (a.cols + 15) / 16 : W.CT, KT = W.KT, F = a.down.K;
    const int ct0 = ctb + int(blockIdx.x) * js, tiles = min(js, CT - int(blockIdx.x) * js);
    uint8_t* lds = reinterpret_cast<uint8_t*>(s_dyn);
    unsigned long long* sums = reinterpret_cast<unsigned long long*>(lds + rows_lds);
    int32_t* lut = reinterpret_cast<int32_t*>(sums + js * 256);   // of the gate
    const size_t at = x * (DOWN ? a.down_stride : a.up_stride);
    const W4Columns from{W.q + at + size_t(ct0) * KT * 1024, W.s + at + size_t(ct0) * KT * (4096 / G), KT};
    // as many tiles of K a chunk as the staging area holds of n rows, chunks of even size
    W4Chunks ch;
    ch.kc = __builtin_amdgcn_readfirstlane(min(KT, max(1, (w4_div(rows_lds >> 4, n * P) - 1) >> 3)));
    ch.n = 1;
    if (ch.kc < KT) {
        ch.n = __builtin_amdgcn_readfirstlane(w4_div(KT + ch.kc - 1, ch.kc));
        ch.kc = __builtin_amdgcn_readfirstlane(w4_div(KT + ch.n - 1, ch.n));
        ch.n = __builtin_amdgcn_readfirstlane(w4_div(KT + ch.kc - 1, ch.kc));
    }
    W4Ring<G, DEPTH> ring;
    ring.start(from, KT, tiles, 0, ch, lane, wave, waves);
    for (int k = threadIdx.x; k < tiles * 256; k += blockDim.x) sums[k] = 0;
    if (int(threadIdx.x) < n) s_max[threadIdx.x] = 0;
    // two columns a thread; its first two's constants are asked for here, in the down product, which has no registers for them, at its
    // end. The barrier that publishes the pairs waits for them, the first tiles and the gate's table, before the rows are asked for; so
    // does the one between chunks for the next chunk's first tiles.
    const int outs = tiles * n * 8, TR = n <= 4 ? 4 : 16;
    const int4* cst = W.cst + size_t(x) * W.CT * 16;
    int4 c0, c1;
    const auto fetch = [&](int k) {
        const int col = (ct0 + w4_div(k >> 3, n)) * 16 + 2 * (k & 7);
        c0 = cst[col];
        c1 = cst[col + 1];
    };
    if (!DOWN && int(threadIdx.x) < outs) fetch(threadIdx.x);
    if constexpr (!DOWN) w4_load_lut(lut, a.Lphi, lane, wave, waves);
    __syncthreads();
    if constexpr (!DOWN)
        if (int(threadIdx.x) < n) s_se[threadIdx.x] = a.e ? a.e[w4_div(s_pair[threadIdx.x], a.topk)] : 0;
    [[maybe_unused]] const auto shift = [&](int r) {
        const int e = moe_shift(a, s_pair[r], lane);
        if (lane == 0) s_se[r] = e;
        return e;
    };
    for (int c = 0;;) {
        const int k0 = c * ch.kc, kc = min(ch.kc, KT - k0);
        if constexpr (DOWN)
            w4_stage_x32(lds, ch.ld(), n, n, k0, kc, F, a.v, [&](int r) { return unsigned(s_pair[r]) * unsigned(F); }, [&](int r) { return c ? s_se[r] : shift(r); }, lane, wave, waves);
        else
            w4_stage<P>(lds, ch.ld(), n, n, k0, kc, a.Kp16, a.hi, a.lo, [&](int r) { return unsigned(w4_div(s_pair[r], a.topk)) * unsigned(a.ld8); });
        __syncthreads();
        if (n <= 4) w4_share<1, 1, P, G>(ring, lds, ch.ld(), n, n, [](int) { return 0; }, sums, lane);
        else w4_share<1, 4, P, G>(ring, lds, ch.ld(), n, n, [](int) { return 0; }, sums, lane);
        if (++c == ch.n) break;
        ring.start(from, KT, tiles, c, ch, lane, wave, waves);
        __syncthreads();
    }
    if (DOWN && int(threadIdx.x) < outs) fetch(threadIdx.x);
    __syncthreads();
    for (int k = threadIdx.x; k < outs; k += blockDim.x) {
        const int c = w4_div(k >> 3, n), t = (k >> 3) - c * n, col = (ct0 + c) * 16 + 2 * (k & 7), pr = s_pair[t];
        if (k != int(threadIdx.x)) fetch(k);
        const longlong2 v = *reinterpret_cast<const longlong2*>(&sums[(c * TR + t) * 16 + 2 * (k & 7)]);
        const int y0 = w4_requant(v.x, P == 2, c0, s_se[t]), y1 = w4_requant(v.y, P == 2, c1, s_se[t]);
        if constexpr (DOWN) {
            *reinterpret_cast<int2*>(a.y + size_t(pr) * MOE_COLS + (col - a.col0)) = make_int2(y0, y1);   // columns past N are not read
        } else if (col < W.N) {
            const int y = geglu_exact(y0, y1, lut);
            a.v[size_t(pr) * F + (col >> 1)] = y;
            atomicMax(&s_max[t], uabs(y));
        }
    }
    if constexpr (!DOWN) {
        __syncthreads();
        if (int(threadIdx.x) < n) a.vmax[size_t(s_pair[threadIdx.x]) * a.up_segs + blockIdx.x] = s_max[threadIdx.x];
    }
}

// Column tiles c of the down products of several pairs: pair c / tiles, the block's column tile c % tiles
struct MoeColumns {
    const uint8_t *q, *s;      // the block's first column tile in expert 0
    size_t stride;
    int KT, tiles;
    int x;                     // lane l: the expert of pair l
    __device__ __forceinline__ int pair(int c) const { return tiles == 1 ? c : __builtin_amdgcn_readfirstlane(w4_div(c, tiles)); }
    template <int G>
    __device__ __forceinline__ void at(int c, int k, const uint8_t*& qc, const uint8_t*& sc) const {
        const int j = pair(c);
        const size_t off = __builtin_amdgcn_readlane(x, j) * stride, tile = size_t(c - j * tiles) * KT + k;
        qc = q + off + tile * 1024;
        sc = s + off + tile * (4096 / G);
    }
};

// Of at most MOE_FEW pairs: all their down products and the sums over the tokens' choices, a segment of column tiles a block, whose
// waves share the tiles of all the pairs evenly. The rows v stand in LDS whole, [plane][pair]. A pair without an expert goes through
// expert 0's tiles and is left out of the sums.
constexpr int MOE_FEW = 24;
template <int G>
__global__ void __launch_bounds__(1024) moe_down_few_kernel(MoeArgs a, int js, int rows_lds) {
    constexpr int DEPTH = 6;   // one token, 4096 x 1536: 5.8 us, 8.5 with 4
    touch_args<int(sizeof(MoeArgs) + 8)>();
    extern __shared__ uint4 s_dyn[];
    __shared__ int s_se[MOE_FEW], s_x[MOE_FEW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = __builtin_amdgcn_readfirstlane(blockDim.x >> 6);
    const W4View& W = a.down;
    const int KT = W.KT, ct0 = int(blockIdx.x) * js, tiles = min(js, W.CT - ct0), F = W.K, ld = KT * 128 + 16, pairs = a.M * a.topk;
    uint8_t* lds = reinterpret_cast<uint8_t*>(s_dyn);
    unsigned long long* sums = reinterpret_cast<unsigned long long*>(lds + rows_lds);   // [pair][column tile][4][16]: the first of the four rows
    unsigned long long* out = sums + pairs * js * 64;                                       // [token][column]
    const int xl = lane < pairs ? a.idx[lane] : -1;
    const MoeColumns from{W.q + size_t(ct0) * KT * 1024, W.s + size_t(ct0) * KT * (4096 / G), a.down_stride, KT, tiles, unsigned(xl) < unsigned(a.experts) ? xl : 0};
    W4Ring<G, DEPTH, MoeColumns> ring;
    ring.start(from, KT, pairs * tiles, 0, W4Chunks{KT, 1}, lane, wave, waves);
    for (int i = threadIdx.x; i < pairs * js * 64 + a.M * js * 16; i += blockDim.x) sums[i] = 0;
    if (int(threadIdx.x) < pairs) s_x[threadIdx.x] = xl;   // the first wave
    const auto shift = [&](int r) {
        const int e = moe_shift(a, r, lane);
        if (lane == 0) s_se[r] = e;
        return e;
    };
    w4_stage_x32(lds, ld, pairs, pairs, 0, KT, F, a.v, [&](int r) { return unsigned(r) * unsigned(F); }, shift, lane, wave, waves);
    __syncthreads();
    // a pair's column a thread, then a token's; what the thread's first ones need besides the sums comes while the products run (before the
    // rows v it would hold those up: 5.0 -> 6.8 us for one token, 1024 x 2048)
    const int items = pairs * tiles * 16, outs = a.M * js * 16;
    int4 c;
    int p, res;
    const auto fetch = [&](int i) {
        const int jj = w4_div(i >> 4, tiles), col = (ct0 + (i >> 4) - jj * tiles) * 16 + (i & 15);
        c = unsigned(s_x[jj]) < unsigned(a.experts) ? W.cst[size_t(s_x[jj]) * W.CT * 16 + col] : make_int4(0, 0, 0, 0);
        p = a.p[jj];
    };
    const auto fetch_res = [&](int i) {
        const int tok = w4_div(i >> 4, js), ct = (i >> 4) - tok * js, col = (ct0 + ct) * 16 + (i & 15);
        res = a.R && ct < tiles && col < W.N ? a.R[size_t(tok) * a.ldy + col] : 0;
    };
    if (int(threadIdx.x) < items) fetch(threadIdx.x);
    if (int(threadIdx.x) < outs) fetch_res(threadIdx.x);
    w4_share<1, 1, 2, G>(ring, lds, ld, pairs, 1, [&](int c2) { return from.pair(c2); }, sums, lane);
    __syncthreads();
    for (int i = threadIdx.x; i < items; i += blockDim.x) {
        const int jj = w4_div(i >> 4, tiles), ct = (i >> 4) - jj * tiles;
        if (i != int(threadIdx.x)) fetch(i);
        if (unsigned(s_x[jj]) >= unsigned(a.experts)) continue;
        const int y = w4_requant(i64(sums[(i >> 4) * 64 + (i & 15)]), true, c, s_se[jj]);
        atomicAdd(&out[(w4_div(jj, a.topk) * js + ct) * 16 + (i & 15)], u64(i64(p)) * u64(i64(y)));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < outs; i += blockDim.x) {
        if (i != int(threadIdx.x)) fetch_res(i);
        const int tok = w4_div(i >> 4, js), ct = (i >> 4) - tok * js, col = (ct0 + ct) * 16 + (i & 15);
        const size_t o = size_t(tok) * a.ldy + col;
        if (ct < tiles && col < W.N) a.Y[o] = add_sat(int(rshr(i64(out[i]), 15)), res);
    }
}

// Y[t] = sat32(sat32(rshr(sum_j p y, 15)) + R[t]) over the columns of a pass, eight choices' loads in flight
__global__ void __launch_bounds__(256) moe_combine_kernel(MoeArgs a) {
    touch_args<int(sizeof(MoeArgs))>();
    const int c = int(blockIdx.x) * 256 + int(threadIdx.x), tok = blockIdx.y;
    if (c >= a.cols) return;
    const size_t o = size_t(tok) * a.ldy + a.col0 + c;
    const int res = a.R ? a.R[o] : 0;
    u64 sum = 0;
    for (int j0 = 0; j0 < a.topk; j0 += 8) {
        int y[8], p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int pr = tok * a.topk + min(j0 + j, a.topk - 1);
            y[j] = a.y[size_t(pr) * MOE_COLS + c];   // of a pair without an expert: whatever stands there, times 0
            p[j] = j0 + j < a.topk && unsigned(a.idx[pr]) < unsigned(a.experts) ? a.p[pr] : 0;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += u64(i64(p[j])) * u64(i64(y[j]));
    }
    a.Y[o] = add_sat(int(rshr(i64(sum), 15)), res);
}

// Shape of the items if the tokens choose their experts evenly: sixteen waves, a whole CU, for the down product from four pairs
// an expert on, where quantising the rows counts, else eight, two items a CU; column tiles a segment for about one item a place,
// with a margin for more experts chosen than expected (a second round of a few items costs as much as the first).
struct MoeShape {
    int waves, js;
};
static double moe_chosen(const MoeArgs& a) { return a.experts * (1.0 - std::pow(1.0 - 1.0 / a.experts, double(a.M) * a.topk)); }   // experts, expected
static MoeShape moe_shape(const MoeArgs& a, int CT, bool down) {
    const double pairs = double(a.M) * a.topk, chosen = moe_chosen(a), tiles = std::max(chosen, pairs / 16);
    const int waves = down && pairs / chosen >= 4.0 ? 16 : 8;
    return {waves, std::max(1, std::min(MOE_JS, int(std::ceil(1.1 * tiles * CT / (waves == 16 ? NCU : 2 * NCU)))))};
}

template <bool DOWN, int P, int G>
static void moe_launch(hipStream_t st, const MoeArgs& a, MoeShape sh) {
    const int CT = DOWN ? cdiv(a.cols, 16) : a.up.CT, KT = DOWN ? a.down.KT : a.up.KT, pairs = a.M * a.topk;
    // row tiles at most; of one token a tile a choice, also where an expert is chosen twice
    const int tiles = a.M == 1 ? pairs : std::min(pairs, std::min(a.experts, pairs) + pairs / 16);
    // the 64-bit sums behind the rows begin at a multiple of 16 bytes
    const int sums = sh.js * 2048, lut = DOWN ? 0 : W4_LUT_LDS, fixed = int(sizeof(MoeFind)) + 256 + sums + lut, rows = std::min(16, pairs);
    const int most = (sh.waves == 16 ? 160 << 10 : 80 << 10) - fixed;
    const int rows_lds = std::max(rows * P * 144, std::min(most & ~15, rows * P * (KT * 128 + 16)));
    hipLaunchKernelGGL((moe_kernel<DOWN, P, G>), dim3(cdiv(CT, sh.js), tiles), dim3(64 * sh.waves), rows_lds + sums + lut, st, a, sh.js, rows_lds);
}
template <int G>
static void moe_down_few(hipStream_t st, const MoeArgs& a, int js, int rows_lds) {
    const int pairs = a.M * a.topk;
    hipLaunchKernelGGL((moe_down_few_kernel<G>), dim3(cdiv(a.down.CT, js)), dim3(1024), rows_lds + pairs * js * 512 + a.M * js * 128, st, a, js, rows_lds);
}
template <bool DOWN, int P>
static void moe_product(hipStream_t st, const MoeArgs& a, int group, MoeShape sh) {
    if (group == 32) moe_launch<DOWN, P, 32>(st, a, sh);
    else if (group == 64) moe_launch<DOWN, P, 64>(st, a, sh);
    else moe_launch<DOWN, P, 128>(st, a, sh);
}

hipError_t launch_moe(hipStream_t st, const MoeArgs& args) {
    MoeArgs a = args;
    const MoeShape up = moe_shape(a, a.up.CT, false);
    a.up_segs = cdiv(a.up.CT, up.js);
    if (a.lo) moe_product<false, 2>(st, a, a.group_up, up);
    else moe_product<false, 1>(st, a, a.group_up, up);
    if (hipError_t e = hipGetLastError()) return e;
    // Few pairs, rows that fit in LDS: their products and the sums at once. One kernel against two, us:
    //   pairs  experts                 one     two
    //     8       8    4096 x 1536     8.6    12.8 + 3.9
    //    12      64    2048 x 1408     9.1     9.2 + 4.6
    //    24      64    2048 x 1408    14.1    11.1 + 4.7
    //    24      32    1024 x 512      8.6     7.0 + 3.9
    //    24       8    2048 x 2048    16.3    10.3 + 4.7
    //    24     256    4096 x 512      9.8    10.6 + 4.7
    //    32      64    2048 x 1408    17.7    14.7 + 4.7
    //    32      16    2048 x 768     11.4     7.8 + 4.0
    //    32     256    4096 x 512     12.0    11.9 + 4.7
    // A pair reads its expert's matrix by itself: not where that is more than 64 MB beyond a read each of the chosen experts (16 pairs of
    // 2 experts: 4096 x 1536, 44 MB, 11.3 against 8.8 + 4.5; 4096 x 4480, 129 MB, 24.5 against 12.8 + 4.6).
    const int pairs = a.M * a.topk, js = std::min(8, cdiv(a.down.CT, NCU)), rows = pairs * 2 * (a.down.KT * 128 + 16);
    if (pairs <= MOE_FEW && rows + pairs * js * 512 + a.M * js * 128 + 2 * MOE_FEW * 4 <= 160 << 10 && (pairs - moe_chosen(a)) * double(a.down_stride) <= 64e6) {
        if (a.group_down == 32) moe_down_few<32>(st, a, js, rows);
        else if (a.group_down == 64) moe_down_few<64>(st, a, js, rows);
        else moe_down_few<128>(st, a, js, rows);
        return hipGetLastError();
    }
    for (a.col0 = 0; a.col0 < a.down.N; a.col0 += MOE_COLS) {
        a.cols = std::min(MOE_COLS, a.down.N - a.col0);
        moe_product<true, 2>(st, a, a.group_down, moe_shape(a, cdiv(a.cols, 16), true));
        if (hipError_t e = hipGetLastError()) return e;
        hipLaunchKernelGGL(moe_combine_kernel, dim3(cdiv(a.cols, 256), a.M), dim3(256), 0, st, a);
        if (hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
}

}  // namespace vk
