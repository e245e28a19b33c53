// A mixture-of-experts layer for few tokens: the router (vgemm_moe_route, one kernel) and the chosen experts' feed-forward on
// 4-bit weights with its combination (vgemm_moe, two kernels: up with GEGLU, down with the sum over a token's choices).
#include <algorithm>

#include "dispatch_rules.h"
#include "moe.h"
#include "norm_math.h"

namespace vk {

// ---------------------------------------------------------------- router

// exp table lookup of the attention: 0 from 2^20 on, else linear between entries z >> 10 and (z >> 10) + 1
__device__ __forceinline__ i64 moe_lutexp(uint32_t z, const i64* __restrict__ L) {
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

constexpr int ROUTE_THREADS = 512;
constexpr int ROUTE_UNROLL = 4;   // experts a wave reads at once

// A block per token. Plane sums stay below 16384 * 2^14 = 2^28.
__global__ void __launch_bounds__(ROUTE_THREADS) moe_route_kernel(RouteArgs a) {
    __shared__ int s_z[MOE_EXPERTS];
    __shared__ int s_top[MOE_TOPK];
    __shared__ unsigned long long s_sum;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = blockIdx.x;
    const int8_t* hi = a.hi + size_t(t) * a.ld8;
    const int8_t* lo = a.lo ? a.lo + size_t(t) * a.ld8 : nullptr;
    const int e = a.e ? a.e[t] : 0;
    if (threadIdx.x == 0) s_sum = 0;
    for (int x0 = wave * ROUTE_UNROLL; x0 < a.experts; x0 += ROUTE_THREADS / 64 * ROUTE_UNROLL) {
        int ch[ROUTE_UNROLL], cl[ROUTE_UNROLL];
#pragma unroll
        for (int i = 0; i < ROUTE_UNROLL; ++i) ch[i] = cl[i] = 0;
        for (int k = lane * 16; k < a.K; k += 1024) {
            const v4i h = *reinterpret_cast<const v4i*>(hi + k);
            const v4i l = lo ? *reinterpret_cast<const v4i*>(lo + k) : v4i{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < ROUTE_UNROLL; ++i) {
                const v4i w = *reinterpret_cast<const v4i*>(a.W + size_t(min(x0 + i, a.experts - 1)) * a.ldw + k);
                ch[i] = dot16(h, w, ch[i]);
                if (lo) cl[i] = dot16(l, w, cl[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < ROUTE_UNROLL; ++i) {
            const int sh = wave_sum32(ch[i]), sl = lo ? wave_sum32(cl[i]) : 0;
            const int x = x0 + i;
            if (lane == 0 && x < a.experts) s_z[x] = w4_requant(lo ? 256LL * sh + sl : i64(sh), lo != nullptr, a.cst[x], e);
        }
    }
    __syncthreads();
    const int i = threadIdx.x;
    const int z = i < a.experts ? s_z[i] : 0;
    if (i < a.experts) {
        // its place: the logits before it in falling order, equal ones by their index
        int rank = 0;
        for (int j = 0; j < a.experts; ++j) {
            const int o = s_z[j];
            rank += (o > z || (o == z && j < i)) ? 1 : 0;
        }
        if (rank < a.topk) {
            a.idx[size_t(t) * a.topk + rank] = i;
            s_top[rank] = z;
        }
        if (a.logits) a.logits[size_t(t) * a.experts + i] = z;
    }
    __syncthreads();
    const uint32_t top = uint32_t(s_top[0]);
    const i64 mine = i < a.topk ? moe_lutexp(top - uint32_t(s_top[i]), a.Lexp) : 0;   // the i-th choice's
    const i64 part = a.renorm ? mine : (i < a.experts ? moe_lutexp(top - uint32_t(z), a.Lexp) : 0);
    if (part) atomicAdd(&s_sum, (unsigned long long)part);
    __syncthreads();
    if (i < a.topk) {
        const u64 sum = s_sum, r = sum ? (u64(1) << 62) / sum : 0;
        const u64 p = (u64(mine) * r + (u64(1) << 46)) >> 47;
        a.p[size_t(t) * a.topk + i] = int(min(p, u64(32767)));
    }
}

hipError_t launch_moe_route(hipStream_t st, const RouteArgs& a, int M) {
    hipLaunchKernelGGL(moe_route_kernel, dim3(M), dim3(ROUTE_THREADS), 0, st, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------- up

// Block (column tile, s) computes the s-th chosen expert's 16 interleaved columns for all its pairs, 16 rows at a time; waves
// split K. Blocks past the chosen experts end at once.
template <int P, int G>
__global__ void __launch_bounds__(512) moe_up_kernel(MoeArgs a) {
    constexpr int NG = 128 / G, DEPTH = 2;
    extern __shared__ uint4 s_dyn[];
    __shared__ int s_cnt[MOE_EXPERTS];
    __shared__ int s_list[MOE_PAIRS];
    __shared__ uint32_t s_max[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int pairs = a.M * a.topk, ct = blockIdx.x, KT = a.up.KT;
    for (int i = threadIdx.x; i < a.experts; i += blockDim.x) s_cnt[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
        const unsigned x = unsigned(a.idx[i]);
        if (x < unsigned(a.experts)) atomicAdd(&s_cnt[x], 1);
    }
    __syncthreads();
    // every wave finds the expert for itself
    int x = -1, left = blockIdx.y;
    for (int c = 0; c < a.experts; c += 64) {
        u64 m = __builtin_amdgcn_ballot_w64(c + lane < a.experts && s_cnt[c + lane] > 0);
        const int n = __builtin_popcountll(m);
        if (left < n) {
            for (; left; --left) m &= m - 1;
            x = c + __builtin_ctzll(m);
            break;
        }
        left -= n;
    }
    if (x < 0) return;
    x = __builtin_amdgcn_readfirstlane(x);
    const int n = __builtin_amdgcn_readfirstlane(s_cnt[x]);
    for (int c = 0, at = 0; c < pairs && at < n; c += 64) {   // each wave writes the same list
        const bool hit = c + lane < pairs && a.idx[c + lane] == x;
        const u64 m = __builtin_amdgcn_ballot_w64(hit);
        if (hit) s_list[at + __builtin_popcountll(m & ((u64(1) << lane) - 1))] = c + lane;
        at += __builtin_popcountll(m);
    }
    wave_lds_fence();
    const uint8_t* q = a.up.q + x * a.up_stride + size_t(ct) * KT * 1024;
    const uint8_t* s = a.up.s + x * a.up_stride + size_t(ct) * KT * 32 * NG;
    const int4* cst = a.up.cst + size_t(x) * a.up.CT * 16;
    const int F = a.up.N / 2;
    for (int r0 = 0; r0 < n; r0 += 16) {
        const int pr = s_list[min(r0 + (lane & 15), n - 1)];   // the lane's pair
        const int tok = pr / a.topk;
        const int8_t* hi = a.hi + size_t(tok) * a.ld8;
        const int8_t* lo = P == 2 ? a.lo + size_t(tok) * a.ld8 : nullptr;
        W4Tile<G> t[DEPTH];
        W4Rows<P> rows[DEPTH][1];
        double acc[1][4] = {{0.0, 0.0, 0.0, 0.0}};
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int kt = wave + d * waves;
            if (kt < KT) {
                t[d].load(q + size_t(kt) * 1024, s + size_t(kt) * 32 * NG, lane);
                rows[d][0].template load<G>(hi, lo, kt * 128, a.Kp16, lane);
            }
        }
        for (int kt = wave; kt < KT; kt += DEPTH * waves) {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                const int kd = kt + d * waves;
                if (kd < KT) {
                    w4_tile<1, P, G>(t[d], rows[d], acc);
                    const int kn = kd + DEPTH * waves;
                    if (kn < KT) {
                        t[d].load(q + size_t(kn) * 1024, s + size_t(kn) * 32 * NG, lane);
                        rows[d][0].template load<G>(hi, lo, kn * 128, a.Kp16, lane);
                    }
                }
            }
        }
        double2* red = reinterpret_cast<double2*>(s_dyn);
#pragma unroll
        for (int h = 0; h < 2; ++h) red[(wave * 2 + h) * 64 + lane] = make_double2(acc[0][2 * h], acc[0][2 * h + 1]);
        if (threadIdx.x < 16) s_max[threadIdx.x] = 0;
        __syncthreads();
        for (int h = wave; h < 2; h += waves) {
            double2 v = red[h * 64 + lane];
            for (int w = 1; w < waves; ++w) {
                const double2 o = red[(w * 2 + h) * 64 + lane];
                v.x += o.x;
                v.y += o.y;
            }
            const int c = ct * 16 + 4 * (lane >> 4) + 2 * h;
            const int e = a.e ? a.e[tok] : 0;
            const int y0 = w4_requant(i64(v.x), P == 2, cst[c], e), y1 = w4_requant(i64(v.y), P == 2, cst[c + 1], e);
            const int y = geglu_exact(y0, y1, a.Lphi);
            if (r0 + (lane & 15) < n && c < a.up.N) {
                a.v[size_t(pr) * F + (c >> 1)] = y;
                atomicMax(&s_max[lane & 15], uabs(y));
            }
        }
        __syncthreads();
        if (threadIdx.x < 16 && r0 + int(threadIdx.x) < n) a.vmax[size_t(s_list[r0 + threadIdx.x]) * a.up.CT + ct] = s_max[threadIdx.x];
        __syncthreads();   // red and s_max are written again
    }
}

// ---------------------------------------------------------------- down

// LDS of the down kernel: the pairs' sums, the waves' staging areas and the tables
constexpr int DOWN_WAVES = 16;
struct alignas(16) DownTables {   // the staging areas and 64-bit sums follow it in LDS
    int cnt[MOE_EXPERTS];      // pairs of an expert, then their first place
    int pos[MOE_PAIRS];        // a pair's place in the order by experts (-1: no expert)
    int pair[MOE_PAIRS];       // the pair at a place
    int se[MOE_PAIRS];         // the shift of the row at a place
    int tile_x[MOE_PAIRS];     // row tiles of at most 16 places: expert,
    int tile_at[MOE_PAIRS];    // first place | rows << 16
    int tiles;
};
static_assert(sizeof(DownTables) % 16 == 0 && (DOWN_WAVES * 2 * 16 * W4_LDR) % 16 == 0, "alignment of what follows the tables");

// A block owns 16 output columns: for every (row tile of an expert's pairs, K tile) its waves take equal shares, quantise the int32 rows
// in their own staging area, and add the sums of a pair and column to 64-bit integers in LDS; then each output sums its
// token's choices. Integer sums: their order does not matter.
template <int G>
__global__ void __launch_bounds__(64 * DOWN_WAVES) moe_down_kernel(MoeArgs a) {
    constexpr int NG = 128 / G, DEPTH = 2;
    extern __shared__ uint4 s_dyn[];
    DownTables& T = *reinterpret_cast<DownTables*>(s_dyn);
    uint8_t* stage_all = reinterpret_cast<uint8_t*>(s_dyn) + sizeof(DownTables);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int pairs = a.M * a.topk, ct = blockIdx.x, KT = a.down.KT, F = a.down.K;
    unsigned long long* sums = reinterpret_cast<unsigned long long*>(stage_all + DOWN_WAVES * 2 * 16 * W4_LDR);   // [place][16]
    for (int i = threadIdx.x; i < a.experts; i += blockDim.x) T.cnt[i] = 0;
    for (int i = threadIdx.x; i < pairs * 16; i += blockDim.x) sums[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
        const unsigned x = unsigned(a.idx[i]);
        T.pos[i] = x < unsigned(a.experts) ? atomicAdd(&T.cnt[x], 1) : -1;
    }
    __syncthreads();
    if (wave == 0) {   // first places and row tiles
        int at = 0, tiles = 0;
        for (int c = 0; c < a.experts; c += 64) {
            const int n = c + lane < a.experts ? T.cnt[c + lane] : 0, nt = (n + 15) >> 4;
            int pn = n, pt = nt;   // inclusive sums over the lanes
            for (int d = 1; d < 64; d <<= 1) {
                const int on = __shfl_up(pn, d), ot = __shfl_up(pt, d);
                if (lane >= d) { pn += on; pt += ot; }
            }
            const int first = at + pn - n, tfirst = tiles + pt - nt;
            if (c + lane < a.experts) T.cnt[c + lane] = first;
            for (int i = 0; i < nt; ++i) {
                T.tile_x[tfirst + i] = c + lane;
                T.tile_at[tfirst + i] = (first + 16 * i) | min(16, n - 16 * i) << 16;
            }
            at += __shfl(pn, 63);
            tiles += __shfl(pt, 63);
        }
        if (lane == 0) T.tiles = tiles;
    }
    __syncthreads();
    for (int i = wave; i < pairs; i += DOWN_WAVES) {   // places and the rows' shifts
        const int x = a.idx[i];
        if (unsigned(x) >= unsigned(a.experts)) continue;
        uint32_t m = 0;
        for (int c = lane; c < a.up.CT; c += 64) m = max(m, a.vmax[size_t(i) * a.up.CT + c]);
        m = wave_umax32(m);
        if (lane == 0) {
            const int at = T.cnt[x] + T.pos[i];
            T.pos[i] = at;
            T.pair[at] = i;
            T.se[at] = rowexp_u32(m);
        }
    }
    __syncthreads();

    const int units = T.tiles * KT, u1 = int((long long)units * (wave + 1) / DOWN_WAVES);
    int u = int((long long)units * wave / DOWN_WAVES);
    uint8_t* lds = stage_all + wave * 2 * 16 * W4_LDR;
    if (u < u1) {
        W4Tile<G> t[DEPTH];
        W4Quads<16> xq;
        const auto weights = [&](W4Tile<G>& tile, int ti, int kt) {
            const int x = __builtin_amdgcn_readfirstlane(T.tile_x[ti]);
            const size_t at = size_t(ct) * KT + kt;
            tile.load(a.down.q + x * a.down_stride + at * 1024, a.down.s + x * a.down_stride + at * 32 * NG, lane);
        };
        const auto quads = [&](int ti, int kt) {
            const int w = __builtin_amdgcn_readfirstlane(T.tile_at[ti]);
            const int* pair = T.pair + (w & 0xffff);
            xq.load([&](int r) { return a.v + size_t(pair[r]) * F; }, w >> 16, kt * 128, F, lane);
        };
        int ti = u / KT, kt = u - ti * KT;      // the unit computed
        int tl = ti, kl = kt, ul = u;           // the unit whose weights are loaded next
        const auto next = [&](int& i, int& k) { if (++k == KT) { k = 0; ++i; } };
#pragma unroll
        for (int d = 0; d < DEPTH; ++d)
            if (ul < u1) {
                weights(t[d], tl, kl);
                next(tl, kl);
                ++ul;
            }
        quads(ti, kt);
        double acc[1][4] = {{0.0, 0.0, 0.0, 0.0}};
        for (; u < u1;) {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                if (u >= u1) break;
                const int w = __builtin_amdgcn_readfirstlane(T.tile_at[ti]), first = w & 0xffff, n = w >> 16;
                wave_lds_fence();
                xq.stage(lds, T.se + first, n, lane);
                wave_lds_fence();
                int tn = ti, kn = kt;
                next(tn, kn);
                if (u + 1 < u1) quads(tn, kn);
                W4Rows<2> rows[1];
                const int r = min(lane & 15, n - 1);
                rows[0].template load<G>(reinterpret_cast<const int8_t*>(lds + r * W4_LDR), reinterpret_cast<const int8_t*>(lds + (16 + r) * W4_LDR), 0, 128, lane);
                w4_tile<1, 2, G>(t[d], rows, acc);
                if (ul < u1) {
                    weights(t[d], tl, kl);
                    next(tl, kl);
                    ++ul;
                }
                if (tn != ti || u + 1 == u1) {   // the last unit of this row tile here
                    if ((lane & 15) < n) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) atomicAdd(&sums[(first + (lane & 15)) * 16 + 4 * (lane >> 4) + k], (unsigned long long)i64(acc[0][k]));
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[0][k] = 0.0;
                }
                ti = tn;
                kt = kn;
                ++u;
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.M * 16; i += blockDim.x) {
        const int tok = i >> 4, c = ct * 16 + (i & 15);
        if (c >= a.down.N) continue;
        u64 sum = 0;
        for (int j = 0; j < a.topk; ++j) {
            const int at = T.pos[tok * a.topk + j];
            if (at < 0) continue;
            const int x = a.idx[tok * a.topk + j];
            const int y = w4_requant(i64(sums[at * 16 + (i & 15)]), true, a.down.cst[size_t(x) * a.down.CT * 16 + c], T.se[at]);
            sum += u64(i64(a.p[tok * a.topk + j])) * u64(i64(y));
        }
        const size_t o = size_t(tok) * a.ldy + c;
        const int y = int(rshr(i64(sum), 15));
        a.Y[o] = a.R ? add_sat(y, a.R[o]) : y;
    }
}

template <int P, int G>
static void moe_up(hipStream_t st, const MoeArgs& a) {
    int waves = 8;
    while (waves > 1 && waves > a.up.KT) waves /= 2;
    const dim3 grid(a.up.CT, std::min(a.experts, a.M * a.topk));
    hipLaunchKernelGGL((moe_up_kernel<P, G>), grid, dim3(64 * waves), size_t(waves) * 2 * 64 * 16, st, a);
}
template <int G>
static void moe_down(hipStream_t st, const MoeArgs& a) {
    const size_t lds = sizeof(DownTables) + DOWN_WAVES * 2 * 16 * W4_LDR + size_t(a.M) * a.topk * 128;
    hipLaunchKernelGGL((moe_down_kernel<G>), dim3(a.down.CT), dim3(64 * DOWN_WAVES), lds, st, a);
}

hipError_t launch_moe(hipStream_t st, const MoeArgs& a) {
    if (a.group_up == 32) a.lo ? moe_up<2, 32>(st, a) : moe_up<1, 32>(st, a);
    else if (a.group_up == 64) a.lo ? moe_up<2, 64>(st, a) : moe_up<1, 64>(st, a);
    else a.lo ? moe_up<2, 128>(st, a) : moe_up<1, 128>(st, a);
    if (hipError_t e = hipGetLastError()) return e;
    if (a.group_down == 32) moe_down<32>(st, a);
    else if (a.group_down == 64) moe_down<64>(st, a);
    else moe_down<128>(st, a);
    return hipGetLastError();
}

}  // namespace vk
