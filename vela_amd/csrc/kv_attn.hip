// Attention of one new token over a paged cache (vgemm_kv_attention), exact in integers: include/vgemm_kv.h states the formulas.
//
// The weights of a softmax need the row's maximum before their sum, and a rounded weight cannot be rescaled exactly. The
// operator is therefore defined on spans of 256 positions: a span's weights are relative to its own maximum, its mean is rounded to 32 bits, and the means
// are joined with the spans' weights. A span needs one pass over its keys and values, the numbers do not depend on which block takes which
// span, and what goes from the first kernel to the join is 4 D bytes a span and query head beside the 512 D bytes of its 8-bit keys and values.
//
// A block of four waves takes a span of one sequence and key head with up to sixteen of its query heads, the columns of the 16x16x64 int8
// matrix instruction. What bounds it is memory: two sequences of 131072 tokens (8 x 128 heads, 8 bits, 32 query heads) take 112 us, 4.8 TB/s of
// cache, against 5.0 for a copy; a span alone is a chain of two loads and ~3.5 us of work: a sequence of 500 tokens (16 x 64, 16 bits), two spans side by side and
// their join in one launch, takes 7.8 us.
//   * Scores: wave w has the positions [64 w, 64 w + 64). The keys are the A operand; row i of subtile ks is position 16 (i / 4) + 4 ks + i % 4, so that
//     lane (fg, query) ends with the scores of the 16 positions from 16 fg on, in order. Quarters of four tokens
//     lie together in a page (vgemm_kv.h), so a load touches four runs of 256 bytes.
//   * Queries are quantised while the first keys are on their way, in signed digits q = 256 h + l (15 bits leave h in [-64, 64]), so that
//     keys of 8 bits need two products a piece and no correction. They stand in LDS: registers are for the keys and values in flight.
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
#include "wave.h"

namespace vk {

namespace {

constexpr int EXP_N = 1025;
constexpr int MAX_DIGITS = 6;         // 15 bits and shifts up to 25 apart
constexpr int P_LD = KV_SPAN + 16;    // bytes of a query's weights in LDS, one digit: rows 4 banks apart
constexpr int TOP_SHIFT = 25;         // of an int32 in 8 bits

// what a wave waits for before it meets the others: its own LDS traffic, not its loads
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ i64 shfl_xor64(i64 v, int d) { return i64(__shfl_xor((long long)v, d)); }

typedef unsigned short us2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ int max_u16x2(int a, int b) {
    return __builtin_bit_cast(int, __builtin_elementwise_max(__builtin_bit_cast(us2, a), __builtin_bit_cast(us2, b)));
}

// floor(n / l) saturated to 32 bits, l > 0, inv = 1 / l: the quotient in double is off by less than one
__device__ __forceinline__ int div_sat(i64 n, i64 l, double inv) {
    double q = floor(double(n) * inv);
    const i64 r = n - i64(cvt_sat(q)) * l;
    if (r < 0) q -= 1.0;
    if (r >= l) q += 1.0;
    return cvt_sat(q);
}
// the same for |n| + l below 2^53, where the remainder is exact in double
__device__ __forceinline__ int div_sat53(double n, double l, double inv) {
    double q = floor(n * inv);
    const double r = fma(-q, l, n);
    q += r >= l ? 1.0 : r < 0.0 ? -1.0 : 0.0;
    return cvt_sat(q);
}

// 1 / l: an estimate and a step of Newton's, off by a few units of the last place; the quotients below are corrected
__device__ __forceinline__ double recip(double l) {
    const double r = __builtin_amdgcn_rcp(l);
    return fma(fma(-l, r, 1.0), r, r);
}

struct Lds {
    uint2 table[EXP_N];                        // entry i: Lexp[i] + 2^14, Lexp[i + 1] - Lexp[i]; the last one stands for 0
    int8_t p[MAX_DIGITS][16][P_LD];
    int mx[4][16], sum[4][16], ev[4];
    i64 x[4][16];
    double scale[16];
    int qsum[16];
    unsigned big[4];
};

// rshr(lutexp(d), 15), at most 32767
__device__ __forceinline__ int weight(const Lds& s, unsigned d) {
    const uint2 t = s.table[min(d >> 10, unsigned(EXP_N - 1))];
    const i64 prod = i64(int(t.y)) * int(d & 1023);
    return int(min((t.x + unsigned(int(prod >> 10))) >> 15, 32767u));
}

// blocks of four waves that a CU holds at a time, by their registers
constexpr int kv_held(int D, int planes) { return D <= 128 && planes == 1 ? 3 : (D + 63) / 64 * planes > 4 ? 1 : 2; }

constexpr int DEAL_ROWS = 2048;   // sequences whose spans are dealt evenly: every wave goes through their lengths, 64 at a time

__device__ __forceinline__ int kv_len(const KvAttnArgs& a, int row) { return int(min(i64(max(min(a.len[row], a.max_len), 0)), i64(a.width) << a.c.lp)); }
__device__ __forceinline__ int kv_first(const KvAttnArgs& a, int n) { return a.window > 0 ? max(0, n - a.window) : 0; }

// G of a span; st.y = 0: none. The greatest has a weight with any table, so that one span alone joins to its own mean.
__device__ __forceinline__ i64 join_weight(const KvAttnArgs& a, int mx, int2 st) {
    const unsigned d = unsigned(mx) - unsigned(st.x);
    if (st.y == 0 || d >= (1u << 20)) return 0;
    const i64 t = a.Lexp[d >> 10], t1 = a.Lexp[(d >> 10) + 1];
    const i64 f = (t + (((t1 - t) * i64(d & 1023)) >> 10) + 64) >> 7;
    return (d == 0 && f == 0 ? 1 : f) * st.y;
}

constexpr int SHORT_SPANS = 4;   // that a block of eight waves takes and joins by itself

// the one of F parts of four that a lane takes: x[KT * sub + t], t < KT = 4 / F
template <int F, class T>
__device__ __forceinline__ T part_of(const T& x0, const T& x1, const T& x2, const T& x3, int sub, int t) {
    if constexpr (F == 1) return t == 0 ? x0 : t == 1 ? x1 : t == 2 ? x2 : x3;
    if constexpr (F == 2) return t == 0 ? (sub ? x2 : x0) : (sub ? x3 : x1);
    const T lo = sub & 1 ? x1 : x0, hi = sub & 1 ? x3 : x2;
    return sub & 2 ? hi : lo;
}
// over a lane's F parts, 16 / F lanes apart in a row of sixteen
template <int F>
__device__ __forceinline__ int parts_max(int v) {
    if constexpr (F >= 2) v = max(v, dpp32<0x128>(v));   // row_ror 8, then 4
    if constexpr (F == 4) v = max(v, dpp32<0x124>(v));
    return v;
}
template <int F>
__device__ __forceinline__ int parts_sum(int v) {
    if constexpr (F >= 2) v += dpp32<0x128>(v);
    if constexpr (F == 4) v += dpp32<0x124>(v);
    return v;
}
template <int N>
__device__ __forceinline__ void load_words(unsigned (&w)[N], const void* p) {
    if constexpr (N == 4) {
        const uint4 v = *static_cast<const uint4*>(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = *static_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
        w[0] = *static_cast<const unsigned*>(p);
    }
}
template <int N, class T>
__device__ __forceinline__ void store_words(void* p, const T (&w)[N]) {
    if constexpr (N == 4) *static_cast<uint4*>(p) = make_uint4(unsigned(w[0]), unsigned(w[1]), unsigned(w[2]), unsigned(w[3]));
    else if constexpr (N == 2) *static_cast<uint2*>(p) = make_uint2(unsigned(w[0]), unsigned(w[1]));
    else *static_cast<unsigned*>(p) = unsigned(w[0]);
}

// EXACT: D == 64 NS, so that the loads' offsets are constants. F: up to 16 / F query heads share a key head; each stands in F columns, whose
// lanes take a F-th of its scores, weights and results (the matrix instructions give all of them in every column): 780 vector instructions a wave and
// span for 128 values in 8 bits with F = 1, about 450 with 4; four queries a key, 32 x 8192 tokens of 64 values 78 -> 68 us, of 128 133 -> 127; eight, F = 2, 82 -> 75 and 140 -> 135.
// chunks > 0: blocks take runs of spans of one sequence and key head, as even as the lengths allow, so that there are about `chunks` runs
// a head over all sequences; every block counts them from the lengths. chunks = 0: a block has one span, or each gridDim.z-th.
// SHORT: a block of eight waves takes a sequence of at most SHORT_SPANS spans, two at a time, each by four waves as elsewhere, and joins them itself.
template <int NS, int PL, bool EXACT, int F, bool SHORT>
__global__ void __launch_bounds__(SHORT ? 512 : 256, SHORT ? 2 : kv_held(64 * NS, PL)) kv_attn_kernel(KvAttnArgs a, int chunks) {
    constexpr int QT = 16 / F, KT = 4 / F, NK = 16 / F, JN = 4 / F;   // queries; a lane's subtiles, keys, and dimensions of four
    constexpr bool EARLY = NS * PL <= 4;       // values asked for beside the keys, and the next span's keys during the softmax: 32 NS PL registers for both
    constexpr int TEAMS = SHORT ? 2 : 1;       // of four waves
    __shared__ __attribute__((aligned(16))) Lds s_of[TEAMS];
    __shared__ __attribute__((aligned(16))) int8_t qs_of[TEAMS][2][16][64 * NS + 16];
    __shared__ __attribute__((aligned(16))) int means[SHORT ? SHORT_SPANS : 1][SHORT ? 16 : 1][SHORT ? 64 * NS : 4];
    __shared__ int2 stats[SHORT ? SHORT_SPANS : 1][SHORT ? 16 : 1];
    touch_args<int(sizeof(KvAttnArgs) + 4)>();
    const int team = SHORT ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
    Lds& s = s_of[team];
    auto& qs = qs_of[team];
    const int tid = SHORT ? threadIdx.x & 255 : threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fg = lane >> 4;
    const int qi = fr & (QT - 1), sub = fr / QT;   // the lane's query, and which part of it
    const bool deal = !SHORT && chunks > 0;
    const int head = blockIdx.x / a.qtiles, q0 = (blockIdx.x % a.qtiles) * 16, nq = min(16, a.group - q0);   // key head, its first query head here and their number
    int row = blockIdx.y, chunk = SHORT ? team : blockIdx.z, split = SHORT ? TEAMS : gridDim.z;
    auto zero_row = [&](int r) {               // a sequence without tokens
        for (int i = tid; i < nq * (EXACT ? 64 * NS : a.c.D); i += 256) a.out[size_t(r) * a.ldo + size_t(head * a.group + q0) * (EXACT ? 64 * NS : a.c.D) + i] = 0;
    };
    int n = 0;
    auto zero_rows = [&]() {                   // of dealt spans: sequences without tokens, which no run covers
        for (int r = blockIdx.y; r < a.rows; r += int(gridDim.y))
            if (kv_len(a, r) == 0) zero_row(r);
    };
    if (deal) {
        // Every wave for itself, without a barrier: a lane has the sequences lane, lane + 64, ...; runs are numbered in the order of lanes.
        auto spans_of = [&](int len) { return (len + KV_SPAN - 1) / KV_SPAN - kv_first(a, len) / KV_SPAN; };
        const int n0 = lane < a.rows ? kv_len(a, lane) : 0, count0 = spans_of(n0);
        int count = count0;
#pragma unroll 4
        for (int r = lane + 64; r < a.rows; r += 64) count += spans_of(kv_len(a, r));
        const int most = min(max(1, (wave_sum(count) + chunks - 1) / chunks), KV_MAX_LEN / KV_SPAN);   // spans of a run
        // runs of at most `most` spans: below 2^16 the product is off by less than 0.5 / most
        const float inv = 1.f / float(most);
        auto runs_of = [&](int spans) { return int((float(spans + most - 1) + 0.5f) * inv); };
        const int runs0 = runs_of(count0);
        int runs = runs0;
#pragma unroll 4
        for (int r = lane + 64; r < a.rows; r += 64) runs += runs_of(spans_of(kv_len(a, r)));
        const int end = wave_scan(runs), y = blockIdx.y;
        if (y >= __builtin_amdgcn_readlane(end, 63)) {
            zero_rows();
            return;
        }
        row = __ffsll((unsigned long long)__ballot(end > y)) - 1;           // the first lane whose runs end behind this one
        chunk = y - __builtin_amdgcn_readlane(end - runs, row);
        split = __builtin_amdgcn_readlane(runs0, row);
        n = __builtin_amdgcn_readlane(n0, row);
        while (chunk >= split) {               // not that lane's first sequence
            chunk -= split;
            row += 64;
            n = __builtin_amdgcn_readfirstlane(kv_len(a, row));
            split = __builtin_amdgcn_readfirstlane(runs_of(spans_of(n)));
        }
    }
    const KvView& c = a.c;
    const int D = EXACT ? 64 * NS : c.D, P = 1 << c.lp, pieces = D >> 4;
    const int32_t* table = a.table + size_t(row) * a.ldt;
    const i64 room = i64(a.width) << c.lp;
    // the pages of span u's sixteen groups, in lanes 0..15 (and again in the others): whatever the sequence's length
    auto fetch = [&](int u) {
        const int pos = u * KV_SPAN + 16 * fr;
        const int page = pos < room ? table[pos >> c.lp] : -1;
        return unsigned(page) < unsigned(c.pages) ? page : -1;
    };
    int page = -1;
    if (!deal && a.window == 0) page = fetch(chunk);   // on its way with the length
    if (!deal) n = kv_len(a, row);
    const int first = kv_first(a, n), u0 = first / KV_SPAN, u1 = (n + KV_SPAN - 1) / KV_SPAN;
    const int qh = head * a.group + q0 + qi;
    // queries: sixteen lanes a query, four neighbouring values at a time
    int4 x[NS];
    {
        const int32_t* q = a.Q + size_t(row) * a.ldq + size_t(head * a.group + q0) * D + (tid >> 4) * D + 4 * fr;
#pragma unroll
        for (int b = 0; b < NS; ++b) x[b] = (tid >> 4) < nq && (EXACT || 4 * fr + 64 * b < D) ? *reinterpret_cast<const int4*>(q + 64 * b) : make_int4(0, 0, 0, 0);
    }
    if (!deal && n == 0 && chunk == 0) zero_row(row);
    // dealt: spans [u, u_end), one after the other; else u, u + split, ...
    int u = deal ? u0 + (u1 - u0) * chunk / split : u0 + chunk;   // at most 2^15 spans: the products stay below 2^30
    const int u_end = deal ? u0 + (u1 - u0) * (chunk + 1) / split : u1, step = deal ? 1 : split;
    if (SHORT ? n == 0 : u >= u_end) return;   // SHORT: a team without a span left goes along, with nothing that counts
    if (deal || a.window) page = fetch(u);

    constexpr int KS = EARLY ? 4 : 2;          // subtiles of keys in registers
    v4i kv[KS][NS][PL], vv[NS][4][PL];
    unsigned ek[KT], ev[KT];
    int evb;
    // a span's group g: where its keys begin (page 0 where there is none)
    auto group = [&](int pages, int u, int g) { return c.keys(max(__shfl(pages, g), 0), head) + (((u * KV_SPAN + 16 * g) & (P - 1)) >> 4) * c.group_bytes(); };
    auto load_tiles = [&](int pages, int u, int k0) {      // subtiles k0, k0 + 1, ...
        const int8_t* kg = group(pages, u, 4 * wave + (fr >> 2)) + (fr & 3) * 16 + fg * 64;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int b = 0; b < NS; ++b)
#pragma unroll
                for (int p = 0; p < PL; ++p)
                    kv[ks][b][p] = EXACT || 4 * b + fg < pieces ? *reinterpret_cast<const v4i*>(kg + p * 16 * D + (k0 + ks) * 4 * D + b * 256) : v4i{0, 0, 0, 0};
    };
    auto load_keys = [&](int pages, int u) {
        load_tiles(pages, u, 0);
        const int pg = __shfl(pages, 4 * wave + fg);
        const uint8_t* sh = c.shifts(max(pg, 0), head) + ((u * KV_SPAN + 64 * wave + 16 * fg) & (P - 1));
        load_words(ek, sh + NK * sub);
        load_words(ev, sh + P + NK * sub);
        evb = sh[P + fr];
    };
    auto load_values = [&](int pages, int u) {
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            const int8_t* vg = group(pages, u, 4 * kt + fg) + c.half_bytes() + fr * 16 + wave * 256;
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int p = 0; p < PL; ++p) vv[i][kt][p] = EXACT || wave + 4 * i < pieces ? *reinterpret_cast<const v4i*>(vg + p * 16 * D + i * 1024) : v4i{0, 0, 0, 0};
        }
    };
    load_keys(page, u);
    if (deal) zero_rows();

    // the table, four entries a thread
    {
        i64 t[5];
#pragma unroll
        for (int i = 0; i < 5; ++i) t[i] = a.Lexp[4 * tid + i];
#pragma unroll
        for (int i = 0; i < 4; ++i) s.table[4 * tid + i] = make_uint2(unsigned(t[i]) + (1u << 14), unsigned(t[i + 1] - t[i]));
        if (tid == 0) s.table[EXP_N - 1] = make_uint2(0, 0);
    }
    {
        unsigned m = 0;
#pragma unroll
        for (int b = 0; b < NS; ++b) m = max(max(m, max(uabs(x[b].x), uabs(x[b].y))), max(uabs(x[b].z), uabs(x[b].w)));
        const int e = max(0, 32 - __clz(int(row_max(m))) - 14);
        int total = 0;
#pragma unroll
        for (int b = 0; b < NS; ++b) {
            const int v[4] = {x[b].x, x[b].y, x[b].z, x[b].w};
            unsigned h = 0, l = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = e ? (v[j] >> e) + ((v[j] >> (e - 1)) & 1) : v[j];
                total += r;
                h |= unsigned(((r + 128) >> 8) & 255) << (8 * j);
                l |= unsigned(r & 255) << (8 * j);
            }
            *reinterpret_cast<unsigned*>(&qs[0][tid >> 4][4 * fr + 64 * b]) = h;
            *reinterpret_cast<unsigned*>(&qs[1][tid >> 4][4 * fr + 64 * b]) = l;
        }
        total = row_sum(total);
        if (fr == 0) {
            s.scale[tid >> 4] = ldexp(double(a.m), e - a.s);
            s.qsum[tid >> 4] = total;
        }
    }
    lds_barrier();
    const double scale = s.scale[qi];
    const int qsum = s.qsum[qi];

    for (;;) {
        const int un = u + step;
        int pagen = -1;
        if (EARLY) {
            load_values(page, u);
            if (un < u_end) pagen = fetch(un);
        }
        // which of the lane's positions count
        const int p0 = u * KV_SPAN + 64 * wave + 16 * fg;
        const bool there = __shfl(page, 4 * wave + fg) >= 0;
        unsigned live;
        {
            const int from = min(max(first - p0 - NK * sub, 0), NK), to = min(max(n - p0 - NK * sub, 0), NK);
            live = there && to > from ? ((1u << to) - 1) & ~((1u << from) - 1) : 0;
        }
        const bool whole = __ballot(live != (1u << NK) - 1) == 0;
        unsigned evw[KT];
        unsigned ekw[KT];
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            ekw[t] = ek[t];
            evw[t] = ev[t];
        }
        // the least and the greatest shift of the values, as the greatest of (ev, 255 - ev) in two halves; a lane a position
        int ends = there && p0 + fr >= first && p0 + fr < n ? evb | (255 - evb) << 16 : 0;
        ends = max_u16x2(ends, dpp32<DPP_XOR1>(ends));
        ends = max_u16x2(ends, dpp32<DPP_XOR2>(ends));
        ends = max_u16x2(ends, dpp32<DPP_HALF_MIRROR>(ends));
        ends = max_u16x2(ends, dpp32<DPP_MIRROR>(ends));
        {
            auto e16 = __builtin_amdgcn_permlane16_swap(ends, ends, false, false);
            ends = max_u16x2(int(e16[0]), int(e16[1]));
            auto e32 = __builtin_amdgcn_permlane32_swap(ends, ends, false, false);
            ends = max_u16x2(int(e32[0]), int(e32[1]));
        }

        int sc[NK];
        int mx = INT_MIN;
        v4i qd[NS][2];   // lane (fg, fr): the values [64 b + 16 fg, + 16) of its query
#pragma unroll
        for (int b = 0; b < NS; ++b)
#pragma unroll
            for (int p = 0; p < 2; ++p) qd[b][p] = *reinterpret_cast<const v4i*>(&qs[p][qi][64 * b + 16 * fg]);
        v4i h[4], mid[4], l[4];
        auto scores = [&](int t, const v4i& h, const v4i& mid, const v4i& l) {   // subtile t of the lane's
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                double S;
                if constexpr (PL == 1) S = double(256 * h[j] + l[j]);
                else S = fma(double(h[j]), 65536.0, fma(double(mid[j]), 256.0, double(l[j] + 128 * qsum)));
                const double up = __builtin_bit_cast(double, u64(1023 + ((ekw[t] >> (8 * j)) & 255)) << 52);
                sc[4 * t + j] = cvt_sat(floor(fma(S * scale, up, 0.5)));
            }
        };
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            if (!EARLY && ks == KS) load_tiles(page, u, KS);
            h[ks] = mid[ks] = l[ks] = v4i{0, 0, 0, 0};
#pragma unroll
            for (int b = 0; b < NS; ++b) {
                h[ks] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv[ks % KS][b][0], qd[b][0], h[ks], 0, 0, 0);
                if constexpr (PL == 1) {
                    l[ks] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv[ks % KS][b][0], qd[b][1], l[ks], 0, 0, 0);
                } else {
                    mid[ks] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv[ks % KS][b][0], qd[b][1], mid[ks], 0, 0, 0);
                    mid[ks] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv[ks % KS][b][1], qd[b][0], mid[ks], 0, 0, 0);
                    l[ks] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv[ks % KS][b][1], qd[b][1], l[ks], 0, 0, 0);
                }
            }
            if (F == 1) scores(ks, h[ks], mid[ks], l[ks]);
        }
        if constexpr (F > 1) {
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                v4i ht, mt = {0, 0, 0, 0}, lt;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    ht[j] = part_of<F>(h[0][j], h[1][j], h[2][j], h[3][j], sub, t);
                    lt[j] = part_of<F>(l[0][j], l[1][j], l[2][j], l[3][j], sub, t);
                    if (PL == 2) mt[j] = part_of<F>(mid[0][j], mid[1][j], mid[2][j], mid[3][j], sub, t);
                }
                scores(t, ht, mt, lt);
            }
        }
        if (!whole)
#pragma unroll
            for (int i = 0; i < NK; ++i) sc[i] = live >> i & 1 ? sc[i] : INT_MIN;
#pragma unroll
        for (int i = 0; i < NK; ++i) mx = max(mx, sc[i]);
        mx = parts_max<F>(across_max(mx));
        if (fg == 0) s.mx[wave][qi] = mx;
        if (lane == 0) s.ev[wave] = ends;
        if (EARLY && un < u_end) load_keys(pagen, un);
        lds_barrier();
        mx = max(max(s.mx[0][qi], s.mx[1][qi]), max(s.mx[2][qi], s.mx[3][qi]));
        ends = max_u16x2(max_u16x2(s.ev[0], s.ev[1]), max_u16x2(s.ev[2], s.ev[3]));
        ends = __builtin_amdgcn_readfirstlane(ends);
        const int lo = 255 - (ends >> 16), hi = max(min(ends & 0xffff, lo + TOP_SHIFT), lo);   // lo = 255 where nothing counts
        const int digits = 2 + (hi - lo + 7) / 8;
        const bool small = digits <= 3 && hi <= 30 - 8 * PL;   // weights of 32 bits, sums that a double holds

        int sum = 0;
        int w[NK];
#pragma unroll
        for (int i = 0; i < NK; ++i) w[i] = weight(s, unsigned(mx) - unsigned(sc[i]));
        if (!whole) {
#pragma unroll
            for (int i = 0; i < NK; ++i) w[i] = live >> i & 1 ? w[i] : 0;
#pragma unroll
            for (int t = 0; t < KT; ++t) {     // shifts of what does not count become the least one
                const unsigned keep = ((live >> (4 * t) & 15) * 0x00204081u & 0x01010101u) * 255u;
                evw[t] = (evw[t] & keep) | (unsigned(lo) * 0x01010101u & ~keep);
            }
        }
#pragma unroll
        for (int i = 0; i < NK; ++i) sum += w[i];
        sum = parts_sum<F>(across_sum(sum));
        if (fg == 0) s.sum[wave][qi] = sum;
        i64 xs = 0;
        int8_t* prow = &s.p[0][qi][64 * wave + 16 * fg + NK * sub];
        if (small) {
            unsigned pk[3][KT];
            int xs32 = 0;                      // at most 256 * 2^23 in all
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const unsigned f = evw[t] - unsigned(lo) * 0x01010101u;   // no byte is below lo
                unsigned y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned v = unsigned(w[4 * t + j]) << (f >> (8 * j) & 31);
                    if (PL == 2) xs32 -= int(v);
                    y[j] = 0x8080u - v;
                }
                const unsigned p01 = __builtin_amdgcn_perm(y[1], y[0], 0x05010400), p23 = __builtin_amdgcn_perm(y[3], y[2], 0x05010400);
                pk[0][t] = __builtin_amdgcn_perm(p23, p01, 0x05040100) ^ 0x80808080u;
                pk[1][t] = __builtin_amdgcn_perm(p23, p01, 0x07060302) ^ 0x80808080u;
                pk[2][t] = __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0602) | __builtin_amdgcn_perm(y[3], y[2], 0x06020c0c);
            }
            if (PL == 2) xs = parts_sum<F>(across_sum(xs32));
            store_words(prow, pk[0]);
            store_words(prow + sizeof s.p[0], pk[1]);
            if (digits == 3) store_words(prow + 2 * sizeof s.p[0], pk[2]);
        } else {
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                i64 x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[j] = -i64(u64(unsigned(w[4 * t + j])) << ((int(evw[t] >> (8 * j) & 255) - lo) & 31));
                    xs += x[j];
                }
                for (int d = 0; d < digits; ++d) {
                    unsigned b = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int y = int(int8_t(x[j]));
                        b |= unsigned(y & 255) << (8 * j);
                        x[j] = (x[j] - y) >> 8;
                    }
                    *reinterpret_cast<unsigned*>(prow + d * int(sizeof s.p[0]) + 4 * t) = b;
                }
            }
            if (PL == 2) {
                for (int d = QT; d < 64; d <<= 1) xs += shfl_xor64(xs, d);
            }
        }
        if (PL == 2 && fg == 0) s.x[wave][qi] = xs;
        lds_barrier();
        sum = s.sum[0][qi] + s.sum[1][qi] + s.sum[2][qi] + s.sum[3][qi];
        if (PL == 2) xs = s.x[0][qi] + s.x[1][qi] + s.x[2][qi] + s.x[3][qi];
        if (!EARLY) load_values(page, u);

        int r[NS][JN];
        auto digit = [&](int t, auto add) {    // the products of one digit, handed over dimension by dimension: the lane's of each four
            v4i pb[4];
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) pb[kt] = *reinterpret_cast<const v4i*>(&s.p[t][qi][64 * kt + 16 * fg]);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                v4i h = {0, 0, 0, 0}, l = {0, 0, 0, 0};
#pragma unroll
                for (int kt = 0; kt < 4; ++kt) {
                    h = __builtin_amdgcn_mfma_i32_16x16x64_i8(vv[i][kt][0], pb[kt], h, 0, 0, 0);
                    if constexpr (PL == 2) l = __builtin_amdgcn_mfma_i32_16x16x64_i8(vv[i][kt][1], pb[kt], l, 0, 0, 0);
                }
                if constexpr (PL == 2)
#pragma unroll
                    for (int j = 0; j < 4; ++j) h[j] = 256 * h[j] + l[j];
#pragma unroll
                for (int j = 0; j < JN; ++j) add(i, j, part_of<F>(h[0], h[1], h[2], h[3], sub, j));
            }
        };
        const double inv = recip(double(max(sum, 1)));
        if (small) {
            // the lower two digits' sums of up to 2^30 are one integer
            int low[NS][JN];
            const auto set = [&](int i, int j, int v) { low[i][j] = v; };
            const auto add = [&](int i, int j, int v) { low[i][j] = low[i][j] * 256 + v; };
            double O[NS][JN];
            if (PL == 2) {                     // sums of two planes: up to 2^30 each
                const auto set2 = [&](int i, int j, int v) { O[i][j] = double(v); };
                const auto add2 = [&](int i, int j, int v) { O[i][j] = fma(O[i][j], 256.0, double(v)); };
                if (digits == 3) {
                    digit(2, set2);
                    digit(1, add2);
                } else {
                    digit(1, set2);
                }
                digit(0, add2);
            } else {
                digit(1, set);
                digit(0, add);
                if (digits == 3) {
                    digit(2, [&](int i, int j, int v) { O[i][j] = fma(double(v), 65536.0, double(low[i][j])); });
                } else {
#pragma unroll
                    for (int i = 0; i < NS; ++i)
#pragma unroll
                        for (int j = 0; j < JN; ++j) O[i][j] = double(low[i][j]);
                }
            }
            const double neg = -__builtin_bit_cast(double, u64(1023 + lo) << 52), half = double(sum >> 1), L = double(sum);
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int j = 0; j < JN; ++j) {
                    const double o = PL == 2 ? fma(double(int(xs)), 128.0, O[i][j]) : O[i][j];
                    r[i][j] = sum ? div_sat53(fma(o, neg, half), L, inv) : 0;
                }
        } else {
            i64 O[NS][JN];
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int j = 0; j < JN; ++j) O[i][j] = 0;
            for (int t = digits - 1; t >= 0; --t) digit(t, [&](int i, int j, int v) { O[i][j] = O[i][j] * 256 + v; });
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int j = 0; j < JN; ++j) r[i][j] = sum ? div_sat(i64(u64(-(O[i][j] + (PL == 2 ? 128 * xs : 0))) << lo) + (sum >> 1), sum, inv) : 0;
        }
        const bool only = u1 - u0 == 1;
        unsigned big = 0;
        if (qi < nq) {
            const size_t at = (size_t(row) * a.Hq + qh) * a.spans + u;
            if (!only && wave == 0 && fg == 0 && sub == 0 && !SHORT) a.stat[at] = make_int2(mx, sum);
            int32_t* y = (only ? a.out + size_t(row) * a.ldo + size_t(qh) * D : a.part + at * D) + 16 * wave + 4 * fg + JN * sub;
            if (SHORT) {
                y = &means[min(u - u0, SHORT_SPANS - 1)][qi][16 * wave + 4 * fg + JN * sub];
                if (u < u1 && wave == 0 && fg == 0 && sub == 0) stats[u - u0][qi] = make_int2(mx, sum);
            }
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                if (!EXACT && wave + 4 * i >= pieces) break;
                if (SHORT && u >= u1) break;
#pragma unroll
                for (int j = 0; j < JN; ++j) big = max(big, uabs(r[i][j]));
                store_words(y + 64 * i, r[i]);
            }
        }
        if (!SHORT && only && a.rowmax) {      // one atomic a block; its only span
            big = unsigned(wave_max(int(big ^ 0x80000000u))) ^ 0x80000000u;
            if (lane == 0) s.big[wave] = big;
            lds_barrier();
            big = max(max(s.big[0], s.big[1]), max(s.big[2], s.big[3]));
            if (tid == 0 && big) atomicMax(a.rowmax + row, big);
        }
        u = un;
        if (SHORT ? u - team >= u1 : u >= u_end) break;
        if (EARLY) {
            page = pagen;
        } else {
            asm volatile("" ::: "memory");     // not among the products, whose values fill the registers
            page = fetch(u);
            load_keys(page, u);
        }
    }
    if constexpr (SHORT) {
        __syncthreads();
        const int count = u1 - u0;
        unsigned big = 0;
        for (int i = threadIdx.x; i < nq * (D >> 2); i += 512) {   // four dimensions of a query head
            const int q = i / (D >> 2), d = 4 * (i % (D >> 2));
            int mx = INT_MIN;
#pragma unroll
            for (int k = 0; k < SHORT_SPANS; ++k)
                if (k < count && stats[k][q].y) mx = max(mx, stats[k][q].x);
            i64 G[SHORT_SPANS], all = 0;
#pragma unroll
            for (int k = 0; k < SHORT_SPANS; ++k) {
                G[k] = k < count ? join_weight(a, mx, stats[k][q]) : 0;
                all += G[k];
            }
            const int h = max(0, 64 - __clzll((long long)all) - 30);
            const i64 half = (i64(1) << h) >> 1;
            i64 x[4] = {0, 0, 0, 0}, T = 0;
#pragma unroll
            for (int k = 0; k < SHORT_SPANS; ++k) {
                if (k >= count) break;
                const int w = int((G[k] + half) >> h);
                const int4 v = *reinterpret_cast<const int4*>(&means[k][q][d]);
                x[0] += i64(w) * v.x;
                x[1] += i64(w) * v.y;
                x[2] += i64(w) * v.z;
                x[3] += i64(w) * v.w;
                T += w;
            }
            const double inv = recip(double(max(T, i64(1))));
            int r[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                r[j] = T ? div_sat(x[j] + (T >> 1), T, inv) : 0;
                big = max(big, uabs(r[j]));
            }
            store_words(a.out + size_t(row) * a.ldo + size_t(head * a.group + q0 + q) * D + d, r);
        }
        if (!a.rowmax) return;
        big = unsigned(wave_max(int(big ^ 0x80000000u))) ^ 0x80000000u;
        if (lane == 0) s.big[wave] = big;
        __syncthreads();
        if (threadIdx.x) return;
        for (int t = 0; t < TEAMS; ++t)
            for (int w = 0; w < 4; ++w) big = max(big, s_of[t].big[w]);
        if (big) atomicMax(a.rowmax + row, big);
    }
}

// ---------------------------------------------------------------- the join

constexpr int JOIN_ONE = 64;       // spans that one wave joins, a lane each for their weights: 8 spans 12.0 us a pass so and 19.3 with eight waves, 64 of 32 sequences 241 and 244
constexpr int JOIN_WAVES = 8;      // waves of a query head where there are more
constexpr int JOIN_CHUNK = 64 * JOIN_WAVES;   // spans whose weights stand in LDS at a time

// A lane has four neighbouring dimensions of every (64 / lanes of a span)-th span, so that a wave reads up to 1 KB at a time. Spans are
// weighed by a lane each. Up to JOIN_ONE spans a wave joins a query head by itself, with the first means on their way before their weights
// are known; beyond that eight waves do, and dims of D dimensions a block where the heads alone would leave CUs idle.
template <int WAVES>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) kv_join_kernel(KvAttnArgs a, int dims) {
    constexpr int AHEAD = 8;
    __shared__ int g_lds[WAVES == 1 ? 1 : JOIN_CHUNK];
    __shared__ int mxs[WAVES];
    __shared__ i64 sums[2][WAVES];
    __shared__ i64 acc[WAVES == 1 ? 1 : WAVES][WAVES == 1 ? 1 : 64 + 1][4];
    touch_args<int(sizeof(KvAttnArgs) + 4)>();
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int D = a.c.D, parts = (D + dims - 1) / dims, row = blockIdx.y;
    const int qh = WAVES == 1 ? int(blockIdx.x) * 4 + wave : int(blockIdx.x) / parts, d0 = WAVES == 1 ? 0 : (int(blockIdx.x) % parts) * dims;
    // without a window the first loads do not wait for the length: they stay within max_len's spans, and what lies behind the sequence's has no weight
    const int n = kv_len(a, row), u0 = a.window ? kv_first(a, n) / KV_SPAN : 0, count = (n + KV_SPAN - 1) / KV_SPAN - u0, most = a.window ? max(count, 1) : a.spans;
    const size_t at = (size_t(row) * a.Hq + min(qh, a.Hq - 1)) * a.spans + u0;
    const int quads = min(dims, D - d0) / 4, per = quads <= 4 ? 4 : quads <= 8 ? 8 : quads <= 16 ? 16 : quads <= 32 ? 32 : 64;   // lanes of a span
    const int groups = 64 / per, quad = lane & (per - 1), sub = lane / per;
    const int32_t* part = a.part + at * D + d0 + 4 * min(quad, quads - 1);
    i64 x[4] = {0, 0, 0, 0}, T = 0;
    auto add = [&](i64 w, int4 v) {
        x[0] += w * v.x;
        x[1] += w * v.y;
        x[2] += w * v.z;
        x[3] += w * v.w;
    };
    if constexpr (WAVES == 1) {
        int4 v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) v[i] = *reinterpret_cast<const int4*>(part + size_t(min(sub + i * groups, most - 1)) * D);
        int2 st = a.stat[at + min(lane, most - 1)];
        if (count <= 1) return;                // the first kernel has written the row
        if (lane >= count) st = make_int2(INT_MIN, 0);
        const int mx = wave_max(st.y ? st.x : INT_MIN);
        const i64 G = join_weight(a, mx, st);
        const int h = max(0, 64 - __clzll((long long)wave_sum64(G)) - 30);
        const int g = int((G + ((i64(1) << h) >> 1)) >> h);   // 0 in the lanes behind the last span
        T = wave_sum64(g);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {      // every lane takes part: what a lane that is switched off holds reads as 0
            const int k = sub + i * groups, w = __shfl(g, k & 63);
            add(k < count ? w : 0, v[i]);
        }
        for (int k = sub + AHEAD * groups; k - sub < count; k += groups) {
            const int w = __shfl(g, k);        // k < 64: count <= JOIN_ONE, and groups divides it
            add(w, *reinterpret_cast<const int4*>(part + size_t(min(k, count - 1)) * D));
        }
    } else {
        // the thread's spans tid + 512 i: the first one's statistics stay in registers
        int4 v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) v[i] = *reinterpret_cast<const int4*>(part + size_t(min(wave * groups + sub + i * WAVES * groups, most - 1)) * D);
        int2 st0 = a.stat[at + min(tid, most - 1)];
        if (count <= 1) return;
        if (tid >= count) st0 = make_int2(INT_MIN, 0);
        int mx = st0.y ? st0.x : INT_MIN;
        for (int k = tid + JOIN_CHUNK; k < count; k += JOIN_CHUNK) {
            const int2 st = a.stat[at + k];
            if (st.y) mx = max(mx, st.x);
        }
        mx = wave_max(mx);
        if (lane == 0) mxs[wave] = mx;
        __syncthreads();
        mx = wave_max(mxs[lane & (WAVES - 1)]);
        const i64 G0 = join_weight(a, mx, st0);
        i64 G = G0;
        for (int k = tid + JOIN_CHUNK; k < count; k += JOIN_CHUNK) G += join_weight(a, mx, a.stat[at + k]);
        G = wave_sum64(G);
        if (lane == 0) sums[0][wave] = G;
        __syncthreads();
        G = wave_sum64(lane < WAVES ? sums[0][lane] : 0);
        const int h = max(0, 64 - __clzll((long long)G) - 30);
        const i64 half = (i64(1) << h) >> 1;
        for (int c = 0; c < count; c += JOIN_CHUNK) {
            const int m = min(JOIN_CHUNK, count - c);
            if (c) __syncthreads();
            if (tid < m) {
                g_lds[tid] = int(((c ? join_weight(a, mx, a.stat[at + c + tid]) : G0) + half) >> h);
                T += g_lds[tid];
            }
            __syncthreads();
            int k = wave * groups + sub;
            if (c == 0) {
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) add(k + i * WAVES * groups < m ? g_lds[k + i * WAVES * groups] : 0, v[i]);
                k += AHEAD * WAVES * groups;
            }
            for (; k < m; k += WAVES * groups) add(g_lds[k], *reinterpret_cast<const int4*>(part + size_t(c + k) * D));
        }
        static_assert(JOIN_CHUNK == 64 * WAVES, "a thread a span of a chunk");
        T = wave_sum64(T);
        if (lane == 0) sums[1][wave] = T;
    }
    for (int d = per; d < 64; d <<= 1)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] += shfl_xor64(x[j], d);
    if constexpr (WAVES > 1) {
        if (sub == 0)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[wave][quad][j] = x[j];
        __syncthreads();
        if (wave) return;
        T = wave_sum64(lane < WAVES ? sums[1][lane] : 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] = 0;
            for (int w = 0; w < WAVES; ++w) x[j] += acc[w][quad][j];
        }
    }
    const bool mine = sub == 0 && quad < quads && qh < a.Hq;
    const double inv = 1.0 / double(T ? T : 1);
    int r[4];
    unsigned big = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        r[j] = T ? div_sat(x[j] + (T >> 1), T, inv) : 0;
        big = max(big, mine ? uabs(r[j]) : 0u);
    }
    if (mine) *reinterpret_cast<int4*>(a.out + size_t(row) * a.ldo + size_t(qh) * D + d0 + 4 * quad) = make_int4(r[0], r[1], r[2], r[3]);
    if (!a.rowmax) return;
    big = unsigned(wave_max(int(big ^ 0x80000000u))) ^ 0x80000000u;
    if constexpr (WAVES == 1) {                // one atomic a block: 32 of them on a row's word cost 2 us
        __shared__ unsigned bigs[4];
        if (lane == 0) bigs[wave] = big;
        __syncthreads();
        big = max(max(bigs[0], bigs[1]), max(bigs[2], bigs[3]));
        if (tid == 0 && big) atomicMax(a.rowmax + row, big);
    } else {
        if (lane == 0 && big) atomicMax(a.rowmax + row, big);
    }
}

constexpr bool kv_short(int D, int planes) { return (D + 63) / 64 * planes <= 4; }   // eight waves' registers are there

template <int NS, int PL, bool EXACT, int F>
void launch_form(hipStream_t st, const KvAttnArgs& a, dim3 g, int chunks) {
    if constexpr (kv_short(64 * NS, PL)) {
        if (chunks < 0) {
            kv_attn_kernel<NS, PL, EXACT, F, true><<<g, 512, 0, st>>>(a, 0);
            return;
        }
    }
    kv_attn_kernel<NS, PL, EXACT, F, false><<<g, 256, 0, st>>>(a, chunks);
}
template <int PL, bool EXACT, int F>
void launch_spans(hipStream_t st, const KvAttnArgs& a, dim3 g, int chunks) {
    switch ((a.c.D + 63) / 64) {
        case 1: launch_form<1, PL, EXACT, F>(st, a, g, chunks); break;
        case 2: launch_form<2, PL, EXACT, F>(st, a, g, chunks); break;
        case 3: launch_form<3, PL, EXACT, F>(st, a, g, chunks); break;
        default: launch_form<4, PL, EXACT, F>(st, a, g, chunks);
    }
}
template <int F>
void launch_spans(hipStream_t st, const KvAttnArgs& a, dim3 g, int chunks) {
    const bool exact = a.c.D % 64 == 0;
    if (a.c.planes == 1) exact ? launch_spans<1, true, F>(st, a, g, chunks) : launch_spans<1, false, F>(st, a, g, chunks);
    else exact ? launch_spans<2, true, F>(st, a, g, chunks) : launch_spans<2, false, F>(st, a, g, chunks);
}
// chunks: the kernel's; -1: SHORT
void launch_spans(hipStream_t st, const KvAttnArgs& a, dim3 g, int chunks) {
    if (a.group <= 4) launch_spans<4>(st, a, g, chunks);
    else if (a.group <= 8) launch_spans<2>(st, a, g, chunks);
    else launch_spans<1>(st, a, g, chunks);
}

}  // namespace

hipError_t launch_kv_attention(hipStream_t st, const KvAttnArgs& a) {
    const int heads = a.c.heads * a.qtiles;
    const int spans = a.window > 0 ? std::min(a.spans, a.window / KV_SPAN + 2) : a.spans;   // that a sequence may have
    const int held = 256 * kv_held(a.c.D, a.c.planes);   // blocks the card holds at a time
    // Few spans a sequence, and a CU for each sequence and head: one launch (500 tokens of 16 heads 9.2 us a pass, 11.0 with the join's launch; 32 x 1000 of 8 heads
    // 17.4 and 21.0). With twice as many, sequences of unequal length wait for the longest twice (64 ragged ones up to 1000: 21.7 and 15.2).
    if (spans > 1 && spans <= SHORT_SPANS && kv_short(a.c.D, a.c.planes) && i64(heads) * a.rows <= 256) {
        launch_spans(st, a, dim3(heads, a.rows), -1);
        return hipGetLastError();
    }
    if (a.rows <= DEAL_ROWS && i64(heads) * a.rows * spans > 2 * held) {
        // Blocks with more than two spans each take them as dealt (256 ragged sequences up to 8000 tokens 136 us a pass, 193 with a block a span; 2 x 131072 129 and
        // 133; 32 x 4096 67.1 and 67.7; 16 x 2000, 1.3 spans a block, 21.0 and 21.2). Runs of a length that gives each of these blocks one, two, three or four: the one whose rounds of blocks would take least if all sequences were
        // of max_len (a run costs its spans and START more; 64 x 8192 tokens in two runs a block 237 us, in one 252), and at least two where the sequences alone are more than the
        // blocks: then the longest are what is waited for.
        const float START = 1.5f;
        const i64 all = i64(a.rows) * spans;
        int chunks = 0;
        float least = 0.f;
        for (int j = i64(a.rows) * heads > held ? 2 : 1; j <= 4; ++j) {
            const int n = std::max(1, j * held / heads);
            const i64 most = (all + n - 1) / n, runs = (spans + most - 1) / most * a.rows;
            const float cost = float((runs * heads + held - 1) / held) * (float(all) / float(runs) + START);
            if (!chunks || cost < least) {
                least = cost;
                chunks = n;
            }
        }
        launch_spans(st, a, dim3(heads, int(std::min<i64>(chunks + a.rows, all))), chunks);   // a sequence adds less than one run to them
    } else {
        const int split = int(std::max<i64>(1, std::min<i64>(spans, 65536 / (heads * i64(a.rows)))));
        launch_spans(st, a, dim3(heads, a.rows, split), 0);
    }
    if (hipError_t e = hipGetLastError()) return e;
    if (a.spans <= 1) return hipSuccess;
    if (spans <= JOIN_ONE) {
        kv_join_kernel<1><<<dim3((a.Hq + 3) / 4, a.rows), 256, 0, st>>>(a, a.c.D);
    } else {
        const int dims = a.rows * a.Hq >= 256 ? a.c.D : 32;   // 2 x 131072, 64 heads of 128: 129 us so, 135 with a block a head; 128 heads 131 and 129
        kv_join_kernel<JOIN_WAVES><<<dim3(a.Hq * ((a.c.D + dims - 1) / dims), a.rows), 64 * JOIN_WAVES, 0, st>>>(a, dims);
    }
    return hipGetLastError();
}

}  // namespace vk
