// Beam search's selection (vgemm_beam_select): for each row of logits the sum of its weights and its best tokens, a span of 4096
// tokens at a time, then per group the best continuations. include/vgemm_kv.h states the formulas.
//
// The sum of a row's weights is defined by spans, as the attention's is, so that one pass over the logits gives a span's maximum, its sum
// and its n best tokens; a second, small kernel joins them. The n best of many values are found by a threshold that at least n of them
// reach -- the n-th greatest of 64 lanes' maxima, found by bits with a ballot each --, and the few that reach it are put in order by counting. Where too many
// do (ties, or the best ones in few lanes), the best are taken one after the other instead.
#include <algorithm>
#include <climits>

#include "kv.h"
#include "norm_math.h"
#include "wave.h"

namespace vk {

namespace {

constexpr int EXP_N = 1025;

__device__ __forceinline__ i64 beam_exp(unsigned d, const int64_t* L) {
    if (d >= (1u << 20)) return 0;
    const i64 a = L[d >> 10], b = L[(d >> 10) + 1];
    return a + (((b - a) * i64(d & 1023)) >> 10);
}

// A logit and its place in the span as one number: greater logits first, then lower places; 0 for what is banned.
__device__ __forceinline__ u64 key_of(int z, int at) { return z == INT_MIN ? 0 : (u64(unsigned(z) ^ 0x80000000u) << 12) + u64(BEAM_SPAN - 1 - at) + 1; }
__device__ __forceinline__ int key_logit(u64 k) { return int(unsigned((k - 1) >> 12) ^ 0x80000000u); }
__device__ __forceinline__ int key_place(u64 k) { return BEAM_SPAN - 1 - int((k - 1) & (BEAM_SPAN - 1)); }

// A value that at least n lanes' v reach, at most `step` below the greatest such one where that lies within `range` (powers of two) of the greatest v;
// 1 where fewer than n lanes have any (v = 0: none).
__device__ __forceinline__ unsigned reached_by(unsigned v, int n, unsigned range, unsigned step) {
    const unsigned top = unsigned(wave_max(int(v ^ 0x80000000u))) ^ 0x80000000u;
    auto enough = [&](unsigned u) { return __popcll(__ballot(v >= u)) >= n; };
    if (top > range && enough(top - range)) {
        unsigned t = top - range;
        for (unsigned b = range >> 1; b >= step; b >>= 1)
            if (enough(t + b)) t += b;
        return t;
    }
    unsigned t = 0;
    for (unsigned b = 1u << 31; b; b >>= 1)
        if (enough(t | b)) t |= b;
    return t > 1 ? t : 1;
}

// orders the wave's own LDS accesses where no barrier does
__device__ __forceinline__ void wave_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

constexpr int LIST = 192;   // keys of a wave that reach the threshold: n and a few more as a rule, at most 64 where they are taken one by one

struct SpanLds {
    uint2 table[EXP_N];     // entry i: Lexp[i], Lexp[i + 1] - Lexp[i]; the last one stands for 0
    u64 list[4 * LIST];     // a wave's own part, or a block's
    i64 sum[4];
    int mx[4], count;
    unsigned reach[4];
};

// lanes below this one among those of mask
__device__ __forceinline__ int below(u64 mask) { return int(__builtin_amdgcn_mbcnt_hi(unsigned(mask >> 32), __builtin_amdgcn_mbcnt_lo(unsigned(mask), 0))); }

// use(key, rank) for each of c keys, its rank the number of greater ones, by `rows` rows of sixteen lanes. Up to 64 keys a row takes one, a lane four of the
// others (4 x 32000 logits: 6.9 -> 5.7 us); beyond that a lane takes one and goes through all.
template <class U>
__device__ __forceinline__ void by_rank(const u64* list, int c, int row, int rows, int l, U use) {
    if (c <= 64) {
        for (int i0 = 0; i0 < c; i0 += rows) {   // whole rows: every lane takes part in the sums
            const int i = i0 + row;
            const u64 k = list[min(i, c - 1)];
            int rank = 0;
#pragma unroll
            for (int j = 0; j < 64; j += 16)
                if (j < c) rank += j + l < c && list[min(j + l, c - 1)] > k;
            rank = row_sum(rank);
            if (l == 0 && i < c) use(k, rank);
        }
    } else {
        for (int i = row * 16 + l; i < c; i += rows * 16) {
            const u64 k = list[i];
            int rank = 0;
            for (int j = 0; j < c; ++j) rank += list[j] > k;
            use(k, rank);
        }
    }
}

struct __attribute__((packed, aligned(4))) Quad { int v[4]; };   // sixteen bytes that lie where rows of any length put them

// One span of one row, by WAVES waves of a block of four: one where there are spans for all CUs (a wave's search, sums and order then serve 64
// values a lane; 200 x 100003 logits take 22 us, 3.6 TB/s, 13 of them the read alone), four where the call's own latency counts (4 x 32000: 5.9 us).
template <int WAVES>
__global__ void __launch_bounds__(256, WAVES == 1 ? 5 : 4) beam_span_kernel(BeamArgs a) {
    constexpr int PER = BEAM_SPAN / (64 * WAVES);
    __shared__ SpanLds s;
    touch_args<int(sizeof(BeamArgs))>();
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = a.b.n;
    const int id = WAVES == 4 ? int(blockIdx.x) : int(blockIdx.x) * 4 + wave, rows = a.b.groups * a.b.beams;
    const int row = min(id / a.spans, rows - 1), span = id % a.spans;
    const size_t out = size_t(row) * a.spans + span;
    const bool in = id < rows * a.spans;
    const i64 score = a.b.score[row];            // on its way with the logits
    const int base = span * BEAM_SPAN, m = in ? min(BEAM_SPAN, a.b.V - base) : 0, t0 = WAVES == 4 ? tid : lane;
    const int32_t* z = a.b.logits + size_t(row) * a.b.ldz + base;
    int v[PER];
    if (m == BEAM_SPAN) {
#pragma unroll
        for (int q = 0; q < PER / 4; ++q) {
            const Quad x = *reinterpret_cast<const Quad*>(z + 4 * (q * 64 * WAVES + t0));
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * q + i] = x.v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = 4 * ((i >> 2) * 64 * WAVES + t0) + (i & 3);
            v[i] = at < m ? z[at] : INT_MIN;
        }
    }
    auto place = [&](int i) { return 4 * ((i >> 2) * 64 * WAVES + t0) + (i & 3); };
    {
        i64 t[5];
#pragma unroll
        for (int i = 0; i < 5; ++i) t[i] = a.b.Lexp[4 * tid + i];
#pragma unroll
        for (int i = 0; i < 4; ++i) s.table[4 * tid + i] = make_uint2(unsigned(t[i]), unsigned(t[i + 1] - t[i]));
        if (tid == 0) s.table[EXP_N - 1] = make_uint2(0, 0);
    }
    if (tid == 0) s.count = 0;
    int mx = INT_MIN;
#pragma unroll
    for (int i = 0; i < PER; ++i) mx = max(mx, v[i]);
    unsigned reach = reached_by(unsigned(mx) ^ 0x80000000u, n, 1u << 20, 1u << 10);   // 16 of the logits, by steps of 1/64
    mx = wave_max(mx);
    if (lane == 0) {
        s.mx[wave] = mx;
        s.reach[wave] = reach;
    }
    __syncthreads();
    if (!in || score == LLONG_MIN) return;     // no such beam: nothing reads its part of the workspace
    if constexpr (WAVES == 4) {
        mx = max(max(s.mx[0], s.mx[1]), max(s.mx[2], s.mx[3]));
        reach = max(max(s.reach[0], s.reach[1]), max(s.reach[2], s.reach[3]));
    }
    const int least = int(reach ^ 0x80000000u);   // above what is banned
    // what reaches the threshold, one after the other in the wave's part of the list, or in the block's from where the wave's begin
    u64* list = WAVES == 4 ? s.list : s.list + wave * LIST;
    int found = 0, at = 0;
    if (WAVES == 4) {
#pragma unroll
        for (int i = 0; i < PER; ++i) found += __popcll(__ballot(v[i] >= least));
        if (found <= LIST) {
            if (lane == 0) at = atomicAdd(&s.count, found);
            at = __builtin_amdgcn_readfirstlane(at);
        }
        found = found <= LIST ? 0 : found;        // to be counted again, or too many
    }
    if (found == 0) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const u64 mask = __ballot(v[i] >= least);
            if (!mask) continue;
            const int to = found + below(mask);
            if (v[i] >= least && to < LIST) list[at + to] = key_of(v[i], place(i));
            found += __popcll(mask);
        }
    }
    const bool over = found > LIST;
    i64 sum = 0;
    // what is banned lies far enough below any maximum but those near it
    const bool low = mx < INT_MIN + (1 << 20);
#pragma unroll
    for (int q = 0; q < PER / 8; ++q) {
#pragma unroll
        for (int i = 8 * q; i < 8 * q + 8; ++i) {
            const unsigned d = low && v[i] == INT_MIN ? ~0u : unsigned(mx) - unsigned(v[i]);
            const uint2 e = s.table[min(d >> 10, unsigned(EXP_N - 1))];
            sum += e.x + unsigned(int((i64(int(e.y)) * int(d & 1023)) >> 10));
        }
        asm volatile("" ::: "memory");   // eight table entries on their way at a time, not 64
    }
    sum = wave_sum64(sum);
    if (over) {                                   // one after the other: each the greatest below the last
        if (WAVES == 4) {
            if (lane == 0) at = atomicAdd(&s.count, n);
            at = __builtin_amdgcn_readfirstlane(at);
        }
        int lz = INT_MAX, lp = -1;                // the last one's logit and place
        for (int k = 0; k < n; ++k) {             // LIST of them there are, and more
            int bz = INT_MIN, bp = 0;
            const int rel = lp - 4 * t0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {       // of equal ones the first: a lane's places rise
                constexpr int STEP = 4 * 64 * WAVES;
                const int at = (i >> 2) * STEP + (i & 3);
                if ((v[i] < lz || (v[i] == lz && at > rel)) && v[i] > bz) {
                    bz = v[i];
                    bp = at;
                }
            }
            u64 best = key_of(bz, 4 * t0 + bp);
            for (int d = 1; d < 64; d <<= 1) best = max(best, u64(__shfl_xor((unsigned long long)best, d)));
            if (lane == 0) list[at + k] = best;
            lz = key_logit(best);
            lp = key_place(best);
        }
        found = n;
    }
    int2* cand = a.cand + out * n;
    auto put = [&](u64 k, int rank) {
        if (rank < n) cand[rank] = make_int2(key_logit(k), base + key_place(k));
    };
    if constexpr (WAVES == 1) {
        wave_lds();
        if (lane == 0) a.stat[out] = BeamStat{sum, mx, 0};
        by_rank(list, found, lane >> 4, 4, lane & 15, put);
        for (int i = found + lane; i < n; i += 64) cand[i] = make_int2(INT_MIN, -1);
    } else {
        if (lane == 0) s.sum[wave] = sum;
        __syncthreads();
        if (tid == 0) a.stat[out] = BeamStat{s.sum[0] + s.sum[1] + s.sum[2] + s.sum[3], mx, 0};
        const int c = s.count;
        by_rank(list, c, tid >> 4, 16, tid & 15, put);
        for (int i = c + tid; i < n; i += 256) cand[i] = make_int2(INT_MIN, -1);
    }
}

// ---------------------------------------------------------------- the groups

struct Best { i64 c; int at; };   // score and list: lower lists first among equal scores
__device__ __forceinline__ bool before(const Best& x, const Best& y) { return x.c > y.c || (x.c == y.c && x.at < y.at); }

constexpr int NEAR = 40;      // bits of a score below the group's best one in a key
constexpr int PLACES = 23;    // bits of beam * V + token
constexpr int CUT = NEAR + PLACES - 32;   // a key's upper 32 bits are what thresholds compare: at least 1 in every key that holds something
constexpr u64 FAR = (u64(1) << NEAR) - 1, HELD = FAR - (u64(1) << (CUT - PLACES));   // distances above HELD are too far for a key
constexpr int BEST_LIST = 1024;

// One group: logZ of its beams, a wave a beam, then the best of its spans' lists, each in falling order: a thread a list or two, by a threshold as
// above over keys of a score's distance from the best one and its place, which the lists' heads give and down to which each list is
// walked. Where the keys do not tell (scores about 2^40 apart, or too many that reach the threshold) the lists are merged n times
// by the best of their heads.
template <int THREADS, int LISTS>
__global__ void __launch_bounds__(THREADS) beam_merge_kernel(BeamArgs a) {
    constexpr int WAVES = THREADS / 64, AHEAD = 2;   // entries of a list that are asked for at the start
    __shared__ i64 off[BEAM_MOST];
    __shared__ Best heads[WAVES];
    __shared__ u64 list[BEST_LIST];
    __shared__ int count, far;
    __shared__ unsigned reach_of[WAVES];
    touch_args<int(sizeof(BeamArgs))>();
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = blockIdx.x, B = a.b.beams, n = a.b.n;
    const int lists = B * a.spans;
    const int2* cand = a.cand + size_t(g) * lists * n;
    int2 first[LISTS][AHEAD];
#pragma unroll
    for (int i = 0; i < LISTS; ++i)
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) first[i][j] = tid + THREADS * i < lists && j < n ? cand[size_t(tid + THREADS * i) * n + j] : make_int2(INT_MIN, -1);
    if (tid == 0) count = far = 0;
    for (int b = wave; b < B; b += WAVES) {
        const int row = g * B + b;
        const i64 score = a.b.score[row];
        const bool in = lane < a.spans && score != LLONG_MIN;
        const BeamStat st = in ? a.stat[size_t(row) * a.spans + lane] : BeamStat{0, INT_MIN, 0};
        const int mx = wave_max(st.mx);
        i64 S = in && st.S ? (beam_exp(unsigned(mx) - unsigned(st.mx), a.b.Lexp) * ((st.S + 2048) >> 12) + (1 << 17)) >> 18 : 0;
        S = max(wave_sum64(S), i64(1));
        const int t = 63 - __clzll((long long)S);
        const i64 f = (t >= 30 ? S >> (t - 30) : S << (30 - t)) - (i64(1) << 30);
        const int i = int(f >> 20);
        const i64 l0 = a.b.Lln[i], l1 = a.b.Lln[i + 1], logz = ((t - 30) * i64(a.b.Lln[EXP_N - 1]) + l0 + (((l1 - l0) * (f & 0xfffff)) >> 20) + (1 << 13)) >> 14;
        if (lane == 0) off[b] = score == LLONG_MIN ? LLONG_MIN : score - mx - logz;
    }
    __syncthreads();
    // LLONG_MIN: no beam (its lists hold anything) or no token
    i64 o[LISTS];
    int f0[LISTS];                               // a beam's place: beam * V
    i64 top = LLONG_MIN;
#pragma unroll
    for (int i = 0; i < LISTS; ++i) {
        const int beam = min(tid + THREADS * i, lists - 1) / a.spans;
        o[i] = off[beam];
        f0[i] = beam * a.b.V;
    }
    auto score_of = [&](int i, int2 k) { return o[i] == LLONG_MIN || k.y < 0 ? LLONG_MIN : o[i] + k.x; };
#pragma unroll
    for (int i = 0; i < LISTS; ++i) top = max(top, score_of(i, first[i][0]));
    top = wave_max64(top);
    if (lane == 0) heads[wave].c = top;
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) top = max(top, heads[w].c);
    auto key = [&](int i, int2 k) {              // 0: none, or too far below the best
        const i64 c = score_of(i, k);
        const u64 d = u64(top) - u64(c);
        return c == LLONG_MIN || d > HELD ? u64(0) : ((FAR - d) << PLACES) | u64((1 << PLACES) - 1 - (f0[i] + k.y));
    };
    u64 best = 0;
#pragma unroll
    for (int i = 0; i < LISTS; ++i) best = max(best, key(i, first[i][0]));
    const unsigned reach_own = reached_by(unsigned(best >> CUT), n, 1u << (20 - (CUT - PLACES)), 1u << (10 - (CUT - PLACES)));   // scores 2^20 below the best, by steps of 2^10
    if (lane == 0) reach_of[wave] = reach_own;
    __syncthreads();
    unsigned reach = 1;
    for (int w = 0; w < WAVES; ++w) reach = max(reach, reach_of[w]);
    // each list's first entries that reach the threshold: all of a wave's get their places at once
    u64 y[LISTS][AHEAD];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < LISTS; ++i)
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            y[i][j] = key(i, first[i][j]);
            mine += y[i][j] && unsigned(y[i][j] >> CUT) >= reach;
        }
    const int upto = wave_scan(mine);
    int slot = 0;
    if (lane == 63) slot = upto ? atomicAdd(&count, upto) : 0;
    slot = __builtin_amdgcn_readlane(slot, 63) + upto - mine;
#pragma unroll
    for (int i = 0; i < LISTS; ++i) {
        bool more = true;                        // a list falls: what follows one that does not reach it does not either
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            more = y[i][j] && unsigned(y[i][j] >> CUT) >= reach;
            if (more && slot < BEST_LIST) list[slot] = y[i][j];
            slot += more;
            if (y[i][j] == 0 && score_of(i, first[i][j]) != LLONG_MIN) far = 1;
        }
        for (int j = AHEAD; more && j < n; ++j) {
            const int2 k = cand[size_t(tid + THREADS * i) * n + j];
            const u64 z = key(i, k);
            more = z && unsigned(z >> CUT) >= reach;
            if (z == 0 && score_of(i, k) != LLONG_MIN) far = 1;
            if (!more) break;
            const int to = atomicAdd(&count, 1);
            if (to < BEST_LIST) list[to] = z;
        }
    }
    __syncthreads();
    const bool told = count >= n || !far;        // else some of the n best are among the far ones
    if (told && count <= BEST_LIST) {
        auto put = [&](int rank, i64 c, int parent, int token) {
            const size_t to = size_t(g) * n + rank;
            a.b.out_score[to] = c;
            a.b.parent[to] = parent;
            a.b.token[to] = token;
        };
        by_rank(list, count, tid >> 4, THREADS / 16, tid & 15, [&](u64 y, int rank) {
            const int f = (1 << PLACES) - 1 - int(y & ((1 << PLACES) - 1));
            if (rank < n) put(rank, i64(u64(top) - (FAR - (y >> PLACES))), g * B + f / a.b.V, f % a.b.V);
        });
        for (int i = count + tid; i < n; i += THREADS) put(i, LLONG_MIN, -1, -1);
        return;
    }
    i64 c[LISTS];              // the heads of this thread's lists, tid + THREADS i
    int at[LISTS];             // and how far they have been taken
    auto head = [&](int i) {
        const int l = tid + THREADS * i;
        c[i] = LLONG_MIN;
        if (l >= lists || at[i] >= n) return;
        c[i] = score_of(i, cand[size_t(l) * n + at[i]]);
    };
#pragma unroll
    for (int i = 0; i < LISTS; ++i) {
        at[i] = 0;
        head(i);
    }
    for (int k = 0; k < n; ++k) {
        Best x{LLONG_MIN, INT_MAX};
#pragma unroll
        for (int i = 0; i < LISTS; ++i) {
            const Best y{c[i], tid + THREADS * i};
            if (c[i] != LLONG_MIN && before(y, x)) x = y;
        }
        for (int d = 32; d; d >>= 1) {
            const Best y{i64(__shfl_xor((long long)x.c, d)), __shfl_xor(x.at, d)};
            if (before(y, x)) x = y;
        }
        if (lane == 0) heads[wave] = x;
        __syncthreads();
        x = heads[0];
        for (int w = 1; w < WAVES; ++w)
            if (before(heads[w], x)) x = heads[w];
        __syncthreads();
        const size_t to = size_t(g) * n + k;
        if (x.at == INT_MAX) {
            if (tid == 0) {
                a.b.out_score[to] = LLONG_MIN;
                a.b.parent[to] = a.b.token[to] = -1;
            }
            continue;
        }
        if ((x.at & (THREADS - 1)) != tid) continue;
#pragma unroll
        for (int i = 0; i < LISTS; ++i)
            if (tid + THREADS * i == x.at) {
                a.b.out_score[to] = x.c;
                a.b.parent[to] = g * B + x.at / a.spans;
                a.b.token[to] = cand[size_t(x.at) * n + at[i]].y;
                ++at[i];
                head(i);
            }
    }
}

}  // namespace

hipError_t launch_beam_select(hipStream_t st, const BeamArgs& a) {
    const int spans = a.b.groups * a.b.beams * a.spans;
    // 512 spans 10.7 us a pass with four waves each and 13.5 with one, 2048 16.8 and 17.7, 4096 23.5 and 22.9, 5000 28.4 and 28.2
    if (spans >= 2048) beam_span_kernel<1><<<(spans + 3) / 4, 256, 0, st>>>(a);
    else beam_span_kernel<4><<<spans, 256, 0, st>>>(a);
    if (hipError_t e = hipGetLastError()) return e;
    // a thread a list
    if (a.b.beams * a.spans <= 256) beam_merge_kernel<256, 1><<<a.b.groups, 256, 0, st>>>(a);
    else beam_merge_kernel<1024, 2><<<a.b.groups, 1024, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace vk
