// Beam search's selection (vgemm_beam_select): for each row of logits the sum of its weights and its best tokens, a span of 4096
// tokens at a time, then per group the best continuations. include/vgemm_kv.h states the formulas.
#include <algorithm>
#include <climits>

#include "kv.h"
#include "norm_math.h"

namespace vk {

namespace {

constexpr int EXP_N = 1025;
constexpr int PER = BEAM_SPAN / 256;   // values of a thread

__device__ __forceinline__ i64 beam_exp(unsigned d, const int64_t* L) {
    if (d >= (1u << 20)) return 0;
    const i64 a = L[d >> 10], b = L[(d >> 10) + 1];
    return a + (((b - a) * i64(d & 1023)) >> 10);
}

// A logit and its place in the span as one number: greater logits first, then lower places; 0 for what is banned or not there.
// 32 + 12 bits, and one that tells the least logit from none.
constexpr int KEY_BITS = 45;
__device__ __forceinline__ u64 key_of(int z, int at) { return z == INT_MIN ? 0 : (u64(unsigned(z) ^ 0x80000000u) << 12) + u64(BEAM_SPAN - 1 - at) + 1; }
__device__ __forceinline__ int key_logit(u64 k) { return int(unsigned((k - 1) >> 12) ^ 0x80000000u); }
__device__ __forceinline__ int key_place(u64 k) { return BEAM_SPAN - 1 - int((k - 1) & (BEAM_SPAN - 1)); }

struct SpanLds {
    uint2 table[EXP_N];        // entry i: Lexp[i], Lexp[i + 1] - Lexp[i]; the last one stands for 0
    u64 list[BEAM_SPAN];       // keys that reach the threshold
    i64 sum[4];
    u64 floor_[4];
    int mx[4], count;
};

// One span of one row. The n-th greatest of a wave's 64 lane maxima is a key that at least n keys of the wave reach, so the greatest of the
// four waves' is a threshold that the span's n best reach; found by bits, with a ballot each. The keys that reach it, a few more than n as
// a rule and at most 16 n a wave, are put in order by counting.
__global__ void __launch_bounds__(256) beam_span_kernel(BeamArgs a) {
    __shared__ SpanLds s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.y, span = blockIdx.x, n = a.b.n;
    const size_t out = size_t(row) * a.spans + span;
    if (a.b.score[row] == LLONG_MIN) return;   // no such beam: nothing reads its part of the workspace
    const int base = span * BEAM_SPAN;
    const int32_t* z = a.b.logits + size_t(row) * a.b.ldz + base;
    const int m = min(BEAM_SPAN, a.b.V - base);
    int v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = tid + 256 * i < m ? z[tid + 256 * i] : INT_MIN;
    for (int i = tid; i < EXP_N; i += 256) {
        const i64 t = a.b.Lexp[i], t1 = a.b.Lexp[min(i + 1, EXP_N - 1)];
        s.table[i] = i < EXP_N - 1 ? make_uint2(unsigned(t), unsigned(t1 - t)) : make_uint2(0, 0);
    }
    if (tid == 0) s.count = 0;
    u64 best = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) best = max(best, key_of(v[i], tid + 256 * i));
    // the greatest t with at least n lane maxima >= t, 0 where fewer lanes have any
    u64 t = 0;
    for (int b = KEY_BITS - 1; b >= 0; --b) {
        const u64 u = t | (u64(1) << b);
        if (__popcll(__ballot(best >= u)) >= n) t = u;
    }
    int mx = best ? key_logit(best) : INT_MIN;
    for (int d = 32; d; d >>= 1) mx = max(mx, __shfl_xor(mx, d));
    if (lane == 0) {
        s.mx[wave] = mx;
        s.floor_[wave] = t;
    }
    __syncthreads();
    mx = max(max(s.mx[0], s.mx[1]), max(s.mx[2], s.mx[3]));
    t = max(max(max(s.floor_[0], s.floor_[1]), max(s.floor_[2], s.floor_[3])), u64(1));
    i64 sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const unsigned d = v[i] == INT_MIN ? ~0u : unsigned(mx) - unsigned(v[i]);
        const uint2 e = s.table[min(d >> 10, unsigned(EXP_N - 1))];
        sum += i64(e.x) + ((i64(int(e.y)) * int(d & 1023)) >> 10);
        const u64 k = key_of(v[i], tid + 256 * i);
        if (k >= t) s.list[atomicAdd(&s.count, 1)] = k;
    }
    for (int d = 32; d; d >>= 1) sum += i64(__shfl_xor((long long)sum, d));
    if (lane == 0) s.sum[wave] = sum;
    __syncthreads();
    const int c = s.count;
    if (tid == 0) a.stat[out] = BeamStat{s.sum[0] + s.sum[1] + s.sum[2] + s.sum[3], mx, 0};
    int2* cand = a.cand + out * n;
    for (int i = tid; i < c; i += 256) {
        const u64 k = s.list[i];
        int rank = 0;
        for (int j = 0; j < c; ++j) rank += s.list[j] > k;
        if (rank < n) cand[rank] = make_int2(key_logit(k), base + key_place(k));
    }
    for (int i = c + tid; i < n; i += 256) cand[i] = make_int2(INT_MIN, -1);
}

struct Best { i64 c; int at; };   // score and list: lower lists first among equal scores
__device__ __forceinline__ bool before(const Best& x, const Best& y) { return x.c > y.c || (x.c == y.c && x.at < y.at); }

// One group: logZ of its beams, a wave a beam, then its spans' lists, each in falling order and all in order of beam and token, merged n
// times by the best of their heads. LLONG_MIN with a list past the last one stands for none.
constexpr int LISTS = BEAM_MOST * (BEAM_V / BEAM_SPAN) / 256;   // lists of a thread
__global__ void __launch_bounds__(256) beam_merge_kernel(BeamArgs a) {
    __shared__ i64 off[BEAM_MOST];
    __shared__ Best heads[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = blockIdx.x, B = a.b.beams, n = a.b.n;
    for (int b = wave; b < B; b += 4) {
        const int row = g * B + b;
        const i64 score = a.b.score[row];
        const bool in = lane < a.spans && score != LLONG_MIN;
        const BeamStat st = in ? a.stat[size_t(row) * a.spans + lane] : BeamStat{0, INT_MIN, 0};
        int mx = st.mx;
        for (int d = 32; d; d >>= 1) mx = max(mx, __shfl_xor(mx, d));
        i64 S = in && st.S ? (beam_exp(unsigned(mx) - unsigned(st.mx), a.b.Lexp) * ((st.S + 2048) >> 12) + (1 << 17)) >> 18 : 0;
        for (int d = 32; d; d >>= 1) S += i64(__shfl_xor((long long)S, d));
        S = max(S, i64(1));
        const int t = 63 - __clzll((long long)S);
        const i64 f = (t >= 30 ? S >> (t - 30) : S << (30 - t)) - (i64(1) << 30);
        const int i = int(f >> 20);
        const i64 l0 = a.b.Lln[i], l1 = a.b.Lln[i + 1], logz = ((t - 30) * i64(a.b.Lln[EXP_N - 1]) + l0 + (((l1 - l0) * (f & 0xfffff)) >> 20) + (1 << 13)) >> 14;
        if (lane == 0) off[b] = score == LLONG_MIN ? LLONG_MIN : score - mx - logz;
    }
    __syncthreads();
    const int lists = B * a.spans;
    const int2* cand = a.cand + size_t(g) * lists * n;
    i64 c[LISTS];              // the heads of this thread's lists, tid + 256 i
    int at[LISTS];             // and how far they have been taken
    auto head = [&](int i) {
        const int list = tid + 256 * i;
        c[i] = LLONG_MIN;
        if (list >= lists || at[i] >= n) return;
        const i64 o = off[list / a.spans];
        if (o == LLONG_MIN) return;
        const int2 k = cand[size_t(list) * n + at[i]];
        if (k.y >= 0) c[i] = o + k.x;
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
            const Best y{c[i], tid + 256 * i};
            if (c[i] != LLONG_MIN && before(y, x)) x = y;
        }
        for (int d = 32; d; d >>= 1) {
            const Best y{i64(__shfl_xor((long long)x.c, d)), __shfl_xor(x.at, d)};
            if (before(y, x)) x = y;
        }
        if (lane == 0) heads[wave] = x;
        __syncthreads();
        x = heads[0];
        for (int w = 1; w < 4; ++w)
            if (before(heads[w], x)) x = heads[w];
        __syncthreads();
        const size_t o = size_t(g) * n + k;
        if (x.at == INT_MAX) {
            if (tid == 0) {
                a.b.out_score[o] = LLONG_MIN;
                a.b.parent[o] = a.b.token[o] = -1;
            }
            continue;
        }
        if ((x.at & 255) != tid) continue;
#pragma unroll
        for (int i = 0; i < LISTS; ++i)
            if (tid + 256 * i == x.at) {
                a.b.out_score[o] = x.c;
                a.b.parent[o] = g * B + x.at / a.spans;
                a.b.token[o] = cand[size_t(x.at) * n + at[i]].y;
                ++at[i];
                head(i);
            }
    }
}

}  // namespace

hipError_t launch_beam_select(hipStream_t st, const BeamArgs& a) {
    beam_span_kernel<<<dim3(a.spans, a.b.groups * a.b.beams), 256, 0, st>>>(a);
    if (hipError_t e = hipGetLastError()) return e;
    beam_merge_kernel<<<a.b.groups, 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace vk
