// The paged key-value cache beside its attention: block tables and slot maps (vgemm_kv_plan), rows into pages and back
// (vgemm_kv_write, vgemm_kv_read), copies of pages (vgemm_kv_copy) and beam search's tables (vgemm_beam_tables).
#include <algorithm>

#include "kv.h"
#include "norm_math.h"
#include "wave.h"

namespace vk {

namespace {

// ---------------------------------------------------------------- block tables and slot maps

__device__ __forceinline__ int clamp_len(int v) { return min(max(v, 0), KV_MAX_LEN); }
__device__ __forceinline__ int sat_pos(i64 v) { return int(v < 0x7fffffffLL ? v : 0x7fffffffLL); }

// the last r with start[r] <= t, of R >= 1 running sums that begin with 0: the request of item t where t is below the sum of all
__device__ __forceinline__ int owner(const int* start, int R, int t) {
    int lo = 0, hi = R;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

struct PlanRow { int len, add, have, more; };
__device__ __forceinline__ PlanRow plan_row(const VgemmKvPlan& p, int lp, int r) {
    PlanRow w;
    w.len = clamp_len(p.len[r]);
    w.add = clamp_len(p.add[r]);
    w.have = (w.len + p.page - 1) >> lp;
    w.more = max(0, min((w.len + w.add + p.page - 1) >> lp, p.width) - w.have);
    return w;
}

// Every block forms the running sums of tokens and new pages of all requests for itself (8 bytes a request from L2, at most 32 KB) and
// serves its share of the token rows and of the new pages: one launch and no traffic between blocks. Table entries that others
// write are not read: a new page's number comes from the free list by the running sum.
__global__ void __launch_bounds__(256) kv_plan_kernel(VgemmKvPlan p, int lp) {
    extern __shared__ int plan_lds[];
    int *tok = plan_lds, *pag = plan_lds + p.R;   // running sums before each request, saturated
    __shared__ i64 part[2][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (p.R + 255) / 256, r0 = min(tid * per, p.R), r1 = min(r0 + per, p.R);
    i64 nt = 0, np = 0;
    for (int r = r0; r < r1; ++r) {
        const PlanRow w = plan_row(p, lp, r);
        nt += w.add;
        np += w.more;
    }
    i64 st = nt, sp = np;                          // running sums over the threads
    for (int d = 1; d < 64; d <<= 1) {
        const i64 a = __shfl_up((long long)st, d), b = __shfl_up((long long)sp, d);
        if (lane >= d) {
            st += a;
            sp += b;
        }
    }
    if (lane == 63) {
        part[0][wave] = st;
        part[1][wave] = sp;
    }
    __syncthreads();
    i64 tokens = 0, used = 0;
    for (int w = 0; w < 4; ++w) {
        if (w < wave) {
            st += part[0][w];
            sp += part[1][w];
        }
        tokens += part[0][w];
        used += part[1][w];
    }
    st -= nt;
    sp -= np;
    const bool first = blockIdx.x == 0;
    for (int r = r0; r < r1; ++r) {
        const PlanRow w = plan_row(p, lp, r);
        tok[r] = sat_pos(st);
        pag[r] = sat_pos(sp);
        if (first && p.start) p.start[r] = tok[r];
        if (first && p.new_len) p.new_len[r] = w.len + w.add;
        st += w.add;
        sp += w.more;
    }
    if (first && tid == 0) {
        if (p.start) p.start[p.R] = sat_pos(tokens);
        if (p.used) p.used[0] = sat_pos(used);
    }
    __syncthreads();
    const int total = sat_pos(tokens), pages = sat_pos(used), nfree = p.R ? p.nfree[0] : 0;
    auto take = [&](int i) {
        const int page = i < nfree ? p.free[i] : -1;
        return unsigned(page) < unsigned(p.pages) ? page : -1;
    };
    const int at = int(blockIdx.x) * 256 + tid, step = int(gridDim.x) * 256;
    for (i64 i = at; i < pages; i += step) {
        const int r = owner(pag, p.R, int(i));
        p.table[size_t(r) * p.ldt + plan_row(p, lp, r).have + int(i) - pag[r]] = take(int(i));
    }
    for (i64 t = at; t < p.tokens; t += step) {
        int slot = -1, pos = -1;
        if (t < total) {
            const int r = owner(tok, p.R, int(t));
            const PlanRow w = plan_row(p, lp, r);
            pos = w.len + int(t) - tok[r];
            const int j = pos >> lp;
            if (j < p.width) {
                const int page = j < w.have ? p.table[size_t(r) * p.ldt + j] : take(pag[r] + j - w.have);
                if (unsigned(page) < unsigned(p.pages)) slot = (page << lp) + (pos & (p.page - 1));
            }
        }
        p.slot[t] = slot;
        if (p.pos) p.pos[t] = pos;
    }
}

// ---------------------------------------------------------------- rows

constexpr int KV_TOKENS = 16;   // of a block: sixteen lanes a token, four neighbouring values at a time

// Where a row lies: page, and the place in it; there = false where the slot is none.
struct Place { bool there; int page, at; };
__device__ __forceinline__ Place place_of(const KvView& c, int slot) {
    const bool there = slot >= 0 && slot < (c.pages << c.lp);
    return Place{there, there ? slot >> c.lp : 0, there ? slot & ((1 << c.lp) - 1) : 0};
}

// Values lie transposed, sixteen tokens a dimension. A block turns its sixteen tokens over in LDS, so that four tokens whose slots follow one another
// from a multiple of four are one word in memory, and lanes that follow one another touch 256 neighbouring bytes. The LDS columns are the
// tokens moved by `off`, which makes a run of tokens that begins anywhere meet those words; tokens of other words go as bytes.
constexpr int TURN = 20;        // columns of a dimension: sixteen and up to three before them
struct Turn {
    int slot[KV_TOKENS];
    int off;
};
__device__ __forceinline__ void turn_init(Turn& t, const KvView& c, const int32_t* slots, int M) {
    if (threadIdx.x < 64) {     // one wave
        const int i = threadIdx.x, at = int(blockIdx.x) * KV_TOKENS + i;
        const int slot = i < KV_TOKENS && at < M ? slots[at] : -1;
        const bool there = place_of(c, slot).there;
        const u64 first = __ballot(there);
        if (i < KV_TOKENS) t.slot[i] = there ? slot : -1;
        if (first ? i == __ffsll((unsigned long long)first) - 1 : i == 0) t.off = first ? (slot - i) & 3 : 0;
    }
}
// the slot of the first of word w's four tokens where they are one word in memory, else -1
__device__ __forceinline__ int turn_word(const Turn& t, int w) {
    const int i = 4 * w - t.off;
    if (i < 0 || i + 3 >= KV_TOKENS) return -1;
    const int s = t.slot[i];
    return s >= 0 && (s & 3) == 0 && t.slot[i + 1] == s + 1 && t.slot[i + 2] == s + 2 && t.slot[i + 3] == s + 3 ? s : -1;
}

template <int PL, bool RUNS>
__global__ void __launch_bounds__(256, 8) kv_write_kernel(KvView c, const int32_t* K, const int32_t* V, int ld, const int32_t* slots, int M) {
    __shared__ Turn turn;
    __shared__ __attribute__((aligned(16))) int8_t vt[RUNS ? PL * 256 * TURN : 16];
    const int tid = threadIdx.x, l = tid & 15, t16 = tid >> 4, t = int(blockIdx.x) * KV_TOKENS + t16, head = blockIdx.y;
    const Place p = place_of(c, t < M ? slots[t] : -1);
    const size_t from = size_t(p.there ? t : 0) * ld + head * c.D;
    // RUNS: keys and values by one block, all their rows asked for at once; else by two
    constexpr int BOTH = RUNS ? 2 : 1;
    int4 v[BOTH][4];
#pragma unroll
    for (int b = 0; b < BOTH; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 4 * l + 64 * i;
            const int32_t* x = ((RUNS ? b : int(blockIdx.z)) ? V : K) + from;
            v[b][i] = p.there && d < c.D ? *reinterpret_cast<const int4*>(x + d) : make_int4(0, 0, 0, 0);
        }
    if (RUNS) {
        turn_init(turn, c, slots, M);
        __syncthreads();
    }
    constexpr int BITS = 8 * PL - 1, TOP = (1 << BITS) - 1;
    int8_t* keys = c.keys(p.page, head) + (p.at >> 4) * c.group_bytes();
#pragma unroll
    for (int b = 0; b < BOTH; ++b) {
        const bool value = RUNS ? b : blockIdx.z;
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(max(m, max(uabs(v[b][i].x), uabs(v[b][i].y))), max(uabs(v[b][i].z), uabs(v[b][i].w)));
        const int e = max(0, 32 - __clz(int(row_max(m))) - BITS);   // __clz(0) is 32
        if (l == 0 && p.there) c.shifts(p.page, head)[(int(value) << c.lp) + p.at] = uint8_t(e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 4 * l + 64 * i;
            if (d >= c.D) break;
            int q[4] = {v[b][i].x, v[b][i].y, v[b][i].z, v[b][i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) q[j] = min(max(e ? (q[j] >> e) + ((q[j] >> (e - 1)) & 1) : q[j], -TOP), TOP);
#pragma unroll
            for (int n = 0; n < PL; ++n) {
                char4 y;
                int8_t* bb = reinterpret_cast<int8_t*>(&y);
#pragma unroll
                for (int j = 0; j < 4; ++j) bb[j] = int8_t(PL == 1 ? q[j] : n == 0 ? q[j] >> 8 : (q[j] & 255) - 128);
                if (RUNS && value) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) vt[(n * c.D + d + j) * TURN + t16 + turn.off] = bb[j];
                } else if (p.there && value) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) keys[c.half_bytes() + n * 16 * c.D + c.value_at(p.at & 15, d + j)] = bb[j];
                } else if (p.there) {
                    *reinterpret_cast<char4*>(keys + n * 16 * c.D + c.key_at(p.at & 15, d)) = y;
                }
            }
        }
    }
    if (!RUNS) return;
    __syncthreads();
    const int words = turn.off ? 5 : 4;
    for (int w = tid & 3; w < words; w += 4) {
        const int s = turn_word(turn, w), i0 = 4 * w - turn.off;
        if (s >= 0) {
            const Place o = place_of(c, s);
            int8_t* dst = c.keys(o.page, head) + c.half_bytes() + (o.at >> 4) * c.group_bytes() + (o.at & 15);
            for (int d = tid >> 2; d < PL * c.D; d += 64) *reinterpret_cast<int*>(dst + 16 * d) = *reinterpret_cast<const int*>(&vt[d * TURN + 4 * w]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (i0 + k < 0 || i0 + k >= KV_TOKENS || turn.slot[i0 + k] < 0) continue;
                const Place o = place_of(c, turn.slot[i0 + k]);
                int8_t* dst = c.keys(o.page, head) + c.half_bytes() + (o.at >> 4) * c.group_bytes() + (o.at & 15);
                for (int d = tid >> 2; d < PL * c.D; d += 64) dst[16 * d] = vt[d * TURN + 4 * w + k];
            }
        }
    }
}

// With RUNS a block reads keys and values where both are asked for (as the write does), the keys' words on their way while the values are turned over.
template <int PL, bool RUNS>
__global__ void __launch_bounds__(256, 8) kv_read_kernel(KvView c, const int32_t* slots, int M, int32_t* K, int32_t* V, int ld) {
    __shared__ Turn turn;
    __shared__ __attribute__((aligned(16))) int8_t vt[RUNS ? PL * 256 * TURN : 16];
    const int tid = threadIdx.x, l = tid & 15, t16 = tid >> 4, t = int(blockIdx.x) * KV_TOKENS + t16, head = blockIdx.y;
    const bool key = RUNS ? K != nullptr : K && !blockIdx.z, value = RUNS ? V != nullptr : !key;
    const Place p = place_of(c, t < M ? slots[t] : -1);
    const uint8_t* sh = c.shifts(p.page, head) + p.at;
    const int ek = min(int(sh[0]), 31), ev = min(int(sh[1 << c.lp]), 31);
    const int8_t* keys = c.keys(p.page, head) + (p.at >> 4) * c.group_bytes();
    char4 k[4][PL];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < PL; ++n) {
            const int d = 4 * l + 64 * i;
            k[i][n] = key && p.there && d < c.D ? *reinterpret_cast<const char4*>(keys + n * 16 * c.D + c.key_at(p.at & 15, d)) : char4{0, 0, 0, 0};
        }
    if (RUNS && value) {
        turn_init(turn, c, slots, M);
        __syncthreads();
        const int words = turn.off ? 5 : 4;
        for (int w = tid & 3; w < words; w += 4) {
            const int s = turn_word(turn, w), i0 = 4 * w - turn.off;
            if (s >= 0) {
                const Place o = place_of(c, s);
                const int8_t* src = c.keys(o.page, head) + c.half_bytes() + (o.at >> 4) * c.group_bytes() + (o.at & 15);
                for (int d = tid >> 2; d < PL * c.D; d += 64) *reinterpret_cast<int*>(&vt[d * TURN + 4 * w]) = *reinterpret_cast<const int*>(src + 16 * d);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (i0 + k < 0 || i0 + k >= KV_TOKENS || turn.slot[i0 + k] < 0) continue;
                    const Place o = place_of(c, turn.slot[i0 + k]);
                    const int8_t* src = c.keys(o.page, head) + c.half_bytes() + (o.at >> 4) * c.group_bytes() + (o.at & 15);
                    for (int d = tid >> 2; d < PL * c.D; d += 64) vt[d * TURN + 4 * w + k] = src[16 * d];
                }
            }
        }
    }
    auto put = [&](int32_t* rows, int e, auto byte) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 4 * l + 64 * i;
            if (d >= c.D) break;
            int q[4] = {0, 0, 0, 0};
            if (p.there) {
#pragma unroll
                for (int n = 0; n < PL; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) q[j] = n == 0 ? byte(i, n, j) : 256 * q[j] + byte(i, n, j) + 128;
#pragma unroll
                for (int j = 0; j < 4; ++j) q[j] = int(sat32(i64(q[j]) << e));
            }
            *reinterpret_cast<int4*>(rows + size_t(t) * ld + head * c.D + d) = make_int4(q[0], q[1], q[2], q[3]);
        }
    };
    if (key && t < M) put(K, ek, [&](int i, int n, int j) { return int(reinterpret_cast<const int8_t*>(&k[i][n])[j]); });
    if (!value) return;
    if (RUNS) __syncthreads();
    if (t >= M) return;
    put(V, ev, [&](int i, int n, int j) {
        const int d = 4 * l + 64 * i + j;
        return int(RUNS ? vt[(n * c.D + d) * TURN + t16 + turn.off] : keys[c.half_bytes() + n * 16 * c.D + c.value_at(p.at & 15, d)]);
    });
}

// ---------------------------------------------------------------- pages and tables by parent

__global__ void __launch_bounds__(256) kv_copy_kernel(KvView c, const int32_t* src, const int32_t* dst) {
    const int i = blockIdx.x, s = src[i], d = dst[i];
    if (unsigned(s) >= unsigned(c.pages) || unsigned(d) >= unsigned(c.pages)) return;
    const size_t bytes = size_t(c.heads) * 2 * c.half_bytes(), sh = (size_t(c.heads) * 2) << c.lp;   // both multiples of 16
    const v4i* a = reinterpret_cast<const v4i*>(c.data + s * bytes);
    v4i* b = reinterpret_cast<v4i*>(c.data + d * bytes);
    const size_t at = size_t(blockIdx.y) * 256 + threadIdx.x, step = size_t(gridDim.y) * 256;
    for (size_t k = at; k < bytes / 16; k += step) b[k] = a[k];
    const v4i* as = reinterpret_cast<const v4i*>(c.shift + s * sh);
    v4i* bs = reinterpret_cast<v4i*>(c.shift + d * sh);
    for (size_t k = at; k < sh / 16; k += step) bs[k] = as[k];
}

__global__ void __launch_bounds__(256) beam_tables_kernel(VgemmBeamTables t, int lp) {
    const int r = blockIdx.x, p = t.parent[r], own = t.fresh[r];
    const bool there = unsigned(p) < unsigned(t.rows);
    const int n = there ? int(min(i64(max(t.len[p], 0)), i64(t.width) << lp)) : 0;
    const int full = n >> lp;
    const int32_t* old = t.table + size_t(there ? p : 0) * t.ldt;
    const int last = n & (t.page - 1) ? old[full] : -1;   // the partly filled page; a fresh one instead of none would hold what nobody has written
    const int fresh = last >= 0 ? own : -1;
    int32_t* row = t.out_table + size_t(r) * t.ldt;
    for (int j = threadIdx.x; j < t.width; j += 256) row[j] = j < full ? old[j] : (j == full ? fresh : -1);
    if (threadIdx.x == 0) {
        t.out_len[r] = n;
        t.src[r] = max(last, -1);
        t.dst[r] = fresh;
    }
}

}  // namespace

hipError_t launch_kv_plan(hipStream_t st, const VgemmKvPlan& p, int lp) {
    // 256 token rows a block, 1024 blocks at most; the new pages, never more than the tokens, are dealt over the same blocks. Without rows one block writes them all.
    const int blocks = std::max(1, std::min(int((int64_t(p.tokens) + 255) / 256), 1024));
    kv_plan_kernel<<<blocks, 256, size_t(p.R) * 8, st>>>(p, lp);
    return hipGetLastError();
}

// Few tokens are mostly a decode step's, each in a page of its own: their bytes go one by one, without LDS and its two barriers. Written and read back, 8
// heads x 128: 24 tokens apart 10.1 us so and 10.7 turned over (the host's time for two calls); in a row, 8 bits, 1000 11.2 and 12.4, 2000 16.5 and 16.2, 4000 27.2 and 22.4; 16 bits,
// 500 9.9 and 10.7, 1000 15.2 and 13.7, 5000 55 and 35.
constexpr int RUNS_FROM = 2048;   // tokens times planes

hipError_t launch_kv_write(hipStream_t st, const KvView& c, const int32_t* K, const int32_t* V, int ld, const int32_t* slot, int M) {
    const bool runs = M >= RUNS_FROM / c.planes;
    const dim3 g((M + KV_TOKENS - 1) / KV_TOKENS, c.heads, runs ? 1 : 2);
    if (c.planes == 1) runs ? kv_write_kernel<1, true><<<g, 256, 0, st>>>(c, K, V, ld, slot, M) : kv_write_kernel<1, false><<<g, 256, 0, st>>>(c, K, V, ld, slot, M);
    else runs ? kv_write_kernel<2, true><<<g, 256, 0, st>>>(c, K, V, ld, slot, M) : kv_write_kernel<2, false><<<g, 256, 0, st>>>(c, K, V, ld, slot, M);
    return hipGetLastError();
}

hipError_t launch_kv_read(hipStream_t st, const KvView& c, const int32_t* slot, int M, int32_t* K, int32_t* V, int ld) {
    const bool runs = M >= RUNS_FROM / c.planes;
    const dim3 g((M + KV_TOKENS - 1) / KV_TOKENS, c.heads, K && V && !runs ? 2 : 1);
    if (c.planes == 1) runs ? kv_read_kernel<1, true><<<g, 256, 0, st>>>(c, slot, M, K, V, ld) : kv_read_kernel<1, false><<<g, 256, 0, st>>>(c, slot, M, K, V, ld);
    else runs ? kv_read_kernel<2, true><<<g, 256, 0, st>>>(c, slot, M, K, V, ld) : kv_read_kernel<2, false><<<g, 256, 0, st>>>(c, slot, M, K, V, ld);
    return hipGetLastError();
}

hipError_t launch_kv_copy(hipStream_t st, const KvView& c, const int32_t* src, const int32_t* dst, int n) {
    const int parts = int(std::min<size_t>(std::max<size_t>(size_t(c.heads) * 2 * c.half_bytes() / (16 * 256 * 4), 1), 64));   // about four 16-byte pieces a thread
    kv_copy_kernel<<<dim3(n, parts), 256, 0, st>>>(c, src, dst);
    return hipGetLastError();
}

hipError_t launch_beam_tables(hipStream_t st, const VgemmBeamTables& t, int lp) {
    beam_tables_kernel<<<t.rows, 256, 0, st>>>(t, lp);
    return hipGetLastError();
}

}  // namespace vk
