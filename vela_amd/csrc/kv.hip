// The paged key-value cache beside its attention: block tables and slot maps (vgemm_kv_plan), rows into pages and back
// (vgemm_kv_write, vgemm_kv_read), copies of pages (vgemm_kv_copy) and beam search's tables (vgemm_beam_tables).
#include <algorithm>

#include "kv.h"
#include "norm_math.h"

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

// the greatest of a 16-lane row's values
__device__ __forceinline__ unsigned row16_max(unsigned v) {
    v = max(v, unsigned(dpp32<DPP_XOR1>(int(v))));
    v = max(v, unsigned(dpp32<DPP_XOR2>(int(v))));
    v = max(v, unsigned(dpp32<DPP_HALF_MIRROR>(int(v))));
    return max(v, unsigned(dpp32<DPP_MIRROR>(int(v))));
}

constexpr int KV_TOKENS = 16;   // of a block: sixteen lanes a token

// sixteen tokens of one head, keys or values (blockIdx.z): a token's sixteen lanes hold four neighbouring values at a time
template <int PL>
__global__ void __launch_bounds__(256) kv_write_kernel(KvView c, const int32_t* K, const int32_t* V, int ld, const int32_t* slots, int M) {
    const int l = threadIdx.x & 15, t = int(blockIdx.x) * KV_TOKENS + (threadIdx.x >> 4), head = blockIdx.y, value = blockIdx.z;
    const int slot = t < M ? slots[t] : -1;
    const bool there = slot >= 0 && slot < (c.pages << c.lp);
    const int32_t* x = (value ? V : K) + size_t(there ? t : 0) * ld + head * c.D;
    int4 v[4];
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = 4 * l + 64 * i;
        v[i] = there && d < c.D ? *reinterpret_cast<const int4*>(x + d) : make_int4(0, 0, 0, 0);
        m = max(max(m, max(uabs(v[i].x), uabs(v[i].y))), max(uabs(v[i].z), uabs(v[i].w)));
    }
    m = row16_max(m);
    constexpr int BITS = 8 * PL - 1, TOP = (1 << BITS) - 1;
    const int e = max(0, 32 - __clz(int(m)) - BITS);   // __clz(0) is 32
    if (!there) return;
    const int page = slot >> c.lp, at = slot & ((1 << c.lp) - 1), t16 = at & 15;
    int8_t* dst = c.keys(page, head) + (value ? c.half_bytes() : 0) + (at >> 4) * c.group_bytes();
    if (l == 0) c.shifts(page, head)[(value << c.lp) + at] = uint8_t(e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = 4 * l + 64 * i;
        if (d >= c.D) break;
        int q[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = min(max(e ? (q[j] >> e) + ((q[j] >> (e - 1)) & 1) : q[j], -TOP), TOP);
#pragma unroll
        for (int p = 0; p < PL; ++p) {
            int8_t* plane = dst + p * 16 * c.D;
            char4 b;
            int8_t* bb = reinterpret_cast<int8_t*>(&b);
#pragma unroll
            for (int j = 0; j < 4; ++j) bb[j] = int8_t(PL == 1 ? q[j] : p == 0 ? q[j] >> 8 : (q[j] & 255) - 128);
            if (value) {
#pragma unroll
                for (int j = 0; j < 4; ++j) plane[c.value_at(t16, d + j)] = bb[j];
            } else {
                *reinterpret_cast<char4*>(plane + c.key_at(t16, d)) = b;
            }
        }
    }
}

template <int PL>
__global__ void __launch_bounds__(256) kv_read_kernel(KvView c, const int32_t* slots, int M, int32_t* K, int32_t* V, int ld) {
    const int l = threadIdx.x & 15, t = int(blockIdx.x) * KV_TOKENS + (threadIdx.x >> 4), head = blockIdx.y;
    const bool value = K ? blockIdx.z : true;
    if (t >= M) return;
    const int slot = slots[t];
    const bool there = slot >= 0 && slot < (c.pages << c.lp);
    int32_t* y = (value ? V : K) + size_t(t) * ld + head * c.D;
    const int page = there ? slot >> c.lp : 0, at = there ? slot & ((1 << c.lp) - 1) : 0, t16 = at & 15;
    const int8_t* src = c.keys(page, head) + (value ? c.half_bytes() : 0) + (at >> 4) * c.group_bytes();
    const int e = there ? min(int(c.shifts(page, head)[(int(value) << c.lp) + at]), 31) : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = 4 * l + 64 * i;
        if (d >= c.D) break;
        int q[4] = {0, 0, 0, 0};
        if (there) {
#pragma unroll
            for (int p = 0; p < PL; ++p) {
                const int8_t* plane = src + p * 16 * c.D;
                char4 b;
                int8_t* bb = reinterpret_cast<int8_t*>(&b);
                if (value) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) bb[j] = plane[c.value_at(t16, d + j)];
                } else {
                    b = *reinterpret_cast<const char4*>(plane + c.key_at(t16, d));
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) q[j] = p == 0 ? bb[j] : 256 * q[j] + bb[j] + 128;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) q[j] = int(sat32(i64(q[j]) << e));
        }
        *reinterpret_cast<int4*>(y + d) = make_int4(q[0], q[1], q[2], q[3]);
    }
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
    const int r = blockIdx.x, p = t.parent[r];
    const bool there = unsigned(p) < unsigned(t.rows);
    const int n = there ? int(min(i64(max(t.len[p], 0)), i64(t.width) << lp)) : 0;
    const int full = n >> lp;
    const bool part = n & (t.page - 1);
    const int32_t* old = t.table + size_t(there ? p : 0) * t.ldt;
    int32_t* row = t.out_table + size_t(r) * t.ldt;
    for (int j = threadIdx.x; j < t.width; j += 256) row[j] = j < full ? old[j] : (j == full && part ? t.fresh[r] : -1);
    if (threadIdx.x == 0) {
        t.out_len[r] = n;
        t.src[r] = part ? old[full] : -1;
        t.dst[r] = part ? t.fresh[r] : -1;
    }
}

}  // namespace

hipError_t launch_kv_plan(hipStream_t st, const VgemmKvPlan& p, int lp) {
    // 256 token rows a block, or 1024 new pages where the rows are few; block 0 alone where there are none
    const int blocks = std::max(1, std::min((p.tokens + 255) / 256, 1024));
    kv_plan_kernel<<<blocks, 256, size_t(p.R) * 8, st>>>(p, lp);
    return hipGetLastError();
}

hipError_t launch_kv_write(hipStream_t st, const KvView& c, const int32_t* K, const int32_t* V, int ld, const int32_t* slot, int M) {
    const dim3 g((M + KV_TOKENS - 1) / KV_TOKENS, c.heads, 2);
    if (c.planes == 1) kv_write_kernel<1><<<g, 256, 0, st>>>(c, K, V, ld, slot, M);
    else kv_write_kernel<2><<<g, 256, 0, st>>>(c, K, V, ld, slot, M);
    return hipGetLastError();
}

hipError_t launch_kv_read(hipStream_t st, const KvView& c, const int32_t* slot, int M, int32_t* K, int32_t* V, int ld) {
    const dim3 g((M + KV_TOKENS - 1) / KV_TOKENS, c.heads, K && V ? 2 : 1);
    if (c.planes == 1) kv_read_kernel<1><<<g, 256, 0, st>>>(c, slot, M, K, V, ld);
    else kv_read_kernel<2><<<g, 256, 0, st>>>(c, slot, M, K, V, ld);
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
