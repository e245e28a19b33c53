// The paged key-value cache (include/vgemm_kv.h): addresses within a page, argument blocks and launchers.
#pragma once
#include "../../include/vgemm_kv.h"
#include "vk_common.h"

namespace vk {

constexpr int KV_SPAN = 256;           // positions whose weights share a maximum
constexpr int KV_PLAN_ROWS = 4096;     // requests of a plan: their running sums stand in LDS
constexpr int KV_MAX_LEN = 1 << 23;    // tokens of a sequence: 2^15 spans of weights below 2^47 add up below 2^62
constexpr int BEAM_SPAN = 4096;        // tokens of the vocabulary whose weights share a maximum
constexpr int BEAM_MOST = 32, BEAM_N = 64, BEAM_V = 1 << 18;

struct KvView {
    int8_t* data;
    uint8_t* shift;
    int pages, lp, heads, D, planes;   // lp: log2 of the tokens of a page

    __host__ __device__ int group_bytes() const { return 16 * D * planes; }
    __host__ __device__ int half_bytes() const { return (D * planes) << lp; }         // a page's keys, or its values, of one head
    __device__ int8_t* keys(int page, int head) const { return data + (size_t(page) * heads + head) * (2u * unsigned(half_bytes())); }
    __device__ uint8_t* shifts(int page, int head) const { return shift + (((size_t(page) * heads + head) * 2) << lp); }
    // offsets in a group of 16 tokens
    __device__ int key_at(int t, int d) const { return (t >> 2) * 4 * D + (d >> 4) * 64 + (t & 3) * 16 + (d & 15); }
    __device__ int value_at(int t, int d) const { return d * 16 + t; }
};

struct KvAttnArgs {
    KvView c;
    const int32_t* Q;
    int ldq, rows, Hq, group, qtiles;
    const int32_t* table;
    int ldt, width;
    const int32_t* len;
    int max_len, window;
    int m, s;
    const long long* Lexp;
    int32_t* out;
    int ldo;
    uint32_t* rowmax;
    int2* stat;         // [rows][Hq][spans] {mx, L}
    int32_t* part;      // [rows][Hq][spans][D]
    int spans;          // of max_len
};

struct BeamStat { long long S; int mx, pad; };
struct BeamArgs {
    VgemmBeam b;
    int spans;
    BeamStat* stat;     // [rows][spans]
    int2* cand;         // [rows][spans][n] {z, token}, in falling order; token -1: none
};

hipError_t launch_kv_plan(hipStream_t st, const VgemmKvPlan& p, int lp);
hipError_t launch_kv_write(hipStream_t st, const KvView& c, const int32_t* K, const int32_t* V, int ld, const int32_t* slot, int M);
hipError_t launch_kv_read(hipStream_t st, const KvView& c, const int32_t* slot, int M, int32_t* K, int32_t* V, int ld);
hipError_t launch_kv_copy(hipStream_t st, const KvView& c, const int32_t* src, const int32_t* dst, int n);
hipError_t launch_kv_attention(hipStream_t st, const KvAttnArgs& a);
hipError_t launch_beam_select(hipStream_t st, const BeamArgs& a);
hipError_t launch_beam_tables(hipStream_t st, const VgemmBeamTables& t, int lp);

}  // namespace vk
