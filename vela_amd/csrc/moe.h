// Launchers of the mixture-of-experts layer (moe.hip).
#pragma once
#include "w4_kernel.h"

namespace vk {

constexpr int MOE_EXPERTS = 512;   // experts a call can have
constexpr int MOE_TOPK = 16;       // choices a token can have
constexpr int MOE_PAIRS = 512;     // (token, choice) pairs one pass over the experts takes
constexpr int MOE_COLS = 8192;     // output columns one pass of the down product takes

struct RouteArgs {
    const int8_t *hi, *lo;
    int ld8;
    const int32_t* e;
    int K;
    const int8_t* W;
    int ldw;
    const int4* cst;
    int experts, topk, renorm;
    const i64* Lexp;
    int32_t *idx, *p, *logits;
};

struct MoeArgs {
    W4View up, down;             // of expert 0; the others follow at the strides
    size_t up_stride, down_stride;
    int experts, group_up, group_down;
    const int8_t *hi, *lo;
    int ld8;
    const int32_t* e;
    int M, topk, Kp16;
    const int32_t *idx, *p, *Lphi;
    int32_t* Y;
    int ldy;
    const int32_t* R;
    int32_t* v;                  // [pairs x F]
    uint32_t* vmax;              // [pairs x up_segs]: max |v| of a segment
    int up_segs;
    int32_t* y;                  // [pairs x MOE_COLS]: the experts' rows
    int col0, cols;              // output columns of this pass
};

hipError_t launch_moe_route(hipStream_t st, const RouteArgs& a, int M);
hipError_t launch_moe(hipStream_t st, const MoeArgs& a);

}  // namespace vk
