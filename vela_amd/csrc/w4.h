// Launchers of the 4-bit products (w4.hip) and the mixture-of-experts layer (moe.hip).
#pragma once
#include "w4_kernel.h"

namespace vk {

struct W4Args {
    W4View w;
    int group;
    // rows: int8 planes (lo null: 8-bit rows) or int32 rows with their maxima
    const int8_t *hi, *lo;
    int ld8;
    const int32_t* e;
    const int32_t* x;
    int ldx;
    const uint32_t* xmax;
    int M, Kp16;
    // epilogue
    int geglu;
    int32_t* Y;
    int ldy;
    const int32_t *R, *Lphi;
    uint32_t* rowmax;
};

hipError_t launch_w4(hipStream_t st, const W4Args& a);
hipError_t launch_w4_pack(hipStream_t st, int N, int K, int group, uint8_t* q, int4* cst, int n, const uint8_t* nib, int ldn, const uint16_t* scale,
                          const uint8_t* zero, int lds, const int32_t* msb);

}  // namespace vk
