// Shared by the few-row products (bfp_few_rows.cu), the router (moe_route.cu) and the C ABI: limits and the argument
// block of the experts.
#pragma once

#include "buda_common.cuh"

namespace buda {

constexpr int kMaxFewRows = 64;      // rows / tokens of one call
constexpr int kMaxExperts = 256;
constexpr int kMaxTop = 16;

struct MoeArgs {
    const void *x;            // bfloat16 [T, H]
    int64_t ldx;
    int T, H, I, E, top, mant_bits, act;
    const float *weights;     // [T, top]
    const int *ids;           // [T, top]
    const void *gate, *up, *down;
    void *y;                  // bfloat16 [T, H]
    int64_t ldy;
    void *h;                  // workspace
};

// Workspace between the expert launches, binary32: every slot's intermediate row, and above kOneSum tokens a row of the result for
// every slot.
constexpr int kOneSum = 3;           // measured at launch_moe_experts
inline int64_t moe_h_bytes(int64_t T, int64_t top, int64_t I) { return T * top * (32 * ((I + 31) / 32)) * 4; }
inline int64_t moe_workspace(int64_t T, int64_t top, int64_t H, int64_t I)
{
    return moe_h_bytes(T, top, I) + (T > kOneSum ? T * top * (32 * ((H + 31) / 32)) * 4 : 0);
}

}  // namespace buda
