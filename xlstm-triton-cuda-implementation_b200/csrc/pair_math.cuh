// Two floats as one operand: the packed fp32 instructions of sm_100.  They run at the rate of the plain ones (128 multiply-adds per
// cycle and SM) in half as many issue slots, which the hardware's exponential and the loads then have.
#pragma once
#include "mlstm_common.cuh"

namespace mlstm {

using f2 = unsigned long long;
__device__ __forceinline__ f2 pack2(float a, float b) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(f2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f2 exp2_2(f2 x) {
    const float2 v = unpack2(x);
    return pack2(fast_exp2(v.x), fast_exp2(v.y));
}

__device__ __forceinline__ float rcp_f(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float sigmoid_f(float x) { return rcp_f(1.0f + fast_exp2(x * -1.44269504088896340736f)); }
// sigmoid of both: two hardware functions each, good to a few units in the last place (exp(-x) = inf gives 0)
__device__ __forceinline__ f2 sigmoid2(f2 x) {
    const float2 e = unpack2(exp2_2(mul2(x, pack2(-1.44269504088896340736f, -1.44269504088896340736f))));
    return pack2(rcp_f(1.0f + e.x), rcp_f(1.0f + e.y));
}

}  // namespace mlstm
