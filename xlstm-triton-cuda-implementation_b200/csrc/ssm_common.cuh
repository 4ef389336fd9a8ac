// Selective state space scan: what its kernels share (ssm.cu: forward and single tokens, ssm_bwd.cu: gradients).
//
// Per channel c with its N states (A [C, N] real, B and C vectors per position and group of channels):
//     delta_t = softplus(dt_t + bias)   (or dt_t + bias)
//     h_t[n]  = exp(delta_t A[n]) h_{t-1}[n] + delta_t x_t B_t[n]
//     y_t     = (sum_n C_t[n] h_t[n] + D x_t) * silu(z_t)
// Everything between the loads and the stores is fp32.
//
// Layout of the work: a CTA owns SSM_CH = 64 neighbouring channels of one group, a lane two of them, so that a position's
// row of 16-bit values is one 128-byte access and every arithmetic instruction is one on a pair of floats (f32x2); the warps of
// the CTA share the N states among them, K each.  B_t[n] and C_t[n] are the same for all channels of a CTA: they lie in shared
// memory twice each, as pairs, and come as one 16-byte broadcast.
#pragma once
#include <initializer_list>
#include <type_traits>

#include "pair_math.cuh"

namespace mlstm {

constexpr int SSM_CH = 64;          // channels per CTA
constexpr int SSM_ROWS = 8;         // positions whose operands a warp holds in registers at a time
constexpr int SSM_MAX_N = 64;       // states per channel
constexpr int SSM_CK = 32;          // positions between two states that the forward keeps for the backward

// strides in elements between batch entries and between positions; the last dimension is contiguous
struct SsmStrides {
    long long b, t;
};

struct SsmArgs {
    const void *x, *dt, *z, *B, *C;
    SsmStrides sx, sdt, sz, sB, sC;
    const float *A, *D, *bias;
    int Bt, S, Ch, G, P, N;             // batch, positions, channels, groups, channels per group, states
    int tiles_g, Cpad;                  // CTAs per group; channels with every group rounded up to whole CTAs
    int softplus;
    int pairs;                          // x, dt, z, y (and dy, and the gradients) can be accessed two channels at a time
    int nseg, seglen;                   // segments that the positions are cut into (seglen a multiple of SSM_CK)
    float* ckpt;                        // [Bt, ceil(S / SSM_CK), N, Cpad] states in front of every SSM_CK positions, or nullptr
    float* seg_end;                     // [Bt, nseg, N, Cpad] what every segment adds to the state
    float* seg_sum;                     // [Bt, nseg, Cpad] sum of delta over every segment
};

__host__ __device__ constexpr int ceil_div(int a, int b) { return (a + b - 1) / b; }

// ---- loads and stores of a pair of neighbouring channels; `pairs`: aligned for one access; n: how many of the two exist
template <typename T>
struct Raw2 { uint32_t v; };
template <>
struct Raw2<float> { float2 v; };

template <typename T>
__device__ __forceinline__ Raw2<T> load_raw2(const T* p, bool pairs, int n) {
    Raw2<T> r;
    if constexpr (sizeof(T) == 4) {
        r.v = make_float2(0.f, 0.f);
        if (n == 2 && pairs) r.v = *reinterpret_cast<const float2*>(p);
        else {
            if (n > 0) r.v.x = p[0];
            if (n > 1) r.v.y = p[1];
        }
    } else {
        r.v = 0u;
        if (n == 2 && pairs) r.v = *reinterpret_cast<const uint32_t*>(p);
        else {
            const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
            if (n > 0) r.v = q[0];
            if (n > 1) r.v |= static_cast<uint32_t>(q[1]) << 16;
        }
    }
    return r;
}
template <typename T>
__device__ __forceinline__ float2 to_float2(Raw2<T> r) {
    if constexpr (sizeof(T) == 4) return r.v;
    else if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&r.v));
    else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r.v));
}
template <typename T>
__device__ __forceinline__ void store_pair(T* p, float2 v, bool pairs, int n) {
    if (n == 2 && pairs) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(p) = v;
        else if constexpr (std::is_same_v<T, __half>) *reinterpret_cast<__half2*>(p) = __float22half2_rn(v);
        else *reinterpret_cast<__nv_bfloat162*>(p) = __float22bfloat162_rn(v);
    } else {
        if (n > 0) p[0] = from_f32<T>(v.x);
        if (n > 1) p[1] = from_f32<T>(v.y);
    }
}

// log(1 + e) for 0 <= e <= 1 by the series of 2 atanh(e / (2 + e)): s = e / (2 + e) <= 1/3, and the first term left out is
// below 2e-8 of the sum.  (1 + e rounds away what a small e has.)
__device__ __forceinline__ float log1p_unit(float e) {
    const float s = __fdividef(e, 2.0f + e), t = s * s;
    float p = fmaf(t, 1.0f / 13.0f, 1.0f / 11.0f);
    p = fmaf(t, p, 1.0f / 9.0f);
    p = fmaf(t, p, 1.0f / 7.0f);
    p = fmaf(t, p, 1.0f / 5.0f);
    p = fmaf(t, p, 1.0f / 3.0f);
    return 2.0f * fmaf(s * t, p, s);
}
__device__ __forceinline__ float softplus_f(float v) { return fmaxf(v, 0.0f) + log1p_unit(__expf(-fabsf(v))); }
__device__ __forceinline__ float sigmoid_f(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

// A in units of log2; -inf as the lowest finite value, so that a step of 0 leaves the state (0 * -inf would be NaN)
__device__ __forceinline__ float decay_rate(float a) {
    const float r = a * 1.44269504088896340736f;
    return r < -3.0e38f ? -3.0e38f : r;
}

// Where a CTA's channels lie: group, first channel, channels of this lane (0, 1 or 2).
struct SsmTile {
    int g, c, n;      // c: first channel of the lane
    int cp;           // its place among the padded channels
};
__device__ __forceinline__ SsmTile ssm_tile(const SsmArgs& p, int tile, int lane) {
    SsmTile r;
    r.g = tile / p.tiles_g;
    const int in_g = (tile - r.g * p.tiles_g) * SSM_CH + 2 * lane;
    r.c = r.g * p.P + in_g;
    r.n = max(0, min(2, p.P - in_g));
    r.cp = tile * SSM_CH + 2 * lane;
    return r;
}

// host helpers (ssm.cu)
int ssm_fill(SsmArgs& a, const void* x, const void* dt, const float* A, const void* B, const void* C, const float* D, const void* z,
             const float* bias, const long long* strides, int Bt, int S, int Ch, int G, int N, int dtype, int softplus);
void ssm_cut(SsmArgs& a, int ctas_per_sm);
bool ssm_pairs(const SsmArgs& a, int es, std::initializer_list<const void*> more);
inline bool ssm_aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace mlstm
