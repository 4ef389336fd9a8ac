// Selective state space scan: what its kernels share (ssm.cu: forward and single tokens, ssm_bwd.cu: gradients).
//
// Per channel c with its N states (A [C, N] real, B and C vectors per position and group of channels):
//     delta_t = softplus(dt_t + bias)   (or dt_t + bias)
//     h_t[n]  = exp(delta_t A[n]) h_{t-1}[n] + delta_t x_t B_t[n]
//     y_t     = (sum_n C_t[n] h_t[n] + D x_t) * silu(z_t)
// Everything between the loads and the stores is fp32.
//
// Layout of the work: a CTA owns SSM_CH = 64 neighbouring channels of one group, a lane two of them, so that a position's
// row of 16-bit values is one 128-byte access and every arithmetic instruction is one on a pair of floats (f32x2); its warps share
// the N states among them.  B_t[n] and C_t[n] are the same for all channels of a CTA: they lie in shared memory twice each, as
// pairs, and come as one 16-byte broadcast.  Where the channels do not fill the chip the positions are cut into segments: a first
// pass takes what every segment adds to the state, and the second one starts each segment from the sum of those in front of it.
#pragma once
#include <atomic>
#include <initializer_list>
#include <type_traits>

#include "pair_math.cuh"

namespace mlstm {

constexpr int SSM_CH = 64;          // channels per CTA
constexpr int SSM_ROWS = 8;         // positions whose operands a warp holds in registers at a time
constexpr int SSM_MAX_N = 64;       // states per channel
constexpr int SSM_WARPS = 4;        // forward: warps that do the recurrence
constexpr int SSM_AIDES = 4;        // forward: warps that prepare and finish
constexpr int SSM_THREADS = 32 * (SSM_WARPS + SSM_AIDES);
constexpr int SSM_CK = 16;          // positions between two states that the forward keeps for the backward

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

// ---- barriers between the two halves of a block: COUNT threads in all, of which some only announce themselves (arrive)
template <int COUNT>
__device__ __forceinline__ void half_sync(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(COUNT) : "memory"); }
template <int COUNT>
__device__ __forceinline__ void half_arrive(int id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(COUNT) : "memory"); }

// ---- loads and stores of a pair of neighbouring channels; PAIRS: aligned for one access; n: how many of the two exist
template <typename T>
struct Raw2 { uint32_t v; };
template <>
struct Raw2<float> { float2 v; };

template <bool PAIRS, typename T>
__device__ __forceinline__ Raw2<T> load_raw2(const T* p, int n) {
    Raw2<T> r;
    if constexpr (PAIRS) {                  // (n is 0 or 2)
        if constexpr (sizeof(T) == 4) r.v = make_float2(0.f, 0.f);
        else r.v = 0u;
        if (n) r.v = *reinterpret_cast<const decltype(r.v)*>(p);
    } else if constexpr (sizeof(T) == 4) {
        r.v = make_float2(n > 0 ? p[0] : 0.f, n > 1 ? p[1] : 0.f);
    } else {
        const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
        r.v = (n > 0 ? q[0] : 0u) | (n > 1 ? static_cast<uint32_t>(q[1]) << 16 : 0u);
    }
    return r;
}
template <typename T>
__device__ __forceinline__ float2 to_float2(Raw2<T> r) {
    if constexpr (sizeof(T) == 4) return r.v;
    else if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&r.v));
    else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r.v));
}
template <bool PAIRS, typename T>
__device__ __forceinline__ void store_pair(T* p, float2 v, int n) {
    if constexpr (PAIRS) {
        if (n == 0) return;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(p) = v;
        else if constexpr (std::is_same_v<T, __half>) *reinterpret_cast<__half2*>(p) = __float22half2_rn(v);
        else *reinterpret_cast<__nv_bfloat162*>(p) = __float22bfloat162_rn(v);
    } else {
        if (n > 0) p[0] = from_f32<T>(v.x);
        if (n > 1) p[1] = from_f32<T>(v.y);
    }
}

// softplus of both: max(v, 0) + log(1 + e), e = exp(-|v|).  The logarithm of 1 + e, which rounds away what a small e has, is taken
// by the series of 2 atanh(s), s = e / (2 + e) <= 1/3; the first term left out is below 2e-8 of the sum.
__device__ __forceinline__ f2 splat2(float a) { return pack2(a, a); }
__device__ __forceinline__ f2 softplus2(float2 v) {
    const f2 e = exp2_2(mul2(pack2(fabsf(v.x), fabsf(v.y)), splat2(-1.44269504088896340736f)));
    const float2 d = unpack2(add2(e, splat2(2.0f)));
    const f2 s = mul2(e, pack2(rcp_f(d.x), rcp_f(d.y))), t = mul2(s, s);
    f2 q = fma2(t, splat2(2.0f / 13.0f), splat2(2.0f / 11.0f));
    q = fma2(t, q, splat2(2.0f / 9.0f));
    q = fma2(t, q, splat2(2.0f / 7.0f));
    q = fma2(t, q, splat2(2.0f / 5.0f));
    q = fma2(t, q, splat2(2.0f / 3.0f));
    q = fma2(t, q, splat2(2.0f));
    return fma2(s, q, pack2(fmaxf(v.x, 0.0f), fmaxf(v.y, 0.0f)));
}
__device__ __forceinline__ float softplus_f(float v) { return unpack2(softplus2(make_float2(v, v))).x; }
// delta of both channels from the pre-activation
__device__ __forceinline__ f2 delta2(float2 raw, f2 bias, int softplus) {
    const f2 v = add2(pack2(raw.x, raw.y), bias);
    return softplus ? softplus2(unpack2(v)) : v;
}

// A in units of log2; -inf (and what is below -1e30) as -1e30: a step of 0 leaves the state (0 * -inf would be NaN), a step above 2e-28
// nothing of it.  Nor does the gradient of such a step overflow, which behind a softplus of -inf is multiplied by a slope of 0.
__device__ __forceinline__ float decay_rate(float a) {
    const float r = a * 1.44269504088896340736f;
    return r < -1.0e30f ? -1.0e30f : r;
}

// exp2(step * rate), the decays of one state over a step.  The hardware's exponential falls short of the value by 2e-8 on average for
// exponents from -0.25 to -1e-3, and by 7e-9 nearer to 0 (measured): a state that lives for a thousand positions would collect
// that a thousand times.  2e-8 in the exponent, added where it is multiplied anyway, takes the larger part of it back; a step of 0
// is still a decay of exactly 1.  (The gradient of A at 4 x 4096 positions, on three sets of inputs: 2.4e-6 off without, 1.6e-6 with it at 1024
// channels, 1.4e-6 and 0.7e-6 at 128, where the positions are cut into more segments and the sums over them are shorter.)
constexpr float DECAY_OFFSET = 2e-8f;
__device__ __forceinline__ f2 decay2(f2 step, f2 rate) { return exp2_2(fma2(step, rate, splat2(DECAY_OFFSET))); }
__device__ __forceinline__ float decay_f(float step, float rate) { return fast_exp2(fmaf(step, rate, DECAY_OFFSET)); }

// add + exp2(sum * rate) h: a state carried over a whole segment whose steps' sum this is.  The decay in two halves: the whole of it may
// be beyond what a float holds where the state behind it is not (steps one by one get there).  A half is at most 2^127: a normal
// number is beyond the range after two of those anyway, and 0 stays 0.  (Written so that NaN stays NaN.  Four quarters, which would
// hold for the states below the normal numbers too: 3 x 1001 x 600, 24 states, fp32 50 us in the place of 43.6.)
__device__ __forceinline__ f2 carry2(f2 sum, f2 rate, f2 h, f2 add) {
    float2 x = unpack2(fma2(mul2(sum, splat2(0.5f)), rate, splat2(DECAY_OFFSET)));
    x.x = x.x > 127.0f ? 127.0f : x.x;
    x.y = x.y > 127.0f ? 127.0f : x.y;
    const f2 e = exp2_2(pack2(x.x, x.y));
    return fma2(mul2(h, e), e, add);
}

// values of a parameter of the lane's two channels
__device__ __forceinline__ f2 param2(const float* p, int c, int n) { return pack2(p && n > 0 ? p[c] : 0.f, p && n > 1 ? p[c + 1] : 0.f); }

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
// Lets a kernel have more shared memory than a plain launch, once for each device (a call of its own costs a microsecond on the host).
template <typename... KArgs>
inline cudaError_t ssm_allow_smem(void (*kern)(KArgs...), size_t bytes, std::atomic<unsigned long long>& done) {
    int dev = 0;
    cudaError_t ce = cudaGetDevice(&dev);
    if (ce != cudaSuccess) return ce;
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
    ce = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (ce == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return ce;
}

}  // namespace mlstm
