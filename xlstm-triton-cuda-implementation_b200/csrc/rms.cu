// Root-mean-square norm with the residual's addition:
//     s = x + residual   (rounded to the residual stream's type: what the next layer adds to is what is normalised here)
//     y = s / sqrt(mean(s^2) + eps) * w
// its result optionally in 8 bits (4 bits of exponent, 3 of mantissa) with one fp32 scale, amax / 448, for a row or for a block
// of 32, 64 or 128 values, and its gradients, with r = 1 / sqrt(mean(s^2) + eps) and u = dy * w:
//     ds = r (u - s r^2 mean(u s)) + (what comes down the stream),   dw = sum over the rows of dy s r.
// Everything between the loads and the stores is fp32.
//
// Bound by HBM: every row is read once and held in registers between the sum over it and its use.  A row belongs to a few lanes of
// a warp or, when it is longer than their registers, to a block.  Measured, bf16: 16384 x 4096 with residual forward 82 us (6.5 TB/s),
// backward 95 us (5.6 TB/s); 8192 x 4096 to 8 bits 52 us (4.5 TB/s: the blocks' barriers); 262144 rows of 128 fp32 values to
// 16 bits forward 40 us (5.0 TB/s), backward 90 (3.7 TB/s: 368 instructions for a warp's two rows, 58 % of the issue slots at four
// warps per scheduler; and 888 blocks where 740 fit, so a second wave of a fifth).
// What is far from its bytes: the backward on an fp32 stream (bf16 x, 16384 x 4096: 270 us where its bytes take 166; held to 64 registers for
// a second block, for which its ring leaves no room), rows above 8192 (4096 x 16384 bf16: forward 100, backward 131 us, of 83 each; the
// forms with 32 values a thread spill), and rows that are no multiple of 8 values or not aligned to 16 bytes, which go value by
// value (16384 x 4095: 208 and 434 us; 262144 rows of 33: 162 and 239).
#include <cuda_fp8.h>

#include "async_copy.cuh"
#include "pair_math.cuh"
#include "reduce_rows.cuh"
#include "vec_cvt.cuh"

namespace mlstm {
namespace {

struct RmsArgs {
    const void *x, *residual, *weight, *dy, *ds;
    void *y, *sum, *q, *dx, *dres;
    float *scale, *part;
    long long rows;
    int D, groups, inner;           // weight row of a row: (row / inner) % groups
    int wdt, ydt, xdt, block;       // element types; block: values per scale
    int lanes;                      // lanes of a warp per row
    float eps, inv_d;
};

template <int V>
__device__ __forceinline__ void store_any(void* p, int dtype, long long at, const float (&f)[V]) {
    if (dtype == MLSTM_DT_F32) store_vec<float, V>(static_cast<float*>(p) + at, from_floats<float, V>(f));
    else if (dtype == MLSTM_DT_F16) store_vec<__half, V>(static_cast<__half*>(p) + at, from_floats<__half, V>(f));
    else store_vec<__nv_bfloat16, V>(static_cast<__nv_bfloat16*>(p) + at, from_floats<__nv_bfloat16, V>(f));
}
template <int V>
__device__ __forceinline__ void load_weight(const RmsArgs& p, long long at, float (&w)[V]) {
    if (!p.weight) {
#pragma unroll
        for (int j = 0; j < V; j++) w[j] = 1.0f;
    } else if (p.wdt == MLSTM_DT_F32) to_floats<float, V>(load_vec<float, V>(static_cast<const float*>(p.weight) + at), w);
    else if (p.wdt == MLSTM_DT_F16) to_floats<__half, V>(load_vec<__half, V>(static_cast<const __half*>(p.weight) + at), w);
    else to_floats<__nv_bfloat16, V>(load_vec<__nv_bfloat16, V>(static_cast<const __nv_bfloat16*>(p.weight) + at), w);
}

// a / b from a * (1 / b), set right by its remainder (Markstein 1990): within 2^-21 of a unit in the last place of the quotient before
// it is rounded, where the remainder does not underflow
__device__ __forceinline__ float quotient(float a, float b, float inv) {
    const float o = a * inv;
    return fmaf(fmaf(-o, b, a), inv, o);
}
__device__ __forceinline__ f2 quotient2(f2 a, f2 minus_b, f2 inv) {
    const f2 o = mul2(a, inv);
    return fma2(fma2(o, minus_b, a), inv, o);
}
constexpr float FP8_MAX = 448.0f, FP8_TINY = 0x1p-80f;      // (remainders underflow where scales are below the latter)

// The scale of a block of values from its largest magnitude (its bits).  A quotient by 448 is 1/14 of a unit away from where two numbers
// are equally near, so this is the rounded one.  Below the normal numbers it is rounded up: the scale of a block that is not all zeros
// is not 0 then, and what is divided by it stays within 448.
__device__ __forceinline__ float block_scale(unsigned top) {
    const float t = __uint_as_float(top);
    if (t >= FP8_TINY && top < 0x7f800000u) return quotient(t, FP8_MAX, 1.0f / FP8_MAX);
    if (top == 0u) return 1.0f;
    return t < FP8_MAX * 0x1p-126f ? __fdiv_ru(t, FP8_MAX) : __fdiv_rn(t, FP8_MAX);
}

// V values in 8 bits: each to the nearest of its quotient by the scale that is returned (of 16-bit inputs one in ten thousand lies on a
// tie, from which a product with an approximate 448 / top goes to the wrong neighbour as often as not).  Where the scale is so
// small that remainders underflow, or no number, it is divided by.  8192 x 4096 bf16, blocks of 128: 50 us without the remainders,
// 52 with them, 59 with a division for each.
template <int V>
__device__ __forceinline__ void store_fp8(uint8_t* q, const float (&v)[V], float scale) {
    float t[V];
    if (scale >= FP8_TINY && scale < __uint_as_float(0x7f800000u)) {
        const float inv = rcp_f(scale);
        if constexpr (V == 8) {
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const float2 o = unpack2(quotient2(pack2(v[j], v[j + 1]), pack2(-scale, -scale), pack2(inv, inv)));
                t[j] = o.x;
                t[j + 1] = o.y;
            }
        } else {
            t[0] = quotient(v[0], scale, inv);
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) t[j] = __fdiv_rn(v[j], scale);
    }
    if constexpr (V == 8) {
        __nv_fp8x2_storage_t o[4];
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = __nv_cvt_float2_to_fp8x2(make_float2(t[2 * j], t[2 * j + 1]), __NV_SATFINITE, __NV_E4M3);
        *reinterpret_cast<uint2*>(q) = make_uint2(o[0] | (static_cast<unsigned>(o[1]) << 16), o[2] | (static_cast<unsigned>(o[3]) << 16));
    } else {
        *q = __nv_cvt_float_to_fp8(t[0], __NV_SATFINITE, __NV_E4M3);
    }
}

// Sum of a pair over the threads of a row: `tpr` lanes of a warp, or the whole block.  Every thread gets it.
template <bool WARP>
__device__ __forceinline__ float2 row_sum(float2 v, float2* sm, int tpr) {
    for (int o = WARP ? tpr >> 1 : 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if (WARP) return v;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (lane == 0) sm[warp] = v;
    __syncthreads();
    v = lane < warps ? sm[lane] : make_float2(0.f, 0.f);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    __syncthreads();                // (sm is used again)
    return v;
}

// T: x, S: the stream (x's type where there is no residual).  A thread's values are V neighbouring ones, K times.
template <typename T, typename S, int V, int K, bool WARP, bool QUANT>
__global__ void __launch_bounds__(WARP ? 128 : 512, WARP ? 8 : V == 8 && K == 2 ? 3 : 1) rms_fwd_kernel(const RmsArgs p) {
    __shared__ float2 sm[32];
    extern __shared__ unsigned amax[];      // QUANT: largest magnitude of every block of the row (as bits: NaN above all)
    grid_dep_wait();
    grid_dep_launch();
    const int tpr = WARP ? p.lanes : blockDim.x, tid = WARP ? threadIdx.x & (tpr - 1) : threadIdx.x;
    const int slot = WARP ? static_cast<int>(threadIdx.x) / tpr : 0;
    const long long row = WARP ? static_cast<long long>(blockIdx.x) * (blockDim.x / tpr) + slot : blockIdx.x;
    const int D = row < p.rows ? p.D : 0;   // (lanes of a warp without a row take part in its sums with nothing)
    const T* x = static_cast<const T*>(p.x) + row * p.D;
    const S* res = p.residual ? static_cast<const S*>(p.residual) + row * p.D : nullptr;
    float v[K][V];
    Vec<T, V> xv[K];
    Vec<S, V> rv[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int e = (k * tpr + tid) * V;
        if (e < D) {
            xv[k] = load_vec<T, V>(x + e);
            if (res) rv[k] = load_vec<S, V>(res + e);
        }
    }
    float2 acc = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int e = (k * tpr + tid) * V;
        if (e < D) {
            to_floats<T, V>(xv[k], v[k]);
            if (res) {
                float r[V];
                to_floats<S, V>(rv[k], r);
#pragma unroll
                for (int j = 0; j < V; j++) v[k][j] += r[j];
                const Vec<S, V> t = from_floats<S, V>(v[k]);
                store_vec<S, V>(static_cast<S*>(p.sum) + row * p.D + e, t);
                to_floats<S, V>(t, v[k]);
            }
#pragma unroll
            for (int j = 0; j < V; j++) acc.x = fmaf(v[k][j], v[k][j], acc.x);
        }
    }
    acc = row_sum<WARP>(acc, sm, tpr);
    const float r = rsqrtf(acc.x * p.inv_d + p.eps);
    const long long wrow = p.groups > 1 ? (row / p.inner) % p.groups * p.D : 0;
    unsigned* top = amax + slot * (p.D / p.block);
    if (QUANT) {
        for (int i = tid; i < p.D / p.block; i += tpr) top[i] = 0u;
        if (WARP) __syncwarp();
        else __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int e = (k * tpr + tid) * V;
        float w[V];
        if (e < D) {
            load_weight<V>(p, wrow + e, w);
#pragma unroll
            for (int j = 0; j < V; j++) v[k][j] = v[k][j] * r * w[j];
        }
        if (!QUANT) {
            if (e < D) store_any<V>(p.y, p.ydt, row * p.D + e, v[k]);
        } else {
            unsigned m = 0u;
            if (e < D) {
#pragma unroll
                for (int j = 0; j < V; j++) m = max(m, __float_as_uint(v[k][j]) & 0x7fffffffu);
            }
            // neighbouring threads of one block of values first (all of a warp's are in one block or every few are)
            const int same = min(tpr < 32 ? tpr : 32, p.block / V > 0 ? p.block / V : 1);
            if ((same & (same - 1)) == 0)
                for (int o = same >> 1; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (e < D) atomicMax(&top[e / p.block], m);       // (the largest: no order to depend on)
        }
    }
    if (QUANT) {
        if (WARP) __syncwarp();
        else __syncthreads();
        const int blocks = p.D / p.block;
        for (int i = tid; i < blocks && D > 0; i += tpr) p.scale[row * blocks + i] = block_scale(top[i]);
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int e = (k * tpr + tid) * V;
            if (e < D) store_fp8<V>(static_cast<uint8_t*>(p.q) + row * p.D + e, v[k], block_scale(top[e / p.block]));
        }
    }
}

// S: the stream's type, T: dy's.  Blocks (or parts of warps) walk over the rows of one group and keep their part of the weight's
// gradient.  Where a thread has eight values of a row (PIPE), its pieces of the next rows are on their way to shared memory
// while it works on one (each thread reads back what it asked for itself: no barrier).
template <typename T, typename S, int V, int K, bool WARP>
struct RmsPipe {
    static constexpr bool ON = V == 8 && K == 1;
    static constexpr int STAGES = 3, NS = sizeof(S) * V / 16, NT = sizeof(T) * V / 16, PIECES = 2 * NS + NT;   // s, ds, dy in 16 bytes
    __host__ __device__ static constexpr size_t bytes(int threads) { return ON ? static_cast<size_t>(STAGES) * PIECES * threads * 16 : 0; }
};
template <typename T, typename S, int V, int K, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 512, WARP ? 4 : V == 8 && K == 1 ? 2 : 1) rms_bwd_kernel(const RmsArgs p) {
    using Pipe = RmsPipe<T, S, V, K, WARP>;
    __shared__ float2 sm[32];
    extern __shared__ __align__(16) unsigned char dyn[];
    grid_dep_wait();
    grid_dep_launch();
    const int tpr = WARP ? p.lanes : blockDim.x, tid = WARP ? threadIdx.x & (tpr - 1) : threadIdx.x;
    const int rpb = WARP ? static_cast<int>(blockDim.x) / tpr : 1, slot = WARP ? static_cast<int>(threadIdx.x) / tpr : 0, g = blockIdx.y;
    const long long rows_g = p.rows / p.groups, step = static_cast<long long>(gridDim.x) * rpb;
    float dw[K][V], w[K][V];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int e = (k * tpr + tid) * V;
#pragma unroll
        for (int j = 0; j < V; j++) dw[k][j] = 0.f;
        if (e < p.D) load_weight<V>(p, static_cast<long long>(g) * p.D + e, w[k]);
    }
    auto row_of = [&](long long i) { return p.groups > 1 ? ((i / p.inner) * p.groups + g) * p.inner + i % p.inner : i; };
    [[maybe_unused]] uint4* ring = reinterpret_cast<uint4*>(dyn) + threadIdx.x;        // [stage][piece][thread]
    [[maybe_unused]] const int pitch = blockDim.x;
    auto fetch = [&](long long i, int stage) {
        if constexpr (Pipe::ON) {
            if (i < rows_g && tid * V < p.D) {
                const long long at = row_of(i) * p.D + tid * V;
                uint4* q = ring + stage * Pipe::PIECES * pitch;
#pragma unroll
                for (int c = 0; c < Pipe::NS; c++) {
                    copy_async<16>(shared_address(q + c * pitch), reinterpret_cast<const uint4*>(static_cast<const S*>(p.x) + at) + c);
                    if (p.ds) copy_async<16>(shared_address(q + (Pipe::NS + c) * pitch), reinterpret_cast<const uint4*>(static_cast<const S*>(p.ds) + at) + c);
                }
#pragma unroll
                for (int c = 0; c < Pipe::NT; c++)
                    copy_async<16>(shared_address(q + (2 * Pipe::NS + c) * pitch), reinterpret_cast<const uint4*>(static_cast<const T*>(p.dy) + at) + c);
            }
            copies_commit();
        }
    };
    int stage = 0;
    const long long first = static_cast<long long>(blockIdx.x) * rpb + slot;
#pragma unroll
    for (int k = 0; k < Pipe::STAGES - 1; k++) fetch(first + k * step, k);
    // (the same number of turns for all lanes of a warp; a lane past the last row takes part in the sums with nothing)
    for (long long i = first; i - slot < rows_g; i += step) {
        const int D = i < rows_g ? p.D : 0;
        const long long row = D ? row_of(i) : 0;
        const S* s = static_cast<const S*>(p.x) + row * p.D;
        const T* dy = static_cast<const T*>(p.dy) + row * p.D;
        const S* ds = p.ds ? static_cast<const S*>(p.ds) + row * p.D : nullptr;
        Vec<S, V> sv[K], dsv[K];
        Vec<T, V> dv[K];
        if constexpr (Pipe::ON) {
            copies_wait<Pipe::STAGES - 2>();
            const uint4* q = ring + stage * Pipe::PIECES * pitch;
#pragma unroll
            for (int c = 0; c < Pipe::NS; c++) {
                reinterpret_cast<uint4*>(&sv[0])[c] = q[c * pitch];
                if (ds) reinterpret_cast<uint4*>(&dsv[0])[c] = q[(Pipe::NS + c) * pitch];
            }
#pragma unroll
            for (int c = 0; c < Pipe::NT; c++) reinterpret_cast<uint4*>(&dv[0])[c] = q[(2 * Pipe::NS + c) * pitch];
            const int into = stage == 0 ? Pipe::STAGES - 1 : stage - 1;      // used up one turn ago
            fetch(i + (Pipe::STAGES - 1) * step, into);
            stage = stage + 1 == Pipe::STAGES ? 0 : stage + 1;
        } else {
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int e = (k * tpr + tid) * V;
                if (e < D) {
                    sv[k] = load_vec<S, V>(s + e);
                    dv[k] = load_vec<T, V>(dy + e);
                    if (ds) dsv[k] = load_vec<S, V>(ds + e);
                }
            }
        }
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < K; k++) {
            if ((k * tpr + tid) * V < D) {
                float a[V], d[V];
                to_floats<S, V>(sv[k], a);
                to_floats<T, V>(dv[k], d);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    acc.x = fmaf(a[j], a[j], acc.x);
                    acc.y = fmaf(a[j] * w[k][j], d[j], acc.y);
                }
            }
        }
        acc = row_sum<WARP>(acc, sm, tpr);
        const float r = rsqrtf(acc.x * p.inv_d + p.eps), m = acc.y * p.inv_d * r * r;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int e = (k * tpr + tid) * V;
            if (e < D) {
                float a[V], d[V], o[V];
                to_floats<S, V>(sv[k], a);
                to_floats<T, V>(dv[k], d);
                if (ds) to_floats<S, V>(dsv[k], o);
                const float m2 = -m * r;                 // r (d w - a m) + ds
#pragma unroll
                for (int j = 0; j < V; j++) {
                    d[j] *= r;
                    o[j] = fmaf(d[j], w[k][j], ds ? fmaf(a[j], m2, o[j]) : a[j] * m2);
                    dw[k][j] = fmaf(d[j], a[j], dw[k][j]);
                }
                store_any<V>(p.dx, p.xdt, row * p.D + e, o);
                if (p.dres) store_vec<S, V>(static_cast<S*>(p.dres) + row * p.D + e, from_floats<S, V>(o));
            }
        }
    }
    if (!p.part) return;
    float* part = p.part + (static_cast<long long>(blockIdx.x) * p.groups + g) * p.D;
    float* sum = reinterpret_cast<float*>(dyn + Pipe::bytes(blockDim.x));
    for (int turn = 0; turn < rpb; turn++) {        // a block's rows at a time, one after the other
        if (WARP && turn > 0) __syncthreads();
        if (slot == turn) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int e = (k * tpr + tid) * V;
                if (e < p.D) {
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        const float t = (turn > 0 ? sum[e + j] : 0.f) + dw[k][j];
                        if (turn == rpb - 1) part[e + j] = t;
                        else sum[e + j] = t;
                    }
                }
            }
        }
    }
}

struct RmsWeightOut {
    AnyOut dw;
    __device__ __forceinline__ void operator()(long long at, float v) const { dw.put(at, v); }
};

constexpr int RMS_MAX_D = 16384;
// How a row is laid over threads: V values each, K times, by `lanes` lanes of a warp (several rows in a block of 128 threads) or, lanes
// = 0, by a whole block of `threads`.
struct RmsPlan {
    int V, K, threads, lanes;
    int rows() const { return lanes ? threads / lanes : 1; }
};
RmsPlan rms_plan(int D, bool wide, bool bwd) {
    const int V = wide ? 8 : 1, K = wide ? (bwd ? 1 : 2) : 16;       // the backward holds three rows and two more of floats
    const int in_warp = wide ? (bwd ? 256 : 1024) : 512;
    if (D <= in_warp) {
        const int k = wide ? (D <= 256 ? 1 : D <= 512 ? 2 : 4) : K;
        int lanes = 32;
        while (wide && lanes > 8 && lanes / 2 * V >= D) lanes /= 2;
        return {V, k, 128, lanes};
    }
    RmsPlan p{V, K, 64, 0};
    while (p.threads * V * p.K < D && p.threads < 512) p.threads *= 2;
    while (p.threads * V * p.K < D) p.K *= 2;
    return p;
}
int rms_bwd_blocks(long long rows_g, int groups, const RmsPlan& pl) {
    const int rpb = pl.rows(), per_sm = pl.lanes ? 6 : 1024 / pl.threads;
    long long want = 148LL * per_sm / groups;
    if (want < 1) want = 1;
    const long long most = (rows_g + rpb - 1) / rpb;
    return static_cast<int>(want < most ? want : most);
}

template <typename T, typename S, bool QUANT>
cudaError_t launch_rms_fwd(RmsArgs a, bool wide, cudaStream_t st) {
    const RmsPlan pl = rms_plan(a.D, wide, false);
    const int rpb = pl.rows();
    a.lanes = pl.lanes;
    const dim3 grid(static_cast<unsigned>((a.rows + rpb - 1) / rpb)), block(pl.threads);
    const size_t smem = QUANT ? static_cast<size_t>(rpb) * (a.D / a.block) * 4 : 0;
    if (pl.V == 1) {
        if (pl.lanes) return launch_plain(rms_fwd_kernel<T, S, 1, 16, true, QUANT>, grid, block, smem, st, a);
        if (pl.K == 16) return launch_plain(rms_fwd_kernel<T, S, 1, 16, false, QUANT>, grid, block, smem, st, a);
        return launch_plain(rms_fwd_kernel<T, S, 1, 32, false, QUANT>, grid, block, smem, st, a);
    }
    if (!pl.lanes && pl.K == 4) return launch_plain(rms_fwd_kernel<T, S, 8, 4, false, QUANT>, grid, block, smem, st, a);
    if (!pl.lanes) return launch_plain(rms_fwd_kernel<T, S, 8, 2, false, QUANT>, grid, block, smem, st, a);
    if (pl.K == 1) return launch_plain(rms_fwd_kernel<T, S, 8, 1, true, QUANT>, grid, block, smem, st, a);
    if (pl.K == 2) return launch_plain(rms_fwd_kernel<T, S, 8, 2, true, QUANT>, grid, block, smem, st, a);
    return launch_plain(rms_fwd_kernel<T, S, 8, 4, true, QUANT>, grid, block, smem, st, a);
}
template <typename T, typename S, int V, int K, bool WARP>
cudaError_t launch_rms_bwd_k(const RmsArgs& a, const RmsPlan& pl, cudaStream_t st) {
    const dim3 grid(rms_bwd_blocks(a.rows / a.groups, a.groups, pl), a.groups), block(pl.threads);
    const size_t smem = RmsPipe<T, S, V, K, WARP>::bytes(pl.threads) + (WARP && a.part ? static_cast<size_t>(a.D) * 4 : 0);
    auto kern = rms_bwd_kernel<T, S, V, K, WARP>;
    if (smem > 48 * 1024) {
        const cudaError_t ce = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (ce != cudaSuccess) return ce;
    }
    return launch_plain(kern, grid, block, smem, st, a);
}
template <typename T, typename S>
cudaError_t launch_rms_bwd(RmsArgs a, bool wide, cudaStream_t st) {
    const RmsPlan pl = rms_plan(a.D, wide, true);
    a.lanes = pl.lanes;
    if (pl.V == 1)
        return pl.lanes ? launch_rms_bwd_k<T, S, 1, 16, true>(a, pl, st)
               : pl.K == 16 ? launch_rms_bwd_k<T, S, 1, 16, false>(a, pl, st) : launch_rms_bwd_k<T, S, 1, 32, false>(a, pl, st);
    if (pl.lanes) return launch_rms_bwd_k<T, S, 8, 1, true>(a, pl, st);
    return pl.K == 1 ? launch_rms_bwd_k<T, S, 8, 1, false>(a, pl, st)
           : pl.K == 2 ? launch_rms_bwd_k<T, S, 8, 2, false>(a, pl, st) : launch_rms_bwd_k<T, S, 8, 4, false>(a, pl, st);
}

inline int elem_size(int dt) { return dt == MLSTM_DT_F32 ? 4 : 2; }
inline bool dtype_ok(int dt) { return dt == MLSTM_DT_F32 || dt == MLSTM_DT_F16 || dt == MLSTM_DT_BF16; }

int rms_check(long long rows, int D, int groups, int inner, int a_dtype, int s_dtype, int w_dtype, bool weight) {
    if (rows <= 0 || D <= 0 || groups <= 0 || inner <= 0) return MLSTM_E_ARG;
    if (!dtype_ok(a_dtype) || !dtype_ok(s_dtype) || (weight && !dtype_ok(w_dtype))) return MLSTM_E_ARG;
    if (s_dtype != a_dtype && s_dtype != MLSTM_DT_F32) return MLSTM_E_ARG;
    if (D > RMS_MAX_D || rows > 0x7fffffffLL || groups > 65535) return MLSTM_E_SHAPE;
    if (groups > 1 && rows % (static_cast<long long>(groups) * inner)) return MLSTM_E_SHAPE;
    return MLSTM_OK;
}
// 8 values at a time: rows of whole 16-byte pieces in every tensor
bool rms_wide(int D, std::initializer_list<const void*> ps) {
    if (D % 8) return false;
    for (const void* q : ps)
        if (!aligned(q, 16)) return false;
    return true;
}

}  // namespace
}  // namespace mlstm

using namespace mlstm;

extern "C" {

int mlstm_rms_fwd(const void* x, const void* residual, const void* weight, void* y, void* sum, float* scale, long long rows, int D,
                  int groups, int inner, int block, float eps, int dtype, int s_dtype, int w_dtype, int y_dtype, void* stream) {
    int rc = rms_check(rows, D, groups, inner, dtype, s_dtype, w_dtype, weight != nullptr);
    if (rc != MLSTM_OK) return rc;
    if (!x || !y || (residual == nullptr) != (sum == nullptr) || (scale == nullptr) != (block == 0)) return MLSTM_E_ARG;
    if (!scale && !dtype_ok(y_dtype)) return MLSTM_E_ARG;
    if (!residual && s_dtype != dtype) return MLSTM_E_ARG;
    if (block < 0 || (block > 0 && (D % block || (block != D && block != 32 && block != 64 && block != 128)))) return MLSTM_E_SHAPE;
    if (!aligned(x, elem_size(dtype)) || !aligned(residual, elem_size(s_dtype)) || !aligned(sum, elem_size(s_dtype)) ||
        !aligned(weight, elem_size(w_dtype)) || (!scale && !aligned(y, elem_size(y_dtype))) || !aligned(scale, 4))
        return MLSTM_E_ALIGN;
    RmsArgs a{};
    a.x = x; a.residual = residual; a.weight = weight; a.sum = sum; a.scale = scale;
    if (scale) a.q = y;
    else a.y = y;
    a.rows = rows; a.D = D; a.groups = groups; a.inner = inner;
    a.wdt = w_dtype; a.ydt = y_dtype; a.block = block ? block : D;
    a.eps = eps; a.inv_d = 1.0f / static_cast<float>(D);
    const bool wide = rms_wide(D, {x, residual, weight, y, sum});
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t ce;
#define RMS_FWD(T, S) (scale ? launch_rms_fwd<T, S, true>(a, wide, st) : launch_rms_fwd<T, S, false>(a, wide, st))
    if (dtype == MLSTM_DT_F32) ce = RMS_FWD(float, float);
    else if (dtype == MLSTM_DT_F16) ce = s_dtype == MLSTM_DT_F32 ? RMS_FWD(__half, float) : RMS_FWD(__half, __half);
    else ce = s_dtype == MLSTM_DT_F32 ? RMS_FWD(__nv_bfloat16, float) : RMS_FWD(__nv_bfloat16, __nv_bfloat16);
#undef RMS_FWD
    if (ce != cudaSuccess) cudaGetLastError();
    return ce == cudaSuccess ? MLSTM_OK : note_cuda_error(ce, "launch of rms_fwd_kernel");
}

size_t mlstm_rms_bwd_workspace(long long rows, int D, int groups, int inner) {
    if (rms_check(rows, D, groups, inner, 0, 0, 0, false) != MLSTM_OK) return 0;
    const long long rows_g = rows / groups;
    const int a = rms_bwd_blocks(rows_g, groups, rms_plan(D, true, true)), b = rms_bwd_blocks(rows_g, groups, rms_plan(D, false, true));
    return static_cast<size_t>(a > b ? a : b) * groups * D * sizeof(float);
}

int mlstm_rms_bwd(const void* dy, const void* ds, const void* s, const void* weight, void* dx, void* dres, void* dweight,
                  void* workspace, size_t workspace_bytes, long long rows, int D, int groups, int inner, float eps, int x_dtype,
                  int s_dtype, int w_dtype, int dy_dtype, void* stream) {
    int rc = rms_check(rows, D, groups, inner, dy_dtype, s_dtype, w_dtype, weight != nullptr);
    if (rc != MLSTM_OK) return rc;
    if (!dy || !s || !dx || !dtype_ok(x_dtype) || (weight == nullptr) != (dweight == nullptr)) return MLSTM_E_ARG;
    if (!aligned(dy, elem_size(dy_dtype)) || !aligned(ds, elem_size(s_dtype)) || !aligned(s, elem_size(s_dtype)) ||
        !aligned(weight, elem_size(w_dtype)) || !aligned(dweight, elem_size(w_dtype)) || !aligned(dx, elem_size(x_dtype)) ||
        !aligned(dres, elem_size(s_dtype)))
        return MLSTM_E_ALIGN;
    if (weight && (!workspace || workspace_bytes < mlstm_rms_bwd_workspace(rows, D, groups, inner) || !aligned(workspace, 16)))
        return MLSTM_E_WORKSPACE;
    RmsArgs a{};
    a.x = s; a.dy = dy; a.ds = ds; a.weight = weight; a.dx = dx; a.dres = dres;
    a.part = weight ? static_cast<float*>(workspace) : nullptr;
    a.rows = rows; a.D = D; a.groups = groups; a.inner = inner;
    a.wdt = w_dtype; a.xdt = x_dtype; a.block = D;
    a.eps = eps; a.inv_d = 1.0f / static_cast<float>(D);
    const bool wide = rms_wide(D, {dy, ds, s, weight, dx, dres});
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t ce;
    if (dy_dtype == MLSTM_DT_F32) ce = launch_rms_bwd<float, float>(a, wide, st);
    else if (dy_dtype == MLSTM_DT_F16) ce = s_dtype == MLSTM_DT_F32 ? launch_rms_bwd<__half, float>(a, wide, st) : launch_rms_bwd<__half, __half>(a, wide, st);
    else ce = s_dtype == MLSTM_DT_F32 ? launch_rms_bwd<__nv_bfloat16, float>(a, wide, st) : launch_rms_bwd<__nv_bfloat16, __nv_bfloat16>(a, wide, st);
    if (ce == cudaSuccess && weight) {
        const int blocks = rms_bwd_blocks(rows / groups, groups, rms_plan(D, wide, true));
        ce = launch_reduce_rows(a.part, blocks, static_cast<long long>(groups) * D, RmsWeightOut{{dweight, w_dtype}}, st);
    }
    if (ce != cudaSuccess) cudaGetLastError();
    return ce == cudaSuccess ? MLSTM_OK : note_cuda_error(ce, "launch of rms_bwd_kernel");
}

}  // extern "C"
