// Root-mean-square norm with the residual's addition:
//     s = x + residual   (rounded to the residual stream's type: what the next layer adds to is what is normalised here)
//     y = s / sqrt(mean(s^2) + eps) * w
// its result optionally in 8 bits (4 bits of exponent, 3 of mantissa) with one fp32 scale, amax / 448, for a row or for a block
// of 32, 64 or 128 values, and its gradients, with r = 1 / sqrt(mean(s^2) + eps) and u = dy * w:
//     ds = r (u - s r^2 mean(u s)) + (what comes down the stream),   dw = sum over the rows of dy s r.
// Everything between the loads and the stores is fp32.
//
// Bound by HBM: every row is read once and held in registers between the sum over it and its use.  A row belongs to one warp
// or, when it is longer than a warp's registers, to one block.
#include <cuda_fp8.h>

#include "reduce_rows.cuh"

namespace mlstm {
namespace {

struct RmsArgs {
    const void *x, *residual, *weight, *dy, *ds;
    void *y, *sum, *q, *dx, *dres;
    float *scale, *part;
    long long rows;
    int D, groups, inner;           // weight row of a row: (row / inner) % groups
    int wdt, ydt, xdt, block;       // element types; block: values per scale
    float eps, inv_d;
};

// V values: 16 bytes of 16-bit values, 2 x 16 of fp32, or a single one
template <typename T, int V>
struct RVec {
    T v[V];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (V == 1) v[0] = *p;
        else {
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(v) / 16); i++)
                reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(p)[i];
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (V == 1) *p = v[0];
        else {
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(v) / 16); i++)
                reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(v)[i];
        }
    }
};
template <typename T, int V>
struct alignas(V == 1 ? sizeof(T) : 16) RVecA : RVec<T, V> {};

template <int V>
__device__ __forceinline__ void store_any(void* p, int dtype, long long at, const float (&f)[V]) {
    if (dtype == MLSTM_DT_F32) {
        RVecA<float, V> o;
#pragma unroll
        for (int j = 0; j < V; j++) o.v[j] = f[j];
        o.store(static_cast<float*>(p) + at);
    } else if (dtype == MLSTM_DT_F16) {
        RVecA<__half, V> o;
#pragma unroll
        for (int j = 0; j < V; j++) o.v[j] = from_f32<__half>(f[j]);
        o.store(static_cast<__half*>(p) + at);
    } else {
        RVecA<__nv_bfloat16, V> o;
#pragma unroll
        for (int j = 0; j < V; j++) o.v[j] = from_f32<__nv_bfloat16>(f[j]);
        o.store(static_cast<__nv_bfloat16*>(p) + at);
    }
}
template <int V>
__device__ __forceinline__ void load_weight(const RmsArgs& p, long long at, float (&w)[V]) {
    if (!p.weight) {
#pragma unroll
        for (int j = 0; j < V; j++) w[j] = 1.0f;
    } else if (p.wdt == MLSTM_DT_F32) {
        RVecA<float, V> r;
        r.load(static_cast<const float*>(p.weight) + at);
#pragma unroll
        for (int j = 0; j < V; j++) w[j] = r.v[j];
    } else if (p.wdt == MLSTM_DT_F16) {
        RVecA<__half, V> r;
        r.load(static_cast<const __half*>(p.weight) + at);
#pragma unroll
        for (int j = 0; j < V; j++) w[j] = to_f32<__half>(r.v[j]);
    } else {
        RVecA<__nv_bfloat16, V> r;
        r.load(static_cast<const __nv_bfloat16*>(p.weight) + at);
#pragma unroll
        for (int j = 0; j < V; j++) w[j] = to_f32<__nv_bfloat16>(r.v[j]);
    }
}

// Sum of a pair over the threads of a row: a warp, or the whole block.  Every thread gets it.
template <bool WARP>
__device__ __forceinline__ float2 row_sum(float2 v, float2* sm) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
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
__global__ void __launch_bounds__(WARP ? 128 : 512) rms_fwd_kernel(const RmsArgs p) {
    __shared__ float2 sm[32];
    extern __shared__ unsigned amax[];      // QUANT: largest magnitude of every block of the row (as bits: NaN above all)
    grid_dep_wait();
    grid_dep_launch();
    const int tpr = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
    const long long row = WARP ? static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= p.rows) return;              // (a whole warp, or never)
    const T* x = static_cast<const T*>(p.x) + row * p.D;
    const S* res = p.residual ? static_cast<const S*>(p.residual) + row * p.D : nullptr;
    float v[K][V];
    RVecA<T, V> xv[K];
    RVecA<S, V> rv[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int e = (k * tpr + tid) * V;
        if (e < p.D) {
            xv[k].load(x + e);
            if (res) rv[k].load(res + e);
        }
    }
    float2 acc = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int e = (k * tpr + tid) * V;
        if (e < p.D) {
            if (res) {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    rv[k].v[j] = from_f32<S>(to_f32<T>(xv[k].v[j]) + to_f32<S>(rv[k].v[j]));
                    v[k][j] = to_f32<S>(rv[k].v[j]);
                }
                rv[k].store(static_cast<S*>(p.sum) + row * p.D + e);
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) v[k][j] = to_f32<T>(xv[k].v[j]);
            }
#pragma unroll
            for (int j = 0; j < V; j++) acc.x = fmaf(v[k][j], v[k][j], acc.x);
        }
    }
    acc = row_sum<WARP>(acc, sm);
    const float r = rsqrtf(acc.x * p.inv_d + p.eps);
    const long long wrow = p.groups > 1 ? (row / p.inner) % p.groups * p.D : 0;
    unsigned* top = amax + (WARP ? (threadIdx.x >> 5) : 0) * (p.D / p.block);
    if (QUANT) {
        for (int i = tid; i < p.D / p.block; i += tpr) top[i] = 0u;
        if (WARP) __syncwarp();
        else __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int e = (k * tpr + tid) * V;
        float w[V];
        if (e < p.D) {
            load_weight<V>(p, wrow + e, w);
#pragma unroll
            for (int j = 0; j < V; j++) v[k][j] = v[k][j] * r * w[j];
        }
        if (!QUANT) {
            if (e < p.D) store_any<V>(p.y, p.ydt, row * p.D + e, v[k]);
        } else {
            unsigned m = 0u;
            if (e < p.D) {
#pragma unroll
                for (int j = 0; j < V; j++) m = max(m, __float_as_uint(v[k][j]) & 0x7fffffffu);
            }
            // neighbouring threads of one block of values first (all of a warp's are in one block or every few are)
            const int same = min(32, p.block / V > 0 ? p.block / V : 1);
            if (same == 32 || (same & (same - 1)) == 0)
                for (int o = same >> 1; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (e < p.D) atomicMax(&top[e / p.block], m);       // (the largest: no order to depend on)
        }
    }
    if (QUANT) {
        if (WARP) __syncwarp();
        else __syncthreads();
        const int blocks = p.D / p.block;
        for (int i = tid; i < blocks; i += tpr) {
            const float s = top[i] == 0u ? 1.0f : __fdiv_rn(__uint_as_float(top[i]), 448.0f);
            p.scale[row * blocks + i] = s;
        }
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int e = (k * tpr + tid) * V;
            if (e < p.D) {
                const unsigned t = top[e / p.block];
                const float inv = t == 0u ? 1.0f : __fdiv_rn(448.0f, __uint_as_float(t));
                uint8_t* q = static_cast<uint8_t*>(p.q) + row * p.D + e;
                if constexpr (V == 8) {
                    __nv_fp8x2_storage_t o[4];
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        o[j] = __nv_cvt_float2_to_fp8x2(make_float2(v[k][2 * j] * inv, v[k][2 * j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
                    *reinterpret_cast<uint2*>(q) = make_uint2(o[0] | (static_cast<unsigned>(o[1]) << 16), o[2] | (static_cast<unsigned>(o[3]) << 16));
                } else {
                    *q = __nv_cvt_float_to_fp8(v[k][0] * inv, __NV_SATFINITE, __NV_E4M3);
                }
            }
        }
    }
}

// S: the stream's type, T: dy's.  Blocks (or warps) walk over the rows of one group and keep their part of the weight's gradient.
template <typename T, typename S, int V, int K, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 512) rms_bwd_kernel(const RmsArgs p) {
    __shared__ float2 sm[32];
    extern __shared__ unsigned dyn[];
    grid_dep_wait();
    grid_dep_launch();
    const int tpr = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int rpb = WARP ? blockDim.x >> 5 : 1, slot = WARP ? threadIdx.x >> 5 : 0, g = blockIdx.y;
    const long long rows_g = p.rows / p.groups;
    float dw[K][V], w[K][V];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int e = (k * tpr + tid) * V;
#pragma unroll
        for (int j = 0; j < V; j++) dw[k][j] = 0.f;
        if (e < p.D) load_weight<V>(p, static_cast<long long>(g) * p.D + e, w[k]);
    }
    for (long long i = static_cast<long long>(blockIdx.x) * rpb + slot; i < rows_g; i += static_cast<long long>(gridDim.x) * rpb) {
        const long long row = p.groups > 1 ? ((i / p.inner) * p.groups + g) * p.inner + i % p.inner : i;
        const S* s = static_cast<const S*>(p.x) + row * p.D;
        const T* dy = static_cast<const T*>(p.dy) + row * p.D;
        const S* ds = p.ds ? static_cast<const S*>(p.ds) + row * p.D : nullptr;
        RVecA<S, V> sv[K], dsv[K];
        RVecA<T, V> dv[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int e = (k * tpr + tid) * V;
            if (e < p.D) {
                sv[k].load(s + e);
                dv[k].load(dy + e);
                if (ds) dsv[k].load(ds + e);
            }
        }
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < K; k++) {
            if ((k * tpr + tid) * V < p.D) {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float a = to_f32<S>(sv[k].v[j]);
                    acc.x = fmaf(a, a, acc.x);
                    acc.y = fmaf(a * w[k][j], to_f32<T>(dv[k].v[j]), acc.y);
                }
            }
        }
        acc = row_sum<WARP>(acc, sm);
        const float r = rsqrtf(acc.x * p.inv_d + p.eps), m = acc.y * p.inv_d * r * r;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int e = (k * tpr + tid) * V;
            if (e < p.D) {
                float out[V];
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float a = to_f32<S>(sv[k].v[j]), d = to_f32<T>(dv[k].v[j]);
                    out[j] = r * (d * w[k][j] - a * m);
                    if (ds) out[j] += to_f32<S>(dsv[k].v[j]);
                    dw[k][j] = fmaf(d * r, a, dw[k][j]);
                }
                store_any<V>(p.dx, p.xdt, row * p.D + e, out);
                if (p.dres) {
                    RVecA<S, V> o;
#pragma unroll
                    for (int j = 0; j < V; j++) o.v[j] = from_f32<S>(out[j]);
                    o.store(static_cast<S*>(p.dres) + row * p.D + e);
                }
            }
        }
    }
    if (!p.part) return;
    float* part = p.part + (static_cast<long long>(blockIdx.x) * p.groups + g) * p.D;
    float* sum = reinterpret_cast<float*>(dyn);
    for (int turn = 0; turn < rpb; turn++) {        // a block's warps, one after the other
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

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

constexpr int RMS_MAX_D = 16384;
// How a row is laid over threads: V values each, K times, by a warp (WARP) or a block of `threads`.
struct RmsPlan {
    int V, K, threads;
    bool warp;
};
RmsPlan rms_plan(int D, bool wide) {
    if (!wide) {
        if (D <= 512) return {1, 16, 128, true};
        int t = 64;
        while (t * 16 < D && t < 512) t *= 2;
        return {1, t * 16 < D ? 32 : 16, t, false};
    }
    if (D <= 256) return {8, 1, 128, true};
    if (D <= 512) return {8, 2, 128, true};
    if (D <= 1024) return {8, 4, 128, true};
    int t = 64;
    while (t * 16 < D && t < 512) t *= 2;
    return {8, t * 16 < D ? 4 : 2, t, false};
}
int rms_bwd_blocks(long long rows_g, int groups, const RmsPlan& pl) {
    const int rpb = pl.warp ? 4 : 1, per_sm = pl.warp ? 8 : pl.threads <= 256 ? 6 : 3;
    long long want = 148LL * per_sm / groups;
    if (want < 1) want = 1;
    const long long most = (rows_g + rpb - 1) / rpb;
    return static_cast<int>(want < most ? want : most);
}

template <typename T, typename S, bool QUANT>
cudaError_t launch_rms_fwd(const RmsArgs& a, bool wide, cudaStream_t st) {
    const RmsPlan pl = rms_plan(a.D, wide);
    const int rpb = pl.warp ? 4 : 1;
    const dim3 grid(static_cast<unsigned>((a.rows + rpb - 1) / rpb)), block(pl.threads);
    const size_t smem = QUANT ? static_cast<size_t>(rpb) * (a.D / a.block) * 4 : 0;
    if (pl.V == 1) {
        if (pl.warp) return launch_plain(rms_fwd_kernel<T, S, 1, 16, true, QUANT>, grid, block, smem, st, a);
        if (pl.K == 16) return launch_plain(rms_fwd_kernel<T, S, 1, 16, false, QUANT>, grid, block, smem, st, a);
        return launch_plain(rms_fwd_kernel<T, S, 1, 32, false, QUANT>, grid, block, smem, st, a);
    }
    if (!pl.warp && pl.K == 4) return launch_plain(rms_fwd_kernel<T, S, 8, 4, false, QUANT>, grid, block, smem, st, a);
    if (!pl.warp) return launch_plain(rms_fwd_kernel<T, S, 8, 2, false, QUANT>, grid, block, smem, st, a);
    if (pl.K == 1) return launch_plain(rms_fwd_kernel<T, S, 8, 1, true, QUANT>, grid, block, smem, st, a);
    if (pl.K == 2) return launch_plain(rms_fwd_kernel<T, S, 8, 2, true, QUANT>, grid, block, smem, st, a);
    return launch_plain(rms_fwd_kernel<T, S, 8, 4, true, QUANT>, grid, block, smem, st, a);
}
template <typename T, typename S>
cudaError_t launch_rms_bwd(const RmsArgs& a, bool wide, cudaStream_t st) {
    const RmsPlan pl = rms_plan(a.D, wide);
    const dim3 grid(rms_bwd_blocks(a.rows / a.groups, a.groups, pl), a.groups), block(pl.threads);
    const size_t smem = pl.warp && a.part ? static_cast<size_t>(a.D) * 4 : 0;
    cudaError_t ce;
    if (pl.V == 1)
        ce = pl.warp ? launch_plain(rms_bwd_kernel<T, S, 1, 16, true>, grid, block, smem, st, a)
             : pl.K == 16 ? launch_plain(rms_bwd_kernel<T, S, 1, 16, false>, grid, block, smem, st, a)
                          : launch_plain(rms_bwd_kernel<T, S, 1, 32, false>, grid, block, smem, st, a);
    else if (!pl.warp && pl.K == 4) ce = launch_plain(rms_bwd_kernel<T, S, 8, 4, false>, grid, block, smem, st, a);
    else if (!pl.warp) ce = launch_plain(rms_bwd_kernel<T, S, 8, 2, false>, grid, block, smem, st, a);
    else if (pl.K == 1) ce = launch_plain(rms_bwd_kernel<T, S, 8, 1, true>, grid, block, smem, st, a);
    else if (pl.K == 2) ce = launch_plain(rms_bwd_kernel<T, S, 8, 2, true>, grid, block, smem, st, a);
    else ce = launch_plain(rms_bwd_kernel<T, S, 8, 4, true>, grid, block, smem, st, a);
    return ce;
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
    const int a = rms_bwd_blocks(rows_g, groups, rms_plan(D, true)), b = rms_bwd_blocks(rows_g, groups, rms_plan(D, false));
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
        const int blocks = rms_bwd_blocks(rows / groups, groups, rms_plan(D, wide));
        ce = launch_reduce_rows(a.part, blocks, static_cast<long long>(groups) * D, RmsWeightOut{{dweight, w_dtype}}, st);
    }
    if (ce != cudaSuccess) cudaGetLastError();
    return ce == cudaSuccess ? MLSTM_OK : note_cuda_error(ce, "launch of rms_bwd_kernel");
}

}  // extern "C"
