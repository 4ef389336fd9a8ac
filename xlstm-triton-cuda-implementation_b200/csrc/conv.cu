// Short causal convolution along the positions, channel by channel, in front of a recurrent mixer:
//     pre_t = bias + sum_k w[k] x_{t - (W - 1) + k},   y_t = pre_t * sigmoid(pre_t)  or  pre_t         (W = 2, 3, 4)
// and its gradients, with d_t = dy_t * y'(pre_t):
//     dx_t = sum_k w[k] d_{t + (W - 1) - k},   dw[k] = sum_t d_t x_{t - (W - 1) + k},   dbias = sum_t d_t.
// In front of position 0 stand the W - 1 inputs carried in, or zeros.  Sums are fp32.
//
// Bound by HBM: x in and y out (forward), x and dy in and dx out (backward).  A thread walks down the positions of its channels
// with the last W inputs in registers, so an input is read once (and W - 1 more at the start of each run of positions, mostly
// from L2); neighbouring threads own neighbouring channels, 16 bytes each, so that rows are read in whole lines.
#include "reduce_rows.cuh"

namespace mlstm {
namespace {

template <typename T, int V>
struct alignas(sizeof(T) * V) CVec {
    T v[V];
};

struct ConvArgs {
    const void *x, *weight, *bias, *initial, *dy;
    void *y, *state_out, *dx;
    float* part;                   // backward: [Bt * blocks along the positions, W + 1, C] partial sums
    long long sxb, sxt;            // strides of x in elements (everything else is contiguous)
    int Bt, S, C, wdt, silu, rows; // rows: positions per thread
};

template <typename T, int V, int W>
__device__ __forceinline__ void load_weights(const ConvArgs& p, int c, float (&w)[W][V], float (&bias)[V]) {
#pragma unroll
    for (int j = 0; j < V; j++) {
#pragma unroll
        for (int k = 0; k < W; k++) w[k][j] = load_any(p.weight, p.wdt, static_cast<long long>(c + j) * W + k);
        bias[j] = p.bias ? load_any(p.bias, p.wdt, c + j) : 0.f;
    }
}
// row t of the inputs, t >= -(W - 1)
template <typename T, int V, int W>
__device__ __forceinline__ CVec<T, V> input_row(const ConvArgs& p, const T* x, int b, int t, int c) {
    CVec<T, V> r;
    if (t >= 0) return *reinterpret_cast<const CVec<T, V>*>(x + t * p.sxt);
    if (p.initial)
        return *reinterpret_cast<const CVec<T, V>*>(static_cast<const T*>(p.initial) +
                                                    (static_cast<size_t>(b) * (W - 1) + (W - 1) + t) * p.C + c);
#pragma unroll
    for (int j = 0; j < V; j++) r.v[j] = from_f32<T>(0.f);
    return r;
}

constexpr int CONV_U = 4;          // rows whose loads are in flight at a time

template <typename T, int V, int W>
__global__ void __launch_bounds__(256) conv_fwd_kernel(const ConvArgs p) {
    grid_dep_wait();
    grid_dep_launch();
    const int c = (blockIdx.x * blockDim.x + threadIdx.x) * V, b = blockIdx.z;
    const int t0 = (blockIdx.y * blockDim.y + threadIdx.y) * p.rows, t1 = min(p.S, t0 + p.rows);
    if (c >= p.C || t0 >= p.S) return;
    float w[W][V], bias[V];
    const T* x = static_cast<const T*>(p.x) + b * p.sxb + c;
    T* y = static_cast<T*>(p.y) + static_cast<size_t>(b) * p.S * p.C + c;
    CVec<T, V> win[W - 1 + CONV_U];
#pragma unroll
    for (int k = 0; k < W - 1; k++) win[k] = input_row<T, V, W>(p, x, b, t0 - (W - 1) + k, c);
    load_weights<T, V, W>(p, c, w, bias);
    for (int t = t0; t < t1; t += CONV_U) {
#pragma unroll
        for (int u = 0; u < CONV_U; u++)
            if (t + u < t1) win[W - 1 + u] = *reinterpret_cast<const CVec<T, V>*>(x + (t + u) * p.sxt);
#pragma unroll
        for (int u = 0; u < CONV_U; u++) {
            if (t + u < t1) {
                CVec<T, V> out;
#pragma unroll
                for (int j = 0; j < V; j++) {
                    float a = bias[j];
#pragma unroll
                    for (int k = 0; k < W; k++) a = fmaf(w[k][j], to_f32<T>(win[u + k].v[j]), a);
                    out.v[j] = from_f32<T>(p.silu ? silu_f(a) : a);
                }
                *reinterpret_cast<CVec<T, V>*>(y + static_cast<size_t>(t + u) * p.C) = out;
            }
        }
#pragma unroll
        for (int k = 0; k < W - 1; k++) win[k] = win[CONV_U + k];
    }
    // The last W - 1 inputs.  Row j of the new state is row j + S of the old one where x is shorter than that: read after
    // nothing but rows in front of it has been written, so that the two may be the same memory.
    if (p.state_out && t0 == 0) {
#pragma unroll
        for (int j = 0; j < W - 1; j++)
            *reinterpret_cast<CVec<T, V>*>(static_cast<T*>(p.state_out) + (static_cast<size_t>(b) * (W - 1) + j) * p.C + c) =
                input_row<T, V, W>(p, x, b, p.S - (W - 1) + j, c);
    }
}

// Backward: a thread's run of positions, and W - 1 more behind it whose d its own dx needs.
template <typename T, int V, int W>
__global__ void __launch_bounds__(256) conv_bwd_kernel(const ConvArgs p) {
    __shared__ float red[256][V];
    grid_dep_wait();
    grid_dep_launch();
    const int c = (blockIdx.x * blockDim.x + threadIdx.x) * V, b = blockIdx.z;
    const int t0 = (blockIdx.y * blockDim.y + threadIdx.y) * p.rows, t1 = min(p.S, t0 + p.rows);
    const bool on = c < p.C && t0 < p.S;
    float dw[W + 1][V];            // dw[W]: the bias
#pragma unroll
    for (int k = 0; k <= W; k++)
#pragma unroll
        for (int j = 0; j < V; j++) dw[k][j] = 0.f;
    if (on) {
        float w[W][V], bias[V], d[W][V];
        const T* x = static_cast<const T*>(p.x) + b * p.sxb + c;
        const size_t base = static_cast<size_t>(b) * p.S * p.C + c;
        const T* dy = static_cast<const T*>(p.dy) + base;
        T* dx = static_cast<T*>(p.dx) + base;
        CVec<T, V> win[W - 1 + CONV_U], g[CONV_U];
#pragma unroll
        for (int k = 0; k < W - 1; k++) win[k] = input_row<T, V, W>(p, x, b, t0 - (W - 1) + k, c);
#pragma unroll
        for (int k = 0; k < W; k++)
#pragma unroll
            for (int j = 0; j < V; j++) d[k][j] = 0.f;
        load_weights<T, V, W>(p, c, w, bias);
        for (int t = t0; t < t1 + W - 1; t += CONV_U) {
#pragma unroll
            for (int u = 0; u < CONV_U; u++) {
                if (t + u < p.S) {
                    win[W - 1 + u] = *reinterpret_cast<const CVec<T, V>*>(x + (t + u) * p.sxt);
                    g[u] = *reinterpret_cast<const CVec<T, V>*>(dy + static_cast<size_t>(t + u) * p.C);
                }
            }
#pragma unroll
            for (int u = 0; u < CONV_U; u++) {
                const int tt = t + u;
#pragma unroll
                for (int j = 0; j < V; j++) {
#pragma unroll
                    for (int k = 0; k < W - 1; k++) d[k][j] = d[k + 1][j];
                    float v = 0.f;
                    if (tt < p.S) {
                        v = to_f32<T>(g[u].v[j]);
                        if (p.silu) {
                            float a = bias[j];
#pragma unroll
                            for (int k = 0; k < W; k++) a = fmaf(w[k][j], to_f32<T>(win[u + k].v[j]), a);
                            const float sg = __fdividef(1.0f, 1.0f + __expf(-a));
                            v *= sg * fmaf(a, 1.0f - sg, 1.0f);
                        }
                        if (tt < t1) {
#pragma unroll
                            for (int k = 0; k < W; k++) dw[k][j] = fmaf(v, to_f32<T>(win[u + k].v[j]), dw[k][j]);
                            dw[W][j] += v;
                        }
                    }
                    d[W - 1][j] = v;
                }
                const int s = tt - (W - 1);
                if (s >= t0 && s < t1) {
                    CVec<T, V> out;
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        float a = 0.f;
#pragma unroll
                        for (int k = 0; k < W; k++) a = fmaf(w[k][j], d[W - 1 - k][j], a);
                        out.v[j] = from_f32<T>(a);
                    }
                    *reinterpret_cast<CVec<T, V>*>(dx + static_cast<size_t>(s) * p.C) = out;
                }
            }
#pragma unroll
            for (int k = 0; k < W - 1; k++) win[k] = win[CONV_U + k];
        }
    }
    // the block's runs of the same channels, one after the other
    const int tid = threadIdx.y * blockDim.x + threadIdx.x;
    const size_t row = static_cast<size_t>(b) * gridDim.y + blockIdx.y;
#pragma unroll
    for (int k = 0; k <= W; k++) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; j++) red[tid][j] = dw[k][j];
        __syncthreads();
        if (threadIdx.y == 0 && c < p.C) {
            for (int r = 1; r < static_cast<int>(blockDim.y); r++)
#pragma unroll
                for (int j = 0; j < V; j++) dw[k][j] += red[r * blockDim.x + threadIdx.x][j];
#pragma unroll
            for (int j = 0; j < V; j++) p.part[(row * (W + 1) + k) * p.C + c + j] = dw[k][j];
        }
    }
}

struct ConvParamOut {
    AnyOut dw, db;
    int W, C;
    __device__ __forceinline__ void operator()(long long at, float v) const {
        const int k = static_cast<int>(at / C), c = static_cast<int>(at - static_cast<long long>(k) * C);
        if (k < W) dw.put(static_cast<long long>(c) * W + k, v);
        else if (db.p) db.put(c, v);
    }
};

inline long long ceil_up(long long a, long long b) { return (a + b - 1) / b; }
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// channels per thread: 16 bytes of them where everything is aligned for that (the backward 8 bytes: its registers), else one
int conv_vec(const ConvArgs& a, int es, bool bwd) {
    const int bytes = bwd && es == 2 ? 8 : 16, v = bytes / es;
    if (a.C % v || a.sxb % v || a.sxt % v) return 1;
    for (const void* q : {a.x, a.initial, a.dy, static_cast<const void*>(a.y), static_cast<const void*>(a.state_out),
                          static_cast<const void*>(a.dx)})
        if (!aligned(q, bytes)) return 1;
    return v;
}

struct ConvGrid {
    dim3 grid, block;
    int rows;
};
constexpr int CONV_BWD_Y = 8;
ConvGrid conv_grid(const ConvArgs& a, int V, bool bwd) {
    const int threads = bwd ? 256 : 128;
    const long long cv = ceil_up(a.C, V);
    ConvGrid g;
    const int y = bwd ? CONV_BWD_Y : a.S <= 8 ? 1 : 4;
    g.block = dim3(threads / y, y, 1);
    const long long bx = ceil_up(cv, g.block.x);
    // the longest runs (the fewest inputs read twice) that still give every SM a few blocks
    g.rows = bwd ? 32 : 64;
    while (g.rows > 8 && bx * a.Bt * ceil_up(a.S, g.rows * y) < 148 * 8) g.rows /= 2;
    g.grid = dim3(static_cast<unsigned>(bx), static_cast<unsigned>(ceil_up(a.S, g.rows * y)), a.Bt);
    return g;
}

template <typename T, int V, int W>
cudaError_t launch_conv_w(ConvArgs& a, bool bwd, cudaStream_t st) {
    const ConvGrid g = conv_grid(a, V, bwd);
    a.rows = g.rows;
    return bwd ? launch_plain(conv_bwd_kernel<T, V, W>, g.grid, g.block, 0, st, a) : launch_plain(conv_fwd_kernel<T, V, W>, g.grid, g.block, 0, st, a);
}
template <typename T, int VMAX>
cudaError_t launch_conv_t(ConvArgs& a, int W, int V, bool bwd, cudaStream_t st) {
    if (V == 1) return W == 2 ? launch_conv_w<T, 1, 2>(a, bwd, st) : W == 3 ? launch_conv_w<T, 1, 3>(a, bwd, st) : launch_conv_w<T, 1, 4>(a, bwd, st);
    return W == 2 ? launch_conv_w<T, VMAX, 2>(a, bwd, st) : W == 3 ? launch_conv_w<T, VMAX, 3>(a, bwd, st) : launch_conv_w<T, VMAX, 4>(a, bwd, st);
}

int conv_check(const void* x, const void* weight, int B, int S, int C, int W, int dtype, int w_dtype, const long long* strides) {
    if (!x || !weight || B <= 0 || S <= 0 || C <= 0) return MLSTM_E_ARG;
    for (int d : {dtype, w_dtype})
        if (d != MLSTM_DT_F32 && d != MLSTM_DT_F16 && d != MLSTM_DT_BF16) return MLSTM_E_ARG;
    if (w_dtype != dtype && w_dtype != MLSTM_DT_F32) return MLSTM_E_ARG;
    if (strides && (strides[0] < 0 || strides[1] < 0)) return MLSTM_E_ARG;
    if (W < 2 || W > 4 || B > 65535 || S > (1 << 23) || C > (1 << 24)) return MLSTM_E_SHAPE;
    return MLSTM_OK;
}

// partial rows of the parameters' gradients, for whichever access width the pointers allow
size_t conv_part_rows(int B, int S, int C) {
    ConvArgs a{};
    a.Bt = B; a.S = S; a.C = C;
    const size_t wide = conv_grid(a, 4, true).grid.y, one = conv_grid(a, 1, true).grid.y;
    return static_cast<size_t>(B) * (wide > one ? wide : one);
}

}  // namespace
}  // namespace mlstm

using namespace mlstm;

extern "C" {

int mlstm_conv_fwd(const void* x, const void* weight, const void* bias, const void* initial, const long long* strides, void* y,
                   void* state_out, int B, int S, int C, int W, int dtype, int w_dtype, int silu, void* stream) {
    const int rc = conv_check(x, weight, B, S, C, W, dtype, w_dtype, strides);
    if (rc != MLSTM_OK) return rc;
    if (!y) return MLSTM_E_ARG;
    const int es = dtype == MLSTM_DT_F32 ? 4 : 2, ws = w_dtype == MLSTM_DT_F32 ? 4 : 2;
    for (const void* q : {x, initial, static_cast<const void*>(y), static_cast<const void*>(state_out)})
        if (!aligned(q, es)) return MLSTM_E_ALIGN;
    if (!aligned(weight, ws) || !aligned(bias, ws)) return MLSTM_E_ALIGN;
    ConvArgs a{};
    a.x = x; a.weight = weight; a.bias = bias; a.initial = initial; a.y = y; a.state_out = state_out;
    a.sxb = strides ? strides[0] : static_cast<long long>(S) * C;
    a.sxt = strides ? strides[1] : C;
    a.Bt = B; a.S = S; a.C = C; a.wdt = w_dtype; a.silu = silu;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int V = conv_vec(a, es, false);
    const cudaError_t ce = dtype == MLSTM_DT_F32 ? launch_conv_t<float, 4>(a, W, V, false, st)
                           : dtype == MLSTM_DT_F16 ? launch_conv_t<__half, 8>(a, W, V, false, st)
                                                   : launch_conv_t<__nv_bfloat16, 8>(a, W, V, false, st);
    if (ce != cudaSuccess) cudaGetLastError();
    return ce == cudaSuccess ? MLSTM_OK : note_cuda_error(ce, "launch of conv_fwd_kernel");
}

size_t mlstm_conv_bwd_workspace(int B, int S, int C, int W, int dtype) {
    const void* any = reinterpret_cast<const void*>(16);
    if (conv_check(any, any, B, S, C, W, dtype, dtype, nullptr) != MLSTM_OK) return 0;
    return conv_part_rows(B, S, C) * (W + 1) * C * sizeof(float);
}

int mlstm_conv_bwd(const void* dy, const void* x, const void* weight, const void* bias, const long long* strides, void* dx,
                   void* dweight, void* dbias, void* workspace, size_t workspace_bytes, int B, int S, int C, int W, int dtype,
                   int w_dtype, int silu, void* stream) {
    const int rc = conv_check(x, weight, B, S, C, W, dtype, w_dtype, strides);
    if (rc != MLSTM_OK) return rc;
    if (!dy || !dx || !dweight || (bias == nullptr) != (dbias == nullptr)) return MLSTM_E_ARG;
    const int es = dtype == MLSTM_DT_F32 ? 4 : 2, ws = w_dtype == MLSTM_DT_F32 ? 4 : 2;
    for (const void* q : {x, dy, static_cast<const void*>(dx)})
        if (!aligned(q, es)) return MLSTM_E_ALIGN;
    for (const void* q : {weight, bias, static_cast<const void*>(dweight), static_cast<const void*>(dbias)})
        if (!aligned(q, ws)) return MLSTM_E_ALIGN;
    if (!workspace || workspace_bytes < mlstm_conv_bwd_workspace(B, S, C, W, dtype) || !aligned(workspace, 16)) return MLSTM_E_WORKSPACE;
    ConvArgs a{};
    a.x = x; a.weight = weight; a.bias = bias; a.dy = dy; a.dx = dx; a.part = static_cast<float*>(workspace);
    a.sxb = strides ? strides[0] : static_cast<long long>(S) * C;
    a.sxt = strides ? strides[1] : C;
    a.Bt = B; a.S = S; a.C = C; a.wdt = w_dtype; a.silu = silu;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int V = conv_vec(a, es, true);
    cudaError_t ce = dtype == MLSTM_DT_F32 ? launch_conv_t<float, 4>(a, W, V, true, st)
                     : dtype == MLSTM_DT_F16 ? launch_conv_t<__half, 4>(a, W, V, true, st)
                                             : launch_conv_t<__nv_bfloat16, 4>(a, W, V, true, st);
    if (ce == cudaSuccess) {
        const int rows = B * static_cast<int>(conv_grid(a, V, true).grid.y);
        ce = launch_reduce_rows(a.part, rows, static_cast<long long>(W + 1) * C,
                                ConvParamOut{{dweight, w_dtype}, {dbias, w_dtype}, W, C}, st);
    }
    if (ce != cudaSuccess) cudaGetLastError();
    return ce == cudaSuccess ? MLSTM_OK : note_cuda_error(ce, "launch of conv_bwd_kernel");
}

}  // extern "C"
