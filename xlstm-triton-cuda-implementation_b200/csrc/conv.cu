// Short causal convolution along the positions, channel by channel, in front of a recurrent mixer:
//     pre_t = bias + sum_k w[k] x_{t - (W - 1) + k},   y_t = pre_t * sigmoid(pre_t)  or  pre_t         (W = 2, 3, 4)
// and its gradients, with d_t = dy_t * y'(pre_t):
//     dx_t = sum_k w[k] d_{t + (W - 1) - k},   dw[k] = sum_t d_t x_{t - (W - 1) + k},   dbias = sum_t d_t.
// In front of position 0 stand the W - 1 inputs carried in, or zeros.  Sums are fp32.
//
// Bound by HBM: x in and y out (forward), x and dy in and dx out (backward).  Neighbouring threads own neighbouring channels, 8 bytes
// each, and walk down the positions, so an input is read once (and W - 1 more at the start of each run, mostly from L2).
// Measured, 4 x 4096 x 4096 bf16, W = 4, silu: forward 52 us (5.2 TB/s; the two hardware functions of silu 62 %, issue slots 69 % busy),
// backward 99 us with the sums of the parameters (151 in all; 4.1 TB/s; 26 instructions per value, 54 % of the issue slots: three warps
// per scheduler at 168 registers do not cover their latencies; four at 128 registers, where the form without silu spills: 3 us more).
// One channel per thread, where widths, strides or addresses allow no more (4 x 4096 x 4095): forward 87, backward 205 us.
#include "async_copy.cuh"
#include "pair_math.cuh"
#include "reduce_rows.cuh"
#include "vec_cvt.cuh"

namespace mlstm {
namespace {

struct ConvArgs {
    const void *x, *weight, *bias, *initial, *dy;
    void *y, *state_out, *dx;
    float* part;                   // backward: [Bt * blocks along the positions, W + 1, C] partial sums
    long long sxb, sxt;            // strides of x in elements (everything else is contiguous)
    int Bt, S, C, wdt, wvec, silu, rows; // rows: positions per thread
};

template <bool BWD>
constexpr int CONV_THREADS = BWD ? 128 : 256;

// N neighbouring values in the widest pieces that N of them allow (p.wvec: the tensor starts on 16 bytes), as floats
template <typename T, int N>
__device__ __forceinline__ void load_row(const T* p, float (&o)[N]) {
    constexpr int bytes = N * sizeof(T), unit = bytes % 16 == 0 ? 16 : bytes % 8 == 0 ? 8 : bytes % 4 == 0 ? 4 : 2;
    using Unit = std::conditional_t<unit == 16, uint4, std::conditional_t<unit == 8, uint2, std::conditional_t<unit == 4, unsigned, unsigned short>>>;
    union {
        Unit u[bytes / unit];
        unsigned short h[bytes / 2];
        float f[bytes / 4 > 0 ? bytes / 4 : 1];
    } raw;
#pragma unroll
    for (int i = 0; i < bytes / unit; i++) raw.u[i] = reinterpret_cast<const Unit*>(p)[i];
#pragma unroll
    for (int i = 0; i < N; i++) {
        if constexpr (sizeof(T) == 4) o[i] = raw.f[i];
        else o[i] = to_f32<T>(*reinterpret_cast<const T*>(&raw.h[i]));
    }
}
template <int N>
__device__ __forceinline__ void load_row_any(const void* p, int dtype, bool vec, long long at, float (&o)[N]) {
    if (!vec) {
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = load_any(p, dtype, at + i);
    } else if (dtype == MLSTM_DT_F32) load_row<float, N>(static_cast<const float*>(p) + at, o);
    else if (dtype == MLSTM_DT_F16) load_row<__half, N>(static_cast<const __half*>(p) + at, o);
    else load_row<__nv_bfloat16, N>(static_cast<const __nv_bfloat16*>(p) + at, o);
}
template <int V, int W>
__device__ __forceinline__ void load_weights(const ConvArgs& p, int c, float (&w)[W][V], float (&bias)[V]) {
    float v[V * W];
    load_row_any<V * W>(p.weight, p.wdt, p.wvec && V > 1, static_cast<long long>(c) * W, v);
    if (p.bias) load_row_any<V>(p.bias, p.wdt, p.wvec && V > 1, c, bias);
#pragma unroll
    for (int j = 0; j < V; j++) {
        if (!p.bias) bias[j] = 0.f;
#pragma unroll
        for (int k = 0; k < W; k++) w[k][j] = v[j * W + k];
    }
}
// row t of the inputs, t >= -(W - 1)
template <typename T, int V, int W>
__device__ __forceinline__ Vec<T, V> input_row(const ConvArgs& p, const T* x, int b, int t, int c) {
    Vec<T, V> r;
    if (t >= 0) return *reinterpret_cast<const Vec<T, V>*>(x + t * p.sxt);
    if (p.initial)
        return *reinterpret_cast<const Vec<T, V>*>(static_cast<const T*>(p.initial) +
                                                    (static_cast<size_t>(b) * (W - 1) + (W - 1) + t) * p.C + c);
#pragma unroll
    for (int j = 0; j < V; j++) r.v[j] = from_f32<T>(0.f);
    return r;
}

// A thread's own rows on their way from memory: groups of U rows, DEPTH groups ahead of the one that is worked on.  They are copied
// to shared memory asynchronously (each thread reads back what it asked for itself, so there is no barrier), which keeps far
// more bytes in flight than there are registers for; single 16-bit values, which cannot be copied so, are loaded plainly.
template <typename T, int V, int U, int DEPTH, int THREADS>
struct RowPipe {
    static constexpr bool ASYNC = V * sizeof(T) >= 4;
    static constexpr int SLOTS = ASYNC ? DEPTH : 1;
    static constexpr int AHEAD = ASYNC ? DEPTH - 1 : 1;      // (into the group that was used up one turn ago)
    using Row = Vec<T, V>;
    using Ring = Row[SLOTS * U][THREADS];
    Ring& ring;
    const T *first, *next;      // the run's first row; the first row of the group to be fetched next
    long long stride;
    int slot_in = 0, slot_out = 0, tid;
    Row raw[ASYNC ? 1 : U];
    __device__ __forceinline__ RowPipe(Ring& r, const T* row0, long long st, int t) : ring(r), first(row0), next(row0), stride(st), tid(t) {}
    // row t + u of the run exists where t + u < n; else zeros
    __device__ __forceinline__ void fetch(int t, int n) {
        if constexpr (ASYNC) {
            const unsigned dst = shared_address(&ring[slot_in * U][tid]);
            constexpr unsigned pitch = THREADS * sizeof(Row);
            if (t + U <= n) {
#pragma unroll
                for (int u = 0; u < U; u++) copy_async<sizeof(Row)>(dst + u * pitch, next + u * stride);
            } else {
#pragma unroll
                for (int u = 0; u < U; u++) copy_async_or_zeros<sizeof(Row)>(dst + u * pitch, t + u < n ? next + u * stride : first, t + u < n);
            }
            slot_in = slot_in + 1 == SLOTS ? 0 : slot_in + 1;
        } else {
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (t + u < n) raw[u] = *reinterpret_cast<const Row*>(next + u * stride);
                else {
#pragma unroll
                    for (int j = 0; j < V; j++) raw[u].v[j] = from_f32<T>(0.f);
                }
            }
        }
        next += U * stride;
    }
    __device__ __forceinline__ void take(float (*out)[V]) {
#pragma unroll
        for (int u = 0; u < U; u++) to_floats<T, V>(ASYNC ? ring[slot_out * U + u][tid] : raw[ASYNC ? 0 : u], out[u]);
        if constexpr (ASYNC) slot_out = slot_out + 1 == SLOTS ? 0 : slot_out + 1;
    }
};
// (backward, with the forward's 52 us: groups of 3 rows 156, of 4 151, of 5 149, of 6 154, of 8 157 us; all before the values behind the
// last position were set to 0, which takes 1.5 us)
constexpr int CONV_U = 4, CONV_DEPTH = 4, CONV_BWD_U = 5, CONV_BWD_DEPTH = 3;

// A thread walks down its run of positions with the last W inputs in registers.
template <typename T, int V, int W, bool SILU>
__global__ void __launch_bounds__(CONV_THREADS<false>, 3) conv_fwd_kernel(const ConvArgs p) {
    grid_dep_wait();
    grid_dep_launch();
    const int c = (blockIdx.x * blockDim.x + threadIdx.x) * V, b = blockIdx.z;
    const int t0 = (blockIdx.y * blockDim.y + threadIdx.y) * p.rows, n = min(p.S - t0, p.rows);
    if (c >= p.C || n <= 0) return;
    const T* x = static_cast<const T*>(p.x) + b * p.sxb + c;
    T* y = static_cast<T*>(p.y) + (static_cast<size_t>(b) * p.S + t0) * p.C + c;
    __shared__ typename RowPipe<T, V, CONV_U, CONV_DEPTH, CONV_THREADS<false>>::Ring ring;
    RowPipe<T, V, CONV_U, CONV_DEPTH, CONV_THREADS<false>> xs(ring, x + t0 * p.sxt, p.sxt, threadIdx.y * blockDim.x + threadIdx.x);
    constexpr int AHEAD = decltype(xs)::AHEAD;
#pragma unroll
    for (int g = 0; g < AHEAD; g++) {
        if (g * CONV_U < n) xs.fetch(g * CONV_U, n);
        copies_commit();
    }
    float w[W][V], bias[V], v[W - 1 + CONV_U][V];
#pragma unroll
    for (int k = 0; k < W - 1; k++) to_floats<T, V>(input_row<T, V, W>(p, x, b, t0 - (W - 1) + k, c), v[k]);
    load_weights<V, W>(p, c, w, bias);
    for (int t = 0; t < n; t += CONV_U) {
        copies_wait<AHEAD - 1>();
        xs.take(v + (W - 1));
        if (t + AHEAD * CONV_U < n) xs.fetch(t + AHEAD * CONV_U, n);
        copies_commit();
#pragma unroll
        for (int u = 0; u < CONV_U; u++) {
            float out[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                out[j] = bias[j];
#pragma unroll
                for (int k = 0; k < W; k++) out[j] = fmaf(w[k][j], v[u + k][j], out[j]);
            }
            if (SILU) {
#pragma unroll
                for (int j = 0; j < V; j++) out[j] *= sigmoid_f(out[j]);
            }
            if (t + u < n) *reinterpret_cast<Vec<T, V>*>(y) = from_floats<T, V>(out);
            y += p.C;
        }
#pragma unroll
        for (int k = 0; k < W - 1; k++)
#pragma unroll
            for (int j = 0; j < V; j++) v[k][j] = v[CONV_U + k][j];
    }
    // The last W - 1 inputs.  Row j of the new state is row j + S of the old one where x is shorter than that: read after
    // nothing but rows in front of it has been written, so that the two may be the same memory.
    if (p.state_out && t0 == 0) {
#pragma unroll
        for (int j = 0; j < W - 1; j++)
            *reinterpret_cast<Vec<T, V>*>(static_cast<T*>(p.state_out) + (static_cast<size_t>(b) * (W - 1) + j) * p.C + c) =
                input_row<T, V, W>(p, x, b, p.S - (W - 1) + j, c);
    }
}

// Backward: the same walk over x and dy, and W - 1 positions further, whose d the run's last dx need.  Arithmetic on pairs of channels.
template <int V>
constexpr int PAIRS = (V + 1) / 2;      // (a single channel: a pair whose second half is idle)
template <int V>
__device__ __forceinline__ void pair_up(const float (&f)[V], f2 (&o)[PAIRS<V>]) {
#pragma unroll
    for (int j = 0; j < PAIRS<V>; j++) o[j] = pack2(f[2 * j], V > 1 ? f[V > 1 ? 2 * j + 1 : 0] : 0.f);
}

template <typename T, int V, int W, bool SILU>
__global__ void __launch_bounds__(CONV_THREADS<true>, 3) conv_bwd_kernel(const ConvArgs p) {
    constexpr int U = CONV_BWD_U, DEPTH = CONV_BWD_DEPTH, P = PAIRS<V>;
    __shared__ f2 red[CONV_THREADS<true>][P];
    __shared__ typename RowPipe<T, V, U, DEPTH, CONV_THREADS<true>>::Ring ring[2];
    const int tid = threadIdx.y * blockDim.x + threadIdx.x;
    grid_dep_wait();
    grid_dep_launch();
    const int c = (blockIdx.x * blockDim.x + threadIdx.x) * V, b = blockIdx.z;
    const int t0 = (blockIdx.y * blockDim.y + threadIdx.y) * p.rows, n = min(p.S - t0, p.rows);
    f2 dw[W + 1][P];               // dw[W]: the bias
#pragma unroll
    for (int k = 0; k <= W; k++)
#pragma unroll
        for (int j = 0; j < P; j++) dw[k][j] = 0;
    if (c < p.C && n > 0) {
        const int have = p.S - t0, last = n + W - 1;             // positions from t0 on that there are; that are walked
        const T* x = static_cast<const T*>(p.x) + b * p.sxb + c;
        const size_t base = (static_cast<size_t>(b) * p.S + t0) * p.C + c;
        T* dx = static_cast<T*>(p.dx) + base;
        const int there = min(have, last);
        RowPipe<T, V, U, DEPTH, CONV_THREADS<true>> xs(ring[0], x + t0 * p.sxt, p.sxt, tid), gs(ring[1], static_cast<const T*>(p.dy) + base, p.C, tid);
        constexpr int AHEAD = decltype(xs)::AHEAD;
#pragma unroll
        for (int g = 0; g < AHEAD; g++) {
            if (g * U < last) {
                xs.fetch(g * U, there);
                gs.fetch(g * U, there);                              // (d = 0 behind the last position)
            }
            copies_commit();
        }
        f2 w[W][P], bias[P], v[W - 1 + U][P], d[W - 1 + U][P];
        {
            float wf[W][V], bf[V];
            load_weights<V, W>(p, c, wf, bf);
            pair_up<V>(bf, bias);
#pragma unroll
            for (int k = 0; k < W; k++) pair_up<V>(wf[k], w[k]);
        }
#pragma unroll
        for (int k = 0; k < W - 1; k++) {
            float f[V];
            to_floats<T, V>(input_row<T, V, W>(p, x, b, t0 - (W - 1) + k, c), f);
            pair_up<V>(f, v[k]);
#pragma unroll
            for (int j = 0; j < P; j++) d[k][j] = 0;
        }
        const f2 one = pack2(1.f, 1.f), minus = pack2(-1.f, -1.f);
        for (int t = 0; t < last; t += U) {
            copies_wait<AHEAD - 1>();
            {
                float f[U][V];
                xs.take(f);
#pragma unroll
                for (int u = 0; u < U; u++) pair_up<V>(f[u], v[W - 1 + u]);
                gs.take(f);
#pragma unroll
                for (int u = 0; u < U; u++) pair_up<V>(f[u], d[W - 1 + u]);
            }
            if (t + AHEAD * U < last) {
                xs.fetch(t + AHEAD * U, there);
                gs.fetch(t + AHEAD * U, there);
            }
            copies_commit();
            // (a group in the middle of the run: no test between its positions, whose chains then overlap)
            auto group = [&](auto whole) {
                constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    f2* g = d[W - 1 + u];
                    if (SILU) {
#pragma unroll
                        for (int j = 0; j < P; j++) {
                            f2 a = bias[j];
#pragma unroll
                            for (int k = 0; k < W; k++) a = fma2(w[k][j], v[u + k][j], a);
                            const f2 sg = sigmoid2(a);                    // silu' = sg (1 + a (1 - sg))
                            g[j] = mul2(mul2(g[j], sg), fma2(a, fma2(sg, minus, one), one));
                        }
                    }
                }
                if (SILU && !WHOLE && t + U > there) {          // (what adds up behind the last position may be no number)
#pragma unroll
                    for (int u = 0; u < U; u++)
#pragma unroll
                        for (int j = 0; j < P; j++)
                            if (t + u >= there) d[W - 1 + u][j] = 0;
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const f2* g = d[W - 1 + u];
                    if (WHOLE || t + u < n) {
#pragma unroll
                        for (int j = 0; j < P; j++) {
#pragma unroll
                            for (int k = 0; k < W; k++) dw[k][j] = fma2(g[j], v[u + k][j], dw[k][j]);
                            dw[W][j] = add2(dw[W][j], g[j]);
                        }
                    }
                    if (WHOLE || (t + u >= W - 1 && t + u < last)) {      // dx_s = sum_k w[k] d_{s + (W - 1) - k}
                        float out[V];
#pragma unroll
                        for (int j = 0; j < P; j++) {
                            f2 a = mul2(w[0][j], d[W - 1 + u][j]);
#pragma unroll
                            for (int k = 1; k < W; k++) a = fma2(w[k][j], d[W - 1 + u - k][j], a);
                            const float2 o = unpack2(a);
                            out[2 * j] = o.x;
                            if (V > 1) out[V > 1 ? 2 * j + 1 : 0] = o.y;
                        }
                        store_vec<T, V>(dx, from_floats<T, V>(out));
                        dx += p.C;
                    }
                }
            };
            static_assert(U >= W - 1, "the first group alone has positions whose dx is another run's");
            if (t > 0 && t + U <= n) group(std::true_type{});
            else group(std::false_type{});
#pragma unroll
            for (int k = 0; k < W - 1; k++)
#pragma unroll
                for (int j = 0; j < P; j++) {
                    v[k][j] = v[U + k][j];
                    d[k][j] = d[U + k][j];
                }
        }
    }
    // the block's runs of the same channels, one after the other
    const size_t row = static_cast<size_t>(b) * gridDim.y + blockIdx.y;
#pragma unroll
    for (int k = 0; k <= W; k++) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < P; j++) red[tid][j] = dw[k][j];
        __syncthreads();
        if (threadIdx.y == 0 && c < p.C) {
            for (int r = 1; r < static_cast<int>(blockDim.y); r++)
#pragma unroll
                for (int j = 0; j < P; j++) dw[k][j] = add2(dw[k][j], red[r * blockDim.x + threadIdx.x][j]);
#pragma unroll
            for (int j = 0; j < P; j++) {
                const float2 o = unpack2(dw[k][j]);
                float* part = p.part + (row * (W + 1) + k) * p.C + c + 2 * j;
                part[0] = o.x;
                if (V > 1) part[1] = o.y;
            }
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

// Bytes of a row that a thread takes where everything is aligned for that.  (16 bytes cost registers, and with them threads: 92 against
// 68 us for 4 x 4096 x 4096 bf16 forward, before the copies were asynchronous; 4 bytes: 69.)
constexpr int CONV_BYTES = 8;
int conv_vec(const ConvArgs& a, int es) {
    constexpr int bytes = CONV_BYTES;
    const int v = bytes / es;
    if (a.C % v || a.sxb % v || a.sxt % v) return 1;
    for (const void* q : {a.x, a.initial, a.dy, static_cast<const void*>(a.y), static_cast<const void*>(a.state_out),
                          static_cast<const void*>(a.dx)})
        if (!aligned(q, bytes)) return 1;
    return v;
}

struct ConvGrid {
    dim3 grid, block;
    int rows;                      // positions per thread
};
ConvGrid conv_grid(const ConvArgs& a, int V, bool bwd) {
    const long long cv = ceil_up(a.C, V);
    ConvGrid g;
    int y = 1;
    const int threads = bwd ? CONV_THREADS<true> : CONV_THREADS<false>;
    while (y < threads / 32 && y * 8 < a.S) y *= 2;
    g.block = dim3(threads / y, y, 1);
    const long long bx = ceil_up(cv, g.block.x);
    // the longest runs (the fewest inputs read twice, and partial sums) that still give every SM eight blocks
    g.rows = 64;
    while (g.rows > 8 && bx * a.Bt * ceil_up(a.S, g.rows * y) < 148 * 8) g.rows /= 2;
    g.grid = dim3(static_cast<unsigned>(bx), static_cast<unsigned>(ceil_up(a.S, g.rows * y)), a.Bt);
    return g;
}

template <typename T, int V, int W, bool BWD>
cudaError_t launch_conv_w(ConvArgs& a, cudaStream_t st) {
    const ConvGrid g = conv_grid(a, V, BWD);
    a.rows = g.rows;
    if constexpr (BWD) return launch_plain(a.silu ? conv_bwd_kernel<T, V, W, true> : conv_bwd_kernel<T, V, W, false>, g.grid, g.block, 0, st, a);
    else return launch_plain(a.silu ? conv_fwd_kernel<T, V, W, true> : conv_fwd_kernel<T, V, W, false>, g.grid, g.block, 0, st, a);
}
template <typename T, bool BWD>
cudaError_t launch_conv_t(ConvArgs& a, int W, int V, cudaStream_t st) {
    constexpr int VMAX = CONV_BYTES / static_cast<int>(sizeof(T));
    if (V == 1) return W == 2 ? launch_conv_w<T, 1, 2, BWD>(a, st) : W == 3 ? launch_conv_w<T, 1, 3, BWD>(a, st) : launch_conv_w<T, 1, 4, BWD>(a, st);
    return W == 2 ? launch_conv_w<T, VMAX, 2, BWD>(a, st) : W == 3 ? launch_conv_w<T, VMAX, 3, BWD>(a, st) : launch_conv_w<T, VMAX, 4, BWD>(a, st);
}
template <bool BWD>
cudaError_t launch_conv(ConvArgs& a, int W, int V, int dtype, cudaStream_t st) {
    return dtype == MLSTM_DT_F32 ? launch_conv_t<float, BWD>(a, W, V, st)
           : dtype == MLSTM_DT_F16 ? launch_conv_t<__half, BWD>(a, W, V, st) : launch_conv_t<__nv_bfloat16, BWD>(a, W, V, st);
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

// bytes of the partial sums of the parameters' gradients with V channels per thread
size_t conv_part_bytes(int B, int S, int C, int W, int V) {
    ConvArgs a{};
    a.Bt = B; a.S = S; a.C = C;
    return static_cast<size_t>(B) * conv_grid(a, V, true).grid.y * (W + 1) * C * sizeof(float);
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
    a.Bt = B; a.S = S; a.C = C; a.wdt = w_dtype; a.wvec = aligned(weight, 16) && aligned(bias, 16); a.silu = silu;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int V = conv_vec(a, es);
    const cudaError_t ce = launch_conv<false>(a, W, V, dtype, st);
    if (ce != cudaSuccess) cudaGetLastError();
    return ce == cudaSuccess ? MLSTM_OK : note_cuda_error(ce, "launch of conv_fwd_kernel");
}

size_t mlstm_conv_bwd_workspace(int B, int S, int C, int W, int dtype) {
    const void* any = reinterpret_cast<const void*>(16);
    if (conv_check(any, any, B, S, C, W, dtype, dtype, nullptr) != MLSTM_OK) return 0;
    // whichever access width the pointers of the call will allow: the grid, and with it the number of partial sums, follows from it
    const size_t wide = conv_part_bytes(B, S, C, W, dtype == MLSTM_DT_F32 ? CONV_BYTES / 4 : CONV_BYTES / 2), one = conv_part_bytes(B, S, C, W, 1);
    return wide > one ? wide : one;
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
    if (!workspace || !aligned(workspace, 16)) return MLSTM_E_WORKSPACE;
    ConvArgs a{};
    a.x = x; a.weight = weight; a.bias = bias; a.dy = dy; a.dx = dx; a.part = static_cast<float*>(workspace);
    a.sxb = strides ? strides[0] : static_cast<long long>(S) * C;
    a.sxt = strides ? strides[1] : C;
    a.Bt = B; a.S = S; a.C = C; a.wdt = w_dtype; a.wvec = aligned(weight, 16) && aligned(bias, 16); a.silu = silu;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int V = conv_vec(a, es);
    if (workspace_bytes < conv_part_bytes(B, S, C, W, V)) return MLSTM_E_WORKSPACE;
    cudaError_t ce = launch_conv<true>(a, W, V, dtype, st);
    if (ce == cudaSuccess) {
        const int rows = B * static_cast<int>(conv_grid(a, V, true).grid.y);
        ce = launch_reduce_rows(a.part, rows, static_cast<long long>(W + 1) * C,
                                ConvParamOut{{dweight, w_dtype}, {dbias, w_dtype}, W, C}, st);
    }
    if (ce != cudaSuccess) cudaGetLastError();
    return ce == cudaSuccess ? MLSTM_OK : note_cuda_error(ce, "launch of conv_bwd_kernel");
}

}  // extern "C"
