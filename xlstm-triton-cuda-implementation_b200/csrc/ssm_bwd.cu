// Selective state space scan: gradients of all inputs (ssm_common.cuh has the forward's formulas and the layout of the work).
//
// With e_t = dy_t * silu(z_t), u_t = exp(delta_t A) h_{t-1} and the gradient g_t of the state behind position t:
//     g_t = C_t e_t + exp(delta_{t+1} A) g_{t+1}
//     dC_t = sum_c e_t h_t          dB_t = sum_c delta_t x_t g_t          dA = sum_t delta_t g_t u_t
//     dx_t = delta_t sum_n g_t B_t + D e_t        ddelta_t = x_t sum_n g_t B_t + sum_n A g_t u_t
//     dz_t = dy_t (sum_n C_t h_t + D x_t) silu'(z_t),   ddt = ddelta * sigmoid(dt + bias) behind a softplus
// The positions are walked from the last to the first in runs of SSM_CK: the states inside a run are computed again from the
// state that the forward kept in front of it, first at every SSM_ROWS positions (to shared memory), then for one group of
// SSM_ROWS at a time in registers, together with the exponentials that the way back needs again.
//
// The sums over the channels (dB, dC) run over a CTA's 64 channels by a transposing butterfly (half of the values change hands at
// every step, so 8 values cost 9 shuffles instead of 40) and over the CTAs of a group in a second kernel; the sums over the
// states run over the warps through shared memory.  No atomics: the same inputs give the same bits.
#include "reduce_rows.cuh"
#include "ssm_common.cuh"

namespace mlstm {
namespace {

struct SsmBwdArgs : SsmArgs {
    const void* dy;                 // [Bt, S, Ch]
    void *dx, *ddt, *dz;            // [Bt, S, Ch]
    float2* bc_part;                // [tiles, batches of this launch, S, N] {dB, dC} of 64 channels
    float* param_part;              // [Bt, nseg, N + 2, Cpad]: dA, dD, dbias
    int b0, nb;                     // batches of this launch: b0 .. b0 + nb - 1
};

constexpr int BWD_SUBS = SSM_CK / SSM_ROWS;

template <int K, int W>
struct SsmBwdSmem {
    float4 dl[SSM_CK][32];                  // delta, delta x
    float2 e[SSM_CK][32];                   // dy silu(z)
    float4 bc[SSM_CK][K * W];               // B, B, C, C
    float2 h[BWD_SUBS][K * W][32];          // the states in front of every SSM_ROWS positions
    float2 red[3][W][SSM_ROWS][32];         // every warp's sums over its states: g B, A g u, C h
    float2 bcg[SSM_ROWS][K * W];            // dB, dC of this CTA's channels
};

// Sums 8 values over the warp; the sum of v[i] arrives in the lanes 4 i .. 4 i + 3.
__device__ __forceinline__ float butterfly8(float (&v)[SSM_ROWS], int lane) {
#pragma unroll
    for (int half = 4, o = 16; half > 0; half >>= 1, o >>= 1) {
        const bool up = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < half; i++) {
            const float keep = up ? v[i + half] : v[i], send = up ? v[i] : v[i + half];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    }
    v[0] += __shfl_xor_sync(0xffffffffu, v[0], 2);
    return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 1);
}

__device__ __forceinline__ float2 delta_of(float2 raw, float2 bias, int softplus) {
    raw.x += bias.x;
    raw.y += bias.y;
    return softplus ? make_float2(softplus_f(raw.x), softplus_f(raw.y)) : raw;
}

// What one segment adds to the gradient of the state in front of it: G = exp(delta A) (G + C e), from the last position back.
template <typename T, int K, int W>
__global__ void __launch_bounds__(32 * W) ssm_back_state_kernel(const SsmBwdArgs p) {
    constexpr int TILE = SSM_ROWS, NP = K * W, IT = TILE / W, BI = (TILE * NP) / (32 * W) > 0 ? (TILE * NP) / (32 * W) : 1;
    __shared__ float4 sm_d[TILE][32];       // delta, e
    __shared__ float2 sm_c[TILE][NP];       // C, C
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = p.b0 + blockIdx.z, seg = blockIdx.y + 1;
    const SsmTile ch = ssm_tile(p, blockIdx.x, lane);
    const int t_begin = seg * p.seglen, t_end = min(p.S, t_begin + p.seglen);
    const bool pairs = p.pairs != 0;
    const T* dtp = static_cast<const T*>(p.dt) + b * p.sdt.b + ch.c;
    const T* zp = p.z ? static_cast<const T*>(p.z) + b * p.sz.b + ch.c : nullptr;
    const T* dyp = static_cast<const T*>(p.dy) + static_cast<size_t>(b) * p.S * p.Ch + ch.c;
    const T* Cp = static_cast<const T*>(p.C) + b * p.sC.b + static_cast<long long>(ch.g) * p.N;
    float2 bias = make_float2(0.f, 0.f);
    if (p.bias) {
        if (ch.n > 0) bias.x = p.bias[ch.c];
        if (ch.n > 1) bias.y = p.bias[ch.c + 1];
    }
    f2 rate[K], G[K], sum = 0;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int n = warp * K + k;
        float r0 = 0.f, r1 = 0.f;
        if (n < p.N) {
            const size_t at = static_cast<size_t>(ch.c) * p.N + n;
            if (ch.n > 0) r0 = decay_rate(p.A[at]);
            if (ch.n > 1) r1 = decay_rate(p.A[at + p.N]);
        }
        rate[k] = pack2(r0, r1);
        G[k] = 0;
    }
    const int tiles = ceil_div(t_end - t_begin, TILE);
    for (int tile = tiles - 1; tile >= 0; tile--) {
        const int t0 = t_begin + tile * TILE;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < IT; i++) {
            const int r = warp + W * i, t = t0 + r, n = t < t_end ? ch.n : 0;
            float2 d = delta_of(to_float2<T>(load_raw2<T>(dtp + t * p.sdt.t, pairs, n)), bias, p.softplus);
            float2 e = to_float2<T>(load_raw2<T>(dyp + static_cast<size_t>(t) * p.Ch, pairs, n));
            if (zp) {
                const float2 z = to_float2<T>(load_raw2<T>(zp + t * p.sz.t, pairs, n));
                e = make_float2(e.x * silu_f(z.x), e.y * silu_f(z.y));
            }
            if (t >= t_end) d = make_float2(0.f, 0.f);
            sm_d[r][lane] = make_float4(d.x, d.y, e.x, e.y);
        }
#pragma unroll
        for (int i = 0; i < BI; i++) {
            const int x = threadIdx.x + i * 32 * W, t = t0 + x / NP, n = x % NP;
            if (x < TILE * NP) {
                const float c = n < p.N && t < t_end ? to_f32<T>(Cp[t * p.sC.t + n]) : 0.f;
                sm_c[x / NP][n] = make_float2(c, c);
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (warp * K + k >= p.N) break;
#pragma unroll
            for (int r = TILE - 1; r >= 0; r--) {
                const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sm_d[r][lane]);
                G[k] = mul2(exp2_2(mul2(v.x, rate[k])), fma2(v.y, *reinterpret_cast<const f2*>(&sm_c[r][warp * K + k]), G[k]));
            }
        }
        if (warp == 0) {
#pragma unroll
            for (int r = 0; r < TILE; r++) sum = add2(sum, *reinterpret_cast<const f2*>(&sm_d[r][lane]));
        }
    }
    const size_t sj = static_cast<size_t>(b) * p.nseg + seg;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int n = warp * K + k;
        if (n < p.N) *reinterpret_cast<f2*>(p.seg_end + (sj * p.N + n) * p.Cpad + ch.cp) = G[k];
    }
    if (warp == 0) *reinterpret_cast<f2*>(p.seg_sum + sj * p.Cpad + ch.cp) = sum;
}

template <typename T, int K, int W, bool GATED>
__global__ void __launch_bounds__(32 * W) ssm_bwd_kernel(const SsmBwdArgs p) {
    constexpr int NP = K * W, IT = SSM_ROWS / W;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    SsmBwdSmem<K, W>& sm = *reinterpret_cast<SsmBwdSmem<K, W>*>(smem_raw);
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bl = blockIdx.z, b = p.b0 + bl, seg = blockIdx.y;
    const SsmTile ch = ssm_tile(p, blockIdx.x, lane);
    const int t_begin = seg * p.seglen, t_end = min(p.S, t_begin + p.seglen);
    const bool pairs = p.pairs != 0;

    const T* xp = static_cast<const T*>(p.x) + b * p.sx.b + ch.c;
    const T* dtp = static_cast<const T*>(p.dt) + b * p.sdt.b + ch.c;
    const T* zp = GATED ? static_cast<const T*>(p.z) + b * p.sz.b + ch.c : nullptr;
    const size_t row0 = static_cast<size_t>(b) * p.S;
    const T* dyp = static_cast<const T*>(p.dy) + row0 * p.Ch + ch.c;
    const T* Bp = static_cast<const T*>(p.B) + b * p.sB.b + static_cast<long long>(ch.g) * p.N;
    const T* Cp = static_cast<const T*>(p.C) + b * p.sC.b + static_cast<long long>(ch.g) * p.N;

    float2 bias = make_float2(0.f, 0.f), skip = make_float2(0.f, 0.f), dskip = make_float2(0.f, 0.f), dbias = make_float2(0.f, 0.f);
    if (p.bias) {
        if (ch.n > 0) bias.x = p.bias[ch.c];
        if (ch.n > 1) bias.y = p.bias[ch.c + 1];
    }
    if (p.D) {
        if (ch.n > 0) skip.x = p.D[ch.c];
        if (ch.n > 1) skip.y = p.D[ch.c + 1];
    }
    f2 rate[K], G[K], dA[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int n = warp * K + k;
        float r0 = 0.f, r1 = 0.f;
        if (n < p.N) {
            const size_t at = static_cast<size_t>(ch.c) * p.N + n;
            if (ch.n > 0) r0 = decay_rate(p.A[at]);
            if (ch.n > 1) r1 = decay_rate(p.A[at + p.N]);
        }
        rate[k] = pack2(r0, r1);
        G[k] = 0;
        dA[k] = 0;
    }
    for (int j = p.nseg - 1; j > seg; j--) {        // the segments behind this one, from the last
        const size_t sj = static_cast<size_t>(b) * p.nseg + j;
        const f2 sum = *reinterpret_cast<const f2*>(p.seg_sum + sj * p.Cpad + ch.cp);
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int n = warp * K + k;
            if (n < p.N)
                G[k] = fma2(exp2_2(mul2(sum, rate[k])), G[k], *reinterpret_cast<const f2*>(p.seg_end + (sj * p.N + n) * p.Cpad + ch.cp));
        }
    }

    const int chunks = ceil_div(t_end - t_begin, SSM_CK);
    for (int chunk = chunks - 1; chunk >= 0; chunk--) {
        const int tc = t_begin + chunk * SSM_CK, subs = ceil_div(min(SSM_CK, t_end - tc), SSM_ROWS);
        f2 h[K];
        {
            const size_t row = static_cast<size_t>(b) * ceil_div(p.S, SSM_CK) + tc / SSM_CK;
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int n = warp * K + k;
                h[k] = n < p.N ? *reinterpret_cast<const f2*>(p.ckpt + (row * p.N + n) * p.Cpad + ch.cp) : 0;
            }
        }
#pragma unroll 4
        for (int r = warp; r < SSM_CK; r += W) {
            const int t = tc + r, n = t < t_end ? ch.n : 0;
            const float2 x = to_float2<T>(load_raw2<T>(xp + t * p.sx.t, pairs, n));
            float2 d = delta_of(to_float2<T>(load_raw2<T>(dtp + t * p.sdt.t, pairs, n)), bias, p.softplus);
            float2 e = to_float2<T>(load_raw2<T>(dyp + static_cast<size_t>(t) * p.Ch, pairs, n));
            if (GATED) {
                const float2 z = to_float2<T>(load_raw2<T>(zp + t * p.sz.t, pairs, n));
                e = make_float2(e.x * silu_f(z.x), e.y * silu_f(z.y));
            }
            if (t >= t_end) d = make_float2(0.f, 0.f);
            sm.dl[r][lane] = make_float4(d.x, d.y, d.x * x.x, d.y * x.y);
            sm.e[r][lane] = e;
        }
#pragma unroll
        for (int i = 0; i < K; i++) {
            const int x = threadIdx.x + i * 32 * W, t = tc + x / NP, n = x % NP;
            const bool in = n < p.N && t < t_end;
            const float bv = in ? to_f32<T>(Bp[t * p.sB.t + n]) : 0.f, cv = in ? to_f32<T>(Cp[t * p.sC.t + n]) : 0.f;
            sm.bc[x / NP][n] = make_float4(bv, bv, cv, cv);
        }
        __syncthreads();
        // the states in front of every SSM_ROWS positions (each warp its own)
#pragma unroll 1
        for (int sub = 0; sub < subs; sub++) {
#pragma unroll
            for (int k = 0; k < K; k++) *reinterpret_cast<f2*>(&sm.h[sub][warp * K + k][lane]) = h[k];
            if (sub + 1 < subs) {
#pragma unroll
                for (int r = 0; r < SSM_ROWS; r++) {
                    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sm.dl[sub * SSM_ROWS + r][lane]);
#pragma unroll
                    for (int k = 0; k < K; k++)
                        h[k] = fma2(exp2_2(mul2(v.x, rate[k])), h[k],
                                    mul2(v.y, *reinterpret_cast<const f2*>(&sm.bc[sub * SSM_ROWS + r][warp * K + k])));
                }
            }
        }
#pragma unroll 1
        for (int sub = subs - 1; sub >= 0; sub--) {
            const int q = sub * SSM_ROWS;
            // for the positions that this thread finishes
            Raw2<T> rx[IT], rdt[IT], rdy[IT];
            [[maybe_unused]] Raw2<T> rz[IT];
#pragma unroll
            for (int i = 0; i < IT; i++) {
                const int t = tc + q + warp + W * i, n = t < t_end ? ch.n : 0;
                rx[i] = load_raw2<T>(xp + t * p.sx.t, pairs, n);
                rdt[i] = load_raw2<T>(dtp + t * p.sdt.t, pairs, n);
                if (GATED) {
                    rz[i] = load_raw2<T>(zp + t * p.sz.t, pairs, n);
                    rdy[i] = load_raw2<T>(dyp + static_cast<size_t>(t) * p.Ch, pairs, n);
                }
            }
            f2 dl[SSM_ROWS], dx[SSM_ROWS], e[SSM_ROWS], sb[SSM_ROWS], su[SSM_ROWS];
            [[maybe_unused]] f2 y[SSM_ROWS];
#pragma unroll
            for (int r = 0; r < SSM_ROWS; r++) {
                const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sm.dl[q + r][lane]);
                dl[r] = v.x;
                dx[r] = v.y;
                e[r] = *reinterpret_cast<const f2*>(&sm.e[q + r][lane]);
                sb[r] = 0;
                su[r] = 0;
                if (GATED) y[r] = 0;
            }
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int n = warp * K + k;
                if (n >= p.N) break;
                f2 a[SSM_ROWS], u[SSM_ROWS], s = *reinterpret_cast<const f2*>(&sm.h[sub][n][lane]);
                float part[SSM_ROWS];
#pragma unroll
                for (int r = 0; r < SSM_ROWS; r++) {
                    const ulonglong2 bc = *reinterpret_cast<const ulonglong2*>(&sm.bc[q + r][n]);
                    a[r] = exp2_2(mul2(dl[r], rate[k]));
                    u[r] = mul2(a[r], s);
                    s = fma2(dx[r], bc.x, u[r]);
                    if (GATED) y[r] = fma2(s, bc.y, y[r]);
                    const float2 c = unpack2(mul2(e[r], s));
                    part[r] = c.x + c.y;
                }
                const float dc = butterfly8(part, lane);
                f2 g = G[k];
#pragma unroll
                for (int r = SSM_ROWS - 1; r >= 0; r--) {
                    const ulonglong2 bc = *reinterpret_cast<const ulonglong2*>(&sm.bc[q + r][n]);
                    g = fma2(bc.y, e[r], g);
                    sb[r] = fma2(g, bc.x, sb[r]);
                    const f2 w = mul2(g, u[r]);
                    su[r] = fma2(w, rate[k], su[r]);
                    dA[k] = fma2(dl[r], w, dA[k]);
                    const float2 c = unpack2(mul2(g, dx[r]));
                    part[r] = c.x + c.y;
                    g = mul2(a[r], g);
                }
                G[k] = g;
                const float db = butterfly8(part, lane);
                if ((lane & 3) == 0) sm.bcg[lane >> 2][n] = make_float2(db, dc);
            }
#pragma unroll
            for (int r = 0; r < SSM_ROWS; r++) {
                *reinterpret_cast<f2*>(&sm.red[0][warp][r][lane]) = sb[r];
                *reinterpret_cast<f2*>(&sm.red[1][warp][r][lane]) = su[r];
                if (GATED) *reinterpret_cast<f2*>(&sm.red[2][warp][r][lane]) = y[r];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < IT; i++) {
                const int r = warp + W * i, t = tc + q + r;
                if (t < t_end) {
                    f2 vs = 0, vu = 0, vy = 0;
#pragma unroll
                    for (int w = 0; w < W; w++) {
                        vs = add2(vs, *reinterpret_cast<const f2*>(&sm.red[0][w][r][lane]));
                        vu = add2(vu, *reinterpret_cast<const f2*>(&sm.red[1][w][r][lane]));
                        if (GATED) vy = add2(vy, *reinterpret_cast<const f2*>(&sm.red[2][w][r][lane]));
                    }
                    const float2 s = unpack2(vs), u = unpack2(vu), x = to_float2<T>(rx[i]), ev = sm.e[q + r][lane];
                    const float4 d = sm.dl[q + r][lane];
                    constexpr float LN2 = 0.69314718055994530942f;      // the rates are in units of log2
                    float2 dd = make_float2(fmaf(x.x, s.x, LN2 * u.x), fmaf(x.y, s.y, LN2 * u.y));
                    if (p.softplus) {
                        const float2 raw = to_float2<T>(rdt[i]);
                        dd.x *= sigmoid_f(raw.x + bias.x);
                        dd.y *= sigmoid_f(raw.y + bias.y);
                    }
                    dbias.x += dd.x;
                    dbias.y += dd.y;
                    dskip.x = fmaf(ev.x, x.x, dskip.x);
                    dskip.y = fmaf(ev.y, x.y, dskip.y);
                    const size_t at = (row0 + t) * p.Ch + ch.c;
                    store_pair<T>(static_cast<T*>(p.ddt) + at, dd, pairs, ch.n);
                    store_pair<T>(static_cast<T*>(p.dx) + at, make_float2(fmaf(d.x, s.x, p.D ? skip.x * ev.x : 0.f), fmaf(d.y, s.y, p.D ? skip.y * ev.y : 0.f)),
                                  pairs, ch.n);
                    if (GATED) {
                        const float2 z = to_float2<T>(rz[i]), dy = to_float2<T>(rdy[i]);
                        float2 yv = unpack2(vy);
                        if (p.D) yv = make_float2(fmaf(skip.x, x.x, yv.x), fmaf(skip.y, x.y, yv.y));
                        const float s0 = sigmoid_f(z.x), s1 = sigmoid_f(z.y);
                        store_pair<T>(static_cast<T*>(p.dz) + at,
                                      make_float2(dy.x * yv.x * s0 * fmaf(z.x, 1.0f - s0, 1.0f), dy.y * yv.y * s1 * fmaf(z.y, 1.0f - s1, 1.0f)),
                                      pairs, ch.n);
                    }
                }
            }
            for (int x = threadIdx.x; x < SSM_ROWS * p.N; x += 32 * W) {
                const int r = x / p.N, n = x - r * p.N, t = tc + q + r;
                if (t < t_end) p.bc_part[((static_cast<size_t>(blockIdx.x) * p.nb + bl) * p.S + t) * p.N + n] = sm.bcg[r][n];
            }
            __syncthreads();
        }
    }
    float* part = p.param_part + (static_cast<size_t>(b) * p.nseg + seg) * (p.N + 2) * p.Cpad + ch.cp;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int n = warp * K + k;
        if (n < p.N) *reinterpret_cast<f2*>(part + static_cast<size_t>(n) * p.Cpad) = dA[k];
    }
    sm.red[0][warp][0][lane] = dskip;
    sm.red[1][warp][0][lane] = dbias;
    __syncthreads();
    if (warp < 2) {
        float2 v = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float2 q = sm.red[warp][w][0][lane];
            v.x += q.x;
            v.y += q.y;
        }
        *reinterpret_cast<float2*>(part + static_cast<size_t>(p.N + warp) * p.Cpad) = v;
    }
}

// dB, dC [Bt, S, G, N]: sums over the CTAs of a group.
template <typename T>
__global__ void __launch_bounds__(256) ssm_bc_sum_kernel(const float2* __restrict__ part, T* __restrict__ dB, T* __restrict__ dC, int tiles_g,
                                                         int G, int N, long long rows, long long row0) {
    grid_dep_wait();
    grid_dep_launch();
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x, per = rows * N;
    if (i >= per) return;
    const int g = blockIdx.y;
    const float2* q = part + static_cast<long long>(g) * tiles_g * per + i;
    float2 s = make_float2(0.f, 0.f);
#pragma unroll 8
    for (int k = 0; k < tiles_g; k++) {
        const float2 v = q[k * per];
        s.x += v.x;
        s.y += v.y;
    }
    const long long r = i / N, at = ((row0 + r) * G + g) * N + (i - r * N);
    dB[at] = from_f32<T>(s.x);
    dC[at] = from_f32<T>(s.y);
}

struct SsmParamOut {
    float *dA, *dD, *dbias;
    int N, Cpad, P, tiles_g;
    __device__ __forceinline__ void operator()(long long col, float v) const {
        const int n = static_cast<int>(col / Cpad), cp = static_cast<int>(col - static_cast<long long>(n) * Cpad);
        const int g = cp / (tiles_g * SSM_CH), in_g = cp - g * tiles_g * SSM_CH;
        if (in_g >= P) return;
        const long long c = static_cast<long long>(g) * P + in_g;
        if (n < N) dA[c * N + n] = v;
        else if (n == N) { if (dD) dD[c] = v; }
        else if (dbias) dbias[c] = v;
    }
};

constexpr size_t SSM_BWD_PART_MAX = 512u << 20;     // bytes of dB, dC partials in scratch at one time (at least one batch entry)
constexpr int SSM_BWD_CTAS = 3;                     // CTAs of 4 warps that an SM is filled with

struct SsmBwdWs {
    float *seg_end, *seg_sum, *param;
    float2* bc;
    int nb;
    size_t bytes;
};
SsmBwdWs ssm_bwd_carve(void* ws, const SsmArgs& a) {
    SsmBwdWs w{};
    uint8_t* base = static_cast<uint8_t*>(ws);
    size_t off = 0;
    auto take = [&](size_t bytes) {
        uint8_t* p = base ? base + off : nullptr;
        off += (bytes + 255) / 256 * 256;
        return p;
    };
    const size_t segs = static_cast<size_t>(a.Bt) * a.nseg;
    if (a.nseg > 1) {
        w.seg_end = reinterpret_cast<float*>(take(segs * a.N * a.Cpad * 4));
        w.seg_sum = reinterpret_cast<float*>(take(segs * a.Cpad * 4));
    }
    w.param = reinterpret_cast<float*>(take(segs * (a.N + 2) * a.Cpad * 4));
    const size_t one = static_cast<size_t>(a.Cpad / SSM_CH) * a.S * a.N * sizeof(float2);
    size_t nb = SSM_BWD_PART_MAX / one;
    if (nb < 1) nb = 1;
    w.nb = nb < static_cast<size_t>(a.Bt) ? static_cast<int>(nb) : a.Bt;
    w.bc = reinterpret_cast<float2*>(take(one * w.nb));
    w.bytes = off;
    return w;
}

template <typename T, int K, int W>
cudaError_t launch_ssm_bwd(SsmBwdArgs a, const SsmBwdWs& w, void* dB, void* dC, cudaStream_t st) {
    const unsigned tiles = static_cast<unsigned>(a.G * a.tiles_g);
    constexpr size_t smem = sizeof(SsmBwdSmem<K, W>);
    auto kern = a.z ? ssm_bwd_kernel<T, K, W, true> : ssm_bwd_kernel<T, K, W, false>;
    cudaError_t ce = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    for (int b0 = 0; b0 < a.Bt && ce == cudaSuccess; b0 += w.nb) {
        a.b0 = b0;
        a.nb = a.Bt - b0 < w.nb ? a.Bt - b0 : w.nb;
        if (a.nseg > 1) ce = launch_plain(ssm_back_state_kernel<T, K, W>, dim3(tiles, a.nseg - 1, a.nb), dim3(32 * W), 0, st, a);
        if (ce == cudaSuccess) ce = launch_plain(kern, dim3(tiles, a.nseg, a.nb), dim3(32 * W), smem, st, a);
        const long long rows = static_cast<long long>(a.nb) * a.S;
        if (ce == cudaSuccess)
            ce = launch_plain(ssm_bc_sum_kernel<T>, dim3(static_cast<unsigned>((rows * a.N + 255) / 256), a.G), dim3(256), 0, st, a.bc_part,
                              static_cast<T*>(dB), static_cast<T*>(dC), a.tiles_g, a.G, a.N, rows, static_cast<long long>(b0) * a.S);
    }
    return ce;
}
template <typename T>
cudaError_t launch_ssm_bwd_n(const SsmBwdArgs& a, const SsmBwdWs& w, void* dB, void* dC, cudaStream_t st) {
    if (a.N <= 4) return launch_ssm_bwd<T, 1, 4>(a, w, dB, dC, st);
    if (a.N <= 8) return launch_ssm_bwd<T, 2, 4>(a, w, dB, dC, st);
    if (a.N <= 16) return launch_ssm_bwd<T, 4, 4>(a, w, dB, dC, st);
    if (a.N <= 32) return launch_ssm_bwd<T, 4, 8>(a, w, dB, dC, st);
    return launch_ssm_bwd<T, 8, 8>(a, w, dB, dC, st);
}

}  // namespace
}  // namespace mlstm

using namespace mlstm;

extern "C" {

size_t mlstm_ssm_bwd_workspace(int B, int S, int C, int G, int N) {
    SsmArgs a;
    const void* any = reinterpret_cast<const void*>(16);
    if (ssm_fill(a, any, any, static_cast<const float*>(any), any, any, nullptr, nullptr, nullptr, nullptr, B, S, C, G, N,
                 MLSTM_DT_F32, 0) != MLSTM_OK)
        return 0;
    ssm_cut(a, SSM_BWD_CTAS);
    return ssm_bwd_carve(nullptr, a).bytes;
}

int mlstm_ssm_bwd(const void* dy, const void* x, const void* dt, const float* A, const void* Bv, const void* Cv, const float* D,
                  const void* z, const float* dt_bias, const long long* strides, const float* checkpoints, void* dx, void* ddt,
                  float* dA, void* dB, void* dC, float* dD, void* dz, float* d_dt_bias, void* workspace, size_t workspace_bytes,
                  int B, int S, int C, int G, int N, int dtype, int softplus, void* stream) {
    SsmBwdArgs a;
    const int rc = ssm_fill(a, x, dt, A, Bv, Cv, D, z, dt_bias, strides, B, S, C, G, N, dtype, softplus);
    if (rc != MLSTM_OK) return rc;
    if (!dy || !checkpoints || !dx || !ddt || !dA || !dB || !dC) return MLSTM_E_ARG;
    if ((D == nullptr) != (dD == nullptr) || (z == nullptr) != (dz == nullptr) || (dt_bias == nullptr) != (d_dt_bias == nullptr)) return MLSTM_E_ARG;
    const int es = dtype == MLSTM_DT_F32 ? 4 : 2;
    for (const void* q : {dy, x, dt, Bv, Cv, z, static_cast<const void*>(dx), static_cast<const void*>(ddt), static_cast<const void*>(dB),
                          static_cast<const void*>(dC), static_cast<const void*>(dz)})
        if (!ssm_aligned(q, es)) return MLSTM_E_ALIGN;
    for (const float* q : {A, D, dt_bias, static_cast<const float*>(dA), static_cast<const float*>(dD), static_cast<const float*>(d_dt_bias)})
        if (!ssm_aligned(q, 4)) return MLSTM_E_ALIGN;
    if (!ssm_aligned(checkpoints, 8)) return MLSTM_E_ALIGN;
    ssm_cut(a, SSM_BWD_CTAS);
    const SsmBwdWs w = ssm_bwd_carve(workspace, a);
    if (!workspace || workspace_bytes < w.bytes || !ssm_aligned(workspace, 16)) return MLSTM_E_WORKSPACE;
    a.seg_end = w.seg_end; a.seg_sum = w.seg_sum; a.param_part = w.param; a.bc_part = w.bc;
    a.ckpt = const_cast<float*>(checkpoints);
    a.dy = dy; a.dx = dx; a.ddt = ddt; a.dz = dz;
    a.pairs = ssm_pairs(a, es, {dy, dx, ddt, dz});
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t ce = dtype == MLSTM_DT_F32 ? launch_ssm_bwd_n<float>(a, w, dB, dC, st)
                     : dtype == MLSTM_DT_F16 ? launch_ssm_bwd_n<__half>(a, w, dB, dC, st) : launch_ssm_bwd_n<__nv_bfloat16>(a, w, dB, dC, st);
    if (ce == cudaSuccess)
        ce = launch_reduce_rows(a.param_part, a.Bt * a.nseg, static_cast<long long>(N + 2) * a.Cpad,
                                SsmParamOut{dA, dD, d_dt_bias, N, a.Cpad, a.P, a.tiles_g}, st);
    if (ce != cudaSuccess) cudaGetLastError();
    return ce == cudaSuccess ? MLSTM_OK : note_cuda_error(ce, "launch of ssm_bwd_kernel");
}

}  // extern "C"
