// Selective state space scan: gradients of all inputs (ssm_common.cuh has the forward's formulas and the layout of the work).
//
// With e_t = dy_t * silu(z_t), u_t = exp(delta_t A) h_{t-1} and the gradient g_t of the state behind position t:
//     g_t = C_t e_t + exp(delta_{t+1} A) g_{t+1}
//     dC_t = sum_c e_t h_t          dB_t = sum_c delta_t x_t g_t          dA = sum_t delta_t g_t u_t
//     dx_t = delta_t sum_n g_t B_t + D e_t        ddelta_t = x_t sum_n g_t B_t + sum_n A g_t u_t
//     dz_t = dy_t (sum_n C_t h_t + D x_t) silu'(z_t),   ddt = ddelta * sigmoid(dt + bias) behind a softplus
// W warps share the N states, K each, and walk the positions from the last to the first in runs of SSM_CK.  The states inside a run are
// computed again from the one that the forward kept in front of it: first the one in its middle, then for BWD_ROWS positions at a
// time all of them, in registers, together with the exponentials that the way back needs again.  All warps prepare and finish
// (delta, e, the sums over the states); the next run's inputs are on their way to shared memory meanwhile.
//
// The sums over the channels (dB, dC) run over a CTA's 64 channels by a transposing butterfly (half of the values change hands at
// every step, so 8 values cost 9 shuffles instead of 40) and over the CTAs of a group in a second kernel; the sums over the
// states run over the warps through shared memory.  No atomics: the same inputs give the same bits.
//
// What bounds it: latency.  255 registers allow eight warps per SM, and a warp's two recurrences, exponentials, broadcasts and
// butterflies are chains: 24 instructions per state and position; with two blocks on every SM issue slots 47 %, shared memory 56 %,
// exponentials 30 % busy.  Measured, bf16, 16 states: 4 x 4096 x 4096 1.77 ms (2.27 with the forward), 2 x 2048 x 4096 0.54 ms (0.73).
// Tried and slower for the first, when it took 2.29 ms with the forward: four positions at a time (163 registers, more states recomputed)
// 2.59; four more warps that prepare and finish, as in the forward 2.86; the channel sums through shared memory 2.38; two states per
// warp at 128 registers, sixteen warps per SM 2.64.  More than 32 states, and 17 to 24, spill 36 to 80 bytes a thread.
#include "async_copy.cuh"
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

constexpr int BWD_ROWS = 8;                            // positions whose states are held in registers at a time
constexpr int BWD_SUBS = SSM_CK / BWD_ROWS;

template <typename T, int K, int W>
struct SsmBwdSmem {
    float4 dl[SSM_CK][32];                  // delta, delta x
    float2 e[SSM_CK][32];                   // dy silu(z)
    float4 bc[SSM_CK][K * W];               // B, B, C, C
    float2 h[BWD_SUBS - 1][K * W][32];      // the states in front of every BWD_ROWS positions but the first
    float2 red[2][3][W][BWD_ROWS][32];      // every warp's sums over its states: g B, A g u, C h
    float2 bcg[2][BWD_ROWS][K * W];         // dB, dC of this CTA's channels
    // what the next run of positions needs, on its way from memory; every thread reads back what it asked for itself
    Raw2<T> raw[2][4][SSM_CK][32];          // x, dt, dy, z
    float2 h0[2][K * W][32];                // the states in front of the run
};

// a pair of channels to shared memory: asynchronously where it is one aligned access
template <bool PAIRS, typename T>
__device__ __forceinline__ void copy_raw2(Raw2<T>* shared, const T* global, int n) {
    if constexpr (PAIRS) {
        if (n) copy_async<2 * sizeof(T)>(shared_address(shared), global);
        else *shared = Raw2<T>{};
    } else {
        *shared = load_raw2<false>(global, n);
    }
}

// Sums R values of two kinds over the warp; those of position i arrive in lane 32 / R * i (and in the lanes up to the next).  The two
// are independent: the latency of one hides the other's.
template <int R>
__device__ __forceinline__ float2 butterfly(float (&v)[R], float (&w)[R], int lane) {
#pragma unroll
    for (int half = R / 2, o = 16; half > 0; half >>= 1, o >>= 1) {
        const bool up = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < half; i++) {
            const float kv = up ? v[i + half] : v[i], sv = up ? v[i] : v[i + half];
            const float kw = up ? w[i + half] : w[i], sw = up ? w[i] : w[i + half];
            v[i] = kv + __shfl_xor_sync(0xffffffffu, sv, o);
            w[i] = kw + __shfl_xor_sync(0xffffffffu, sw, o);
        }
    }
#pragma unroll
    for (int o = 16 / R; o > 0; o >>= 1) {
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
        w[0] += __shfl_xor_sync(0xffffffffu, w[0], o);
    }
    return make_float2(v[0], w[0]);
}

// What one segment adds to the gradient of the state in front of it: G = exp(delta A) (G + C e), from the last position back.
template <typename T, int K, int W, bool PAIRS>
__global__ void __launch_bounds__(32 * W) ssm_back_state_kernel(const SsmBwdArgs p) {
    constexpr int TILE = SSM_ROWS, NP = K * W, IT = TILE / W, BI = (TILE * NP + 32 * W - 1) / (32 * W);
    __shared__ float4 sm_d[TILE][32];       // delta, e
    __shared__ float2 sm_c[TILE][NP];       // C, C
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = p.b0 + blockIdx.z, seg = blockIdx.y + 1;
    const SsmTile ch = ssm_tile(p, blockIdx.x, lane);
    const int t_begin = seg * p.seglen, t_end = min(p.S, t_begin + p.seglen);
    const T* dtp = static_cast<const T*>(p.dt) + b * p.sdt.b + ch.c;
    const T* zp = p.z ? static_cast<const T*>(p.z) + b * p.sz.b + ch.c : nullptr;
    const T* dyp = static_cast<const T*>(p.dy) + static_cast<size_t>(b) * p.S * p.Ch + ch.c;
    const T* Cp = static_cast<const T*>(p.C) + b * p.sC.b + static_cast<long long>(ch.g) * p.N;
    const f2 bias = param2(p.bias, ch.c, ch.n);
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
    Raw2<T> rdt[IT], rdy[IT], rz[IT];               // the next tile (the one in front), on its way
    T rC[BI];
    auto fetch = [&](int tile) {
        const int t0 = t_begin + tile * TILE;
#pragma unroll
        for (int i = 0; i < IT; i++) {
            const int t = t0 + warp + W * i, n = t < t_end ? ch.n : 0;
            rdt[i] = load_raw2<PAIRS>(dtp + t * p.sdt.t, n);
            rdy[i] = load_raw2<PAIRS>(dyp + static_cast<size_t>(t) * p.Ch, n);
            if (zp) rz[i] = load_raw2<PAIRS>(zp + t * p.sz.t, n);
        }
#pragma unroll
        for (int i = 0; i < BI; i++) {
            const int x = threadIdx.x + i * 32 * W, t = t0 + x / NP, n = x % NP;
            rC[i] = x < TILE * NP && n < p.N && t < t_end ? Cp[t * p.sC.t + n] : from_f32<T>(0.f);
        }
    };
    fetch(tiles - 1);
    for (int tile = tiles - 1; tile >= 0; tile--) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < IT; i++) {
            const int r = warp + W * i;
            f2 d = delta2(to_float2<T>(rdt[i]), bias, p.softplus);
            const float2 dy = to_float2<T>(rdy[i]);
            f2 e = pack2(dy.x, dy.y);
            if (zp) {
                const float2 z = to_float2<T>(rz[i]);
                e = mul2(e, mul2(pack2(z.x, z.y), sigmoid2(pack2(z.x, z.y))));
            }
            if (t_begin + tile * TILE + r >= t_end) d = 0;
            *reinterpret_cast<ulonglong2*>(&sm_d[r][lane]) = make_ulonglong2(d, e);
        }
#pragma unroll
        for (int i = 0; i < BI; i++) {
            const int x = threadIdx.x + i * 32 * W;
            const float c = to_f32<T>(rC[i]);
            if (x < TILE * NP) sm_c[x / NP][x % NP] = make_float2(c, c);
        }
        if (tile > 0) fetch(tile - 1);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (warp * K + k >= p.N) break;
#pragma unroll
            for (int r = TILE - 1; r >= 0; r--) {
                const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sm_d[r][lane]);
                G[k] = mul2(decay2(v.x, rate[k]), fma2(v.y, *reinterpret_cast<const f2*>(&sm_c[r][warp * K + k]), G[k]));
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

template <typename T, int K, int W, bool GATED, bool PAIRS, bool FULL>
__global__ void __launch_bounds__(32 * W) ssm_bwd_kernel(SsmBwdArgs p) {
    constexpr int NP = K * W, IT = SSM_CK / W, SIT = BWD_ROWS / W > 0 ? BWD_ROWS / W : 1, BSTEP = 32 * W / NP, BI = (SSM_CK + BSTEP - 1) / BSTEP;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    SsmBwdSmem<T, K, W>& sm = *reinterpret_cast<SsmBwdSmem<T, K, W>*>(smem_raw);
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bl = blockIdx.z, b = p.b0 + bl, seg = blockIdx.y;
    const SsmTile ch = ssm_tile(p, blockIdx.x, lane);
    const int t_begin = seg * p.seglen, t_end = min(p.S, t_begin + p.seglen);

    const int chunks = ceil_div(t_end - t_begin, SSM_CK), t_last = t_begin + (chunks - 1) * SSM_CK;
    // rows of this thread in the run that is fetched next (the last one first): tc + warp + W i
    const T* xp = static_cast<const T*>(p.x) + b * p.sx.b + (t_last + warp) * p.sx.t + ch.c;
    const T* dtp = static_cast<const T*>(p.dt) + b * p.sdt.b + (t_last + warp) * p.sdt.t + ch.c;
    const T* zp = GATED ? static_cast<const T*>(p.z) + b * p.sz.b + (t_last + warp) * p.sz.t + ch.c : nullptr;
    const size_t row0 = static_cast<size_t>(b) * p.S;
    const T* dyp = static_cast<const T*>(p.dy) + (row0 + t_last + warp) * p.Ch + ch.c;
    const int bt = threadIdx.x < NP * BSTEP ? threadIdx.x / NP : SSM_CK, bn = threadIdx.x % NP;    // (SSM_CK: a thread with none)
    const T* Bp = static_cast<const T*>(p.B) + b * p.sB.b + (t_last + bt) * p.sB.t + static_cast<long long>(ch.g) * p.N + bn;
    const T* Cp = static_cast<const T*>(p.C) + b * p.sC.b + (t_last + bt) * p.sC.t + static_cast<long long>(ch.g) * p.N + bn;
    const float* kept = p.ckpt + ((static_cast<size_t>(b) * ceil_div(p.S, SSM_CK) + t_last / SSM_CK) * p.N + warp * K) * p.Cpad + ch.cp;

    const f2 bias = param2(p.bias, ch.c, ch.n), skip = param2(p.D, ch.c, ch.n);
    f2 dskip = 0, dbias = 0;
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
                G[k] = carry2(sum, rate[k], G[k], *reinterpret_cast<const f2*>(p.seg_end + (sj * p.N + n) * p.Cpad + ch.cp));
        }
    }

    T rB[BI], rC[BI];
    auto fetch = [&](int left, int buf) {           // left: positions of the segment from the run on
#pragma unroll
        for (int i = 0; i < IT; i++) {
            const int r = warp + W * i, n = r < left ? ch.n : 0;
            copy_raw2<PAIRS>(&sm.raw[buf][0][r][lane], xp + (W * i) * p.sx.t, n);
            copy_raw2<PAIRS>(&sm.raw[buf][1][r][lane], dtp + (W * i) * p.sdt.t, n);
            copy_raw2<PAIRS>(&sm.raw[buf][2][r][lane], dyp + static_cast<size_t>(W * i) * p.Ch, n);
            if (GATED) copy_raw2<PAIRS>(&sm.raw[buf][3][r][lane], zp + (W * i) * p.sz.t, n);
        }
        xp -= SSM_CK * p.sx.t;
        dtp -= SSM_CK * p.sdt.t;
        dyp -= static_cast<size_t>(SSM_CK) * p.Ch;
        if (GATED) zp -= SSM_CK * p.sz.t;
#pragma unroll
        for (int k = 0; k < K; k++)
            if (warp * K + k < p.N) copy_async<8>(shared_address(&sm.h0[buf][warp * K + k][lane]), kept + static_cast<size_t>(k) * p.Cpad);
        kept -= static_cast<size_t>(p.N) * p.Cpad;
        copies_commit();
#pragma unroll
        for (int i = 0; i < BI; i++) {
            const bool in = bn < p.N && bt + BSTEP * i < min(left, SSM_CK);
            rB[i] = in ? Bp[(BSTEP * i) * p.sB.t] : from_f32<T>(0.f);
            rC[i] = in ? Cp[(BSTEP * i) * p.sC.t] : from_f32<T>(0.f);
        }
        Bp -= SSM_CK * p.sB.t;
        Cp -= SSM_CK * p.sC.t;
    };
    fetch(t_end - t_last, (chunks - 1) & 1);
    for (int chunk = chunks - 1; chunk >= 0; chunk--) {
        const int tc = t_begin + chunk * SSM_CK, subs = ceil_div(min(SSM_CK, t_end - tc), BWD_ROWS), buf = chunk & 1;
        copies_wait<0>();
        // (the run behind this one has been read: its last barrier lies in front of everything that is written here)
#pragma unroll
        for (int i = 0; i < IT; i++) {
            const int r = warp + W * i;
            const float2 x = to_float2<T>(sm.raw[buf][0][r][lane]), dy = to_float2<T>(sm.raw[buf][2][r][lane]);
            f2 d = delta2(to_float2<T>(sm.raw[buf][1][r][lane]), bias, p.softplus), e = pack2(dy.x, dy.y);
            if (GATED) {
                const float2 z = to_float2<T>(sm.raw[buf][3][r][lane]);
                e = mul2(e, mul2(pack2(z.x, z.y), sigmoid2(pack2(z.x, z.y))));
            }
            if (tc + r >= t_end) d = 0;
            *reinterpret_cast<ulonglong2*>(&sm.dl[r][lane]) = make_ulonglong2(d, mul2(d, pack2(x.x, x.y)));
            *reinterpret_cast<f2*>(&sm.e[r][lane]) = e;
        }
#pragma unroll
        for (int i = 0; i < BI; i++) {
            const float bv = to_f32<T>(rB[i]), cv = to_f32<T>(rC[i]);
            if (bt + BSTEP * i < SSM_CK) sm.bc[bt + BSTEP * i][bn] = make_float4(bv, bv, cv, cv);
        }
        __syncthreads();
        if (chunk > 0) fetch(SSM_CK, buf ^ 1);
        // the states in front of every BWD_ROWS positions (each warp its own)
        if (subs > 1) {
            f2 s[K];
#pragma unroll
            for (int k = 0; k < K; k++) s[k] = *reinterpret_cast<const f2*>(&sm.h0[buf][warp * K + k][lane]);
#pragma unroll 1
            for (int sub = 1; sub < subs; sub++) {
#pragma unroll
                for (int r = 0; r < BWD_ROWS; r++) {
                    const int row = (sub - 1) * BWD_ROWS + r;
                    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sm.dl[row][lane]);
#pragma unroll
                    for (int k = 0; k < K; k++)
                        s[k] = fma2(decay2(v.x, rate[k]), s[k], mul2(v.y, *reinterpret_cast<const f2*>(&sm.bc[row][warp * K + k])));
                }
#pragma unroll
                for (int k = 0; k < K; k++) *reinterpret_cast<f2*>(&sm.h[sub - 1][warp * K + k][lane]) = s[k];
            }
        }
#pragma unroll 1
        for (int sub = subs - 1; sub >= 0; sub--) {
            const int q = sub * BWD_ROWS, turn = sub & 1;
            const float2* front = sub ? &sm.h[sub - 1][0][lane] : &sm.h0[buf][0][lane];
            f2 dl[BWD_ROWS], dx[BWD_ROWS], e[BWD_ROWS], sb[BWD_ROWS], su[BWD_ROWS];
            [[maybe_unused]] f2 y[BWD_ROWS];
#pragma unroll
            for (int r = 0; r < BWD_ROWS; r++) {
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
                if (!FULL && n >= p.N) break;           // (FULL: N = K W.  A branch here would keep the states' chains apart)
                f2 a[BWD_ROWS], u[BWD_ROWS], s = *reinterpret_cast<const f2*>(front + n * 32);
                float pc[BWD_ROWS], pb[BWD_ROWS];
#pragma unroll
                for (int r = 0; r < BWD_ROWS; r++) {
                    const ulonglong2 bc = *reinterpret_cast<const ulonglong2*>(&sm.bc[q + r][n]);
                    a[r] = decay2(dl[r], rate[k]);
                    u[r] = mul2(a[r], s);
                    s = fma2(dx[r], bc.x, u[r]);
                    if (GATED) y[r] = fma2(s, bc.y, y[r]);
                    const float2 c = unpack2(mul2(e[r], s));
                    pc[r] = c.x + c.y;
                }
                f2 g = G[k];
#pragma unroll
                for (int r = BWD_ROWS - 1; r >= 0; r--) {
                    const ulonglong2 bc = *reinterpret_cast<const ulonglong2*>(&sm.bc[q + r][n]);
                    g = fma2(bc.y, e[r], g);
                    sb[r] = fma2(g, bc.x, sb[r]);
                    const f2 w = mul2(g, u[r]);
                    su[r] = fma2(w, rate[k], su[r]);
                    dA[k] = fma2(dl[r], w, dA[k]);
                    const float2 c = unpack2(mul2(g, dx[r]));
                    pb[r] = c.x + c.y;
                    g = mul2(a[r], g);
                }
                G[k] = g;
                const float2 sums = butterfly<BWD_ROWS>(pb, pc, lane);
                if (lane % (32 / BWD_ROWS) == 0) sm.bcg[turn][lane / (32 / BWD_ROWS)][n] = sums;
            }
#pragma unroll
            for (int r = 0; r < BWD_ROWS; r++) {
                *reinterpret_cast<f2*>(&sm.red[turn][0][warp][r][lane]) = sb[r];
                *reinterpret_cast<f2*>(&sm.red[turn][1][warp][r][lane]) = su[r];
                if (GATED) *reinterpret_cast<f2*>(&sm.red[turn][2][warp][r][lane]) = y[r];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < SIT; i++) {
                const int r = warp + W * i, t = tc + q + r;
                if (t < t_end && (SIT * W == BWD_ROWS || r < BWD_ROWS)) {
                    f2 vs = 0, vu = 0, vy = 0;
#pragma unroll
                    for (int w = 0; w < W; w++) {
                        vs = add2(vs, *reinterpret_cast<const f2*>(&sm.red[turn][0][w][r][lane]));
                        vu = add2(vu, *reinterpret_cast<const f2*>(&sm.red[turn][1][w][r][lane]));
                        if (GATED) vy = add2(vy, *reinterpret_cast<const f2*>(&sm.red[turn][2][w][r][lane]));
                    }
                    const float2 xv = to_float2<T>(sm.raw[buf][0][q + r][lane]);
                    const f2 x = pack2(xv.x, xv.y), ev = *reinterpret_cast<const f2*>(&sm.e[q + r][lane]);
                    const f2 d = *reinterpret_cast<const f2*>(&sm.dl[q + r][lane]);
                    f2 dd = fma2(x, vs, mul2(splat2(0.69314718055994530942f), vu));      // (the rates are in units of log2)
                    if (p.softplus) {
                        const float2 raw = to_float2<T>(sm.raw[buf][1][q + r][lane]);
                        dd = mul2(dd, sigmoid2(add2(pack2(raw.x, raw.y), bias)));
                    }
                    dbias = add2(dbias, dd);
                    dskip = fma2(ev, x, dskip);
                    const size_t at = (row0 + t) * p.Ch + ch.c;
                    store_pair<PAIRS>(static_cast<T*>(p.ddt) + at, unpack2(dd), ch.n);
                    store_pair<PAIRS>(static_cast<T*>(p.dx) + at, unpack2(p.D ? fma2(d, vs, mul2(skip, ev)) : mul2(d, vs)), ch.n);
                    if (GATED) {
                        const float2 zv = to_float2<T>(sm.raw[buf][3][q + r][lane]), dy = to_float2<T>(sm.raw[buf][2][q + r][lane]);
                        if (p.D) vy = fma2(skip, x, vy);
                        const f2 z = pack2(zv.x, zv.y), sg = sigmoid2(z);        // silu' = sg (1 + z (1 - sg))
                        const f2 slope = mul2(sg, fma2(z, fma2(sg, splat2(-1.0f), splat2(1.0f)), splat2(1.0f)));
                        store_pair<PAIRS>(static_cast<T*>(p.dz) + at, unpack2(mul2(pack2(dy.x, dy.y), mul2(vy, slope))), ch.n);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < (BWD_ROWS + BSTEP - 1) / BSTEP; i++) {
                const int r = bt + BSTEP * i, t = tc + q + r;
                if (r < BWD_ROWS && t < t_end && bn < p.N)
                    p.bc_part[((static_cast<size_t>(blockIdx.x) * p.nb + bl) * p.S + t) * p.N + bn] = sm.bcg[turn][r][bn];
            }
        }
    }
    float* part = p.param_part + (static_cast<size_t>(b) * p.nseg + seg) * (p.N + 2) * p.Cpad + ch.cp;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int n = warp * K + k;
        if (n < p.N) *reinterpret_cast<f2*>(part + static_cast<size_t>(n) * p.Cpad) = dA[k];
    }
    __syncthreads();
    *reinterpret_cast<f2*>(&sm.red[0][0][warp][0][lane]) = dskip;
    *reinterpret_cast<f2*>(&sm.red[0][1][warp][0][lane]) = dbias;
    __syncthreads();
    if (warp < 2) {
        f2 v = 0;
#pragma unroll
        for (int w = 0; w < W; w++) v = add2(v, *reinterpret_cast<const f2*>(&sm.red[0][warp][w][0][lane]));
        *reinterpret_cast<f2*>(part + static_cast<size_t>(p.N + warp) * p.Cpad) = v;
    }
}

// dB, dC [Bt, S, G, N]: sums over the CTAs of a group, for the groups from g0 on.
template <typename T>
__global__ void __launch_bounds__(256) ssm_bc_sum_kernel(const float2* __restrict__ part, T* __restrict__ dB, T* __restrict__ dC, int tiles_g,
                                                         int G, int g0, int N, long long rows, long long row0) {
    grid_dep_wait();
    grid_dep_launch();
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x, per = rows * N;
    if (i >= per) return;
    const int g = g0 + blockIdx.y;
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
// Four states per warp and four warps: two CTAs fill an SM's registers.  Where the channels give at most one CTA to an SM, or there are
// more states, eight warps.  (With two states each, so one CTA of eight warps per SM, forward and backward of 4 x 4096 x 4096 take
// 2.65 against 2.27 ms, but those of 2 x 2048 x 4096 0.73 against 0.81 ms.)
bool ssm_bwd_wide(const SsmArgs& a) { return a.N > 16 || (a.N > 8 && static_cast<long long>(a.G) * a.tiles_g * a.Bt <= 148); }
void ssm_bwd_cut(SsmArgs& a) { ssm_cut(a, ssm_bwd_wide(a) ? 1 : 2); }

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
    constexpr size_t smem = sizeof(SsmBwdSmem<T, K, W>);
    static std::atomic<unsigned long long> done[6];
    const int v = (!a.pairs ? 0 : a.N == K * W ? 2 : 1) + (a.z ? 3 : 0);
    void (*const kerns[6])(SsmBwdArgs) = {ssm_bwd_kernel<T, K, W, false, false, false>, ssm_bwd_kernel<T, K, W, false, true, false>,
                                          ssm_bwd_kernel<T, K, W, false, true, true>,   ssm_bwd_kernel<T, K, W, true, false, false>,
                                          ssm_bwd_kernel<T, K, W, true, true, false>,   ssm_bwd_kernel<T, K, W, true, true, true>};
    auto kern = kerns[v];
    cudaError_t ce = ssm_allow_smem(kern, smem, done[v]);
    for (int b0 = 0; b0 < a.Bt && ce == cudaSuccess; b0 += w.nb) {
        a.b0 = b0;
        a.nb = a.Bt - b0 < w.nb ? a.Bt - b0 : w.nb;
        if (a.nseg > 1) ce = launch_plain(a.pairs ? ssm_back_state_kernel<T, K, W, true> : ssm_back_state_kernel<T, K, W, false>, dim3(tiles, a.nseg - 1, a.nb), dim3(32 * W), 0, st, a);
        if (ce == cudaSuccess) ce = launch_plain(kern, dim3(tiles, a.nseg, a.nb), dim3(32 * W), smem, st, a);
        const long long rows = static_cast<long long>(a.nb) * a.S;
        constexpr int MOST = 65535;             // places of a grid's second dimension
        for (int g0 = 0; g0 < a.G && ce == cudaSuccess; g0 += MOST)
            ce = launch_plain(ssm_bc_sum_kernel<T>, dim3(static_cast<unsigned>((rows * a.N + 255) / 256), a.G - g0 < MOST ? a.G - g0 : MOST), dim3(256), 0, st,
                              a.bc_part, static_cast<T*>(dB), static_cast<T*>(dC), a.tiles_g, a.G, g0, a.N, rows, static_cast<long long>(b0) * a.S);
    }
    return ce;
}
// (Three states per warp for 24 and six for 48: 901 and 1479 us for 2 x 2048 x 2048 positions and channels, bf16, forward included,
// against 1014 and 1836 with four and eight, which leave the last two warps without any.)
template <typename T>
cudaError_t launch_ssm_bwd_n(const SsmBwdArgs& a, const SsmBwdWs& w, void* dB, void* dC, cudaStream_t st) {
    if (a.N <= 4) return launch_ssm_bwd<T, 1, 4>(a, w, dB, dC, st);
    if (a.N <= 8) return launch_ssm_bwd<T, 2, 4>(a, w, dB, dC, st);
    if (a.N <= 16) return ssm_bwd_wide(a) ? launch_ssm_bwd<T, 2, 8>(a, w, dB, dC, st) : launch_ssm_bwd<T, 4, 4>(a, w, dB, dC, st);
    if (a.N <= 24) return launch_ssm_bwd<T, 3, 8>(a, w, dB, dC, st);
    if (a.N <= 32) return launch_ssm_bwd<T, 4, 8>(a, w, dB, dC, st);
    if (a.N <= 48) return launch_ssm_bwd<T, 6, 8>(a, w, dB, dC, st);
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
    ssm_bwd_cut(a);
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
        if (!aligned(q, es)) return MLSTM_E_ALIGN;
    for (const float* q : {A, D, dt_bias, static_cast<const float*>(dA), static_cast<const float*>(dD), static_cast<const float*>(d_dt_bias)})
        if (!aligned(q, 4)) return MLSTM_E_ALIGN;
    if (!aligned(checkpoints, 8)) return MLSTM_E_ALIGN;
    ssm_bwd_cut(a);
    const SsmBwdWs w = ssm_bwd_carve(workspace, a);
    if (!workspace || workspace_bytes < w.bytes || !aligned(workspace, 16)) return MLSTM_E_WORKSPACE;
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
