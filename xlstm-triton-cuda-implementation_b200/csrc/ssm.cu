// Selective state space scan: forward over prompts, and the step for a few new tokens (ssm_common.cuh has the formulas and the
// layout of the work).
#include "ssm_common.cuh"

namespace mlstm {
namespace {

// positions staged in shared memory at a time (with eight warps half as many: what they hand over fits the 48 KB of a plain launch)
template <int W>
constexpr int SSM_TILE = W == 8 ? 8 : 16;

struct SsmFwdArgs : SsmArgs {
    const float* initial;           // [Bt, Ch, N] or nullptr
    void* y;                        // [Bt, S, Ch]
    float* state_out;               // [Bt, Ch, N] or nullptr
};

template <int K, int W>
struct SsmFwdSmem {
    float4 dl[SSM_TILE<W>][32];                    // delta, delta x of the lane's two channels
    float4 bc[SSM_TILE<W>][K * W];                 // B, B, C, C
    float2 y[W][SSM_TILE<W>][32];                  // every warp's part of the output
};

// One CTA: 64 channels, one segment.  OUT: outputs (and the states that are kept); else only what the segment adds to the state.
template <typename T, int K, int W, bool OUT>
__global__ void __launch_bounds__(32 * W) ssm_fwd_kernel(const SsmFwdArgs p) {
    constexpr int TILE = SSM_TILE<W>, NP = K * W, IT = TILE / W, BI = (TILE * NP + 32 * W - 1) / (32 * W);
    __shared__ SsmFwdSmem<K, W> sm;
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.z, seg = blockIdx.y;
    const SsmTile ch = ssm_tile(p, blockIdx.x, lane);
    const int t_begin = seg * p.seglen, t_end = min(p.S, t_begin + p.seglen);
    const bool pairs = p.pairs != 0;

    const T* xp = static_cast<const T*>(p.x) + b * p.sx.b + ch.c;
    const T* dtp = static_cast<const T*>(p.dt) + b * p.sdt.b + ch.c;
    const T* zp = p.z ? static_cast<const T*>(p.z) + b * p.sz.b + ch.c : nullptr;
    const T* Bp = static_cast<const T*>(p.B) + b * p.sB.b + static_cast<long long>(ch.g) * p.N;
    const T* Cp = static_cast<const T*>(p.C) + b * p.sC.b + static_cast<long long>(ch.g) * p.N;

    float2 bias = make_float2(0.f, 0.f), skip = make_float2(0.f, 0.f);
    if (p.bias) {
        if (ch.n > 0) bias.x = p.bias[ch.c];
        if (ch.n > 1) bias.y = p.bias[ch.c + 1];
    }
    if (OUT && p.D) {
        if (ch.n > 0) skip.x = p.D[ch.c];
        if (ch.n > 1) skip.y = p.D[ch.c + 1];
    }
    f2 rate[K], h[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int n = warp * K + k;
        float r0 = 0.f, r1 = 0.f, h0 = 0.f, h1 = 0.f;
        if (n < p.N) {
            const size_t at = static_cast<size_t>(ch.c) * p.N + n;
            if (ch.n > 0) r0 = decay_rate(p.A[at]);
            if (ch.n > 1) r1 = decay_rate(p.A[at + p.N]);
            // (cut into segments: the first pass keeps the state carried in for the second one, whose last CTAs may
            // overwrite it, as state_out may be the same memory)
            if (p.initial && (OUT ? p.nseg == 1 : seg == 0)) {
                const size_t hb = static_cast<size_t>(b) * p.Ch * p.N + at;
                if (ch.n > 0) h0 = p.initial[hb];
                if (ch.n > 1) h1 = p.initial[hb + p.N];
            }
        }
        rate[k] = pack2(r0, r1);
        h[k] = pack2(h0, h1);
    }
    if (!OUT && seg == 0) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int n = warp * K + k;
            if (n < p.N)
                *reinterpret_cast<f2*>(p.seg_end + ((static_cast<size_t>(b) * p.nseg + p.nseg - 1) * p.N + n) * p.Cpad + ch.cp) = h[k];
            h[k] = 0;
        }
    }
    if (OUT && p.nseg > 1) {      // the state in front of this segment: what was carried in, and the segments before this one
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int n = warp * K + k;
            if (n < p.N)
                h[k] = *reinterpret_cast<const f2*>(p.seg_end + ((static_cast<size_t>(b) * p.nseg + p.nseg - 1) * p.N + n) * p.Cpad + ch.cp);
        }
        for (int j = 0; j < seg; j++) {
            const size_t sj = (static_cast<size_t>(b) * p.nseg + j);
            const f2 sum = *reinterpret_cast<const f2*>(p.seg_sum + sj * p.Cpad + ch.cp);
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int n = warp * K + k;
                if (n < p.N)
                    h[k] = fma2(exp2_2(mul2(sum, rate[k])), h[k],
                                *reinterpret_cast<const f2*>(p.seg_end + (sj * p.N + n) * p.Cpad + ch.cp));
            }
        }
    }

    Raw2<T> rx[IT], rdt[IT], rz[IT];
    T rB[BI], rC[BI];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int i = 0; i < IT; i++) {
            const int t = t0 + warp + W * i, n = t < t_end ? ch.n : 0;
            rx[i] = load_raw2<T>(xp + t * p.sx.t, pairs, n);
            rdt[i] = load_raw2<T>(dtp + t * p.sdt.t, pairs, n);
            if (OUT && zp) rz[i] = load_raw2<T>(zp + t * p.sz.t, pairs, n);
        }
#pragma unroll
        for (int i = 0; i < BI; i++) {
            const int e = threadIdx.x + i * 32 * W, t = t0 + e / NP, n = e % NP;
            const bool in = e < TILE * NP && n < p.N && t < t_end;
            rB[i] = in ? Bp[t * p.sB.t + n] : from_f32<T>(0.f);
            if (OUT) rC[i] = in ? Cp[t * p.sC.t + n] : from_f32<T>(0.f);
        }
    };
    [[maybe_unused]] f2 sum = 0;
    fetch(t_begin);
    for (int t0 = t_begin; t0 < t_end; t0 += TILE) {
        [[maybe_unused]] float2 x[IT], z[IT];
#pragma unroll
        for (int i = 0; i < IT; i++) {
            const int r = warp + W * i;
            x[i] = to_float2<T>(rx[i]);
            if (OUT && zp) z[i] = to_float2<T>(rz[i]);
            float2 d = to_float2<T>(rdt[i]);
            d.x += bias.x;
            d.y += bias.y;
            if (p.softplus) d = make_float2(softplus_f(d.x), softplus_f(d.y));
            if (t0 + r >= t_end) d = make_float2(0.f, 0.f);     // a step of 0 leaves the state
            sm.dl[r][lane] = make_float4(d.x, d.y, d.x * x[i].x, d.y * x[i].y);
        }
#pragma unroll
        for (int i = 0; i < BI; i++) {
            const int e = threadIdx.x + i * 32 * W;
            const float bv = to_f32<T>(rB[i]), cv = OUT ? to_f32<T>(rC[i]) : 0.f;
            if (e < TILE * NP) sm.bc[e / NP][e % NP] = make_float4(bv, bv, cv, cv);
        }
        __syncthreads();
        if (t0 + TILE < t_end) fetch(t0 + TILE);
        if (OUT && p.ckpt && t0 % SSM_CK == 0) {
            const size_t row = static_cast<size_t>(b) * ceil_div(p.S, SSM_CK) + t0 / SSM_CK;
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int n = warp * K + k;
                if (n < p.N) *reinterpret_cast<f2*>(p.ckpt + (row * p.N + n) * p.Cpad + ch.cp) = h[k];
            }
        }
#pragma unroll 1
        for (int half = 0; half < TILE; half += SSM_ROWS) {
            f2 dl[SSM_ROWS], dx[SSM_ROWS];
            [[maybe_unused]] f2 y[SSM_ROWS];
#pragma unroll
            for (int r = 0; r < SSM_ROWS; r++) {
                const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sm.dl[half + r][lane]);
                dl[r] = v.x;
                dx[r] = v.y;
                if (OUT) y[r] = 0;
                else if (warp == 0) sum = add2(sum, v.x);
            }
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (warp * K + k >= p.N) break;         // (the same for the whole warp)
                f2 s = h[k];
#pragma unroll
                for (int r = 0; r < SSM_ROWS; r++) {
                    const ulonglong2 bc = *reinterpret_cast<const ulonglong2*>(&sm.bc[half + r][warp * K + k]);
                    s = fma2(exp2_2(mul2(dl[r], rate[k])), s, mul2(dx[r], bc.x));
                    if (OUT) y[r] = fma2(s, bc.y, y[r]);
                }
                h[k] = s;
            }
            if (OUT) {
#pragma unroll
                for (int r = 0; r < SSM_ROWS; r++) *reinterpret_cast<f2*>(&sm.y[warp][half + r][lane]) = y[r];
            }
        }
        __syncthreads();
        if (OUT) {
#pragma unroll
            for (int i = 0; i < IT; i++) {
                const int r = warp + W * i;
                if (t0 + r < t_end) {
                    float2 v = make_float2(skip.x * x[i].x, skip.y * x[i].y);
                    if (!p.D) v = make_float2(0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < W; w++) {
                        const float2 part = sm.y[w][r][lane];
                        v.x += part.x;
                        v.y += part.y;
                    }
                    if (zp) v = make_float2(v.x * silu_f(z[i].x), v.y * silu_f(z[i].y));
                    store_pair<T>(static_cast<T*>(p.y) + (static_cast<size_t>(b) * p.S + t0 + r) * p.Ch + ch.c, v, pairs, ch.n);
                }
            }
        }
    }
    if (!OUT) {
        const size_t sj = static_cast<size_t>(b) * p.nseg + seg;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int n = warp * K + k;
            if (n < p.N) *reinterpret_cast<f2*>(p.seg_end + (sj * p.N + n) * p.Cpad + ch.cp) = h[k];
        }
        if (warp == 0) *reinterpret_cast<f2*>(p.seg_sum + sj * p.Cpad + ch.cp) = sum;
    } else if (p.state_out && seg == p.nseg - 1) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int n = warp * K + k;
            const float2 v = unpack2(h[k]);
            const size_t at = (static_cast<size_t>(b) * p.Ch + ch.c) * p.N + n;
            if (n < p.N) {
                if (ch.n > 0) p.state_out[at] = v.x;
                if (ch.n > 1) p.state_out[at + p.N] = v.y;
            }
        }
    }
}

template <typename T, int K, int W>
cudaError_t launch_ssm_fwd(const SsmFwdArgs& a, cudaStream_t st) {
    const unsigned tiles = static_cast<unsigned>(a.G * a.tiles_g);
    if (a.nseg > 1) {
        const cudaError_t ce = launch_plain(ssm_fwd_kernel<T, K, W, false>, dim3(tiles, a.nseg - 1, a.Bt), dim3(32 * W), 0, st, a);
        if (ce != cudaSuccess) return ce;
    }
    return launch_plain(ssm_fwd_kernel<T, K, W, true>, dim3(tiles, a.nseg, a.Bt), dim3(32 * W), 0, st, a);
}
template <typename T>
cudaError_t launch_ssm_fwd_n(const SsmFwdArgs& a, cudaStream_t st) {
    if (a.N <= 4) return launch_ssm_fwd<T, 1, 4>(a, st);
    if (a.N <= 8) return launch_ssm_fwd<T, 2, 4>(a, st);
    if (a.N <= 16) return launch_ssm_fwd<T, 4, 4>(a, st);
    if (a.N <= 32) return launch_ssm_fwd<T, 8, 4>(a, st);
    return launch_ssm_fwd<T, 8, 8>(a, st);
}

// ---------------------------------------------------------------------------------------------- a few new tokens
constexpr int STEP_TOKENS = 8;
constexpr int STEP_THREADS = 128;

struct SsmStepArgs : SsmArgs {
    const float* initial;
    void* y;
    float* state_out;
    int lanes;                       // lanes per channel (a power of two), four states each
    int vec;                         // states can be accessed four at a time
};

template <typename T>
__global__ void __launch_bounds__(STEP_THREADS) ssm_step_kernel(const SsmStepArgs p) {
    grid_dep_wait();
    grid_dep_launch();
    const int L = p.lanes, per = STEP_THREADS / L, b = blockIdx.y;
    const int sub = threadIdx.x & (L - 1), c = blockIdx.x * per + static_cast<int>(threadIdx.x) / L, n0 = sub * 4;
    const bool on = c < p.Ch;
    const int cc = on ? c : 0, nn = on ? max(0, min(4, p.N - n0)) : 0, g = cc / p.P;
    float h[4] = {0.f, 0.f, 0.f, 0.f}, rate[4] = {0.f, 0.f, 0.f, 0.f};
    const size_t at = static_cast<size_t>(cc) * p.N + n0, hb = static_cast<size_t>(b) * p.Ch * p.N + at;
    if (p.vec && nn == 4) {
        const float4 r = *reinterpret_cast<const float4*>(p.A + at);
        rate[0] = r.x; rate[1] = r.y; rate[2] = r.z; rate[3] = r.w;
        if (p.initial) {
            const float4 v = *reinterpret_cast<const float4*>(p.initial + hb);
            h[0] = v.x; h[1] = v.y; h[2] = v.z; h[3] = v.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (j < nn) {
                rate[j] = p.A[at + j];
                if (p.initial) h[j] = p.initial[hb + j];
            }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) rate[j] = decay_rate(rate[j]);
    const float bias = p.bias ? p.bias[cc] : 0.f, skip = p.D ? p.D[cc] : 0.f;
    for (int t = 0; t < p.S; t++) {
        const float x = to_f32<T>(static_cast<const T*>(p.x)[b * p.sx.b + t * p.sx.t + cc]);
        float d = to_f32<T>(static_cast<const T*>(p.dt)[b * p.sdt.b + t * p.sdt.t + cc]) + bias;
        if (p.softplus) d = softplus_f(d);
        const float dx = d * x;
        const T* Bp = static_cast<const T*>(p.B) + b * p.sB.b + t * p.sB.t + static_cast<long long>(g) * p.N + n0;
        const T* Cp = static_cast<const T*>(p.C) + b * p.sC.b + t * p.sC.t + static_cast<long long>(g) * p.N + n0;
        float y = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j < nn) {
                h[j] = fmaf(fast_exp2(d * rate[j]), h[j], dx * to_f32<T>(Bp[j]));
                y = fmaf(h[j], to_f32<T>(Cp[j]), y);
            }
        }
        for (int o = L >> 1; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
        if (on && sub == 0) {
            if (p.D) y = fmaf(skip, x, y);
            if (p.z) y *= silu_f(to_f32<T>(static_cast<const T*>(p.z)[b * p.sz.b + t * p.sz.t + cc]));
            static_cast<T*>(p.y)[(static_cast<size_t>(b) * p.S + t) * p.Ch + c] = from_f32<T>(y);
        }
    }
    if (p.state_out) {
        if (p.vec && nn == 4) *reinterpret_cast<float4*>(p.state_out + hb) = make_float4(h[0], h[1], h[2], h[3]);
        else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (j < nn) p.state_out[hb + j] = h[j];
        }
    }
}

template <typename T>
cudaError_t launch_ssm_step(const SsmStepArgs& a, cudaStream_t st) {
    const int per = STEP_THREADS / a.lanes;
    return launch_plain(ssm_step_kernel<T>, dim3(ceil_div(a.Ch, per), a.Bt), dim3(STEP_THREADS), 0, st, a);
}

// How many segments the positions are cut into: one where the channels alone fill the chip.  Cutting costs a second pass over
// the exponentials (the state that a segment adds, then its outputs), so a cut in two gains nothing.
int ssm_segments(const SsmArgs& a, int ctas_per_sm) {
    const long long ctas = static_cast<long long>(a.G) * a.tiles_g * a.Bt, want = 148LL * ctas_per_sm;
    const int most = ceil_div(a.S, 2 * SSM_CK) < 64 ? ceil_div(a.S, 2 * SSM_CK) : 64;
    const long long n = ctas > 0 ? want / ctas : 1;
    return n < 3 ? 1 : static_cast<int>(n < most ? n : most);
}

}  // namespace

int ssm_fill(SsmArgs& a, const void* x, const void* dt, const float* A, const void* B, const void* C, const float* D, const void* z,
             const float* bias, const long long* strides, int Bt, int S, int Ch, int G, int N, int dtype, int softplus) {
    if (!x || !dt || !A || !B || !C) return MLSTM_E_ARG;
    if (Bt <= 0 || S <= 0 || Ch <= 0 || G <= 0 || N <= 0) return MLSTM_E_ARG;
    if (dtype != MLSTM_DT_F32 && dtype != MLSTM_DT_F16 && dtype != MLSTM_DT_BF16) return MLSTM_E_ARG;
    if (Ch % G != 0 || N > SSM_MAX_N || Bt > 65535) return MLSTM_E_SHAPE;
    if (S > 0x7fffffff - 2 * SSM_CK || Ch > (1 << 24)) return MLSTM_E_SHAPE;
    a = SsmArgs{};
    a.x = x; a.dt = dt; a.z = z; a.B = B; a.C = C; a.A = A; a.D = D; a.bias = bias;
    a.Bt = Bt; a.S = S; a.Ch = Ch; a.G = G; a.P = Ch / G; a.N = N;
    a.tiles_g = ceil_div(a.P, SSM_CH);
    a.Cpad = G * a.tiles_g * SSM_CH;
    a.softplus = softplus;
    const long long row = Ch, vec = static_cast<long long>(G) * N;
    const long long plain[10] = {row * S, row, row * S, row, vec * S, vec, vec * S, vec, row * S, row};
    const long long* s = strides ? strides : plain;
    for (int k = 0; k < 10; k++)
        if (s[k] < 0) return MLSTM_E_ARG;
    a.sx = {s[0], s[1]};
    a.sdt = {s[2], s[3]};
    a.sB = {s[4], s[5]};
    a.sC = {s[6], s[7]};
    a.sz = {s[8], s[9]};
    return MLSTM_OK;
}

namespace {

struct SsmWs {
    float *seg_end, *seg_sum;
    size_t bytes;
};
SsmWs ssm_carve(void* ws, const SsmArgs& a) {
    SsmWs w{};
    if (a.nseg <= 1) return w;
    const size_t segs = static_cast<size_t>(a.Bt) * a.nseg, end = segs * a.N * a.Cpad * 4, sum = segs * a.Cpad * 4;
    w.bytes = end + sum;
    if (ws) {
        w.seg_end = static_cast<float*>(ws);
        w.seg_sum = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + end);
    }
    return w;
}

}  // namespace

void ssm_cut(SsmArgs& a, int ctas_per_sm) {
    a.nseg = ssm_segments(a, ctas_per_sm);
    a.seglen = ceil_div(ceil_div(a.S, a.nseg), SSM_CK) * SSM_CK;
    a.nseg = ceil_div(a.S, a.seglen);
}

// Whether channels can be accessed two at a time.
bool ssm_pairs(const SsmArgs& a, int es, std::initializer_list<const void*> more) {
    if ((a.Ch & 1) || (a.G > 1 && (a.P & 1))) return false;
    if ((a.sx.b | a.sx.t | a.sdt.b | a.sdt.t) & 1) return false;
    if (a.z && ((a.sz.b | a.sz.t) & 1)) return false;
    uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.dt) | reinterpret_cast<uintptr_t>(a.z);
    for (const void* q : more) bits |= reinterpret_cast<uintptr_t>(q);
    return (bits & (2 * es - 1)) == 0;
}

namespace {

constexpr int SSM_FWD_CTAS = 4;     // CTAs of 4 warps that an SM is filled with

}  // namespace
}  // namespace mlstm

using namespace mlstm;

extern "C" {

int mlstm_ssm_step_max_tokens(void) { return STEP_TOKENS; }

size_t mlstm_ssm_checkpoint_floats(int B, int S, int C, int G, int N) {
    if (B <= 0 || S <= 0 || C <= 0 || G <= 0 || N <= 0 || C % G != 0 || N > SSM_MAX_N) return 0;
    return static_cast<size_t>(B) * ceil_div(S, SSM_CK) * N * G * ceil_div(C / G, SSM_CH) * SSM_CH;
}

size_t mlstm_ssm_fwd_workspace(int B, int S, int C, int G, int N) {
    SsmArgs a;
    const void* any = reinterpret_cast<const void*>(16);
    if (ssm_fill(a, any, any, static_cast<const float*>(any), any, any, nullptr, nullptr, nullptr, nullptr, B, S, C, G, N,
                 MLSTM_DT_F32, 0) != MLSTM_OK)
        return 0;
    ssm_cut(a, SSM_FWD_CTAS);
    return ssm_carve(nullptr, a).bytes;
}

int mlstm_ssm_fwd(const void* x, const void* dt, const float* A, const void* Bv, const void* Cv, const float* D, const void* z,
                  const float* dt_bias, const float* initial, const long long* strides, void* y, float* state_out,
                  float* checkpoints, void* workspace, size_t workspace_bytes, int B, int S, int C, int G, int N, int dtype,
                  int softplus, void* stream) {
    SsmArgs base;
    const int rc = ssm_fill(base, x, dt, A, Bv, Cv, D, z, dt_bias, strides, B, S, C, G, N, dtype, softplus);
    if (rc != MLSTM_OK) return rc;
    if (!y) return MLSTM_E_ARG;
    const int es = dtype == MLSTM_DT_F32 ? 4 : 2;
    for (const void* q : {x, dt, Bv, Cv, z, static_cast<const void*>(y)})
        if (!ssm_aligned(q, es)) return MLSTM_E_ALIGN;
    for (const void* q : {static_cast<const void*>(A), static_cast<const void*>(D), static_cast<const void*>(dt_bias),
                          static_cast<const void*>(initial), static_cast<const void*>(state_out)})
        if (!ssm_aligned(q, 4)) return MLSTM_E_ALIGN;
    if (!ssm_aligned(checkpoints, 8)) return MLSTM_E_ALIGN;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t ce;
    if (S <= STEP_TOKENS && !checkpoints) {
        SsmStepArgs a;
        static_cast<SsmArgs&>(a) = base;
        a.initial = initial; a.y = y; a.state_out = state_out;
        a.lanes = 1;
        while (a.lanes * 4 < N) a.lanes *= 2;
        a.vec = N % 4 == 0 && ssm_aligned(A, 16) && ssm_aligned(initial, 16) && ssm_aligned(state_out, 16);
        ce = dtype == MLSTM_DT_F32 ? launch_ssm_step<float>(a, st)
             : dtype == MLSTM_DT_F16 ? launch_ssm_step<__half>(a, st) : launch_ssm_step<__nv_bfloat16>(a, st);
    } else {
        SsmFwdArgs a;
        static_cast<SsmArgs&>(a) = base;
        ssm_cut(a, SSM_FWD_CTAS);
        const SsmWs w = ssm_carve(workspace, a);
        if (w.bytes && (!workspace || workspace_bytes < w.bytes || !ssm_aligned(workspace, 16))) return MLSTM_E_WORKSPACE;
        a.seg_end = w.seg_end; a.seg_sum = w.seg_sum;
        a.ckpt = checkpoints; a.initial = initial; a.y = y; a.state_out = state_out;
        a.pairs = ssm_pairs(a, es, {y});
        ce = dtype == MLSTM_DT_F32 ? launch_ssm_fwd_n<float>(a, st)
             : dtype == MLSTM_DT_F16 ? launch_ssm_fwd_n<__half>(a, st) : launch_ssm_fwd_n<__nv_bfloat16>(a, st);
    }
    if (ce != cudaSuccess) cudaGetLastError();
    return ce == cudaSuccess ? MLSTM_OK : note_cuda_error(ce, "launch of the state space scan");
}

}  // extern "C"
