// Selective state space scan: forward over prompts, and the step for a few new tokens (ssm_common.cuh has the formulas and the
// layout of the work).
//
// Forward.  Four warps of a CTA do the recurrence, K of the N states each, eight positions of their operands in registers at a time;
// four more prepare what these read (delta, delta x, B, C) and finish what they leave (the sum over the warps' states, D x, the
// gate).  The two halves work on different tiles of 16 positions at the same time, two buffers each way, handed over by named
// barriers.  (All eight warps doing both, one tile after the other: 0.86 against 0.54 ms for 4 x 4096 x 4096, 16 states.)
// Bound by the exponentials: one per state and position on the hardware's special function unit, 16 a cycle and SM, and four for
// every softplus and gate; 1.1e9 of them take 0.24 ms.  Measured, bf16, 16 states: 4 x 4096 positions x 4096 channels 0.50 ms (256
// CTAs on 148 SMs: 86 % of the slots filled; the unit 63 to 76 % busy while they are, with 8 instructions per state and position
// in the other slots), 1 x 16384 x 1024 0.21 ms in 18 segments (two passes).  A polynomial for part of the exponentials would
// take as many issue slots as it frees: not built.
#include "ssm_common.cuh"
#include "vec_cvt.cuh"

namespace mlstm {
namespace {

constexpr int SSM_TILE = 16;        // positions handed over at a time

struct SsmFwdArgs : SsmArgs {
    const float* initial;           // [Bt, Ch, N] or nullptr
    void* y;                        // [Bt, S, Ch]
    float* state_out;               // [Bt, Ch, N] or nullptr
};

template <int K>
struct SsmFwdSmem {
    float4 dl[2][SSM_TILE][32];                         // delta, delta x of the lane's two channels
    float4 bc[2][SSM_TILE][K * SSM_WARPS];              // B, B, C, C
    float2 y[2][SSM_WARPS][SSM_TILE][32];               // every warp's part of the output
};
// barriers, one for each buffer
enum : int { BAR_FULL = 1, BAR_EMPTY = 3, BAR_Y_FULL = 5, BAR_Y_EMPTY = 7 };

// One CTA: 64 channels, one segment.  OUT: outputs (and the states that are kept); else only what the segment adds to the state.
// Tile i uses buffer i & 1 of everything.  A buffer's first use waits for nothing, and what the last two uses leave is not
// announced, so every barrier is met exactly as often by either half.
template <typename T, int K, bool OUT, bool PAIRS, bool FULL>
__global__ void __launch_bounds__(SSM_THREADS, 2) ssm_fwd_kernel(const SsmFwdArgs p) {
    constexpr int TILE = SSM_TILE, W = SSM_WARPS, NP = K * W;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    SsmFwdSmem<K>& sm = *reinterpret_cast<SsmFwdSmem<K>*>(smem_raw);
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, b = blockIdx.z, seg = blockIdx.y;
    const SsmTile ch = ssm_tile(p, blockIdx.x, lane);
    const int t_begin = seg * p.seglen, t_end = min(p.S, t_begin + p.seglen), tiles = ceil_div(t_end - t_begin, TILE);

    if (threadIdx.x >= 32 * W) {
        constexpr int AW = SSM_AIDES, AT = 32 * AW, IT = TILE / AW, BSTEP = AT / NP, BI = (TILE + BSTEP - 1) / BSTEP;
        static_assert(TILE % AW == 0 && NP <= AT && BI * BSTEP >= TILE, "every value of a tile has a thread");
        const bool gated = OUT && p.z;
        const int tid = threadIdx.x - 32 * W, warp = tid >> 5;
        // rows of this thread: t0 + warp + AW i; positions and state of its B, C: t0 + bt + BSTEP i, bn
        const T* xp = static_cast<const T*>(p.x) + b * p.sx.b + (t_begin + warp) * p.sx.t + ch.c;
        const T* dtp = static_cast<const T*>(p.dt) + b * p.sdt.b + (t_begin + warp) * p.sdt.t + ch.c;
        const T* zp = gated ? static_cast<const T*>(p.z) + b * p.sz.b + (t_begin + warp) * p.sz.t + ch.c : nullptr;
        T* yp = OUT ? static_cast<T*>(p.y) + (static_cast<size_t>(b) * p.S + t_begin + warp) * p.Ch + ch.c : nullptr;
        const int bt = tid < NP * BSTEP ? tid / NP : TILE, bn = tid % NP;      // (TILE: a thread with none)
        const T* Bp = static_cast<const T*>(p.B) + b * p.sB.b + (t_begin + bt) * p.sB.t + static_cast<long long>(ch.g) * p.N + bn;
        const T* Cp = static_cast<const T*>(p.C) + b * p.sC.b + (t_begin + bt) * p.sC.t + static_cast<long long>(ch.g) * p.N + bn;
        const f2 bias = param2(p.bias, ch.c, ch.n), skip = OUT ? param2(p.D, ch.c, ch.n) : 0;
        Raw2<T> rx[IT], rdt[IT], rz[IT];
        T rB[BI], rC[BI];
        auto fetch = [&](int left) {            // left: positions of the segment from the tile on
#pragma unroll
            for (int i = 0; i < IT; i++) {
                const int n = warp + AW * i < left ? ch.n : 0;
                rx[i] = load_raw2<PAIRS>(xp + (AW * i) * p.sx.t, n);
                rdt[i] = load_raw2<PAIRS>(dtp + (AW * i) * p.sdt.t, n);
                if (gated) rz[i] = load_raw2<PAIRS>(zp + (AW * i) * p.sz.t, n);
            }
            xp += TILE * p.sx.t;
            dtp += TILE * p.sdt.t;
            if (gated) zp += TILE * p.sz.t;
#pragma unroll
            for (int i = 0; i < BI; i++) {
                const bool in = bn < p.N && bt + BSTEP * i < min(left, TILE);
                rB[i] = in ? Bp[(BSTEP * i) * p.sB.t] : from_f32<T>(0.f);
                if (OUT) rC[i] = in ? Cp[(BSTEP * i) * p.sC.t] : from_f32<T>(0.f);
            }
            Bp += TILE * p.sB.t;
            Cp += TILE * p.sC.t;
        };
        f2 part[IT], gate[IT], next_part[IT], next_gate[IT];     // D x and silu(z) of the positions that this thread finishes
        auto stage = [&](int tile) {                             // (the tile has been fetched)
            const int buf = tile & 1, left = t_end - t_begin - tile * TILE;
            if (tile >= 2) half_sync<SSM_THREADS>(BAR_EMPTY + buf);
#pragma unroll
            for (int i = 0; i < IT; i++) {
                const int r = warp + AW * i;
                const float2 x = to_float2<T>(rx[i]);
                f2 d = delta2(to_float2<T>(rdt[i]), bias, p.softplus);
                if (r >= left) d = 0;           // a step of 0 leaves the state
                const f2 xv = pack2(x.x, x.y);
                *reinterpret_cast<ulonglong2*>(&sm.dl[buf][r][lane]) = make_ulonglong2(d, mul2(d, xv));
                if (OUT) next_part[i] = p.D ? mul2(skip, xv) : 0;
                if (gated) {
                    const float2 z = to_float2<T>(rz[i]);
                    next_gate[i] = mul2(pack2(z.x, z.y), sigmoid2(pack2(z.x, z.y)));
                }
            }
#pragma unroll
            for (int i = 0; i < BI; i++) {
                const float bv = to_f32<T>(rB[i]), cv = OUT ? to_f32<T>(rC[i]) : 0.f;
                if (bt + BSTEP * i < TILE) sm.bc[buf][bt + BSTEP * i][bn] = make_float4(bv, bv, cv, cv);
            }
            half_arrive<SSM_THREADS>(BAR_FULL + buf);
            if (left > TILE) fetch(left - TILE);
        };
        fetch(t_end - t_begin);
        stage(0);
        for (int tile = 0; tile < tiles; tile++) {
            if (OUT) {
#pragma unroll
                for (int i = 0; i < IT; i++) {
                    part[i] = next_part[i];
                    if (gated) gate[i] = next_gate[i];
                }
            }
            if (tile + 1 < tiles) stage(tile + 1);
            if (OUT) {
                const int buf = tile & 1, left = t_end - t_begin - tile * TILE;
                half_sync<SSM_THREADS>(BAR_Y_FULL + buf);
#pragma unroll
                for (int i = 0; i < IT; i++) {
                    const int r = warp + AW * i;
                    f2 v = part[i];
#pragma unroll
                    for (int w = 0; w < W; w++) v = add2(v, *reinterpret_cast<const f2*>(&sm.y[buf][w][r][lane]));
                    if (gated) v = mul2(v, gate[i]);
                    if (r < left) store_pair<PAIRS>(yp + static_cast<size_t>(AW * i) * p.Ch, unpack2(v), ch.n);
                }
                yp += static_cast<size_t>(TILE) * p.Ch;
                if (tile + 2 < tiles) half_arrive<SSM_THREADS>(BAR_Y_EMPTY + buf);
            }
        }
        return;
    }

    const int warp = threadIdx.x >> 5;
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
    auto seg_state = [&](int j, int n) { return p.seg_end + ((static_cast<size_t>(b) * p.nseg + j) * p.N + n) * p.Cpad + ch.cp; };
    if (!OUT && seg == 0) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int n = warp * K + k;
            if (n < p.N) *reinterpret_cast<f2*>(seg_state(p.nseg - 1, n)) = h[k];
            h[k] = 0;
        }
    }
    if (OUT && p.nseg > 1) {      // the state in front of this segment: what was carried in, and the segments before this one
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int n = warp * K + k;
            if (n < p.N) h[k] = *reinterpret_cast<const f2*>(seg_state(p.nseg - 1, n));
        }
        for (int j = 0; j < seg; j++) {
            const f2 sum = *reinterpret_cast<const f2*>(p.seg_sum + (static_cast<size_t>(b) * p.nseg + j) * p.Cpad + ch.cp);
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int n = warp * K + k;
                if (n < p.N) h[k] = carry2(sum, rate[k], h[k], *reinterpret_cast<const f2*>(seg_state(j, n)));
            }
        }
    }
    [[maybe_unused]] f2 sum = 0;
    for (int tile = 0; tile < tiles; tile++) {
        const int buf = tile & 1;
        if (OUT && p.ckpt && tile % (SSM_CK / TILE) == 0) {
            const size_t row = static_cast<size_t>(b) * ceil_div(p.S, SSM_CK) + (t_begin + tile * TILE) / SSM_CK;
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int n = warp * K + k;
                if (n < p.N) *reinterpret_cast<f2*>(p.ckpt + (row * p.N + n) * p.Cpad + ch.cp) = h[k];
            }
        }
        half_sync<SSM_THREADS>(BAR_FULL + buf);
        if (OUT && tile >= 2) half_sync<SSM_THREADS>(BAR_Y_EMPTY + buf);
#pragma unroll 1
        for (int half = 0; half < TILE; half += SSM_ROWS) {
            f2 dl[SSM_ROWS], dx[SSM_ROWS];
            [[maybe_unused]] f2 y[SSM_ROWS];
#pragma unroll
            for (int r = 0; r < SSM_ROWS; r++) {
                const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sm.dl[buf][half + r][lane]);
                dl[r] = v.x;
                dx[r] = v.y;
                if (OUT) y[r] = 0;
                else if (warp == 0) sum = add2(sum, v.x);
            }
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (!FULL && warp * K + k >= p.N) break;        // (FULL: N = 4 K.  A branch here would keep the states' chains apart)
                f2 s = h[k];
#pragma unroll
                for (int r = 0; r < SSM_ROWS; r++) {
                    const ulonglong2 bc = *reinterpret_cast<const ulonglong2*>(&sm.bc[buf][half + r][warp * K + k]);
                    s = fma2(decay2(dl[r], rate[k]), s, mul2(dx[r], bc.x));
                    if (OUT) y[r] = fma2(s, bc.y, y[r]);
                }
                h[k] = s;
            }
            if (OUT) {
#pragma unroll
                for (int r = 0; r < SSM_ROWS; r++) *reinterpret_cast<f2*>(&sm.y[buf][warp][half + r][lane]) = y[r];
            }
        }
        if (OUT) half_arrive<SSM_THREADS>(BAR_Y_FULL + buf);
        if (tile + 2 < tiles) half_arrive<SSM_THREADS>(BAR_EMPTY + buf);
    }
    if (!OUT) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int n = warp * K + k;
            if (n < p.N) *reinterpret_cast<f2*>(seg_state(seg, n)) = h[k];
        }
        if (warp == 0) *reinterpret_cast<f2*>(p.seg_sum + (static_cast<size_t>(b) * p.nseg + seg) * p.Cpad + ch.cp) = sum;
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

template <typename T, int K, bool OUT>
cudaError_t launch_ssm_fwd_pass(const SsmFwdArgs& a, int segs, cudaStream_t st) {
    constexpr size_t smem = sizeof(SsmFwdSmem<K>);
    static std::atomic<unsigned long long> done[3];
    const int v = !a.pairs ? 0 : a.N == K * SSM_WARPS ? 2 : 1;
    auto kern = v == 2 ? ssm_fwd_kernel<T, K, OUT, true, true> : v == 1 ? ssm_fwd_kernel<T, K, OUT, true, false> : ssm_fwd_kernel<T, K, OUT, false, false>;
    const cudaError_t ce = ssm_allow_smem(kern, smem, done[v]);
    if (ce != cudaSuccess) return ce;
    return launch_plain(kern, dim3(static_cast<unsigned>(a.G * a.tiles_g), segs, a.Bt), dim3(SSM_THREADS), smem, st, a);
}
template <typename T, int K>
cudaError_t launch_ssm_fwd(const SsmFwdArgs& a, cudaStream_t st) {
    if (a.nseg > 1) {
        const cudaError_t ce = launch_ssm_fwd_pass<T, K, false>(a, a.nseg - 1, st);
        if (ce != cudaSuccess) return ce;
    }
    return launch_ssm_fwd_pass<T, K, true>(a, a.nseg, st);
}
// States per warp: as few as hold all N.  (Six for 24 states, twelve for 48: 157 and 307 us for 2 x 2048 x 2048 positions and channels, bf16,
// against 210 and 415 with eight and sixteen, which leave the last warp without any.)
template <typename T>
cudaError_t launch_ssm_fwd_n(const SsmFwdArgs& a, cudaStream_t st) {
    if (a.N <= 4) return launch_ssm_fwd<T, 1>(a, st);
    if (a.N <= 8) return launch_ssm_fwd<T, 2>(a, st);
    if (a.N <= 16) return launch_ssm_fwd<T, 4>(a, st);
    if (a.N <= 24) return launch_ssm_fwd<T, 6>(a, st);
    if (a.N <= 32) return launch_ssm_fwd<T, 8>(a, st);
    if (a.N <= 48) return launch_ssm_fwd<T, 12>(a, st);
    return launch_ssm_fwd<T, 16>(a, st);
}

// ---------------------------------------------------------------------------------------------- a few new tokens
constexpr int STEP_TOKENS = 8;
constexpr int STEP_THREADS = 128;
constexpr int STEP_CH = 4;           // channels per group of lanes

struct SsmStepArgs : SsmArgs {
    const float* initial;
    void* y;
    float* state_out;
};

// L lanes share STEP_CH neighbouring channels, four states of each per lane; every channel's input, step and output are one lane's
// (lane i % L for channel i), which hands them to the others.  A group works on several sequences, one after the other, so
// that A is read once for them.  VEC: N = 4 L, states and B, C in whole pieces, all four channels in one group.
// Bound by the states, read and written once: 256 sequences x 4096 channels x 16 states, 134 MB, in 35 us (3.9 TB/s; 63 us with one
// channel per group, whose softplus every lane takes for itself).
template <typename T, int L, bool VEC>
__global__ void __launch_bounds__(STEP_THREADS) ssm_step_kernel(const SsmStepArgs p) {
    constexpr int CH = STEP_CH, OWN = (CH + L - 1) / L;      // channels whose values this lane takes
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, sub = lane & (L - 1), lead = lane - sub;
    const int c0 = ((blockIdx.x * STEP_THREADS + threadIdx.x) / L) * CH, n0 = sub * 4;
    const int nn = max(0, min(4, p.N - n0));
    int c[CH];
    bool on[CH];
    float rate[CH][4], bias[OWN], skip[OWN];
#pragma unroll
    for (int i = 0; i < CH; i++) {
        on[i] = c0 + i < p.Ch;
        c[i] = on[i] ? c0 + i : 0;
        const float* A = p.A + static_cast<size_t>(c[i]) * p.N + n0;
        if (VEC) {
            const float4 r = on[i] ? *reinterpret_cast<const float4*>(A) : make_float4(0.f, 0.f, 0.f, 0.f);
            rate[i][0] = r.x; rate[i][1] = r.y; rate[i][2] = r.z; rate[i][3] = r.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) rate[i][j] = j < nn ? A[j] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; j++) rate[i][j] = decay_rate(rate[i][j]);
    }
    int mine[OWN];                           // (0 where there is none: read, and not written)
    bool have[OWN];
#pragma unroll
    for (int o = 0; o < OWN; o++) {
        const int i = o * L + sub;
        have[o] = i < CH && c0 + i < p.Ch;
        mine[o] = have[o] ? c0 + i : 0;
        bias[o] = p.bias ? p.bias[mine[o]] : 0.f;
        skip[o] = p.D ? p.D[mine[o]] : 0.f;
    }
    float next[CH][4];                       // the states of the sequence after the one that is worked on, on their way
    auto fetch = [&](int b) {
#pragma unroll
        for (int i = 0; i < CH; i++) {
            const float* H = p.initial + (static_cast<size_t>(b) * p.Ch + c[i]) * p.N + n0;
#pragma unroll
            for (int j = 0; j < 4; j++) next[i][j] = 0.f;
            if (p.initial && on[i]) {
                if (VEC) {
                    const float4 v = *reinterpret_cast<const float4*>(H);
                    next[i][0] = v.x; next[i][1] = v.y; next[i][2] = v.z; next[i][3] = v.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (j < nn) next[i][j] = H[j];
                }
            }
        }
    };
    fetch(blockIdx.y);
    for (int b = blockIdx.y; b < p.Bt; b += gridDim.y) {
        float h[CH][4];
#pragma unroll
        for (int i = 0; i < CH; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) h[i][j] = next[i][j];
        if (b + static_cast<int>(gridDim.y) < p.Bt) fetch(b + gridDim.y);
        for (int t = 0; t < p.S; t++) {
            float x[OWN], d[OWN], gate[OWN];
#pragma unroll
            for (int o = 0; o < OWN; o++) {
                x[o] = to_f32<T>(static_cast<const T*>(p.x)[b * p.sx.b + t * p.sx.t + mine[o]]);
                d[o] = to_f32<T>(static_cast<const T*>(p.dt)[b * p.sdt.b + t * p.sdt.t + mine[o]]) + bias[o];
                if (p.z) gate[o] = to_f32<T>(static_cast<const T*>(p.z)[b * p.sz.b + t * p.sz.t + mine[o]]);
            }
            float Bv[4], Cv[4];
            const T* Bp = static_cast<const T*>(p.B) + b * p.sB.b + t * p.sB.t + n0;
            const T* Cp = static_cast<const T*>(p.C) + b * p.sC.b + t * p.sC.t + n0;
            auto vectors = [&](int g) {
                const T *B = Bp + static_cast<long long>(g) * p.N, *C = Cp + static_cast<long long>(g) * p.N;
                if (VEC) {
                    to_floats<T, 4>(load_vec<T, 4>(B), Bv);
                    to_floats<T, 4>(load_vec<T, 4>(C), Cv);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        Bv[j] = j < nn ? to_f32<T>(B[j]) : 0.f;
                        Cv[j] = j < nn ? to_f32<T>(C[j]) : 0.f;
                    }
                }
            };
            if (VEC) vectors(c[0] / p.P);
#pragma unroll
            for (int o = 0; o < OWN; o++)
                if (p.softplus) d[o] = softplus_f(d[o]);
            float y[OWN];
#pragma unroll
            for (int o = 0; o < OWN; o++) y[o] = 0.f;
#pragma unroll
            for (int i = 0; i < CH; i++) {
                const float di = __shfl_sync(0xffffffffu, d[i / L], lead + i % L), xi = __shfl_sync(0xffffffffu, x[i / L], lead + i % L);
                if (!VEC) vectors(c[i] / p.P);
                const float dx = di * xi;
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (VEC || j < nn) {
                        h[i][j] = fmaf(decay_f(di, rate[i][j]), h[i][j], dx * Bv[j]);
                        s = fmaf(h[i][j], Cv[j], s);
                    }
                }
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                if (i % L == sub) y[i / L] = s;
            }
#pragma unroll
            for (int o = 0; o < OWN; o++) {
                if (p.D) y[o] = fmaf(skip[o], x[o], y[o]);
                if (p.z) y[o] *= gate[o] * sigmoid_f(gate[o]);
                if (have[o]) static_cast<T*>(p.y)[(static_cast<size_t>(b) * p.S + t) * p.Ch + mine[o]] = from_f32<T>(y[o]);
            }
        }
        if (p.state_out) {
#pragma unroll
            for (int i = 0; i < CH; i++) {
                float* H = p.state_out + (static_cast<size_t>(b) * p.Ch + c[i]) * p.N + n0;
                if (!on[i]) continue;
                if (VEC) *reinterpret_cast<float4*>(H) = make_float4(h[i][0], h[i][1], h[i][2], h[i][3]);
                else {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (j < nn) H[j] = h[i][j];
                }
            }
        }
    }
}

template <typename T, int L>
cudaError_t launch_ssm_step_l(const SsmStepArgs& a, bool vec, cudaStream_t st) {
    const int per = STEP_THREADS / L * STEP_CH, gx = ceil_div(a.Ch, per);
    // as many sequences per group as leave every SM some sixteen blocks
    int gy = ceil_div(148 * 16, gx);
    gy = gy < a.Bt ? gy : a.Bt;
    gy = ceil_div(a.Bt, ceil_div(a.Bt, gy));
    return vec && a.N == 4 * L ? launch_plain(ssm_step_kernel<T, L, true>, dim3(gx, gy), dim3(STEP_THREADS), 0, st, a)
                               : launch_plain(ssm_step_kernel<T, L, false>, dim3(gx, gy), dim3(STEP_THREADS), 0, st, a);
}
template <typename T>
cudaError_t launch_ssm_step(const SsmStepArgs& a, bool vec, cudaStream_t st) {
    if (a.N <= 4) return launch_ssm_step_l<T, 1>(a, vec, st);
    if (a.N <= 8) return launch_ssm_step_l<T, 2>(a, vec, st);
    if (a.N <= 16) return launch_ssm_step_l<T, 4>(a, vec, st);
    if (a.N <= 32) return launch_ssm_step_l<T, 8>(a, vec, st);
    return launch_ssm_step_l<T, 16>(a, vec, st);
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

constexpr int SSM_FWD_CTAS = 2;     // CTAs that an SM is filled with

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
        if (!aligned(q, es)) return MLSTM_E_ALIGN;
    for (const void* q : {static_cast<const void*>(A), static_cast<const void*>(D), static_cast<const void*>(dt_bias),
                          static_cast<const void*>(initial), static_cast<const void*>(state_out)})
        if (!aligned(q, 4)) return MLSTM_E_ALIGN;
    if (!aligned(checkpoints, 8)) return MLSTM_E_ALIGN;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t ce;
    if (S <= STEP_TOKENS && !checkpoints) {
        SsmStepArgs a;
        static_cast<SsmArgs&>(a) = base;
        a.initial = initial; a.y = y; a.state_out = state_out;
        // whole pieces of four states, and of four values of B and C; four channels of one group
        const long long strides4 = a.sB.b | a.sB.t | a.sC.b | a.sC.t;
        const bool vec = N % 4 == 0 && a.P % STEP_CH == 0 && (strides4 & 3) == 0 && aligned(A, 16) && aligned(initial, 16) &&
                         aligned(state_out, 16) && aligned(Bv, 4 * es) && aligned(Cv, 4 * es);
        ce = dtype == MLSTM_DT_F32 ? launch_ssm_step<float>(a, vec, st)
             : dtype == MLSTM_DT_F16 ? launch_ssm_step<__half>(a, vec, st) : launch_ssm_step<__nv_bfloat16>(a, vec, st);
    } else {
        SsmFwdArgs a;
        static_cast<SsmArgs&>(a) = base;
        ssm_cut(a, SSM_FWD_CTAS);
        const SsmWs w = ssm_carve(workspace, a);
        if (w.bytes && (!workspace || workspace_bytes < w.bytes || !aligned(workspace, 16))) return MLSTM_E_WORKSPACE;
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
