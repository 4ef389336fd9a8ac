// Sums over the rows of a matrix of partial results [rows, cols] fp32, always in the same order: what the gradients of shared
// parameters are finished with (no atomics, so the same inputs give the same bits).
#pragma once
#include "mlstm_common.cuh"

namespace mlstm {

constexpr int RR_COLS = 32;

// out(column, sum): stores one sum.  A block takes 32 columns; RR_GROUPS groups of threads take every RR_GROUPS-th row: 32 where there
// are rows for them, 4 where there are few (2 rows of 73728 columns: 14 us with 32).
template <int RR_GROUPS, typename Out>
__global__ void __launch_bounds__(RR_COLS * RR_GROUPS) reduce_rows_kernel(const float* __restrict__ part, int rows, long long cols, Out out) {
    __shared__ float sm[RR_GROUPS][RR_COLS];
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const long long c = static_cast<long long>(blockIdx.x) * RR_COLS + lane;
    float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
    if (c < cols) {
        int r = grp;
        for (; r + 3 * RR_GROUPS < rows; r += 4 * RR_GROUPS) {
            s0 += part[static_cast<long long>(r) * cols + c];
            s1 += part[static_cast<long long>(r + RR_GROUPS) * cols + c];
            s2 += part[static_cast<long long>(r + 2 * RR_GROUPS) * cols + c];
            s3 += part[static_cast<long long>(r + 3 * RR_GROUPS) * cols + c];
        }
        for (; r < rows; r += RR_GROUPS) s0 += part[static_cast<long long>(r) * cols + c];
    }
    sm[grp][lane] = (s0 + s1) + (s2 + s3);
    __syncthreads();
    if (grp == 0 && c < cols) {
        float s = 0.f;
#pragma unroll
        for (int g = 0; g < RR_GROUPS; g++) s += sm[g][lane];
        out(c, s);
    }
}

template <typename Out>
cudaError_t launch_reduce_rows(const float* part, int rows, long long cols, const Out& out, cudaStream_t st) {
    const dim3 grid(static_cast<unsigned>((cols + RR_COLS - 1) / RR_COLS));
    if (rows > 32) return launch_plain(reduce_rows_kernel<32, Out>, grid, dim3(RR_COLS * 32), 0, st, part, rows, cols, out);
    return launch_plain(reduce_rows_kernel<4, Out>, grid, dim3(RR_COLS * 4), 0, st, part, rows, cols, out);
}

// a value stored in one of the element types
struct AnyOut {
    void* p;
    int dtype;
    __device__ __forceinline__ void put(long long at, float v) const {
        if (dtype == MLSTM_DT_F32) static_cast<float*>(p)[at] = v;
        else if (dtype == MLSTM_DT_F16) static_cast<__half*>(p)[at] = from_f32<__half>(v);
        else static_cast<__nv_bfloat16*>(p)[at] = from_f32<__nv_bfloat16>(v);
    }
};
__device__ __forceinline__ float load_any(const void* p, int dtype, long long at) {
    if (dtype == MLSTM_DT_F32) return static_cast<const float*>(p)[at];
    if (dtype == MLSTM_DT_F16) return to_f32<__half>(static_cast<const __half*>(p)[at]);
    return to_f32<__nv_bfloat16>(static_cast<const __nv_bfloat16*>(p)[at]);
}

}  // namespace mlstm
