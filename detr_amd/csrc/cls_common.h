// What the kernels of the classification losses share: the class map's codes, the workgroup's sum, the kernel that adds the
// workgroups' partial sums, and the checks of the entry points.
#pragma once

#include "dm_common.h"

namespace {

constexpr int CLS_THREADS = 256;
constexpr int CLS_MAX_BLOCKS = DM_CLS_LOSS_PARTIALS / 2;     // two partial sums per workgroup

// Sum over the workgroup, valid in thread 0: butterflies inside the wave, then the waves in index order.
__device__ __forceinline__ double block_sum(double v, double *lds)
{
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();                 // (the previous use of lds has been read)
    if (lane == 0) lds[wave] = v;
    __syncthreads();
    double total = 0.0;
    if (threadIdx.x == 0)
        for (int w = 0; w < CLS_THREADS / 64; ++w) total += lds[w];
    return total;
}

struct FocalParams {
    float alpha, gamma, scale;
    int64_t ignore_index;
    int use_ignore;
};

// What the class map says about a row, in 32 bits: the class (0 .. C, C = no object), or one of two codes.
constexpr int ROW_IGNORED = -1;     // contributes nothing
constexpr int ROW_BAD = -2;         // a class the reference's one_hot refuses: contributes nothing, and is reported

__device__ __forceinline__ int row_code(int64_t label, unsigned C, const FocalParams &fp)
{
    if (fp.use_ignore && label == fp.ignore_index) return ROW_IGNORED;
    if (label < 0 || label > (int64_t)C) return ROW_BAD;
    return (int)label;
}

// The workgroups' partial sums in index order.  FOCAL: loss = scale * sum.  Otherwise loss = numerator / denominator,
// loss_out[1] = 1 / denominator (what the backward pass scales the stored gradient by).
template <bool FOCAL>
__global__ __launch_bounds__(CLS_THREADS) void cls_loss_finish_kernel(const double *__restrict__ partials, const int blocks,
                                                                      const float scale, float *__restrict__ loss_out)
{
    __shared__ double lds[CLS_THREADS / 64];
    double a = 0.0, b = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < blocks; i += CLS_THREADS) {
        if (FOCAL) a += partials[i];
        else { a += partials[2 * i]; b += partials[2 * i + 1]; }
    }
    a = block_sum(a, lds);
    if (!FOCAL) b = block_sum(b, lds);
    if (threadIdx.x == 0) {
        if (FOCAL) {
            loss_out[0] = (float)(a * (double)scale);
        } else {
            loss_out[0] = (float)(a / b);
            loss_out[1] = (float)(1.0 / b);
        }
    }
}

inline int check_common(const void *logits, const int64_t *target_cls, int64_t rows, int C, float *loss_out, double *partials,
                        int32_t *status)
{
    if (rows < 0 || C < 1) return DM_E_INVALID_ARG;
    if (!loss_out || !partials || !status) return DM_E_INVALID_ARG;
    if (rows > 0 && (!logits || !target_cls)) return DM_E_INVALID_ARG;
    if ((unsigned long long)rows * (unsigned long long)C >= (1ull << 31)) return DM_E_UNSUPPORTED;
    return DM_OK;
}

}  // namespace
