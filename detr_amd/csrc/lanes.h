// Element types, loads of four elements at any alignment, and reductions over groups of lanes, shared by the loss kernels
// that take float32, bfloat16 and float16 logits.
#pragma once

#include "dm_common.h"

namespace dm {

typedef _Float16 half_t;
typedef __bf16 bf16_t;

// Four consecutive elements.  The vector is aligned like one element: rows of odd length start anywhere, and gfx950 takes
// wide global accesses at any address.
template <typename T>
struct Quad {
    typedef T type __attribute__((ext_vector_type(4), aligned(sizeof(T))));
};

// Elements c .. c + 3 of a row of n as float32, `fill` past its end.
template <typename T>
__device__ __forceinline__ void load_quad(const T *row, unsigned c, unsigned n, float fill, float (&v)[4])
{
    if (c + 4 <= n) {
        const typename Quad<T>::type t = *reinterpret_cast<const typename Quad<T>::type *>(row + c);
        v[0] = (float)t.x; v[1] = (float)t.y; v[2] = (float)t.z; v[3] = (float)t.w;
    } else {
#pragma unroll
        for (unsigned k = 0; k < 4; ++k) v[k] = c + k < n ? (float)row[c + k] : fill;
    }
}

// The same way back, each value rounded once to the row's type.
template <typename T>
__device__ __forceinline__ void store_quad(T *row, unsigned c, unsigned n, const float (&v)[4])
{
    if (c + 4 <= n) {
        typename Quad<T>::type t;
        t.x = (T)v[0]; t.y = (T)v[1]; t.z = (T)v[2]; t.w = (T)v[3];
        *reinterpret_cast<typename Quad<T>::type *>(row + c) = t;
    } else {
#pragma unroll
        for (unsigned k = 0; k < 4; ++k)
            if (c + k < n) row[c + k] = (T)v[k];
    }
}

// The value of a partner lane at every step of a reduction over groups of L consecutive lanes (L a power of two): lanes
// that hold partial results of the same part of the group trade with those of the other part.  Steps 1 to 8 are DPP moves
// inside a row of 16 lanes (the mirrors pair the right parts because the steps before have made each part's lanes equal).
template <int STEP>
__device__ __forceinline__ int partner(int v)
{
    if (STEP == 1) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true);        // quad_perm [1,0,3,2]
    if (STEP == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true);        // quad_perm [2,3,0,1]
    if (STEP == 4) return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, true);       // row_half_mirror
    if (STEP == 8) return __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, true);       // row_mirror
    return __shfl_xor(v, STEP);
}
template <int STEP>
__device__ __forceinline__ unsigned partner(unsigned v) { return (unsigned)partner<STEP>((int)v); }
template <int STEP>
__device__ __forceinline__ float partner(float v) { return __int_as_float(partner<STEP>(__float_as_int(v))); }

struct Max { template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a > b ? a : b; } };
struct Min { template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a < b ? a : b; } };
struct Add { template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; } };

// Over the group of L lanes that the lane belongs to; every lane gets the result.
template <int L, typename Op, typename V>
__device__ __forceinline__ V over_group(V v, Op op)
{
    if (L >= 2) v = op(v, partner<1>(v));
    if (L >= 4) v = op(v, partner<2>(v));
    if (L >= 8) v = op(v, partner<4>(v));
    if (L >= 16) v = op(v, partner<8>(v));
    if (L >= 32) v = op(v, partner<16>(v));
    if (L >= 64) v = op(v, partner<32>(v));
    return v;
}

}  // namespace dm
