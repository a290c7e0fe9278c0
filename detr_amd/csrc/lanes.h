// Element types, loads of four elements at any alignment, and reductions over groups of lanes, shared by the loss kernels
// that take float32, bfloat16 and float16 logits.
#pragma once

#include <type_traits>

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

// A row that L lanes share; WIDE: of DM_F32, else of DM_BF16 or DM_F16 as `dtype` says.  A lane holds NQ quads of four
// elements, the lanes' quads side by side.  `fetch_row` only asks for the memory, so that a kernel can ask for its next row
// before it works on this one; `row_values` makes float32 of what came: `raw_values`, then `place_row`.  There is no branch
// between the loads (each would wait for the one before it): a quad that reaches past the row is read at the row's last four
// elements and moved into place afterwards.  One lane with one quad also takes rows of fewer than four elements.  (What is read
// is of the row in every case.)
template <int NQ, bool WIDE>
struct RawRow {
    unsigned q[NQ][WIDE ? 4 : 2];
};

template <int NQ, int L, bool WIDE>
__device__ __forceinline__ RawRow<NQ, WIDE> fetch_row(const void *base, size_t first, unsigned sub, unsigned n)
{
    typedef unsigned Four __attribute__((ext_vector_type(4), aligned(4)));
    typedef unsigned Two __attribute__((ext_vector_type(2), aligned(2)));
    RawRow<NQ, WIDE> raw;
    if (NQ == 1 && L == 1 && n < 4) {
        if (WIDE) {
            const unsigned *row = static_cast<const unsigned *>(base) + first;
            for (unsigned k = 0; k < 4; ++k) raw.q[0][k & (WIDE ? 3 : 1)] = row[min(k, n - 1)];
        } else {
            const uint16_t *row = static_cast<const uint16_t *>(base) + first;
            raw.q[0][0] = row[0] | (unsigned)row[min(1u, n - 1)] << 16;
            raw.q[0][1] = row[n - 1] | (unsigned)row[n - 1] << 16;
        }
        return raw;
    }
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const unsigned c = min(4 * (q * L + sub), n - 4);
        if (WIDE) {
            const Four t = *reinterpret_cast<const Four *>(static_cast<const float *>(base) + first + c);
            raw.q[q][0] = t.x;
            raw.q[q][1] = t.y;
            raw.q[q][WIDE ? 2 : 0] = t.z;
            raw.q[q][WIDE ? 3 : 1] = t.w;
        } else {
            const Two t = *reinterpret_cast<const Two *>(static_cast<const uint16_t *>(base) + first + c);
            raw.q[q][0] = t.x;
            raw.q[q][1] = t.y;
        }
    }
    return raw;
}

template <int NQ, bool WIDE>
__device__ __forceinline__ void raw_values(const RawRow<NQ, WIDE> &raw, int dtype, float (&x)[4 * NQ])
{
    if (WIDE) {
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int k = 0; k < 4; ++k) x[4 * q + k] = __uint_as_float(raw.q[q][WIDE ? k : 0]);
    } else if (dtype == DM_BF16) {
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                x[4 * q + 2 * k] = __uint_as_float(raw.q[q][k] << 16);
                x[4 * q + 2 * k + 1] = __uint_as_float(raw.q[q][k] & 0xFFFF0000u);
            }
    } else {
        typedef half_t Halves __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const Halves h = __builtin_bit_cast(Halves, raw.q[q][k]);
                x[4 * q + 2 * k] = (float)h.x;
                x[4 * q + 2 * k + 1] = (float)h.y;
            }
    }
}

// Quads that were read further to the left into their places, `fill` behind the row's end.
template <int NQ, int L>
__device__ __forceinline__ void place_row(float (&x)[4 * NQ], unsigned sub, unsigned n, float fill)
{
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        if (4 * (q + 1) * L <= n) continue;                    // (the same for all lanes)
        const unsigned c = 4 * (q * L + sub);
        float *v = x + 4 * q;
        if ((n & 3) == 0 || n < 4) {
#pragma unroll
            for (unsigned k = 0; k < 4; ++k) v[k] = c + k < n ? v[k] : fill;
        } else {
            const unsigned moved = c - min(c, n - 4);
            const bool one = moved & 1, two = moved & 2, out = moved >= 4;
            const float v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3];
            const float a0 = one ? v1 : v0, a1 = one ? v2 : v1, a2 = one ? v3 : v2, a3 = one ? fill : v3;
            v[0] = out ? fill : two ? a2 : a0;
            v[1] = out ? fill : two ? a3 : a1;
            v[2] = out || two ? fill : a2;
            v[3] = out || two ? fill : a3;
        }
    }
}

// The same for 16-bit elements before they are made float32, a quad at once; `pair`: two elements to fill with.
template <int NQ, int L>
__device__ __forceinline__ void place_raw(RawRow<NQ, false> &raw, unsigned sub, unsigned n, unsigned pair)
{
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        if (4 * (q + 1) * L <= n) continue;                    // (the same for all lanes)
        const unsigned c = 4 * (q * L + sub);
        // moved: places that the quad is to move down; n < 4: it was read in place, what is behind the end is made `fill`
        const unsigned moved = n < 4 ? 0 : c - min(c, n - 4);
        const unsigned long long v = (unsigned long long)raw.q[q][1] << 32 | raw.q[q][0];
        const unsigned long long all = (unsigned long long)pair << 32 | pair;
        const unsigned left = n < 4 ? min(n - min(c, n), 4u) : 4 - min(moved, 4u);      // elements of the row in the quad
        const unsigned long long low = moved >= 4 ? 0ull : v >> (16 * (moved & 3));
        const unsigned long long keep = left >= 4 ? ~0ull : (1ull << (16 * left)) - 1;
        const unsigned long long r = (low & keep) | (all & ~keep);
        raw.q[q][0] = (unsigned)r;
        raw.q[q][1] = (unsigned)(r >> 32);
    }
}

template <int NQ, int L, bool WIDE>
__device__ __forceinline__ void row_values(const RawRow<NQ, WIDE> &raw, int dtype, unsigned sub, unsigned n, float fill, float (&x)[4 * NQ])
{
    raw_values<NQ, WIDE>(raw, dtype, x);
    place_row<NQ, L>(x, sub, n, fill);
}

template <int NQ, int L, bool WIDE>
__device__ __forceinline__ void store_row(void *base, int dtype, size_t first, unsigned sub, unsigned n, const float (&x)[4 * NQ])
{
    auto store = [&](auto *row) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const float v[4] = {x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
            store_quad(row, 4 * (q * L + sub), n, v);
        }
    };
    if (WIDE) store(static_cast<float *>(base) + first);
    else if (dtype == DM_BF16) store(static_cast<bf16_t *>(base) + first);
    else store(static_cast<half_t *>(base) + first);
}

// Largest and smallest of three, in one instruction.  (fmaxf would first quiet each argument, as IEEE asks of a signalling NaN.)  A quiet
// NaN is passed over, a signalling one may come out.
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

__device__ __forceinline__ float min3(float a, float b, float c)
{
    float r;
    asm("v_min3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
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

template <int STEP>
__device__ __forceinline__ unsigned long long partner(unsigned long long v)
{
    return (unsigned long long)partner<STEP>((unsigned)(v >> 32)) << 32 | partner<STEP>((unsigned)v);
}
template <int STEP>
__device__ __forceinline__ double partner(double v)
{
    return __builtin_bit_cast(double, partner<STEP>(__builtin_bit_cast(unsigned long long, v)));
}

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

// The largest over the group, each step one instruction: the maximum takes the partner's value itself.  (Two wait states
// between a register's result and its reading by a DPP operand, which the compiler does not see inside.)  No NaN.
#define DM_MAX_DPP(v, control) asm("s_nop 1\n\tv_max_f32_dpp %0, %1, %1 " control " row_mask:0xf bank_mask:0xf" : "=v"(v) : "v"(v))
template <int L>
__device__ __forceinline__ float largest(float v)
{
    if (L >= 2) DM_MAX_DPP(v, "quad_perm:[1,0,3,2]");
    if (L >= 4) DM_MAX_DPP(v, "quad_perm:[2,3,0,1]");
    if (L >= 8) DM_MAX_DPP(v, "row_half_mirror");
    if (L >= 16) DM_MAX_DPP(v, "row_mirror");
    if (L >= 32) v = __builtin_amdgcn_fmed3f(v, partner<16>(v), __builtin_huge_valf());
    if (L >= 64) v = __builtin_amdgcn_fmed3f(v, partner<32>(v), __builtin_huge_valf());
    return v;
}
#undef DM_MAX_DPP
#define DM_MAX_DPP(v, control) asm("s_nop 1\n\tv_max_i32_dpp %0, %1, %1 " control " row_mask:0xf bank_mask:0xf" : "=v"(v) : "v"(v))
template <int L>
__device__ __forceinline__ int largest(int v)
{
    if (L >= 2) DM_MAX_DPP(v, "quad_perm:[1,0,3,2]");
    if (L >= 4) DM_MAX_DPP(v, "quad_perm:[2,3,0,1]");
    if (L >= 8) DM_MAX_DPP(v, "row_half_mirror");
    if (L >= 16) DM_MAX_DPP(v, "row_mirror");
    if (L >= 32) v = max(v, partner<16>(v));
    if (L >= 64) v = max(v, partner<32>(v));
    return v;
}
#undef DM_MAX_DPP

// The middle one of three.
__device__ __forceinline__ float median(float a, float b, float c) { return __builtin_amdgcn_fmed3f(a, b, c); }
__device__ __forceinline__ int median(int a, int b, int c)
{
    int r;
    asm("v_med3_i32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// The sum over the lanes of a row of 16 whose number is the same modulo L (L <= 16): every lane gets that of its own.
template <int L, typename V>
__device__ __forceinline__ V over_row16(V v)
{
    auto turned = [](V a, auto step) {
        int i;
        __builtin_memcpy(&i, &a, 4);
        i = __builtin_amdgcn_update_dpp(0, i, 0x120 + decltype(step)::value, 0xF, 0xF, true);      // row_ror
        V r;
        __builtin_memcpy(&r, &i, 4);
        return r;
    };
    if (L <= 8) v += turned(v, std::integral_constant<int, 8>());
    if (L <= 4) v += turned(v, std::integral_constant<int, 4>());
    if (L <= 2) v += turned(v, std::integral_constant<int, 2>());
    if (L <= 1) v += turned(v, std::integral_constant<int, 1>());
    return v;
}

}  // namespace dm
