// The classification losses with 8 bits per logit kept for the backward pass, for gfx950 (MI355X): the forward pass reads
// the logits once, sums the loss and leaves one byte per logit; the backward pass computes the gradient from the bytes.
// Against keeping the float32 gradient (cls_loss_kernels.hip) the state between the two is a quarter, and a step moves
// 4 + 1 and 1 + 4 bytes per float32 logit instead of 4 + 4 and 4 + 4.
//
// The code.  A block of logits shares a step 2^e, the finest from 2^-16 up to a coarsest one for which the whole numbers
// rint(x 2^-e) of the block span at most 255; a logit's byte is how many steps it lies below the block's largest, 255 at
// most.  With a power of two every operation of this is exact in float32 -- the byte does not depend on the arithmetic it
// was found with -- and the logit is off by at most half a step.
//   focal           blocks of 128 consecutive logits of the flat array, clamped to +-20 first: sigmoid(-20) = 2e-9 is below
//                   the rounding of a float32 gradient of order one, and one masked logit does not take the block's
//                   resolution away.  The span is 40 at most, so 2^-2 always suffices and no byte is cut off at 255.
//                   Rows that do not count are part of the array, and so of the ranges, but a padded row may hold anything:
//                   what lies beyond +-20 there, or is no number, counts as 0.
//                   A head per block, 32 bits: largest whole number << 8 | e.  With a gamma below zero none of this would hold
//                   (a slope falls off like exp((1 + gamma) z) only): refused.
//   cross entropy   a block is a row: the softmax does not change when a row's largest logit is taken off, so e is all that
//                   is kept beside the bytes.  2^-3 at most: logits further below the largest than 31.9 are cut off there,
//                   at a probability of e^-31.9 = 1e-14.  (Logits beyond +-2^20 count as +-2^20.)
// e = -128 marks a block with a NaN (cross entropy: a row whose softmax is NaN); its gradient is NaN.
//
// The gradient is that of the loss at the decoded logits; the loss itself is of the logits as they came.
//
// Measured in a step (a copy of a GiB runs at 5.1 TB/s, a kernel of a few workgroups takes 4 us among others), forward and backward:
//   focal           256 x 900 x 91 float32 (84 MB of logits, 21 of bytes): 27.5 and 25.6 us, 4 TB/s, bound by 50 and 35 vector
//                   instructions per logit, an exponential, a logarithm and a reciprocal among them; the same of bfloat16: 26.9 and
//                   25.5; with a fifth of the rows ignored: 34.3 and 28.4 (what does not count is asked of each quad of a wave that
//                   meets such a row); 4 x 300 x 1203 bfloat16: 7.8 and 5.9; 64 x 600 x 2 float32: 4.6 and 4.2
//   cross entropy   256 x 900 x 92 float32 (85 MB, 21 MB): 22.5 and 19.1 us, 4.7 and 5.6 TB/s, at the rate of a copy; of bfloat16
//                   20.9 and 16.4; 16 x 301 x 1205 float16 (12 MB, 6 MB): 10.3 and 8.3
// The sums of the workgroups' partial sums take 2 to 4 us more; one workgroup by itself makes the loss as well.  The host's part of
// a call and its backward pass, about 45 us, most of it the autograd engine's, covers all of these.
#include <algorithm>
#include <climits>

#include "cls_common.h"
#include "lanes.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int FINEST = -16, FOCAL_COARSEST = -2, CE_COARSEST = -3, NOT_A_NUMBER = -128;
constexpr float FOCAL_CLAMP = 20.0f, CE_CLAMP = 1048576.0f;

// A byte (a whole number from 0 to 255) into place k of a word.
__device__ __forceinline__ unsigned pack_code(unsigned word, unsigned k, float code)
{
    return __builtin_amdgcn_cvt_pk_u8_f32(code, k, word);
}

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }

// The exponent of the step of a block whose logits lie in [low, high].  With high - low in [2^E, 2^(E+1)) the span at
// 2^(E-9) is above 510 and at 2^(E-6) below 130: two trials after the first candidate E - 8.
__device__ __forceinline__ int step_exponent(float high, float low, int coarsest)
{
    int e = (int)((__float_as_uint(high - low) >> 23) & 255u) - 127 - 8;
    e = min(max(e, FINEST), coarsest);
#pragma unroll
    for (int trial = 0; trial < 2; ++trial) {
        const float inverse = power_of_two(-e);
        const bool wide = __builtin_rintf(high * inverse) - __builtin_rintf(low * inverse) > 255.0f;
        e += wide && e < coarsest ? 1 : 0;
    }
    return e;
}

// softplus(z) and sigmoid(z)^gamma with z = -x for the positive logit and z = x for the others (the loss of a logit is
// alpha_t times their product), and the derivative of that product.  e = exp(-|z|) serves all: sigmoid(z) = 1 / (1 + e) or
// e / (1 + e), softplus(z) = max(z, 0) + log1p(e), sigmoid(z)^gamma = exp(-gamma softplus(-z)).
struct FocalParts {
    float softplus, power, sigmoid, rest;      // rest = 1 - sigmoid
};
template <bool GAMMA2>
__device__ __forceinline__ FocalParts focal_parts(float z, float gamma)
{
    FocalParts f;
    const float e = __builtin_amdgcn_exp2f(-__builtin_fabsf(z) * LOG2E);
    const float one_e = 1.0f + e, r = __builtin_amdgcn_rcpf(one_e);
    const bool up = z >= 0.0f;
    f.sigmoid = (up ? 1.0f : e) * r;
    f.rest = (up ? e : 1.0f) * r;
    // log1p(e) = log(1 + e) + what the rounding of 1 + e dropped, over 1 + e
    const float l1p = __builtin_fmaf(e - (one_e - 1.0f), r, __builtin_amdgcn_logf(one_e) * LN2);
    f.softplus = (up ? z : 0.0f) + l1p;
    // (NaN: fminf passes it over, e carries it)
    if (GAMMA2) f.power = f.sigmoid * f.sigmoid;
    else f.power = __builtin_amdgcn_exp2f(-gamma * LOG2E * __builtin_fminf((up ? 0.0f : -z) + l1p, 1e30f));      // (0 x infinity)
    return f;
}

// The focal kernels' share of the flat array: 8 lanes take a block of 128 logits, each four quads of four consecutive ones,
// 32 logits apart (a load of the 8 lanes is 128 bytes of float32).  With four logits per lane, and 32 lanes to agree on a
// block's step, the agreement cost as much as half of the loss itself.
constexpr unsigned BLOCK = 128, LANES = 8, QUADS = 4, BLOCKS_AT_A_TIME = CLS_THREADS / LANES;

// Rows and columns of a lane's quads, walked by additions: from quad to quad of a block, and from block to block.
struct Walk {
    unsigned row, col, C, quad_row, quad_col, block_row, block_col;
    __device__ __forceinline__ Walk(unsigned block, unsigned stride, unsigned sub, unsigned C_) : C(C_)
    {
        const unsigned first = block * BLOCK + 4 * sub, apart = 4 * LANES, far = stride * BLOCK;
        row = first / C;
        col = first - row * C;
        quad_row = apart / C;
        quad_col = apart - quad_row * C;
        block_row = far / C;
        block_col = far - block_row * C;
    }
    __device__ __forceinline__ void step(unsigned &r, unsigned &c, unsigned rows, unsigned cols) const
    {
        c += cols;
        const bool over = c >= C;
        c = over ? c - C : c;
        r += rows + (over ? 1u : 0u);
    }
    __device__ __forceinline__ void next_quad(unsigned &r, unsigned &c) const { step(r, c, quad_row, quad_col); }
    __device__ __forceinline__ void next_block() { step(row, col, block_row, block_col); }
};

// The rows of a lane's quads.  With two or more classes four consecutive logits lie in at most two rows (quads start at
// multiples of four of the flat array, so that also holds for two classes); with one, each is a row.
template <bool ONE_CLASS>
struct BlockRows {
    static constexpr unsigned ROWS = ONE_CLASS ? 4 : 2;
    int64_t label[QUADS][ROWS];
    unsigned col[QUADS];
    int hot[QUADS][ROWS];       // place of the row's positive logit in the quad, if it is there
    bool skipped;               // some row may not count: `dropped` has to be asked

    // (first: of the lane's logits in the flat array)
    __device__ __forceinline__ void ask(const int64_t *cls, const Walk &at, unsigned first, unsigned rows)
    {
        unsigned r = at.row, c = at.col;
#pragma unroll
        for (unsigned q = 0; q < QUADS; ++q) {
            col[q] = c;
#pragma unroll
            for (unsigned k = 0; k < ROWS; ++k) label[q][k] = cls[min((ONE_CLASS ? first + 4 * LANES * q : r) + k, rows - 1)];
            if (!ONE_CLASS) at.next_quad(r, c);
        }
    }
    __device__ __forceinline__ void settle(unsigned C, const FocalParams &fp)
    {
        unsigned largest = 0, high = 0;
#pragma unroll
        for (unsigned q = 0; q < QUADS; ++q)
#pragma unroll
            for (unsigned k = 0; k < ROWS; ++k) {
                const unsigned low = (unsigned)label[q][k];
                high |= (unsigned)((uint64_t)label[q][k] >> 32);
                largest = max(largest, low);
                // (a class that is none is nowhere: its row's neighbours in the quad are others'.  Modulo 2^32, where no other place
                // comes round to 0 to 3 again: low - col lies between -2^31 and 2^31, low + C - col below 2^32)
                const unsigned place = low + (ONE_CLASS ? k : k ? C - col[q] : 0u - col[q]);
                hot[q][k] = low < C ? (int)place : INT_MIN;
            }
        skipped = high != 0 || largest > C;
        if (fp.use_ignore && (uint64_t)fp.ignore_index <= C) {
#pragma unroll
            for (unsigned q = 0; q < QUADS; ++q)
#pragma unroll
                for (unsigned k = 0; k < ROWS; ++k) skipped |= (unsigned)label[q][k] == (unsigned)fp.ignore_index;
        }
    }
    __device__ __forceinline__ bool positive(unsigned q, unsigned k) const
    {
        if (ONE_CLASS) return hot[q][k] == (int)k;
        return hot[q][0] == (int)k || hot[q][1] == (int)k;
    }
    // Which of a quad's logits (a bit each) are of rows that do not count.
    __device__ __forceinline__ unsigned dropped(unsigned q, unsigned C, const FocalParams &fp, bool *bad) const
    {
        unsigned of_row[ROWS];
#pragma unroll
        for (unsigned k = 0; k < ROWS; ++k) {
            const int code = row_code(label[q][k], C, fp);
            *bad |= code == ROW_BAD;
            of_row[k] = code < 0 ? 15u : 0u;
        }
        if (ONE_CLASS) return (of_row[0] & 1u) | (of_row[1] & 2u) | (of_row[ROWS - 2] & 4u) | (of_row[ROWS - 1] & 8u);
        const unsigned first = (1u << min(C - col[q], 4u)) - 1;      // of the first row
        return (of_row[0] & first) | (of_row[1] & ~first);
    }
};

// Loss, bytes and heads.  codes NULL: the loss alone.  One exponential per logit serves the softplus, the sigmoid and its
// power; the block's step is found from its extremes (8 lanes, three exchanges) while the logits are still in registers.
template <typename T, bool GAMMA2, bool ONE_CLASS>
__global__ __launch_bounds__(CLS_THREADS) void focal_saved_kernel(const T *__restrict__ x, const int64_t *__restrict__ cls,
                                                                  const unsigned n, const unsigned C, const unsigned rows,
                                                                  const FocalParams fp, unsigned *__restrict__ codes,
                                                                  int32_t *__restrict__ heads, double *__restrict__ partials,
                                                                  float *__restrict__ loss_out, int32_t *__restrict__ status)
{
    typedef typename dm::Quad<T>::type Four;
    __shared__ double lds[CLS_THREADS / 64];
    const unsigned blocks = n / BLOCK, stride = gridDim.x * BLOCKS_AT_A_TIME;      // whole blocks
    const unsigned sub = threadIdx.x & (LANES - 1), lane = threadIdx.x & 63;
    const float alpha1 = fp.alpha >= 0.0f ? fp.alpha : 1.0f, alpha0 = fp.alpha >= 0.0f ? 1.0f - fp.alpha : 1.0f;
    double acc = 0.0;                // (in 64 bits from block to block: a lane may walk hundreds of equal ones)
    bool bad = false;

    // a block with its logits and rows; whole: all 128 are there
    auto work = [&](unsigned block, float (&v)[4 * QUADS], BlockRows<ONE_CLASS> &rows_of, bool whole) {
        const unsigned first = block * BLOCK + 4 * sub;
        rows_of.settle(C, fp);
        // logits of rows that do not count, or behind the last one, add no loss, whatever they hold: at an infinity on their class's
        // side it is 0.  The former have their place in the block's range, as 0 what lies beyond the clamp.  (Their bytes, which
        // saturate, are not asked for.)
        bool some_out = false;
        float low_before = FOCAL_CLAMP, high_before = -FOCAL_CLAMP;
        if (rows_of.skipped || !whole) {
            some_out = true;
#pragma unroll
            for (unsigned q = 0; q < QUADS; ++q) {
                const unsigned at = first + 4 * LANES * q, there = whole ? 4u : at < n ? min(n - at, 4u) : 0u;
                const unsigned none = rows_of.dropped(q, C, fp, &bad), out = none | (15u << there);
#pragma unroll
                for (unsigned k = 0; k < 4; ++k) {
                    const float x = v[4 * q + k], clamped = __builtin_amdgcn_fmed3f(x, -FOCAL_CLAMP, FOCAL_CLAMP);
                    const float held = none >> k & 1 && clamped != x ? 0.0f : clamped;
                    low_before = k < there ? dm::min3(low_before, held, held) : low_before;
                    high_before = k < there ? dm::max3(high_before, held, held) : high_before;
                    if (out >> k & 1) v[4 * q + k] = rows_of.positive(q, k) ? __builtin_huge_valf() : -__builtin_huge_valf();
                }
            }
        }
        float c[4 * QUADS], high = -FOCAL_CLAMP, low = FOCAL_CLAMP, sum = 0.0f;
        bool nan = false;
#pragma unroll
        for (unsigned q = 0; q < QUADS; ++q) {
            float term[4];
#pragma unroll
            for (unsigned k = 0; k < 4; ++k) {
                const float x = v[4 * q + k];
                const bool positive = rows_of.positive(q, k);
                const FocalParts f = focal_parts<GAMMA2>(positive ? -x : x, fp.gamma);
                term[k] = (positive ? alpha1 : alpha0) * (f.softplus * f.power);
                c[4 * q + k] = __builtin_amdgcn_fmed3f(x, -FOCAL_CLAMP, FOCAL_CLAMP);
                nan |= x != x;
            }
            low = dm::min3(dm::min3(low, c[4 * q], c[4 * q + 1]), c[4 * q + 2], c[4 * q + 3]);
            high = dm::max3(dm::max3(high, c[4 * q], c[4 * q + 1]), c[4 * q + 2], c[4 * q + 3]);
            sum += (term[0] + term[1]) + (term[2] + term[3]);
        }
        acc += (double)sum;
        if (!codes) return;
        low = some_out ? low_before : low;
        high = some_out ? high_before : high;
        high = dm::largest<LANES>(high);
        low = -dm::largest<LANES>(-low);
        const bool block_nan = ((__ballot(nan) >> (lane & ~(LANES - 1))) & ((1u << LANES) - 1)) != 0;
        const int e = step_exponent(high, low, FOCAL_COARSEST);
        const float inverse = power_of_two(-e);
        const float top = __builtin_rintf(high * inverse);
#pragma unroll
        for (unsigned q = 0; q < QUADS; ++q) {
            unsigned packed = 0;
#pragma unroll
            for (unsigned k = 0; k < 4; ++k) packed = pack_code(packed, k, top - __builtin_rintf(c[4 * q + k] * inverse));
            codes[block * (BLOCK / 4) + LANES * q + sub] = packed;
        }
        if (sub == 0) heads[block] = block_nan ? (NOT_A_NUMBER & 255) : (int)top * 256 | (e & 255);
    };

    unsigned block = blockIdx.x * BLOCKS_AT_A_TIME + threadIdx.x / LANES;
    Walk at(block, stride, sub, C);
    // (the lanes of a block run the same trips)
    for (; block < blocks; block += stride) {
        const unsigned first = block * BLOCK + 4 * sub;
        Four t[QUADS];
#pragma unroll
        for (unsigned q = 0; q < QUADS; ++q) t[q] = *reinterpret_cast<const Four *>(x + first + 4 * LANES * q);
        BlockRows<ONE_CLASS> rows_of;
        rows_of.ask(cls, at, first, rows);
        at.next_block();
        float v[4 * QUADS];
#pragma unroll
        for (unsigned q = 0; q < QUADS; ++q) {
            v[4 * q] = (float)t[q].x;
            v[4 * q + 1] = (float)t[q].y;
            v[4 * q + 2] = (float)t[q].z;
            v[4 * q + 3] = (float)t[q].w;
        }
        work(block, v, rows_of, true);
    }
    // the last block, if it is not a whole one
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x < LANES && n % BLOCK != 0) {
        const unsigned first = blocks * BLOCK + 4 * sub;
        float v[4 * QUADS];
#pragma unroll
        for (unsigned q = 0; q < QUADS; ++q)
#pragma unroll
            for (unsigned k = 0; k < 4; ++k) v[4 * q + k] = (float)x[min(first + 4 * LANES * q + k, n - 1)];
        const Walk last(blocks, 0, sub, C);
        BlockRows<ONE_CLASS> rows_of;
        rows_of.ask(cls, last, first, rows);
        work(blocks, v, rows_of, false);
    }
    if (bad) dm::raise_status(status, DM_ST_LABEL_RANGE);
    const double total = block_sum(acc, lds);
    if (threadIdx.x == 0) {
        if (gridDim.x == 1) loss_out[0] = (float)(total * (double)fp.scale);
        else partials[blockIdx.x] = total;
    }
}

// The gradient of the logits that the bytes stand for, with the same exponential, logarithm and reciprocal per logit.
template <typename T, bool GAMMA2, bool ONE_CLASS>
__global__ __launch_bounds__(CLS_THREADS) void focal_from_saved_kernel(const unsigned *__restrict__ codes,
                                                                       const int32_t *__restrict__ heads,
                                                                       const int64_t *__restrict__ cls, const unsigned n,
                                                                       const unsigned C, const unsigned rows, const FocalParams fp,
                                                                       const float *__restrict__ grad_loss, T *__restrict__ grad)
{
    typedef typename dm::Quad<T>::type Four;
    const unsigned blocks = (n + BLOCK - 1) / BLOCK, whole = n / BLOCK, stride = gridDim.x * BLOCKS_AT_A_TIME;
    const unsigned sub = threadIdx.x & (LANES - 1);
    const float scale = fp.scale * grad_loss[0];
    const float gamma = GAMMA2 ? 2.0f : fp.gamma;
    // (the gradient of a positive logit has the other sign)
    const float alpha1 = -scale * (fp.alpha >= 0.0f ? fp.alpha : 1.0f), alpha0 = scale * (fp.alpha >= 0.0f ? 1.0f - fp.alpha : 1.0f);
    unsigned block = blockIdx.x * BLOCKS_AT_A_TIME + threadIdx.x / LANES;
    Walk at(block, stride, sub, C);
    for (; block < blocks; block += stride) {
        const unsigned first = block * BLOCK + 4 * sub;
        unsigned packed[QUADS];
#pragma unroll
        for (unsigned q = 0; q < QUADS; ++q) packed[q] = codes[block * (BLOCK / 4) + LANES * q + sub];
        const int head = heads[block];
        BlockRows<ONE_CLASS> rows_of;
        rows_of.ask(cls, at, first, rows);
        at.next_block();
        rows_of.settle(C, fp);
        const int e = (int)(int8_t)(head & 255);
        const float step = e == NOT_A_NUMBER ? __builtin_nanf("") : power_of_two(e);
        const float top = (float)(head >> 8) * step;
#pragma unroll
        for (unsigned q = 0; q < QUADS; ++q) {
            float g[4];
#pragma unroll
            for (unsigned k = 0; k < 4; ++k) {
                const bool positive = rows_of.positive(q, k);
                const float x = __builtin_fmaf((float)((packed[q] >> (8 * k)) & 255u), -step, top);      // (exact)
                const FocalParts f = focal_parts<GAMMA2>(positive ? -x : x, fp.gamma);
                const float slope = f.power * __builtin_fmaf(gamma, f.softplus * f.rest, f.sigmoid);
                g[k] = (positive ? alpha1 : alpha0) * slope;
            }
            if (rows_of.skipped) {
                bool bad = false;
                const unsigned out = rows_of.dropped(q, C, fp, &bad);
#pragma unroll
                for (unsigned k = 0; k < 4; ++k) g[k] = out >> k & 1 ? 0.0f : g[k];
            }
            if (block < whole) {
                Four t;
                t.x = (T)g[0]; t.y = (T)g[1]; t.z = (T)g[2]; t.w = (T)g[3];
                *reinterpret_cast<Four *>(grad + first + 4 * LANES * q) = t;
            } else {
                dm::store_quad(grad, first + 4 * LANES * q, n, g);
            }
        }
    }
}

// What a row of the class map weighs in the cross entropy: 0 when it is ignored or its class is none of the row's.
__device__ __forceinline__ float row_weight(int64_t y, unsigned C, int64_t ignore_index, const float *weight, bool *bad)
{
    if (y == ignore_index) return 0.0f;
    if (y < 0 || y >= (int64_t)C) {
        *bad = true;
        return 0.0f;
    }
    return weight ? weight[y] : 1.0f;
}

// A workgroup's sums: of the only one they are the loss (as cls_loss_finish_kernel makes it).
__device__ __forceinline__ void ce_sums(double num, double den, double *partials, float *loss_out)
{
    if (gridDim.x == 1) {
        loss_out[0] = (float)(num / den);
        loss_out[1] = (float)(1.0 / den);
    } else {
        partials[2 * blockIdx.x] = num;
        partials[2 * blockIdx.x + 1] = den;
    }
}

// The bytes of the classes c .. c + 3 of a row of C, at any alignment.
__device__ __forceinline__ void store_codes(uint8_t *row, unsigned c, unsigned C, unsigned packed)
{
    typedef unsigned Word __attribute__((aligned(1)));
    if (c + 4 <= C) {
        *reinterpret_cast<Word *>(row + c) = packed;
    } else {
#pragma unroll
        for (unsigned k = 0; k < 3; ++k)
            if (c + k < C) row[c + k] = (uint8_t)(packed >> (8 * k));
    }
}

// L lanes share a row and keep it in registers, NQ quads of four logits each; the next row is asked for before this one is
// worked on.
template <int NQ, int L, bool WIDE>
__global__ __launch_bounds__(CLS_THREADS) void ce_saved_kernel(const void *__restrict__ x, const int dtype, const int64_t *__restrict__ cls,
                                                               const float *__restrict__ weight, const unsigned rows,
                                                               const unsigned C, const int64_t ignore_index,
                                                               uint8_t *__restrict__ codes, int8_t *__restrict__ steps,
                                                               double *__restrict__ partials, float *__restrict__ loss_out,
                                                               int32_t *__restrict__ status)
{
    __shared__ double lds[CLS_THREADS / 64];
    constexpr int N = 4 * NQ;
    const unsigned sub = threadIdx.x & (L - 1);
    constexpr unsigned ROWS = CLS_THREADS / L;
    const unsigned stride = gridDim.x * ROWS;
    const float inf = __builtin_huge_valf();
    double num = 0.0, den = 0.0;     // (a lane may walk thousands of rows, and equal ones round to the same side)
    bool bad = false;
    dm::RawRow<NQ, WIDE> next;
    int64_t next_y = 0;
    auto fetch = [&](unsigned row) {
        const unsigned r = min(row, rows - 1);
        next_y = cls[r];
        next = dm::fetch_row<NQ, L, WIDE>(x, (size_t)r * C, sub, C);
    };
    if (blockIdx.x * ROWS < rows) fetch(blockIdx.x * ROWS + threadIdx.x / L);
    // (every lane makes the same trips: the reductions need all lanes of a row)
    for (unsigned r0 = blockIdx.x * ROWS; r0 < rows; r0 += stride) {
        const unsigned row = r0 + threadIdx.x / L;
        const bool live = row < rows;
        const dm::RawRow<NQ, WIDE> raw = next;
        const int64_t y = next_y;
        const float w = live ? row_weight(y, C, ignore_index, weight, &bad) : 0.0f;
        // the row's own logit, once more (by all its lanes, before the next row is asked for: it is waited for first)
        const size_t own_at = (size_t)(live ? row : 0) * C + (w != 0.0f ? (unsigned)y : 0u);
        const float own = WIDE ? static_cast<const float *>(x)[own_at]
                          : dtype == DM_BF16 ? (float)static_cast<const dm::bf16_t *>(x)[own_at] : (float)static_cast<const dm::half_t *>(x)[own_at];
        if (r0 + stride < rows) fetch(row + stride);
        float v[N];
        dm::raw_values<NQ, WIDE>(raw, dtype, v);
        float mx = -inf, low = inf;
        if (codes) {
            // (logits of the row that were read twice do not change its smallest)
#pragma unroll
            for (int j = 0; j < N; ++j) low = __builtin_amdgcn_fmed3f(low, v[j], -inf);
            low = -dm::largest<L>(-low);
        }
        dm::place_row<NQ, L>(v, sub, C, -inf);
#pragma unroll
        for (int j = 0; j < N; j += 2) mx = dm::max3(mx, v[j], v[j + 1]);      // (a NaN makes the sum NaN, whatever is found here)
        mx = dm::largest<L>(mx);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) sum += __builtin_amdgcn_exp2f((v[j] - mx) * LOG2E);      // (past the row: exp2(-inf) = 0)
        sum = dm::over_group<L>(sum, dm::Add());
        if (sub == 0 && w != 0.0f) {
            num += (double)(w * ((mx + __builtin_amdgcn_logf(sum) * LN2) - own));
            den += (double)w;
        }
        if (!codes) continue;
        const float high = __builtin_amdgcn_fmed3f(mx, -CE_CLAMP, CE_CLAMP);
        low = __builtin_amdgcn_fmed3f(low, -CE_CLAMP, CE_CLAMP);
        const int e = step_exponent(high, low, CE_COARSEST);
        const float inverse = power_of_two(-e), top = __builtin_rintf(high * inverse);
        // (the clamp changes no byte while the largest lies well inside it: what is below -2^20 is cut off at 255 anyway)
        if (__any(!(__builtin_fabsf(mx) < CE_CLAMP / 2))) {
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = __builtin_amdgcn_fmed3f(v[j], -CE_CLAMP, CE_CLAMP);
        }
        uint8_t *out = codes + (size_t)row * C;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            unsigned packed = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                packed = pack_code(packed, k, __builtin_amdgcn_fmed3f(top - __builtin_rintf(v[4 * q + k] * inverse), 0.0f, 255.0f));
            const unsigned c = 4 * (q * L + sub);
            if (live) store_codes(out, c, C, packed);
        }
        if (sub == 0 && live) steps[row] = (int8_t)(sum == sum ? e : NOT_A_NUMBER);
    }
    if (bad) dm::raise_status(status, DM_ST_LABEL_RANGE);
    const double a = block_sum(num, lds);
    const double b = block_sum(den, lds);
    if (threadIdx.x == 0) ce_sums(a, b, partials, loss_out);
}

// softmax of the decoded row less its own class, times weight and scale: the row's largest decodes to 0, so there is no maximum
// to find, and a byte's exponential is one product and one instruction.
template <int NQ, int L, bool WIDE>
__global__ __launch_bounds__(CLS_THREADS) void ce_from_saved_kernel(const uint8_t *__restrict__ codes, const int8_t *__restrict__ steps,
                                                                    const int64_t *__restrict__ cls, const float *__restrict__ weight,
                                                                    const unsigned rows, const unsigned C,
                                                                    const int64_t ignore_index, const float *__restrict__ inv_weight,
                                                                    const float *__restrict__ grad_loss, const int dtype,
                                                                    void *__restrict__ grad)
{
    typedef unsigned Word __attribute__((aligned(1)));
    constexpr int N = 4 * NQ;
    const unsigned sub = threadIdx.x & (L - 1);
    constexpr unsigned ROWS = CLS_THREADS / L;
    const unsigned stride = gridDim.x * ROWS;
    const float scale = inv_weight[0] * grad_loss[0];
    unsigned next[NQ];
    int next_e = 0;
    int64_t next_y = 0;
    auto fetch = [&](unsigned row) {
        const unsigned r = min(row, rows - 1);
        next_y = cls[r];
        next_e = steps[r];
        const uint8_t *in = codes + (size_t)r * C;
        if (NQ == 1 && L == 1 && C < 4) {
            next[0] = in[0] | (unsigned)in[min(1u, C - 1)] << 8 | (unsigned)in[C - 1] << 16;
            return;
        }
#pragma unroll
        for (int q = 0; q < NQ; ++q) next[q] = *reinterpret_cast<const Word *>(in + min(4 * (q * L + sub), C - 4));
    };
    if (blockIdx.x * ROWS < rows) fetch(blockIdx.x * ROWS + threadIdx.x / L);
    for (unsigned r0 = blockIdx.x * ROWS; r0 < rows; r0 += stride) {
        const unsigned row = r0 + threadIdx.x / L;
        const bool live = row < rows;
        const int64_t y = next_y;
        const int e = next_e;
        float p[N];
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int k = 0; k < 4; ++k) p[4 * q + k] = (float)((next[q] >> (8 * k)) & 255u);
        if (r0 + stride < rows) fetch(row + stride);
        bool bad = false;
        const float w = row_weight(y, C, ignore_index, weight, &bad);
        dm::place_row<NQ, L>(p, sub, C, __builtin_huge_valf());
        const float step = e == NOT_A_NUMBER ? __builtin_nanf("") : -power_of_two(e) * LOG2E;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            p[j] = __builtin_amdgcn_exp2f(p[j] * step);
            sum += p[j];
        }
        sum = dm::over_group<L>(sum, dm::Add());
        const float inv = __builtin_amdgcn_rcpf(sum), ws = w * scale;
        // the place of the row's own logit in the lane's quads (its first is at 4 sub)
        const unsigned hot = w != 0.0f ? (unsigned)y - 4 * sub : 0xFFFFFFFFu;
#pragma unroll
        for (int j = 0; j < N; ++j) p[j] = (p[j] * inv - (hot == (unsigned)(4 * (j >> 2) * L + (j & 3)) ? 1.0f : 0.0f)) * ws;
        if (w == 0.0f) {
#pragma unroll
            for (int j = 0; j < N; ++j) p[j] = 0.0f;
        }
        if (live) dm::store_row<NQ, L, WIDE>(grad, dtype, (size_t)row * C, sub, C, p);
    }
}

// Rows too long for a wavefront's registers: a workgroup per row, which it walks twice (forward: largest, smallest and sum
// of exponentials in one pass, the bytes in the second, out of the cache; backward: the sum, then the gradient).  In a step 354 MB of
// float32 logits of 4096 classes take 144 and 155 us, of 2048 classes in registers 120 and 76: every exponential is taken twice.
constexpr int WIDE_WAVES = CLS_THREADS / 64;

struct RowStats {
    float mx, mn, sum;      // sum of exp(x - mx)
};
__device__ __forceinline__ RowStats join(const RowStats &a, const RowStats &b)
{
    RowStats r;
    r.mx = fmaxf(a.mx, b.mx);
    r.mn = fminf(a.mn, b.mn);
    // (two parts at -infinity have equal maxima: no difference is taken of them, a sum of zero stays zero)
    const float fa = a.mx == r.mx ? 1.0f : __builtin_amdgcn_exp2f((a.mx - r.mx) * LOG2E);
    const float fb = b.mx == r.mx ? 1.0f : __builtin_amdgcn_exp2f((b.mx - r.mx) * LOG2E);
    r.sum = a.sum * fa + b.sum * fb;
    return r;
}

template <typename T>
__global__ __launch_bounds__(CLS_THREADS) void ce_saved_wide_kernel(const T *__restrict__ x, const int64_t *__restrict__ cls,
                                                                    const float *__restrict__ weight, const unsigned rows,
                                                                    const unsigned C, const int64_t ignore_index,
                                                                    uint8_t *__restrict__ codes, int8_t *__restrict__ steps,
                                                                    double *__restrict__ partials, float *__restrict__ loss_out,
                                                                    int32_t *__restrict__ status)
{
    __shared__ RowStats lds[WIDE_WAVES];
    const float inf = __builtin_huge_valf();
    double num = 0.0, den = 0.0;
    bool bad = false;
    for (unsigned row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *lg = x + (size_t)row * C;
        RowStats s{-inf, inf, 0.0f};
        for (unsigned c = 4 * threadIdx.x; c < C; c += 4 * CLS_THREADS) {
            float t[4];
            dm::load_quad(lg, c, C, -inf, t);
            const float m4 = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
            const float m = fmaxf(s.mx, m4);
            const float keep = s.mx == m ? 1.0f : __builtin_amdgcn_exp2f((s.mx - m) * LOG2E);
            float add = 0.0f;
#pragma unroll
            for (unsigned k = 0; k < 4; ++k) {
                // (-infinity adds nothing, also while nothing larger has been met; a NaN, or an infinity over itself, is NaN)
                if (c + k < C) {
                    add += t[k] == -inf ? 0.0f : __builtin_amdgcn_exp2f((t[k] - m) * LOG2E);
                    s.mn = fminf(s.mn, t[k]);
                }
            }
            s.sum = s.sum * keep + add;
            s.mx = m;
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1)
            s = join(s, RowStats{__shfl_xor(s.mx, off), __shfl_xor(s.mn, off), __shfl_xor(s.sum, off)});
        __syncthreads();                 // (the previous row's use of lds is over)
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
        __syncthreads();
        s = lds[0];
        for (int w = 1; w < WIDE_WAVES; ++w) s = join(s, lds[w]);
        const float sum = s.mx == -inf ? __builtin_nanf("") : s.sum;       // (nothing but -infinity: NaN, as in a softmax)
        if (threadIdx.x == 0) {
            const int64_t y = cls[row];
            const float w = row_weight(y, C, ignore_index, weight, &bad);
            if (w != 0.0f) {
                num += (double)(w * ((s.mx + __builtin_amdgcn_logf(sum) * LN2) - (float)lg[y]));
                den += (double)w;
            }
        }
        if (!codes) continue;
        const float high = fminf(fmaxf(s.mx, -CE_CLAMP), CE_CLAMP), low = fminf(fmaxf(s.mn, -CE_CLAMP), CE_CLAMP);
        const int e = step_exponent(high, low, CE_COARSEST);
        const float inverse = power_of_two(-e), top = __builtin_rintf(high * inverse);
        uint8_t *out = codes + (size_t)row * C;
        for (unsigned c = 4 * threadIdx.x; c < C; c += 4 * CLS_THREADS) {
            float t[4];
            dm::load_quad(lg, c, C, -inf, t);
            unsigned packed = 0;
#pragma unroll
            for (unsigned k = 0; k < 4; ++k) {
                const float z = __builtin_amdgcn_fmed3f(t[k], -CE_CLAMP, CE_CLAMP);
                packed = pack_code(packed, k, __builtin_amdgcn_fmed3f(top - __builtin_rintf(z * inverse), 0.0f, 255.0f));
            }
            store_codes(out, c, C, packed);
        }
        if (threadIdx.x == 0) steps[row] = (int8_t)(sum == sum ? e : NOT_A_NUMBER);
    }
    if (bad) dm::raise_status(status, DM_ST_LABEL_RANGE);
    if (threadIdx.x == 0) ce_sums(num, den, partials, loss_out);
}

template <typename T>
__global__ __launch_bounds__(CLS_THREADS) void ce_from_saved_wide_kernel(const uint8_t *__restrict__ codes,
                                                                         const int8_t *__restrict__ steps,
                                                                         const int64_t *__restrict__ cls,
                                                                         const float *__restrict__ weight, const unsigned rows,
                                                                         const unsigned C, const int64_t ignore_index,
                                                                         const float *__restrict__ inv_weight,
                                                                         const float *__restrict__ grad_loss, T *__restrict__ grad)
{
    __shared__ float lds[WIDE_WAVES];
    const float scale = inv_weight[0] * grad_loss[0];
    for (unsigned row = blockIdx.x; row < rows; row += gridDim.x) {
        const size_t base = (size_t)row * C;
        const int e = steps[row];
        const float step = e == NOT_A_NUMBER ? __builtin_nanf("") : -power_of_two(e) * LOG2E;
        float sum = 0.0f;
        for (unsigned c = 4 * threadIdx.x; c < C; c += 4 * CLS_THREADS) {
            float t[4];
            dm::load_quad(codes + base, c, C, __builtin_huge_valf(), t);
#pragma unroll
            for (int k = 0; k < 4; ++k) sum += __builtin_amdgcn_exp2f(t[k] * step);
        }
        sum = dm::over_group<64>(sum, dm::Add());
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
        __syncthreads();
        sum = lds[0];
        for (int w = 1; w < WIDE_WAVES; ++w) sum += lds[w];
        bool bad = false;
        const int64_t y = cls[row];
        const float w = row_weight(y, C, ignore_index, weight, &bad);
        const float inv = __builtin_amdgcn_rcpf(sum), ws = w * scale;
        for (unsigned c = 4 * threadIdx.x; c < C; c += 4 * CLS_THREADS) {
            float t[4], g[4];
            dm::load_quad(codes + base, c, C, __builtin_huge_valf(), t);
#pragma unroll
            for (unsigned k = 0; k < 4; ++k)
                g[k] = w == 0.0f ? 0.0f : (__builtin_amdgcn_exp2f(t[k] * step) * inv - ((int64_t)(c + k) == y ? 1.0f : 0.0f)) * ws;
            dm::store_quad(grad + base, c, C, g);
        }
    }
}

// ---- host side ----

template <typename T>
void launch_focal_saved(const void *logits, const int64_t *cls, unsigned n, unsigned C, unsigned rows, const FocalParams &fp,
                        uint8_t *codes, int32_t *heads, double *partials, float *loss_out, int32_t *status, int blocks, hipStream_t st)
{
    auto kernel = fp.gamma == 2.0f ? (C == 1 ? focal_saved_kernel<T, true, true> : focal_saved_kernel<T, true, false>)
                                   : (C == 1 ? focal_saved_kernel<T, false, true> : focal_saved_kernel<T, false, false>);
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(CLS_THREADS), 0, st, static_cast<const T *>(logits), cls, n, C, rows, fp,
                       reinterpret_cast<unsigned *>(codes), heads, partials, loss_out, status);
}
template <typename T>
void launch_focal_from_saved(const uint8_t *codes, const int32_t *heads, const int64_t *cls, unsigned n, unsigned C, unsigned rows,
                             const FocalParams &fp, const float *grad_loss, void *grad, int blocks, hipStream_t st)
{
    auto kernel = fp.gamma == 2.0f ? (C == 1 ? focal_from_saved_kernel<T, true, true> : focal_from_saved_kernel<T, true, false>)
                                   : (C == 1 ? focal_from_saved_kernel<T, false, true> : focal_from_saved_kernel<T, false, false>);
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(CLS_THREADS), 0, st, reinterpret_cast<const unsigned *>(codes), heads, cls, n, C,
                       rows, fp, grad_loss, static_cast<T *>(grad));
}

// Workgroups for a number of trips: as many as the chip holds at once (six per CU at these kernels' registers), each with the
// same number of trips.  (256 x 900 x 91 logits are 5119 trips of the focal kernels: with 1707 workgroups, the most of which
// each makes three, 171 of them wait for the others' end, 27.9 us; 1280 that make four take 26.8.)
// One for up to `alone` trips, which then makes the loss itself.
unsigned even_blocks(unsigned trips, unsigned alone)
{
    if (trips <= alone) return 1;
    constexpr unsigned RESIDENT = 6 * 256;
    static_assert(RESIDENT <= (unsigned)CLS_MAX_BLOCKS, "a partial sum for each");
    const unsigned each = std::max(1u, (trips + RESIDENT - 1) / RESIDENT);
    return std::max(1u, (trips + each - 1) / each);
}

// Trips of a forward pass that one workgroup makes by itself: calls of one, two and three trips of the focal kernel (4096 logits each)
// take 8.2, 8.2 and 9.7 us among others instead of 8.3, 11.0 and 11.1, of four 11.3 instead of 11.2; four trips of the cross
// entropy 8.0 to 9.9 instead of 11.1, eight 9.3 to 17.3.
constexpr unsigned FOCAL_ALONE = 3, CE_ALONE = 4;

int focal_blocks(unsigned n, unsigned alone)
{
    const unsigned per_block = BLOCK * BLOCKS_AT_A_TIME;
    return (int)even_blocks(n / per_block + (n % per_block != 0), alone);
}

constexpr unsigned WIDEST = 2048;      // logits of a row that a wavefront keeps in registers

// Quads of four logits per lane, and lanes per row.  Two quads and twice the lanes make longer runs of stores: the backward pass
// takes 118, 119 and 88 us for 354 MB of float32 gradients of 24, 32 and 64 classes, with twelve or sixteen logits per lane 153, 179
// and 126.  The forward pass of 16-bit logits is bound by instructions, and lanes behind the row's end are wasted ones: 12, 24
// and 48 classes take 79, 73 and 67 us for 177 MB with twelve logits per lane, 94, 95 and 94 with eight.  (1537 to 1792 classes take
// the form of 2048, an eighth of its quads empty: one of seven quads has not been built.)
struct Form {
    int NQ, L;
};
Form ce_form(unsigned C, bool filled)      // filled: no more lanes than the row needs
{
    if (C <= 8) return {C <= 4 ? 1 : 2, 1};
    if (C <= 16) return filled && C <= 12 ? Form{3, 1} : Form{2, 2};
    if (C <= 32) return filled && C <= 24 ? Form{3, 2} : Form{2, 4};
    if (C <= 64) return filled && C <= 48 ? Form{3, 4} : Form{2, 8};
    if (C <= 128) return {C <= 96 ? 3 : 4, 8};
    if (C <= 256) return {C <= 192 ? 3 : 4, 16};
    if (C <= 512) return {C <= 384 ? 3 : 4, 32};
    if (C <= 1024) return {C <= 768 ? 3 : 4, 64};
    return {C <= 1280 ? 5 : C <= 1536 ? 6 : 8, 64};
}
template <bool FILLED, typename F>
void with_ce_form(unsigned C, F &&f)
{
    auto as = [&](auto nq, auto l) { f(nq, l); };
#define DM_FORM(NQ_, L_) as(std::integral_constant<int, NQ_>(), std::integral_constant<int, L_>())
    const Form form = ce_form(C, FILLED);
    if constexpr (FILLED) {
        if (form.NQ == 3 && form.L <= 4) return form.L == 1 ? DM_FORM(3, 1) : form.L == 2 ? DM_FORM(3, 2) : DM_FORM(3, 4);
    }
    switch (form.L) {
    case 1: return form.NQ == 1 ? DM_FORM(1, 1) : DM_FORM(2, 1);
    case 2: return DM_FORM(2, 2);
    case 4: return DM_FORM(2, 4);
    case 8: return form.NQ == 2 ? DM_FORM(2, 8) : form.NQ == 3 ? DM_FORM(3, 8) : DM_FORM(4, 8);
    case 16: return form.NQ == 3 ? DM_FORM(3, 16) : DM_FORM(4, 16);
    case 32: return form.NQ == 3 ? DM_FORM(3, 32) : DM_FORM(4, 32);
    default:
        switch (form.NQ) {
        case 3: return DM_FORM(3, 64);
        case 4: return DM_FORM(4, 64);
        case 5: return DM_FORM(5, 64);
        case 6: return DM_FORM(6, 64);
        default: return DM_FORM(8, 64);
        }
    }
#undef DM_FORM
}
unsigned ce_blocks(unsigned rows, unsigned C, bool filled, unsigned alone)
{
    const unsigned rows_per_block = C <= WIDEST ? (unsigned)(CLS_THREADS / ce_form(C, filled).L) : 1u;
    return even_blocks(rows / rows_per_block + (rows % rows_per_block != 0), C <= WIDEST ? alone : 0);
}
template <typename T>
void launch_ce_saved(const void *logits, int dtype, const int64_t *cls, const float *weight, unsigned rows, unsigned C, int64_t ignore_index,
                     uint8_t *codes, int8_t *steps, double *partials, float *loss_out, int32_t *status, unsigned blocks, hipStream_t st)
{
    if (C > WIDEST) {
        hipLaunchKernelGGL(ce_saved_wide_kernel<T>, dim3(blocks), dim3(CLS_THREADS), 0, st, static_cast<const T *>(logits), cls, weight,
                           rows, C, ignore_index, codes, steps, partials, loss_out, status);
        return;
    }
    with_ce_form<sizeof(T) == 2>(C, [&](auto nq, auto l) {
        hipLaunchKernelGGL((ce_saved_kernel<decltype(nq)::value, decltype(l)::value, sizeof(T) == 4>), dim3(blocks), dim3(CLS_THREADS), 0,
                           st, logits, dtype, cls, weight, rows, C, ignore_index, codes, steps, partials, loss_out, status);
    });
}
template <typename T>
void launch_ce_from_saved(const uint8_t *codes, const int8_t *steps, int dtype, const int64_t *cls, const float *weight, unsigned rows,
                          unsigned C, int64_t ignore_index, const float *inv_weight, const float *grad_loss, void *grad, unsigned blocks,
                          hipStream_t st)
{
    if (C > WIDEST) {
        hipLaunchKernelGGL(ce_from_saved_wide_kernel<T>, dim3(blocks), dim3(CLS_THREADS), 0, st, codes, steps, cls, weight, rows, C,
                           ignore_index, inv_weight, grad_loss, static_cast<T *>(grad));
        return;
    }
    with_ce_form<false>(C, [&](auto nq, auto l) {
        hipLaunchKernelGGL((ce_from_saved_kernel<decltype(nq)::value, decltype(l)::value, sizeof(T) == 4>), dim3(blocks), dim3(CLS_THREADS),
                           0, st, codes, steps, cls, weight, rows, C, ignore_index, inv_weight, grad_loss, dtype, grad);
    });
}

bool known(int dtype) { return dtype == DM_F32 || dtype == DM_BF16 || dtype == DM_F16; }

int check_from_saved(const uint8_t *codes, const void *marks, int dtype, const int64_t *target_cls, int64_t rows, int C,
                     const float *grad_loss, const void *grad_out)
{
    if (rows < 0 || C < 1 || !known(dtype)) return DM_E_INVALID_ARG;
    if (rows > 0 && (!codes || !marks || !target_cls || !grad_loss || !grad_out)) return DM_E_INVALID_ARG;
    if ((unsigned long long)rows * (unsigned long long)C >= (1ull << 31)) return DM_E_UNSUPPORTED;
    return DM_OK;
}

}  // namespace

extern "C" int dm_focal_loss_saved(const void *logits, int dtype, const int64_t *target_cls, int64_t rows, int C, float alpha,
                                   float gamma, float scale, int64_t ignore_index, int use_ignore, float *loss_out,
                                   uint8_t *codes, int32_t *heads, double *partials, int32_t *status, void *stream)
{
    int rc = check_common(logits, target_cls, rows, C, loss_out, partials, status);
    if (rc != DM_OK) return rc;
    if (!known(dtype) || (codes != nullptr) != (heads != nullptr) || gamma < 0.0f) return DM_E_INVALID_ARG;
    if (((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(heads)) & 3) != 0) return DM_E_INVALID_ARG;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const unsigned n = (unsigned)(rows * C);
    const int blocks = focal_blocks(n, FOCAL_ALONE);
    const FocalParams fp{alpha, gamma, scale, ignore_index, use_ignore};
    auto launch = dtype == DM_F32 ? launch_focal_saved<float> : dtype == DM_BF16 ? launch_focal_saved<dm::bf16_t> : launch_focal_saved<dm::half_t>;
    launch(logits, target_cls, n, (unsigned)C, (unsigned)rows, fp, codes, heads, partials, loss_out, status, blocks, st);
    rc = dm::check_hip(hipGetLastError(), "focal_saved_kernel launch");
    if (rc != DM_OK || blocks == 1) return rc;
    hipLaunchKernelGGL(cls_loss_finish_kernel<true>, dim3(1), dim3(CLS_THREADS), 0, st, partials, blocks, scale, loss_out);
    return dm::check_hip(hipGetLastError(), "cls_loss_finish_kernel launch");
}

extern "C" int dm_focal_loss_from_saved(const uint8_t *codes, const int32_t *heads, int dtype, const int64_t *target_cls,
                                        int64_t rows, int C, float alpha, float gamma, float scale, int64_t ignore_index,
                                        int use_ignore, const float *grad_loss, void *grad_out, void *stream)
{
    const int rc = check_from_saved(codes, heads, dtype, target_cls, rows, C, grad_loss, grad_out);
    if (rc != DM_OK) return rc;
    if (gamma < 0.0f) return DM_E_INVALID_ARG;
    if (((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(heads)) & 3) != 0) return DM_E_INVALID_ARG;
    if (rows == 0) return DM_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const unsigned n = (unsigned)(rows * C);
    const int blocks = focal_blocks(n, 0);
    const FocalParams fp{alpha, gamma, scale, ignore_index, use_ignore};
    auto launch = dtype == DM_F32 ? launch_focal_from_saved<float>
                  : dtype == DM_BF16 ? launch_focal_from_saved<dm::bf16_t> : launch_focal_from_saved<dm::half_t>;
    launch(codes, heads, target_cls, n, (unsigned)C, (unsigned)rows, fp, grad_loss, grad_out, blocks, st);
    return dm::check_hip(hipGetLastError(), "focal_from_saved_kernel launch");
}

extern "C" int dm_cross_entropy_saved(const void *logits, int dtype, const int64_t *target_cls, const float *weight, int64_t rows,
                                      int C, int64_t ignore_index, float *loss_out, uint8_t *codes, int8_t *steps,
                                      double *partials, int32_t *status, void *stream)
{
    int rc = check_common(logits, target_cls, rows, C, loss_out, partials, status);
    if (rc != DM_OK) return rc;
    if (!known(dtype) || (codes != nullptr) != (steps != nullptr)) return DM_E_INVALID_ARG;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const unsigned blocks = ce_blocks((unsigned)rows, (unsigned)C, dtype != DM_F32, CE_ALONE);
    auto launch = dtype == DM_F32 ? launch_ce_saved<float> : dtype == DM_BF16 ? launch_ce_saved<dm::bf16_t> : launch_ce_saved<dm::half_t>;
    launch(logits, dtype, target_cls, weight, (unsigned)rows, (unsigned)C, ignore_index, codes, steps, partials, loss_out, status, blocks, st);
    rc = dm::check_hip(hipGetLastError(), "ce_saved_kernel launch");
    if (rc != DM_OK || blocks == 1) return rc;
    hipLaunchKernelGGL(cls_loss_finish_kernel<false>, dim3(1), dim3(CLS_THREADS), 0, st, partials, (int)blocks, 1.0f, loss_out);
    return dm::check_hip(hipGetLastError(), "cls_loss_finish_kernel launch");
}

extern "C" int dm_cross_entropy_from_saved(const uint8_t *codes, const int8_t *steps, int dtype, const int64_t *target_cls,
                                           const float *weight, int64_t rows, int C, int64_t ignore_index, const float *inv_weight,
                                           const float *grad_loss, void *grad_out, void *stream)
{
    const int rc = check_from_saved(codes, steps, dtype, target_cls, rows, C, grad_loss, grad_out);
    if (rc != DM_OK) return rc;
    if (rows == 0) return DM_OK;
    if (!inv_weight) return DM_E_INVALID_ARG;
    auto launch = dtype == DM_F32 ? launch_ce_from_saved<float>
                  : dtype == DM_BF16 ? launch_ce_from_saved<dm::bf16_t> : launch_ce_from_saved<dm::half_t>;
    launch(codes, steps, dtype, target_cls, weight, (unsigned)rows, (unsigned)C, ignore_index, inv_weight, grad_loss, grad_out,
           ce_blocks((unsigned)rows, (unsigned)C, false, 0), static_cast<hipStream_t>(stream));
    return dm::check_hip(hipGetLastError(), "ce_from_saved_kernel launch");
}
