// Balance loss of expert routers with per-expert counts, and its gradient, for gfx950 (MI355X).
//
// Per group (a set of router logits, or one image of it) of n rows that count, over E experts:
//     f_e = E c_e / sum c,   P_e = 1/n sum_rows p_e,   balance = sum_e f_e P_e,   z = 1/n sum_rows logsumexp(x)^2
// with c_e the number of rows whose top k logits include e.  The gradient
//     dx_e = g_balance / n * p_e (f_e - sum_j f_j p_j) + g_z / n * 2 logsumexp(x) p_e
// needs the counts of the whole group, so forward and backward each read the logits once: nothing per row is kept.  f is
// stored less one (the p of a row sum to one, so a constant drops out): near balance f_e - sum f p would lose its digits.
//
// Forward: workgroups walk chunks of an image's rows, a group of lanes per row; sums over rows stay in registers of the
// lane that owns the expert (in float32 for RUN rows, then they go to 64 bits in shared memory), and leave once per workgroup,
// into a slot of the workspace.  A second kernel adds the slots in index order in 64 bits: no two lanes add to one place, the
// same bits every run.  A group that one workgroup walks needs no second kernel.
//
// What bounds it, as measured (a copy of a GiB runs at 5.1 TB/s, a kernel of a few workgroups takes 4 us among others):
//   memory          6 x 256 x 900 x 64 float32, top 4 (354 MB): forward 107 us, sums and loss 5 each, backward 123 (708 MB at
//                   5.8 TB/s).  Forward, sums and loss by themselves, over and over, take 75 (4.7 TB/s); in a step they wait for the
//                   gradients of the one before, of which the caches hold up to 256 MB, to be written.
//   instructions    16-bit logits with many choices: 2 x 64 x 1050 x 160 bfloat16, sigmoid scores, top 8 (43 MB): forward 36 us,
//                   sums and loss 7, backward 27; 6 x 256 x 900 x 64 bfloat16, softmax, top 4 (177 MB): 70, 9 and 89; counts alone
//                   of 256 x 900 x 256, top 8 (118 MB): 44 us, the vector units busy four fifths of it.  Of the 20 instructions per
//                   logit 6 keep the list and 3 make the order; taking the heads off the lists (for the top 8 seven rounds that
//                   wait for one another) costs a lane about a hundred a row, however few logits it holds.
//   the launches    6 x 64 x 600 x 16 float32 (15 MB): 11.2, 5.4 and 8.6 us; 1 x 300 x 8, where one workgroup makes the loss as
//                   well: 6.1 and 2.8.
#include <algorithm>
#include <climits>

#include "lanes.h"

namespace {

constexpr int RT_THREADS = 256;
constexpr int RT_WAVES = RT_THREADS / 64;
constexpr int RT_MAX_EXPERTS = 1024;
constexpr unsigned RUN = 64;         // rows whose scores a lane adds in float32: equal ones round to the same side
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// One set as the kernels see it: `images` images of Q rows (a contiguous set asked for as one group is one image of B * Q
// rows), each cut into `chunks` chunks of `chunk_rows`.
struct RouterSetK {
    const void *logits;
    const uint8_t *mask;
    const int64_t *experts;
    void *grad;
    int64_t image_stride;      // elements
    unsigned Q, images, chunks, chunk_rows;
    unsigned first_block;      // of the set in the launch; its slots start there too
};
struct RouterSets {
    RouterSetK s[DM_MAX_SETS_PER_LAUNCH];
    int S;
    unsigned E, k;
    unsigned per_image;        // a group per image
    unsigned first_group[DM_MAX_SETS_PER_LAUNCH];
};

// Words of a workgroup's slot: sum of p per expert (float), count per expert (uint32), sum of lse^2 (double), rows (uint32).
__host__ __device__ constexpr unsigned slot_words(unsigned E) { return 2 * E + 4; }

struct Place {
    int set;
    unsigned image, row0, rows;      // the rows row0 .. row0 + rows - 1 of the image
};
__device__ __forceinline__ Place place_of(const RouterSets &a, unsigned block)
{
    int set = 0;
    while (set + 1 < a.S && block >= a.s[set + 1].first_block) ++set;
    const RouterSetK &s = a.s[set];
    const unsigned local = block - s.first_block;
    const unsigned image = local / s.chunks, row0 = (local - image * s.chunks) * s.chunk_rows;
    return Place{set, image, row0, row0 < s.Q ? min(s.chunk_rows, s.Q - row0) : 0u};
}

// The scores of a row before they are divided by their sum, and what turns them into p: w_e / sum w.
// Sigmoid: sigmoid(x) times a constant of the row that keeps the largest from underflowing: with c = min(max x, 0),
// t = exp(-|x| - c), sigmoid(x) exp(-c) = (x >= 0 ? 1 : t) / (1 + t exp(c)).  `rest` = 1 - sigmoid(x).
__device__ __forceinline__ float softmax_weight(float x, float mx) { return __builtin_amdgcn_exp2f((x - mx) * LOG2E); }
// All of a lane's.  exp(x - max) as 2^(x log2 e - (max log2 e)): the rounding of the product with the row's largest is the
// same for the whole row, it drops out of p and is within the rounding of the logarithm of the sum.  Not so far from zero,
// where that rounding is a step of the exponent and more.
template <int N>
__device__ __forceinline__ void softmax_weights(float (&x)[N], float mx)
{
    if (__any(!(__builtin_fabsf(mx) < 1024.0f))) {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = softmax_weight(x[j], mx);
        return;
    }
    const float base = mx * LOG2E;
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[j], LOG2E, -base));
}
template <int N, bool REST>
__device__ __forceinline__ void sigmoid_weights(float (&x)[N], float mx, float (&rest)[REST ? N : 1])
{
    auto weigh = [&](int j, float t, float r) {
        const bool up = x[j] >= 0.0f;
        if (REST) rest[REST ? j : 0] = (up ? t : 1.0f) * r;
        x[j] = (up ? 1.0f : t) * r;
    };
    if (__any(mx < 0.0f)) {
        const float c = fminf(mx, 0.0f), exp_c = __builtin_amdgcn_exp2f(c * LOG2E);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float t = __builtin_amdgcn_exp2f((-__builtin_fabsf(x[j]) - c) * LOG2E);
            weigh(j, t, __builtin_amdgcn_rcpf(__builtin_fmaf(t, exp_c, 1.0f)));
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float t = __builtin_amdgcn_exp2f(-__builtin_fabsf(x[j]) * LOG2E);
        weigh(j, t, __builtin_amdgcn_rcpf(1.0f + t));
    }
}

// What the choice compares: an order in which no two of a row are equal where that can be had, and its least.
//   float32   the logits, with what is never chosen (-infinity, NaN) at -infinity.  Equal ones are seen to afterwards.
//   16 bits   equal logits are frequent, and are to go to the lowest index: the logit as a 16-bit number of the same order
//             (sign and magnitude to two's complement, which also makes the two zeros one), two at a time, in the upper half
//             of an int, and 1023 - expert in the lower; -infinity lies below `least`, a NaN is put there
template <bool WIDE>
struct Order;
template <>
struct Order<true> {
    typedef float Type;
    static __device__ __forceinline__ Type never() { return -__builtin_huge_valf(); }
    static __device__ __forceinline__ Type above_all() { return __builtin_huge_valf(); }
    static __device__ __forceinline__ Type least(int) { return -__FLT_MAX__; }
    static __device__ __forceinline__ float logit(Type y, int) { return y; }
};
template <>
struct Order<false> {
    typedef int Type;
    typedef short Pair __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ Type never() { return INT_MIN; }
    static __device__ __forceinline__ Type above_all() { return INT_MAX; }
    static __device__ __forceinline__ unsigned infinity(int dtype) { return dtype == DM_BF16 ? 0x7F80u : 0x7C00u; }
    static __device__ __forceinline__ Type least(int dtype) { return (int)((1u - infinity(dtype)) << 16); }
    static __device__ __forceinline__ float logit(Type y, int dtype)
    {
        const int v = y >> 16, sign = v >> 31;
        const unsigned u = (unsigned)((v ^ sign) - sign) | ((unsigned)sign & 0x8000u);
        return dtype == DM_BF16 ? __uint_as_float(u << 16) : (float)__builtin_bit_cast(dm::half_t, (uint16_t)u);
    }
    // two logits; low: 1023 - expert of each; over: not 0 for a NaN
    static __device__ __forceinline__ void of(unsigned raw, unsigned low0, unsigned low1, unsigned inf2, Type *y0, Type *y1, unsigned *over)
    {
        const unsigned magnitude = raw & 0x7FFF7FFFu;
        const Pair sign = __builtin_bit_cast(Pair, raw) >> 15;
        const unsigned key = __builtin_bit_cast(unsigned, __builtin_bit_cast(Pair, magnitude ^ __builtin_bit_cast(unsigned, sign)) - sign);
        unsigned beyond;
        asm("v_pk_sub_u16 %0, %1, %2 clamp" : "=v"(beyond) : "v"(magnitude), "v"(inf2));
        *over |= beyond;
        *y0 = (int)(key << 16 | low0);
        *y1 = (int)((key & 0xFFFF0000u) | low1);
    }
};

// A lane's logits in their order.
template <int NQ, int L>
__device__ __forceinline__ void in_order(const dm::RawRow<NQ, true> &raw, int dtype, unsigned sub, unsigned E, bool counts,
                                         float (&y)[4 * NQ], bool *nan)
{
    const float ninf = -__builtin_huge_valf();
    dm::row_values<NQ, L, true>(raw, dtype, sub, E, ninf, y);
    if (!counts) {
#pragma unroll
        for (int j = 0; j < 4 * NQ; ++j) y[j] = ninf;
    }
    *nan = false;
#pragma unroll
    for (int j = 0; j < 4 * NQ; ++j) {
        const bool is = y[j] != y[j];
        *nan |= is;
        y[j] = is ? ninf : y[j];
    }
}
template <int NQ, int L>
__device__ __forceinline__ void in_order(dm::RawRow<NQ, false> &raw, int dtype, unsigned sub, unsigned E, bool counts,
                                         int (&y)[4 * NQ], bool *nan)
{
    const unsigned inf = Order<false>::infinity(dtype), inf2 = inf << 16 | inf, pair = inf2 | 0x80008000u;
    dm::place_raw<NQ, L>(raw, sub, E, pair);
    if (!counts) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) raw.q[q][0] = raw.q[q][1] = pair;
    }
    unsigned over = 0;
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const unsigned low = 1023u - (4 * (q * L + sub) + 2 * h);
            Order<false>::of(raw.q[q][h], low, low - 1, inf2, &y[4 * q + 2 * h], &y[4 * q + 2 * h + 1], &over);
        }
    *nan = false;                                              // (the scores are made of the logits as they came)
    if (__any(over)) {
#pragma unroll
        for (int j = 0; j < 4 * NQ; ++j)
            if (((raw.q[j >> 2][(j >> 1) & 1] >> (16 * (j & 1))) & 0x7FFFu) > inf) y[j] = Order<false>::never();
    }
}

// What a group's loss is made of, and where it goes.
struct Results {
    const int64_t *given_counts;
    float *balance, *z;
    int64_t *counts;
    float *slope, *inv_rows;
};
constexpr int LOSS_THREADS = 256, LOSS_WAVES = LOSS_THREADS / 64, LOSS_EACH = RT_MAX_EXPERTS / LOSS_THREADS;
struct LossSums {
    unsigned long long rows[LOSS_WAVES], total[LOSS_WAVES];
    double z[LOSS_WAVES], dot[LOSS_WAVES];
};

// The loss of a group, and what its gradient needs, by LOSS_THREADS threads.  A thread brings the counts and the sums of p of its
// experts tid, tid + LOSS_THREADS, ..., and its share of the rows that count and of the sum of lse^2.
__device__ __forceinline__ void group_loss(const Results &out, const unsigned E, const size_t group, const long long (&counts)[LOSS_EACH],
                                           const double (&sums)[LOSS_EACH], unsigned long long rows, double zs, LossSums &lds)
{
    const unsigned tid = threadIdx.x;
    double dot = 0.0;
    unsigned long long total = 0;
#pragma unroll
    for (int j = 0; j < LOSS_EACH; ++j) {                      // (0 behind the last expert)
        dot += (double)counts[j] * sums[j];
        total += (unsigned long long)counts[j];
    }
    // over the wave, then over the waves, in every thread
    rows = dm::over_group<64>(rows, dm::Add());
    total = dm::over_group<64>(total, dm::Add());
    zs = dm::over_group<64>(zs, dm::Add());
    dot = dm::over_group<64>(dot, dm::Add());
    if ((tid & 63) == 0) {
        lds.rows[tid >> 6] = rows;
        lds.total[tid >> 6] = total;
        lds.z[tid >> 6] = zs;
        lds.dot[tid >> 6] = dot;
    }
    __syncthreads();
    rows = lds.rows[0];
    total = lds.total[0];
    zs = lds.z[0];
    dot = lds.dot[0];
#pragma unroll
    for (int w = 1; w < LOSS_WAVES; ++w) {
        rows += lds.rows[w];
        total += lds.total[w];
        zs += lds.z[w];
        dot += lds.dot[w];
    }
    const long long all = (long long)total;
    const double inv_n = rows ? 1.0 / (double)rows : 0.0;
    const double per_count = all > 0 ? (double)E / (double)all : 0.0;
    if (tid == 0) {
        out.balance[group] = (float)(dot * per_count * inv_n);
        if (out.z) out.z[group] = (float)(zs * inv_n);
        out.inv_rows[group] = (float)inv_n;
    }
#pragma unroll
    for (int j = 0; j < LOSS_EACH; ++j) {
        const unsigned e = tid + j * LOSS_THREADS;
        if (e < E) out.slope[group * E + e] = all > 0 ? (float)((double)counts[j] * per_count - 1.0) : 0.0f;
    }
}

// K: the longest list of largest logits that a lane keeps, k at most; 16: any k (a lane has no more logits than that).
//
// The choice.  A lane inserts its logits into a sorted list of its K largest, one instruction per place (the new place i is
// the median of the old i - 1, the old i and the logit); then k times the largest head of the row's lanes is taken off its
// list, and the last one taken, T, is the row's k-th largest: the experts with a logit of at least T are the chosen ones.
// Where equal logits lie across the border, or T came out too low because equal heads went together, more than k are: those
// rows are chosen again, one by one (float32 only, 16-bit logits are made unequal): k rounds over all logits, each a maximum, a
// search for its lowest place and a selection.  With lists 6 x 256 x 900 x 64 float32 take, sums and loss among them, 73, 78, 90 and
// 125 us for the top 2, 4, 8 and 16 and 148 for the top 17; with such rounds for every row the top 17 took 320.
//
// The next row is asked for before this one is worked on, and no branch lies between its loads: one row in flight is what a
// lane has registers for (two were slower), and with three workgroups per CU that keeps the memory busy.
//
// whole: every group has one workgroup, which makes the group's loss itself instead of leaving its sums.
template <int NQ, int L, int K, bool WIDE, bool COUNT_ONLY>
__global__ __launch_bounds__(RT_THREADS) void router_forward_kernel(const RouterSets a, const int dtype, const int sigmoid,
                                                                    const int whole, unsigned *__restrict__ slots,
                                                                    const Results out, int32_t *__restrict__ status)
{
    constexpr int N = 4 * NQ;                                  // logits of a row per lane
    constexpr int PARTS = L <= 16 ? 4 : 64 / L;                // partial sums of p that a wave leaves
    constexpr unsigned WIDTH = N * L;                          // E, rounded up to what the lanes hold
    __shared__ unsigned hist[WIDTH];
    __shared__ double psum_lds[COUNT_ONLY ? 1 : RT_WAVES * PARTS][COUNT_ONLY ? 1 : WIDTH];
    __shared__ double z_lds[RT_WAVES];
    __shared__ unsigned n_lds[RT_WAVES];
    __shared__ LossSums loss_lds;
    const unsigned E = a.E, k = a.k;
    const float ninf = -__builtin_huge_valf();
    for (unsigned e = threadIdx.x; e < WIDTH; e += RT_THREADS) hist[e] = 0;
    if constexpr (!COUNT_ONLY)
        for (unsigned i = threadIdx.x; i < RT_WAVES * PARTS * WIDTH; i += RT_THREADS) psum_lds[0][i] = 0.0;
    __syncthreads();

    const Place at = place_of(a, blockIdx.x);
    const RouterSetK &set = a.s[at.set];
    const size_t image_at = (size_t)at.image * (size_t)set.image_stride;
    const size_t image_row = (size_t)at.image * set.Q;
    const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned sub = lane & (L - 1);
    constexpr unsigned ROWS = RT_THREADS / L;                  // rows of the workgroup at a time
    float psum[N] = {};
    unsigned cnt[N] = {};
    double z = 0.0;
    unsigned n = 0;
    bool bad = false;

    // (every lane makes the same trips: the reductions need all lanes of a row's group)
    const unsigned local = threadIdx.x / L;
    dm::RawRow<NQ, WIDE> next;
    uint8_t next_counts = 1;
    auto fetch = [&](unsigned r) {
        const size_t row = (size_t)at.row0 + (r < at.rows ? r : 0);
        next = dm::fetch_row<NQ, L, WIDE>(set.logits, image_at + row * E, sub, E);
        if (set.mask) next_counts = set.mask[image_row + row];
    };
    if (at.rows) fetch(local);
    unsigned r0 = 0, run = 0;
    do {
        run = COUNT_ONLY ? at.rows : min(at.rows, r0 + RUN * ROWS);
        for (; r0 < run; r0 += ROWS) {
            const unsigned r = r0 + local;
            const bool there = r < at.rows;
            const size_t row = (size_t)at.row0 + (there ? r : 0);
            dm::RawRow<NQ, WIDE> raw = next;
            const bool counts = there && next_counts != 0;
            if (r0 + ROWS < at.rows) fetch(r + ROWS);
            typedef Order<WIDE> O;
            typename O::Type y[N];
            bool nan;
            in_order<NQ, L>(raw, dtype, sub, E, counts, y, &nan);
            constexpr int PLACES = K < N ? K : N;
            typename O::Type list[PLACES];
#pragma unroll
            for (int i = 0; i < PLACES; ++i) list[i] = O::never();
#pragma unroll
            for (int j = 0; j < N; ++j) {
#pragma unroll
                for (int i = PLACES - 1; i >= 1; --i)
                    if (i <= j) list[i] = dm::median(list[i - 1], list[i], y[j]);      // (place j is empty before the j-th)
                list[0] = j ? dm::median(list[0], y[j], O::above_all()) : y[0];
            }
            const typename O::Type top = dm::largest<L>(list[0]);
            if (COUNT_ONLY || !set.experts) {
                typename O::Type last = O::never();
                if (L == 1) {
#pragma unroll
                    for (int i = 0; i < PLACES; ++i) last = i + 1 == (int)k ? list[i] : last;
                } else {
                    last = top;
                    // the heads that equal `last` off their lists, as far as `places`, and the largest head that is left (the median of a
                    // place, the next and the least is the next, of the largest the place itself)
                    auto next_largest = [&](int places) {
                        const typename O::Type gone = list[0] == last ? O::never() : O::above_all();
#pragma unroll
                        for (int j = 0; j < PLACES; ++j)
                            if (j < places) list[j] = dm::median(list[j], j + 1 < PLACES ? list[j + 1] : O::never(), gone);
                        last = dm::largest<L>(list[0]);
                    };
                    if (K == 16 && k > 16) {
                        for (unsigned i = 1; i < k; ++i) next_largest(PLACES);
                    } else {
#pragma unroll
                        for (int i = 1; i < K; ++i)
                            if (i < (int)k) next_largest(K - i);       // (what could come up after the k-th is not moved any more)
                    }
                }
                last = max(last, O::least(dtype));                 // (fewer than k: all that can be)
                unsigned chosen = 0;
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const unsigned one = y[j] >= last ? 1u : 0u;
                    cnt[j] += one;
                    if (WIDE) chosen += one;
                }
                if (WIDE) chosen = dm::over_group<L>(chosen, dm::Add());
                if (WIDE && __any(chosen > k)) {
#pragma unroll
                    for (int j = 0; j < N; ++j) cnt[j] -= y[j] >= last ? 1u : 0u;
                    // k times the largest that is left, of the lowest expert that has it
                    typename O::Type left[N];
#pragma unroll
                    for (int j = 0; j < N; ++j) left[j] = y[j];
                    for (unsigned i = 0; i < k; ++i) {
                        typename O::Type best = O::never();
#pragma unroll
                        for (int j = 0; j < N; ++j) best = dm::median(best, left[j], O::above_all());
                        best = dm::largest<L>(best);
                        unsigned first = 0xFFFFFFFFu;
#pragma unroll
                        for (int j = N - 1; j >= 0; --j)
                            if (left[j] == best) first = (unsigned)(4 * ((j >> 2) * L + sub) + (j & 3));
                        first = dm::over_group<L>(first, dm::Min());
                        if (best < O::least(dtype)) first = 0xFFFFFFFFu;
#pragma unroll
                        for (int j = 0; j < N; ++j) {
                            const bool hit = first == (unsigned)(4 * ((j >> 2) * L + sub) + (j & 3));
                            cnt[j] += hit ? 1u : 0u;
                            left[j] = hit ? O::never() : left[j];
                        }
                    }
                }
            }
            if constexpr (!COUNT_ONLY) {
                // the scores, of the logits as they came
                const float mx = top < O::least(dtype) ? 0.0f : O::logit(top, dtype);
                float x[N];
                if constexpr (WIDE) {
#pragma unroll
                    for (int j = 0; j < N; ++j) x[j] = y[j];
                } else {
                    dm::raw_values<NQ, WIDE>(raw, dtype, x);
                }
                float sum = nan ? __builtin_nanf("") : 0.0f;
                if (sigmoid) {
                    float none[1];
                    sigmoid_weights<N, false>(x, mx, none);
                } else {
                    softmax_weights(x, mx);
                }
#pragma unroll
                for (int j = 0; j < N; ++j) sum += x[j];
                sum = dm::over_group<L>(sum, dm::Add());
                const bool live = sum != 0.0f;                     // (a NaN makes it NaN)
                const float inv = live ? __builtin_amdgcn_rcpf(sum) : 0.0f;
#pragma unroll
                for (int j = 0; j < N; ++j) psum[j] = __builtin_fmaf(x[j], inv, psum[j]);
                if (live && sub == 0) {
                    const float lse = mx + __builtin_amdgcn_logf(sum) * LN2;
                    z += (double)lse * (double)lse;
                    ++n;
                }
                if (set.experts && live)
                    for (unsigned j = sub; j < k; j += L) {
                        const int64_t e = set.experts[(image_row + row) * k + j];
                        if (e >= 0 && e < (int64_t)E) atomicAdd(&hist[(unsigned)e], 1u);
                        else bad |= e != -1;
                    }
            }
        }
        if constexpr (!COUNT_ONLY) {
            // the run's sums of p into the workgroup's: the rows of a wave whose lanes are 16 apart or more have a part each, and every
            // place of it one lane that writes it
            unsigned thread = threadIdx.x;
            asm("" : "+v"(thread));                                // (or places are worked out before the walk, and kept in registers)
            double *part = psum_lds[thread / (L <= 16 ? 16 : L)] + 4 * (thread & (L - 1));
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (L <= 16) psum[j] = dm::over_row16<L>(psum[j]);
            }
            if ((thread & 15) < L || L > 16) {
                // (one instruction without an answer to wait for; nobody else adds to the place)
#pragma unroll
                for (int j = 0; j < N; ++j)
                    __hip_atomic_fetch_add(part + 4 * (j >> 2) * L + (j & 3), (double)psum[j], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) psum[j] = 0.0f;
        }
    } while (r0 < at.rows);
    if (bad) dm::raise_status(status, DM_ST_LABEL_RANGE);

#pragma unroll
    for (int j = 0; j < N; ++j) {
        if (L <= 16) cnt[j] = dm::over_row16<L>(cnt[j]);
        if (((lane & 15) < L || L > 16) && cnt[j]) atomicAdd(&hist[4 * ((j >> 2) * L + sub) + (j & 3)], cnt[j]);
    }
    if (!COUNT_ONLY) {
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) {
            z += __shfl_xor(z, off);
            n += __shfl_xor(n, off);
        }
        if (lane == 0) {
            z_lds[wave] = z;
            n_lds[wave] = n;
        }
    }
    __syncthreads();
    if (whole) {
        static_assert(RT_THREADS == LOSS_THREADS, "");
        const size_t group = a.first_group[at.set] + (a.per_image ? at.image : 0);
        long long counts[LOSS_EACH];
        double sums[LOSS_EACH];
#pragma unroll
        for (int j = 0; j < LOSS_EACH; ++j) {
            const unsigned e = threadIdx.x + j * RT_THREADS;
            counts[j] = 0;
            sums[j] = 0.0;
            if (e < E) {
                counts[j] = (long long)hist[e];
                out.counts[group * E + e] = counts[j];
                if (!COUNT_ONLY) {
                    double s = psum_lds[0][e];      // (the parts in order)
#pragma unroll
                    for (int w = 1; w < RT_WAVES * PARTS; ++w) s += psum_lds[w][e];
                    sums[j] = s;
                    if (out.given_counts) counts[j] = out.given_counts[group * E + e];
                }
            }
        }
        if (!COUNT_ONLY) {
            const bool brings = threadIdx.x < RT_WAVES;
            group_loss(out, E, group, counts, sums, brings ? n_lds[threadIdx.x] : 0, brings ? z_lds[threadIdx.x] : 0.0, loss_lds);
        }
        return;
    }
    unsigned *slot = slots + (size_t)blockIdx.x * slot_words(E);
    for (unsigned e = threadIdx.x; e < E; e += RT_THREADS) {
        if (!COUNT_ONLY) {
            double s = psum_lds[0][e];
#pragma unroll
            for (int w = 1; w < RT_WAVES * PARTS; ++w) s += psum_lds[w][e];
            slot[e] = __float_as_uint((float)s);
        }
        slot[E + e] = hist[e];
    }
    if (!COUNT_ONLY && threadIdx.x == 0) {
        double s = z_lds[0];
        unsigned rows = n_lds[0];
        for (int w = 1; w < RT_WAVES; ++w) {
            s += z_lds[w];
            rows += n_lds[w];
        }
        *reinterpret_cast<double *>(slot + 2 * E) = s;
        slot[2 * E + 2] = rows;
    }
}

// The slots of a group's workgroups added in index order: `cols` experts at a time (a power of two, 64 at most), a thread per
// expert and every FINISH_THREADS / cols-th slot, their sums joined in order.  Then the loss of the sums.
// Bound by the latency of its loads: 5 us for 125 slots of 64 experts in each of six groups, 7 to 9 for 768 slots of one.
//   SUMS and LOSS   a workgroup per group does both
//   SUMS alone      gridDim.y workgroups per group, each its share of the experts; the sums go to counts and means
//   LOSS alone      a workgroup per group, from counts and means
// Two launches are taken for few groups of many experts, where one workgroup would read a megabyte of slots by itself.  (One
// launch in which the last of a group's workgroups makes the loss is slower: the fences it needs write the caches back.)
constexpr int FINISH_THREADS = 1024, FINISH_WAVES = FINISH_THREADS / 64;

template <bool SUMS, bool LOSS>
__global__ __launch_bounds__(FINISH_THREADS) void router_finish_kernel(const RouterSets a, const unsigned *__restrict__ slots,
                                                                       const unsigned cols, double *__restrict__ means, const Results out)
{
    __shared__ double p_lds[FINISH_WAVES][64];
    __shared__ unsigned long long c_lds[FINISH_WAVES][64];
    __shared__ double P[RT_MAX_EXPERTS];
    __shared__ long long C[RT_MAX_EXPERTS];
    __shared__ LossSums loss_lds;
    const unsigned E = a.E, words = slot_words(E), tid = threadIdx.x, group = blockIdx.x;
    int set = 0;
    while (set + 1 < a.S && group >= a.first_group[set + 1]) ++set;
    const RouterSetK &s = a.s[set];
    const unsigned image = group - a.first_group[set];                   // (0 unless per_image)
    const unsigned slots_of_group = a.per_image ? s.chunks : s.images * s.chunks;
    const unsigned *first = slots + (size_t)(s.first_block + image * s.chunks) * words;
    if (SUMS) {
        const unsigned col = tid & (cols - 1), slice = tid / cols, slices = FINISH_THREADS / cols;
        const bool with_p = means != nullptr || LOSS;
        for (unsigned e0 = blockIdx.y * cols; e0 < E; e0 += gridDim.y * cols) {
            const unsigned e = e0 + col;
            double p = 0.0;
            unsigned long long c = 0;
            // (eight slots are asked for before the first is added)
            for (unsigned i = slice; i < slots_of_group; i += 8 * slices) {
                float part[8];
                unsigned times[8];
#pragma unroll
                for (unsigned u = 0; u < 8; ++u) {
                    const bool there = e < E && i + u * slices < slots_of_group;
                    const unsigned *slot = first + (size_t)(there ? i + u * slices : 0) * words + (there ? e : 0);
                    part[u] = there && with_p ? __uint_as_float(slot[0]) : 0.0f;
                    times[u] = there ? slot[E] : 0u;
                }
#pragma unroll
                for (unsigned u = 0; u < 8; ++u) {
                    p += (double)part[u];
                    c += times[u];
                }
            }
            // (cols: 1 to 64; the lanes of an expert are cols apart)
            for (unsigned off = cols; off < 64; off <<= 1) {
                p += __shfl_xor(p, off);
                c += __shfl_xor(c, off);
            }
            if ((tid & 63) < cols) {
                p_lds[tid >> 6][col] = p;
                c_lds[tid >> 6][col] = c;
            }
            __syncthreads();
            if (tid < cols && e < E) {
#pragma unroll
                for (int i = 1; i < FINISH_WAVES; ++i) {
                    p += p_lds[i][col];
                    c += c_lds[i][col];
                }
                out.counts[(size_t)group * E + e] = (int64_t)c;
                if (LOSS) {
                    P[e] = p;
                    C[e] = (long long)c;
                } else if (means) {
                    means[(size_t)group * E + e] = p;
                }
            }
            __syncthreads();
        }
    }
    if (!LOSS || tid >= LOSS_THREADS) return;
    const int64_t *given = out.given_counts ? out.given_counts : SUMS ? nullptr : out.counts;
    long long counts[LOSS_EACH];
    double sums[LOSS_EACH];
#pragma unroll
    for (int j = 0; j < LOSS_EACH; ++j) {
        const unsigned e = tid + j * LOSS_THREADS;
        counts[j] = 0;
        sums[j] = 0.0;
        if (e < E) {
            counts[j] = given ? given[(size_t)group * E + e] : C[e];
            sums[j] = SUMS ? P[e] : means[(size_t)group * E + e];
        }
    }
    double zs = 0.0;
    unsigned long long rows = 0;
#pragma unroll 4
    for (unsigned i = tid; i < slots_of_group; i += LOSS_THREADS) {
        const unsigned *slot = first + (size_t)i * words;
        zs += *reinterpret_cast<const double *>(slot + 2 * E);
        rows += slot[2 * E + 2];
    }
    group_loss(out, E, group, counts, sums, rows, zs, loss_lds);
}

// The logits once more, their scores and their share in the gradient, a row per group of lanes as above: the row's dot product
// with f needs all of its scores, and reading 4 bytes again costs less than 4 bytes kept in between and read.  Memory bound
// from float32 logits (5.8 TB/s read and written in a step of 354 MB of logits, 4.8 when it is repeated by itself over 708 MB).
template <int NQ, int L, bool WIDE>
__global__ __launch_bounds__(RT_THREADS) void router_backward_kernel(const RouterSets a, const int dtype, const int sigmoid,
                                                                     const float *__restrict__ slope,
                                                                     const float *__restrict__ inv_rows,
                                                                     const float *__restrict__ grad_balance,
                                                                     const float *__restrict__ grad_z)
{
    constexpr int N = 4 * NQ;
    const unsigned E = a.E;
    const float ninf = -__builtin_huge_valf();
    const Place at = place_of(a, blockIdx.x);
    const RouterSetK &set = a.s[at.set];
    const size_t image_at = (size_t)at.image * (size_t)set.image_stride;
    const size_t image_row = (size_t)at.image * set.Q;
    const unsigned group = a.first_group[at.set] + (a.per_image ? at.image : 0);
    const float inv_n = inv_rows[group];
    const float gb = grad_balance ? grad_balance[group] * inv_n : 0.0f;
    const float gz = grad_z ? 2.0f * (grad_z[group] * inv_n) : 0.0f;
    const unsigned sub = threadIdx.x & (L - 1);
    constexpr unsigned ROWS = RT_THREADS / L;
    float f[N];
    dm::row_values<NQ, L, true>(dm::fetch_row<NQ, L, true>(slope, (size_t)group * E, sub, E), DM_F32, sub, E, 0.0f, f);
    const unsigned local = threadIdx.x / L;
    dm::RawRow<NQ, WIDE> next;
    uint8_t next_counts = 1;
    auto fetch = [&](unsigned r) {
        const size_t row = (size_t)at.row0 + (r < at.rows ? r : 0);
        next = dm::fetch_row<NQ, L, WIDE>(set.logits, image_at + row * E, sub, E);
        if (set.mask) next_counts = set.mask[image_row + row];
    };
    if (at.rows) fetch(local);
    for (unsigned r0 = 0; r0 < at.rows; r0 += ROWS) {
        const unsigned r = r0 + local;
        const bool there = r < at.rows;
        const size_t row = (size_t)at.row0 + (there ? r : 0);
        dm::RawRow<NQ, WIDE> raw = next;
        const bool counts = next_counts != 0;
        if (r0 + ROWS < at.rows) fetch(r + ROWS);
        float x[N];
        if constexpr (WIDE) {
            dm::row_values<NQ, L, WIDE>(raw, dtype, sub, E, ninf, x);
        } else {
            dm::place_raw<NQ, L>(raw, sub, E, dtype == DM_BF16 ? 0xFF80FF80u : 0xFC00FC00u);
            dm::raw_values<NQ, WIDE>(raw, dtype, x);
        }
        if (!counts) {
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = ninf;
        }
        float mx = ninf;                                       // (a NaN makes the whole row NaN, whatever is found here)
#pragma unroll
        for (int j = 0; j < N; j += 2) mx = dm::max3(mx, x[j], x[j + 1]);
        mx = dm::largest<L>(mx);
        mx = mx == ninf ? 0.0f : mx;
        float sum = 0.0f, dot = 0.0f;
        float rest[N];
        if (sigmoid) {
            sigmoid_weights<N, true>(x, mx, rest);
        } else {
            softmax_weights(x, mx);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            sum += x[j];
            dot = __builtin_fmaf(x[j], f[j], dot);
        }
        sum = dm::over_group<L>(sum, dm::Add());
        dot = dm::over_group<L>(dot, dm::Add());
        const bool live = sum != 0.0f;
        const float inv = live ? __builtin_amdgcn_rcpf(sum) : 0.0f;
        dot *= inv;
        // p (gb (f - dot) + gz lse); of a row that does not count 0 times 0, whatever comes from upstream; with no gradient of z no
        // product with lse at all: a sigmoid row may hold an infinite logit (its score is 1), and 0 times that is NaN
        const float zpart = live && grad_z ? gz * (mx + __builtin_amdgcn_logf(sum) * LN2) : 0.0f;
        const float bpart = live ? gb : 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = (x[j] * inv) * __builtin_fmaf(bpart, f[j] - dot, zpart);
        if (sigmoid) {
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] *= rest[j];
        }
        if (there) dm::store_row<NQ, L, WIDE>(set.grad, dtype, (image_row + row) * E, sub, E, x);
    }
}

// ---- host side ----

struct Shape {
    int S, B, E;
    bool per_image, merged;      // merged: every set is one run of B * Q rows
};

int check_shape(const DmRouterSet *sets, int S, int B, int E, int per_image, Shape *sh)
{
    if (S < 0 || B < 0 || E < 1 || (S > 0 && !sets)) return DM_E_INVALID_ARG;
    if (E > RT_MAX_EXPERTS) return DM_E_UNSUPPORTED;
    if ((long long)S * (per_image ? B : 1) >= (1ll << 31)) return DM_E_UNSUPPORTED;
    bool dense = true;
    for (int s = 0; s < S; ++s) {
        if (sets[s].Q < 0) return DM_E_INVALID_ARG;
        const long long image = (long long)sets[s].Q * E;
        if (sets[s].image_stride != 0 && sets[s].image_stride < image) return DM_E_INVALID_ARG;
        if ((long long)B * sets[s].Q >= (1ll << 31)) return DM_E_UNSUPPORTED;
        dense &= sets[s].image_stride == 0 || sets[s].image_stride == image || B <= 1;
    }
    *sh = Shape{S, B, E, per_image != 0, dense && !per_image};
    return DM_OK;
}

// Quads of four logits per lane, and lanes per row.
//   Forward: as few lanes as can hold the row with sixteen logits each.  Every reduction over lanes is paid per row, every
//   lane behind the row's end as well: 354 MB of float32 logits of 16, 48, 64 and 96 experts (top 2, 4, 4, 4) take 79, 79, 79 and
//   80 us, with half as many logits per lane 105, 101, 89 and 117 us.  (More than sixteen have not been measured.)
//   Backward, float32: four logits per lane and up to sixteen lanes, whose store is a run of memory; in the forward pass's
//   forms 12, 24 and 48 experts take 171, 169 and 157 us for 354 MB read and written instead of 152, 149 and 149.
//   Backward, 16 bits: bound by instructions, not memory, where lanes lie behind the row's end: 12, 20, 33 and 96 experts take
//   91, 95, 101 and 86 us for 177 MB read and written with twelve logits per lane, 103, 114, 145 and 96 us with four or eight.
struct Form {
    int NQ, L;
};
Form forward_form(unsigned E)
{
    if (E <= 8) return {E <= 4 ? 1 : 2, 1};
    if (E <= 16) return {E <= 12 ? 3 : 4, 1};
    if (E <= 32) return {E <= 24 ? 3 : 4, 2};
    if (E <= 64) return {E <= 48 ? 3 : 4, 4};
    if (E <= 128) return {E <= 96 ? 3 : 4, 8};
    if (E <= 256) return {E <= 192 ? 3 : 4, 16};
    return {4, E <= 512 ? 32 : 64};
}
Form backward_form(unsigned E, bool wide)
{
    if (E <= 4) return {1, 1};
    if (E <= 8) return {1, 2};
    if (E <= 16) return !wide && E <= 12 ? Form{3, 1} : Form{1, 4};
    if (E <= 32) return !wide && E <= 24 ? Form{3, 2} : Form{1, 8};
    if (E <= 64) return !wide && E <= 48 ? Form{3, 4} : Form{1, 16};
    if (E <= 128) return E <= 96 ? Form{3, 8} : Form{2, 16};
    if (E <= 256) return {E <= 192 ? 3 : 4, 16};
    return {4, E <= 512 ? 32 : 64};
}

// Chunks per image of a set, and their rows: over all sets of the call as many workgroups as the chip holds at once (with
// 1020 workgroups of the float32 kernel a second round of a few of them doubled the time), each with the same number of trips.
// Per CU, at the kernels' registers: three of the forward kernel, eight of the backward kernel.  (Five of the forward kernel fit
// for 16 bits: no faster, and two thirds more slots to add.)
struct Pass {
    int resident, lanes;         // workgroups, lanes per row
    bool whole;                  // one workgroup per group
};
Pass forward_pass(const DmRouterSet *sets, const Shape &sh)
{
    // Groups of up to WHOLE_TRIPS trips by one workgroup each: no second launch, whose time a few trips one after the other cost
    // less than.  Six sets of four trips: counts and forward pass of 8 experts 6.7 and 9.5 us among others instead of 8.8 and 11.6,
    // of 64 6.7 and 10.1 instead of 9.9 and 12.6, of 256 (bfloat16, top 8) 7.9 and 10.8 instead of 11.6 and 15.1; of eight trips
    // 7.6 and 11.3 instead of 8.8 and 11.6, but 9.7 and 14.9 instead of 9.8 and 12.6, and 12.1 and 16.9 instead of 11.9 and 15.5.
    constexpr long long WHOLE_TRIPS = 4;
    const int lanes = forward_form((unsigned)sh.E).L;
    bool whole = sh.merged || sh.per_image;
    for (int s = 0; s < sh.S && whole; ++s)
        whole = (sh.merged ? (long long)sh.B * sets[s].Q : (long long)sets[s].Q) <= WHOLE_TRIPS * (RT_THREADS / lanes);
    return {3 * 256, lanes, whole};
}
Pass backward_pass(const Shape &sh, bool wide) { return {8 * 256, backward_form((unsigned)sh.E, wide).L, false}; }
struct Chunks {
    unsigned count, rows;
};
Chunks chunks_of(const Shape &sh, int Q, const Pass &pass)
{
    const long long images = sh.merged ? 1 : sh.B;
    const long long rows = sh.merged ? (long long)sh.B * Q : Q;
    const long long trip = RT_THREADS / pass.lanes;
    const long long trips = std::max(1ll, (rows + trip - 1) / trip);
    const long long want = std::max(1ll, pass.resident / std::max(1ll, std::min<long long>(sh.S, DM_MAX_SETS_PER_LAUNCH) * images));
    const long long each = pass.whole ? trips : (trips + want - 1) / want;
    return Chunks{(unsigned)((trips + each - 1) / each), (unsigned)(each * trip)};
}

// The kernel arguments of sets first .. first + n - 1; returns the launch's workgroups.
unsigned long long describe(const DmRouterSet *sets, int first, int n, const Shape &sh, int k, const Pass &pass, RouterSets *a)
{
    a->S = n;
    a->E = (unsigned)sh.E;
    a->k = (unsigned)k;
    a->per_image = sh.per_image;
    unsigned long long blocks = 0;
    for (int i = 0; i < n; ++i) {
        const DmRouterSet &in = sets[first + i];
        RouterSetK &s = a->s[i];
        s.logits = in.logits;
        s.mask = in.mask;
        s.experts = in.experts;
        s.grad = in.grad;
        s.image_stride = in.image_stride ? in.image_stride : (int64_t)in.Q * sh.E;
        s.images = sh.merged ? 1u : (unsigned)sh.B;
        s.Q = sh.merged ? (unsigned)sh.B * (unsigned)in.Q : (unsigned)in.Q;
        const Chunks c = chunks_of(sh, in.Q, pass);
        s.chunks = c.count;
        s.chunk_rows = c.rows;
        s.first_block = (unsigned)blocks;
        a->first_group[i] = (unsigned)i * (sh.per_image ? (unsigned)sh.B : 1u);
        blocks += (unsigned long long)s.images * s.chunks;
    }
    return blocks;
}

// (the sets of a call go through launches of up to DM_MAX_SETS_PER_LAUNCH, one after the other, over the same workspace)
unsigned long long most_blocks(const DmRouterSet *sets, const Shape &sh, const Pass &pass)
{
    unsigned long long most = 0;
    for (int first = 0; first < sh.S; first += DM_MAX_SETS_PER_LAUNCH) {
        unsigned long long blocks = 0;
        for (int s = first; s < std::min(sh.S, first + DM_MAX_SETS_PER_LAUNCH); ++s)
            blocks += (unsigned long long)(sh.merged ? 1 : sh.B) * chunks_of(sh, sets[s].Q, pass).count;
        most = std::max(most, blocks);
    }
    return most;
}

typedef void (*ForwardKernel)(RouterSets, int, int, int, unsigned *, Results, int32_t *);
typedef void (*BackwardKernel)(RouterSets, int, int, const float *, const float *, const float *, const float *);

template <int NQ, int L, int K>
ForwardKernel forward_of(bool wide, bool count_only)
{
    return wide ? (count_only ? router_forward_kernel<NQ, L, K, true, true> : router_forward_kernel<NQ, L, K, true, false>)
                : (count_only ? router_forward_kernel<NQ, L, K, false, true> : router_forward_kernel<NQ, L, K, false, false>);
}
template <int NQ, int L>
ForwardKernel forward_with(unsigned k, bool wide, bool count_only)
{
    if (k <= 2) return forward_of<NQ, L, 2>(wide, count_only);
    if (k <= 4) return forward_of<NQ, L, 4>(wide, count_only);
    if (k <= 8) return forward_of<NQ, L, 8>(wide, count_only);
    return forward_of<NQ, L, 16>(wide, count_only);
}
ForwardKernel forward_for(unsigned E, unsigned k, bool wide, bool count_only)
{
    const Form f = forward_form(E);
    switch (f.L) {
    case 1:
        return f.NQ == 1 ? forward_with<1, 1>(k, wide, count_only) : f.NQ == 2 ? forward_with<2, 1>(k, wide, count_only)
               : f.NQ == 3 ? forward_with<3, 1>(k, wide, count_only) : forward_with<4, 1>(k, wide, count_only);
    case 2: return f.NQ == 3 ? forward_with<3, 2>(k, wide, count_only) : forward_with<4, 2>(k, wide, count_only);
    case 4: return f.NQ == 3 ? forward_with<3, 4>(k, wide, count_only) : forward_with<4, 4>(k, wide, count_only);
    case 8: return f.NQ == 3 ? forward_with<3, 8>(k, wide, count_only) : forward_with<4, 8>(k, wide, count_only);
    case 16: return f.NQ == 3 ? forward_with<3, 16>(k, wide, count_only) : forward_with<4, 16>(k, wide, count_only);
    case 32: return forward_with<4, 32>(k, wide, count_only);
    default: return forward_with<4, 64>(k, wide, count_only);
    }
}
template <bool WIDE>
BackwardKernel backward_for(unsigned E)
{
    const Form f = backward_form(E, WIDE);
    switch (f.L) {
    case 1: if constexpr (!WIDE) { if (f.NQ == 3) return router_backward_kernel<3, 1, WIDE>; } return router_backward_kernel<1, 1, WIDE>;
    case 2: if constexpr (!WIDE) { if (f.NQ == 3) return router_backward_kernel<3, 2, WIDE>; } return router_backward_kernel<1, 2, WIDE>;
    case 4: if constexpr (!WIDE) { if (f.NQ == 3) return router_backward_kernel<3, 4, WIDE>; } return router_backward_kernel<1, 4, WIDE>;
    case 8: return f.NQ == 3 ? router_backward_kernel<3, 8, WIDE> : router_backward_kernel<1, 8, WIDE>;
    case 16:
        return f.NQ == 1 ? router_backward_kernel<1, 16, WIDE> : f.NQ == 2 ? router_backward_kernel<2, 16, WIDE>
               : f.NQ == 3 ? router_backward_kernel<3, 16, WIDE> : router_backward_kernel<4, 16, WIDE>;
    case 32: return router_backward_kernel<4, 32, WIDE>;
    default: return router_backward_kernel<4, 64, WIDE>;
    }
}

// (a launch has fewer than 2^32 threads)
constexpr unsigned long long MOST_BLOCKS = (1ull << 32) / RT_THREADS - 1, MOST_GROUPS = (1ull << 32) / FINISH_THREADS - 1;

// Workspace: the slots of a launch's workgroups, then the sums of p of its groups.
struct Workspace {
    unsigned long long blocks, groups;
    int64_t bytes(int E) const { return (int64_t)(std::max(1ull, blocks) * slot_words((unsigned)E) * 4 + groups * (unsigned long long)E * 8); }
};
Workspace workspace_of(const DmRouterSet *sets, const Shape &sh)
{
    const unsigned long long groups = sh.per_image ? (unsigned long long)sh.B : 1ull;      // of a set
    return Workspace{most_blocks(sets, sh, forward_pass(sets, sh)), (unsigned long long)std::min(sh.S, DM_MAX_SETS_PER_LAUNCH) * groups};
}

int forward(const DmRouterSet *sets, int S, int B, int E, int top_k, int dtype, int scores, int per_image,
            const int64_t *given_counts, float *balance, float *z, int64_t *counts, float *slope, float *inv_rows,
            void *workspace, int64_t workspace_bytes, int32_t *status, hipStream_t st)
{
    Shape sh;
    int rc = check_shape(sets, S, B, E, per_image, &sh);
    if (rc != DM_OK) return rc;
    if (dtype != DM_F32 && dtype != DM_BF16 && dtype != DM_F16) return DM_E_INVALID_ARG;
    if (scores != DM_SCORES_SOFTMAX && scores != DM_SCORES_SIGMOID) return DM_E_INVALID_ARG;
    if (top_k < 1) return DM_E_INVALID_ARG;
    const long long groups = (long long)S * (per_image ? B : 1);
    if (groups == 0) return DM_OK;
    if (!counts || !status) return DM_E_INVALID_ARG;
    int given = -1;                  // (of the sets with rows: all or none come with indices)
    for (int s = 0; s < S; ++s) {
        if (B == 0 || sets[s].Q == 0) continue;
        const int has = sets[s].experts != nullptr;
        if (!sets[s].logits || (given >= 0 && has != given) || (!has && top_k > E)) return DM_E_INVALID_ARG;
        given = has;
    }
    if (given == 1 && !balance) return DM_E_INVALID_ARG;       // (the counts of given indices need no logits)
    const Workspace need = workspace_of(sets, sh);
    if (need.blocks > MOST_BLOCKS || need.groups > MOST_GROUPS) return DM_E_UNSUPPORTED;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 || workspace_bytes < need.bytes(E)) return DM_E_INVALID_ARG;
    const Pass pass = forward_pass(sets, sh);
    unsigned *slots = static_cast<unsigned *>(workspace);
    double *means = reinterpret_cast<double *>(slots + (size_t)std::max(1ull, need.blocks) * slot_words((unsigned)E));
    for (int first = 0; first < S; first += DM_MAX_SETS_PER_LAUNCH) {
        RouterSets a;
        const int n = std::min(S - first, DM_MAX_SETS_PER_LAUNCH);
        const unsigned blocks = (unsigned)describe(sets, first, n, sh, top_k, pass, &a);
        const size_t g0 = (size_t)first * (per_image ? (size_t)B : 1);
        const unsigned gn = (unsigned)n * (per_image ? (unsigned)B : 1u);
        const Results out{given_counts ? given_counts + g0 * E : nullptr, balance ? balance + g0 : nullptr, z ? z + g0 : nullptr,
                          counts + g0 * E, slope ? slope + g0 * E : nullptr, inv_rows ? inv_rows + g0 : nullptr};
        hipLaunchKernelGGL(forward_for((unsigned)E, given == 1 ? 1u : (unsigned)top_k, dtype == DM_F32, balance == nullptr), dim3(blocks),
                           dim3(RT_THREADS), 0, st, a, dtype, scores == DM_SCORES_SIGMOID ? 1 : 0, pass.whole ? 1 : 0, slots, out, status);
        rc = dm::check_hip(hipGetLastError(), "router_forward_kernel launch");
        if (rc != DM_OK) return rc;
        if (pass.whole) continue;
        unsigned cols = 1;
        while (cols < 64 && cols < (unsigned)E) cols <<= 1;
        auto finish = [&](auto kernel, unsigned parts, unsigned width, int threads) {
            hipLaunchKernelGGL(kernel, dim3(gn, parts), dim3(threads), 0, st, a, slots, width, means, out);
        };
        // (one workgroup adds 720 slots of 64 experts in 20 us, four of 16 experts each in 4)
        const bool few = gn <= 64 && (unsigned long long)blocks * (unsigned)E > 4096ull * gn && E > 16;
        const unsigned width = few ? 16u : cols, parts = few ? (unsigned)(E + 15) / 16 : 1u;
        if (!balance) {
            means = nullptr;
            finish(router_finish_kernel<true, false>, parts, width, FINISH_THREADS);
        } else if (few) {
            finish(router_finish_kernel<true, false>, parts, width, FINISH_THREADS);
            finish(router_finish_kernel<false, true>, 1u, cols, LOSS_THREADS);
        } else {
            finish(router_finish_kernel<true, true>, 1u, cols, FINISH_THREADS);
        }
        rc = dm::check_hip(hipGetLastError(), "router_finish_kernel launch");
        if (rc != DM_OK) return rc;
    }
    return DM_OK;
}

}  // namespace

extern "C" int64_t dm_balance_workspace(const DmRouterSet *sets, int S, int B, int E, int per_image)
{
    Shape sh;
    const int rc = check_shape(sets, S, B, E, per_image, &sh);
    if (rc != DM_OK) return rc;
    return workspace_of(sets, sh).bytes(E);
}

extern "C" int dm_balance_loss(const DmRouterSet *sets, int S, int B, int E, int top_k, int dtype, int scores, int per_image,
                               const int64_t *given_counts, float *balance, float *z, int64_t *counts, float *slope,
                               float *inv_rows, void *workspace, int64_t workspace_bytes, int32_t *status, void *stream)
{
    if (S > 0 && (!per_image || B > 0) && (!balance || !slope || !inv_rows)) return DM_E_INVALID_ARG;
    if (S > 0 && (!per_image || B > 0) && !z && scores == DM_SCORES_SOFTMAX) return DM_E_INVALID_ARG;
    return forward(sets, S, B, E, top_k, dtype, scores, per_image, given_counts, balance, z, counts, slope, inv_rows, workspace,
                   workspace_bytes, status, static_cast<hipStream_t>(stream));
}

extern "C" int dm_expert_counts(const DmRouterSet *sets, int S, int B, int E, int top_k, int dtype, int per_image,
                                int64_t *counts, void *workspace, int64_t workspace_bytes, int32_t *status, void *stream)
{
    return forward(sets, S, B, E, top_k, dtype, DM_SCORES_SOFTMAX, per_image, nullptr, nullptr, nullptr, counts, nullptr, nullptr,
                   workspace, workspace_bytes, status, static_cast<hipStream_t>(stream));
}

extern "C" int dm_balance_backward(const DmRouterSet *sets, int S, int B, int E, int dtype, int scores, int per_image,
                                   const float *slope, const float *inv_rows, const float *grad_balance, const float *grad_z,
                                   void *stream)
{
    Shape sh;
    int rc = check_shape(sets, S, B, E, per_image, &sh);
    if (rc != DM_OK) return rc;
    if (dtype != DM_F32 && dtype != DM_BF16 && dtype != DM_F16) return DM_E_INVALID_ARG;
    if (scores != DM_SCORES_SOFTMAX && scores != DM_SCORES_SIGMOID) return DM_E_INVALID_ARG;
    if (scores == DM_SCORES_SIGMOID && grad_z) return DM_E_INVALID_ARG;
    if (S == 0 || B == 0) return DM_OK;
    if (!slope || !inv_rows) return DM_E_INVALID_ARG;
    for (int s = 0; s < S; ++s)
        if (sets[s].Q > 0 && (!sets[s].logits || !sets[s].grad)) return DM_E_INVALID_ARG;
    if (most_blocks(sets, sh, backward_pass(sh, dtype == DM_F32)) > MOST_BLOCKS) return DM_E_UNSUPPORTED;
    hipStream_t st = static_cast<hipStream_t>(stream);
    for (int first = 0; first < S; first += DM_MAX_SETS_PER_LAUNCH) {
        RouterSets a;
        const int n = std::min(S - first, DM_MAX_SETS_PER_LAUNCH);
        const unsigned blocks = (unsigned)describe(sets, first, n, sh, 0, backward_pass(sh, dtype == DM_F32), &a);
        const size_t g0 = (size_t)first * (per_image ? (size_t)B : 1);
        hipLaunchKernelGGL(dtype == DM_F32 ? backward_for<true>((unsigned)E) : backward_for<false>((unsigned)E), dim3(blocks),
                           dim3(RT_THREADS), 0, st, a, dtype, scores == DM_SCORES_SIGMOID ? 1 : 0, slope + g0 * E, inv_rows + g0,
                           grad_balance ? grad_balance + g0 : nullptr, grad_z ? grad_z + g0 : nullptr);
        rc = dm::check_hip(hipGetLastError(), "router_backward_kernel launch");
        if (rc != DM_OK) return rc;
    }
    return DM_OK;
}
