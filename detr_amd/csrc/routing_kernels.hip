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
// lane that owns the expert, and leave once per workgroup, into a slot of the workspace.  A second kernel adds the slots in
// index order in 64 bits: no float atomics, the same bits every run.
#include <algorithm>

#include "lanes.h"

namespace {

constexpr int RT_THREADS = 256;
constexpr int RT_WAVES = RT_THREADS / 64;
constexpr int RT_MAX_EXPERTS = 1024;
constexpr int FINISH_THREADS = 1024;
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

// Order of the logits as an unsigned key; 0 for those that are never chosen (-infinity, NaN).  -0 counts as +0.
__device__ __forceinline__ unsigned order_key(float x)
{
    const unsigned u = __float_as_uint(x + 0.0f);
    const unsigned key = u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
    return x > -__builtin_huge_valf() ? key : 0u;
}
__device__ __forceinline__ float value_of_key(unsigned key)
{
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// The scores of a row before they are divided by their sum, and what turns them into p: w_e / sum w.
// Sigmoid: sigmoid(x) times a constant of the row that keeps the largest from underflowing: with c = min(max x, 0),
// t = exp(-|x| - c), sigmoid(x) exp(-c) = (x >= 0 ? 1 : t) / (1 + t exp(c)).  `rest` = 1 - sigmoid(x).
__device__ __forceinline__ float softmax_weight(float x, float mx) { return __builtin_amdgcn_exp2f((x - mx) * LOG2E); }
__device__ __forceinline__ float sigmoid_weight(float x, float c, float exp_c, float *rest)
{
    const float t = __builtin_amdgcn_exp2f((-__builtin_fabsf(x) - c) * LOG2E);
    const float r = __builtin_amdgcn_rcpf(1.0f + t * exp_c);
    *rest = (x >= 0.0f ? t : 1.0f) * r;
    return (x >= 0.0f ? 1.0f : t) * r;
}

template <typename T, int NQ, int L, bool COUNT_ONLY>
__global__ __launch_bounds__(RT_THREADS) void router_forward_kernel(const RouterSets a, const int sigmoid, unsigned *__restrict__ slots,
                                                                    int32_t *__restrict__ status)
{
    constexpr int N = 4 * NQ;                                  // logits of a row per lane
    __shared__ unsigned hist[RT_MAX_EXPERTS];
    __shared__ float psum_lds[COUNT_ONLY ? 1 : RT_WAVES][COUNT_ONLY ? 1 : RT_MAX_EXPERTS];
    __shared__ double z_lds[RT_WAVES];
    __shared__ unsigned n_lds[RT_WAVES];
    const unsigned E = a.E, k = a.k;
    const float ninf = -__builtin_huge_valf();
    for (unsigned e = threadIdx.x; e < E; e += RT_THREADS) hist[e] = 0;
    __syncthreads();

    const Place at = place_of(a, blockIdx.x);
    const RouterSetK &set = a.s[at.set];
    const T *base = static_cast<const T *>(set.logits) + (size_t)at.image * (size_t)set.image_stride;
    const size_t image_row = (size_t)at.image * set.Q;
    const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned sub = lane & (L - 1);
    constexpr unsigned ROWS = RT_THREADS / L;                  // rows of the workgroup at a time
    float psum[N] = {};
    unsigned cnt[N] = {};
    float z = 0.0f;
    unsigned n = 0;
    bool bad = false;

    // (every lane makes the same trips: the reductions need all lanes of a row's group)
    for (unsigned r0 = 0; r0 < at.rows; r0 += ROWS) {
        const unsigned r = r0 + threadIdx.x / L;
        const bool there = r < at.rows;
        const size_t row = (size_t)at.row0 + (there ? r : 0);
        const bool wanted = there && (!set.mask || set.mask[image_row + row] != 0);
        float x[N];
        unsigned key[N];
        unsigned top = 0;
        bool any_nan = false;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            float v[4] = {ninf, ninf, ninf, ninf};
            if (wanted) dm::load_quad(base + row * E, 4 * (q * L + sub), E, ninf, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[4 * q + j] = v[j];
                key[4 * q + j] = order_key(v[j]);
                top = max(top, key[4 * q + j]);
                any_nan |= v[j] != v[j];
            }
        }
        top = dm::over_group<L>(top, dm::Max());
        bool live;
        if (!COUNT_ONLY) {
            const float mx = top ? value_of_key(top) : 0.0f;
            const float c = fminf(mx, 0.0f), exp_c = __builtin_amdgcn_exp2f(c * LOG2E);
            float sum = 0.0f, rest;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                x[j] = sigmoid ? (x[j] == ninf ? 0.0f : sigmoid_weight(x[j], c, exp_c, &rest)) : softmax_weight(x[j], mx);
                sum += x[j];
            }
            sum = dm::over_group<L>(sum, dm::Add());
            live = sum != 0.0f;                                // (a NaN makes it NaN)
            const float inv = live ? __builtin_amdgcn_rcpf(sum) : 0.0f;
#pragma unroll
            for (int j = 0; j < N; ++j) psum[j] += x[j] * inv;
            if (live && sub == 0) {
                const float lse = mx + __builtin_amdgcn_logf(sum) * LN2;
                z += lse * lse;
                ++n;
            }
        } else {
            live = dm::over_group<L>((unsigned)(top != 0 || any_nan), dm::Max()) != 0;
        }
        if (set.experts) {
            if (live)
                for (unsigned j = sub; j < k; j += L) {
                    const int64_t e = set.experts[(image_row + row) * k + j];
                    if (e >= 0 && e < (int64_t)E) atomicAdd(&hist[(unsigned)e], 1u);
                    else bad |= e != -1;
                }
        } else {
            // k times the largest key that is left, of the lowest expert that has it
            for (unsigned i = 0; i < k; ++i) {
                unsigned best = 0;
#pragma unroll
                for (int j = 0; j < N; ++j) best = max(best, key[j]);
                best = dm::over_group<L>(best, dm::Max());
                unsigned first = 0xFFFFFFFFu;
#pragma unroll
                for (int j = N - 1; j >= 0; --j)
                    if (key[j] == best) first = (unsigned)(4 * ((j >> 2) * L + sub) + (j & 3));
                first = dm::over_group<L>(first, dm::Min());
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const bool hit = best != 0 && first == (unsigned)(4 * ((j >> 2) * L + sub) + (j & 3));
                    cnt[j] += hit ? 1u : 0u;
                    key[j] = hit ? 0u : key[j];
                }
            }
        }
    }
    if (bad) dm::raise_status(status, DM_ST_LABEL_RANGE);

    // the wave's rows, then the waves in index order
#pragma unroll
    for (int j = 0; j < N; ++j) {
#pragma unroll
        for (int off = L; off < 64; off <<= 1) {
            if (!COUNT_ONLY) psum[j] += __shfl_xor(psum[j], off);
            cnt[j] += __shfl_xor(cnt[j], off);
        }
        const unsigned e = 4 * ((j >> 2) * L + sub) + (j & 3);
        if (lane < L && e < E) {
            if (!COUNT_ONLY) psum_lds[wave][e] = psum[j];
            if (cnt[j]) atomicAdd(&hist[e], cnt[j]);
        }
    }
    double zd = z;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        zd += __shfl_xor(zd, off);
        n += __shfl_xor(n, off);
    }
    if (lane == 0) {
        z_lds[wave] = zd;
        n_lds[wave] = n;
    }
    __syncthreads();
    unsigned *slot = slots + (size_t)blockIdx.x * slot_words(E);
    for (unsigned e = threadIdx.x; e < E; e += RT_THREADS) {
        if (!COUNT_ONLY) {
            float s = psum_lds[0][e];
            for (int w = 1; w < RT_WAVES; ++w) s += psum_lds[w][e];
            slot[e] = __float_as_uint(s);
        }
        slot[E + e] = hist[e];
    }
    if (threadIdx.x == 0) {
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

// One workgroup per group: the slots of its workgroups added in index order, columns of COLS experts at a time, a thread
// per expert and every FINISH_THREADS / COLS-th slot.
__global__ __launch_bounds__(FINISH_THREADS) void router_finish_kernel(const RouterSets a, const unsigned *__restrict__ slots,
                                                                       const unsigned cols, const int64_t *__restrict__ given_counts,
                                                                       float *__restrict__ balance, float *__restrict__ z,
                                                                       int64_t *__restrict__ counts, float *__restrict__ slope,
                                                                       float *__restrict__ inv_rows)
{
    __shared__ double p_lds[FINISH_THREADS];
    __shared__ unsigned long long c_lds[FINISH_THREADS];
    __shared__ double P[RT_MAX_EXPERTS];
    __shared__ long long C[RT_MAX_EXPERTS];
    const unsigned E = a.E, words = slot_words(E), tid = threadIdx.x;
    int set = 0;
    while (set + 1 < a.S && blockIdx.x >= a.first_group[set + 1]) ++set;
    const RouterSetK &s = a.s[set];
    const unsigned image = blockIdx.x - a.first_group[set];              // (0 unless per_image)
    const unsigned slots_of_group = a.per_image ? s.chunks : s.images * s.chunks;
    const unsigned *first = slots + (size_t)(s.first_block + image * s.chunks) * words;
    const unsigned slices = FINISH_THREADS / cols, col = tid & (cols - 1), slice = tid / cols;
    for (unsigned e0 = 0; e0 < E; e0 += cols) {
        double p = 0.0;
        unsigned long long c = 0;
        if (e0 + col < E)
            for (unsigned i = slice; i < slots_of_group; i += slices) {
                const unsigned *slot = first + (size_t)i * words;
                if (balance) p += (double)__uint_as_float(slot[e0 + col]);
                c += slot[E + e0 + col];
            }
        __syncthreads();
        p_lds[tid] = p;
        c_lds[tid] = c;
        __syncthreads();
        if (tid < cols && e0 + tid < E) {
            for (unsigned i = 1; i < slices; ++i) {
                p += p_lds[i * cols + tid];
                c += c_lds[i * cols + tid];
            }
            P[e0 + tid] = p;
            C[e0 + tid] = (long long)c;
            counts[(size_t)blockIdx.x * E + e0 + tid] = (int64_t)c;
        }
    }
    if (!balance) return;
    // the rows that count and the sum of lse^2
    double zs = 0.0;
    unsigned long long rows = 0;
    for (unsigned i = tid; i < slots_of_group; i += FINISH_THREADS) {
        const unsigned *slot = first + (size_t)i * words;
        zs += *reinterpret_cast<const double *>(slot + 2 * E);
        rows += slot[2 * E + 2];
    }
    __syncthreads();
    p_lds[tid] = zs;
    c_lds[tid] = rows;
    if (given_counts)
        for (unsigned e = tid; e < E; e += FINISH_THREADS) C[e] = given_counts[(size_t)blockIdx.x * E + e];
    for (unsigned half = FINISH_THREADS / 2; half >= 1; half >>= 1) {
        __syncthreads();
        if (tid < half) {
            p_lds[tid] += p_lds[tid + half];
            c_lds[tid] += c_lds[tid + half];
        }
    }
    __syncthreads();
    const double inv_n = c_lds[0] ? 1.0 / (double)c_lds[0] : 0.0;
    const double z_mean = p_lds[0] * inv_n;
    // sum of the counts, then sum_e c_e P_e
    __syncthreads();
    long long total = 0;
    double dot = 0.0;
    for (unsigned e = tid; e < E; e += FINISH_THREADS) {
        total += C[e];
        dot += (double)C[e] * P[e];
    }
    p_lds[tid] = dot;
    c_lds[tid] = (unsigned long long)total;
    for (unsigned half = FINISH_THREADS / 2; half >= 1; half >>= 1) {
        __syncthreads();
        if (tid < half) {
            p_lds[tid] += p_lds[tid + half];
            c_lds[tid] += c_lds[tid + half];
        }
    }
    __syncthreads();
    const long long all = (long long)c_lds[0];
    const double per_count = all > 0 ? (double)E / (double)all : 0.0;
    if (tid == 0) {
        balance[blockIdx.x] = (float)(p_lds[0] * per_count * inv_n);
        if (z) z[blockIdx.x] = (float)z_mean;
        inv_rows[blockIdx.x] = (float)inv_n;
    }
    for (unsigned e = tid; e < E; e += FINISH_THREADS)
        slope[(size_t)blockIdx.x * E + e] = all > 0 ? (float)((double)C[e] * per_count - 1.0) : 0.0f;
}

template <typename T, int NQ, int L>
__global__ __launch_bounds__(RT_THREADS) void router_backward_kernel(const RouterSets a, const int sigmoid,
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
    const T *base = static_cast<const T *>(set.logits) + (size_t)at.image * (size_t)set.image_stride;
    const size_t image_row = (size_t)at.image * set.Q;
    T *out = static_cast<T *>(set.grad) + image_row * E;
    const unsigned group = a.first_group[at.set] + (a.per_image ? at.image : 0);
    const float inv_n = inv_rows[group];
    const float gb = grad_balance ? grad_balance[group] * inv_n : 0.0f;
    const float gz = grad_z ? 2.0f * (grad_z[group] * inv_n) : 0.0f;
    const unsigned sub = threadIdx.x & (L - 1);
    constexpr unsigned ROWS = RT_THREADS / L;
    float f[N];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        float v[4];
        dm::load_quad(slope + (size_t)group * E, 4 * (q * L + sub), E, 0.0f, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[4 * q + j] = v[j];
    }
    for (unsigned r0 = 0; r0 < at.rows; r0 += ROWS) {
        const unsigned r = r0 + threadIdx.x / L;
        const bool there = r < at.rows;
        const size_t row = (size_t)at.row0 + (there ? r : 0);
        const bool wanted = there && (!set.mask || set.mask[image_row + row] != 0);
        float x[N];
        float mx = ninf;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            float v[4] = {ninf, ninf, ninf, ninf};
            if (wanted) dm::load_quad(base + row * E, 4 * (q * L + sub), E, ninf, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[4 * q + j] = v[j];
                mx = fmaxf(mx, v[j]);                          // (NaN is passed over)
            }
        }
        mx = dm::over_group<L>(mx, dm::Max());
        mx = mx == ninf ? 0.0f : mx;
        const float c = fminf(mx, 0.0f), exp_c = __builtin_amdgcn_exp2f(c * LOG2E);
        float sum = 0.0f, dot = 0.0f;
        float rest[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            rest[j] = 1.0f;
            x[j] = sigmoid ? (x[j] == ninf ? 0.0f : sigmoid_weight(x[j], c, exp_c, &rest[j])) : softmax_weight(x[j], mx);
            sum += x[j];
            dot += x[j] * f[j];
        }
        sum = dm::over_group<L>(sum, dm::Add());
        dot = dm::over_group<L>(dot, dm::Add());
        const bool live = sum != 0.0f;
        const float inv = live ? __builtin_amdgcn_rcpf(sum) : 0.0f;
        dot *= inv;
        const float lse = live ? mx + __builtin_amdgcn_logf(sum) * LN2 : 0.0f;
        const float zpart = gz * lse;
        if (there) {
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = 4 * q + j;
                    v[j] = live ? x[i] * inv * (gb * (f[i] - dot) + zpart) * rest[i] : 0.0f;
                }
                dm::store_quad(out + row * E, 4 * (q * L + sub), E, v);
            }
        }
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

constexpr unsigned ROWS_AT_A_TIME = RT_THREADS / 64;

// Chunks per image of a set: enough workgroups to fill the chip over all sets of the call, none with less than one trip.
unsigned chunks_of(const Shape &sh, int Q)
{
    const long long images = sh.merged ? 1 : sh.B;
    const long long rows = sh.merged ? (long long)sh.B * Q : Q;
    const long long want = std::max(1ll, 1024 / std::max(1ll, (long long)sh.S * images));
    return (unsigned)std::max(1ll, std::min(want, (rows + ROWS_AT_A_TIME - 1) / ROWS_AT_A_TIME));
}

// The kernel arguments of sets first .. first + n - 1; returns the launch's workgroups.
unsigned long long describe(const DmRouterSet *sets, int first, int n, const Shape &sh, int k, RouterSets *a)
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
        s.chunks = chunks_of(sh, in.Q);
        s.chunk_rows = (s.Q + s.chunks - 1) / s.chunks;
        s.first_block = (unsigned)blocks;
        a->first_group[i] = (unsigned)i * (sh.per_image ? (unsigned)sh.B : 1u);
        blocks += (unsigned long long)s.images * s.chunks;
    }
    return blocks;
}

// (the sets of a call go through launches of up to DM_MAX_SETS_PER_LAUNCH, one after the other, over the same workspace)
unsigned long long most_blocks(const DmRouterSet *sets, const Shape &sh)
{
    unsigned long long most = 0;
    for (int first = 0; first < sh.S; first += DM_MAX_SETS_PER_LAUNCH) {
        unsigned long long blocks = 0;
        for (int s = first; s < std::min(sh.S, first + DM_MAX_SETS_PER_LAUNCH); ++s)
            blocks += (unsigned long long)(sh.merged ? 1 : sh.B) * chunks_of(sh, sets[s].Q);
        most = std::max(most, blocks);
    }
    return most;
}

typedef void (*ForwardKernel)(RouterSets, int, unsigned *, int32_t *);
typedef void (*BackwardKernel)(RouterSets, int, const float *, const float *, const float *, const float *);

template <typename T, int NQ>
ForwardKernel forward_of(bool count_only)
{
    return count_only ? router_forward_kernel<T, NQ, 64, true> : router_forward_kernel<T, NQ, 64, false>;
}
template <typename T>
ForwardKernel forward_for(unsigned E, bool count_only)
{
    if (E <= 256) return forward_of<T, 1>(count_only);
    if (E <= 512) return forward_of<T, 2>(count_only);
    return forward_of<T, 4>(count_only);
}
template <typename T>
BackwardKernel backward_for(unsigned E)
{
    if (E <= 256) return router_backward_kernel<T, 1, 64>;
    if (E <= 512) return router_backward_kernel<T, 2, 64>;
    return router_backward_kernel<T, 4, 64>;
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
    const unsigned long long blocks_needed = most_blocks(sets, sh);
    if (blocks_needed >= (1ull << 31)) return DM_E_UNSUPPORTED;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
        workspace_bytes < (int64_t)(blocks_needed * slot_words((unsigned)E) * 4)) return DM_E_INVALID_ARG;
    unsigned *slots = static_cast<unsigned *>(workspace);
    unsigned cols = 1;
    while (cols < 64 && cols < (unsigned)E) cols <<= 1;
    for (int first = 0; first < S; first += DM_MAX_SETS_PER_LAUNCH) {
        RouterSets a;
        const int n = std::min(S - first, DM_MAX_SETS_PER_LAUNCH);
        const unsigned blocks = (unsigned)describe(sets, first, n, sh, top_k, &a);
        if (blocks) {
            const bool count_only = balance == nullptr;
            ForwardKernel kernel = dtype == DM_F32    ? forward_for<float>((unsigned)E, count_only)
                                   : dtype == DM_BF16 ? forward_for<dm::bf16_t>((unsigned)E, count_only)
                                                      : forward_for<dm::half_t>((unsigned)E, count_only);
            hipLaunchKernelGGL(kernel, dim3(blocks), dim3(RT_THREADS), 0, st, a, scores == DM_SCORES_SIGMOID ? 1 : 0, slots, status);
            rc = dm::check_hip(hipGetLastError(), "router_forward_kernel launch");
            if (rc != DM_OK) return rc;
        }
        const size_t g0 = (size_t)first * (per_image ? (size_t)B : 1);
        const unsigned gn = (unsigned)n * (per_image ? (unsigned)B : 1u);
        hipLaunchKernelGGL(router_finish_kernel, dim3(gn), dim3(FINISH_THREADS), 0, st, a, slots, cols,
                           given_counts ? given_counts + g0 * E : nullptr, balance ? balance + g0 : nullptr,
                           z ? z + g0 : nullptr, counts + g0 * E, slope ? slope + g0 * E : nullptr,
                           inv_rows ? inv_rows + g0 : nullptr);
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
    return (int64_t)(std::max(1ull, most_blocks(sets, sh)) * slot_words((unsigned)E) * 4);
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
    if (most_blocks(sets, sh) >= (1ull << 31)) return DM_E_UNSUPPORTED;
    hipStream_t st = static_cast<hipStream_t>(stream);
    for (int first = 0; first < S; first += DM_MAX_SETS_PER_LAUNCH) {
        RouterSets a;
        const int n = std::min(S - first, DM_MAX_SETS_PER_LAUNCH);
        const unsigned blocks = (unsigned)describe(sets, first, n, sh, 0, &a);
        BackwardKernel kernel = dtype == DM_F32    ? backward_for<float>((unsigned)E)
                                : dtype == DM_BF16 ? backward_for<dm::bf16_t>((unsigned)E)
                                                   : backward_for<dm::half_t>((unsigned)E);
        const size_t g0 = (size_t)first * (per_image ? (size_t)B : 1);
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(RT_THREADS), 0, st, a, scores == DM_SCORES_SIGMOID ? 1 : 0,
                           slope + g0 * E, inv_rows + g0, grad_balance ? grad_balance + g0 : nullptr,
                           grad_z ? grad_z + g0 : nullptr);
        rc = dm::check_hip(hipGetLastError(), "router_backward_kernel launch");
        if (rc != DM_OK) return rc;
    }
    return DM_OK;
}
