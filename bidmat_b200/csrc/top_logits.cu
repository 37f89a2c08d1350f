// The k largest logits of every token column as a sparse matrix, with the column's log-sum-exp.
//
// Values are compared as whole numbers in the order of the floats, and with the lower row first where they are equal.
// A CTA, or a cluster of up to 8 where columns are few, goes over a column once, 4 vectors per thread at a time (a round):
//   1. The first round gives a bound.  Each thread's vectors form a group, or four; with at least k groups, the k-th
//      largest of the groups' maxima is a value that k of the round's values reach, so nothing below it is among the
//      column's k largest.  And it is tight: in no particular order, of 8192 values in 256 groups about 70 reach it for
//      k = 64.
//   2. A vector whose largest value is above the bound is set aside, which costs the others one comparison.  Every few
//      rounds the vectors set aside are gone through by all threads, element by element, and what is above the bound is
//      listed.  (Rounds that set aside more than there is room for are repeated one by one.)  When the list has grown, its
//      k-th largest entry becomes the bound.  Rows ascend from round to round, so of equal values the later ones need not
//      be looked at once there are k.
//   3. In the end the parts of a cluster are put together in its first CTA; what the k-th largest entry leaves (k, or a
//      few more) goes to the place that its rank gives.
// With many long columns the exponentials of the log-sum-exp and the steps between the rounds share the time with the
// reading (131072 x 2048 bf16, k = 64: 160 us with the log-sum-exp, 112 us without, 82 us to read), with few columns the chain
// of the steps counts (32768 x 1 fp32, k = 40: 9.4 us).  Parts kept in shared memory and bounded each by itself took 517 us and 14 us: short-lived
// CTAs spent most of their time on the bounds and on waiting for the cluster.
#include <cuda_runtime.h>

#include "tokens_stream.cuh"

using namespace bidmat;
namespace cg = cooperative_groups;

namespace {

typedef unsigned long long Entry;           // order key above, complement of the row below

__device__ __forceinline__ Entry entry_of(unsigned key, unsigned row) { return ((Entry)key << 32) | (0xffffffffu - row); }
__device__ __forceinline__ unsigned key_of(Entry e) { return (unsigned)(e >> 32); }
__device__ __forceinline__ unsigned row_of(Entry e) { return 0xffffffffu - (unsigned)e; }

struct TopArgs {
    int nrows, ncols, k;
    long long ldx;
    float t, c;
    int *ir, *ic, *jc;
    float *data, *lse;
};

constexpr int kTop = 256;                                   // threads
constexpr int kRound = 4;                                   // vectors per thread and round
constexpr int kSlack = 64;                                  // entries beyond k that a selection may leave
constexpr int kBatch = kTop * 4;                            // values that are listed between two looks at the length
constexpr int kList = kBatch + BIDMAT_B200_TOP_MAX_K + kSlack;

struct TopShared {
    Entry list[kList];
    uint4 aside[kTop * kRound];
    int aside_at[kTop * kRound];
    unsigned hist[256];
    float2 sums[kTop / 32];
    int length, set_aside;
    int digit, above, inside;
};

// One of the at most two vectors of a column that are not the column's alone.
template <typename T> __device__ __noinline__ uint4 partial_vector(const T *column, int rows, int i) {
    return Column<T>(column, rows).load_partial(i);
}

// The largest b = d 2^shift that at least k of the list's n entries reach, for the first shift from 56 down in steps of
// 8 to `last` with which no more than k + kSlack do; how many reach it.  By the whole CTA, k <= n.
__device__ __forceinline__ Entry select(TopShared &sh, int n, int k, int last, int *reach) {
    const int tid = threadIdx.x, lane = tid & 31;
    Entry b = 0;
    int left = k;                                           // the k-th largest is the left-th of those that agree with b
    *reach = n;
    for (int shift = 56; shift >= last; shift -= 8) {
        sh.hist[tid] = 0;
        __syncthreads();
        const Entry mask = shift == 56 ? 0 : ~(Entry)0 << (shift + 8);
        for (int i = tid; i < n; i += kTop) {
            const Entry e = sh.list[i];
            if ((e & mask) == b) atomicAdd(&sh.hist[(unsigned)(e >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (tid < 32) {                                     // lane 0 has the highest eight digits
            int own[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) sum += own[i] = (int)sh.hist[255 - 8 * lane - i];
            int before = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before += v;
            }
            before -= sum;
            if (before < left && left <= before + sum) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (before < left && left <= before + own[i]) {
                        sh.digit = 255 - 8 * lane - i;
                        sh.above = before;
                        sh.inside = own[i];
                    }
                    before += own[i];
                }
            }
        }
        __syncthreads();
        b |= (Entry)sh.digit << shift;
        left -= sh.above;
        *reach = k - left + sh.inside;
        if (sh.inside - left <= kSlack) break;
    }
    return b;
}

// Leaves the entries that reach b; there is room for them in front.
__device__ __forceinline__ void keep_from(TopShared &sh, int n, Entry b) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid == 0) sh.length = 0;
    Entry mine[(kList + kTop - 1) / kTop];
#pragma unroll
    for (int k = 0; k < (kList + kTop - 1) / kTop; k++) mine[k] = tid + k * kTop < n ? sh.list[tid + k * kTop] : 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < (kList + kTop - 1) / kTop; k++)
        if (tid + k * kTop < n && mine[k] >= b) sh.list[atomicAdd(&sh.length, 1)] = mine[k];
    __syncthreads();
}

// Cuts the list to its k largest and a few; what they reach.
__device__ __noinline__ Entry cut(TopShared &sh, int k) {
    int reach;
    const Entry b = select(sh, sh.length, k, 0, &reach);
    keep_from(sh, sh.length, b);
    return b;
}

// Goes through the vectors that were set aside: what is above `bound` is listed.  Where the list gets long it is cut, and
// what its k largest reach is the new bound; the entries of a round come in no order, so within it rows count as well.
template <typename T> __device__ __noinline__ unsigned go_through(TopShared &sh, int row0, int rows, int k, unsigned bound) {
    constexpr int N = Pack<T>::N, PER = kBatch / N;         // vectors per batch
    const int n = sh.set_aside;
    Entry from = bound == 0xffffffffu ? ~(Entry)0 : (Entry)(bound + 1) << 32;
    for (int first = 0; first < n; first += PER) {
        // All threads cut or none does.  Some may read the length before others have added to it, but the last to add reads all
        // of it; and nobody adds again before every thread has read it.
        if (__syncthreads_or(sh.length > kList - kBatch)) from = max(from, cut(sh, k));
        const int last = min(n, first + PER);
        for (int i = first * N + (int)threadIdx.x; i < last * N; i += kTop) {
            const unsigned key = order_key(to_float(reinterpret_cast<const T *>(sh.aside)[i]));
            const int row = row0 + sh.aside_at[i / N] * N + (i & (N - 1));
            const Entry e = entry_of(key, (unsigned)row);
            if (e >= from && row >= 0 && row < rows) sh.list[atomicAdd(&sh.length, 1)] = e;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.set_aside = 0;
    if (sh.length >= 2 * k + 128) from = max(from, cut(sh, k));
    // later rows are larger: what equals the k-th of the list comes behind it
    return from == (Entry)(bound + 1) << 32 ? bound : key_of(from);
}

// A bound as a float, of which NaN wants everything; 0x7fffffff, the key below zero's, would be the other zero.
__device__ __forceinline__ float limit_of(unsigned key) { return order_value(key == 0x7fffffffu ? key - 1 : key); }

// This thread's vectors of the round that starts at r0, -infinity behind v1.
template <typename T>
__device__ __forceinline__ void read_round(const Column<T> &x, int f0, int f1, int v1, int r0, uint4 (&r)[kRound]) {
    constexpr int N = Pack<T>::N;
    if (r0 >= f0 && r0 + kTop * kRound <= f1) {
        const T *p = x.base + (long long)(r0 + (int)threadIdx.x) * N;
#pragma unroll
        for (int k = 0; k < kRound; k++) r[k] = load16(p + k * kTop * N);
    } else {
#pragma unroll
        for (int k = 0; k < kRound; k++) {
            const int i = r0 + (int)threadIdx.x + k * kTop;
            r[k] = i >= f0 && i < f1 ? x.load(i) : (i < v1 ? partial_vector(x.base + x.shift, x.rows, i) : Pack<T>::lowest());
        }
    }
}

// Sets aside what may be above the limit, as far as there is room.
__device__ __forceinline__ void set_aside(TopShared &sh, const uint4 (&r)[kRound], const float (&top)[kRound], float limit, int r0, int v1) {
#pragma unroll
    for (int k = 0; k < kRound; k++)
        if (!(top[k] <= limit) && (r0 + kTop * kRound <= v1 || r0 + (int)threadIdx.x + k * kTop < v1)) {
            const int at = atomicAdd(&sh.set_aside, 1);
            if (at < kTop * kRound) {
                sh.aside[at] = r[k];
                sh.aside_at[at] = r0 + (int)threadIdx.x + k * kTop;
            }
        }
}

// The rounds from r0 to r1 once more, one at a time, because more had to be set aside than there was room for.
template <typename T>
__device__ __noinline__ unsigned repeat(TopShared &sh, const T *column, int rows, int f0, int f1, int v1, int r0, int r1, int k, unsigned bound) {
    const Column<T> x(column, rows);
    for (; r0 < r1; r0 += kTop * kRound) {
        __syncthreads();
        if (threadIdx.x == 0) sh.set_aside = 0;
        __syncthreads();
        uint4 r[kRound];
        float top[kRound];
        read_round(x, f0, f1, v1, r0, r);
#pragma unroll
        for (int i = 0; i < kRound; i++) top[i] = Pack<T>::max_nan(r[i]);
        set_aside(sh, r, top, limit_of(bound), r0, v1);
        __syncthreads();
        bound = go_through<T>(sh, -x.shift, x.rows, k, bound);
    }
    return bound;
}

template <typename T, bool LSE>
__global__ void __launch_bounds__(kTop, LSE ? 3 : 4) top_kernel(TopArgs a, int groups, const T *X) {
    __shared__ TopShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, part = (int)cluster.block_rank(), parts = (int)cluster.num_blocks();
    const int col = (int)(blockIdx.x / (unsigned)parts);
    const Column<T> x(X + col * a.ldx, a.nrows);
    int v0, v1;
    my_part(x.nvec, part, parts, &v0, &v1);
    const int row0 = -x.shift;                                  // row of position 0
    if (tid == 0) sh.length = sh.set_aside = 0;
    unsigned bound = 0;                                         // values with a larger key are wanted
    float limit = limit_of(bound);
    SumExp s;
    const int step = kTop * kRound, f0 = max(v0, x.full0), f1 = min(v1, x.full1);
    // Rounds between two barriers: one at first, then as many as are likely to find room for what they set aside.
    const int block = a.k <= 128 ? 4 : (a.k <= 256 ? 2 : 1);
    uint4 next[kRound];
    if (v0 < v1) read_round(x, f0, f1, v1, v0, next);
    for (int b0 = v0; b0 < v1;) {
        const int b1 = min(v1, b0 + (b0 == v0 ? step : block * step));
        unsigned first = 0;
        for (int r0 = b0; r0 < b1; r0 += step) {
            uint4 r[kRound];
            float top[kRound];
#pragma unroll
            for (int k = 0; k < kRound; k++) r[k] = next[k];
            if (r0 + step < v1) read_round(x, f0, f1, v1, r0 + step, next);
#pragma unroll
            for (int k = 0; k < kRound; k++) top[k] = Pack<T>::max_nan(r[k]);
            if (LSE) add_vectors<T, kRound>(s, r, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), a.c);
            if (r0 == v0) {
                // 16 bits of the k-th largest maximum are enough; what equals them is wanted here
                if (groups == kTop) {
                    sh.list[tid] = (Entry)order_key(larger_nan(larger_nan(top[0], top[1]), larger_nan(top[2], top[3]))) << 32;
                } else {
#pragma unroll
                    for (int k = 0; k < kRound; k++) sh.list[tid + k * kTop] = (Entry)order_key(top[k]) << 32;
                }
                __syncthreads();
                int reach;
                first = key_of(select(sh, groups, a.k, 48, &reach));
                // groups of nothing but -infinity, or of nothing at all, give no bound
                bound = first > order_key(-INFINITY) ? first - 1 : 0;
                limit = limit_of(bound);
            }
            set_aside(sh, r, top, limit, r0, v1);
        }
        __syncthreads();
        const int aside = sh.set_aside;
        const unsigned before = bound;
        if (aside > kTop * kRound) bound = repeat(sh, x.base + x.shift, x.rows, f0, f1, v1, b0, b1, a.k, bound);
        else if (aside > 0) bound = go_through<T>(sh, row0, a.nrows, a.k, bound);
        if (b0 == v0 && before > 0) bound = max(bound, first);
        limit = limit_of(bound);
        __syncthreads();
        b0 = b1;
    }
    if (LSE) {
        warp_join(s, a.c);
        if (lane == 0) sh.sums[tid >> 5] = make_float2(s.m, s.s);
    }
    __syncthreads();
    if (sh.length > a.k + kSlack) cut(sh, a.k);
    if (parts > 1) {
        cluster.sync();
        if (part == 0) {
            for (int p = 1; p < parts; p++) {
                const int m = *cluster.map_shared_rank(&sh.length, p);
                if (sh.length + m > kList) cut(sh, a.k);
                const int n = sh.length;
                const Entry *from = cluster.map_shared_rank(sh.list, p);
                for (int i = tid; i < m; i += kTop) sh.list[n + i] = from[i];
                __syncthreads();
                if (tid == 0) sh.length = n + m;
                __syncthreads();
            }
        }
    }
    if (LSE && part == 0 && tid < 32) {
        s = SumExp();
        for (int i = lane; i < parts * (kTop / 32); i += 32) {
            const float2 v = *cluster.map_shared_rank(&sh.sums[i % (kTop / 32)], i / (kTop / 32));
            join(s, v.x, v.y, a.c);
        }
        warp_join(s, a.c);
        if (lane == 0) a.lse[col] = (float)(s.m / (double)a.t + s.log_sum(a.c));
    }
    if (parts > 1) cluster.sync();                              // a part stays until it has been read
    if (part != 0) return;
    if (sh.length > a.k + kSlack) cut(sh, a.k);
    const int n = sh.length;
    for (int i = tid; i < n; i += kTop) {
        const Entry e = sh.list[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; j++) rank += sh.list[j] > e;
        if (rank >= a.k) continue;
        const long long o = (long long)col * a.k + rank;
        a.ir[o] = (int)row_of(e);
        a.ic[o] = col;
        a.data[o] = order_value(key_of(e));
    }
    if (tid == 0) {
        a.jc[col] = col * a.k;
        if (col == a.ncols - 1) a.jc[a.ncols] = (col + 1) * a.k;
    }
}

// A CTA per column, or as many as the machine holds at a time (three or four per SM): a second wave would cost more than a
// CTA's longer way (100003 x 257 fp16: 28 us in one part, 43 us in three).
template <typename T> cudaError_t launch_top(const TopArgs &a, const void *X, cudaStream_t st) {
    const long long bytes = (long long)a.nrows * (long long)sizeof(T);
    const long long fill = 3 * kSMs / a.ncols, worth = (bytes + 8191) / 8192;
    long long parts = fill < worth ? fill : worth;
    if (parts < 1) parts = 1;
    if (parts > 8) parts = 8;
    if ((long long)a.ncols * parts > 0x7fffffffLL) parts = 1;
    const int groups = a.k <= kTop / 2 ? kTop : kTop * kRound;
    const auto kernel = a.lse ? top_kernel<T, true> : top_kernel<T, false>;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = cluster_config(&attr, (unsigned)(a.ncols * parts), kTop, (int)parts, 0, st);
    return cudaLaunchKernelEx(&cfg, kernel, a, groups, (const T *)X);
}

}  // namespace

extern "C" int bidmat_b200_top_logits(int nrows, int ncols, const void *X, long long ldx, int dtype, int k,
                                      float temperature, int *Sir, int *Sic, int *Sjc, float *Sdata, float *lse,
                                      bidmat_stream_t stream) {
    if (nrows < 1 || nrows > kMostRows || ncols < 0 || ncols > kMostRows || !dtype_ok(dtype)) return (int)cudaErrorInvalidValue;
    if (k < 1 || k > nrows || k > BIDMAT_B200_TOP_MAX_K) return (int)cudaErrorInvalidValue;
    if (!temperature_ok(temperature)) return (int)cudaErrorInvalidValue;
    if ((long long)k * ncols > 0x7fffffffLL || !Sjc) return (int)cudaErrorInvalidValue;
    cudaStream_t st = as_stream(stream);
    if (ncols == 0) return (int)cudaMemsetAsync(Sjc, 0, sizeof(int), st);
    if (!dense_ok(X, ldx, nrows, dtype) || !Sir || !Sic || !Sdata) return (int)cudaErrorInvalidValue;
    const TopArgs a{nrows, ncols, k, ldx, temperature, (float)(kLog2e / (double)temperature), Sir, Sic, Sjc, Sdata, lse};
    cudaError_t err = cudaSuccess;
#define CALL_TOP(T) err = launch_top<T>(a, X, st)
    DISPATCH_DTYPE(dtype, CALL_TOP);
#undef CALL_TOP
    if (err == cudaSuccess) g_launches += 1;
    return (int)err;
}
