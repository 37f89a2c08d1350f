// The k largest logits of every token column as a sparse matrix, with the column's log-sum-exp.
//
// Values are compared as whole numbers in the order of the floats, and with the lower row first where they are equal.
//
// Columns up to 1.5 MB: a cluster of up to 8 CTAs per column, each with a part of it in shared memory.
//   1. Each thread's vectors form one to four groups, of which it finds the largest value.  With at least k groups in a
//      part, the k-th largest of those maxima is a bound: k values of the part are as large or larger, so nothing below
//      the bound is among the column's k largest.  And it is tight: for values in no particular order little more than k
//      pass it (of 16384 values in 256 groups about 70 for k = 64, 180 for k = 128).
//   2. The values at or above the bound are collected; threads whose maximum is below it have nothing to look at.
//      If there are too many (equal values, a part with fewer groups than k) the part's k largest are found exactly.
//   3. The cluster's first CTA gathers what the parts have found, finds the k-th largest by bisection, and writes
//      every entry at the place that its rank among the survivors gives.
// So X is read once.  Bound by memory: 131072 x 2048 bf16, k = 64, with the log-sum-exp TIMEA.
//
// Longer columns: one CTA per column, four rounds over eight bits of the values each.
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
    int nrows, k;
    long long ldx;
    float t, c;
    int *ir, *ic, *jc;
    float *data, *lse;
};

constexpr int kTop = 256;                   // threads of a part
constexpr int kCollect = BIDMAT_B200_TOP_MAX_K + 64;      // entries that a part can hand on

// The values of a part that pass the bound, in an order of chance.
template <typename T>
__device__ __forceinline__ void collect(const uint4 *kept, int n, int groups, const float (&top)[4], unsigned bound, int row0, int rows,
                                        Entry *list, int limit, int *count) {
    constexpr int N = Pack<T>::N;
#pragma unroll
    for (int g = 0; g < 4; g++) {
        if (g >= groups || order_key(top[g]) < bound) continue;
        for (int i = threadIdx.x + g * kTop; i < n; i += groups * kTop) {
            const uint4 r = kept[i];
            if (order_key(Pack<T>::max_nan(r)) < bound) continue;
            float v[N];
            Pack<T>::unpack(r, v);
#pragma unroll
            for (int j = 0; j < N; j++) {
                const unsigned key = order_key(v[j]);
                const int row = row0 + i * N + j;
                if (key < bound || row < 0 || row >= rows) continue;
                const int at = atomicAdd(count, 1);
                if (at < limit) list[at] = entry_of(key, (unsigned)row);
            }
        }
    }
}

// The part's k largest exactly (k <= values of the part): list[0 .. k).  By the whole CTA.
template <typename T>
__device__ __noinline__ void select_part(const uint4 *kept, int n, int row0, int rows, int k, Entry *list, unsigned *hist, int *shared) {
    constexpr int N = Pack<T>::N;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T *x = reinterpret_cast<const T *>(kept);
    const int lo = row0 < 0 ? -row0 : 0, hi = min(n * N, rows - row0);          // positions that are the column's
    unsigned prefix = 0, left = (unsigned)k;    // the k-th largest agrees with prefix; it is the left-th of those
    for (int shift = 24; shift >= 0; shift -= 8) {
        hist[tid] = 0;
        __syncthreads();
        const unsigned mask = shift == 24 ? 0u : ~0u << (shift + 8);
        for (int u = lo + tid; u < hi; u += kTop) {
            const unsigned key = order_key(to_float(x[u]));
            if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            unsigned m = left;
            int b = 255;
            while (b > 0 && hist[b] < m) m -= hist[b--];
            shared[0] = (int)(prefix | ((unsigned)b << shift));
            shared[1] = (int)m;
        }
        __syncthreads();
        prefix = (unsigned)shared[0];
        left = (unsigned)shared[1];
    }
    __syncthreads();
    if (tid == 0) shared[0] = 0;
    __syncthreads();
    unsigned equal = 0;                         // equal values in the rows before this stretch
    for (int u0 = lo; u0 < hi; u0 += kTop) {
        const int u = u0 + tid;
        const unsigned key = u < hi ? order_key(to_float(x[u])) : 0u;
        if (u < hi && key > prefix) list[atomicAdd(&shared[0], 1)] = entry_of(key, (unsigned)(row0 + u));
        const bool tie = u < hi && key == prefix && equal < left;
        if (__syncthreads_or(tie)) {
            const unsigned vote = __ballot_sync(0xffffffffu, tie);
            if (lane == 0) hist[warp] = __popc(vote);
            __syncthreads();
            unsigned at = equal + __popc(vote & ((1u << lane) - 1u));
            for (int w = 0; w < warp; w++) at += hist[w];
            if (tie && at < left) list[(unsigned)k - left + at] = entry_of(key, (unsigned)(row0 + u));
            for (int w = 0; w < kTop / 32; w++) equal += hist[w];
            __syncthreads();
        }
    }
    __syncthreads();
}

template <typename T, bool LSE>
__global__ void __launch_bounds__(kTop, 5) top_part_kernel(TopArgs a, Layout l, int groups, int limit, const T *X) {
    constexpr int N = Pack<T>::N, W = kTop / 32;
    __shared__ Entry list[kCollect];
    __shared__ unsigned hist[kTop];
    unsigned *maxima = reinterpret_cast<unsigned *>(list);      // of the groups, before there are entries
    static_assert(sizeof(list) >= 4 * kTop * sizeof(unsigned), "the groups' maxima share the list's memory");
    __shared__ float2 sums[W];
    __shared__ int count, shared[2];
    __shared__ unsigned bound;
    extern __shared__ uint4 kept[];
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31;
    const int col = (int)(blockIdx.x / (unsigned)l.parts), part = (int)(blockIdx.x % (unsigned)l.parts);
    const Slice<T> x(X, a.ldx, a.nrows, l, col, part);
    const T *const end = X + (l.ncols - 1) * a.ldx + a.nrows;
    x.template copy<kTop>(kept, X, end);
    if (tid == 0) count = 0;
    const int row0 = x.v0 * N - x.shift;                        // row of position 0
    x.template arrive<kTop>(kept, X, end, X + col * a.ldx, a.nrows);

    // 1. groups and their maxima
    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (groups == 1) {
#pragma unroll 4
        for (int i = tid; i < x.n; i += kTop) top[0] = larger_nan(top[0], Pack<T>::max_nan(kept[i]));
    } else {
#pragma unroll
        for (int g = 0; g < 4; g++)
            for (int i = tid + g * kTop; i < x.n && g < groups; i += groups * kTop) top[g] = larger_nan(top[g], Pack<T>::max_nan(kept[i]));
    }
#pragma unroll
    for (int g = 0; g < 4; g++)
        if (g < groups) maxima[g * kTop + tid] = order_key(top[g]);
    if (LSE) {
        SumExp s;
        s.m = top[0];
#pragma unroll
        for (int g = 1; g < 4; g++) s.m = larger_nan(s.m, top[g]);
        const float ref = s.ref();
        const unsigned long long mr = pair(-ref, -ref), cc = pair(a.c, a.c);
        unsigned long long acc = pair(0.f, 0.f);
#pragma unroll 2
        for (int i = tid; i < x.n; i += kTop) {
            float v[N];
            Pack<T>::unpack(kept[i], v);
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const float2 q = exp_pair(v[j], v[j + 1], mr, cc);
                acc = add2(acc, pair(q.x, q.y));
            }
        }
        const float2 q = unpair(acc);
        s.s = q.x + q.y;
        warp_join(s, a.c);
        if (lane == 0) sums[tid >> 5] = make_float2(s.m, s.s);
    }
    __syncthreads();
    // the bound: 16 bits of the k-th largest maximum are enough
    if (tid < 32) {
        unsigned key[4 * kTop / 32];
#pragma unroll
        for (int i = 0; i < 4 * kTop / 32; i++) key[i] = i < groups * (kTop / 32) ? maxima[i * 32 + lane] : 0u;
        unsigned b = 0;
        for (int bit = 31; bit >= 16; bit--) {
            const unsigned tryb = b | (1u << bit);
            int n = 0;
#pragma unroll
            for (int i = 0; i < kTop / 32; i++) n += key[i] >= tryb;
            if (groups > 1) {
#pragma unroll
                for (int i = kTop / 32; i < 4 * kTop / 32; i++) n += key[i] >= tryb;
            }
            if (__reduce_add_sync(0xffffffffu, n) >= a.k) b = tryb;
        }
        if (lane == 0) bound = b;
    }
    __syncthreads();
    // 2. what passes it
    collect<T>(kept, x.n, groups, top, bound, row0, a.nrows, list, limit, &count);
    __syncthreads();
    int found = count;
    if (found > limit) {                                        // more than limit >= k values
        select_part<T>(kept, x.n, row0, a.nrows, a.k, list, hist, shared);
        found = a.k;
    }
    __syncthreads();
    if (tid == 0) count = found;

    // 3. the cluster's first CTA puts them together
    if (l.parts > 1) {
        cluster.sync();
        if (part != 0) {
            cluster.sync();                                     // stays until it has been read
            return;
        }
    }
    __syncthreads();
    Entry *all = reinterpret_cast<Entry *>(kept);               // the part is no longer needed
    int total = 0;
    for (int p = 0; p < l.parts; p++) {
        const Entry *from = p ? cluster.map_shared_rank(list, p) : list;
        const int m = p ? *cluster.map_shared_rank(&count, p) : count;
        for (int i = tid; i < m; i += kTop) all[total + i] = from[i];
        total += m;
    }
    if (LSE && tid < 32) {
        SumExp s;
        for (int i = lane; i < l.parts * W; i += 32) {
            const float2 v = *cluster.map_shared_rank(&sums[i % W], i / W);
            join(s, v.x, v.y, a.c);
        }
        warp_join(s, a.c);
        if (lane == 0) {
            const double L = s.m == -INFINITY ? (double)(s.s == 0.f ? -INFINITY : NAN) : s.m / (double)a.t + log((double)s.s);
            a.lse[col] = (float)L;
        }
    }
    if (l.parts > 1) cluster.sync();
    else __syncthreads();
    // the largest b that at least k entries reach: by value, and among equal values by row where they are many
    if (tid < 64) hist[tid] = 0;
    __syncthreads();
    Entry b = 0;
    int reach = total;
    for (int bit = 63; bit >= 0 && (bit >= 32 ? reach > a.k : reach > a.k + 64); bit--) {
        const Entry tryb = b | ((Entry)1 << bit);
        int n = 0;
        for (int i = tid; i < total; i += kTop) n += all[i] >= tryb;
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0 && n) atomicAdd(&hist[bit], (unsigned)n);
        __syncthreads();
        n = (int)hist[bit];
        if (n >= a.k) {
            b = tryb;
            reach = n;
        }
    }
    // survivors side by side, then each to its rank
    if (tid == 0) count = 0;
    __syncthreads();
    for (int i = tid; i < total; i += kTop)
        if (all[i] >= b) list[atomicAdd(&count, 1)] = all[i];
    __syncthreads();
    for (int i = tid; i < reach; i += kTop) {
        const Entry e = list[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < reach; j++) rank += list[j] > e;
        if (rank >= a.k) continue;
        const long long o = (long long)col * a.k + rank;
        a.ir[o] = (int)row_of(e);
        a.ic[o] = col;
        a.data[o] = order_value(key_of(e));
    }
    if (tid == 0) {
        a.jc[col] = col * a.k;
        if (col == l.ncols - 1) a.jc[l.ncols] = (col + 1) * a.k;
    }
}

// ---------------------------------------------------------------- longer columns

constexpr int kTopThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kTopThreads)
top_long_kernel(int nrows, int ncols, const T *__restrict__ X, long long ldx, int k, float temperature,
                  int *__restrict__ Sir, int *__restrict__ Sic, int *__restrict__ Sjc, float *__restrict__ Sdata,
                  float *__restrict__ lse) {
    __shared__ unsigned hist[256];
    __shared__ unsigned long long list[BIDMAT_B200_TOP_MAX_K];
    __shared__ double red[kTopThreads / 32];
    __shared__ unsigned warp_cnt[kTopThreads / 32];
    __shared__ unsigned s_prefix, s_left, s_fill;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long c = blockIdx.x;
    const T *x = X + c * ldx;

    unsigned prefix = 0, left = k;      // the k-th largest agrees with prefix; it is the left-th of those
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kTopThreads) hist[i] = 0;
        __syncthreads();
        const unsigned mask = shift == 24 ? 0u : ~0u << (shift + 8);
        for (int v = tid; v < nrows; v += kTopThreads) {
            const unsigned key = order_key(to_float(x[v]));
            if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            unsigned n = left;
            int b = 255;
            while (b > 0 && hist[b] < n) n -= hist[b--];
            s_prefix = prefix | ((unsigned)b << shift);
            s_left = n;
        }
        __syncthreads();
        prefix = s_prefix;
        left = s_left;
    }
    for (int i = tid; i < BIDMAT_B200_TOP_MAX_K; i += kTopThreads) list[i] = 0;
    if (tid == 0) s_fill = 0;
    __syncthreads();
    unsigned equal = 0;                 // equal values in the rows before this stretch
    for (int v0 = 0; v0 < nrows; v0 += kTopThreads) {
        const int v = v0 + tid;
        const unsigned key = v < nrows ? order_key(to_float(x[v])) : 0u;
        const unsigned long long entry = ((unsigned long long)key << 32) | (0xffffffffu - (unsigned)v);
        if (v < nrows && key > prefix) list[atomicAdd(&s_fill, 1u)] = entry;
        const bool tie = v < nrows && key == prefix;
        if (__syncthreads_or(tie && equal < left)) {
            const unsigned vote = __ballot_sync(0xffffffffu, tie);
            if (lane == 0) warp_cnt[warp] = __popc(vote);
            __syncthreads();
            unsigned at = equal + __popc(vote & ((1u << lane) - 1u));
            for (int w = 0; w < warp; w++) at += warp_cnt[w];
            if (tie && at < left) list[k - left + at] = entry;
            for (int w = 0; w < kTopThreads / 32; w++) equal += warp_cnt[w];
            __syncthreads();
        }
    }
    __syncthreads();
    int n = 1;
    while (n < k) n <<= 1;
    for (int size = 2; size <= n; size <<= 1)
        for (int step = size >> 1; step; step >>= 1) {
            for (int i = tid; i < n; i += kTopThreads) {
                const int j = i ^ step;
                if (j > i) {
                    const bool down = (i & size) == 0;
                    const unsigned long long p = list[i], q = list[j];
                    if ((p < q) == down) { list[i] = q; list[j] = p; }
                }
            }
            __syncthreads();
        }
    for (int i = tid; i < k; i += kTopThreads) {
        const long long o = c * k + i;
        Sir[o] = (int)(0xffffffffu - (unsigned)list[i]);
        Sic[o] = (int)c;
        Sdata[o] = order_value((unsigned)(list[i] >> 32));
    }
    if (tid == 0) {
        Sjc[c] = (int)(c * k);
        if (c == ncols - 1) Sjc[ncols] = (int)((c + 1) * k);
    }
    if (lse) {
        const float m = order_value((unsigned)(list[0] >> 32));
        const float u = m == -INFINITY ? 0.f : m;
        double s = 0.0;
        for (int v = tid; v < nrows; v += kTopThreads) s += expf((to_float(x[v]) - u) / temperature);
        s = warp_sum(s);
        if (lane == 0) red[warp] = s;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kTopThreads / 32; w++) s += red[w];
            lse[c] = (float)((double)u / temperature + log(s));
        }
    }
}

// ---------------------------------------------------------------- host side

constexpr long long kPartBytes = 32768, kMostPartBytes = 196608;

// Parts as in the distillation: 32 KB each where that takes 8 of them or fewer, more where columns are few.  Groups: so
// many that the k-th largest maximum is well inside them.
template <typename T>
cudaError_t launch_top(const TopArgs &a, int ncols, const void *X, cudaStream_t st) {
    const long long nvec = most_vectors<T>(X, a.ldx, a.nrows, ncols), bytes = nvec * 16;
    long long parts = (bytes + kPartBytes - 1) / kPartBytes;
    const long long fill = (296 + ncols - 1) / ncols, worth = (nvec + kTop - 1) / kTop;
    if (parts < fill) parts = fill < worth ? fill : worth;
    if (parts > 8) parts = 8;
    const long long per = ((nvec + parts - 1) / parts + 7) & ~7LL;
    if (per * 16 > kMostPartBytes || (long long)ncols * parts > 0x7fffffffLL) {
        top_long_kernel<T><<<ncols, kTopThreads, 0, st>>>(a.nrows, ncols, (const T *)X, a.ldx, a.k, a.t, a.ir, a.ic, a.jc, a.data, a.lse);
        return cudaGetLastError();
    }
    // what the parts hand on has to fit the place of the first one's part
    long long limit = per * 2 / parts;
    if (limit < a.k) limit = a.k;
    if (limit > kCollect) limit = kCollect;
    const size_t smem = (size_t)(per * 16 > parts * limit * 8 ? per * 16 : parts * limit * 8);
    const int groups = a.k <= kTop / 2 ? 1 : (a.k <= kTop ? 2 : 4);
    const auto kernel = a.lse ? top_part_kernel<T, true> : top_part_kernel<T, false>;
    if (smem > 40000) {
        const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (err != cudaSuccess) return err;
    }
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = cluster_config(&attr, (unsigned)(ncols * parts), kTop, (int)parts, smem, st);
    return cudaLaunchKernelEx(&cfg, kernel, a, layout<T>(X, a.ldx, ncols, (int)parts, per), groups, (int)limit, (const T *)X);
}

}  // namespace

extern "C" int bidmat_b200_top_logits(int nrows, int ncols, const void *X, long long ldx, int dtype, int k,
                                      float temperature, int *Sir, int *Sic, int *Sjc, float *Sdata, float *lse,
                                      bidmat_stream_t stream) {
    if (nrows < 1 || nrows > kMostRows || ncols < 0 || ncols > kMostRows || !dtype_ok(dtype)) return (int)cudaErrorInvalidValue;
    if (k < 1 || k > nrows || k > BIDMAT_B200_TOP_MAX_K) return (int)cudaErrorInvalidValue;
    if (!isfinite(temperature) || temperature <= 0.f) return (int)cudaErrorInvalidValue;
    if ((long long)k * ncols > 0x7fffffffLL || !Sjc) return (int)cudaErrorInvalidValue;
    cudaStream_t st = as_stream(stream);
    if (ncols == 0) return (int)cudaMemsetAsync(Sjc, 0, sizeof(int), st);
    if (!dense_ok(X, ldx, nrows, dtype) || !Sir || !Sic || !Sdata) return (int)cudaErrorInvalidValue;
    const TopArgs a{nrows, k, ldx, temperature, (float)(kLog2e / (double)temperature), Sir, Sic, Sjc, Sdata, lse};
    cudaError_t err = cudaSuccess;
#define CALL_TOP(T) err = launch_top<T>(a, ncols, X, st)
    DISPATCH_DTYPE(dtype, CALL_TOP);
#undef CALL_TOP
    g_launches += 1;
    return (int)err;
}
