// The k largest logits of every token column as a sparse matrix, with the column's log-sum-exp.
//
// Values are compared as whole numbers in the order of the floats.  The k-th largest is found by four rounds
// over eight bits each (a histogram of the values that still agree with the prefix), then everything above it
// is collected, then as many equal values as are missing, lowest rows first, and the k entries are sorted.
#include <cuda_runtime.h>

#include "tokens_common.cuh"

using namespace bidmat;

namespace {

constexpr int kTopThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kTopThreads)
top_logits_kernel(int nrows, int ncols, const T *__restrict__ X, long long ldx, int k, float temperature,
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

}  // namespace

extern "C" int bidmat_b200_top_logits(int nrows, int ncols, const void *X, long long ldx, int dtype, int k,
                                      float temperature, int *Sir, int *Sic, int *Sjc, float *Sdata, float *lse,
                                      bidmat_stream_t stream) {
    if (nrows < 1 || ncols < 0 || !dtype_ok(dtype)) return (int)cudaErrorInvalidValue;
    if (k < 1 || k > nrows || k > BIDMAT_B200_TOP_MAX_K) return (int)cudaErrorInvalidValue;
    if (!isfinite(temperature) || temperature <= 0.f) return (int)cudaErrorInvalidValue;
    if ((long long)k * ncols > 0x7fffffffLL || !Sjc) return (int)cudaErrorInvalidValue;
    cudaStream_t st = as_stream(stream);
    if (ncols == 0) return (int)cudaMemsetAsync(Sjc, 0, sizeof(int), st);
    if (!dense_ok(X, ldx, nrows, dtype) || !Sir || !Sic || !Sdata) return (int)cudaErrorInvalidValue;
#define CALL_TOP(T)                                                                                             \
    top_logits_kernel<T><<<ncols, kTopThreads, 0, st>>>(nrows, ncols, (const T *)X, ldx, k, temperature, Sir, Sic, \
                                                        Sjc, Sdata, lse)
    DISPATCH_DTYPE(dtype, CALL_TOP);
#undef CALL_TOP
    g_launches += 1;
    return (int)cudaGetLastError();
}
