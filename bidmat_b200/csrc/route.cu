// Routing of token columns to experts, and its gradient.
//
//   s = softmax or sigmoid of a column of scores; key = s + bias (without a bias: the score itself, which has
//   the same order); optionally only the experts of the best groups compete; the k best keys are picked, ties
//   to the lower row; weights are s of the picked rows, optionally divided by their sum, times a scale.
//
// The order of two experts whose keys are closer than fp32 can tell has to come out right, so keys that are
// sums with a bias are compared in 64 bits.
#include <cuda_runtime.h>

#include "tokens_common.cuh"

using namespace bidmat;

namespace {

constexpr int kRouteWarps = 4;      // columns in flight per CTA, one warp each

struct RouteArgs {
    int nrows, ncols, k, score, ngroups, topgroups, grouptop, renorm;
    long long ldx;
    float scale;
};

// Best (key, row) over the warp: larger key, then lower row.  row < 0: no candidate.
__device__ __forceinline__ void warp_best(double &key, int &row) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const double k2 = __shfl_xor_sync(0xffffffffu, key, o);
        const int r2 = __shfl_xor_sync(0xffffffffu, row, o);
        if (r2 >= 0 && (row < 0 || k2 > key || (k2 == key && r2 < row))) { key = k2; row = r2; }
    }
}

template <typename T>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_kernel(RouteArgs a, const T *__restrict__ X, const float *__restrict__ bias, int *__restrict__ Sir,
             int *__restrict__ Sic, int *__restrict__ Sjc, float *__restrict__ Sdata) {
    extern __shared__ double route_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long c = (long long)blockIdx.x * kRouteWarps + warp;
    if (c >= a.ncols) return;
    double *rank = route_smem + (size_t)warp * (a.nrows + a.ngroups);      // s + bias, -inf where unavailable
    double *gval = rank + a.nrows;
    const T *x = X + c * a.ldx;
    const double inf = INFINITY;

    bool bad = false;
    double m = -inf;
    for (int e = lane; e < a.nrows; e += 32) {
        const double v = to_float(x[e]);
        bad |= !(v < inf);
        m = v > m ? v : m;
    }
    bad = __any_sync(0xffffffffu, bad);
    m = warp_max(m);
    if (m == -inf) m = 0.0;
    double sum = 0.0;
    if (a.score == BIDMAT_B200_SOFTMAX && !bad) {
        for (int e = lane; e < a.nrows; e += 32) sum += exp((double)to_float(x[e]) - m);
        sum = warp_sum(sum);
    }
    auto score_of = [&](int e) -> double {
        const double v = to_float(x[e]);
        return a.score == BIDMAT_B200_SOFTMAX ? exp(v - m) / sum : 1.0 / (1.0 + exp(-v));
    };
    if (!bad) {
        for (int e = lane; e < a.nrows; e += 32) {
            const double v = to_float(x[e]);
            double r = v > -inf ? score_of(e) + (bias ? (double)bias[e] : 0.0) : -inf;
            if (r != r) r = -inf;
            rank[e] = r;
        }
        __syncwarp();
        const int gsize = a.nrows / a.ngroups;
        if (a.ngroups > 1) {
            for (int g = lane; g < a.ngroups; g += 32) {
                double b1 = -inf, b2 = -inf;
                for (int e = g * gsize; e < (g + 1) * gsize; e++) {
                    const double r = rank[e];
                    if (r > b1) { b2 = b1; b1 = r; } else if (r > b2) b2 = r;
                }
                gval[g] = (a.grouptop == 2 && b2 > -inf) ? b1 + b2 : b1;
            }
            __syncwarp();
            // a group stays if fewer than topgroups groups come before it
            bool drop[BIDMAT_B200_ROUTE_MAX_ROWS / 32];
            int n = 0;
            for (int g = lane; g < a.ngroups; g += 32, n++) {
                int before = 0;
                for (int h = 0; h < a.ngroups; h++)
                    before += gval[h] > gval[g] || (gval[h] == gval[g] && h < g);
                drop[n] = before >= a.topgroups;
            }
            n = 0;
            for (int g = lane; g < a.ngroups; g += 32, n++)
                if (drop[n])
                    for (int e = g * gsize; e < (g + 1) * gsize; e++) rank[e] = -inf;
            __syncwarp();
        }
    } else {
        for (int e = lane; e < a.nrows; e += 32) rank[e] = -inf;
        __syncwarp();
    }
    // k rounds: the best one that is left; then, in the order of the rows, the others with weight zero.
    // NaN marks a row that is taken.
    double w = 0.0;
    int pick = 0;
    for (int i = 0; i < a.k; i++) {
        double key = -inf;
        int row = -1;
        for (int e = lane; e < a.nrows; e += 32) {
            const double r = rank[e];
            if (r != r) continue;
            const double v = r == -inf ? -inf : (bias ? r : (double)to_float(x[e]));
            if (row < 0 || v > key) { key = v; row = e; }
        }
        warp_best(key, row);
        if ((row & 31) == lane) rank[row] = NAN;
        if (lane == i) {
            pick = row;
            w = key > -inf ? score_of(row) : 0.0;
        }
        __syncwarp();
    }
    if (a.renorm) {
        const double tot = warp_sum(w);
        w = tot > 0.0 ? w / tot : 0.0;
    }
    if (lane < a.k) {
        const long long o = c * a.k + lane;
        Sir[o] = pick;
        Sic[o] = (int)c;
        Sdata[o] = bad ? NAN : (float)(w * a.scale);
    }
    if (lane == 0) {
        Sjc[c] = (int)(c * a.k);
        if (c == a.ncols - 1) Sjc[a.ncols] = (int)((c + 1) * a.k);
    }
}

// The gradient of the weights goes back to the scores (w, g: weight and gradient of an entry, D = sum of w g):
//   softmax, renormalised: w (g - D/scale)            sigmoid, renormalised: w (1 - s) (g - D/scale)
//   softmax:  w g at the entries, - p D everywhere    sigmoid:               w (1 - s) g
template <typename T>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_grad_kernel(RouteArgs a, int nnz, const T *X, const int *__restrict__ Sir,
                  const int *__restrict__ Sjc, const float *__restrict__ Sdata, const float *__restrict__ dS,
                  T *dX, long long lddx) {
    extern __shared__ float route_grad_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long c = (long long)blockIdx.x * kRouteWarps + warp;
    if (c >= a.ncols) return;
    float *col = route_grad_smem + (size_t)warp * a.nrows;
    const T *x = X + c * a.ldx;
    const int j0 = max(Sjc[c], 0), j1 = min(Sjc[c + 1], nnz);
    float d = 0.f;
    for (int j = j0 + lane; j < j1; j += 32) d = fmaf(Sdata[j], dS[j], d);
    d = warp_sum(d);
    if (a.score == BIDMAT_B200_SOFTMAX && !a.renorm) {
        float m = -INFINITY, sum = 0.f;
        for (int e = lane; e < a.nrows; e += 32) m = fmaxf(m, to_float(x[e]));
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (m == -INFINITY) m = 0.f;
        for (int e = lane; e < a.nrows; e += 32) {
            const float v = expf(to_float(x[e]) - m);
            col[e] = v;
            sum += v;
        }
        sum = warp_sum(sum);
        const float f = sum > 0.f ? -d / sum : (sum == 0.f ? 0.f : NAN);
        for (int e = lane; e < a.nrows; e += 32) col[e] *= f;
    } else {
        for (int e = lane; e < a.nrows; e += 32) col[e] = 0.f;
    }
    __syncwarp();
    const float back = a.renorm ? d / a.scale : 0.f;
    for (int j = j0; j < j1; j += 32) {
        const bool on = j + lane < j1;
        const int row = on ? Sir[j + lane] : -1;
        float v = 0.f;
        if (row >= 0 && row < a.nrows) {
            v = Sdata[j + lane] * (dS[j + lane] - back);
            if (a.score == BIDMAT_B200_SIGMOID) v *= 1.f / (1.f + expf(to_float(x[row])));
        }
        // one lane at a time: a row that comes twice gets its terms in their order
        for (int l = 0; l < min(32, j1 - j); l++) {
            if (l == lane && row >= 0 && row < a.nrows) col[row] += v;
            __syncwarp();
        }
    }
    for (int e = lane; e < a.nrows; e += 32) dX[c * lddx + e] = from_float<T>(col[e]);
}

bool route_sizes_ok(int nrows, int ncols, int score, float scale) {
    return nrows >= 1 && nrows <= BIDMAT_B200_ROUTE_MAX_ROWS && ncols >= 0 &&
           (score == BIDMAT_B200_SOFTMAX || score == BIDMAT_B200_SIGMOID) && isfinite(scale) && scale != 0.f;
}

}  // namespace

extern "C" int bidmat_b200_route(int nrows, int ncols, const void *X, long long ldx, int dtype, int k, int score,
                                 const float *bias, int ngroups, int topgroups, int grouptop, int renorm, float scale,
                                 int *Sir, int *Sic, int *Sjc, float *Sdata, bidmat_stream_t stream) {
    if (!route_sizes_ok(nrows, ncols, score, scale) || !dtype_ok(dtype)) return (int)cudaErrorInvalidValue;
    if (ngroups < 1 || nrows % ngroups || topgroups < 1 || topgroups > ngroups || (grouptop != 1 && grouptop != 2))
        return (int)cudaErrorInvalidValue;
    if (k < 1 || k > BIDMAT_B200_ROUTE_MAX_K || k > (long long)topgroups * (nrows / ngroups))
        return (int)cudaErrorInvalidValue;
    if ((long long)k * ncols > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    if (!Sjc) return (int)cudaErrorInvalidValue;
    cudaStream_t st = as_stream(stream);
    if (ncols == 0) return (int)cudaMemsetAsync(Sjc, 0, sizeof(int), st);
    if (!dense_ok(X, ldx, nrows, dtype) || !Sir || !Sic || !Sdata) return (int)cudaErrorInvalidValue;
    const RouteArgs a{nrows, ncols, k, score, ngroups, topgroups, grouptop, renorm, ldx, scale};
    const unsigned grid = (unsigned)((ncols + kRouteWarps - 1) / kRouteWarps);
    const size_t smem = (size_t)kRouteWarps * (nrows + ngroups) * sizeof(double);
    cudaError_t err = cudaSuccess;
#define CALL_ROUTE(T)                                                                                           \
    err = cudaFuncSetAttribute(route_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);       \
    if (err == cudaSuccess)                                                                                    \
        route_kernel<T><<<grid, kRouteWarps * 32, smem, st>>>(a, (const T *)X, bias, Sir, Sic, Sjc, Sdata)
    DISPATCH_DTYPE(dtype, CALL_ROUTE);
#undef CALL_ROUTE
    if (err != cudaSuccess) return (int)err;
    g_launches += 1;
    return (int)cudaGetLastError();
}

extern "C" int bidmat_b200_route_grad(int nrows, int ncols, int nnz, const void *X, long long ldx, int dtype, int score,
                                      int renorm, float scale, const int *Sir, const int *Sjc, const float *Sdata,
                                      const float *dS, void *dX, long long lddx, bidmat_stream_t stream) {
    if (!route_sizes_ok(nrows, ncols, score, scale) || !dtype_ok(dtype) || nnz < 0) return (int)cudaErrorInvalidValue;
    if (ncols == 0) return 0;
    if (!dense_ok(X, ldx, nrows, dtype) || !dense_ok(dX, lddx, nrows, dtype) || !Sjc) return (int)cudaErrorInvalidValue;
    if (nnz > 0 && (!Sir || !Sdata || !dS)) return (int)cudaErrorInvalidValue;
    if (X == dX && ldx != lddx) return (int)cudaErrorInvalidValue;
    cudaStream_t st = as_stream(stream);
    RouteArgs a{};
    a.nrows = nrows; a.ncols = ncols; a.score = score; a.renorm = renorm; a.ldx = ldx; a.scale = scale;
    const unsigned grid = (unsigned)((ncols + kRouteWarps - 1) / kRouteWarps);
    const size_t smem = (size_t)kRouteWarps * nrows * sizeof(float);
#define CALL_GRAD(T)                                                                                               \
    route_grad_kernel<T><<<grid, kRouteWarps * 32, smem, st>>>(a, nnz, (const T *)X, Sir, Sjc, Sdata, dS, (T *)dX, lddx)
    DISPATCH_DTYPE(dtype, CALL_GRAD);
#undef CALL_GRAD
    g_launches += 1;
    return (int)cudaGetLastError();
}
