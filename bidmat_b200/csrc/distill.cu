// Distillation of token columns from a teacher's top logits: loss and gradient.
//
// x: a student's column of logits, (row, z): the teacher's entries of that column, t: the temperature.
//   p_i = exp(z_i/t - Lt), Lt the log-sum-exp of the entries (or given), P = sum p_i
//   L = log sum_v exp(x_v/t)
//   loss = sum_i p_i (log p_i - (x_i/t - L)) = sum_i p_i (z_i - x_i)/t + P (L - Lt)
//   d(w loss)/dx_v = w/t (P exp(x_v/t - L) - p_v)
// The second form of the loss keeps the difference z - x, so it stays exact where the two agree.  What is
// computed once per entry or once per column is in fp64; the sum over the rows is in fp32 per thread.
#include <cuda_runtime.h>

#include "tokens_common.cuh"

using namespace bidmat;

namespace {

constexpr int kDistThreads = 512;

struct Teacher {
    const int *ir, *jc;
    const float *data, *lse;
    int nnz;
};

// Sum / maximum over the CTA, the same value in every thread.
template <bool MAX> __device__ double block_reduce(double v, double *red) {
    v = MAX ? warp_max(v) : warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < kDistThreads / 32; w++) v = MAX ? max_nan(v, red[w]) : v + red[w];
    return v;
}

// LOSS: write the loss; XLSE: write L (else, without LOSS, L is read); GRAD: write the gradient.
template <typename T, bool LOSS, bool GRAD>
__global__ void __launch_bounds__(kDistThreads)
distill_kernel(int nrows, const T *__restrict__ X, long long ldx, float temperature, Teacher z,
               const float *__restrict__ weights, const float *__restrict__ lse_in, float *__restrict__ loss,
               float *__restrict__ lse_out, T *__restrict__ dX, long long lddx) {
    __shared__ double red[kDistThreads / 32];
    const int tid = threadIdx.x;
    const long long c = blockIdx.x;
    const T *x = X + c * ldx;
    const int j0 = max(z.jc[c], 0), j1 = min(z.jc[c + 1], z.nnz);
    const float w = weights ? weights[c] : 1.f;
    const double t = temperature;

    if (GRAD && (w == 0.f || j1 <= j0)) {          // no say in the result: not read
        for (int v = tid; v < nrows; v += kDistThreads) dX[c * lddx + v] = from_float<T>(0.f);
        if (LOSS && tid == 0) loss[c] = 0.f;
        return;
    }
    double L = 0.0;
    if (LOSS) {
        float m = -INFINITY;
        for (int v = tid; v < nrows; v += kDistThreads) m = fmaxf(m, to_float(x[v]));
        m = (float)block_reduce<true>(m, red);
        const float u = m == -INFINITY ? 0.f : m;
        float s = 0.f;
        for (int v = tid; v < nrows; v += kDistThreads) s += expf((to_float(x[v]) - u) / temperature);
        L = u / t + log(block_reduce<false>(s, red));
        if (lse_out && tid == 0) lse_out[c] = (float)L;
    } else {
        L = lse_in[c];
    }
    double lt;
    if (z.lse) {
        lt = z.lse[c];
    } else {
        double m = -INFINITY, s = 0.0;
        for (int j = j0 + tid; j < j1; j += kDistThreads) m = max_nan(m, z.data[j] / t);
        m = block_reduce<true>(m, red);
        if (m == -INFINITY) m = 0.0;
        for (int j = j0 + tid; j < j1; j += kDistThreads) s += exp(z.data[j] / t - m);
        s = block_reduce<false>(s, red);
        lt = s == 0.0 ? INFINITY : m + log(s);     // nothing finite: all p are zero
    }
    double P = 0.0, sum = 0.0;
    for (int j = j0 + tid; j < j1; j += kDistThreads) {
        const int row = z.ir[j];
        const double p = (row >= 0 && row < nrows) ? exp(z.data[j] / t - lt) : NAN;
        P += p;
        if (LOSS && p > 0.0) sum += p * ((z.data[j] - (double)to_float(x[row])) / t);
    }
    P = block_reduce<false>(P, red);
    if (LOSS) {
        sum = block_reduce<false>(sum, red);
        if (tid == 0) loss[c] = P == 0.0 ? 0.f : (float)((GRAD ? (double)w : 1.0) * (sum + P * (L - lt)));
    }
    if (GRAD) {
        const double f = P * w / t;
        for (int v = tid; v < nrows; v += kDistThreads)
            dX[c * lddx + v] = from_float<T>(P == 0.0 ? 0.f : (float)(f * exp((double)to_float(x[v]) / t - L)));
        __syncthreads();
        for (int j = j0 + tid; j < j1; j += kDistThreads) {
            const int row = z.ir[j];
            if (row < 0 || row >= nrows || P == 0.0) continue;
            double p = 0.0;                         // a row that comes twice: its first entry sums them
            bool first = true;
            for (int i = j0; i < j1; i++)
                if (z.ir[i] == row) {
                    if (i < j) first = false;
                    p += exp(z.data[i] / t - lt);
                }
            if (first)
                dX[c * lddx + row] = from_float<T>((float)(w / t * (P * exp((double)to_float(x[row]) / t - L) - p)));
        }
    }
}

int check(int nrows, int ncols, int nnz, const void *X, long long ldx, int dtype, float temperature, const int *Zir,
          const int *Zjc, const float *Zdata) {
    if (nrows < 1 || ncols < 0 || nnz < 0 || !dtype_ok(dtype)) return (int)cudaErrorInvalidValue;
    if (!isfinite(temperature) || temperature <= 0.f) return (int)cudaErrorInvalidValue;
    if (ncols == 0) return 0;
    if (!dense_ok(X, ldx, nrows, dtype) || !Zjc || (nnz > 0 && (!Zir || !Zdata))) return (int)cudaErrorInvalidValue;
    return 0;
}

}  // namespace

extern "C" int bidmat_b200_distill(int nrows, int ncols, int nnz, const void *X, long long ldx, int dtype,
                                   float temperature, const int *Zir, const int *Zjc, const float *Zdata,
                                   const float *Zlse, float *loss, float *Xlse, bidmat_stream_t stream) {
    const int bad = check(nrows, ncols, nnz, X, ldx, dtype, temperature, Zir, Zjc, Zdata);
    if (bad) return bad;
    if (ncols == 0) return 0;
    if (!loss || !Xlse) return (int)cudaErrorInvalidValue;
    cudaStream_t st = as_stream(stream);
    const Teacher z{Zir, Zjc, Zdata, Zlse, nnz};
#define CALL_LOSS(T)                                                                                             \
    distill_kernel<T, true, false><<<ncols, kDistThreads, 0, st>>>(nrows, (const T *)X, ldx, temperature, z, nullptr, \
                                                                   nullptr, loss, Xlse, (T *)nullptr, 0)
    DISPATCH_DTYPE(dtype, CALL_LOSS);
#undef CALL_LOSS
    g_launches += 1;
    return (int)cudaGetLastError();
}

extern "C" int bidmat_b200_distill_grad(int nrows, int ncols, int nnz, const void *X, long long ldx, int dtype,
                                        float temperature, const int *Zir, const int *Zjc, const float *Zdata,
                                        const float *Zlse, const float *Xlse, const float *weights, void *dX,
                                        long long lddx, bidmat_stream_t stream) {
    const int bad = check(nrows, ncols, nnz, X, ldx, dtype, temperature, Zir, Zjc, Zdata);
    if (bad) return bad;
    if (ncols == 0) return 0;
    if (!Xlse || !dense_ok(dX, lddx, nrows, dtype)) return (int)cudaErrorInvalidValue;
    cudaStream_t st = as_stream(stream);
    const Teacher z{Zir, Zjc, Zdata, Zlse, nnz};
#define CALL_GRAD(T)                                                                                             \
    distill_kernel<T, false, true><<<ncols, kDistThreads, 0, st>>>(nrows, (const T *)X, ldx, temperature, z, weights, \
                                                                   Xlse, nullptr, nullptr, (T *)dX, lddx)
    DISPATCH_DTYPE(dtype, CALL_GRAD);
#undef CALL_GRAD
    g_launches += 1;
    return (int)cudaGetLastError();
}

extern "C" int bidmat_b200_distill_with_grad(int nrows, int ncols, int nnz, const void *X, long long ldx, int dtype,
                                             float temperature, const int *Zir, const int *Zjc, const float *Zdata,
                                             const float *Zlse, const float *weights, float *loss, void *dX,
                                             long long lddx, bidmat_stream_t stream) {
    const int bad = check(nrows, ncols, nnz, X, ldx, dtype, temperature, Zir, Zjc, Zdata);
    if (bad) return bad;
    if (ncols == 0) return 0;
    if (!loss || !dense_ok(dX, lddx, nrows, dtype)) return (int)cudaErrorInvalidValue;
    cudaStream_t st = as_stream(stream);
    const Teacher z{Zir, Zjc, Zdata, Zlse, nnz};
#define CALL_BOTH(T)                                                                                             \
    distill_kernel<T, true, true><<<ncols, kDistThreads, 0, st>>>(nrows, (const T *)X, ldx, temperature, z, weights, \
                                                                  nullptr, loss, nullptr, (T *)dX, lddx)
    DISPATCH_DTYPE(dtype, CALL_BOTH);
#undef CALL_BOTH
    g_launches += 1;
    return (int)cudaGetLastError();
}
