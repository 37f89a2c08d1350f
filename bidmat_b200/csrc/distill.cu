// Distillation of token columns from a teacher's top logits: loss and gradient.
//
// x: a student's column of logits, (row, z): the teacher's entries of that column, t: the temperature.
//   p_i = exp(z_i/t - Lt), Lt the log-sum-exp of the entries (or given), P = sum p_i
//   L = log sum_v exp(x_v/t)
//   loss = sum_i p_i (log p_i - (x_i/t - L)) = sum_i p_i (z_i - x_i)/t + P (L - Lt)
//   d(w loss)/dx_v = w/t (P exp(x_v/t - L) - p_v)
// The second form of the loss keeps the difference z - x, so it stays exact where the two agree.  What is
// computed once per entry or once per column is in fp64; exponentials over the rows and their sums are in fp32.
//
// All three functions are bound by memory: one read of X, for the gradient one write of dX.
#include <cuda_runtime.h>

#include "tokens_stream.cuh"

using namespace bidmat;
namespace cg = cooperative_groups;

namespace {

constexpr int kStream = 256;              // threads that go over the rows; one more warp looks after the teacher
constexpr int kThreadsAll = kStream + 32;
constexpr int kMarkRows = 32768;          // rows per stretch of a gradient: one mark bit each

struct Teacher {
    const int *ir, *jc;
    const float *data, *lse;
    int nnz;
};

// A column's entries and what they amount to.
struct Entries {
    int j0, j1;
    double lt, P;      // log-sum-exp and mass; P = 0: nothing to learn from, P = NaN: a row outside the matrix
    double cross;      // sum p (z - x)/t
};

// By one warp; x may be null when the loss is not wanted.
template <typename T>
__device__ __forceinline__ Entries read_entries(const Teacher &z, int j0, int j1, long long c, int nrows, double t, const T *x) {
    const int lane = threadIdx.x & 31;
    Entries e;
    e.j0 = j0;
    e.j1 = j1;
    if (z.lse) {
        e.lt = z.lse[c];
    } else {
        double m = -INFINITY, s = 0.0;
        for (int j = j0 + lane; j < j1; j += 32) m = max_nan(m, z.data[j] / t);
        m = warp_max(m);
        const double u = m == -INFINITY ? 0.0 : m;
        for (int j = j0 + lane; j < j1; j += 32) s += exp(z.data[j] / t - u);
        s = warp_sum(s);
        e.lt = s == 0.0 ? INFINITY : u + log(s);       // nothing finite: every p is zero
    }
    e.P = e.cross = 0.0;
    for (int j = j0 + lane; j < j1; j += 32) {
        const int row = z.ir[j];
        const double p = (row >= 0 && row < nrows) ? exp(z.data[j] / t - e.lt) : NAN;
        e.P += p;
        if (x && p > 0.0) e.cross += p * (((double)z.data[j] - (double)to_float(x[row])) / t);
    }
    e.P = warp_sum(e.P);
    e.cross = warp_sum(e.cross);
    return e;
}

// Rows of the vectors [v0, v1) of the gradient: f exp((x - ref)/t) everywhere, and w/t (P q - p) at the
// teacher's rows, q = exp((x - ref)/t) qf.  The rows with an entry are marked first, written by the threads of the entries, and
// left out by the threads that go over the rows; so the column may be overwritten in place.
template <typename T, int THREADS>
__device__ __forceinline__ void write_gradient(const Column<T> &x, T *dx, const Teacher &z, const Entries &e, int v0, int v1,
                                               double t, double w, float ref, double qf, float f, float c, unsigned *marks) {
    constexpr int N = Pack<T>::N;
    constexpr int U = 4;
    const int tid = threadIdx.x;
    T *out = dx - x.shift;                                  // position u is out[u]
    const bool wide = ((reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    for (int a0 = v0; a0 < v1; a0 += kMarkRows / N) {
        const int a1 = min(v1, a0 + kMarkRows / N);
        const long long u0 = (long long)a0 * N, u1 = (long long)a1 * N;
        __syncthreads();
        for (int i = tid; i < kMarkRows / 32; i += THREADS) marks[i] = 0;
        __syncthreads();
        bool twice = false;
        for (int j = e.j0 + tid; j < e.j1; j += THREADS) {
            const int row = z.ir[j];
            const long long u = (long long)row + x.shift - u0;
            if (row < 0 || row >= x.rows || u < 0 || u >= u1 - u0) continue;
            twice |= (atomicOr(&marks[u >> 5], 1u << (u & 31)) >> (u & 31)) & 1u;
        }
        twice = __syncthreads_or(twice);
        for (int j = e.j0 + tid; j < e.j1; j += THREADS) {
            const int row = z.ir[j];
            const long long u = (long long)row + x.shift - u0;
            if (row < 0 || row >= x.rows || u < 0 || u >= u1 - u0) continue;
            double p = exp(z.data[j] / t - e.lt);
            bool mine = true;
            if (twice) {                                    // a row's first entry adds them up in their order
                p = 0.0;
                for (int i = e.j0; i < e.j1; i++)
                    if (z.ir[i] == row) {
                        mine &= i >= j;
                        p += exp(z.data[i] / t - e.lt);
                    }
            }
            if (mine) {
                const double q = exp(((double)to_float(x.base[u + u0]) - ref) / t) * qf;
                out[u + u0] = from_float<T>((float)(w / t * (e.P * q - p)));
            }
        }
        auto scaled = [&](const uint4 &r) {
            const unsigned long long mr = pair(-ref, -ref), cc = pair(c, c), ff = pair(f, f);
            float v[N];
            Pack<T>::unpack(r, v);
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const float2 q = exp_pair(v[j], v[j + 1], mr, cc);
                const float2 y = unpair(mul2(pair(q.x, q.y), ff));
                v[j] = y.x;
                v[j + 1] = y.y;
            }
            return Pack<T>::pack(v);
        };
        // what of vector i is neither marked nor `skip`
        auto store = [&](int i, const uint4 &y, unsigned skip) {
            const int b = (i - a0) * N;
            skip |= (marks[b >> 5] >> (b & 31)) & ((1u << N) - 1u);
            if (wide && !skip) {
                store16(out + (long long)i * N, y);
            } else {
#pragma unroll
                for (int j = 0; j < N; j++)
                    if (!((skip >> j) & 1u)) out[(long long)i * N + j] = reinterpret_cast<const T *>(&y)[j];
            }
        };
        const int f1 = min(a1, x.full1);
        int i = max(a0, x.full0) + tid;
        for (; i < f1 - (U - 1) * THREADS; i += U * THREADS) {
            uint4 r[U];
#pragma unroll
            for (int k = 0; k < U; k++) r[k] = x.load(i + k * THREADS);
#pragma unroll
            for (int k = 0; k < U; k++) store(i + k * THREADS, scaled(r[k]), 0);
        }
        for (; i < f1; i += THREADS) store(i, scaled(x.load(i)), 0);
        if (tid < 2) {
            const int p = x.partial(tid, a0, a1);
            if (p >= 0) {
                unsigned skip = 0;
                for (int j = 0; j < N; j++) skip |= x.inside(p, j) ? 0u : 1u << j;
                store(p, scaled(x.load_partial(p)), skip);
            }
        }
    }
}

template <typename T, int THREADS>
__device__ __forceinline__ void write_zeros(const Column<T> &x, T *dx, int v0, int v1) {
    constexpr int N = Pack<T>::N;
    T *out = dx - x.shift;
    const bool wide = ((reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    for (int i = v0 + (int)threadIdx.x; i < v1; i += THREADS) {
        if (wide && i >= x.full0 && i < x.full1) {
            store16(out + (long long)i * N, make_uint4(0, 0, 0, 0));
        } else {
            for (int j = 0; j < N; j++)
                if (x.inside(i, j)) out[(long long)i * N + j] = from_float<T>(0.f);
        }
    }
}

// The part of nvec vectors that CTA `rank` of `size` has: whole 128-byte lines but for the last.
__device__ __forceinline__ void my_part(int nvec, int rank, int size, int *v0, int *v1) {
    const int per = (((nvec + size - 1) / size) + 7) & ~7;
    *v0 = (int)min((long long)nvec, (long long)rank * per);
    *v1 = (int)min((long long)nvec, (long long)(rank + 1) * per);
}

struct DistillArgs {
    int nrows;
    long long ldx, lddx;
    float t, c;
    Teacher z;
    const float *weights, *lse_in;
    float *loss, *lse_out;
};

// One cluster per column.  GRAD: also write the gradient, after the CTAs have joined their sums.
template <typename T, bool GRAD>
__global__ void __launch_bounds__(kThreadsAll, 4)
distill_kernel(DistillArgs a, const T *X, T *dX) {
    __shared__ float2 parts[kStream / 32];
    __shared__ float2 joined[8];                   // (m, s) of every CTA of the cluster
    __shared__ Entries entries;
    __shared__ unsigned marks[GRAD ? kMarkRows / 32 : 1];
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, rank = (int)cluster.block_rank(), size = (int)cluster.num_blocks();
    const long long col = blockIdx.x / size;
    const double t = a.t;
    const Column<T> x(X + col * a.ldx, a.nrows);
    int v0, v1;
    my_part(x.nvec, rank, size, &v0, &v1);
    const float w = a.weights ? a.weights[col] : 1.f;
    const int j0 = max(a.z.jc[col], 0), j1 = min(a.z.jc[col + 1], a.z.nnz);
    if (GRAD && (w == 0.f || j1 <= j0)) {          // the whole cluster goes this way
        write_zeros<T, kThreadsAll>(x, dX + col * a.lddx, v0, v1);
        if (rank == 0 && tid == 0) a.loss[col] = 0.f;
        return;
    }
    cluster_arrive();                              // waited for before the first access to another CTA's memory
    if (tid >= kStream) {
        if (rank == 0) {
            const Entries e = read_entries<T>(a.z, j0, j1, col, a.nrows, t, X + col * a.ldx);
            if (tid == kStream) entries = e;
        }
    } else {
        SumExp s = sum_exp_slice<T, kStream>(x, v0, v1, a.c);
        warp_join(s, a.c);
        if ((tid & 31) == 0) parts[tid >> 5] = make_float2(s.m, s.s);
    }
    cluster_wait();
    __syncthreads();
    if (tid == 0) {
        SumExp s;
        for (int i = 0; i < kStream / 32; i++) join(s, parts[i].x, parts[i].y, a.c);
        for (int r = 0; r < size; r++)
            if (GRAD || r == 0) *cluster.map_shared_rank(&joined[rank], r) = make_float2(s.m, s.s);
    }
    if (GRAD && rank == 0 && tid > 0 && tid < size) *cluster.map_shared_rank(&entries, tid) = entries;
    cluster.sync();
    if (!GRAD && (rank != 0 || tid != 0)) return;
    SumExp s;
    for (int r = 0; r < size; r++) join(s, joined[r].x, joined[r].y, a.c);
    const Entries e = entries;
    if (rank == 0 && tid == 0) {
        const double L = s.m == -INFINITY ? (double)(s.s == 0.f ? -INFINITY : NAN) : s.m / t + log((double)s.s);
        if (a.lse_out) a.lse_out[col] = (float)L;
        a.loss[col] = e.P == 0.0 ? 0.f : (float)((GRAD ? (double)w : 1.0) * (e.cross + e.P * (L - e.lt)));
    }
    if (GRAD) {
        if (e.P == 0.0) {
            write_zeros<T, kThreadsAll>(x, dX + col * a.lddx, v0, v1);
        } else {
            const double qf = 1.0 / (double)s.s;
            write_gradient<T, kThreadsAll>(x, dX + col * a.lddx, a.z, e, v0, v1, t, w, s.ref(), qf, (float)(e.P * w / t * qf), a.c, marks);
        }
    }
}

// The gradient from a saved log-sum-exp: `size` CTAs per column, each on its own.
template <typename T>
__global__ void __launch_bounds__(kStream, 5)
distill_grad_kernel(DistillArgs a, int size, const T *X, T *dX) {
    __shared__ Entries entries;
    __shared__ unsigned marks[kMarkRows / 32];
    const int tid = threadIdx.x, rank = (int)(blockIdx.x % size);
    const long long col = blockIdx.x / size;
    const double t = a.t;
    const Column<T> x(X + col * a.ldx, a.nrows);
    int v0, v1;
    my_part(x.nvec, rank, size, &v0, &v1);
    const float w = a.weights ? a.weights[col] : 1.f;
    const int j0 = max(a.z.jc[col], 0), j1 = min(a.z.jc[col + 1], a.z.nnz);
    bool none = w == 0.f || j1 <= j0;
    if (!none) {
        if (tid < 32) {
            const Entries e = read_entries<T>(a.z, j0, j1, col, a.nrows, t, nullptr);
            if (tid == 0) entries = e;
        }
        __syncthreads();
        none = entries.P == 0.0;
    }
    if (none) {
        write_zeros<T, kStream>(x, dX + col * a.lddx, v0, v1);
        return;
    }
    const Entries e = entries;
    const double L = a.lse_in[col];
    const float ref = (float)(L * t);
    const double qf = exp(ref / t - L);
    write_gradient<T, kStream>(x, dX + col * a.lddx, a.z, e, v0, v1, t, w, ref, qf, (float)(e.P * w / t * qf), a.c, marks);
}

// CTAs of a cluster per column: enough of them to fill the machine (4 per SM), each with at least 8 KB.
int cluster_for(int ncols, int nrows, int dtype, bool grad) {
    const long long bytes = (long long)nrows * (long long)dtype_size(dtype);
    int size = 1;
    while (size < 8 && bytes / (2 * size) >= 8192 && ((long long)ncols * size < 592 || (grad && bytes / size > 65536))) size *= 2;
    return size;
}

template <typename T, bool GRAD>
cudaError_t launch_distill(const DistillArgs &a, int ncols, int size, const void *X, void *dX, cudaStream_t st) {
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = cluster_config(&attr, (unsigned)ncols * (unsigned)size, kThreadsAll, size, 0, st);
    return cudaLaunchKernelEx(&cfg, distill_kernel<T, GRAD>, a, (const T *)X, (T *)dX);
}

DistillArgs arguments(int nrows, long long ldx, long long lddx, float t, const Teacher &z, const float *weights, const float *lse_in,
                      float *loss, float *lse_out) {
    return DistillArgs{nrows, ldx, lddx, t, (float)(kLog2e / (double)t), z, weights, lse_in, loss, lse_out};
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
    const DistillArgs a = arguments(nrows, ldx, 0, temperature, Teacher{Zir, Zjc, Zdata, Zlse, nnz}, nullptr, nullptr, loss, Xlse);
    const int size = cluster_for(ncols, nrows, dtype, false);
    if ((long long)ncols * size > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    cudaError_t err = cudaSuccess;
#define CALL_LOSS(T) err = launch_distill<T, false>(a, ncols, size, X, nullptr, as_stream(stream))
    DISPATCH_DTYPE(dtype, CALL_LOSS);
#undef CALL_LOSS
    g_launches += 1;
    return (int)err;
}

extern "C" int bidmat_b200_distill_grad(int nrows, int ncols, int nnz, const void *X, long long ldx, int dtype,
                                        float temperature, const int *Zir, const int *Zjc, const float *Zdata,
                                        const float *Zlse, const float *Xlse, const float *weights, void *dX,
                                        long long lddx, bidmat_stream_t stream) {
    const int bad = check(nrows, ncols, nnz, X, ldx, dtype, temperature, Zir, Zjc, Zdata);
    if (bad) return bad;
    if (ncols == 0) return 0;
    if (!Xlse || !dense_ok(dX, lddx, nrows, dtype)) return (int)cudaErrorInvalidValue;
    if (X == dX && ldx != lddx) return (int)cudaErrorInvalidValue;
    const DistillArgs a = arguments(nrows, ldx, lddx, temperature, Teacher{Zir, Zjc, Zdata, Zlse, nnz}, weights, Xlse, nullptr, nullptr);
    // CTAs per column: eight per SM in all, stretches of 2048 rows or more, one stretch of marks at most where that gives enough
    long long size = ((long long)nrows + kMarkRows - 1) / kMarkRows;
    const long long fill = (1184 + (long long)ncols - 1) / ncols;
    if (size < fill) size = fill;
    const long long most = ((long long)nrows + 2047) / 2048;
    if (size > most) size = most;
    if (size * ncols > 0x7fffffffLL) size = 0x7fffffffLL / ncols;
    cudaStream_t st = as_stream(stream);
#define CALL_GRAD(T)                                                                                                     distill_grad_kernel<T><<<(unsigned)(size * ncols), kStream, 0, st>>>(a, (int)size, (const T *)X, (T *)dX)
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
    if (X == dX && ldx != lddx) return (int)cudaErrorInvalidValue;
    const DistillArgs a = arguments(nrows, ldx, lddx, temperature, Teacher{Zir, Zjc, Zdata, Zlse, nnz}, weights, nullptr, loss, nullptr);
    const int size = cluster_for(ncols, nrows, dtype, true);
    if ((long long)ncols * size > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    cudaError_t err = cudaSuccess;
#define CALL_BOTH(T) err = launch_distill<T, true>(a, ncols, size, X, dX, as_stream(stream))
    DISPATCH_DTYPE(dtype, CALL_BOTH);
#undef CALL_BOTH
    g_launches += 1;
    return (int)err;
}
