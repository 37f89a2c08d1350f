// Distillation of token columns from a teacher's top logits: loss and gradient.
//
// x: a student's column of logits, (row, z): the teacher's entries of that column, t: the temperature.
//   p_i = exp(z_i/t - Lt), Lt the log-sum-exp of the entries (or given), P = sum p_i
//   L = log sum_v exp(x_v/t)
//   loss = sum_i p_i (log p_i - (x_i/t - L)) = sum_i p_i (z_i - x_i)/t + P (L - Lt)
//   d(w loss)/dx_v = w/t (P exp(x_v/t - L) - p_v)
// The second form of the loss keeps the difference z - x, so it stays exact where the two agree; z is taken relative to the
// entries' largest, x to the largest logit at an entry, so that neither loses anything where all are masked by a large number.
// Masses and the loss are in fp64; exponentials over the rows, their sums and the gradient are in fp32.  So is the gradient at a
// column's first 128 entries, which a warp has in registers with their masses (fp64 there would make the chain that the other
// warps wait for longer); further entries, and those of a row that comes twice, are gone through again in fp64.
//
// All three functions are bound by memory: one read of X, for the gradient one write of dX.
#include <cuda_runtime.h>

#include "tokens_stream.cuh"

using namespace bidmat;
namespace cg = cooperative_groups;

namespace {

constexpr int kStream = 256;              // threads that go over the rows; one more warp looks after the teacher
constexpr int kMarkRows = 32768;          // rows per stretch of a gradient: one mark bit each

struct Teacher {
    const int *ir, *jc;
    const float *data, *lse;
    int nnz;
};

// What a column's entries amount to.
struct Entries {
    double zr, lt;     // p = exp((z - zr)/t - lt): the largest z and the log-sum-exp relative to it, or 0 and the one given
    double P;          // mass; 0: nothing to learn from, NaN: a row outside the matrix
    double xr;         // a logit next to the largest at an entry
    double cross;      // sum p ((z - zr) - (x - xr))/t
};

// p of an entry, 0 for -infinity also where the log-sum-exp is -infinity (a teacher's column of nothing else).
__device__ __forceinline__ double mass(float z, double zr, double it, double lt) {
    return z == -INFINITY ? 0.0 : exp((z - zr) * it - lt);
}

// Entries that a warp has in registers: the first 32 R of a column.
constexpr int R = 4;
struct Held {
    int j0, j1;
    int row[R];         // -1: none
    float z[R];
};
__device__ __forceinline__ void hold(Held &h, const Teacher &z, int j0, int j1) {
    const int lane = threadIdx.x & 31;
    h.j0 = j0;
    h.j1 = j1;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int j = j0 + 32 * r + lane;
        h.z[r] = j < j1 ? z.data[j] : -INFINITY;
        h.row[r] = j < j1 ? z.ir[j] : -1;
    }
}

// By one warp.  x: the student's column, read WITH_X.  xr, pr: the student's logits and the masses of the
// entries held.  it: 1/t; differences times it are as near as differences over t.  One exponential each.
template <typename T, bool WITH_X>
__device__ __forceinline__ Entries weigh_entries(const Held &h, const Teacher &z, long long c, int nrows, double it, const T *x,
                                                 float (&xr)[R], float (&pr)[R]) {
    const int lane = threadIdx.x & 31;
    double lt = 0.0, zr = 0.0, near = 0.0;
    if (z.lse) lt = z.lse[c];
    bool outside = false;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const bool in = h.row[r] >= 0 && h.row[r] < nrows;
        outside |= !in && h.j0 + 32 * r + lane < h.j1;
        xr[r] = WITH_X && in ? to_float(x[h.row[r]]) : 0.f;
    }
    const int rest = h.j0 + 32 * R + lane;
    if (!z.lse) {
        double m = -INFINITY;
#pragma unroll
        for (int r = 0; r < R; r++) m = max_nan(m, (double)h.z[r]);
        for (int j = rest; j < h.j1; j += 32) m = max_nan(m, (double)z.data[j]);
        m = warp_max(m);
        zr = m == -INFINITY ? 0.0 : m;
    }
    if (WITH_X) {                       // the largest of those held is near enough
        float top = -INFINITY;
#pragma unroll
        for (int r = 0; r < R; r++)
            if (h.row[r] >= 0 && h.row[r] < nrows && fabsf(xr[r]) < INFINITY) top = fmaxf(top, xr[r]);
        top = warp_top(top);
        near = top == -INFINITY ? 0.f : top;
    }
    double s = 0.0, cross = 0.0;
    auto add = [&](float zj, float xj) {
        const double e = mass(zj, zr, it, lt);
        s += e;
        if (WITH_X && e > 0.0) cross += e * (((zj - zr) - (xj - near)) * it);
        return e;
    };
#pragma unroll
    for (int r = 0; r < R; r++) {
        pr[r] = 0.f;
        if (h.j0 + 32 * r < h.j1) pr[r] = (float)add(h.z[r], xr[r]);
    }
    for (int j = rest; j < h.j1; j += 32) {
        const int rj = z.ir[j];
        const bool in = rj >= 0 && rj < nrows;
        outside |= !in;
        add(z.data[j], WITH_X && in ? to_float(x[rj]) : 0.f);
    }
    s = warp_sum(s);
    if (WITH_X) cross = warp_sum(cross);
    outside = __any_sync(0xffffffffu, outside);
    Entries e;
    e.zr = zr;
    e.xr = near;
    if (z.lse) {
        e.lt = lt;
        e.P = s;
        e.cross = cross;
    } else {
        e.lt = s == 0.0 ? INFINITY : log(s);               // nothing finite: every p is zero
        e.P = s == 0.0 ? 0.0 : s / s;                       // one, or NaN
        e.cross = cross / s;
#pragma unroll
        for (int r = 0; r < R; r++) pr[r] = s == 0.0 ? 0.f : pr[r] / (float)s;
    }
    if (outside) e.P = e.cross = NAN;
    return e;
}

// What the gradient of a column is made of: f exp((x - ref)/t) at every row, w/t (P qf exp((x - ref)/t) - p) at
// the teacher's.
struct Slope {
    float t, c, w, ref, f;
    double it, qf, zr, lt, P;
};

// One stretch of the gradient is the vectors [a0, a1) of a column, at most kMarkRows rows.  The rows with an
// entry are marked first, are written by the threads that have the entries and left out by those that
// go over the rows; so the column may be overwritten in place (what a vector holds at a marked row is not used).

// A barrier of the first THREADS threads only.
template <int THREADS> __device__ __forceinline__ void sync_first() { asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory"); }

// The first THREADS threads mark the stretch's entries; `twice` is set when a row comes twice.  To be seen by
// others after a barrier.
template <typename T, int THREADS>
__device__ __forceinline__ void mark_entries(const Column<T> &x, const Teacher &z, int j0, int j1, int a0, int a1, unsigned *marks,
                                             int *twice) {
    constexpr int N = Pack<T>::N;
    const int tid = threadIdx.x;
    for (int i = tid; i < (a1 - a0) * N / 32 + 1; i += THREADS) marks[i] = 0;
    if (tid == 0) *twice = 0;
    sync_first<THREADS>();
    for (int j = j0 + tid; j < j1; j += THREADS) {
        const int row = z.ir[j];
        const long long u = (long long)row + x.shift - (long long)a0 * N;
        if (row < 0 || row >= x.rows || u < 0 || u >= (long long)(a1 - a0) * N) continue;
        if ((atomicOr(&marks[u >> 5], 1u << (u & 31)) >> (u & 31)) & 1u) *twice = 1;
    }
}

// The rows with an entry, by `count` threads of which this is number `who`.
template <typename T>
__device__ __forceinline__ void write_entries(const Column<T> &x, T *out, const Teacher &z, int j0, int j1, int a0, int a1,
                                              const Slope &g, bool twice, int who, int count) {
    constexpr int N = Pack<T>::N;
    for (int j = j0 + who; j < j1; j += count) {
        const int row = z.ir[j];
        const long long u = (long long)row + x.shift - (long long)a0 * N;
        if (row < 0 || row >= x.rows || u < 0 || u >= (long long)(a1 - a0) * N) continue;
        double p = mass(z.data[j], g.zr, g.it, g.lt);
        if (twice) {                                    // a row's first entry adds them up in their order
            bool mine = true;
            p = 0.0;
            for (int i = j0; i < j1; i++)
                if (z.ir[i] == row) {
                    mine &= i >= j;
                    p += mass(z.data[i], g.zr, g.it, g.lt);
                }
            if (!mine) continue;
        }
        const float xv = to_float(x.base[u + (long long)a0 * N]);
        const double q = exp(((double)xv - g.ref) * g.it) * g.qf;
        out[u + (long long)a0 * N] = from_float<T>(g.P == 0.0 ? 0.f : (float)(g.w * g.it * (g.P * q - p)));
    }
}

// The other rows.
template <typename T, int THREADS>
__device__ __forceinline__ void write_rows(const Column<T> &x, T *out, int a0, int a1, const Slope &g, const unsigned *marks) {
    constexpr int N = Pack<T>::N;
    constexpr int U = 4;
    const int tid = threadIdx.x;
    const bool wide = ((reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const unsigned long long mr = pair(-g.ref, -g.ref), cc = pair(g.c, g.c), ff = pair(g.f, g.f);
    auto scaled = [&](const uint4 &r) {
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
    // what of vector i is neither marked nor in `skip`
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

// The vectors [v0, v1) of the gradient, read again, stretch by stretch.
template <typename T, int THREADS>
__device__ __forceinline__ void write_gradient(const Column<T> &x, T *out, const Teacher &z, int j0, int j1, int v0, int v1,
                                               const Slope &g, unsigned *marks, int *twice) {
    for (int a0 = v0; a0 < v1; a0 += kMarkRows / Pack<T>::N) {
        const int a1 = min(v1, a0 + kMarkRows / Pack<T>::N);
        __syncthreads();
        if (threadIdx.x < kStream) mark_entries<T, kStream>(x, z, j0, j1, a0, a1, marks, twice);
        __syncthreads();
        write_entries<T>(x, out, z, j0, j1, a0, a1, g, *twice, (int)threadIdx.x, THREADS);
        write_rows<T, THREADS>(x, out, a0, a1, g, marks);
    }
}

template <typename T, int THREADS>
__device__ __forceinline__ void write_zeros(const Column<T> &x, T *out, int v0, int v1) {
    constexpr int N = Pack<T>::N;
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

struct DistillArgs {
    int nrows;
    long long ldx, lddx;
    float t, c;
    double it;                      // 1/t
    Teacher z;
    const float *weights, *lse_in;
    float *loss, *lse_out;
};

// ---------------------------------------------------------------- columns that fit shared memory
//
// A CTA has a part of a column, which starts on its way to shared memory as the first thing.  Meanwhile one more warp
// goes through the entries: a chain of dependent loads and fp64 exponentials that takes about as long.  It marks the
// entries' rows, which the other warps leave out when they write, and writes those itself.
//   BOTH: the CTAs of a cluster have one column.  Every warp sums up its rows and sends (m, s) to every CTA.
//   GRAD: the log-sum-exp is given; CTAs have nothing to do with one another.
// CTAs are short-lived and three to five of them share an SM, so that one's loads overlap another's arithmetic and stores.
enum Mode { GRAD, BOTH };

// The sum of what every warp of the cluster has sent here.
template <int W> __device__ __forceinline__ SumExp receive(unsigned long long *arrived, const float2 *joined, int count, float c) {
    const bool ok = mail_wait(arrived, 0);
    SumExp s;
    for (int i = threadIdx.x & 31; i < count; i += 32) join(s, joined[i].x, joined[i].y, c);
    warp_join(s, c);
    if (!ok) s.s = NAN;             // never seen; an answer that cannot be mistaken for one
    return s;
}

template <bool WITH_LSE>
__device__ __forceinline__ void write_loss(const DistillArgs &a, long long col, const SumExp &s, const Entries &e, float w) {
    const double l = s.log_sum(a.c);
    if (WITH_LSE) a.lse_out[col] = (float)(s.m * a.it + l);
    a.loss[col] = e.P == 0.0 ? 0.f : (float)((double)w * (e.cross + e.P * ((s.m - e.xr) * a.it + l - e.lt)));
}

template <typename T, int THREADS, Mode MODE>
__global__ void __launch_bounds__(THREADS + 32, THREADS == 64 ? 14 : (MODE == GRAD ? 5 : 3))
distill_part_kernel(DistillArgs a, Layout l, const T *X, T *dX) {
    constexpr int N = Pack<T>::N, W = THREADS / 32;
    __shared__ float2 joined[MODE == GRAD ? 1 : 8 * W];         // (m, s) of every warp of the cluster
    __shared__ unsigned long long arrived;
    __shared__ float2 slope;                                    // factor P w/t, in GRAD times the rest of the reference; reference
    __shared__ int twice;                                       // 1: a row came twice, 2: the gradient is zero
    extern __shared__ uint4 kept[];                             // the part's vectors, then its marks: a byte per vector, a bit per element
    unsigned char *marks = reinterpret_cast<unsigned char *>(kept + l.per);
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31;
    const int col = (int)(blockIdx.x / (unsigned)l.parts), part = (int)(blockIdx.x % (unsigned)l.parts);
    const Slice<T> x(X, a.ldx, a.nrows, l, col, part);
    const int j0 = max(a.z.jc[col], 0), j1 = min(a.z.jc[col + 1], a.z.nnz);
    const float w = a.weights ? a.weights[col] : 1.f;
    const float lse = MODE == GRAD ? a.lse_in[col] : 0.f;
    const T *const end = X + (l.ncols - 1) * a.ldx + a.nrows;
    T *out = dX + (col * a.lddx + ((long long)x.v0 * N - x.shift));     // position 0 of the part

    if (w == 0.f || j1 <= j0) {         // nothing is read; the whole cluster goes this way
        const Column<T> whole(X + col * a.ldx, a.nrows);
        write_zeros<T, THREADS + 32>(whole, dX + col * a.lddx - x.shift, x.v0, x.v0 + x.n);
        if (MODE == BOTH && part == 0 && tid == 0) a.loss[col] = 0.f;
        return;
    }
    if (tid < THREADS) x.template copy<THREADS>(kept, X, end);
    if (MODE == BOTH) {
        if (tid == 0) {
            mail_init(&arrived);
            mail_init_done();
            mail_expect(&arrived, l.parts * W * 8);
        }
        // Every CTA has its barrier before anything is sent to it.  The warp that reads the student's logits of all entries, in
        // every part of the column, arrives when it has read them: dX may be X, and no part is written before the sums are here.
        if (part != 0 || tid < THREADS) cluster_arrive();
    }
    if (tid >= THREADS) {
        Held h;
        float xr[R], pr[R];
        hold(h, a.z, j0, j1);
        for (int i = lane; i < (l.per + 15) / 16; i += 32) reinterpret_cast<uint4 *>(marks)[i] = make_uint4(0, 0, 0, 0);
        if (lane == 0) twice = 0;
        __syncwarp();
        auto mark = [&](int u) {                                // a position of the part
            const int byte = u / N, bit = (byte & 3) * 8 + (u & (N - 1));
            return (atomicOr(reinterpret_cast<unsigned *>(marks) + (byte >> 2), 1u << bit) >> bit) & 1u;
        };
        auto mark_row = [&](int r) {
            const int u = r + x.shift - x.v0 * N;
            if (r >= 0 && r < a.nrows && u >= 0 && u < x.n * N && mark(u)) atomicOr(&twice, 1);
        };
        if (lane < x.head) mark(lane);
        if (lane < x.tail) mark(x.last * N + N - 1 - lane);
#pragma unroll
        for (int r = 0; r < R; r++) mark_row(h.row[r]);
        for (int j = j0 + 32 * R + lane; j < j1; j += 32) mark_row(a.z.ir[j]);
        // only CTA 0 needs the student's logits of all entries, for the loss
        Entries e = MODE == BOTH && part == 0 ? weigh_entries<T, true>(h, a.z, col, a.nrows, a.it, X + col * a.ldx, xr, pr)
                                              : weigh_entries<T, false>(h, a.z, col, a.nrows, a.it, nullptr, xr, pr);
        float ref = 0.f, qf = 1.f;
        if (MODE == GRAD) {
            ref = (float)((double)lse * a.t);
            qf = (float)exp(ref / (double)a.t - lse);           // what the rounding of the reference leaves
        }
        if (lane == 0) {
            slope = make_float2((float)e.P * w / a.t * qf, ref);
            if (e.P == 0.0) atomicOr(&twice, 2);
        }
        if (MODE == BOTH) {
            if (part == 0) cluster_arrive();
            cluster_wait();
        }
        __syncthreads();                                        // marks, slope; the part is in shared memory
        if (MODE == BOTH) {
            const SumExp s = receive<W>(&arrived, joined, l.parts * W, a.c);
            ref = s.ref();
            qf = (float)(1.0 / s.exact(a.c));
            if (part == 0 && lane == 0) write_loss<false>(a, col, s, e, w);
        }
        const bool plain = (twice & 1) == 0;
        if (plain) {
#pragma unroll
            for (int r = 0; r < R; r++) {
                const int u = h.row[r] + x.shift - x.v0 * N;
                if (h.row[r] >= 0 && h.row[r] < a.nrows && u >= 0 && u < x.n * N) {
                    const float q = exp2_fast((to_float(reinterpret_cast<const T *>(kept)[u]) - ref) * a.c) * qf;
                    out[u] = from_float<T>(e.P == 0.0 ? 0.f : w / a.t * ((float)e.P * q - pr[r]));
                }
            }
        }
        if (!plain || j1 - j0 > 32 * R) {
            const Slope g{a.t, a.c, w, ref, 0.f, a.it, (double)qf, e.zr, e.lt, e.P};
            const Column<T> whole(X + col * a.ldx, a.nrows);
            write_entries<T>(whole, dX + col * a.lddx - x.shift, a.z, plain ? j0 + 32 * R : j0, j1, x.v0, x.v0 + x.n, g, !plain, lane, 32);
        }
        return;
    }

    x.template arrive<THREADS>(kept, X, end, X + col * a.ldx, a.nrows);
    float f, ref;
    SumExp sum;                     // of the column
    if (MODE == BOTH) {
        SumExp s;
#pragma unroll 4
        for (int i = tid; i < x.n; i += THREADS) s.m = fmaxf(s.m, Pack<T>::max(kept[i]));
        const float k0 = __fmul_rn(s.ref(), a.c);
        if (moderate(k0)) {
            const unsigned long long cc = pair(a.c, a.c), mk = pair(-k0, -k0);
            unsigned long long acc = pair(0.f, 0.f);
#pragma unroll 2
            for (int i = tid; i < x.n; i += THREADS) {
                float v[N];
                Pack<T>::unpack(kept[i], v);
#pragma unroll
                for (int j = 0; j < N; j += 2) {
                    const float2 q = exp_pair_from(v[j], v[j + 1], cc, mk);
                    acc = add2(acc, pair(q.x, q.y));
                }
            }
            const float2 q = unpair(acc);
            s.s = q.x + q.y;
        } else {
            for (int i = tid; i < x.n; i += THREADS) s.s += sum_of_differences<T>(kept[i], s.ref(), a.c);
        }
        warp_join(s, a.c);
        cluster_wait();
        if (lane < l.parts) mail_send(&joined[part * W + (tid >> 5)], &arrived, lane, make_float2(s.m, s.s));
        __syncthreads();
        sum = receive<W>(&arrived, joined, l.parts * W, a.c);
        ref = sum.ref();
        f = slope.x / sum.s;
    } else {
        __syncthreads();
        f = slope.x;
        ref = slope.y;
    }
    const bool zero = (twice & 2) != 0, wide = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    auto store = [&](int i, const uint4 &y) {
        const unsigned skip = marks[i];
        if (wide && !skip) {
            store16(out + (long long)i * N, y);
        } else {
#pragma unroll
            for (int j = 0; j < N; j++)
                if (!((skip >> j) & 1u)) out[(long long)i * N + j] = reinterpret_cast<const T *>(&y)[j];
        }
    };
    // Exponents relative to the reference, for 16-bit gradients with the factor among them.  Its logarithm makes for a second
    // rounding that no sum makes up for, so the reference has to be small for that: with |k0| <= 256 and a factor within fp32's
    // range it is at most half a step below 512, 2^-16 of an exponent, and that of k0 in GRAD 2^-17, together 1.6e-5 of the value
    // (half a step of fp16 is 4.9e-4).
    constexpr bool FOLD = sizeof(T) == 2;
    const float k0 = __fmul_rn(ref, a.c), shift = FOLD ? k0 - log2f(fabsf(f)) : k0;
    const bool quick = FOLD ? fabsf(k0) <= 256.f && !(f < 0.f) : MODE == BOTH && moderate(k0);
    if (zero) {
        for (int i = tid; i < x.n; i += THREADS) store(i, make_uint4(0, 0, 0, 0));
    } else if (quick) {
        const unsigned long long cc = pair(a.c, a.c), mk = pair(-shift, -shift), ff = pair(f, f);
#pragma unroll 2
        for (int i = tid; i < x.n; i += THREADS) {
            float v[N];
            Pack<T>::unpack(kept[i], v);
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                float2 y = exp_pair_from(v[j], v[j + 1], cc, mk);
                if (!FOLD) y = unpair(mul2(pair(y.x, y.y), ff));
                v[j] = y.x;
                v[j + 1] = y.y;
            }
            store(i, Pack<T>::pack(v));
        }
    } else {
        // differences first: references that are not moderate, or not small, or negative weights in 16 bits, fp32 gradients
        // from a saved log-sum-exp.  They are relative to the reference itself, and so is the sum.
        const float f1 = MODE == BOTH ? slope.x / (float)sum.exact(a.c) : f;
        const unsigned long long mr = pair(-ref, -ref), cc = pair(a.c, a.c), ff = pair(f1, f1);
#pragma unroll 2
        for (int i = tid; i < x.n; i += THREADS) {
            float v[N];
            Pack<T>::unpack(kept[i], v);
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const float2 q = exp_pair(v[j], v[j + 1], mr, cc);
                const float2 y = unpair(mul2(pair(q.x, q.y), ff));
                v[j] = y.x;
                v[j + 1] = y.y;
            }
            store(i, Pack<T>::pack(v));
        }
    }
}

// ---------------------------------------------------------------- columns of any length
//
// One cluster per column, also for the loss alone; the column is read twice for the gradient.  The last warp of CTA 0
// looks after the entries, the others sum up their rows, and every warp leaves its sum with every CTA, or with CTA 0.
template <typename T, bool GRADIENT>
__global__ void __launch_bounds__(kStream + 32, GRADIENT ? 4 : 6)
distill_long_kernel(DistillArgs a, const T *X, T *dX) {
    constexpr int W = kStream / 32;
    __shared__ float2 joined[8 * W];               // (m, s) of every warp of the cluster
    __shared__ Entries entries;
    __shared__ unsigned marks[GRADIENT ? kMarkRows / 32 + 1 : 1];
    __shared__ int twice;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, rank = (int)cluster.block_rank(), size = (int)cluster.num_blocks();
    const long long col = blockIdx.x / size;
    const Column<T> x(X + col * a.ldx, a.nrows);
    int v0, v1;
    my_part(x.nvec, rank, size, &v0, &v1);
    T *out = GRADIENT ? dX + col * a.lddx - x.shift : nullptr;           // position u is out[u]
    const float w = GRADIENT && a.weights ? a.weights[col] : 1.f;
    const int j0 = max(a.z.jc[col], 0), j1 = min(a.z.jc[col + 1], a.z.nnz);
    if (GRADIENT && (w == 0.f || j1 <= j0)) {          // the whole cluster goes this way
        write_zeros<T, kStream + 32>(x, out, v0, v1);
        if (rank == 0 && tid == 0) a.loss[col] = 0.f;
        return;
    }
    cluster_arrive();                              // waited for before the first access to another CTA's memory
    if (tid >= kStream) {
        Entries e;
        if (rank == 0) {
            Held h;
            float xr[R], pr[R];
            hold(h, a.z, j0, j1);
            e = weigh_entries<T, true>(h, a.z, col, a.nrows, a.it, X + col * a.ldx, xr, pr);
        }
        cluster_wait();
        if (rank == 0 && lane < (GRADIENT ? size : 1)) *cluster.map_shared_rank(&entries, lane) = e;
    } else {
        SumExp s = sum_exp_slice<T, kStream, 4>(x, v0, v1, a.c);
        warp_join(s, a.c);
        cluster_wait();
        if (lane < (GRADIENT ? size : 1)) *cluster.map_shared_rank(&joined[rank * W + (tid >> 5)], lane) = make_float2(s.m, s.s);
    }
    cluster_arrive();
    if (!GRADIENT && (rank != 0 || tid >= 32)) return;
    cluster_wait();
    SumExp s;
    for (int i = lane; i < size * W; i += 32) join(s, joined[i].x, joined[i].y, a.c);
    warp_join(s, a.c);
    const Entries &e = entries;
    if (rank == 0 && tid == 0) write_loss<!GRADIENT>(a, col, s, e, w);
    if (GRADIENT) {
        if (e.P == 0.0) {
            write_zeros<T, kStream + 32>(x, out, v0, v1);
            return;
        }
        const double sum = s.exact(a.c);
        const Slope g{a.t, a.c, w, s.ref(), (float)e.P * w / (a.t * (float)sum), a.it, 1.0 / sum, e.zr, e.lt, e.P};
        write_gradient<T, kStream + 32>(x, out, a.z, j0, j1, v0, v1, g, marks, &twice);
    }
}

// ---------------------------------------------------------------- host side

// Parts, 131072 x 2048 bf16.  BOTH: of 64 KB, three CTAs on an SM, 195 us; 32 KB and five CTAs 225 us, 48 KB and four 212 us,
// 96 KB and two 221 us: with fewer parts fewer CTAs wait for one another.  GRAD: nobody waits, 32 KB and five CTAs.  A cluster has
// at most 8 parts, so columns above 512 KB get parts of up to 96 KB and those above 768 KB are read twice.  Where columns
// are few they are cut into more parts, to give every SM two CTAs.  Columns of up to 32 KB have CTAs of 96 threads
// (8000 x 8192 bf16, BOTH: 83 us, 122 us with 288 threads).
constexpr long long kGradBytes = 32768, kBothBytes = 65536, kMostPartBytes = 98304, kShortBytes = 32768;

template <typename T, int THREADS, Mode MODE>
cudaError_t launch_part(const DistillArgs &a, int ncols, int parts, long long nvec, const void *X, void *dX, cudaStream_t st) {
    const auto kernel = distill_part_kernel<T, THREADS, MODE>;
    const long long per = ((nvec + parts - 1) / parts + 7) & ~7LL;         // whole 128-byte lines
    const size_t smem = (size_t)per * 16 + (((size_t)per + 15) & ~size_t(15));
    const cudaError_t err = allow_shared(kernel, smem, (size_t)kMostPartBytes + kMostPartBytes / 16);
    if (err != cudaSuccess) return err;
    if ((long long)ncols * parts > 0x7fffffffLL) return cudaErrorInvalidValue;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = cluster_config(&attr, (unsigned)(ncols * parts), THREADS + 32, MODE == GRAD ? 1 : parts, smem, st);
    const Layout l = layout<T>(X, a.ldx, ncols, parts, per);
    return cudaLaunchKernelEx(&cfg, kernel, a, l, (const T *)X, (T *)dX);
}

template <typename T, bool GRADIENT>
cudaError_t launch_long(const DistillArgs &a, int ncols, int size, const void *X, void *dX, cudaStream_t st) {
    if ((long long)ncols * size > 0x7fffffffLL) return cudaErrorInvalidValue;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = cluster_config(&attr, (unsigned)(ncols * size), kStream + 32, size, 0, st);
    return cudaLaunchKernelEx(&cfg, distill_long_kernel<T, GRADIENT>, a, (const T *)X, (T *)dX);
}

template <typename T, Mode MODE>
cudaError_t launch_distill(const DistillArgs &a, int ncols, const void *X, void *dX, cudaStream_t st) {
    const long long nvec = most_vectors<T>(X, a.ldx, a.nrows, ncols), bytes = nvec * 16;
    const long long most = MODE == GRAD ? nvec : 8;
    const bool small = bytes <= kShortBytes;
    const long long part_bytes = MODE == GRAD ? kGradBytes : kBothBytes;
    long long parts = (bytes + part_bytes - 1) / part_bytes;
    const long long fill = (2 * kSMs + ncols - 1) / ncols, worth = (nvec + (small ? 63 : 255)) / (small ? 64 : 256);
    if (parts < fill) parts = fill < worth ? fill : worth;
    if (parts > most) parts = most;
    if (small) return launch_part<T, 64, MODE>(a, ncols, (int)parts, nvec, X, dX, st);
    if (bytes <= parts * kMostPartBytes) return launch_part<T, 256, MODE>(a, ncols, (int)parts, nvec, X, dX, st);
    return launch_long<T, true>(a, ncols, 8, X, dX, st);
}

// Without a gradient nothing has to stay on the chip, and a CTA is best kept on one column as long as there are
// enough of them, six per SM (131072 x 2048 bf16: 88 us in one part, 87 us in two, 95 us in three, 102 us in five).
template <typename T> cudaError_t launch_loss(const DistillArgs &a, int ncols, const void *X, cudaStream_t st) {
    const long long bytes = (long long)a.nrows * (long long)sizeof(T);
    const long long fill = 6 * kSMs / ncols, worth = (bytes + 8191) / 8192;
    long long parts = fill < worth ? fill : worth;
    if (parts < 1) parts = 1;
    if (parts > 8) parts = 8;
    return launch_long<T, false>(a, ncols, (int)parts, X, nullptr, st);
}

DistillArgs arguments(int nrows, long long ldx, long long lddx, float t, const Teacher &z, const float *weights, const float *lse_in,
                      float *loss, float *lse_out) {
    return DistillArgs{nrows, ldx, lddx, t, (float)(kLog2e / (double)t), 1.0 / (double)t, z, weights, lse_in, loss, lse_out};
}

int check(int nrows, int ncols, int nnz, const void *X, long long ldx, int dtype, float temperature, const int *Zir,
          const int *Zjc, const float *Zdata) {
    if (nrows < 1 || nrows > kMostRows || ncols < 0 || ncols > kMostRows || nnz < 0 || nnz > kMostEntries || !dtype_ok(dtype))
        return (int)cudaErrorInvalidValue;
    if (!temperature_ok(temperature)) return (int)cudaErrorInvalidValue;
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
    cudaError_t err = cudaSuccess;
#define CALL_LOSS(T) err = launch_loss<T>(a, ncols, X, as_stream(stream))
    DISPATCH_DTYPE(dtype, CALL_LOSS);
#undef CALL_LOSS
    if (err == cudaSuccess) g_launches += 1;
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
    cudaError_t err = cudaSuccess;
#define CALL_GRAD(T) err = launch_distill<T, GRAD>(a, ncols, X, dX, as_stream(stream))
    DISPATCH_DTYPE(dtype, CALL_GRAD);
#undef CALL_GRAD
    if (err == cudaSuccess) g_launches += 1;
    return (int)err;
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
    cudaError_t err = cudaSuccess;
#define CALL_BOTH(T) err = launch_distill<T, BOTH>(a, ncols, X, dX, as_stream(stream))
    DISPATCH_DTYPE(dtype, CALL_BOTH);
#undef CALL_BOTH
    if (err == cudaSuccess) g_launches += 1;
    return (int)err;
}
