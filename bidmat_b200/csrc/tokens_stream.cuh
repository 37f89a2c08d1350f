// Long columns read in 16-byte vectors, split over the CTAs of a cluster.
//
// A column of V elements starts at any element: it is treated as a row of 16-byte vectors from the aligned
// address at or below its first element.  Position u = row + shift, shift = elements between that address and
// the column; vector i holds the positions [i N, (i+1) N), N = 16 / sizeof(T).  Only the first and the last
// vector can be partial.  They are read one element at a time, or whole where their other elements belong to the matrix as
// well (between its first element and its last), and written one element at a time.
//
// A thread keeps (m, s): the largest x so far and the sum of 2^(x c - k) over its rows, c = log2(e)/t and k = m c as fp32
// rounds it.  That takes one instruction for two differences.  The terms are then relative to 2^k and not to 2^(m c), which
// exact() makes up for by the factor 2^(k - m c), the exponent taken in fp64, where m c has no rounding.  Up to |k| = 2^24 it
// is at most a half.  Beyond that (a mask of -1e9 that leaves nothing, logits over a temperature of 1e-7) the differences
// x - m come first instead, so that such a column neither overflows nor loses its distribution.
#pragma once
#include <cooperative_groups.h>

#include "tokens_common.cuh"

namespace bidmat {

constexpr double kLog2e = 1.4426950408889634074;

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The larger one, NaN if either is.
__device__ __forceinline__ float larger_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// N elements of one 16-byte vector as floats and back; lowest: all -infinity.  max leaves NaN out, max_nan is NaN if any element is.
template <typename T> struct Pack;
template <> struct Pack<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ uint4 lowest() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
    static __device__ __forceinline__ void unpack(const uint4 &r, float (&v)[N]) {
        v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[N]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
    static __device__ __forceinline__ float max(const uint4 &r) {
        return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
    }
    static __device__ __forceinline__ float max_nan(const uint4 &r) {
        return larger_nan(larger_nan(__uint_as_float(r.x), __uint_as_float(r.y)), larger_nan(__uint_as_float(r.z), __uint_as_float(r.w)));
    }
};
template <> struct Pack<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ uint4 lowest() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
    static __device__ __forceinline__ void unpack(const uint4 &r, float (&v)[N]) {
        const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[N]) {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const unsigned *>(&p);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float max(const uint4 &r) {
        const __nv_bfloat162 *p = reinterpret_cast<const __nv_bfloat162 *>(&r);
        const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
        return fmaxf(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ float max_nan(const uint4 &r) {
        const __nv_bfloat162 *p = reinterpret_cast<const __nv_bfloat162 *>(&r);
        const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3]));
        return larger_nan(__low2float(m), __high2float(m));
    }
};
template <> struct Pack<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ uint4 lowest() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
    static __device__ __forceinline__ void unpack(const uint4 &r, float (&v)[N]) {
        const __half2 *p = reinterpret_cast<const __half2 *>(&r);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(p[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[N]) {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __half2 p = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const unsigned *>(&p);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float max(const uint4 &r) {
        const __half2 *p = reinterpret_cast<const __half2 *>(&r);
        const __half2 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
        return fmaxf(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ float max_nan(const uint4 &r) {
        const __half2 *p = reinterpret_cast<const __half2 *>(&r);
        const __half2 m = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3]));
        return larger_nan(__low2float(m), __high2float(m));
    }
};

// Plain (coherent) loads: in place, the same kernel writes the column.
__device__ __forceinline__ void store16(void *p, const uint4 &r) {
    asm volatile("st.global.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w) : "memory");
}
__device__ __forceinline__ uint4 load16(const void *p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p)
                 : "memory");
    return r;
}

// One column as vectors.
template <typename T> struct Column {
    static constexpr int N = Pack<T>::N;
    const T *base;      // aligned address of vector 0
    int shift, rows, nvec;
    int full0, full1;   // the vectors that are the column's alone; before and behind at most one each is partial
    __device__ __forceinline__ Column(const T *x, int nrows) : rows(nrows) {
        shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
        base = x - shift;
        const long long end = (long long)shift + nrows;
        nvec = (int)((end + N - 1) / N);
        full0 = shift ? 1 : 0;
        full1 = (int)(end / N);
        if (full1 < full0) full1 = full0;       // everything inside the first vector
    }
    // position j of vector i belongs to the column
    __device__ __forceinline__ bool inside(int i, int j) const {
        const long long u = (long long)i * N + j;
        return u >= shift && u < (long long)shift + rows;
    }
    __device__ __forceinline__ uint4 load(int i) const { return load16(base + (long long)i * N); }
    // a partial vector, -infinity where it is not the column's
    __device__ __forceinline__ uint4 load_partial(int i) const {
        float v[N];
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = inside(i, j) ? to_float(base[(long long)i * N + j]) : -INFINITY;
        return Pack<T>::pack(v);
    }
    // vector i with -infinity where it is not the column's
    __device__ __forceinline__ uint4 only_inside(int i, const uint4 &r) const {
        float v[N];
        Pack<T>::unpack(r, v);
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = inside(i, j) ? v[j] : -INFINITY;
        return Pack<T>::pack(v);
    }
    // The partial vectors among [v0, v1): number 0 and 1, or -1.
    __device__ __forceinline__ int partial(int number, int v0, int v1) const {
        const int i = number == 0 ? 0 : nvec - 1;
        if (i >= full0 && i < full1) return -1;
        if (number == 1 && i == 0 && full0 > 0) return -1;          // one vector, counted as the first
        if (number == 0 && full0 == 0) return -1;                   // the first is full; the last is number 1
        return i >= v0 && i < v1 ? i : -1;
    }
};

// Asynchronous copies of 16 bytes to shared memory; their thread waits for all of its own.
__device__ __forceinline__ void copy16(void *smem, const void *p) {
    const unsigned dst = (unsigned)__cvta_generic_to_shared(smem);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(p) : "memory");
}
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// The two halves of a cluster-wide barrier.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait;" ::: "memory"); }

// A barrier in shared memory that counts arriving bytes, for values that other CTAs of the cluster send here.
__device__ __forceinline__ unsigned smem_address(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mail_init(unsigned long long *bar) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_address(bar)) : "memory");
}
__device__ __forceinline__ void mail_init_done() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void mail_expect(unsigned long long *bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_address(bar)), "r"(bytes) : "memory");
}
// Two floats to the same place of CTA `rank`, whose barrier counts them when they are there.
__device__ __forceinline__ void mail_send(float2 *to, unsigned long long *bar, int rank, float2 v) {
    unsigned dst, b;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(smem_address(to)), "r"(rank));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(smem_address(bar)), "r"(rank));
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1,%2}, [%3];" ::"r"(dst), "f"(v.x), "f"(v.y),
                 "r"(b)
                 : "memory");
}
// Waits for phase `parity`, with a limit of about a second; false when it ran out.
__device__ __forceinline__ bool mail_wait(unsigned long long *bar, unsigned parity) {
    const unsigned b = smem_address(bar);
    for (int i = 0; i < (1 << 20); i++) {
        unsigned ok;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, 1000;\nselp.u32 %0, 1, 0, p;\n}"
                     : "=r"(ok)
                     : "r"(b), "r"(parity)
                     : "memory");
        if (ok) return true;
    }
    return false;
}

// k of a maximum, and whether exponents are taken relative to it.
__device__ __forceinline__ bool moderate(float k) { return fabsf(k) <= 16777216.f; }
// The exponent that brings a sum relative to m1 up to m2 >= m1.  Where only one of them is moderate the other's sum is
// relative to the maximum itself.
__device__ __forceinline__ float rise(float m1, float m2, float c) {
    const float k1 = __fmul_rn(m1, c), k2 = __fmul_rn(m2, c);
    if (moderate(k1) && moderate(k2)) return k1 - k2;
    return (m1 - m2) * c - (moderate(k1) ? fmaf(m1, c, -k1) : 0.f) + (moderate(k2) ? fmaf(m2, c, -k2) : 0.f);
}

struct SumExp {
    float m = -INFINITY, s = 0.f;
    // what is subtracted: m, or 0 while everything was -infinity (the sum is then 0)
    __device__ __forceinline__ float ref() const { return m == -INFINITY ? 0.f : m; }
    __device__ __forceinline__ void raise(float top, float c) {
        s = s == 0.f ? 0.f : s * exp2_fast(rise(m, top, c));     // a NaN stays
        m = top;
    }
    // the sum of exp((x - m)/t)
    __device__ __forceinline__ double exact(float c) const {
        const float k = __fmul_rn(ref(), c);
        return moderate(k) ? s * exp2(k - (double)ref() * c) : (double)s;
    }
    // log sum exp((x - m)/t), or log sum exp(x/t) of a column of -infinity or NaN
    __device__ __forceinline__ double log_sum(float c) const {
        if (m == -INFINITY) return s == 0.f ? -INFINITY : NAN;
        return log(exact(c));
    }
};

// Two floats per instruction.
__device__ __forceinline__ unsigned long long pair(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1,%2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(unsigned long long r) {
    float2 v;
    asm("mov.b64 {%0,%1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
    return v;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// 2^(a c - k), 2^(b c - k)
__device__ __forceinline__ float2 exp_pair_from(float a, float b, unsigned long long cc, unsigned long long minus_k) {
    const float2 e = unpair(fma2(pair(a, b), cc, minus_k));
    return make_float2(exp2_fast(e.x), exp2_fast(e.y));
}
// 2^((a - ref) c), 2^((b - ref) c)
__device__ __forceinline__ float2 exp_pair(float a, float b, unsigned long long minus_ref, unsigned long long cc) {
    const float2 e = unpair(mul2(add2(pair(a, b), minus_ref), cc));
    return make_float2(exp2_fast(e.x), exp2_fast(e.y));
}

// The sum of 2^((x - ref) c) over a vector: for maxima that are not moderate.
template <typename T> __device__ __noinline__ float sum_of_differences(const uint4 r, float ref, float c) {
    constexpr int N = Pack<T>::N;
    float v[N], sum = 0.f;
    Pack<T>::unpack(r, v);
    for (int j = 0; j < N; j++) sum += exp2_fast((v[j] - ref) * c);
    return sum;
}

// top: the vectors' maximum.
template <typename T, int K> __device__ __forceinline__ void add_vectors(SumExp &a, const uint4 (&r)[K], float top, float c) {
    constexpr int N = Pack<T>::N;
    if (top > a.m) a.raise(top, c);
    const float ref = a.ref(), k0 = __fmul_rn(ref, c);
    if (moderate(k0)) {
        const unsigned long long cc = pair(c, c), mk = pair(-k0, -k0);
        unsigned long long acc[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
        for (int k = 0; k < K; k++) {
            float v[N];
            Pack<T>::unpack(r[k], v);
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const float2 e = exp_pair_from(v[j], v[j + 1], cc, mk);
                acc[(j >> 1) & 1] = add2(acc[(j >> 1) & 1], pair(e.x, e.y));
            }
        }
        const float2 e = unpair(add2(acc[0], acc[1]));
        a.s += e.x + e.y;
    } else {
#pragma unroll
        for (int k = 0; k < K; k++) a.s += sum_of_differences<T>(r[k], ref, c);
    }
}

__device__ __forceinline__ void join(SumExp &a, float m, float s, float c) {
    if (m > a.m) {
        a.raise(m, c);
        a.s += s;
    } else {
        a.s += s == 0.f ? 0.f : (m == a.m ? s : s * exp2_fast(rise(m, a.m, c)));
    }
}
// Largest of the warp's values (none of them NaN).
__device__ __forceinline__ float warp_top(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
// The same result in every lane: the sums are brought up to the largest maximum, then added.
__device__ __forceinline__ void warp_join(SumExp &a, float c) {
    const float m = warp_top(a.m);
    a.s = a.m == m || a.s == 0.f ? a.s : a.s * exp2_fast(rise(a.m, m, c));
    a.m = m;
    a.s = warp_sum(a.s);
}

// The part of nvec vectors that CTA `rank` of `size` has: whole 128-byte lines but for the last.
__device__ __forceinline__ void my_part(int nvec, int rank, int size, int *v0, int *v1) {
    const int per = (((nvec + size - 1) / size) + 7) & ~7;
    *v0 = (int)min((long long)nvec, (long long)rank * per);
    *v1 = (int)min((long long)nvec, (long long)(rank + 1) * per);
}

// The vectors [v0, v1) of a column, U loads in flight per thread.
template <typename T, int THREADS, int U>
__device__ __forceinline__ SumExp sum_exp_slice(const Column<T> &x, int v0, int v1, float c) {
    SumExp a;
    const int f1 = min(v1, x.full1);
    int i = max(v0, x.full0) + (int)threadIdx.x;
    for (; i < f1 - (U - 1) * THREADS; i += U * THREADS) {
        uint4 r[U];
#pragma unroll
        for (int u = 0; u < U; u++) r[u] = x.load(i + u * THREADS);
        float top = Pack<T>::max(r[0]);
#pragma unroll
        for (int u = 1; u < U; u++) top = fmaxf(top, Pack<T>::max(r[u]));
        add_vectors<T, U>(a, r, top, c);
    }
    for (; i < f1; i += THREADS) {
        const uint4 r[1] = {x.load(i)};
        add_vectors<T, 1>(a, r, Pack<T>::max(r[0]), c);
    }
    if (threadIdx.x < 2) {
        const int p = x.partial((int)threadIdx.x, v0, v1);
        if (p >= 0) {
            const uint4 r[1] = {x.load_partial(p)};
            add_vectors<T, 1>(a, r, Pack<T>::max(r[0]), c);
        }
    }
    return a;
}

// What the columns have in common: a column's vectors start `shift` elements before it.
struct Layout {
    int ncols, parts, per;          // parts of a column, vectors per part
    int shift0, ldmod;              // shift of column 0; how it moves from column to column
};
// A part of a column: vectors base[0 .. n), the first of them number v0 of the column.
template <typename T> struct Slice {
    static constexpr int N = Pack<T>::N;
    const T *base;
    int v0, n, shift;
    int head, tail;                 // positions of vector 0 and of vector `last` that are not the column's
    int last;                       // the column's last vector, relative to v0
    __device__ __forceinline__ Slice(const T *X, long long ld, int rows, const Layout &l, int col, int part) {
        shift = (l.shift0 + (col & (N - 1)) * l.ldmod) & (N - 1);
        v0 = part * l.per;
        const int nvec = (shift + rows + N - 1) / N;
        n = max(min(nvec - v0, l.per), 0);
        base = X + (col * ld + ((long long)v0 * N - shift));
        head = v0 == 0 ? shift : 0;
        last = nvec - 1 - v0;
        tail = last >= 0 && last < n ? nvec * N - shift - rows : 0;
    }
    // vector 0, the last vector lie in the matrix that goes from X to end
    __device__ __forceinline__ bool whole_head(const T *X) const { return base >= X; }
    __device__ __forceinline__ bool whole_tail(const T *end) const { return base + ((long long)last + 1) * N <= end; }
    // Starts the copies of a thread's vectors (tid, tid + THREADS, ...) to shared memory.  Partial vectors are copied
    // whole where their neighbours belong to the matrix as well.
    template <int THREADS> __device__ __forceinline__ void copy(uint4 *kept, const T *X, const T *end) const {
        const int tid = threadIdx.x, lo = head && !whole_head(X), hi = n - (tail && !whole_tail(end));
        const T *p = base + (long long)tid * N;
        uint4 *to = kept + tid;
        int i = tid;
        if (i < lo) { i += THREADS; p += THREADS * N; to += THREADS; }
#pragma unroll 4
        for (; i < hi; i += THREADS, p += THREADS * N, to += THREADS) copy16(to, p);
    }
    // Waits for them; partial vectors get -infinity where they are not the column's.
    template <int THREADS>
    __device__ __forceinline__ void arrive(uint4 *kept, const T *X, const T *end, const T *column, int rows) const {
        const int tid = threadIdx.x;
        copies_wait();
        if ((head && tid == 0) || (tail && tid == (last & (THREADS - 1)))) {
            const Column<T> whole(column, rows);
            const bool one = head && tail && last == 0;
            if (head && tid == 0)
                kept[0] = whole_head(X) && !(one && !whole_tail(end)) ? whole.only_inside(0, kept[0]) : whole.load_partial(0);
            if (tail && tid == (last & (THREADS - 1)) && !one)
                kept[last] = whole_tail(end) ? whole.only_inside(last + v0, kept[last]) : whole.load_partial(last + v0);
        }
    }
};

// ------------------------------------------------------------------ host side
// Vectors of the longest column, for the addresses that the columns really have.
template <typename T> long long most_vectors(const void *X, long long ldx, int nrows, int ncols) {
    constexpr int N = Pack<T>::N;
    const bool even = is16(X) && (ncols == 1 || ldx % N == 0);
    return ((long long)nrows + (even ? N - 1 : 2 * N - 2)) / N;
}
template <typename T> Layout layout(const void *X, long long ldx, int ncols, int parts, long long per) {
    return Layout{ncols, parts, (int)per, (int)((reinterpret_cast<uintptr_t>(X) & 15) / sizeof(T)), (int)(ldx & (Pack<T>::N - 1))};
}

// Clusters of `size` CTAs along x.
inline cudaLaunchConfig_t cluster_config(cudaLaunchAttribute *attr, unsigned grid, unsigned threads, int size, size_t smem,
                                         cudaStream_t st) {
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = (unsigned)size;
    attr->val.clusterDim.y = 1;
    attr->val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

}  // namespace bidmat
