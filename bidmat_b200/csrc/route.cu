// Routing of token columns to experts, and its gradient.
//
//   s = softmax or sigmoid of a column of scores; key = s + bias (without a bias: the score itself, which has
//   the same order); optionally only the experts of the best groups compete; the k best keys are picked, ties
//   to the lower row; weights are s of the picked rows, optionally divided by their sum, times a scale.
//
// The order of two experts whose keys are closer than fp32 can tell has to come out right, so keys that are
// sums with a bias are compared in 64 bits.
#include <cuda_runtime.h>

#include "tokens_stream.cuh"

using namespace bidmat;

namespace {

constexpr int kRouteWarps = 4;      // warps per CTA
constexpr int kListed = 4;          // rows per lane that a list has room for

struct RouteArgs {
    int nrows, ncols, k, score, ngroups, topgroups, grouptop, renorm;
    long long ldx;
    float scale;
    int gsize;                      // rows of a group
    int wide, wide_out;             // columns can be read, written 16 bytes at a time
    int stride, lists_at, doubles_at, warp_bytes;       // shared memory per warp: floats per column, bytes
    int *ir, *ic, *jc;
    float *data;
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

// The same for a column of which only the rows with an fp32 key of `cut` or more come into question: one row per lane.
// False if there are more than 32 of them, or fewer than k.
template <typename T>
__device__ __noinline__ bool route_few(const RouteArgs a, const T *__restrict__ x, const float *__restrict__ bias, long long c, float cut,
                                       const float *val, int *rows) {
    const int lane = threadIdx.x & 31;
    int n = 0;
    for (int e0 = 0; e0 < a.nrows; e0 += 32) {
        const bool in = e0 + lane < a.nrows && val[e0 + lane] >= cut;
        const unsigned vote = __ballot_sync(0xffffffffu, in);
        const int at = n + __popc(vote & ((1u << lane) - 1u));
        if (in && at < 32) rows[at] = e0 + lane;
        n += __popc(vote);
    }
    if (n > 32 || n < a.k) return false;
    double m = 0.0, sum = 1.0;
    if (a.score == BIDMAT_B200_SOFTMAX) {
        float top = -INFINITY;
        for (int e = lane; e < a.nrows; e += 32) top = fmaxf(top, to_float(x[e]));
        m = warp_max((double)top);
        sum = 0.0;
        for (int e = lane; e < a.nrows; e += 32) sum += exp((double)to_float(x[e]) - m);
        sum = warp_sum(sum);
    }
    __syncwarp();
    const int row = lane < n ? rows[lane] : -1;
    double s = 0.0, key = -INFINITY;
    if (row >= 0) {
        const double v = to_float(x[row]);
        s = a.score == BIDMAT_B200_SOFTMAX ? exp(v - m) / sum : 1.0 / (1.0 + exp(-v));
        key = s + bias[row];
    }
    int rank = 0;
    for (int j = 0; j < n; j++) {                   // rows ascend with the lanes
        const double other = __shfl_sync(0xffffffffu, key, j);
        rank += other > key || (other == key && j < lane);
    }
    const bool pick = row >= 0 && rank < a.k;
    if (a.renorm) {
        const double tot = warp_sum(pick ? s : 0.0);
        s = tot > 0.0 ? s / tot : 0.0;
    }
    if (pick) {
        const long long o = c * a.k + rank;
        a.ir[o] = row;
        a.data[o] = (float)(s * a.scale);
    }
    return true;
}

// One column by one warp with everything that is compared in 64 bits.  val: nrows floats, rank: nrows + ngroups
// doubles of shared memory.  groups: choose the groups as well; else val is -infinity where a row is out of the running.
template <typename T>
__device__ __noinline__ void route_exact(const RouteArgs a, const T *__restrict__ x, const float *__restrict__ bias, long long c,
                                         bool groups, float *val, double *rank) {
    const int lane = threadIdx.x & 31;
    double *gval = rank + a.nrows;                  // rank: s + bias, -inf where out of the running
    const double inf = INFINITY;
    double m = -inf, sum = 0.0;
    if (groups || a.score == BIDMAT_B200_SOFTMAX) {
        float top = -INFINITY;
        for (int e = lane; e < a.nrows; e += 32) {
            const float v = to_float(x[e]);
            top = fmaxf(top, v);
            rank[e] = v;
            if (groups) val[e] = v;
        }
        m = warp_max((double)top);
        if (m == -inf) m = 0.0;
        if (a.score == BIDMAT_B200_SOFTMAX) {
            for (int e = lane; e < a.nrows; e += 32) sum += exp(rank[e] - m);
            sum = warp_sum(sum);
        }
    }
    __syncwarp();
    auto score_of = [&](int e) -> double {
        const double v = to_float(x[e]);
        return a.score == BIDMAT_B200_SOFTMAX ? exp(v - m) / sum : 1.0 / (1.0 + exp(-v));
    };
    const bool by_score = groups || bias;           // else the scores' own order does
#pragma unroll 4
    for (int e = lane; e < a.nrows; e += 32) {
        double r = val[e];
        if (by_score && r > -inf) r = score_of(e) + (bias ? (double)bias[e] : 0.0);
        else if (by_score) r = -inf;
        if (r != r) r = -inf;
        rank[e] = r;
    }
    __syncwarp();
    if (groups) {
        const int gsize = a.gsize;
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
        unsigned drop = 0;
        int n = 0;
        for (int g = lane; g < a.ngroups; g += 32, n++) {
            int before = 0;
            for (int h = 0; h < a.ngroups; h++)
                before += gval[h] > gval[g] || (gval[h] == gval[g] && h < g);
            drop |= (before >= a.topgroups ? 1u : 0u) << n;
        }
        n = 0;
        for (int g = lane; g < a.ngroups; g += 32, n++)
            if ((drop >> n) & 1u)
                for (int e = g * gsize; e < (g + 1) * gsize; e++) rank[e] = -inf;
        __syncwarp();
    }
    double w = -inf;
    int pick = 0;
    // The k-th largest of the lanes' maxima is a bound that k rows reach; if no more than 32 do, each is ranked by counting.
    auto key_of_row = [&](int e) { return rank[e] == -inf || bias ? rank[e] : (double)val[e]; };
    double top = -inf;
    for (int e = lane; e < a.nrows; e += 32) top = fmax(top, key_of_row(e));
    int place = 0;
#pragma unroll 4
    for (int j = 0; j < 32; j++) {
        const double t = __shfl_sync(0xffffffffu, top, j);
        place += t > top || (t == top && j < lane);
    }
    const double reach = __shfl_sync(0xffffffffu, top, __ffs(__ballot_sync(0xffffffffu, place == a.k - 1)) - 1);
    int n = 0;
    for (int e = lane; e < a.nrows; e += 32) n += key_of_row(e) >= reach ? 1 : 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if (reach > -inf && n <= 32) {
        double key = -inf;
        int row = -1, have = 0;
        for (int e0 = 0; e0 < a.nrows; e0 += 32) {  // lane i gets the i-th of them, in the order of the rows
            const bool in = e0 + lane < a.nrows && key_of_row(e0 + lane) >= reach;
            unsigned vote = __ballot_sync(0xffffffffu, in);
            const int more = __popc(vote);
            if (lane >= have && lane < have + more) {
                for (int i = have; i < lane; i++) vote &= vote - 1;
                row = e0 + __ffs(vote) - 1;
                key = key_of_row(row);
            }
            have += more;
        }
        int r = 0;
        for (int j = 0; j < n; j++) {
            const double t = __shfl_sync(0xffffffffu, key, j);
            r += t > key || (t == key && j < lane);
        }
        for (int j = 0; j < n; j++) {               // rank i goes to lane i
            const int at = __shfl_sync(0xffffffffu, r, j), from = __shfl_sync(0xffffffffu, row, j);
            if (at == lane) {
                pick = from;
                w = 0.0;                            // a pick
            }
        }
    } else {
        // k rounds: the best one that is left; then, in the order of the rows, the others with weight zero.
        // NaN marks a row that is taken.
        for (int i = 0; i < a.k; i++) {
            double key = -inf;
            int row = -1;
            for (int e = lane; e < a.nrows; e += 32) {
                const double r = rank[e];
                if (r != r) continue;
                const double v = r == -inf || bias ? r : (double)val[e];
                if (row < 0 || v > key) { key = v; row = e; }
            }
            warp_best(key, row);
            if ((row & 31) == lane) rank[row] = NAN;
            if (lane == i) {
                pick = row;
                w = key;
            }
            __syncwarp();
        }
    }
    w = lane < a.k && w > -inf ? score_of(pick) : 0.0;
    if (a.renorm) {
        const double tot = warp_sum(w);
        w = tot > 0.0 ? w / tot : 0.0;
    }
    if (lane < a.k) {
        const long long o = c * a.k + lane;
        a.ir[o] = pick;
        a.data[o] = (float)(w * a.scale);
    }
}

// An entry: order key above, complement of the row below.
typedef unsigned long long Entry;
__device__ __forceinline__ Entry entry_of(float key, int row) { return ((Entry)order_key(key) << 32) | (0xffffffffu - (unsigned)row); }
__device__ __forceinline__ int row_of(Entry e) { return (int)(0xffffffffu - (unsigned)e); }
__device__ __forceinline__ float key_of(Entry e) { return order_value((unsigned)(e >> 32)); }

// G lanes have a column, each every G-th of its rows.  The (k+1)-th largest of the lanes' maxima is a bound that k + 1
// rows reach; few more do, so the rows that reach it are listed and each is ranked by counting the ones before it.
// (256 x 4096 fp32 with bias and groups: 9.8 us, 36 us with sorted lists in the lanes' registers that are joined by exchanges;
// 160 x 65537 bf16 with groups: 36 and 47 us.)
//
// Where the order is that of scores plus bias, or of groups by their scores, it is found in fp32 first.  A sigmoid
// s = 1/(1 + e) is then off by at most s (1 - s) (2^-22 + |x| 2^-23) + 1.5 s 2^-23 < 2^-22 (the exponential, the sum and the
// reciprocal), a softmax by at most 2^-20 of the column's largest (the sum's error besides).  Two sums of two of them that
// differ by more than four times that, or sums with a bias that differ by more than twice that, and by more than
// 2^-22 of their size for the roundings of the sums, are in the right order; so are keys made of the same two numbers.  The size
// of a group's sum is that of its two parts, which may have opposite signs with a bias.  A column with two neighbours closer than
// that, one in some thousand, goes to route_few or route_exact.
constexpr float kNearSigmoid = 9.5367432e-07f, kNearSoftmax = 3.8146973e-06f, kNearPart = 2.3841858e-07f;

__device__ __forceinline__ bool near(float a, float b, float within) {
    return !(fabsf(a - b) > within + kNearPart * fmaxf(fabsf(a), fabsf(b)));
}

template <typename T> __device__ __forceinline__ bool same_numbers(const T *x, const float *bias, int r, int t) {
    return to_float(x[r]) == to_float(x[t]) && bias[r] == bias[t];
}

// Whether behind the k picks is a row that may come before the last one: in the list of n, whose keys descend, the one with the
// largest key that does not reach the bound, or one of those that equal `bound` (if not -infinity) and found no room in the list.
// A lane looks at every G-th.
template <typename T, int G>
__device__ __noinline__ bool another_near(const Entry *sorted, int n, int k, const T *x, const float *bias, float within, float rejected,
                                          float bound, const float *val, int nrows) {
    const int sub = threadIdx.x & (G - 1);
    const Entry last = sorted[k - 1];
    for (int j = k + sub; j < n; j += G) {
        const Entry q = sorted[j];
        if (!near(key_of(last), key_of(q), within)) break;
        if (!same_numbers(x, bias, row_of(last), row_of(q))) return true;
    }
    if (rejected > -INFINITY && near(key_of(last), rejected, within)) return true;
    if (bound > -INFINITY && near(key_of(last), bound, within))
        for (int e = sub; e < nrows; e += G)
            if (val[e] == bound && !same_numbers(x, bias, row_of(last), e)) return true;
    return false;
}

template <typename T, int G, bool BIAS>
__global__ void __launch_bounds__(kRouteWarps * 32, 8)
route_kernel(RouteArgs a, const T *__restrict__ X, const float *__restrict__ bias) {
    constexpr int C = 32 / G;                       // columns per warp
    constexpr int L = kListed * G, P = kListed;     // rows that can be listed, per column and per lane
    extern __shared__ double route_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane & (G - 1), which = lane / G;
    const unsigned mine = G == 32 ? 0xffffffffu : ((1u << G) - 1u) << (which * G);
    const long long c = ((long long)blockIdx.x * kRouteWarps + warp) * C + which;
    // shared memory of the warp: the keys in fp32 (scores, or scores plus bias) and the groups of each column; one column in fp64
    char *const base = reinterpret_cast<char *>(route_smem) + (size_t)warp * a.warp_bytes;
    float *val = reinterpret_cast<float *>(base) + which * a.stride;
    float *gval = val + ((a.nrows + 3) & ~3);
    Entry *list = reinterpret_cast<Entry *>(base + a.lists_at) + which * 2 * L, *sorted = list + L;
    const bool on = c < a.ncols;
    const T *x = X + (on ? c : 0) * a.ldx;
    const bool softmax = a.score == BIDMAT_B200_SOFTMAX;
    // scores of all rows are needed for a bias, for groups that are not ranked by their best score alone, and for softmax
    // weights as they are
    const bool group_scores = a.ngroups > 1 && a.grouptop == 2;
    const bool total = softmax && (BIAS || group_scores || !a.renorm);

    // A lane reads 16 bytes at a time where it can.  What each of its vectors has largest falls to one of two groups.
    constexpr int N = Pack<T>::N;
    const int quads = (a.nrows + 3) / 4;            // of val, which is padded with -infinity
    bool bad = false;
    float m = -INFINITY, sum = 0.f, top0 = -INFINITY, top1 = -INFINITY;
    if (a.wide) {
        for (int i = sub; i * N < a.nrows; i += 2 * G) {
            const uint4 none = Pack<T>::lowest();
            const bool second = (i + G) * N < a.nrows;
            const uint4 r0 = on ? *reinterpret_cast<const uint4 *>(x + i * N) : none;
            const uint4 r1 = on && second ? *reinterpret_cast<const uint4 *>(x + (i + G) * N) : none;
            top0 = larger_nan(top0, Pack<T>::max_nan(r0));
            top1 = larger_nan(top1, Pack<T>::max_nan(r1));
            float v[N];
            Pack<T>::unpack(r0, v);
#pragma unroll
            for (int j = 0; j < N; j += 4) *reinterpret_cast<float4 *>(val + i * N + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            if (second) {
                Pack<T>::unpack(r1, v);
#pragma unroll
                for (int j = 0; j < N; j += 4)
                    *reinterpret_cast<float4 *>(val + (i + G) * N + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            }
        }
    } else {
#pragma unroll 4
        for (int e = sub; e < quads * 4; e += G) {
            const float v = on && e < a.nrows ? to_float(x[e]) : -INFINITY;
            if ((e / G) & 1) top1 = larger_nan(top1, v);
            else top0 = larger_nan(top0, v);
            val[e] = v;
        }
    }
    m = larger_nan(top0, top1);
    bad = !(m < INFINITY);
    __syncwarp();
    bad = (__ballot_sync(0xffffffffu, bad) & mine) != 0;
    if (total) {
#pragma unroll
        for (int o = G / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (m == -INFINITY || bad) m = 0.f;
        for (int q = sub; q < quads; q += G) {
            const float4 v = reinterpret_cast<const float4 *>(val)[q];
            sum += (exp2_fast((v.x - m) * (float)kLog2e) + exp2_fast((v.y - m) * (float)kLog2e)) +
                   (exp2_fast((v.z - m) * (float)kLog2e) + exp2_fast((v.w - m) * (float)kLog2e));
        }
#pragma unroll
        for (int o = G / 2; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    const float inverse = total ? 1.f / sum : 0.f;
    const float within = softmax ? kNearSoftmax * fminf(inverse, 1.f) : kNearSigmoid;
    // for comparisons
    auto quick_score = [&](float v) {
        return softmax ? exp2_fast((v - m) * (float)kLog2e) * inverse : __fdividef(1.f, 1.f + exp2_fast(-v * (float)kLog2e));
    };
    // for weights
    auto score_of = [&](float v) { return softmax ? expf(v - m) / sum : 1.f / (1.f + expf(-v)); };
    if (BIAS) {
#pragma unroll 4
        for (int e = sub; e < a.nrows; e += G) {
            const float v = val[e];
            const float r = quick_score(v) + bias[e];
            val[e] = v > -INFINITY && r > -INFINITY ? r : -INFINITY;
        }
    }
    __syncwarp();
    bool again = false, groups_again = false;       // two neighbours too close
    if (a.ngroups > 1) {
        // a lane takes whole groups, four rows at once where that divides them; groups that would meet in one bank are begun at
        // another place in every lane
        float *goff = gval + a.ngroups;             // BIAS: what the roundings of a group's sum may come to
        const int size = a.gsize, four = (size & 3) ? 0 : size / 4;
        auto first_of = [&](int g) { return (size & 31) ? 0 : g % four; };
        for (int g = sub; g < a.ngroups; g += G) {
            float b1 = -INFINITY, b2 = -INFINITY;
            auto add = [&](float v) {
                if (!BIAS && group_scores && v > -INFINITY) v = quick_score(v);
                b2 = fmaxf(b2, fminf(b1, v));
                b1 = fmaxf(b1, v);
            };
            if (four) {
                const float4 *member = reinterpret_cast<const float4 *>(val) + g * four;
                const int turn = first_of(g);
                for (int i = turn, left = four; left > 0; left--) {
                    const float4 v = member[i];
                    add(v.x);
                    add(v.y);
                    add(v.z);
                    add(v.w);
                    if (++i == four) i = 0;
                }
            } else {
                for (int i = 0; i < size; i++) add(val[g * size + i]);
            }
            const bool both = a.grouptop == 2 && b2 > -INFINITY;
            gval[g] = both ? fmaxf(b1 + b2, -3.4028235e38f) : b1;       // not that of a group of nothing
            if (BIAS) goff[g] = kNearPart * fabsf(b1) + (both ? kNearPart * fabsf(b2) : 0.f);
        }
        __syncwarp();
        // at least, at most: of the groups kept, of those dropped
        float worst = INFINITY, best = -INFINITY;
        unsigned drop = 0;                          // of this lane's groups
        int n = 0;
        for (int g = sub; g < a.ngroups; g += G, n++) {
            const float v = gval[g];
            int before = 0;
            for (int h = 0; h < a.ngroups; h++) {
                const float u = gval[h];
                before += u > v || (u == v && h < g);
            }
            const float off = BIAS ? goff[g] : 0.f;
            if (before < a.topgroups) worst = fminf(worst, v - off);
            else best = fmaxf(best, v > -INFINITY ? v + off : v), drop |= 1u << (n & 31);
        }
        __syncwarp();
#pragma unroll
        for (int o = G / 2; o; o >>= 1) {
            worst = fminf(worst, __shfl_xor_sync(0xffffffffu, worst, o));
            best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
        }
        groups_again = (BIAS || group_scores) && best > -INFINITY && (BIAS ? !(worst - best > within) : near(worst, best, within));
        n = 0;
        for (int g = sub; g < a.ngroups; g += G, n++) {
            if (!((drop >> (n & 31)) & 1u)) continue;
            if (four) {
                float4 *member = reinterpret_cast<float4 *>(val) + g * four;
                const int turn = first_of(g);
                for (int i = turn, left = four; left > 0; left--) {
                    member[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                    if (++i == four) i = 0;
                }
            } else {
                for (int i = 0; i < size; i++) val[g * size + i] = -INFINITY;
            }
        }
        __syncwarp();
    }
    // the bound
    const int before_me = (1 << sub) - 1;
    // ... of two maxima per lane, or of one where that is plenty: the bound stays well inside them, so that few more reach it
    const bool two = G < 32 || a.k > 12;
    // Other keys than the scores, or not all of them, or so few vectors that k + 1 of their maxima, of whole vectors each, are no
    // bound to speak of: then the lists overflow and every column goes to route_exact.  (32768 columns, bf16, this and the vectors'
    // maxima: 64 rows, k = 8: 11.7 and 63.5 us; 96 rows, k = 8: 12.7 and 15.6 us; 128 rows, k = 8, not taken: 13.0 and 12.4 us.)
    if (BIAS || a.ngroups > 1 || (a.wide && 2 * a.nrows < 3 * N * (a.k + 1))) {
        // every 2 G-th row, so that a group's rows fall to as many maxima as there are
        top0 = top1 = -INFINITY;
        int e = sub;
#pragma unroll 4
        for (; e + G < 4 * quads; e += 2 * G) {
            top0 = fmaxf(top0, val[e]);
            top1 = fmaxf(top1, val[e + G]);
        }
        if (e < 4 * quads) top0 = fmaxf(top0, val[e]);
    }
    float bound = -INFINITY;                        // so few rows that all of them can be listed
    if (a.nrows > 2 * G) {
        if (!two) top0 = fmaxf(top0, top1);
        int place0 = two && top1 > top0, place1 = top0 >= top1;
#pragma unroll
        for (int o = 1; o < G; o++) {
            const int from = (sub + o) & (G - 1);
            const float t0 = __shfl_sync(0xffffffffu, top0, from, G);
            place0 += from < sub ? t0 >= top0 : t0 > top0;
            if (two) {
                const float t1 = __shfl_sync(0xffffffffu, top1, from, G);
                place0 += from < sub ? t1 >= top0 : t1 > top0;
                place1 += from < sub ? (t0 >= top1) + (t1 >= top1) : (t0 > top1) + (t1 > top1);
            }
        }
        const int kth = min(a.k, two ? 2 * G - 1 : G - 1);
        const unsigned who0 = __ballot_sync(0xffffffffu, place0 == kth) & mine, who1 = __ballot_sync(0xffffffffu, two && place1 == kth) & mine;
        const float bound0 = __shfl_sync(0xffffffffu, top0, who0 ? __ffs(who0) - 1 : 0), bound1 = __shfl_sync(0xffffffffu, top1, who1 ? __ffs(who1) - 1 : 0);
        bound = who0 ? bound0 : bound1;
    }
    // the rows that reach it
    // bit 4 i + j of the mask: row 4 (sub + G i) + j
    unsigned mask = 0;
    float rejected = -INFINITY;
    const float reach = fmaxf(bound, -3.4028235e38f);       // -infinity is never listed
    {
        int bit = 0;
#pragma unroll 2
        for (int q = sub; q < quads; q += G, bit += 4) {
            const float4 v = reinterpret_cast<const float4 *>(val)[q];
            unsigned in = 0;
            if (v.x >= reach) in |= 1u;
            if (v.y >= reach) in |= 2u;
            if (v.z >= reach) in |= 4u;
            if (v.w >= reach) in |= 8u;
            mask |= in << bit;
            if (BIAS) {
                if (!(in & 1u)) rejected = fmaxf(rejected, v.x);
                if (!(in & 2u)) rejected = fmaxf(rejected, v.y);
                if (!(in & 4u)) rejected = fmaxf(rejected, v.z);
                if (!(in & 8u)) rejected = fmaxf(rejected, v.w);
            }
        }
    }
    auto masked_row = [&](int bit) { return 4 * (sub + G * (bit >> 2)) + (bit & 3); };
    int at = __popc(mask);
    const int own = at;
#pragma unroll
    for (int o = 1; o < G; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, at, o, G);
        if (sub >= o) at += v;
    }
    int n = __shfl_sync(0xffffffffu, at, G - 1, G);
    at -= own;
    bool left_out = false;                          // rows whose keys equal the bound in fp32
    if (__any_sync(0xffffffffu, n > L)) {
        // more than the list holds: those above the bound, and of those that equal it the lowest rows
        const bool over = n > L;
        unsigned above = 0;
        for (int i = 0; masked_row(i) < 4 * quads; i++) above |= (val[masked_row(i)] > bound ? 1u : 0u) << i;
        int n1 = __popc(above);
        const int own1 = n1;
        for (int o = 1; o < G; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, n1, o, G);
            if (sub >= o) n1 += v;
        }
        const int first = n1 - own1;
        n1 = __shfl_sync(0xffffffffu, n1, G - 1, G);
        if (over && n1 + a.k > L) again = true;     // one lane has too many of the largest
        int taken = n1;
        for (int e = sub; e - sub < a.nrows; e += G) {
            const bool tie = over && !again && e < a.nrows && val[e] == bound;
            const unsigned vote = (__ballot_sync(0xffffffffu, tie) & mine) >> (which * G);
            const int to = taken + __popc(vote & before_me);
            if (tie && to < L) list[to] = entry_of(bound, e);
            taken += __popc(vote);
        }
        left_out = taken > L;
        if (over) {
            mask = again ? 0 : above;
            at = first;
            n = again ? 0 : min(taken, L);
        }
    }
    for (; mask; mask &= mask - 1) {
        const int e = masked_row(__ffs(mask) - 1);
        list[at++] = entry_of(val[e], e);
    }
    __syncwarp();
    // ranks
    {
        Entry en[P];
        int rank[P];
#pragma unroll
        for (int p = 0; p < P; p++) {
            en[p] = sub + p * G < n ? list[sub + p * G] : 0;
            rank[p] = 0;
        }
        if (__all_sync(0xffffffffu, n <= 2 * G)) {
#pragma unroll 2
            for (int j = 0; j < n; j++) {
                const Entry other = list[j];
                rank[0] += other > en[0];
                rank[1] += other > en[1];
            }
        } else {
            for (int j = 0; j < n; j++) {
                const Entry other = list[j];
#pragma unroll
                for (int p = 0; p < P; p++) rank[p] += other > en[p];
            }
        }
#pragma unroll
        for (int p = 0; p < P; p++)
            if (sub + p * G < n) sorted[rank[p]] = en[p];
    }
    __syncwarp();
    const bool none = n == 0 && !again;
    if (!none && n < a.k) again = true;             // fewer than k rows: the others are found there
    const Entry pick = sub < min(a.k, n) ? sorted[sub] : 0;
    if (BIAS) {
        // Neighbours among the picks, and the last one with all that may come before it: behind rows that are made of the same
        // numbers as the last pick there may be others.
#pragma unroll
        for (int o = G / 2; o; o >>= 1) rejected = fmaxf(rejected, __shfl_xor_sync(0xffffffffu, rejected, o));
        bool further = left_out;
        if (pick != 0) {
            if (sub + 1 < n) {
                const Entry q = sorted[sub + 1];
                if (near(key_of(pick), key_of(q), within)) {
                    if (!same_numbers(x, bias, row_of(pick), row_of(q))) again = true;
                    else if (sub + 1 == a.k) further = true;
                }
            } else if (rejected > -INFINITY && near(key_of(pick), rejected, within)) {
                again = true;
            }
        }
        if (__any_sync(0xffffffffu, further) && n >= a.k)       // few columns
            again |= another_near<T, G>(sorted, n, a.k, x, bias, within, rejected, left_out ? bound : -INFINITY, val, a.nrows);
    }
    const unsigned redo_groups = __ballot_sync(0xffffffffu, groups_again && !bad && on);
    const bool relative = softmax && !total;        // only the picks matter: relative to the largest of them
    const int row = none || bad || pick == 0 ? sub : row_of(pick);
    float w = 0.f;
    if (pick != 0 && !bad) {
        const float v = BIAS ? to_float(x[row]) : val[row];
        w = relative ? expf(v - val[row_of(sorted[0])]) : score_of(v);
    }
    float wsum = w;
    if (a.renorm) {
#pragma unroll
        for (int o = G / 2; o; o >>= 1) wsum += __shfl_xor_sync(0xffffffffu, wsum, o);
        // Scores that leave the range of fp32, or come near enough to its end to lose bits that the sum of the picks, small
        // itself, would bring back into the weights.
        if ((!(wsum > 1e-30f) || (pick != 0 && w < 1e-31f && wsum < 1e-7f)) && !none && !bad) again = true;
    } else if (!softmax && pick != 0 && !bad && w < 1e-30f) {
        again = true;
    }
    if (on && sub < a.k) {
        const long long o = c * a.k + sub;
        a.ir[o] = row;
        a.ic[o] = (int)c;
        a.data[o] = bad ? NAN : (a.renorm ? (wsum > 0.f ? w / wsum : 0.f) : w) * a.scale;
    }
    if (on && sub == 0) {
        a.jc[c] = (int)(c * a.k);
        if (c == a.ncols - 1) a.jc[a.ncols] = (int)((c + 1) * a.k);
    }
    // columns that fp32 cannot order
    const unsigned redo = __ballot_sync(0xffffffffu, again && !bad && on) | redo_groups;
    for (int w2 = 0; w2 < C; w2++) {
        const unsigned of = G == 32 ? 0xffffffffu : ((1u << G) - 1u) << (w2 * G);
        if (!(redo & of)) continue;
        const float last = __shfl_sync(0xffffffffu, pick != 0 ? key_of(pick) : -INFINITY, w2 * G + a.k - 1);
        // no row that is out of the running, also where the last pick's key is the lowest number or so
        const float cut = fmaxf(last - 2.f * (__shfl_sync(0xffffffffu, within, w2 * G) + kNearPart * fabsf(last)), -3.4028235e38f);
        const long long col = ((long long)blockIdx.x * kRouteWarps + warp) * C + w2;
        const T *xc = X + col * a.ldx;
        float *v = reinterpret_cast<float *>(base) + w2 * a.stride;
        double *rank = reinterpret_cast<double *>(base + a.doubles_at);
        const bool groups = (redo_groups & of) != 0;
        __syncwarp();
        if (groups || !BIAS || !(last > -INFINITY) ||
            !route_few<T>(a, xc, bias, col, cut, v, reinterpret_cast<int *>(rank)))
            route_exact<T>(a, xc, bias, col, groups, v, rank);
        __syncwarp();
    }
}

// The gradient of the weights goes back to the scores (w, g: weight and gradient of an entry, D = sum of w g):
//   softmax, renormalised: w (g - D/scale)            sigmoid, renormalised: w (1 - s) (g - D/scale)
//   softmax:  w g at the entries, - p D everywhere    sigmoid:               w (1 - s) g
//
// G lanes have a column.  It is put together in shared memory in fp32: what every row gets, then the entries, one lane at a
// time, so that a row that comes twice gets its terms in their order.  Bound by memory for many columns (160 x 65537 bf16,
// softmax: 17.6 us for 7.2 us of copying), by latency for few (256 x 4096 fp32: 3.5 us).
template <typename T, int G>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_grad_kernel(RouteArgs a, int nnz, const T *X, const int *__restrict__ Sir, const int *__restrict__ Sjc,
                  const float *__restrict__ Sdata, const float *__restrict__ dS, T *dX, long long lddx) {
    constexpr int C = 32 / G, N = Pack<T>::N, V = 32 / N;       // columns per warp, vectors per lane: 32 G rows at most
    extern __shared__ float4 route_grad_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane & (G - 1), which = lane / G;
    const long long c = ((long long)blockIdx.x * kRouteWarps + warp) * C + which;
    const bool on = c < a.ncols;
    float *col = reinterpret_cast<float *>(route_grad_smem) + (size_t)(warp * C + which) * a.stride;
    const T *x = X + (on ? c : 0) * a.ldx;
    const int j0 = on ? max(Sjc[c], 0) : 0, j1 = on ? min(Sjc[c + 1], nnz) : 0;
    const bool everywhere = a.score == BIDMAT_B200_SOFTMAX && !a.renorm;
    auto over_lanes = [&](float v) {
#pragma unroll
        for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    uint4 r[V];
    if (everywhere) {
#pragma unroll
        for (int k = 0; k < V; k++) {
            const int i = sub + k * G;
            r[k] = Pack<T>::lowest();
            if (on && i * N < a.nrows) {
                if (a.wide) {
                    r[k] = *reinterpret_cast<const uint4 *>(x + i * N);
                } else {
                    float v[N];
#pragma unroll
                    for (int j = 0; j < N; j++) v[j] = i * N + j < a.nrows ? to_float(x[i * N + j]) : -INFINITY;
                    r[k] = Pack<T>::pack(v);
                }
            }
        }
    }
    float d = 0.f;
    for (int j = j0 + sub; j < j1; j += G) d = fmaf(Sdata[j], dS[j], d);
    d = over_lanes(d);
    if (everywhere) {
        float m = -INFINITY, sum = 0.f;
#pragma unroll
        for (int k = 0; k < V; k++) m = fmaxf(m, Pack<T>::max(r[k]));
#pragma unroll
        for (int o = G / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (m == -INFINITY) m = 0.f;
        const unsigned long long mr = pair(-m, -m), cc = pair((float)kLog2e, (float)kLog2e);
        float e[V * N];
#pragma unroll
        for (int k = 0; k < V; k++) {
            float v[N];
            Pack<T>::unpack(r[k], v);
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const float2 q = exp_pair(v[j], v[j + 1], mr, cc);
                e[k * N + j] = q.x;
                e[k * N + j + 1] = q.y;
                sum += q.x + q.y;
            }
        }
        sum = over_lanes(sum);
        const float f = sum > 0.f ? -d / sum : (sum == 0.f ? 0.f : NAN);
#pragma unroll
        for (int k = 0; k < V; k++)
            if ((sub + k * G) * N < a.nrows)
#pragma unroll
                for (int j = 0; j < N; j += 4)
                    *reinterpret_cast<float4 *>(col + (sub + k * G) * N + j) =
                        make_float4(e[k * N + j] * f, e[k * N + j + 1] * f, e[k * N + j + 2] * f, e[k * N + j + 3] * f);
    } else {
        for (int i = sub; i * 4 < a.nrows; i += G) *reinterpret_cast<float4 *>(col + i * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncwarp();
    const float inverse = 1.f / a.scale;            // infinite for a subnormal scale
    const float back = a.renorm ? (fabsf(inverse) < INFINITY ? d * inverse : d / a.scale) : 0.f;
    for (int j = j0; __any_sync(0xffffffffu, j < j1); j += G) {
        const bool have = j + sub < j1;
        const int row = have ? Sir[j + sub] : -1;
        const bool in = row >= 0 && row < a.nrows;
        float v = 0.f;
        if (in) {
            v = Sdata[j + sub] * (dS[j + sub] - back);
            if (a.score == BIDMAT_B200_SIGMOID) v *= 1.f / (1.f + expf(to_float(x[row])));
        }
        const int most = __reduce_max_sync(0xffffffffu, min(j1 - j, G));
        for (int l = 0; l < most; l++) {
            if (l == sub && in) col[row] += v;
            __syncwarp();
        }
    }
    if (!on) return;
    T *out = dX + c * lddx;
    for (int i = sub; i * N < a.nrows; i += G) {
        float v[N];
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const float4 q = *reinterpret_cast<const float4 *>(col + i * N + j);
            v[j] = q.x;
            v[j + 1] = q.y;
            v[j + 2] = q.z;
            v[j + 3] = q.w;
        }
        if (a.wide_out) {
            store16(out + i * N, Pack<T>::pack(v));
        } else {
#pragma unroll
            for (int j = 0; j < N; j++)
                if (i * N + j < a.nrows) out[i * N + j] = from_float<T>(v[j]);
        }
    }
}

template <typename T, int G, bool BIAS>
cudaError_t launch_route_as(RouteArgs a, const void *X, const float *bias, cudaStream_t st) {
    constexpr int C = 32 / G;
    const auto kernel = route_kernel<T, G, BIAS>;
    a.wide = is16(X) && a.nrows % Pack<T>::N == 0 && (a.ldx % Pack<T>::N == 0 || a.ncols == 1);
    auto place = [](RouteArgs &b) {
        b.stride = (((b.nrows + 3) / 4 * 4 + b.ngroups * (BIAS ? 2 : 1) + 31) & ~31) + 8;       // columns 8 banks apart
        b.lists_at = C * b.stride * (int)sizeof(float);
        b.doubles_at = b.lists_at + C * 2 * kListed * G * (int)sizeof(Entry);
        b.warp_bytes = (b.doubles_at + (b.nrows + b.ngroups) * (int)sizeof(double) + 15) & ~15;
        return (size_t)kRouteWarps * b.warp_bytes;
    };
    RouteArgs most = a;
    most.nrows = most.ngroups = 32 * G;             // launch_route
    const size_t smem = place(a);
    const cudaError_t err = allow_shared(kernel, smem, place(most));
    if (err != cudaSuccess) return err;
    const long long per = (long long)kRouteWarps * C;
    kernel<<<(unsigned)((a.ncols + per - 1) / per), kRouteWarps * 32, smem, st>>>(a, (const T *)X, bias);
    return cudaGetLastError();
}

// Eight or sixteen lanes per column where each then has no more than 32 rows and one pick, a whole warp for more.
template <typename T> cudaError_t launch_route(const RouteArgs &a, const void *X, const float *bias, cudaStream_t st) {
    if (a.nrows <= 256 && a.k <= 8)
        return bias ? launch_route_as<T, 8, true>(a, X, bias, st) : launch_route_as<T, 8, false>(a, X, bias, st);
    if (a.nrows <= 512 && a.k <= 16)
        return bias ? launch_route_as<T, 16, true>(a, X, bias, st) : launch_route_as<T, 16, false>(a, X, bias, st);
    return bias ? launch_route_as<T, 32, true>(a, X, bias, st) : launch_route_as<T, 32, false>(a, X, bias, st);
}

template <typename T, int G>
cudaError_t launch_grad_as(RouteArgs a, int nnz, const void *X, const int *Sir, const int *Sjc, const float *Sdata, const float *dS,
                           void *dX, long long lddx, cudaStream_t st) {
    constexpr int N = Pack<T>::N;
    a.stride = ((a.nrows + 31) & ~31) + 8;
    a.wide = is16(X) && a.nrows % N == 0 && (a.ldx % N == 0 || a.ncols == 1);
    a.wide_out = is16(dX) && a.nrows % N == 0 && (lddx % N == 0 || a.ncols == 1);
    const size_t smem = (size_t)kRouteWarps * (32 / G) * a.stride * sizeof(float);
    const long long per = (long long)kRouteWarps * (32 / G);
    route_grad_kernel<T, G><<<(unsigned)((a.ncols + per - 1) / per), kRouteWarps * 32, smem, st>>>(a, nnz, (const T *)X, Sir, Sjc, Sdata, dS,
                                                                                                (T *)dX, lddx);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_grad(const RouteArgs &a, int nnz, const void *X, const int *Sir, const int *Sjc, const float *Sdata, const float *dS,
                        void *dX, long long lddx, cudaStream_t st) {
    return a.nrows <= 256 ? launch_grad_as<T, 8>(a, nnz, X, Sir, Sjc, Sdata, dS, dX, lddx, st)
                          : launch_grad_as<T, 32>(a, nnz, X, Sir, Sjc, Sdata, dS, dX, lddx, st);
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
    RouteArgs a{nrows, ncols, k, score, ngroups, topgroups, grouptop, renorm, ldx, scale, nrows / ngroups, 0, 0, 0, 0, 0, 0, Sir, Sic, Sjc, Sdata};
    cudaError_t err = cudaSuccess;
#define CALL_ROUTE(T) err = launch_route<T>(a, X, bias, st)
    DISPATCH_DTYPE(dtype, CALL_ROUTE);
#undef CALL_ROUTE
    if (err != cudaSuccess) return (int)err;
    g_launches += 1;
    return (int)cudaGetLastError();
}

extern "C" int bidmat_b200_route_grad(int nrows, int ncols, int nnz, const void *X, long long ldx, int dtype, int score,
                                      int renorm, float scale, const int *Sir, const int *Sjc, const float *Sdata,
                                      const float *dS, void *dX, long long lddx, bidmat_stream_t stream) {
    if (!route_sizes_ok(nrows, ncols, score, scale) || !dtype_ok(dtype) || nnz < 0 || nnz > kMostEntries)
        return (int)cudaErrorInvalidValue;
    if (ncols == 0) return 0;
    if (!dense_ok(X, ldx, nrows, dtype) || !dense_ok(dX, lddx, nrows, dtype) || !Sjc) return (int)cudaErrorInvalidValue;
    if (nnz > 0 && (!Sir || !Sdata || !dS)) return (int)cudaErrorInvalidValue;
    if (X == dX && ldx != lddx) return (int)cudaErrorInvalidValue;
    cudaStream_t st = as_stream(stream);
    RouteArgs a{};
    a.nrows = nrows; a.ncols = ncols; a.score = score; a.renorm = renorm; a.ldx = ldx; a.scale = scale;
    cudaError_t err = cudaSuccess;
#define CALL_GRAD(T) err = launch_grad<T>(a, nnz, X, Sir, Sjc, Sdata, dS, dX, lddx, st)
    DISPATCH_DTYPE(dtype, CALL_GRAD);
#undef CALL_GRAD
    if (err == cudaSuccess) g_launches += 1;
    return (int)err;
}
