// Sampling a token from each row of logits (sm_100a), from given random numbers.
//
//     w_i = exp((z_i - max z) / T)
//     top k:  the k largest z, equal ones by lowest index
//     top p:  of those the shortest run, largest first (equal ones by lowest index), whose
//             weight is at least p of theirs
//     min p:  of those the ones with w_i >= min p
//     token:  the first i in index order whose weights up to it pass u times their sum
//
// What is kept is a run of the ranking by (z descending, index ascending), so it is
// given by its last entry: (tau, ti) keeps z > tau, and z == tau up to index ti.
//
// A sum next to a border decides a token, and sums of 131072 weights in float32 are
// off by more than the distance between neighbours: weights and sums are doubles, in a
// fixed order (a lane, a warp, then the warps in order), so a call's result is the
// same every time. No order of atomics reaches it: what they collect is counted in
// whole numbers, or sorted.
//
// A row is read by a cluster of C CTAs; warp q of all of theirs has the q-th piece of the
// row in every pass, so that sums in index order are sums over warps. The k-th largest
// entry and the end of the mass p are found by bins over the range of the logits: counts or
// fixed-point weights of 2048 equal bins, then the bin in question is made the range,
// until it holds one value or few enough entries to sort. Whole-number bins only choose
// where to look: the weights before the bin are summed again as doubles, and a bin
// that was chosen wrongly by the rounding of the fixed-point weights is left for its neighbour.
#include <algorithm>
#include <cooperative_groups.h>

#include "mms_common.cuh"
#include "mms_serve.h"

namespace cg = cooperative_groups;

namespace mms {

namespace {

constexpr int THREADS = 512, NW = THREADS / 32;
constexpr int BINS = 2048;
constexpr int CAP = 2048;               // entries that are sorted rather than divided further
constexpr float NEG_INF = -__builtin_huge_valf();

// Larger keys for larger floats; -0 and 0 are one value.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// What the CTAs of a row tell one another.
struct Part {
    double mass, bin_mass;              // weight of the bins before the one in question, and of it
    float lo, hi;                       // smallest and largest value of the bin
    float before, after;                // smallest value of the bins before, largest of those after
    int bin_count;
    float top;                          // largest value, and its lowest index
    int top_at;
    float least;                        // smallest value above -inf
    int nan;
};

struct Shared {
    unsigned long long bins[BINS];      // counts, or fixed-point weights
    unsigned long long list[CAP];       // (key, index), to be sorted so that the largest value comes first
    unsigned long long warp_bins[NW];
    double warp_mass[NW];               // of the CTA's warps
    double all_mass[8 * NW];            // of all the row's warps
    int warp_count[NW], all_count[8 * NW];
    Part part, warp_part[NW];
    int listed;
    float tau;
    int ti;
    int bin;
    int token;
    double weight;
};

// The row as one CTA sees it.
template <typename E, int C>
struct Row {
    static constexpr int VEC = 16 / (int)sizeof(E);
    const E *p;
    int vocab, off;                     // entries before p back to a 16-byte boundary
    int from, to;                       // this warp's piece, counted from that boundary
    float top;
    double rate;                        // 1 / T
    float tau;
    int ti;

    __device__ __forceinline__ double weight(float v) const {
        if (isinf(top)) return v == top ? 1.0 : 0.0;
        return exp(((double)v - (double)top) * rate);
    }
    __device__ __forceinline__ bool kept(float v, int i) const { return v > tau || (v == tau && i <= ti); }

    // f(value, index) over the piece, 32 * VEC entries at a time; lane l has VEC neighbours
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        const int lane = threadIdx.x & 31;
        constexpr int UN = 2;
        for (int at = from; at < to; at += 32 * VEC * UN) {
            E v[UN][VEC];
#pragma unroll
            for (int q = 0; q < UN; ++q) read(v[q], at + (q * 32 + lane) * VEC);
#pragma unroll
            for (int q = 0; q < UN; ++q)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const int i = at + (q * 32 + lane) * VEC + j - off;
                    if (i >= 0 && i < vocab && i + off < to) f(to_f(v[q][j]), i);
                }
        }
    }
    // entries at .. at + VEC - 1 of the piece; those outside the row are left as they are
    __device__ __forceinline__ void read(E (&v)[VEC], int at) const {
        if (at >= off && at + VEC <= vocab + off) {
            *reinterpret_cast<uint4 *>(v) = __ldg(reinterpret_cast<const uint4 *>(p - off + at));
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (at + j >= off && at + j < vocab + off) v[j] = p[at + j - off];
        }
    }
};

template <int C>
__device__ __forceinline__ void row_sync() {
    if constexpr (C > 1) cg::this_cluster().sync();
    else __syncthreads();
}
template <int C, typename T>
__device__ __forceinline__ T *of_rank(T *p, int r) {
    if constexpr (C > 1) return cg::this_cluster().map_shared_rank(p, r);
    else return p;
}
template <int C>
__device__ __forceinline__ int rank_of() {
    if constexpr (C > 1) return (int)cg::this_cluster().block_rank();
    else return 0;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ int warp_sum(int v) { return __reduce_add_sync(0xffffffffu, v); }

// Every warp's value (lane-wise `v`) to sh.all_mass of all CTAs, in the row's order.
template <int C>
__device__ double row_sums(Shared &sh, double v)
{
    const int warp = threadIdx.x >> 5;
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) sh.warp_mass[warp] = v;
    row_sync<C>();
    for (int i = threadIdx.x; i < C * NW; i += THREADS) sh.all_mass[i] = of_rank<C>(sh.warp_mass, i / NW)[i % NW];
    row_sync<C>();
    double total = 0.0;
    for (int i = 0; i < C * NW; ++i) total += sh.all_mass[i];
    return total;
}
template <int C>
__device__ int row_counts(Shared &sh, int v)
{
    const int warp = threadIdx.x >> 5;
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) sh.warp_count[warp] = v;
    row_sync<C>();
    for (int i = threadIdx.x; i < C * NW; i += THREADS) sh.all_count[i] = of_rank<C>(sh.warp_count, i / NW)[i % NW];
    row_sync<C>();
    int total = 0;
    for (int i = 0; i < C * NW; ++i) total += sh.all_count[i];
    return total;
}

__device__ __forceinline__ void join(Part &a, const Part &b)
{
    a.mass += b.mass, a.bin_mass += b.bin_mass, a.bin_count += b.bin_count;
    a.lo = fminf(a.lo, b.lo), a.hi = fmaxf(a.hi, b.hi);
    a.before = fminf(a.before, b.before), a.after = fmaxf(a.after, b.after);
    if (b.top > a.top || (b.top == a.top && b.top_at < a.top_at)) a.top = b.top, a.top_at = b.top_at;
    a.least = fminf(a.least, b.least);
    a.nan |= b.nan;
}
__device__ __forceinline__ Part no_part()
{
    return Part{0.0, 0.0, -NEG_INF, NEG_INF, -NEG_INF, NEG_INF, 0, NEG_INF, 0x7fffffff, -NEG_INF, 0};
}

// Parts of all lanes joined in the row's order; every thread gets the whole.
template <int C>
__device__ Part row_part(Shared &sh, Part v)
{
    const int warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Part b;
        b.mass = __shfl_xor_sync(0xffffffffu, v.mass, o), b.bin_mass = __shfl_xor_sync(0xffffffffu, v.bin_mass, o);
        b.lo = __shfl_xor_sync(0xffffffffu, v.lo, o), b.hi = __shfl_xor_sync(0xffffffffu, v.hi, o);
        b.before = __shfl_xor_sync(0xffffffffu, v.before, o), b.after = __shfl_xor_sync(0xffffffffu, v.after, o);
        b.bin_count = __shfl_xor_sync(0xffffffffu, v.bin_count, o);
        b.top = __shfl_xor_sync(0xffffffffu, v.top, o), b.top_at = __shfl_xor_sync(0xffffffffu, v.top_at, o);
        b.least = __shfl_xor_sync(0xffffffffu, v.least, o), b.nan = __shfl_xor_sync(0xffffffffu, v.nan, o);
        join(v, b);
    }
    if ((threadIdx.x & 31) == 0) sh.warp_part[warp] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        v = sh.warp_part[0];
        for (int i = 1; i < NW; ++i) join(v, sh.warp_part[i]);
        sh.part = v;
    }
    row_sync<C>();
    v = *of_rank<C>(&sh.part, 0);
    for (int r = 1; r < C; ++r) join(v, *of_rank<C>(&sh.part, r));
    row_sync<C>();
    return v;
}

// The list sorted ascending, padded with ones to a power of two.
__device__ void sort_list(unsigned long long *list, int n)
{
    int m = 2;
    while (m < n) m *= 2;
    for (int i = n + threadIdx.x; i < m; i += THREADS) list[i] = ~0ull;
    for (int size = 2; size <= m; size *= 2)
        for (int gap = size / 2; gap > 0; gap /= 2) {
            __syncthreads();
            for (int i = threadIdx.x; i < m / 2; i += THREADS) {
                const int a = 2 * i - (i & (gap - 1)), b = a + gap;
                const unsigned long long x = list[a], y = list[b];
                if ((x > y) == ((a & size) == 0)) list[a] = y, list[b] = x;
            }
        }
    __syncthreads();
}

// The index of the n-th (from 1) kept entry equal to `value`.
template <typename E, int C>
__device__ int nth_equal(Shared &sh, const Row<E, C> &row, float value, int n)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = rank_of<C>();
    int mine = 0;
    row.each([&](float v, int i) { mine += v == value && row.kept(v, i); });
    row_counts<C>(sh, mine);
    int w = 0, left = n;
    while (w < C * NW - 1 && left > sh.all_count[w]) left -= sh.all_count[w++];
    if (w == rank * NW + warp) {
        constexpr int VEC = Row<E, C>::VEC;
        for (int at = row.from; at < row.to; at += 32 * VEC) {
            E v[VEC];
            row.read(v, at + lane * VEC);
            unsigned hits = 0;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int i = at + lane * VEC + j - row.off;
                if (i >= 0 && i < row.vocab && i + row.off < row.to && to_f(v[j]) == value && row.kept(value, i)) hits |= 1u << j;
            }
            int upto = __popc(hits);
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int b = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += b;
            }
            const int before = upto - __popc(hits), all = __shfl_sync(0xffffffffu, upto, 31);
            if (left > before && left <= upto) {
                for (int k = left - before; k > 1; --k) hits &= hits - 1;
                const int i = at + lane * VEC + __ffs(hits) - 1 - row.off;
                for (int r = 0; r < C; ++r) of_rank<C>(&sh, r)->ti = i;
            }
            if (left <= all) break;
            left -= all;
        }
    }
    row_sync<C>();
    return sh.ti;
}

// Cuts what is kept to the shortest run of the ranking that reaches `target`: so many
// entries (MASS false), or so much weight. Where all of it does not, nothing changes.
// Every round ends in a smaller [a, b]; MOST bounds them all the same.
template <bool MASS, typename E, int C>
__device__ void cut(Shared &sh, Row<E, C> &row, double target, float least)
{
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = rank_of<C>();
    float a = fmaxf(least, row.tau), b = row.top;          // the last entry of the run lies in [a, b]
    double above = 0.0;                                    // what lies above b
    // fixed point of the bins' weights: sums of all entries stay below 2^63
    const double unit = MASS ? exp2((double)min(45, 62 - (32 - __clz(row.vocab)))) : 1.0;
    constexpr int MOST = 100;
    for (int round = 0; round < MOST; ++round) {
        const double scale = BINS / ((double)b - (double)a);
        auto bin_of = [&](float v) { return a == b ? 0 : min(BINS - 1, (int)(((double)b - (double)v) * scale)); };
        // where no sum reaches the target by the rounding of the weights: the bin of the smallest value
        const int last = a == b ? 0 : BINS - 1;
        for (int i = tid; i < BINS; i += THREADS) sh.bins[i] = 0;
        if (tid == 0) sh.listed = 0, sh.bin = last;
        __syncthreads();
        row.each([&](float v, int i) {
            if (v <= b && v >= a && row.kept(v, i))
                atomicAdd(&sh.bins[bin_of(v)], MASS ? (unsigned long long)(row.weight(v) * unit) : 1ull);
        });
        row_sync<C>();
        // each thread's bins of the whole row, then where the sum reaches the target
        constexpr int PER = BINS / THREADS;
        unsigned long long mine[PER], sum = 0;
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            mine[q] = 0;
            for (int r = 0; r < C; ++r) mine[q] += of_rank<C>(sh.bins, r)[tid * PER + q];
            sum += mine[q];
        }
        unsigned long long upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const unsigned long long v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 31) sh.warp_bins[warp] = upto;
        __syncthreads();
        for (int w = 0; w < warp; ++w) upto += sh.warp_bins[w];
        upto -= sum;
        const double want = fmax(0.0, (target - above) * unit);
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const double lo = (double)upto;
            upto += mine[q];
            if (lo < want && (double)upto >= want) atomicMin(&sh.bin, tid * PER + q);
        }
        row_sync<C>();                                     // the bins are read, the bin is known
        const int bin = sh.bin;
        // the bins before it and it itself, as doubles; its entries to the list
        Part p = no_part();
        row.each([&](float v, int i) {
            if (v > b || v < a || !row.kept(v, i)) return;
            const int k = bin_of(v);
            const double w = MASS ? (k <= bin ? row.weight(v) : 0.0) : 1.0;
            if (k < bin) {
                p.mass += w;
                p.before = fminf(p.before, v);
            } else if (k > bin) {
                p.after = fmaxf(p.after, v);
            } else {
                p.bin_mass += w;
                p.lo = fminf(p.lo, v), p.hi = fmaxf(p.hi, v);
                ++p.bin_count;
                const int at = atomicAdd(&of_rank<C>(&sh, 0)->listed, 1);
                if (at < CAP) of_rank<C>(&sh, 0)->list[at] = (unsigned long long)(~key_of(v)) << 32 | (unsigned)i;
            }
        });
        p = row_part<C>(sh, p);
        const double ahead = above + p.mass;
        if (p.before <= b && ahead >= target) {            // rounding: it is in a bin before
            a = p.before;
            continue;
        }
        if (p.bin_count == 0 || ahead + p.bin_mass < target) {
            if (p.after < a) break;                        // all of it does not reach the target
            above = ahead + p.bin_mass;                    // rounding: it is in a bin behind
            b = p.after;
            continue;
        }
        if (p.lo == p.hi) {
            const double each = MASS ? row.weight(p.lo) : 1.0;
            const int n = (int)fmin((double)p.bin_count, fmax(1.0, ceil((target - ahead) / each)));
            if (n < p.bin_count) {
                const int ti = nth_equal(sh, row, p.lo, n);
                row.ti = ti;
            } else if (p.lo != row.tau) {
                row.ti = 0x7fffffff;
            }
            row.tau = p.lo;
            return;
        }
        if (p.bin_count <= CAP) {
            if (rank == 0) {
                sort_list(sh.list, p.bin_count);
                if (tid == 0) {
                    double sum = ahead;
                    int i = 0;
                    for (; i < p.bin_count - 1; ++i) {
                        sum += MASS ? row.weight(of_key(~(uint32_t)(sh.list[i] >> 32))) : 1.0;
                        if (sum >= target) break;
                    }
                    sh.tau = of_key(~(uint32_t)(sh.list[i] >> 32));
                    sh.ti = (int)(uint32_t)sh.list[i];
                }
            }
            row_sync<C>();
            row.tau = of_rank<C>(&sh, 0)->tau;
            row.ti = of_rank<C>(&sh, 0)->ti;
            row_sync<C>();
            return;
        }
        a = p.lo, b = p.hi, above = ahead;
    }
    if (a != row.tau) row.ti = 0x7fffffff;
    row.tau = a;
}

template <typename E, int C>
__global__ void __launch_bounds__(THREADS)
sample_kernel(const __grid_constant__ SampleArgs s)
{
    __shared__ Shared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = rank_of<C>(), at = blockIdx.x / C;
    constexpr int VEC = Row<E, C>::VEC;
    Row<E, C> row;
    row.p = reinterpret_cast<const E *>(s.logits) + at * s.ld;
    row.vocab = s.vocab;
    row.off = (int)((reinterpret_cast<uintptr_t>(row.p) & 15) / sizeof(E));
    const int piece = ((s.vocab + row.off + C * NW - 1) / (C * NW) + 32 * VEC - 1) / (32 * VEC) * (32 * VEC);
    row.from = (int)min((long long)(rank * NW + warp) * piece, (long long)s.vocab + row.off);
    row.to = (int)min((long long)row.from + piece, (long long)s.vocab + row.off);
    row.tau = NEG_INF, row.ti = -1, row.top = 0.f;

    Part p = no_part();
    row.each([&](float v, int i) {
        p.nan |= v != v;
        if (v > p.top) p.top = v, p.top_at = i;
        if (v > NEG_INF) p.least = fminf(p.least, v);
    });
    p = row_part<C>(sh, p);
    row.top = p.top;
    if (isinf(p.top)) row.tau = p.top, row.ti = 0x7fffffff;        // nothing beside it has weight
    const float t = s.temperature ? s.temperature[at] : s.temperature1;
    const long long k = s.top_k.p ? s.top_k.at(at) : s.top_k1;
    const float top_p = s.top_p ? s.top_p[at] : s.top_p1;
    const float min_p = fminf(s.min_p ? s.min_p[at] : s.min_p1, 1.f);
    row.rate = 1.0 / (double)t;
    // nothing to draw from, or nothing to draw
    const bool none = p.nan || !(p.top > NEG_INF) || t != t || top_p != top_p;
    if (none || t <= 0.f || k == 1 || top_p <= 0.f) {
        if (rank == 0 && tid == 0) {
            s.token[at] = none ? -1 : p.top_at;
            if (s.logprob) s.logprob[at] = none ? __int_as_float(0x7fc00000) : 0.f;
        }
        if constexpr (C > 1) cg::this_cluster().sync();    // no CTA leaves while another reads its memory
        return;
    }
    if (k > 0 && k < s.vocab) cut<false>(sh, row, (double)k, p.least);
    if (top_p < 1.f) {
        double mass = 0.0;
        row.each([&](float v, int i) {
            if (row.kept(v, i)) mass += row.weight(v);
        });
        const double all = row_sums<C>(sh, mass);
        cut<true>(sh, row, (double)top_p * all, p.least);
    }
    double mass = 0.0;
    auto weight = [&](float v, int i) {
        const double w = row.kept(v, i) ? row.weight(v) : 0.0;
        return w >= (double)min_p ? w : 0.0;
    };
    row.each([&](float v, int i) { mass += weight(v, i); });
    const double all = row_sums<C>(sh, mass);
    const float u = s.uniform[at];
    const double want = (u > 0.f ? fmin((double)u, 1.0) : 0.0) * all;
    // the warp whose piece passes it (or the last that has any weight), then the entry
    int w = -1;
    double upto = 0.0, base = 0.0;
    for (int i = 0; i < C * NW; ++i) {
        const double m = sh.all_mass[i];
        if (m > 0.0 && (w < 0 || upto <= want)) w = i, base = upto;
        upto += m;
    }
    if (w == rank * NW + warp) {
        int token = -1;
        double of_token = 0.0;
        for (int a = row.from; a < row.to; a += 32 * VEC) {
            E v[VEC];
            row.read(v, a + lane * VEC);
            double ws[VEC], sum = 0.0;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int i = a + lane * VEC + j - row.off;
                ws[j] = i >= 0 && i < row.vocab && i + row.off < row.to ? weight(to_f(v[j]), i) : 0.0;
                sum += ws[j];
            }
            double incl = sum;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const double b = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += b;
            }
            // the lane's first entry past `want`, else its last with weight
            double run = base + incl - sum;
            int hit = -1, last = -1;
            double hit_w = 0.0, last_w = 0.0;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                run += ws[j];
                if (ws[j] > 0.0) {
                    const int i = a + lane * VEC + j - row.off;
                    if (hit < 0 && run > want) hit = i, hit_w = ws[j];
                    last = i, last_w = ws[j];
                }
            }
            const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), any = __ballot_sync(0xffffffffu, last >= 0);
            if (hits) {
                const int l = __ffs(hits) - 1;
                token = __shfl_sync(0xffffffffu, hit, l), of_token = __shfl_sync(0xffffffffu, hit_w, l);
                break;
            }
            if (any) {
                const int l = 31 - __clz(any);
                token = __shfl_sync(0xffffffffu, last, l), of_token = __shfl_sync(0xffffffffu, last_w, l);
            }
            base += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) {
            s.token[at] = token;
            if (s.logprob) s.logprob[at] = (float)log(of_token / all);
        }
    }
    if constexpr (C > 1) cg::this_cluster().sync();
}

template <typename E, int C>
cudaError_t sample_of(const SampleArgs &a, cudaStream_t stream)
{
    cudaLaunchConfig_t c{};
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = C, cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    c.gridDim = dim3((unsigned)((long long)a.rows * C));
    c.blockDim = dim3(THREADS);
    c.stream = stream;
    c.attrs = &cluster;
    c.numAttrs = C > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&c, sample_kernel<E, C>, a);
}

// CTAs a row: as many (up to 8, a portable cluster) as still fit the GPU at 2 an SM, none of
// fewer than 2048 entries.
template <typename E>
cudaError_t sample_by_rows(const SampleArgs &a, cudaStream_t stream)
{
    const long long most = std::min<long long>(2LL * N_SM / a.rows, a.vocab / 2048);
    if (most >= 8) return sample_of<E, 8>(a, stream);
    if (most >= 4) return sample_of<E, 4>(a, stream);
    if (most >= 2) return sample_of<E, 2>(a, stream);
    return sample_of<E, 1>(a, stream);
}

}  // namespace

cudaError_t launch_sample(const SampleArgs &a, cudaStream_t stream)
{
    return a.bf16 ? sample_by_rows<__nv_bfloat16>(a, stream) : sample_by_rows<float>(a, stream);
}

}  // namespace mms
