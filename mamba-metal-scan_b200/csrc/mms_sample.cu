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
// off by more than the distance between neighbours. Weights are computed in float64
// and held as whole numbers of 2^-44 of the largest (fewer bits above 2^18 entries, so that
// no sum passes 2^62): their sums are exact in any order, so bins may be filled by atomics
// and a call's result is the same every time.
//
// A row is read by a cluster of C CTAs; warp q of all of theirs has the q-th piece of the
// row in every pass, so that sums in index order are sums over warps.
//   k up to about 256 C: every warp has the j-th largest of its 32 lanes' maxima, j = k / warps
//     rounded up; the m-th largest of these, m = k / j rounded up, has k entries above it or
//     equal, and not many more. Those are listed and sorted, and all else happens on the list.
//   else: the end of the run of k entries, or of the mass p, is found by bins over the
//     range of the logits, counts and weights of 2048 equal bins. If the entries down to the bin in
//     question fit the list, all else happens there; otherwise that bin becomes the range,
//     until it holds one value or few enough entries to sort, and another pass draws.
//   bf16, where k is not small or there is a p, and a row has one or two CTAs: there are few different values, so
//     one pass counts each of 5633 of them (magnitudes 2^-16 to 64 and 0; the others are listed one by one),
//     and every cut and sum follows from the counts; one more pass, with the weights from a
//     table, draws. Only where a cut falls among the values that are not counted, or too many are
//     not, the bins above find it. (p = 0.9: 256 x 131072 by one CTA 141 us, by bins 283; 60 x 20000 by
//     two 39 and 53. By eight the tables cost more than their part of a row: 1 x 32768 49 and 41. Without a
//     cut the table loses too: 60 x 131072, 45 us and 34. Logits most of which are not counted pay for both: 256 x
//     131072 of standard deviation 2000 at a temperature of 1000, 317 us, float32 rows of them, bins alone, 281.)
// The row is read from HBM once; the later passes, one to five, find it in L2. What bounds a
// pass over all weights is their arithmetic (12 operations in float64 and some 30 others an
// entry), not the bytes.

#include <float.h>

#include <algorithm>
#include <cooperative_groups.h>

#include "mms_common.cuh"
#include "mms_serve.h"

namespace cg = cooperative_groups;

namespace mms {

namespace {

using u64 = unsigned long long;
constexpr int THREADS = 512, NW = THREADS / 32;
constexpr int BINS = 2048;
constexpr int CAP = 2048;               // entries that are sorted rather than divided further
constexpr int PER = BINS / THREADS;     // bins, and list entries, of a thread
static_assert(CAP == BINS, "one scan serves both");
constexpr int RANKED = 128;             // entries that are sorted by counting, at most
constexpr float NEG_INF = -__builtin_huge_valf();
constexpr int BITS = 44;                // of weights, fewer above 2^18 entries
constexpr int LIMBS_MAX = 1 << 17;      // entries whose weights' 15-bit parts add up in 32 bits
constexpr int EVERY = 0x7fffffff;       // ti: all entries equal to tau

// Larger keys for larger floats; -0 and 0 are one value.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// The values of bf16 rows that are counted, in descending order: 2^6 (1 - 2^-8) .. 2^-16, 0, -2^-16 ..
// Between and around them lie the others, in four gaps: above, between the counted ones and 0 on
// either side, below.
constexpr int CORE_LOW = 0x3780, CORE = 0x4280 - CORE_LOW;           // bits of 2^-16; magnitudes
constexpr int ZERO = CORE + 2, VALUES = 2 * CORE + 5;                // gap, CORE, gap, 0, gap, CORE, gap
constexpr int PER_VALUE = (VALUES + THREADS - 1) / THREADS;
// Where a counted value (bf16 bits) lies in the tables: positive ones by magnitude, then negative
// ones, then 0; -1 for the others.
__device__ __forceinline__ int value_slot(uint32_t b) {
    const uint32_t off = (b & 0x7fffu) - CORE_LOW;
    return off < (uint32_t)CORE ? (int)(off + (b >> 15) * CORE) : (b & 0x7fffu) == 0 ? 2 * CORE : -1;
}
// A gap's slot behind them.
__device__ __forceinline__ int gap_slot(uint32_t b) {
    return 2 * CORE + 1 + ((b & 0x7fffu) < CORE_LOW ? 1 + (b >> 15) : 3 * (b >> 15));
}
__device__ __forceinline__ bool is_gap(int place) {
    return place == 0 || place == ZERO - 1 || place == ZERO + 1 || place == VALUES - 1;
}
// the slot of a place in the descending order
__device__ __forceinline__ int slot_at(int place) {
    if (is_gap(place)) return 2 * CORE + 1 + (place == 0 ? 0 : place == ZERO - 1 ? 1 : place == ZERO + 1 ? 2 : 3);
    return place == ZERO ? 2 * CORE : place < ZERO ? CORE - place : CORE + (place - ZERO - 2);
}
__device__ __forceinline__ float value_at(int place) {               // of one that is no gap
    if (place == ZERO) return 0.f;
    const uint32_t b = place < ZERO ? (uint32_t)(CORE_LOW + CORE - place) : 0x8000u + CORE_LOW + (place - ZERO - 2);
    return __uint_as_float(b << 16);
}

struct Shared {
    union {
        struct {
            union {
                unsigned limbs[2][BINS];    // weights of bins, 15 bits of each weight in one sum, ..
                u64 bins[BINS];             // .. or whole
            };
            unsigned counts[BINS];
            union {
                unsigned limb2[BINS];       // the uppermost 15 bits
                u64 list[CAP];
            };
            u64 row_bins[BINS];             // the whole row's bins, of C > 1
            unsigned row_counts[BINS];
            float queue[NW][64];            // a warp's entries that wait for a whole warp of them
        };
        struct {
            u64 table[VALUES];              // a value's weight; a gap's whole (by slot)
            unsigned found[VALUES];         // its count
            float others[CAP];
        };
    };
    double powers[16];                  // 2^(j / 16)
    u64 warp_sum[NW];                   // of the CTA's warps
    u64 all_sum[8 * NW];                // of all the row's warps
    float warp_max[NW], warp_pivot[NW], warp_lo[NW], warp_hi[NW];
    float all_pivot[8 * NW], pivot;
    u64 before;                         // what lies before the bin in question
    u64 scan[NW];
    int listed, bin, least, tau_key, ti, others_count;
    unsigned entries;                   // of the range, down to the bin in question
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

// the next smaller float
__device__ __forceinline__ float below(float v) {
    const int b = __float_as_int(v);
    return v == 0.f ? -1e-45f : __int_as_float(v > 0.f ? b - 1 : b + 1);
}
// max that hands a NaN on
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
template <typename F>
__device__ __forceinline__ float warp_fold(float v, F f) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_scan(u64 v) {          // inclusive
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const u64 b = __shfl_up_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) >= o) v += b;
    }
    return v;
}
// What the threads before this one hold together (sh.scan; every thread gets the whole in `all`).
__device__ __forceinline__ u64 block_before(Shared &sh, u64 v, u64 &all) {
    const int warp = threadIdx.x >> 5;
    const u64 upto = warp_scan(v);
    __syncthreads();                                       // sh.scan of a call before
    if ((threadIdx.x & 31) == 31) sh.scan[warp] = upto;
    __syncthreads();
    u64 r = upto - v;
    all = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        if (w < warp) r += sh.scan[w];
        all += sh.scan[w];
    }
    return r;
}

// 16 bytes of a row.
template <typename E>
struct Words {
    static constexpr int VEC = 16 / (int)sizeof(E);
    uint4 q;
    __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w; }
    __device__ __forceinline__ float at(int j) const {
        if constexpr (sizeof(E) == 4) return __uint_as_float(word(j));
        else return __uint_as_float(j & 1 ? word(j >> 1) & 0xffff0000u : word(j >> 1) << 16);
    }
    // the largest, or a NaN if there is one
    __device__ __forceinline__ float most() const {
        if constexpr (sizeof(E) == 4) {
            return max_nan(max_nan(at(0), at(1)), max_nan(at(2), at(3)));
        } else {
            auto two = [](uint32_t w) { return reinterpret_cast<const __nv_bfloat162 &>(w); };
            const __nv_bfloat162 a = __hmax2_nan(two(q.x), two(q.y)), b = __hmax2_nan(two(q.z), two(q.w));
            const __nv_bfloat162 m = __hmax2_nan(a, b);
            return max_nan(__low2float(m), __high2float(m));
        }
    }
};

// The row as one CTA sees it. Places count from the 16-byte boundary at or before its start.
template <typename E, int C>
struct Row {
    static constexpr int VEC = Words<E>::VEC, STEP = 32 * VEC;
    const E *p;                         // that boundary
    int off, end;                       // first place, and the one behind the last
    int piece;                          // places of a warp's piece, whole steps
    float top, floor;                   // the largest; no weight is left here and below
    double limit, rate;                 // the largest as a finite number; 1 / T
    int bits;                           // weights are whole numbers of 2^-bits
    const double *powers;
    float tau;
    int ti;

    __device__ __forceinline__ int from(int w) const { return (int)min((long long)w * piece, (long long)end); }

    // (v - top) / T
    __device__ __forceinline__ double exponent(float v) const { return ((double)fminf(v, FLT_MAX) - limit) * rate; }
    // 2^bits e^exponent, rounded. e^x = 2^(k / 16) e^r, |r| <= log(2) / 32, the first factor from a
    // table, the second to r^6: what is left out is r^7 / 5040 < 5e-16 (table-driven exponentials
    // after Tang, 1989). At `floor` and below, where x is -34 or less, it is 0.
    __device__ __forceinline__ u64 weight(float v) const {
        constexpr double ROUND = 6755399441055744.0;       // 1.5 * 2^52: the sum's last bit is worth 1
        constexpr double STEP16 = 0.69314718055994531 / 16.0;
        const double x = ((double)fmaxf(fminf(v, FLT_MAX), floor) - limit) * rate;
        const double m = fma(x, 1.0 / STEP16, ROUND);
        const int k = __double2loint(m);
        const double r = fma(m - ROUND, -STEP16, x);
        double e = fma(r, 1.0 / 720.0, 1.0 / 120.0);
        e = fma(e, r, 1.0 / 24.0);
        e = fma(e, r, 1.0 / 6.0);
        e = fma(e, r, 0.5);
        e = fma(e, r, 1.0);
        e = fma(e, r, 1.0);
        e *= powers[k & 15];
        e = __hiloint2double(__double2hiint(e) + (((k >> 4) + bits) << 20), __double2loint(e));
        const u64 w = (u64)__double_as_longlong(e + 4503599627370496.0) & ((1ull << 52) - 1);
        return v > floor ? w : 0;
    }
    // w to a bin. Shared memory adds 32 bits at a time: three sums of 15 bits of each weight hold it (of
    // rows above LIMBS_MAX, 64 bits in a loop), and most weights have the lowest 15 alone.
    __device__ __forceinline__ void add(Shared &sh, int bin, u64 w) const {
        atomicAdd(&sh.counts[bin], 1u);
        if (end - off > LIMBS_MAX) {
            atomicAdd(&sh.bins[bin], w);
        } else {
            atomicAdd(&sh.limbs[0][bin], (unsigned)w & 0x7fffu);
            const unsigned up = (unsigned)(w >> 15);
            if (up) {
                atomicAdd(&sh.limbs[1][bin], up & 0x7fffu);
                if (up >> 15) atomicAdd(&sh.limb2[bin], up >> 15);
            }
        }
    }
    __device__ __forceinline__ u64 weight_of(const Shared &o, int bin) const {
        return end - off > LIMBS_MAX ? o.bins[bin] : o.limbs[0][bin] + ((u64)o.limbs[1][bin] << 15) + ((u64)o.limb2[bin] << 30);
    }
    __device__ __forceinline__ bool kept(float v, int i) const { return v > tau || (v == tau && i <= ti); }

    // 16 bytes at a place; entries outside the row are -inf
    __device__ __forceinline__ Words<E> read(int at) const {
        Words<E> v;
        if (at >= off && at + VEC <= end) {
            v.q = __ldg(reinterpret_cast<const uint4 *>(p + at));
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(E) == 4) {
                    w[i] = at + i >= off && at + i < end ? __float_as_uint(to_f(p[at + i])) : 0xff800000u;
                } else {
                    uint32_t h[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int a = at + 2 * i + j;
                        h[j] = a >= off && a < end ? __float_as_uint(to_f(p[a])) >> 16 : 0xff80u;
                    }
                    w[i] = h[0] | h[1] << 16;
                }
            }
            v.q = make_uint4(w[0], w[1], w[2], w[3]);
        }
        return v;
    }
    // f(words, place of the first) over the warp's share [a, b) of the row, a multiple of STEP;
    // UN loads at a time (one where f is long: its code is there UN + 1 times, and a pass whose code
    // does not fit the instruction caches waits for it). Entries of a step are all within [a, b) or
    // outside the row.
    template <int UN, typename F>
    __device__ __forceinline__ void words(int a, int b, F f) const {
        const int lane = threadIdx.x & 31;
        int at = a;
        if constexpr (UN > 1) {
            for (; at + (UN - 1) * STEP < b; at += UN * STEP) {
                Words<E> v[UN];
#pragma unroll
                for (int q = 0; q < UN; ++q) v[q] = read(at + q * STEP + lane * VEC);
#pragma unroll
                for (int q = 0; q < UN; ++q) f(v[q], at + q * STEP + lane * VEC);
            }
        }
        if (at >= b) return;
        Words<E> next = read(at + lane * VEC);
#pragma unroll 1
        for (; at < b; at += STEP) {
            const Words<E> v = next;
            if (at + STEP < b) next = read(at + STEP + lane * VEC);
            f(v, at + lane * VEC);
        }
    }
    // f(value, index) for entries above -inf
    template <typename F>
    __device__ __forceinline__ void each(int a, int b, F f) const {
        words<1>(a, b, [&](const Words<E> &v, int at) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float x = v.at(j);
                if (x > NEG_INF) f(x, at + j - off);
            }
        });
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        const int w = rank_of<C>() * NW + (threadIdx.x >> 5);
        each(from(w), from(w + 1), f);
    }
};

// Every warp's value to sh.all_sum of all CTAs, in the row's order.
template <int C>
__device__ __forceinline__ void row_sums(Shared &sh, u64 v)
{
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) sh.warp_sum[threadIdx.x >> 5] = v;
    row_sync<C>();
    if (threadIdx.x < C * NW) sh.all_sum[threadIdx.x] = of_rank<C>(sh.warp_sum, threadIdx.x / NW)[threadIdx.x % NW];
    row_sync<C>();
}
// A float of every warp joined over the row (`mine` and `all` in shared memory).
template <int C, typename F>
__device__ __forceinline__ float row_fold(float (&mine)[NW], float v, F f)
{
    v = warp_fold(v, f);
    if ((threadIdx.x & 31) == 0) mine[threadIdx.x >> 5] = v;
    row_sync<C>();
    // lane l of every warp joins the warps l, l + 32, ... of the row
    const int lane = threadIdx.x & 31;
    v = of_rank<C>(mine, (lane % (C * NW)) / NW)[lane % NW];
    for (int i = lane + 32; i < C * NW; i += 32) v = f(v, of_rank<C>(mine, i / NW)[i % NW]);
    return warp_fold(v, f);
}

// The first n entries of sh.list sorted ascending (behind them: ones, up to a power of two, or what was there).
__device__ void sort_list(u64 *list, int n)
{
    if (n <= RANKED) {                                     // every entry's place by counting
        __syncthreads();
        const int i = threadIdx.x;
        const u64 mine = i < n ? list[i] : 0;
        int place = 0;
        if (i < n)
            for (int q = 0; q < n; ++q) place += list[q] < mine || (list[q] == mine && q < i);
        __syncthreads();
        if (i < n) list[place] = mine;
        __syncthreads();
        return;
    }
    // A bitonic network of m entries, four of them in a thread's registers: steps of 1 and 2 entries
    // there, up to 64 between the lanes of a warp, from 128 on (10 of 66 steps for 2048) in shared memory.
    int m = 256;
    while (m < n) m *= 2;
    __syncthreads();
    const int t = threadIdx.x;
    const bool in = t < m / 4;                             // (whole warps)
    ulonglong2 *mine = reinterpret_cast<ulonglong2 *>(list) + 2 * t;
    u64 v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = in && 4 * t + e < n ? list[4 * t + e] : ~0ull;
    auto keep = [](u64 &x, u64 other, bool low) { x = low == (other < x) ? other : x; };
    auto order = [](u64 &x, u64 &y, bool up) {
        const bool swap = (y < x) == up;
        const u64 a = swap ? y : x, b = swap ? x : y;
        x = a, y = b;
    };
#pragma unroll 1
    for (int size = 2; size <= m; size *= 2) {
        const bool up = (4 * t & size) == 0;
#pragma unroll 1
        for (int gap = size / 2; gap >= 128; gap /= 2) {
            __syncthreads();
            if (in) mine[0] = make_ulonglong2(v[0], v[1]), mine[1] = make_ulonglong2(v[2], v[3]);
            __syncthreads();
            if (in) {
                const ulonglong2 *other = reinterpret_cast<const ulonglong2 *>(list) + 2 * (t ^ gap / 4);
                const ulonglong2 a = other[0], b = other[1];
                const bool low = ((t & gap / 4) == 0) == up;
                keep(v[0], a.x, low), keep(v[1], a.y, low), keep(v[2], b.x, low), keep(v[3], b.y, low);
            }
        }
        if (!in) continue;
#pragma unroll 1
        for (int gap = min(size / 2, 64); gap >= 4; gap /= 2) {
            const bool low = ((t & gap / 4) == 0) == up;
#pragma unroll
            for (int e = 0; e < 4; ++e) keep(v[e], __shfl_xor_sync(0xffffffffu, v[e], gap / 4), low);
        }
        if (size > 2) order(v[0], v[2], up), order(v[1], v[3], up);
        order(v[0], v[1], up), order(v[2], v[3], size > 2 && up);
    }
    __syncthreads();
    if (in) mine[0] = make_ulonglong2(v[0], v[1]), mine[1] = make_ulonglong2(v[2], v[3]);
    __syncthreads();
}
// List entries that sort by rank (z descending, index ascending), and by index.
__device__ __forceinline__ u64 ranked(float v, int i) { return (u64)(~key_of(v)) << 32 | (unsigned)i; }
__device__ __forceinline__ float ranked_value(u64 e) { return of_key(~(uint32_t)(e >> 32)); }

// An entry to the CTA's list (counted, but not kept, above CAP).
__device__ __forceinline__ void to_list(Shared &sh, float v, int i) {
    const int at = atomicAdd(&sh.listed, 1);
    if (at < CAP) sh.list[at] = ranked(v, i);
}
// All CTAs' lists to the first one's, if it holds them; how many entries that are (all CTAs get it).
template <int C>
__device__ int join_lists(Shared &sh) {
    row_sync<C>();
    if constexpr (C == 1) return sh.listed;
    int n[C], all = 0;
#pragma unroll
    for (int r = 0; r < C; ++r) all += n[r] = *of_rank<C>(&sh.listed, r);
    if (rank_of<C>() == 0 && all <= CAP) {
        int to = n[0];
#pragma unroll
        for (int r = 1; r < C; ++r) {
            for (int i = threadIdx.x; i < n[r]; i += THREADS) sh.list[to + i] = of_rank<C>(sh.list, r)[i];
            to += n[r];
        }
    }
    row_sync<C>();
    return all;
}

// The first index of 0 .. n - 1 at which the sums of value(i) reach `target` (n - 1 if none does).
template <typename F>
__device__ int reached(Shared &sh, int n, u64 target, F value)
{
    u64 v[PER], sum = 0, all;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
        const int i = threadIdx.x * PER + q;
        v[q] = i < n ? value(i) : 0;
        sum += v[q];
    }
    if (threadIdx.x == 0) sh.least = n - 1;
    u64 upto = block_before(sh, sum, all);
#pragma unroll
    for (int q = 0; q < PER; ++q) {
        const u64 lo = upto;
        upto += v[q];
        if (lo < target && upto >= target) atomicMin(&sh.least, threadIdx.x * PER + q);
    }
    __syncthreads();
    return sh.least;
}

// ceil(share * sum) as the sum that has to be reached
__device__ __forceinline__ u64 share_of(float share, u64 sum) {
    return max(1ull, (u64)ceil((double)share * (double)sum));
}
// sums above this one pass u * sum; below `sum`, as u is below 1
__device__ __forceinline__ u64 border_of(float u, u64 sum) {
    u = u > 0.f ? fminf(u, 1.f - 0x1p-24f) : 0.f;
    return min((u64)((double)u * (double)sum), sum - 1);
}

// The index of the n-th (from 1) kept entry equal to `value`.
template <typename E, int C>
__device__ int nth_equal(Shared &sh, const Row<E, C> &row, float value, int n)
{
    const int lane = threadIdx.x & 31, mine = rank_of<C>() * NW + (threadIdx.x >> 5);
    u64 count = 0;
    row.each([&](float v, int i) { count += v == value && row.kept(v, i); });
    row_sums<C>(sh, count);
    int w = 0;
    u64 left = n;
    while (w < C * NW - 1 && left > sh.all_sum[w]) left -= sh.all_sum[w++];
    if (w == mine) {
        for (int at = row.from(w); at < row.from(w + 1); at += row.STEP) {
            const Words<E> v = row.read(at + lane * row.VEC);
            unsigned hits = 0;
#pragma unroll
            for (int j = 0; j < Row<E, C>::VEC; ++j)
                if (v.at(j) == value && row.kept(value, at + lane * row.VEC + j - row.off)) hits |= 1u << j;
            const u64 upto = warp_scan(__popc(hits)), before = upto - __popc(hits);
            const u64 all = __shfl_sync(0xffffffffu, upto, 31);
            if (left > before && left <= upto) {
                for (u64 k = left - before; k > 1; --k) hits &= hits - 1;
                const int i = at + lane * row.VEC + __ffs(hits) - 1 - row.off;
                for (int r = 0; r < C; ++r) of_rank<C>(&sh, r)->ti = i;
            }
            if (left <= all) break;
            left -= all;
        }
    }
    row_sync<C>();
    return sh.ti;
}

// Cuts what is kept to the shortest run of the ranking that reaches `target` entries
// (MASS false) or the share `share` of the weight kept before; then `target` is the weight
// that it has to reach. [a, b]: the range that the end of the run lies in, smaller in every
// round; MOST bounds the rounds all the same. Returns the entries that it put into the list, if
// all that is kept is there, else 0.
template <bool MASS, typename E, int C>
__device__ int cut(Shared &sh, Row<E, C> &row, u64 &target, float share)
{
    const int tid = threadIdx.x, rank = rank_of<C>();
    float a = fmaxf(row.tau, fmaxf(row.floor, -FLT_MAX)), b = row.top;   // (at the floor and below nothing weighs anything)
    u64 above = 0;                                         // what lies above b
    const bool all_in = row.tau == NEG_INF;
    // an entry this light is not in the run: all that are make up less than half of 1 - share
    const u64 light = MASS ? (u64)(0.5 * (1.0 - (double)share) / row.end * (double)(1ull << row.bits)) : 0;
    constexpr int MOST = 100;
    for (int round = 0; round < MOST; ++round) {
        // bins of equal width from b down; halves, so that no difference overflows
        const float width = 0.5f * b - 0.5f * a, scale = BINS / width;
        const bool fine = width >= 1e-34f;                 // (scale is finite)
        const double scale2 = BINS / ((double)b - (double)a);
        auto bin_of = [&](float v) {
            const float f = fine ? (0.5f * b - 0.5f * v) * scale : (float)(((double)b - (double)v) * scale2);
            return a == b ? 0 : min(BINS - 1, (int)f);
        };
        for (int i = tid; i < BINS; i += THREADS) {
            sh.counts[i] = 0;
            if (MASS) sh.bins[i] = 0, sh.limb2[i] = 0;
        }
        if (tid == 0) sh.listed = 0;
        __syncthreads();
        u64 beside = 0;                                    // kept and not in a bin, in the first round
        row.each([&](float v, int i) {
            if (!(v >= a && v <= b) || !(all_in || row.kept(v, i))) return;
            if constexpr (MASS) {
                const u64 w = row.weight(v);
                if (w <= light) {
                    beside += w;
                } else {
                    const int k = bin_of(v);
                    row.add(sh, k, w);
                }
            } else {
                atomicAdd(&sh.counts[bin_of(v)], 1u);
            }
        });
        if (MASS && round == 0) row_sums<C>(sh, beside);
        else row_sync<C>();
        u64 mine[PER], sum = 0, all;
        unsigned counts[PER];
        if constexpr (C > 1) {
            // The whole row's bins: of two CTAs each adds up all, of more each its part and then takes the
            // others' parts. (In parts: 77 x 50021 by two, p = 0.9, 80 us for 77; 1 x 32768 by eight, 33 for 37.)
            constexpr bool SHARED = C > 2;
            constexpr int PART = SHARED ? BINS / C : BINS;
            const int first = SHARED ? rank * PART : 0;
            for (int i = first + tid; i < first + PART; i += THREADS) {
                unsigned n = 0;
                u64 w = 0;
#pragma unroll
                for (int r = 0; r < C; ++r) {
                    n += of_rank<C>(sh.counts, r)[i];
                    if (MASS) w += row.weight_of(*of_rank<C>(&sh, r), i);
                }
                sh.row_counts[i] = n;
                if (MASS) sh.row_bins[i] = w;
            }
            if (SHARED) row_sync<C>();
#pragma unroll
            for (int q = 0; q < PER; ++q) {
                const int i = tid + q * THREADS, r = i / PART;
                if (!SHARED || r == rank) continue;
                sh.row_counts[i] = of_rank<C>(sh.row_counts, r)[i];
                if (MASS) sh.row_bins[i] = of_rank<C>(sh.row_bins, r)[i];
            }
            __syncthreads();
        }
        // each thread's bins, then where the sum reaches the target
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            counts[q] = C > 1 ? sh.row_counts[tid * PER + q] : sh.counts[tid * PER + q];
            mine[q] = !MASS ? counts[q] : C > 1 ? sh.row_bins[tid * PER + q] : row.weight_of(sh, tid * PER + q);
            sum += mine[q];
        }
        u64 upto = block_before(sh, sum, all);
        if (MASS && round == 0) {
            u64 kept = all;
            for (int w = 0; w < C * NW; ++w) kept += sh.all_sum[w];
            target = share_of(share, kept);
        }
        if (above + all < target) {                        // all of the range is kept, and more is not there
            row_sync<C>();
            break;
        }
        u64 dummy;
        unsigned entries = (unsigned)block_before(sh, (u64)counts[0] + counts[1] + counts[2] + counts[3], dummy);
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const u64 lo = above + upto;
            upto += mine[q];
            entries += counts[q];
            if (lo < target && above + upto >= target) sh.bin = tid * PER + q, sh.before = lo, sh.entries = entries;
        }
        row_sync<C>();                                     // bins read, the bin known
        const int bin = sh.bin;
        const u64 before = sh.before;
        const bool whole = round == 0 && sh.entries <= CAP;          // all that is kept fits the list
        float lo = -NEG_INF, hi = NEG_INF;
        row.each([&](float v, int i) {
            if (!(v >= a && v <= b) || !(all_in || row.kept(v, i))) return;
            const int k = bin_of(v);
            if (whole ? k > bin : k != bin) return;
            if (MASS && row.weight(v) <= light) return;    // (not in the bins either)
            lo = fminf(lo, v), hi = fmaxf(hi, v);
            to_list(sh, v, i);
        });
        if (!whole) {
            lo = row_fold<C>(sh.warp_lo, lo, [](float x, float y) { return fminf(x, y); });
            hi = row_fold<C>(sh.warp_hi, hi, [](float x, float y) { return fmaxf(x, y); });
        }
        const int n = join_lists<C>(sh);
        if (whole) return min(n, CAP);
        if (lo == hi) {
            const u64 each = MASS ? row.weight(lo) : 1ull;
            const u64 need = (target - before + each - 1) / each;
            if (need < (u64)n) {
                row.ti = nth_equal(sh, row, lo, (int)need);
            } else {
                if (lo != row.tau) row.ti = EVERY;
                row_sync<C>();
            }
            row.tau = lo;
            return 0;
        }
        if (n <= CAP) {
            if (rank == 0) {
                sort_list(sh.list, n);
                const int i = reached(sh, n, target - before,
                                      [&](int q) { return MASS ? row.weight(ranked_value(sh.list[q])) : 1ull; });
                if (tid == 0) sh.tau_key = (int)key_of(ranked_value(sh.list[i])), sh.ti = (int)(uint32_t)sh.list[i];
            }
            row_sync<C>();
            row.tau = of_key((uint32_t)of_rank<C>(&sh, 0)->tau_key);
            row.ti = of_rank<C>(&sh, 0)->ti;
            row_sync<C>();
            return 0;
        }
        a = lo, b = hi, above = before;
        row_sync<C>();
    }
    return 0;                                              // nothing to cut: what is below the range weighs nothing
}

// Where the sums of value(place) over the counted values reach `target`: the place (sh.bin), the sum
// before it (sh.before); false if they do not. All CTAs of the row hold the same.
template <typename F>
__device__ bool value_reached(Shared &sh, u64 target, F value)
{
    u64 v[PER_VALUE], sum = 0, all;
#pragma unroll
    for (int q = 0; q < PER_VALUE; ++q) {
        const int i = threadIdx.x * PER_VALUE + q;
        v[q] = i < VALUES ? value(i) : 0;
        sum += v[q];
    }
    u64 upto = block_before(sh, sum, all);
#pragma unroll
    for (int q = 0; q < PER_VALUE; ++q) {
        const u64 lo = upto;
        upto += v[q];
        if (lo < target && upto >= target) sh.bin = threadIdx.x * PER_VALUE + q, sh.before = lo;
    }
    __syncthreads();
    return all >= target;
}

// Weights by value (sh.table) and what the row keeps, from the counts of its values (sh.found of
// this CTA's part, sh.others). False where a cut falls into a gap.
template <typename E, int C>
__device__ bool cut_counted(Shared &sh, Row<E, C> &row, long long k, float top_p, u64 least)
{
    const int tid = threadIdx.x;
    for (int i = tid; i < VALUES; i += THREADS) sh.table[slot_at(i)] = is_gap(i) ? 0 : row.weight(value_at(i));
    __syncthreads();
    for (int i = tid; i < sh.others_count; i += THREADS) {
        const int slot = gap_slot(__float_as_uint(sh.others[i]) >> 16);
        atomicAdd(&sh.table[slot], row.weight(sh.others[i]));
        atomicAdd(&sh.found[slot], 1u);
    }
    row_sync<C>();
    if constexpr (C > 1) {
        // the whole row's, into registers, then back
        unsigned n[PER_VALUE];
        u64 gap = 0;
#pragma unroll
        for (int q = 0; q < PER_VALUE; ++q) {
            const int i = tid + q * THREADS;
            n[q] = 0;
            if (i < VALUES)
                for (int r = 0; r < C; ++r) n[q] += of_rank<C>(sh.found, r)[i];
        }
        if (tid < VALUES - 2 * CORE - 1)
            for (int r = 0; r < C; ++r) gap += of_rank<C>(sh.table, r)[2 * CORE + 1 + tid];
        row_sync<C>();
#pragma unroll
        for (int q = 0; q < PER_VALUE; ++q)
            if (tid + q * THREADS < VALUES) sh.found[tid + q * THREADS] = n[q];
        if (tid < VALUES - 2 * CORE - 1) sh.table[2 * CORE + 1 + tid] = gap;
        __syncthreads();
    }
    int last = VALUES - 1;                                 // the last place that is kept, and how many of it
    unsigned of_last = sh.found[slot_at(last)];
    auto kept_of = [&](int i) -> u64 { return i < last ? sh.found[slot_at(i)] : i == last ? of_last : 0; };
    // the run ends in place sh.bin with `need` of its entries
    auto end_at = [&](u64 need) {
        if (is_gap(sh.bin) && need < kept_of(sh.bin)) return false;
        of_last = (unsigned)min(need, kept_of(sh.bin));
        last = sh.bin;
        return true;
    };
    if (k > 0 && k < row.end - row.off && value_reached(sh, (u64)k, [&](int i) { return (u64)sh.found[slot_at(i)]; }))
        if (!end_at((u64)k - sh.before)) return false;
    if (top_p < 1.f) {
        auto weight = [&](int i) -> u64 {
            const u64 n = kept_of(i);
            return n ? (is_gap(i) ? 1 : n) * sh.table[slot_at(i)] : 0;
        };
        u64 mine = 0, all;
        for (int i = tid; i < VALUES; i += THREADS) mine += weight(i);
        block_before(sh, mine, all);
        const u64 target = share_of(top_p, all);
        if (value_reached(sh, target, weight)) {
            if (is_gap(sh.bin)) return false;
            const u64 each = sh.table[slot_at(sh.bin)];
            end_at((target - sh.before + each - 1) / each);
        }
    }
    if (is_gap(last) && last != VALUES - 1) return false;  // a gap's smallest is wanted
    if (last != VALUES - 1) {
        const unsigned there = sh.found[slot_at(last)];
        row.tau = value_at(last), row.ti = EVERY;
        if (of_last < there) {
            Row<E, C> whole = row;
            whole.tau = NEG_INF;
            row.ti = nth_equal(sh, whole, row.tau, (int)of_last);
        }
    }
    __syncthreads();
    // the table for the draw: 0 for what is not kept (of the last value, beyond ti, the draw sees to it)
    for (int i = tid; i < VALUES; i += THREADS) {
        const int slot = slot_at(i);
        if (i > last || (!is_gap(i) && sh.table[slot] < least)) sh.table[slot] = 0;
    }
    __syncthreads();
    return true;
}

// The rest of a row whose candidates are all in sh.list: n entries, of which the k first in rank count,
// and of those the ones that reach `target`, or (0) the share top_p of their weight.
template <typename E, int C>
__device__ void finish_list(Shared &sh, const Row<E, C> &row, const SampleArgs &s, int at, int n, int k, float top_p,
                            u64 target, u64 least)
{
    const int tid = threadIdx.x;
    sort_list(sh.list, n);
    n = min(n, k);
    // the cuts are prefixes of the sorted list
    u64 sum = 0, all;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
        const int i = tid + q * THREADS;
        if (i < n) {
            const u64 w = row.weight(ranked_value(sh.list[i]));
            sh.bins[i] = w;
            sum += w;
        }
    }
    block_before(sh, sum, all);                            // (two barriers: sh.bins is written)
    if (top_p < 1.f) n = reached(sh, n, target ? target : share_of(top_p, all), [&](int i) { return sh.bins[i]; }) + 1;
    __syncthreads();
    // by index: (index, key), the ones too light last
#pragma unroll
    for (int q = 0; q < PER; ++q) {
        const int i = tid + q * THREADS;
        if (i < n) {
            const u64 e = sh.list[i];
            sh.list[i] = sh.bins[i] >= least ? (e & 0xffffffffull) << 32 | (uint32_t)~(uint32_t)(e >> 32) : ~0ull;
        }
    }
    sort_list(sh.list, n);
    auto weight_at = [&](int i) { return sh.list[i] == ~0ull ? 0ull : row.weight(of_key((uint32_t)sh.list[i])); };
    sum = 0;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
        const int i = tid + q * THREADS;
        if (i < n) {
            const u64 w = weight_at(i);
            sh.bins[i] = w;
            sum += w;
        }
    }
    block_before(sh, sum, all);
    const int i = reached(sh, n, border_of(s.uniform[at], all) + 1, [&](int q) { return sh.bins[q]; });
    if (tid == 0) {
        const u64 e = sh.list[i];
        s.token[at] = (int64_t)(e >> 32);
        if (s.logprob)
            s.logprob[at] = (float)(row.exponent(of_key((uint32_t)e)) - log(ldexp((double)all, -row.bits)));
    }
}

template <typename E, int C>
__global__ void __launch_bounds__(THREADS, C > 2 ? 1 : 2)
sample_kernel(const __grid_constant__ SampleArgs s)
{
    extern __shared__ __align__(16) unsigned char memory[];
    Shared &sh = *reinterpret_cast<Shared *>(memory);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = rank_of<C>(), at = blockIdx.x / C;
    Row<E, C> row;
    constexpr int VEC = Row<E, C>::VEC, STEP = Row<E, C>::STEP;
    const E *start = reinterpret_cast<const E *>(s.logits) + at * s.ld;
    row.off = (int)((reinterpret_cast<uintptr_t>(start) & 15) / sizeof(E));
    row.p = start - row.off;
    row.end = s.vocab + row.off;
    row.piece = ((row.end + C * NW - 1) / (C * NW) + STEP - 1) / STEP * STEP;
    row.powers = sh.powers;
    row.bits = min(BITS, 62 - (32 - __clz(s.vocab - 1)));
    row.tau = NEG_INF, row.ti = EVERY;
    const int w = rank * NW + warp;
    if (tid < 16) sh.powers[tid] = exp2(tid / 16.0);
    if (tid == 0) sh.listed = 0, sh.least = EVERY, sh.others_count = 0;
    const float t = s.temperature ? s.temperature[at] : s.temperature1;
    const long long k = s.top_k.p ? s.top_k.at(at) : s.top_k1;
    const float top_p = s.top_p ? s.top_p[at] : s.top_p1;
    const float share = s.min_p ? s.min_p[at] : s.min_p1, min_p = fminf(share, 1.f);
    // k entries at least are as large as the m-th largest of the warps' j-th largest of their lanes'
    // maxima, m j >= k; with j from the pieces that are whole there are m warps
    const int pieces = max(1, row.end / row.piece);
    const int j = (int)min((k + pieces - 1) / pieces, 1000ll);
    const bool listed = k > 1 && k < s.vocab && j <= 16;
    constexpr bool MAY_COUNT = sizeof(E) == 2 && C <= 2;
    bool counted = MAY_COUNT && ((k > 0 && k < s.vocab) || top_p < 1.f) && !listed && k != 1 && t > 0.f && top_p > 0.f;
    if (counted)
        for (int i = tid; i < VALUES; i += THREADS) sh.found[i] = 0;
    __syncthreads();
    // the largest value (NaN if there is one)
    float most = NEG_INF;
    if (counted) {
        row.template words<1>(row.from(w), row.from(w + 1), [&](const Words<E> &v, int) {
            most = max_nan(most, v.most());
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const uint32_t b = __float_as_uint(v.at(i)) >> 16;
                const int slot = value_slot(b);
                if (slot >= 0) atomicAdd(&sh.found[slot], 1u);
                if (slot < 0 && b != 0xff80u) {
                    const int to = atomicAdd(&sh.others_count, 1);
                    if (to < CAP) sh.others[to] = v.at(i);
                }
            }
        });
    } else {
        row.template words<4>(row.from(w), row.from(w + 1), [&](const Words<E> &v, int) { most = max_nan(most, v.most()); });
    }
    if (listed) {
        uint32_t mine = most == most ? key_of(most) : 0, best = 0;
        for (int q = 0; q < j; ++q) {
            best = __reduce_max_sync(0xffffffffu, mine);
            const unsigned has = __ballot_sync(0xffffffffu, mine == best);
            if (lane == __ffs(has) - 1) mine = 0;
        }
        if (lane == 0) sh.warp_pivot[warp] = best ? of_key(best) : NEG_INF;
    }
    row.top = row_fold<C>(sh.warp_max, most, [](float x, float y) { return max_nan(x, y); });
    row.rate = 1.0 / (double)t;
    row.limit = (double)fminf(row.top, FLT_MAX);
    // (beside +inf not even FLT_MAX, as which an infinite logit is computed, has weight)
    row.floor = isinf(row.top) ? FLT_MAX
                               : fminf(below(row.top), __double2float_rd(row.limit - 34.0 * (double)t));
    // nothing to draw from, or nothing to draw
    const bool none = !(row.top > NEG_INF) || t != t || top_p != top_p || share != share;
    if (none || t <= 0.f || k == 1 || top_p <= 0.f) {
        int first = EVERY;
        if (!none)
            row.each([&](float v, int i) {
                if (v == row.top) first = min(first, i);
            });
        first = __reduce_min_sync(0xffffffffu, first);
        if (lane == 0) atomicMin(&of_rank<C>(&sh, 0)->least, first);
        row_sync<C>();
        if (rank == 0 && tid == 0) {
            s.token[at] = none ? -1 : sh.least;
            if (s.logprob) s.logprob[at] = none ? __int_as_float(0x7fc00000) : 0.f;
        }
        return;
    }
    const u64 least = min_p > 0.f ? (u64)ceil(ldexp((double)min_p, row.bits)) : 0;
    if (listed) {
        const int m = ((int)k + j - 1) / j;
        if (tid < C * NW) sh.all_pivot[tid] = of_rank<C>(sh.warp_pivot, tid / NW)[tid % NW];
        __syncthreads();
        if (tid < C * NW) {
            const float mine = sh.all_pivot[tid];
            int above = 0;
#pragma unroll 8
            for (int q = 0; q < C * NW; ++q) above += sh.all_pivot[q] > mine || (sh.all_pivot[q] == mine && q < tid);
            if (above == m - 1) sh.pivot = mine;
        }
        __syncthreads();
        const float pivot = sh.pivot;
        row.each([&](float v, int i) {
            if (v >= pivot) to_list(sh, v, i);
        });
        const int n = join_lists<C>(sh);
        if (n <= CAP) {
            if (rank == 0) finish_list(sh, row, s, at, n, (int)k, top_p, 0, least);
            return;
        }
    }
    if constexpr (MAY_COUNT) {
        for (int r = 0; r < C; ++r) counted = counted && *of_rank<C>(&sh.others_count, r) <= CAP;
        counted = counted && !isinf(row.top) && cut_counted(sh, row, k, top_p, least);
    }
    if (!counted) {
        row_sync<C>();                                     // what was counted gives way to bins
        row.tau = isinf(row.top) ? row.top : NEG_INF;      // (nothing beside it has weight)
        u64 target = (u64)k;
        int in_list = k > 0 && k < s.vocab ? cut<false>(sh, row, target, 0.f) : 0;
        const bool few = in_list > 0;
        if (!few && top_p < 1.f) in_list = cut<true>(sh, row, target, top_p);
        if (in_list > 0) {
            if (rank == 0) finish_list(sh, row, s, at, in_list, few ? (int)k : in_list, top_p, few ? 0 : target, least);
            return;
        }
    }
    auto weight = [&](float v, int i) -> u64 {
        if (counted) {
            const int slot = value_slot(__float_as_uint(v) >> 16);
            if (slot >= 0) return v == row.tau && i > row.ti ? 0 : sh.table[slot];
        }
        if (!row.kept(v, i)) return 0;
        const u64 x = row.weight(v);
        return x >= least ? x : 0;
    };
    u64 mass = 0;
    if (counted) {
        const bool part = row.ti != EVERY;                 // of the entries equal to tau
        row.template words<1>(row.from(w), row.from(w + 1), [&](const Words<E> &v, int place) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float x = v.at(i);
                const int slot = value_slot(__float_as_uint(x) >> 16);
                if (slot >= 0) mass += sh.table[slot];
                if (slot < 0 && x > NEG_INF) mass += weight(x, place + i - row.off);
                if (part && x == row.tau && place + i - row.off > row.ti) mass -= sh.table[slot];
            }
        });
    } else if (row.tau == NEG_INF) {
        row.each([&](float v, int i) { mass += weight(v, i); });
    } else {
        // few of the entries are kept: their weights are computed 32 at a time
        float *queue = sh.queue[warp];
        int waiting = 0;
        auto heavy = [&](float v) {
            const u64 x = row.weight(v);
            return x >= least ? x : 0;
        };
        row.template words<1>(row.from(w), row.from(w + 1), [&](const Words<E> &v, int place) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float x = v.at(i);
                const bool in = row.kept(x, place + i - row.off);
                const unsigned who = __ballot_sync(0xffffffffu, in);
                if (in) queue[waiting + __popc(who & ((1u << lane) - 1))] = x;
                waiting += __popc(who);
                if (waiting >= 32) {
                    __syncwarp();
                    mass += heavy(queue[lane]);
                    const float rest = queue[32 + lane];
                    __syncwarp();
                    waiting -= 32;
                    if (lane < waiting) queue[lane] = rest;          // (the places behind are the next entries')
                }
            }
        });
        __syncwarp();
        if (lane < waiting) mass += heavy(queue[lane]);
    }
    row_sums<C>(sh, mass);
    u64 all = 0;
    for (int i = 0; i < C * NW; ++i) all += sh.all_sum[i];
    const u64 border = border_of(s.uniform[at], all);
    // the piece, the part of it, then the entry, that pass the border
    int hit = 0;
    u64 base = 0;
    while (hit < C * NW - 1 && base + sh.all_sum[hit] <= border) base += sh.all_sum[hit++];
    if (hit / NW == rank) {
        const int a = row.from(hit), b = row.from(hit + 1);
        const int part = ((b - a + NW - 1) / NW + STEP - 1) / STEP * STEP;
        auto part_from = [&](int q) { return min(a + q * part, b); };
        mass = 0;
        row.each(part_from(warp), part_from(warp + 1), [&](float v, int i) { mass += weight(v, i); });
        mass = warp_sum(mass);
        if (lane == 0) sh.scan[warp] = mass;
        __syncthreads();
        int q = 0;
        while (q < NW - 1 && base + sh.scan[q] <= border) base += sh.scan[q++];
        if (q == warp) {
            for (int x = part_from(q); x < part_from(q + 1); x += STEP) {
                const Words<E> v = row.read(x + lane * VEC);
                u64 ws[VEC], sum = 0;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    ws[i] = v.at(i) > NEG_INF ? weight(v.at(i), x + lane * VEC + i - row.off) : 0;
                    sum += ws[i];
                }
                const u64 incl = warp_scan(sum);
                u64 run = base + incl - sum;
                if (run <= border && run + sum > border) {
                    bool done = false;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        run += ws[i];
                        if (!done && run > border) {
                            done = true;
                            s.token[at] = x + lane * VEC + i - row.off;
                            if (s.logprob)
                                s.logprob[at] = (float)(row.exponent(v.at(i)) - log(ldexp((double)all, -row.bits)));
                        }
                    }
                }
                base += __shfl_sync(0xffffffffu, incl, 31);
                if (base > border) break;
            }
        }
    }
}

template <typename E, int C>
cudaError_t sample_of(const SampleArgs &a, cudaStream_t stream)
{
    const cudaError_t e = smem_opt_in<sample_kernel<E, C>>(sizeof(Shared));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t c{};
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = C, cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    c.gridDim = dim3((unsigned)((long long)a.rows * C));
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = sizeof(Shared);
    c.stream = stream;
    c.attrs = &cluster;
    c.numAttrs = C > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&c, sample_kernel<E, C>, a);
}

// CTAs a row: as many (up to 8, a portable cluster) as the GPU holds, 2 an SM or, of larger
// clusters, whose joins need more registers, one; none of fewer than 2048 entries.
template <typename E>
cudaError_t sample_by_rows(const SampleArgs &a, cudaStream_t stream)
{
    const long long most = std::min<long long>(N_SM / a.rows, a.vocab / 2048);
    if (most >= 8) return sample_of<E, 8>(a, stream);
    if (most >= 4) return sample_of<E, 4>(a, stream);
    if (2LL * N_SM / a.rows >= 2 && a.vocab >= 4096) return sample_of<E, 2>(a, stream);
    return sample_of<E, 1>(a, stream);
}

}  // namespace

cudaError_t launch_sample(const SampleArgs &a, cudaStream_t stream)
{
    return a.bf16 ? sample_by_rows<__nv_bfloat16>(a, stream) : sample_by_rows<float>(a, stream);
}

}  // namespace mms
