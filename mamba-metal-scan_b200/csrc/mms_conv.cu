// Short depthwise causal convolution with SiLU for sm_100a, forward, backward
// and over packed sequences with their last inputs kept in a cache.
//
//     pre[t, d] = bias[d] + sum_k w[d, k] x[t - K + 1 + k, d]      y = pre * sigmoid(pre), or pre
//     ds = dy * act'(pre),   dx[t] = sum_k w[k] ds[t + K - 1 - k],
//     dw[k] = sum_t ds[t] x[t - K + 1 + k],   dbias = sum_t ds[t]
//
// A few FMAs an element beside x and y (forward, 2 elements moved), x, dy and dx (backward, 3), and with
// SiLU two MUFU operations. Of 4 x 4096 x 8192 (floor at HBM's rate in brackets): float32 is bound by HBM,
// forward 172 us (167), backward 266 (250); bf16 not, forward 94 (83): MUFU at 68 %, backward 172 (125):
// instructions, the FMA pipe at 52 % with the three CTAs an SM that 168 registers leave. The reference transposes to
// channels first, calls a convolution and a SiLU and transposes back (reference
// mamba_metal/model.py:175-177, 214-219); here rows stay as they are in memory,
// channels innermost: a thread owns VEC neighbouring channels, a warp 32 * VEC,
// so that every access is a whole line, and x may be a view with strides (a half
// of in_proj's output).
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "mms_common.cuh"
#include "mms_serve.h"

namespace mms {

namespace {

constexpr int WARPS = 4;                // per CTA, each with rows of its own and the same channels
constexpr int THREADS = 32 * WARPS;
// Rows of packed sequences a warp walks. (With 16, 32 and 64, us: 37 prompts, 8192 x 2304, float32 33.6, 31.4, 31.1,
// bf16 28.8, 26.3, 26.8, 1319 CTAs of 32 rows where 740 run at a time; 9 prompts, 2048 x 1432, float32 8.2, 10.4, 15.7;
// 37 prompts, 32768 x 2304, float32 112, 104, 107.)
constexpr int TAIL_ROWS = 32;
// Rows that a warp loads at once, and computes while the next are on their way: 64 bytes a lane and
// array. (Backward with half of them at 4 CTAs an SM: 201 us of 4 x 4096 x 8192 in bf16, so 174;
// a quarter, 228; a forward that loads a tile and then computes it, 177, so 91.)
template <typename E>
constexpr int FWD_STEP = sizeof(E) == 4 ? 4 : 8;
template <typename E>
constexpr int BWD_STEP = sizeof(E) == 4 ? 4 : 8;

// VEC neighbouring channels of a row as they are stored, and as NP pairs of floats (one
// channel alone: the second of its pair is 0).
template <int VEC>
constexpr int NP = (VEC + 1) / 2;

template <typename E, int VEC>
struct Pack {
    static constexpr int WORDS = VEC == 1 ? 1 : VEC * (int)sizeof(E) / 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ float2 pair(int p) const {
        if constexpr (sizeof(E) == 4) return VEC == 1 ? f2(__uint_as_float(w[0]), 0.f)
                                                      : f2(__uint_as_float(w[2 * p % WORDS]), __uint_as_float(w[(2 * p + 1) % WORDS]));
        else return f2(__uint_as_float(w[p] << 16), VEC == 1 ? 0.f : __uint_as_float(w[p] & 0xffff0000u));
    }
};

template <typename E, int VEC>
__device__ __forceinline__ Pack<E, VEC> nothing() {
    Pack<E, VEC> o;
#pragma unroll
    for (int i = 0; i < o.WORDS; ++i) o.w[i] = 0;
    return o;
}
template <typename E, int VEC>
__device__ __forceinline__ Pack<E, VEC> load(const E *p) {
    Pack<E, VEC> o;
    if constexpr (VEC == 1 && sizeof(E) == 2) o.w[0] = *reinterpret_cast<const uint16_t *>(p);
    else if constexpr (VEC == 1) o.w[0] = *reinterpret_cast<const uint32_t *>(p);
    else if constexpr (sizeof(E) == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        o.w[0] = v.x, o.w[1] = v.y;
    } else {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        o.w[0] = v.x, o.w[1] = v.y, o.w[2] = v.z, o.w[3] = v.w;
    }
    return o;
}
template <typename E, int VEC>
__device__ __forceinline__ void store(E *p, const float2 (&v)[NP<VEC>]) {
    if constexpr (VEC == 1) {
        *p = from_f<E>(v[0].x);
    } else if constexpr (sizeof(E) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    } else {
        const __nv_bfloat162 a = __float22bfloat162_rn(v[0]), b = __float22bfloat162_rn(v[1]);
        *reinterpret_cast<uint2 *>(p) = make_uint2(reinterpret_cast<const uint32_t &>(a), reinterpret_cast<const uint32_t &>(b));
    }
}

// sigmoid(v) = 1 / (1 + e^-v) on MUFU's ex2 and reciprocal
__device__ __forceinline__ float2 sigmoid2(float2 v) {
    const float2 d = add2(ex2x2(mul2(v, f2(-MMS_LOG2E, -MMS_LOG2E))), f2(1.f, 1.f));
    float2 r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(d.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(d.y));
    return r;
}
__device__ __forceinline__ float2 act(float2 v, bool silu) { return silu ? mul2(v, sigmoid2(v)) : v; }

// A channel group's taps. KT: taps the code is unrolled for; with fewer of them
// (K < KT) the first KT - K stand for none and are skipped, not multiplied by zero:
// an infinite input there must not turn into a NaN.
template <typename E, int KT, int VEC>
struct Taps {
    float2 w[KT][NP<VEC>], bias[NP<VEC>];
    __device__ __forceinline__ void read(const E *wp, const E *bp, int d, int K) {
#pragma unroll
        for (int p = 0; p < NP<VEC>; ++p) {
            const int c0 = d + 2 * p, c1 = VEC == 1 ? c0 : c0 + 1;
            bias[p] = bp ? f2(to_f(bp[c0]), to_f(bp[c1])) : f2(0.f, 0.f);
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                const int kk = k - (KT - K);
                w[k][p] = kk >= 0 ? f2(to_f(wp[(long long)c0 * K + kk]), to_f(wp[(long long)c1 * K + kk])) : f2(0.f, 0.f);
            }
        }
    }
    // the sum over rows x[0 .. KT - 1]
    template <typename Row>
    __device__ __forceinline__ void sum(float2 (&acc)[NP<VEC>], int K, Row row) const {
#pragma unroll
        for (int p = 0; p < NP<VEC>; ++p) acc[p] = bias[p];
#pragma unroll
        for (int k = 0; k < KT; ++k)
            if (k >= KT - K) {
#pragma unroll
                for (int p = 0; p < NP<VEC>; ++p) acc[p] = fma2(w[k][p], row(k, p), acc[p]);
            }
    }
};

// K as the code knows it: KT itself where the kernel is for exactly KT taps.
template <int KT, bool EXACT>
__device__ __forceinline__ int taps_of(int K) { return EXACT ? KT : K; }

// ---------------------------------------------------------------- forward

// The rows [t0, t1) from xp, row t0; `above`: how many rows before t0 there are (zeros above them).
// out(t, sums) takes each row's sum of taps.
template <typename E, int KT, int VEC, typename Out>
__device__ __forceinline__ void walk(const E *xp, long long ldt, int t0, int t1, int above, int K,
                                     const Taps<E, KT, VEC> &taps, Out out)
{
    constexpr int STEP = FWD_STEP<E>;
    Pack<E, VEC> xs[STEP + KT - 1], next[STEP];            // rows t - KT + 1 .. t + STEP - 1, the STEP behind them
    auto rows_in = [&](int t) {
        if (t + STEP <= t1) {
#pragma unroll
            for (int u = 0; u < STEP; ++u) {
                next[u] = load<E, VEC>(xp);
                xp += ldt;
            }
        } else {
#pragma unroll
            for (int u = 0; u < STEP; ++u) {
                next[u] = t + u < t1 ? load<E, VEC>(xp) : nothing<E, VEC>();
                xp += ldt;
            }
        }
    };
#pragma unroll
    for (int j = 0; j < KT - 1; ++j) {
        const int back = KT - 1 - j;
        xs[j] = back <= above ? load<E, VEC>(xp - back * ldt) : nothing<E, VEC>();
    }
    rows_in(t0);
    for (int t = t0; t < t1; t += STEP) {
#pragma unroll
        for (int u = 0; u < STEP; ++u) xs[KT - 1 + u] = next[u];
        rows_in(t + STEP);
#pragma unroll
        for (int u = 0; u < STEP; ++u) {
            float2 acc[NP<VEC>];
            taps.sum(acc, K, [&](int k, int p) { return xs[u + k].pair(p); });
            out(t + u, acc);
        }
#pragma unroll
        for (int j = 0; j < KT - 1; ++j) xs[j] = xs[j + STEP];
    }
}

template <typename E, int KT, bool EXACT, int VEC>
__global__ void __launch_bounds__(THREADS)
conv_fwd_kernel(const E *__restrict__ x, long long ldb, long long ldt, const E *__restrict__ w,
                const E *__restrict__ bias, E *__restrict__ y, int T, int D, int K_in, bool silu, int nd, int segs,
                int len, long long units)
{
    const int K = taps_of<KT, EXACT>(K_in);
    const long long unit = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5);   // (b, segment, channel block)
    if (unit >= units) return;
    const int d = (int)(unit % nd) * 32 * VEC + (threadIdx.x & 31) * VEC;
    const int seg = (int)(unit / nd % segs), b = (int)(unit / nd / segs);
    const int t0 = seg * len, t1 = min(T, t0 + len);
    if (d >= D) return;
    Taps<E, KT, VEC> taps;
    taps.read(w, bias, d, K);
    E *yp = y + ((long long)b * T + t0) * D + d;
    walk<E, KT, VEC>(x + b * ldb + t0 * ldt + d, ldt, t0, t1, t0, K, taps, [&](int t, float2 (&acc)[NP<VEC>]) {
#pragma unroll
        for (int p = 0; p < NP<VEC>; ++p) acc[p] = act(acc[p], silu);
        if (t < t1) store<E, VEC>(yp, acc);
        yp += D;
    });
}

// --------------------------------------------------------------- backward

// A warp walks `len` rows of one sequence, ds rolling through registers: after
// ds[t] the row dx[t - KT + 1] is complete. The KT - 1 rows behind its own are
// computed as well, for dx alone. dw and dbias stay in registers; the CTA's four
// warps are joined in shared memory and leave one partial sum a CTA.
template <typename E, int KT, bool EXACT, int VEC>
__global__ void __launch_bounds__(THREADS, KT <= 4 ? 3 : 2)
conv_bwd_kernel(const E *__restrict__ x, long long ldb, long long ldt, const E *__restrict__ w,
                const E *__restrict__ bias, const E *__restrict__ dy, E *__restrict__ dx,
                float *__restrict__ part, int T, int D, int K_in, bool silu, int nd, int segs, int len, long long rows)
{
    constexpr int P = NP<VEC>, STEP = BWD_STEP<E>;
    const int K = taps_of<KT, EXACT>(K_in);
    __shared__ float2 sums[WARPS][KT + 1][P][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int d = (blockIdx.x % nd) * 32 * VEC + lane * VEC;
    const long long row = (long long)(blockIdx.x / nd) * WARPS + warp;     // (b, segment)
    const int seg = (int)(row % segs), b = (int)(row / segs);
    const int t0 = seg * len, t1 = min(T, t0 + len);
    float2 dw[KT][P], db[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        db[p] = f2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < KT; ++k) dw[k][p] = f2(0.f, 0.f);
    }
    if (d < D && row < rows) {
        const E *xp = x + b * ldb + d + t0 * ldt;          // row t
        const E *gp = dy + ((long long)b * T + t0) * D + d;
        E *op = dx + ((long long)b * T + t0 - (KT - 1)) * D + d;  // row t - KT + 1
        Taps<E, KT, VEC> taps;
        taps.read(w, bias, d, K);
        Pack<E, VEC> xs[STEP + KT - 1], xn[STEP], gn[STEP];       // rows t - KT + 1 .. t + STEP - 1, the next
        float2 ds[STEP + KT - 1][P];
        const int end = min(T, t1 + KT - 1);               // rows that are read
        auto rows_in = [&](int t) {
            if (t + STEP <= end) {
#pragma unroll
                for (int u = 0; u < STEP; ++u) {
                    xn[u] = load<E, VEC>(xp), gn[u] = load<E, VEC>(gp);
                    xp += ldt, gp += D;
                }
            } else {
#pragma unroll
                for (int u = 0; u < STEP; ++u) {
                    const bool in = t + u < end;
                    xn[u] = in ? load<E, VEC>(xp) : nothing<E, VEC>();
                    gn[u] = in ? load<E, VEC>(gp) : nothing<E, VEC>();
                    xp += ldt, gp += D;
                }
            }
        };
#pragma unroll
        for (int j = 0; j < KT - 1; ++j) {
            const int back = KT - 1 - j;
            xs[j] = t0 >= back ? load<E, VEC>(xp - back * ldt) : nothing<E, VEC>();
#pragma unroll
            for (int p = 0; p < P; ++p) ds[j][p] = f2(0.f, 0.f);
        }
        rows_in(t0);
        // inner: all rows of the step are the warp's own, and so are those whose dx they complete
        auto step = [&](int t, auto inner) {
            constexpr bool INNER = decltype(inner)::value;
            Pack<E, VEC> g[STEP];
#pragma unroll
            for (int u = 0; u < STEP; ++u) xs[KT - 1 + u] = xn[u], g[u] = gn[u];
            rows_in(t + STEP);
#pragma unroll
            for (int u = 0; u < STEP; ++u) {
                float2 pre[P];
                if (silu) taps.sum(pre, K, [&](int k, int p) { return xs[u + k].pair(p); });
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    float2 s = g[u].pair(p);
                    if (silu) {                            // dy sg (1 + pre (1 - sg))
                        const float2 sg = sigmoid2(pre[p]);
                        const float2 rest = fma2(sg, f2(-1.f, -1.f), f2(1.f, 1.f));
                        s = mul2(s, mul2(sg, fma2(pre[p], rest, f2(1.f, 1.f))));
                    }
                    ds[KT - 1 + u][p] = INNER || t + u < T ? s : f2(0.f, 0.f);
                }
                if (INNER || t + u < t1) {
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        db[p] = add2(db[p], ds[KT - 1 + u][p]);
#pragma unroll
                        for (int k = 0; k < KT; ++k) dw[k][p] = fma2(ds[KT - 1 + u][p], xs[u + k].pair(p), dw[k][p]);
                    }
                }
                const int to = t + u - (KT - 1);
                if (INNER || (to >= t0 && to < t1)) {
                    float2 o[P];
#pragma unroll
                    for (int p = 0; p < P; ++p) o[p] = f2(0.f, 0.f);
#pragma unroll
                    for (int k = 0; k < KT; ++k)
                        if (k >= KT - K) {
#pragma unroll
                            for (int p = 0; p < P; ++p) o[p] = fma2(taps.w[k][p], ds[KT - 1 + u - k][p], o[p]);
                        }
                    store<E, VEC>(op, o);
                }
                op += D;
            }
#pragma unroll
            for (int j = 0; j < KT - 1; ++j) {
                xs[j] = xs[j + STEP];
#pragma unroll
                for (int p = 0; p < P; ++p) ds[j][p] = ds[j + STEP][p];
            }
        };
        for (int t = t0; t < t1 + KT - 1; t += STEP) {
            if (t - (KT - 1) >= t0 && t + STEP <= t1) step(t, std::true_type{});
            else step(t, std::false_type{});
        }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int k = 0; k < KT; ++k) sums[warp][k][p][lane] = dw[k][p];
        sums[warp][KT][p][lane] = db[p];
    }
    __syncthreads();
    // part[CTA's rows][K + 1][D]
    float *pb = part + (long long)(blockIdx.x / nd) * (K + 1) * D + (blockIdx.x % nd) * 32 * VEC;
    const int left = D - (blockIdx.x % nd) * 32 * VEC;
    for (int o = threadIdx.x; o < (KT + 1) * P * 32; o += THREADS) {
        const int c = o % (P * 32), k = o / (P * 32);
        const int at = VEC == 1 ? c : 2 * c;               // its first channel in the CTA
        if (at >= left || k < KT - K) continue;
        const int p = c % P, l = c / P;
        float2 s = sums[0][k][p][l];
#pragma unroll
        for (int q = 1; q < WARPS; ++q) s = add2(s, sums[q][k][p][l]);
        float *to = pb + (long long)(k - (KT - K)) * D + at;
        to[0] = s.x;
        if (VEC > 1) to[1] = s.y;
    }
}

// dw (D, K) and dbias (D) from the partial sums, in a fixed order: row q of 8 takes
// every eighth partial sum, then the rows are joined.
template <typename E>
__global__ void __launch_bounds__(256)
conv_reduce_kernel(const float *__restrict__ part, E *__restrict__ dw, E *__restrict__ dbias, int parts, int D, int K)
{
    __shared__ float rows[8][32];
    const int c = threadIdx.x & 31, q = threadIdx.x >> 5;
    const int d = blockIdx.x * 32 + c, k = blockIdx.y;
    float s = 0.f;
    if (d < D)
        for (int p = q; p < parts; p += 8) s += part[((long long)p * (K + 1) + k) * D + d];
    rows[q][c] = s;
    __syncthreads();
    if (q == 0 && d < D) {
        for (int r = 1; r < 8; ++r) s += rows[r][c];
        if (k < K) dw[(long long)d * K + k] = from_f<E>(s);
        else if (dbias) dbias[d] = from_f<E>(s);
    }
}

// ----------------------------------------------------------------- packed

// Packed sequences in one launch of two kinds of warps that write different rows,
// so that none waits for another though the cache is updated in place:
//   heads  (sequence, channel block): the outputs that still see the old window,
//          rows 0 .. min(length, K - 1) - 1, and then the new window;
//   tails  (32 rows, channel block): the rows at place K - 1 and later of their
//          sequence, which depend on x alone; rows of no sequence get zeros.
template <typename E, int KT, bool EXACT, int VEC>
__global__ void __launch_bounds__(THREADS)
conv_packed_kernel(const E *__restrict__ x, long long ldx, const E *__restrict__ w, const E *__restrict__ bias,
                   E *__restrict__ window, E *__restrict__ y, Sequences seq, int D, int K_in, bool silu, int nd,
                   long long heads, long long units)
{
    const int K = taps_of<KT, EXACT>(K_in);
    const int lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5);
    if (unit >= units) return;
    const int d = (int)(unit % nd) * 32 * VEC + lane * VEC;
    if (unit < heads) {
        if (d >= D) return;
        const int s = (int)(unit / nd);
        const int first = seq.start(s), end = seq.starts.p ? max(first, seq.start(s + 1)) : s + 1;
        const int len = end - first, K1 = K - 1;
        const long long from = seq.from(s), to = seq.to(s);
        // rows[0 .. KT - 2] the old window (as pairs of floats), then the first inputs
        E old[KT > 1 ? KT - 1 : 1][VEC];
        float2 rows[2 * (KT - 1) + 1][NP<VEC>];
#pragma unroll
        for (int j = 0; j < KT - 1; ++j) {
            const int jw = j - (KT - K);                   // its place in the window
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                old[j][i] = from >= 0 && jw >= 0 ? window[(from * D + d + i) * K1 + jw] : from_f<E>(0.f);
            const bool in = j < len && j < K1;
            const Pack<E, VEC> v = in ? load<E, VEC>(x + (first + j) * ldx + d) : nothing<E, VEC>();
#pragma unroll
            for (int p = 0; p < NP<VEC>; ++p) {
                rows[j][p] = VEC == 1 ? f2(to_f(old[j][0]), 0.f) : f2(to_f(old[j][2 * p]), to_f(old[j][(2 * p + 1) % VEC]));
                rows[KT - 1 + j][p] = v.pair(p);
            }
        }
        if (to >= 0) {
            // the last K - 1 of the window and the inputs behind it
#pragma unroll
            for (int j = 0; j < KT - 1; ++j) {
                if (j >= K1) continue;
                const int p = len - K1 + j;                // its row; below 0: in the old window
                E v[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[i] = p >= 0 ? x[(first + p) * ldx + d + i] : from_f<E>(0.f);
#pragma unroll
                for (int q = 0; q < KT - 1; ++q) {         // (constant indices: registers)
                    const bool here = p < 0 && q - (KT - K) == p + K1;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) v[i] = here ? old[q][i] : v[i];
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) window[(to * D + d + i) * K1 + j] = v[i];
            }
        }
        Taps<E, KT, VEC> taps;
        taps.read(w, bias, d, K);
#pragma unroll
        for (int r = 0; r < KT - 1; ++r) {
            if (r >= K1 || r >= len) continue;
            float2 acc[NP<VEC>];
            taps.sum(acc, K, [&](int k, int p) { return rows[r + k][p]; });
#pragma unroll
            for (int p = 0; p < NP<VEC>; ++p) acc[p] = act(acc[p], silu);
            store<E, VEC>(y + (long long)(first + r) * D + d, acc);
        }
        return;
    }
    const int r0 = (int)((unit - heads) / nd) * TAIL_ROWS, r1 = min(seq.rows, r0 + TAIL_ROWS);
    auto start = [&](int i) { return seq.start(i); };
    const int n = seq.count + 1;
    // the sequence of the row that is next, its first row and the one behind its last
    int s = seq.starts.p ? Sequences::last_at_most(n, r0, start) : 0, first = 0, next = seq.rows;
    auto bounds = [&]() {
        first = s < 0 ? 0 : seq.start(s), next = s + 1 < n ? seq.start(s + 1) : seq.rows;
    };
    if (seq.starts.p) bounds();
    Taps<E, KT, VEC> taps;
    const bool act_lane = d < D;
    if (act_lane) taps.read(w, bias, d, K);
    E *yp = y + (long long)r0 * D + d;
    walk<E, KT, VEC>(x + r0 * ldx + (act_lane ? d : 0), ldx, r0, r1, r0, K, taps, [&](int r, float2 (&acc)[NP<VEC>]) {
        if (r < r1) {
            if (r >= next) {                               // (all lanes)
                s = Sequences::last_at_most(n, r, start);
                bounds();
            }
            const bool nobody = s < 0 || s >= seq.count;
            if (act_lane && (nobody || !seq.starts.p || r - first >= K - 1)) {
#pragma unroll
                for (int p = 0; p < NP<VEC>; ++p) acc[p] = nobody ? f2(0.f, 0.f) : act(acc[p], silu);
                store<E, VEC>(yp, acc);
            }
        }
        yp += D;
    });
}

// ------------------------------------------------------------------ launch

// 4 channels a thread where every row starts at a whole group of 4: 16 (float32) or
// 8 (bf16) bytes an access; one channel otherwise.
template <typename E>
bool groups_of_4(int D, std::initializer_list<const void *> arrays, std::initializer_list<long long> strides)
{
    bool ok = D % 4 == 0;
    for (const void *p : arrays) ok = ok && reinterpret_cast<uintptr_t>(p) % (4 * sizeof(E)) == 0;
    for (long long s : strides) ok = ok && s % 4 == 0;
    return ok;
}

// Rows a warp walks: as many as make 8 CTAs an SM, so that the halo of K - 1 rows and the
// backward's partial sums stay small beside them; at least 16, at most 128. Of those 8 the registers let 6 run at a
// time forward (80 of 4 taps) and 3 backward (168), so that 16 x 512 x 1432, 24 rows a warp, is 1.2 and 2.4
// waves. (Aiming at 4, 6, 8 and 16, us, forward and backward with its sums: that size in float32 18.7, 17.0, 19.8,
// 19.4 and 40.2, 34.4, 38.6, 39.8, in bf16 13.9, 13.9, 14.3, 14.3 and 30.5, 30.4, 34.3, 38.1; 4 x 4096 x 8192,
// bf16, 128 rows up to 8 and 112 at 16: 94 to 91 and 172, at 16 176; 2 x 2048 x 1024, 16 rows for all, 7.7 and 18.1.)
int rows_of_warp(int Bt, int T, int D)
{
    const long long nd = (D + 127) / 128;                  // (the same for one channel a thread: the sums' layout)
    const long long want = std::max<long long>(1, 8LL * N_SM * WARPS / (nd * Bt));
    const long long len = (T + want - 1) / want;
    return (int)std::min<long long>(128, std::max<long long>(16, (len + 7) / 8 * 8));
}

int parts_of(int Bt, int T, int len) { return (int)(((long long)Bt * ((T + len - 1) / len) + WARPS - 1) / WARPS); }

// The kernels for 2, 3 and 4 taps are unrolled for exactly those; 1 and 5 to 8 taps
// run one that is unrolled for 8.
template <typename F>
cudaError_t by_taps(int K, F f)
{
    switch (K) {
    case 2: return f(std::integral_constant<int, 2>{}, std::true_type{});
    case 3: return f(std::integral_constant<int, 3>{}, std::true_type{});
    case 4: return f(std::integral_constant<int, 4>{}, std::true_type{});
    default: return f(std::integral_constant<int, 8>{}, std::false_type{});
    }
}

template <typename E, int VEC>
cudaError_t fwd_of(const ConvArgs &a, cudaStream_t stream)
{
    const int nd = (a.D + 32 * VEC - 1) / (32 * VEC), len = rows_of_warp(a.Bt, a.T, a.D), segs = (a.T + len - 1) / len;
    const long long units = (long long)a.Bt * segs * nd, blocks = (units + WARPS - 1) / WARPS;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    return by_taps(a.K, [&](auto kt, auto exact) {
        conv_fwd_kernel<E, decltype(kt)::value, decltype(exact)::value, VEC><<<(unsigned)blocks, THREADS, 0, stream>>>(
            (const E *)a.x, a.ldb, a.ldt, (const E *)a.w, (const E *)a.bias, (E *)a.y, a.T, a.D, a.K, a.silu, nd, segs,
            len, units);
        return cudaGetLastError();
    });
}

template <typename E, int VEC>
cudaError_t bwd_of(const ConvArgs &a, cudaStream_t stream)
{
    const int nd = (a.D + 32 * VEC - 1) / (32 * VEC), len = rows_of_warp(a.Bt, a.T, a.D), segs = (a.T + len - 1) / len;
    const int parts = parts_of(a.Bt, a.T, len);
    const long long blocks = (long long)parts * nd;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    const cudaError_t e = by_taps(a.K, [&](auto kt, auto exact) {
        conv_bwd_kernel<E, decltype(kt)::value, decltype(exact)::value, VEC><<<(unsigned)blocks, THREADS, 0, stream>>>(
            (const E *)a.x, a.ldb, a.ldt, (const E *)a.w, (const E *)a.bias, (const E *)a.dy, (E *)a.dx, a.part, a.T,
            a.D, a.K, a.silu, nd, segs, len, (long long)a.Bt * segs);
        return cudaGetLastError();
    });
    if (e != cudaSuccess) return e;
    conv_reduce_kernel<E><<<dim3((a.D + 31) / 32, a.K + 1), 256, 0, stream>>>(a.part, (E *)a.dw, (E *)a.dbias, parts,
                                                                             a.D, a.K);
    return cudaGetLastError();
}

template <typename E, int VEC>
cudaError_t packed_of(const ConvPackedArgs &a, cudaStream_t stream)
{
    const int nd = (a.D + 32 * VEC - 1) / (32 * VEC);
    // single tokens have no tails unless there is no window
    const long long heads = a.K > 1 || a.seq.starts.p ? (long long)a.seq.count * nd : 0;
    const long long tails = a.seq.starts.p || a.K == 1 ? (long long)((a.seq.rows + TAIL_ROWS - 1) / TAIL_ROWS) * nd : 0;
    const long long blocks = (heads + tails + WARPS - 1) / WARPS;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    if (blocks == 0) return cudaSuccess;
    return by_taps(a.K, [&](auto kt, auto exact) {
        conv_packed_kernel<E, decltype(kt)::value, decltype(exact)::value, VEC>
            <<<(unsigned)blocks, THREADS, 0, stream>>>((const E *)a.x, a.ldx, (const E *)a.w, (const E *)a.bias,
                                                       (E *)a.window, (E *)a.y, a.seq, a.D, a.K, a.silu, nd, heads,
                                                       heads + tails);
        return cudaGetLastError();
    });
}

}  // namespace

size_t conv_workspace_bytes(int Bt, int T, int D, int K)
{
    return (size_t)parts_of(Bt, T, rows_of_warp(Bt, T, D)) * (K + 1) * D * sizeof(float);
}

cudaError_t launch_conv_fwd(const ConvArgs &a, cudaStream_t stream)
{
    if (a.bf16)
        return groups_of_4<__nv_bfloat16>(a.D, {a.x, a.y}, {a.ldb, a.ldt}) ? fwd_of<__nv_bfloat16, 4>(a, stream)
                                                                           : fwd_of<__nv_bfloat16, 1>(a, stream);
    return groups_of_4<float>(a.D, {a.x, a.y}, {a.ldb, a.ldt}) ? fwd_of<float, 4>(a, stream) : fwd_of<float, 1>(a, stream);
}

cudaError_t launch_conv_bwd(const ConvArgs &a, cudaStream_t stream)
{
    if (a.bf16)
        return groups_of_4<__nv_bfloat16>(a.D, {a.x, a.dy, a.dx}, {a.ldb, a.ldt})
                   ? bwd_of<__nv_bfloat16, 4>(a, stream) : bwd_of<__nv_bfloat16, 1>(a, stream);
    return groups_of_4<float>(a.D, {a.x, a.dy, a.dx}, {a.ldb, a.ldt}) ? bwd_of<float, 4>(a, stream)
                                                                      : bwd_of<float, 1>(a, stream);
}

cudaError_t launch_conv_packed(const ConvPackedArgs &a, cudaStream_t stream)
{
    if (a.bf16)
        return groups_of_4<__nv_bfloat16>(a.D, {a.x, a.y}, {a.ldx}) ? packed_of<__nv_bfloat16, 4>(a, stream)
                                                                    : packed_of<__nv_bfloat16, 1>(a, stream);
    return groups_of_4<float>(a.D, {a.x, a.y}, {a.ldx}) ? packed_of<float, 4>(a, stream) : packed_of<float, 1>(a, stream);
}

}  // namespace mms
