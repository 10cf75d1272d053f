// Selective scan over packed sequences that go on from stored states (sm_100a):
// prompts of unequal lengths behind one another, their pieces, and single tokens.
//
//     h_t = exp(-dt_t Aneg) h_{t-1} + dt_t B_t x_t,   y_t = sum_n C_tn h_tn    (h before the first: the cache)
//     out_t = (y_t + d_skip) * silu(z_t)              (each part where it is given)
//
// The reference's cache goes on by single tokens of one batch only (reference
// mamba_metal/model.py:203-221, 228-241).
//
// Prompts are bound by the exponentials, one a state and step (MUFU, 16 an SM and
// clock). A thread holds up to 16 states of one channel in registers, as the forward
// scan does; G = 1, 2 or 4 lanes share a channel of up to 16, 32 or 64 states. A
// sequence is cut into segments of `seg` rows, so that one long prompt fills the GPU
// as well as many short ones, whatever the lengths, which the host does not know:
//   first   segments whose state is known, the first ones of short sequences, with their
//           outputs; of the others but a sequence's last the state at the end from nothing
//           and the sum of dt (a state's decay over the segment is exp(-Aneg sum dt));
//   rest    all other segments with their outputs, each from the chain of the ends before it.
// The ends are sums over the rows, v_n = sum_t exp(-Aneg_n sum_{t' > t} dt) dt_t B_tn x_t, from
// the last row back: a state's rows are left out where the decay is flushed to 0
// (below 2^-126), which leaves a quarter of the exponentials where dt is around 0.14
// and Aneg 1 to 16. (Walking forward through all of them: 16384 x 2048 x 16, float32, 343 us.
// Adding what enters a segment to outputs computed from nothing, with the same
// exponentials left out: 313 us, 381 instead of 226 for 8192 x 2304 x 16 in bf16; it reads and
// writes the outputs once more.)
//
// Unit u of a launch is segment i of sequence s with u = s + start_s / seg + i: as
// a sequence of n rows has at most (start_s + n) / seg - start_s / seg + 1
// segments, no two share a number, and a search over the starts finds s.
//
// Single tokens without a list of starts are bound by the states' bytes, read and
// written once: 4 states a lane, G lanes a channel, several sequences a thread so that
// their loads are in flight together and Aneg is read once.
#include <algorithm>
#include <type_traits>

#include "mms_common.cuh"
#include "mms_serve.h"

namespace mms {

namespace {

constexpr int THREADS = 128;
constexpr int TT = 8;                   // rows of a tile of B and C
#ifndef MMS_SUB
#define MMS_SUB 4
#endif
constexpr int SUB = MMS_SUB;            // rows of x, dt and z in registers
constexpr float GONE = -126.f;          // log2 of the decays below, which ex2 flushes to 0
// A sequence's first segment is done in full in the first launch if it has at most FEW
// segments; of longer ones its end comes first, like the others', so that the launch does not
// end with its CTAs alone.
#ifndef MMS_PACKED_FEW
#define MMS_PACKED_FEW 3
#endif
constexpr int FEW = MMS_PACKED_FEW;
#ifndef MMS_PACKED_POLY
#define MMS_PACKED_POLY 1
#endif
#ifndef MMS_PACKED_MINB
#define MMS_PACKED_MINB 4
#endif
#ifndef MMS_PACKED_FILL
#define MMS_PACKED_FILL 4
#endif

template <typename E, typename BE>
struct Args {
    const E *x, *dt, *z;
    const BE *B, *C;
    long long ldx, lddt, ldB, ldC, ldz;
    const float *aneg, *d_skip;
    float *state;
    E *y;
    Sequences seq;
    int D, N;
    Proj pj;
    float *ends, *sums;                 // end states (row, D, N) and sums of dt (row, D) of segments
    float *entry;                       // (row, D, N) what sequences of more than FEW segments go on from
    int seg, nd;                        // rows of a segment, channel blocks
    int units;                          // units of segments; the blocks behind them clear rows of no sequence
};

// NS states of a channel on each of G lanes.
template <int NS_, int G_>
struct Split {
    static constexpr int NS = NS_, G = G_, NP = NS_ * G_, DPB = THREADS / G_;
};

// What a CTA of a segment's launch is to do.
struct Unit {
    int s, i, segs, t0, t1;             // sequence, segment of how many, rows
    int row;                            // of the sequence in the workspace
};
template <typename E, typename BE>
__device__ __forceinline__ bool find_unit(const Args<E, BE> &a, int unit, Unit &u)
{
    u.s = Sequences::last_at_most(a.seq.count, unit, [&](int i) { return i + a.seq.start(i) / a.seg; });
    if (u.s < 0) return false;
    const int first = a.seq.start(u.s), end = max(first, a.seq.start(u.s + 1));
    u.row = first / a.seg;
    u.i = unit - (u.s + u.row);
    u.segs = max(1, (end - first + a.seg - 1) / a.seg);
    u.t0 = first + u.i * a.seg, u.t1 = min(end, u.t0 + a.seg);
    return u.i >= 0 && u.i < u.segs;
}

// A tile of TT rows of B and C as float32 in shared memory: this thread's share of it.
template <int NP, int ARR>
struct Share {
    static constexpr int PER = (TT * ARR * NP + THREADS - 1) / THREADS;
    float v[PER];
    template <typename BE>
    __device__ __forceinline__ void read(const BE *B, long long ldB, const BE *C, long long ldC, int N, int t, int t1) {
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int o = threadIdx.x + q * THREADS, n = o % NP, arr = o / NP % ARR, j = o / (NP * ARR);
            v[q] = 0.f;
            if (j < TT && n < N && t + j < t1) v[q] = arr ? to_f(C[(t + j) * ldC + n]) : to_f(B[(t + j) * ldB + n]);
        }
    }
    __device__ __forceinline__ void write(float (*bc)[ARR][NP]) const {
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int o = threadIdx.x + q * THREADS, n = o % NP, arr = o / NP % ARR, j = o / (NP * ARR);
            if (j < TT) bc[j][arr][n] = v[q];
        }
    }
};

// ------------------------------------------------------------- segments

// The rows [t0, t1) from state h, with their outputs. Rows come through registers
// SUB at a time, the next ones requested as soon as these are converted; B and C through
// shared memory, TT rows at a time. POLY of a thread's 8 pairs of exponentials are taken
// from MUFU to the FMA pipe (16384 x 2048 x 16: 0 pairs 360 us, 1 343, 2 366, in the form with two
// walks).
template <typename E, typename BE, typename S>
__device__ __forceinline__ void walk(const Args<E, BE> &a, float (*bc)[TT][2][S::NP], float2 (&h)[S::NS / 2],
                                      const float2 (&nan2)[S::NS / 2], int t0, int t1, int d, int g, bool act)
{
    constexpr int NS = S::NS;
    constexpr int POLY = MMS_PACKED_POLY * NS / 16;
    const bool gate = a.z != nullptr;
    const float skip = a.d_skip && act ? a.d_skip[d] : 0.f;
    const int ds = act ? d : 0;                            // a channel that is there
    const E *xp = a.x + t0 * a.ldx + ds, *dp = a.dt + t0 * a.lddt + ds;
    const E *zp = gate ? a.z + t0 * a.ldz + ds : a.x;
    const long long ldz = gate ? a.ldz : 0;
    long long yo = (long long)t0 * a.D + ds;
    E xr[SUB], dr[SUB], zr[SUB];
    auto rows_in = [&](int left) {                         // the next SUB rows, of which `left` are there
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
            if (j < left) {
                xr[j] = *xp, dr[j] = *dp;
                if (gate) zr[j] = *zp;
            } else {
                xr[j] = dr[j] = from_f<E>(0.f);
            }
            xp += a.ldx, dp += a.lddt, zp += ldz;
        }
    };
    Share<S::NP, 2> next;
    next.read(a.B, a.ldB, a.C, a.ldC, a.N, t0, t1);
    rows_in(t1 - t0);
    next.write(bc[0]);
    __syncthreads();
    int buf = 0;
    for (int t = t0; t < t1; t += TT, buf ^= 1) {
        const bool more = t + TT < t1;
        if (more) next.read(a.B, a.ldB, a.C, a.ldC, a.N, t + TT, t1);
#pragma unroll
        for (int sub = 0; sub < TT; sub += SUB) {
            const int left = t1 - t - sub;                 // rows from here on
            if (sub > 0 && left <= 0) break;
            float xf[SUB], df[SUB], gf[SUB];
#pragma unroll
            for (int j = 0; j < SUB; ++j) xf[j] = to_f(xr[j]), df[j] = to_f(dr[j]), gf[j] = 1.f;
            if (a.pj.on) {
#pragma unroll
                for (int j = 0; j < SUB; ++j) df[j] = j < left ? fmaf(a.pj.range, sigmoid_fast(df[j]), a.pj.lo) : 0.f;
            }
            if (gate) {
#pragma unroll
                for (int j = 0; j < SUB; ++j) gf[j] = to_f(zr[j]) * sigmoid_fast(to_f(zr[j]));
            }
            rows_in(left - SUB);
            // rows behind the last have dt = 0: decay 1, nothing added
#pragma unroll
            for (int j = 0; j < SUB; ++j) {
                const float2 dt2 = f2(df[j], df[j]), bx2 = f2(df[j] * xf[j], df[j] * xf[j]);
                const float4 *bp = reinterpret_cast<const float4 *>(&bc[buf][sub + j][0][g * NS]);
                const float4 *cp = reinterpret_cast<const float4 *>(&bc[buf][sub + j][1][g * NS]);
                float2 acc[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
                for (int q = 0; q < NS / 4; ++q) {
                    const float4 Bv = bp[q], Cv = cp[q];
                    const float2 e0 = mul2(dt2, nan2[2 * q]), e1 = mul2(dt2, nan2[2 * q + 1]);
                    h[2 * q] = fma2(2 * q < POLY ? ex2_poly2(e0) : ex2x2(e0), h[2 * q], mul2(bx2, lo(Bv)));
                    h[2 * q + 1] = fma2(2 * q + 1 < POLY ? ex2_poly2(e1) : ex2x2(e1), h[2 * q + 1], mul2(bx2, hi(Bv)));
                    acc[0] = fma2(lo(Cv), h[2 * q], acc[0]);
                    acc[1] = fma2(hi(Cv), h[2 * q + 1], acc[1]);
                }
                acc[0] = add2(acc[0], acc[1]);
                float yv = acc[0].x + acc[0].y;
#pragma unroll
                for (int o = S::G / 2; o > 0; o >>= 1) yv += __shfl_xor_sync(0xffffffffu, yv, o);
                yv = (yv + skip) * gf[j];
                if (act && g == 0 && j < left) a.y[yo] = from_f<E>(yv);
                yo += a.D;
            }
        }
        if (more) {
            next.write(bc[buf ^ 1]);                       // the tile before was read before the last barrier
            __syncthreads();
        }
    }
}

// What the rows [t0, t1) leave of nothing, v, and the sum of their dt, from the last row back.
// An x or B that is not finite stays in the state for good, whatever its decay: a product
// with 0 keeps it, also where its row is left out.
template <typename E, typename BE, typename S>
__device__ __forceinline__ float leave(const Args<E, BE> &a, float (*bc)[TT][1][S::NP], float (&lost)[S::NP],
                                       float2 (&v)[S::NS / 2], const float2 (&nan2)[S::NS / 2], int t0, int t1, int d,
                                       int g, bool act)
{
    constexpr int NPAIR = S::NS / 2;
    const int tid = threadIdx.x, ds = act ? d : 0;
    const E *xp = a.x + (t1 - 1) * a.ldx + ds, *dp = a.dt + (t1 - 1) * a.lddt + ds;
    E xr[TT], dr[TT];                                      // rows t - 1, t - 2, ..
    auto rows_in = [&](int left) {
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            if (j < left) {
                xr[j] = *xp, dr[j] = *dp;
            } else {
                xr[j] = dr[j] = from_f<E>(0.f);
            }
            xp -= a.ldx, dp -= a.lddt;
        }
    };
    if (tid < S::NP) lost[tid] = 0.f;
    // (rows of B in front of t0 are other segments', or not there: read() takes rows from t0 on)
    Share<S::NP, 1> next;
    float bad_b = 0.f;
    auto b_in = [&](int t) {                               // rows t - 1 down to t - TT
#pragma unroll
        for (int q = 0; q < next.PER; ++q) {
            const int o = tid + q * THREADS, n = o % S::NP, j = o / S::NP;
            next.v[q] = 0.f;
            if (j < TT && n < a.N && t - 1 - j >= t0) next.v[q] = to_f(a.B[(t - 1 - j) * a.ldB + n]);
            bad_b = fmaf(next.v[q], 0.f, bad_b);
        }
    };
#pragma unroll
    for (int q = 0; q < NPAIR; ++q) v[q] = f2(0.f, 0.f);
    b_in(t1);
    rows_in(t1 - t0);
    next.write(bc[0]);
    __syncthreads();
    float total = 0.f, bad_x = 0.f;
    int buf = 0;
    for (int t = t1; t > t0; t -= TT, buf ^= 1) {
        const int left = t - t0;
        float sum[TT], bx[TT], least = INFINITY, most = -INFINITY;
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            float dtv = to_f(dr[j]);
            if (a.pj.on) dtv = j < left ? fmaf(a.pj.range, sigmoid_fast(dtv), a.pj.lo) : 0.f;
            sum[j] = total;                                // of the rows behind
            least = fminf(least, total), most = fmaxf(most, total);
            total += dtv;
            bx[j] = dtv * to_f(xr[j]);
            bad_x = fmaf(bx[j], 0.f, bad_x);
        }
        const bool more = left > TT;
        if (more) {
            b_in(t - TT);
            rows_in(left - TT);
        }
#pragma unroll
        for (int q = 0; q < NPAIR; ++q) {
            // the pair's largest decay in the tile
            const float top = fmaxf(fmaxf(nan2[q].x * least, nan2[q].x * most), fmaxf(nan2[q].y * least, nan2[q].y * most));
            if (!__any_sync(0xffffffffu, act && !(top < GONE))) continue;
#pragma unroll
            for (int j = 0; j < TT; ++j) {
                const float2 e = ex2x2(mul2(f2(sum[j], sum[j]), nan2[q]));
                const float2 Bv = *reinterpret_cast<const float2 *>(&bc[buf][j][0][g * S::NS + 2 * q]);
                v[q] = fma2(mul2(e, f2(bx[j], bx[j])), Bv, v[q]);
            }
        }
        if (more) {
            next.write(bc[buf ^ 1]);                       // the tile before was read before the last barrier
            __syncthreads();
        }
    }
    if (bad_b != bad_b) lost[tid % S::NP] = bad_b;         // (whichever of those that found one)
    __syncthreads();
#pragma unroll
    for (int q = 0; q < NPAIR; ++q)
        v[q] = add2(v[q], f2(bad_x + lost[g * S::NS + 2 * q], bad_x + lost[g * S::NS + 2 * q + 1]));
    return total;
}

template <typename S>
__device__ __forceinline__ void read_state(float2 (&h)[S::NS / 2], const float *p, int N, int g, bool act)
{
#pragma unroll
    for (int q = 0; q < S::NS / 4; ++q) {
        const int n = g * S::NS + 4 * q;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (act && n < N) v = *reinterpret_cast<const float4 *>(p + n);
        h[2 * q] = lo(v);
        h[2 * q + 1] = hi(v);
    }
}

template <typename S>
__device__ __forceinline__ void write_state(const float2 (&h)[S::NS / 2], float *p, int N, int g, bool act)
{
#pragma unroll
    for (int q = 0; q < S::NS / 4; ++q) {
        const int n = g * S::NS + 4 * q;
        if (act && n < N) st4(p + n, make_float4(h[2 * q].x, h[2 * q].y, h[2 * q + 1].x, h[2 * q + 1].y));
    }
}

// -Aneg * log2(e) of the lane's states, 0 behind the last
template <typename S>
__device__ __forceinline__ void read_rates(float2 (&nan2)[S::NS / 2], const float *aneg, int N, int g, bool act, bool raw)
{
    read_state<S>(nan2, aneg, N, g, act);
#pragma unroll
    for (int q = 0; q < S::NS / 2; ++q) {
        float2 v = nan2[q];
        if (raw) v = f2(softplus(v.x), softplus(v.y));
        const bool in = act && g * S::NS + 2 * q < N;
        nan2[q] = in ? f2(-v.x * MMS_LOG2E, -v.y * MMS_LOG2E) : f2(0.f, 0.f);
    }
}

template <typename E, typename BE, typename S, bool REST>
__global__ void __launch_bounds__(THREADS, MMS_PACKED_MINB)
scan_segments_kernel(const __grid_constant__ Args<E, BE> a)
{
    __shared__ __align__(16) float bc[2 * TT * 2 * S::NP];
    __shared__ float lost[S::NP];
    constexpr int NPAIR = S::NS / 2;
    const int tid = threadIdx.x, g = tid % S::G;
    const int unit = blockIdx.x / a.nd;
    if (!REST && unit >= a.units) {                        // rows of no sequence: zeros
        const int behind = a.seq.start(a.seq.count), before = a.seq.start(0);
        const long long lead = (long long)before * a.D, all = lead + (long long)(a.seq.rows - behind) * a.D;
        const long long step = (long long)(gridDim.x - a.units * a.nd) * THREADS;
        for (long long i = (long long)(blockIdx.x - a.units * a.nd) * THREADS + tid; i < all; i += step)
            a.y[i < lead ? i : (long long)behind * a.D + (i - lead)] = from_f<E>(0.f);
        return;
    }
    Unit u;
    if (!find_unit(a, unit, u)) return;
    const bool late = u.i > 0 || u.segs > FEW;             // its outputs come in the second launch
    if (REST ? !late : u.i > 0 && u.i == u.segs - 1) return;

    const int d = (blockIdx.x % a.nd) * S::DPB + tid / S::G;
    const bool act = d < a.D;
    const size_t at = (size_t)(act ? d : 0) * a.N, DN = (size_t)a.D * a.N;
    float2 nan2[NPAIR], h[NPAIR];
    read_rates<S>(nan2, a.aneg + at, a.N, g, act, a.pj.on);
    // a sequence of more than FEW segments has more than FEW * seg rows: the next one's is another
    float *entry = a.entry + (size_t)(u.row / FEW) * DN + at;
    if (REST && u.i > 0) {
        // the first segment's end, then of each one between what was left of it and its own
        read_state<S>(h, a.ends + u.row * DN + at, a.N, g, act);
#pragma unroll 2
        for (int j = 1; j < u.i; ++j) {
            float2 v[NPAIR];
            read_state<S>(v, a.ends + (u.row + j) * DN + at, a.N, g, act);
            const float dtv = act ? a.sums[(size_t)(u.row + j) * a.D + d] : 0.f;
#pragma unroll
            for (int q = 0; q < NPAIR; ++q) h[q] = fma2(ex2x2(mul2(f2(dtv, dtv), nan2[q])), h[q], v[q]);
        }
    } else {
        const long long from = REST || u.i > 0 ? -1 : a.seq.from(u.s);
        const float *src = REST ? entry : a.state + (from >= 0 ? from : 0) * DN + at;
        read_state<S>(h, src, a.N, g, act && (REST || from >= 0));
        // (its last segment may write the place that it was read from)
        if (!REST && u.i == 0 && late) write_state<S>(h, entry, a.N, g, act);
    }
    if (REST || !late) {
        walk<E, BE, S>(a, reinterpret_cast<float(*)[TT][2][S::NP]>(bc), h, nan2, u.t0, u.t1, d, g, act);
        if (u.i == u.segs - 1) {
            const long long to = a.seq.to(u.s);
            if (to >= 0) write_state<S>(h, a.state + to * DN + at, a.N, g, act);
            return;
        }
        if (REST) return;
    } else {
        float2 v[NPAIR];
        const float total = leave<E, BE, S>(a, reinterpret_cast<float(*)[TT][1][S::NP]>(bc), lost, v, nan2, u.t0, u.t1,
                                            d, g, act);
        if (act && g == 0) a.sums[(size_t)(u.row + u.i) * a.D + d] = total;
#pragma unroll
        for (int q = 0; q < NPAIR; ++q) h[q] = fma2(ex2x2(mul2(f2(total, total), nan2[q])), h[q], v[q]);
    }
    write_state<S>(h, a.ends + (u.row + u.i) * DN + at, a.N, g, act);
}

// --------------------------------------------------------- single tokens

template <typename BE>
__device__ __forceinline__ float4 four(const BE *p)
{
    if constexpr (sizeof(BE) == 4) {
        return ld4(p);
    } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
        return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u),
                           __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
    }
}

constexpr int TOKEN_THREADS = 256;

// Lane g of a channel's G holds states 4g .. 4g + 3 of SEQ sequences.
template <typename E, typename BE, int G, int SEQ>
__global__ void __launch_bounds__(TOKEN_THREADS)
scan_token_kernel(const __grid_constant__ Args<E, BE> a)
{
    const int tid = blockIdx.x % a.nd * TOKEN_THREADS + threadIdx.x;
    const int d = tid / G, g = threadIdx.x % G, n = 4 * g;
    const int s0 = blockIdx.x / a.nd * SEQ;
    const bool chan = d < a.D, act = chan && n < a.N;
    const size_t DN = (size_t)a.D * a.N, at = (size_t)d * a.N + n;
    float4 hv[SEQ], Bv[SEQ], Cv[SEQ];
    float xv[SEQ], dtv[SEQ], zv[SEQ];
    long long to[SEQ];
#pragma unroll
    for (int q = 0; q < SEQ; ++q) {
        const int s = s0 + q;
        const bool in = s < a.seq.count;
        const long long from = in ? a.seq.from(s) : -1;
        to[q] = in ? a.seq.to(s) : -1;
        hv[q] = Bv[q] = Cv[q] = make_float4(0.f, 0.f, 0.f, 0.f);
        xv[q] = dtv[q] = zv[q] = 0.f;
        if (act && from >= 0) hv[q] = *reinterpret_cast<const float4 *>(a.state + from * DN + at);
        if (act && in) {
            Bv[q] = four(a.B + s * a.ldB + n);
            Cv[q] = four(a.C + s * a.ldC + n);
        }
        if (chan && in) {
            xv[q] = to_f(a.x[s * a.ldx + d]);
            dtv[q] = to_f(a.dt[s * a.lddt + d]);
            if (a.z) zv[q] = to_f(a.z[s * a.ldz + d]);
        }
    }
    float4 av = make_float4(0.f, 0.f, 0.f, 0.f);
    if (act) av = ld4(a.aneg + at);
    if (a.pj.on) av = make_float4(softplus(av.x), softplus(av.y), softplus(av.z), softplus(av.w));
    const float2 n0 = f2(-av.x * MMS_LOG2E, -av.y * MMS_LOG2E), n1 = f2(-av.z * MMS_LOG2E, -av.w * MMS_LOG2E);
    const float skip = a.d_skip && chan ? a.d_skip[d] : 0.f;
#pragma unroll
    for (int q = 0; q < SEQ; ++q) {
        if (a.pj.on) dtv[q] = fmaf(a.pj.range, sigmoid_fast(dtv[q]), a.pj.lo);
        const float2 dt2 = f2(dtv[q], dtv[q]), bx2 = f2(dtv[q] * xv[q], dtv[q] * xv[q]);
        const float2 h0 = fma2(ex2x2(mul2(dt2, n0)), lo(hv[q]), mul2(bx2, lo(Bv[q])));
        const float2 h1 = fma2(ex2x2(mul2(dt2, n1)), hi(hv[q]), mul2(bx2, hi(Bv[q])));
        if (act && to[q] >= 0) st4(a.state + to[q] * DN + at, make_float4(h0.x, h0.y, h1.x, h1.y));
        const float2 acc = fma2(hi(Cv[q]), h1, mul2(lo(Cv[q]), h0));
        float yv = acc.x + acc.y;
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) yv += __shfl_xor_sync(0xffffffffu, yv, o, G);
        yv += skip;
        if (a.z) yv *= zv[q] * sigmoid_fast(zv[q]);
        if (chan && g == 0 && s0 + q < a.seq.count) a.y[(long long)(s0 + q) * a.D + d] = from_f<E>(yv);
    }
}

// ----------------------------------------------------------------- launch

int lanes_of(int N) { return N <= 16 ? 1 : N <= 32 ? 2 : 4; }

// Rows of a segment: as few as give every SM 4 CTAs (16 warps, what the registers hold)
// when the rows belong to one sequence, at least 64, a whole number of tiles.
int segment_rows(int rows, int D, int N)
{
    const long long nd = (D + THREADS / lanes_of(N) - 1) / (THREADS / lanes_of(N));
    const long long want = std::max<long long>(1, (long long)MMS_PACKED_FILL * N_SM / nd);
    const long long seg = std::max<long long>(64, (rows + want - 1) / want);
    return (int)std::min<long long>((seg + TT - 1) / TT * TT, 1 << 30);
}

// A call's units and its workspace (bytes from the start, regions of whole 256 bytes):
// segments before the last of their sequence, of which there is at most one for every `seg`
// rows; entries of sequences of more than FEW segments, told apart by start / (FEW * seg).
struct Plan {
    int seg;
    long long nd, units;
    bool more;                          // a sequence can have a second segment
    size_t sums = 0, entry = 0, total = 0;
    Plan(int rows, int count, int D, int N) : seg(segment_rows(rows, D, N)) {
        nd = ((long long)D * lanes_of(N) + THREADS - 1) / THREADS;
        units = (long long)count + rows / seg;
        more = rows > seg;
        const size_t ends = rows / seg, d = D;
        auto up = [](size_t n) { return (n + 255) / 256 * 256; };
        sums = up(ends * d * N * 4);
        entry = sums + up(ends * d * 4);
        total = !more ? 0 : entry + (ends >= FEW ? up((ends / FEW + 1) * d * N * 4) : 0);
    }
};

template <typename E, typename BE>
Args<E, BE> args_of(const ScanPackedArgs &p)
{
    Args<E, BE> a{};
    a.x = (const E *)p.x, a.dt = (const E *)p.dt, a.z = (const E *)p.z;
    a.B = (const BE *)p.B, a.C = (const BE *)p.C;
    a.ldx = p.ldx, a.lddt = p.lddt, a.ldB = p.ldB, a.ldC = p.ldC, a.ldz = p.ldz;
    a.aneg = p.aneg, a.d_skip = p.d_skip, a.state = p.state, a.y = (E *)p.y;
    a.seq = p.seq, a.D = p.D, a.N = p.N, a.pj = p.proj;
    return a;
}

template <typename E, typename BE, typename S>
cudaError_t segments_of(const ScanPackedArgs &p, cudaStream_t stream)
{
    Args<E, BE> a = args_of<E, BE>(p);
    const Plan plan(p.seq.rows, p.seq.count, p.D, p.N);
    char *ws = static_cast<char *>(p.workspace);
    a.seg = plan.seg, a.nd = (int)plan.nd, a.units = (int)plan.units;
    a.ends = (float *)ws, a.sums = (float *)(ws + plan.sums), a.entry = (float *)(ws + plan.entry);
    const long long clear = 2 * N_SM, blocks = plan.units * plan.nd;
    if (blocks + clear > 0x7fffffffLL) return cudaErrorInvalidValue;
    scan_segments_kernel<E, BE, S, false><<<(unsigned)(blocks + clear), THREADS, 0, stream>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || !plan.more) return e;
    scan_segments_kernel<E, BE, S, true><<<(unsigned)blocks, THREADS, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename E, typename BE, int G>
cudaError_t tokens_of(const ScanPackedArgs &p, cudaStream_t stream)
{
    Args<E, BE> a = args_of<E, BE>(p);
    a.nd = (p.D * G + TOKEN_THREADS - 1) / TOKEN_THREADS;
    // 4 sequences a thread once that still leaves 8 CTAs an SM, else one: the shorter chain of loads
    const bool many = (long long)a.nd * p.seq.count >= 4LL * 8 * N_SM;
    const long long blocks = (long long)a.nd * (many ? (p.seq.count + 3) / 4 : p.seq.count);
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    if (many) scan_token_kernel<E, BE, G, 4><<<(unsigned)blocks, TOKEN_THREADS, 0, stream>>>(a);
    else scan_token_kernel<E, BE, G, 1><<<(unsigned)blocks, TOKEN_THREADS, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename E, typename BE>
cudaError_t packed_of(const ScanPackedArgs &p, cudaStream_t stream)
{
    if (!p.seq.starts.p) {
        switch (groups_for(p.N)) {
        case 1: return tokens_of<E, BE, 1>(p, stream);
        case 2: return tokens_of<E, BE, 2>(p, stream);
        case 4: return tokens_of<E, BE, 4>(p, stream);
        case 8: return tokens_of<E, BE, 8>(p, stream);
        default: return tokens_of<E, BE, 16>(p, stream);
        }
    }
    if (p.N <= 4) return segments_of<E, BE, Split<4, 1>>(p, stream);
    if (p.N <= 8) return segments_of<E, BE, Split<8, 1>>(p, stream);
    if (p.N <= 16) return segments_of<E, BE, Split<16, 1>>(p, stream);
    if (p.N <= 32) return segments_of<E, BE, Split<16, 2>>(p, stream);
    return segments_of<E, BE, Split<16, 4>>(p, stream);
}

}  // namespace

size_t scan_packed_workspace_bytes(int rows, int count, int D, int N) { return Plan(rows, count, D, N).total; }

cudaError_t launch_scan_packed(const ScanPackedArgs &p, cudaStream_t stream)
{
    using BF = __nv_bfloat16;
    if (!p.bf16) return packed_of<float, float>(p, stream);
    return p.bc_bf16 ? packed_of<BF, BF>(p, stream) : packed_of<BF, float>(p, stream);
}

}  // namespace mms
