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
//   first   the first segment of a sequence in full; of those between it and the last
//           only the end state from nothing and the sum of dt (the decay of a state
//           over the segment is exp(-Aneg sum dt));
//   rest    all later segments, each from the chain of the end states before it.
// A sequence of one segment is done in the first launch, with one exponential a state
// and step; only the segments between the first and the last take two. Of a sequence of
// more than FEW segments the first is taken like those between: the launch would
// otherwise end with its CTAs alone, which have half as much again to do.
//
// Unit u of a launch is segment i of sequence s with u = s + start_s / seg + i: as
// a sequence of n rows has at most (start_s + n) / seg - start_s / seg + 1
// segments, no two share a number, and a binary search over the starts finds s.
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
constexpr int SUB = 4;                  // rows of x, dt and z in registers
constexpr int FEW = 3;                  // segments of a sequence whose first is done in full at once
#ifndef MMS_PACKED_POLY
#define MMS_PACKED_POLY 1
#endif
#ifndef MMS_PACKED_MINB
#define MMS_PACKED_MINB 4
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
    float *entry;                       // (row, D, N) what long sequences go on from
    int seg, nd;                        // rows of a segment, channel blocks
    int units;                          // units of segments; the blocks behind them clear rows of no sequence
};

// NS states of a channel on each of G lanes.
template <int NS_, int G_>
struct Split {
    static constexpr int NS = NS_, G = G_, NP = NS_ * G_, DPB = THREADS / G_;
};

// ------------------------------------------------------------- segments

// The rows [t0, t1) from state h; FULL: with outputs, else h from what it is and the
// sum of dt. Rows come through registers SUB at a time, the next ones requested as
// soon as these are converted; B and C as float32 through shared memory, TT rows at a time.
// POLY of a thread's pairs of exponentials are taken from MUFU to the FMA pipe.
template <bool FULL, typename E, typename BE, typename S>
__device__ __forceinline__ float walk(const Args<E, BE> &a, float (*bc)[TT][2][S::NP], float2 (&h)[S::NS / 2],
                                      const float2 (&nan2)[S::NS / 2], int t0, int t1, int d, int g, bool act)
{
    constexpr int NS = S::NS, NP = S::NP;
    constexpr int ARR = FULL ? 2 : 1;                      // B, and C where it is wanted
    constexpr int PER = (TT * ARR * NP + THREADS - 1) / THREADS;
    constexpr int POLY = MMS_PACKED_POLY * NS / 16;
    const int tid = threadIdx.x;
    const bool gate = FULL && a.z != nullptr;
    const float skip = FULL && a.d_skip && act ? a.d_skip[d] : 0.f;
    const int ds = act ? d : 0;                            // a channel that is there
    const E *xp = a.x + t0 * a.ldx + ds, *dp = a.dt + t0 * a.lddt + ds;
    const E *zp = gate ? a.z + t0 * a.ldz + ds : a.x;
    const long long ldz = gate ? a.ldz : 0;
    E *yp = a.y + (long long)t0 * a.D + ds;
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
            xp += a.ldx, dp += a.lddt;
            if (FULL) zp += ldz;
        }
    };
    float next[PER];
    auto bc_in = [&](int t) {                              // this thread's share of a tile of B and C
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int o = tid + q * THREADS, n = o % NP, arr = o / NP % ARR, j = o / (NP * ARR);
            float v = 0.f;
            if (j < TT && n < a.N && t + j < t1)
                v = arr ? to_f(a.C[(t + j) * a.ldC + n]) : to_f(a.B[(t + j) * a.ldB + n]);
            next[q] = v;
        }
    };
    auto bc_out = [&](int buf) {
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int o = tid + q * THREADS, n = o % NP, arr = o / NP % ARR, j = o / (NP * ARR);
            if (j < TT) bc[buf][j][arr][n] = next[q];
        }
    };
    bc_in(t0);
    rows_in(t1 - t0);
    bc_out(0);
    __syncthreads();
    float total = 0.f;
    int buf = 0;
    for (int t = t0; t < t1; t += TT, buf ^= 1) {
        const bool more = t + TT < t1;
        if (more) bc_in(t + TT);
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
                if (!FULL) total += df[j];
                const float4 *bp = reinterpret_cast<const float4 *>(&bc[buf][sub + j][0][g * NS]);
                const float4 *cp = reinterpret_cast<const float4 *>(&bc[buf][sub + j][1][g * NS]);
                float2 acc[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
                for (int q = 0; q < NS / 4; ++q) {
                    const float4 Bv = bp[q];
                    const float2 e0 = mul2(dt2, nan2[2 * q]), e1 = mul2(dt2, nan2[2 * q + 1]);
                    h[2 * q] = fma2(2 * q < POLY ? ex2_poly2(e0) : ex2x2(e0), h[2 * q], mul2(bx2, lo(Bv)));
                    h[2 * q + 1] = fma2(2 * q + 1 < POLY ? ex2_poly2(e1) : ex2x2(e1), h[2 * q + 1], mul2(bx2, hi(Bv)));
                    if (FULL) {
                        const float4 Cv = cp[q];
                        acc[0] = fma2(lo(Cv), h[2 * q], acc[0]);
                        acc[1] = fma2(hi(Cv), h[2 * q + 1], acc[1]);
                    }
                }
                if (FULL) {
                    acc[0] = add2(acc[0], acc[1]);
                    float yv = acc[0].x + acc[0].y;
#pragma unroll
                    for (int o = S::G / 2; o > 0; o >>= 1) yv += __shfl_xor_sync(0xffffffffu, yv, o);
                    yv = (yv + skip) * gf[j];
                    if (act && g == 0 && j < left) *yp = from_f<E>(yv);
                    yp += a.D;
                }
            }
        }
        if (more) {
            bc_out(buf ^ 1);                               // the tile before was read before the last barrier
            __syncthreads();
        }
    }
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
scan_packed_kernel(const __grid_constant__ Args<E, BE> a)
{
    __shared__ __align__(16) float bc[2][TT][2][S::NP];
    const int tid = threadIdx.x, g = tid % S::G;
    const int unit = blockIdx.x / a.nd;
    if (unit >= a.units) {                                 // rows of no sequence: zeros
        const int behind = a.seq.start(a.seq.count), before = a.seq.start(0);
        const long long lead = (long long)before * a.D, all = lead + (long long)(a.seq.rows - behind) * a.D;
        const long long step = (long long)(gridDim.x - a.units * a.nd) * THREADS;
        for (long long i = (long long)(blockIdx.x - a.units * a.nd) * THREADS + tid; i < all; i += step)
            a.y[i < lead ? i : (long long)behind * a.D + (i - lead)] = from_f<E>(0.f);
        return;
    }
    const int s = Sequences::last_at_most(a.seq.count, unit, [&](int i) { return i + a.seq.start(i) / a.seg; });
    if (s < 0) return;
    const int first = a.seq.start(s), end = max(first, a.seq.start(s + 1));
    const int i = unit - (s + first / a.seg);
    const int segs = max(1, (end - first + a.seg - 1) / a.seg);
    if (i < 0 || i >= segs) return;
    const bool split = segs > FEW;                         // its first segment is left for the second launch, too
    if (REST ? i == 0 && !split : i > 0 && i == segs - 1) return;

    const int d = (blockIdx.x % a.nd) * S::DPB + tid / S::G;
    const bool act = d < a.D;
    const size_t at = (size_t)(act ? d : 0) * a.N;
    const int t0 = first + i * a.seg, t1 = min(end, t0 + a.seg);
    float2 nan2[S::NS / 2], h[S::NS / 2];
    read_rates<S>(nan2, a.aneg + at, a.N, g, act, a.pj.on);
    const long long row = first / a.seg;                   // of the sequence's first end state
    const size_t DN = (size_t)a.D * a.N;
    // a sequence of more than FEW segments has more than FEW * seg rows: the next one's is another
    float *entry = a.entry + (size_t)(first / (FEW * a.seg)) * DN + at;
    if (i == 0) {
        const long long from = a.seq.from(s);
        if (REST) read_state<S>(h, entry, a.N, g, act);
        else read_state<S>(h, a.state + (from >= 0 ? from : 0) * DN + at, a.N, g, act && from >= 0);
        // (its last segment may write the place that it was read from)
        if (!REST && split) write_state<S>(h, entry, a.N, g, act);
    } else if (REST) {
        // the states at the ends of the segments before: of the first as it is, of the others
        // what was left of the one before and their own
        read_state<S>(h, a.ends + row * DN + at, a.N, g, act);
#pragma unroll 2
        for (int j = 1; j < i; ++j) {
            float2 v[S::NS / 2];
            read_state<S>(v, a.ends + (row + j) * DN + at, a.N, g, act);
            const float dtv = act ? a.sums[(row + j) * a.D + d] : 0.f;
#pragma unroll
            for (int q = 0; q < S::NS / 2; ++q) h[q] = fma2(ex2x2(mul2(f2(dtv, dtv), nan2[q])), h[q], v[q]);
        }
    } else {
#pragma unroll
        for (int q = 0; q < S::NS / 2; ++q) h[q] = f2(0.f, 0.f);
    }
    if (REST || (i == 0 && !split)) {
        walk<true, E, BE, S>(a, bc, h, nan2, t0, t1, d, g, act);
    } else {
        const float total = walk<false, E, BE, S>(a, bc, h, nan2, t0, t1, d, g, act);
        if (act && g == 0) a.sums[(row + i) * a.D + d] = total;
    }
    if (i == segs - 1) {
        const long long to = a.seq.to(s);
        if (to >= 0) write_state<S>(h, a.state + to * DN + at, a.N, g, act);
    } else if (!REST) {
        write_state<S>(h, a.ends + (row + i) * DN + at, a.N, g, act);
    }
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
    const long long want = std::max<long long>(1, 4LL * N_SM / nd);
    const long long seg = std::max<long long>(64, (rows + want - 1) / want);
    return (int)std::min<long long>((seg + TT - 1) / TT * TT, 1 << 30);
}

// Sequences of more than FEW segments are told apart by start / (FEW * seg).
int entries_of(int rows, int seg) { return rows > FEW * seg ? rows / (FEW * seg) + 1 : 0; }

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
    const int rows = p.seq.rows;
    a.seg = segment_rows(rows, p.D, p.N);
    a.nd = (p.D + S::DPB - 1) / S::DPB;
    a.ends = static_cast<float *>(p.workspace);
    a.entry = a.ends + (size_t)(rows / a.seg) * p.D * p.N;
    a.sums = a.entry + (size_t)entries_of(rows, a.seg) * p.D * p.N;
    const long long units = (long long)p.seq.count + rows / a.seg;
    const long long clear = 2 * N_SM;
    if (units * a.nd + clear > 0x7fffffffLL) return cudaErrorInvalidValue;
    a.units = (int)units;
    scan_packed_kernel<E, BE, S, false><<<(unsigned)(units * a.nd + clear), THREADS, 0, stream>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || rows <= a.seg) return e;       // no sequence can have a second segment
    scan_packed_kernel<E, BE, S, true><<<(unsigned)(units * a.nd), THREADS, 0, stream>>>(a);
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

// Segments before the last of their sequence, at most one for every `seg` rows, and entries.
size_t scan_packed_workspace_bytes(int rows, int count, int D, int N)
{
    (void)count;
    const int seg = segment_rows(rows, D, N);
    const size_t ends = rows / seg, entries = entries_of(rows, seg);
    return (ends * (N + 1) + entries * N) * D * sizeof(float);
}

cudaError_t launch_scan_packed(const ScanPackedArgs &p, cudaStream_t stream)
{
    using BF = __nv_bfloat16;
    if (!p.bf16) return packed_of<float, float>(p, stream);
    return p.bc_bf16 ? packed_of<BF, BF>(p, stream) : packed_of<BF, float>(p, stream);
}

}  // namespace mms
