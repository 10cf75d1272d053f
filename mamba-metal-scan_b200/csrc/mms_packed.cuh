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
// clock), and by the instructions and shared memory reads around them. A thread holds up to 8
// states of two neighbouring channels in registers; G = 1, 2, 4 or 8 lanes share the two, for
// up to 8, 16, 32 or 64 states. A sequence is cut into segments of `seg` rows, so that one long
// prompt fills the GPU as well as many short ones, whatever the lengths, which the host does not know:
//   first   sequences of one segment, with their outputs; of others' segments but the last
//           the state at the end from nothing and the sum of dt (a state's decay over the
//           segment is exp(-Aneg sum dt));
//   join    (where there are many segments) the ends one after another become states;
//   rest    the segments of the other sequences with their outputs, each from the state before it.
// The ends are sums over the rows, v_n = sum_t exp(-Aneg_n sum_{t' > t} dt) dt_t B_tn x_t, from
// the last row back: a state's rows are left out where the decay is flushed to 0
// (below 2^-126), which leaves two fifths of the exponentials where dt is around 0.14
// and Aneg 1 to 16; smaller steps leave more (logits for dt of 0.001 to 0.1, as the model's: 8192 x 2304 x 16, float32,
// 16 prompts, 241 us for 204, 16384 x 2048 x 16, one prompt, 347 for 274). (Walking forward through all of them: 16384 x 2048 x 16, float32, 343 us;
// adding what enters a segment to outputs computed from nothing, with the same
// exponentials left out: 313 us, 381 instead of 226 for 8192 x 2304 x 16 in bf16, as it reads and
// writes the outputs once more.)
//
// 16384 x 2048 x 16, float32, one prompt: 278 us (100 first, 175 rest: MUFU at 49 and 70 % of its
// rate, 13 of 16 warps an SM that its registers allow). 8192 x 2304 x 16, bf16, 16 prompts: 205 us;
// 3001 x 1433 x 64, 63 tokens and 7 prompts: 227 us (rest: MUFU 52 %, shared memory 70 %).
// Not kept: a launch set up while the one before runs (griddepcontrol, 5 to 10 us slower: CTAs
// that are to leave at once hold the places of others); more warps of fewer states.
//
// Single tokens without a list of starts are bound by the states' bytes, read and
// written once: 4 states a lane, G lanes a channel. 256 x 2304 x 16: 22.4 us, 3.4 TB/s (75.5 MB; 5.4
// warps an issue wait for memory, the ALUs are at 49 %).
#pragma once

#include <float.h>

#include <algorithm>
#include <type_traits>

#include "mms_common.cuh"
#include "mms_serve.h"
#include "mms_stage.cuh"
#include "mms_units.h"

namespace mms {

namespace {

constexpr int THREADS = 128;
constexpr int TT = 8;                   // rows of a tile in shared memory
constexpr int STAGES = 3;               // tiles of x, dt and z
constexpr float GONE = -126.f;          // log2 of the decays below, which ex2 flushes to 0
constexpr int CTAS = 4;                 // an SM: what the registers hold
// Rows that a segment takes straight from memory. (None: 512 single tokens in a list of starts, 1432 x 16,
// float32, 105 for 75 us, 1000 of them and a prompt, 4096 rows, 289 for 225, 3001 x 1433 x 64 with 63, 274 for 261;
// 16 prompts alone, 8192 x 2304 x 16, 197 for 203, as the code is shorter. Up to 4: the same as 2.)
constexpr int DIRECT = 2;
// A segment's state is chained from the ends of those before it, by each segment for itself or, in calls
// with MANY more whole segments than sequences or 2 MANY of them in all, for sequences of more than CHAIN by a
// launch between the two. (16384 x 256 x 16, one prompt, 256 segments: 96 us, without that launch 255; 4096 x
// 1024 x 16, 4 prompts, 73 segments: 76 and 92; 512 x 1432 x 16, one prompt, 16 segments: 43 and 39; 8192 x 2304 x
// 16, 16 prompts, 32 segments: 224 and 211. Beside as many sequences as segments, whose lengths the host
// does not know: 16384 x 64 x 16, a prompt and 480 single tokens, 77 and 219; 8192 x 256 x 16, 512 sequences of
// 16 rows, which have nothing to join, 32 and 24.)
constexpr int MANY = 32, CHAIN = 4;

template <typename E>
struct Args {
    const E *x, *dt, *z;
    const void *B, *C;                  // float32, or bf16 where bc_bf16
    bool bc_bf16;
    long long ldx, lddt, ldB, ldC, ldz;
    const float *aneg, *d_skip;
    float *state;
    E *y;
    Sequences seq;
    int D, N;
    Proj pj;
    float *ends, *sums;                 // end states (row, D, N) and sums of dt (row, D) of segments
    float *entry;                       // (row, D, N) what sequences of several segments go on from
    int seg, nd;                        // rows of a segment, channel blocks
    int chain;                          // sequences of more segments are joined by a launch
    int fulls, units;                   // units of whole segments, of all; the blocks behind them clear rows of no sequence
};

// A thread holds NS states of 2 neighbouring channels; G lanes share the two. Lane g has the pairs
// g, G + g, 2G + g, .. of states: where the rates rise with the state, as they do at
// first, a warp's lanes then come to decays of 0 together.
template <int NS_, int G_>
struct Split {
    static constexpr int NS = NS_, G = G_, NP = NS_ * G_, NPAIR = NS_ / 2, DPB = 2 * THREADS / G_;
    // the first state of lane g's pair q, and where state n lies in a row of B or C: lane by lane
    __device__ static __forceinline__ int state(int g, int q) { return 2 * (q * G + g); }
    __device__ static __forceinline__ int place(int n) { return n / 2 % G * NS + n / 2 / G * 2 + n % 2; }
};
// The states of a thread: [channel][pair of states].
template <typename S>
using States = float2[2][S::NPAIR];

template <typename E>
__device__ __forceinline__ bool find_unit(const Args<E> &a, int unit, Unit &u)
{
    const int s = unit < a.fulls ? Sequences::last_at_most(a.seq.count, unit, [&](int i) { return a.seq.start(i) / a.seg; })
                                 : unit - a.fulls;
    return s >= 0 && unit_rows(unit, a.fulls, a.seg, s, a.seq.start(s), a.seq.start(s + 1), u);
}

// -Aneg log2(e), -FLT_MAX at least: what is -inf there (an Aneg above 2.3e38) would turn a step of 0, as the
// rows behind a sequence's last have it in a tile, into a NaN of every state. A NaN stays one.
__device__ __forceinline__ float rate_of(float aneg)
{
    float v;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(-aneg * MMS_LOG2E), "f"(-FLT_MAX));
    return v;
}

// An element of B or C.
__device__ __forceinline__ float bc_at(const void *p, long long i, bool bf16)
{
    return bf16 ? to_f(static_cast<const __nv_bfloat16 *>(p)[i]) : static_cast<const float *>(p)[i];
}

// A tile of TT rows of B and C as float32 in shared memory: this thread's share of it.
template <typename S, int ARR>
struct Share {
    static constexpr int NP = S::NP, PER = (TT * ARR * NP + THREADS - 1) / THREADS;
    float v[PER];
    template <typename E>
    __device__ __forceinline__ void read(const Args<E> &a, int t, int t0, int t1) {
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int o = threadIdx.x + q * THREADS, n = o % NP, arr = o / NP % ARR, j = o / (NP * ARR);
            v[q] = 0.f;
            if (j < TT && n < a.N && t + j >= t0 && t + j < t1)
                v[q] = bc_at(arr ? a.C : a.B, (t + j) * (arr ? a.ldC : a.ldB) + n, a.bc_bf16);
        }
    }
    __device__ __forceinline__ void write(float (*bc)[ARR][NP]) const {
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int o = threadIdx.x + q * THREADS, n = o % NP, arr = o / NP % ARR, j = o / (NP * ARR);
            if (j < TT) bc[j][arr][S::place(n)] = v[q];
        }
    }
};

// Rows t .. t + TT - 1 of ARR of x, dt and z, channels d0 .. d0 + DPB - 1, to a tile [row][array][channel];
// zeros for rows outside [t0, t1) and channels behind the last. VEC: 16 bytes at a time (D, the
// strides and the bases whole 16 bytes); else one element, bf16 ones through registers.
template <bool VEC, int ARR, int DPB, typename E>
__device__ __forceinline__ void stage(const Args<E> &a, E *tile, int d0, int t, int t0, int t1)
{
    constexpr int EPV = VEC ? 16 / (int)sizeof(E) : 1, CH = DPB / EPV, ALL = TT * ARR * CH;
    constexpr int UN = VEC ? ALL / THREADS + 1 : 4;        // (all 48 elements at once spill)
#pragma unroll UN
    for (int k0 = 0; k0 < ALL; k0 += THREADS) {
        const int k = k0 + threadIdx.x;
        if (ALL % THREADS && k >= ALL) break;
        const int q = k % CH, arr = k / CH % ARR, r = k / (CH * ARR), d = d0 + EPV * q;
        const bool in = t + r >= t0 && t + r < t1 && d < a.D;
        const E *src = arr == 0 ? a.x + (t + r) * a.ldx : arr == 1 ? a.dt + (t + r) * a.lddt : a.z + (t + r) * a.ldz;
        E *to = tile + (r * ARR + arr) * DPB + EPV * q;
        if constexpr (VEC) cp16(to, in ? src + d : a.x, in);
        else if constexpr (sizeof(E) == 4) cp4(to, in ? src + d : a.x, in);
        else *to = in ? src[d] : from_f<E>(0.f);
    }
    cp_commit();
}

// Both channels' values of a tile's row.
template <typename E>
__device__ __forceinline__ float2 both(const E *p)
{
    if constexpr (sizeof(E) == 4) {
        return *reinterpret_cast<const float2 *>(p);
    } else {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(p);
        return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
}

// dt from its logit.
__device__ __forceinline__ float step_of(const Proj &pj, float v) { return fmaf(pj.range, sigmoid_fast(v), pj.lo); }

// Lanes that share channels share these too: each computes some rows of its warp's channels and
// leaves them for the others, dt from its logits and (G > 2; with two the lanes have an output each)
// silu(z). float32 tiles take them in place, for bf16 ones there is a second tile.
template <typename E, typename S>
struct Ready {
    static constexpr int G = S::G, W = 64 / G, DPB = S::DPB;             // channels of a warp
    static constexpr int ARRAYS = G == 1 ? 0 : G == 2 ? 1 : 2;
    static constexpr bool APART = sizeof(E) == 2;
    static constexpr int SIZE = APART && ARRAYS ? ARRAYS * TT * DPB : 1;
    template <int ARR, typename F>
    __device__ static __forceinline__ void make(E *tile, float *apart, int arr, F f) {
        const int lane = threadIdx.x & 31, c0 = threadIdx.x / 32 * W;
#pragma unroll
        for (int q = 0; q < TT * W / 32; ++q) {
            const int e = lane + 32 * q, r = e / W, c = c0 + e % W;
            E *at = tile + (r * ARR + arr) * DPB + c;
            const float v = f(r, to_f(*at));
            if constexpr (APART) apart[((arr - 1) * TT + r) * DPB + c] = v;
            else *at = v;
        }
    }
    // both channels' of a row: c channels into the CTA
    template <int ARR>
    __device__ static __forceinline__ const float *at(const E *tile, const float *apart, int arr, int r, int c) {
        if constexpr (APART) return apart + ((arr - 1) * TT + r) * DPB + c;
        else return tile + (r * ARR + arr) * DPB + c;
    }
};

// ------------------------------------------------------------- segments

// The rows [t0, t1) from states h, with their outputs. Every value of B and C that a lane takes
// from shared memory serves its two channels: read for one channel each, 8 of them 16
// bytes at a time a row, they take as long as the row's 16 exponentials
// (shared memory returns 128 bytes a clock, 16 for the lanes of a quarter warp that all
// read the same). All exponentials are MUFU's: with one, two or three of a thread's 8 pairs on the FMA pipe the
// second launch took 184, 198 and 215 us, without 183 (16384 x 2048 x 16, float32, at that time).
template <bool VEC, bool GATE, bool RAW, typename E, typename S>
__device__ __forceinline__ void walk(const Args<E> &a, float (*bc)[TT][2][S::NP], E *tiles, float *apart,
                                     States<S> &h, const States<S> &nan2, int t0, int t1, int d0)
{
    constexpr int G = S::G, DPB = S::DPB, ARR = GATE ? 3 : 2, TILE = TT * ARR * DPB;
    using R = Ready<E, S>;
    constexpr bool DT = RAW && R::ARRAYS > 0, Z = GATE && R::ARRAYS > 1;
    const int tid = threadIdx.x, g = tid % G, c = 2 * (tid / G);
    // the channels whose outputs this lane writes: both, or one of them (lanes 0 and 1 of G)
    const int own = G == 1 ? 0 : g & 1;
    const int d = d0 + c + own;
    const bool out0 = g < 2 && d < a.D, out1 = G == 1 && d + 1 < a.D;
    const float skip0 = a.d_skip && out0 ? a.d_skip[d] : 0.f, skip1 = a.d_skip && out1 ? a.d_skip[d + 1] : 0.f;
    Share<S, 2> next;
    next.read(a, t0, t0, t1);
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) stage<VEC, ARR, DPB>(a, tiles + s * TILE, d0, t0 + s * TT, t0, t1);
    next.write(bc[0]);
    E *yp = a.y + (long long)t0 * a.D + (out0 ? d : 0);
    int buf = 0, at = 0;                                   // of B and C, of the tile
    for (int t = t0; t < t1; t += TT, buf ^= 1) {
        cp_wait<STAGES - 2>();
        __syncthreads();                                   // the tile is there, the one before it read
        const int ahead = at == 0 ? STAGES - 1 : at - 1;
        stage<VEC, ARR, DPB>(a, tiles + ahead * TILE, d0, t + (STAGES - 1) * TT, t0, t1);
        const bool more = t + TT < t1;
        if (more) next.read(a, t + TT, t0, t1);
        E *tile = tiles + at * TILE;
        const E *row = tile + c;
        const int left = t1 - t;
        // (rows behind the last have dt = 0)
        if (DT) R::template make<ARR>(tile, apart, 1, [&](int r, float v) { return r < left ? step_of(a.pj, v) : 0.f; });
        if (Z) R::template make<ARR>(tile, apart, 2, [&](int, float v) { return v * sigmoid_fast(v); });
        if (DT || Z) __syncwarp();
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            const float2 xv = both(row + j * ARR * DPB);
            float2 dtv;
            if (DT) dtv = *reinterpret_cast<const float2 *>(R::template at<ARR>(tile, apart, 1, j, c));
            else dtv = both(row + (j * ARR + 1) * DPB);
            if (RAW && !DT) dtv = j < left ? f2(step_of(a.pj, dtv.x), step_of(a.pj, dtv.y)) : f2(0.f, 0.f);
            const float2 bx = mul2(dtv, xv);
            const float4 *bp = reinterpret_cast<const float4 *>(&bc[buf][j][0][g * S::NS]);
            const float4 *cp = reinterpret_cast<const float4 *>(&bc[buf][j][1][g * S::NS]);
            float2 acc[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
            for (int q = 0; q < S::NPAIR / 2; ++q) {
                const float4 Bv = bp[q], Cv = cp[q];
#pragma unroll
                for (int ch = 0; ch < 2; ++ch) {
                    const float dt1 = ch ? dtv.y : dtv.x, bx1 = ch ? bx.y : bx.x;
                    const float2 e0 = mul2(f2(dt1, dt1), nan2[ch][2 * q]), e1 = mul2(f2(dt1, dt1), nan2[ch][2 * q + 1]);
                    h[ch][2 * q] = fma2(ex2x2(e0), h[ch][2 * q], mul2(f2(bx1, bx1), lo(Bv)));
                    h[ch][2 * q + 1] = fma2(ex2x2(e1), h[ch][2 * q + 1], mul2(f2(bx1, bx1), hi(Bv)));
                    acc[ch] = fma2(lo(Cv), h[ch][2 * q], acc[ch]);
                    acc[ch] = fma2(hi(Cv), h[ch][2 * q + 1], acc[ch]);
                }
            }
            float y0 = acc[0].x + acc[0].y, y1 = acc[1].x + acc[1].y;
            if (G > 1) {                                   // lanes of even g go on with the first channel
                const float mine = own ? y1 : y0, other = own ? y0 : y1;
                y0 = mine + __shfl_xor_sync(0xffffffffu, other, 1);
#pragma unroll
                for (int o = 2; o < G; o *= 2) y0 += __shfl_xor_sync(0xffffffffu, y0, o);
            }
            y0 += skip0, y1 += skip1;
            if (Z) {
                y0 *= *R::template at<ARR>(tile, apart, 2, j, c + own);
            } else if (GATE) {
                const float z0 = to_f(row[(j * ARR + 2) * DPB + own]);
                y0 *= z0 * sigmoid_fast(z0);
                if (G == 1) {
                    const float z1 = to_f(row[(j * ARR + 2) * DPB + 1]);
                    y1 *= z1 * sigmoid_fast(z1);
                }
            }
            if (out0 && j < left) *yp = from_f<E>(y0);
            if (out1 && j < left) yp[1] = from_f<E>(y1);
            yp += a.D;
        }
        if (more) next.write(bc[buf ^ 1]);
        at = at + 1 < STAGES ? at + 1 : 0;
    }
    cp_wait<0>();
    __syncthreads();
}

// walk() for a few rows, without shared memory: a single token among prompts needs neither tiles nor
// their unused rows.
template <typename E, typename S>
__device__ __forceinline__ void walk_direct(const Args<E> &a, States<S> &h, const States<S> &nan2, int t0, int t1,
                                            int d, int channels)
{
    constexpr int G = S::G;
    const int g = threadIdx.x % G, own = G == 1 ? 0 : g & 1;
    const bool out0 = g < 2 && own < channels, out1 = G == 1 && channels > 1;
    const int c0 = channels > 0 ? d : 0, c1 = channels > 1 ? d + 1 : c0, mine = own ? c1 : c0;
    const float skip0 = a.d_skip ? a.d_skip[mine] : 0.f, skip1 = a.d_skip ? a.d_skip[c1] : 0.f;
    for (long long t = t0; t < t1; ++t) {
        float2 Bv[S::NPAIR], Cv[S::NPAIR];
#pragma unroll
        for (int q = 0; q < S::NPAIR; ++q) {
            const int n = S::state(g, q);
            const bool in = n < a.N;
            auto pair = [&](const void *p, long long i) {
                return in ? f2(bc_at(p, i, a.bc_bf16), bc_at(p, i + 1, a.bc_bf16)) : f2(0.f, 0.f);
            };
            Bv[q] = pair(a.B, t * a.ldB + n), Cv[q] = pair(a.C, t * a.ldC + n);
        }
        const float2 xv = f2(to_f(a.x[t * a.ldx + c0]), to_f(a.x[t * a.ldx + c1]));
        float2 dtv = f2(to_f(a.dt[t * a.lddt + c0]), to_f(a.dt[t * a.lddt + c1]));
        float z0 = 0.f, z1 = 0.f;
        if (a.z) z0 = to_f(a.z[t * a.ldz + mine]), z1 = to_f(a.z[t * a.ldz + c1]);
        if (a.pj.on) dtv = f2(step_of(a.pj, dtv.x), step_of(a.pj, dtv.y));
        const float2 bx = mul2(dtv, xv);
        float2 acc[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
        for (int q = 0; q < S::NPAIR; ++q)
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
                const float dt1 = ch ? dtv.y : dtv.x, bx1 = ch ? bx.y : bx.x;
                h[ch][q] = fma2(ex2x2(mul2(f2(dt1, dt1), nan2[ch][q])), h[ch][q], mul2(f2(bx1, bx1), Bv[q]));
                acc[ch] = fma2(Cv[q], h[ch][q], acc[ch]);
            }
        float y0 = acc[0].x + acc[0].y, y1 = acc[1].x + acc[1].y;
        if (G > 1) {
            const float keep = own ? y1 : y0, other = own ? y0 : y1;
            y0 = keep + __shfl_xor_sync(0xffffffffu, other, 1);
#pragma unroll
            for (int o = 2; o < G; o *= 2) y0 += __shfl_xor_sync(0xffffffffu, y0, o);
        }
        y0 += skip0, y1 += skip1;
        if (a.z) y0 *= z0 * sigmoid_fast(z0), y1 *= z1 * sigmoid_fast(z1);
        if (out0) a.y[t * a.D + mine] = from_f<E>(y0);
        if (out1) a.y[t * a.D + c1] = from_f<E>(y1);
    }
}

// What the rows [t0, t1) leave of nothing, v, and the sums of their dt, from the last row back.
// An x or B that is not finite stays in the state for good, whatever its decay: a product
// with 0 keeps it, also where its row is left out.
template <bool VEC, bool RAW, typename E, typename S>
__device__ __forceinline__ float2 leave(const Args<E> &a, float (*bc)[TT][1][S::NP], float (&lost)[S::NP], E *tiles,
                                        float *apart, States<S> &v, const States<S> &nan2, int t0, int t1, int d0, int channels)
{
    constexpr int G = S::G, DPB = S::DPB, TILE = TT * 2 * DPB;
    using R = Ready<E, S>;
    constexpr bool DT = RAW && R::ARRAYS > 0;
    const int tid = threadIdx.x, g = tid % G, c = 2 * (tid / G);
    if (tid < S::NP) lost[tid] = 0.f;
    Share<S, 1> next;
    float bad_b = 0.f;
    auto b_in = [&](int t) { next.read(a, t, t0, t1); };   // rows t .. t + TT - 1
    auto b_out = [&](int buf) {
#pragma unroll
        for (int q = 0; q < next.PER; ++q) bad_b = fmaf(next.v[q], 0.f, bad_b);
        next.write(bc[buf]);
    };
#pragma unroll
    for (int ch = 0; ch < 2; ++ch)
#pragma unroll
        for (int q = 0; q < S::NPAIR; ++q) v[ch][q] = f2(0.f, 0.f);
    b_in(t1 - TT);
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) stage<VEC, 2, DPB>(a, tiles + s * TILE, d0, t1 - (s + 1) * TT, t0, t1);
    b_out(0);
    float2 total = f2(0.f, 0.f), bad_x = f2(0.f, 0.f);
    int buf = 0, at = 0;
    for (int t = t1 - TT; t > t0 - TT; t -= TT, buf ^= 1) {        // rows t .. t + TT - 1
        cp_wait<STAGES - 2>();
        __syncthreads();
        const int ahead = at == 0 ? STAGES - 1 : at - 1;
        stage<VEC, 2, DPB>(a, tiles + ahead * TILE, d0, t - (STAGES - 1) * TT, t0, t1);
        const bool more = t > t0;
        if (more) b_in(t - TT);
        E *tile = tiles + at * TILE;
        const E *row = tile + c;
        if (DT) {
            R::template make<2>(tile, apart, 1, [&](int r, float v) { return t + r >= t0 ? step_of(a.pj, v) : 0.f; });
            __syncwarp();
        }
        float2 sum[TT], bx[TT], least = f2(0.f, 0.f);
        const float2 behind = total;                       // of the rows behind the tile
#pragma unroll
        for (int j = TT - 1; j >= 0; --j) {
            float2 dtv;
            if (DT) dtv = *reinterpret_cast<const float2 *>(R::template at<2>(tile, apart, 1, j, c));
            else dtv = both(row + (2 * j + 1) * DPB);
            if (RAW && !DT) dtv = t + j >= t0 ? f2(step_of(a.pj, dtv.x), step_of(a.pj, dtv.y)) : f2(0.f, 0.f);
            sum[j] = total;                                // of the rows behind
            least = f2(fminf(least.x, dtv.x), fminf(least.y, dtv.y));
            total = add2(total, dtv);
            bx[j] = mul2(dtv, both(row + 2 * j * DPB));
            bad_x = fma2(bx[j], f2(0.f, 0.f), bad_x);
        }
#pragma unroll
        for (int q = 0; q < S::NPAIR; ++q) {
            // With no dt below 0 and a rate that is none either, the tile's largest decay is its last row's.
            bool gone = fminf(least.x, least.y) >= 0.f;
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
                const float r = fmaxf(nan2[ch][q].x, nan2[ch][q].y), top = r * (ch ? behind.y : behind.x);
                if (ch < channels) gone = gone && r <= 0.f && top < GONE;
            }
            if (!__any_sync(0xffffffffu, S::state(g, q) < a.N && channels && !gone)) continue;
#pragma unroll
            for (int j = TT - 1; j >= 0; --j) {
                const float2 Bv = *reinterpret_cast<const float2 *>(&bc[buf][j][0][g * S::NS + 2 * q]);
#pragma unroll
                for (int ch = 0; ch < 2; ++ch) {
                    const float s1 = ch ? sum[j].y : sum[j].x, b1 = ch ? bx[j].y : bx[j].x;
                    const float2 e = ex2x2(mul2(f2(s1, s1), nan2[ch][q]));
                    v[ch][q] = fma2(mul2(e, f2(b1, b1)), Bv, v[ch][q]);
                }
            }
        }
        if (more) b_out(buf ^ 1);
        at = at + 1 < STAGES ? at + 1 : 0;
    }
    cp_wait<0>();
    if (bad_b != bad_b) lost[S::place(tid % S::NP)] = bad_b;         // (whichever of those that found one)
    __syncthreads();
#pragma unroll
    for (int q = 0; q < S::NPAIR; ++q) {
        const float2 bad = *reinterpret_cast<const float2 *>(&lost[g * S::NS + 2 * q]);
        v[0][q] = add2(v[0][q], add2(bad, f2(bad_x.x, bad_x.x)));
        v[1][q] = add2(v[1][q], add2(bad, f2(bad_x.y, bad_x.y)));
    }
    return total;
}

// This lane's states of channels d and d + 1 from p, channel d's; zeros where a channel or state is not there.
template <typename S>
__device__ __forceinline__ void read_states(States<S> &h, const float *p, int N, int g, int channels)
{
#pragma unroll
    for (int ch = 0; ch < 2; ++ch)
#pragma unroll
        for (int q = 0; q < S::NPAIR; ++q) {
            const int n = S::state(g, q);
            h[ch][q] = ch < channels && n < N ? *reinterpret_cast<const float2 *>(p + ch * N + n) : f2(0.f, 0.f);
        }
}

template <typename S>
__device__ __forceinline__ void write_states(const States<S> &h, float *p, int N, int g, int channels)
{
#pragma unroll
    for (int ch = 0; ch < 2; ++ch)
#pragma unroll
        for (int q = 0; q < S::NPAIR; ++q) {
            const int n = S::state(g, q);
            if (ch < channels && n < N) *reinterpret_cast<float2 *>(p + ch * N + n) = h[ch][q];
        }
}

// The rates of the lane's states, 0 where there is none
template <typename S>
__device__ __forceinline__ void read_rates(States<S> &nan2, const float *aneg, int N, int g, int channels, bool raw)
{
    read_states<S>(nan2, aneg, N, g, channels);
#pragma unroll
    for (int ch = 0; ch < 2; ++ch)
#pragma unroll
        for (int q = 0; q < S::NPAIR; ++q) {
            float2 v = nan2[ch][q];
            if (raw) v = f2(softplus(v.x), softplus(v.y));
            nan2[ch][q] = ch < channels && S::state(g, q) < N ? f2(rate_of(v.x), rate_of(v.y)) : f2(0.f, 0.f);
        }
}

// h moved over a segment whose dt have these sums, and what the segment leaves of nothing
template <typename S>
__device__ __forceinline__ void carry(States<S> &h, const States<S> &nan2, float2 sums, const States<S> &v)
{
#pragma unroll
    for (int ch = 0; ch < 2; ++ch) {
        const float s = ch ? sums.y : sums.x;
#pragma unroll
        for (int q = 0; q < S::NPAIR; ++q) h[ch][q] = fma2(ex2x2(mul2(f2(s, s), nan2[ch][q])), h[ch][q], v[ch][q]);
    }
}

template <typename E, typename S, bool REST, bool VEC>
__global__ void __launch_bounds__(THREADS, CTAS)
scan_segments_kernel(const __grid_constant__ Args<E> a)
{
    __shared__ __align__(16) float bc[2 * TT * 2 * S::NP];
    __shared__ __align__(8) float lost[S::NP];
    __shared__ __align__(8) float apart[Ready<E, S>::SIZE];
    extern __shared__ __align__(16) unsigned char rows[];
    E *tiles = reinterpret_cast<E *>(rows);
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
    const bool late = u.segs > 1;                          // its outputs come in the second launch
    if (REST ? !late : u.i > 0 && u.i == u.segs - 1) return;

    const int d0 = (blockIdx.x % a.nd) * S::DPB, d = d0 + 2 * (tid / S::G);
    const int channels = min(2, max(0, a.D - d));          // of the lane's that are there
    const size_t at = channels ? (size_t)d * a.N : 0, DN = (size_t)a.D * a.N;
    States<S> nan2, h;
    read_rates<S>(nan2, a.aneg + at, a.N, g, channels, a.pj.on);
    float *entry = a.entry + u.row * DN + at;
    if (REST && u.i > 0) {
        const bool joined = u.segs > a.chain;
        read_states<S>(h, a.ends + (u.row + (joined ? u.i - 1 : 0)) * DN + at, a.N, g, channels);
        // the first segment's end, then of each one between what was left of it and its own
        constexpr int AT_ONCE = 3;                         // ends that are read at a time
        for (int j = 1; j < u.i && !joined; j += AT_ONCE) {
            States<S> v[AT_ONCE];
            float2 sums[AT_ONCE];
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const int c = j + k < u.i ? channels : 0;
                read_states<S>(v[k], a.ends + (u.row + j + k) * DN + at, a.N, g, c);
                const float *s = a.sums + (size_t)(u.row + j + k) * a.D + d;
                sums[k] = f2(c > 0 ? s[0] : 0.f, c > 1 ? s[1] : 0.f);
            }
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k)
                if (j + k < u.i) carry<S>(h, nan2, sums[k], v[k]);
        }
    } else {
        const long long from = REST || u.i > 0 ? -1 : a.seq.from(u.s);
        const float *src = REST ? entry : a.state + (from >= 0 ? from : 0) * DN + at;
        read_states<S>(h, src, a.N, g, REST || from >= 0 ? channels : 0);
        // (its last segment may write the place that it was read from)
        if (!REST && u.i == 0 && late) write_states<S>(h, entry, a.N, g, channels);
    }
    if (REST || !late) {
        auto tile = reinterpret_cast<float(*)[TT][2][S::NP]>(bc);
        auto all = [&](auto gate, auto raw) {
            walk<VEC, decltype(gate)::value, decltype(raw)::value, E, S>(a, tile, tiles, apart, h, nan2, u.t0, u.t1, d0);
        };
        using Yes = std::true_type;
        using No = std::false_type;
        if (u.t1 - u.t0 <= DIRECT) walk_direct<E, S>(a, h, nan2, u.t0, u.t1, d, channels);
        else if (a.z && a.pj.on) all(Yes{}, Yes{});
        else if (a.z) all(Yes{}, No{});
        else if (a.pj.on) all(No{}, Yes{});
        else all(No{}, No{});
        if (u.i == u.segs - 1) {
            const long long to = a.seq.to(u.s);
            if (to >= 0) write_states<S>(h, a.state + to * DN + at, a.N, g, channels);
            return;
        }
        if (REST) return;
    } else {
        States<S> v;
        auto tile = reinterpret_cast<float(*)[TT][1][S::NP]>(bc);
        const float2 total = a.pj.on ? leave<VEC, true, E, S>(a, tile, lost, tiles, apart, v, nan2, u.t0, u.t1, d0, channels)
                                     : leave<VEC, false, E, S>(a, tile, lost, tiles, apart, v, nan2, u.t0, u.t1, d0, channels);
        float *s = a.sums + (size_t)(u.row + u.i) * a.D + d;
        if (g == 0 && channels > 0) s[0] = total.x;
        if (g == 0 && channels > 1) s[1] = total.y;
        carry<S>(h, nan2, total, v);
    }
    write_states<S>(h, a.ends + (u.row + u.i) * DN + at, a.N, g, channels);
}

// The ends of segments, each from nothing but a sequence's first, become states: h moved over a segment, and
// what it leaves. A thread has four states of a channel; a block a sequence, or the one whose first
// segment is its unit, whichever are fewer; AHEAD segments are on their way at a time.
constexpr int JOIN_THREADS = 128, AHEAD = 12;
template <typename E>
__global__ void __launch_bounds__(JOIN_THREADS)
scan_join_kernel(const __grid_constant__ Args<E> a, int blocks, bool by_sequence)
{
    Unit u;
    if (by_sequence) {
        const int s = blockIdx.x / blocks, start = a.seq.start(s);
        u.row = start / a.seg, u.segs = (a.seq.start(s + 1) - start + a.seg - 1) / a.seg;
        if (u.segs <= a.chain) return;
    } else if (!find_unit(a, blockIdx.x / blocks, u) || u.i > 0 || u.segs <= a.chain) {
        return;
    }
    const int e = (blockIdx.x % blocks * JOIN_THREADS + (int)threadIdx.x) * 4;      // of a place's D * N
    const size_t DN = (size_t)a.D * a.N;
    if (e >= (int)DN) return;
    const int d = e / a.N;
    float4 r = ld4(a.aneg + e);
    if (a.pj.on) r = make_float4(softplus(r.x), softplus(r.y), softplus(r.z), softplus(r.w));
    const float2 n0 = f2(rate_of(r.x), rate_of(r.y)), n1 = f2(rate_of(r.z), rate_of(r.w));
    float *end = a.ends + u.row * DN + e;
    const float *sums = a.sums + (size_t)u.row * a.D + d;
    const float4 first = *reinterpret_cast<const float4 *>(end);
    float2 h0 = lo(first), h1 = hi(first);
    const int n = u.segs - 1;
    for (int j = 1; j < n; j += AHEAD) {
        float4 v[AHEAD];
        float s[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (j + k < n) v[k] = *reinterpret_cast<const float4 *>(end + (j + k) * DN), s[k] = sums[(size_t)(j + k) * a.D];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (j + k >= n) break;
            h0 = fma2(ex2x2(mul2(f2(s[k], s[k]), n0)), h0, lo(v[k]));
            h1 = fma2(ex2x2(mul2(f2(s[k], s[k]), n1)), h1, hi(v[k]));
            st4(end + (j + k) * DN, make_float4(h0.x, h0.y, h1.x, h1.y));
        }
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

// Lane g of a channel's G holds states 4g .. 4g + 3. A CTA takes `per` sequences one after another,
// the next one's state and the places of the one after it on their way meanwhile.
template <typename E, typename BE, int G>
__global__ void __launch_bounds__(TOKEN_THREADS)
scan_token_kernel(const __grid_constant__ Args<E> a, int per)
{
    const BE *Bp = static_cast<const BE *>(a.B), *Cp = static_cast<const BE *>(a.C);
    const int block = blockIdx.x % a.nd;
    const int d = (block * TOKEN_THREADS + (int)threadIdx.x) / G, g = threadIdx.x % G, n = 4 * g;
    const int s0 = blockIdx.x / a.nd * per, s1 = min(a.seq.count, s0 + per);
    const bool chan = d < a.D, act = chan && n < a.N;
    const size_t DN = (size_t)a.D * a.N;
    float *state = a.state + (act ? (size_t)d * a.N + n : 0);
    const int ds = chan ? d : 0, ns = act ? n : 0;
    float4 av = make_float4(0.f, 0.f, 0.f, 0.f);
    if (act) av = ld4(a.aneg + (size_t)d * a.N + n);
    const float skip = a.d_skip && chan ? a.d_skip[d] : 0.f;
    auto from_of = [&](int s) { return s < s1 ? (int)a.seq.from(s) : -1; };
    auto state_of = [&](int from) {
        return act && from >= 0 ? *reinterpret_cast<const float4 *>(state + from * DN) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    int from = from_of(s0), from_next = from_of(s0 + 1), to = (int)a.seq.to(s0);
    float4 hv = state_of(from);
    if (a.pj.on) av = make_float4(softplus(av.x), softplus(av.y), softplus(av.z), softplus(av.w));
    const float2 n0 = f2(rate_of(av.x), rate_of(av.y)), n1 = f2(rate_of(av.z), rate_of(av.w));
    for (int s = s0; s < s1; ++s) {
        float4 Bv = four(Bp + s * a.ldB + ns), Cv = four(Cp + s * a.ldC + ns);
        const float xv = to_f(a.x[s * a.ldx + ds]);
        float dtv = to_f(a.dt[s * a.lddt + ds]), zv = 0.f;
        if (a.z) zv = to_f(a.z[s * a.ldz + ds]);
        const float4 h_next = state_of(from_next);
        const int to_next = s + 1 < s1 ? (int)a.seq.to(s + 1) : -1;
        from_next = from_of(s + 2);
        if (a.pj.on) dtv = fmaf(a.pj.range, sigmoid_fast(dtv), a.pj.lo);
        const float2 dt2 = f2(dtv, dtv), bx2 = f2(dtv * xv, dtv * xv);
        const float2 h0 = fma2(ex2x2(mul2(dt2, n0)), lo(hv), mul2(bx2, lo(Bv)));
        const float2 h1 = fma2(ex2x2(mul2(dt2, n1)), hi(hv), mul2(bx2, hi(Bv)));
        if (act && to >= 0) st4(state + to * DN, make_float4(h0.x, h0.y, h1.x, h1.y));
        const float2 acc = fma2(hi(Cv), h1, mul2(lo(Cv), h0));
        float yv = act ? acc.x + acc.y : 0.f;
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) yv += __shfl_xor_sync(0xffffffffu, yv, o, G);
        yv += skip;
        if (a.z) yv *= zv * sigmoid_fast(zv);
        if (chan && g == 0) a.y[(long long)s * a.D + d] = from_f<E>(yv);
        hv = h_next, to = to_next;
    }
}

// ----------------------------------------------------------------- launch

// Lanes that share two channels in the segments' launches.
int lanes_of(int N) { return N <= 8 ? 1 : N <= 16 ? 2 : N <= 32 ? 4 : 8; }

long long channel_blocks(int D, int N)
{
    const int dpb = 2 * THREADS / lanes_of(N);
    return (D + dpb - 1) / dpb;
}

// Rows of a segment: as few as give every SM its CTAs when the rows belong to one sequence, at
// least 32, a whole number of tiles. (Half as many: 16384 x 2048 x 16, one prompt, 293 for 276 us; 8192 x
// 2304 x 16, 16 prompts of four draws, 212 for 205; 16384 x 2048 x 16, 32 prompts, bf16, 414 for 426. At least 64: 2048 x 1432 x
// 16, one prompt, 78 for 66 us.)
int segment_rows(int rows, int D, int N)
{
    const long long nd = channel_blocks(D, N);
    const long long want = std::max<long long>(1, (long long)CTAS * N_SM / nd);
    const long long seg = std::max<long long>(32, (rows + want - 1) / want);
    return (int)std::min<long long>((seg + TT - 1) / TT * TT, 1 << 30);
}

// A call's units and its workspace (bytes from the start, regions of whole 256 bytes):
// segments before the last of their sequence, of which there is at most one for every `seg`
// rows, and as many entries of sequences.
struct Plan {
    int seg;
    long long nd, fulls, units;
    bool more;                          // a sequence can have a second segment
    size_t sums = 0, entry = 0, total = 0;
    Plan(int rows, int count, int D, int N) : seg(segment_rows(rows, D, N)) {
        nd = channel_blocks(D, N);
        fulls = rows / seg, units = fulls + count;
        more = rows > seg;
        const size_t ends = fulls, d = D;
        auto up = [](size_t n) { return (n + 255) / 256 * 256; };
        sums = up(ends * d * N * 4);
        entry = sums + up(ends * d * 4);
        total = !more ? 0 : entry + up(ends * d * N * 4);
    }
};

template <typename E>
Args<E> args_of(const ScanPackedArgs &p)
{
    Args<E> a{};
    a.x = (const E *)p.x, a.dt = (const E *)p.dt, a.z = (const E *)p.z;
    a.B = p.B, a.C = p.C, a.bc_bf16 = p.bc_bf16;
    a.ldx = p.ldx, a.lddt = p.lddt, a.ldB = p.ldB, a.ldC = p.ldC, a.ldz = p.ldz;
    a.aneg = p.aneg, a.d_skip = p.d_skip, a.state = p.state, a.y = (E *)p.y;
    a.seq = p.seq, a.D = p.D, a.N = p.N, a.pj = p.proj;
    return a;
}

// the tiles of the widest CTA (256 channels, N up to 8, float32 with a gate)
constexpr size_t MAX_TILES = (size_t)STAGES * TT * 3 * 2 * THREADS * sizeof(float);

template <typename E, typename S>
cudaError_t segments_of(const ScanPackedArgs &p, cudaStream_t stream)
{
    Args<E> a = args_of<E>(p);
    const Plan plan(p.seq.rows, p.seq.count, p.D, p.N);
    char *ws = static_cast<char *>(p.workspace);
    const bool joined = plan.fulls >= 2 * MANY || plan.fulls >= MANY + p.seq.count;
    a.seg = plan.seg, a.nd = (int)plan.nd, a.chain = joined ? CHAIN : 0x7fffffff, a.fulls = (int)plan.fulls, a.units = (int)plan.units;
    a.ends = (float *)ws, a.sums = (float *)(ws + plan.sums), a.entry = (float *)(ws + plan.entry);
    const long long clear = 2 * N_SM, blocks = plan.units * plan.nd;
    const long long sequences = std::min<long long>(plan.fulls, p.seq.count);      // that can have several segments
    const int joins = (int)(((long long)p.D * p.N / 4 + JOIN_THREADS - 1) / JOIN_THREADS);
    if (blocks + clear > 0x7fffffffLL || sequences * joins > 0x7fffffffLL) return cudaErrorInvalidValue;
    auto launch = [&](auto vec) {
        constexpr bool VEC = decltype(vec)::value;
        const size_t smem = (size_t)STAGES * TT * (a.z ? 3 : 2) * S::DPB * sizeof(E);
        cudaError_t e = smem_opt_in<scan_segments_kernel<E, S, false, VEC>>(MAX_TILES);
        if (e == cudaSuccess) e = smem_opt_in<scan_segments_kernel<E, S, true, VEC>>(MAX_TILES);
        if (e != cudaSuccess) return e;
        scan_segments_kernel<E, S, false, VEC><<<(unsigned)(blocks + clear), THREADS, smem, stream>>>(a);
        e = cudaGetLastError();
        if (e != cudaSuccess || !plan.more) return e;
        if (joined) {
            scan_join_kernel<E><<<(unsigned)(sequences * joins), JOIN_THREADS, 0, stream>>>(a, joins, sequences < plan.fulls);
            e = cudaGetLastError();
            if (e != cudaSuccess) return e;
        }
        scan_segments_kernel<E, S, true, VEC><<<(unsigned)blocks, THREADS, smem, stream>>>(a);
        return cudaGetLastError();
    };
    // whole 16 bytes of rows
    auto whole = [&](const void *p, long long ld) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (long long)sizeof(E) % 16 == 0;
    };
    if (p.D * sizeof(E) % 16 == 0 && whole(p.x, p.ldx) && whole(p.dt, p.lddt) && (!p.z || whole(p.z, p.ldz)))
        return launch(std::true_type{});
    return launch(std::false_type{});
}

template <typename E, typename BE, int G>
cudaError_t tokens_of(const ScanPackedArgs &p, cudaStream_t stream)
{
    Args<E> a = args_of<E>(p);
    a.nd = (p.D * G + TOKEN_THREADS - 1) / TOKEN_THREADS;
    // as many sequences a CTA, up to 8, as leave every SM 8 CTAs
    const int per = (int)std::min<long long>(8, std::max<long long>(1, (long long)a.nd * p.seq.count / (8 * N_SM)));
    const long long blocks = (long long)a.nd * ((p.seq.count + per - 1) / per);
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    scan_token_kernel<E, BE, G><<<(unsigned)blocks, TOKEN_THREADS, 0, stream>>>(a, per);
    return cudaGetLastError();
}

template <typename E, typename BE>
cudaError_t tokens_by_states(const ScanPackedArgs &p, cudaStream_t stream)
{
    switch (groups_for(p.N)) {
    case 1: return tokens_of<E, BE, 1>(p, stream);
    case 2: return tokens_of<E, BE, 2>(p, stream);
    case 4: return tokens_of<E, BE, 4>(p, stream);
    case 8: return tokens_of<E, BE, 8>(p, stream);
    default: return tokens_of<E, BE, 16>(p, stream);
    }
}

template <typename E>
cudaError_t segments_by_states(const ScanPackedArgs &p, cudaStream_t stream)
{
    if (p.N <= 4) return segments_of<E, Split<4, 1>>(p, stream);
    if (p.N <= 8) return segments_of<E, Split<8, 1>>(p, stream);
    if (p.N <= 16) return segments_of<E, Split<8, 2>>(p, stream);
    if (p.N <= 32) return segments_of<E, Split<8, 4>>(p, stream);
    return segments_of<E, Split<8, 8>>(p, stream);
}

}  // namespace

}  // namespace mms
