// The matrix products of the head's losses on the 5th-generation tensor cores,
// with what follows them on a tile (MmKind in mms_head.h).
//
// A CTA pair computes tiles of 256 rows and up to 256 columns: each CTA holds
// 128 rows of a and half the columns' b in shared memory (6 stages of 64
// summed elements, 32 KB each, filled by TMA with the 128-byte swizzle), one
// thread of the leader issues tcgen05.mma.cta_group::2, and each CTA's 128
// rows of the product stand in its tensor memory, in two buffers of 256
// columns, so that the multiplies of the next tile run under the epilogue of
// this one. Persistent: one pair per two SMs walks the tiles.
//
// Warps: 0..7 epilogue (a warp reads the 32 lanes of its number mod 4; the two
// halves of the columns go to two warps), 8 loads, 9 multiplies (leader) and
// owns the tensor memory. The epilogue's two warpgroups take registers from
// the third one (168 a thread at launch -> 224 and 56: 2 x 224 + 56 = 3 x 168).
//
// Measured at 8192 x 131072 x 2048, bf16 (4.4 TFLOP each): log-sum-exp 3.2 ms,
// dz 3.1, dx 3.5, dw 3.9 (1.37, 1.41, 1.26, 1.13 PFLOP/s; the library's
// sustained rate is 1.38). Without the epilogues' work they run at 1.6; what
// bounds them is power and the copies from L2, 45 to 50 bytes a clock and SM.
// Four stages measure the same as six.
//
// Tile order: the dimension with fewer tiles runs fastest, in groups of 16,
// so the concurrent tiles share one side's panels in L2 and the long side is
// read from HBM once.
//
// float32 factors are two fp16 planes each (see mms_head.cu) and a product the
// sum of three of their products (not the second by the second). A stage then
// holds both planes of both factors (3 stages of 64 KB) and each is copied
// once for its three uses: 64 KB for 12 multiplies where one pair of planes
// after the other takes 96 KB. At 8192 x 32768 x 640 that is 3.1 ms for the
// four products against 3.6: the copies no longer bound them.
//
// The tensor core adds each 16 summed elements to its fp32 sum with truncation,
// not rounding, so a long sum drifts towards zero: each addition loses up to
// 2^-23 of the sum so far (measured: 1.1e-5 of a result at 8192 elements, 1.1e-3
// at 262144). The sum is therefore cut into parts: each
// goes to its own tensor memory buffer and the epilogue warps add the parts up
// in registers, rounding to nearest (`PARTS`). Where the result stays float32,
// parts of 512 cost nothing beside the multiplies; of 256, 25 % of the
// log-sum-exp at 8192 x 131072 x 2048 (4.15 ms against 3.31); of 128, 80 %. With
// two planes by two each
// element is added three times, so parts are of 256 (3.17 ms for the four
// products; of 384 3.06 ms but errors up to 1.5e-6, of 192 3.37 ms). Where 16
// bits are kept of the result, sums of more than 2048 elements are cut into parts
// of as many (a drift of 2^-16 at most, and so the backward's q of 2^-16 of its
// logit). At 8192 x 131072 x 2048, forward and backward, that is within the spread of
// runs (16.0 ms; dx and dw alone take 7 % more where power does not bound them);
// parts of 512 for dz too would be 5 % more, everywhere 8 %.
//
// The epilogue turns a warp's 32 rows x 32 columns through shared memory, in
// 16-byte pieces (16-bit results already rounded and packed), so that its
// stores and the reads of `acc` cover whole sectors of a row. Its arithmetic
// is on packed pairs with independent sums. At 8192 x 32768 x 64 (bf16), where
// it is all there is, a tile of the log-sum-exp takes 6.2 k clocks and of dz
// 8.0 k (7.0 and 10 k with scalar sums and turns; the exponentials alone
// 2.0 k); under a product of 2048 elements, 16.4 k, it is hidden. Loading the
// next 32 columns of tensor memory ahead measured the same, and spilled.
//
// Tiles that do not fill a last round of the 74 pairs are split along the
// summed dimension; their partial sums go to a workspace that a second kernel
// adds up in order.
//
// Every wait is bounded. A wait that runs out sets a flag for
// mms_device_status; all roles leave, the leader waits (bounded) for the
// copies in flight, and the pair leaves together.
#include <cuda_fp16.h>

#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "mms_common.cuh"
#include "mms_head.h"
#include "mms_kernels.h"
#include "mms_stage.cuh"
#include "mms_tma.cuh"
#include "mms_umma.cuh"

namespace mms {

namespace {

constexpr int TM = 256, BK = 64, THREADS = 384;
constexpr int HALF = 16384;                                  // bytes of one CTA's a (or b) per stage
constexpr int GROUP = 16;
constexpr int PART = 512;                                    // summed elements per part
constexpr int PART_BOTH = 256;                               // the same for two planes by two
constexpr int PART_LONG = 2048;                              // the same where 16 bits are kept of the result
constexpr int TURN = 32 * 33;                                // floats of a warp's tile to turn
// Stages: two planes by two stand side by side in one stage, and are read once for all three passes.
constexpr int STAGE_BYTES = 6 * 2 * HALF;                    // of all stages
constexpr size_t SMEM = 1024 + (size_t)STAGE_BYTES + 8 * TURN * 4;

__device__ unsigned int g_mm_timeout;

struct Tiles {
    int mt, nt, bn;         // tiles of rows and columns, columns per tile (a multiple of 32)
    int half;               // of them, columns of the first four epilogue warps (at most 128)
    int whole, splits;      // tiles done by one item each; items of every other tile
    int items;
    int steps, kb;          // steps of BK summed elements, and of them in an item of a split tile
    int part;               // steps per part of a sum
};

int passes_of(int planes_a, int planes_b) { return planes_a + planes_b - 1; }

// Columns per tile and splits of the tiles beyond whole rounds: the cheapest
// by a model of a pair's clocks. A step of 64 summed elements is the larger of
// the multiplies (2 clocks a column, at full rate) and the copies of 16 KB +
// 64 bytes a column into each CTA; two planes by two need fewer copies, but
// narrow tiles pay there for the parts (d = 640: dx 0.88 ms at 128 columns,
// 0.71 at 224), so the same model serves; an item ends with an epilogue that nothing
// overlaps on the last one. Splits pay a write and a read of their partial
// sums and one more launch.
Tiles plan(MmKind kind, int m, int n, int k, int passes, size_t split_bytes)
{
    constexpr int PAIRS = N_SM / 2;
    Tiles best{};
    double least = 0;
    for (int bn = 256; bn >= 64; bn -= 32) {
        Tiles q;
        q.mt = (m + TM - 1) / TM;
        q.nt = (n + bn - 1) / bn;
        q.bn = bn;
        q.half = bn > 128 ? 128 : (bn / 2 + 31) / 32 * 32;
        q.steps = (k + BK - 1) / BK;
        const int tiles = q.mt * q.nt, rest = tiles % PAIRS;
        const double step = std::max(2.0 * bn, 234 + 0.92 * bn) * passes;
        const double whole = (double)(tiles / PAIRS) * (q.steps * step + 300);
        for (int s = 1; s <= (kind == MM_OUT && rest ? PAIRS : 1); ++s) {
            q.kb = (q.steps + s - 1) / s;
            if (s > 1 && (q.kb < 4 || rest * s > 4 * PAIRS || (size_t)rest * s * TM * bn * 4 > split_bytes)) break;
            q.splits = (q.steps + q.kb - 1) / q.kb;
            if (q.splits != s) continue;
            q.whole = s > 1 ? tiles - rest : tiles;
            q.items = q.whole + (tiles - q.whole) * s;
            double cost = whole + (rest * s + PAIRS - 1) / PAIRS * (q.kb * step + 300) + 1500 + 10 * bn;
            if (s > 1) cost += 5000 + 2.0 * rest * s * TM * bn * 4 / 3000;
            if (!best.mt || cost < 0.97 * least) {
                best = q;
                least = cost;
            }
        }
    }
    return best;
}

// Tile number t as (row tile, column tile).
__device__ __forceinline__ void tile_of(const Tiles &q, int t, int &mi, int &ni) {
    const bool rows_fast = q.mt <= q.nt;
    const int fast = rows_fast ? q.mt : q.nt, slow = rows_fast ? q.nt : q.mt;
    const int g = t / (GROUP * slow), base = g * GROUP;
    const int w = min(GROUP, fast - base), r = t - g * GROUP * slow;
    const int f = base + r % w, s = r / w;
    mi = rows_fast ? f : s;
    ni = rows_fast ? s : f;
}

// The rows and steps that are live (MmArgs::live): rows of results, rows that
// tiles cover (at least one tile, so that there is something to write), steps.
struct Live {
    int rows, tile_rows, steps;
};
template <bool AT>
__device__ __forceinline__ Live live_of(const MmArgs &a, const Tiles &q) {
    const int n = a.live ? *a.live : INT_MAX;
    if (AT) return Live{a.m, a.m, min(q.steps, max(1, (min(n, a.k) + BK - 1) / BK))};
    return Live{min(a.m, n), min(a.m, max(1, n)), q.steps};
}

// The plan for the live rows: their tiles alone, dense over the pairs; those
// beyond whole rounds split into up to LIVE_ITEMS items.
constexpr int LIVE_ITEMS = 4 * N_SM / 2;
template <int KIND, bool AT>
__device__ __forceinline__ Tiles live_plan(const MmArgs &a, Tiles q, const Live &l) {
    if (AT || !a.live) return q;
    constexpr int PAIRS = N_SM / 2;
    q.mt = (l.tile_rows + TM - 1) / TM;
    const int tiles = q.mt * q.nt, rest = tiles % PAIRS;
    q.whole = q.items = tiles;
    q.splits = 1;
    if (KIND == MM_OUT && rest && (size_t)LIVE_ITEMS * TM * q.bn * 4 <= a.split_bytes) {
        // rounds of items times their steps; partial sums cost 8 steps for the launch and a third
        // of one (256 KB written and read) for each item
        int least = q.steps, best = 1;
        for (int i = 2; i <= 9; ++i) {
            const int s = i == 9 ? PAIRS / rest : i;
            if (s < 2 || rest * s > LIVE_ITEMS || s * 4 > q.steps) continue;
            const int cost = (rest * s + PAIRS - 1) / PAIRS * ((q.steps + s - 1) / s) + 8 + rest * s / 3;
            if (cost < least) {
                least = cost;
                best = s;
            }
        }
        q.kb = (q.steps + best - 1) / best;
        q.splits = (q.steps + q.kb - 1) / q.kb;
        if (q.splits > 1) {
            q.whole = tiles - rest;
            q.items = q.whole + rest * q.splits;
        }
    }
    return q;
}

// Item t: its tile, and its steps of the sum; `split` its number among the
// items of split tiles, or -1.
// False if there is nothing to do: no live rows in the tile, or no live steps in the item.
__device__ __forceinline__ bool item_of(const Tiles &q, const Live &l, int t, int &mi, int &ni, int &split,
                                        int &begin, int &end) {
    int tile;
    if (t < q.whole) {
        tile = t;
        split = -1;
        begin = 0;
        end = l.steps;
    } else {
        split = t - q.whole;
        tile = q.whole + split / q.splits;
        begin = split % q.splits * q.kb;
        end = min(l.steps, begin + q.kb);
    }
    tile_of(q, tile, mi, ni);
    return mi * TM < l.tile_rows && begin < end;
}

__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, uint32_t limit) {
    for (uint32_t i = 0; i < limit; ++i)
        if (mbar_try(bar, parity)) return true;
    return false;
}

// The planes of pass c of (planes_a, planes_b): the last pass is (0, 0), before
// it (0, 1) if b has two, and first (1, 0).
__device__ __forceinline__ void planes_of(int passes, int c, int &pa, int &pb) {
    pa = passes > 1 && c == 0;
    pb = passes > 2 && c == 1;
}

// v[i] without an indexed register file: halves of the candidates by each bit of i.
__device__ __forceinline__ float pick32(const float (&v)[32], int i) {
    float t[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) t[j] = i & 16 ? v[j + 16] : v[j];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = i & 8 ? t[j + 8] : t[j];
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = i & 4 ? t[j + 4] : t[j];
#pragma unroll
    for (int j = 0; j < 2; ++j) t[j] = i & 2 ? t[j + 2] : t[j];
    return i & 1 ? t[1] : t[0];
}

// What follows the product on 32 columns of one row per lane.
template <int KIND>
struct Epilogue {
    float f;                    // the product's factor
    float mx, s;                // MM_LSE: running maximum and sum
    int at, nth;                // MM_LSE: the next column whose product is asked for, its number in the list
    float2 lse2;                // MM_GRAD
    float rs;
    int rows;                   // rows of results
    __device__ __forceinline__ void next(const MmArgs &a, int m) {
        const int c = nth < a.lists.k ? a.lists.col[(size_t)m * a.lists.k + nth] : INT_MAX;
        at = c == INT_MAX ? c : c - a.first_col;
    }
    // m: this lane's row, n: the first column that this warp will see
    __device__ __forceinline__ void begin(const MmArgs &a, const Live &l, int m, int n) {
        // dz's padding rows up to the tile's end are written too
        rows = KIND == MM_GRAD ? min(a.m, (l.tile_rows + TM - 1) / TM * TM) : l.rows;
        const bool in = m < rows;
        f = a.c;
        if (a.row_mul) f *= in ? a.row_mul[m] : 0.f;
        if (a.mul) f *= *a.mul;
        if (KIND == MM_LSE) {
            mx = -INFINITY;
            s = 0.f;
            at = INT_MAX;
            nth = 0;
            // as 0 it would make NaN of the -inf behind the last column; the products it stands for are below 2^-60
            f = fmaxf(f, 1.17549435e-38f);
            if (a.target && in) {
                const long long t = a.target[a.row_of ? a.row_of[m] : m] - a.first_col;
                if (t >= 0 && t < a.n) at = (int)t;
            }
            if (a.lists.col && in && n < a.n) {
                nth = a.lists.before[(size_t)((a.first_col + n) / LIST_BLOCK) * a.lists.rows + m];
                next(a, m);
            }
        }
        if (KIND == MM_GRAD) {
            lse2 = in ? a.lse2[m] : make_float2(0.f, 0.f);
            rs = in ? a.rs[m] : 0.f;
            if (rs != 0.f && a.g_unit != 0.f) rs = a.g_unit;
        }
    }
    __device__ static __forceinline__ size_t out_row(const int *row_of, int m0, int r) {
        return row_of ? row_of[r] : m0 + r;
    }
    // m0: the row of lane 0; rows and columns beyond the product are left out.
    __device__ __forceinline__ void chunk(const MmArgs &a, const Tiles &q, int split, int m0, int n, int tile_col,
                                          float (&v)[32], float *turn) {
        if (n >= a.n || (KIND != MM_LSE && m0 >= rows)) return;        // the whole warp
        if (KIND == MM_LSE) {
            lse(a, m0, n, v);
            return;
        }
        const int lane = threadIdx.x % 32, left = min(32, rows - m0), cols = min(32, a.n - n);
        const float2 fp = f2(f, f);
        if (KIND == MM_GRAD) {
            const float2 x = f2(-lse2.x, -lse2.x), y = f2(-lse2.y, -lse2.y), r = f2(rs, rs);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
                const float2 e = ex2x2(add2(fma2(f2(v[i], v[i + 1]), fp, x), y)), g = mul2(r, e);
                v[i] = g.x;
                v[i + 1] = g.y;
            }
            if (__any_sync(~0u, rs == 0.f))
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = rs == 0.f ? 0.f : v[i];
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = pack(a.fp16, v[2 * i], v[2 * i + 1]);
            uint16_t *g = a.g + (size_t)m0 * a.ldg + n;
            turn16(w, turn, left, (cols + 7) / 8, g, a.ldg, nullptr, 0);
            if (a.gplanes > 1) {
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = pack_rest(a.fp16, v[2 * i], v[2 * i + 1], w[i]);
                turn16(w, turn, left, (cols + 7) / 8, g + a.gplane, a.ldg, nullptr, 0);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const float2 p = mul2(f2(v[i], v[i + 1]), fp);
            v[i] = p.x;
            v[i + 1] = p.y;
        }
        const int *row_of = a.row_of ? a.row_of + m0 : nullptr;
        if (split < 0 && a.out_bf16 && !a.acc && cols == 32 && a.n % 8 == 0) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = pack(false, v[2 * i], v[2 * i + 1]);
            turn16(w, turn, left, 4, static_cast<uint16_t *>(a.out) + n, a.n, row_of, m0);
            return;
        }
        __syncwarp();
        const float *acc = a.acc ? a.acc + (size_t)m0 * a.n + n : nullptr;
        if (split < 0 && (cols < 32 || a.n % (a.out_bf16 ? 8 : 4))) {
            // ragged columns, or rows that do not start at whole pieces: a row at a time
#pragma unroll
            for (int i = 0; i < 32; ++i) turn[lane * 33 + i] = v[i];
            __syncwarp();
            if (lane >= cols) return;
            const auto store = [&](auto *out) {
                using O = typename std::remove_pointer<decltype(out)>::type;
                if (row_of || acc || left < 32) {
#pragma unroll 4
                    for (int r = 0; r < left; ++r)
                        out[out_row(row_of, m0, r) * a.n + n + lane] =
                            from_f<O>(turn[r * 33 + lane] + (acc ? acc[(size_t)r * a.n + lane] : 0.f));
                } else {
                    O *p = out + (size_t)m0 * a.n + n + lane;
#pragma unroll
                    for (int r = 0; r < 32; ++r) p[(size_t)r * a.n] = from_f<O>(turn[r * 33 + lane]);
                }
            };
            if (a.out_bf16) store(static_cast<__nv_bfloat16 *>(a.out));
            else store(static_cast<float *>(a.out));
            return;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            st4(turn + lane * 32 + ((j ^ (lane & 7)) << 2), make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
        __syncwarp();
        const int c = lane % 8 * 4;                            // 4 columns, 4 rows at a time
        if (split >= 0) {
            float *p = a.split + ((size_t)split * TM + m0 % TM) * q.bn + tile_col + c;
#pragma unroll
            for (int r = lane / 8; r < 32; r += 4) st4(p + (size_t)r * q.bn, turned(turn, r, lane % 8));
            return;
        }
#pragma unroll
        for (int r = lane / 8; r < 32; r += 4) {
            if (r >= left) break;
            float4 w = turned(turn, r, lane % 8);
            if (acc) {
                // not through the read-only path: out may be the same array
                const float4 t = *reinterpret_cast<const float4 *>(acc + (size_t)r * a.n + c);
                w = make_float4(w.x + t.x, w.y + t.y, w.z + t.z, w.w + t.w);
            }
            const size_t o = out_row(row_of, m0, r) * a.n + n + c;
            if (a.out_bf16)
                *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + o) =
                    make_uint2(pack(false, w.x, w.y), pack(false, w.z, w.w));
            else
                st4(static_cast<float *>(a.out) + o, w);
        }
    }
    __device__ static __forceinline__ float4 turned(const float *turn, int r, int piece) {
        return *reinterpret_cast<const float4 *>(turn + r * 32 + ((piece ^ (r & 7)) << 2));
    }
    __device__ static __forceinline__ uint32_t pack(bool fp16, float x, float y) {
        if (fp16) {
            const __half2 h = __floats2half2_rn(x, y);
            return *reinterpret_cast<const uint32_t *>(&h);
        }
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    // what the 16-bit parts in p left of x and y
    __device__ static __forceinline__ uint32_t pack_rest(bool fp16, float x, float y, uint32_t p) {
        float2 h;
        if (fp16) h = __half22float2(*reinterpret_cast<const __half2 *>(&p));
        else h = f2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u));
        return pack(fp16, x - h.x, y - h.y);
    }
    // This lane's row of 32 16-bit values to rows of `out` (at its column n) with stride ld, 4 lanes a
    // row: `pieces` of 8 columns, `left` rows. In shared memory piece j of row r lies at j ^ (r / 2 % 4).
    __device__ static __forceinline__ void turn16(const uint32_t (&w)[16], float *turn, int left, int pieces,
                                                  uint16_t *out, long long ld, const int *row_of, int m0) {
        const int lane = threadIdx.x % 32;
        uint4 *t = reinterpret_cast<uint4 *>(turn);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j)
            t[lane * 4 + (j ^ (lane >> 1 & 3))] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        __syncwarp();
        const int j = lane % 4;
        if (j >= pieces) return;
#pragma unroll
        for (int r = lane / 4; r < 32; r += 8)
            if (r < left)
                *reinterpret_cast<uint4 *>(out + out_row(row_of, m0, r) * ld + 8 * j) = t[r * 4 + (j ^ (r >> 1 & 3))];
    }
    __device__ __forceinline__ void lse(const MmArgs &a, int m0, int n, float (&v)[32]) {
        if (n + 32 > a.n)
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (n + i >= a.n) v[i] = -INFINITY;
        float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int i = 4; i < 32; ++i) top[i % 4] = fmaxf(top[i % 4], v[i]);
        while (at < n + 32) {
            const int m = m0 + threadIdx.x % 32;
            if (at >= n) {
                const size_t to = a.target ? m : (size_t)m * a.lists.k + a.lists.pos[(size_t)m * a.lists.k + nth];
                const float z = pick32(v, at - n), p = z * f;
                a.at[to] = p;
                a.rest[to] = rounding_of(z, f, p);
            }
            if (a.target) {
                at = INT_MAX;
            } else {
                ++nth;
                next(a, m);
            }
        }
        const float now = fmaxf(mx, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * f);   // f > 0
        const float ref = now == -INFINITY ? 0.f : now;
        const float2 fp = f2(f, f), rp = f2(-ref, -ref);
        float2 t[4];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float2 e = ex2x2(fma2(f2(v[2 * i], v[2 * i + 1]), fp, rp));
            t[i % 4] = i < 4 ? e : add2(t[i % 4], e);
        }
        const float2 u = add2(add2(t[0], t[1]), add2(t[2], t[3]));
        s = fmaf(s, ex2(mx - ref), u.x + u.y);
        mx = now;
    }
    __device__ __forceinline__ void end(const MmArgs &a, int m, int i) {
        if (KIND == MM_LSE && m < rows) a.part[(size_t)i * a.m + m] = make_float2(mx, s);
    }
};

template <int KIND, bool AT, bool BT, bool PARTS, bool BOTH>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
mm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
          const MmArgs a, const Tiles planned, uint32_t limit, int skip)
{
    chain_next();
    constexpr int STAGES = BOTH ? 3 : 6, PLANES = BOTH ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[2 * STAGES + 5];
    __shared__ uint32_t tmem_slot;
    __shared__ int failed, issued;
    const uint32_t tiles = (smem_u32(smem_raw) + 1023) / 1024 * 1024;
    const uint32_t rank = cluster_rank();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t full = smem_u32(bars), empty = full + 8 * STAGES, tfull = empty + 8 * STAGES,
                   tempty = tfull + 16, drain = tempty + 16;

    if (threadIdx.x == 0) {
        failed = issued = 0;
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(tfull + 8 * i, 1);
            mbar_init(tempty + 8 * i, 16);           // 8 epilogue warps of each CTA
        }
        mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 9) tmem_alloc_pair(smem_u32(&tmem_slot));
    umma_fence_before();
    __syncthreads();
    cluster_sync();
    umma_fence_after();
    chain_wait();
    asm volatile("fence.proxy.async.global;\n" ::: "memory");      // the copies read what kernels before have stored
    const uint32_t tmem = tmem_slot;
    const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;
    const int passes = BOTH ? 1 : a.a.planes + a.b.planes - 1;      // over the stages
    const int bhalf = planned.bn / 2;
    const int bblocks = BT ? (bhalf + 63) / 64 : 0;
    const Live live = live_of<AT>(a, planned);
    const Tiles q = live_plan<KIND, AT>(a, planned, live);

    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
    if (warp == 8 && lane == 0) {
        const uint32_t b_bytes = BT ? bblocks * 8192u : bhalf * 128u;
        int it = 0;
        bool ok = true;
        for (int t = pair; ok && t < q.items; t += pairs) {
            int split, k_begin, k_end, mi, ni;
            if (!item_of(q, live, t, mi, ni, split, k_begin, k_end)) continue;
            const int m0 = mi * TM + rank * 128, n0 = ni * q.bn + rank * bhalf;
            // the second CTA may have no rows: its part of a then stays as it is, and so does its product
            const bool some = m0 < live.tile_rows;
            const uint32_t a_bytes = HALF + (mi * TM + 128 < live.tile_rows ? HALF : 0);
            for (int k_first = k_begin; ok && k_first < k_end; k_first += q.part)
            for (int c = 0; ok && c < passes; ++c) {
                int pa, pb;
                planes_of(passes, c, pa, pb);
                for (int kb = k_first; kb < min(k_end, k_first + q.part); ++kb, ++it) {
                    const int st = it % STAGES;
                    if (!wait_bar(empty + 8 * st, ((it / STAGES) & 1) ^ 1, limit)) {
                        ok = false;
                        break;
                    }
                    if (it == skip) continue;
                    const uint32_t bar = leader_addr(full + 8 * st);
                    if (rank == 0) mbar_expect(full + 8 * st, PLANES * (a_bytes + 2 * b_bytes));
                    const uint32_t sa = tiles + st * PLANES * 2 * HALF, sb = sa + PLANES * HALF;
                    const int k0 = kb * BK;
#pragma unroll
                    for (int p = 0; p < PLANES; ++p) {
                        const uint32_t da = sa + p * HALF, db = sb + p * HALF;
                        if (BOTH) pa = pb = p;
                        if (!some) {
                        } else if (AT) {
                            tma3_pair(da, &map_a, m0, k0, pa, bar);
                            tma3_pair(da + 8192, &map_a, m0 + 64, k0, pa, bar);
                        } else {
                            tma3_pair(da, &map_a, k0, m0, pa, bar);
                        }
                        if (BT) {
                            for (int b = 0; b < bblocks; ++b)
                                tma3_pair(db + b * 8192, &map_b, n0 + 64 * b, k0, pb, bar);
                        } else {
                            tma3_pair(db, &map_b, k0, n0, pb, bar);
                        }
                    }
                    issued = it + 1;
                }
            }
        }
        if (!ok) failed = 1;
    } else if (warp == 9 && lane == 0 && rank == 0) {
        const uint32_t idesc = umma_idesc(q.bn, a.fp16, AT, BT);
        int it = 0, use = 0;
        bool ok = true;
        for (int t = pair; ok && t < q.items; t += pairs) {
        int split, k_begin, k_end, mi, ni;
        if (!item_of(q, live, t, mi, ni, split, k_begin, k_end)) continue;
        for (int k_first = k_begin; k_first < k_end; k_first += q.part, ++use) {
            const int buf = use & 1;
            if (!wait_bar(tempty + 8 * buf, ((use >> 1) & 1) ^ 1, limit)) {
                ok = false;
                break;
            }
            umma_fence_after();
            const int steps = passes * min(q.part, k_end - k_first);
            for (int i = 0; i < steps; ++i, ++it) {
                const int st = it % STAGES;
                if (!wait_bar(full + 8 * st, (it / STAGES) & 1, limit)) {
                    ok = false;
                    break;
                }
                umma_fence_after();
                const uint32_t sa = tiles + st * PLANES * 2 * HALF, sb = sa + PLANES * HALF;
#pragma unroll
                for (int c = 0; c < (BOTH ? 3 : 1); ++c) {      // (1, 0), (0, 1), (0, 0): the small products first
                    const uint32_t pa = sa + (BOTH && c == 0 ? HALF : 0), pb = sb + (BOTH && c == 1 ? HALF : 0);
                    const uint64_t da = AT ? umma_desc(pa, 8192, 1024) : umma_desc(pa, 16, 1024);
                    const uint64_t db = BT ? umma_desc(pb, 8192, 1024) : umma_desc(pb, 16, 1024);
#pragma unroll
                    for (int k = 0; k < BK / 16; ++k)   // 16 elements on: 32 bytes along a row, or 16 rows
                        umma_pair(tmem + buf * 256, da + (AT ? 2048 / 16 : 32 / 16) * k,
                                  db + (BT ? 2048 / 16 : 32 / 16) * k, idesc, i > 0 || c > 0 || k > 0);
                }
                umma_commit_pair(empty + 8 * st);
            }
            if (!ok) break;
            umma_commit_pair(tfull + 8 * buf);
        }
        }
        if (!ok) failed = 1;
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
                     ::"r"(drain) : "memory");
        wait_bar(drain, 0, limit);
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;\n");
        const int quad = warp % 4, side = warp / 4;
        const uint32_t lane_base = tmem + ((uint32_t)quad << 21);
        // this warp has read its share of a buffer: the next multiplies may overwrite it
        const auto release = [&](uint32_t bar) {
            umma_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(leader_addr(bar));
        };
        const int c0 = side * q.half, cols = side ? q.bn - q.half : q.half;
        float *turn = reinterpret_cast<float *>(smem_raw + (tiles - smem_u32(smem_raw)) + STAGE_BYTES) + warp * TURN;
        int use = 0;
        bool ok = true;
        for (int t = pair; ok && t < q.items; t += pairs) {
            int split, k_begin, k_end, mi, ni;
            if (!item_of(q, live, t, mi, ni, split, k_begin, k_end)) continue;
            const int m0 = mi * TM + rank * 128 + quad * 32, m = m0 + lane;
            Epilogue<KIND> ep;
            ep.begin(a, live, m, ni * q.bn + c0);
            float2 sum[4][16];                               // unused without PARTS
            for (int k_first = k_begin; k_first < k_end; k_first += q.part, ++use) {
                const int buf = use & 1;
                // every lane polls; the warp leaves together
                ok = wait_bar(tfull + 8 * buf, (use >> 1) & 1, limit);
                if (__any_sync(~0u, !ok)) {
                    if (lane == 0) failed = 1;
                    ok = false;
                    break;
                }
                umma_fence_after();
                const uint32_t from = lane_base + buf * 256 + c0;
                if (PARTS) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (32 * c >= cols) continue;
                        float v[32];
                        tmem_load32(from + 32 * c, v);
                        tmem_wait(v);
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            sum[c][i] = k_first > k_begin ? add2(sum[c][i], f2(v[2 * i], v[2 * i + 1]))
                                                          : f2(v[2 * i], v[2 * i + 1]);
                    }
                    release(tempty + 8 * buf);
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float v[32];
                        if (32 * c < cols) {
                            tmem_load32(from + 32 * c, v);
                            tmem_wait(v);
                        }
                        if (c == 3) release(tempty + 8 * buf);
                        if (32 * c < cols)
                            ep.chunk(a, q, split, m0, ni * q.bn + c0 + 32 * c, c0 + 32 * c, v, turn);
                    }
                }
            }
            if (!ok) break;
            if (PARTS && KIND == MM_LSE) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (32 * c < cols)
                        ep.chunk(a, q, split, m0, ni * q.bn + c0 + 32 * c, c0 + 32 * c,
                                 reinterpret_cast<float (&)[32]>(sum[c]), turn);
            } else if (PARTS) {
                // one copy of the code, the sums moving up: unrolled it spills registers
#pragma unroll 1
                for (int c = 0; 32 * c < cols; ++c) {
                    ep.chunk(a, q, split, m0, ni * q.bn + c0 + 32 * c, c0 + 32 * c,
                             reinterpret_cast<float (&)[32]>(sum[0]), turn);
#pragma unroll
                    for (int j = 0; j < 3; ++j)
#pragma unroll
                        for (int i = 0; i < 16; ++i) sum[j][i] = sum[j + 1][i];
                }
            }
            ep.end(a, m, ni * 2 + side);
        }
    }
    __syncwarp();
    umma_fence_before();
    __syncthreads();
    if (failed && threadIdx.x == 0) {
        atomicOr(&g_mm_timeout, 1u);
        if (rank == 0)                              // both CTAs' copies complete on the leader's barriers
            for (int it = max(0, issued - STAGES); it < issued; ++it)
                if (it != skip) wait_bar(full + 8 * (it % STAGES), (it / STAGES) & 1, limit);
    }
    __syncthreads();
    cluster_sync();
    if (warp == 9) tmem_free_pair(tmem);
}

bool encode(PFN_cuTensorMapEncodeTiled_v12000 fn, CUtensorMap *map, const Factor &f, int rows, int k, int box_rows)
{
    const cuuint64_t dim[3] = {(cuuint64_t)(f.t ? rows : k), (cuuint64_t)(f.t ? k : rows), (cuuint64_t)f.planes};
    const cuuint64_t stride[2] = {(cuuint64_t)f.ld * 2, (cuuint64_t)(f.planes == 1 ? f.ld : f.plane) * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)(f.t ? BK : box_rows), 1}, one[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<uint16_t *>(f.p), dim, stride, box, one,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int KIND, bool AT, bool BT, bool PARTS, bool BOTH>
cudaError_t launch(const MmArgs &a, Tiles q, cudaStream_t stream)
{
    // one round of tiles is short anyway: finer parts, as far as the multiplies hide them (a part costs the
    // epilogue some 1900 clocks, a step 512 a pass)
    q.part = !PARTS ? q.steps
             : KIND != MM_LSE && !BOTH ? PART_LONG / BK
             : q.items <= N_SM / 2 ? (BOTH ? 2 : 4) : (BOTH ? PART_BOTH : PART) / BK;
    const auto fn = tma_encoder();
    CUtensorMap ma, mb;
    if (!fn || !tma_context() || !encode(fn, &ma, a.a, a.m, a.k, 128) || !encode(fn, &mb, a.b, a.n, a.k, q.bn / 2))
        return cudaErrorInvalidValue;
    constexpr auto kernel = mm_kernel<KIND, AT, BT, PARTS, BOTH>;
    const cudaError_t e = smem_opt_in<kernel>(SMEM);
    if (e != cudaSuccess) return e;
    const int pairs = a.live && !AT ? N_SM / 2 : std::min(N_SM / 2, q.items);
    launch_chained(kernel, 2 * pairs, THREADS, SMEM, stream, ma, mb, a, q, tma_wait_limit(), tma_skip_item());
    return cudaGetLastError();
}

template <int KIND, bool AT, bool BT>
cudaError_t launch_as(const MmArgs &a, const Tiles &q, bool parts, bool both, cudaStream_t stream)
{
    if (both)
        return parts ? launch<KIND, AT, BT, true, true>(a, q, stream) : launch<KIND, AT, BT, false, true>(a, q, stream);
    return parts ? launch<KIND, AT, BT, true, false>(a, q, stream) : launch<KIND, AT, BT, false, false>(a, q, stream);
}

// out = acc + the partial sums of the split tiles, in order; a CTA per 4 rows of a tile,
// a thread per 4 columns.
template <typename T, bool AT>
__global__ void __launch_bounds__(256) split_sum_kernel(const MmArgs a, const Tiles planned)
{
    chained();
    int mi, ni;
    const Live live = live_of<AT>(a, planned);
    const Tiles q = live_plan<MM_OUT, AT>(a, planned, live);
    if (q.whole + (int)blockIdx.y >= q.mt * q.nt) return;
    tile_of(q, q.whole + blockIdx.y, mi, ni);
    const int splits = min(q.splits, (live.steps + q.kb - 1) / q.kb);
    const float *p = a.split + (size_t)blockIdx.y * q.splits * TM * q.bn;
    const int i = threadIdx.x * 4, r = blockIdx.x * 4 + i / q.bn, c = i % q.bn, m = mi * TM + r, n = ni * q.bn + c;
    if (i >= 4 * q.bn || m >= live.rows || n >= a.n) return;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int k = 0; k < splits; ++k) {
        const float4 t = *reinterpret_cast<const float4 *>(p + ((size_t)k * TM + r) * q.bn + c);
        s = make_float4(s.x + t.x, s.y + t.y, s.z + t.z, s.w + t.w);
    }
    const float *acc = a.acc ? a.acc + (size_t)m * a.n + n : nullptr;
    T *out = static_cast<T *>(a.out) + (size_t)(a.row_of ? a.row_of[m] : m) * a.n + n;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (n + j < a.n) out[j] = from_f<T>(comp(s, j) + (acc ? acc[j] : 0.f));
}

template <bool AT>
void split_sum(const MmArgs &a, const Tiles &q, int rest, cudaStream_t stream)
{
    const dim3 grid(TM / 4, rest);
    if (a.out_bf16) launch_chained(split_sum_kernel<__nv_bfloat16, AT>, grid, 256, 0, stream, a, q);
    else launch_chained(split_sum_kernel<float, AT>, grid, 256, 0, stream, a, q);
}

}  // namespace

int mm_lse_parts(int m, int n, int k, int planes_a, int planes_b)
{
    return 2 * plan(MM_LSE, m, n, k, passes_of(planes_a, planes_b), 0).nt;
}

size_t mm_split_bytes(int m, int n, int k, int planes_a, int planes_b, bool live)
{
    if (live) return (size_t)LIVE_ITEMS * TM * MM_COLS * 4;
    const Tiles q = plan(MM_OUT, m, n, k, passes_of(planes_a, planes_b), ~(size_t)0);
    return (size_t)(q.items - q.whole) * TM * q.bn * 4;
}

cudaError_t launch_mm(MmKind kind, const MmArgs &a, cudaStream_t stream)
{
    const Tiles q = plan(kind, a.m, a.n, a.k, passes_of(a.a.planes, a.b.planes), a.split_bytes);
    const int steps = q.whole || a.live ? q.steps : q.kb;       // live rows split as the device finds it
    const bool both = a.a.planes == 2 && a.b.planes == 2;
    const bool parts = kind != MM_LSE && !both ? steps > PART_LONG / BK
                                               : steps * BK > (both ? PART_BOTH : PART) ||
                                                     (q.items <= N_SM / 2 && steps > (both ? 2 : 4));
    if (kind == MM_LSE) return launch_as<MM_LSE, false, false>(a, q, parts, both, stream);
    if (kind == MM_GRAD) return launch_as<MM_GRAD, false, false>(a, q, parts, both, stream);
    const cudaError_t e = a.a.t ? launch_as<MM_OUT, true, true>(a, q, parts, both, stream)
                                : launch_as<MM_OUT, false, true>(a, q, parts, both, stream);
    // the live rows' tiles are not known here: as many CTAs as they may need
    const int rest = a.live && !a.a.t ? std::min(N_SM / 2 - 1, q.mt * q.nt) : q.mt * q.nt - q.whole;
    if (e != cudaSuccess || !rest) return e;
    if (a.a.t) split_sum<true>(a, q, rest, stream);
    else split_sum<false>(a, q, rest, stream);
    return cudaGetLastError();
}

int mm_take_timeout()
{
    unsigned int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_mm_timeout, sizeof(v)) != cudaSuccess) return -1;
    if (v) {
        const unsigned int z = 0;
        cudaMemcpyToSymbol(g_mm_timeout, &z, sizeof(z));
    }
    return v != 0;
}

}  // namespace mms
