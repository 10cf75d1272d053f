// Losses of a language model's head without its logits (sm_100a): softmax
// cross entropy and distillation from a teacher's top k, forward and backward.
//
// With z = x w^T (rows x vocab) and c = log2(e) / tau (tau = 1 for the cross
// entropy), in units of log 2:
//     lse2[m]   = (top, log2 sum_v 2^(c z[m, v] - top)),  top = max_v c z[m, v]
//     logq2[m, j] = c z[m, index[m, j]] - lse2, the log-probability there
//     CE  loss  = -ln2 logq2
//     KD  loss  = tau^2 sum_j p_j (log p_j - ln2 logq2_j)
// and for an upstream factor r[m] (dloss, times 1 / count for a mean, times
// tau for the distillation; 0 for a row that is left out):
//     dz[m, v]  = r (2^(c z - lse2) - sum of p_j with index_j = v)
//     dx = dz w,   dw = dz^T x
// The two halves of lse2 stay apart, and the logits at the indices keep their
// rounding errors (`rest`): sums would round at the magnitude of the logits,
// where the difference of a likely entry's logit to lse2 is small and exact.
// z is computed once forward (2 rows vocab dim flops) and again backward, in
// pieces of the vocabulary small enough that dz's piece stays in a bounded
// workspace (piece_size); the two products with dz follow piece by piece (6 more).
//
// Rows that do not count (an ignored target, an empty list) take no part: with
// more than MAP_ROWS rows a map lists those that do (map_kernel), x is staged
// in that order, everything between works on the listed rows, and the products
// read their number from the device. The host never learns it.
//
// Forward:   products (MM_LSE) -> one (max, sum) per row and half tile, joined
//            by lse_kernel. The logits at the indices are the product's own
//            values, so that its errors cancel against lse2's; the
//            distillation's lists are sorted for that (order_kernel,
//            before_kernel). Then a loss kernel; one block adds the rows up.
//            Up to few_rows() rows (few_kernel) w is read once, as it is, by
//            the CUDA cores: nothing is staged. The backward then takes dz from
//            the same sums (few_grad_kernel), and the distillation's logits
//            come from dot products in the same order (pick_kernel).
// Backward:  x staged, and r with it, left-out rows as zeros (so that nothing
//            in them, NaN included, reaches dw); per piece: product
//            MM_GRAD, sparse_kernel sets dz at the indices (from logq2, in
//            fp32; as expm1(log q) + 1 - p where p is near 1, so that nothing
//            cancels), then MM_OUT twice.
//
// bf16 backward: dz needs more bits than bf16's 8 beside the result's own
// rounding. Above FEW_ROWS rows it is one plane of scaled fp16 (2^-11 of a value
// at most; in bf16, 2^-8, gradients were 14 to 37 % further from float64 than
// their own rounding, now 1 %), and x and w follow it into fp16, scaled by
// powers of two, which holds a bf16 value exactly down to 2^-31 of the largest:
// r = M E with E a power of two and M in [1, 2),
//   dz = 2^14 M (q - p),  dx = E dz w,  dw = dz^T (E x)
// so that dz is all that is rounded; below 2^-28 it loses bits to fp16's range
// (2^-39 absolute). The price is w's copy and maximum (against one plane of
// bf16: 512 x 65536 x 2048 507 -> 650 us, 2048 rows 1.80 -> 1.95 ms, 8192 x 131072
// x 2048 15.5 -> 16.0; unaligned rows, copied anyway, 1000 x 50021 x 1001 504 ->
// 540). Up to FEW_ROWS rows, where w's bytes are what counts, w is taken as it is
// and dz is two planes of bf16 (2^-17; one more pass of two products): without r
// where it is the same for all rows (mean, sum), as r (q - p) where it is not. At
// 257 rows of 65536 x 2048 that takes 613 us, fp16 618; at 512 rows 730 and 650.
//
// float32: factors are split into two fp16 planes, 22 bits, after a scaling by
// a power of two that brings the largest element into [2^14, 2^15); the
// product of the second planes (below 2^-22 of a term) is left out. Elements
// below 2^-16 of the largest lose bits to fp16's range, one for each power of
// two (2^-20: 19 bits left, 2^-28: 11): 2^-39 of the largest is the absolute
// bound. So a vocabulary row of w far above the rest, by 2^16 and more, costs
// the others bits that float32 sums would keep. Three passes of the tensor
// cores; three bf16 planes would keep float32's range but need six. The scalings
// follow the output's rows where they can, so that rows do not disturb one
// another:
//   z  = x w^T    x scaled row by row, w as a whole
//   dz = 2^14 (q - p) without r, in [-2^14, 2^14]
//   dx = r dz w   r in the epilogue
//   dw = dz^T (r x)   r x scaled as a whole
#include <cuda_fp16.h>

#include <limits.h>

#include <algorithm>

#include "mms_common.cuh"
#include "mms_head.h"
#include "mms_kernels.h"
#include "mms_scan.h"

namespace mms {

namespace {

constexpr float LN2 = 0.6931471805599453f;
constexpr size_t PIECE_BYTES = (size_t)512 << 20;   // a staged or dz piece; or up to this much more
constexpr size_t PIECE_MOST = (size_t)2 << 30;      // for PIECE_ENTRIES of the vocabulary
constexpr int PIECE_ENTRIES = 4096;
constexpr int FEW_ROWS = 256;
constexpr int MAP_ROWS = 512;                       // two tiles of rows: with fewer there is little to leave out
// Rows that the CUDA cores take: at 50176 x 1024 they need (us, forward) 34, 49, 45, 68 for 1, 2,
// 4, 8 rows of float32, where staging alone is 100; in bf16 20, 20, 36, 58, the tensor cores 31.
int few_rows(bool bf16) { return bf16 ? 2 : 8; }
constexpr int FEW_BLOCKS = 148 * 4;
constexpr int STAGE_GRID = 148 * 16;                // CTAs of a staging pass, at most
constexpr float DZ_UNIT = 16384.f;                  // the scale of dz's planes in fp16

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }
size_t up256(size_t v) { return (v + 255) / 256 * 256; }
long long padded(int dim) { return (dim + 7) / 8 * 8; }     // rows of 16-byte multiples

// Pieces of the vocabulary (each a multiple of MM_COLS rows of w but the
// last): as few equal ones as keep `bytes_per_row` (per vocabulary entry)
// times the piece below PIECE_BYTES, or below PIECE_MOST for pieces of
// PIECE_ENTRIES, so that their products stay long and the float32 sums of dx are
// not read and written too often (7 % of the time with 4096 entries a piece); of MM_COLS
// where even those are more (dz above 4 M rows).
int piece_size(int vocab, size_t bytes_per_row)
{
    const size_t long_ones = std::min<size_t>(PIECE_ENTRIES, PIECE_MOST / bytes_per_row);
    const int most = (int)std::min<size_t>(vocab, std::max({(size_t)MM_COLS, long_ones, PIECE_BYTES / bytes_per_row}));
    // whole tiles: equal pieces rounded up would pass the bound
    const int whole = most >= vocab ? vocab : most / MM_COLS * MM_COLS, pieces = ceil_div(vocab, whole);
    const long long v = ceil_div(ceil_div(vocab, pieces), MM_COLS) * (long long)MM_COLS;
    return (int)std::min<long long>(v, vocab);
}

// Both directions: planes of x and w, and whether they are staged, and then as scaled fp16.
struct Layout {
    bool stage_x, stage_w, scaled;
    int planes, piece, last;        // vocabulary entries of a piece, of the last one
    size_t xs, ws, row_mul, muls;   // staged x, w; scaled: their scales (muls: w's, r x's, and w's maximum where
                                    // the forward did not keep it)
    size_t total;
};

// What the forward keeps for the backward.
struct Kept {
    float2 *lse2;       // (rows)
    float *logq2;       // (rows, k)
    float *prob;        // (rows, k), distillation
    float *count;       // (2): the rows that count; float32: the largest |w|
    int *map, *live;    // more than MAP_ROWS rows: those that count, and their number
};

// Row i of the listed rows, and how many there are.
struct RowMap {
    const int *map, *live;
    __device__ __forceinline__ int n(int rows) const { return live ? *live : rows; }
    __device__ __forceinline__ int row(int i) const { return map ? map[i] : i; }
};

struct FwdLayout : Layout {
    bool few;
    size_t col, pos, before;        // the distillation's sorted lists
    size_t flags;                   // the distillation's rows that count
    size_t part, rowloss, rest;
};

struct BwdLayout : Layout {
    bool few;
    int gplanes;
    long long ldg;
    size_t xr, g, dxacc, rs, pow, tops, split, split_bytes;
};

size_t common_layout(Layout &l, int rows, int vocab, int dim, size_t per_entry)
{
    const size_t row = (size_t)padded(dim) * 2 * l.planes;
    l.piece = piece_size(vocab, std::max<size_t>(l.stage_w ? row : 1, per_entry));
    l.last = vocab - (vocab - 1) / l.piece * l.piece;
    size_t o = 0;
    l.muls = o; o += 256;
    l.row_mul = o; o += l.scaled ? up256((size_t)rows * sizeof(float)) : 0;
    l.xs = o; o += l.stage_x ? up256(row * rows) : 0;
    l.ws = o; o += l.stage_w ? up256(row * l.piece) : 0;
    return o;
}

FwdLayout fwd_layout(int rows, int vocab, int dim, int k, bool bf16, long long ldx, long long ldw)
{
    FwdLayout l;
    l.few = rows <= few_rows(bf16);
    l.planes = bf16 || l.few ? 1 : 2;
    l.scaled = l.planes > 1;
    l.stage_x = !l.few && (!bf16 || ldx % 8 || rows > MAP_ROWS);
    l.stage_w = !l.few && (!bf16 || ldw % 8);
    size_t o = common_layout(l, rows, vocab, dim, (size_t)rows * sizeof(float2) / 32 + 1);
    const int parts = l.few ? FEW_BLOCKS : std::max(mm_lse_parts(rows, l.piece, dim, l.planes, l.planes),
                                                    mm_lse_parts(rows, l.last, dim, l.planes, l.planes));
    l.part = o; o += up256((size_t)(parts + 1) * rows * sizeof(float2));
    l.rowloss = o; o += up256((size_t)rows * sizeof(float));
    l.rest = o; o += up256((size_t)rows * std::max(k, 1) * sizeof(float));
    const size_t lists = l.few ? 0 : (size_t)rows * k, blocks = lists ? (size_t)(vocab - 1) / LIST_BLOCK + 1 : 0;
    l.flags = o; o += k && rows > MAP_ROWS ? up256(rows) : 0;
    l.col = o; o += up256(lists * sizeof(int));
    l.pos = o; o += up256(lists * sizeof(uint16_t));
    l.before = o; o += up256(blocks * rows * sizeof(uint16_t));
    l.total = o;
    return l;
}

BwdLayout bwd_layout(int rows, int vocab, int dim, bool bf16, long long ldw)
{
    BwdLayout l;
    l.planes = bf16 ? 1 : 2;
    l.few = rows <= few_rows(bf16);
    l.scaled = !bf16 || rows > FEW_ROWS;
    l.gplanes = bf16 && l.scaled ? 1 : 2;
    l.stage_x = true;
    l.stage_w = l.scaled || ldw % 8;
    size_t o = common_layout(l, rows, vocab, dim, (size_t)rows * 2 * l.gplanes);
    l.ldg = (l.piece + 7) / 8 * 8;
    l.xr = o; o += l.scaled ? up256((size_t)padded(dim) * 2 * l.planes * rows) : 0;
    l.g = o; o += up256((size_t)rows * l.ldg * 2 * l.gplanes);
    l.dxacc = o; o += l.piece < vocab ? up256((size_t)rows * dim * sizeof(float)) : 0;
    l.rs = o; o += up256((size_t)rows * sizeof(float));
    l.pow = o; o += bf16 && l.scaled ? up256((size_t)rows * sizeof(float)) : 0;
    l.tops = o; o += l.scaled ? up256(STAGE_GRID * sizeof(float)) : 0;
    // partial sums; the last, smaller piece splits as far as this room goes
    l.split_bytes = std::max(mm_split_bytes(rows, dim, l.piece, l.gplanes, l.planes, rows > MAP_ROWS),
                             mm_split_bytes(l.piece, dim, rows, l.gplanes, l.planes, false));
    l.split = o; o += up256(l.split_bytes);
    l.total = o;
    return l;
}

// ------------------------------------------------------------------- staging

// Powers of two: 2^e as two factors (e may be beyond float32's exponents).
struct Pow2 {
    float a, b;
    __device__ __forceinline__ float operator()(float v) const { return v * a * b; }
};
__device__ __forceinline__ float pow2(int e) { return ldexpf(1.f, e); }
// The exponent that brings `top` into [2^14, 2^15); 0 for 0.
__device__ __forceinline__ int exponent_for(float top) {
    return top == 0.f ? 0 : 14 - max((int)(__float_as_uint(top) >> 23) - 127, -126);
}
__device__ __forceinline__ Pow2 scale_by(int e) { return Pow2{pow2(e / 2), pow2(e - e / 2)}; }
__device__ __forceinline__ float finite_abs(float v) {
    v = fabsf(v);
    return v <= 3.4028234e38f ? v : 0.f;
}

// 8 elements of a row from column c on; 0 beyond `cols`. Where the row is not
// 16-byte aligned: bf16 from the two aligned pieces around them if both lie
// within the row (which any 8 but the first and the last do), else one by one.
template <typename T>
__device__ __forceinline__ void load8(const T *__restrict__ p, int c, int cols, float (&v)[8]) {
    const int off = (int)(reinterpret_cast<uintptr_t>(p + c) % 16);     // bytes past an aligned place
    if (c + 8 <= cols && off == 0) {
        uint4 q[sizeof(T) / 2];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) q[i] = __ldg(reinterpret_cast<const uint4 *>(p + c) + i);
        const T *e = reinterpret_cast<const T *>(q);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f(e[i]);
    } else if (sizeof(T) == 2 && c >= off / 2 && c - off / 2 + 16 <= cols) {
        const uint4 *q = reinterpret_cast<const uint4 *>(p + c - off / 2);
        const uint4 a = __ldg(q), b = __ldg(q + 1);
        uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        if (off & 4)
#pragma unroll
            for (int i = 0; i < 7; ++i) w[i] = w[i + 1];
        if (off & 8)
#pragma unroll
            for (int i = 0; i < 5; ++i) w[i] = w[i + 2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t t = __funnelshift_r(w[i], w[i + 1], off % 4 * 8);
            v[2 * i] = __uint_as_float(t << 16);
            v[2 * i + 1] = __uint_as_float(t & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? to_f(p[c + i]) : 0.f;
    }
}

// The CTA's maximum of v >= 0 (256 threads), in every thread.
__device__ __forceinline__ float block_max(float v) {
    __shared__ float sh[8];
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
    if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) v = fmaxf(v, sh[i]);
    return v;
}

// The same in pairs; VEC: every piece of 8 is whole and aligned.
template <bool VEC, typename T>
__device__ __forceinline__ void load8(const T *__restrict__ p, int c, int cols, float2 (&v)[4]) {
    if (!VEC) {
        load8(p, c, cols, reinterpret_cast<float (&)[8]>(v));
    } else if (sizeof(T) == 4) {
        const float4 a = ld4(reinterpret_cast<const float *>(p + c)), b = ld4(reinterpret_cast<const float *>(p + c) + 4);
        v[0] = lo(a); v[1] = hi(a); v[2] = lo(b); v[3] = hi(b);
    } else {
        const uint4 q = __ldg(reinterpret_cast<const uint4 *>(p + c));
        const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = f2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
    }
}

// How a staged matrix is scaled: not at all (bf16), each row to its own
// maximum, or all of it to the maximum that `top` holds.
enum StageKind { ST_COPY, ST_ROWS, ST_WHOLE };

// Where the backward's row factors r come from: computed where x is staged.
struct RowFactors {
    const float *dloss, *count, *prob, *logq2;
    const int64_t *index;
    int64_t ignore;
    int k, reduction;
    float tau;
    float *rs;                  // written: r of each row; NaN where an index that counts lies outside the
                                // vocabulary (logq2 is NaN there)
    float *pow;                 // written, if not null: E of each row, and DZ_UNIT M to rs; r = M E with E a
                                // power of two
    float *whole;               // written, may be null: the factor of all rows that count, where it is the same
};

struct StageArgs {
    const void *src;
    long long lds;
    uint16_t *out;
    long long ld, plane;
    int rows, cols;
    RowMap rows_map;            // row i of `out` comes from there; rows beyond them are 0
    RowFactors from;            // ST_COPY, ST_ROWS: if from.dloss, rows with r = 0 become 0
    const float *rs;            // ST_WHOLE: factors of the rows, or null
    float *mul;                 // ST_ROWS: 2^-e of each row; ST_WHOLE: of all
    float *top;                 // ST_WHOLE: maxima whose largest sets the scale, `tops` of them
    int tops;                   // ST_ROWS: the CTAs' maxima of |r| (or E) times the row's go to `top` (if not null),
                                //          and with `zero` a zero there
    float *zero;
};

// r of row i, by LP lanes together (all lanes of the warp call).
template <int LP>
__device__ __forceinline__ float row_factor(const RowFactors &f, RowMap rm, int i, int live, int lane) {
    float r = f.reduction == MMS_REDUCE_NONE ? (i < live ? f.dloss[rm.row(i)] : 0.f) : f.dloss[0];
    r *= f.tau;
    if (f.reduction == MMS_REDUCE_MEAN) r = *f.count == 0.f ? 0.f : r / *f.count;    // no row counts: gradients of 0
    if (i == 0 && lane == 0 && f.whole) *f.whole = r;
    int some = 0, bad = 0;
    if (i < live) {
        if (!f.prob) some = rm.live || f.index[i] != f.ignore;
        for (int j = lane; j < f.k; j += LP) {
            const float z = f.logq2[(size_t)i * f.k + j], p = f.prob ? f.prob[(size_t)i * f.k + j] : 1.f;
            some |= f.prob && !(p == 0.f);              // NaN counts
            bad |= z != z && !(p == 0.f);
        }
    }
#pragma unroll
    for (int o = LP / 2; o; o >>= 1) {
        some |= __shfl_xor_sync(~0u, some, o, LP);
        bad |= __shfl_xor_sync(~0u, bad, o, LP);
    }
    return !some ? 0.f : bad && r != 0.f ? __int_as_float(0x7fc00000) : r;
}

// r's E: its exponent alone, 1 where r is 0 or not finite (M = r then).
__device__ __forceinline__ float pow2_of(float r) {
    const uint32_t e = __float_as_uint(r) >> 23 & 255;
    return r == 0.f || e == 255 ? 1.f : __uint_as_float(max(e, 1u) << 23);
}

// LP lanes a row, 8 columns a lane and step. Bound by memory: 32768 x 640 of
// float32 weights in 26 us (84 MB in, 84 out: 6.4 TB/s); 50021 x 1001 bf16,
// whose rows are not aligned, in 42 us (4.8 TB/s).
template <typename T, int KIND, int LP>
__global__ void __launch_bounds__(256) stage_kernel(const StageArgs a)
{
    chained();
    const int lane = threadIdx.x % LP;
    float top = 0.f;
    Pow2 whole{1.f, 1.f};
    if (KIND == ST_WHOLE) {
        for (int i = threadIdx.x; i < a.tops; i += 256) top = fmaxf(top, a.top[i]);
        const int e = exponent_for(block_max(top));
        whole = scale_by(e);
        if (blockIdx.x == 0 && threadIdx.x == 0) *a.mul = pow2(-e);
    }
    if (KIND == ST_ROWS && a.zero && blockIdx.x == 0 && threadIdx.x == 0) *a.zero = 0.f;
    constexpr int RW = 32 / LP;                             // rows a warp has at once
    constexpr bool REST = KIND != ST_COPY && sizeof(T) == 4;    // a second plane: bf16 needs none in fp16
    // a last tile's padding is 0: nothing behind it is read
    const int live = a.rows_map.n(a.rows), rows = min(a.rows, (max(live, 1) + 255) / 256 * 256);
    for (int r0 = (blockIdx.x * 8 + threadIdx.x / 32) * RW; r0 < rows; r0 += gridDim.x * 8 * RW) {
        const int r = r0 + threadIdx.x % 32 / LP;           // lanes beyond the rows stay for the shuffles
        const bool in = r < rows;
        const T *src = static_cast<const T *>(a.src) + (size_t)(r < live ? a.rows_map.row(r) : 0) * a.lds;
        uint16_t *out = a.out + (size_t)r * a.ld;
        float rs = r >= live ? 0.f : a.rs ? a.rs[r] : 1.f;
        if (KIND != ST_WHOLE && a.from.dloss) {
            rs = row_factor<LP>(a.from, a.rows_map, r, live, lane);
            const float pow = a.from.pow ? pow2_of(rs) : 1.f;
            if (in && lane == 0) a.from.rs[r] = a.from.pow ? rs / pow * DZ_UNIT : rs;
            if (a.from.pow && rs != 0.f) rs = pow;
            if (in && lane == 0 && a.from.pow) a.from.pow[r] = rs;
        }
        const int cols = rs == 0.f ? 0 : a.cols;            // nothing of a left-out row is read
        Pow2 by{1.f, 1.f};
        if (KIND == ST_ROWS) {
            float m = 0.f;
            for (int c = lane * 8; c < cols; c += LP * 8) {
                float v[8];
                load8(src, c, cols, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_abs(v[i]));
            }
#pragma unroll
            for (int o = LP / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o, LP));
            const int e = exponent_for(m);
            by = scale_by(e);
            if (in && lane == 0) a.mul[r] = pow2(-e);
            top = fmaxf(top, finite_abs(rs * m));
        }
        if (KIND == ST_WHOLE) by = whole;
        for (int c = lane * 8; in && c < a.cols; c += LP * 8) {
            float v[8];
            load8(src, c, cols, v);
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint16_t h[2], l[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float x = v[2 * i + j];
                    if (KIND == ST_COPY) {
                        if (rs != rs) x = rs;               // a bad index: dw shows it
                        h[j] = __bfloat16_as_ushort(__float2bfloat16_rn(x));
                    } else {
                        x = by(KIND == ST_WHOLE ? rs * x : x);
                        const __half q = __float2half_rn(x);
                        h[j] = __half_as_ushort(q);
                        if (REST) l[j] = __half_as_ushort(__float2half_rn(x - __half2float(q)));
                    }
                }
                hi[i] = h[0] | (uint32_t)h[1] << 16;
                if (REST) lo[i] = l[0] | (uint32_t)l[1] << 16;
            }
            *reinterpret_cast<uint4 *>(out + c) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if (REST)
                *reinterpret_cast<uint4 *>(out + a.plane + c) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    }
    if (KIND == ST_ROWS && a.top) {
        top = block_max(top);
        if (threadIdx.x == 0) a.top[blockIdx.x] = top;
    }
}

// The largest finite magnitude of a matrix (*top starts at 0), whose last row
// has `last` columns; VEC: every row begins at 16 bytes. A warp reads a row, 4
// pieces a lane at a time; one atomic a CTA, a few thousand on one address
// would take longer than the reads. 131072 x 2048 bf16: 95 us (5.6 TB/s).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
top_kernel(const T *__restrict__ src, long long lds, int rows, int cols, int last, float *top)
{
    chained();
    constexpr int PIECE = VEC ? 16 / (int)sizeof(T) : 8;
    const int lane = threadIdx.x % 32;
    float m = 0.f;
    for (long long r = (long long)blockIdx.x * 8 + threadIdx.x / 32; r < rows; r += gridDim.x * 8) {
        const T *p = src + (size_t)r * lds;
        const int n = r + 1 < rows ? cols : last;
        if (VEC) {
            const uint4 *q = reinterpret_cast<const uint4 *>(p);
            for (int c = lane; c < n / PIECE; c += 128) {
                uint4 t[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) t[k] = c + 32 * k < n / PIECE ? __ldg(q + c + 32 * k) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int i = 0; i < PIECE; ++i) m = fmaxf(m, finite_abs(to_f(reinterpret_cast<const T *>(t + k)[i])));
            }
            const int c = n / PIECE * PIECE + lane;
            if (c < n) m = fmaxf(m, finite_abs(to_f(p[c])));
        } else {
#pragma unroll 2
            for (int c = lane * PIECE; c < n; c += 32 * PIECE) {
                float v[8];
                load8(p, c, n, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_abs(v[i]));
            }
        }
    }
    m = block_max(m);                                       // non-negative floats compare as their bits
    if (threadIdx.x == 0 && m > 0.f) atomicMax(reinterpret_cast<unsigned *>(top), __float_as_uint(m));
}

int grid_of(long long rows, int per_block) { return (int)std::min<long long>((rows + per_block - 1) / per_block, STAGE_GRID); }

int stage_grid(int rows, int cols) { return grid_of(rows, cols <= 64 ? 32 : cols <= 128 ? 16 : 8); }

template <typename T, int KIND>
void stage(const StageArgs &a, cudaStream_t s)
{
    const int grid = stage_grid(a.rows, a.cols);
    if (a.cols <= 64) launch_chained(stage_kernel<T, KIND, 8>, grid, 256, 0, s, a);
    else if (a.cols <= 128) launch_chained(stage_kernel<T, KIND, 16>, grid, 256, 0, s, a);
    else launch_chained(stage_kernel<T, KIND, 32>, grid, 256, 0, s, a);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
    return v;
}

// The distillation's logq2[m, j] = c * (x[m] . w[index[m, j]]), a warp each;
// NaN for an index outside the vocabulary, 0 for an entry that is left out.
template <typename T>
__global__ void __launch_bounds__(256)
pick_kernel(const T *__restrict__ x, long long ldx, const T *__restrict__ w, long long ldw,
            const int64_t *__restrict__ index, int k, float c, float *__restrict__ logq2,
            float *__restrict__ rest, long long n, int vocab, int dim)
{
    chained();
    const long long e = (long long)blockIdx.x * 8 + threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    if (e >= n) return;
    const int64_t v = index[e];
    float s = 0.f;
    if (v < 0) {
    } else if (v >= vocab) {
        s = __int_as_float(0x7fc00000);
    } else {
        const T *xr = x + e / k * ldx, *wr = w + v * ldw;
        float2 acc = f2(0.f, 0.f);
        for (int i = lane * 8; i < dim; i += 256) {
            float2 p[4], q[4];
            load8<false>(xr, i, dim, p);
            load8<false>(wr, i, dim, q);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc = fma2(p[j], q[j], acc);
        }
        s = warp_sum(acc.x + acc.y);
    }
    if (lane) return;
    const float p = s * c;
    logq2[e] = p;
    rest[e] = rounding_of(s, c, p);
}

// (max, sum) pairs join to the pair of both; a NaN in either sum stays. The
// sums are double: where one term has nearly all the probability, a thousand
// small ones added to a float32 near 1 would lose what its gradient is made of.
struct Part {
    float x;
    double y;
    // the same with the larger maximum m
    __device__ __forceinline__ Part at(float m) const { return Part{m, y * ex2(x - (m == -INFINITY ? 0.f : m))}; }
};
__device__ __forceinline__ Part join(Part a, Part b) {
    const float m = fmaxf(a.x, b.x);
    return Part{m, a.at(m).y + b.at(m).y};
}

// Up to few_rows() rows: a warp takes 4 rows of w at a time, its lanes 8 columns
// each, against R rows of x (L1 holds them). Bound by reading w once. These
// are the 4 R dot products, in every lane; pick_kernel adds in the same order.
template <typename T, int R, bool VEC>
__device__ __forceinline__ void few_dots(const T *__restrict__ x, long long ldx, const T *__restrict__ w,
                                         long long ldw, int rows, int vocab, int dim, int v, float (&s)[R][4]) {
    const T *wr[4], *xr[R];
    float2 acc[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) xr[r] = x + (size_t)min(r, rows - 1) * ldx;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        wr[i] = w + (size_t)min(v + i, vocab - 1) * ldw;
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][i] = f2(0.f, 0.f);
    }
#pragma unroll(sizeof(T) == 2 ? 2 : 1)
    for (int k = threadIdx.x % 32 * 8; k < dim; k += 256) {
        float2 q[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) load8<VEC>(wr[i], k, dim, q[i]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float2 p[4];
            load8<VEC>(xr[r], k, dim, p);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[r][i] = fma2(p[j], q[i][j], acc[r][i]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[r][i] = warp_sum(acc[r][i].x + acc[r][i].y);
}

struct FewArgs {
    const void *x, *w;
    long long ldx, ldw;
    float c;
    int rows, vocab, dim;
    const int64_t *target;      // forward: the cross entropy's, whose logits go to `at`
    float *at, *rest;
    float2 *part;
    const float2 *lse2;         // backward
    const float *rs;
    float unit;
    uint16_t *g;
    long long ldg, gplane;
    int v0, n;                  // this piece
    bool fp16;
};

// The log-sum-exp over a share of w's rows per CTA.
template <typename T, int R, bool VEC>
__global__ void __launch_bounds__(256) few_kernel(const FewArgs a)
{
    chained();
    __shared__ Part sh[8][R];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const float c = a.c;
    Part run[R];
    long long at[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        run[r] = Part{-INFINITY, 0.};
        at[r] = a.target && r < a.rows ? a.target[r] : -1;
    }
    for (int v = (blockIdx.x * 8 + warp) * 4; v < a.vocab; v += gridDim.x * 32) {
        float s[R][4];
        few_dots<T, R, VEC>(static_cast<const T *>(a.x), a.ldx, static_cast<const T *>(a.w), a.ldw, a.rows, a.vocab, a.dim, v, s);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float m = run[r].x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (v + i >= a.vocab) s[r][i] = -INFINITY;
                if (v + i == at[r] && lane == 0) {
                    a.at[r] = s[r][i] * c;
                    a.rest[r] = rounding_of(s[r][i], c, s[r][i] * c);
                }
                m = fmaxf(m, s[r][i] * c);
            }
            const float ref = m == -INFINITY ? 0.f : m;
            float e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = ex2(fmaf(s[r][i], c, -ref));
            run[r] = Part{m, run[r].y * ex2(run[r].x - ref) + ((double)e[0] + e[1]) + ((double)e[2] + e[3])};
        }
    }
    if (lane == 0)
#pragma unroll
        for (int r = 0; r < R; ++r) sh[warp][r] = run[r];
    __syncthreads();
    if (threadIdx.x < a.rows) {
        Part t = sh[0][threadIdx.x];
#pragma unroll
        for (int i = 1; i < 8; ++i) t = join(t, sh[i][threadIdx.x]);
        // without the top's own 1, beside which float32 would lose the rest (less_one in lse_kernel)
        a.part[(size_t)blockIdx.x * a.rows + threadIdx.x] = make_float2(t.x, (float)(t.y - 1.));
    }
}

// dz of a piece of the vocabulary, two planes.
template <typename T, int R, bool VEC>
__global__ void __launch_bounds__(256) few_grad_kernel(const FewArgs a)
{
    chained();
    const int lane = threadIdx.x % 32, row = lane / 4, i = lane % 4;
    const bool in = row < a.rows;
    const float2 l = in ? a.lse2[row] : make_float2(0.f, 0.f);
    const float rs = in ? a.rs[row] : 0.f, by = rs != 0.f && a.unit != 0.f ? a.unit : rs;
    for (int v = (blockIdx.x * 8 + threadIdx.x / 32) * 4; v < a.n; v += gridDim.x * 32) {
        float s[R][4];
        few_dots<T, R, VEC>(static_cast<const T *>(a.x), a.ldx, static_cast<const T *>(a.w) + (size_t)a.v0 * a.ldw, a.ldw,
                 a.rows, a.n, a.dim, v, s);
        float z = 0.f;                                      // lane 4 r + i takes s[r][i]
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) z = r == row && j == i ? s[r][j] : z;
        if (!in || v + i >= a.n) continue;
        float d = by == 0.f ? 0.f : by * ex2(fmaf(z, a.c, -l.x) - l.y);
        uint16_t *o = a.g + (size_t)row * a.ldg + v + i;
        for (int q = 0; q < 2; ++q, o += a.gplane) {
            if (a.fp16) {
                const __half t = __float2half_rn(d);
                *o = __half_as_ushort(t);
                d -= __half2float(t);
            } else {
                const __nv_bfloat16 t = __float2bfloat16_rn(d);
                *o = __bfloat16_as_ushort(t);
                d -= to_f(t);
            }
        }
    }
}

template <typename T, int R, bool VEC>
void launch_few_rows(const FewArgs &a, int blocks, bool backward, cudaStream_t s)
{
    if (backward) launch_chained(few_grad_kernel<T, R, VEC>, blocks, 256, 0, s, a);
    else launch_chained(few_kernel<T, R, VEC>, blocks, 256, 0, s, a);
}

template <typename T, bool VEC>
void launch_few_vec(const FewArgs &a, int blocks, bool backward, cudaStream_t s)
{
    if (a.rows == 1) launch_few_rows<T, 1, VEC>(a, blocks, backward, s);
    else if (a.rows == 2) launch_few_rows<T, 2, VEC>(a, blocks, backward, s);
    else if (a.rows <= 4) launch_few_rows<T, 4, VEC>(a, blocks, backward, s);
    else launch_few_rows<T, 8, VEC>(a, blocks, backward, s);
}

template <typename T>
void launch_few(const FewArgs &a, int blocks, bool backward, cudaStream_t s)
{
    constexpr int PER16 = 16 / (int)sizeof(T);              // bases are 16-byte aligned
    if (a.dim % 8 == 0 && a.ldx % PER16 == 0 && a.ldw % PER16 == 0) launch_few_vec<T, true>(a, blocks, backward, s);
    else launch_few_vec<T, false>(a, blocks, backward, s);
}

FewArgs few_args(const HeadArgs &a, float c)
{
    FewArgs f{};
    f.x = a.x; f.w = a.w; f.ldx = a.ldx; f.ldw = a.ldw; f.c = c;
    f.rows = a.rows; f.vocab = a.vocab; f.dim = a.dim; f.fp16 = !a.bf16;
    return f;
}

// The distillation's lists in ascending order, a warp a row: an entry's place
// is the number of entries before it. Indices outside the vocabulary go last.
__global__ void __launch_bounds__(256)
order_kernel(const int64_t *__restrict__ index, int k, int rows, RowMap rm, int vocab, int *__restrict__ col,
             uint16_t *__restrict__ pos, float *__restrict__ logq2, float *__restrict__ rest)
{
    chained();
    extern __shared__ int sh_index[];
    const int m = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
    if (m >= rm.n(rows)) return;
    int *v = sh_index + threadIdx.x / 32 * k;
    const int64_t *from = index + (size_t)rm.row(m) * k;
    for (int j = lane; j < k; j += 32) {
        const int64_t t = from[j];
        v[j] = t < 0 || t >= vocab ? INT_MAX : (int)t;
        // no product will come for these
        if (v[j] == INT_MAX) {
            logq2[(size_t)m * k + j] = t < 0 ? 0.f : __int_as_float(0x7fc00000);
            rest[(size_t)m * k + j] = 0.f;
        }
    }
    __syncwarp();
    for (int j = lane; j < k; j += 32) {
        const int t = v[j];
        int place = 0;
#pragma unroll 8
        for (int i = 0; i < k; ++i) place += v[i] < t || (v[i] == t && i < j);
        col[(size_t)m * k + place] = t;
        pos[(size_t)m * k + place] = (uint16_t)j;
    }
}

// before[b * rows + m]: entries of row m below column LIST_BLOCK * b. A thread a row
// (32 a CTA, so that the stores are whole sectors) and its CTA's blocks' eighth.
__global__ void __launch_bounds__(256)
before_kernel(const int *col, int k, int rows, RowMap rm, int blocks, uint16_t *__restrict__ before)
{
    chained();
    const int m = blockIdx.x * 32 + threadIdx.x % 32;
    if (m >= rm.n(rows)) return;
    const int each = (blocks + 8 * gridDim.y - 1) / (8 * gridDim.y);
    const int b0 = min(blocks, (int)(blockIdx.y * 8 + threadIdx.x / 32) * each), b1 = min(blocks, b0 + each);
    const int *c = col + (size_t)m * k;
    int lo = 0, hi = k;                                     // the first entry not below b0's column
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (c[mid] < (long long)b0 * LIST_BLOCK) lo = mid + 1;
        else hi = mid;
    }
    int at = lo < k ? c[lo] : INT_MAX;
    for (int b = b0; b < b1; ++b) {
        while (at < (long long)b * LIST_BLOCK) at = ++lo < k ? c[lo] : INT_MAX;
        before[(size_t)b * rows + m] = (uint16_t)lo;
    }
}

constexpr int AT_ONCE = 8;

// One row a lane, 32 threads a row over the tiles. Parts 1..ntiles, and part
// 0 (the pieces before) unless `first`. Writes part 0, or in the last piece
// lse2 and, from the target's logit in logq2, the cross entropy's row loss;
// with `total` (up to 32 rows) total_kernel's work too. less_one: the parts' sums are less the 1 of
// their maximum.
__global__ void __launch_bounds__(1024)
lse_kernel(float2 *part, bool less_one, int ntiles, bool first, bool last, int rows, RowMap rm, float2 *__restrict__ lse2,
           const int64_t *__restrict__ target, int64_t ignore, int vocab, float *__restrict__ logq2,
           const float *rest, float *__restrict__ loss, int reduction,
           float *__restrict__ total, float *__restrict__ count)
{
    chained();
    __shared__ Part sh[32][33];
    __shared__ float row_loss[32];
    const int m = blockIdx.x * 32 + threadIdx.x, live = rm.n(rows);
    Part v{-INFINITY, 0.};
    if (m < live)
        for (int t0 = threadIdx.y + (first ? 1 : 0); t0 <= ntiles; t0 += 32 * AT_ONCE) {
            // all loads, then the maximum, then independent terms: no chain of joins
            float2 p[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i)
                p[i] = t0 + 32 * i <= ntiles ? part[(size_t)(t0 + 32 * i) * rows + m] : make_float2(-INFINITY, 0.f);
            float top = v.x;
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) top = fmaxf(top, p[i].x);
            v = v.at(top);
            // a float32 sum and what it lost: converting each term to double bounds the kernel (888 parts of
            // 16 rows 11.1 us, this way 7.7)
            const float ref = top == -INFINITY ? 0.f : top;
            float s = 0.f, lost = 0.f;
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const float e = ex2(p[i].x - ref), z = __fmul_rn(p[i].y, e), y = less_one ? e : z, n = s + y, d = n - s;
                lost += (s - (n - d)) + (y - d) + (less_one ? z : 0.f);
                s = n;
            }
            v.y += (double)s + lost;
        }
    sh[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    // transposed: a warp joins the 32 values of one row
    v = sh[threadIdx.x][threadIdx.y];
    v = v.at(warp_max(v.x));
#pragma unroll
    for (int o = 16; o; o >>= 1) v.y += __shfl_xor_sync(~0u, v.y, o);
    const int r = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && r < live) {
        if (!last) {
            part[r] = make_float2(v.x, (float)v.y);
        }
        const float log_sum = last ? (float)log2(v.y) : 0.f;
        if (last) lse2[r] = make_float2(v.x, log_sum);
        if (last && target) {
            const int64_t t = target[rm.row(r)];
            float l = 0.f;
            if (t != ignore) l = t < 0 || t >= vocab ? __int_as_float(0x7fc00000) : ((logq2[r] - v.x) + rest[r]) - log_sum;
            logq2[r] = l;
            loss[reduction == MMS_REDUCE_NONE ? rm.row(r) : r] = row_loss[threadIdx.y] = -LN2 * l;
        }
    }
    if (!total) return;                                     // one CTA has all rows
    __syncthreads();
    if (threadIdx.y) return;
    const bool in = threadIdx.x < rows;
    const float s = warp_sum(in ? row_loss[threadIdx.x] : 0.f);
    const float n = warp_sum(in && target[threadIdx.x] != ignore ? 1.f : 0.f);
    if (threadIdx.x == 0) {
        *count = n;
        if (reduction != MMS_REDUCE_NONE) *total = reduction == MMS_REDUCE_MEAN ? s / n : s;
    }
}

// Distillation's row loss, a warp a row: the teacher's softmax over its
// entries, kept as prob, against the student's log-probabilities.
__global__ void __launch_bounds__(256)
kd_kernel(const int64_t *__restrict__ index, const float *__restrict__ logits, int k, float tau,
          const float2 *lse2, float *__restrict__ logq2,
          const float *rest, float *__restrict__ prob, float *__restrict__ loss, int rows, RowMap rm,
          int reduction)
{
    chained();
    const int m = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
    if (m >= rm.n(rows)) return;
    const size_t o = (size_t)m * k;
    index += (size_t)rm.row(m) * k;
    logits += (size_t)rm.row(m) * k;
    const float inv = 1.f / tau;
    const float2 l2 = lse2[m];
    float top = -INFINITY;
    for (int j = lane; j < k; j += 32)
        if (index[j] >= 0) top = fmaxf(top, logits[j]);
    top = warp_max(top);
    float sum = 0.f;
    for (int j = lane; j < k; j += 32)
        if (index[j] >= 0 && !(top == -INFINITY && logits[j] == -INFINITY))
            sum += expf((logits[j] - top) * inv);
    sum = warp_sum(sum);
    const float log_sum = logf(sum), over = 1.f / sum;
    const bool some = sum != 0.f;                       // NaN counts as some
    float acc = 0.f;
    for (int j = lane; j < k; j += 32) {
        float p = 0.f;
        const float lq = ((logq2[o + j] - l2.x) + rest[o + j]) - l2.y;
        logq2[o + j] = lq;
        if (some && index[j] >= 0) {
            const float t = (logits[j] - top) * inv;
            p = expf(t) * over;
            if (p != 0.f) acc += p * ((t - log_sum) - LN2 * lq);
        }
        prob[o + j] = p;
    }
    acc = warp_sum(acc);
    if (lane == 0) loss[reduction == MMS_REDUCE_NONE ? rm.row(m) : m] = some ? tau * tau * acc : 0.f;
}

// Whether row m counts.
__device__ __forceinline__ bool row_counts(const int64_t *index, const float *prob, int k,
                                           int64_t ignore, size_t m) {
    if (!prob) return index[m] != ignore;
    for (int j0 = 0; j0 < k; j0 += 8) {                 // 8 loads at once
        bool some = false;
#pragma unroll
        for (int j = j0; j < j0 + 8; ++j) some |= j < k && !(prob[m * k + j] == 0.f);   // NaN counts
        if (some) return true;
    }
    return false;
}

// count, and loss = the rows' sum (over count for a mean), in a fixed order.
__global__ void __launch_bounds__(1024)
total_kernel(const float *rowloss, const int64_t *__restrict__ index,
             const float *prob, int k, int64_t ignore, int rows, RowMap rm, int reduction,
             float *__restrict__ loss, float *__restrict__ count)
{
    chained();
    __shared__ float sh[2][32];
    float s = 0.f, n = 0.f;
    const int live = rm.n(rows);
    for (int m = threadIdx.x; m < live; m += 1024) {
        if (reduction != MMS_REDUCE_NONE) s += rowloss[m];
        n += rm.live || row_counts(index, prob, k, ignore, m) ? 1.f : 0.f;
    }
    s = warp_sum(s);
    n = warp_sum(n);
    if (threadIdx.x % 32 == 0) {
        sh[0][threadIdx.x / 32] = s;
        sh[1][threadIdx.x / 32] = n;
    }
    __syncthreads();
    if (threadIdx.x >= 32) return;
    s = warp_sum(sh[0][threadIdx.x]);
    n = warp_sum(sh[1][threadIdx.x]);
    if (threadIdx.x == 0) {
        *count = n;
        if (reduction != MMS_REDUCE_NONE) *loss = reduction == MMS_REDUCE_MEAN ? s / n : s;
    }
}

// flags[m]: whether the teacher's list has an entry with index >= 0 and a logit above -inf.
__global__ void __launch_bounds__(256)
flags_kernel(const int64_t *__restrict__ index, const float *__restrict__ logits, int k, int rows,
             uint8_t *__restrict__ flags)
{
    chained();
    const int m = blockIdx.x * 8 + threadIdx.x / 32;
    if (m >= rows) return;
    bool some = false;
    for (int j = threadIdx.x % 32; j < k; j += 32)
        some |= index[(size_t)m * k + j] >= 0 && logits[(size_t)m * k + j] != -INFINITY;
    some = __any_sync(~0u, some);
    if (threadIdx.x % 32 == 0) flags[m] = some;
}

// The rows that count, in order, and their number: one CTA, 1024 rows at a time.
__global__ void __launch_bounds__(1024)
map_kernel(const int64_t *__restrict__ target, int64_t ignore, const uint8_t *flags, int rows,
           int *__restrict__ map, int *__restrict__ live)
{
    chained();
    __shared__ int sh[32];
    int base = 0;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    for (int m0 = 0; m0 < rows; m0 += 1024) {
        const int m = m0 + threadIdx.x;
        const bool in = m < rows && (flags ? flags[m] != 0 : target[m] != ignore);
        const unsigned vote = __ballot_sync(~0u, in);
        if (lane == 0) sh[warp] = __popc(vote);
        __syncthreads();
        int at = sh[lane];                                  // inclusive sums of the 32 warps' counts
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(~0u, at, o);
            if (lane >= o) at += t;
        }
        const int all = __shfl_sync(~0u, at, 31);
        const int before = warp ? __shfl_sync(~0u, at, warp - 1) : 0;
        if (in) map[base + before + __popc(vote & ((1u << lane) - 1))] = m;
        base += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) *live = base;
}

// dz at the sparse entries that lie in this piece of the vocabulary; `unit` in
// place of r if it is not 0.
__global__ void __launch_bounds__(256)
sparse_kernel(const int64_t *__restrict__ index, const float *prob,
              const float *logq2, const float *rs, float unit, int k, int rows, RowMap rm, int v0, int v1,
              uint16_t *__restrict__ g, long long ldg, long long gplane, int planes, bool fp16)
{
    chained();
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x, m = e / k;
    if (m >= rm.n(rows)) return;
    const int64_t *list = index + (size_t)rm.row((int)m) * k;
    const int64_t v = list[e - m * k];
    if (v < v0 || v >= v1) return;
    const float r = rs[m];
    if (r == 0.f) return;                               // dz is 0 there already
    uint16_t *o = g + m * ldg + (v - v0);
    float p = 1.f;
    if (prob) {                                         // an index may occur twice: the first one writes
        p = 0.f;
        for (int j = 0; j < k; ++j) {
            if (list[j] != v) continue;
            if (m * k + j < e) return;
            p += prob[m * k + j];
        }
    }
    // q - p without rounding at 1 where both are small, nor losing 1 - q where p is near 1
    const float lq = LN2 * logq2[e];
    float d = (unit != 0.f ? unit : r) * (p > 0.5f ? expm1f(lq) + (1.f - p) : expf(lq) - p);
    for (int q = 0; q < planes; ++q, o += gplane) {
        if (fp16) {
            const __half t = __float2half_rn(d);
            *o = __half_as_ushort(t);
            d -= __half2float(t);
        } else {
            const __nv_bfloat16 t = __float2bfloat16_rn(d);
            *o = __bfloat16_as_ushort(t);
            d -= to_f(t);
        }
    }
}

uint16_t *u16(void *base, size_t off) { return reinterpret_cast<uint16_t *>(static_cast<char *>(base) + off); }
size_t kept_layout(int rows, int k, bool kd, char *base, Kept &o)
{
    size_t at = 0;
    const auto take = [&](size_t bytes) { char *p = base + at; at += (bytes + 15) / 16 * 16; return p; };
    o.lse2 = reinterpret_cast<float2 *>(take((size_t)rows * sizeof(float2)));
    o.logq2 = reinterpret_cast<float *>(take((size_t)rows * k * sizeof(float)));
    o.prob = kd ? reinterpret_cast<float *>(take((size_t)rows * k * sizeof(float))) : nullptr;
    o.count = reinterpret_cast<float *>(take(2 * sizeof(float)));
    const bool mapped = rows > MAP_ROWS;
    o.live = mapped ? reinterpret_cast<int *>(take(sizeof(int))) : nullptr;
    o.map = mapped ? reinterpret_cast<int *>(take((size_t)rows * sizeof(int))) : nullptr;
    return at;
}
Kept kept_of(const HeadArgs &a)
{
    Kept o;
    kept_layout(a.rows, a.k, a.kd, static_cast<char *>(a.kept), o);
    return o;
}

float *fl(void *base, size_t off) { return reinterpret_cast<float *>(static_cast<char *>(base) + off); }

// Where w's largest magnitude is: the float32 forward keeps it for the backward
// (count[1]), but for few rows, where it does not need it, as the bf16 one never does.
bool finds_top(const HeadArgs &a, const Layout &l)
{
    return l.scaled && (!a.backward || a.bf16 || a.rows <= few_rows(a.bf16));
}
float *w_top(const HeadArgs &a, const Layout &l)
{
    return a.backward && finds_top(a, l) ? fl(a.workspace, l.muls) + 3 : kept_of(a).count + 1;
}
template <typename T>
void top_of(const HeadArgs &a, float *top, cudaStream_t s)
{
    int rows = a.vocab, cols = a.dim, last = a.dim;
    long long ld = a.ldw;
    if (ld == cols && ld * sizeof(T) % 16) {                // rows without gaps: aligned ones of another length
        const long long n = (long long)rows * cols;
        ld = cols = 2048;
        rows = ceil_div(n, cols);
        last = (int)(n - (rows - 1) * ld);
    }
    const auto run = [&](auto kernel) {
        launch_chained(kernel, std::min(ceil_div(rows, 8), 148 * 8), 256, 0, s, static_cast<const T *>(a.w), ld, rows, cols,
                       last, top);
    };
    if (ld * sizeof(T) % 16 == 0) run(top_kernel<T, true>);
    else run(top_kernel<T, false>);
}
void top_of_w(const HeadArgs &a, float *top, cudaStream_t s)
{
    if (a.bf16) top_of<__nv_bfloat16>(a, top, s);
    else top_of<float>(a, top, s);
}

template <int KIND>
void stage_scaled(const HeadArgs &a, const StageArgs &st, cudaStream_t s)
{
    if (a.bf16) stage<__nv_bfloat16, KIND>(st, s);
    else stage<float, KIND>(st, s);
}

// Rows [v0, v0 + n) of w as a factor: staged, or w itself.
Factor w_factor(const HeadArgs &a, const Layout &l, int v0, int n, cudaStream_t s)
{
    if (!l.stage_w) return Factor{static_cast<const uint16_t *>(a.w) + (size_t)v0 * a.ldw, a.ldw, 0, 1, false};
    const long long ld = padded(a.dim);
    StageArgs st{};
    st.src = static_cast<const char *>(a.w) + (size_t)v0 * a.ldw * (a.bf16 ? 2 : 4);
    st.lds = a.ldw;
    st.out = u16(a.workspace, l.ws); st.ld = ld; st.plane = ld * l.piece;
    st.rows = n; st.cols = a.dim;
    st.mul = fl(a.workspace, l.muls);
    st.top = w_top(a, l); st.tops = 1;
    if (l.scaled) stage_scaled<ST_WHOLE>(a, st, s);
    else stage<__nv_bfloat16, ST_COPY>(st, s);
    return Factor{st.out, ld, st.plane, l.planes, false};
}

// x as a factor of z: staged, or x itself. Backward: with the rows' factors
// (`from`), and if scaled the maxima of r x. The place of w's maximum is zeroed
// for top_of_w.
Factor x_factor(const HeadArgs &a, const Layout &l, const RowFactors &from, float *tops, RowMap rm, cudaStream_t s)
{
    if (!l.stage_x) return Factor{static_cast<const uint16_t *>(a.x), a.ldx, 0, 1, false};
    const long long ld = padded(a.dim);
    StageArgs st{};
    st.src = a.x; st.lds = a.ldx;
    st.out = u16(a.workspace, l.xs); st.ld = ld; st.plane = ld * a.rows;
    st.rows = a.rows; st.cols = a.dim; st.rows_map = rm;
    st.from = from;
    st.mul = fl(a.workspace, l.row_mul);
    st.top = tops;
    st.zero = finds_top(a, l) ? w_top(a, l) : nullptr;
    if (l.scaled) stage_scaled<ST_ROWS>(a, st, s);
    else stage<__nv_bfloat16, ST_COPY>(st, s);
    return Factor{st.out, ld, st.plane, l.planes, false};
}

}  // namespace

size_t head_kept_bytes(int rows, int k, bool kd)
{
    Kept o;
    return kept_layout(rows, k, kd, nullptr, o);
}

size_t head_workspace_bytes(int rows, int vocab, int dim, int k, bool bf16, long long ldx, long long ldw,
                            bool backward)
{
    return backward ? bwd_layout(rows, vocab, dim, bf16, ldw).total
                    : fwd_layout(rows, vocab, dim, k, bf16, ldx, ldw).total;
}

cudaError_t launch_head_fwd(const HeadArgs &a, cudaStream_t stream)
{
    chain_begin();
    const FwdLayout l = fwd_layout(a.rows, a.vocab, a.dim, a.kd ? a.k : 0, a.bf16, a.ldx, a.ldw);
    const Kept o = kept_of(a);
    const RowMap rm{o.map, o.live};
    const float c = MMS_LOG2E / a.tau;
    const bool none = a.reduction == MMS_REDUCE_NONE;
    float2 *part = reinterpret_cast<float2 *>(fl(a.workspace, l.part));
    float *rowloss = none ? a.loss : fl(a.workspace, l.rowloss), *rest = fl(a.workspace, l.rest);
    float *total = a.kd || a.rows > 32 ? nullptr : a.loss;
    const int64_t *target = a.kd ? nullptr : a.index;
    cudaError_t e;
    if (rm.live) {
        uint8_t *flags = a.kd ? static_cast<uint8_t *>(a.workspace) + l.flags : nullptr;
        if (a.kd) launch_chained(flags_kernel, ceil_div(a.rows, 8), 256, 0, stream, a.index, a.logits, a.k, a.rows, flags);
        launch_chained(map_kernel, 1, 1024, 0, stream, a.index, a.ignore_index, flags, a.rows, o.map, o.live);
        // the rows that are left out
        if (none && (e = cudaMemsetAsync(a.loss, 0, (size_t)a.rows * sizeof(float), stream)) != cudaSuccess) return e;
    }
    Lists lists{};
    if (a.kd && l.few) {
        const int n = a.rows * a.k;
        if (a.bf16)
            launch_chained(pick_kernel<__nv_bfloat16>, ceil_div(n, 8), 256, 0, stream,
                static_cast<const __nv_bfloat16 *>(a.x), a.ldx, static_cast<const __nv_bfloat16 *>(a.w), a.ldw,
                a.index, a.k, c, o.logq2, rest, n, a.vocab, a.dim);
        else
            launch_chained(pick_kernel<float>, ceil_div(n, 8), 256, 0, stream,
                static_cast<const float *>(a.x), a.ldx, static_cast<const float *>(a.w), a.ldw, a.index, a.k, c,
                o.logq2, rest, n, a.vocab, a.dim);
    } else if (a.kd) {
        int *col = reinterpret_cast<int *>(fl(a.workspace, l.col));
        uint16_t *pos = u16(a.workspace, l.pos), *before = u16(a.workspace, l.before);
        launch_chained(order_kernel, ceil_div(a.rows, 8), 256, 8 * a.k * sizeof(int), stream, a.index, a.k, a.rows, rm, a.vocab,
                                                                                col, pos, o.logq2, rest);
        // few rows: more CTAs a row, down to 4 blocks a thread
        const int blocks = (a.vocab - 1) / LIST_BLOCK + 1, ctas = ceil_div(a.rows, 32);
        const dim3 grid(ctas, std::max(1, std::min(2 * 148 / ctas, blocks / 32)));
        launch_chained(before_kernel, grid, 256, 0, stream, col, a.k, a.rows, rm, blocks, before);
        lists = Lists{col, pos, before, a.k, a.rows};
    }
    if (l.few) {
        const int blocks = std::min(ceil_div(a.vocab, 32), FEW_BLOCKS);
        FewArgs f = few_args(a, c);
        f.target = target; f.at = o.logq2; f.rest = rest; f.part = part + a.rows;
        if (a.bf16) launch_few<__nv_bfloat16>(f, blocks, false, stream);
        else launch_few<float>(f, blocks, false, stream);
        launch_chained(lse_kernel, 1, dim3(32, 32), 0, stream, part, true, blocks, true, true, a.rows, rm, o.lse2, target,
                                                  a.ignore_index, a.vocab, o.logq2, rest, rowloss, a.reduction,
                                                  total, o.count);
    }
    const Factor x = l.few ? Factor{} : x_factor(a, l, RowFactors{}, nullptr, rm, stream);
    if (finds_top(a, l)) top_of_w(a, w_top(a, l), stream);
    for (int v0 = l.few ? a.vocab : 0; v0 < a.vocab; v0 += l.piece) {
        const int nv = std::min(l.piece, a.vocab - v0);
        MmArgs mm{};
        mm.a = x;
        mm.b = w_factor(a, l, v0, nv, stream);
        mm.fp16 = !a.bf16;
        mm.m = a.rows; mm.n = nv; mm.k = a.dim; mm.c = c;
        mm.live = rm.live;
        mm.row_of = rm.map;
        if (l.scaled) {
            mm.row_mul = fl(a.workspace, l.row_mul);
            mm.mul = fl(a.workspace, l.muls);
        }
        mm.part = part + a.rows;                        // part 0: the pieces before
        mm.target = target;
        mm.lists = lists;
        mm.first_col = v0;
        mm.at = o.logq2;
        mm.rest = rest;
        if ((e = launch_mm(MM_LSE, mm, stream)) != cudaSuccess) return e;
        launch_chained(lse_kernel, ceil_div(a.rows, 32), dim3(32, 32), 0, stream,
            part, false, mm_lse_parts(a.rows, nv, a.dim, l.planes, l.planes), v0 == 0, v0 + nv == a.vocab, a.rows, rm,
            o.lse2, target, a.ignore_index, a.vocab, o.logq2, rest, rowloss, a.reduction, total, o.count);
    }
    if (a.kd)
        launch_chained(kd_kernel, ceil_div(a.rows, 8), 256, 0, stream, a.index, a.logits, a.k, a.tau, o.lse2, o.logq2, rest,
                                                          o.prob, rowloss, a.rows, rm, a.reduction);
    if (!total)
        launch_chained(total_kernel, 1, 1024, 0, stream, rowloss, a.index, o.prob, a.k, a.ignore_index, a.rows, rm, a.reduction,
                                             a.loss, o.count);
    return cudaGetLastError();
}

cudaError_t launch_head_bwd(const HeadArgs &a, cudaStream_t stream)
{
    chain_begin();
    const BwdLayout l = bwd_layout(a.rows, a.vocab, a.dim, a.bf16, a.ldw);
    const Kept o = kept_of(a);
    const RowMap rm{o.map, o.live};
    const float c = MMS_LOG2E / a.tau;
    // unscaled, all rows alike: dz without r, which comes in with the products' factors
    const bool uniform = !l.scaled && a.reduction != MMS_REDUCE_NONE;
    float *rs = fl(a.workspace, l.rs), *acc = fl(a.workspace, l.dxacc);
    float *pow = a.bf16 && l.scaled ? fl(a.workspace, l.pow) : nullptr;
    const float *row_by = pow ? pow : rs;               // what dz is without: E or r
    float *muls = fl(a.workspace, l.muls), *row_mul = fl(a.workspace, l.row_mul);
    cudaError_t e;
    // the rows that are left out
    if (rm.live && a.dx &&
        (e = cudaMemsetAsync(a.dx, 0, (size_t)a.rows * a.dim * (a.bf16 ? 2 : 4), stream)) != cudaSuccess)
        return e;
    const RowFactors from{a.dloss, o.count, o.prob, o.logq2, a.index, a.ignore_index, a.k, a.reduction, a.tau, rs,
                          pow, uniform ? muls + 1 : nullptr};
    const Factor x = x_factor(a, l, from, l.scaled ? fl(a.workspace, l.tops) : nullptr, rm, stream);
    if (finds_top(a, l)) top_of_w(a, w_top(a, l), stream);
    Factor xr = x;                                      // the factor of dw: x, r x or E x
    if (l.scaled) {
        StageArgs st{};
        st.src = a.x; st.lds = a.ldx;
        st.out = u16(a.workspace, l.xr); st.ld = x.ld; st.plane = x.plane;
        st.rows = a.rows; st.cols = a.dim; st.rows_map = rm;
        st.rs = row_by;
        st.mul = muls + 1;
        st.top = fl(a.workspace, l.tops); st.tops = stage_grid(a.rows, a.dim);
        stage_scaled<ST_WHOLE>(a, st, stream);
        xr.p = st.out;
    }
    xr.t = true;
    const long long n = (long long)a.rows * a.k, gplane = (long long)a.rows * l.ldg;
    const float unit = !a.bf16 ? DZ_UNIT : uniform ? 1.f : 0.f;
    uint16_t *g = u16(a.workspace, l.g);
    for (int v0 = 0; v0 < a.vocab; v0 += l.piece) {
        const int nv = std::min(l.piece, a.vocab - v0);
        const bool first = v0 == 0, last = v0 + nv == a.vocab;
        MmArgs mm{};
        mm.a = x;
        mm.b = w_factor(a, l, v0, nv, stream);
        mm.fp16 = l.scaled;
        mm.m = a.rows; mm.n = nv; mm.k = a.dim; mm.c = c;
        mm.live = rm.live;
        if (l.scaled) {
            mm.row_mul = row_mul;
            mm.mul = muls;
        }
        mm.lse2 = o.lse2; mm.rs = rs; mm.g_unit = unit;
        mm.g = g; mm.ldg = l.ldg; mm.gplane = gplane; mm.gplanes = l.gplanes;
        if (l.few) {
            FewArgs f = few_args(a, c);
            f.lse2 = o.lse2; f.rs = rs; f.unit = unit; f.g = g; f.ldg = l.ldg; f.gplane = gplane;
            f.v0 = v0; f.n = nv;
            const int blocks = std::min(ceil_div(nv, 32), FEW_BLOCKS);
            if (a.bf16) launch_few<__nv_bfloat16>(f, blocks, true, stream);
            else launch_few<float>(f, blocks, true, stream);
        } else if ((e = launch_mm(MM_GRAD, mm, stream)) != cudaSuccess) {
            return e;
        }
        launch_chained(sparse_kernel, ceil_div(n, 256), 256, 0, stream, a.index, o.prob, o.logq2, rs, unit, a.k, a.rows, rm, v0,
                                                            v0 + nv, g, l.ldg, gplane, l.gplanes, l.scaled);
        MmArgs out{};
        out.fp16 = l.scaled;
        out.c = l.scaled ? 1.f / DZ_UNIT : 1.f;
        out.n = a.dim;
        out.live = rm.live;
        out.split = fl(a.workspace, l.split);
        out.split_bytes = l.split_bytes;
        out.a = Factor{g, l.ldg, gplane, l.gplanes, false};
        if (a.dx) {
            out.b = mm.b;
            out.b.t = true;
            out.m = a.rows; out.k = nv;
            out.row_mul = l.scaled || uniform ? row_by : nullptr;
            out.mul = l.scaled ? muls : nullptr;
            out.acc = first ? nullptr : acc;
            out.out = last ? a.dx : acc;
            out.out_bf16 = last && a.bf16;
            out.row_of = last ? rm.map : nullptr;
            if ((e = launch_mm(MM_OUT, out, stream)) != cudaSuccess) return e;
            out.row_of = nullptr;
        }
        if (a.dw) {
            out.a.t = true;
            out.b = xr;
            out.m = nv; out.k = a.rows;
            out.row_mul = nullptr;
            out.mul = l.scaled || uniform ? muls + 1 : nullptr;
            out.acc = nullptr;
            out.out = static_cast<char *>(a.dw) + (size_t)v0 * a.dim * (a.bf16 ? 2 : 4);
            out.out_bf16 = a.bf16;
            if ((e = launch_mm(MM_OUT, out, stream)) != cudaSuccess) return e;
        }
    }
    return cudaGetLastError();
}

}  // namespace mms
