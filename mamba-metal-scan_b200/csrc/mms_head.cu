// Losses of a language model's head without its logits (sm_100a): softmax
// cross entropy and distillation from a teacher's top k, forward and backward.
//
// With z = x w^T (rows x vocab) and c = log2(e) / tau (tau = 1 for the cross
// entropy), in units of log 2:
//     lse2[m]   = log2 sum_v 2^(c z[m, v])
//     picked[m, j] = c z[m, index[m, j]]
//     CE  loss  = ln2 (lse2 - picked)
//     KD  loss  = tau^2 sum_j p_j (log p_j - ln2 (picked_j - lse2))
// and for an upstream factor r[m] (dloss, times 1 / count for a mean, times
// tau for the distillation; 0 for a row that is left out):
//     dz[m, v]  = r (2^(c z - lse2) - sum of p_j with index_j = v)
//     dx = dz w,   dw = dz^T x
// z is computed once forward (2 rows vocab dim flops) and again backward, in
// pieces of the vocabulary small enough that dz's piece stays in a bounded
// workspace; the two products with dz follow piece by piece (6 more).
//
// Forward:   products (MM_LSE) -> one (max, sum) per row and half tile;
//            pick_kernel: the dot products at the indices; lse_kernel joins
//            the parts; a loss kernel; for mean / sum one block adds rows up.
// Backward:  rows_kernel: r; stage_kernel: x with the left-out rows as zeros
//            (so that nothing in them, NaN included, reaches dw); per piece:
//            product MM_GRAD, sparse_kernel sets dz at the indices (from
//            picked, in fp32, as r (expm1(log q) + 1 - p): no cancellation
//            when a target's probability is near 1), then MM_OUT twice.
//
// fp32 factors are split into three bf16 planes (8 bits of mantissa each):
// the products of planes i + j <= 2 leave out terms below 2^-24.
#include <algorithm>

#include "mms_common.cuh"
#include "mms_head.h"
#include "mms_scan.h"

namespace mms {

namespace {

constexpr float LN2 = 0.6931471805599453f;
constexpr size_t PIECE_BYTES = (size_t)256 << 20;   // bound on one staged or dz piece

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }
size_t up256(size_t v) { return (v + 255) / 256 * 256; }
long long padded(int dim) { return (dim + 7) / 8 * 8; }     // rows of 16-byte multiples

// Pieces of the vocabulary (each a multiple of MM_COLS rows of w but the
// last): as few equal ones as keep `bytes_per_row` (per vocabulary entry)
// times the piece below PIECE_BYTES, at least 4096 entries each so that a
// piece's products stay long.
int piece_size(int vocab, size_t bytes_per_row)
{
    const long long most = std::max<long long>(4096, (long long)(PIECE_BYTES / bytes_per_row));
    const int pieces = ceil_div(vocab, most);
    const long long v = ceil_div(ceil_div(vocab, pieces), MM_COLS) * (long long)MM_COLS;
    return (int)std::min<long long>(v, vocab);
}

struct FwdLayout {
    bool stage_x, stage_w;
    int planes, piece;
    size_t xs, ws, part, rowloss, total;
};

FwdLayout fwd_layout(int rows, int vocab, int dim, bool bf16, long long ldx, long long ldw)
{
    FwdLayout l;
    l.planes = bf16 ? 1 : 3;
    l.stage_x = !bf16 || ldx % 8;
    l.stage_w = !bf16 || ldw % 8;
    const size_t row = (size_t)padded(dim) * 2 * l.planes;
    l.piece = piece_size(vocab, std::max<size_t>(l.stage_w ? row : 1,
                                                 (size_t)rows * sizeof(float2) / 64 + 1));
    const int last = vocab - (vocab - 1) / l.piece * l.piece;
    size_t o = 0;
    l.xs = o; o += l.stage_x ? up256(row * rows) : 0;
    l.ws = o; o += l.stage_w ? up256(row * l.piece) : 0;
    l.part = o; o += up256((size_t)(std::max(mm_lse_parts(rows, l.piece, dim, l.planes),
                                            mm_lse_parts(rows, last, dim, l.planes)) + 1) * rows * sizeof(float2));
    l.rowloss = o; o += up256((size_t)rows * sizeof(float));
    l.total = o;
    return l;
}

struct BwdLayout {
    bool stage_w;
    int planes, piece;
    long long ldg;
    size_t xs, ws, g, dxacc, rs, split, split_bytes, total;
};

BwdLayout bwd_layout(int rows, int vocab, int dim, bool bf16, long long ldw)
{
    BwdLayout l;
    l.planes = bf16 ? 1 : 3;
    l.stage_w = !bf16 || ldw % 8;
    const size_t row = (size_t)padded(dim) * 2 * l.planes;
    l.piece = piece_size(vocab, std::max<size_t>(l.stage_w ? row : 1, (size_t)rows * 2 * l.planes));
    l.ldg = (l.piece + 7) / 8 * 8;
    size_t o = 0;
    l.xs = o; o += up256(row * rows);
    l.ws = o; o += l.stage_w ? up256(row * l.piece) : 0;
    l.g = o; o += up256((size_t)rows * l.ldg * 2 * l.planes);
    l.dxacc = o; o += l.piece < vocab ? up256((size_t)rows * dim * sizeof(float)) : 0;
    l.rs = o; o += up256((size_t)rows * sizeof(float));
    // partial sums; the last, smaller piece splits as far as this room goes
    l.split_bytes = std::max(mm_split_bytes(rows, dim, l.piece, l.planes),
                             mm_split_bytes(l.piece, dim, rows, l.planes));
    l.split = o; o += up256(l.split_bytes);
    l.total = o;
    return l;
}

// out[p, r, 0..cols) = the bf16 planes of src[r, 0..cols); rows with rs = 0
// (if given) as zeros. Row stride ld of out, planes apart by `plane`.
template <typename T>
__global__ void __launch_bounds__(256)
stage_kernel(const T *__restrict__ src, long long lds, const float *__restrict__ rs,
             __nv_bfloat16 *__restrict__ out, long long ld, long long plane, int rows, int cols,
             int planes)
{
    const long long total = (long long)rows * cols;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total;
         i += (long long)gridDim.x * 256) {
        const long long r = i / cols;
        const int c = (int)(i - r * cols);
        float v = to_f(src[r * lds + c]);
        if (rs && rs[r] == 0.f) v = 0.f;
        for (int p = 0; p < planes; ++p) {
            const __nv_bfloat16 q = __float2bfloat16_rn(v);
            out[p * plane + r * ld + c] = q;
            v -= to_f(q);
        }
    }
}

template <typename T>
void stage(const void *src, long long lds, const float *rs, __nv_bfloat16 *out, long long ld,
           long long plane, int rows, int cols, int planes, cudaStream_t stream)
{
    const long long blocks = ((long long)rows * cols + 255) / 256;
    stage_kernel<T><<<(int)std::min<long long>(blocks, 148 * 16), 256, 0, stream>>>(
        static_cast<const T *>(src), lds, rs, out, ld, plane, rows, cols, planes);
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

// picked[m, j] = c * (x[m] . w[index[m, j]]), a warp each; NaN for an index
// outside the vocabulary, 0 for an entry that is left out.
template <typename T>
__global__ void __launch_bounds__(256)
pick_kernel(const T *__restrict__ x, long long ldx, const T *__restrict__ w, long long ldw,
            const int64_t *__restrict__ index, bool kd, int64_t ignore, int k, float c,
            float *__restrict__ picked, long long n, int vocab, int dim)
{
    const long long e = (long long)blockIdx.x * 8 + threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    if (e >= n) return;
    const int64_t v = index[e];
    float s = 0.f;
    if (kd ? v < 0 : v == ignore) {
    } else if (v < 0 || v >= vocab) {
        s = __int_as_float(0x7fc00000);
    } else {
        const T *xr = x + e / k * ldx, *wr = w + v * ldw;
        for (int i = lane; i < dim; i += 32) s = fmaf(to_f(xr[i]), to_f(wr[i]), s);
        s = warp_sum(s) * c;
    }
    if (lane == 0) picked[e] = s;
}

// (max, sum) pairs join to the pair of both; a NaN in either sum stays.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x);
    if (m == -INFINITY) return make_float2(m, a.y + b.y);
    return make_float2(m, a.y * ex2(a.x - m) + b.y * ex2(b.x - m));
}

// One row a lane, 32 threads a row over the tiles. Parts 1..ntiles, and part
// 0 (the pieces before) unless `first`. Writes part 0, or in the last piece
// lse2 and the cross entropy's row loss.
__global__ void __launch_bounds__(1024)
lse_kernel(float2 *part, int ntiles, bool first, bool last, int rows, float *__restrict__ lse2,
           const int64_t *__restrict__ target, int64_t ignore, const float *__restrict__ picked,
           float *__restrict__ loss)
{
    __shared__ float2 sh[32][33];
    const int m = blockIdx.x * 32 + threadIdx.x;
    float2 v = make_float2(-INFINITY, 0.f);
    if (m < rows)
        for (int t = threadIdx.y + (first ? 1 : 0); t <= ntiles; t += 32)
            v = join(v, part[(size_t)t * rows + m]);
    sh[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    // transposed: a warp joins the 32 values of one row
    v = sh[threadIdx.x][threadIdx.y];
#pragma unroll
    for (int o = 16; o; o >>= 1)
        v = join(v, make_float2(__shfl_xor_sync(~0u, v.x, o), __shfl_xor_sync(~0u, v.y, o)));
    const int r = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x || r >= rows) return;
    if (!last) {
        part[r] = v;
        return;
    }
    const float l = v.x + log2f(v.y);
    lse2[r] = l;
    if (target) loss[r] = target[r] == ignore ? 0.f : LN2 * (l - picked[r]);
}

// Distillation's row loss, a warp a row: the teacher's softmax over its
// entries, kept as prob, against the student's log-probabilities.
__global__ void __launch_bounds__(256)
kd_kernel(const int64_t *__restrict__ index, const float *__restrict__ logits, int k, float tau,
          const float *__restrict__ lse2, const float *__restrict__ picked,
          float *__restrict__ prob, float *__restrict__ loss, int rows)
{
    const int m = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
    if (m >= rows) return;
    const size_t o = (size_t)m * k;
    const float inv = 1.f / tau, l2 = lse2[m];
    float top = -INFINITY;
    for (int j = lane; j < k; j += 32)
        if (index[o + j] >= 0) top = fmaxf(top, logits[o + j]);
    top = warp_max(top);
    float sum = 0.f;
    for (int j = lane; j < k; j += 32)
        if (index[o + j] >= 0 && !(top == -INFINITY && logits[o + j] == -INFINITY))
            sum += expf((logits[o + j] - top) * inv);
    sum = warp_sum(sum);
    const float log_sum = logf(sum), over = 1.f / sum;
    const bool some = sum != 0.f;                       // NaN counts as some
    float acc = 0.f;
    for (int j = lane; j < k; j += 32) {
        float p = 0.f;
        if (some && index[o + j] >= 0) {
            const float t = (logits[o + j] - top) * inv;
            p = expf(t) * over;
            if (p != 0.f) acc += p * ((t - log_sum) - LN2 * (picked[o + j] - l2));
        }
        prob[o + j] = p;
    }
    acc = warp_sum(acc);
    if (lane == 0) loss[m] = some ? tau * tau * acc : 0.f;
}

// Whether row m counts.
__device__ __forceinline__ bool row_counts(const int64_t *index, const float *prob, int k,
                                           int64_t ignore, size_t m) {
    if (!prob) return index[m] != ignore;
    for (int j = 0; j < k; ++j)
        if (!(prob[m * k + j] == 0.f)) return true;     // NaN counts
    return false;
}

// count, and loss = the rows' sum (over count for a mean), in a fixed order.
__global__ void __launch_bounds__(1024)
total_kernel(const float *__restrict__ rowloss, const int64_t *__restrict__ index,
             const float *__restrict__ prob, int k, int64_t ignore, int rows, int reduction,
             float *__restrict__ loss, float *__restrict__ count)
{
    __shared__ float sh[2][32];
    float s = 0.f, n = 0.f;
    for (int m = threadIdx.x; m < rows; m += 1024) {
        s += rowloss[m];
        n += row_counts(index, prob, k, ignore, m) ? 1.f : 0.f;
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

// rs[m]: the upstream factor of row m's dz; NaN where an index that counts
// lies outside the vocabulary (picked is NaN there).
__global__ void rows_kernel(const float *__restrict__ dloss, const float *__restrict__ count,
                            const int64_t *__restrict__ index, const float *__restrict__ prob,
                            const float *__restrict__ picked, int k, int64_t ignore, int reduction,
                            float tau, float *__restrict__ rs, int rows)
{
    const int m = blockIdx.x * blockDim.x + threadIdx.x;
    if (m >= rows) return;
    float r = dloss[reduction == MMS_REDUCE_NONE ? m : 0] * tau;
    if (reduction == MMS_REDUCE_MEAN) r /= *count;
    if (!row_counts(index, prob, k, ignore, m)) r = 0.f;
    if (r != 0.f)
        for (int j = 0; j < k; ++j) {
            const float z = picked[(size_t)m * k + j];
            if (z != z && !(prob && prob[(size_t)m * k + j] == 0.f)) r = z;
        }
    rs[m] = r;
}

// dz at the sparse entries that lie in this piece of the vocabulary.
__global__ void __launch_bounds__(256)
sparse_kernel(const int64_t *__restrict__ index, const float *__restrict__ prob,
              const float *__restrict__ picked, const float *__restrict__ lse2,
              const float *__restrict__ rs, int k, long long n, int v0, int v1,
              __nv_bfloat16 *__restrict__ g, long long ldg, long long gplane, int planes)
{
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    if (e >= n) return;
    const int64_t v = index[e];
    if (v < v0 || v >= v1) return;
    const long long m = e / k;
    const float r = rs[m];
    if (r == 0.f) return;                               // dz is 0 there already
    float p = 1.f;
    if (prob) {                                         // an index may occur twice
        p = 0.f;
        for (int j = 0; j < k; ++j)
            if (index[m * k + j] == v) p += prob[m * k + j];
    }
    float d = r * (expm1f(LN2 * (picked[e] - lse2[m])) + (1.f - p));
    for (int q = 0; q < planes; ++q) {
        const __nv_bfloat16 t = __float2bfloat16_rn(d);
        g[q * gplane + m * ldg + (v - v0)] = t;
        d -= to_f(t);
    }
}

__nv_bfloat16 *bf(void *base, size_t off) {
    return reinterpret_cast<__nv_bfloat16 *>(static_cast<char *>(base) + off);
}
float *fl(void *base, size_t off) { return reinterpret_cast<float *>(static_cast<char *>(base) + off); }

void stage_any(bool bf16, const void *src, long long lds, const float *rs, __nv_bfloat16 *out,
               long long ld, long long plane, int rows, int cols, int planes, cudaStream_t stream)
{
    if (bf16) stage<__nv_bfloat16>(src, lds, rs, out, ld, plane, rows, cols, planes, stream);
    else stage<float>(src, lds, rs, out, ld, plane, rows, cols, planes, stream);
}

// Rows [v0, v0 + n) of w as a factor: staged, or w itself.
Factor w_factor(const HeadArgs &a, bool staged, __nv_bfloat16 *ws, int piece, int planes, int v0,
                int n, bool t, cudaStream_t stream)
{
    if (!staged) return Factor{static_cast<const __nv_bfloat16 *>(a.w) + (size_t)v0 * a.ldw, a.ldw, 0, t};
    const long long ld = padded(a.dim), plane = ld * piece;
    const char *src = static_cast<const char *>(a.w) + (size_t)v0 * a.ldw * (a.bf16 ? 2 : 4);
    stage_any(a.bf16, src, a.ldw, nullptr, ws, ld, plane, n, a.dim, planes, stream);
    return Factor{ws, ld, plane, t};
}

}  // namespace

size_t head_workspace_bytes(int rows, int vocab, int dim, bool bf16, long long ldx, long long ldw,
                            bool backward)
{
    return backward ? bwd_layout(rows, vocab, dim, bf16, ldw).total
                    : fwd_layout(rows, vocab, dim, bf16, ldx, ldw).total;
}

cudaError_t launch_head_fwd(const HeadArgs &a, cudaStream_t stream)
{
    const FwdLayout l = fwd_layout(a.rows, a.vocab, a.dim, a.bf16, a.ldx, a.ldw);
    const float c = MMS_LOG2E / a.tau;
    float2 *part = reinterpret_cast<float2 *>(fl(a.workspace, l.part));
    float *rowloss = a.reduction == MMS_REDUCE_NONE ? a.loss : fl(a.workspace, l.rowloss);
    const long long n = (long long)a.rows * a.k;
    const int pick_grid = ceil_div(n, 8);
    if (a.bf16)
        pick_kernel<__nv_bfloat16><<<pick_grid, 256, 0, stream>>>(
            static_cast<const __nv_bfloat16 *>(a.x), a.ldx, static_cast<const __nv_bfloat16 *>(a.w),
            a.ldw, a.index, a.kd, a.ignore_index, a.k, c, a.picked, n, a.vocab, a.dim);
    else
        pick_kernel<float><<<pick_grid, 256, 0, stream>>>(
            static_cast<const float *>(a.x), a.ldx, static_cast<const float *>(a.w), a.ldw, a.index,
            a.kd, a.ignore_index, a.k, c, a.picked, n, a.vocab, a.dim);
    Factor x{static_cast<const __nv_bfloat16 *>(a.x), a.ldx, 0, false};
    if (l.stage_x) {
        x = Factor{bf(a.workspace, l.xs), padded(a.dim), padded(a.dim) * a.rows, false};
        stage_any(a.bf16, a.x, a.ldx, nullptr, bf(a.workspace, l.xs), x.ld, x.plane, a.rows, a.dim,
                  l.planes, stream);
    }
    for (int v0 = 0; v0 < a.vocab; v0 += l.piece) {
        const int nv = std::min(l.piece, a.vocab - v0);
        const bool last = v0 + nv == a.vocab;
        MmArgs mm{};
        mm.a = x;
        mm.b = w_factor(a, l.stage_w, bf(a.workspace, l.ws), l.piece, l.planes, v0, nv, false, stream);
        mm.m = a.rows; mm.n = nv; mm.k = a.dim; mm.planes = l.planes; mm.c = c;
        mm.part = part + a.rows;                        // part 0: the pieces before
        cudaError_t e = launch_mm(MM_LSE, mm, stream);
        if (e != cudaSuccess) return e;
        lse_kernel<<<ceil_div(a.rows, 32), dim3(32, 32), 0, stream>>>(
            part, mm_lse_parts(a.rows, nv, a.dim, l.planes), v0 == 0, last, a.rows, a.lse2,
            a.kd ? nullptr : a.index, a.ignore_index, a.picked, rowloss);
    }
    if (a.kd)
        kd_kernel<<<ceil_div(a.rows, 8), 256, 0, stream>>>(a.index, a.logits, a.k, a.tau, a.lse2,
                                                          a.picked, a.prob, rowloss, a.rows);
    total_kernel<<<1, 1024, 0, stream>>>(rowloss, a.index, a.kd ? a.prob : nullptr, a.k,
                                         a.ignore_index, a.rows, a.reduction, a.loss, a.count);
    return cudaGetLastError();
}

cudaError_t launch_head_bwd(const HeadArgs &a, cudaStream_t stream)
{
    const BwdLayout l = bwd_layout(a.rows, a.vocab, a.dim, a.bf16, a.ldw);
    const float c = MMS_LOG2E / a.tau;
    const float *prob = a.kd ? a.c_prob : nullptr;
    float *rs = fl(a.workspace, l.rs), *acc = fl(a.workspace, l.dxacc);
    rows_kernel<<<ceil_div(a.rows, 256), 256, 0, stream>>>(a.dloss, a.c_count, a.index, prob,
                                                           a.c_picked, a.k, a.ignore_index,
                                                           a.reduction, a.tau, rs, a.rows);
    const long long ldx = padded(a.dim), n = (long long)a.rows * a.k;
    __nv_bfloat16 *xs = bf(a.workspace, l.xs), *g = bf(a.workspace, l.g);
    stage_any(a.bf16, a.x, a.ldx, rs, xs, ldx, ldx * a.rows, a.rows, a.dim, l.planes, stream);
    const long long gplane = (long long)a.rows * l.ldg;
    for (int v0 = 0; v0 < a.vocab; v0 += l.piece) {
        const int nv = std::min(l.piece, a.vocab - v0);
        const bool first = v0 == 0, last = v0 + nv == a.vocab;
        MmArgs mm{};
        mm.planes = l.planes;
        mm.a = Factor{xs, ldx, ldx * a.rows, false};
        mm.b = w_factor(a, l.stage_w, bf(a.workspace, l.ws), l.piece, l.planes, v0, nv, false, stream);
        mm.m = a.rows; mm.n = nv; mm.k = a.dim; mm.c = c;
        mm.lse2 = a.c_lse2; mm.rs = rs; mm.g = g; mm.ldg = l.ldg; mm.gplane = gplane;
        cudaError_t e = launch_mm(MM_GRAD, mm, stream);
        if (e != cudaSuccess) return e;
        sparse_kernel<<<ceil_div(n, 256), 256, 0, stream>>>(a.index, prob, a.c_picked, a.c_lse2, rs,
                                                            a.k, n, v0, v0 + nv, g, l.ldg, gplane,
                                                            l.planes);
        MmArgs out{};
        out.planes = l.planes;
        out.split = fl(a.workspace, l.split);
        out.split_bytes = l.split_bytes;
        if (a.dx) {
            out.a = Factor{g, l.ldg, gplane, false};
            out.b = mm.b;
            out.b.t = true;
            out.m = a.rows; out.n = a.dim; out.k = nv; out.ldo = a.dim;
            out.acc = first ? nullptr : acc;
            out.out = last ? a.dx : acc;
            out.out_bf16 = last && a.bf16;
            if ((e = launch_mm(MM_OUT, out, stream)) != cudaSuccess) return e;
        }
        if (a.dw) {
            out.a = Factor{g, l.ldg, gplane, true};
            out.b = Factor{xs, ldx, ldx * a.rows, true};
            out.m = nv; out.n = a.dim; out.k = a.rows; out.ldo = a.dim;
            out.acc = nullptr;
            out.out = static_cast<char *>(a.dw) + (size_t)v0 * a.dim * (a.bf16 ? 2 : 4);
            out.out_bf16 = a.bf16;
            if ((e = launch_mm(MM_OUT, out, stream)) != cudaSuccess) return e;
        }
    }
    return cudaGetLastError();
}

}  // namespace mms
