// Internal interface of the head's losses (mms_head.cu) and their matrix
// products (mms_head_mm.cu), and of the residual norm (mms_norm.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mms {

// A factor of a product: `planes` matrices of 16-bit floats, apart by `plane`
// elements, whose sum is the factor. Element (r, k), with k the summed index,
// is at p[r * ld + k], or at p[k * ld + r] if `t`.
struct Factor {
    const uint16_t *p;
    long long ld, plane;
    int planes;
    bool t;
};

// The three products of the losses, s[m, n] = f sum_k a(m, k) b(n, k) with
// f = c * (row_mul ? row_mul[m] : 1) * (mul ? *mul : 1):
//   MM_LSE    each row's log-sum-exp over parts of the columns:
//             part[i * m + row] = (max, sum of 2^(s - max)), in units of log 2,
//             i < mm_lse_parts()
//   MM_GRAD   g[m, n] = r 2^(s - lse2[m].x - lse2[m].y) as planes of 16-bit floats; 0 where
//             rs[m] is 0; r = rs[m], or the constant g_unit if that is not 0
//   MM_OUT    out[m, n] = s (+ acc[m, n]), float32 or bf16
enum MmKind { MM_LSE, MM_GRAD, MM_OUT };
constexpr int MM_COLS = 256;            // columns of the widest tile

// Columns of each row in ascending order: col[m * k + i] (INT_MAX: none), the
// place pos[m * k + i] each had before, and before[b * rows + m], how many of
// them lie below column LIST_BLOCK * b.
constexpr int LIST_BLOCK = 128;
struct Lists {
    const int *col;
    const uint16_t *pos, *before;
    int k, rows;
};

// What a * b lost by rounding to p; 0 where p is not finite.
__device__ __forceinline__ float rounding_of(float a, float b, float p) {
    const float r = fmaf(a, b, -p);
    return r == r ? r : 0.f;
}

struct MmArgs {
    Factor a, b;
    bool fp16;                  // the planes are fp16, else bf16
    int m, n, k;
    // How many of a's rows there are, or (a transposed) of the summed elements:
    // *live <= m (k); null: all. The rest is not read but for the padding that
    // fills a last step (64 elements) or tile (256 rows; MM_GRAD writes those
    // rows, as zeros where rs is 0).
    const int *live;
    const int *row_of;          // row m's place in target and in out (not in `acc`, nor in partial sums); null: m
    float c;
    const float *row_mul, *mul;
    float2 *part;               // MM_LSE
    // MM_LSE: the products at given columns. One a row: where target[row_of[m]] - first_col
    // is a column, at[m] + rest[m] = s, rest the rounding of at. Or `lists` of them
    // (see Lists) at m * k + pos.
    const int64_t *target;
    Lists lists;                // lists.col may be null
    float *at, *rest;
    int first_col;              // of column 0
    const float2 *lse2;         // MM_GRAD: (top, log2 of the sum of 2^(s - top))
    const float *rs;            // MM_GRAD
    float g_unit;               // MM_GRAD
    uint16_t *g;                // MM_GRAD
    long long ldg, gplane;      // MM_GRAD
    int gplanes;                // MM_GRAD
    const float *acc;           // MM_OUT: added, row stride n; may be null
    void *out;                  // MM_OUT, row stride n
    bool out_bf16;              // MM_OUT
    float *split;               // MM_OUT: room for partial sums,
    size_t split_bytes;         //         mm_split_bytes() or less
};

// Planes: 1 x 1, 2 x 1 or 2 x 2; the product of the second planes is left out.
int mm_lse_parts(int m, int n, int k, int planes_a, int planes_b);
// live: for a product whose `live` rows are fewer than m
size_t mm_split_bytes(int m, int n, int k, int planes_a, int planes_b, bool live);
// Factors: 16-byte aligned, ld and plane multiples of 8. `g`: 16-byte aligned,
// ldg and gplane multiples of 8, its rows are written up to the next multiple
// of 8 columns. `out` 16-byte aligned.
cudaError_t launch_mm(MmKind kind, const MmArgs &a, cudaStream_t stream);
// 1 if a wait of the products timed out since the last call (and clears it),
// 0 if not, -1 if the flag could not be read.
int mm_take_timeout();

// The two losses share everything but their sparse part: row m has the
// entries index[m, 0..k), and for the distillation their probabilities.
struct HeadArgs {
    const void *x, *w;
    long long ldx, ldw;
    int rows, vocab, dim;
    bool bf16;
    const int64_t *index;       // target or teacher_index
    int64_t ignore_index;       // cross entropy
    const float *logits;        // distillation, forward
    int k;
    bool kd;
    float tau;
    int reduction;
    float *loss;
    void *kept;                 // written by the forward, read by the backward (KeptLayout)
    const float *dloss;
    void *dx, *dw;
    void *workspace;
    bool backward;
};

size_t head_kept_bytes(int rows, int k, bool kd);
// k: entries of the distillation's lists, 0 for the cross entropy
size_t head_workspace_bytes(int rows, int vocab, int dim, int k, bool bf16, long long ldx, long long ldw,
                            bool backward);
cudaError_t launch_head_fwd(const HeadArgs &a, cudaStream_t stream);
cudaError_t launch_head_bwd(const HeadArgs &a, cudaStream_t stream);

struct NormArgs {
    const void *x, *y, *gate, *weight, *post, *scale;
    long long ldg;
    float eps;
    void *h, *u;
    float *stat;
    const float *c_stat;
    const void *dh, *du;
    void *dx, *dy, *dgate, *dweight, *dpost, *dscale;
    void *workspace;
    int rows, dim;
    bool bf16;
};

size_t norm_workspace_bytes(int rows, int dim);
cudaError_t launch_norm_fwd(const NormArgs &a, cudaStream_t stream);
cudaError_t launch_norm_bwd(const NormArgs &a, cudaStream_t stream);

}  // namespace mms
