// Internal interface of the head's losses (mms_head.cu) and their matrix
// products (mms_head_mm.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mms {

// A factor of a product: 1 bf16 matrix, or 3 (planes apart by `plane`
// elements) whose sum is the fp32 matrix. Element (r, k), with k the summed
// index, is at p[r * ld + k], or at p[k * ld + r] if `t`.
struct Factor {
    const __nv_bfloat16 *p;
    long long ld, plane;
    bool t;
};

// The three products of the losses, s[m, n] = sum_k a(m, k) b(n, k):
//   MM_LSE    each row's log-sum-exp over parts of the columns:
//             part[i * m + row] = (max, sum of 2^(c s - max)), in units of log 2,
//             i < mm_lse_parts()
//   MM_GRAD   g[m, n] = rs[m] 2^(c s - lse2[m]) (0 where rs[m] is 0), as bf16 planes
//   MM_OUT    out[m, n] = s (+ acc[m, n]), float32 or bf16
enum MmKind { MM_LSE, MM_GRAD, MM_OUT };
constexpr int MM_COLS = 256;            // columns of the widest tile

struct MmArgs {
    Factor a, b;
    int m, n, k;
    int planes;                 // 1 or 3, of both factors (and of g)
    float c;                    // MM_LSE, MM_GRAD
    float2 *part;               // MM_LSE
    const float *lse2, *rs;     // MM_GRAD
    __nv_bfloat16 *g;           // MM_GRAD
    long long ldg, gplane;      // MM_GRAD
    const float *acc;           // MM_OUT: added, (m, n) with row stride ldo; may be null
    void *out;                  // MM_OUT
    long long ldo;              // MM_OUT (= n where split may be used)
    bool out_bf16;              // MM_OUT
    float *split;               // MM_OUT: room for partial sums over parts of k,
    size_t split_bytes;         //         mm_split_bytes() or less
};

int mm_lse_parts(int m, int n, int k, int planes);
size_t mm_split_bytes(int m, int n, int k, int planes);

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
    float *loss, *lse2, *picked, *prob, *count;     // forward outputs
    const float *dloss, *c_lse2, *c_picked, *c_prob, *c_count;   // backward inputs
    void *dx, *dw;
    void *workspace;
};

size_t head_workspace_bytes(int rows, int vocab, int dim, bool bf16, long long ldx, long long ldw,
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
