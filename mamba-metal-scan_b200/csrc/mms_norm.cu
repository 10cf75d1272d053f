// Residual sum after a block fused with the norms around it (sm_100a):
//     a = y silu(gate);  b = post a r1;  h = x + scale b;  u = weight h r2
//     r1 = 1 / sqrt(mean(a^2) + eps),    r2 = 1 / sqrt(mean(h^2) + eps)
// and with n = h r2, t = weight du, the gradients
//     dh' = dh + r2 (t - n mean(t n))            dx = dh'
//     dscale = sum over rows of dh' b,           db = scale dh'
//     dpost = sum over rows of db a r1,          s = post db
//     da = r1 (s - a r1 mean(s a r1))
//     dy = da silu(gate),                        dgate = da y silu'(gate)
//     dweight = sum over rows of du n
// All of it in fp32 from the inputs as stored; outputs are rounded once.
#include "mms_common.cuh"
#include "mms_head.h"

namespace mms {

namespace {

constexpr int NT = 256;
constexpr int MAX_BLOCKS = 148 * 4;

int blocks_for(int rows) { return rows < MAX_BLOCKS ? rows : MAX_BLOCKS; }

__device__ __forceinline__ float block_sum(float v, float *sh) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) v += sh[i];
    __syncthreads();
    return v;
}

template <typename T>
struct Row {
    const T *x, *y, *gate, *w, *post, *scale;
    __device__ __forceinline__ float gate_at(int i, float &sig) const {
        const float z = to_f(gate[i]);
        sig = 1.f / (1.f + expf(-z));
        return z * sig;
    }
    __device__ __forceinline__ float a_at(int i) const {
        float s;
        return gate ? to_f(y[i]) * gate_at(i, s) : to_f(y[i]);
    }
    __device__ __forceinline__ float b_at(int i, float r1) const {
        const float a = a_at(i);
        return post ? a * r1 * to_f(post[i]) : a;
    }
    __device__ __forceinline__ float h_at(int i, float r1) const {
        const float b = b_at(i, r1);
        return to_f(x[i]) + (scale ? b * to_f(scale[i]) : b);
    }
};

template <typename T>
__device__ __forceinline__ Row<T> row_of(const NormArgs &a, size_t r) {
    return Row<T>{static_cast<const T *>(a.x) + r * a.dim, static_cast<const T *>(a.y) + r * a.dim,
                  a.gate ? static_cast<const T *>(a.gate) + r * a.ldg : nullptr,
                  static_cast<const T *>(a.weight), static_cast<const T *>(a.post),
                  static_cast<const T *>(a.scale)};
}

template <typename T>
__global__ void __launch_bounds__(NT) norm_fwd_kernel(const NormArgs a)
{
    __shared__ float sh[NT / 32];
    const float inv = 1.f / a.dim;
    for (size_t r = blockIdx.x; r < (size_t)a.rows; r += gridDim.x) {
        const Row<T> row = row_of<T>(a, r);
        float r1 = 0.f, s = 0.f;
        if (a.post) {
            for (int i = threadIdx.x; i < a.dim; i += NT) {
                const float v = row.a_at(i);
                s += v * v;
            }
            r1 = rsqrtf(block_sum(s, sh) * inv + a.eps);
            s = 0.f;
        }
        for (int i = threadIdx.x; i < a.dim; i += NT) {
            const float v = row.h_at(i, r1);
            s += v * v;
        }
        const float r2 = rsqrtf(block_sum(s, sh) * inv + a.eps);
        for (int i = threadIdx.x; i < a.dim; i += NT) {
            const float v = row.h_at(i, r1);
            static_cast<T *>(a.h)[r * a.dim + i] = from_f<T>(v);
            static_cast<T *>(a.u)[r * a.dim + i] = from_f<T>(v * r2 * to_f(row.w[i]));
        }
        if (threadIdx.x == 0 && a.stat) {
            a.stat[2 * r] = r1;
            a.stat[2 * r + 1] = r2;
        }
    }
}

// Partial sums over the rows of one block: part[(which * blocks + block) * dim + i].
template <typename T>
__global__ void __launch_bounds__(NT) norm_bwd_kernel(const NormArgs a)
{
    __shared__ float sh[NT / 32];
    const float inv = 1.f / a.dim;
    const size_t plane = (size_t)gridDim.x * a.dim;
    float *pw = static_cast<float *>(a.workspace) + (size_t)blockIdx.x * a.dim;
    float *ps = pw + plane, *pp = ps + plane;
    for (int i = threadIdx.x; i < a.dim; i += NT) pw[i] = ps[i] = pp[i] = 0.f;
    for (size_t r = blockIdx.x; r < (size_t)a.rows; r += gridDim.x) {
        const Row<T> row = row_of<T>(a, r);
        const T *dh = static_cast<const T *>(a.dh) + r * a.dim, *du = static_cast<const T *>(a.du) + r * a.dim;
        const float r1 = a.c_stat[2 * r], r2 = a.c_stat[2 * r + 1];
        float s = 0.f;
        for (int i = threadIdx.x; i < a.dim; i += NT) s += to_f(du[i]) * to_f(row.w[i]) * row.h_at(i, r1);
        const float mean = block_sum(s, sh) * inv * r2;
        const auto dh_at = [&](int i, float h) {
            return to_f(dh[i]) + r2 * (to_f(du[i]) * to_f(row.w[i]) - h * r2 * mean);
        };
        float mean1 = 0.f;
        if (a.post) {
            s = 0.f;
            for (int i = threadIdx.x; i < a.dim; i += NT) {
                const float d = dh_at(i, row.h_at(i, r1)) * (a.scale ? to_f(row.scale[i]) : 1.f);
                s += d * to_f(row.post[i]) * row.a_at(i);
            }
            mean1 = block_sum(s, sh) * inv * r1;
        }
        for (int i = threadIdx.x; i < a.dim; i += NT) {
            const size_t o = r * a.dim + i;
            const float av = row.a_at(i), b = row.b_at(i, r1), h = row.h_at(i, r1);
            const float d = dh_at(i, h);
            pw[i] += to_f(du[i]) * h * r2;
            float v = d;
            if (a.scale) {
                ps[i] += d * b;
                v *= to_f(row.scale[i]);
            }
            if (a.post) {
                pp[i] += v * av * r1;
                v = r1 * (v * to_f(row.post[i]) - av * r1 * mean1);
            }
            if (a.gate) {
                float sig;
                const float z = to_f(row.gate[i]), sl = row.gate_at(i, sig);
                static_cast<T *>(a.dgate)[o] = from_f<T>(v * to_f(row.y[i]) * (sig * (1.f + z * (1.f - sig))));
                v *= sl;
            }
            static_cast<T *>(a.dx)[o] = from_f<T>(d);
            static_cast<T *>(a.dy)[o] = from_f<T>(v);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(NT) norm_reduce_kernel(const NormArgs a, int blocks)
{
    const int i = blockIdx.x * NT + threadIdx.x, which = blockIdx.y;
    T *out = static_cast<T *>(which == 0 ? a.dweight : which == 1 ? a.dscale : a.dpost);
    if (i >= a.dim || !out) return;
    const float *p = static_cast<const float *>(a.workspace) + (size_t)which * blocks * a.dim + i;
    float s = 0.f;
    for (int b = 0; b < blocks; ++b) s += p[(size_t)b * a.dim];
    out[i] = from_f<T>(s);
}

}  // namespace

size_t norm_workspace_bytes(int rows, int dim)
{
    return (size_t)3 * blocks_for(rows) * dim * sizeof(float);
}

cudaError_t launch_norm_fwd(const NormArgs &a, cudaStream_t stream)
{
    const int grid = a.rows < 148 * 16 ? a.rows : 148 * 16;
    if (a.bf16) norm_fwd_kernel<__nv_bfloat16><<<grid, NT, 0, stream>>>(a);
    else norm_fwd_kernel<float><<<grid, NT, 0, stream>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_norm_bwd(const NormArgs &a, cudaStream_t stream)
{
    const int blocks = blocks_for(a.rows);
    if (a.bf16) norm_bwd_kernel<__nv_bfloat16><<<blocks, NT, 0, stream>>>(a);
    else norm_bwd_kernel<float><<<blocks, NT, 0, stream>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const dim3 grid((a.dim + NT - 1) / NT, 3);
    if (a.bf16) norm_reduce_kernel<__nv_bfloat16><<<grid, NT, 0, stream>>>(a, blocks);
    else norm_reduce_kernel<float><<<grid, NT, 0, stream>>>(a, blocks);
    return cudaGetLastError();
}

}  // namespace mms
