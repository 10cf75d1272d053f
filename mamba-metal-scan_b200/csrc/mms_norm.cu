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
//
// Bound by HBM: forward 4 arrays (5 with a gate), backward 5 to 8. So a row
// passes through registers once: a CTA takes a row at a time, each thread E
// elements of it in 16-byte pieces (single elements where rows are not
// 16-byte aligned), and the one or two sums a row needs are block reductions.
// A thread owns the same columns in every row, so the backward's sums over
// rows stay in its registers; the CTAs' partial sums meet in the workspace in
// a fixed order. Rows too long for that (above 512 x 16 elements) are read
// again for each sum.
#include <algorithm>

#include "mms_common.cuh"
#include "mms_head.h"
#include "mms_kernels.h"

namespace mms {

namespace {

constexpr int MAX_ROW_BLOCKS = 148 * 8;         // backward CTAs, at most
constexpr int ROW_THREADS = 512;                // threads of a row held in registers, at most

// Sum over the CTA; `sh` has two sets of 32 used in turn, so that one barrier a sum is enough.
struct BlockSum {
    float (*sh)[32];
    int turn;
    __device__ __forceinline__ float operator()(float v) {
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
        const int warps = blockDim.x / 32;
        if (warps == 1) return v;
        float *s = sh[turn ^= 1];
        if (threadIdx.x % 32 == 0) s[threadIdx.x / 32] = v;
        __syncthreads();
        v = threadIdx.x % 32 < warps ? s[threadIdx.x % 32] : 0.f;
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
        return v;
    }
};

// E elements of a row per thread: 16-byte pieces at (i * blockDim + thread) if
// VEC, else single elements there. Elements past the row read as 0.
template <typename T, int E, bool VEC>
struct Cols {
    static constexpr int VW = VEC ? 16 / (int)sizeof(T) : 1, NV = E / VW;
    __device__ static __forceinline__ int at(int v) { return (v * blockDim.x + threadIdx.x) * VW; }
    __device__ static __forceinline__ void load(const T *__restrict__ p, int dim, float (&o)[E]) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = at(v);
            if (VEC) {
                uint4 q = make_uint4(0, 0, 0, 0);
                if (c < dim) q = __ldg(reinterpret_cast<const uint4 *>(p + c));
                const T *e = reinterpret_cast<const T *>(&q);
#pragma unroll
                for (int j = 0; j < VW; ++j) o[v * VW + j] = to_f(e[j]);
            } else {
                o[v] = c < dim ? to_f(p[c]) : 0.f;
            }
        }
    }
    __device__ static __forceinline__ void store(T *__restrict__ p, int dim, const float (&o)[E]) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = at(v);
            if (c >= dim) continue;
            if (VEC) {
                uint4 q;
                T *e = reinterpret_cast<T *>(&q);
#pragma unroll
                for (int j = 0; j < VW; ++j) e[j] = from_f<T>(o[v * VW + j]);
                *reinterpret_cast<uint4 *>(p + c) = q;
            } else {
                p[c] = from_f<T>(o[v]);
            }
        }
    }
};

// POST, GATE, SCALE: bits of F.
enum { POST = 1, GATE = 2, SCALE = 4 };

template <typename T, int E, bool VEC, int F>
__global__ void __launch_bounds__(ROW_THREADS) norm_fwd_kernel(const NormArgs a)
{
    using C = Cols<T, E, VEC>;
    __shared__ float sh[2][32];
    BlockSum sum{sh, 0};
    const float inv = 1.f / a.dim;
    float w[E];
    for (size_t r = blockIdx.x; r < (size_t)a.rows; r += gridDim.x) {
        const size_t o = r * a.dim;
        float h[E], b[E];
        C::load(static_cast<const T *>(a.y) + o, a.dim, b);
        C::load(static_cast<const T *>(a.x) + o, a.dim, h);
        if (F & GATE) {
            float z[E];
            C::load(static_cast<const T *>(a.gate) + r * a.ldg, a.dim, z);
#pragma unroll
            for (int i = 0; i < E; ++i) b[i] *= z[i] * sigmoid_fast(z[i]);
        }
        float r1 = 0.f;
        if (F & POST) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) s = fmaf(b[i], b[i], s);
            C::load(static_cast<const T *>(a.post), a.dim, w);
            r1 = rsqrtf(sum(s) * inv + a.eps);
#pragma unroll
            for (int i = 0; i < E; ++i) b[i] *= r1 * w[i];
        }
        if (F & SCALE) {
            C::load(static_cast<const T *>(a.scale), a.dim, w);
#pragma unroll
            for (int i = 0; i < E; ++i) b[i] *= w[i];
        }
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            h[i] += b[i];
            s = fmaf(h[i], h[i], s);
        }
        C::store(static_cast<T *>(a.h) + o, a.dim, h);
        C::load(static_cast<const T *>(a.weight), a.dim, w);
        const float r2 = rsqrtf(sum(s) * inv + a.eps);
#pragma unroll
        for (int i = 0; i < E; ++i) h[i] *= r2 * w[i];
        C::store(static_cast<T *>(a.u) + o, a.dim, h);
        if (threadIdx.x == 0) {
            a.stat[2 * r] = r1;
            a.stat[2 * r + 1] = r2;
        }
    }
}

// Sums over this CTA's rows go to part[(which * gridDim + block) * dim + column],
// which = 0 dweight, 1 dscale, 2 dpost.
template <typename T, int E, bool VEC, int F>
__global__ void __launch_bounds__(ROW_THREADS) norm_bwd_kernel(const NormArgs a)
{
    using C = Cols<T, E, VEC>;
    __shared__ float sh[2][32];
    BlockSum sum{sh, 0};
    const float inv = 1.f / a.dim;
    float sw[E], ss[E], sp[E];
#pragma unroll
    for (int i = 0; i < E; ++i) sw[i] = ss[i] = sp[i] = 0.f;
    for (size_t r = blockIdx.x; r < (size_t)a.rows; r += gridDim.x) {
        const size_t o = r * a.dim;
        float h[E], t[E], y[E], z[E], v[E], w[E], d[E];
        C::load(static_cast<const T *>(a.du) + o, a.dim, t);
        C::load(static_cast<const T *>(a.x) + o, a.dim, h);
        C::load(static_cast<const T *>(a.y) + o, a.dim, y);
        if (F & GATE) C::load(static_cast<const T *>(a.gate) + r * a.ldg, a.dim, z);
        C::load(static_cast<const T *>(a.dh) + o, a.dim, d);
        const float r1 = F & POST ? a.c_stat[2 * r] : 1.f, r2 = a.c_stat[2 * r + 1];
        // v = a r1 (the normed a, or a itself), h
        if (F & POST) C::load(static_cast<const T *>(a.post), a.dim, w);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            v[i] = y[i];
            if (F & GATE) v[i] *= z[i] * sigmoid_fast(z[i]);
            if (F & POST) v[i] *= r1;
        }
        float sc[E];
        if (F & SCALE) C::load(static_cast<const T *>(a.scale), a.dim, sc);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            float b = v[i];
            if (F & POST) b *= w[i];
            if (F & SCALE) b *= sc[i];
            h[i] = (h[i] + b) * r2;                          // n
        }
        float s = 0.f;
        float ww[E];
        C::load(static_cast<const T *>(a.weight), a.dim, ww);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            sw[i] = fmaf(t[i], h[i], sw[i]);
            t[i] *= ww[i];
            s = fmaf(t[i], h[i], s);
        }
        const float mean = sum(s) * inv;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            d[i] = fmaf(r2, t[i] - h[i] * mean, d[i]);       // dh'
            t[i] = d[i];
            if (F & SCALE) {
                ss[i] = fmaf(d[i], F & POST ? v[i] * w[i] : v[i], ss[i]);
                t[i] *= sc[i];                               // db
            }
            if (F & POST) {
                sp[i] = fmaf(t[i], v[i], sp[i]);
                t[i] *= w[i];
                s = fmaf(t[i], v[i], s);
            }
        }
        C::store(static_cast<T *>(a.dx) + o, a.dim, d);
        if (F == 0) continue;                                // dy has dx's values
        if (F & POST) {
            const float mean1 = sum(s) * inv;
#pragma unroll
            for (int i = 0; i < E; ++i) t[i] = r1 * (t[i] - v[i] * mean1);
        }
        if (F & GATE) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float sig = sigmoid_fast(z[i]);
                d[i] = t[i] * y[i] * (sig * (1.f + z[i] * (1.f - sig)));
                t[i] *= z[i] * sig;
            }
            C::store(static_cast<T *>(a.dgate) + o, a.dim, d);
        }
        C::store(static_cast<T *>(a.dy) + o, a.dim, t);
    }
    const size_t plane = (size_t)gridDim.x * a.dim;
    float *part = static_cast<float *>(a.workspace) + (size_t)blockIdx.x * a.dim;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int c = C::at(i / C::VW) + i % C::VW;
        if (c >= a.dim) continue;
        part[c] = sw[i];
        if (F & SCALE) part[plane + c] = ss[i];
        if (F & POST) part[2 * plane + c] = sp[i];
    }
}

// ------------------------------------------------------------- rows of any length

template <typename T>
struct Row {
    const T *x, *y, *gate, *w, *post, *scale;
    __device__ __forceinline__ float a_at(int i) const {
        if (!gate) return to_f(y[i]);
        const float z = to_f(gate[i]);
        return to_f(y[i]) * (z * sigmoid_fast(z));
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
__global__ void __launch_bounds__(1024) norm_fwd_long_kernel(const NormArgs a)
{
    __shared__ float sh[2][32];
    BlockSum sum{sh, 0};
    const float inv = 1.f / a.dim;
    for (size_t r = blockIdx.x; r < (size_t)a.rows; r += gridDim.x) {
        const Row<T> row = row_of<T>(a, r);
        float r1 = 0.f, s = 0.f;
        if (a.post) {
            for (int i = threadIdx.x; i < a.dim; i += blockDim.x) {
                const float v = row.a_at(i);
                s += v * v;
            }
            r1 = rsqrtf(sum(s) * inv + a.eps);
            s = 0.f;
        }
        for (int i = threadIdx.x; i < a.dim; i += blockDim.x) {
            const float v = row.h_at(i, r1);
            s += v * v;
        }
        const float r2 = rsqrtf(sum(s) * inv + a.eps);
        for (int i = threadIdx.x; i < a.dim; i += blockDim.x) {
            const float v = row.h_at(i, r1);
            static_cast<T *>(a.h)[r * a.dim + i] = from_f<T>(v);
            static_cast<T *>(a.u)[r * a.dim + i] = from_f<T>(v * r2 * to_f(row.w[i]));
        }
        if (threadIdx.x == 0) {
            a.stat[2 * r] = r1;
            a.stat[2 * r + 1] = r2;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(1024) norm_bwd_long_kernel(const NormArgs a)
{
    __shared__ float sh[2][32];
    BlockSum sum{sh, 0};
    const float inv = 1.f / a.dim;
    const size_t plane = (size_t)gridDim.x * a.dim;
    float *pw = static_cast<float *>(a.workspace) + (size_t)blockIdx.x * a.dim;
    float *ps = pw + plane, *pp = ps + plane;
    for (int i = threadIdx.x; i < a.dim; i += blockDim.x) {
        pw[i] = 0.f;
        if (a.scale) ps[i] = 0.f;
        if (a.post) pp[i] = 0.f;
    }
    for (size_t r = blockIdx.x; r < (size_t)a.rows; r += gridDim.x) {
        const Row<T> row = row_of<T>(a, r);
        const T *dh = static_cast<const T *>(a.dh) + r * a.dim, *du = static_cast<const T *>(a.du) + r * a.dim;
        const float r1 = a.c_stat[2 * r], r2 = a.c_stat[2 * r + 1];
        float s = 0.f;
        for (int i = threadIdx.x; i < a.dim; i += blockDim.x) s += to_f(du[i]) * to_f(row.w[i]) * row.h_at(i, r1);
        const float mean = sum(s) * inv * r2;
        const auto dh_at = [&](int i, float h) {
            return to_f(dh[i]) + r2 * (to_f(du[i]) * to_f(row.w[i]) - h * r2 * mean);
        };
        float mean1 = 0.f;
        if (a.post) {
            s = 0.f;
            for (int i = threadIdx.x; i < a.dim; i += blockDim.x) {
                const float d = dh_at(i, row.h_at(i, r1)) * (a.scale ? to_f(row.scale[i]) : 1.f);
                s += d * to_f(row.post[i]) * row.a_at(i);
            }
            mean1 = sum(s) * inv * r1;
        }
        for (int i = threadIdx.x; i < a.dim; i += blockDim.x) {
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
                const float z = to_f(row.gate[i]), sig = sigmoid_fast(z);
                static_cast<T *>(a.dgate)[o] = from_f<T>(v * to_f(row.y[i]) * (sig * (1.f + z * (1.f - sig))));
                v *= z * sig;
            }
            static_cast<T *>(a.dx)[o] = from_f<T>(d);
            if (a.dy != a.dx) static_cast<T *>(a.dy)[o] = from_f<T>(v);
        }
    }
}

// 32 columns a CTA, 32 threads a column over the partial sums.
template <typename T>
__global__ void __launch_bounds__(1024) norm_reduce_kernel(const NormArgs a, int blocks)
{
    __shared__ float sh[32][33];
    const int which = blockIdx.y, col = blockIdx.x * 32 + threadIdx.x;
    T *out = static_cast<T *>(which == 0 ? a.dweight : which == 1 ? a.dscale : a.dpost);
    if (!out) return;
    const float *p = static_cast<const float *>(a.workspace) + (size_t)which * blocks * a.dim;
    float s = 0.f;
    if (col < a.dim)
#pragma unroll 4
        for (int b = threadIdx.y; b < blocks; b += 32) s += p[(size_t)b * a.dim + col];
    sh[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    s = sh[threadIdx.x][threadIdx.y];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    const int c = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && c < a.dim) out[c] = from_f<T>(s);
}

bool rows_aligned(const NormArgs &a)
{
    const int e = a.bf16 ? 2 : 4;
    const void *p[] = {a.x, a.y, a.gate, a.weight, a.post, a.scale, a.h, a.u, a.dh, a.du, a.dx, a.dy, a.dgate};
    for (const void *q : p)
        if (reinterpret_cast<uintptr_t>(q) % 16) return false;
    return (long long)a.dim * e % 16 == 0 && (!a.gate || a.ldg * e % 16 == 0);
}

// E and threads of a CTA for a row of `dim` elements in pieces of `vw`: the
// fewest elements a thread that ROW_THREADS threads can do; 0 if 16 are too few.
struct Shape {
    int e, threads;
};
Shape shape_for(int dim, int vw)
{
    for (int e = std::max(vw, 4); e <= 16; e *= 2) {
        const int threads = ((dim + e - 1) / e + 31) / 32 * 32;
        if (threads <= ROW_THREADS) return Shape{e, threads};
    }
    return Shape{0, 1024};
}

// CTAs of a kernel that fit the GPU at once (asked once per kernel and size).
template <auto KERNEL>
int resident(int threads)
{
    static std::atomic<int> known[ROW_THREADS / 32 + 1];
    int n = known[threads / 32].load(std::memory_order_relaxed);
    if (!n) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, threads, 0) != cudaSuccess || n < 1) n = 1;
        known[threads / 32].store(n, std::memory_order_relaxed);
    }
    return n * N_SM;
}

template <typename T, int E, bool VEC, int F>
cudaError_t run(const NormArgs &a, int threads, bool backward, int *blocks, cudaStream_t stream)
{
    if (backward) {
        *blocks = std::min({a.rows, resident<norm_bwd_kernel<T, E, VEC, F>>(threads), MAX_ROW_BLOCKS});
        norm_bwd_kernel<T, E, VEC, F><<<*blocks, threads, 0, stream>>>(a);
    } else {
        const int grid = std::min(a.rows, resident<norm_fwd_kernel<T, E, VEC, F>>(threads));
        norm_fwd_kernel<T, E, VEC, F><<<grid, threads, 0, stream>>>(a);
    }
    return cudaGetLastError();
}

template <typename T, int E, bool VEC>
cudaError_t run_flags(const NormArgs &a, int threads, bool backward, int *blocks, cudaStream_t s)
{
    switch ((a.post ? POST : 0) | (a.gate ? GATE : 0) | (a.scale ? SCALE : 0)) {
    case 0: return run<T, E, VEC, 0>(a, threads, backward, blocks, s);
    case 1: return run<T, E, VEC, 1>(a, threads, backward, blocks, s);
    case 2: return run<T, E, VEC, 2>(a, threads, backward, blocks, s);
    case 3: return run<T, E, VEC, 3>(a, threads, backward, blocks, s);
    case 4: return run<T, E, VEC, 4>(a, threads, backward, blocks, s);
    case 5: return run<T, E, VEC, 5>(a, threads, backward, blocks, s);
    case 6: return run<T, E, VEC, 6>(a, threads, backward, blocks, s);
    default: return run<T, E, VEC, 7>(a, threads, backward, blocks, s);
    }
}

template <typename T>
cudaError_t run_type(const NormArgs &a, bool backward, int *blocks, cudaStream_t s)
{
    const bool vec = rows_aligned(a);
    constexpr int VW = 16 / (int)sizeof(T);
    const Shape q = shape_for(a.dim, vec ? VW : 1);
    if (vec) {
        if constexpr (VW == 4)
            if (q.e == 4) return run_flags<T, 4, true>(a, q.threads, backward, blocks, s);
        if (q.e == 8) return run_flags<T, 8, true>(a, q.threads, backward, blocks, s);
        if (q.e == 16) return run_flags<T, 16, true>(a, q.threads, backward, blocks, s);
    } else {
        if (q.e == 4) return run_flags<T, 4, false>(a, q.threads, backward, blocks, s);
        if (q.e == 8) return run_flags<T, 8, false>(a, q.threads, backward, blocks, s);
        if (q.e == 16) return run_flags<T, 16, false>(a, q.threads, backward, blocks, s);
    }
    *blocks = std::min(a.rows, N_SM * 2);
    if (backward) norm_bwd_long_kernel<T><<<*blocks, 1024, 0, s>>>(a);
    else norm_fwd_long_kernel<T><<<*blocks, 1024, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

size_t norm_workspace_bytes(int rows, int dim)
{
    return (size_t)3 * std::min(rows, MAX_ROW_BLOCKS) * dim * sizeof(float);
}

cudaError_t launch_norm_fwd(const NormArgs &a, cudaStream_t stream)
{
    int blocks;
    return a.bf16 ? run_type<__nv_bfloat16>(a, false, &blocks, stream) : run_type<float>(a, false, &blocks, stream);
}

cudaError_t launch_norm_bwd(const NormArgs &a, cudaStream_t stream)
{
    int blocks = 0;
    const cudaError_t e = a.bf16 ? run_type<__nv_bfloat16>(a, true, &blocks, stream)
                                 : run_type<float>(a, true, &blocks, stream);
    if (e != cudaSuccess) return e;
    const dim3 grid((a.dim + 31) / 32, a.post || a.scale ? 3 : 1);
    if (a.bf16) norm_reduce_kernel<__nv_bfloat16><<<grid, dim3(32, 32), 0, stream>>>(a, blocks);
    else norm_reduce_kernel<float><<<grid, dim3(32, 32), 0, stream>>>(a, blocks);
    return cudaGetLastError();
}

}  // namespace mms
