// Residual sum after a block fused with the norms around it (sm_100a):
//     a = y silu(gate);  b = post a r1;  h = x + scale b;  u = weight h r2
//     r1 = 1 / sqrt(mean(a^2) + eps),    r2 = 1 / sqrt(mean(h^2) + eps)
// and with n = h r2, t = weight du, the gradients
//     dh' = dh + r2 (t - n mean(t n))            dx = dh'
//     dscale = post sum over rows of dh' a r1,   db = scale dh'
//     dpost = scale sum over rows of dh' a r1,   s = post db
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
// a fixed order. The backward's five reads a row come a row ahead, by
// cp.async into shared memory where each thread finds its own pieces again (no
// barrier), and its arithmetic is on packed pairs. It is close to issue bound,
// so nothing is computed twice: post and scale act as one product (in registers
// for all rows), their gradients come from one sum over the rows, sum of dh' a r1,
// and silu(gate) and its slope wait in shared memory for da. Measured:
// 16384 x 4096 bf16 with all options forward 118 us (5.7 TB/s), backward 194 us
// (5.5 TB/s; 233 us with both sums and the sigmoids twice, 307 us with loads at
// the top of the row and scalar arithmetic too); 8192 x 640 float32 sum and norm
// 12 and 18 us, partly from L2. Rows too long for that (above 512 x 16 elements)
// are read again for each sum.
#include <algorithm>

#include "mms_common.cuh"
#include "mms_head.h"
#include "mms_kernels.h"
#include "mms_stage.cuh"

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
    // the same pieces by cp.async to `dst` (one piece of 16 bytes a thread and v), and from there
    __device__ static __forceinline__ void fetch(uint4 *dst, const T *__restrict__ p, int dim) {
#pragma unroll
        for (int v = 0; v < NV; ++v) cp16(dst + v * blockDim.x + threadIdx.x, p + (at(v) < dim ? at(v) : 0), at(v) < dim);
    }
    __device__ static __forceinline__ void take(const uint4 *src, float (&o)[E]) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const uint4 q = src[v * blockDim.x + threadIdx.x];
            const T *e = reinterpret_cast<const T *>(&q);
#pragma unroll
            for (int j = 0; j < VW; ++j) o[v * VW + j] = to_f(e[j]);
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
    chained();
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
        if (threadIdx.x == 0 && a.stat) {
            a.stat[2 * r] = r1;
            a.stat[2 * r + 1] = r2;
        }
    }
}

// silu'(z) = sig (1 + z (1 - sig)) = sig + z sig - (z sig) sig
__device__ __forceinline__ float2 silu_slope(float2 zs, float2 sig) {
    return fma2(zs, fma2(sig, f2(-1.f, -1.f), f2(1.f, 1.f)), sig);
}

template <int P>
__device__ __forceinline__ float (&flat(float2 (&v)[P]))[2 * P] {
    return reinterpret_cast<float (&)[2 * P]>(v);
}

// The backward's reads of a row, in the order of their places in shared memory.
enum { IN_DU, IN_X, IN_Y, IN_DH, IN_GATE };
// Rows in shared memory, this one and the next, where ROW_THREADS leave room for
// them (5 x 512 x 16 bytes a row and piece); 0: loads at the top of the row.
template <typename T, int E, bool VEC>
__host__ __device__ constexpr int fetch_rows() {
    return !VEC || E * sizeof(T) > 32 ? 0 : 2;
}

template <typename T, int E, bool VEC, int F>
__host__ __device__ constexpr int fetch_bytes(int threads) {
    return fetch_rows<T, E, VEC>() * (F & GATE ? 5 : 4) * threads * E * (int)sizeof(T);
}

template <typename T, int E, bool VEC, int F>
struct RowReader {
    using C = Cols<T, E, VEC>;
    static constexpr int N = F & GATE ? 5 : 4, R = fetch_rows<T, E, VEC>();
    const NormArgs &a;
    uint4 *smem;                                // [R][N][NV * threads]
    size_t r;
    int slot;
    __device__ __forceinline__ const T *src(int which, size_t row) const {
        const size_t o = row * a.dim;
        switch (which) {
        case IN_DU: return static_cast<const T *>(a.du) + o;
        case IN_X: return static_cast<const T *>(a.x) + o;
        case IN_Y: return static_cast<const T *>(a.y) + o;
        case IN_DH: return static_cast<const T *>(a.dh) + o;
        default: return static_cast<const T *>(a.gate) + row * a.ldg;
        }
    }
    __device__ __forceinline__ uint4 *place(int which, int s) const {
        return smem + (size_t)(s * N + which) * C::NV * blockDim.x;
    }
    __device__ __forceinline__ void fetch(size_t row, int s) {
        if constexpr (R > 0) {
            if (row < (size_t)a.rows)
#pragma unroll
                for (int w = 0; w < N; ++w) C::fetch(place(w, s), src(w, row), a.dim);
            cp_commit();                        // also without a row: the waits count groups
        }
    }
    __device__ __forceinline__ void begin(size_t row) {
        r = row;
        slot = 0;
        for (int i = 0; i < R - 1; ++i) fetch(r + (size_t)i * gridDim.x, i);
    }
    // This row is there; one more is on its way, into the place that the row before left.
    __device__ __forceinline__ void ready() {
        fetch(r + (size_t)(R - 1) * gridDim.x, slot == 0 ? R - 1 : slot - 1);
        if constexpr (R > 0) cp_wait<R - 1>();
    }
    __device__ __forceinline__ void get(int which, float (&o)[E]) const {
        if constexpr (R > 0) C::take(place(which, slot), o);
        else C::load(src(which, r), a.dim, o);
    }
    __device__ __forceinline__ void next() {
        r += gridDim.x;
        slot = slot == R - 1 ? 0 : slot + 1;
    }
};

// With a gate and rows in shared memory: silu(gate) and y silu'(gate) of a row stay there from the
// pass that computes a to the one that uses them (each thread its own).
template <typename T, int E, bool VEC, int F>
__host__ __device__ constexpr bool keeps_gate() {
    return F & GATE && fetch_rows<T, E, VEC>() > 0;
}

template <typename T, int E, bool VEC, int F>
constexpr int bwd_smem(int threads) {
    return fetch_bytes<T, E, VEC, F>(threads) + (keeps_gate<T, E, VEC, F>() ? threads * E * 8 : 0);
}

// Sums over this CTA's rows go to part[(which * gridDim + block) * dim + column]: which = 0 those of
// du n; 1 those of dh' v (v = a r1, or a without post), whose products with post and scale are dscale
// and dpost.
template <typename T, int E, bool VEC, int F>
__global__ void __launch_bounds__(ROW_THREADS) norm_bwd_kernel(const NormArgs a)
{
    chained();
    using C = Cols<T, E, VEC>;
    extern __shared__ uint4 rows_smem[];
    __shared__ float sh[2][32];
    BlockSum sum{sh, 0};
    const float inv = 1.f / a.dim;
    constexpr int P = E / 2;                                 // packed pairs: half the instructions
    constexpr bool KEEP = keeps_gate<T, E, VEC, F>();
    float2 sw[P], sv[P], ps[P];                              // ps = post scale
#pragma unroll
    for (int i = 0; i < P; ++i) {
        sw[i] = sv[i] = f2(0.f, 0.f);
        ps[i] = f2(1.f, 1.f);
    }
    if (F & POST) C::load(static_cast<const T *>(a.post), a.dim, flat(ps));
    if (F & SCALE) {
        float2 w[P];
        C::load(static_cast<const T *>(a.scale), a.dim, flat(w));
#pragma unroll
        for (int i = 0; i < P; ++i) ps[i] = F & POST ? mul2(ps[i], w[i]) : w[i];
    }
    RowReader<T, E, VEC, F> in{a, rows_smem, 0, 0};
    float4 *kept = KEEP ? reinterpret_cast<float4 *>(rows_smem) +
                              (size_t)fetch_bytes<T, E, VEC, F>(blockDim.x) / 16 + threadIdx.x : nullptr;
    for (in.begin(blockIdx.x); in.r < (size_t)a.rows; in.next()) {
        in.ready();
        const size_t o = in.r * a.dim;
        float2 h[P], t[P], v[P], d[P];
        const float r1 = F & POST ? a.c_stat[2 * in.r] : 1.f, r2 = a.c_stat[2 * in.r + 1];
        const float2 r1p = f2(r1, r1), r2p = f2(r2, r2);
        // v = a r1 (the normed a, or a itself), h = n
        in.get(IN_Y, flat(v));
        if (F & GATE) {
            in.get(IN_GATE, flat(d));
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const float2 sig = f2(sigmoid_fast(d[i].x), sigmoid_fast(d[i].y)), zs = mul2(d[i], sig);
                if (KEEP) {
                    const float2 g = mul2(v[i], silu_slope(zs, sig));
                    kept[i * blockDim.x] = make_float4(zs.x, zs.y, g.x, g.y);
                }
                v[i] = mul2(v[i], zs);
            }
        }
        in.get(IN_X, flat(h));
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if (F & POST) v[i] = mul2(v[i], r1p);
            h[i] = mul2(F & (POST | SCALE) ? fma2(v[i], ps[i], h[i]) : add2(h[i], v[i]), r2p);
        }
        in.get(IN_DU, flat(t));
        float2 s = f2(0.f, 0.f);
        C::load(static_cast<const T *>(a.weight), a.dim, flat(d));
#pragma unroll
        for (int i = 0; i < P; ++i) {
            sw[i] = fma2(t[i], h[i], sw[i]);
            t[i] = mul2(t[i], d[i]);
            s = fma2(t[i], h[i], s);
        }
        const float mean = sum(s.x + s.y) * inv;
        const float2 meanp = f2(-mean, -mean);
        in.get(IN_DH, flat(d));
#pragma unroll
        for (int i = 0; i < P; ++i) d[i] = fma2(r2p, fma2(h[i], meanp, t[i]), d[i]);        // dh'
        C::store(static_cast<T *>(a.dx) + o, a.dim, flat(d));
        if (F == 0) continue;                                // dy has dx's values
        s = f2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if (F & (POST | SCALE)) {
                sv[i] = fma2(d[i], v[i], sv[i]);
                d[i] = mul2(d[i], ps[i]);
            }
            if (F & POST) s = fma2(d[i], v[i], s);
        }
        if (F & POST) {
            const float mean1 = sum(s.x + s.y) * inv;
            const float2 mean1p = f2(-mean1, -mean1);
#pragma unroll
            for (int i = 0; i < P; ++i) d[i] = mul2(r1p, fma2(v[i], mean1p, d[i]));
        }
        if (F & GATE) {
            if (KEEP) {
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const float4 k = kept[i * blockDim.x];
                    t[i] = mul2(d[i], f2(k.z, k.w));
                    d[i] = mul2(d[i], f2(k.x, k.y));
                }
            } else {
                in.get(IN_GATE, flat(h));
                in.get(IN_Y, flat(v));
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const float2 sig = f2(sigmoid_fast(h[i].x), sigmoid_fast(h[i].y)), zs = mul2(h[i], sig);
                    t[i] = mul2(d[i], mul2(v[i], silu_slope(zs, sig)));
                    d[i] = mul2(d[i], zs);
                }
            }
            C::store(static_cast<T *>(a.dgate) + o, a.dim, flat(t));
        }
        C::store(static_cast<T *>(a.dy) + o, a.dim, flat(d));
    }
    const size_t plane = (size_t)gridDim.x * a.dim;
    float *part = static_cast<float *>(a.workspace) + (size_t)blockIdx.x * a.dim;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int c = C::at(i / C::VW) + i % C::VW;
        if (c >= a.dim) continue;
        part[c] = flat(sw)[i];
        if (F & (POST | SCALE)) part[plane + c] = flat(sv)[i];
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
    chained();
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
        if (threadIdx.x == 0 && a.stat) {
            a.stat[2 * r] = r1;
            a.stat[2 * r + 1] = r2;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(1024) norm_bwd_long_kernel(const NormArgs a)
{
    chained();
    __shared__ float sh[2][32];
    BlockSum sum{sh, 0};
    const float inv = 1.f / a.dim;
    const size_t plane = (size_t)gridDim.x * a.dim;
    float *pw = static_cast<float *>(a.workspace) + (size_t)blockIdx.x * a.dim;
    float *pv = pw + plane;
    const bool any = a.post || a.scale;
    for (int i = threadIdx.x; i < a.dim; i += blockDim.x) {
        pw[i] = 0.f;
        if (any) pv[i] = 0.f;
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
            const float av = row.a_at(i), h = row.h_at(i, r1);
            const float d = dh_at(i, h);
            pw[i] += to_f(du[i]) * h * r2;
            float v = d;
            if (any) pv[i] += d * (a.post ? av * r1 : av);
            if (a.scale) v *= to_f(row.scale[i]);
            if (a.post) {
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
    chained();
    __shared__ float sh[32][33];
    const int which = blockIdx.y, col = blockIdx.x * 32 + threadIdx.x;
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
    if (threadIdx.x || c >= a.dim) return;
    const T *post = static_cast<const T *>(a.post), *scale = static_cast<const T *>(a.scale);
    if (which == 0) static_cast<T *>(a.dweight)[c] = from_f<T>(s);
    if (which == 1 && scale) static_cast<T *>(a.dscale)[c] = from_f<T>(post ? s * to_f(post[c]) : s);
    if (which == 1 && post) static_cast<T *>(a.dpost)[c] = from_f<T>(scale ? s * to_f(scale[c]) : s);
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
int resident(int threads, int smem)
{
    static std::atomic<int> known[ROW_THREADS / 32 + 1];
    int n = known[threads / 32].load(std::memory_order_relaxed);
    if (!n) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, threads, smem) != cudaSuccess || n < 1) n = 1;
        known[threads / 32].store(n, std::memory_order_relaxed);
    }
    return n * N_SM;
}

template <typename T, int E, bool VEC, int F>
cudaError_t run(const NormArgs &a, int threads, bool backward, int *blocks, cudaStream_t stream)
{
    if (backward) {
        const int smem = bwd_smem<T, E, VEC, F>(threads);
        const cudaError_t e = smem_opt_in<norm_bwd_kernel<T, E, VEC, F>>(bwd_smem<T, E, VEC, F>(ROW_THREADS));
        if (e != cudaSuccess) return e;
        *blocks = std::min({a.rows, resident<norm_bwd_kernel<T, E, VEC, F>>(threads, smem), MAX_ROW_BLOCKS});
        launch_chained(norm_bwd_kernel<T, E, VEC, F>, *blocks, threads, smem, stream, a);
    } else {
        const int grid = std::min(a.rows, resident<norm_fwd_kernel<T, E, VEC, F>>(threads, 0));
        launch_chained(norm_fwd_kernel<T, E, VEC, F>, grid, threads, 0, stream, a);
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
    if (backward) launch_chained(norm_bwd_long_kernel<T>, *blocks, 1024, 0, s, a);
    else launch_chained(norm_fwd_long_kernel<T>, *blocks, 1024, 0, s, a);
    return cudaGetLastError();
}

}  // namespace

size_t norm_workspace_bytes(int rows, int dim)
{
    return (size_t)2 * std::min(rows, MAX_ROW_BLOCKS) * dim * sizeof(float);
}

cudaError_t launch_norm_fwd(const NormArgs &a, cudaStream_t stream)
{
    chain_begin();
    int blocks;
    return a.bf16 ? run_type<__nv_bfloat16>(a, false, &blocks, stream) : run_type<float>(a, false, &blocks, stream);
}

cudaError_t launch_norm_bwd(const NormArgs &a, cudaStream_t stream)
{
    chain_begin();
    int blocks = 0;
    const cudaError_t e = a.bf16 ? run_type<__nv_bfloat16>(a, true, &blocks, stream)
                                 : run_type<float>(a, true, &blocks, stream);
    if (e != cudaSuccess) return e;
    const dim3 grid((a.dim + 31) / 32, a.post || a.scale ? 2 : 1);
    if (a.bf16) launch_chained(norm_reduce_kernel<__nv_bfloat16>, grid, dim3(32, 32), 0, stream, a, blocks);
    else launch_chained(norm_reduce_kernel<float>, grid, dim3(32, 32), 0, stream, a, blocks);
    return cudaGetLastError();
}

}  // namespace mms
