// The matrix products of the head's losses, with what follows them on a tile.
#include "mms_common.cuh"
#include "mms_head.h"

namespace mms {

namespace {

constexpr int BM = 64, BK = 16;

__device__ __forceinline__ float factor_at(const Factor &f, int planes, int r, int k) {
    const __nv_bfloat16 *p = f.p + (f.t ? (size_t)k * f.ld + r : (size_t)r * f.ld + k);
    float v = to_f(p[0]);
    if (planes == 3) v += to_f(p[f.plane]) + to_f(p[2 * f.plane]);
    return v;
}

// One CTA: 64 rows, 64 columns (MM_LSE: MM_LSE_TILE columns, 64 at a time).
template <int KIND>
__global__ void __launch_bounds__(256) mm_kernel(const MmArgs a)
{
    __shared__ float sa[BK][BM + 4], sb[BK][BM + 4];
    __shared__ float2 red[BM][16];
    constexpr int SUB = KIND == MM_LSE ? MM_LSE_TILE / BM : 1;
    const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
    const int m0 = blockIdx.x * BM;
    float2 run = make_float2(-INFINITY, 0.f);
    for (int sub = 0; sub < SUB; ++sub) {
        const int n0 = (blockIdx.y * SUB + sub) * BM;
        if (n0 >= a.n) break;
        float acc[4][4] = {};
        for (int k0 = 0; k0 < a.k; k0 += BK) {
            for (int i = tid; i < BK * BM; i += 256) {
                const int ra = a.a.t ? i % BM : i / BK, ka = a.a.t ? i / BM : i % BK;
                sa[ka][ra] = m0 + ra < a.m && k0 + ka < a.k ? factor_at(a.a, a.planes, m0 + ra, k0 + ka) : 0.f;
                const int rb = a.b.t ? i % BM : i / BK, kb = a.b.t ? i / BM : i % BK;
                sb[kb][rb] = n0 + rb < a.n && k0 + kb < a.k ? factor_at(a.b, a.planes, n0 + rb, k0 + kb) : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < BK; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], acc[i][j]);
            __syncthreads();
        }
        if (KIND == MM_LSE) {
            for (int i = 0; i < 4; ++i) {
                float mx = -INFINITY, s = 0.f;
                for (int j = 0; j < 4; ++j)
                    if (n0 + tx * 4 + j < a.n) mx = fmaxf(mx, a.c * acc[i][j]);
                for (int j = 0; j < 4; ++j)
                    if (n0 + tx * 4 + j < a.n && !(mx == -INFINITY && a.c * acc[i][j] == -INFINITY))
                        s += ex2(a.c * acc[i][j] - mx);
                red[ty * 4 + i][tx] = make_float2(mx, s);
            }
            __syncthreads();
            if (tid < BM)
                for (int j = 0; j < 16; ++j) {
                    const float2 v = red[tid][j];
                    const float mx = fmaxf(run.x, v.x);
                    if (mx != -INFINITY)
                        run = make_float2(mx, run.y * ex2(run.x - mx) + v.y * ex2(v.x - mx));
                    else
                        run.y += v.y;               // NaN, if any
                }
            __syncthreads();
        }
        for (int i = 0; i < 4 && KIND != MM_LSE; ++i) {
            const int m = m0 + ty * 4 + i;
            if (m >= a.m) break;
            for (int j = 0; j < 4; ++j) {
                const int n = n0 + tx * 4 + j;
                if (n >= a.n) break;
                if (KIND == MM_GRAD) {
                    const float rs = a.rs[m];
                    float v = rs == 0.f ? 0.f : rs * ex2(a.c * acc[i][j] - a.lse2[m]);
                    for (int p = 0; p < a.planes; ++p) {
                        const __nv_bfloat16 q = __float2bfloat16_rn(v);
                        a.g[p * a.gplane + (size_t)m * a.ldg + n] = q;
                        v -= to_f(q);
                    }
                } else {
                    const size_t o = (size_t)m * a.ldo + n;
                    const float v = acc[i][j] + (a.acc ? a.acc[o] : 0.f);
                    if (a.out_bf16) static_cast<__nv_bfloat16 *>(a.out)[o] = __float2bfloat16_rn(v);
                    else static_cast<float *>(a.out)[o] = v;
                }
            }
        }
    }
    if (KIND == MM_LSE && tid < BM && m0 + tid < a.m)
        a.part[(size_t)blockIdx.y * a.m + m0 + tid] = run;
}

}  // namespace

cudaError_t launch_mm(MmKind kind, const MmArgs &a, cudaStream_t stream)
{
    const int bn = kind == MM_LSE ? MM_LSE_TILE : BM;
    const dim3 grid((a.m + BM - 1) / BM, (a.n + bn - 1) / bn);
    if (kind == MM_LSE) mm_kernel<MM_LSE><<<grid, 256, 0, stream>>>(a);
    else if (kind == MM_GRAD) mm_kernel<MM_GRAD><<<grid, 256, 0, stream>>>(a);
    else mm_kernel<MM_OUT><<<grid, 256, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace mms
