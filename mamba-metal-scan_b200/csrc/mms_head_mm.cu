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
// Warps: 0 loads, 1 multiplies (leader), 2 owns the tensor memory, 4..11
// epilogue (a warp reads the 32 lanes of its number mod 4; the two halves of
// the columns go to two warps).
//
// Tile order: the dimension with fewer tiles runs fastest, in groups of 16,
// so the concurrent tiles share one side's panels in L2 and the long side is
// read from HBM once.
//
// float32 factors are three bf16 planes each; a product then runs over the
// six pairs of planes with i + j <= 2, smallest terms first.
//
// Every wait is bounded. A wait that runs out sets a flag for
// mms_device_status; all roles leave, the leader waits (bounded) for the
// copies in flight, and the pair leaves together.
#include <algorithm>

#include "mms_common.cuh"
#include "mms_head.h"
#include "mms_kernels.h"
#include "mms_stage.cuh"
#include "mms_tma.cuh"
#include "mms_umma.cuh"

namespace mms {

namespace {

constexpr int TM = 256, BK = 64, STAGES = 6, THREADS = 384;
constexpr int HALF = 16384;                                  // bytes of one CTA's a (or b) per stage
constexpr int GROUP = 16;
constexpr size_t SMEM = 1024 + (size_t)STAGES * 2 * HALF + 256;

__device__ unsigned int g_mm_timeout;

struct Tiles {
    int mt, nt, bn;         // tiles of rows and columns, columns per tile
    int kb;                 // steps of BK summed elements
};

__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, uint32_t limit) {
    for (uint32_t i = 0; i < limit; ++i)
        if (mbar_try(bar, parity)) return true;
    return false;
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

// The pair of planes of pass c (of 6): a's in the low half, smallest products first.
__device__ __forceinline__ void planes_of(int passes, int c, int &pa, int &pb) {
    if (passes == 1) {
        pa = pb = 0;
        return;
    }
    // (1,1) (0,2) (2,0) (0,1) (1,0) (0,0)
    const int ta = 0x010201, tb = 0x001021;      // digit c
    pa = ta >> (4 * c) & 15;
    pb = tb >> (4 * c) & 15;
}

__device__ __forceinline__ void store_planes(const MmArgs &a, int m, int n, const float (&v)[32]) {
    float t[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) t[i] = v[i];
    for (int p = 0; p < a.planes; ++p) {
        __nv_bfloat16 *g = a.g + p * a.gplane + (size_t)m * a.ldg + n;
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
            if (n + i >= a.n) break;             // ldg is a multiple of 8: whole pieces fit the row
            __nv_bfloat16 q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                q[j] = __float2bfloat16_rn(t[i + j]);
                t[i + j] -= to_f(q[j]);
            }
            *reinterpret_cast<uint4 *>(g + i) = *reinterpret_cast<const uint4 *>(q);
        }
    }
}

// What follows the product on 32 columns of one row.
template <int KIND>
struct Epilogue {
    float mx, s;                // MM_LSE: running maximum and sum
    float lse2, rs;             // MM_GRAD
    __device__ __forceinline__ void begin(const MmArgs &a, int m) {
        if (KIND == MM_LSE) {
            mx = -INFINITY;
            s = 0.f;
        }
        if (KIND == MM_GRAD) {
            lse2 = m < a.m ? a.lse2[m] : 0.f;
            rs = m < a.m ? a.rs[m] : 0.f;
        }
    }
    __device__ __forceinline__ void chunk(const MmArgs &a, int m, int n, float (&v)[32]) {
        if (n >= a.n) return;
        if (KIND == MM_LSE) {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                v[i] = n + i < a.n ? v[i] * a.c : -INFINITY;
                top = fmaxf(top, v[i]);
            }
            const float now = fmaxf(mx, top), ref = now == -INFINITY ? 0.f : now;
            float t = s * ex2(mx - ref);
#pragma unroll
            for (int i = 0; i < 32; ++i) t += ex2(v[i] - ref);
            mx = now;
            s = t;
        } else if (KIND == MM_GRAD) {
            if (m >= a.m) return;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = rs == 0.f ? 0.f : rs * ex2(v[i] * a.c - lse2);
            store_planes(a, m, n, v);
        } else {
            if (m >= a.m) return;
            const size_t o = (size_t)m * a.ldo + n;
            const int left = min(32, a.n - n);
            if (a.acc) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (i < left) v[i] += a.acc[o + i];
            }
            if (a.out_bf16) {
                __nv_bfloat16 *p = static_cast<__nv_bfloat16 *>(a.out) + o;
                if (left == 32 && a.ldo % 8 == 0) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        __nv_bfloat16 q[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) q[j] = __float2bfloat16_rn(v[i + j]);
                        *reinterpret_cast<uint4 *>(p + i) = *reinterpret_cast<const uint4 *>(q);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (i < left) p[i] = __float2bfloat16_rn(v[i]);
                }
            } else {
                float *p = static_cast<float *>(a.out) + o;
                if (left == 32 && a.ldo % 4 == 0) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) st4(p + i, make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]));
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (i < left) p[i] = v[i];
                }
            }
        }
    }
    // `part` column of the 128-column half tile
    __device__ __forceinline__ void end(const MmArgs &a, int m, int half_tile) {
        if (KIND == MM_LSE && m < a.m && (long long)half_tile * MM_LSE_TILE < a.n)
            a.part[(size_t)half_tile * a.m + m] = make_float2(mx, s);
    }
};

template <int KIND, bool AT, bool BT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
mm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
          const MmArgs a, const Tiles q, uint32_t limit, int skip)
{
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
    if (warp == 2) tmem_alloc_pair(smem_u32(&tmem_slot));
    umma_fence_before();
    __syncthreads();
    cluster_sync();
    umma_fence_after();
    const uint32_t tmem = tmem_slot;
    const int pair = blockIdx.x / 2, pairs = gridDim.x / 2, ntiles = q.mt * q.nt;
    const int passes = a.planes == 3 ? 6 : 1;
    const int bhalf = q.bn / 2;
    const int bblocks = BT ? (bhalf + 63) / 64 : 0;

    if (warp == 0 && lane == 0) {
        const uint32_t b_bytes = BT ? bblocks * 8192u : bhalf * 128u;
        int it = 0;
        bool ok = true;
        for (int t = pair; ok && t < ntiles; t += pairs) {
            int mi, ni;
            tile_of(q, t, mi, ni);
            const int m0 = mi * TM + rank * 128, n0 = ni * q.bn + rank * bhalf;
            for (int c = 0; ok && c < passes; ++c) {
                int pa, pb;
                planes_of(passes, c, pa, pb);
                for (int kb = 0; kb < q.kb; ++kb, ++it) {
                    const int st = it % STAGES;
                    if (!wait_bar(empty + 8 * st, ((it / STAGES) & 1) ^ 1, limit)) {
                        ok = false;
                        break;
                    }
                    if (it == skip) continue;
                    const uint32_t bar = leader_addr(full + 8 * st);
                    if (rank == 0) mbar_expect(full + 8 * st, 2 * (HALF + b_bytes));
                    const uint32_t sa = tiles + st * 2 * HALF, sb = sa + HALF;
                    const int k0 = kb * BK;
                    if (AT) {
                        tma3_pair(sa, &map_a, m0, k0, pa, bar);
                        tma3_pair(sa + 8192, &map_a, m0 + 64, k0, pa, bar);
                    } else {
                        tma3_pair(sa, &map_a, k0, m0, pa, bar);
                    }
                    if (BT) {
                        for (int b = 0; b < bblocks; ++b)
                            tma3_pair(sb + b * 8192, &map_b, n0 + 64 * b, k0, pb, bar);
                    } else {
                        tma3_pair(sb, &map_b, k0, n0, pb, bar);
                    }
                    issued = it + 1;
                }
            }
        }
        if (!ok) failed = 1;
    } else if (warp == 1 && lane == 0 && rank == 0) {
        const uint32_t idesc = umma_idesc(q.bn, AT, BT);
        int it = 0, use = 0;
        bool ok = true;
        for (int t = pair; ok && t < ntiles; t += pairs, ++use) {
            const int buf = use & 1;
            if (!wait_bar(tempty + 8 * buf, ((use >> 1) & 1) ^ 1, limit)) {
                ok = false;
                break;
            }
            umma_fence_after();
            const int steps = passes * q.kb;
            for (int i = 0; i < steps; ++i, ++it) {
                const int st = it % STAGES;
                if (!wait_bar(full + 8 * st, (it / STAGES) & 1, limit)) {
                    ok = false;
                    break;
                }
                umma_fence_after();
                const uint32_t sa = tiles + st * 2 * HALF, sb = sa + HALF;
                const uint64_t da = AT ? umma_desc(sa, 8192, 1024) : umma_desc(sa, 16, 1024);
                const uint64_t db = BT ? umma_desc(sb, 8192, 1024) : umma_desc(sb, 16, 1024);
#pragma unroll
                for (int k = 0; k < BK / 16; ++k)       // 16 elements on: 32 bytes along a row, or 16 rows
                    umma_pair(tmem + buf * 256, da + (AT ? 2048 / 16 : 32 / 16) * k,
                              db + (BT ? 2048 / 16 : 32 / 16) * k, idesc, i > 0 || k > 0);
                umma_commit_pair(empty + 8 * st);
            }
            if (ok) umma_commit_pair(tfull + 8 * buf);
        }
        if (!ok) failed = 1;
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
                     ::"r"(drain) : "memory");
        wait_bar(drain, 0, limit);
    } else if (warp >= 4) {
        const int quad = warp % 4, side = (warp - 4) / 4;
        const uint32_t lane_base = tmem + ((uint32_t)quad << 21);
        int use = 0;
        for (int t = pair; t < ntiles; t += pairs, ++use) {
            const int buf = use & 1;
            int mi, ni;
            tile_of(q, t, mi, ni);
            const int m = mi * TM + rank * 128 + quad * 32 + lane;
            Epilogue<KIND> ep;
            ep.begin(a, m);
            // every lane polls; the warp leaves together
            const bool ok = wait_bar(tfull + 8 * buf, (use >> 1) & 1, limit);
            if (__any_sync(~0u, !ok)) {
                if (lane == 0) failed = 1;
                break;
            }
            umma_fence_after();
            const int c0 = side * 128, c1 = min(q.bn, c0 + 128);
            for (int c = c0; c < c1; c += 32) {
                float v[32];
                tmem_load32(lane_base + buf * 256 + c, v);
                tmem_wait();
                if (c + 32 >= c1) {
                    umma_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(leader_addr(tempty + 8 * buf));
                }
                ep.chunk(a, m, ni * q.bn + c, v);
            }
            if (c0 >= c1 && lane == 0) mbar_arrive_cluster(leader_addr(tempty + 8 * buf));
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
    if (warp == 2) tmem_free_pair(tmem);
}

bool encode(PFN_cuTensorMapEncodeTiled_v12000 fn, CUtensorMap *map, const Factor &f, int planes, int rows, int k,
            int box_rows)
{
    const cuuint64_t dim[3] = {(cuuint64_t)(f.t ? rows : k), (cuuint64_t)(f.t ? k : rows), (cuuint64_t)planes};
    const cuuint64_t stride[2] = {(cuuint64_t)f.ld * 2, (cuuint64_t)(planes == 1 ? f.ld : f.plane) * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)(f.t ? BK : box_rows), 1}, one[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16 *>(f.p), dim, stride, box, one,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int KIND, bool AT, bool BT>
cudaError_t launch(const MmArgs &a, cudaStream_t stream)
{
    Tiles q;
    q.bn = 256;
    q.mt = (a.m + TM - 1) / TM;
    q.kb = (a.k + BK - 1) / BK;
    q.nt = (a.n + q.bn - 1) / q.bn;
    const auto fn = tma_encoder();
    CUtensorMap ma, mb;
    if (!fn || !tma_context() || !encode(fn, &ma, a.a, a.planes, a.m, a.k, 128) ||
        !encode(fn, &mb, a.b, a.planes, a.n, a.k, q.bn / 2))
        return cudaErrorInvalidValue;
    constexpr auto kernel = mm_kernel<KIND, AT, BT>;
    const cudaError_t e = smem_opt_in<kernel>(SMEM);
    if (e != cudaSuccess) return e;
    const int pairs = std::min(N_SM / 2, q.mt * q.nt);
    kernel<<<2 * pairs, THREADS, SMEM, stream>>>(ma, mb, a, q, tma_wait_limit(), tma_skip_item());
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_mm(MmKind kind, const MmArgs &a, cudaStream_t stream)
{
    if (kind == MM_LSE) return launch<MM_LSE, false, false>(a, stream);
    if (kind == MM_GRAD) return launch<MM_GRAD, false, false>(a, stream);
    return a.a.t ? launch<MM_OUT, true, true>(a, stream) : launch<MM_OUT, false, true>(a, stream);
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
