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
// Tile order: the dimension with fewer tiles runs fastest, in groups of 16,
// so the concurrent tiles share one side's panels in L2 and the long side is
// read from HBM once.
//
// float32 factors are three bf16 planes each; a product then runs over the
// six pairs of planes with i + j <= 2, smallest terms first.
//
// The tensor core adds each 16 summed elements to its fp32 sum with truncation,
// not rounding, so a long sum drifts towards zero by about n 2^-25 of itself
// over n additions (measured: 1.1e-5 at 8192 elements). Where the result
// stays float32 the sum is therefore cut into parts of PART elements: each
// goes to its own tensor memory buffer and the epilogue warps add the parts up
// in registers, rounding to nearest (`PARTS`).
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
constexpr int PART = 256;                                    // summed elements (of each pair of planes) per part
constexpr size_t SMEM = 1024 + (size_t)STAGES * 2 * HALF + 256;

__device__ unsigned int g_mm_timeout;

struct Tiles {
    int mt, nt, bn;         // tiles of rows and columns, columns per tile (a multiple of 64)
    int splits, kb;         // work items per tile, steps of BK summed elements of each
    int steps;              // steps of the whole sum
    int part;               // steps per part of a sum
};

// Columns per tile and splits of the sum: the cheapest by a model of the clocks
// of a pair. A step of 64 summed elements is the larger of the multiplies
// (2 clocks a column, at full rate) and the copies of 16 KB + 64 bytes a
// column into each CTA; an item ends with an epilogue that nothing overlaps
// on the last one; the waves are those of 74 pairs. Splits pay a write and a
// read of their partial sums and one more launch.
Tiles plan(MmKind kind, int m, int n, int k, int planes, size_t split_bytes)
{
    Tiles best{};
    double least = 0;
    const int passes = planes == 3 ? 6 : 1;
    const int steps = (k + BK - 1) / BK;
    for (int bn = 256; bn >= 64; bn -= 64) {
        Tiles q;
        q.mt = (m + TM - 1) / TM;
        q.nt = (n + bn - 1) / bn;
        q.bn = bn;
        q.steps = steps;
        const long long tiles = (long long)q.mt * q.nt;
        const double step = std::max(2.0 * bn, 234 + 0.92 * bn) * passes;
        for (int s = 1; s <= (kind == MM_OUT ? 74 : 1); ++s) {
            if (s > 1 && (tiles * s > 74 * 8 || steps < 4 * s || (size_t)s * m * n * 4 > split_bytes)) break;
            q.kb = (steps + s - 1) / s;
            q.splits = (steps + q.kb - 1) / q.kb;
            if (q.splits != s) continue;
            const double waves = (double)((tiles * s + N_SM / 2 - 1) / (N_SM / 2));
            double cost = waves * (q.kb * step + 300) + 1500 + 10 * bn;
            if (s > 1) cost += 5000 + (2.0 * s + 1) * m * n * 4 / 3000;
            if (!best.mt || cost < 0.97 * least) {
                best = q;
                least = cost;
            }
        }
    }
    return best;
}

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
    __device__ __forceinline__ void chunk(const MmArgs &a, int split, int m, int n, float (&v)[32]) {
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
            const size_t o = ((size_t)split * a.m + m) * a.ldo + n;
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
    __device__ __forceinline__ void end(const MmArgs &a, int m, int i) {
        if (KIND == MM_LSE && m < a.m)
            a.part[(size_t)i * a.m + m] = make_float2(mx, s);
    }
};

template <int KIND, bool AT, bool BT, bool PARTS>
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
    if (warp == 9) tmem_alloc_pair(smem_u32(&tmem_slot));
    umma_fence_before();
    __syncthreads();
    cluster_sync();
    umma_fence_after();
    const uint32_t tmem = tmem_slot;
    const int pair = blockIdx.x / 2, pairs = gridDim.x / 2, items = q.mt * q.nt * q.splits;
    const int passes = a.planes == 3 ? 6 : 1;
    const int bhalf = q.bn / 2;
    const int bblocks = BT ? (bhalf + 63) / 64 : 0;

    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
    if (warp == 8 && lane == 0) {
        const uint32_t b_bytes = BT ? bblocks * 8192u : bhalf * 128u;
        int it = 0;
        bool ok = true;
        for (int t = pair; ok && t < items; t += pairs) {
            int mi, ni;
            tile_of(q, t / q.splits, mi, ni);
            const int k_begin = t % q.splits * q.kb, k_end = min(q.steps, k_begin + q.kb);
            const int m0 = mi * TM + rank * 128, n0 = ni * q.bn + rank * bhalf;
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
    } else if (warp == 9 && lane == 0 && rank == 0) {
        const uint32_t idesc = umma_idesc(q.bn, AT, BT);
        int it = 0, use = 0;
        bool ok = true;
        for (int t = pair; ok && t < items; t += pairs) {
        const int k_begin = t % q.splits * q.kb, k_end = min(q.steps, k_begin + q.kb);
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
                const uint32_t sa = tiles + st * 2 * HALF, sb = sa + HALF;
                const uint64_t da = AT ? umma_desc(sa, 8192, 1024) : umma_desc(sa, 16, 1024);
                const uint64_t db = BT ? umma_desc(sb, 8192, 1024) : umma_desc(sb, 16, 1024);
#pragma unroll
                for (int k = 0; k < BK / 16; ++k)       // 16 elements on: 32 bytes along a row, or 16 rows
                    umma_pair(tmem + buf * 256, da + (AT ? 2048 / 16 : 32 / 16) * k,
                              db + (BT ? 2048 / 16 : 32 / 16) * k, idesc, i > 0 || k > 0);
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
        const int cols = q.bn / 2, c0 = side * cols;
        int use = 0;
        bool ok = true;
        for (int t = pair; ok && t < items; t += pairs) {
            int mi, ni;
            tile_of(q, t / q.splits, mi, ni);
            const int split = t % q.splits, k_begin = split * q.kb, k_end = min(q.steps, k_begin + q.kb);
            const int m = mi * TM + rank * 128 + quad * 32 + lane;
            Epilogue<KIND> ep;
            ep.begin(a, m);
            float2 sum[PARTS ? 4 : 1][16];
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
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float v[32];
                    if (32 * c < cols) {
                        tmem_load32(lane_base + buf * 256 + c0 + 32 * c, v);
                        tmem_wait();
                        if (PARTS) {
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                sum[c][i] = k_first > k_begin ? add2(sum[c][i], f2(v[2 * i], v[2 * i + 1]))
                                                    : f2(v[2 * i], v[2 * i + 1]);
                        }
                    }
                    if (c == 3) {                       // read: the next multiplies may overwrite it
                        umma_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(leader_addr(tempty + 8 * buf));
                    }
                    if (!PARTS && 32 * c < cols) ep.chunk(a, split, m, ni * q.bn + c0 + 32 * c, v);
                }
            }
            if (!ok) break;
            if (PARTS) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (32 * c < cols)
                        ep.chunk(a, split, m, ni * q.bn + c0 + 32 * c, reinterpret_cast<float (&)[32]>(sum[c]));
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

template <int KIND, bool AT, bool BT, bool PARTS>
cudaError_t launch(const MmArgs &a, Tiles q, cudaStream_t stream)
{
    q.part = PARTS ? PART / BK : q.kb;
    const auto fn = tma_encoder();
    CUtensorMap ma, mb;
    if (!fn || !tma_context() || !encode(fn, &ma, a.a, a.planes, a.m, a.k, 128) ||
        !encode(fn, &mb, a.b, a.planes, a.n, a.k, q.bn / 2))
        return cudaErrorInvalidValue;
    constexpr auto kernel = mm_kernel<KIND, AT, BT, PARTS>;
    const cudaError_t e = smem_opt_in<kernel>(SMEM);
    if (e != cudaSuccess) return e;
    const int pairs = std::min(N_SM / 2, q.mt * q.nt * q.splits);
    kernel<<<2 * pairs, THREADS, SMEM, stream>>>(ma, mb, a, q, tma_wait_limit(), tma_skip_item());
    return cudaGetLastError();
}

// out = acc + the splits' partial sums, in order.
template <typename T>
__global__ void __launch_bounds__(256)
split_sum_kernel(const float *__restrict__ part, int splits, const float *__restrict__ acc, T *__restrict__ out,
                 long long n)
{
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        float s = acc ? acc[i] : 0.f;
        for (int k = 0; k < splits; ++k) s += part[k * n + i];
        out[i] = from_f<T>(s);
    }
}

}  // namespace

int mm_lse_parts(int m, int n, int k, int planes) { return 2 * plan(MM_LSE, m, n, k, planes, 0).nt; }

size_t mm_split_bytes(int m, int n, int k, int planes)
{
    const Tiles q = plan(MM_OUT, m, n, k, planes, ~(size_t)0);
    return q.splits > 1 ? (size_t)q.splits * m * n * 4 : 0;
}

cudaError_t launch_mm(MmKind kind, const MmArgs &a, cudaStream_t stream)
{
    const Tiles q = plan(kind, a.m, a.n, a.k, a.planes, a.split_bytes);
    // float32 results in parts; what is rounded to bf16 anyway (2^-9) in one sum
    const bool parts = q.kb * BK > PART && (kind == MM_LSE || a.planes == 3);
    if (kind == MM_LSE)
        return parts ? launch<MM_LSE, false, false, true>(a, q, stream)
                     : launch<MM_LSE, false, false, false>(a, q, stream);
    if (kind == MM_GRAD)
        return parts ? launch<MM_GRAD, false, false, true>(a, q, stream)
                     : launch<MM_GRAD, false, false, false>(a, q, stream);
    MmArgs o = a;
    if (q.splits > 1) {
        o.out = a.split;
        o.out_bf16 = false;
        o.acc = nullptr;
        o.ldo = a.n;
    }
    const cudaError_t e = a.a.t ? parts ? launch<MM_OUT, true, true, true>(o, q, stream)
                                        : launch<MM_OUT, true, true, false>(o, q, stream)
                                : parts ? launch<MM_OUT, false, true, true>(o, q, stream)
                                        : launch<MM_OUT, false, true, false>(o, q, stream);
    if (e != cudaSuccess || q.splits == 1) return e;
    const long long n = (long long)a.m * a.n;           // out is contiguous (ldo == n)
    const int grid = (int)std::min<long long>((n + 255) / 256, N_SM * 16);
    if (a.out_bf16)
        split_sum_kernel<<<grid, 256, 0, stream>>>(a.split, q.splits, a.acc, static_cast<__nv_bfloat16 *>(a.out), n);
    else
        split_sum_kernel<<<grid, 256, 0, stream>>>(a.split, q.splits, a.acc, static_cast<float *>(a.out), n);
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
