// Internal interface of the causal convolution (mms_conv.cu), the packed scan
// (mms_packed.cuh) and sampling (mms_sample.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "mms_kernels.h"

namespace mms {

constexpr int CONV_MAX_K = 8;           // taps of the convolution

struct ConvArgs {
    const void *x;                      // element (b, t, d) at x[b * ldb + t * ldt + d]
    long long ldb, ldt;
    const void *w, *bias;               // (D, K), (D) or NULL
    void *y;                            // (Bt, T, D)
    const void *dy;                     // backward: (Bt, T, D)
    void *dx, *dw, *dbias;
    float *part;                        // backward: conv_workspace_bytes()
    int Bt, T, D, K;
    bool silu, bf16;
};

size_t conv_workspace_bytes(int Bt, int T, int D, int K);
cudaError_t launch_conv_fwd(const ConvArgs &a, cudaStream_t stream);
cudaError_t launch_conv_bwd(const ConvArgs &a, cudaStream_t stream);

// Whole numbers of 32 or 64 bits on the device.
struct Ints {
    const void *p;
    bool wide;
    __device__ __forceinline__ long long at(long long i) const {
        return wide ? reinterpret_cast<const long long *>(p)[i] : (long long)reinterpret_cast<const int *>(p)[i];
    }
};

// Sequences of packed rows: sequence s has the rows starts[s] .. starts[s + 1] - 1
// (starts.p NULL: row s alone), goes on from place slots[s] of a cache of `places`
// (slots.p NULL: place s; outside the cache: from nothing) and leaves its state in
// place out_slots[s] (NULL: slots; outside: nowhere).
struct Sequences {
    Ints starts, slots, out_slots;
    int count, rows, places;

    // starts[s] brought into [0, rows], so that no list leads outside the arrays
    __device__ __forceinline__ int start(int s) const {
        if (!starts.p) return s;
        const long long v = starts.at(s);
        return (int)(v < 0 ? 0 : v > rows ? rows : v);
    }
    // the place in the cache, -1 for none
    __device__ __forceinline__ long long place(const Ints &list, int s) const {
        const long long v = list.p ? list.at(s) : s;
        return v >= 0 && v < places ? v : -1;
    }
    __device__ __forceinline__ long long from(int s) const { return place(slots, s); }
    __device__ __forceinline__ long long to(int s) const { return place(out_slots.p ? out_slots : slots, s); }
    // The last s in [0, n) with key(s) <= v for ascending keys, -1 if there is none; by a whole
    // warp, 32 keys at a time (two loads deep up to 1024 sequences).
    template <typename Key>
    __device__ static __forceinline__ int last_at_most(int n, int v, Key key) {
        const int lane = threadIdx.x & 31;
        int lo = 0;
        while (n > 32) {
            const int step = (n + 31) / 32, i = lane * step;
            const int below = __popc(__ballot_sync(0xffffffffu, i < n && key(lo + i) <= v));
            if (below == 0) return lo - 1;
            lo += (below - 1) * step;
            n = min(step, n - (below - 1) * step);
        }
        return lo + __popc(__ballot_sync(0xffffffffu, lane < n && key(lo + lane) <= v)) - 1;
    }
};

struct ConvPackedArgs {
    const void *x;                      // (rows, D), row stride ldx
    long long ldx;
    const void *w, *bias;
    void *window;                       // (places, D, K - 1)
    void *y;                            // (rows, D)
    Sequences seq;
    int D, K;
    bool silu, bf16;
};

cudaError_t launch_conv_packed(const ConvPackedArgs &a, cudaStream_t stream);

struct ScanPackedArgs {
    const void *x, *dt, *B, *C, *z;     // (rows, D), (rows, N): row strides below; z NULL: no gate
    long long ldx, lddt, ldB, ldC, ldz;
    const float *aneg, *d_skip;         // (D, N), (D) or NULL
    float *state;                       // (places, D, N)
    void *y;                            // (rows, D)
    void *workspace;
    Sequences seq;
    int D, N;
    Proj proj;
    bool bf16, bc_bf16;                 // storage of x, dt, z, y; of B and C
};

size_t scan_packed_workspace_bytes(int rows, int count, int D, int N);
cudaError_t launch_scan_packed(const ScanPackedArgs &a, cudaStream_t stream);
cudaError_t launch_scan_packed_bf16(const ScanPackedArgs &a, cudaStream_t stream);   // its part with bf16 set

struct SampleArgs {
    const void *logits;                 // (rows, vocab), row stride ld
    long long ld;
    const float *uniform;               // (rows)
    // one value a row, or (NULL) the same for all
    const float *temperature, *top_p, *min_p;
    Ints top_k;
    float temperature1, top_p1, min_p1;
    long long top_k1;
    int64_t *token;                     // (rows)
    float *logprob;                     // (rows) or NULL
    int rows, vocab;
    bool bf16;
};

cudaError_t launch_sample(const SampleArgs &a, cudaStream_t stream);

}  // namespace mms
