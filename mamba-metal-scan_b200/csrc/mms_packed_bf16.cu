// The scan over packed sequences with x, dt, z and y in bf16 (a file of its own: they compile side by side).
#include "mms_packed.cuh"

namespace mms {

cudaError_t launch_scan_packed_bf16(const ScanPackedArgs &p, cudaStream_t stream)
{
    using BF = __nv_bfloat16;
    if (p.seq.starts.p) return segments_by_states<BF>(p, stream);
    return p.bc_bf16 ? tokens_by_states<BF, BF>(p, stream) : tokens_by_states<BF, float>(p, stream);
}

}  // namespace mms
