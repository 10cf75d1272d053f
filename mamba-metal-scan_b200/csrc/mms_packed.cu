// The scan over packed sequences in float32; which launches a call takes.
#include "mms_packed.cuh"

namespace mms {

size_t scan_packed_workspace_bytes(int rows, int count, int D, int N) { return Plan(rows, count, D, N).total; }

cudaError_t launch_scan_packed(const ScanPackedArgs &p, cudaStream_t stream)
{
    if (p.bf16) return launch_scan_packed_bf16(p, stream);
    return p.seq.starts.p ? segments_by_states<float>(p, stream) : tokens_by_states<float, float>(p, stream);
}

}  // namespace mms
