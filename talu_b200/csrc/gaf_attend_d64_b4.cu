// Instances of the attention kernel for heads of 64 values in 4-bit codes.
#include "gaf_attend.cuh"

namespace tgaf {
namespace attend {

cudaError_t launch_d64_b4(const Params &p, const CUtensorMap &tmap, int nt, int limbs, int sm_count, cudaStream_t stream) {
    if (p.a.kv.group == 32u) return launch_rows<64, 4, 32>(p, tmap, nt, limbs, sm_count, stream);
    return launch_rows<64, 4, 64>(p, tmap, nt, limbs, sm_count, stream);
}

}  // namespace attend
}  // namespace tgaf
