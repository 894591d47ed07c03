// Instances of the attention kernel for heads of 128 values in 8-bit codes.
#include "gaf_attend.cuh"

namespace tgaf {
namespace attend {

cudaError_t launch_d128_b8(const Params &p, const CUtensorMap &tmap, int nt, int limbs, int sm_count, cudaStream_t stream) {
    if (p.a.kv.group == 32u) return launch_rows<128, 8, 32>(p, tmap, nt, limbs, sm_count, stream);
    if (p.a.kv.group == 128u) return launch_rows<128, 8, 128>(p, tmap, nt, limbs, sm_count, stream);
    return launch_rows<128, 8, 64>(p, tmap, nt, limbs, sm_count, stream);
}

}  // namespace attend
}  // namespace tgaf
