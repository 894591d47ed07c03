// Instances of the tcgen05 attention kernel.
#include "gaf_attend_wide.cuh"

namespace tgaf {
namespace attend {

cudaError_t launch_wide(const Params &p, const CUtensorMap &tmap, int sm_count, cudaStream_t stream) {
    const KvView &kv = p.a.kv;
    if (kv.head_dim == 64u) {
        if (kv.bits == 4u) return kv.group == 32u ? launch_wide<64, 4, 32>(p, tmap, sm_count, stream) : launch_wide<64, 4, 64>(p, tmap, sm_count, stream);
        return kv.group == 32u ? launch_wide<64, 8, 32>(p, tmap, sm_count, stream) : launch_wide<64, 8, 64>(p, tmap, sm_count, stream);
    }
    if (kv.bits == 4u)
        return kv.group == 32u ? launch_wide<128, 4, 32>(p, tmap, sm_count, stream)
             : kv.group == 64u ? launch_wide<128, 4, 64>(p, tmap, sm_count, stream) : launch_wide<128, 4, 128>(p, tmap, sm_count, stream);
    return kv.group == 32u ? launch_wide<128, 8, 32>(p, tmap, sm_count, stream)
         : kv.group == 64u ? launch_wide<128, 8, 64>(p, tmap, sm_count, stream) : launch_wide<128, 8, 128>(p, tmap, sm_count, stream);
}

}  // namespace attend
}  // namespace tgaf
