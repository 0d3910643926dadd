// Decode over the fp8 e4m3 cache (paged_decode.cuh built for it).
#include "paged_decode.cuh"

namespace gb200 {

int launch_paged_decode_e4m3(granite_cuda_compute* c, const GraniteCudaPagedDecodeArgs& a, const CacheView& view) {
    return launch_decode_as<kElemE4M3, true>(c, a, false, 0, nullptr, view);
}

}  // namespace gb200
