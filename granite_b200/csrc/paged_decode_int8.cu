// Decode over the int8 cache (paged_decode.cuh built for it).
#include "paged_decode.cuh"

namespace gb200 {

int launch_paged_decode_int8(granite_cuda_compute* c, const GraniteCudaPagedDecodeArgs& a, const CacheView& view) {
    return launch_decode_as<kElemInt8, true>(c, a, false, 0, nullptr, view);
}

}  // namespace gb200
