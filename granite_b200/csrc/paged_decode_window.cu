// Decode over a sliding window over the fp16 caches (paged_decode.cuh built for it).
#include "paged_decode.cuh"

namespace gb200 {

int launch_paged_decode_window(granite_cuda_compute* c, const GraniteCudaPagedDecodeArgs& a, bool contiguous, uint32_t max_seq, const CacheView& view) {
    return launch_decode_as<kElemF16, true>(c, a, contiguous, max_seq, nullptr, view);
}

}  // namespace gb200
