// tc_attn.hip -- which attention kernels serve a call, and their scratch.
#include "tc_attn_common.hpp"
#include "tc_kernels.hpp"

namespace tc {

size_t attn_scratch_bytes(int num_cu) { return attn_part_bytes(num_cu); }

hipError_t launch_attn(const AttnArgs &a, int ctype, int num_cu, void *scratch, hipStream_t st) {
    switch (ctype) {
        case kF16: return launch_attn_cache<kF16>(a, num_cu, scratch, st);
        case kBF16: return launch_attn_cache<kBF16>(a, num_cu, scratch, st);
        case kI8: return launch_attn_cache<kI8>(a, num_cu, scratch, st);
        default: return launch_attn_cache<kE4M3>(a, num_cu, scratch, st);
    }
}

}  // namespace tc
