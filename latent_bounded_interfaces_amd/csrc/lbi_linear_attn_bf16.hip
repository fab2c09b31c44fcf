// Linear attention over chunks, bf16 storage.
#include "lbi_linear_attn_launch.h"

namespace lbi {
namespace linear_attn {

// A state that the caller keeps takes all 24 significant bits of the decayed values, one that only feeds 16-bit results 16 of them.
int run_bf16(const Call& call, bool exact_last, hipStream_t stream) {
    return exact_last ? by_pieces<bf16_raw, 3>(call, stream) : by_pieces<bf16_raw, 2>(call, stream);
}

}  // namespace linear_attn
}  // namespace lbi
