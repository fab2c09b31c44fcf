// Linear attention over chunks, bf16 storage.
#include "lbi_linear_attn_launch.h"

namespace lbi {
namespace linear_attn {

// exact: a state takes all 24 significant bits of the decayed values, in every forward call, so that its results do not go by whether the state is returned,
// and in pullbacks that return the state's cotangent.  Otherwise it takes 16 of them: then it only feeds 16-bit results through a copy of 8 bits, which
// is what their error goes by (us, 24 bits / 16: a basis of 4 for 64 heads of 4096 of 128 556 / 502, of 2 307 / 275, one direction for 96 of 1024 of 64 42 / 39; forwards,
// 64 chains of 4096 of 128 103 / 89, 512 462 / 451, 96 of 1024 of 64 27 / 26).
int run_bf16(const Call& call, bool exact, hipStream_t stream) {
    if (call.T <= MOST_TWICE) return by_pieces<bf16_raw, 3, true>(call, stream);
    return exact ? by_pieces<bf16_raw, 3, false>(call, stream) : by_pieces<bf16_raw, 2, false>(call, stream);
}

}  // namespace linear_attn
}  // namespace lbi
