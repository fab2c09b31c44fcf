// Linear attention over chunks, fp16 storage.
#include "lbi_linear_attn_launch.h"

namespace lbi {
namespace linear_attn {

int run_f16(const Call& call, hipStream_t stream) {
    return call.T <= MOST_TWICE ? by_pieces<_Float16, 2, true>(call, stream) : by_pieces<_Float16, 2, false>(call, stream);
}

}  // namespace linear_attn
}  // namespace lbi
