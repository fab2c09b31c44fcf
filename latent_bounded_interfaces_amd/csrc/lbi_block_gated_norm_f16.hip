// The norms behind and before a block, fp16 branches.
#include "lbi_block_gated_norm_kernel.h"

namespace lbi {
namespace block_norm {

int forward_f16(const Forward& f, bool same, hipStream_t stream) { return same ? forward<_Float16, _Float16>(f, stream) : forward<_Float16, float>(f, stream); }
int pullback_f16(const Pullback& f, bool same, hipStream_t stream) { return same ? pullback<_Float16, _Float16>(f, stream) : pullback<_Float16, float>(f, stream); }

}  // namespace block_norm
}  // namespace lbi
