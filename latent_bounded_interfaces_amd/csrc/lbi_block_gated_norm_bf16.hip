// The norms behind and before a block, bf16 branches.
#include "lbi_block_gated_norm_kernel.h"

namespace lbi {
namespace block_norm {

int forward_bf16(const Forward& f, bool same, hipStream_t stream) { return same ? forward<bf16_raw, bf16_raw>(f, stream) : forward<bf16_raw, float>(f, stream); }
int pullback_bf16(const Pullback& f, bool same, hipStream_t stream) { return same ? pullback<bf16_raw, bf16_raw>(f, stream) : pullback<bf16_raw, float>(f, stream); }

}  // namespace block_norm
}  // namespace lbi
