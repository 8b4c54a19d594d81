// k_attention_bf16.hip -- the attention kernels over bf16 tensors.
#include "fg_attention_kernel.h"

namespace fg {
namespace attn {
template int forward<kBF16>(hipStream_t, const Args &, bool, bool);
template int combine<kBF16>(hipStream_t, const Args &);
template int backward<kBF16>(hipStream_t, const Args &, bool);
}  // namespace attn
}  // namespace fg
