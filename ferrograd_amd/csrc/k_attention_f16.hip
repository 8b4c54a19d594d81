// k_attention_f16.hip -- the attention kernels over fp16 tensors.
#include "fg_attention_kernel.h"

namespace fg {
namespace attn {
template int forward<kF16>(hipStream_t, const Args &, bool, bool);
template int combine<kF16>(hipStream_t, const Args &);
template int backward<kF16>(hipStream_t, const Args &, bool);
}  // namespace attn
}  // namespace fg
