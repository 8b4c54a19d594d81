// k_attention_f32.hip -- the attention kernels over fp32 tensors.
#include "fg_attention_kernel.h"

namespace fg {
namespace attn {
template int forward<kF32>(hipStream_t, const Args &, bool, bool);
template int combine<kF32>(hipStream_t, const Args &);
template int backward<kF32>(hipStream_t, const Args &, bool);
}  // namespace attn
}  // namespace fg
