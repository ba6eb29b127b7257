// flare_qattn_bf16_8.hip -- softmax attention of bf16 queries over a cache of 8 bits.
#include "flare_attn_fwd.h"
#include "flare_qattn.h"

namespace flare {
namespace attn {
template int forward_bits<__hip_bfloat16, 8>(const AttnArgs&, hipStream_t);
template int rows_e<__hip_bfloat16, 8>(const AttnArgs&, int, hipStream_t);
}  // namespace attn
}  // namespace flare
