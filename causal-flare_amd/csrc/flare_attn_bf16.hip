// flare_attn_bf16.hip -- softmax attention over bf16 tensors.
#include "flare_attn_bwd.h"
#include "flare_attn_fwd.h"

namespace flare {
namespace attn {
template int forward_e<__hip_bfloat16>(const AttnArgs&, hipStream_t);
template int backward_e<__hip_bfloat16>(const AttnArgs&, float*, float*, float*, hipStream_t);
}  // namespace attn
}  // namespace flare
