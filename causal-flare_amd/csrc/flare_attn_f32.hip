// flare_attn_f32.hip -- softmax attention over f32 tensors.
#include "flare_attn_bwd.h"
#include "flare_attn_fwd.h"

namespace flare {
namespace attn {
template int forward_e<float>(const AttnArgs&, hipStream_t);
template int backward_e<float>(const AttnArgs&, float*, float*, float*, hipStream_t);
}  // namespace attn
}  // namespace flare
