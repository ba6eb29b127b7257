// flare_attn_f16.hip -- softmax attention over f16 tensors.
#include "flare_attn_bwd.h"
#include "flare_attn_fwd.h"

namespace flare {
namespace attn {
template int forward_e<__half>(const AttnArgs&, hipStream_t);
template int backward_e<__half>(const AttnArgs&, float*, float*, float*, hipStream_t);
}  // namespace attn
}  // namespace flare
