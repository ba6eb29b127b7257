// flare_qattn_f32_8.hip -- softmax attention of f32 queries over a cache of 8 bits.
#include "flare_qattn.h"

namespace flare {
namespace attn {
template int rows_e<float, 8>(const AttnArgs&, int, hipStream_t);
}  // namespace attn
}  // namespace flare
