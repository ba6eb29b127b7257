// flare_qattn_f32_4.hip -- softmax attention of f32 queries over a cache of 4 bits.
#include "flare_qattn.h"

namespace flare {
namespace attn {
template int rows_e<float, 4>(const AttnArgs&, int, hipStream_t);
}  // namespace attn
}  // namespace flare
