// The dense head's products in bf16.
#include "dense_tile.h"

namespace sft {
namespace dense {
SFT_DENSE_TYPE(bf16_t)
}  // namespace dense
}  // namespace sft
