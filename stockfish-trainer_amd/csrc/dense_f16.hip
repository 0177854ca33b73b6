// The dense head's products in f16.
#include "dense_tile.h"

namespace sft {
namespace dense {
SFT_DENSE_TYPE(f16_t)
}  // namespace dense
}  // namespace sft
