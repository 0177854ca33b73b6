// The dense head's products in f32.
#include "dense_tile.h"

namespace sft {
namespace dense {
SFT_DENSE_TYPE(float)
}  // namespace dense
}  // namespace sft
