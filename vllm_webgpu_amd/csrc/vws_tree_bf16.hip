// vws_tree_bf16.hip -- the drafted trees' attention over a bfloat16 cache (see vws_tree_kernel.h).
#include "vws_tree_kernel.h"

namespace vws {
VWS_TREES(uint16_t)
}  // namespace vws
