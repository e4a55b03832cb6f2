// vws_tree_f16.hip -- the drafted trees' attention over a binary16 cache (see vws_tree_kernel.h).
#include "vws_tree_kernel.h"

namespace vws {
VWS_TREES(_Float16)
}  // namespace vws
