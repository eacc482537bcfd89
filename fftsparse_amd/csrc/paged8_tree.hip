// Paged attention of trees of new tokens, over 8-bit pages: that form of the kernels in paged_kernel.h.
#include "paged_kernel.h"

namespace fs {

FS_PAGED_FORM(run_tree8) { return run<true, k8 | kTree>(k, dtype, D, few, true, w, work, B, Lq, s, fn); }

}  // namespace fs
