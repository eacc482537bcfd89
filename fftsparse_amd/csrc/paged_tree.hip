// Paged attention of trees of new tokens: that form of the kernels in paged_kernel.h.
#include "paged_kernel.h"

namespace fs {

FS_PAGED_FORM(run_tree) { return run<true, kTree>(k, dtype, D, few, true, w, work, B, Lq, s, fn); }

}  // namespace fs
