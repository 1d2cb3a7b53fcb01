// linear_kernel for one tile shape (CTAs per tile, columns)
#include "linear_kernel.cuh"

namespace act { namespace linear { ACT_LINEAR_INSTANTIATE(1, 64) } }
