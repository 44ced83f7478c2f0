// Grouped products of f16 matrices: see grouped_kernels.h.
#include "grouped_kernels.h"

MGGB_GROUPED_TYPE(f16, __half)
