// Grouped products of bf16 matrices: see grouped_kernels.h.
#include "grouped_kernels.h"

MGGB_GROUPED_TYPE(bf16, __nv_bfloat16)
