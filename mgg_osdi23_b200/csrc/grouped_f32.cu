// Grouped products of f32 matrices: see grouped_kernels.h.
#include "grouped_kernels.h"

MGGB_GROUPED_TYPE(f32, float)

namespace mggb {
size_t grouped_scratch(long long n, int groups, int K, int M, bool f32) { return cut(n, groups, K, M, f32).bytes; }
}  // namespace mggb
