// One status word for the kernels of the row operators: each keeps its own on the device.
#include "common.h"

namespace mggb {
int layer_norm_status(int* status, int reset);
int class_logprob_status(int* status, int reset);
int grouped_dense_status(int* status, int reset);
}  // namespace mggb

extern "C" int mggb_operator_device_status(int* status, int reset) {
    MGGB_REQUIRE(status, "operator_device_status: NULL output");
    int (*const parts[])(int*, int) = {mggb::layer_norm_status, mggb::class_logprob_status, mggb::grouped_dense_status};
    *status = 0;
    for (auto part : parts) {
        int one = 0;
        const int rc = part(&one, reset);
        if (rc != MGGB_OK) return rc;
        if (one && !*status) *status = one;
    }
    return MGGB_OK;
}
