// One status word for the kernels of the row operators: each keeps its own on the device.  The limit of their waits.
#include "common.h"

namespace mggb {
int layer_norm_status(int* status, int reset);
int class_logprob_status(int* status, int reset);
int grouped_dense_status(int* status, int reset);

static std::atomic<unsigned> g_polls{ASYNC_SPIN_LIMIT};
unsigned wait_polls() { return g_polls.load(std::memory_order_relaxed); }
}  // namespace mggb

extern "C" int mggb_operator_wait_limit(int64_t polls, int64_t* before) {
    MGGB_REQUIRE(polls >= -1 && polls <= mggb::ASYNC_SPIN_LIMIT, "operator_wait_limit: need 0 <= polls <= %u, or -1 for the default, got %lld",
                 mggb::ASYNC_SPIN_LIMIT, (long long)polls);
    const unsigned was = mggb::g_polls.exchange(polls < 0 ? mggb::ASYNC_SPIN_LIMIT : (unsigned)polls);
    if (before) *before = was;
    return MGGB_OK;
}

extern "C" int mggb_operator_device_status(int* status, int reset) {
    MGGB_REQUIRE(status, "operator_device_status: NULL output");
    int (*const parts[])(int*, int) = {mggb::layer_norm_status, mggb::class_logprob_status, mggb::grouped_dense_status};
    *status = 0;
    MGGB_CUDA(cudaDeviceSynchronize());        // a read of the words alone would not wait for streams that do not block the default one
    for (auto part : parts) {
        int one = 0;
        const int rc = part(&one, reset);
        if (rc != MGGB_OK) return rc;
        if (one && !*status) *status = one;
    }
    return MGGB_OK;
}
