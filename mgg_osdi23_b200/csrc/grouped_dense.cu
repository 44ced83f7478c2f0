// Entry points of the dense products grouped by node type; the kernels are in grouped_kernels.h, compiled once per type.
#include "elem.h"
#include "overlap.h"

namespace mggb {
#define DECLARE(NAME)                                                                                                                          \
    int grouped_forward_##NAME(void*, const void*, const void*, const int32_t*, int, long long, int, int, cudaStream_t);                       \
    int grouped_backward_##NAME(void*, float*, const void*, const void*, const void*, const int32_t*, int, long long, int, int, void*,         \
                                cudaStream_t);                                                                                                 \
    int grouped_status_##NAME(int*, int);
DECLARE(f32)
DECLARE(bf16)
DECLARE(f16)
size_t grouped_scratch(long long n, int groups, int K, int M, bool f32);

int grouped_dense_status(int* status, int reset) {
    *status = 0;
    for (auto part : {grouped_status_f32, grouped_status_bf16, grouped_status_f16}) {
        int one = 0;
        const int rc = part(&one, reset);
        if (rc != MGGB_OK) return rc;
        if (one && !*status) *status = one;
    }
    return MGGB_OK;
}
}  // namespace mggb

namespace {

using namespace mggb;

int check_sizes(const char* who, int groups, long long n, int K, int M) {
    MGGB_REQUIRE(n >= 0 && K >= 1 && M >= 1, "%s: need n >= 0, dim1 >= 1, dim2 >= 1 (n=%lld dim1=%d dim2=%d)", who, n, K, M);
    MGGB_REQUIRE(n <= 0x7FFFFFFFLL, "%s: row positions are int32: n=%lld is too large", who, n);
    MGGB_REQUIRE(groups >= 1, "%s: need groups >= 1, got %d", who, groups);
    if (groups > MGGB_MAX_GROUPS || K > MGGB_MAX_GROUPED_DIM || M > MGGB_MAX_GROUPED_DIM)
        return fail(MGGB_ERR_UNSUPPORTED, "%s: at most %d groups and dimensions of at most %d (groups=%d dim1=%d dim2=%d)", who, MGGB_MAX_GROUPS,
                    MGGB_MAX_GROUPED_DIM, groups, K, M);
    return MGGB_OK;
}

}  // namespace

extern "C" {

int mggb_grouped_dense_forward(void* out, const void* x, const void* w, const int32_t* group_ptr, int groups, int64_t n, int dim1, int dim2,
                               int dtype, void* stream) {
    MGGB_REQUIRE_DTYPE(dtype, "grouped_dense_forward");
    const int rc = check_sizes("grouped_dense_forward", groups, n, dim1, dim2);
    if (rc != MGGB_OK || n == 0) return rc;
    MGGB_REQUIRE(out && x && w && group_ptr, "grouped_dense_forward: NULL argument");
    MGGB_REQUIRE(out != x && out != w, "grouped_dense_forward: out must not alias an input");
    const uint64_t s = elem_bytes(dtype), n_x = n * dim1 * s, n_y = n * dim2 * s, n_w = (uint64_t)groups * dim1 * dim2 * s;
    MGGB_REQUIRE(!runs_meet(out, n_y, x, n_x) && !runs_meet(out, n_y, w, n_w), "grouped_dense_forward: out lies partly over an input");
    const auto run = dtype == MGGB_F32 ? grouped_forward_f32 : dtype == MGGB_BF16 ? grouped_forward_bf16 : grouped_forward_f16;
    return run(out, x, w, group_ptr, groups, n, dim1, dim2, (cudaStream_t)stream);
}

int mggb_grouped_dense_backward_scratch_bytes(int64_t n, int groups, int dim1, int dim2, int dtype, size_t* bytes) {
    MGGB_REQUIRE(bytes, "grouped_dense_backward_scratch_bytes: NULL output");
    MGGB_REQUIRE_DTYPE(dtype, "grouped_dense_backward_scratch_bytes");
    const int rc = check_sizes("grouped_dense_backward_scratch_bytes", groups, n, dim1, dim2);
    if (rc != MGGB_OK) return rc;
    *bytes = grouped_scratch(n, groups, dim1, dim2, dtype == MGGB_F32);      // sums in fp32; the type decides how they are cut
    return MGGB_OK;
}

int mggb_grouped_dense_backward(void* dx, float* dw, const void* dy, const void* x, const void* w, const int32_t* group_ptr, int groups, int64_t n,
                                int dim1, int dim2, int dtype, void* scratch, size_t scratch_bytes, void* stream) {
    MGGB_REQUIRE_DTYPE(dtype, "grouped_dense_backward");
    int rc = check_sizes("grouped_dense_backward", groups, n, dim1, dim2);
    if (rc != MGGB_OK) return rc;
    MGGB_REQUIRE(group_ptr, "grouped_dense_backward: NULL group_ptr");
    MGGB_REQUIRE(dx || dw || n == 0, "grouped_dense_backward: no output given");
    MGGB_REQUIRE(n == 0 || dy, "grouped_dense_backward: NULL dy");
    MGGB_REQUIRE(n == 0 || !dx || w, "grouped_dense_backward: dx needs w");
    MGGB_REQUIRE(n == 0 || !dw || x, "grouped_dense_backward: dw needs x");
    MGGB_REQUIRE(n == 0 || !dx || (dx != dy && dx != w && dx != x), "grouped_dense_backward: dx must not alias an input");
    MGGB_REQUIRE(n == 0 || !dw || (dw != dy && dw != x && dw != dx), "grouped_dense_backward: dw must not alias dy, x or dx");
    if (dw) {
        size_t need = 0;
        rc = mggb_grouped_dense_backward_scratch_bytes(n, groups, dim1, dim2, dtype, &need);
        if (rc != MGGB_OK) return rc;
        MGGB_REQUIRE(need == 0 || (scratch && scratch_bytes >= need), "grouped_dense_backward: scratch of %zu bytes needed, %zu given", need, scratch ? scratch_bytes : (size_t)0);
        MGGB_REQUIRE(need == 0 || (uintptr_t)scratch % 16 == 0, "grouped_dense_backward: scratch must be 16-byte aligned");
    }
    const uint64_t s = elem_bytes(dtype), n_x = n * dim1 * s, n_y = n * dim2 * s, n_w = (uint64_t)groups * dim1 * dim2 * s, n_dw = (uint64_t)groups * dim1 * dim2 * 4;
    MGGB_REQUIRE(n == 0 || !dx || !(runs_meet(dx, n_x, dy, n_y) || runs_meet(dx, n_x, w, n_w) || (x && runs_meet(dx, n_x, x, n_x))),
                 "grouped_dense_backward: dx lies partly over an input");
    MGGB_REQUIRE(n == 0 || !dw || !(runs_meet(dw, n_dw, dy, n_y) || runs_meet(dw, n_dw, x, n_x) || (dx && runs_meet(dw, n_dw, dx, n_x))),
                 "grouped_dense_backward: dw lies partly over dy, x or dx");
    const auto run = dtype == MGGB_F32 ? grouped_backward_f32 : dtype == MGGB_BF16 ? grouped_backward_bf16 : grouped_backward_f16;
    return run(dx, dw, dy, x, w, group_ptr, groups, n, dim1, dim2, scratch, (cudaStream_t)stream);
}

}  // extern "C"
