// Dense products grouped by node type: rows group_ptr[g] .. group_ptr[g+1]-1 of x go through w[g] (dim1 x dim2).
//     out = x w[g]        dx = dy w[g]^T        dw[g] = x_g^T dy_g
// The sizes of the groups are read on the device; row positions are clamped to [0, n] and made non-decreasing, so that
// no group_ptr makes a kernel touch a row outside the matrices or two groups write one row.
// Stands beside dense_beg_new_forward (include/gnn_layer.cuh:42-46), whose weight is one for all nodes.
#include <algorithm>
#include "elem.h"

namespace {

using mggb::from_f32;
using mggb::to_f32;

constexpr int GT = 32;                 // tile edge

// First row of group g, clamped and made monotone by a running maximum over what came before.
struct GroupWalk {
    const int32_t* ptr;
    long long n;
    int first;
    __device__ GroupWalk(const int32_t* p, long long rows) : ptr(p), n(rows), first(0) { first = clamp(p[0]); }
    __device__ int clamp(int v) const { return (int)max(0LL, min((long long)v, n)); }
    __device__ int next(int g) { return max(first, clamp(ptr[g + 1])); }     // end of group g
};

// out[row, col] = sum_k a(row, k) * w(k, col) for the rows of one tile; TRANS: w(k, col) = w[col][k].
template <typename T, bool TRANS>
__global__ void __launch_bounds__(GT* 8) grouped_rows_kernel(T* __restrict__ out, const T* __restrict__ a, const T* __restrict__ w,
                                                             const int32_t* __restrict__ ptr, int groups, long long n, int K, int N) {
    __shared__ float As[GT][GT + 1], Ws[GT][GT + 1];
    __shared__ int s_g, s_row, s_end;
    if (threadIdx.x == 0) {
        GroupWalk walk(ptr, n);
        long long t = blockIdx.x;
        s_g = -1;
        for (int g = 0; g < groups; g++) {
            const int end = walk.next(g), tiles = (end - walk.first + GT - 1) / GT;
            if (t < tiles) { s_g = g; s_row = walk.first + (int)t * GT; s_end = end; break; }
            t -= tiles;
            walk.first = end;
        }
    }
    __syncthreads();
    if (s_g < 0) return;
    const int row0 = s_row, rows = min(GT, s_end - row0), col0 = blockIdx.y * GT;
    const T* wg = w + (long long)s_g * K * N;
    const int tx = threadIdx.x % GT, ty = threadIdx.x / GT;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < K; k0 += GT) {
        for (int i = ty; i < GT; i += 8) {
            As[i][tx] = (i < rows && k0 + tx < K) ? to_f32(a[(long long)(row0 + i) * K + k0 + tx]) : 0.f;
            if (TRANS) Ws[tx][i] = (col0 + i < N && k0 + tx < K) ? to_f32(wg[(long long)(col0 + i) * K + k0 + tx]) : 0.f;
            else       Ws[i][tx] = (k0 + i < K && col0 + tx < N) ? to_f32(wg[(long long)(k0 + i) * N + col0 + tx]) : 0.f;
        }
        __syncthreads();
        for (int k = 0; k < GT; k++)
            for (int j = 0; j < 4; j++) acc[j] += As[ty + 8 * j][k] * Ws[k][tx];
        __syncthreads();
    }
    for (int j = 0; j < 4; j++)
        if (ty + 8 * j < rows && col0 + tx < N) out[(long long)(row0 + ty + 8 * j) * N + col0 + tx] = from_f32<T>(acc[j]);
}

template <typename T>
__global__ void __launch_bounds__(GT* 8) grouped_dw_kernel(float* __restrict__ dw, const T* __restrict__ x, const T* __restrict__ dy,
                                                           const int32_t* __restrict__ ptr, long long n, int K, int N) {
    __shared__ float Xs[GT][GT + 1], Ds[GT][GT + 1];
    __shared__ int s_row, s_end;
    const int g = blockIdx.z, k0 = blockIdx.y * GT, n0 = blockIdx.x * GT;
    if (threadIdx.x == 0) {
        GroupWalk walk(ptr, n);
        for (int i = 0; i < g; i++) walk.first = walk.next(i);
        s_row = walk.first;
        s_end = walk.next(g);
    }
    __syncthreads();
    const int tx = threadIdx.x % GT, ty = threadIdx.x / GT;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int r0 = s_row; r0 < s_end; r0 += GT) {
        for (int i = ty; i < GT; i += 8) {
            const bool ok = r0 + i < s_end;
            Xs[i][tx] = (ok && k0 + tx < K) ? to_f32(x[(long long)(r0 + i) * K + k0 + tx]) : 0.f;
            Ds[i][tx] = (ok && n0 + tx < N) ? to_f32(dy[(long long)(r0 + i) * N + n0 + tx]) : 0.f;
        }
        __syncthreads();
        for (int r = 0; r < GT; r++)
            for (int j = 0; j < 4; j++) acc[j] += Xs[r][ty + 8 * j] * Ds[r][tx];
        __syncthreads();
    }
    for (int j = 0; j < 4; j++)
        if (k0 + ty + 8 * j < K && n0 + tx < N) dw[((long long)g * K + k0 + ty + 8 * j) * N + n0 + tx] = acc[j];
}

template <typename T>
int forward(void* out, const void* x, const void* w, const int32_t* ptr, int groups, long long n, int K, int N, cudaStream_t st) {
    const dim3 grid((unsigned)(n / GT + groups), (N + GT - 1) / GT);
    grouped_rows_kernel<T, false><<<grid, GT * 8, 0, st>>>((T*)out, (const T*)x, (const T*)w, ptr, groups, n, K, N);
    MGGB_CUDA(cudaGetLastError());
    return MGGB_OK;
}

template <typename T>
int backward(void* dx, float* dw, const void* dy, const void* x, const void* w, const int32_t* ptr, int groups, long long n, int K, int N, cudaStream_t st) {
    if (dx && n > 0) {
        const dim3 grid((unsigned)(n / GT + groups), (K + GT - 1) / GT);
        grouped_rows_kernel<T, true><<<grid, GT * 8, 0, st>>>((T*)dx, (const T*)dy, (const T*)w, ptr, groups, n, N, K);
        MGGB_CUDA(cudaGetLastError());
    }
    if (dw) {
        const dim3 grid((N + GT - 1) / GT, (K + GT - 1) / GT, groups);
        grouped_dw_kernel<T><<<grid, GT * 8, 0, st>>>(dw, (const T*)x, (const T*)dy, ptr, n, K, N);
        MGGB_CUDA(cudaGetLastError());
    }
    return MGGB_OK;
}

int check_sizes(const char* who, int groups, long long n, int K, int N) {
    MGGB_REQUIRE(n >= 0 && K >= 1 && N >= 1, "%s: need n >= 0, dim1 >= 1, dim2 >= 1 (n=%lld dim1=%d dim2=%d)", who, n, K, N);
    MGGB_REQUIRE(n <= 0x7FFFFFFFLL, "%s: row positions are int32: n=%lld is too large", who, n);
    MGGB_REQUIRE(groups >= 1, "%s: need groups >= 1, got %d", who, groups);
    if (groups > MGGB_MAX_GROUPS || K > MGGB_MAX_GROUPED_DIM || N > MGGB_MAX_GROUPED_DIM)
        return mggb::fail(MGGB_ERR_UNSUPPORTED, "%s: at most %d groups and dimensions of at most %d (groups=%d dim1=%d dim2=%d)", who, MGGB_MAX_GROUPS,
                          MGGB_MAX_GROUPED_DIM, groups, K, N);
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
    return MGGB_BY_DTYPE(dtype, forward, out, x, w, group_ptr, groups, n, dim1, dim2, (cudaStream_t)stream);
}

int mggb_grouped_dense_backward_scratch_bytes(int64_t n, int groups, int dim1, int dim2, int dtype, size_t* bytes) {
    MGGB_REQUIRE(bytes, "grouped_dense_backward_scratch_bytes: NULL output");
    MGGB_REQUIRE_DTYPE(dtype, "grouped_dense_backward_scratch_bytes");
    const int rc = check_sizes("grouped_dense_backward_scratch_bytes", groups, n, dim1, dim2);
    if (rc != MGGB_OK) return rc;
    *bytes = 0;
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
    size_t need = 0;
    rc = mggb_grouped_dense_backward_scratch_bytes(n, groups, dim1, dim2, dtype, &need);
    if (rc != MGGB_OK) return rc;
    MGGB_REQUIRE(!dw || need == 0 || (scratch && scratch_bytes >= need), "grouped_dense_backward: scratch of %zu bytes needed, %zu given", need, scratch ? scratch_bytes : (size_t)0);
    return MGGB_BY_DTYPE(dtype, backward, dx, dw, dy, x, w, group_ptr, groups, n, dim1, dim2, (cudaStream_t)stream);
}

}  // extern "C"
