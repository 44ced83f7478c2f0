// Layer norm over the features of each row, forward and backward.
//     mean = sum(x) / D,  rstd = 1 / sqrt(sum((x - mean)^2) / D + eps),  xhat = (x - mean) * rstd,  y = xhat * w + b
//     g = dy * w;  dx = rstd * (g - mean(g) - xhat * mean(g * xhat));  dw = sum over rows of dy * xhat;  db = sum of dy
// No counterpart in the reference, whose models have no normalisation between layers.
#include <algorithm>
#include "elem.h"

namespace {

using mggb::from_f32;
using mggb::to_f32;

constexpr int LN_THREADS = 128;

// Sum of v over the block; every thread gets it.
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = mggb::warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.f;
    for (int i = 0; i < LN_THREADS / 32; i++) s += red[i];
    return s;
}

template <typename T>
__global__ void __launch_bounds__(LN_THREADS) ln_forward_kernel(T* __restrict__ out, const T* __restrict__ x, const float* __restrict__ w,
                                                                const float* __restrict__ b, float eps, float* __restrict__ mean_out,
                                                                float* __restrict__ rstd_out, long long n, int D, long long ld_out, long long ld_x) {
    __shared__ float red[LN_THREADS / 32];
    for (long long row = blockIdx.x; row < n; row += gridDim.x) {
        const T* xr = x + row * ld_x;
        float s = 0.f;
        for (int c = threadIdx.x; c < D; c += LN_THREADS) s += to_f32(xr[c]);
        const float mean = block_sum(s, red) / D;
        float q = 0.f;
        for (int c = threadIdx.x; c < D; c += LN_THREADS) { const float d = to_f32(xr[c]) - mean; q += d * d; }
        const float rstd = 1.f / sqrtf(block_sum(q, red) / D + eps);
        for (int c = threadIdx.x; c < D; c += LN_THREADS) {
            float v = (to_f32(xr[c]) - mean) * rstd;
            if (w) v *= w[c];
            if (b) v += b[c];
            out[row * ld_out + c] = from_f32<T>(v);
        }
        if (threadIdx.x == 0) {
            if (mean_out) mean_out[row] = mean;
            if (rstd_out) rstd_out[row] = rstd;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(LN_THREADS) ln_dx_kernel(T* __restrict__ dx, const T* __restrict__ dy, const T* __restrict__ x,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd,
                                                           const float* __restrict__ w, long long n, int D, long long ld_dx, long long ld_dy, long long ld_x) {
    __shared__ float red[LN_THREADS / 32];
    for (long long row = blockIdx.x; row < n; row += gridDim.x) {
        const T *xr = x + row * ld_x, *gr = dy + row * ld_dy;
        const float mu = mean[row], r = rstd[row];
        float a = 0.f, c1 = 0.f;
        for (int c = threadIdx.x; c < D; c += LN_THREADS) {
            const float g = to_f32(gr[c]) * (w ? w[c] : 1.f);
            a += g;
            c1 += g * ((to_f32(xr[c]) - mu) * r);
        }
        a = block_sum(a, red) / D;
        c1 = block_sum(c1, red) / D;
        for (int c = threadIdx.x; c < D; c += LN_THREADS) {
            const float g = to_f32(gr[c]) * (w ? w[c] : 1.f);
            dx[row * ld_dx + c] = from_f32<T>(r * (g - a - (to_f32(xr[c]) - mu) * r * c1));
        }
    }
}

// Partial sums of one range of rows for 128 columns: part[split][0] = dw, part[split][1] = db.
template <typename T>
__global__ void __launch_bounds__(LN_THREADS) ln_dw_partial_kernel(float* __restrict__ part, const T* __restrict__ dy, const T* __restrict__ x,
                                                                   const float* __restrict__ mean, const float* __restrict__ rstd, long long n, int D,
                                                                   long long ld_dy, long long ld_x) {
    const int c = blockIdx.x * LN_THREADS + threadIdx.x;
    if (c >= D) return;
    const long long step = (n + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * step, r1 = min(n, r0 + step);
    float dw = 0.f, db = 0.f;
    for (long long row = r0; row < r1; row++) {
        const float g = to_f32(dy[row * ld_dy + c]);
        dw += g * ((to_f32(x[row * ld_x + c]) - mean[row]) * rstd[row]);
        db += g;
    }
    part[((long long)blockIdx.y * 2) * D + c] = dw;
    part[((long long)blockIdx.y * 2 + 1) * D + c] = db;
}

__global__ void ln_dw_reduce_kernel(float* __restrict__ dw, float* __restrict__ db, const float* __restrict__ part, int splits, int D) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= D) return;
    float a = 0.f, b = 0.f;
    for (int s = 0; s < splits; s++) {
        a += part[((long long)s * 2) * D + c];
        b += part[((long long)s * 2 + 1) * D + c];
    }
    if (dw) dw[c] = a;
    if (db) db[c] = b;
}

// Row ranges the weight's gradient is split into.
int ln_splits(long long n) { return (int)std::max<long long>(1, std::min<long long>(2LL * mggb::sm_count(), n / 16)); }

int row_grid(long long n) { return (int)std::min<long long>(n, 16LL * mggb::sm_count()); }

template <typename T>
int forward(void* out, const void* x, const float* w, const float* b, float eps, float* mean, float* rstd, long long n, int D,
            long long ld_out, long long ld_x, cudaStream_t st) {
    ln_forward_kernel<T><<<row_grid(n), LN_THREADS, 0, st>>>((T*)out, (const T*)x, w, b, eps, mean, rstd, n, D, ld_out, ld_x);
    MGGB_CUDA(cudaGetLastError());
    return MGGB_OK;
}

template <typename T>
int backward(void* dx, float* dw, float* db, const void* dy, const void* x, const float* mean, const float* rstd, const float* w,
             long long n, int D, long long ld_dx, long long ld_dy, long long ld_x, float* part, cudaStream_t st) {
    if (dw || db) {
        const int splits = ln_splits(n);
        const dim3 grid((D + LN_THREADS - 1) / LN_THREADS, splits);
        ln_dw_partial_kernel<T><<<grid, LN_THREADS, 0, st>>>(part, (const T*)dy, (const T*)x, mean, rstd, n, D, ld_dy, ld_x);
        MGGB_CUDA(cudaGetLastError());
        ln_dw_reduce_kernel<<<(D + 127) / 128, 128, 0, st>>>(dw, db, part, splits, D);
        MGGB_CUDA(cudaGetLastError());
    }
    if (n > 0 && dx) {
        ln_dx_kernel<T><<<row_grid(n), LN_THREADS, 0, st>>>((T*)dx, (const T*)dy, (const T*)x, mean, rstd, w, n, D, ld_dx, ld_dy, ld_x);
        MGGB_CUDA(cudaGetLastError());
    }
    return MGGB_OK;
}

}  // namespace

extern "C" {

int mggb_layer_norm_forward(void* out, const void* x, const float* weight, const float* bias, float eps, float* mean, float* rstd,
                            int64_t n, int dim, int64_t ld_out, int64_t ld_x, int dtype, void* stream) {
    MGGB_REQUIRE(n >= 0 && dim >= 1, "layer_norm_forward: need n >= 0, dim >= 1 (n=%lld dim=%d)", (long long)n, dim);
    MGGB_REQUIRE_DTYPE(dtype, "layer_norm_forward");
    MGGB_REQUIRE(eps >= 0.f, "layer_norm_forward: eps must not be negative or NaN");
    MGGB_REQUIRE(ld_out >= dim && ld_x >= dim, "layer_norm_forward: row strides must be at least dim");
    if (n == 0) return MGGB_OK;
    MGGB_REQUIRE(out && x, "layer_norm_forward: NULL argument");
    MGGB_REQUIRE(out != x || ld_out == ld_x, "layer_norm_forward: in place needs equal row strides");
    return MGGB_BY_DTYPE(dtype, forward, out, x, weight, bias, eps, mean, rstd, n, dim, ld_out, ld_x, (cudaStream_t)stream);
}

int mggb_layer_norm_backward_scratch_bytes(int64_t n, int dim, size_t* bytes) {
    MGGB_REQUIRE(bytes, "layer_norm_backward_scratch_bytes: NULL output");
    MGGB_REQUIRE(n >= 0 && dim >= 1, "layer_norm_backward_scratch_bytes: need n >= 0, dim >= 1 (n=%lld dim=%d)", (long long)n, dim);
    *bytes = (size_t)ln_splits(n) * 2 * dim * sizeof(float);
    return MGGB_OK;
}

int mggb_layer_norm_backward(void* dx, float* dweight, float* dbias, const void* dy, const void* x, const float* mean, const float* rstd,
                             const float* weight, int64_t n, int dim, int64_t ld_dx, int64_t ld_dy, int64_t ld_x, int dtype,
                             void* scratch, size_t scratch_bytes, void* stream) {
    MGGB_REQUIRE(n >= 0 && dim >= 1, "layer_norm_backward: need n >= 0, dim >= 1 (n=%lld dim=%d)", (long long)n, dim);
    MGGB_REQUIRE_DTYPE(dtype, "layer_norm_backward");
    MGGB_REQUIRE(ld_dx >= dim && ld_dy >= dim && ld_x >= dim, "layer_norm_backward: row strides must be at least dim");
    MGGB_REQUIRE(n == 0 || (dy && x && mean && rstd), "layer_norm_backward: NULL argument");
    MGGB_REQUIRE(n == 0 || dx || dweight || dbias, "layer_norm_backward: no output given");
    MGGB_REQUIRE(n == 0 || !dx || ((dx != dy || ld_dx == ld_dy) && (dx != x || ld_dx == ld_x)), "layer_norm_backward: in place needs equal row strides");
    if (dweight || dbias) {
        size_t need = 0;
        const int rc = mggb_layer_norm_backward_scratch_bytes(n, dim, &need);
        if (rc != MGGB_OK) return rc;
        MGGB_REQUIRE(scratch && scratch_bytes >= need, "layer_norm_backward: scratch of %zu bytes needed, %zu given", need, scratch ? scratch_bytes : (size_t)0);
        MGGB_REQUIRE((uintptr_t)scratch % 16 == 0, "layer_norm_backward: scratch must be 16-byte aligned");
    }
    return MGGB_BY_DTYPE(dtype, backward, dx, dweight, dbias, dy, x, mean, rstd, weight, n, dim, ld_dx, ld_dy, ld_x, (float*)scratch, (cudaStream_t)stream);
}

}  // extern "C"
