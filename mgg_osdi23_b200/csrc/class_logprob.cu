// Log probabilities of given classes, with the distribution's entropy and its most likely classes, and their gradient.
//     m = max_c z_c,  S = sum_c e^(z_c - m),  L = log S
//     logprob = (z_y - m) - L            H = L - sum_c e^(z_c - m) (z_c - m) / S
//     dz_c = dlogprob * (1[c = y] - p_c) - dH * p_c * (log p_c + H),   log p_c = (z_c - m) - L
// The row's statistics are kept as the pair (m, L), not as m + L: with large scores the sum would lose the low bits of L
// and every probability of the backward pass with them.
// Stands beside softmax_new_forward (include/gnn_layer.cuh:36-40); no counterpart in the reference.
#include <algorithm>
#include <cfloat>
#include "elem.h"

namespace {

using mggb::from_f32;
using mggb::to_f32;

constexpr int LP_THREADS = 128;

// Order of the values as integers: larger value = larger key, NaN above everything, -0 == +0.
__device__ __forceinline__ int order_key(float v) {
    if (v != v) return 0x7F800001;      // the next key above infinity's
    const int b = __float_as_int(v + 0.f);
    return b ^ ((b >> 31) & 0x7FFFFFFF);
}

// (key, class): larger key first, then smaller class.
__device__ __forceinline__ unsigned long long rank_of(int key, int c) {
    return ((unsigned long long)((unsigned)key ^ 0x80000000u) << 32) | (0xFFFFFFFFu - (unsigned)c);
}

struct LogprobOut {
    float *logprob, *stats, *entropy;
    int32_t* top_ids;
    float* top_logprobs;
    int top;
};

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) logprob_forward_kernel(const LogprobOut o, const T* __restrict__ z, long long ld,
                                                                     const int32_t* __restrict__ labels, long long n, int C) {
    __shared__ float red[2][LP_THREADS / 32];
    __shared__ unsigned long long best[LP_THREADS / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (long long row = blockIdx.x; row < n; row += gridDim.x) {
        const T* zr = z + row * ld;
        // fmaxf drops NaN operands: a NaN comes back through the sums below
        float m = -INFINITY;
        for (int c = threadIdx.x; c < C; c += LP_THREADS) m = fmaxf(m, to_f32(zr[c]));
        for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
        __syncthreads();
        if (lane == 0) red[0][warp] = m;
        __syncthreads();
        for (int i = 0; i < LP_THREADS / 32; i++) m = fmaxf(m, red[0][i]);
        float s = 0.f, t = 0.f;
        for (int c = threadIdx.x; c < C; c += LP_THREADS) {
            const float v = to_f32(zr[c]);
            const float d = v == -INFINITY ? -INFINITY : v - m;
            const float e = expf(d);
            s += e;
            if (!(e <= 0.f)) t += e * d;
        }
        s = mggb::warp_sum(s);
        t = mggb::warp_sum(t);
        __syncthreads();
        if (lane == 0) { red[0][warp] = s; red[1][warp] = t; }
        __syncthreads();
        s = t = 0.f;
        for (int i = 0; i < LP_THREADS / 32; i++) { s += red[0][i]; t += red[1][i]; }
        // a row that is masked out as a whole (all -inf): no class has a probability, entropy 0
        const bool nothing = m == -INFINITY && s == 0.f;
        const float L = nothing ? 0.f : logf(s);
        if (threadIdx.x == 0) {
            if (o.logprob) {
                const int y = labels[row];
                float lp = 0.f;
                if (y >= 0 && y < C) lp = nothing ? -INFINITY : (to_f32(zr[y]) - m) - L;
                o.logprob[row] = lp;
            }
            if (o.stats) { o.stats[2 * row] = m; o.stats[2 * row + 1] = L; }
            if (o.entropy) o.entropy[row] = nothing ? 0.f : L - t / s;
        }
        unsigned long long last = ~0ull;
        for (int k = 0; k < o.top; k++) {
            unsigned long long b = 0;
            for (int c = threadIdx.x; c < C; c += LP_THREADS) {
                const unsigned long long r = rank_of(order_key(to_f32(zr[c])), c);
                if (r < last && r > b) b = r;
            }
            for (int off = 16; off; off >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, off));
            __syncthreads();
            if (lane == 0) best[warp] = b;
            __syncthreads();
            for (int i = 0; i < LP_THREADS / 32; i++) b = max(b, best[i]);
            last = b;
            if (threadIdx.x == 0) {
                const int c = (int)(0xFFFFFFFFu - (unsigned)b);
                o.top_ids[row * o.top + k] = c;
                if (o.top_logprobs) o.top_logprobs[row * o.top + k] = nothing ? -INFINITY : (to_f32(zr[c]) - m) - L;
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) logprob_backward_kernel(T* dz, const T* z, long long ld_dz, long long ld_z,
                                                                      const int32_t* __restrict__ labels, const float* __restrict__ stats,
                                                                      const float* __restrict__ dlogprob, const float* __restrict__ entropy,
                                                                      const float* __restrict__ dentropy, long long n, int C) {
    for (long long row = blockIdx.x; row < n; row += gridDim.x) {
        const float m = stats[2 * row], L = stats[2 * row + 1];
        const int y = labels ? labels[row] : -1;
        const float up = (y >= 0 && y < C && dlogprob) ? dlogprob[row] : 0.f;
        const float H = dentropy ? entropy[row] : 0.f, dH = dentropy ? dentropy[row] : 0.f;
        for (int c = threadIdx.x; c < C; c += LP_THREADS) {
            const float v = to_f32(z[row * ld_z + c]);
            const float lp = (v - m) - L;
            const float p = expf(lp);
            float g = -up * p;
            if (c == y) g += up;
            if (dH != 0.f && !(p <= 0.f)) g -= dH * p * (lp + H);
            if (m == -INFINITY && L == 0.f) g = 0.f;      // a row that is masked out as a whole
            dz[row * ld_dz + c] = from_f32<T>(g);
        }
    }
}

int row_grid(long long n) { return (int)std::min<long long>(n, 16LL * mggb::sm_count()); }

template <typename T>
int forward(const LogprobOut& o, const void* z, long long ld, const int32_t* labels, long long n, int C, cudaStream_t st) {
    logprob_forward_kernel<T><<<row_grid(n), LP_THREADS, 0, st>>>(o, (const T*)z, ld, labels, n, C);
    MGGB_CUDA(cudaGetLastError());
    return MGGB_OK;
}

template <typename T>
int backward(void* dz, const void* z, long long ld_dz, long long ld_z, const int32_t* labels, const float* stats, const float* dlp,
             const float* H, const float* dH, long long n, int C, cudaStream_t st) {
    logprob_backward_kernel<T><<<row_grid(n), LP_THREADS, 0, st>>>((T*)dz, (const T*)z, ld_dz, ld_z, labels, stats, dlp, H, dH, n, C);
    MGGB_CUDA(cudaGetLastError());
    return MGGB_OK;
}

}  // namespace

extern "C" {

int mggb_class_logprob_forward(float* logprob, float* stats, float* entropy, int32_t* top_ids, float* top_logprobs, int top,
                               const void* logits, int64_t ld_logits, const int32_t* labels, int64_t n, int classes, int dtype, void* stream) {
    MGGB_REQUIRE(n >= 0 && classes >= 1, "class_logprob_forward: need n >= 0, classes >= 1 (n=%lld classes=%d)", (long long)n, classes);
    MGGB_REQUIRE_DTYPE(dtype, "class_logprob_forward");
    MGGB_REQUIRE(ld_logits >= classes, "class_logprob_forward: the row stride must be at least classes");
    MGGB_REQUIRE(top >= 0 && top <= MGGB_MAX_TOP && top <= classes, "class_logprob_forward: top must be 0..min(%d, classes), got %d", MGGB_MAX_TOP, top);
    if (n == 0) return MGGB_OK;
    MGGB_REQUIRE(logits, "class_logprob_forward: NULL logits");
    MGGB_REQUIRE((logprob == nullptr) == (labels == nullptr), "class_logprob_forward: logprob and labels go together");
    MGGB_REQUIRE(top == 0 || top_ids, "class_logprob_forward: top > 0 needs top_ids");
    MGGB_REQUIRE(logprob || stats || entropy || top > 0, "class_logprob_forward: no output given");
    const LogprobOut o{logprob, stats, entropy, top_ids, top_logprobs, top};
    return MGGB_BY_DTYPE(dtype, forward, o, logits, ld_logits, labels, n, classes, (cudaStream_t)stream);
}

int mggb_class_logprob_backward(void* dlogits, const void* logits, int64_t ld_dlogits, int64_t ld_logits, const int32_t* labels,
                                const float* stats, const float* dlogprob, const float* entropy, const float* dentropy,
                                int64_t n, int classes, int dtype, void* stream) {
    MGGB_REQUIRE(n >= 0 && classes >= 1, "class_logprob_backward: need n >= 0, classes >= 1 (n=%lld classes=%d)", (long long)n, classes);
    MGGB_REQUIRE_DTYPE(dtype, "class_logprob_backward");
    MGGB_REQUIRE(ld_logits >= classes && ld_dlogits >= classes, "class_logprob_backward: row strides must be at least classes");
    if (n == 0) return MGGB_OK;
    MGGB_REQUIRE(dlogits && logits && stats, "class_logprob_backward: NULL argument");
    MGGB_REQUIRE((dlogprob == nullptr) == (labels == nullptr), "class_logprob_backward: dlogprob and labels go together");
    MGGB_REQUIRE((dentropy == nullptr) || entropy, "class_logprob_backward: dentropy needs the forward pass's entropy");
    MGGB_REQUIRE(dlogprob || dentropy, "class_logprob_backward: no gradient given");
    MGGB_REQUIRE(dlogits != logits || ld_dlogits == ld_logits, "class_logprob_backward: in place needs equal row strides");
    return MGGB_BY_DTYPE(dtype, backward, dlogits, logits, ld_dlogits, ld_logits, labels, stats, dlogprob, entropy, dentropy, n, classes, (cudaStream_t)stream);
}

}  // extern "C"
