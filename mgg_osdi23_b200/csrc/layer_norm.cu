// Layer norm over the features of each row, forward and backward.
//     mean = sum(x) / D,  rstd = 1 / sqrt(sum((x - mean)^2) / D + eps),  xhat = (x - mean) * rstd,  y = xhat * w + b
//     g = dy * w;  dx = rstd * (g - mean(g) - xhat * mean(g * xhat));  dw = sum over rows of dy * xhat;  db = sum of dy
// No counterpart in the reference, whose models have no normalisation between layers.
//
// Bound by HBM: the forward pass has to read and write each element once, the backward pass to read two and write one.
// A row therefore stays in registers between its reductions and its result, in the vectors it was loaded as, and the
// gradients of weight and bias are summed in registers by threads that keep the same columns for every row they take.
// Two shapes of the same code:
//   rows up to 128 vectors   1 to 32 lanes of a warp per row, up to 4 vectors per lane; reductions by shuffles only.
//                            Several narrow rows share a warp: a lane always has 4 loads in flight.
//   wider rows               one block per row, 1 to 8 vectors per thread; reductions through shared memory.
// Rows too wide for that (above 8192 vectors) are read again for every pass over them (from L2).
#include <algorithm>
#include "elem.h"

namespace {

using mggb::from_f32;
using mggb::Pack;
using mggb::to_f32;

constexpr int ROW_THREADS = 256;    // block of the kernels that put several rows in a warp or block
constexpr int MAX_TPR = 1024;       // threads per row of the block-per-row kernels
constexpr int MAX_TPR_BWD = 512;    // of the backward pass: 16 elements a thread with their sums want up to 128 registers

// Sum over the lanes of a group of lpr (a power of two) neighbouring lanes; every lane gets it.
__device__ __forceinline__ float group_sum(float v, int lpr) {
    for (int off = lpr >> 1; off; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// Sums over the block.  Consecutive calls alternate between two rows of `red`, so one barrier each is enough.
struct BlockSum {
    float (*red)[2][32];
    int turn;
    __device__ __forceinline__ float2 operator()(float a, float b) {
        const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        a = mggb::warp_sum(a);
        b = mggb::warp_sum(b);
        if (lane == 0) { red[turn][0][warp] = a; red[turn][1][warp] = b; }
        __syncthreads();
        a = mggb::warp_sum(lane < warps ? red[turn][0][lane] : 0.f);
        b = mggb::warp_sum(lane < warps ? red[turn][1][lane] : 0.f);
        turn ^= 1;
        return make_float2(a, b);
    }
    __device__ __forceinline__ float operator()(float a) {
        const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        a = mggb::warp_sum(a);
        if (lane == 0) red[turn][0][warp] = a;
        __syncthreads();
        a = mggb::warp_sum(lane < warps ? red[turn][0][lane] : 0.f);
        turn ^= 1;
        return a;
    }
};

// VE consecutive floats of a parameter vector; 16-byte loads when the caller's pointers allow it.
template <int VE>
__device__ __forceinline__ void load_params(float (&v)[VE], const float* __restrict__ p, int vec_ok) {
    if (VE % 4 == 0 && vec_ok) {
#pragma unroll
        for (int i = 0; i < VE / 4; i++) *reinterpret_cast<float4*>(&v[4 * i]) = __ldg(reinterpret_cast<const float4*>(p) + i);
    } else if (VE == 2 && vec_ok) {
        *reinterpret_cast<float2*>(&v[0]) = __ldg(reinterpret_cast<const float2*>(p));
    } else {
#pragma unroll
        for (int i = 0; i < VE; i++) v[i] = __ldg(p + i);
    }
}

struct FwdArgs {
    void* out;
    const void* x;
    const float *w, *b;
    float eps;
    float *mean, *rstd;
    long long n, ld_out, ld_x;
    int D, nvec, lpr, param_vec;
};

template <typename T, int VB, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? MAX_TPR : ROW_THREADS) ln_forward_kernel(const FwdArgs A) {
    constexpr int VE = Pack<T, VB>::VE;
    constexpr int U = BLOCK || NV > 4 ? 1 : 4 / NV;       // rows a group of lanes has in flight
    __shared__ float red[2][2][32];
    BlockSum block_sum{red, 0};
    const int tpr = BLOCK ? blockDim.x : A.lpr;
    const int l = BLOCK ? threadIdx.x : threadIdx.x & (A.lpr - 1);
    const int groups = BLOCK ? 1 : ROW_THREADS / A.lpr, group = BLOCK ? 0 : threadIdx.x / A.lpr;
    const float D = (float)A.D;
    for (long long row0 = (long long)blockIdx.x * groups * U; row0 < A.n; row0 += (long long)gridDim.x * groups * U) {
        Pack<T, VB> v[U][NV];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long row = row0 + u * groups + group;
            const T* xr = (const T*)A.x + row * A.ld_x;
#pragma unroll
            for (int j = 0; j < NV; j++)
                if (row < A.n && l + j * tpr < A.nvec) v[u][j].load(xr + (l + j * tpr) * VE);
        }
        float mean[U], rstd[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < NV; j++)
#pragma unroll
                for (int i = 0; i < VE; i++) s += v[u][j].get(i);
            mean[u] = (BLOCK ? block_sum(s) : group_sum(s, A.lpr)) / D;
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            float q = 0.f;
#pragma unroll
            for (int j = 0; j < NV; j++)
                if (l + j * tpr < A.nvec) {
#pragma unroll
                    for (int i = 0; i < VE; i++) { const float d = v[u][j].get(i) - mean[u]; q += d * d; }
                }
            rstd[u] = 1.f / sqrtf((BLOCK ? block_sum(q) : group_sum(q, A.lpr)) / D + A.eps);
        }
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = (l + j * tpr) * VE;
            if (l + j * tpr >= A.nvec) continue;
            float w[VE], b[VE];
            if (A.w) load_params<VE>(w, A.w + c, A.param_vec);
            if (A.b) load_params<VE>(b, A.b + c, A.param_vec);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const long long row = row0 + u * groups + group;
                if (row >= A.n) continue;
#pragma unroll
                for (int i = 0; i < VE; i++) {
                    float y = (v[u][j].get(i) - mean[u]) * rstd[u];
                    if (A.w) y *= w[i];
                    if (A.b) y += b[i];
                    v[u][j].set(i, y);
                }
                v[u][j].store((T*)A.out + row * A.ld_out + c);
            }
        }
        if (l == 0) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const long long row = row0 + u * groups + group;
                if (row < A.n && A.mean) A.mean[row] = mean[u];
                if (row < A.n && A.rstd) A.rstd[row] = rstd[u];
            }
        }
    }
}

// Rows of more vectors than a block keeps in registers.
template <typename T>
__global__ void __launch_bounds__(MAX_TPR) ln_forward_wide_kernel(const FwdArgs A) {
    __shared__ float red[2][2][32];
    BlockSum block_sum{red, 0};
    for (long long row = blockIdx.x; row < A.n; row += gridDim.x) {
        const T* xr = (const T*)A.x + row * A.ld_x;
        float s = 0.f;
        for (int c = threadIdx.x; c < A.D; c += blockDim.x) s += to_f32(xr[c]);
        const float mean = block_sum(s) / (float)A.D;
        float q = 0.f;
        for (int c = threadIdx.x; c < A.D; c += blockDim.x) { const float d = to_f32(xr[c]) - mean; q += d * d; }
        const float rstd = 1.f / sqrtf(block_sum(q) / (float)A.D + A.eps);
        for (int c = threadIdx.x; c < A.D; c += blockDim.x) {
            float y = (to_f32(xr[c]) - mean) * rstd;
            if (A.w) y *= __ldg(A.w + c);
            if (A.b) y += __ldg(A.b + c);
            ((T*)A.out)[row * A.ld_out + c] = from_f32<T>(y);
        }
        if (threadIdx.x == 0) {
            if (A.mean) A.mean[row] = mean;
            if (A.rstd) A.rstd[row] = rstd;
        }
    }
}

struct BwdArgs {
    void* dx;
    const void *dy, *x;
    const float *mean, *rstd, *w;
    float* part;                     // [blocks][2][D]: the blocks' sums of dy * xhat and dy; NULL when not wanted
    long long n, ld_dx, ld_dy, ld_x;
    int D, nvec, lpr, param_vec;
};

template <typename T, int VB, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? MAX_TPR_BWD : ROW_THREADS, BLOCK ? 1 : 2) ln_backward_kernel(const BwdArgs A) {
    constexpr int VE = Pack<T, VB>::VE;
    constexpr int U = BLOCK || NV * VE > 8 ? 1 : (NV * VE > 4 ? 2 : 4);
    extern __shared__ float sums[];                       // [2][D] (lane-group kernels only)
    __shared__ float red[2][2][32];
    BlockSum block_sum{red, 0};
    const int tpr = BLOCK ? blockDim.x : A.lpr;
    const int l = BLOCK ? threadIdx.x : threadIdx.x & (A.lpr - 1);
    const int groups = BLOCK ? 1 : ROW_THREADS / A.lpr, group = BLOCK ? 0 : threadIdx.x / A.lpr;
    const float D = (float)A.D;
    float aw[NV][VE], ab[NV][VE];
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int i = 0; i < VE; i++) aw[j][i] = ab[j][i] = 0.f;
    for (long long row0 = (long long)blockIdx.x * groups * U; row0 < A.n; row0 += (long long)gridDim.x * groups * U) {
        Pack<T, VB> x[U][NV], g[U][NV];
        float mean[U], rstd[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long row = row0 + u * groups + group;
            const T *xr = (const T*)A.x + row * A.ld_x, *gr = (const T*)A.dy + row * A.ld_dy;
#pragma unroll
            for (int j = 0; j < NV; j++)
                if (row < A.n && l + j * tpr < A.nvec) {
                    x[u][j].load(xr + (l + j * tpr) * VE);
                    g[u][j].load(gr + (l + j * tpr) * VE);
                }
            mean[u] = row < A.n ? __ldg(A.mean + row) : 0.f;
            rstd[u] = row < A.n ? __ldg(A.rstd + row) : 0.f;
        }
        float a[U], c[U];
#pragma unroll
        for (int u = 0; u < U; u++) a[u] = c[u] = 0.f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (l + j * tpr >= A.nvec) continue;
            float w[VE];
            if (A.w) load_params<VE>(w, A.w + (l + j * tpr) * VE, A.param_vec);
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < VE; i++) {
                    // a row past the end has dy = 0 and rstd = 0: it adds nothing
                    const float dy = g[u][j].get(i), xhat = (x[u][j].get(i) - mean[u]) * rstd[u];
                    aw[j][i] += dy * xhat;
                    ab[j][i] += dy;
                    const float gi = A.w ? dy * w[i] : dy;
                    a[u] += gi;
                    c[u] += gi * xhat;
                }
        }
        if (!A.dx) continue;
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (BLOCK) {
                const float2 s = block_sum(a[u], c[u]);
                a[u] = s.x / D;
                c[u] = s.y / D;
            } else {
                a[u] = group_sum(a[u], A.lpr) / D;
                c[u] = group_sum(c[u], A.lpr) / D;
            }
        }
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (l + j * tpr >= A.nvec) continue;
            float w[VE];
            if (A.w) load_params<VE>(w, A.w + (l + j * tpr) * VE, A.param_vec);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const long long row = row0 + u * groups + group;
                if (row >= A.n) continue;
#pragma unroll
                for (int i = 0; i < VE; i++) {
                    const float dy = g[u][j].get(i), xhat = (x[u][j].get(i) - mean[u]) * rstd[u];
                    g[u][j].set(i, rstd[u] * ((A.w ? dy * w[i] : dy) - a[u] - xhat * c[u]));
                }
                g[u][j].store((T*)A.dx + row * A.ld_dx + (l + j * tpr) * VE);
            }
        }
    }
    if (!A.part) return;
    float* part = A.part + (long long)blockIdx.x * 2 * A.D;
    if (BLOCK) {
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (l + j * tpr < A.nvec) {
#pragma unroll
                for (int i = 0; i < VE; i++) {
                    part[(l + j * tpr) * VE + i] = aw[j][i];
                    part[A.D + (l + j * tpr) * VE + i] = ab[j][i];
                }
            }
        return;
    }
    // groups of one warp meet by shuffles, warps in shared memory one after the other (a fixed order)
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int i = 0; i < VE; i++)
            for (int off = A.lpr; off < 32; off <<= 1) {
                aw[j][i] += __shfl_xor_sync(0xffffffffu, aw[j][i], off);
                ab[j][i] += __shfl_xor_sync(0xffffffffu, ab[j][i], off);
            }
    for (int wp = 0; wp < ROW_THREADS / 32; wp++) {
        if ((threadIdx.x >> 5) == wp && (threadIdx.x & 31) < A.lpr) {
#pragma unroll
            for (int j = 0; j < NV; j++)
                if (l + j * tpr < A.nvec) {
#pragma unroll
                    for (int i = 0; i < VE; i++) {
                        const int col = (l + j * tpr) * VE + i;
                        sums[col] = (wp ? sums[col] : 0.f) + aw[j][i];
                        sums[A.D + col] = (wp ? sums[A.D + col] : 0.f) + ab[j][i];
                    }
                }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * A.D; i += ROW_THREADS) part[i] = sums[i];
}

// Rows of more vectors than a block keeps in registers: dx row by row, the weight's gradient column by column.
template <typename T>
__global__ void __launch_bounds__(MAX_TPR) ln_dx_wide_kernel(const BwdArgs A) {
    __shared__ float red[2][2][32];
    BlockSum block_sum{red, 0};
    for (long long row = blockIdx.x; row < A.n; row += gridDim.x) {
        const T *xr = (const T*)A.x + row * A.ld_x, *gr = (const T*)A.dy + row * A.ld_dy;
        const float mu = A.mean[row], r = A.rstd[row];
        float a = 0.f, c1 = 0.f;
        for (int c = threadIdx.x; c < A.D; c += blockDim.x) {
            const float g = to_f32(gr[c]) * (A.w ? __ldg(A.w + c) : 1.f);
            a += g;
            c1 += g * ((to_f32(xr[c]) - mu) * r);
        }
        const float2 s = block_sum(a, c1);
        a = s.x / (float)A.D;
        c1 = s.y / (float)A.D;
        for (int c = threadIdx.x; c < A.D; c += blockDim.x) {
            const float g = to_f32(gr[c]) * (A.w ? __ldg(A.w + c) : 1.f);
            ((T*)A.dx)[row * A.ld_dx + c] = from_f32<T>(r * (g - a - (to_f32(xr[c]) - mu) * r * c1));
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(128) ln_dw_wide_kernel(const BwdArgs A) {
    const int c = blockIdx.x * 128 + threadIdx.x;
    if (c >= A.D) return;
    const long long step = (A.n + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * step, r1 = min(A.n, r0 + step);
    float dw = 0.f, db = 0.f;
    for (long long row = r0; row < r1; row++) {
        const float g = to_f32(((const T*)A.dy)[row * A.ld_dy + c]);
        dw += g * ((to_f32(((const T*)A.x)[row * A.ld_x + c]) - A.mean[row]) * A.rstd[row]);
        db += g;
    }
    A.part[((long long)blockIdx.y * 2) * A.D + c] = dw;
    A.part[((long long)blockIdx.y * 2 + 1) * A.D + c] = db;
}

// Column sums of the blocks' partial sums: 32 columns per block, 16 warps take every 16th block, then meet in order.
__global__ void __launch_bounds__(512) ln_dw_reduce_kernel(float* __restrict__ dw, float* __restrict__ db, const float* __restrict__ part,
                                                           int parts, int D) {
    __shared__ float s[16][33];
    const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + lane;
    float a = 0.f;
    if (col < 2 * D)
        for (int p = wp; p < parts; p += 16) a += part[(long long)p * 2 * D + col];
    s[wp][lane] = a;
    __syncthreads();
    if (wp == 0 && col < 2 * D) {
        for (int i = 1; i < 16; i++) a += s[i][lane];
        if (col < D) { if (dw) dw[col] = a; }
        else if (db) db[col - D] = a;
    }
}

// Blocks whose sums of the weight's gradient are kept apart: enough to fill the machine at this width, never more than
// 8192 * 2 * 4 bytes per SM in all.
int ln_parts(long long n, int D) {
    const long long per_sm = std::max(1, std::min(8, 8192 / D));
    return (int)std::max<long long>(1, std::min<long long>(n, per_sm * mggb::sm_count()));
}

int pow2_at_least(int v) {
    int p = 1;
    while (p < v) p <<= 1;
    return p;
}

// How a row of nvec vectors is laid over threads: lanes of a warp or a whole block, and vectors per thread.
struct Layout {
    int lpr, nv, tpr;      // lpr > 0: lanes per row; otherwise tpr threads of a block per row
};

// at_most: vectors per lane or thread.  A lane group is at least 8 lanes wide where the row has that many vectors, so that
// a group's load covers 128 bytes or more.
Layout layout(int nvec, int at_most, int lane_max) {
    if (nvec <= lane_max) {
        const int nv_cap = std::min(4, at_most);
        const int lpr = std::min(32, std::max(pow2_at_least((nvec + nv_cap - 1) / nv_cap), std::min(8, pow2_at_least(nvec))));
        return {lpr, pow2_at_least((nvec + lpr - 1) / lpr), 0};
    }
    int nv = 1;
    while (nv < at_most && (nvec + nv - 1) / nv > 256) nv <<= 1;
    return {0, nv, ((nvec + nv - 1) / nv + 31) / 32 * 32};
}

template <typename T, int VB>
int launch_forward(FwdArgs A, cudaStream_t st) {
    constexpr int VE = Pack<T, VB>::VE;
    A.nvec = A.D / VE;
    const Layout L = layout(A.nvec, 8, 128);
    const int sms = mggb::sm_count();
    if (L.lpr) {
        A.lpr = L.lpr;
        const long long rows = (long long)ROW_THREADS / L.lpr * (4 / L.nv);
        const int grid = (int)std::min<long long>((A.n + rows - 1) / rows, 8LL * sms);
        if (L.nv == 1) ln_forward_kernel<T, VB, 1, false><<<grid, ROW_THREADS, 0, st>>>(A);
        else if (L.nv == 2) ln_forward_kernel<T, VB, 2, false><<<grid, ROW_THREADS, 0, st>>>(A);
        else ln_forward_kernel<T, VB, 4, false><<<grid, ROW_THREADS, 0, st>>>(A);
    } else if (L.tpr <= MAX_TPR) {
        const int grid = (int)std::min<long long>(A.n, (long long)sms * std::max(1, 2048 / L.tpr));
        if (L.nv == 1) ln_forward_kernel<T, VB, 1, true><<<grid, L.tpr, 0, st>>>(A);
        else if (L.nv == 2) ln_forward_kernel<T, VB, 2, true><<<grid, L.tpr, 0, st>>>(A);
        else if (L.nv == 4) ln_forward_kernel<T, VB, 4, true><<<grid, L.tpr, 0, st>>>(A);
        else ln_forward_kernel<T, VB, 8, true><<<grid, L.tpr, 0, st>>>(A);
    } else {
        ln_forward_wide_kernel<T><<<(int)std::min<long long>(A.n, 2LL * sms), MAX_TPR, 0, st>>>(A);
    }
    MGGB_CUDA(cudaGetLastError());
    return MGGB_OK;
}

template <typename T>
int forward(FwdArgs A, cudaStream_t st) {
    const int s = sizeof(T);
    const int a = mggb::common_alignment({(uint64_t)A.x, (uint64_t)A.out, (uint64_t)A.ld_x * s, (uint64_t)A.ld_out * s, (uint64_t)A.D * s});
    A.param_vec = ((uint64_t)A.w | (uint64_t)A.b) % 16 == 0;
    if (a == 16) return launch_forward<T, 16>(A, st);
    if (sizeof(T) == 4 && a == 8) return launch_forward<T, sizeof(T) == 4 ? 8 : 4>(A, st);
    if (a >= 4) return launch_forward<T, 4>(A, st);
    return launch_forward<T, sizeof(T)>(A, st);
}

template <typename T, int VB>
int launch_backward(BwdArgs A, float* dw, float* db, cudaStream_t st) {
    constexpr int VE = Pack<T, VB>::VE;
    A.nvec = A.D / VE;
    const Layout L = layout(A.nvec, std::min(8, 16 / VE), 128);
    const int sms = mggb::sm_count();
    int parts = ln_parts(A.n, A.D);
    if (A.n == 0) {
        parts = 0;
    } else if (L.lpr) {
        A.lpr = L.lpr;
        const int u = L.nv * VE > 8 ? 1 : (L.nv * VE > 4 ? 2 : 4);
        const long long rows = (long long)ROW_THREADS / L.lpr * u;
        const int grid = parts = (int)std::min<long long>((A.n + rows - 1) / rows, std::min(parts, 2 * sms));
        const size_t smem = A.part ? (size_t)2 * A.D * sizeof(float) : 0;
        if (L.nv == 1) ln_backward_kernel<T, VB, 1, false><<<grid, ROW_THREADS, smem, st>>>(A);
        else if (L.nv == 2) ln_backward_kernel<T, VB, 2, false><<<grid, ROW_THREADS, smem, st>>>(A);
        else ln_backward_kernel<T, VB, 4, false><<<grid, ROW_THREADS, smem, st>>>(A);
    } else if (L.tpr <= MAX_TPR_BWD) {
        const auto kernel = L.nv == 1 ? ln_backward_kernel<T, VB, 1, true> : L.nv == 2 ? ln_backward_kernel<T, VB, 2, true>
                          : L.nv == 4 ? ln_backward_kernel<T, VB, VE <= 4 ? 4 : 1, true> : ln_backward_kernel<T, VB, VE <= 2 ? 8 : 1, true>;
        // one wave: blocks that have to wait for others would find their rows late
        int resident = 1;
        if (parts > sms) MGGB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, L.tpr, 0));
        parts = std::min(parts, sms * std::max(1, resident));
        kernel<<<parts, L.tpr, 0, st>>>(A);
    } else {
        if (A.part) {
            const dim3 grid((A.D + 127) / 128, parts);
            ln_dw_wide_kernel<T><<<grid, 128, 0, st>>>(A);       // before dx, which may be dy or x
        }
        if (A.dx) ln_dx_wide_kernel<T><<<(int)std::min<long long>(A.n, 2LL * sms), MAX_TPR, 0, st>>>(A);
    }
    MGGB_CUDA(cudaGetLastError());
    if (A.part) {
        ln_dw_reduce_kernel<<<(2 * A.D + 31) / 32, 512, 0, st>>>(dw, db, A.part, parts, A.D);
        MGGB_CUDA(cudaGetLastError());
    }
    return MGGB_OK;
}

template <typename T>
int backward(BwdArgs A, float* dw, float* db, cudaStream_t st) {
    const int s = sizeof(T);
    const int a = mggb::common_alignment({(uint64_t)A.x, (uint64_t)A.dy, (uint64_t)A.dx, (uint64_t)A.ld_x * s, (uint64_t)A.ld_dy * s,
                                          A.dx ? (uint64_t)A.ld_dx * s : 0, (uint64_t)A.D * s});
    A.param_vec = (uint64_t)A.w % 16 == 0;
    if (a == 16) return launch_backward<T, 16>(A, dw, db, st);
    if (sizeof(T) == 4 && a == 8) return launch_backward<T, sizeof(T) == 4 ? 8 : 4>(A, dw, db, st);
    if (a >= 4) return launch_backward<T, 4>(A, dw, db, st);
    return launch_backward<T, sizeof(T)>(A, dw, db, st);
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
    const FwdArgs A{out, x, weight, bias, eps, mean, rstd, n, ld_out, ld_x, dim, 0, 0, 0};
    return MGGB_BY_DTYPE(dtype, forward, A, (cudaStream_t)stream);
}

int mggb_layer_norm_backward_scratch_bytes(int64_t n, int dim, size_t* bytes) {
    MGGB_REQUIRE(bytes, "layer_norm_backward_scratch_bytes: NULL output");
    MGGB_REQUIRE(n >= 0 && dim >= 1, "layer_norm_backward_scratch_bytes: need n >= 0, dim >= 1 (n=%lld dim=%d)", (long long)n, dim);
    *bytes = (size_t)ln_parts(n, dim) * 2 * dim * sizeof(float);
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
    const bool params = dweight || dbias;
    if (params) {
        size_t need = 0;
        const int rc = mggb_layer_norm_backward_scratch_bytes(n, dim, &need);
        if (rc != MGGB_OK) return rc;
        MGGB_REQUIRE(scratch && scratch_bytes >= need, "layer_norm_backward: scratch of %zu bytes needed, %zu given", need, scratch ? scratch_bytes : (size_t)0);
        MGGB_REQUIRE((uintptr_t)scratch % 16 == 0, "layer_norm_backward: scratch must be 16-byte aligned");
    } else if (n == 0) {
        return MGGB_OK;
    }
    const BwdArgs A{dx, dy, x, mean, rstd, weight, params ? (float*)scratch : nullptr, n, ld_dx, ld_dy, ld_x, dim, 0, 0, 0};
    return MGGB_BY_DTYPE(dtype, backward, A, dweight, dbias, (cudaStream_t)stream);
}

}  // extern "C"
