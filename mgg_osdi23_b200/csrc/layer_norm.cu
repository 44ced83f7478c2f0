// Layer norm over the features of each row, forward and backward.
//     mean = sum(x) / D,  rstd = 1 / sqrt(sum((x - mean)^2) / D + eps),  xhat = (x - mean) * rstd,  y = xhat * w + b
//     g = dy * w;  dx = rstd * (g - mean(g) - xhat * mean(g * xhat));  dw = sum over rows of dy * xhat;  db = sum of dy
// No counterpart in the reference, whose models have no normalisation between layers.
//
// Bound by HBM: the forward pass has to read and write each element once, the backward pass to read two and write one.
// A row therefore stays in registers between its reductions and its result, in the vectors it was loaded as, and the
// gradients of weight and bias are summed in registers by threads that keep the same columns for every row they take.
// Forward, two shapes of the same code:
//   rows up to 128 vectors   1 to 32 lanes of a warp per row, up to 4 vectors per lane; reductions by shuffles only.
//                            Several narrow rows share a warp: a lane always has 4 loads in flight.
//   wider rows               one block per row, 1 to 8 vectors per thread; reductions through shared memory.
// Backward: teams of 1 to 16 warps take their rows from rings of bulk copies (see ln_backward_kernel).
// Rows too wide for registers are read again for every pass over them (from L2).
// Measured: forward 2,449,029 x 100 fp32 343 us (5.8 TB/s, 0.89 of the copy rate); backward 232,965 x 602 fp32 335 us (0.78; loads
// into registers instead of the rings: 421), 8192 x 4096 bf16 59 us.
#include <algorithm>
#include <cfloat>
#include <utility>
#include "async.h"
#include "elem.h"
#include "overlap.h"

namespace {

using namespace mggb;

constexpr int ROW_THREADS = 256;    // block of the kernels that put several rows in a warp or block
constexpr int MAX_TPR = 1024;       // threads per row of the block-per-row kernels
constexpr int BWD_THREADS = 512;    // block of the backward pass: 20 elements a thread with their sums want up to 128 registers
constexpr int BWD_WARPS = BWD_THREADS / 32;
constexpr int MAX_STAGES = 8;       // steps of a team's ring
constexpr int RING_BYTES = 216 * 1024;

// Sum over the lanes of a group of lpr (a power of two) neighbouring lanes; every lane gets it.
__device__ __forceinline__ float group_sum(float v, int lpr) {
#pragma unroll
    for (int off = 16; off; off >>= 1)
        if (off < lpr) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// Sums over the block.  Consecutive calls alternate between two rows of `red`, so one barrier each is enough.
struct BlockSum {
    float (*red)[2][32];
    int turn;
    __device__ __forceinline__ float2 operator()(float a, float b) {
        const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        a = warp_sum(a);
        b = warp_sum(b);
        if (lane == 0) { red[turn][0][warp] = a; red[turn][1][warp] = b; }
        __syncthreads();
        a = warp_sum(lane < warps ? red[turn][0][lane] : 0.f);
        b = warp_sum(lane < warps ? red[turn][1][lane] : 0.f);
        turn ^= 1;
        return make_float2(a, b);
    }
    __device__ __forceinline__ float operator()(float a) {
        const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        a = warp_sum(a);
        if (lane == 0) red[turn][0][warp] = a;
        __syncthreads();
        a = warp_sum(lane < warps ? red[turn][0][lane] : 0.f);
        turn ^= 1;
        return a;
    }
};

// VE consecutive floats of a parameter vector (fill where there is none); ALIGNED: p is a multiple of 16 bytes away.
template <int VE, bool ALIGNED>
__device__ __forceinline__ void load_params(float (&v)[VE], const float* p, bool have, float fill) {
    if (!have) {
#pragma unroll
        for (int i = 0; i < VE; i++) v[i] = fill;
    } else if (VE % 4 == 0 && ALIGNED) {
#pragma unroll
        for (int i = 0; i < VE / 4; i++) *reinterpret_cast<float4*>(&v[4 * i]) = __ldg(reinterpret_cast<const float4*>(p) + i);
    } else if (VE == 2 && ALIGNED) {
        *reinterpret_cast<float2*>(&v[0]) = __ldg(reinterpret_cast<const float2*>(p));
    } else {
#pragma unroll
        for (int i = 0; i < VE; i++) v[i] = __ldg(p + i);
    }
}

// s / D from the rounded reciprocal and one correction: within an ulp, at a fifth of a division's instructions.
__device__ __forceinline__ float divide(float s, float D, float inv_D) {
    const float q = s * inv_D;
    return fmaf(fmaf(-q, D, s), inv_D, q);
}

struct FwdArgs {
    void* out;
    const void* x;
    const float *w, *b;
    float eps;
    float *mean, *rstd;
    long long n, ld_out, ld_x;
    int D, nvec, param_vec;
};

// LPR: lanes per row, 0 for a whole block per row.
template <typename T, int VB, int NV, int LPR>
__global__ void __launch_bounds__(LPR ? ROW_THREADS : MAX_TPR) ln_forward_kernel(const FwdArgs A) {
    constexpr int VE = Pack<T, VB>::VE;
    constexpr bool BLOCK = LPR == 0;
    constexpr int U = BLOCK || NV > 4 ? 1 : 4 / NV;       // rows a group of lanes has in flight
    constexpr int GROUPS = BLOCK ? 1 : ROW_THREADS / (BLOCK ? 1 : LPR);
    __shared__ float red[2][2][32];
    BlockSum block_sum{red, 0};
    const int tpr = BLOCK ? blockDim.x : LPR;
    const int l = BLOCK ? threadIdx.x : threadIdx.x % (BLOCK ? 1 : LPR);
    const long long row0 = (long long)blockIdx.x * (GROUPS * U) + (BLOCK ? 0 : threadIdx.x / (BLOCK ? 1 : LPR));
    const int left = (int)min(A.n - row0, (long long)(GROUPS * U));      // rows row0 + u * GROUPS with u * GROUPS < left exist
    const float D = (float)A.D, inv_D = 1.f / D;
    const T* x = (const T*)A.x + row0 * A.ld_x + l * VE;
    float v[U][NV][VE];
    {
        Pack<T, VB> raw[U][NV];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < NV; j++)
                if (u * GROUPS < left && l + j * tpr < A.nvec) raw[u][j].load(x + u * GROUPS * A.ld_x + j * tpr * VE);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < NV; j++) raw[u][j].widen(v[u][j]);
    }
    float mean[U], rstd[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int i = 0; i < VE; i++) s += v[u][j][i];
        mean[u] = divide(BLOCK ? block_sum(s) : group_sum(s, LPR), D, inv_D);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float qj = 0.f;
#pragma unroll
            for (int i = 0; i < VE; i++) {
                v[u][j][i] -= mean[u];
                qj = fmaf(v[u][j][i], v[u][j][i], qj);
            }
            q += l + j * tpr < A.nvec ? qj : 0.f;
        }
        rstd[u] = rsqrtf((BLOCK ? block_sum(q) : group_sum(q, LPR)) * inv_D + A.eps);
    }
    T* out = (T*)A.out + row0 * A.ld_out + l * VE;
    auto store_rows = [&](auto aligned) {
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (l + j * tpr >= A.nvec) continue;
            const int c = (l + j * tpr) * VE;
            float w[VE], b[VE];
            load_params<VE, decltype(aligned)::value>(w, A.w + c, A.w != nullptr, 1.f);
            load_params<VE, decltype(aligned)::value>(b, A.b + c, A.b != nullptr, 0.f);
#pragma unroll
            for (int u = 0; u < U; u++) {
                float y[VE];
#pragma unroll
                for (int i = 0; i < VE; i++) y[i] = fmaf(v[u][j][i] * rstd[u], w[i], b[i]);
                Pack<T, VB> o;
                o.narrow(y);
                if (u * GROUPS < left) o.store(out + u * GROUPS * A.ld_out + j * tpr * VE);
            }
        }
    };
    if (A.param_vec) store_rows(std::true_type());
    else store_rows(std::false_type());
    if (l == 0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (u * GROUPS < left && A.mean) A.mean[row0 + u * GROUPS] = mean[u];
            if (u * GROUPS < left && A.rstd) A.rstd[row0 + u * GROUPS] = rstd[u];
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
    int D, nvec, lpr;
    int rows, stages, slot;          // rows of a team's step, steps in its ring, bytes of one matrix's rows of one step
    unsigned polls;                  // of a barrier before a wait gives up
};

__device__ int g_ln_status = 0;      // 1: a bounded wait for rows expired

template <int P>
__device__ __forceinline__ float& at(float2 (&v)[P], int i) { return i & 1 ? v[i >> 1].y : v[i >> 1].x; }

// A team of W warps takes rows (W = 1: rows of 32 / lpr groups of lanes, U each) step by step from a ring in shared
// memory that it fills itself by bulk copies, several steps ahead: the loads in flight cost no registers and do not wait
// for the reductions.  A thread keeps the same NV vectors of columns for all rows, and their gradients' sums.
template <typename T, int VB, int NV, bool TEAM>
__global__ void __launch_bounds__(BWD_THREADS, 1) ln_backward_kernel(const BwdArgs A, const int W) {
    constexpr int VE = Pack<T, VB>::VE;
    constexpr int E = NV * VE, P = (E + 1) / 2;
    constexpr int U = TEAM || E > 8 ? 1 : (E > 4 ? 2 : 4);
    extern __shared__ __align__(128) unsigned char smem[];            // [D] weight (when there is one), then the teams' rings
    float* weight = reinterpret_cast<float*>(smem);
    unsigned char* ring_all = smem + (A.w ? (A.D * 4 + 127) / 128 * 128 : 0);
    __shared__ unsigned long long bars[BWD_WARPS * MAX_STAGES];
    __shared__ float2 red[2][BWD_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int teams = BWD_WARPS / (TEAM ? W : 1), team = TEAM ? warp / W : warp;
    const int tpr = TEAM ? 32 * W : A.lpr;                              // threads per row
    const int l = TEAM ? threadIdx.x - team * tpr : lane & (A.lpr - 1);
    const int groups = TEAM ? 1 : 32 / A.lpr, group = TEAM ? 0 : lane / A.lpr;
    const bool issuer = TEAM ? warp == team * W : true;                 // the team's copying warp
    unsigned char* ring = ring_all + (size_t)team * A.stages * 2 * A.slot;
    const uint32_t ring_base = smem_addr(ring), bar0 = smem_addr(bars + team * MAX_STAGES);
    const float inv_D = 1.f / (float)A.D;

    if (issuer && lane == 0)
        for (int s = 0; s < A.stages; s++) bar_init(bar0 + 8 * s, 1);
    bar_init_fence();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (A.w)
        for (int i = threadIdx.x; i < A.D; i += BWD_THREADS) weight[i] = __ldg(A.w + i);
    __syncthreads();

    const long long first = (long long)blockIdx.x * teams + team, stride = (long long)gridDim.x * teams;
    const long long all = (A.n + A.rows - 1) / A.rows;
    const int steps = first < all ? (int)((all - first + stride - 1) / stride) : 0;
    const bool joined_x = A.ld_x == A.D, joined_g = A.ld_dy == A.D;
    const int row_bytes = A.D * (int)sizeof(T), pitch = (row_bytes + 15 + 16) / 16 * 16;
    auto issue = [&](long long row0, int s) {                           // copying warp only
        const int rows = (int)min((long long)A.rows, A.n - row0);
        const uint32_t dst = ring_base + s * 2 * A.slot;
        unsigned char* dst_ptr = ring + s * 2 * A.slot;
        unsigned bytes = copy_rows<T>(dst, dst_ptr, A.x, A.ld_x, A.D, A.n, row0, rows, pitch, bar0 + 8 * s);
        bytes += copy_rows<T>(dst + A.slot, dst_ptr + A.slot, A.dy, A.ld_dy, A.D, A.n, row0, rows, pitch, bar0 + 8 * s);
        bytes = __reduce_add_sync(0xffffffffu, bytes);
        __syncwarp();
        if (lane == 0) bar_expect(bar0 + 8 * s, bytes);                 // also publishes the plain stores of the odd bytes
    };
    if (issuer)
        for (int k = 0; k < min(steps, A.stages); k++) issue((first + k * stride) * A.rows, k);

    // a thread's E elements in pairs, column j * VE + i at place j * VE + i
    float2 aw[P], ab[P];
#pragma unroll
    for (int p = 0; p < P; p++) aw[p] = ab[p] = make_float2(0.f, 0.f);
    int turn = 0, s = 0;
    unsigned phase = 0;
    bool ok = true;
    long long row0 = first * A.rows;
    const long long row_step = stride * A.rows;
    // where row 0 of a step begins in its slot: at the same offset inside 16 bytes as in memory
    const bool steady_x = (A.ld_x * sizeof(T)) % 16 == 0, steady_g = (A.ld_dy * sizeof(T)) % 16 == 0;
    const bool ragged = E % 2 != 0 || NV * tpr > A.nvec;                // some threads hold places without an element
    // the rows' statistics come a step ahead: their latency would stand between every step's arrival and its refill
    float mean[U], rstd[U], mean_next[U], rstd_next[U];
    auto load_stats = [&](long long row) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long r = row + u * groups + group;
            const bool live = u * groups + group < A.rows && r < A.n;
            mean_next[u] = live ? __ldg(A.mean + r) : 0.f;
            rstd_next[u] = live ? __ldg(A.rstd + r) : 0.f;
        }
    };
    load_stats(row0);
    for (int k = 0; k < steps; k++, row0 += row_step) {
        bool huge = false;
#pragma unroll
        for (int u = 0; u < U; u++) {
            mean[u] = mean_next[u];
            rstd[u] = rstd_next[u];
            huge = huge || (!TEAM && ragged && !(fabsf(mean[u] * rstd[u]) <= FLT_MAX));
        }
        load_stats(row0 + row_step);
        // after a wait that ran out nothing is issued or stored any more, but the team's warps keep meeting at its barrier
        if (ok) {
            ok = __all_sync(0xffffffffu, bar_wait(bar0 + 8 * s, phase, A.polls));
            // copies still on their way: of this step and of those that were asked for behind it
            for (int i = k; !ok && issuer && i < min(steps, k + A.stages); i++) bar_wait(bar0 + 8 * (i % A.stages), (unsigned)(i / A.stages) & 1);
        }
        const unsigned char* slot = ring + s * 2 * A.slot;
        const int left = (int)min(A.n - row0, (long long)A.rows);
        float2 xh[U][P], g[U][P];
        float a[U], c[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int r = u * groups + group;
            const bool live = r < left;
            const int mx = (int)(((uint64_t)A.x + (steady_x ? 0 : (row0 + (joined_x ? 0 : r)) * A.ld_x * sizeof(T))) & 15);
            const int mg = (int)(((uint64_t)A.dy + (steady_g ? 0 : (row0 + (joined_g ? 0 : r)) * A.ld_dy * sizeof(T))) & 15);
            const unsigned char *px = slot + mx + r * (joined_x ? row_bytes : pitch) + l * VB;
            const unsigned char *pg = slot + A.slot + mg + r * (joined_g ? row_bytes : pitch) + l * VB;
            if (E % 2) xh[u][P - 1].y = g[u][P - 1].y = 0.f;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                Pack<T, VB> xv, gv;
                if (live && l + j * tpr < A.nvec) {
                    xv.raw = *reinterpret_cast<const typename Pack<T, VB>::R*>(px + j * tpr * VB);
                    gv.raw = *reinterpret_cast<const typename Pack<T, VB>::R*>(pg + j * tpr * VB);
                }
#pragma unroll
                for (int i = 0; i < VE; i++) {
                    at(xh[u], j * VE + i) = xv.get(i);
                    at(g[u], j * VE + i) = gv.get(i);
                }
            }
        }
        if (!TEAM) {                       // a warp's own ring: refilled as soon as its lanes have read the slot
            __syncwarp();
            if (ok && k + A.stages < steps) issue(row0 + A.stages * row_step, s);
        }
        float2 a2[U], c2[U];
#pragma unroll
        for (int u = 0; u < U; u++) a2[u] = c2[u] = make_float2(0.f, 0.f);
        // what is not there has dy = 0 and x = 0: with xhat finite it adds nothing
        auto mean_at = [&](int u, int e) { return TEAM && (e >= E || l + e / VE * tpr >= A.nvec) ? 0.f : mean[u]; };
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int u = 0; u < U; u++) {
                xh[u][p] = mul2(add2(xh[u][p], make_float2(-mean_at(u, 2 * p), -mean_at(u, 2 * p + 1))), make_float2(rstd[u], rstd[u]));
                aw[p] = fma2(g[u][p], xh[u][p], aw[p]);
                ab[p] = add2(ab[p], g[u][p]);
            }
        // its xhat is -mean * rstd: where that overflows, 0 times it must not reach the row's sums
        if (huge) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (E % 2) xh[u][P - 1].y = 0.f;
#pragma unroll
                for (int j = 0; j < NV; j++)
                    if (l + j * tpr >= A.nvec) {
#pragma unroll
                        for (int i = 0; i < VE; i++) at(xh[u], j * VE + i) = 0.f;
                    }
            }
        }
        if (A.w) {
#pragma unroll
            for (int j = 0; j < NV; j++) {
                float w[VE];
                const float* pw = weight + (l + j * tpr) * VE;
                if (l + j * tpr < A.nvec) {
                    if constexpr (VE % 4 == 0) {
#pragma unroll
                        for (int i = 0; i < VE; i += 4) *reinterpret_cast<float4*>(&w[i]) = *reinterpret_cast<const float4*>(pw + i);
                    } else if constexpr (VE == 2) {
                        *reinterpret_cast<float2*>(&w[0]) = *reinterpret_cast<const float2*>(pw);
                    } else {
                        w[0] = *pw;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < VE; i++) w[i] = 0.f;
                }
#pragma unroll
                for (int u = 0; u < U; u++)
                    if constexpr (VE > 1) {
#pragma unroll
                        for (int i = 0; i < VE; i += 2) g[u][(j * VE + i) / 2] = mul2(g[u][(j * VE + i) / 2], make_float2(w[i], w[i + 1]));
                    } else {
                        at(g[u], j) *= w[0];
                    }
            }
        }
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int u = 0; u < U; u++) {
                a2[u] = add2(a2[u], g[u][p]);
                c2[u] = fma2(g[u][p], xh[u][p], c2[u]);
            }
        // row sums
#pragma unroll
        for (int u = 0; u < U; u++) {
            a[u] = a2[u].x + a2[u].y;
            c[u] = c2[u].x + c2[u].y;
            if (TEAM) {
                a[u] = warp_sum(a[u]);
                c[u] = warp_sum(c[u]);
                if (lane == 0) red[turn][warp] = make_float2(a[u], c[u]);
                // behind this barrier every thread of the team has read its part of the slot, too
                asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(tpr) : "memory");
                a[u] = c[u] = 0.f;
                for (int i = 0; i < W; i++) {
                    const float2 t = red[turn][team * W + i];
                    a[u] += t.x;
                    c[u] += t.y;
                }
                turn ^= 1;
                if (issuer && ok && k + A.stages < steps) issue(row0 + A.stages * row_step, s);
            } else {
                a[u] = group_sum(a[u], A.lpr);
                c[u] = group_sum(c[u], A.lpr);
            }
        }
        if (++s == A.stages) { s = 0; phase ^= 1; }
        if (!A.dx || !ok) continue;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int r = u * groups + group;
            const float am = a[u] * inv_D, cm = c[u] * inv_D;
            T* out = (T*)A.dx + (row0 + r) * A.ld_dx + l * VE;
#pragma unroll
            for (int p = 0; p < P; p++)
                g[u][p] = mul2(fma2(make_float2(-cm, -cm), xh[u][p], add2(g[u][p], make_float2(-am, -am))), make_float2(rstd[u], rstd[u]));
#pragma unroll
            for (int j = 0; j < NV; j++) {
                float d[VE];
#pragma unroll
                for (int i = 0; i < VE; i++) d[i] = at(g[u], j * VE + i);
                Pack<T, VB> o;
                o.narrow(d);
                if (r < left && l + j * tpr < A.nvec) o.store(out + j * tpr * VE);
            }
        }
    }
    if (!ok) atomicExch(&g_ln_status, 1);
    __syncthreads();                       // every copy has landed (each was waited for), every slot has been read
    if (!A.part) return;
    float* part = A.part + (long long)blockIdx.x * 2 * A.D;
    if (!TEAM) {                           // lane groups of a warp meet by shuffles
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int i = 0; i < VE; i++)
                for (int off = A.lpr; off < 32; off <<= 1) {
                    at(aw, j * VE + i) += __shfl_xor_sync(0xffffffffu, at(aw, j * VE + i), off);
                    at(ab, j * VE + i) += __shfl_xor_sync(0xffffffffu, at(ab, j * VE + i), off);
                }
    }
    // teams meet in shared memory (the ring's, now free) one after the other: a fixed order
    float* sums = reinterpret_cast<float*>(ring_all);
    for (int t = 0; t < teams; t++) {
        if (team == t && group == 0) {
#pragma unroll
            for (int j = 0; j < NV; j++)
                if (l + j * tpr < A.nvec) {
#pragma unroll
                    for (int i = 0; i < VE; i++) {
                        const int col = (l + j * tpr) * VE + i;
                        sums[col] = (t ? sums[col] : 0.f) + at(aw, j * VE + i);
                        sums[A.D + col] = (t ? sums[A.D + col] : 0.f) + at(ab, j * VE + i);
                    }
                }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * A.D; i += BWD_THREADS) part[i] = sums[i];
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

// Column sums of the blocks' partial sums: 32 columns per block, 32 warps take every 32nd block, then meet in order.
__global__ void __launch_bounds__(1024) ln_dw_reduce_kernel(float* __restrict__ dw, float* __restrict__ db, const float* __restrict__ part,
                                                            int parts, int D) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + lane;
    float a = 0.f;
    asm volatile("griddepcontrol.wait;" ::: "memory");       // the partial sums are complete
    if (col < 2 * D)
#pragma unroll 8
        for (int p = wp; p < parts; p += 32) a += part[(long long)p * 2 * D + col];
    s[wp][lane] = a;
    __syncthreads();
    // warp w sums columns w, each lane one of the 32 partial sums
    a = warp_sum(s[lane][wp]);
    const int c = blockIdx.x * 32 + wp;
    if (lane == 0 && c < 2 * D) {
        if (c < D) { if (dw) dw[c] = a; }
        else if (db) db[c - D] = a;
    }
}

// Blocks whose sums of the weight's gradient are kept apart.
int ln_parts(long long n) { return (int)std::max<long long>(1, std::min<long long>(n, sm_count())); }

int pow2_at_least(int v) {
    int p = 1;
    while (p < v) p <<= 1;
    return p;
}

template <typename T, int VB>
int launch_forward(FwdArgs A, cudaStream_t st) {
    constexpr int VE = Pack<T, VB>::VE, MOST = VE <= 4 ? 8 : 4;
    A.nvec = A.D / VE;
    if (A.nvec <= 128) {
        // narrow rows: 8 lanes at least where the row has that many vectors (128 bytes per group and load with 16-byte
        // vectors), then 4 vectors per lane, then more lanes
        const int lpr = std::min(32, std::max(pow2_at_least((A.nvec + 3) / 4), std::min(8, pow2_at_least(A.nvec))));
        const int nv = pow2_at_least((A.nvec + lpr - 1) / lpr);
        const auto kernel = lpr == 1 ? ln_forward_kernel<T, VB, 1, 1> : lpr == 2 ? ln_forward_kernel<T, VB, 1, 2> : lpr == 4 ? ln_forward_kernel<T, VB, 1, 4>
                          : lpr == 16 ? ln_forward_kernel<T, VB, 4, 16> : lpr == 32 ? ln_forward_kernel<T, VB, 4, 32>
                          : nv == 1 ? ln_forward_kernel<T, VB, 1, 8> : nv == 2 ? ln_forward_kernel<T, VB, 2, 8> : ln_forward_kernel<T, VB, 4, 8>;
        const long long rows = (long long)ROW_THREADS / lpr * (4 / (lpr < 8 ? 1 : lpr > 8 ? 4 : nv));
        kernel<<<(unsigned)((A.n + rows - 1) / rows), ROW_THREADS, 0, st>>>(A);
    } else {
        int nv = 1;
        while (nv < MOST && (A.nvec + nv - 1) / nv > 256) nv <<= 1;
        const int tpr = ((A.nvec + nv - 1) / nv + 31) / 32 * 32;
        if (tpr <= MAX_TPR) {
            const auto kernel = nv == 1 ? ln_forward_kernel<T, VB, 1, 0> : nv == 2 ? ln_forward_kernel<T, VB, 2, 0> : nv == 4 ? ln_forward_kernel<T, VB, 4, 0>
                              : ln_forward_kernel<T, VB, MOST, 0>;
            kernel<<<(unsigned)A.n, tpr, 0, st>>>(A);
        } else {
            ln_forward_wide_kernel<T><<<(int)std::min<long long>(A.n, 2LL * sm_count()), MAX_TPR, 0, st>>>(A);
        }
    }
    MGGB_CUDA(cudaGetLastError());
    return MGGB_OK;
}

template <typename T>
int forward(FwdArgs A, cudaStream_t st) {
    const int s = sizeof(T);
    const int a = common_alignment({(uint64_t)A.x, (uint64_t)A.out, (uint64_t)A.ld_x * s, (uint64_t)A.ld_out * s, (uint64_t)A.D * s});
    A.param_vec = ((uint64_t)A.w | (uint64_t)A.b) % 16 == 0;
    if (a == 16) return launch_forward<T, 16>(A, st);
    if (sizeof(T) == 4 && a == 8) return launch_forward<T, sizeof(T) == 4 ? 8 : 4>(A, st);
    if (a >= 4) return launch_forward<T, 4>(A, st);
    return launch_forward<T, sizeof(T)>(A, st);
}

// Vectors per thread the backward kernel is built for: at most 20 elements.
template <int VE> struct BwdVectors;
template <> struct BwdVectors<8> { static constexpr int v[] = {1, 2}; };
template <> struct BwdVectors<4> { static constexpr int v[] = {1, 2, 3, 4, 5}; };
template <> struct BwdVectors<2> { static constexpr int v[] = {1, 2, 4, 6, 8, 10}; };
template <> struct BwdVectors<1> { static constexpr int v[] = {1, 2, 4, 8, 12, 16, 20}; };

template <typename T, int VB, int I>
int launch_backward_nv(BwdArgs A, int nv, int W, int* parts, cudaStream_t st) {
    constexpr int VE = Pack<T, VB>::VE;
    using V = BwdVectors<VE>;
    if constexpr (I < (int)(sizeof(V::v) / sizeof(int))) {
        if (V::v[I] != nv) return launch_backward_nv<T, VB, I + 1>(A, nv, W, parts, st);
        constexpr int NV = V::v[I];
        const int u = W > 1 || NV * VE > 8 ? 1 : (NV * VE > 4 ? 2 : 4);
        const int teams = BWD_WARPS / W;
        A.rows = W > 1 ? 1 : 32 / A.lpr * u;
        const int row_bytes = A.D * (int)sizeof(T), pitch = (row_bytes + 31) / 16 * 16;
        A.slot = std::max((A.rows * row_bytes + 31) / 16 * 16, (A.ld_x == A.D && A.ld_dy == A.D) ? 0 : A.rows * pitch);
        const int weight_bytes = A.w ? (A.D * 4 + 127) / 128 * 128 : 0;
        A.stages = std::min(MAX_STAGES, (RING_BYTES - weight_bytes) / (teams * 2 * A.slot));
        const long long steps = (A.n + A.rows - 1) / A.rows;
        *parts = (int)std::min<long long>((steps + teams - 1) / teams, sm_count());
        const int smem = weight_bytes + std::max(teams * A.stages * 2 * A.slot, A.part ? 2 * A.D * 4 : 0);
        const auto kernel = W > 1 ? ln_backward_kernel<T, VB, NV, true> : ln_backward_kernel<T, VB, NV, false>;
        MGGB_CUDA((W > 1 ? allow_shared<ln_backward_kernel<T, VB, NV, true>>() : allow_shared<ln_backward_kernel<T, VB, NV, false>>()));
        kernel<<<*parts, BWD_THREADS, smem, st>>>(A, W);
        MGGB_CUDA(cudaGetLastError());
        return MGGB_OK;
    }
    return fail(MGGB_ERR_UNSUPPORTED, "layer_norm_backward: no kernel for %d vectors", nv);
}

template <typename T, int VB>
int launch_backward(BwdArgs A, float* dw, float* db, cudaStream_t st) {
    constexpr int VE = Pack<T, VB>::VE;
    using V = BwdVectors<VE>;
    constexpr int kinds = sizeof(V::v) / sizeof(int), most = V::v[kinds - 1];
    A.nvec = A.D / VE;
    int parts = 0;
    int W = 1;
    while (W < BWD_WARPS && A.nvec > 32 * W * most) W *= 2;
    if (A.n > 0 && A.nvec <= 32 * W * most) {
        // a row on fewer than 32 lanes only while each lane has up to 4 vectors of it: 128 bytes per group and load or more
        int threads = 32 * W;
        if (W == 1) threads = std::min(32, std::max(pow2_at_least((A.nvec + std::min(4, most) - 1) / std::min(4, most)), std::min(8, pow2_at_least(A.nvec))));
        A.lpr = threads;
        int nv = most;
        for (int i = kinds - 1; i >= 0; i--)
            if (V::v[i] * threads >= A.nvec) nv = V::v[i];
        const int rc = launch_backward_nv<T, VB, 0>(A, nv, W, &parts, st);
        if (rc != MGGB_OK) return rc;
    } else if (A.n > 0) {
        if (A.part) {
            parts = ln_parts(A.n);
            const dim3 grid((A.D + 127) / 128, parts);
            ln_dw_wide_kernel<T><<<grid, 128, 0, st>>>(A);       // before dx, which may be dy or x
            MGGB_CUDA(cudaGetLastError());
        }
        if (A.dx) ln_dx_wide_kernel<T><<<(int)std::min<long long>(A.n, 2LL * sm_count()), MAX_TPR, 0, st>>>(A);
        MGGB_CUDA(cudaGetLastError());
    }
    if (A.part) {
        // launched while the kernel before it still runs; its blocks wait for that kernel's end
        cudaLaunchConfig_t config = {};
        cudaLaunchAttribute attr[1];
        config.gridDim = dim3((2 * A.D + 31) / 32);
        config.blockDim = dim3(1024);
        config.stream = st;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        config.attrs = attr;
        config.numAttrs = 1;
        MGGB_CUDA(cudaLaunchKernelEx(&config, ln_dw_reduce_kernel, dw, db, (const float*)A.part, parts, A.D));
    }
    return MGGB_OK;
}

template <typename T>
int backward(BwdArgs A, float* dw, float* db, cudaStream_t st) {
    const int s = sizeof(T);
    const int a = common_alignment({(uint64_t)A.x, (uint64_t)A.dy, (uint64_t)A.dx, (uint64_t)A.ld_x * s, (uint64_t)A.ld_dy * s,
                                          A.dx ? (uint64_t)A.ld_dx * s : 0, (uint64_t)A.D * s});
    if (a == 16) return launch_backward<T, 16>(A, dw, db, st);
    if (sizeof(T) == 4 && a == 8) return launch_backward<T, sizeof(T) == 4 ? 8 : 4>(A, dw, db, st);
    if (a >= 4) return launch_backward<T, 4>(A, dw, db, st);
    return launch_backward<T, sizeof(T)>(A, dw, db, st);
}

}  // namespace

namespace mggb {
int layer_norm_status(int* status, int reset) {
    MGGB_CUDA(cudaMemcpyFromSymbol(status, g_ln_status, sizeof(int)));
    const int zero = 0;
    if (reset && *status) MGGB_CUDA(cudaMemcpyToSymbol(g_ln_status, &zero, sizeof(int)));     // what was not read is not cleared
    return MGGB_OK;
}
}  // namespace mggb

extern "C" {

int mggb_layer_norm_forward(void* out, const void* x, const float* weight, const float* bias, float eps, float* mean, float* rstd,
                            int64_t n, int dim, int64_t ld_out, int64_t ld_x, int dtype, void* stream) {
    MGGB_REQUIRE(n >= 0 && dim >= 1 && dim <= 1 << 28, "layer_norm_forward: need n >= 0, 1 <= dim <= 2^28 (n=%lld dim=%d)", (long long)n, dim);
    MGGB_REQUIRE_DTYPE(dtype, "layer_norm_forward");
    MGGB_REQUIRE(eps >= 0.f, "layer_norm_forward: eps must not be negative or NaN");
    MGGB_REQUIRE(ld_out >= dim && ld_x >= dim, "layer_norm_forward: row strides must be at least dim");
    if (n == 0) return MGGB_OK;
    MGGB_REQUIRE(out && x, "layer_norm_forward: NULL argument");
    MGGB_REQUIRE(out != x || ld_out == ld_x, "layer_norm_forward: in place needs equal row strides");
    const int s = elem_bytes(dtype);
    MGGB_REQUIRE(out == x || !rows_meet(out, ld_out * s, x, ld_x * s, n, (uint64_t)dim * s), "layer_norm_forward: out lies partly over x");
    const FwdArgs A{out, x, weight, bias, eps, mean, rstd, n, ld_out, ld_x, dim, 0, 0};
    return MGGB_BY_DTYPE(dtype, forward, A, (cudaStream_t)stream);
}

int mggb_layer_norm_backward_scratch_bytes(int64_t n, int dim, size_t* bytes) {
    MGGB_REQUIRE(bytes, "layer_norm_backward_scratch_bytes: NULL output");
    MGGB_REQUIRE(n >= 0 && dim >= 1 && dim <= 1 << 28, "layer_norm_backward_scratch_bytes: need n >= 0, 1 <= dim <= 2^28 (n=%lld dim=%d)", (long long)n, dim);
    *bytes = (size_t)ln_parts(n) * 2 * dim * sizeof(float);
    return MGGB_OK;
}

int mggb_layer_norm_backward(void* dx, float* dweight, float* dbias, const void* dy, const void* x, const float* mean, const float* rstd,
                             const float* weight, int64_t n, int dim, int64_t ld_dx, int64_t ld_dy, int64_t ld_x, int dtype,
                             void* scratch, size_t scratch_bytes, void* stream) {
    MGGB_REQUIRE(n >= 0 && dim >= 1 && dim <= 1 << 28, "layer_norm_backward: need n >= 0, 1 <= dim <= 2^28 (n=%lld dim=%d)", (long long)n, dim);
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
    const int s = elem_bytes(dtype);
    for (const auto& in : {std::make_pair(dy, ld_dy), std::make_pair(x, ld_x)})
        MGGB_REQUIRE(!dx || dx == in.first || !rows_meet(dx, ld_dx * s, in.first, in.second * s, n, (uint64_t)dim * s),
                     "layer_norm_backward: dx lies partly over an input");
    const BwdArgs A{dx, dy, x, mean, rstd, weight, params ? (float*)scratch : nullptr, n, ld_dx, ld_dy, ld_x, dim, 0, 0, 0, 0, 0, wait_polls()};
    return MGGB_BY_DTYPE(dtype, backward, A, dweight, dbias, (cudaStream_t)stream);
}

}  // extern "C"
