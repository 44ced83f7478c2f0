// Dense products grouped by node type, on the 5th-generation tensor cores (tcgen05, sm_100a): rows group_ptr[g] ..
// group_ptr[g+1]-1 of x go through w[g] (dim1 x dim2).
//     out = x w[g]        dx = dy w[g]^T        dw[g] = x_g^T dy_g
// Stands beside dense_beg_new_forward (include/gnn_layer.cuh:42-46), whose weight is one for all nodes.
//
// All three are one kernel, D[m, n] = sum_k A[m, k] B[n, k], with the output's COLUMNS on m and its ROWS on n:
//             m (128 per tile)   n (up to 256)    k             A                      B
//     out     columns, dim2      rows of a group  dim1          w[g]^T   m contiguous  x    k contiguous
//     dx      columns, dim1      rows of a group  dim2          w[g]     k contiguous  dy   k contiguous
//     dw      columns, dim2      rows, dim1       group's rows  dy^T     m contiguous  x^T  n contiguous
// The ragged side of a group is then the instruction's N, which may be any multiple of 16: a group's last few rows cost what
// they are, not a whole tile.  And an accumulator lane is an output column, so a warp stores 32 consecutive columns of a row
// at once, from registers.  No operand is transposed: the tensor core reads either order from 64- or 128-byte swizzled tiles.
//
// Precision.  16-bit operands go in as they are, products and sums are fp32.  An fp32 operand is cut into three bf16 numbers
// that add up to it exactly (8 + 8 + 8 bits of mantissa, by truncation); of the nine partial products the six above 2^-24
// are taken, so the result is fp32-equivalent.  Cost: six bf16 instructions, the same as a pair of TF32
// numbers with all partial products but one would take, and three times 2 bytes of shared memory per element.  What the
// tensor core cuts off its sums, and when a sum leaves it, stands beside launch_tiles.
//
// The sizes of the groups are read on the device: every block turns group_ptr into a list of units of work (one tile over the
// whole sum; for dw, one tile over a chunk of a group's rows) and takes every gridDim-th.  Positions are clamped to [0, n]
// and made non-decreasing, so no group_ptr makes a kernel touch a row outside the matrices or two units write one row.
//
// Measured: 600,000 x 128 -> 128 fp32 in 4 groups 145 us (floor 95); 61 x 2048 -> 2048 bf16 in 8 groups 21 us (floor 10); 16,384 x
// 2048 -> 2048 bf16 in 16 groups, both gradients 336 to 390 us with the power cap (floor 162).
//
// One persistent block per SM, its warps in roles joined by mbarriers:
//     producers   16-bit operands whose rows are multiples of 16 bytes: one thread issues TMA copies of 64-wide boxes.
//                 Otherwise (fp32, odd widths): two groups of eight warps take every other k-chunk, load it into registers,
//                 cut it into its parts and store them in the tile's layout; while one group stores, the other's loads are
//                 in flight.
//     one thread  issues tcgen05.mma and commits to mbarriers; for dw by TMA its warp clears rows behind a group's last one.
//     four warps  (eight beside TMA) read finished accumulators (two, in tensor memory) and store them.
// Narrow products would leave most of a 128-wide tile empty and pay its latency; the fp32 pipes take them (see each kernel):
//     narrow_rows_kernel    out and dx with few terms and fewer than 32 columns: a thread per row
//     row_dots_kernel       out and dx with at most 8 columns and many terms: a warp per 4 rows, terms over lanes
//     narrow_weight_kernel  dw of small weights: 4 x 4 elements per lane, rows over warps
// Every wait is bounded; on expiry the block records it (mggb_operator_device_status), lets go of its copies and its tensor
// memory and returns.
#pragma once
#include <cuda.h>
#include <algorithm>
#include <cstring>
#include "async.h"
#include "elem.h"

namespace {

using namespace mggb;

enum { FORWARD = 0, GRAD_X = 1, GRAD_W = 2 };

constexpr int TILE_M = 128;
constexpr int MAX_TILE_N = 256, SMALL_TILE_N = 64;
constexpr int MAX_STAGES = 10;
constexpr int PRODUCERS = 256;               // threads of one producer group (register path), 2^8
constexpr int SMEM_BUDGET = 222 * 1024;

__device__ int g_grouped_status = 0;         // which wait expired first: 1 full, 2 empty, 3 accumulator ready, 4 accumulator free

struct Args {
    const int32_t* ptr;
    const void *a, *b;                       // the matrices behind A and B (register path)
    void* out;
    float* partial;                          // dw: chunks of groups that have more than one, [slot][dim1][dim2]
    int* multi;                              // dw: list of those groups: count, then (group, first slot, chunks) each
    long long n;
    int groups, M, N, K;                     // M: output columns; N: output rows of dw; K: length of the sum of out and dx
    int tile_n, m_tiles, n_tiles, stages, chunk_rows;
    int keep;                                // 1: a unit's whole A stays in shared memory for the units after it that have the same
    int seg;                                 // k per accumulator: longer sums are added up in fp32 outside the tensor core
    int split;                               // 1: fp32 parts' small products go to an accumulator of their own
    int pair;                                // 1: fp32 sums of two k-chunks, the small products of both first
    int bufs;                                // accumulators (pairs of them with split) in tensor memory: 2, or 1 where they are wide
    unsigned tmem_cols;
    unsigned polls;                          // of a barrier before a wait gives up
};

// A group's rows and where its units begin.
struct Plan {
    int *start, *unit, *slot;                // [groups + 1] each; slot only for dw
};

struct Unit {
    int g, row0, rows, m0, n0, chunk, chunks;
};

// ---- pieces ------------------------------------------------------------------------------------------------

// LIMIT_FIRST: the limit is looked at before a poll, else behind one that failed.  Before it costs the single threads 40 ns per
// wait; the producers' warps are better off with it (15,066 x 84 -> 1903 bf16, dw: 132 us instead of 175).
template <bool LIMIT_FIRST = false>
__device__ __forceinline__ bool wait_or_abort(const Args& P, uint32_t bar, unsigned parity, volatile int* abort_flag, int code) {
    for (unsigned i = 0; !LIMIT_FIRST || i < P.polls; i++) {
        if (bar_try(bar, parity)) return true;
        if (*abort_flag) return false;
        if (!LIMIT_FIRST && i + 1 >= P.polls) break;
    }
    *abort_flag = code;
    atomicCAS(&g_grouped_status, 0, code);
    return false;
}

// Shared-memory matrix descriptor.  swizzle: 2 = 128 bytes, 4 = 64 bytes.
//   k contiguous: rows of 128 (64) bytes in groups of eight, `stride` bytes from group to group; `lead` unused
//   m or n contiguous: blocks of 64 elements (128 bytes) by k rows; `stride` from eight k rows to the next eight, `lead` from
//   one block of 64 to the next
__device__ __forceinline__ uint64_t matrix_desc(uint32_t addr, uint32_t lead, uint32_t stride, uint32_t swizzle) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)((lead >> 4) & 0x3FFFu) << 16 | (uint64_t)((stride >> 4) & 0x3FFFu) << 32 |
           (uint64_t)1 << 46 | (uint64_t)swizzle << 61;
}

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

template <typename T, int MODE>
struct Shape {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int PARTS = F32 ? 3 : 1;
    static constexpr int BK = F32 ? 32 : 64;                       // k per stage
    static constexpr bool A_MN = MODE != GRAD_X, B_MN = MODE == GRAD_W;
    static constexpr int A_PART = TILE_M * BK * 2;                 // bytes of one part of a tile of A
    static constexpr int ROW = BK * 2;                             // bytes of a k-contiguous row
    __host__ __device__ static int b_part(int tile_n) { return tile_n * BK * 2; }
    __host__ __device__ static int stage(int tile_n, bool keep) { return PARTS * ((keep ? 0 : A_PART) + b_part(tile_n)); }
    // where 16 bytes (8 elements) go: k contiguous, row `o`, piece `ch` of its k
    __device__ static uint32_t at_k(int o, int ch) { return (uint32_t)(o * ROW + ((ch ^ (ROW == 128 ? o & 7 : (o >> 1) & 3)) << 4)); }
    // m or n contiguous, k row `o`, piece `ch` along m or n
    __device__ static uint32_t at_mn(int o, int ch) { return (uint32_t)((ch >> 3) * (BK * 128) + o * 128 + (((ch & 7) ^ (o & 7)) << 4)); }
};

// ---- units of work -------------------------------------------------------------------------------------------

// One warp: turns group_ptr into the plan.
template <int MODE>
__device__ void make_plan(const Args& P, const Plan& plan) {
    const int lane = threadIdx.x & 31;
    auto clamp = [&](int v) { return (int)max(0LL, min((long long)v, P.n)); };
    int reached = clamp(P.ptr[0]), units = 0, slots = 0;
    for (int g0 = 0; g0 < P.groups; g0 += 32) {
        const int g = g0 + lane;
        int end = g < P.groups ? clamp(P.ptr[g + 1]) : 0;
        end = max(end, reached);
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, end, off);
            if (lane >= off) end = max(end, o);
        }
        int start = __shfl_up_sync(0xffffffffu, end, 1);
        if (lane == 0) start = reached;
        const int rows = end - start;
        int mine = 0;
        if (g < P.groups) mine = MODE == GRAD_W ? max(1, (int)(((long long)rows + P.chunk_rows - 1) / P.chunk_rows)) : (int)(((long long)rows + P.tile_n - 1) / P.tile_n);
        int sum = mine, slot_sum = MODE == GRAD_W && mine > 1 ? mine : 0;
        const int own_slots = slot_sum;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, sum, off), q = __shfl_up_sync(0xffffffffu, slot_sum, off);
            if (lane >= off) { sum += o; slot_sum += q; }
        }
        if (g < P.groups) {
            plan.start[g] = start;
            plan.unit[g] = units + sum - mine;
            if (MODE == GRAD_W) plan.slot[g] = slots + slot_sum - own_slots;
            if (g == P.groups - 1) {
                plan.start[P.groups] = end;
                plan.unit[P.groups] = units + sum;
                if (MODE == GRAD_W) plan.slot[P.groups] = slots + slot_sum;
            }
        }
        reached = __shfl_sync(0xffffffffu, end, 31);
        units += __shfl_sync(0xffffffffu, sum, 31);
        slots += __shfl_sync(0xffffffffu, slot_sum, 31);
    }
}

// One thread of one block: the groups whose chunks have to be added up.
__device__ __forceinline__ void list_multi(const Args& P, const Plan& plan) {
    int count = 0;
    for (int g = 0; g < P.groups; g++)
        if (plan.slot[g + 1] > plan.slot[g]) {
            P.multi[1 + 3 * count] = g;
            P.multi[2 + 3 * count] = plan.slot[g];
            P.multi[3 + 3 * count] = plan.slot[g + 1] - plan.slot[g];
            count++;
        }
    P.multi[0] = count;
}

// This block's units one after the other: every gridDim-th, without a division or a search per unit.
template <int MODE>
struct Walk {
    int t, r, g, dt, dr, tiles, all;               // row tile or chunk, (m, n) tile, group; steps from unit to unit
    __device__ __forceinline__ Walk(const Args& P, const Plan& plan) {
        tiles = P.m_tiles * (MODE == GRAD_W ? P.n_tiles : 1);
        t = blockIdx.x / tiles;
        r = blockIdx.x - t * tiles;
        dt = gridDim.x / tiles;
        dr = gridDim.x - dt * tiles;
        g = 0;
        all = plan.unit[P.groups];
    }
    __device__ __forceinline__ bool more() const { return t < all; }
    __device__ __forceinline__ void next() {
        t += dt;
        r += dr;
        if (r >= tiles) { r -= tiles; t++; }
    }
    __device__ __forceinline__ Unit unit(const Args& P, const Plan& plan) {
        while (plan.unit[g + 1] <= t) g++;
        Unit w;
        int mt = r, nt = 0;
        if (MODE == GRAD_W) {
            nt = r / P.m_tiles;
            mt = r - nt * P.m_tiles;
        }
        w.m0 = mt * TILE_M;
        w.n0 = nt * P.tile_n;
        w.g = g;
        w.chunk = t - plan.unit[g];
        w.chunks = plan.unit[g + 1] - plan.unit[g];
        const int step = MODE == GRAD_W ? P.chunk_rows : P.tile_n;
        w.row0 = (int)(plan.start[g] + (long long)w.chunk * step);
        w.rows = min(step, plan.start[g + 1] - w.row0);
        return w;
    }
};

// ---- register path -------------------------------------------------------------------------------------------

// One producer thread's share of an operand's tile: pieces of VW bytes (VE elements) along the contiguous side, neighbouring
// threads on neighbouring pieces, a thread's pieces all at the same place of a row and `step` rows apart.  VW divides the
// addresses and the row lengths, so a piece is inside its row or outside.
// TILE: the largest number of m or n; MN: m or n (not k) is the contiguous side; BIG: one of the launch's tiles is above 128.
template <typename T, int MODE, int VW, bool MN, int TILE, bool BIG>
struct Loader {
    using S = Shape<T, MODE>;
    static constexpr int VE = VW / (int)sizeof(T);
    static constexpr int BATCHES = VW == 2 && BIG ? 2 : 1;          // single 16-bit elements would fill the registers at once
    static constexpr int PIECES = TILE * S::BK / (PRODUCERS * VE * BATCHES);
    // With 8 rows (a swizzle period) or a multiple between a thread's pieces, known here, their places differ by constants.
    static constexpr int STEP = !MN ? PRODUCERS * VE / S::BK : TILE == TILE_M ? PRODUCERS * VE / TILE_M : 0;
    static constexpr bool EVEN = STEP > 0 && STEP % 8 == 0;
    using V = Pack<T, VW>;
    V v[PIECES];
    int first, step_log2, inner;         // this thread's first row, rows between its pieces (a power of two), element in the row
    int count;                           // its pieces of this tile
    int ends;                            // where its pieces that are worth storing end

    // tile: m or n of this launch's tiles (a power of two)
    __device__ __forceinline__ void init(int tile) {
        const int per_row_log2 = 31 - __clz((MN ? tile : S::BK) / VE), p = threadIdx.x & (PRODUCERS - 1);
        first = p >> per_row_log2;
        inner = (p & ((1 << per_row_log2) - 1)) * VE;
        step_log2 = 8 - per_row_log2;
        count = tile * S::BK / (PRODUCERS * VE);
    }
    // base: element (0, 0) of the tile in the row-major matrix, ld its row length; rows from outer_end and elements from
    // inner_end on are taken as 0
    __device__ __forceinline__ void load(const T* base, int ld, int outer_end, int inner_end, int batch) {
        const int step = STEP ? STEP : 1 << step_log2, skip = batch * PIECES;
        const int rows = (outer_end - first + step - 1) >> step_log2;
        // m and n past the end may hold anything (they make results that nobody stores), k past the end has to be 0
        ends = MN ? (inner < inner_end ? count : 0) : min(count, rows);
        const T* p = base + (long long)(first + skip * step) * ld + inner;
        const long long ahead = (long long)step * ld;
        const int have = inner < inner_end ? min(rows, count) - skip : 0;
        if (have >= PIECES) {
#pragma unroll
            for (int i = 0; i < PIECES; i++, p += ahead) load_now(v[i].raw, p);
        } else {
#pragma unroll
            for (int i = 0; i < PIECES; i++, p += ahead) {
                v[i] = V();
                if (i < have) load_now(v[i].raw, p);
            }
        }
    }
    __device__ static __forceinline__ uint32_t place(int o, int inner) { return (MN ? S::at_mn(o, inner >> 3) : S::at_k(o, inner >> 3)) + (inner & 7) * 2; }
    // the fp32 parts are bf16 numbers cut off, not rounded: x = x0 + x1 + x2 exactly
    __device__ __forceinline__ void store(uint32_t tile, int part_bytes, int batch) const {
        const int step = STEP ? STEP : 1 << step_log2;
        int o0 = first + batch * PIECES * step;
        asm volatile("" : "+r"(o0));                       // the pieces' places are computed here, not kept in registers
        const uint32_t at0 = tile + place(o0, inner);
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            if (i + batch * PIECES >= ends) break;
            const uint32_t at = EVEN ? at0 + i * STEP * (MN ? 128 : S::ROW) : tile + place(o0 + i * step, inner);
            if constexpr (S::F32) {
                uint32_t part[3][VE];                      // parts in the upper halves
#pragma unroll
                for (int e = 0; e < VE; e++) {
                    const uint32_t x0 = __float_as_uint(v[i].get(e));
                    const uint32_t x1 = __float_as_uint(__uint_as_float(x0) - __uint_as_float(x0 & 0xFFFF0000u));
                    part[0][e] = x0;
                    part[1][e] = x1;
                    part[2][e] = __float_as_uint(__uint_as_float(x1) - __uint_as_float(x1 & 0xFFFF0000u));
                }
#pragma unroll
                for (int s = 0; s < 3; s++) {
                    if constexpr (VE == 4)
                        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at + s * part_bytes), "r"(__byte_perm(part[s][0], part[s][1], 0x7632)),
                                     "r"(__byte_perm(part[s][2], part[s][3], 0x7632)) : "memory");
                    else if constexpr (VE == 2)
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + s * part_bytes), "r"(__byte_perm(part[s][0], part[s][1], 0x7632)) : "memory");
                    else
                        asm volatile("st.shared.b16 [%0], %1;" ::"r"(at + s * part_bytes), "h"((unsigned short)(part[s][0] >> 16)) : "memory");
                }
            } else if constexpr (VW == 16) {
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[i].raw.x), "r"(v[i].raw.y), "r"(v[i].raw.z), "r"(v[i].raw.w) : "memory");
            } else if constexpr (VW == 4) {
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(v[i].raw) : "memory");
            } else {
                asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"(v[i].raw) : "memory");
            }
        }
    }
};

// BIG: tiles of up to 256 rows; otherwise up to 64, whose single 16-bit elements fit a thread's registers at once.
template <typename T, int MODE, int VA, int VB, bool BIG>
__device__ __forceinline__ void produce(const Args& P, const Plan& plan, uint32_t ring, uint32_t kept, uint32_t full0, uint32_t empty0, uint32_t kept_full, uint32_t kept_free,
                        volatile int* abort_flag, int group) {
    using S = Shape<T, MODE>;
    const int b_part = S::b_part(P.tile_n), stage_bytes = S::stage(P.tile_n, P.keep);
    using LA = Loader<T, MODE, VA, S::A_MN, TILE_M, BIG>;
    using LB = Loader<T, MODE, VB, S::B_MN, BIG ? MAX_TILE_N : SMALL_TILE_N, BIG>;
    LA a;
    LB b;
    a.init(TILE_M);
    b.init(P.tile_n);
    unsigned c = 0;                                        // k-chunks of this block before this unit
    int s = 0;                                             // stage of the next k-chunk, whoever's
    unsigned phase = 1;                                    // parity of the stage's previous release
    bool first_round = true;
    auto advance = [&]() {
        if (++s == P.stages) { s = 0; phase ^= 1; first_round = false; }
    };
    int kept_g = -1, kept_m = 0;                           // whose A is kept
    unsigned kept_phase = 1;
    for (Walk<MODE> walk(P, plan); walk.more(); walk.next()) {
        const Unit w = walk.unit(P, plan);
        const int K = MODE == GRAD_W ? w.rows : P.K;
        const T *A, *B;
        int lda, ldb, n_left;
        const int m_left = P.M - w.m0;
        if (MODE == FORWARD) {                             // w[g] [K][M], x [n][K]
            lda = P.M; ldb = P.K;
            A = (const T*)P.a + (long long)w.g * P.K * P.M + w.m0;
            B = (const T*)P.b + (long long)w.row0 * ldb;
            n_left = w.rows;
        } else if (MODE == GRAD_X) {                       // w[g] [M][K], dy [n][K]
            lda = P.K; ldb = P.K;
            A = (const T*)P.a + ((long long)w.g * P.M + w.m0) * P.K;
            B = (const T*)P.b + (long long)w.row0 * ldb;
            n_left = w.rows;
        } else {                                           // dy [n][M], x [n][N]
            lda = P.M; ldb = P.N;
            A = (const T*)P.a + (long long)w.row0 * lda + w.m0;
            B = (const T*)P.b + (long long)w.row0 * ldb + w.n0;
            n_left = P.N - w.n0;
        }
        auto load_a = [&](int k0, int batch) {
            if (S::A_MN) a.load(A + (long long)k0 * lda, lda, min(S::BK, K - k0), m_left, batch);
            else a.load(A + k0, lda, min(TILE_M, m_left), K - k0, batch);
        };
        auto load_b = [&](int k0, int batch) {
            if (S::B_MN) b.load(B + (long long)k0 * ldb, ldb, min(S::BK, K - k0), n_left, batch);
            else b.load(B + k0, ldb, n_left, K - k0, batch);
        };
        if (P.keep && (w.g != kept_g || w.m0 != kept_m)) {
            // another A: both groups bring it, every other k-chunk each, when the last product with the old one is done
            if (kept_g >= 0 && !wait_or_abort<true>(P, kept_free, kept_phase, abort_flag, 2)) return;
            kept_g = w.g;
            kept_m = w.m0;
            kept_phase ^= 1;
            for (int k0 = group * S::BK; k0 < K; k0 += 2 * S::BK)
#pragma unroll 1
                for (int batch = 0; batch < LA::BATCHES; batch++) {
                    load_a(k0, batch);
                    a.store(kept + (k0 / S::BK) * (S::PARTS * S::A_PART), S::A_PART, batch);
                }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            bar_arrive(kept_full);
        }
        const int chunks = (K + S::BK - 1) / S::BK;
        int i = (c & 1) == (unsigned)group ? 0 : 1;        // this group's k-chunks of the unit: every other one
        if (i == 1 && chunks > 0) advance();
        for (; i < chunks; i += 2) {
            const int batches = P.keep ? LB::BATCHES : max(LA::BATCHES, LB::BATCHES);
#pragma unroll 1
            for (int batch = 0; batch < batches; batch++) {
                if (!P.keep && batch < LA::BATCHES) load_a(i * S::BK, batch);
                if (batch < LB::BATCHES) load_b(i * S::BK, batch);
                if (batch == 0 && !first_round && !wait_or_abort<true>(P, empty0 + 8 * s, phase, abort_flag, 2)) return;
                const uint32_t stage = ring + s * stage_bytes;
                if (!P.keep && batch < LA::BATCHES) a.store(stage, S::A_PART, batch);
                if (batch < LB::BATCHES) b.store(stage + (P.keep ? 0 : S::PARTS * S::A_PART), b_part, batch);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // visible to the tensor core
            bar_arrive(full0 + 8 * s);
            advance();
            if (i + 1 < chunks) advance();                 // the other group's
        }
        c += chunks;
    }
}

// ---- TMA path ------------------------------------------------------------------------------------------------

// One thread.  Boxes past the end of a matrix are not asked for; inside a box what lies past the end arrives as 0.
// Returns how many k-chunks were asked for.
template <typename T, int MODE>
__device__ long long issue_copies(const Args& P, const Plan& plan, const CUtensorMap* map_a, const CUtensorMap* map_b, uint32_t ring, uint32_t full0, uint32_t empty0,
                             volatile int* abort_flag) {
    using S = Shape<T, MODE>;
    constexpr int BOX = 64 * S::BK * 2;                    // bytes of a box of 64 m or n by BK
    const int stage_bytes = S::stage(P.tile_n, false);
    long long c = 0;
    int s = 0;
    unsigned phase = 1;
    bool ok = true;
    for (Walk<MODE> walk(P, plan); walk.more() && ok; walk.next()) {
        const Unit w = walk.unit(P, plan);
        const int K = MODE == GRAD_W ? w.rows : P.K;
        const int a_boxes = S::A_MN ? min(TILE_M / 64, (P.M - w.m0 + 63) / 64) : 1;
        const int b_boxes = S::B_MN ? min(P.tile_n / 64, (P.N - w.n0 + 63) / 64) : 1;
        const unsigned bytes = (S::A_MN ? a_boxes * BOX : S::A_PART) + (S::B_MN ? b_boxes * BOX : S::b_part(P.tile_n));
        for (int k0 = 0; k0 < K && ok; k0 += S::BK, c++) {
            if (c >= P.stages && !(ok = wait_or_abort(P, empty0 + 8 * s, phase, abort_flag, 2))) break;
            const uint32_t a = ring + s * stage_bytes, b = a + S::A_PART, bar = full0 + 8 * s;
            bar_expect(bar, bytes);
            if (MODE == FORWARD)
                for (int i = 0; i < a_boxes; i++) tma_3d(a + i * BOX, map_a, w.m0 + 64 * i, k0, w.g, bar);
            else if (MODE == GRAD_X)
                tma_3d(a, map_a, k0, w.m0, w.g, bar);
            else
                for (int i = 0; i < a_boxes; i++) tma_2d(a + i * BOX, map_a, w.m0 + 64 * i, w.row0 + k0, bar);
            if (MODE != GRAD_W) tma_2d(b, map_b, k0, w.row0, bar);
            else
                for (int i = 0; i < b_boxes; i++) tma_2d(b + i * BOX, map_b, w.n0 + 64 * i, w.row0 + k0, bar);
            if (++s == P.stages) { s = 0; phase ^= 1; }
        }
    }
    return c;
}

// The same thread, when the block gives up, whoever's wait ran out: what was asked for has to land before the block's shared
// memory goes to another.  Chunk j is in stage j % stages, and the stage's (j / stages)-th filling; all but the last filling
// of each stage had landed before the stage was asked for again.
__device__ __forceinline__ void await_copies(const Args& P, long long asked, uint32_t full0) {
    for (long long j = max(0LL, asked - P.stages); j < asked; j++) bar_wait(full0 + 8 * (int)(j % P.stages), (unsigned)(j / P.stages) & 1);
}

// ---- tensor core ---------------------------------------------------------------------------------------------

// Lanes 1 to 31 of the multiplying warp, for dw by TMA.  The last copies of a unit bring rows behind its last one.  Those up to
// the next multiple of 16, an instruction's k, count as 0 in both operands (a NaN there must not meet a 0 here); the others are
// not multiplied.  Lane 0 meets these lanes when the copies have landed and again when the rows are cleared.
template <typename T>
__device__ void clear_rows(const Args& P, const Plan& plan, unsigned char* ring) {
    using S = Shape<T, GRAD_W>;
    const int stage_bytes = S::stage(P.tile_n, false), boxes = (stage_bytes + S::BK * 128 - 1) / (S::BK * 128);
    unsigned chunks = 0;                                 // k-chunks up to and with this unit's last
    for (Walk<GRAD_W> walk(P, plan); walk.more(); walk.next()) {
        const Unit w = walk.unit(P, plan);
        chunks += (w.rows + S::BK - 1) / S::BK;
        const int rows = w.rows % S::BK, end = (rows + 15) / 16 * 16;
        if (rows == 0) continue;
        unsigned char* stage = ring + (chunks - 1) % P.stages * stage_bytes;
        __syncwarp();
        for (int x = 0; x < boxes; x++)
            for (int i = rows * 128 + ((threadIdx.x & 31) - 1) * 16; i < end * 128; i += 31 * 16) *reinterpret_cast<uint4*>(stage + x * S::BK * 128 + i) = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
    }
}
// Lane 0 after an expired wait: the others expect it at every clearing.
template <typename T>
__device__ void attend_clearings(const Args& P, const Plan& plan, int done) {
    for (Walk<GRAD_W> walk(P, plan); walk.more(); walk.next())
        if (walk.unit(P, plan).rows % Shape<T, GRAD_W>::BK && --done < 0) {
            __syncwarp();
            __syncwarp();
        }
}

// Lane 0 alone: a lane whose own wait has run out cannot then be missing where the warp's others wait for it.  (All lanes waiting
// and voting would do, too, and takes 60 ns more per k-chunk; so does one that keeps a flag instead of returning.)  Returns how
// many clearings there have been.
template <typename T, int MODE, bool TMA>
__device__ int multiply(const Args& P, const Plan& plan, uint32_t ring, uint32_t kept, uint32_t full0, uint32_t empty0, uint32_t ready0, uint32_t free0,
                         uint32_t kept_full, uint32_t kept_free, uint32_t tmem, volatile int* abort_flag) {
    using S = Shape<T, MODE>;
    constexpr bool CLEARS = TMA && MODE == GRAD_W;
    const int b_part = S::b_part(P.tile_n), stage_bytes = S::stage(P.tile_n, P.keep);
    constexpr uint32_t FORMAT = std::is_same<T, __half>::value ? 0u : 1u;       // f16 or bf16
    const uint32_t idesc0 = (1u << 4) | (FORMAT << 7) | (FORMAT << 10) | ((S::A_MN ? 1u : 0u) << 15) | ((S::B_MN ? 1u : 0u) << 16) | ((uint32_t)(TILE_M >> 4) << 24);
    constexpr uint32_t SW_K = S::ROW == 128 ? 2u : 4u, STRIDE_K = 8u * S::ROW;
    constexpr uint32_t STEP_K = 32u, STEP_MN = 2048u;                           // bytes from 16 k to the next 16
    auto desc_a = [&](uint32_t base) { return S::A_MN ? matrix_desc(base, S::BK * 128, 1024, 2) : matrix_desc(base, 16, STRIDE_K, SW_K); };
    auto desc_b = [&](uint32_t base) { return S::B_MN ? matrix_desc(base, S::BK * 128, 1024, 2) : matrix_desc(base, 16, STRIDE_K, SW_K); };
    constexpr uint32_t STEP_A = S::A_MN ? STEP_MN : STEP_K, STEP_B = S::B_MN ? STEP_MN : STEP_K;
    int s = 0, kept_g = -1, kept_m = 0;
    unsigned phase = 0, kept_phase = 0;
    int buf = 0;                                         // the next accumulator, and whether it has been used before
    unsigned used = 0;
    bool first_use = true;
    // pairs of parts, smallest products first
    constexpr int PAIRS = S::F32 ? 6 : 1;
    constexpr int PA[6] = {0, 1, 2, 0, 1, 0}, PB[6] = {2, 1, 0, 1, 0, 0};
    int done = 0;
    for (Walk<MODE> walk(P, plan); walk.more(); walk.next()) {
        const Unit w = walk.unit(P, plan);
        if (!TMA && P.keep && (w.g != kept_g || w.m0 != kept_m)) {
            if (kept_g >= 0) mma_commit(kept_free);      // everything so far has been issued: the old A is free when it is done
            kept_g = w.g;
            kept_m = w.m0;
            if (!wait_or_abort(P, kept_full, kept_phase, abort_flag, 1)) return done;
            kept_phase ^= 1;
        }
        const int K = MODE == GRAD_W ? w.rows : P.K;
        const int cols = MODE == GRAD_W ? min(P.tile_n, P.N - w.n0) : w.rows;
        const uint32_t idesc = idesc0 | ((uint32_t)((cols + 15) / 16 * 2) << 17);
        uint32_t d = 0;
        if constexpr (S::F32 && MODE != GRAD_W)
            if (P.pair) {
                // a stage is kept until both have landed: at least two
                if (!first_use && !wait_or_abort(P, free0 + 8 * buf, used, abort_flag, 4)) return done;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                d = tmem + (uint32_t)(buf * P.tile_n);
                const int s1 = s + 1 == P.stages ? 0 : s + 1;
                const uint64_t da[2] = {desc_a(kept), desc_a(kept + S::PARTS * S::A_PART)}, db[2] = {desc_b(ring + s * stage_bytes), desc_b(ring + s1 * stage_bytes)};
                auto issue = [&](int c, int first, int last) {
#pragma unroll
                    for (int i = first; i < last; i++)
#pragma unroll
                        for (int ks = 0; ks < S::BK / 16; ks++)
                            mma_f16(d, da[c] + ((PA[i] * S::A_PART + ks * STEP_A) >> 4), db[c] + ((PB[i] * b_part + ks * STEP_B) >> 4), idesc, c > 0 || i > 0 || ks > 0);
                };
                if (!wait_or_abort(P, full0 + 8 * s, phase, abort_flag, 1)) return done;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                issue(0, 0, PAIRS - 1);
                if (!wait_or_abort(P, full0 + 8 * s1, s1 == 0 ? phase ^ 1 : phase, abort_flag, 1)) return done;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                issue(1, 0, PAIRS - 1);
                issue(0, PAIRS - 1, PAIRS);
                mma_commit(empty0 + 8 * s);
                issue(1, PAIRS - 1, PAIRS);
                mma_commit(empty0 + 8 * s1);
                mma_commit(ready0 + 8 * buf);
                for (int i = 0; i < 2; i++)
                    if (++s == P.stages) { s = 0; phase ^= 1; }
                if (++buf == P.bufs) {
                    buf = 0;
                    if (!first_use) used ^= 1;
                    first_use = false;
                }
                continue;
            }
        int in_seg = 0;                                  // k0's place in its segment
        for (int k0 = 0; k0 == 0 || k0 < K; k0 += S::BK) {
            if (in_seg == 0) {
                if (!first_use && !wait_or_abort(P, free0 + 8 * buf, used, abort_flag, 4)) return done;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                d = tmem + (uint32_t)(buf * (P.split ? 2 : 1) * P.tile_n);
            }
            if (K <= 0) {                                // a group without rows: its results are 0 whatever the accumulator holds
                mma_commit(ready0 + 8 * buf);
                break;
            }
            const uint32_t stage0 = ring + s * stage_bytes;
            const uint32_t a = P.keep ? kept + (k0 / S::BK) * (S::PARTS * S::A_PART) : stage0, b = P.keep ? stage0 : stage0 + S::PARTS * S::A_PART;
            const uint64_t da = desc_a(a), db = desc_b(b);       // made before the wait: from its end to the next copies every cycle counts
            if (!wait_or_abort(P, full0 + 8 * s, phase, abort_flag, 1)) return done;
            if constexpr (CLEARS)
                if (K - k0 < S::BK) {
                    __syncwarp();
                    __syncwarp();
                    done++;
                }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int i = 0; i < PAIRS; i++) {
                const int pa = S::F32 ? PA[i] : 0, pb = S::F32 ? PB[i] : 0;
                const bool small = P.split && i < PAIRS - 1, first = i == 0 || (P.split && i == PAIRS - 1);
#pragma unroll
                for (int ks = 0; ks < S::BK / 16; ks++)
                    if (!CLEARS || ks * 16 < K - k0)
                        mma_f16(small ? d + P.tile_n : d, da + ((pa * S::A_PART + ks * STEP_A) >> 4), db + ((pb * b_part + ks * STEP_B) >> 4), idesc, in_seg > 0 || !first || ks > 0);
            }
            mma_commit(empty0 + 8 * s);              // the stage may be filled again once these are done
            if (in_seg + S::BK >= P.seg || k0 + S::BK >= K) mma_commit(ready0 + 8 * buf);      // the accumulator is complete
            if (++s == P.stages) { s = 0; phase ^= 1; }
            const bool full = in_seg + S::BK >= P.seg;
            if ((full || k0 + S::BK >= K) && ++buf == P.bufs) {
                buf = 0;
                if (!first_use) used ^= 1;
                first_use = false;
            }
            in_seg = full ? 0 : in_seg + S::BK;
        }
        if (K <= 0 && ++buf == P.bufs) {
            buf = 0;
            if (!first_use) used ^= 1;
            first_use = false;
        }
    }
    return done;
}

// ---- results -------------------------------------------------------------------------------------------------

__device__ __forceinline__ void read_columns(uint32_t (&r)[16], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
}
__device__ __forceinline__ void write_columns(uint32_t at, const float (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
                 ::"f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]),
                   "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "r"(at)
                 : "memory");
}
// SHARES: warps per quarter of the tensor memory's lanes, which take every SHARES-th block of output rows.  A sum of several
// segments is added up in fp32, rounding to nearest (the tensor core cuts what it adds): an fp32 result in the output itself
// (only this thread writes the element, and it is still in L2), a 16-bit one in columns of tensor memory behind the
// accumulators, which this warp alone touches, so that it is rounded to 16 bits once.
template <typename T, int MODE, int SHARES>
__device__ void store_results(const Args& P, const Plan& plan, uint32_t ready0, uint32_t free0, uint32_t tmem, volatile int* abort_flag, int first_warp) {
    using O = typename std::conditional<MODE == GRAD_W, float, T>::type;
    constexpr bool IN_OUTPUT = std::is_same<O, float>::value;
    constexpr int CW = 16;                                                     // output rows per block
    const int quarter = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;       // a warp reads tensor-memory lanes 32 * (warp % 4) ..
    const int share = SHARES > 1 ? ((int)(threadIdx.x >> 5) - first_warp) >> 2 : 0;
    int buf = 0;
    unsigned used = 0;
    for (Walk<MODE> walk(P, plan); walk.more(); walk.next()) {
        const Unit w = walk.unit(P, plan);
        const int K = MODE == GRAD_W ? w.rows : P.K;
        const int m = w.m0 + quarter * 32 + lane;
        const int cols = MODE == GRAD_W ? min(P.tile_n, P.N - w.n0) : w.rows;
        O* base;
        if (MODE == GRAD_W)
            base = (O*)(w.chunks > 1 ? P.partial + (long long)(plan.slot[w.g] + w.chunk) * P.N * P.M : (float*)P.out + (long long)w.g * P.N * P.M) + (long long)w.n0 * P.M + m;
        else
            base = (O*)P.out + (long long)w.row0 * P.M + m;
        for (int k0 = 0; k0 == 0 || k0 < K; k0 += P.seg) {
            if (!__all_sync(0xffffffffu, wait_or_abort(P, ready0 + 8 * buf, used, abort_flag, 3))) return;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t at0 = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * (P.split ? 2 : 1) * P.tile_n);
            auto block = [&](int c0, float (&v)[CW]) {
                uint32_t r[CW];
                read_columns(r, at0 + c0);
                if constexpr (Shape<T, MODE>::F32) {
                    if (P.split) {
                        uint32_t q[CW];
                        read_columns(q, at0 + P.tile_n + c0);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int j = 0; j < CW; j++) v[j] = __uint_as_float(r[j]) + __uint_as_float(q[j]);
                        return;
                    }
                }
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int j = 0; j < CW; j++) v[j] = __uint_as_float(r[j]);
            };
            auto store = [&](int c0, float (&v)[CW]) {
                if (m >= P.M) return;
                O* out = base + (long long)c0 * P.M;
                if (MODE == GRAD_W && K <= 0) {
#pragma unroll
                    for (int j = 0; j < CW; j++) v[j] = 0.f;          // a group without rows: nothing was accumulated
                }
                if constexpr (IN_OUTPUT) {
                    if (k0 > 0) {
                        const O* before = out;
                        float b[CW];
#pragma unroll
                        for (int j = 0; j < CW; j++, before += P.M) b[j] = c0 + j < cols ? (float)*before : 0.f;
#pragma unroll
                        for (int j = 0; j < CW; j++) v[j] += b[j];
                    }
                }
                if (c0 + CW <= cols) {
#pragma unroll
                    for (int j = 0; j < CW; j++, out += P.M) *out = from_f32<O>(v[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < CW; j++, out += P.M)
                        if (c0 + j < cols) *out = from_f32<O>(v[j]);
                }
            };
            const bool sum = !IN_OUTPUT && K > P.seg;
            const uint32_t sum0 = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(P.bufs * P.tile_n);
            for (int c0 = CW * share; c0 < cols; c0 += CW * SHARES) {
                float v[CW];
                block(c0, v);
                if (sum && k0 > 0) {
                    uint32_t r[CW];
                    read_columns(r, sum0 + c0);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int j = 0; j < CW; j++) v[j] += __uint_as_float(r[j]);
                }
                if (sum && k0 + P.seg < K) write_columns(sum0 + c0, v);
                else store(c0, v);
            }
            if (sum) asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");        // the next segment reads them
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            bar_arrive(free0 + 8 * buf);
            if (++buf == P.bufs) { buf = 0; used ^= 1; }
        }
    }
}

// ---- kernel --------------------------------------------------------------------------------------------------

// Warps per quarter of tensor memory's lanes that store results, and threads of a block.
template <int MODE, bool TMA>
struct Roles {
    static constexpr int SHARES = TMA ? 2 : 1, THREADS = (TMA ? 32 : 2 * PRODUCERS) + 32 + 128 * SHARES;
};

template <typename T, int MODE, bool TMA, int VA, int VB, bool BIG>
__global__ void __launch_bounds__((Roles<MODE, TMA>::THREADS), 1)
grouped_kernel(const Args P, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    using S = Shape<T, MODE>;
    unsigned char* kept = ring + (size_t)P.stages * S::stage(P.tile_n, P.keep);
    int* lists = reinterpret_cast<int*>(kept + (P.keep ? (size_t)((P.K + S::BK - 1) / S::BK) * S::PARTS * S::A_PART : 0));
    const Plan plan{lists, lists + P.groups + 1, lists + 2 * (P.groups + 1)};
    __shared__ unsigned long long bars[2 * MAX_STAGES + 7];
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;                // which wait ran out first in this block; 0: none
    constexpr int PRODUCER_WARPS = TMA ? 1 : 2 * PRODUCERS / 32, SHARES = Roles<MODE, TMA>::SHARES;
    const int warp = threadIdx.x >> 5;
    const uint32_t full0 = smem_addr(bars), empty0 = full0 + 8 * MAX_STAGES, ready0 = empty0 + 8 * MAX_STAGES, free0 = ready0 + 16,
                   drained = free0 + 16, kept_full = drained + 8, kept_free = kept_full + 8;

    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < P.stages; s++) {
            bar_init(full0 + 8 * s, TMA ? 1 : PRODUCERS);
            bar_init(empty0 + 8 * s, 1);
        }
        for (int b = 0; b < 2; b++) {
            bar_init(ready0 + 8 * b, 1);
            bar_init(free0 + 8 * b, 128 * SHARES);
        }
        bar_init(drained, 1);
        bar_init(kept_full, 2 * PRODUCERS);
        bar_init(kept_free, 1);
        bar_init_fence();
    }
    if (warp == PRODUCER_WARPS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(P.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (MODE == GRAD_W) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp == PRODUCER_WARPS + 1) make_plan<MODE>(P, plan);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;
    long long asked = 0;                            // k-chunks that this thread has asked for by TMA

    if (warp < PRODUCER_WARPS) {
        if constexpr (TMA) {
            if (threadIdx.x == 0) asked = issue_copies<T, MODE>(P, plan, &map_a, &map_b, smem_addr(ring), full0, empty0, &s_abort);
        } else {
            produce<T, MODE, VA, VB, BIG>(P, plan, smem_addr(ring), smem_addr(kept), full0, empty0, kept_full, kept_free, &s_abort, threadIdx.x / PRODUCERS);
        }
    } else if (warp == PRODUCER_WARPS) {
        if ((threadIdx.x & 31) == 0) {
            const int done = multiply<T, MODE, TMA>(P, plan, smem_addr(ring), smem_addr(kept), full0, empty0, ready0, free0, kept_full, kept_free, tmem, &s_abort);
            if (TMA && MODE == GRAD_W && s_abort) attend_clearings<T>(P, plan, done);
        } else if (TMA && MODE == GRAD_W) {
            clear_rows<T>(P, plan, ring);
        }
    } else {
        if (MODE == GRAD_W && blockIdx.x == 0 && P.multi && warp == PRODUCER_WARPS + 1 && (threadIdx.x & 31) == 0) {
            list_multi(P, plan);
        }
        __syncwarp();
        store_results<T, MODE, SHARES>(P, plan, ready0, free0, tmem, &s_abort, PRODUCER_WARPS + 1);
    }
    __syncwarp();                                   // lane 0 of the copying and of the multiplying warp comes last
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (TMA && threadIdx.x == 0 && s_abort) await_copies(P, asked, full0);
    if (warp == PRODUCER_WARPS) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (s_abort) {                              // instructions still under way read shared memory and write tensor memory
            if ((threadIdx.x & 31) == 0) {
                mma_commit(drained);
                bar_wait(drained, 0);
            }
            __syncwarp();
        }
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P.tmem_cols) : "memory");
    }
}

// ---- narrow products on the fp32 pipes ---------------------------------------------------------------------------

constexpr int NARROW_ROWS = 128;

// q / d for q < 2^31
struct Divide {
    unsigned d, magic, shift;
    __device__ __forceinline__ unsigned operator()(unsigned q) const { return (__umulhi(q, magic) + q) >> shift; }
};
Divide divide_by(unsigned d) {
    Divide r{d, 0, 0};
    while ((1ull << r.shift) < d) r.shift++;
    r.magic = (unsigned)(((1ull << 32) * ((1ull << r.shift) - d)) / d + 1);
    return r;
}

// `rows` rows of `len` elements, one run of memory, to shared memory as fp32 rows `pitch` apart; 16 bytes at a time where the
// address allows.  A thread's loads are issued in batches before the first is used, and a vector is told its row once.
template <typename T, int THREADS>
__device__ __forceinline__ void lay_rows(float* dst, int pitch, const T* p, int rows, int len, const Divide& by_len) {
    constexpr int VE = 16 / (int)sizeof(T), UV = 4, US = 8;
    const int count = rows * len;
    int done = 0;
    if ((uint64_t)p % 16 == 0) {
        const int vecs = count / VE;
        for (int i0 = threadIdx.x; i0 < vecs; i0 += THREADS * UV) {
            Pack<T, 16> v[UV];
#pragma unroll
            for (int u = 0; u < UV; u++)
                if (i0 + u * THREADS < vecs) load_now(v[u].raw, p + (i0 + u * THREADS) * VE);
#pragma unroll
            for (int u = 0; u < UV; u++)
                if (i0 + u * THREADS < vecs) {
                    const int i = (i0 + u * THREADS) * VE, r = by_len(i);
                    int c = i - r * len;
                    float* d = dst + r * pitch + c;
#pragma unroll
                    for (int e = 0; e < VE; e++) {
                        *d++ = v[u].get(e);
                        if (++c == len) { c = 0; d += pitch - len; }
                    }
                }
        }
        done = vecs * VE;
    }
    for (int i0 = done + threadIdx.x; i0 < count; i0 += THREADS * US) {
        T v[US];
#pragma unroll
        for (int u = 0; u < US; u++)
            if (i0 + u * THREADS < count) v[u] = __ldg(p + i0 + u * THREADS);
#pragma unroll
        for (int u = 0; u < US; u++)
            if (i0 + u * THREADS < count) {
                const int i = i0 + u * THREADS, r = by_len(i);
                dst[r * pitch + (i - r * len)] = to_f32(v[u]);
            }
    }
}

// out[row, 0..M) = sum_k in[row, k] * w[g](k, m), M <= MC, a thread per row and its columns in registers.  A block's rows are
// one run of memory in and out; in shared memory they are an odd number of words apart, so neighbouring threads read different
// banks, and the weight's row k is read by all threads at once.
template <typename T, int MODE, int MC>
__global__ void __launch_bounds__(NARROW_ROWS, 8) narrow_rows_kernel(const Args P, const Divide by_k) {
    extern __shared__ __align__(16) float narrow_smem[];
    const int K = P.K, M = P.M, pitch = K | 1, t = threadIdx.x;
    int* lists = reinterpret_cast<int*>(narrow_smem);
    const Plan plan{lists, lists + P.groups + 1, nullptr};
    float* w = narrow_smem + (2 * (P.groups + 1) + 3) / 4 * 4;        // [K][MC]
    float* x = w + K * MC;                                          // [rows][pitch], then the results
    if (t < 32) make_plan<MODE>(P, plan);
    __syncthreads();
    int kept_g = -1;
    for (Walk<MODE> walk(P, plan); walk.more(); walk.next()) {
        const Unit u = walk.unit(P, plan);
        if (u.g != kept_g) {
            kept_g = u.g;
            const T* wg = (const T*)P.a + (long long)u.g * K * M;
            for (int i = t; i < K * MC; i += NARROW_ROWS) {
                const int k = i / MC, m = i - k * MC;
                w[i] = m < M ? to_f32(MODE == FORWARD ? wg[k * M + m] : wg[m * K + k]) : 0.f;
            }
        }
        lay_rows<T, NARROW_ROWS>(x, pitch, (const T*)P.b + (long long)u.row0 * K, u.rows, K, by_k);
        __syncthreads();
        T* out = (T*)P.out + (long long)u.row0 * M;
        float acc[MC];
#pragma unroll
        for (int m = 0; m < MC; m++) acc[m] = 0.f;
        const float* xr = x + t * pitch;
        if (t < u.rows)
#pragma unroll 4
            for (int k = 0; k < K; k++) {
                const float v = xr[k];
#pragma unroll
                for (int m = 0; m < MC; m += 4) {
                    const float4 q = *reinterpret_cast<const float4*>(w + k * MC + m);
                    acc[m] = fmaf(v, q.x, acc[m]);
                    acc[m + 1] = fmaf(v, q.y, acc[m + 1]);
                    acc[m + 2] = fmaf(v, q.z, acc[m + 2]);
                    acc[m + 3] = fmaf(v, q.w, acc[m + 3]);
                }
            }
        // through shared memory, so that the block's rows leave as the one run they are
        __syncthreads();
        T* y = reinterpret_cast<T*>(x);
        if (t < u.rows)
#pragma unroll
            for (int m = 0; m < MC; m++)
                if (m < M) y[t * M + m] = from_f32<T>(acc[m]);
        __syncthreads();
        for (int i = t; i < u.rows * M; i += NARROW_ROWS) out[i] = y[i];
        __syncthreads();
    }
}

// At most 8 columns, any number of terms: a warp takes 4 rows, its lanes VE neighbouring terms each, so x is streamed in whole
// lines.  KEEP: the weight lies in shared memory, a row per column, as fp32 (read without conflicts, once for the 4 rows);
// otherwise (more terms than fit) it comes from the caches.  Bound by reading x.
constexpr int DOT_ROWS = 4, DOT_COLS = 8, DOT_THREADS = 256, DOT_KEEP_BYTES = 100 * 1024;
template <typename T, int MODE, int VB, int MC, bool KEEP>
__global__ void __launch_bounds__(DOT_THREADS) row_dots_kernel(const Args P) {
    constexpr int VE = VB / (int)sizeof(T);
    extern __shared__ __align__(16) float narrow_smem[];
    const int K = P.K, M = P.M, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pitch = (K + 3) / 4 * 4;
    int* lists = reinterpret_cast<int*>(narrow_smem);
    const Plan plan{lists, lists + P.groups + 1, nullptr};
    float* w = narrow_smem + (2 * (P.groups + 1) + 3) / 4 * 4;        // KEEP: [MC][pitch]
    if (warp == 0) make_plan<MODE>(P, plan);
    __syncthreads();
    int kept_g = -1;
    for (Walk<MODE> walk(P, plan); walk.more(); walk.next()) {
        const Unit u = walk.unit(P, plan);
        const T* wg = (const T*)P.a + (long long)u.g * K * M;
        if (KEEP && u.g != kept_g) {
            kept_g = u.g;
            __syncthreads();
            for (int m = 0; m < MC; m++)
                for (int k = threadIdx.x; k < K; k += DOT_THREADS)
                    w[m * pitch + k] = m < M ? to_f32(MODE == FORWARD ? wg[(long long)k * M + m] : wg[(long long)m * K + k]) : 0.f;
            __syncthreads();
        }
        for (int r0 = warp * DOT_ROWS; r0 < u.rows; r0 += DOT_THREADS / 32 * DOT_ROWS) {
            const T* x = (const T*)P.b + ((long long)u.row0 + r0) * K;
            const int rows = min(DOT_ROWS, u.rows - r0);
            float acc[DOT_ROWS][MC];
#pragma unroll
            for (int r = 0; r < DOT_ROWS; r++)
#pragma unroll
                for (int m = 0; m < MC; m++) acc[r][m] = 0.f;
            for (int k = lane * VE; k < K; k += 32 * VE) {
                Pack<T, VB> v[DOT_ROWS];
#pragma unroll
                for (int r = 0; r < DOT_ROWS; r++)
                    if (r < rows) v[r].raw = __ldcs(reinterpret_cast<const typename Pack<T, VB>::R*>(x + (long long)r * K + k));
#pragma unroll
                for (int m = 0; m < MC; m++) {
                    float q[VE];
                    if constexpr (KEEP) {
                        const float* wk = w + m * pitch + k;
                        if constexpr (VE % 4 == 0) {
#pragma unroll
                            for (int e = 0; e < VE; e += 4) *reinterpret_cast<float4*>(&q[e]) = *reinterpret_cast<const float4*>(wk + e);
                        } else {
#pragma unroll
                            for (int e = 0; e < VE; e++) q[e] = wk[e];
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < VE; e++)
                            q[e] = m < M ? to_f32(__ldg(MODE == FORWARD ? wg + (long long)(k + e) * M + m : wg + (long long)m * K + k + e)) : 0.f;
                    }
#pragma unroll
                    for (int r = 0; r < DOT_ROWS; r++)
#pragma unroll
                        for (int e = 0; e < VE; e++) acc[r][m] = fmaf(v[r].get(e), q[e], acc[r][m]);
                }
            }
            // lane r * MC + m keeps the sum of its row and column
            float mine = 0.f;
#pragma unroll
            for (int r = 0; r < DOT_ROWS; r++)
#pragma unroll
                for (int m = 0; m < MC; m++) {
                    const float s = warp_sum(acc[r][m]);
                    if (lane == r * MC + m) mine = s;
                }
            const int r = lane / MC, m = lane % MC;
            if (r < rows && m < M) ((T*)P.out)[((long long)u.row0 + r0 + r) * M + m] = from_f32<T>(mine);
        }
    }
}

// dw of a weight of at most 256 blocks of 4 x 4 (64 x 64): P.tile_n rows of x and dy at a time in shared memory, rows dealt to warps, each lane keeping up
// to 4 blocks of 4 x 4 elements in registers (two 16-byte reads for 16 multiply-adds); weights of more than 128 such blocks
// are dealt to two sets of warps.  The warps' sums meet in shared memory in their order, a float4 per lane side by side (element by
// element at the weight's own pitch that cost more than the products).  856 x 64 -> 64 fp32 in 2 groups 16 us, 50,000 x 11 -> 132 38 us
// (with scalar sums and rounds of 12 KiB throughout: 28 and 78).
constexpr int NW_THREADS = 256;
template <typename T, int TL>
__global__ void __launch_bounds__(NW_THREADS, TL == 1 ? 4 : TL == 2 ? 3 : 2) narrow_weight_kernel(const Args P, const Divide by_k, const Divide by_m) {
    extern __shared__ __align__(16) float narrow_smem[];
    const int K = P.N, M = P.M, kq = (K + 3) / 4, mq = (M + 3) / 4, kp = kq * 4, mp = mq * 4;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    int* lists = reinterpret_cast<int*>(narrow_smem);
    const Plan plan{lists, lists + P.groups + 1, lists + 2 * (P.groups + 1)};
    const int step = P.tile_n;
    float* x = narrow_smem + (3 * (P.groups + 1) + 3) / 4 * 4;        // [step][kp]
    float* y = x + step * kp;                                       // [step][mp]
    float4* sums = reinterpret_cast<float4*>(y + step * mp);        // [4 rows of a block][blocks]: lanes side by side
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp == 0) make_plan<GRAD_W>(P, plan);
    for (int i = t; i < step * (kp + mp); i += NW_THREADS) x[i] = 0.f;     // the columns past K and M stay 0
    __syncthreads();
    if (blockIdx.x == 0 && t == 0 && P.multi) list_multi(P, plan);
    const int blocks = kq * mq, sets = blocks > 32 * TL ? 2 : 1, set = warp % sets, row_warp = warp / sets, row_warps = NW_THREADS / 32 / sets;
    for (Walk<GRAD_W> walk(P, plan); walk.more(); walk.next()) {
        const Unit u = walk.unit(P, plan);
        float acc[TL][4][4];
        int kb[TL], mb[TL];
#pragma unroll
        for (int i = 0; i < TL; i++) {
            const int b = min((set * TL + i) * 32 + lane, blocks - 1);
            kb[i] = b / mq * 4;
            mb[i] = b % mq * 4;
#pragma unroll
            for (int a = 0; a < 4; a++)
#pragma unroll
                for (int c = 0; c < 4; c++) acc[i][a][c] = 0.f;
        }
        for (int r0 = 0; r0 < u.rows; r0 += step) {
            const int rows = min(step, u.rows - r0);
            lay_rows<T, NW_THREADS>(x, kp, (const T*)P.b + ((long long)u.row0 + r0) * K, rows, K, by_k);
            lay_rows<T, NW_THREADS>(y, mp, (const T*)P.a + ((long long)u.row0 + r0) * M, rows, M, by_m);
            __syncthreads();
            for (int r = row_warp; r < rows; r += row_warps) {
#pragma unroll
                for (int i = 0; i < TL; i++) {
                    if ((set * TL + i) * 32 >= blocks) break;
                    const float4 a = *reinterpret_cast<const float4*>(x + r * kp + kb[i]), b = *reinterpret_cast<const float4*>(y + r * mp + mb[i]);
                    const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                    for (int p = 0; p < 4; p++)
#pragma unroll
                        for (int q = 0; q < 4; q++) acc[i][p][q] = fmaf(av[p], bv[q], acc[i][p][q]);
                }
            }
            __syncthreads();
        }
        for (int rw = 0; rw < row_warps; rw++) {
            if (row_warp == rw) {
#pragma unroll
                for (int i = 0; i < TL; i++) {
                    const int b = (set * TL + i) * 32 + lane;
                    if (b >= blocks) break;
#pragma unroll
                    for (int p = 0; p < 4; p++) {
                        float4 s = rw ? sums[p * blocks + b] : make_float4(0.f, 0.f, 0.f, 0.f);
                        s.x += acc[i][p][0];
                        s.y += acc[i][p][1];
                        s.z += acc[i][p][2];
                        s.w += acc[i][p][3];
                        sums[p * blocks + b] = s;
                    }
                }
            }
            __syncthreads();
        }
        float* out = u.chunks > 1 ? P.partial + (long long)(plan.slot[u.g] + u.chunk) * K * M : (float*)P.out + (long long)u.g * K * M;
        for (int i = t; i < K * M; i += NW_THREADS) {
            const int k = (int)by_m(i), m = i - k * M;
            out[i] = reinterpret_cast<const float*>(sums + (k & 3) * blocks + (k >> 2) * mq + (m >> 2))[m & 3];
        }
        __syncthreads();
    }
}

// dw of the groups that were cut into chunks: 128 elements per block, 8 warps take every 8th chunk, then meet in order.
__global__ void __launch_bounds__(256) grouped_reduce_kernel(float* __restrict__ dw, const float* __restrict__ partial, const int* __restrict__ multi, long long size,
                                                             int vec_ok) {
    __shared__ float4 part[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");       // the kernel before this one has written what is read here
    for (int i = blockIdx.y; i < multi[0]; i += gridDim.y) {
        const int g = multi[1 + 3 * i], slot = multi[2 + 3 * i], count = multi[3 + 3 * i];
        for (long long e0 = (long long)blockIdx.x * 128; e0 < size; e0 += (long long)gridDim.x * 128) {
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            if (vec_ok) {
                const long long e = e0 + 4 * lane;
                if (e < size) {
                    const float* p = partial + (slot + warp) * size + e;
#pragma unroll 4
                    for (int c = warp; c < count; c += 8, p += 8 * size) {
                        const float4 v = __ldcs(reinterpret_cast<const float4*>(p));
                        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
                    }
                }
            } else {
                const long long e = e0 + lane;
                const float* p = partial + (slot + warp) * size + e;
                const bool b0 = e < size, b1 = e + 32 < size, b2 = e + 64 < size, b3 = e + 96 < size;
#pragma unroll 4
                for (int c = warp; c < count; c += 8, p += 8 * size) {
                    if (b0) s.x += __ldcs(p);
                    if (b1) s.y += __ldcs(p + 32);
                    if (b2) s.z += __ldcs(p + 64);
                    if (b3) s.w += __ldcs(p + 96);
                }
            }
            part[warp][lane] = s;
            __syncthreads();
            if (threadIdx.x < 128) {
                const int l = vec_ok ? threadIdx.x / 4 : threadIdx.x % 32, q = vec_ok ? threadIdx.x % 4 : threadIdx.x / 32;
                float t = 0.f;
#pragma unroll
                for (int w = 0; w < 8; w++) t += reinterpret_cast<const float*>(&part[w][l])[q];
                if (e0 + threadIdx.x < size) dw[g * size + e0 + threadIdx.x] = t;
            }
            __syncthreads();
        }
    }
}

// ---- launches ------------------------------------------------------------------------------------------------

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// Looked up through the runtime, so that the library does not link against the driver library.
EncodeTiledFn encode_tiled() {
    static const EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

// A row-major tensor of 16-bit elements with `dims` dimensions (innermost first), read in boxes of 64 by `rows`, 128-byte
// swizzled.
int make_map(CUtensorMap* map, const void* base, bool bf16, int dims, cuuint64_t d0, cuuint64_t d1, cuuint64_t d2, int rows) {
    const cuuint64_t dim[3] = {d0, d1, d2}, stride[2] = {d0 * 2, d0 * d1 * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)rows, 1}, step[3] = {1, 1, 1};
    const CUresult r = encode_tiled()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, dims, const_cast<void*>(base), dim, stride, box,
                                      step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(MGGB_ERR_CUDA, "grouped_dense: cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return MGGB_OK;
}

template <typename T, int MODE, bool TMA, int VA, int VB, bool BIG>
int launch_tiles(Args P, const CUtensorMap& map_a, const CUtensorMap& map_b, long long max_units, cudaStream_t st) {
    using S = Shape<T, MODE>;
    const int lists = (P.groups + 1) * 4 * (MODE == GRAD_W ? 3 : 2);
    const int room = SMEM_BUDGET - 1024 - lists;
    // The weight of a node type is used for many row tiles: where it is small, it is brought and cut into its parts once.
    const int kept = MODE == GRAD_W ? 0 : (int)std::min<long long>(1 << 30, (long long)((P.K + S::BK - 1) / S::BK) * S::PARTS * S::A_PART);
    P.keep = !TMA && MODE != GRAD_W && room - kept >= 2 * S::stage(P.tile_n, true) ? 1 : 0;
    P.stages = std::min(MAX_STAGES, (room - (P.keep ? kept : 0)) / S::stage(P.tile_n, P.keep));
    // The tensor core cuts what it adds at the accumulator's last places instead of rounding, always towards zero.  Measured per
    // instruction, where it is most (terms of one sign, products of 22 bits): 2e-7 of the accumulator, whose mean is half its
    // end's size.  Products of two bf16 numbers have 16 bits and lose next to nothing until the sum is 2^8 times their size.
    //   fp32: the five small products have an accumulator of their own, whose cuts do not count, and the sum is handed over every
    //       512 terms: 2e-7 of a sum of one sign, 5e-7 in the norm of mixed signs.  In one accumulator 128 terms lose 3e-6 and
    //       0.9e-6.  The second accumulator's price: 600,000 x 128 -> 128 149 us instead of 120, since two pairs of 256 rows do
    //       not fit tensor memory and the next tile waits until one has been stored.  Up to 64 terms, two k-chunks, one
    //       accumulator is as exact: all small products come first (1e-7; 600,000 x 64 -> 64 81 us, 103 with a second one)
    //   dw of 16-bit rows: handed over every 768 terms: f16 4e-6 and 0.9e-6, bf16 1e-7 and 5e-7 (every 256 would divide f16's
    //       by three, but each time dw is read and written: 16,384 x 2048 -> 2048 271 us instead of 171)
    //   16-bit results: every 2048 terms, 128 instructions: 1.3e-5, a fortieth of f16's half step of 4.9e-4.  Without an end
    //       65,536 terms would lose 4.1e-4.  8192 x 4096 -> 2048 bf16 in 4 groups 160 us (151 without)
    P.pair = S::F32 && MODE != GRAD_W && P.K > S::BK && P.K <= 2 * S::BK && P.keep ? 1 : 0;
    P.split = S::F32 && (MODE == GRAD_W || P.K > S::BK) && !P.pair ? 1 : 0;
    P.seg = S::F32 ? 512 : MODE == GRAD_W ? 768 : 2048;
    const unsigned wide = (P.split ? 2u : 1u) * P.tile_n, sum = !S::F32 && MODE != GRAD_W && P.K > P.seg ? P.tile_n : 0;
    P.bufs = 2 * wide + sum <= 512 ? 2 : 1;
    P.tmem_cols = 32;
    while (P.tmem_cols < P.bufs * wide + sum) P.tmem_cols <<= 1;
    const int smem = 1024 + P.stages * S::stage(P.tile_n, P.keep) + (P.keep ? kept : 0) + lists;
    const auto kernel = grouped_kernel<T, MODE, TMA, VA, VB, BIG>;
    MGGB_CUDA((allow_shared<grouped_kernel<T, MODE, TMA, VA, VB, BIG>>()));
    // a multiple of the column tiles, so that a block stays with one of them (and its part of the weight)
    const int sms = sm_count();
    const unsigned grid = (unsigned)std::min<long long>(max_units, P.keep && P.m_tiles < sms ? sms / P.m_tiles * P.m_tiles : sms);
    kernel<<<grid, Roles<MODE, TMA>::THREADS, smem, st>>>(P, map_a, map_b);
    MGGB_CUDA(cudaGetLastError());
    return MGGB_OK;
}

template <typename T, int MODE, bool TMA, int VA, int VB>
int launch(const Args& P, const CUtensorMap& map_a, const CUtensorMap& map_b, long long max_units, cudaStream_t st) {
    constexpr bool SINGLES = VA == 2 || VB == 2;            // 16-bit elements one by one
    if (!SINGLES || P.tile_n > SMALL_TILE_N) return launch_tiles<T, MODE, TMA, VA, VB, true>(P, map_a, map_b, max_units, st);
    return launch_tiles<T, MODE, TMA, VA, VB, !SINGLES>(P, map_a, map_b, max_units, st);
}

// The widest loads that never straddle the end of a row: 16 bytes, 8 (fp32 only) or 4, or single elements.
template <typename T>
int load_width(const void* p, int row) {
    const int a = common_alignment({(uint64_t)p, (uint64_t)row * sizeof(T)});
    return a == 8 && sizeof(T) == 2 ? 4 : std::max(a, (int)sizeof(T));
}

template <typename T, int MODE, int VA>
int launch_b(const Args& P, int vb, const CUtensorMap& none, long long max_units, cudaStream_t st) {
    if (vb == 16) return launch<T, MODE, false, VA, 16>(P, none, none, max_units, st);
    if (sizeof(T) == 4 && vb == 8) return launch<T, MODE, false, VA, sizeof(T) == 4 ? 8 : 4>(P, none, none, max_units, st);
    if (vb >= 4) return launch<T, MODE, false, VA, 4>(P, none, none, max_units, st);
    return launch<T, MODE, false, VA, (int)sizeof(T)>(P, none, none, max_units, st);
}

// a: the matrix behind A; b: behind B.  Picks the path by what the addresses and row lengths allow.
template <typename T, int MODE>
int dispatch(const Args& P, long long max_units, cudaStream_t st) {
    using S = Shape<T, MODE>;
    const int la = MODE == GRAD_X ? P.K : P.M, lb = MODE == GRAD_W ? P.N : P.K;         // row lengths
    const int va = load_width<T>(P.a, la), vb = load_width<T>(P.b, lb);
    CUtensorMap map_a, map_b;
    memset(&map_a, 0, sizeof(map_a));
    memset(&map_b, 0, sizeof(map_b));
    if constexpr (!S::F32) {
        if (va == 16 && vb == 16 && encode_tiled() != nullptr) {
            const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
            int rc;
            if (MODE == FORWARD) rc = make_map(&map_a, P.a, bf16, 3, P.M, P.K, P.groups, 64);
            else if (MODE == GRAD_X) rc = make_map(&map_a, P.a, bf16, 3, P.K, P.M, P.groups, TILE_M);
            else rc = make_map(&map_a, P.a, bf16, 2, P.M, P.n, 1, 64);
            if (rc != MGGB_OK) return rc;
            rc = MODE == GRAD_W ? make_map(&map_b, P.b, bf16, 2, P.N, P.n, 1, 64) : make_map(&map_b, P.b, bf16, 2, P.K, P.n, 1, P.tile_n);
            if (rc != MGGB_OK) return rc;
            return launch<T, MODE, true, 16, 16>(P, map_a, map_b, max_units, st);
        }
    }
    if (va == 16) return launch_b<T, MODE, 16>(P, vb, map_a, max_units, st);
    if (sizeof(T) == 4 && va == 8) return launch_b<T, MODE, sizeof(T) == 4 ? 8 : 4>(P, vb, map_a, max_units, st);
    if (va >= 4) return launch_b<T, MODE, 4>(P, vb, map_a, max_units, st);
    return launch_b<T, MODE, (int)sizeof(T)>(P, vb, map_a, max_units, st);
}

// Rows of a tile of out or dx: as many as still give every SM a tile, about twice an average group at most (most groups then
// fit one tile, and the copies do not bring many rows of others).
int rows_tile(long long n, int groups, int m_tiles) {
    int t = 32;
    while (t < MAX_TILE_N && t < 2 * (n / groups) && n / (2 * t) * m_tiles >= sm_count()) t *= 2;
    return t;
}

template <typename T, int MODE>
int launch_narrow_rows(Args P, cudaStream_t st) {
    P.tile_n = NARROW_ROWS;
    P.m_tiles = 1;
    const int mc = P.M <= 8 ? 8 : P.M <= 16 ? 16 : 32;
    const int smem = ((2 * (P.groups + 1) + 3) / 4 * 4 + P.K * mc + NARROW_ROWS * std::max(P.K | 1, P.M)) * 4;
    const int per_sm = std::max(1, std::min(12, 200 * 1024 / smem));
    const long long units = P.n / NARROW_ROWS + std::min<long long>(P.groups, P.n);
    const unsigned grid = (unsigned)std::min<long long>(units, (long long)per_sm * sm_count());
    const Divide by_k = divide_by(P.K);
    if (mc == 8) {
        MGGB_CUDA((allow_shared<narrow_rows_kernel<T, MODE, 8>>()));
        narrow_rows_kernel<T, MODE, 8><<<grid, NARROW_ROWS, smem, st>>>(P, by_k);
    } else if (mc == 16) {
        MGGB_CUDA((allow_shared<narrow_rows_kernel<T, MODE, 16>>()));
        narrow_rows_kernel<T, MODE, 16><<<grid, NARROW_ROWS, smem, st>>>(P, by_k);
    } else {
        MGGB_CUDA((allow_shared<narrow_rows_kernel<T, MODE, 32>>()));
        narrow_rows_kernel<T, MODE, 32><<<grid, NARROW_ROWS, smem, st>>>(P, by_k);
    }
    MGGB_CUDA(cudaGetLastError());
    return MGGB_OK;
}

template <typename T, int MODE, int VB, int MC>
int launch_row_dots_mc(Args P, cudaStream_t st) {
    const int per_block = DOT_THREADS / 32 * DOT_ROWS;
    const long long kept = (long long)MC * ((P.K + 3) / 4 * 4) * 4;
    const bool keep = kept <= DOT_KEEP_BYTES;
    const int smem = (2 * (P.groups + 1) + 3) / 4 * 16 + (keep ? (int)kept : 0);
    const int per_sm = std::max(1, std::min(8, 200 * 1024 / smem));
    // rows per tile: several rounds of the block's warps where there are enough rows (the weight is brought once per group)
    P.tile_n = per_block;
    while (P.tile_n < 8 * per_block && P.n / (2 * P.tile_n) >= (long long)per_sm * sm_count()) P.tile_n *= 2;
    P.m_tiles = 1;
    const long long units = P.n / P.tile_n + std::min<long long>(P.groups, P.n);
    const unsigned grid = (unsigned)std::min<long long>(units, (long long)per_sm * sm_count());
    if (keep) {
        MGGB_CUDA((allow_shared<row_dots_kernel<T, MODE, VB, MC, true>>()));
        row_dots_kernel<T, MODE, VB, MC, true><<<grid, DOT_THREADS, smem, st>>>(P);
    } else {
        row_dots_kernel<T, MODE, VB, MC, false><<<grid, DOT_THREADS, smem, st>>>(P);
    }
    MGGB_CUDA(cudaGetLastError());
    return MGGB_OK;
}

template <typename T, int MODE, int VB>
int launch_row_dots(const Args& P, cudaStream_t st) {
    return P.M <= 2 ? launch_row_dots_mc<T, MODE, VB, 2>(P, st) : P.M <= 4 ? launch_row_dots_mc<T, MODE, VB, 4>(P, st) : launch_row_dots_mc<T, MODE, VB, 8>(P, st);
}

template <typename T, int MODE>
int rows_product(void* out, const void* a, const void* b, const int32_t* ptr, int groups, long long n, int K, int M, cudaStream_t st) {
    Args P{};
    P.ptr = ptr; P.a = a; P.b = b; P.out = out; P.n = n; P.groups = groups; P.M = M; P.K = K; P.polls = wait_polls();
    // Which products the fp32 pipes take, from measurements of all three kernels at K = 8 to 128 (and 256 to 2016), M = 2 to 64 and
    // 10,000 to 600,000 rows; us at 600,000 rows in 4 groups (below 100,000 rows the narrow kernels are ahead longer, by 2 to 4 us):
    //   narrow rows, tiles   fp32: 80 x 4 78, 143 (87 by row dots); 112 x 8 126, 146; 128 x 8 179, 144; 48 x 16 75, 77; 64 x 16 92, 79 (up to
    //                        64 terms the tiles need one accumulator); 65 x 16 104, 153; 88 x 16 147, 153; 100 x 16 163, 150; 40 x 31 79,
    //                        79; 48 x 31 95, 80.  bf16: 64 x 5 47, 68; 64 x 8 48, 47; 80 x 8 68, 60; 25 x 16 51, 81; 40 x 16 56, 43; 25 x 24
    //                        68, 81; 40 x 24 80, 49.  32 columns and more lie in few banks on their way out: 16 x 32 fp32 115, 66
    //   row dots, tiles      fp32: 100 x 4 89, 149 (114 by narrow rows); 602 x 8 542, 795; 256 x 8 282, 236.  bf16: 100 x 2 62, 79; 2016 x 1
    //                        416, 843; 100 x 4 98, 79; 602 x 4 285, 228 (but 13, 29 at 10,000 rows); 1024 x 3 295, 434; 602 x 8 510, 211
    //                        (17, 25 at 10,000 rows)
    constexpr bool F32 = sizeof(T) == 4;
    const bool narrow = M <= 8    ? K <= (F32 ? M <= 4 ? 80 : 112 : 64)
                        : M <= 16 ? (F32 ? K <= 48 || (K > 64 && K <= 88) : K <= 32)
                                  : M < 32 && K <= (F32 ? 40 : 24);
    if (narrow) return launch_narrow_rows<T, MODE>(P, st);
    if (M <= (F32 ? 4 : 2) || (K > 512 && (M <= 4 || (M <= DOT_COLS && (F32 || n <= 16384))))) {
        const int v = load_width<T>(b, K);
        if (v == 16) return launch_row_dots<T, MODE, 16>(P, st);
        if (v >= 4) return launch_row_dots<T, MODE, 4>(P, st);
        return launch_row_dots<T, MODE, (int)sizeof(T)>(P, st);
    }
    P.m_tiles = (M + TILE_M - 1) / TILE_M;
    P.tile_n = rows_tile(n, groups, P.m_tiles);
    return dispatch<T, MODE>(P, (n / P.tile_n + std::min<long long>(groups, n)) * P.m_tiles, st);
}

// How dw's sums over rows are cut.
struct Cut {
    bool narrow;                     // narrow_weight_kernel
    int tile_n, m_tiles, n_tiles, chunk_rows;
    long long slots, multi;          // at most so many chunks of groups with several, and so many such groups
    size_t list_bytes, bytes;
};
Cut cut(long long n, int groups, int K, int M, bool f32) {
    Cut c;
    c.tile_n = K <= 64 ? 64 : K <= 128 ? 128 : 256;
    // The fp32 pipes' time grows with the weight's blocks of 4 x 4, the tensor cores' with its tiles; few rows have shorter trips
    // here.  us at 600,000 rows in 4 groups, narrow kernel and tiles, fp32: 16 x 16 53, 144; 64 x 16 (64 blocks) 150, 152; 64 x 64 300,
    // 155; 602 x 4 (3 tiles) 606, 989; at 100,000 rows 64 x 64 62, 45, at 10,000 19, 27.  bf16: 24 x 19 66, 101; 16 x 16 58, 40
    // (TMA) but at 10,000 rows 10.4, 12.5; 47 x 16 113, 68; 64 x 64 322, 44.
    const long long blocks = (long long)((K + 3) / 4) * ((M + 3) / 4), whole = (long long)((M + TILE_M - 1) / TILE_M) * ((K + c.tile_n - 1) / c.tile_n);
    c.narrow = f32 ? blocks <= 256 && (n <= 65536 || blocks <= 64 * whole) : blocks <= 32 && (n <= 16384 || K % 8 != 0 || M % 8 != 0);
    c.n_tiles = c.narrow ? 1 : (K + c.tile_n - 1) / c.tile_n;
    c.m_tiles = c.narrow ? 1 : (M + TILE_M - 1) / TILE_M;
    // chunks so that the units are about two per SM (of at least 512 rows), or eight of the narrow kernel's smaller blocks
    const long long tiles = (long long)c.m_tiles * c.n_tiles, want = std::max(1LL, (c.narrow ? 4LL : 2LL) * sm_count() / tiles);
    c.chunk_rows = (int)std::min<long long>(0x7FFFFFC0LL, std::max(c.narrow ? 128LL : 512LL, (n / want + 63) / 64 * 64));
    c.multi = n > 0 ? (n - 1) / c.chunk_rows : 0;                 // a group of several chunks has more than chunk_rows rows
    c.slots = std::min(2 * c.multi, c.multi + groups);
    c.multi = std::min<long long>(c.multi, groups);
    c.list_bytes = c.slots ? (size_t)(4 * (1 + 3 * c.multi) + 255) / 256 * 256 : 0;
    c.bytes = c.list_bytes + (size_t)c.slots * K * M * 4;
    return c;
}

template <typename T, int TL>
int launch_narrow_weight(Args P, long long max_units, cudaStream_t st) {
    const int kp = (P.N + 3) / 4 * 4, mp = (P.M + 3) / 4 * 4;
    // rows per round: 12 KiB of them, more while an SM has fewer than five units (a round is a trip to memory); a multiple of 8,
    // so that a round starts on 16 bytes if the chunk does
    const int room = (int)std::max(12LL, 64LL * sm_count() / std::max<long long>(max_units, sm_count())) * 1024;
    P.tile_n = std::max(16, std::min({128, P.chunk_rows, room / ((kp + mp) * 4)}) / 8 * 8);
    const int smem = ((3 * (P.groups + 1) + 3) / 4 * 4 + P.tile_n * (kp + mp) + kp * mp) * 4;
    MGGB_CUDA((allow_shared<narrow_weight_kernel<T, TL>>()));
    const unsigned grid = (unsigned)std::min<long long>(max_units, (long long)std::max(1, std::min(4, 200 * 1024 / smem)) * sm_count());
    narrow_weight_kernel<T, TL><<<grid, NW_THREADS, smem, st>>>(P, divide_by(P.N), divide_by(P.M));
    MGGB_CUDA(cudaGetLastError());
    return MGGB_OK;
}

template <typename T>
int weight_product(float* dw, const void* dy, const void* x, const int32_t* ptr, int groups, long long n, int K, int M, void* scratch, cudaStream_t st) {
    const Cut c = cut(n, groups, K, M, sizeof(T) == 4);
    Args P{};
    P.ptr = ptr; P.a = dy; P.b = x; P.out = dw; P.n = n; P.groups = groups; P.M = M; P.N = K; P.polls = wait_polls();
    P.tile_n = c.tile_n; P.m_tiles = c.m_tiles; P.n_tiles = c.n_tiles; P.chunk_rows = c.chunk_rows;
    P.multi = c.slots ? (int*)scratch : nullptr;
    P.partial = c.slots ? (float*)((char*)scratch + c.list_bytes) : nullptr;
    const long long max_units = (n / c.chunk_rows + groups) * c.m_tiles * c.n_tiles;
    int rc;
    if (c.narrow) {
        const int blocks = ((K + 3) / 4) * ((M + 3) / 4);
        if constexpr (sizeof(T) == 4)
            rc = blocks <= 32 ? launch_narrow_weight<T, 1>(P, max_units, st) : blocks <= 64 ? launch_narrow_weight<T, 2>(P, max_units, st)
                                                                                            : launch_narrow_weight<T, 4>(P, max_units, st);
        else
            rc = launch_narrow_weight<T, 1>(P, max_units, st);
    } else {
        rc = dispatch<T, GRAD_W>(P, max_units, st);
    }
    if (rc != MGGB_OK || c.slots == 0) return rc;
    const long long size = (long long)K * M;
    // launched while the kernel before it still runs; its blocks wait for that kernel's end
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attr[1];
    config.gridDim = dim3((unsigned)std::min<long long>((size + 127) / 128, 16LL * sm_count()), (unsigned)std::min(c.multi, 1024LL));
    config.blockDim = dim3(256);
    config.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    MGGB_CUDA(cudaLaunchKernelEx(&config, grouped_reduce_kernel, dw, (const float*)P.partial, (const int*)P.multi, size, size % 4 == 0 ? 1 : 0));
    return MGGB_OK;
}

template <typename T>
int forward(void* out, const void* x, const void* w, const int32_t* ptr, int groups, long long n, int K, int M, cudaStream_t st) {
    return rows_product<T, FORWARD>(out, w, x, ptr, groups, n, K, M, st);
}

template <typename T>
int backward(void* dx, float* dw, const void* dy, const void* x, const void* w, const int32_t* ptr, int groups, long long n, int K, int M, void* scratch,
             cudaStream_t st) {
    if (n == 0) {
        if (dw) MGGB_CUDA(cudaMemsetAsync(dw, 0, (size_t)groups * K * M * 4, st));
        return MGGB_OK;
    }
    if (dx) {
        const int rc = rows_product<T, GRAD_X>(dx, w, dy, ptr, groups, n, M, K, st);
        if (rc != MGGB_OK) return rc;
    }
    return dw ? weight_product<T>(dw, dy, x, ptr, groups, n, K, M, scratch, st) : MGGB_OK;
}

}  // namespace

// One translation unit per element type: its entry points, and its kernels' status word.
#define MGGB_GROUPED_TYPE(NAME, T)                                                                                                             \
    namespace mggb {                                                                                                                           \
    int grouped_forward_##NAME(void* out, const void* x, const void* w, const int32_t* ptr, int groups, long long n, int K, int M,            \
                               cudaStream_t st) {                                                                                              \
        return forward<T>(out, x, w, ptr, groups, n, K, M, st);                                                                                \
    }                                                                                                                                          \
    int grouped_backward_##NAME(void* dx, float* dw, const void* dy, const void* x, const void* w, const int32_t* ptr, int groups,            \
                                long long n, int K, int M, void* scratch, cudaStream_t st) {                                                   \
        return backward<T>(dx, dw, dy, x, w, ptr, groups, n, K, M, scratch, st);                                                               \
    }                                                                                                                                          \
    int grouped_status_##NAME(int* status, int reset) {                                                                                        \
        MGGB_CUDA(cudaMemcpyFromSymbol(status, g_grouped_status, sizeof(int)));                                                                \
        const int zero = 0;                                                                                                                    \
        if (reset && *status) MGGB_CUDA(cudaMemcpyToSymbol(g_grouped_status, &zero, sizeof(int)));                                             \
        return MGGB_OK;                                                                                                                        \
    }                                                                                                                                          \
    }
