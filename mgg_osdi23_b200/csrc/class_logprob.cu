// Log probabilities of given classes, with the distribution's entropy and its most likely classes, and their gradient.
//     m = max_c z_c,  S = sum_c e^(z_c - m),  L = log S
//     logprob = (z_y - m) - L            H = L - sum_c e^(z_c - m) (z_c - m) / S
//     dz_c = dlogprob * (1[c = y] - p_c) - dH * p_c * (log p_c + H),   log p_c = (z_c - m) - L
// The row's statistics are kept as the pair (m, L), not as m + L: with large scores the sum would lose the low bits of L
// and every probability of the backward pass with them.
// Stands beside softmax_new_forward (include/gnn_layer.cuh:36-40); no counterpart in the reference.
//
// The forward pass has to read every logit once and is bound by HBM where the alternatives leave it time.  Three kernels,
// by the number of classes:
//   up to 128      a thread owns a row.  A block's rows arrive in shared memory by bulk copies (whatever their alignment);
//                  no value crosses lanes.  The k best are kept as VALUES by a chain of max / min; their classes are
//                  found afterwards from the bit mask of the scores that reach the k-th value.
//   up to 1024     a warp owns a row, in registers.
//   above          a block owns a row, or a cluster of blocks where there are fewer rows than would fill the machine;
//                  the parts meet through the blocks' shared memory.
// The last two find the k best through a threshold: the k-th largest of the lanes' (or groups of lanes') maxima is
// reached by at least k scores and by few more, which are collected and ranked by counting.  Where too many reach it
// (ties, or so many masked classes that the threshold is -inf), the k best are found one after the other instead: a row of
// equal scores, or with 5 classes left, costs 64 x 100,000 bf16 69 us instead of 14, 2048 x 32,768 481 instead of 51.
// The backward pass is elementwise from (m, L): vectors over the whole matrix, whatever the row length; up to 128 classes a
// thread per row.
// Measured: 2,449,029 x 47 fp32, top 5: 145 us (floor 94; a rotation of the reads where a row's words are even costs 30 %);
// 64 x 100,000 bf16, top 8: 12.7 us (9.1 without alternatives); 2048 x 32,768 bf16: 49 us (36); backward 232,965 x 41 fp32:
// 16.4 us (27 with a row search per vector), 2048 x 32,768 bf16 with entropy: 53 us (0.78 of the copy rate).
#include <algorithm>
#include <cfloat>
#include "async.h"
#include "elem.h"
#include "overlap.h"

namespace {

using namespace mggb;

constexpr int NARROW_ROWS = 128;      // rows (and threads) of a block of the thread-per-row kernel
constexpr int NARROW_CLASSES = 128;
constexpr int WARP_CLASSES = 1024;
constexpr int WARP_ROWS = 8;          // warps of a block of the warp-per-row kernel
constexpr int WIDE_THREADS = 256;
constexpr int CAND = 1024;            // scores collected per block before the slow selection takes over
constexpr int WARP_CAND = 64;
constexpr int HOLD_VECS = 16;         // vectors (a multiple of 4) whose maxima a thread keeps between the passes of the block-per-row kernel

__device__ int g_lp_status = 0;       // 1: a bounded wait for rows expired

// e^d as 2^(d log2 e) on the special-function unit, relative error below 2^-22 + |d| 2^-24: what counts in a sum of
// exponentials that contains e^0, where a term with large |d| is small.
__device__ __forceinline__ float exp_fast(float d) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * 1.4426950408889634f));
    return r;
}

// Order of the scores as integers: larger score = larger key, NaN above everything, -0 == +0.
__device__ __forceinline__ int order_key(float v) {
    if (v != v) return 0x7F800001;      // the next key above infinity's
    const int b = __float_as_int(v + 0.f);
    return b ^ ((b >> 31) & 0x7FFFFFFF);
}
__device__ __forceinline__ float key_score(int key) {
    return key == 0x7F800001 ? __int_as_float(0x7FC00000) : __int_as_float(key ^ ((key >> 31) & 0x7FFFFFFF));
}

// (score, class) as one number: larger score first, then smaller class.
__device__ __forceinline__ unsigned long long rank_of(float v, int c) {
    return ((unsigned long long)((unsigned)order_key(v) ^ 0x80000000u) << 32) | (0xFFFFFFFFu - (unsigned)c);
}
__device__ __forceinline__ int rank_class(unsigned long long r) { return (int)(0xFFFFFFFFu - (unsigned)r); }
__device__ __forceinline__ float rank_score(unsigned long long r) { return key_score((int)((unsigned)(r >> 32) ^ 0x80000000u)); }

// Running maximum m, s = sum e^(z - m), t = sum e^(z - m) (z - m).  While m is -inf (nothing but masked scores so far) the
// exponents are taken against 0: s is then 0, or NaN if there was a NaN.
struct Sums {
    float m, s, t;
    __device__ __forceinline__ Sums() : m(-INFINITY), s(0.f), t(0.f) {}
    __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }
    // takes the maximum M >= m; what it rescales by is bounded so that 0 * (a huge difference) stays 0
    __device__ __forceinline__ void raise(float M) {
        const float d = m == -INFINITY ? 0.f : fmaxf(m - M, -1e4f);
        const float f = exp_fast(d);
        t = f * fmaf(d, s, t);
        s *= f;
        m = M;
    }
    __device__ __forceinline__ void add(float z, float from) {       // from = base()
        const float d = z - from, e = exp_fast(d);
        s += e;
        t = fmaf(e, fmaxf(d, -FLT_MAX), t);                           // e = 0 at d = -inf
    }
    template <int N>
    __device__ static __forceinline__ float largest(const float (&z)[N]) {
        float c = z[0];
#pragma unroll
        for (int i = 1; i < N; i++) c = fmaxf(c, z[i]);               // passes over NaN: it comes back through s
        return c;
    }
    // z, of which `most` is the largest
    template <int N>
    __device__ __forceinline__ void add_all(const float (&z)[N], float most) {
        if (most > m) raise(most);
        const float from = base();
        if constexpr (N % 2 == 0) {
            float2 s2 = make_float2(0.f, 0.f), t2 = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const float2 d = add2(make_float2(z[i], z[i + 1]), make_float2(-from, -from));
                const float2 q = mul2(d, make_float2(1.4426950408889634f, 1.4426950408889634f));
                float2 e;
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(q.x));
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(q.y));
                s2 = add2(s2, e);
                t2 = fma2(e, make_float2(fmaxf(d.x, -FLT_MAX), fmaxf(d.y, -FLT_MAX)), t2);
            }
            s += s2.x + s2.y;
            t += t2.x + t2.y;
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) add(z[i], from);
        }
    }
    __device__ __forceinline__ void merge(float om, float os, float ot) {
        Sums o;
        o.m = om; o.s = os; o.t = ot;
        const float M = fmaxf(m, om);
        if (M > m) raise(M);
        if (M > om) o.raise(M);
        s += o.s;
        t += o.t;
    }
    __device__ __forceinline__ bool nothing() const { return m == -INFINITY && s == 0.f; }
    __device__ __forceinline__ float L() const { return nothing() ? 0.f : logf(s); }
    __device__ __forceinline__ float entropy(float L) const { return nothing() ? 0.f : L - t / s; }
    // log probability of a score; -inf throughout in a row that is masked out as a whole
    __device__ __forceinline__ float logprob(float z, float L) const { return nothing() ? -INFINITY : (z - m) - L; }
};

struct FwdArgs {
    const void* z;
    const int32_t* labels;
    float *logprob, *stats, *entropy;
    int32_t* top_ids;
    float* top_logprobs;
    long long n, ld;
    int C, top;
    unsigned polls;                      // of a barrier before a wait gives up
};

// What one thread writes for a row: everything but the alternatives.  zy is the score at the label (or anything).
__device__ __forceinline__ void write_row(const FwdArgs& A, long long row, const Sums& S, float L, bool has, float zy) {
    if (A.logprob) A.logprob[row] = has ? S.logprob(zy, L) : 0.f;
    if (A.stats) reinterpret_cast<float2*>(A.stats)[row] = make_float2(S.m, L);
    if (A.entropy) A.entropy[row] = S.entropy(L);
}

// ---- a thread per row ------------------------------------------------------------------------------

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// v (falling) becomes the K largest values of itself, a and b: with hi >= lo of the two, the i-th is the largest of v[i],
// min(v[i-1], hi) and min(v[i-2], lo).  Seven instructions per score at K = 5, where taking them one by one needs nine.
template <int K>
__device__ __forceinline__ void keep_best(float (&v)[K], float a, float b) {
    const float hi = fmaxf(a, b), lo = fminf(a, b);
#pragma unroll
    for (int i = K - 1; i >= 2; i--) v[i] = max3(v[i], fminf(v[i - 1], hi), fminf(v[i - 2], lo));
    if (K > 1) v[K > 1 ? 1 : 0] = max3(v[K > 1 ? 1 : 0], fminf(v[0], hi), lo);
    v[0] = fmaxf(v[0], hi);
}

// A block's tile of up to NARROW_ROWS rows in shared memory, and thread t's row in it.
template <typename T>
struct NarrowTile {
    const T* z;
    int turn;
    bool ok;
    // every thread; `tile` holds NARROW_ROWS rows of `pitch` bytes, or one run of them where the matrix has no gaps
    __device__ __forceinline__ NarrowTile(unsigned char* tile, unsigned long long* bar, const void* base, long long ld, int C, long long n, long long row0,
                                          int rows, int pitch, unsigned polls, int32_t* status) {
        const int t = threadIdx.x;
        if (t == 0) {
            bar_init(smem_addr(bar), 1);
            bar_init_fence();
        }
        __syncthreads();
        if (t < 32) {
            unsigned bytes = copy_rows<T>(smem_addr(tile), tile, base, ld, C, n, row0, rows, pitch, smem_addr(bar));
            bytes = __reduce_add_sync(0xffffffffu, bytes);
            __syncwarp();
            if (t == 0) bar_expect(smem_addr(bar), bytes);
        }
        const bool joined = ld == C;
        z = reinterpret_cast<const T*>(tile + (((uint64_t)base + (row0 + (joined ? 0 : t)) * ld * sizeof(T)) & 15)) +
            (size_t)t * (joined ? C : pitch / (int)sizeof(T));
        // Rows of an even number of words start in few banks: neighbouring threads then start at other classes, so that a
        // warp's 32 reads fall into 32 banks.
        const int words = (joined ? C * (int)sizeof(T) : pitch) / 4;
        const int g = min(32, words & -words);
        turn = words > 0 && g > 1 ? (t & 31) / (32 / g) * (4 / (int)sizeof(T)) % C : 0;
        ok = bar_wait(smem_addr(bar), 0, polls);
        if (!ok) {
            *status = 1;
            bar_wait(smem_addr(bar), 0);          // the copy still lands
        }
    }
};

// TURN: rows of an even number of words (see NarrowTile), at two more instructions per score and pass.
template <typename T, int K, bool TURN>
__global__ void __launch_bounds__(NARROW_ROWS) logprob_narrow_kernel(const FwdArgs A, const int pitch) {
    constexpr int KV = K > 0 ? K : 1;
    extern __shared__ __align__(128) unsigned char tile[];
    __shared__ unsigned long long bar;
    const int t = threadIdx.x, C = A.C;
    const long long row0 = (long long)blockIdx.x * NARROW_ROWS;
    const int rows = (int)min((long long)NARROW_ROWS, A.n - row0);
    const int y = A.labels && t < rows ? A.labels[row0 + t] : -1;
    const NarrowTile<T> N(tile, &bar, A.z, A.ld, C, A.n, row0, rows, pitch, A.polls, &g_lp_status);
    const T* z = N.z;

    float v[KV];
    int id[KV];
    if (t < rows && N.ok) {
#pragma unroll
        for (int k = 0; k < KV; k++) { v[k] = -INFINITY; id[k] = 0x7FFFFFFF; }
        // position p is class p + turn, from the start again behind the last class
        auto klass = [&](int p) {
            if (!TURN) return p;
            const int c = p + N.turn;
            return c < C ? c : c - C;
        };
        int p = 0;
#pragma unroll 4
        for (; p + 2 <= C; p += 2) keep_best<KV>(v, to_f32(z[klass(p)]), to_f32(z[klass(p + 1)]));
        if (p < C) keep_best<KV>(v, to_f32(z[klass(p)]), -INFINITY);
        Sums S;
        S.m = v[0];
        const float from = S.base();
        float last = v[0];                     // the last value of the ranking that is wanted
#pragma unroll
        for (int k = 0; k < K; k++)
            if (k < A.top) last = v[k];
        unsigned hits[NARROW_CLASSES / 32];
#pragma unroll
        for (int w = 0; w < NARROW_CLASSES / 32; w++) {
            hits[w] = 0;
#pragma unroll
            for (int g = 0; g < 32; g += 8) {
                const int left = C - (32 * w + g);
                if (left <= 0) break;
                const T* zg = z + 32 * w + g;
                if (left >= 8) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float x = to_f32(TURN ? z[klass(32 * w + g + i)] : zg[i]);
                        S.add(x, from);
                        if (K > 0 && x >= last) hits[w] |= 1u << (g + i);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 7; i++)
                        if (i < left) {
                            const float x = to_f32(TURN ? z[klass(32 * w + g + i)] : zg[i]);
                            S.add(x, from);
                            if (K > 0 && x >= last) hits[w] |= 1u << (g + i);
                        }
                }
            }
        }
        const float L = S.L();
        const bool has = y >= 0 && y < C;
        write_row(A, row0 + t, S, L, has, has ? to_f32(z[y]) : 0.f);
        if (K > 0) {
            if (S.s == S.s) {
                // The scores that reach the last value, in any order: each goes to the first place of its value that holds a
                // larger class, whose holder moves on; of more ties than places the smallest classes stay.
                while (true) {
                    int c;
                    if (hits[0]) { c = __ffs(hits[0]) - 1; hits[0] &= hits[0] - 1; }
                    else if (hits[1]) { c = __ffs(hits[1]) + 31; hits[1] &= hits[1] - 1; }
                    else if (hits[2]) { c = __ffs(hits[2]) + 63; hits[2] &= hits[2] - 1; }
                    else if (hits[3]) { c = __ffs(hits[3]) + 95; hits[3] &= hits[3] - 1; }
                    else break;
                    c = klass(c);
                    const float x = to_f32(z[c]);
#pragma unroll
                    for (int k = 0; k < K; k++)
                        if (v[k] == x && id[k] > c) {
                            const int o = id[k];
                            id[k] = c;
                            c = o;
                        }
                }
            } else {
                // a NaN or +inf in the row: one place after the other
                unsigned long long before = ~0ull;
#pragma unroll
                for (int k = 0; k < K; k++)
                    if (k < A.top) {
                        unsigned long long b = 0;
                        for (int c = 0; c < C; c++) {
                            const unsigned long long r = rank_of(to_f32(z[c]), c);
                            if (r < before && r > b) b = r;
                        }
                        before = b;
                        id[k] = rank_class(b);
                        v[k] = rank_score(b);
                    }
            }
#pragma unroll
            for (int k = 0; k < K; k++) v[k] = S.logprob(v[k], L);
        }
    }
    if (K > 0) {
        // the rankings leave through shared memory: a row's few words next to the next row's
        __syncthreads();
        int32_t* ids = reinterpret_cast<int32_t*>(tile);
        float* lps = reinterpret_cast<float*>(tile) + NARROW_ROWS * A.top;
#pragma unroll
        for (int k = 0; k < K; k++)
            if (k < A.top && t < rows && N.ok) { ids[t * A.top + k] = id[k]; lps[t * A.top + k] = v[k]; }
        __syncthreads();
        if (N.ok)
            for (int i = t; i < rows * A.top; i += NARROW_ROWS) {
                A.top_ids[row0 * A.top + i] = ids[i];
                if (A.top_logprobs) A.top_logprobs[row0 * A.top + i] = lps[i];
            }
    }
}

// ---- vectors of a row of any alignment ---------------------------------------------------------------

// Elements [0, count) at p: up to VE - 1 single elements until p is a multiple of 16 bytes, vectors, single elements.
template <typename T>
struct Run {
    static constexpr int VE = 16 / (int)sizeof(T);
    const T* p;
    int head, nvec, tail0, count;
    __device__ __forceinline__ Run(const T* q, int n) : p(q), count(n) {
        head = min(n, (int)((16 - ((uint64_t)q & 15)) & 15) / (int)sizeof(T));
        nvec = (n - head) / VE;
        tail0 = head + nvec * VE;
    }
};

// ---- a warp per row ----------------------------------------------------------------------------------

template <typename T, int NV>
__global__ void __launch_bounds__(WARP_ROWS * 32) logprob_warp_kernel(const FwdArgs A) {
    constexpr int VE = 16 / (int)sizeof(T), E = NV * VE + 2;
    __shared__ unsigned long long cand[WARP_ROWS][WARP_CAND];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, C = A.C;
    const long long row = (long long)blockIdx.x * WARP_ROWS + warp;
    if (row >= A.n) return;
    const Run<T> R((const T*)A.z + row * A.ld, C);
    // place 0: a single element in front, places 1 .. NV * VE: vectors, the last place: a single element behind
    float x[E];
    x[0] = lane < R.head ? to_f32(R.p[lane]) : -INFINITY;
    x[E - 1] = R.tail0 + lane < C ? to_f32(R.p[R.tail0 + lane]) : -INFINITY;
    {
        Pack<T, 16> raw[NV];
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (lane + 32 * j < R.nvec) raw[j].load(R.p + R.head + (lane + 32 * j) * VE);
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int i = 0; i < VE; i++) x[1 + j * VE + i] = lane + 32 * j < R.nvec ? raw[j].get(i) : -INFINITY;
    }
    auto class_at = [&](int i) { return i == 0 ? lane : i == E - 1 ? R.tail0 + lane : R.head + (lane + 32 * ((i - 1) / VE)) * VE + (i - 1) % VE; };
    auto exists = [&](int i) { return i == 0 ? lane < R.head : i == E - 1 ? R.tail0 + lane < C : lane + 32 * ((i - 1) / VE) < R.nvec; };

    float mine = x[0];
#pragma unroll
    for (int i = 1; i < E; i++) mine = fmaxf(mine, x[i]);
    Sums S;
    S.m = key_score(__reduce_max_sync(0xffffffffu, order_key(mine)));
    S.add_all(x, S.m);
    S.s = warp_sum(S.s);
    S.t = warp_sum(S.t);
    const float L = S.L();
    if (lane == 0) {
        const int y = A.labels ? A.labels[row] : -1;
        const bool has = y >= 0 && y < C;
        write_row(A, row, S, L, has, has ? to_f32(R.p[y]) : 0.f);
    }
    if (A.top == 0) return;

    // the top-th largest of the lanes' maxima
    int key = order_key(mine), limit = 0;
    for (int k = 0; k < A.top; k++) {
        limit = __reduce_max_sync(0xffffffffu, key);
        const unsigned who = __ballot_sync(0xffffffffu, key == limit);
        if (lane == __ffs(who) - 1) key = (int)0x80000000;
    }
    const float low = key_score(limit);
    int found = 0;
#pragma unroll
    for (int i = 0; i < E; i++) {
        const bool hit = exists(i) && !(x[i] < low);                  // a NaN is never below
        const unsigned who = __ballot_sync(0xffffffffu, hit);
        if (who) {
            const int at = found + __popc(who & ((1u << lane) - 1));
            if (hit && at < WARP_CAND) cand[warp][at] = rank_of(x[i], class_at(i));
            found += __popc(who);
        }
    }
    __syncwarp();
    auto put = [&](int place, unsigned long long r) {
        A.top_ids[row * A.top + place] = rank_class(r);
        if (A.top_logprobs) A.top_logprobs[row * A.top + place] = S.logprob(rank_score(r), L);
    };
    if (found <= WARP_CAND) {
        for (int i = lane; i < found; i += 32) {
            const unsigned long long r = cand[warp][i];
            int place = 0;
            for (int j = 0; j < found; j++) place += cand[warp][j] > r;
            if (place < A.top) put(place, r);
        }
        return;
    }
    unsigned long long before = ~0ull;
    for (int k = 0; k < A.top; k++) {
        unsigned long long b = 0;
#pragma unroll
        for (int i = 0; i < E; i++) {
            const unsigned long long r = exists(i) ? rank_of(x[i], class_at(i)) : 0;
            if (r < before && r > b) b = r;
        }
#pragma unroll
        for (int off = 16; off; off >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, off));
        before = b;
        if (lane == 0) put(k, b);
    }
}

// ---- a block or a cluster of blocks per row ------------------------------------------------------------

struct WideShared {
    int key[WIDE_THREADS / 32];
    float s[WIDE_THREADS / 32], t[WIDE_THREADS / 32];
    float sum[3];                                   // the block's Sums
    int keys[WIDE_THREADS];                         // the threads' maxima
    int limit, found;
    unsigned long long cand[CAND];
    unsigned long long best[MGGB_MAX_TOP];          // the block's alternatives, in order
    unsigned long long slow[WIDE_THREADS / 32];
};

// address of a block's shared variable as another block of the cluster sees it
__device__ __forceinline__ uint32_t in_block(const void* p, int block) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(block));
    return a;
}
__device__ __forceinline__ float read_f32(uint32_t a) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ unsigned long long read_u64(uint32_t a) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// HOLD: a slice of at most HOLD_VECS * WIDE_THREADS vectors, whose maxima are kept between the two passes: the second
// then looks at the few vectors that reach the threshold only.
template <typename T, bool HOLD>
__global__ void __launch_bounds__(WIDE_THREADS, 4) logprob_wide_kernel(const FwdArgs A, const int blocks) {
    constexpr int VE = 16 / (int)sizeof(T), UN = 4;
    __shared__ WideShared sh;
    __shared__ float most[HOLD ? HOLD_VECS : 1][WIDE_THREADS];      // a thread's own, at no conflicts
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, C = A.C;
    const int part = blocks > 1 ? (int)(blockIdx.x % blocks) : 0;
    const long long row = blockIdx.x / blocks;
    const T* zr = (const T*)A.z + row * A.ld;
    const int step = (C + blocks - 1) / blocks, c0 = min(C, part * step), c1 = min(C, c0 + step);
    const Run<T> R(zr + c0, c1 - c0);
    const T* body = R.p + R.head;

    // running maximum and sums per thread
    Sums S;
    Pack<T, 16> raw[UN];
    auto load = [&](int i) {
#pragma unroll
        for (int u = 0; u < UN; u++)
            if (i + u * WIDE_THREADS < R.nvec) load_now(raw[u].raw, body + (size_t)(i + u * WIDE_THREADS) * VE);
    };
    auto take = [&](int u) {
        float z[VE];
        raw[u].widen(z);
        const float big = Sums::largest(z);
        S.add_all(z, big);
        return big;
    };
    float single = -INFINITY;                       // a single element in front of the vectors (or behind, from thread 32 on)
    int single_class = 0;
    if (tid < R.head) { single = to_f32(R.p[tid]); single_class = c0 + tid; }
    else if (tid >= 32 && R.tail0 + tid - 32 < R.count) { single = to_f32(R.p[R.tail0 + tid - 32]); single_class = c0 + R.tail0 + tid - 32; }
    const bool has_single = tid < R.head || (tid >= 32 && R.tail0 + tid - 32 < R.count);
    for (int i = tid, q = 0; i - tid < R.nvec; i += UN * WIDE_THREADS, q += UN) {
        load(i);
#pragma unroll
        for (int u = 0; u < UN; u++) {
            float big = -INFINITY;
            if (i + u * WIDE_THREADS < R.nvec) big = take(u);
            if (HOLD && A.top > 0) most[q + u][tid] = big;
        }
    }
    if (has_single) { const float z[1] = {single}; S.add_all(z, single); }
    // The block's maximum, then every thread's sums against it.  The threads of one lane number form a group:
    // the groups' maxima bound the k best from below.
    int key = order_key(S.m);
    if (A.top > 0) sh.keys[tid] = key;
    key = __reduce_max_sync(0xffffffffu, key);
    if (lane == 0) sh.key[warp] = key;
    if (tid == 0) sh.found = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WIDE_THREADS / 32; w++) key = max(key, sh.key[w]);
    S.raise(key_score(key));
    S.s = warp_sum(S.s);
    S.t = warp_sum(S.t);
    if (lane == 0) { sh.s[warp] = S.s; sh.t[warp] = S.t; }
    if (A.top > 0 && warp == 0) {
        int mine = sh.keys[lane], place = 0;
#pragma unroll
        for (int w = 1; w < WIDE_THREADS / 32; w++) mine = max(mine, sh.keys[32 * w + lane]);
#pragma unroll
        for (int j = 0; j < 32; j++) {
            const int o = __shfl_sync(0xffffffffu, mine, j);
            place += o > mine || (o == mine && j < lane);
        }
        if (place == A.top - 1) sh.limit = mine;
    }
    __syncthreads();
    S.s = S.t = 0.f;
#pragma unroll
    for (int w = 0; w < WIDE_THREADS / 32; w++) { S.s += sh.s[w]; S.t += sh.t[w]; }

    if (A.top > 0) {
        const float low = key_score(sh.limit);
        auto look = [&](float v, int c) {
            if (!(v < low)) {                                         // a NaN is never below
                const int at = atomicAdd(&sh.found, 1);
                if (at < CAND) sh.cand[at] = rank_of(v, c);           // in any order: they are ranked by what they are
            }
        };
        auto look_at = [&](int j) {                                   // vector j of the slice
            Pack<T, 16> v;
            v.raw = __ldg(reinterpret_cast<const uint4*>(body + (size_t)j * VE));
#pragma unroll
            for (int e = 0; e < VE; e++) look(v.get(e), c0 + R.head + j * VE + e);
        };
        const bool odd = !(S.s == S.s);                               // a NaN somewhere (or +inf): maxima do not tell
        if (has_single) look(single, single_class);
        if constexpr (HOLD) {
            for (int j = tid, q = 0; j < R.nvec; j += WIDE_THREADS, q++)
                if (odd || most[q][tid] >= low) look_at(j);
        } else {
            for (int i = tid; i < R.nvec; i += UN * WIDE_THREADS) {
                load(i);
#pragma unroll
                for (int u = 0; u < UN; u++) {
                    const int j = i + u * WIDE_THREADS;
                    float z[VE];
                    raw[u].widen(z);
                    if (j < R.nvec && (odd || Sums::largest(z) >= low)) look_at(j);
                }
            }
        }
        __syncthreads();
        const int found = sh.found, want = min(A.top, c1 - c0);
        if (found <= CAND) {
            for (int j = tid; j < found; j += WIDE_THREADS) {
                const unsigned long long r = sh.cand[j];
                int place = 0;
                for (int q = 0; q < found; q++) place += sh.cand[q] > r;
                if (place < want) sh.best[place] = r;
            }
        } else {
            unsigned long long before = ~0ull;
            for (int k = 0; k < want; k++) {
                unsigned long long b = 0;
                for (int c = c0 + tid; c < c1; c += WIDE_THREADS) {
                    const unsigned long long r = rank_of(to_f32(zr[c]), c);
                    if (r < before && r > b) b = r;
                }
#pragma unroll
                for (int off = 16; off; off >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, off));
                if (lane == 0) sh.slow[warp] = b;
                __syncthreads();
                for (int w = 0; w < WIDE_THREADS / 32; w++) b = max(b, sh.slow[w]);
                __syncthreads();
                before = b;
                if (tid == 0) sh.best[k] = b;
            }
        }
        if (tid >= want && tid < A.top) sh.best[tid] = 0;             // a slice shorter than top
    }
    if (blocks > 1) {
        if (tid == 0) { sh.sum[0] = S.m; sh.sum[1] = S.s; sh.sum[2] = S.t; }
        cluster_sync();
        if (part == 0) {
            S = Sums();
            for (int b = 0; b < blocks; b++) S.merge(read_f32(in_block(&sh.sum[0], b)), read_f32(in_block(&sh.sum[1], b)), read_f32(in_block(&sh.sum[2], b)));
            const int all = blocks * A.top;                           // at most 8 * MGGB_MAX_TOP = the block's threads
            if (tid < all) sh.cand[tid] = read_u64(in_block(&sh.best[tid % A.top], tid / A.top));
            __syncthreads();
            unsigned long long r = 0;
            int place = A.top;
            if (tid < all) {
                r = sh.cand[tid];
                place = 0;
                for (int q = 0; q < all; q++) place += sh.cand[q] > r;
            }
            __syncthreads();
            if (r != 0 && place < A.top) sh.cand[place] = r;
        }
        cluster_sync();                                               // nobody leaves while its shared memory is read
        if (part != 0) return;
        if (tid < A.top) sh.best[tid] = sh.cand[tid];
    }
    __syncthreads();
    const float L = S.L();
    if (tid == 0) {
        const int y = A.labels ? A.labels[row] : -1;
        const bool has = y >= 0 && y < C;
        write_row(A, row, S, L, has, has ? to_f32(zr[y]) : 0.f);
    }
    if (tid < A.top) {
        A.top_ids[row * A.top + tid] = rank_class(sh.best[tid]);
        if (A.top_logprobs) A.top_logprobs[row * A.top + tid] = S.logprob(rank_score(sh.best[tid]), L);
    }
}

// ---- backward ------------------------------------------------------------------------------------------

struct BwdArgs {
    void* dz;
    const void* z;
    const int32_t* labels;
    const float *stats, *dlogprob, *entropy, *dentropy;
    long long n, ld_dz, ld_z, total;     // total: vectors
    unsigned C, magic, shift;            // q / C = (umulhi(q, magic) + q) >> shift for q < 2^31
    int row_vec;                         // vectors per row where none straddles rows; 0: the matrix is one run of elements
    unsigned polls;                      // of a barrier before a wait gives up
};

constexpr int BWD_THREADS = 256, BWD_UNROLL = 4;

// What the elements of a row share.  In a row that is masked out as a whole everything is taken as 0: its exponentials are.
struct RowTerms {
    float m, L, up, H, dH;
    int y;
    __device__ __forceinline__ void load(const BwdArgs& A, long long row) {
        const float2 s = __ldg(reinterpret_cast<const float2*>(A.stats) + row);
        const bool nothing = s.x == -INFINITY && s.y == 0.f;
        m = nothing ? 0.f : s.x;
        L = s.y;
        y = A.labels ? __ldg(A.labels + row) : -1;
        up = 0.f;
        if ((unsigned)y < A.C && !nothing) up = __ldg(A.dlogprob + row);
        else y = -1;
        H = A.dentropy && !nothing ? __ldg(A.entropy + row) : 0.f;
        dH = A.dentropy && !nothing ? __ldg(A.dentropy + row) : 0.f;
    }
    // without the label's own term; the bound keeps p = 0 times log p at 0
    template <bool ENTROPY>
    __device__ __forceinline__ float gradient(float z) const {
        const float lp = (z - m) - L, p = exp_fast(lp);
        return ENTROPY ? __fmul_rn(p, fmaf(-dH, fmaxf(lp, -1e30f), -fmaf(dH, H, up))) : __fmul_rn(p, -up);
    }
    template <bool ENTROPY>
    __device__ __forceinline__ float2 gradient2(float2 z) const {
        const float2 lp = add2(add2(z, make_float2(-m, -m)), make_float2(-L, -L));
        const float2 e = mul2(lp, make_float2(1.4426950408889634f, 1.4426950408889634f));
        float2 p;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p.x) : "f"(e.x));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p.y) : "f"(e.y));
        if (!ENTROPY) return mul2(p, make_float2(-up, -up));
        const float k = fmaf(dH, H, up);
        return mul2(p, fma2(make_float2(-dH, -dH), make_float2(fmaxf(lp.x, -1e30f), fmaxf(lp.y, -1e30f)), make_float2(-k, -k)));
    }
};

template <typename T, int VB, bool ENTROPY>
__global__ void __launch_bounds__(BWD_THREADS) logprob_backward_kernel(const BwdArgs A) {
    constexpr int VE = Pack<T, VB>::VE;
    // A block takes BWD_UNROLL * BWD_THREADS consecutive vectors; its first one's row and column are found once, the rest by
    // 32-bit arithmetic from there.
    const long long v0 = (long long)blockIdx.x * (BWD_THREADS * BWD_UNROLL);
    const unsigned unit = A.row_vec ? (unsigned)A.row_vec : A.C;         // vectors or elements per row
    const long long q0 = A.row_vec ? v0 : v0 * VE;
    const long long base_row = q0 / unit;
    const unsigned base_rest = (unsigned)(q0 - base_row * unit);
    const long long elements = A.n * (long long)A.C;
    const int left = (int)min(A.total - v0, (long long)(BWD_THREADS * BWD_UNROLL));
    Pack<T, VB> x[BWD_UNROLL];
    unsigned row[BWD_UNROLL];                                            // from base_row
    int col[BWD_UNROLL];
#pragma unroll
    for (int u = 0; u < BWD_UNROLL; u++) {
        const int i = u * BWD_THREADS + threadIdx.x;
        const unsigned q = base_rest + (A.row_vec ? i : i * VE);
        row[u] = (__umulhi(q, A.magic) + q) >> A.shift;
        col[u] = (int)(q - row[u] * unit) * (A.row_vec ? VE : 1);
        const T* p = (const T*)A.z + (base_row + row[u]) * A.ld_z + col[u];
        if (i < left) {
            if (VE == 1 || A.row_vec || i + 1 < left || (v0 + i + 1) * VE <= elements) x[u].load(p);
            else {
#pragma unroll
                for (int e = 0; e < VE; e++)                             // the matrix ends inside its last vector
                    if ((v0 + i) * VE + e < elements) x[u].e[e] = p[e];
            }
        }
    }
    RowTerms t;
    unsigned have = ~0u;
#pragma unroll
    for (int u = 0; u < BWD_UNROLL; u++) {
        const int i = u * BWD_THREADS + threadIdx.x;
        if (i >= left) break;
        if (row[u] != have) t.load(A, base_row + row[u]);
        have = row[u];
        float g[VE];
        if (VE == 1 || col[u] + VE <= (int)A.C) {
            if constexpr (VE > 1) {
#pragma unroll
                for (int e = 0; e < VE; e += 2) {
                    const float2 d = t.gradient2<ENTROPY>(make_float2(x[u].get(e), x[u].get(e + 1)));
                    g[e] = d.x;
                    g[e + 1] = d.y;
                }
            } else {
                g[0] = t.gradient<ENTROPY>(x[u].get(0));
            }
            if ((unsigned)(t.y - col[u]) < (unsigned)VE) {
#pragma unroll
                for (int e = 0; e < VE; e++)
                    if (col[u] + e == t.y) g[e] = __fadd_rn(g[e], t.up);
            }
        } else {                                                         // a vector over the end of a row
            int c = col[u];
#pragma unroll
            for (int e = 0; e < VE; e++) {
                if (c == (int)A.C) {
                    c = 0;
                    have++;
                    if (base_row + have < A.n) t.load(A, base_row + have);
                }
                g[e] = __fadd_rn(t.gradient<ENTROPY>(x[u].get(e)), c == t.y ? t.up : 0.f);
                c++;
            }
        }
        Pack<T, VB> o;
        o.narrow(g);
        T* p = (T*)A.dz + (base_row + row[u]) * A.ld_dz + col[u];
        if (VE == 1 || A.row_vec || i + 1 < left || (v0 + i + 1) * VE <= elements) o.store(p);
        else {
#pragma unroll
            for (int e = 0; e < VE; e++)
                if ((v0 + i) * VE + e < elements) p[e] = o.e[e];
        }
    }
}

// Rows of few classes in one run of 16-byte aligned memory: a thread owns a row, so that the row's terms are read once and
// no element has to be told its row.  The tile is changed in place and leaves as it came.
template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(NARROW_ROWS) logprob_backward_narrow_kernel(const BwdArgs A) {
    extern __shared__ __align__(128) unsigned char tile[];
    __shared__ unsigned long long bar;
    const int t = threadIdx.x, C = (int)A.C;
    const long long row0 = (long long)blockIdx.x * NARROW_ROWS;
    const int rows = (int)min((long long)NARROW_ROWS, A.n - row0);
    RowTerms r;
    if (t < rows) r.load(A, row0 + t);
    const NarrowTile<T> N(tile, &bar, A.z, C, C, A.n, row0, rows, 0, A.polls, &g_lp_status);
    if (t < rows && N.ok) {
        T* z = const_cast<T*>(N.z);
        auto change = [&](int from, int to) {
#pragma unroll 8
            for (int c = from; c < to; c++) z[c] = from_f32<T>(__fadd_rn(r.template gradient<ENTROPY>(to_f32(z[c])), c == r.y ? r.up : 0.f));
        };
        change(N.turn, C);
        change(0, N.turn);
    }
    __syncthreads();
    if (!N.ok) return;
    T* out = (T*)A.dz + row0 * C;
    const int count = rows * C, vecs = count / (16 / (int)sizeof(T));
    for (int i = t; i < vecs; i += NARROW_ROWS) __stcs(reinterpret_cast<uint4*>(out) + i, reinterpret_cast<const uint4*>(tile)[i]);
    for (int i = vecs * (16 / (int)sizeof(T)) + t; i < count; i += NARROW_ROWS) out[i] = reinterpret_cast<const T*>(tile)[i];
}

// ---- launches --------------------------------------------------------------------------------------------

template <typename T, int K>
int launch_narrow(const FwdArgs& A, cudaStream_t st) {
    const int row_bytes = A.C * (int)sizeof(T), pitch = (row_bytes + 31) / 16 * 16;
    const int rows = A.ld == A.C ? (NARROW_ROWS * row_bytes + 31) / 16 * 16 : NARROW_ROWS * pitch;
    const int smem = std::max(rows, NARROW_ROWS * A.top * 8);
    const bool odd = ((A.ld == A.C ? row_bytes : pitch) / 4) % 2 != 0;      // in words: as NarrowTile decides
    const auto kernel = odd ? logprob_narrow_kernel<T, K, false> : logprob_narrow_kernel<T, K, true>;
    MGGB_CUDA((odd ? allow_shared<logprob_narrow_kernel<T, K, false>>() : allow_shared<logprob_narrow_kernel<T, K, true>>()));
    kernel<<<(unsigned)((A.n + NARROW_ROWS - 1) / NARROW_ROWS), NARROW_ROWS, smem, st>>>(A, pitch);
    MGGB_CUDA(cudaGetLastError());
    return MGGB_OK;
}

template <typename T>
int forward(const FwdArgs& A, cudaStream_t st) {
    if (A.C <= NARROW_CLASSES) {
        if (A.top == 0) return launch_narrow<T, 0>(A, st);
        if (A.top == 1) return launch_narrow<T, 1>(A, st);
        if (A.top <= 3) return launch_narrow<T, 3>(A, st);
        if (A.top <= 5) return launch_narrow<T, 5>(A, st);
        if (A.top <= 8) return launch_narrow<T, 8>(A, st);
        if (A.top <= 16) return launch_narrow<T, 16>(A, st);
        return launch_narrow<T, 32>(A, st);
    }
    if (A.C <= WARP_CLASSES) {
        constexpr int VE = 16 / (int)sizeof(T);
        const unsigned grid = (unsigned)((A.n + WARP_ROWS - 1) / WARP_ROWS);
        const int nvec = A.C / VE;
        if (nvec <= 32) logprob_warp_kernel<T, 1><<<grid, WARP_ROWS * 32, 0, st>>>(A);
        else if (nvec <= 64) logprob_warp_kernel<T, 2><<<grid, WARP_ROWS * 32, 0, st>>>(A);
        else if (nvec <= 128) logprob_warp_kernel<T, 4><<<grid, WARP_ROWS * 32, 0, st>>>(A);
        else logprob_warp_kernel<T, VE == 4 ? 8 : 4><<<grid, WARP_ROWS * 32, 0, st>>>(A);
        MGGB_CUDA(cudaGetLastError());
        return MGGB_OK;
    }
    // blocks per row: enough for four on every SM, each with at least 4096 classes
    int blocks = 1;
    while (blocks < 8 && A.n * blocks < 4LL * sm_count() && A.C / (2 * blocks) >= 4096) blocks *= 2;
    MGGB_REQUIRE(A.n <= 0x7FFFFFFFLL / 8, "class_logprob_forward: n=%lld rows of %d classes are too many for one launch", A.n, A.C);
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attr[1];
    config.gridDim = dim3((unsigned)(A.n * blocks));
    config.blockDim = dim3(WIDE_THREADS);
    config.stream = st;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = blocks > 1 ? 1 : 0;
    const int slice = (A.C + blocks - 1) / blocks;
    const auto kernel = slice / (16 / (int)sizeof(T)) <= HOLD_VECS * WIDE_THREADS ? logprob_wide_kernel<T, true> : logprob_wide_kernel<T, false>;
    MGGB_CUDA(cudaLaunchKernelEx(&config, kernel, A, blocks));
    return MGGB_OK;
}

template <typename T, int VB>
int launch_backward(BwdArgs A, bool joined, cudaStream_t st) {
    constexpr int VE = Pack<T, VB>::VE;
    A.row_vec = joined ? 0 : (int)A.C / VE;
    A.total = joined ? (A.n * (long long)A.C + VE - 1) / VE : A.n * A.row_vec;
    const unsigned unit = joined ? A.C : (unsigned)A.row_vec;
    A.shift = 0;
    while (A.shift < 32 && (1ull << A.shift) < unit) A.shift++;
    A.magic = (unsigned)(((1ull << 32) * ((1ull << A.shift) - unit)) / unit + 1);
    const long long per = BWD_THREADS * BWD_UNROLL;
    MGGB_REQUIRE((A.total + per - 1) / per <= 0x7FFFFFFFLL, "class_logprob_backward: n=%lld rows of %u classes are too many for one launch", A.n, A.C);
    const auto kernel = A.dentropy ? logprob_backward_kernel<T, VB, true> : logprob_backward_kernel<T, VB, false>;
    kernel<<<(unsigned)((A.total + per - 1) / per), BWD_THREADS, 0, st>>>(A);
    MGGB_CUDA(cudaGetLastError());
    return MGGB_OK;
}

template <typename T>
int backward(const BwdArgs& A, cudaStream_t st) {
    const int s = sizeof(T);
    // a matrix without gaps is one run of elements: 16-byte vectors whatever the row length
    const bool joined = A.ld_z == (long long)A.C && A.ld_dz == (long long)A.C;
    const int a = joined ? common_alignment({(uint64_t)A.z, (uint64_t)A.dz})
                         : common_alignment({(uint64_t)A.z, (uint64_t)A.dz, (uint64_t)A.ld_z * s, (uint64_t)A.ld_dz * s, (uint64_t)A.C * s});
    if (joined && a == 16 && A.C <= NARROW_CLASSES) {
        const int smem = (NARROW_ROWS * (int)A.C * s + 31) / 16 * 16;
        const auto kernel = A.dentropy ? logprob_backward_narrow_kernel<T, true> : logprob_backward_narrow_kernel<T, false>;
        MGGB_CUDA((A.dentropy ? allow_shared<logprob_backward_narrow_kernel<T, true>>() : allow_shared<logprob_backward_narrow_kernel<T, false>>()));
        kernel<<<(unsigned)((A.n + NARROW_ROWS - 1) / NARROW_ROWS), NARROW_ROWS, smem, st>>>(A);
        MGGB_CUDA(cudaGetLastError());
        return MGGB_OK;
    }
    if (a == 16) return launch_backward<T, 16>(A, joined, st);
    if (a >= 4) return launch_backward<T, 4>(A, joined, st);
    return launch_backward<T, sizeof(T)>(A, joined, st);
}

}  // namespace

namespace mggb {
int class_logprob_status(int* status, int reset) {
    MGGB_CUDA(cudaMemcpyFromSymbol(status, g_lp_status, sizeof(int)));
    const int zero = 0;
    if (reset && *status) MGGB_CUDA(cudaMemcpyToSymbol(g_lp_status, &zero, sizeof(int)));     // what was not read is not cleared
    return MGGB_OK;
}
}  // namespace mggb

extern "C" {

int mggb_class_logprob_forward(float* logprob, float* stats, float* entropy, int32_t* top_ids, float* top_logprobs, int top,
                               const void* logits, int64_t ld_logits, const int32_t* labels, int64_t n, int classes, int dtype, void* stream) {
    MGGB_REQUIRE(n >= 0 && classes >= 1 && classes <= 1 << 30, "class_logprob_forward: need n >= 0, 1 <= classes <= 2^30 (n=%lld classes=%d)", (long long)n, classes);
    MGGB_REQUIRE_DTYPE(dtype, "class_logprob_forward");
    MGGB_REQUIRE(ld_logits >= classes, "class_logprob_forward: the row stride must be at least classes");
    MGGB_REQUIRE(top >= 0 && top <= MGGB_MAX_TOP && top <= classes, "class_logprob_forward: top must be 0..min(%d, classes), got %d", MGGB_MAX_TOP, top);
    if (n == 0) return MGGB_OK;
    MGGB_REQUIRE(logits, "class_logprob_forward: NULL logits");
    MGGB_REQUIRE((logprob == nullptr) == (labels == nullptr), "class_logprob_forward: logprob and labels go together");
    MGGB_REQUIRE(top == 0 || top_ids, "class_logprob_forward: top > 0 needs top_ids");
    MGGB_REQUIRE(logprob || stats || entropy || top > 0, "class_logprob_forward: no output given");
    MGGB_REQUIRE((uintptr_t)stats % 8 == 0, "class_logprob_forward: stats must be 8-byte aligned");
    const FwdArgs A{logits, labels, logprob, stats, entropy, top_ids, top_logprobs, n, ld_logits, classes, top, wait_polls()};
    return MGGB_BY_DTYPE(dtype, forward, A, (cudaStream_t)stream);
}

int mggb_class_logprob_backward(void* dlogits, const void* logits, int64_t ld_dlogits, int64_t ld_logits, const int32_t* labels,
                                const float* stats, const float* dlogprob, const float* entropy, const float* dentropy,
                                int64_t n, int classes, int dtype, void* stream) {
    MGGB_REQUIRE(n >= 0 && classes >= 1 && classes <= 1 << 30, "class_logprob_backward: need n >= 0, 1 <= classes <= 2^30 (n=%lld classes=%d)", (long long)n, classes);
    MGGB_REQUIRE_DTYPE(dtype, "class_logprob_backward");
    MGGB_REQUIRE(ld_logits >= classes && ld_dlogits >= classes, "class_logprob_backward: row strides must be at least classes");
    if (n == 0) return MGGB_OK;
    MGGB_REQUIRE(dlogits && logits && stats, "class_logprob_backward: NULL argument");
    MGGB_REQUIRE((dlogprob == nullptr) == (labels == nullptr), "class_logprob_backward: dlogprob and labels go together");
    MGGB_REQUIRE((dentropy == nullptr) || entropy, "class_logprob_backward: dentropy needs the forward pass's entropy");
    MGGB_REQUIRE(dlogprob || dentropy, "class_logprob_backward: no gradient given");
    MGGB_REQUIRE(dlogits != logits || ld_dlogits == ld_logits, "class_logprob_backward: in place needs equal row strides");
    const int s = elem_bytes(dtype);
    MGGB_REQUIRE(dlogits == logits || !rows_meet(dlogits, ld_dlogits * s, logits, ld_logits * s, n, (uint64_t)classes * s),
                 "class_logprob_backward: dlogits lies partly over logits");
    MGGB_REQUIRE((uintptr_t)stats % 8 == 0, "class_logprob_backward: stats must be 8-byte aligned");
    const BwdArgs A{dlogits, logits, labels, stats, dlogprob, entropy, dentropy, n, ld_dlogits, ld_logits, 0, (unsigned)classes, 0, 0, 0, wait_polls()};
    return MGGB_BY_DTYPE(dtype, backward, A, (cudaStream_t)stream);
}

}  // extern "C"
