// Layer norm of rows, forward and backward.
//
//   mean = sum(x) / d;  var = sum((x - mean)^2) / d;  rstd = 1 / sqrt(var + eps);  h = (x - mean) * rstd
//   y = h * gamma + beta
//   g = dy * gamma;  dx = rstd * (g - sum(g) / d - h * sum(g * h) / d);  dgamma = sum over rows of dy * h;  dbeta = of dy
//
// The variance is taken after the mean: the difference of the mean of squares and the squared mean loses all digits on rows
// whose offset is large against their spread.  All sums are fp32 in a fixed order.
#include "ops.cuh"

#include <float.h>
#include <math.h>

namespace omoe {

namespace {

constexpr int kRowsMax = 0x7fff0000;  // row numbers, and the rows a grid takes at a time beyond them, fit 32 bits
constexpr int kWideThreads = 512;

// Sum over a block of kWideThreads, the same value in every thread.
__device__ __forceinline__ float block_sum(float v, float *s) {
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kWideThreads / 32; i++) sum += s[i];
    return sum;
}

// ---- rows of any width ---------------------------------------------------------------------------------------------
// A block walks its row three times (forward) or twice (backward), from cache after the first; the column sums read everything once
// more.  What does not fit the registers below, and what those do not have in stages (two fp32 rows of more than 8192).
template <typename XT, typename YT, int V>
__global__ void __launch_bounds__(kWideThreads)
norm_wide_kernel(const XT *__restrict__ x, int64_t ldx, const float *__restrict__ gamma, const float *__restrict__ beta,
                 float eps, YT *__restrict__ y, int64_t ldy, float *__restrict__ mean_out, float *__restrict__ rstd_out, int d) {
    __shared__ float s[kWideThreads / 32];
    const int64_t t = blockIdx.x;
    pdl_trigger();
    pdl_wait();
    const XT *row = x + t * ldx;
    Frag<XT, V> f;
    float v[V], sum = 0.f;
#pragma unroll 4
    for (int c = threadIdx.x * V; c < d; c += kWideThreads * V) {
        f.load_cached(row + c);
        f.get(v);
#pragma unroll
        for (int i = 0; i < V; i++) sum += v[i];
    }
    const float mean = block_sum(sum, s) / (float)d;
    sum = 0.f;
#pragma unroll 4
    for (int c = threadIdx.x * V; c < d; c += kWideThreads * V) {
        f.load_cached(row + c);
        f.get(v);
#pragma unroll
        for (int i = 0; i < V; i++) sum = fmaf(v[i] - mean, v[i] - mean, sum);
    }
    const float rstd = rsqrtf(block_sum(sum, s) / (float)d + eps);
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[t] = mean;
        if (rstd_out) rstd_out[t] = rstd;
    }
    for (int c = threadIdx.x * V; c < d; c += kWideThreads * V) {
        Frag<float, V> p;
        Frag<YT, V> out;
        float w[V], b[V];
        f.load_cached(row + c);
        f.get(v);
#pragma unroll
        for (int i = 0; i < V; i++) { w[i] = 1.f; b[i] = 0.f; }
        if (gamma) { p.load_cached(gamma + c); p.get(w); }
        if (beta) { p.load_cached(beta + c); p.get(b); }
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = fmaf((v[i] - mean) * rstd, w[i], b[i]);
        out.set(v);
        out.store(y + t * ldy + c);
    }
}

template <typename XT, typename YT, int V>
__global__ void __launch_bounds__(kWideThreads)
norm_bwd_wide_kernel(const YT *__restrict__ dy, int64_t lddy, const XT *__restrict__ x, int64_t ldx,
                     const float *__restrict__ gamma, const float *__restrict__ mean, const float *__restrict__ rstd,
                     XT *__restrict__ dx, int64_t lddx, int d) {
    __shared__ float s[2][kWideThreads / 32];
    const int64_t t = blockIdx.x;
    pdl_trigger();
    pdl_wait();
    const float m = mean[t], r = rstd[t];
    float sum = 0.f, dot = 0.f;
    float g[V], h[V];
    auto take = [&](int c) {  // g = dy * gamma and h of V columns
        Frag<YT, V> fy;
        Frag<XT, V> fx;
        fy.load_cached(dy + t * lddy + c);
        fx.load_cached(x + t * ldx + c);
        fy.get(g);
        fx.get(h);
        if (gamma) {
            Frag<float, V> p;
            float w[V];
            p.load_cached(gamma + c);
            p.get(w);
#pragma unroll
            for (int i = 0; i < V; i++) g[i] *= w[i];
        }
#pragma unroll
        for (int i = 0; i < V; i++) h[i] = (h[i] - m) * r;
    };
#pragma unroll 2
    for (int c = threadIdx.x * V; c < d; c += kWideThreads * V) {
        take(c);
#pragma unroll
        for (int i = 0; i < V; i++) {
            sum += g[i];
            dot = fmaf(g[i], h[i], dot);
        }
    }
    const float mg = block_sum(sum, s[0]) / (float)d, mh = block_sum(dot, s[1]) / (float)d;
#pragma unroll 2
    for (int c = threadIdx.x * V; c < d; c += kWideThreads * V) {
        Frag<XT, V> out;
        take(c);
#pragma unroll
        for (int i = 0; i < V; i++) g[i] = r * (g[i] - mg - h[i] * mh);
        out.set(g);
        out.store(dx + t * lddx + c);
    }
}

// Column sums of a slice of the rows: partial[slice][0][d] of dy * h, [1][d] of dy.  A thread has V columns of all of the slice's rows.
constexpr int kColThreads = 256;
template <typename XT, typename YT, int V>
__global__ void __launch_bounds__(kColThreads)
norm_cols_kernel(const YT *__restrict__ dy, int64_t lddy, const XT *__restrict__ x, int64_t ldx,
                 const float *__restrict__ mean, const float *__restrict__ rstd, float *__restrict__ partial, int T, int d,
                 int slice) {
    constexpr int U = V == 8 ? 2 : 4;  // rows whose loads are on their way together (twice as many take the registers of half the blocks)
    const int64_t c = ((int64_t)blockIdx.x * kColThreads + threadIdx.x) * V;
    pdl_trigger();
    pdl_wait();
    if (c >= d) return;
    const int64_t t0 = (int64_t)blockIdx.y * slice, t1 = min((int64_t)T, t0 + slice);
    float a[V], b[V];
#pragma unroll
    for (int i = 0; i < V; i++) a[i] = b[i] = 0.f;
    for (int64_t t = t0; t < t1; t += U) {
        Frag<YT, V> fy[U];
        Frag<XT, V> fx[U];
        float m[U], r[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (t + u < t1) {
                fy[u].load(dy + (t + u) * lddy + c);
                fx[u].load(x + (t + u) * ldx + c);
                m[u] = mean[t + u];
                r[u] = rstd[t + u];
            }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (t + u < t1) {
                float g[V], h[V];
                fy[u].get(g);
                fx[u].get(h);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    a[i] = fmaf(g[i], (h[i] - m[u]) * r[u], a[i]);
                    b[i] += g[i];
                }
            }
    }
    float *to = partial + (int64_t)blockIdx.y * 2 * d + c;
    Frag<float, V> f;
    f.set(a);
    f.store(to);
    f.set(b);
    f.store(to + d);
}

// ---- rows that fit a block's registers ----------------------------------------------------------------------------
//
// A block of B threads works on B / G rows at a time: G threads hold a row, P vectors of V elements each, and walk the rows of the
// grid with a stride.  The forms for few threads (FEW) take for a row the whole warps that it needs instead, and as many rows as then
// fit the block: few_forward and few_backward.  Rows arrive in a ring of S stages in shared memory by asynchronous copies that a warp makes for
// its own columns alone, so the ring needs no block barrier, and the loads of the next S - 1 rows are on their way while a
// row is reduced.  The reductions are what threads of a row meet for: warp shuffles, then one named barrier each.
// Bound by the issue of instructions before it is by HBM, hence pairs of values in the packed fp32 instructions, sums that
// share their shuffles, and no divisions.
template <int G>
constexpr int kFwdBlock = G > 512 ? G : 512;
// Backward one block per SM leaves half the column sums to join that two do (16384 x 4096 of bf16 73 us against 76, x 1544 of fp32 57
// against 62); but long rows of fp32 are faster in two (109 us against 121), and 16 rows at a time would run out of barriers.
template <typename XT, int V, int G, int P>
constexpr int kBwdBlock = G == 1024 || (V == 8 && P == 1 && G != 64 && !(G == 512 && sizeof(XT) == 4)) ? 1024 : 512;

// Two fp32 values in one register pair.
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack2(float a, float b) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(f2 v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float both(f2 v) {
    float a, b;
    unpack2(v, a, b);
    return a + b;
}

__device__ __forceinline__ void copy16(uint32_t to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the last N groups of this warp's copies have landed, and its lanes are done with the stage they read before.
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
    __syncwarp();
}
__device__ __forceinline__ uint4 shared16(uint32_t at) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
    return r;
}

// The rows ahead.  V = 8: S stages of shared memory.  In a stage every warp has, for each vector of its threads, the 256 columns
// they hold as they lie in the row, in pieces of 16 bytes; the lanes copy neighbouring pieces.  A thread's 8 columns are one
// piece of bf16 and two of fp32; there pieces 8 .. 15 of every 16 are swapped in pairs, so that eight lanes reading their first
// pieces meet all banks.
// V = 1 (rows that are not aligned): one row ahead, in registers.
template <typename T, int B, int V, int G, int P, int S>
struct Ahead {
    static constexpr int kPieces = sizeof(T) / 2;  // of a thread's vector
    static constexpr int kVector = B * 16 * kPieces, kStage = kVector * P;
    uint32_t first, second, put;  // this thread's pieces, and where it puts what it copies
    int col;                      // the first column it copies
    // vectors behind the row's end are zeros in every stage from the start
    __device__ __forceinline__ Ahead(uint32_t ring, int d, int in_row) {
        const int lane = threadIdx.x & 31;
        const uint32_t warp = ring + (threadIdx.x - lane) * 16 * kPieces;
        const int swap = kPieces == 2 ? lane >> 2 & 1 : 0;
        first = warp + (lane * kPieces ^ swap) * 16;
        second = warp + ((lane * kPieces + 1) ^ swap) * 16;
        put = warp + (kPieces == 2 ? lane ^ (lane >> 3 & 1) : lane) * 16;
        col = (in_row - lane) * 8 + lane * (8 / kPieces);
#pragma unroll
        for (int p = 0; p < P; p++)
            if ((p * G + in_row) * 8 >= d)
                for (int i = 0; i < S; i++) {
                    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(first + i * kStage + p * kVector), "r"(0) : "memory");
                    if constexpr (kPieces == 2)
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(second + i * kStage + p * kVector), "r"(0) : "memory");
                }
        __syncwarp();
    }
    // from: the row's element `col`
    __device__ __forceinline__ void fetch(int stage, const T *from, int d) const {
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int q = 0; q < kPieces; q++) {
                const int c = p * G * 8 + q * 128;
                if (col + c < d) copy16(put + stage * kStage + p * kVector + q * 512, from + c);
            }
    }
    // pairs 4p .. 4p + 3 of this thread
    __device__ __forceinline__ void take(int stage, int p, f2 (&v)[4]) const {
        const uint4 a = shared16(first + stage * kStage + p * kVector);
        if constexpr (kPieces == 1) {
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        } else {
            const uint4 b = shared16(second + stage * kStage + p * kVector);
            v[0] = pack2(__uint_as_float(a.x), __uint_as_float(a.y));
            v[1] = pack2(__uint_as_float(a.z), __uint_as_float(a.w));
            v[2] = pack2(__uint_as_float(b.x), __uint_as_float(b.y));
            v[3] = pack2(__uint_as_float(b.z), __uint_as_float(b.w));
        }
    }
};
template <typename T, int B, int G, int P, int S>
struct Ahead<T, B, 1, G, P, S> {
    static constexpr int kStage = 0;
    Frag<T, 1> next[P];
    int col;
    __device__ __forceinline__ Ahead(uint32_t, int, int in_row) : col(in_row) {
#pragma unroll
        for (int p = 0; p < P; p++) next[p].zero();
    }
    __device__ __forceinline__ void fetch(int, const T *from, int d) {
#pragma unroll
        for (int p = 0; p < P; p++)
            if (col + p * G < d) next[p].load(from + p * G);
    }
    // all of this thread's elements, two by two
    __device__ __forceinline__ void take(int, int p, f2 (&v)[P / 2]) const {
#pragma unroll
        for (int i = 0; i < P / 2; i++) {
            float a[1], b[1];
            next[2 * i].get(a);
            next[2 * i + 1].get(b);
            v[i] = pack2(a[0], b[0]);
        }
    }
};

// What a thread holds of a row, in groups of pairs that are read and stored together: a vector each (V = 8), or all of its
// single elements (V = 1).
template <int V, int G, int P, bool FEW>
struct Part {
    static constexpr int kGroups = V == 8 ? P : 1, kPairs = V == 8 ? 4 : P / 2;
    int d, mine;  // the row's width, the thread's number in the row
    __device__ __forceinline__ int in_row() const { return FEW ? mine : threadIdx.x % G; }
    __device__ __forceinline__ int col(int q) const { return V == 8 ? (q * G + in_row()) * 8 : in_row(); }
    __device__ __forceinline__ bool has(int q) const { return col(q) < d; }
    // single elements: zeros in place of what lies behind the row's end
    __device__ __forceinline__ void mask(int q, f2 (&v)[kPairs]) const {
#pragma unroll
        for (int i = 0; i < kPairs; i++) {
            if constexpr (V == 1) {
                float a, b;
                unpack2(v[i], a, b);
                v[i] = pack2(in_row() + 2 * i * G < d ? a : 0.f, in_row() + (2 * i + 1) * G < d ? b : 0.f);
            }
        }
    }
    // sum + a * b; of single elements only where the row has them (the first half of its threads' elements it always has, but on one warp)
    __device__ __forceinline__ f2 add_product(int i, f2 a, f2 b, f2 sum) const {
        if constexpr (V == 1) {
            if (G == 32 || 4 * i >= P) {
                float c, e;
                unpack2(b, c, e);
                b = pack2(in_row() + 2 * i * G < d ? c : 0.f, in_row() + (2 * i + 1) * G < d ? e : 0.f);
            }
        }
        return fma2(a, b, sum);
    }
    __device__ __forceinline__ void load(const float *p, int q, float missing, f2 (&v)[kPairs]) const {
#pragma unroll
        for (int i = 0; i < kPairs; i++) v[i] = pack2(missing, missing);
        if (!p || !has(q)) return;
        if constexpr (V == 8) {
            Frag<float, 8> f;
            f.load_cached(p + col(q));
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = pack2(f.r[2 * i], f.r[2 * i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < kPairs; i++) {
                const int a = in_row() + 2 * i * G, b = a + G;
                v[i] = pack2(a < d ? __ldg(p + a) : missing, b < d ? __ldg(p + b) : missing);
            }
        }
    }
    // p: element col(0) of the row
    template <typename T>
    __device__ __forceinline__ void store(T *p, int q, const f2 (&v)[kPairs]) const {
        float w[2 * kPairs];
#pragma unroll
        for (int i = 0; i < kPairs; i++) unpack2(v[i], w[2 * i], w[2 * i + 1]);
        if constexpr (V == 8) {
            if (!has(q)) return;
            Frag<T, 8> f;
            f.set(w);
            f.store(p + q * G * 8);
        } else {
#pragma unroll
            for (int i = 0; i < 2 * kPairs; i++)
                if (in_row() + i * G < d) p[i * G] = (T)w[i];
        }
    }
};

// p, rows of `bytes` bytes further on.
template <typename T>
__device__ __forceinline__ T *rows_on(T *p, int rows, uint32_t bytes) {
    return reinterpret_cast<T *>(reinterpret_cast<uintptr_t>(p) + (uint64_t)(uint32_t)rows * bytes);
}

// Blocks that share an SM: what the registers allow.
template <int G>
constexpr int kFwdBlocks = 1024 / kFwdBlock<G>;
template <typename XT, int V, int G, int P>
constexpr int kBwdBlocks = P > 4 || (V == 8 && P > 1) ? 1 : 1024 / kBwdBlock<XT, V, G, P>;
// Rows that a forward block's threads take at a time.  Where many threads share a row of bf16, two rows share their barriers and
// shuffles (16384 x 4096: 44 us, one by one 50; 40000 x 1536 on 256 threads a row: 44 and 55); fp32 is bound by HBM either way, and
// narrower rows are faster one by one (65536 x 1024: 49 us and 45).
template <typename XT, int V, int G, int P>
constexpr int kFwdRows = V == 8 && G >= 256 && (P == 1 || G == 1024) && sizeof(XT) == 2 ? 2 : 1;
// Stages that fit a block's share of shared memory.  Forward two beside those of two goes (16384 x 4096 of bf16 with four 45.3 us, with six
// 43.9).  Backward three for bf16 (with four 65536 x 256 takes 23.3 us, 22.4 with three), four for fp32, and two where two blocks
// of long fp32 rows share an SM (x 4096 to bf16, 8192 to 30011 rows: 52 to 186 us, with four 57 to 215).
constexpr int stages(int stage_bytes, int blocks, int most) {
    const int fit = stage_bytes ? 212992 / blocks / stage_bytes : 2;
    return fit > most ? most : fit;
}
template <typename XT, int V, int G, int P>
constexpr int kFwdStages = V == 1 ? 2 : stages(kFwdBlock<G> * P * V * (int)sizeof(XT), kFwdBlocks<G>, 2 + 2 * kFwdRows<XT, V, G, P>);
template <typename XT, typename YT, int V, int G, int P>
constexpr int kBwdStages = V == 1 ? 2 : stages(kBwdBlock<XT, V, G, P> * P * V * (int)(sizeof(XT) + sizeof(YT)), kBwdBlocks<XT, V, G, P>,
                                                  sizeof(XT) == 2 ? 3 : G == 512 ? 2 : 4);

// The threads of a block, by row.
template <int B, int G, bool FEW>
struct Block {
    // rows at a time: B / G, or as many as a block can have of at least G / 2 + 32 threads each
    static constexpr int kRows = FEW ? 2 * B / (G + 64) : B / G;
    static_assert(G == 32 || kRows == 1 || kRows < 16, "a named barrier for every row");
    static constexpr int kWords = kRows * 2 * (G / 32);  // two for every warp that a row can have
    int row_threads;
    __device__ __forceinline__ int threads() const { return FEW ? row_threads : G; }
    __device__ __forceinline__ int all() const { return FEW ? (int)blockDim.x : B; }
    __device__ __forceinline__ int rows() const { return FEW ? all() / row_threads : B / G; }
    __device__ __forceinline__ int in_row() const { return threadIdx.x % threads(); }
    __device__ __forceinline__ unsigned warp() const { return FEW ? (unsigned)in_row() >> 5 : threadIdx.x % G >> 5; }
    __device__ __forceinline__ void row_barrier() const {
        if constexpr (G == B) __syncthreads();
        else if constexpr (FEW) asm volatile("bar.sync %0, %1;" ::"r"((int)threadIdx.x / row_threads + 1), "r"(row_threads) : "memory");
        else asm volatile("bar.sync %0, %1;" ::"r"((int)threadIdx.x / G + 1), "n"(G) : "memory");
    }
    // the words of warps that the rows do not have stay zero
    __device__ __forceinline__ void clear(float (&words)[2][kWords]) const {
        if constexpr (FEW) {
            for (int i = threadIdx.x; i < 2 * kWords; i += all()) words[i / kWords][i % kWords] = 0.f;
            __syncthreads();
        }
    }
};

// The sum of v over the threads of a row, in all of them.  s: words of this row; between two uses the threads of the row
// have to meet at another barrier.
template <int B, int G, bool FEW>
__device__ __forceinline__ float row_sum(float v, float *s, const Block<B, G, FEW> &block) {
    constexpr int W = G / 32;
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if constexpr (W > 1) {
        const int lane = threadIdx.x & 31;
        if (lane == 0) s[block.warp()] = v;
        block.row_barrier();
        v = s[lane & (W - 1)];
#pragma unroll
        for (int m = W / 2; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    }
    return v;
}

// Two sums at once: after one exchange the lower half of a warp adds up a and the upper half b.
template <int B, int G, bool FEW>
__device__ __forceinline__ void row_sums(float &a, float &b, float *s, const Block<B, G, FEW> &block) {
    constexpr int W = G / 32;
    const int lane = threadIdx.x & 31, half = lane >> 4;
    float v = half ? b : a;
    v += __shfl_xor_sync(0xffffffffu, half ? a : b, 16);
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if constexpr (W > 1) {
        if ((lane & 15) == 0) s[half * W + block.warp()] = v;
        block.row_barrier();
        v = s[half * W + (lane & (W - 1) & 15)];
        if constexpr (W == 32) v += s[half * W + 16 + (lane & 15)];
#pragma unroll
        for (int m = W / 2 > 8 ? 8 : W / 2; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    }
    a = __shfl_sync(0xffffffffu, v, 0);
    b = __shfl_sync(0xffffffffu, v, 16);
}

// gamma or beta of this thread's columns: in registers (KEPT), or from cache for every row.
template <int V, int G, int P, bool FEW, bool KEPT>
struct Param {
    using Mine = Part<V, G, P, FEW>;
    const float *p;
    float missing;
    f2 kept[KEPT ? Mine::kGroups : 1][Mine::kPairs];
    __device__ __forceinline__ Param(const float *from, const Mine &part, float absent) : p(from), missing(absent) {
        if constexpr (KEPT)
#pragma unroll
            for (int q = 0; q < Mine::kGroups; q++) part.load(p, q, missing, kept[q]);
    }
    __device__ __forceinline__ void get(const Mine &part, int q, f2 (&v)[Mine::kPairs]) const {
        if constexpr (KEPT) {
#pragma unroll
            for (int i = 0; i < Mine::kPairs; i++) v[i] = kept[q][i];
        } else part.load(p, q, missing, v);
    }
};

// 1 / d in two parts.  A sum times 1 / d rounded once is off by up to two roundings of the quotient: where d * fl(1 / d) is not 1 (d = 328), a row
// of equal numbers 1024 gets a mean of 1023.99994 and y = 0.019 instead of 0.  With both parts the quotient is rounded once but for 2^-48 of it.
// `high` lies below 1 / d and `low` is positive, so that an infinite sum keeps its infinite mean.
struct Inverse {
    float nearest, high, low;
    explicit Inverse(int d) : nearest(1.f / (float)d), high(nearest) {
        if ((double)high * d > 1.0) high = nextafterf(high, 0.f);  // exact in 64 bits
        low = fmaxf((float)(1.0 / d - (double)high), FLT_MIN);
    }
    __device__ __forceinline__ float mean(float sum) const { return fmaf(sum, high, sum * low); }
};

template <typename XT, typename YT, int V, int G, int P, bool FEW>
__global__ void __launch_bounds__(kFwdBlock<G>, kFwdBlocks<G>)
norm_kernel(const XT *__restrict__ x, uint32_t x_pitch, const float *__restrict__ gamma, const float *__restrict__ beta, float eps,
            YT *__restrict__ y, uint32_t y_pitch, float *__restrict__ mean_out, float *__restrict__ rstd_out, int T, int d, Inverse inv,
            int row_threads) {
    using Mine = Part<V, G, P, FEW>;
    constexpr int B = kFwdBlock<G>, S = kFwdStages<XT, V, G, P>, R = kFwdRows<XT, V, G, P>, Q = Mine::kGroups, N = Mine::kPairs;
    static_assert(S >= 2 * R, "rows are read from some stages while others fill");
    extern __shared__ __align__(16) char sm[];
    __shared__ float s_sum[2][Block<B, G, FEW>::kWords];
    const int group = FEW ? threadIdx.x / row_threads : threadIdx.x / G;
    const int step = gridDim.x * (FEW ? blockDim.x / row_threads : B / G);
    const Block<B, G, FEW> block{row_threads};
    block.clear(s_sum);
    const Mine part = {d, block.in_row()};
    Ahead<XT, B, V, G, P, S> ahead((uint32_t)__cvta_generic_to_shared(sm), d, part.in_row());
    pdl_trigger();
    pdl_wait();
    // Kept also where a thread has two vectors (8192 x 8192 of bf16 43 us, read from cache 55), but on 1024 threads only from fp32 to bf16
    // (4096 x 16384: 65 and 76; from bf16 60 and 57, fp32 to fp32 95 and 90).
    constexpr bool kKept = P * V <= 8 || (V == 8 && (G < 1024 || (sizeof(XT) == 4 && sizeof(YT) == 2)));
    const Param<V, G, P, FEW, kKept> scale(gamma, part, 1.f), shift(beta, part, 0.f);
    int t = blockIdx.x * (FEW ? blockDim.x / row_threads : B / G) + group;  // T and the rows of 2 S strides stay below 2^31: kRowsMax
    int next = t;  // the row to fetch
    x += ahead.col;
    y += part.col(0);
    auto fetch = [&](int stage) {
        if (next < T) ahead.fetch(stage, rows_on(x, next, x_pitch), d);
        copies_commit();
        next += step;
    };
#pragma unroll
    for (int i = 0; i < S - R; i++) fetch(i);
    float *s_mean = s_sum[0] + group * (2 * G / 32), *s_var = s_sum[1] + group * (2 * G / 32);
    auto rows = [&](int stage) {  // R rows from `stage` on
        f2 v[R][Q][N];
        float sum[2] = {0.f, 0.f}, mean[2], rstd[2];
        copies_wait<S - 2 * R>();
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int q = 0; q < Q; q++) ahead.take(stage + r, q, v[r][q]);
#pragma unroll
        for (int r = 0; r < R; r++) fetch((stage + S - R + r) % S);
#pragma unroll
        for (int r = 0; r < R; r++) {
            f2 pair = 0ull;
#pragma unroll
            for (int q = 0; q < Q; q++)
#pragma unroll
                for (int i = 0; i < N; i++) pair = add2(pair, v[r][q][i]);
            sum[r] = both(pair);
        }
        if constexpr (R == 2) row_sums(sum[0], sum[1], s_mean, block);
        else sum[0] = row_sum(sum[0], s_mean, block);
#pragma unroll
        for (int r = 0; r < R; r++) {
            mean[r] = inv.mean(sum[r]);
            const f2 minus = pack2(-mean[r], -mean[r]);
            f2 pair = 0ull;
#pragma unroll
            for (int q = 0; q < Q; q++) {
                if (V == 8 && !part.has(q)) continue;  // a branch: all but one warp of a row go the same way
#pragma unroll
                for (int i = 0; i < N; i++) v[r][q][i] = add2(v[r][q][i], minus);
                part.mask(q, v[r][q]);
#pragma unroll
                for (int i = 0; i < N; i++) pair = fma2(v[r][q][i], v[r][q][i], pair);
            }
            sum[r] = both(pair);
        }
        if constexpr (R == 2) row_sums(sum[0], sum[1], s_var, block);
        else sum[0] = row_sum(sum[0], s_var, block);
#pragma unroll
        for (int r = 0; r < R; r++) rstd[r] = rsqrtf(fmaf(sum[r], inv.nearest, eps));
        if (part.in_row() == 0) {
#pragma unroll
            for (int r = 0; r < R; r++)
                if (t + r * step < T) {
                    if (mean_out) mean_out[t + r * step] = mean[r];
                    if (rstd_out) rstd_out[t + r * step] = rstd[r];
                }
        }
#pragma unroll
        for (int q = 0; q < Q; q++) {
            f2 w[N], b[N];
            scale.get(part, q, w);
            shift.get(part, q, b);
#pragma unroll
            for (int r = 0; r < R; r++) {
                if (t + r * step >= T) break;
                const f2 rr = pack2(rstd[r], rstd[r]);
                f2 out[N];
#pragma unroll
                for (int i = 0; i < N; i++) out[i] = fma2(mul2(v[r][q][i], rr), w[i], b[i]);
                part.store(rows_on(y, t + r * step, y_pitch), q, out);
            }
        }
    };
    // a copy of the loop's body for every stage that a row can lie in, so that stages are constants
    constexpr int kPhases = V == 1 ? 1 : S / R;
    static_assert(V == 1 || S % R == 0, "whole groups of rows");
    while (t < T) {
#pragma unroll
        for (int phase = 0; phase < kPhases; phase++) {
            if (t >= T) break;
            rows(phase * R);
            t += R * step;
        }
    }
}

// The column sums of dy * h and dy stay in registers over all of a block's rows; each block leaves them in `partial`.  With
// several vectors per thread the row itself does not fit beside them and is read from its stage again for dx.
// Columns that the row does not have must not meet the others in the sum of g * h: they have g = 0, but h = (0 - mean) * rstd, and
// where that is infinite (a row of equal numbers 2^100, eps 1e-30) the product is NaN.  At the limit of the registers every form needs a way of its
// own: a thread with one vector behind the row's end has mean = rstd = 0 (kNone); in the forms for few threads, where these loads diverge
// (20000 x 2224 of bf16 54 us, with them 60), it adds nothing in the end; of several vectors those that may be missing (the second half: by_width)
// have rstd = 0; single elements are masked in the product.  Against sums that take them in: 16384 x 4096 of bf16 68 us both, 65536 x 264 34 and 33,
// 4096 x 16384 from fp32 146 and 144, of bf16 113 and 116.
template <typename XT, typename YT, int V, int G, int P, bool FEW>
__global__ void __launch_bounds__(kBwdBlock<XT, V, G, P>, kBwdBlocks<XT, V, G, P>)
norm_bwd_kernel(const YT *__restrict__ dy, uint32_t dy_pitch, const XT *__restrict__ x, uint32_t x_pitch, const float *__restrict__ gamma,
                const float *__restrict__ mean, const float *__restrict__ rstd, XT *__restrict__ dx, uint32_t dx_pitch,
                float *__restrict__ partial, int T, int d, int row_threads) {
    using Mine = Part<V, G, P, FEW>;
    constexpr int B = kBwdBlock<XT, V, G, P>, S = kBwdStages<XT, YT, V, G, P>, Q = Mine::kGroups, N = Mine::kPairs;
    constexpr bool kAgain = Q > 1;
    static_assert(S >= 2, "a row is read from one stage while another one fills");
    extern __shared__ __align__(16) char sm[];
    __shared__ float s_sum[2][Block<B, G, FEW>::kWords];
    const int group = FEW ? threadIdx.x / row_threads : threadIdx.x / G;
    const int step = gridDim.x * (FEW ? blockDim.x / row_threads : B / G);
    const Block<B, G, FEW> block{row_threads};
    block.clear(s_sum);
    const Mine part = {d, block.in_row()};
    f2 dg[Q][N], db[Q][N];
#pragma unroll
    for (int q = 0; q < Q; q++)
#pragma unroll
        for (int i = 0; i < N; i++) dg[q][i] = db[q][i] = 0ull;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(sm);
    Ahead<XT, B, V, G, P, S> ahead_x(ring, d, part.in_row());
    Ahead<YT, B, V, G, P, S> ahead_y(ring + S * Ahead<XT, B, V, G, P, S>::kStage, d, part.in_row());
    const float inv = 1.f / (float)d;
    pdl_trigger();
    pdl_wait();
    const Param<V, G, P, FEW, P * V <= 8> scale(gamma, part, 1.f);
    int t = blockIdx.x * (FEW ? blockDim.x / row_threads : B / G) + group, next = t;
    x += ahead_x.col;
    dy += ahead_y.col;
    dx += part.col(0);
    auto fetch = [&](int stage) {
        if (next < T) {
            ahead_x.fetch(stage, rows_on(x, next, x_pitch), d);
            ahead_y.fetch(stage, rows_on(dy, next, dy_pitch), d);
        }
        copies_commit();
        next += step;
    };
#pragma unroll
    for (int i = 0; i < S - 1; i++) fetch(i);
    constexpr bool kNone = V == 8 && P == 1 && !FEW;
    float m = 0.f, r = 0.f;
    if (t < T && (!kNone || part.has(0))) {
        m = mean[t];
        r = rstd[t];
    }
    auto row = [&](int stage, int turn) {
        f2 h[Q][N], g[Q][N], sum_g = 0ull, sum_gh = 0ull;
        const f2 minus = pack2(-m, -m), rr = pack2(r, r);
        if (t + step < T && (!kNone || part.has(0))) {
            m = mean[t + step];
            r = rstd[t + step];
        }
        copies_wait<S - 2>();
        if constexpr (!kAgain) {
            ahead_x.take(stage, 0, h[0]);
            ahead_y.take(stage, 0, g[0]);
        }
        fetch((stage + S - 1) % S);
#pragma unroll
        for (int q = 0; q < Q; q++) {
            if constexpr (kAgain) {
                ahead_x.take(stage, q, h[q]);
                ahead_y.take(stage, q, g[q]);
            }
            f2 w[N];
            scale.get(part, q, w);
#pragma unroll
            for (int i = 0; i < N; i++) {
                h[q][i] = mul2(add2(h[q][i], minus), kAgain && 2 * q >= P && !part.has(q) ? 0ull : rr);
                dg[q][i] = fma2(g[q][i], h[q][i], dg[q][i]);
                db[q][i] = add2(db[q][i], g[q][i]);
                g[q][i] = mul2(g[q][i], w[i]);
                sum_g = add2(sum_g, g[q][i]);
                sum_gh = part.add_product(i, g[q][i], h[q][i], sum_gh);
            }
        }
        float mg = both(sum_g), mh = both(sum_gh);
        if (FEW && !part.has(0)) mh = 0.f;
        row_sums(mg, mh, s_sum[turn] + group * (2 * G / 32), block);
        const f2 less = pack2(-mg * inv, -mg * inv), slope = pack2(-mh * inv, -mh * inv);
#pragma unroll
        for (int q = 0; q < Q; q++) {
            f2 out[N];
            if constexpr (kAgain) {
                f2 w[N];
                ahead_x.take(stage, q, h[q]);
                ahead_y.take(stage, q, g[q]);
                scale.get(part, q, w);
#pragma unroll
                for (int i = 0; i < N; i++) {
                    h[q][i] = mul2(add2(h[q][i], minus), rr);
                    g[q][i] = mul2(g[q][i], w[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < N; i++) out[i] = mul2(fma2(h[q][i], slope, add2(g[q][i], less)), rr);
            part.store(rows_on(dx, t, dx_pitch), q, out);
        }
    };
    // as in the forward kernel; an even number of copies, for the two sets of sums that take turns
    constexpr int kPhases = S % 2 ? 2 * S : S;
    while (t < T) {
#pragma unroll
        for (int phase = 0; phase < kPhases; phase++) {
            if (t >= T) break;
            row(phase % S, phase % 2);
            t += step;
        }
    }
    if (!partial) return;
    // column sums of the block: the rows' groups joined through shared memory, in order
    float *sums = partial + (int64_t)blockIdx.x * 2 * d;
    if constexpr (G == B) {
#pragma unroll
        for (int q = 0; q < Q; q++) {
            part.store(sums + part.col(0), q, dg[q]);
            part.store(sums + d + part.col(0), q, db[q]);
        }
    } else {
        const int cols = block.threads() * P * V;  // that a row's threads cover
        float *s = reinterpret_cast<float *>(sm);
        copies_wait<0>();
        __syncthreads();
#pragma unroll
        for (int q = 0; q < Q; q++)
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int c = V == 8 ? part.col(q) + 2 * i : part.in_row() + 2 * i * G, next_c = V == 8 ? 1 : G;
                float *a = s + group * 2 * cols + c, *b = a + cols;
                unpack2(dg[q][i], a[0], a[next_c]);
                unpack2(db[q][i], b[0], b[next_c]);
            }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * cols; i += block.all()) {
            const int which = i / cols, col = i % cols;
            if (col >= d) continue;
            float sum = 0.f;
#pragma unroll
            for (int q = 0; q < block.rows(); q++) sum += s[(q * 2 + which) * cols + col];
            sums[which * d + col] = sum;
        }
    }
}

// dgamma and dbeta from n partial sums: 32 columns per block, a warp takes every 32nd sum, then the warps' are joined.
__global__ void __launch_bounds__(1024)
norm_join_kernel(const float *__restrict__ partial, int n, int d, float *__restrict__ dgamma, float *__restrict__ dbeta) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float *out = blockIdx.y ? dbeta : dgamma;
    pdl_trigger();
    pdl_wait();
    if (!out) return;
    float sum = 0.f;
    if (c < d)
#pragma unroll 10
        for (int i = warp; i < n; i += 32) sum += partial[((int64_t)i * 2 + blockIdx.y) * d + c];
    s[warp][lane] = sum;
    __syncthreads();
    sum = s[lane][warp];  // warp's column, the sum of warp `lane`
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    if (lane == 0 && blockIdx.x * 32 + warp < d) out[blockIdx.x * 32 + warp] = sum;
}

// Row slices of norm_cols_kernel, whose column sums are kept apart: as many as give every SM kColBlocks blocks, but eight at least, so that
// no sum is longer than an eighth of the rows.
constexpr int kSlicesMin = 8, kSlicesMax = 64, kColBlocks = 4;
// Blocks of norm_bwd_kernel, and with that column sums kept apart: two on each of up to 160 SMs.
constexpr int kBwdBlocksMax = 320;

int slices_of(int T, int d, int per_thread, int sms) {
    int want = ceil_div(sms * kColBlocks, ceil_div(d, kColThreads * per_thread));
    want = want < kSlicesMin ? kSlicesMin : want;
    const int most = T < kSlicesMax ? (T < 1 ? 1 : T) : kSlicesMax;
    return want < most ? want : most;
}

// Calls f with the vector width, threads per row and vectors per thread (integral constants) for rows of width d, or
// returns false where they do not fit a block's registers.  Vectors: the fewest threads that hold the row with one each, then two, with
// the exceptions below.
// Single elements: eight per thread, then sixteen (fewer elements and more threads per row: 20000 x 1001 of bf16 forward 53 us with four on 512
// threads, 21 with eight on 128, 35 with sixteen on 64).
template <int N>
using Int = std::integral_constant<int, N>;
template <bool BACK, typename XT, typename YT, typename F>
bool by_width(bool vec, int T, int d, F f) {
    if (vec) {
        // Two vectors on half the threads halve the shuffles and barriers; forward that is faster for rows of bf16 from bf16 where
        // many of them (60000 x 640: 35 us, with two vectors 30; 6000: 5.4 and 5.6) are not too wide (x 896: 41 and 35, 65536 x 1024: 44
        // and 48), ...
        if constexpr (!BACK && sizeof(XT) == 2 && sizeof(YT) == 2)
            if (T >= 8000 && d > 512 && d <= 896) return f(Int<8>(), Int<64>(), Int<2>()), true;
        // ... and where a row has an SM to itself otherwise and now two share it: to bf16 from bf16 (8192 x 8192: 47 and 43, 8000 x 5120: 33
        // and 35) and from fp32 (8000 x 5888: 51 and 44, 8192 x 8192: 63 and 68), not to fp32 (8192 x 8192: 82 and 97).
        if constexpr (!BACK && sizeof(YT) == 2)
            if (sizeof(XT) == 2 ? d > 5120 && d <= 8192 : d > 4096 && d <= 7168) return f(Int<8>(), Int<512>(), Int<2>()), true;
        if (d <= 256) f(Int<8>(), Int<32>(), Int<1>());
        else if (d <= 512) f(Int<8>(), Int<64>(), Int<1>());
        else if (d <= 1024) f(Int<8>(), Int<128>(), Int<1>());
        else if (d <= 2048) f(Int<8>(), Int<256>(), Int<1>());
        else if (d <= 4096) f(Int<8>(), Int<512>(), Int<1>());
        else if (d <= 8192) f(Int<8>(), Int<1024>(), Int<1>());
        else if (d <= 16384) {
            // backward, two vectors' column sums spill from 64 registers; four vectors have 128
            if constexpr (BACK) f(Int<8>(), Int<512>(), Int<4>());
            else f(Int<8>(), Int<1024>(), Int<2>());
        } else return false;
    } else {
        if (d <= 256) f(Int<1>(), Int<32>(), Int<8>());
        else if (d <= 512) f(Int<1>(), Int<64>(), Int<8>());
        else if (d <= 1024) f(Int<1>(), Int<128>(), Int<8>());
        else if (d <= 2048) f(Int<1>(), Int<256>(), Int<8>());
        else if (d <= 4096) f(Int<1>(), Int<512>(), Int<8>());
        else if (d <= 8192) f(Int<1>(), Int<512>(), Int<16>());
        else return false;
    }
    return true;
}

// The whole warps that a row of width d needs where a thread holds one vector, in threads.
int few_threads(int d) { return ceil_div(d, 256) * 32; }
// Which kernels have a form for few threads.  Forward it gains wherever y is bf16 (20000 x 2224 from fp32: 60 us, with few threads 43;
// from bf16 41 and 31; 40000 x 1536 from bf16 44 and 40).  Rows of fp32 results are slower several at a time (40000 x 1200: 64 and 72), so
// there only those of a whole block have it (10000 x 4352: 73 and 63).
template <typename YT, int V, int G, int P>
constexpr bool few_forward = V == 8 && P == 1 && G >= 128 && (sizeof(YT) == 2 || G == 1024);
// Backward, where more rows fit a block: for bf16 x (40000 x 1200 of bf16: 68 us, with few threads 54; 20000 x 2224: 68 and 54), and for
// fp32 x with bf16 dy in the middle (40000 x 1200: 103 and 87, but 60000 x 640: 67 and 71); not with both fp32 (40000 x 1200: 90 and 96).
template <typename XT, typename YT, int V, int G, int P>
constexpr bool few_backward = V == 8 && P == 1 && G >= 128 && G < kBwdBlock<XT, V, G, P> && (sizeof(XT) == 2 || (sizeof(YT) == 2 && G == 256));

template <typename K>
cudaError_t allow_smem(K kern, size_t bytes, PerDeviceOnce &once) {
    bool *done = once.slot();
    if (done && *done) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && done) *done = true;
    return e;
}

}  // namespace
}  // namespace omoe

using namespace omoe;

extern "C" {

int omoe_layer_norm(const void *x_dev, int64_t ldx, int32_t x_dtype, const float *gamma_dev, const float *beta_dev, float eps,
                    void *y_dev, int64_t ldy, int32_t y_dtype, float *mean_dev, float *rstd_dev, int32_t T, int32_t d,
                    void *cuda_stream) {
    const char *fn = "omoe_layer_norm";
    if (T < 0) return ops_fail(OMOE_ERR_INVALID, fn, "T must not be negative");
    if (T > kRowsMax) return ops_fail(OMOE_ERR_TOO_LARGE, fn, "T is beyond the limit");
    if (!(eps >= 0.f)) return ops_fail(OMOE_ERR_INVALID, fn, "eps must not be negative");
    const Rows x = {x_dev, ldx, x_dtype, T, d}, y = {y_dev, ldy, y_dtype, T, d};
    if (const char *bad = rows_wrong(x)) return ops_fail(OMOE_ERR_INVALID, fn, bad);
    if (const char *bad = rows_wrong(y)) return ops_fail(OMOE_ERR_INVALID, fn, bad);
    if (misaligned(gamma_dev, 4) || misaligned(beta_dev, 4) || misaligned(mean_dev, 4) || misaligned(rstd_dev, 4))
        return ops_fail(OMOE_ERR_INVALID, fn, "fp32 buffers must be 4-byte aligned");
    const Rows all[] = {y, words(mean_dev, T), words(rstd_dev, T), x, words(gamma_dev, d), words(beta_dev, d)};
    if (int rc = ops_apart(all, 6, 3, fn)) return rc;
    if (T == 0) return ops_ok();
    const int sms = ops_sm_count();
    if (!sms) return ops_fail(OMOE_ERR_CUDA, fn, "no device");
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    const Inverse inverse(d);
    return ops_launched(by_types(x_dtype, y_dtype, [&](auto *xt, auto *yt) {
        using XT = std::remove_pointer_t<decltype(xt)>;
        using YT = std::remove_pointer_t<decltype(yt)>;
        cudaError_t e = cudaSuccess;
        // (parameters that may lie anywhere, behind a branch in the kernels, cost the aligned ones: 65536 x 1024 of bf16 44 -> 45 us, 4096 x 16384
        // 58 -> 66 and backward 113 -> 138)
        const bool vec = rows_vector(x) && rows_vector(y) && !misaligned(gamma_dev, 32) && !misaligned(beta_dev, 32);
        if (by_width<false, XT, YT>(vec, T, d,
                     [&](auto v, auto g, auto p) {
                         constexpr int V = decltype(v)::value, G = decltype(g)::value, P = decltype(p)::value;
                         constexpr size_t smem = kFwdStages<XT, V, G, P> * Ahead<XT, kFwdBlock<G>, V, G, P, 2>::kStage;
                         auto launch = [&](auto kern, PerDeviceOnce &once, int row) {
                             e = allow_smem(kern, smem, once);
                             if (e != cudaSuccess) return;
                             const int at_once = kFwdBlock<G> / row, threads = at_once * row;
                             const int blocks = ceil_div(T, at_once), most = 1024 / threads * sms;
                             e = launch_ex(kern, dim3(blocks < most ? blocks : most), dim3(threads), smem, s, ops_pdl(),
                                           static_cast<const XT *>(x_dev), (uint32_t)(ldx * sizeof(XT)), gamma_dev, beta_dev, eps,
                                           static_cast<YT *>(y_dev), (uint32_t)(ldy * sizeof(YT)), mean_dev, rstd_dev, T, d, inverse, row);
                         };
                         static PerDeviceOnce once;
                         if constexpr (few_forward<YT, V, G, P>) {
                             static PerDeviceOnce once_few;
                             if (few_threads(d) < G) return launch(norm_kernel<XT, YT, V, G, P, true>, once_few, few_threads(d));
                         }
                         launch(norm_kernel<XT, YT, V, G, P, false>, once, G);
                     }))
            return e;
        auto wide = [&](auto kern) {
            return launch_ex(kern, dim3(T), dim3(kWideThreads), 0, s, ops_pdl(), static_cast<const XT *>(x_dev), ldx, gamma_dev,
                             beta_dev, eps, static_cast<YT *>(y_dev), ldy, mean_dev, rstd_dev, d);
        };
        return vec ? wide(norm_wide_kernel<XT, YT, 8>) : wide(norm_wide_kernel<XT, YT, 1>);
    }), fn);
}

int64_t omoe_layer_norm_backward_workspace(int32_t T, int32_t d) {
    if (T < 0 || d < 1) return OMOE_ERR_INVALID;
    return (int64_t)(T < kBwdBlocksMax ? (T < 1 ? 1 : T) : kBwdBlocksMax) * 2 * d * sizeof(float);
}

int omoe_layer_norm_backward(const void *dy_dev, int64_t lddy, int32_t dy_dtype, const void *x_dev, int64_t ldx, int32_t x_dtype,
                             const float *gamma_dev, const float *mean_dev, const float *rstd_dev, void *dx_dev, int64_t lddx,
                             float *dgamma_dev, float *dbeta_dev, int32_t T, int32_t d, void *workspace_dev,
                             int64_t workspace_bytes, void *cuda_stream) {
    const char *fn = "omoe_layer_norm_backward";
    if (T < 0) return ops_fail(OMOE_ERR_INVALID, fn, "T must not be negative");
    if (T > kRowsMax) return ops_fail(OMOE_ERR_TOO_LARGE, fn, "T is beyond the limit");
    const Rows dx = {dx_dev, lddx, x_dtype, T, d}, dy = {dy_dev, lddy, dy_dtype, T, d}, x = {x_dev, ldx, x_dtype, T, d};
    for (const Rows *r : {&dx, &dy, &x})
        if (const char *bad = rows_wrong(*r)) return ops_fail(OMOE_ERR_INVALID, fn, bad);
    if (T > 0 && (!mean_dev || !rstd_dev)) return ops_fail(OMOE_ERR_INVALID, fn, "null buffer");
    if (misaligned(gamma_dev, 4) || misaligned(mean_dev, 4) || misaligned(rstd_dev, 4) || misaligned(dgamma_dev, 4) ||
        misaligned(dbeta_dev, 4))
        return ops_fail(OMOE_ERR_INVALID, fn, "fp32 buffers must be 4-byte aligned");
    if (workspace_bytes < omoe_layer_norm_backward_workspace(T, d) || !workspace_dev || misaligned(workspace_dev, 32))
        return ops_fail(OMOE_ERR_INVALID, fn, "the workspace is missing, misaligned or too small");
    const Rows all[] = {dx, words(dgamma_dev, d), words(dbeta_dev, d), words(workspace_dev, omoe_layer_norm_backward_workspace(T, d) / 4),
                        dy, x, words(gamma_dev, d), words(mean_dev, T), words(rstd_dev, T)};
    if (int rc = ops_apart(all, 9, 4, fn)) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    const int sms = ops_sm_count();
    if (!sms) return ops_fail(OMOE_ERR_CUDA, fn, "no device");
    float *partial = static_cast<float *>(workspace_dev);
    const int cols = ceil_div(d, 32);
    const bool params = dgamma_dev || dbeta_dev;
    return ops_launched(by_types(x_dtype, dy_dtype, [&](auto *xt, auto *yt) {
        using XT = std::remove_pointer_t<decltype(xt)>;
        using YT = std::remove_pointer_t<decltype(yt)>;
        const YT *g = static_cast<const YT *>(dy_dev);
        const XT *in = static_cast<const XT *>(x_dev);
        cudaError_t e = cudaSuccess;
        int sums = 0;  // column sums in the workspace
        const bool vec = rows_vector(x) && rows_vector(dy) && rows_vector(dx) && !misaligned(gamma_dev, 32);
        if (T > 0 && by_width<true, XT, YT>(vec, T, d,
                              [&](auto v, auto gg, auto p) {
                                  constexpr int V = decltype(v)::value, G = decltype(gg)::value, P = decltype(p)::value;
                                  constexpr int S = kBwdStages<XT, YT, V, G, P>, B = kBwdBlock<XT, V, G, P>;
                                  if constexpr (S >= 2) {
                                      constexpr size_t ring = S * (Ahead<XT, B, V, G, P, S>::kStage + Ahead<YT, B, V, G, P, S>::kStage);
                                      constexpr size_t join = G < B ? 2 * B * P * V * sizeof(float) : 0;
                                      constexpr size_t smem = ring > join ? ring : join;
                                      auto launch = [&](auto kern, PerDeviceOnce &once, int row) {
                                          e = allow_smem(kern, smem, once);
                                          if (e != cudaSuccess) return;
                                          const int at_once = B / row, blocks = ceil_div(T, at_once);
                                          int most = kBwdBlocks<XT, V, G, P> * sms;
                                          most = most < kBwdBlocksMax ? most : kBwdBlocksMax;
                                          sums = blocks < most ? blocks : most;
                                          e = launch_ex(kern, dim3(sums), dim3(at_once * row), smem, s, ops_pdl(), g,
                                                        (uint32_t)(lddy * sizeof(YT)), in, (uint32_t)(ldx * sizeof(XT)), gamma_dev, mean_dev,
                                                        rstd_dev, static_cast<XT *>(dx_dev), (uint32_t)(lddx * sizeof(XT)),
                                                        params ? partial : nullptr, T, d, row);
                                      };
                                      static PerDeviceOnce once;
                                      if constexpr (few_backward<XT, YT, V, G, P>) {
                                          static PerDeviceOnce once_few;
                                          if (B / few_threads(d) > B / G)
                                              return launch(norm_bwd_kernel<XT, YT, V, G, P, true>, once_few, few_threads(d));
                                      }
                                      launch(norm_bwd_kernel<XT, YT, V, G, P, false>, once, G);
                                  }
                              }) && (e != cudaSuccess || sums > 0)) {
            if (e != cudaSuccess || !params) return e;
            return launch_ex(norm_join_kernel, dim3(cols, 2), dim3(1024), 0, s, ops_pdl(), partial, sums, d, dgamma_dev, dbeta_dev);
        }
        int slices = 0;
        auto wide = [&](auto kern, auto cols_kern, int V) {
            cudaError_t e = cudaSuccess;
            slices = slices_of(T, d, V, sms);
            if (T > 0)
                e = launch_ex(kern, dim3(T), dim3(kWideThreads), 0, s, ops_pdl(), g, lddy, in, ldx, gamma_dev, mean_dev, rstd_dev,
                              static_cast<XT *>(dx_dev), lddx, d);
            if (e != cudaSuccess || !params) return e;
            return launch_ex(cols_kern, dim3(ceil_div(d, kColThreads * V), slices), dim3(kColThreads), 0, s, ops_pdl(), g, lddy, in, ldx, mean_dev, rstd_dev,
                             partial, T, d, ceil_div(T, slices));
        };
        e = vec ? wide(norm_bwd_wide_kernel<XT, YT, 8>, norm_cols_kernel<XT, YT, 8>, 8)
                : wide(norm_bwd_wide_kernel<XT, YT, 1>, norm_cols_kernel<XT, YT, 1>, 1);
        if (e != cudaSuccess || !params) return e;
        return launch_ex(norm_join_kernel, dim3(cols, 2), dim3(1024), 0, s, ops_pdl(), partial, slices, d, dgamma_dev, dbeta_dev);
    }), fn);
}

}  // extern "C"
