// Layer norm of rows, forward and backward.
//
//   mean = sum(x) / d;  var = sum((x - mean)^2) / d;  rstd = 1 / sqrt(var + eps);  h = (x - mean) * rstd
//   y = h * gamma + beta
//   g = dy * gamma;  dx = rstd * (g - sum(g) / d - h * sum(g * h) / d);  dgamma = sum over rows of dy * h;  dbeta = of dy
//
// The variance is taken after the mean: the difference of the mean of squares and the squared mean loses all digits on rows
// whose offset is large against their spread.  All sums are fp32 in a fixed order.
#include "ops.cuh"

namespace omoe {

namespace {

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

// Any width: a block walks its row three times, from cache after the first.
template <typename XT, typename YT>
__global__ void __launch_bounds__(kWideThreads)
norm_wide_kernel(const XT *__restrict__ x, int64_t ldx, const float *__restrict__ gamma, const float *__restrict__ beta,
                 float eps, YT *__restrict__ y, int64_t ldy, float *__restrict__ mean_out, float *__restrict__ rstd_out, int d) {
    __shared__ float s[kWideThreads / 32];
    const int64_t t = blockIdx.x;
    pdl_trigger();
    pdl_wait();
    const XT *row = x + t * ldx;
    float sum = 0.f;
    for (int c = threadIdx.x; c < d; c += kWideThreads) sum += (float)row[c];
    const float mean = block_sum(sum, s) / (float)d;
    sum = 0.f;
    for (int c = threadIdx.x; c < d; c += kWideThreads) {
        const float v = (float)row[c] - mean;
        sum = fmaf(v, v, sum);
    }
    const float rstd = 1.f / sqrtf(block_sum(sum, s) / (float)d + eps);
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[t] = mean;
        if (rstd_out) rstd_out[t] = rstd;
    }
    for (int c = threadIdx.x; c < d; c += kWideThreads) {
        const float h = ((float)row[c] - mean) * rstd;
        y[t * ldy + c] = (YT)fmaf(h, gamma ? gamma[c] : 1.f, beta ? beta[c] : 0.f);
    }
}

template <typename XT, typename YT>
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
    for (int c = threadIdx.x; c < d; c += kWideThreads) {
        const float g = (float)dy[t * lddy + c] * (gamma ? gamma[c] : 1.f);
        sum += g;
        dot = fmaf(g, ((float)x[t * ldx + c] - m) * r, dot);
    }
    const float mg = block_sum(sum, s[0]) / (float)d, mh = block_sum(dot, s[1]) / (float)d;
    for (int c = threadIdx.x; c < d; c += kWideThreads) {
        const float g = (float)dy[t * lddy + c] * (gamma ? gamma[c] : 1.f), h = ((float)x[t * ldx + c] - m) * r;
        dx[t * lddx + c] = (XT)(r * (g - mg - h * mh));
    }
}

// Column sums of a slice of the rows: partial[slice][0][d] of dy * h, [1][d] of dy.
template <typename XT, typename YT>
__global__ void __launch_bounds__(256)
norm_cols_kernel(const YT *__restrict__ dy, int64_t lddy, const XT *__restrict__ x, int64_t ldx,
                 const float *__restrict__ mean, const float *__restrict__ rstd, float *__restrict__ partial, int T, int d,
                 int slice) {
    __shared__ float s[2][8][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    pdl_trigger();
    pdl_wait();
    const int64_t t0 = (int64_t)blockIdx.y * slice, t1 = min((int64_t)T, t0 + slice);
    float a = 0.f, b = 0.f;
    if (c < d)
        for (int64_t t = t0 + warp; t < t1; t += 8) {
            const float g = (float)dy[t * lddy + c];
            a = fmaf(g, ((float)x[t * ldx + c] - mean[t]) * rstd[t], a);
            b += g;
        }
    s[0][warp][lane] = a;
    s[1][warp][lane] = b;
    __syncthreads();
    if (warp < 2 && c < d) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) sum += s[warp][i][lane];
        partial[((int64_t)blockIdx.y * 2 + warp) * d + c] = sum;
    }
}

// ---- rows that fit a block's registers ----------------------------------------------------------------------------
//
// A block of 512 threads works on 512 / G rows at a time: G threads hold a row, P vectors of V elements each, and walk
// the rows of the grid with a stride.  Rows arrive in a ring of S stages in shared memory by asynchronous copies; a thread
// copies exactly the vectors it will read, so the ring needs no barrier, and the loads of the next S - 1 rows are on
// their way while a row is reduced.  The reductions are what threads of a row meet for: warp shuffles, then one named barrier each.
constexpr int kBlock = 512;

__device__ __forceinline__ void copy16(uint32_t to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// This thread's vectors of the rows ahead.  V = 8: S stages of shared memory.  V = 1 (rows that are not 16-byte aligned):
// one row ahead, in registers.
template <typename T, int V, int P, int S>
struct Ahead {
    uint32_t slot;
    static constexpr int kBytes = V * sizeof(T);
    // vectors behind the row's end are zeros in every stage from the start
    __device__ __forceinline__ Ahead(uint32_t ring, const int (&c)[P], int d) : slot(ring + threadIdx.x * 16) {
#pragma unroll
        for (int p = 0; p < P; p++)
            if (c[p] >= d)
                for (int i = 0; i < S; i++)
#pragma unroll
                    for (int q = 0; q < kBytes / 16; q++)
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(slot + ((i * P + p) * (kBytes / 16) + q) * (kBlock * 16)), "r"(0) : "memory");
    }
    static constexpr int kStage = kBlock * P * kBytes;
    __device__ __forceinline__ void fetch(int stage, const T *row, const int (&c)[P], int d) {
#pragma unroll
        for (int p = 0; p < P; p++)
            if (c[p] < d)
#pragma unroll
                for (int q = 0; q < kBytes / 16; q++)
                    copy16(slot + ((stage * P + p) * (kBytes / 16) + q) * (kBlock * 16), reinterpret_cast<const char *>(row + c[p]) + q * 16);
    }
    __device__ __forceinline__ void take(int stage, float (&v)[P][V]) const {
#pragma unroll
        for (int p = 0; p < P; p++) {
            uint4 r[kBytes / 16];
#pragma unroll
            for (int q = 0; q < kBytes / 16; q++)
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r[q].x), "=r"(r[q].y), "=r"(r[q].z), "=r"(r[q].w)
                             : "r"(slot + ((stage * P + p) * (kBytes / 16) + q) * (kBlock * 16)) : "memory");
            if constexpr (sizeof(T) == 2) unpack8(r[0], v[p]);
            else {
                const uint32_t w[8] = {r[0].x, r[0].y, r[0].z, r[0].w, r[1].x, r[1].y, r[1].z, r[1].w};
#pragma unroll
                for (int i = 0; i < 8; i++) v[p][i] = __uint_as_float(w[i]);
            }
        }
    }
};
template <typename T, int P, int S>
struct Ahead<T, 1, P, S> {
    Frag<T, 1> next[P];
    __device__ __forceinline__ Ahead(uint32_t, const int (&)[P], int) {
#pragma unroll
        for (int p = 0; p < P; p++) next[p].zero();
    }
    static constexpr int kStage = 0;
    __device__ __forceinline__ void fetch(int, const T *row, const int (&c)[P], int d) {
#pragma unroll
        for (int p = 0; p < P; p++)
            if (c[p] < d) next[p].load(row + c[p]);
    }
    __device__ __forceinline__ void take(int, float (&v)[P][1]) const {
#pragma unroll
        for (int p = 0; p < P; p++) next[p].get(v[p]);
    }
};

// Stages that fit a block's share of shared memory, where BLOCKS of them share an SM.
constexpr int stages(int stage_bytes, int blocks) {
    const int fit = stage_bytes ? 212992 / blocks / stage_bytes : 2;
    return fit > 6 ? 6 : fit;
}
// two blocks per SM, or one where that leaves fewer than three stages
template <typename XT, int V, int P>
constexpr int kFwdStages = V == 1 ? 2 : stages(kBlock * P * V * (int)sizeof(XT), kBlock * P * V * sizeof(XT) * 6 <= 212992 ? 2 : 1);
template <int P>
constexpr int kBwdBlocks = P == 1 ? 2 : 1;  // per SM: what the registers allow
template <typename XT, typename YT, int V, int P>
constexpr int kBwdStages = V == 1 ? 2 : stages(kBlock * P * V * (int)(sizeof(XT) + sizeof(YT)), kBwdBlocks<P>);

template <int G>
__device__ __forceinline__ void row_barrier() {
    if constexpr (G == kBlock) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"((int)threadIdx.x / G + 1), "n"(G) : "memory");
}

// The sum of v over the G threads of a row, in all of them.  s: G / 32 words of this row; between two uses the
// threads of the row have to meet at another barrier.
template <int G>
__device__ __forceinline__ float row_sum(float v, float *s) {
    constexpr int W = G / 32;
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if constexpr (W > 1) {
        const int lane = threadIdx.x & 31;
        if (lane == 0) s[(threadIdx.x % G) >> 5] = v;
        row_barrier<G>();
        v = s[lane & (W - 1)];
#pragma unroll
        for (int m = W / 2; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    }
    return v;
}

// Two sums at once, 2 * (G / 32) words: after one exchange the lower half of a warp adds up a and the upper half b.
template <int G>
__device__ __forceinline__ void row_sums(float &a, float &b, float *s) {
    constexpr int W = G / 32;
    const int lane = threadIdx.x & 31, half = lane >> 4;
    float v = half ? b : a;
    v += __shfl_xor_sync(0xffffffffu, half ? a : b, 16);
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if constexpr (W > 1) {
        if ((lane & 15) == 0) s[half * W + ((threadIdx.x % G) >> 5)] = v;
        row_barrier<G>();
        v = s[half * W + (lane & (W - 1))];
#pragma unroll
        for (int m = W / 2; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    }
    a = __shfl_sync(0xffffffffu, v, 0);
    b = __shfl_sync(0xffffffffu, v, 16);
}

// gamma or beta of this thread's columns: in registers where a thread has one vector, else from cache for every row.
template <int V, int P>
struct Param {
    static constexpr bool kKept = P * V <= 8;
    const float *p;
    float kept[kKept ? P : 1][V];
    __device__ __forceinline__ Param(const float *from, const int (&c)[P], int d, float missing) : p(from) {
        if constexpr (kKept)
#pragma unroll
            for (int q = 0; q < P; q++) {
#pragma unroll
                for (int i = 0; i < V; i++) kept[q][i] = missing;
                if (p && c[q] < d) {
                    Frag<float, V> f;
                    f.load_cached(p + c[q]);
                    f.get(kept[q]);
                }
            }
    }
    __device__ __forceinline__ void get(int q, int col, float missing, float (&v)[V]) const {
        if constexpr (kKept) {
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = kept[q][i];
        } else if (p) {
            Frag<float, V> f;
            f.load_cached(p + col);
            f.get(v);
        } else {
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = missing;
        }
    }
};

template <typename XT, typename YT, int V, int G, int P>
__global__ void __launch_bounds__(kBlock, 2)
norm_kernel(const XT *__restrict__ x, int64_t ldx, const float *__restrict__ gamma, const float *__restrict__ beta, float eps,
            YT *__restrict__ y, int64_t ldy, float *__restrict__ mean_out, float *__restrict__ rstd_out, int T, int d) {
    extern __shared__ __align__(16) char sm[];
    __shared__ float s_sum[2][kBlock / 32];
    constexpr int S = kFwdStages<XT, V, P>;
    static_assert(S >= 2, "a row is read from one stage while another one fills");
    const int group = threadIdx.x / G, in_row = threadIdx.x % G;
    const int64_t step = (int64_t)gridDim.x * (kBlock / G);
    int c[P];
#pragma unroll
    for (int p = 0; p < P; p++) c[p] = (p * G + in_row) * V;
    Ahead<XT, V, P, S> ahead((uint32_t)__cvta_generic_to_shared(sm), c, d);
    const float n = (float)d;
    pdl_trigger();
    pdl_wait();
    const Param<V, P> scale(gamma, c, d, 1.f), shift(beta, c, d, 0.f);
    int64_t t = (int64_t)blockIdx.x * (kBlock / G) + group, next = t;
#pragma unroll
    for (int i = 0; i < S - 1; i++, next += step) {
        if (next < T) ahead.fetch(i, x + next * ldx, c, d);
        copies_commit();
    }
    float *s_mean = s_sum[0] + group * (G / 32), *s_var = s_sum[1] + group * (G / 32);
    for (int stage = 0; t < T; t += step) {
        float v[P][V], sum = 0.f;
        copies_wait<S - 2>();
        ahead.take(stage, v);
        if (next < T) ahead.fetch(stage == 0 ? S - 1 : stage - 1, x + next * ldx, c, d);
        copies_commit();
        next += step;
        stage = stage + 1 == S ? 0 : stage + 1;
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int i = 0; i < V; i++) sum += v[p][i];
        const float mean = row_sum<G>(sum, s_mean) / n;
        sum = 0.f;
#pragma unroll
        for (int p = 0; p < P; p++)
            if (c[p] < d)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    v[p][i] -= mean;
                    sum = fmaf(v[p][i], v[p][i], sum);
                }
        const float rstd = 1.f / sqrtf(row_sum<G>(sum, s_var) / n + eps);
        if (in_row == 0) {
            if (mean_out) mean_out[t] = mean;
            if (rstd_out) rstd_out[t] = rstd;
        }
#pragma unroll
        for (int p = 0; p < P; p++)
            if (c[p] < d) {
                float w[V], b[V];
                Frag<YT, V> out;
                scale.get(p, c[p], 1.f, w);
                shift.get(p, c[p], 0.f, b);
#pragma unroll
                for (int i = 0; i < V; i++) w[i] = fmaf(v[p][i] * rstd, w[i], b[i]);
                out.set(w);
                out.store(y + t * ldy + c[p]);
            }
    }
}

template <typename XT, typename YT, int V, int G, int P>
__global__ void __launch_bounds__(kBlock, kBwdBlocks<P>)
norm_bwd_kernel(const YT *__restrict__ dy, int64_t lddy, const XT *__restrict__ x, int64_t ldx, const float *__restrict__ gamma,
                const float *__restrict__ mean, const float *__restrict__ rstd, XT *__restrict__ dx, int64_t lddx,
                float *__restrict__ partial, int T, int d) {
    extern __shared__ __align__(16) char sm[];
    __shared__ float s_sum[2][2 * kBlock / 32];
    constexpr int S = kBwdStages<XT, YT, V, P>;
    static_assert(S >= 2, "a row is read from one stage while another one fills");
    const int group = threadIdx.x / G, in_row = threadIdx.x % G;
    const int64_t step = (int64_t)gridDim.x * (kBlock / G);
    int c[P];
    float dg[P][V], db[P][V];
#pragma unroll
    for (int p = 0; p < P; p++) {
        c[p] = (p * G + in_row) * V;
#pragma unroll
        for (int i = 0; i < V; i++) dg[p][i] = db[p][i] = 0.f;
    }
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(sm);
    Ahead<XT, V, P, S> ahead_x(ring, c, d);
    Ahead<YT, V, P, S> ahead_y(ring + S * Ahead<XT, V, P, S>::kStage, c, d);
    const float n = (float)d;
    pdl_trigger();
    pdl_wait();
    const Param<V, P> scale(gamma, c, d, 1.f);
    int64_t t = (int64_t)blockIdx.x * (kBlock / G) + group, next = t;
#pragma unroll
    for (int i = 0; i < S - 1; i++, next += step) {
        if (next < T) {
            ahead_x.fetch(i, x + next * ldx, c, d);
            ahead_y.fetch(i, dy + next * lddy, c, d);
        }
        copies_commit();
    }
    float m = 0.f, r = 0.f;
    if (t < T) {
        m = mean[t];
        r = rstd[t];
    }
    for (int stage = 0, odd = 0; t < T; t += step, odd ^= 1) {
        float h[P][V], g[P][V], mg = 0.f, mh = 0.f;
        copies_wait<S - 2>();
        ahead_x.take(stage, h);
        ahead_y.take(stage, g);
        if (next < T) {
            const int to = stage == 0 ? S - 1 : stage - 1;
            ahead_x.fetch(to, x + next * ldx, c, d);
            ahead_y.fetch(to, dy + next * lddy, c, d);
        }
        copies_commit();
        next += step;
        stage = stage + 1 == S ? 0 : stage + 1;
        const float m0 = m, r0 = r;
        if (t + step < T) {
            m = mean[t + step];
            r = rstd[t + step];
        }
#pragma unroll
        for (int p = 0; p < P; p++)
            if (c[p] < d) {
                float w[V];
                scale.get(p, c[p], 1.f, w);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    h[p][i] = (h[p][i] - m0) * r0;
                    dg[p][i] = fmaf(g[p][i], h[p][i], dg[p][i]);
                    db[p][i] += g[p][i];
                    g[p][i] *= w[i];
                    mg += g[p][i];
                    mh = fmaf(g[p][i], h[p][i], mh);
                }
            }
        row_sums<G>(mg, mh, s_sum[odd] + group * (2 * G / 32));
        mg /= n;
        mh /= n;
#pragma unroll
        for (int p = 0; p < P; p++)
            if (c[p] < d) {
                Frag<XT, V> out;
                float v[V];
#pragma unroll
                for (int i = 0; i < V; i++) v[i] = r0 * fmaf(-h[p][i], mh, g[p][i] - mg);
                out.set(v);
                out.store(dx + t * lddx + c[p]);
            }
    }
    if (!partial) return;
    // column sums of the block: the rows' groups joined through shared memory, in order
    float *to = partial + (int64_t)blockIdx.x * 2 * d;
    if constexpr (G == kBlock) {
#pragma unroll
        for (int p = 0; p < P; p++)
            if (c[p] < d) {
                Frag<float, V> f;
                f.set(dg[p]);
                f.store(to + c[p]);
                f.set(db[p]);
                f.store(to + d + c[p]);
            }
    } else {
        constexpr int W = G * P * V;  // columns a group covers
        float *s = reinterpret_cast<float *>(sm);
        copies_wait<0>();
        __syncthreads();
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int i = 0; i < V; i++) {
                s[(group * 2) * W + c[p] + i] = dg[p][i];
                s[(group * 2 + 1) * W + c[p] + i] = db[p][i];
            }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * W; i += kBlock) {
            const int which = i / W, col = i % W;
            if (col >= d) continue;
            float sum = 0.f;
#pragma unroll
            for (int q = 0; q < kBlock / G; q++) sum += s[(q * 2 + which) * W + col];
            to[which * d + col] = sum;
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

// Row slices of the wide kernels whose column sums are kept apart.
constexpr int kSlicesMax = 64;
// Blocks of norm_bwd_kernel, and with that column sums kept apart: two on each of up to 160 SMs.
constexpr int kBwdBlocksMax = 320;

int slices_of(int T) { return T < kSlicesMax ? (T < 1 ? 1 : T) : kSlicesMax; }

// Calls f with the vector width, threads per row and vectors per thread (integral constants) for rows of width d, or
// returns false where they do not fit a block's registers.  Vectors: the fewest threads that hold the row with one each, then all of the
// block with more.  Single elements: four per thread.
template <int N>
using Int = std::integral_constant<int, N>;
template <typename F>
bool by_width(bool vec, int d, F f) {
    if (vec) {
        if (d <= 256) f(Int<8>(), Int<32>(), Int<1>());
        else if (d <= 512) f(Int<8>(), Int<64>(), Int<1>());
        else if (d <= 1024) f(Int<8>(), Int<128>(), Int<1>());
        else if (d <= 2048) f(Int<8>(), Int<256>(), Int<1>());
        else if (d <= 4096) f(Int<8>(), Int<512>(), Int<1>());
        else if (d <= 8192) f(Int<8>(), Int<512>(), Int<2>());
        else if (d <= 16384) f(Int<8>(), Int<512>(), Int<4>());
        else return false;
    } else {
        if (d <= 128) f(Int<1>(), Int<32>(), Int<4>());
        else if (d <= 512) f(Int<1>(), Int<128>(), Int<4>());
        else if (d <= 2048) f(Int<1>(), Int<512>(), Int<4>());
        else if (d <= 4096) f(Int<1>(), Int<512>(), Int<8>());
        else return false;
    }
    return true;
}

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
    if (!(eps >= 0.f)) return ops_fail(OMOE_ERR_INVALID, fn, "eps must not be negative");
    const Rows x = {x_dev, ldx, x_dtype, T, d}, y = {y_dev, ldy, y_dtype, T, d};
    if (const char *bad = rows_wrong(x)) return ops_fail(OMOE_ERR_INVALID, fn, bad);
    if (const char *bad = rows_wrong(y)) return ops_fail(OMOE_ERR_INVALID, fn, bad);
    if (rows_overlap(y, x)) return ops_fail(OMOE_ERR_INVALID, fn, "an output overlaps another buffer");
    if (misaligned(gamma_dev, 4) || misaligned(beta_dev, 4) || misaligned(mean_dev, 4) || misaligned(rstd_dev, 4))
        return ops_fail(OMOE_ERR_INVALID, fn, "fp32 buffers must be 4-byte aligned");
    if (T == 0) return ops_ok();
    const int sms = ops_sm_count();
    if (!sms) return ops_fail(OMOE_ERR_CUDA, fn, "no device");
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    return ops_launched(by_types(x_dtype, y_dtype, [&](auto *xt, auto *yt) {
        using XT = std::remove_pointer_t<decltype(xt)>;
        using YT = std::remove_pointer_t<decltype(yt)>;
        cudaError_t e = cudaSuccess;
        if (by_width(rows_vector(x) && rows_vector(y) && !misaligned(gamma_dev, 16) && !misaligned(beta_dev, 16), d,
                     [&](auto v, auto g, auto p) {
                         constexpr int V = decltype(v)::value, G = decltype(g)::value, P = decltype(p)::value;
                         constexpr size_t smem = kFwdStages<XT, V, P> * Ahead<XT, V, P, 2>::kStage;
                         static PerDeviceOnce once;
                         e = allow_smem(norm_kernel<XT, YT, V, G, P>, smem, once);
                         if (e != cudaSuccess) return;
                         const int blocks = ceil_div(T, kBlock / G), most = 2 * sms;
                         e = launch_ex(norm_kernel<XT, YT, V, G, P>, dim3(blocks < most ? blocks : most), dim3(kBlock), smem, s, ops_pdl(),
                                       static_cast<const XT *>(x_dev), ldx, gamma_dev, beta_dev, eps, static_cast<YT *>(y_dev), ldy,
                                       mean_dev, rstd_dev, T, d);
                     }))
            return e;
        return launch_ex(norm_wide_kernel<XT, YT>, dim3(T), dim3(kWideThreads), 0, s, ops_pdl(), static_cast<const XT *>(x_dev),
                         ldx, gamma_dev, beta_dev, eps, static_cast<YT *>(y_dev), ldy, mean_dev, rstd_dev, d);
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
    const Rows dx = {dx_dev, lddx, x_dtype, T, d}, dy = {dy_dev, lddy, dy_dtype, T, d}, x = {x_dev, ldx, x_dtype, T, d};
    for (const Rows *r : {&dx, &dy, &x})
        if (const char *bad = rows_wrong(*r)) return ops_fail(OMOE_ERR_INVALID, fn, bad);
    if (rows_overlap(dx, dy) || rows_overlap(dx, x)) return ops_fail(OMOE_ERR_INVALID, fn, "an output overlaps another buffer");
    if (T > 0 && (!mean_dev || !rstd_dev)) return ops_fail(OMOE_ERR_INVALID, fn, "null buffer");
    if (misaligned(gamma_dev, 4) || misaligned(mean_dev, 4) || misaligned(rstd_dev, 4) || misaligned(dgamma_dev, 4) ||
        misaligned(dbeta_dev, 4))
        return ops_fail(OMOE_ERR_INVALID, fn, "fp32 buffers must be 4-byte aligned");
    if (workspace_bytes < omoe_layer_norm_backward_workspace(T, d) || !workspace_dev || misaligned(workspace_dev, 16))
        return ops_fail(OMOE_ERR_INVALID, fn, "the workspace is missing, misaligned or too small");
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    const int sms = ops_sm_count();
    if (!sms) return ops_fail(OMOE_ERR_CUDA, fn, "no device");
    float *partial = static_cast<float *>(workspace_dev);
    const int slices = slices_of(T), cols = ceil_div(d, 32);
    const bool params = dgamma_dev || dbeta_dev;
    return ops_launched(by_types(x_dtype, dy_dtype, [&](auto *xt, auto *yt) {
        using XT = std::remove_pointer_t<decltype(xt)>;
        using YT = std::remove_pointer_t<decltype(yt)>;
        const YT *g = static_cast<const YT *>(dy_dev);
        const XT *in = static_cast<const XT *>(x_dev);
        cudaError_t e = cudaSuccess;
        int sums = 0;  // column sums in the workspace
        if (T > 0 && by_width(rows_vector(x) && rows_vector(dy) && rows_vector(dx) && !misaligned(gamma_dev, 16), d,
                              [&](auto v, auto gg, auto p) {
                                  constexpr int V = decltype(v)::value, G = decltype(gg)::value, P = decltype(p)::value;
                                  constexpr int S = kBwdStages<XT, YT, V, P>;
                                  if constexpr (S >= 2) {
                                      constexpr size_t ring = S * (Ahead<XT, V, P, S>::kStage + Ahead<YT, V, P, S>::kStage);
                                      constexpr size_t join = G < kBlock ? 2 * kBlock * P * V * sizeof(float) : 0;
                                      constexpr size_t smem = ring > join ? ring : join;
                                      static PerDeviceOnce once;
                                      e = allow_smem(norm_bwd_kernel<XT, YT, V, G, P>, smem, once);
                                      if (e != cudaSuccess) return;
                                      const int blocks = ceil_div(T, kBlock / G);
                                      int most = kBwdBlocks<P> * sms;
                                      most = most < kBwdBlocksMax ? most : kBwdBlocksMax;
                                      sums = blocks < most ? blocks : most;
                                      e = launch_ex(norm_bwd_kernel<XT, YT, V, G, P>, dim3(sums), dim3(kBlock), smem, s, ops_pdl(), g, lddy, in,
                                                    ldx, gamma_dev, mean_dev, rstd_dev, static_cast<XT *>(dx_dev), lddx,
                                                    params ? partial : nullptr, T, d);
                                  }
                              }) && (e != cudaSuccess || sums > 0)) {
            if (e != cudaSuccess || !params) return e;
            return launch_ex(norm_join_kernel, dim3(cols, 2), dim3(1024), 0, s, ops_pdl(), partial, sums, d, dgamma_dev, dbeta_dev);
        }
        if (T > 0) {
            e = launch_ex(norm_bwd_wide_kernel<XT, YT>, dim3(T), dim3(kWideThreads), 0, s, ops_pdl(), g, lddy, in, ldx, gamma_dev,
                          mean_dev, rstd_dev, static_cast<XT *>(dx_dev), lddx, d);
            if (e != cudaSuccess || !params) return e;
        }
        if (!params) return e;
        e = launch_ex(norm_cols_kernel<XT, YT>, dim3(cols, slices), dim3(256), 0, s, ops_pdl(), g, lddy, in, ldx, mean_dev,
                      rstd_dev, partial, T, d, ceil_div(T, slices));
        if (e != cudaSuccess) return e;
        return launch_ex(norm_join_kernel, dim3(cols, 2), dim3(1024), 0, s, ops_pdl(), partial, slices, d, dgamma_dev, dbeta_dev);
    }), fn);
}

}  // extern "C"
