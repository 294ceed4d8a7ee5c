// The global norm of many gradient tensors, and clipping by it.
//
// All tensors together are one sequence of chunks of 32 KB (a tensor's last one may be shorter), dealt out to the blocks in turn.  The table of
// tensors travels as a kernel parameter, so a call needs no copy and a captured graph keeps its own.
#include "ops.cuh"

#include <float.h>
#include <math.h>
#include <stdlib.h>

#include <algorithm>

namespace omoe {

namespace {

constexpr int kThreads = 256;
constexpr int kVectors = 8;  // of 16 bytes, that a thread has in flight; with 4 the sum of 1.4 GB takes 5 % longer, of bf16 half as long again
inline __host__ __device__ int chunk_elems(int dtype) { return kThreads * kVectors * 16 / (dtype == OMOE_BF16 ? 2 : 4); }
constexpr int kSlots = OMOE_GRAD_WORKSPACE_BYTES / 8;  // blocks' sums in the workspace

struct Entry {
    const void *in;
    void *out;
    int64_t count;
    int32_t first;  // chunk
    int32_t dtype;
};
// The tensors of one launch.  A parameter is copied with every launch, 32 KB of them for longer than 16 MB of gradients take; so there
// are tables of several sizes, the largest what fits the kernel parameters.
template <int N>
struct Table {
    Entry e[N];
    int32_t n, chunks;
};

// The sum of 16 values' squares.  In fp32 first, with four chains; where that overflows, or is so small that squares
// have lost digits, again in fp64 (the squares of fp32 values are exact there and their sum stays in range).
__device__ __forceinline__ double squares(const float *v) {
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; i++) s[i & 3] = fmaf(v[i], v[i], s[i & 3]);
    const float sum = (s[0] + s[1]) + (s[2] + s[3]);
    if (sum > 1e-20f && sum < 1e37f) return (double)sum;
    double d = 0.0;
#pragma unroll
    for (int i = 0; i < 16; i++) d = fma((double)v[i], (double)v[i], d);
    return d;
}

__device__ __forceinline__ double block_sum(double v, double *s) {
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    double sum = 0.0;
    for (int i = 0; i < (int)(blockDim.x >> 5); i++) sum += s[i];
    __syncthreads();
    return sum;
}

// The chunk's elements as this thread sees them.  Aligned chunks: vectors of 16 bytes, thread after thread, and what is left behind the
// last whole vector one element per thread in `rest`.  Others: element by element.
template <typename T>
struct Chunk {
    static constexpr int V = 16 / sizeof(T);
    uint4 r[kVectors];
    float rest;
    static __device__ __forceinline__ void unpack(const uint4 &r, float *v) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (V == 4) v[j] = __uint_as_float(w[j]);
            else {
                v[2 * j] = __uint_as_float(w[j] << 16);
                v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
        }
    }
    static __device__ __forceinline__ uint4 pack(const float *v) {
        if constexpr (V == 4)
            return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        else
            return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    }
    __device__ __forceinline__ void load(const T *p, int n) {
        const int whole = n / V;
        const uint4 *from = reinterpret_cast<const uint4 *>(p) + threadIdx.x;
#pragma unroll
        for (int i = 0; i < kVectors; i++) {
            r[i] = make_uint4(0, 0, 0, 0);
            if (i * kThreads + (int)threadIdx.x < whole) r[i] = from[i * kThreads];
        }
        rest = whole * V + (int)threadIdx.x < n ? (float)p[whole * V + threadIdx.x] : 0.f;
    }
    __device__ __forceinline__ void store(T *p, int n, float c) const {
        const int whole = n / V;
        uint4 *to = reinterpret_cast<uint4 *>(p) + threadIdx.x;
#pragma unroll
        for (int i = 0; i < kVectors; i++)
            if (i * kThreads + (int)threadIdx.x < whole) {
                float v[V];
                unpack(r[i], v);
#pragma unroll
                for (int j = 0; j < V; j++) v[j] *= c;
                to[i * kThreads] = pack(v);
            }
        if (whole * V + (int)threadIdx.x < n) p[whole * V + threadIdx.x] = (T)(rest * c);
    }
    __device__ __forceinline__ double sum() const {
        double s = (double)rest * (double)rest;
        constexpr int W = 16 / V;  // vectors whose squares are summed at a time
#pragma unroll
        for (int i = 0; i < kVectors; i += W) {
            float v[16];
#pragma unroll
            for (int j = 0; j < W; j++) unpack(r[i + j], v + j * V);
            s += squares(v);
        }
        return s;
    }
};
template <typename T>
__device__ double sum_elements(const T *p, int n) {
    double s = 0.0;
    for (int i0 = threadIdx.x; i0 < n; i0 += 16 * kThreads) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = i0 + i * kThreads < n ? (float)p[i0 + i * kThreads] : 0.f;
        s += squares(v);
    }
    return s;
}
template <typename T>
__device__ void scale_elements(const T *p, T *o, int n, float c) {
    for (int i0 = threadIdx.x; i0 < n; i0 += 16 * kThreads) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = i0 + i * kThreads < n ? (float)p[i0 + i * kThreads] : 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (i0 + i * kThreads < n) o[i0 + i * kThreads] = (T)(v[i] * c);
    }
}

// Calls f(entry, first element, elements) for this block's chunks: every gridDim.x-th, so that the blocks move through memory side by
// side, from the front or from the back (what the other pass read last is still in L2).
template <bool BACK, int N, typename F>
__device__ __forceinline__ void walk(const Table<N> &t, F f) {
    for (int k = blockIdx.x; k < t.chunks; k += gridDim.x) {
        const int c = BACK ? t.chunks - 1 - k : k;
        int i = 0;
        for (int b = t.n; i + 1 < b;) {  // the last tensor that starts at or before chunk c
            const int mid = (i + b) >> 1;
            if (t.e[mid].first <= c) i = mid;
            else b = mid;
        }
        const Entry &e = t.e[i];
        const int elems = chunk_elems(e.dtype);
        const int64_t at = (int64_t)(c - e.first) * elems;
        f(e, at, (int)min((int64_t)elems, e.count - at));
    }
}

template <int N>
__global__ void __launch_bounds__(kThreads)
grad_squares_kernel(const __grid_constant__ Table<N> t, double *__restrict__ slots, int add) {
    __shared__ double s[kThreads / 32];
    pdl_trigger();
    pdl_wait();
    double sum = 0.0;
    walk<false>(t, [&](const Entry &e, int64_t at, int n) {
        auto add = [&](auto *p) {
            if (reinterpret_cast<uintptr_t>(p) & 15u) sum += sum_elements(p + at, n);
            else {
                Chunk<std::remove_const_t<std::remove_pointer_t<decltype(p)>>> x;
                x.load(p + at, n);
                sum += x.sum();
            }
        };
        if (e.dtype == OMOE_F32) add(static_cast<const float *>(e.in));
        else add(static_cast<const __nv_bfloat16 *>(e.in));
    });
    sum = block_sum(sum, s);
    if (threadIdx.x == 0) slots[blockIdx.x] = add ? slots[blockIdx.x] + sum : sum;
}

__device__ __forceinline__ float norm_of(const double *slots, int n, double *s) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) sum += slots[i];
    return (float)sqrt(block_sum(sum, s));
}

__global__ void __launch_bounds__(kThreads)
grad_norm_kernel(const double *__restrict__ slots, int n, float *__restrict__ norm) {
    __shared__ double s[kThreads / 32];
    pdl_trigger();
    pdl_wait();
    const float v = norm_of(slots, n, s);
    if (threadIdx.x == 0) *norm = v;
}

// c = min(1, max_norm / (norm + 1e-6)); 1 where the norm is not finite.  Every block works it out, from the sums of the blocks
// that squared (slots) or from the norm handed over.
template <int N>
__global__ void __launch_bounds__(kThreads)
grad_scale_kernel(const __grid_constant__ Table<N> t, const double *__restrict__ slots, int n_slots, const float *norm_in,
                  float *norm_out, float max_norm, int in_place) {
    __shared__ double s[kThreads / 32];
    pdl_trigger();
    pdl_wait();
    const float norm = slots ? norm_of(slots, n_slots, s) : *norm_in;
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    float c = 1.f;
    if (norm < INFINITY) c = (float)fmin(1.0, (double)max_norm / ((double)norm + 1e-6));
    if (in_place && c == 1.f) return;
    walk<true>(t, [&](const Entry &e, int64_t at, int n) {
        auto scale = [&](const auto *p, auto *o) {
            if ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(o)) & 15u) scale_elements(p + at, o + at, n, c);
            else {
                Chunk<std::remove_pointer_t<decltype(o)>> x;
                x.load(p + at, n);
                x.store(o + at, n, c);
            }
        };
        if (e.dtype == OMOE_F32) scale(static_cast<const float *>(e.in), static_cast<float *>(e.out));
        else scale(static_cast<const __nv_bfloat16 *>(e.in), static_cast<__nv_bfloat16 *>(e.out));
    });
}

struct Span {
    uintptr_t lo, hi;
    int32_t i;
};

// The spans of a list by address, empty tensors left out; returns how many.
int spans_of(const omoe_tensor *t, int n, Span *s) {
    int m = 0;
    bool sorted = true;
    for (int i = 0; i < n; i++) {
        if (t[i].count == 0) continue;
        s[m].lo = reinterpret_cast<uintptr_t>(t[i].ptr);
        s[m].hi = s[m].lo + (uintptr_t)t[i].count * (t[i].dtype == OMOE_BF16 ? 2 : 4);
        s[m].i = i;
        sorted = sorted && (m == 0 || s[m - 1].lo <= s[m].lo);
        m++;
    }
    if (!sorted) std::sort(s, s + m, [](const Span &a, const Span &b) { return a.lo < b.lo; });
    return m;
}

int check_list(const omoe_tensor *grads, const omoe_tensor *out, int n, bool writes, const char *fn) {
    if (n < 0 || (n > 0 && !grads)) return ops_fail(OMOE_ERR_INVALID, fn, "bad list of tensors");
    for (int i = 0; i < n; i++) {
        const omoe_tensor &g = grads[i];
        if (g.dtype != OMOE_F32 && g.dtype != OMOE_BF16) return ops_fail(OMOE_ERR_INVALID, fn, "a dtype is neither OMOE_F32 nor OMOE_BF16");
        if (g.count < 0 || g.count > ((int64_t)1 << 42)) return ops_fail(OMOE_ERR_INVALID, fn, "a tensor's count is out of range");
        if (g.count > 0 && !g.ptr) return ops_fail(OMOE_ERR_INVALID, fn, "null tensor");
        const uintptr_t elem = g.dtype == OMOE_BF16 ? 2 : 4;
        if (misaligned(g.ptr, elem)) return ops_fail(OMOE_ERR_INVALID, fn, "a tensor is not aligned to its element type");
        if (!out) continue;
        if (out[i].count != g.count || out[i].dtype != g.dtype) return ops_fail(OMOE_ERR_INVALID, fn, "out[i] must have the count and dtype of grads[i]");
        if (g.count > 0 && !out[i].ptr) return ops_fail(OMOE_ERR_INVALID, fn, "null tensor");
        if (misaligned(out[i].ptr, elem)) return ops_fail(OMOE_ERR_INVALID, fn, "a tensor is not aligned to its element type");
    }
    if (!writes || n == 0) return OMOE_OK;
    Span *s = static_cast<Span *>(malloc(sizeof(Span) * 2 * (size_t)n));
    if (!s) return ops_fail(OMOE_ERR_NOMEM, fn, "out of host memory");
    const int m = spans_of(out ? out : grads, n, s);
    bool bad = false;
    for (int i = 1; i < m; i++) bad = bad || s[i].lo < s[i - 1].hi;
    if (out && !bad) {  // a gradient may be met by its own output alone, and only where it starts
        Span *g = s + n;
        const int mg = spans_of(grads, n, g);
        for (int i = 0, j = 0; i < mg && !bad; i++) {
            while (j < m && s[j].hi <= g[i].lo) j++;
            for (int q = j; q < m && s[q].lo < g[i].hi; q++) bad = bad || !(s[q].i == g[i].i && s[q].lo == g[i].lo);
        }
    }
    free(s);
    return bad ? ops_fail(OMOE_ERR_INVALID, fn, "tensors of the list overlap") : OMOE_OK;
}

// Blocks per SM of the two passes: more than four sum no faster, and eight scale up to 4 % faster than six.
constexpr int kSumBlocks = 4, kScaleBlocks = 8;
int grid_of(int chunks, int most) {
    if (most > kSlots) most = kSlots;
    return chunks < most ? chunks : most;
}

// Launches f(table, blocks, is it the first) for the tensors of the list, as many at a time as a table takes.
template <int N, typename F>
cudaError_t tables(const omoe_tensor *grads, const omoe_tensor *out, int n, int most, F f) {
    Table<N> t;
    bool first = true;
    for (int i = 0; i < n;) {
        t.n = 0;
        int64_t chunks = 0;
        for (; i < n && t.n < N; i++) {
            if (grads[i].count == 0) continue;
            const int elems = chunk_elems(grads[i].dtype);
            const int64_t c = (grads[i].count + elems - 1) / elems;
            if (chunks + c > INT32_MAX / 2) break;  // chunk numbers and a grid beyond them fit; never for the first: count <= 2^42
            t.e[t.n++] = {grads[i].ptr, out ? out[i].ptr : grads[i].ptr, grads[i].count, (int32_t)chunks, grads[i].dtype};
            chunks += c;
        }
        if (t.n == 0) break;
        t.chunks = (int32_t)chunks;
        cudaError_t e = f(t, grid_of(t.chunks, most), first);
        if (e != cudaSuccess) return e;
        first = false;
    }
    return cudaSuccess;
}

int used(const omoe_tensor *t, int n) {
    int m = 0;
    for (int i = 0; i < n; i++) m += t[i].count > 0;
    return m;
}

template <typename F>
cudaError_t by_count(const omoe_tensor *grads, const omoe_tensor *out, int n, int most, F f) {
    const int m = used(grads, n);
    if (m <= 16) return tables<16>(grads, out, n, most, f);
    if (m <= 64) return tables<64>(grads, out, n, most, f);
    if (m <= 256) return tables<256>(grads, out, n, most, f);
    if (m <= 500) return tables<500>(grads, out, n, most, f);
    return tables<1000>(grads, out, n, most, f);
}

// Blocks' sums of squares into the workspace; *slots is how many there are.
cudaError_t launch_squares(const omoe_tensor *grads, int n, double *ws, int sms, cudaStream_t s, int *slots) {
    *slots = 0;
    auto go = [&](const auto &t, int blocks, bool first) {
        using Tab = std::remove_cv_t<std::remove_reference_t<decltype(t)>>;
        constexpr int N = sizeof(Tab::e) / sizeof(Entry);
        if (first) *slots = blocks;
        // later tables add to the slots of the first one
        const int b = first ? blocks : (blocks < *slots ? blocks : *slots);
        return launch_ex(grad_squares_kernel<N>, dim3(b), dim3(kThreads), 0, s, ops_pdl(), t, ws, first ? 0 : 1);
    };
    return by_count(grads, nullptr, n, sms * kSumBlocks, go);
}

cudaError_t launch_scale(const omoe_tensor *grads, const omoe_tensor *out, int n, const double *ws, int slots, const float *norm_in,
                         float *norm_out, float max_norm, int sms, cudaStream_t s) {
    auto go = [&](const auto &t, int blocks, bool first) {
        using Tab = std::remove_cv_t<std::remove_reference_t<decltype(t)>>;
        constexpr int N = sizeof(Tab::e) / sizeof(Entry);
        return launch_ex(grad_scale_kernel<N>, dim3(blocks), dim3(kThreads), 0, s, ops_pdl(), t, ws, slots, norm_in,
                         first ? norm_out : nullptr, max_norm, out ? 0 : 1);
    };
    return by_count(grads, out, n, sms * kScaleBlocks, go);
}

// True where [p, p + bytes) meets a tensor of the lists.
bool meets(const void *p, size_t bytes, const omoe_tensor *grads, const omoe_tensor *out, int n) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p), hi = lo + bytes;
    for (int i = 0; i < n; i++) {
        const uintptr_t size = (uintptr_t)grads[i].count * (grads[i].dtype == OMOE_BF16 ? 2 : 4);
        const uintptr_t a = reinterpret_cast<uintptr_t>(grads[i].ptr), b = out ? reinterpret_cast<uintptr_t>(out[i].ptr) : a;
        if (size && ((a < hi && lo < a + size) || (b < hi && lo < b + size))) return true;
    }
    return false;
}
const char kMeets[] = "norm_dev or the workspace overlaps a tensor of the list";

const char *norm_args_wrong(const float *norm, const void *ws, int64_t bytes) {
    if (!norm || misaligned(norm, 4)) return "norm_dev is null or misaligned";
    const uintptr_t at = reinterpret_cast<uintptr_t>(norm), w = reinterpret_cast<uintptr_t>(ws);
    if (ws && at + 4 > w && at < w + OMOE_GRAD_WORKSPACE_BYTES) return "norm_dev lies in the workspace";
    if (!ws || misaligned(ws, 16) || bytes < OMOE_GRAD_WORKSPACE_BYTES) return "the workspace is missing, misaligned or too small";
    return nullptr;
}

}  // namespace
}  // namespace omoe

using namespace omoe;

extern "C" {

int omoe_grad_norm(const omoe_tensor *grads, int32_t n, float *norm_dev, void *workspace_dev, int64_t workspace_bytes,
                   void *cuda_stream) {
    const char *fn = "omoe_grad_norm";
    if (int rc = check_list(grads, nullptr, n, false, fn)) return rc;
    if (const char *bad = norm_args_wrong(norm_dev, workspace_dev, workspace_bytes)) return ops_fail(OMOE_ERR_INVALID, fn, bad);
    if (meets(norm_dev, 4, grads, nullptr, n) || meets(workspace_dev, OMOE_GRAD_WORKSPACE_BYTES, grads, nullptr, n))
        return ops_fail(OMOE_ERR_INVALID, fn, kMeets);
    const int sms = ops_sm_count();
    if (!sms) return ops_fail(OMOE_ERR_CUDA, fn, "no device");
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    double *ws = static_cast<double *>(workspace_dev);
    int slots = 0;
    cudaError_t e = launch_squares(grads, n, ws, sms, s, &slots);
    if (e == cudaSuccess) e = launch_ex(grad_norm_kernel, dim3(1), dim3(kThreads), 0, s, ops_pdl(), ws, slots, norm_dev);
    return ops_launched(e, fn);
}

int omoe_grad_scale(const omoe_tensor *grads, const omoe_tensor *out, int32_t n, const float *norm_dev, float max_norm,
                    void *cuda_stream) {
    const char *fn = "omoe_grad_scale";
    if (int rc = check_list(grads, out, n, true, fn)) return rc;
    if (!norm_dev || misaligned(norm_dev, 4)) return ops_fail(OMOE_ERR_INVALID, fn, "norm_dev is null or misaligned");
    if (!(max_norm >= 0.f)) return ops_fail(OMOE_ERR_INVALID, fn, "max_norm must not be negative");
    if (meets(norm_dev, 4, grads, out, n)) return ops_fail(OMOE_ERR_INVALID, fn, kMeets);
    const int sms = ops_sm_count();
    if (!sms) return ops_fail(OMOE_ERR_CUDA, fn, "no device");
    return ops_launched(launch_scale(grads, out, n, nullptr, 0, norm_dev, nullptr, max_norm, sms, static_cast<cudaStream_t>(cuda_stream)), fn);
}

int omoe_grad_clip(const omoe_tensor *grads, const omoe_tensor *out, int32_t n, float max_norm, float *norm_dev,
                   void *workspace_dev, int64_t workspace_bytes, void *cuda_stream) {
    const char *fn = "omoe_grad_clip";
    if (int rc = check_list(grads, out, n, true, fn)) return rc;
    if (const char *bad = norm_args_wrong(norm_dev, workspace_dev, workspace_bytes)) return ops_fail(OMOE_ERR_INVALID, fn, bad);
    if (!(max_norm >= 0.f)) return ops_fail(OMOE_ERR_INVALID, fn, "max_norm must not be negative");
    if (meets(norm_dev, 4, grads, out, n) || meets(workspace_dev, OMOE_GRAD_WORKSPACE_BYTES, grads, out, n))
        return ops_fail(OMOE_ERR_INVALID, fn, kMeets);
    const int sms = ops_sm_count();
    if (!sms) return ops_fail(OMOE_ERR_CUDA, fn, "no device");
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    double *ws = static_cast<double *>(workspace_dev);
    if (used(grads, n) == 0) return ops_launched(launch_ex(grad_norm_kernel, dim3(1), dim3(kThreads), 0, s, ops_pdl(), ws, 0, norm_dev), fn);
    int slots = 0;
    cudaError_t e = launch_squares(grads, n, ws, sms, s, &slots);
    if (e == cudaSuccess) e = launch_scale(grads, out, n, ws, slots, nullptr, norm_dev, max_norm, sms, s);
    return ops_launched(e, fn);
}

}  // extern "C"
