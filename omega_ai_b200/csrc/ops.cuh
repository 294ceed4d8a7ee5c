// What the operators without a handle share (token_sort.cu, layer_norm.cu, grad_norm.cu): error text, checks of row
// matrices, and fragments of rows as vectors or single elements.
#pragma once

#include "common.cuh"

namespace omoe {

// Sets omoe_ops_error() of this host thread to "fn: msg" and returns code.
int ops_fail(int code, const char *fn, const char *msg);
int ops_ok();
// Launch status to return code.
int ops_launched(cudaError_t e, const char *fn);
// SMs of the current device (asked once per device), 0 when there is none.
int ops_sm_count();
// Programmatic dependent launch is on (OMOE_PDL=0 switches it off).
bool ops_pdl();

// A row matrix of a call: `rows` rows of d elements, ld elements apart.
struct Rows {
    const void *p;
    int64_t ld;
    int32_t dtype;
    int64_t rows;
    int64_t d;
    size_t elem() const { return dtype == OMOE_BF16 ? 2 : 4; }
};
// nullptr, or what is wrong with it.
const char *rows_wrong(const Rows &r);
// n contiguous elements of 4 bytes; none where p is null
inline Rows words(const void *p, int64_t n) { return {p, n, OMOE_F32, p && n > 0 ? 1 : 0, n}; }
// True where an element of `a` is also one of `b`.  Two column windows of the same matrix do not overlap.
bool rows_overlap(const Rows &a, const Rows &b);
// Status of a call whose first n_out buffers are written, with the text set: none of them may meet another one.
int ops_apart(const Rows *all, int n, int n_out, const char *fn);
// True when every group of 8 elements of a row is aligned to its size (16 bytes of bf16, 32 of fp32).
inline bool rows_vector(const Rows &r) {
    return r.d % 8 == 0 && reinterpret_cast<uintptr_t>(r.p) % (8 * r.elem()) == 0 && (r.rows <= 1 || r.ld % 8 == 0);
}
inline bool misaligned(const void *p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

// Calls f with two null pointers of the element types of a and b.
template <typename F>
inline cudaError_t by_types(int32_t a, int32_t b, F f) {
    using bf16 = __nv_bfloat16;
    if (a == OMOE_F32) return b == OMOE_F32 ? f((float *)nullptr, (float *)nullptr) : f((float *)nullptr, (bf16 *)nullptr);
    return b == OMOE_F32 ? f((bf16 *)nullptr, (float *)nullptr) : f((bf16 *)nullptr, (bf16 *)nullptr);
}

// V consecutive elements of a row as they lie in memory: 8 (16 bytes of bf16, 32 of fp32) or 1.  load() is for what is read once,
// load_cached() for what is read again and not written by the kernel.
template <typename T, int V>
struct Frag;
template <>
struct Frag<__nv_bfloat16, 8> {
    uint4 r;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { r = __ldcs(reinterpret_cast<const uint4 *>(p)); }
    __device__ __forceinline__ void load_cached(const __nv_bfloat16 *p) { r = __ldg(reinterpret_cast<const uint4 *>(p)); }
    __device__ __forceinline__ void store(__nv_bfloat16 *p) const { *reinterpret_cast<uint4 *>(p) = r; }
    __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&v)[8]) const { unpack8(r, v); }
    __device__ __forceinline__ void set(const float (&v)[8]) { r = pack8(v); }
};
template <>
struct Frag<float, 8> {
    // one 32-byte access: two of 16 bytes would each touch half of every 32-byte sector of the warp's lines
    float r[8];
    __device__ __forceinline__ void load(const float *p) {
        asm volatile("ld.global.cs.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]) : "l"(p) : "memory");
    }
    __device__ __forceinline__ void load_cached(const float *p) {
        asm volatile("ld.global.nc.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]) : "l"(p));
    }
    __device__ __forceinline__ void store(float *p) const {
        asm volatile("st.global.v8.f32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]),
                     "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]), "l"(p) : "memory");
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] = 0.f;
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = r[i];
    }
    __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] = v[i];
    }
};
template <>
struct Frag<float, 1> {
    float r;
    __device__ __forceinline__ void load(const float *p) { r = __ldcs(p); }
    __device__ __forceinline__ void load_cached(const float *p) { r = __ldg(p); }
    __device__ __forceinline__ void store(float *p) const { *p = r; }
    __device__ __forceinline__ void zero() { r = 0.f; }
    __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = r; }
    __device__ __forceinline__ void set(const float (&v)[1]) { r = v[0]; }
};
template <>
struct Frag<__nv_bfloat16, 1> {
    __nv_bfloat16 r;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { r = __ldcs(p); }
    __device__ __forceinline__ void load_cached(const __nv_bfloat16 *p) { r = __ldg(p); }
    __device__ __forceinline__ void store(__nv_bfloat16 *p) const { *p = r; }
    __device__ __forceinline__ void zero() { r = __float2bfloat16_rn(0.f); }
    __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = __bfloat162float(r); }
    __device__ __forceinline__ void set(const float (&v)[1]) { r = __float2bfloat16_rn(v[0]); }
};

// Element type change of a fragment; between equal types a copy.
template <typename A, typename B, int V>
__device__ __forceinline__ void convert(const Frag<A, V> &a, Frag<B, V> &b) {
    float v[V];
    a.get(v);
    b.set(v);
}
template <typename A, int V>
__device__ __forceinline__ void convert(const Frag<A, V> &a, Frag<A, V> &b) { b = a; }

}  // namespace omoe
