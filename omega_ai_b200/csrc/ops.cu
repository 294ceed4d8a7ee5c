// Error text and argument checks of the operators without a handle.
#include "ops.cuh"

#include <stdlib.h>

namespace omoe {

namespace {
thread_local char g_ops_err[256] = "";
}

int ops_fail(int code, const char *fn, const char *msg) {
    snprintf(g_ops_err, sizeof(g_ops_err), "%s: %s", fn, msg);
    return code;
}

int ops_ok() {
    g_ops_err[0] = 0;
    return OMOE_OK;
}

int ops_launched(cudaError_t e, const char *fn) {
    return e == cudaSuccess ? ops_ok() : ops_fail(OMOE_ERR_CUDA, fn, cudaGetErrorString(e));
}

int ops_sm_count() {
    static int count[kMaxDevices] = {};  // the same value whoever writes it
    int dev = -1, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev >= 0 && dev < kMaxDevices && count[dev] > 0) return count[dev];
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    if (dev >= 0 && dev < kMaxDevices) count[dev] = n;
    return n;
}

bool ops_pdl() {
    static const bool on = !(getenv("OMOE_PDL") && atoi(getenv("OMOE_PDL")) == 0);
    return on;
}

const char *rows_wrong(const Rows &r) {
    if (r.dtype != OMOE_F32 && r.dtype != OMOE_BF16) return "a dtype is neither OMOE_F32 nor OMOE_BF16";
    if (r.d <= 0) return "d must be positive";
    if (r.ld < r.d || r.ld >= ((int64_t)1 << 30)) return "a leading dimension is smaller than d or out of range";
    if (r.rows > 0 && !r.p) return "null buffer";
    if (misaligned(r.p, r.elem())) return "a buffer is not aligned to its element type";
    return nullptr;
}

bool rows_overlap(const Rows &a, const Rows &b) {
    if (a.rows <= 0 || b.rows <= 0 || !a.p || !b.p) return false;
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a.p), b0 = reinterpret_cast<uintptr_t>(b.p);
    const uintptr_t wa = a.d * a.elem(), wb = b.d * b.elem(), pa = a.ld * a.elem(), pb = b.ld * b.elem();
    if (a0 + (a.rows - 1) * pa + wa <= b0 || b0 + (b.rows - 1) * pb + wb <= a0) return false;
    if (pa == pb || a.rows == 1 || b.rows == 1) {
        // windows of one matrix: disjoint where neither reaches the other within the common pitch
        const uintptr_t pitch = a.rows == 1 ? pb : pa;
        if (a.rows == 1 && b.rows == 1) return true;
        if (wa <= pitch && wb <= pitch) {
            const uintptr_t shift = a0 >= b0 ? (a0 - b0) % pitch : (pitch - (b0 - a0) % pitch) % pitch;
            if (shift >= wb && shift + wa <= pitch) return false;
        }
    }
    return true;
}

int ops_apart(const Rows *all, int n, int n_out, const char *fn) {
    for (int i = 0; i < n_out; i++)
        for (int j = i + 1; j < n; j++)
            if (rows_overlap(all[i], all[j])) return ops_fail(OMOE_ERR_INVALID, fn, "an output overlaps another buffer");
    return OMOE_OK;
}

}  // namespace omoe

extern "C" const char *omoe_ops_error(void) { return omoe::g_ops_err; }
