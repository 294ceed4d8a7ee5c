// Token rows sorted by expert and back, with weights applied, and the gradients of both.
//
// The plan is a stable counting sort of the T*top_k picks by expert.  The rows are moved by the inverse of it (the row
// of every pick), so that a token's row is read once for all its picks and a sum over a token's picks runs in pick
// order: nothing here needs an atomic, and the same inputs give the same bits.
#include "ops.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace omoe {

namespace {

constexpr int64_t kRowsMax = 0x7fff0000;  // row numbers, and a block's worth beyond them, fit 32 bits
constexpr int kPlanWarps = 32;
constexpr int kPlanBatch = 8;    // picks a lane loads together
constexpr int kPlanCtasMax = 16;  // the largest cluster; 8 where the device cannot hold one of 16
constexpr size_t kPlanSmem = 220 * 1024;
static_assert(sizeof(int32_t) * (OMOE_SORT_MAX_EXPERTS * (4 + kPlanCtasMax + kPlanWarps) + 1) <= kPlanSmem, "the tables of the most experts fit");

// One cluster does the whole plan.  Every warp owns a contiguous run of picks and counts its picks of every expert in
// shared memory, numbering them as it goes: lanes with the same expert are found by ballots over the bits of its number (a warp-wide
// match takes longer the more experts meet in a warp).  After sums over the warps, which every CTA stores into the shared memory of
// all, and over the CTAs every warp knows where its first pick of each expert goes.  A run of up to 256 picks stays in
// registers, a longer one keeps its numbers in pos meanwhile.
// perm is a scatter: written pick by pick every store touches up to 32 lines, and few SMs have to make them all (by eight, 49152 picks on 64
// experts took 13.5 us, through lists 10.8; sixteen CTAs that send their totals take 7.8).  So the CTA's picks are put in order in shared memory first, `list` of them at most, and leave
// as one run per expert.  Bound by latency: the walk, the barriers, the copies.
__global__ void __launch_bounds__(kPlanWarps * 32)
sort_plan_kernel(const int32_t *__restrict__ idx, int n, int E, int align, int rows_cap, int warp_run, int list,
                 int32_t *__restrict__ pos, int32_t *__restrict__ perm, int32_t *__restrict__ counts,
                 int32_t *__restrict__ offsets) {
    extern __shared__ int32_t sm[];
    cg::cluster_group cluster = cg::this_cluster();
    const int nw = blockDim.x >> 5, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int ctas = cluster.num_blocks(), cta = cluster.block_rank();
    int32_t *s_totals = sm;             // [CTAs][E] the CTAs' picks of every expert, each stored by the CTA itself
    int32_t *s_total = s_totals + cta * E;
    int32_t *s_count = s_totals + ctas * E;  // [E] all picks
    int32_t *s_first = s_count + E;     // [E+1] first row of every expert
    int32_t *s_start = s_first + E + 1; // [E] first row of this CTA's picks of the expert
    int32_t *s_local = s_start + E;     // [E] where they start in the CTA's list
    int32_t *s_hist = s_local + E;      // [warps][E]
    int32_t *s_list = s_hist + nw * E;  // [list] pick numbers by expert
    uint16_t *s_expert = reinterpret_cast<uint16_t *>(s_list + list);  // [list]
    int32_t *hist = s_hist + warp * E;

    // the others' shared memory may be stored to once all CTAs have started; waited for below
    if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    pdl_trigger();
    for (int e = lane; e < E; e += 32) hist[e] = 0;
    const int64_t lo64 = (int64_t)(cta * nw + warp) * warp_run;
    const int lo = (int)min((int64_t)n, lo64), hi = (int)min((int64_t)n, lo64 + warp_run);
    pdl_wait();
    __syncwarp();
    const int bits = 32 - __clz(E);  // of the keys 0..E, E standing for no expert
    int32_t key[kPlanBatch], rank[kPlanBatch];
    for (int i0 = lo; i0 < hi; i0 += kPlanBatch * 32) {
#pragma unroll
        for (int u = 0; u < kPlanBatch; u++) {
            const int i = i0 + u * 32 + lane;
            const int e = i < hi ? idx[i] : -1;
            key[u] = e >= 0 && e < E ? e : E;
        }
#pragma unroll
        for (int u = 0; u < kPlanBatch; u++) {
            const int i = i0 + u * 32 + lane;
            if (i0 + u * 32 >= hi) break;
            uint32_t same = 0xffffffffu;  // lanes with this lane's key
            for (int b = 0; b < bits; b++) {
                const int bit = (int)((uint32_t)key[u] << (31 - b)) >> 31;  // 0 or all ones
                same &= ~(__ballot_sync(0xffffffffu, bit) ^ (uint32_t)bit);
            }
            const uint32_t before = same & ((1u << lane) - 1);
            rank[u] = 0;
            if (key[u] < E) rank[u] = hist[key[u]] + __popc(before);
            __syncwarp();
            if (key[u] < E && !before) hist[key[u]] += __popc(same);
            __syncwarp();
            if (warp_run > kPlanBatch * 32 && i < hi) pos[i] = rank[u];  // kept there until the expert's first row is known
        }
    }
    __syncthreads();
    if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
        int run = 0;
#pragma unroll 8
        for (int w = 0; w < nw; w++) {
            const int c = s_hist[w * E + e];
            s_hist[w * E + e] = run;
            run += c;
        }
        for (int c = 0; c < ctas; c++) cluster.map_shared_rank(s_total, c)[e] = run;
    }
    if (ctas > 1) cluster.sync();  // the last access to another CTA's memory
    else __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
        int before = 0, all = 0;
#pragma unroll 4
        for (int c = 0; c < ctas; c++) {
            const int v = s_totals[c * E + e];
            if (c < cta) before += v;
            all += v;
        }
        s_count[e] = all;
        s_start[e] = before;  // the expert's first row is added below
    }
    __syncthreads();
    if (warp == 0) {
        int row = 0, local = 0;
        for (int e0 = 0; e0 < E; e0 += 32) {
            const int e = e0 + lane;
            const int c = e < E ? s_total[e] : 0, p = e < E ? (s_count[e] + align - 1) / align * align : 0;
            int rows = p, mine = c;  // inclusive sums over the lanes
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int r = __shfl_up_sync(0xffffffffu, rows, o), m = __shfl_up_sync(0xffffffffu, mine, o);
                if (lane >= o) { rows += r; mine += m; }
            }
            if (e < E) {
                s_first[e] = row + rows - p;
                s_start[e] += row + rows - p;
                s_local[e] = local + mine - c;
            }
            row += __shfl_sync(0xffffffffu, rows, 31);
            local += __shfl_sync(0xffffffffu, mine, 31);
        }
        if (lane == 0) s_first[E] = row;
    }
    __syncthreads();
    for (int i0 = lo; i0 < hi; i0 += kPlanBatch * 32) {
        if (warp_run > kPlanBatch * 32) {
#pragma unroll
            for (int u = 0; u < kPlanBatch; u++) {
                const int i = i0 + u * 32 + lane;
                const int e = i < hi ? idx[i] : -1;
                key[u] = e >= 0 && e < E ? e : E;
                rank[u] = i < hi ? pos[i] : 0;
            }
        }
#pragma unroll
        for (int u = 0; u < kPlanBatch; u++) {
            const int i = i0 + u * 32 + lane, e = key[u];
            if (i >= hi) continue;
            int row = -1;
            if (e < E) {
                const int q = hist[e] + rank[u];  // among the CTA's picks of the expert
                row = s_start[e] + q;
                if (list) {
                    s_list[s_local[e] + q] = i;
                    s_expert[s_local[e] + q] = (uint16_t)e;
                } else if (row < rows_cap) perm[row] = i;
            }
            pos[i] = row;
        }
    }
    // what is the same for all CTAs is shared out: counts and offsets, and perm where there is no pick
    for (int e = cta * blockDim.x + threadIdx.x; e < E; e += ctas * blockDim.x) {
        counts[e] = s_count[e];
        offsets[e] = s_first[e];
    }
    if (cta == 0 && threadIdx.x == 0) offsets[E] = s_first[E];
    for (int e = align > 1 ? cta * nw + warp : E; e < E; e += ctas * nw)
        for (int r = s_first[e] + s_count[e] + lane; r < s_first[e + 1] && r < rows_cap; r += 32) perm[r] = -1;
    for (int64_t r = (int64_t)s_first[E] + cta * blockDim.x + threadIdx.x; r < rows_cap; r += ctas * blockDim.x) perm[r] = -1;
    if (list) {
        __syncthreads();
        const int mine = s_local[E - 1] + s_total[E - 1];
        for (int q = threadIdx.x; q < mine; q += blockDim.x) {
            const int e = s_expert[q], row = s_start[e] + q - s_local[e];
            if (row < rows_cap) perm[row] = s_list[q];
        }
    }
}

// A warp takes one chunk of a token's columns: U vectors per lane.  Rows of up to 256 columns get one (a warp that has nothing to do for
// most of its vectors still issues for them: 20 us against 10 for the way back of 16384 x 128 and 8 picks).  Else two; sums over picks
// four where those chunks fill the GPU's warps by themselves (16384 x 4096, 2 picks: 65 us against 71; 4096 x 1024: 5.5 against 5.4).
template <int V, int U>
constexpr int kChunk = 32 * V * U;
// Calls f(V, U) (integral constants) for T rows of width d.
template <typename F>
int by_chunk(bool vec, int64_t T, int d, bool sums, F f) {
    using std::integral_constant;
    if (!vec) return f(integral_constant<int, 1>(), integral_constant<int, 8>());
    if (d <= 256) return f(integral_constant<int, 8>(), integral_constant<int, 1>());
    if (sums && T * ceil_div(d, kChunk<8, 4>) > (int64_t)64 * ops_sm_count())
        return f(integral_constant<int, 8>(), integral_constant<int, 4>());
    return f(integral_constant<int, 8>(), integral_constant<int, 2>());
}

// The rows of a token's picks, a pick per lane; picks without a row, or with one that no plan makes, are negative.
__device__ __forceinline__ int pick_row(const int32_t *pos, int64_t t, int k, int lane, int rows_cap) {
    int r = -1;
    if (lane < k) r = pos[t * k + lane];
    return r < rows_cap ? r : -1;
}

// Padding rows of an expert are zeroed by kPadRows at a time, each slice by a warp or block of its own: one warp for all of an
// expert's up to 127 rows took longer than the whole copy.
constexpr int kPadRows = 8, kPadSlicesMax = 128;
int pad_slices(int align) {
    const int n = (align - 1 + kPadRows - 1) / kPadRows;
    return n < kPadSlicesMax ? n : kPadSlicesMax;
}

// Zeros for the padding rows of slice `item` (experts times slices), columns c0, c0 + step, ... below c1.
template <typename T, int V>
__device__ __forceinline__ void zero_padding(T *rows, int64_t ld, const int32_t *counts, const int32_t *offsets, int item, int slices,
                                             int c0, int c1, int step, int rows_cap) {
    const int e = item / slices, first = offsets[e] + counts[e], last = min(offsets[e + 1], rows_cap);
    if (first < 0) return;
    Frag<T, V> z;
    z.zero();
    for (int r0 = first + item % slices * kPadRows; r0 < last; r0 += slices * kPadRows)
        for (int c = c0; c < c1; c += step)
#pragma unroll
            for (int r = 0; r < kPadRows; r++)
                if (r0 + r < last) z.store(rows + (int64_t)(r0 + r) * ld + c);
}

// xs[pos] = x: a warp reads a chunk of a token's row once and stores it for every pick.  HBM bound.
template <typename XT, typename OT, int V, int U>
__global__ void __launch_bounds__(256)
sort_rows_kernel(const XT *__restrict__ x, int64_t ldx, OT *__restrict__ xs, int64_t ldxs, const int32_t *__restrict__ pos,
                 const int32_t *__restrict__ counts, const int32_t *__restrict__ offsets, int T, int k, int pads, int slices, int d,
                 int n_chunks, int rows_cap) {
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t t = item / n_chunks;
    const int c0 = (int)(item % n_chunks) * kChunk<V, U> + lane * V;
    pdl_trigger();
    pdl_wait();
    if (t >= T) {
        if (t - T < pads)
            zero_padding<OT, V>(xs, ldxs, counts, offsets, (int)(t - T), slices, c0, min(d, c0 - lane * V + kChunk<V, U>), 32 * V, rows_cap);
        return;
    }
    const int r = pick_row(pos, t, k, lane, rows_cap);
    Frag<XT, V> in[U];
    Frag<OT, V> out[U];
    // before the picks are there: a token that turns out to have none was read for nothing, the others have waited once, not twice
#pragma unroll
    for (int u = 0; u < U; u++)
        if (c0 + u * 32 * V < d) in[u].load(x + t * ldx + c0 + u * 32 * V);
    uint32_t picks = __ballot_sync(0xffffffffu, r >= 0);
    if (!picks) return;
#pragma unroll
    for (int u = 0; u < U; u++) convert(in[u], out[u]);
    for (; picks; picks &= picks - 1) {
        OT *to = xs + (int64_t)__shfl_sync(0xffffffffu, r, __ffs(picks) - 1) * ldxs;
#pragma unroll
        for (int u = 0; u < U; u++)
            if (c0 + u * 32 * V < d) out[u].store(to + c0 + u * 32 * V);
    }
}

// y[t] = sum over the picks of w * ys[pos] (W) or of ys[pos]: a warp per chunk of a token's columns, two picks' loads in
// flight.  fp32 sums in pick order.  HBM bound.
template <typename XT, typename OT, int V, int U, bool W>
__global__ void __launch_bounds__(256)
unsort_rows_kernel(const XT *__restrict__ ys, int64_t ldys, OT *__restrict__ y, int64_t ldy, const int32_t *__restrict__ pos,
                   const float *__restrict__ w, int T, int k, int d, int n_chunks, int rows_cap) {
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t t = item / n_chunks;
    const int c0 = (int)(item % n_chunks) * kChunk<V, U> + lane * V;
    pdl_trigger();
    pdl_wait();
    if (t >= T) return;
    const int r = pick_row(pos, t, k, lane, rows_cap);
    float wl = 1.f;
    if (W && lane < k) wl = w[t * k + lane];
    uint32_t picks = __ballot_sync(0xffffffffu, r >= 0);
    float acc[U][V];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int i = 0; i < V; i++) acc[u][i] = 0.f;
    while (picks) {
        const int j0 = __ffs(picks) - 1;
        picks &= picks - 1;
        const int j1 = picks ? __ffs(picks) - 1 : -1;
        picks &= picks - 1;  // stays 0 where it is
        Frag<XT, V> a[U], b[U];
        const XT *p0 = ys + (int64_t)__shfl_sync(0xffffffffu, r, j0) * ldys;
        const XT *p1 = ys + (int64_t)__shfl_sync(0xffffffffu, r, j1 < 0 ? j0 : j1) * ldys;
        const float w0 = __shfl_sync(0xffffffffu, wl, j0), w1 = __shfl_sync(0xffffffffu, wl, j1 < 0 ? j0 : j1);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (c0 + u * 32 * V < d) {
                a[u].load(p0 + c0 + u * 32 * V);
                if (j1 >= 0) b[u].load(p1 + c0 + u * 32 * V);
            }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (c0 + u * 32 * V < d) {
                float v[V];
                a[u].get(v);
#pragma unroll
                for (int i = 0; i < V; i++) acc[u][i] = W ? fmaf(w0, v[i], acc[u][i]) : acc[u][i] + v[i];
                if (j1 >= 0) {
                    b[u].get(v);
#pragma unroll
                    for (int i = 0; i < V; i++) acc[u][i] = W ? fmaf(w1, v[i], acc[u][i]) : acc[u][i] + v[i];
                }
            }
    }
#pragma unroll
    for (int u = 0; u < U; u++)
        if (c0 + u * 32 * V < d) {
            Frag<OT, V> o;
            o.set(acc[u]);
            o.store(y + t * ldy + c0 + u * 32 * V);
        }
}

// dys[pos] = w * dy and dw = <dy, ys[pos]>: `threads` threads per token read dy once; a thread's columns are
// added up for every pick in registers, then over the token's threads in a fixed order.  K bounds k.  HBM bound.
template <typename DT, typename YT, int V, int K>
__global__ void __launch_bounds__(512)
unsort_bwd_kernel(const DT *__restrict__ dy, int64_t lddy, const YT *__restrict__ ys, int64_t ldys, YT *__restrict__ dys,
                  int64_t lddys, const int32_t *__restrict__ pos, const int32_t *__restrict__ counts,
                  const int32_t *__restrict__ offsets, const float *__restrict__ w, float *__restrict__ dw, int T, int k, int pads,
                  int slices, int d, int rows_cap, int threads) {
    constexpr int U = V > 1 ? 1 : K <= 4 ? 4 : 2;  // single elements: several columns' loads together
    constexpr int J = K <= 6 || (sizeof(YT) * V <= 16 && K <= 8) ? K : 4;  // picks whose vectors are held at a time
    __shared__ float s_dot[16][K];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, of_token = threadIdx.x % threads;
    const int64_t t = (int64_t)blockIdx.x * (blockDim.x / threads) + threadIdx.x / threads;
    pdl_trigger();
    pdl_wait();
    if (t >= T && t - T < pads) zero_padding<YT, V>(dys, lddys, counts, offsets, (int)(t - T), slices, of_token * V, d, threads * V, rows_cap);
    float dot[K];
#pragma unroll
    for (int j = 0; j < K; j++) dot[j] = 0.f;
    if (t < T) {
        int row[K];
        float wt[K];
#pragma unroll
        for (int j = 0; j < K; j++) {
            row[j] = j < k ? pos[t * k + j] : -1;
            if (row[j] >= rows_cap) row[j] = -1;
            wt[j] = w && j < k ? w[t * k + j] : 1.f;
        }
        for (int c0 = of_token * V; c0 < d; c0 += threads * V * U) {
            Frag<DT, V> g[U];
            Frag<YT, V> y[U][J], o;
            float gv[V], v[V];
#pragma unroll
            for (int u = 0; u < U; u++)
                if (c0 + u * threads * V < d) g[u].load(dy + t * lddy + c0 + u * threads * V);
#pragma unroll
            for (int j0 = 0; j0 < K; j0 += J) {
                if (dw)
#pragma unroll
                    for (int u = 0; u < U; u++)
#pragma unroll
                        for (int j = 0; j < J; j++)
                            if (row[j0 + j] >= 0 && c0 + u * threads * V < d)
                                y[u][j].load(ys + (int64_t)row[j0 + j] * ldys + c0 + u * threads * V);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int c = c0 + u * threads * V;
                    if (U > 1 && c >= d) break;
                    g[u].get(gv);
#pragma unroll
                    for (int j = 0; j < J; j++)
                        if (row[j0 + j] >= 0) {
#pragma unroll
                            for (int i = 0; i < V; i++) v[i] = wt[j0 + j] * gv[i];
                            o.set(v);
                            o.store(dys + (int64_t)row[j0 + j] * lddys + c);
                            if (dw) {
                                y[u][j].get(v);
#pragma unroll
                                for (int i = 0; i < V; i++) dot[j0 + j] = fmaf(gv[i], v[i], dot[j0 + j]);
                            }
                        }
                }
            }
        }
    }
    if (!dw) return;
#pragma unroll
    for (int j = 0; j < K; j++) {
#pragma unroll
        for (int m = 16; m >= 1; m >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], m);
        if (lane == 0) s_dot[warp][j] = dot[j];
    }
    if (threads > 32) __syncthreads();
    else __syncwarp();
    if (t < T && of_token < k) {
        float sum = 0.f;
        for (int i = 0; i < threads / 32; i++) sum += s_dot[warp + i][of_token];
        dw[t * k + of_token] = sum;
    }
}

const char *plan_wrong(const omoe_sort *p) {
    if (!p) return "null plan";
    if (p->n_tokens < 0 || p->top_k < 1 || p->n_experts < 1 || p->row_align < 1) return "bad sizes in the plan";
    if (!p->counts || !p->offsets || (p->n_tokens > 0 && !p->pos) || (p->rows_cap > 0 && !p->perm)) return "null buffer in the plan";
    if (misaligned(p->pos, 4) || misaligned(p->perm, 4) || misaligned(p->counts, 4) || misaligned(p->offsets, 4))
        return "the plan's buffers must be 4-byte aligned";
    return nullptr;
}

// The plan of a call on rows: status, with the text set.
int check_plan(const omoe_sort *p, const char *fn) {
    if (const char *bad = plan_wrong(p)) return ops_fail(OMOE_ERR_INVALID, fn, bad);
    const int64_t need = omoe_sort_rows_cap(p->n_tokens, p->top_k, p->n_experts, p->row_align);
    if (need < 0) return ops_fail((int)need, fn, "the plan's sizes are beyond the limits");
    if (p->rows_cap < need) return ops_fail(OMOE_ERR_TOO_LARGE, fn, "rows_cap is smaller than omoe_sort_rows_cap()");
    if (p->rows_cap > kRowsMax) return ops_fail(OMOE_ERR_TOO_LARGE, fn, "rows_cap is beyond the limit");
    return OMOE_OK;
}

int check_rows(const Rows *m, int n, const char *fn) {
    for (int i = 0; i < n; i++)
        if (const char *bad = rows_wrong(m[i])) return ops_fail(OMOE_ERR_INVALID, fn, bad);
    return OMOE_OK;
}
// The plan's buffers as a call on rows reads them.
Rows pos_of(const omoe_sort *p) { return words(p->pos, (int64_t)p->n_tokens * p->top_k); }
Rows counts_of(const omoe_sort *p) { return words(p->counts, p->n_experts); }
Rows offsets_of(const omoe_sort *p) { return words(p->offsets, (int64_t)p->n_experts + 1); }

// The CTAs of the largest cluster that the current device can hold with all of kPlanSmem, asked once per device.
cudaError_t plan_ctas(int *most) {
    static int known[kMaxDevices] = {};  // the same value whoever writes it
    int dev = -1;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices && known[dev]) {
        *most = known[dev];
        return cudaSuccess;
    }
    e = cudaFuncSetAttribute(sort_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPlanSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(sort_plan_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kPlanCtasMax);
    cfg.blockDim = dim3(kPlanWarps * 32);
    cfg.dynamicSmemBytes = kPlanSmem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = kPlanCtasMax;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int clusters = 0;
    e = cudaOccupancyMaxActiveClusters(&clusters, sort_plan_kernel, &cfg);
    if (e != cudaSuccess) return e;
    *most = clusters > 0 ? kPlanCtasMax : 8;
    if (dev < kMaxDevices) known[dev] = *most;
    return cudaSuccess;
}

// Blocks of eight warps for `tokens` rows cut into chunks.
int64_t row_blocks(int64_t tokens, int d, int chunk) { return (tokens * ceil_div(d, chunk) + 7) / 8; }
const char kTooMany[] = "the rows need too many blocks";

}  // namespace
}  // namespace omoe

using namespace omoe;

extern "C" {

int64_t omoe_sort_rows_cap(int32_t n_tokens, int32_t top_k, int32_t n_experts, int32_t row_align) {
    if (n_tokens < 0 || top_k < 1 || n_experts < 1 || row_align < 1) return OMOE_ERR_INVALID;
    if (n_experts > OMOE_SORT_MAX_EXPERTS || top_k > kMaxTopK) return OMOE_ERR_TOO_LARGE;
    const int64_t n = (int64_t)n_tokens * top_k, padded = n < n_experts ? n : n_experts;
    const int64_t rows = (n + padded * (row_align - 1) + row_align - 1) / row_align * row_align;
    return rows > kRowsMax ? OMOE_ERR_TOO_LARGE : rows;
}

int omoe_sort_plan(const omoe_sort *plan, const int32_t *topk_idx_dev, void *cuda_stream) {
    const char *fn = "omoe_sort_plan";
    if (int rc = check_plan(plan, fn)) return rc;
    if (plan->n_tokens > 0 && !topk_idx_dev) return ops_fail(OMOE_ERR_INVALID, fn, "null buffer");
    if (misaligned(topk_idx_dev, 4)) return ops_fail(OMOE_ERR_INVALID, fn, "topk_idx_dev must be 4-byte aligned");
    const Rows all[] = {pos_of(plan), words(plan->perm, plan->rows_cap), counts_of(plan), offsets_of(plan),
                        words(topk_idx_dev, (int64_t)plan->n_tokens * plan->top_k)};
    if (int rc = ops_apart(all, 5, 4, fn)) return rc;
    const int n = plan->n_tokens * plan->top_k, E = plan->n_experts;  // below 2^31: check_plan
    int most = 0;  // CTAs of a cluster
    if (cudaError_t e = plan_ctas(&most)) return ops_launched(e, fn);
    // a warp takes 64 picks before a second CTA joins; the CTAs of the largest cluster share the rest
    const int64_t want = ((int64_t)n + 63) / 64;
    int ctas = 1;
    while (ctas < most && want > ctas * kPlanWarps) ctas *= 2;
    const int warps = want < 8 ? 8 : want > kPlanWarps ? kPlanWarps : (int)want;  // eight for the experts' sums alone
    const int64_t run = round_up(((int64_t)n + ctas * warps - 1) / (ctas * warps), 32);
    const size_t tables = sizeof(int32_t) * ((size_t)E * (4 + ctas + warps) + 1);
    int64_t list = warps * run;  // picks of a CTA; beyond what fits they are scattered one by one
    if (tables + list * 6 > kPlanSmem) list = 0;
    const size_t smem = tables + list * 6;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(warps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(cuda_stream);
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ctas;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = ops_pdl() ? 2 : 1;
    return ops_launched(cudaLaunchKernelEx(&cfg, sort_plan_kernel, topk_idx_dev, n, E, (int)plan->row_align,
                                           (int)plan->rows_cap, (int)run, (int)list, plan->pos, plan->perm, plan->counts,
                                           plan->offsets), fn);
}

int omoe_sort_rows(const omoe_sort *plan, const void *x_dev, int64_t ldx, int32_t x_dtype, void *xs_dev, int64_t ldxs,
                   int32_t xs_dtype, int32_t d, void *cuda_stream) {
    const char *fn = "omoe_sort_rows";
    if (int rc = check_plan(plan, fn)) return rc;
    const int T = plan->n_tokens, E = plan->n_experts;
    const Rows x = {x_dev, ldx, x_dtype, T, d}, xs = {xs_dev, ldxs, xs_dtype, plan->rows_cap, d};
    const Rows all[] = {xs, x, pos_of(plan), counts_of(plan), offsets_of(plan)};
    if (int rc = check_rows(all, 2, fn)) return rc;
    if (int rc = ops_apart(all, 5, 1, fn)) return rc;
    if (T == 0) return ops_ok();
    const bool vec = rows_vector(x) && rows_vector(xs);
    const int slices = pad_slices(plan->row_align), pads = E * slices;
    const int64_t tokens = (int64_t)T + pads;  // a slice of an expert's padding is one more "token"
    return by_chunk(vec, T, d, false, [&](auto v, auto u) {
        constexpr int V = decltype(v)::value, U = decltype(u)::value, C = kChunk<V, U>;
        const int64_t blocks = row_blocks(tokens, d, C);
        if (blocks > INT32_MAX) return ops_fail(OMOE_ERR_TOO_LARGE, fn, kTooMany);
        return ops_launched(by_types(x_dtype, xs_dtype, [&](auto *xt, auto *ot) {
            using XT = std::remove_pointer_t<decltype(xt)>;
            using OT = std::remove_pointer_t<decltype(ot)>;
            return launch_ex(sort_rows_kernel<XT, OT, V, U>, dim3((unsigned)blocks), dim3(256), 0, static_cast<cudaStream_t>(cuda_stream),
                             ops_pdl(), static_cast<const XT *>(x_dev), ldx, static_cast<OT *>(xs_dev), ldxs, plan->pos, plan->counts,
                             plan->offsets, T, plan->top_k, pads, slices, d, ceil_div(d, C), (int)plan->rows_cap);
        }), fn);
    });
}

static int unsort(const omoe_sort *plan, const void *ys_dev, int64_t ldys, int32_t ys_dtype, const float *w_dev, void *y_dev,
                  int64_t ldy, int32_t y_dtype, int32_t d, void *cuda_stream, const char *fn) {
    if (int rc = check_plan(plan, fn)) return rc;
    const int T = plan->n_tokens;
    const Rows y = {y_dev, ldy, y_dtype, T, d}, ys = {ys_dev, ldys, ys_dtype, T ? plan->rows_cap : 0, d};
    const Rows all[] = {y, ys, words(w_dev, (int64_t)T * plan->top_k), pos_of(plan)};
    if (int rc = check_rows(all, 2, fn)) return rc;
    if (misaligned(w_dev, 4)) return ops_fail(OMOE_ERR_INVALID, fn, "the weights must be 4-byte aligned");
    if (int rc = ops_apart(all, 4, 1, fn)) return rc;
    if (T == 0) return ops_ok();
    const bool vec = rows_vector(y) && rows_vector(ys);
    return by_chunk(vec, T, d, true, [&](auto v, auto u) {
        constexpr int V = decltype(v)::value, U = decltype(u)::value, C = kChunk<V, U>;
        const int64_t blocks = row_blocks(T, d, C);
        if (blocks > INT32_MAX) return ops_fail(OMOE_ERR_TOO_LARGE, fn, kTooMany);
        return ops_launched(by_types(ys_dtype, y_dtype, [&](auto *xt, auto *ot) {
            using XT = std::remove_pointer_t<decltype(xt)>;
            using OT = std::remove_pointer_t<decltype(ot)>;
            auto go = [&](auto kern) {
                return launch_ex(kern, dim3((unsigned)blocks), dim3(256), 0, static_cast<cudaStream_t>(cuda_stream), ops_pdl(),
                                 static_cast<const XT *>(ys_dev), ldys, static_cast<OT *>(y_dev), ldy, plan->pos, w_dev, T, plan->top_k,
                                 d, ceil_div(d, C), (int)plan->rows_cap);
            };
            return w_dev ? go(unsort_rows_kernel<XT, OT, V, U, true>) : go(unsort_rows_kernel<XT, OT, V, U, false>);
        }), fn);
    });
}

int omoe_sort_rows_backward(const omoe_sort *plan, const void *dxs_dev, int64_t lddxs, int32_t dxs_dtype, void *dx_dev,
                            int64_t lddx, int32_t dx_dtype, int32_t d, void *cuda_stream) {
    return unsort(plan, dxs_dev, lddxs, dxs_dtype, nullptr, dx_dev, lddx, dx_dtype, d, cuda_stream, "omoe_sort_rows_backward");
}

int omoe_unsort_rows(const omoe_sort *plan, const void *ys_dev, int64_t ldys, int32_t ys_dtype, const float *w_dev, void *y_dev,
                     int64_t ldy, int32_t y_dtype, int32_t d, void *cuda_stream) {
    return unsort(plan, ys_dev, ldys, ys_dtype, w_dev, y_dev, ldy, y_dtype, d, cuda_stream, "omoe_unsort_rows");
}

int omoe_unsort_rows_backward(const omoe_sort *plan, const void *dy_dev, int64_t lddy, int32_t dy_dtype, const void *ys_dev,
                              int64_t ldys, int32_t ys_dtype, const float *w_dev, void *dys_dev, int64_t lddys, float *dw_dev,
                              int32_t d, void *cuda_stream) {
    const char *fn = "omoe_unsort_rows_backward";
    if (int rc = check_plan(plan, fn)) return rc;
    const int T = plan->n_tokens, E = plan->n_experts, k = plan->top_k;
    const Rows dys = {dys_dev, lddys, ys_dtype, T ? plan->rows_cap : 0, d}, dy = {dy_dev, lddy, dy_dtype, T, d};
    const Rows ys = {ys_dev, ldys, ys_dtype, T && dw_dev ? plan->rows_cap : 0, d};
    const Rows rows[] = {dys, dy, ys};
    if (int rc = check_rows(rows, dw_dev ? 3 : 2, fn)) return rc;
    if (misaligned(w_dev, 4) || misaligned(dw_dev, 4)) return ops_fail(OMOE_ERR_INVALID, fn, "the weights must be 4-byte aligned");
    const Rows all[] = {dys, words(dw_dev, (int64_t)T * k), dy, ys, words(w_dev, (int64_t)T * k), pos_of(plan), counts_of(plan), offsets_of(plan)};
    if (int rc = ops_apart(all, 8, 2, fn)) return rc;
    if (T == 0) return ops_ok();
    const int slices = pad_slices(plan->row_align);
    const bool vec = rows_vector(dys) && rows_vector(dy) && (!dw_dev || rows_vector(ys));
    const int pads = E * slices;
    int threads = 32;  // per token: two vectors or eight elements each, up to a block of 512
    while (threads < 512 && threads * (vec ? 16 : 8) < d) threads *= 2;
    const int block = threads < 128 ? 128 : threads;
    const int64_t blocks = ((int64_t)T + pads + block / threads - 1) / (block / threads);
    if (blocks > INT32_MAX) return ops_fail(OMOE_ERR_TOO_LARGE, fn, kTooMany);
    return ops_launched(by_types(dy_dtype, ys_dtype, [&](auto *dt, auto *yt) {
        using DT = std::remove_pointer_t<decltype(dt)>;
        using YT = std::remove_pointer_t<decltype(yt)>;
        auto go = [&](auto kern) {
            return launch_ex(kern, dim3((unsigned)blocks), dim3(block), 0, static_cast<cudaStream_t>(cuda_stream), ops_pdl(),
                             static_cast<const DT *>(dy_dev), lddy, static_cast<const YT *>(ys_dev), ldys,
                             static_cast<YT *>(dys_dev), lddys, plan->pos, plan->counts, plan->offsets, w_dev, dw_dev, T, k, pads, slices,
                             d, (int)plan->rows_cap, threads);
        };
        auto by_k = [&](auto v) {
            constexpr int V = decltype(v)::value;
            if (k <= 2) return go(unsort_bwd_kernel<DT, YT, V, 2>);
            if (k <= 4) return go(unsort_bwd_kernel<DT, YT, V, 4>);
            if (k <= 6) return go(unsort_bwd_kernel<DT, YT, V, 6>);
            if (k <= 8) return go(unsort_bwd_kernel<DT, YT, V, 8>);
            return go(unsort_bwd_kernel<DT, YT, V, 16>);
        };
        return vec ? by_k(std::integral_constant<int, 8>()) : by_k(std::integral_constant<int, 1>());
    }), fn);
}

}  // extern "C"
