// Routes of a mixture-of-experts block sorted by expert, and back: the plan
// (a stable counting sort of the routed ids), the tokens' rows in that order,
// the experts' rows weighted and added per token, and the gradients.
//
// Route p = t k + j is token t's j-th expert.  Sorted by expert, routes of one
// expert in order of p, it has row place[p]; source is the inverse.  A route
// without an expert (id -1, or outside [0, E), which also sets a status bit)
// comes behind all others, and its place is kept as ~row.
//
// Kernels:
//   k_expert_count   routes per expert of each segment (more than one segment)
//   k_expert_place   the sort
//   k_expert_rows    rows[place[p]] = x[t]
//   k_expert_combine out[t] = sum_j s[p] y[place[p]] (+ residual[t])
//   k_expert_grad    dy[place[p]] = s[p] dout[t], ds[p] = <dout[t], y[place[p]]>

#include <algorithm>

#include "vmi_device.h"
#include "vmi_internal.h"

namespace {

constexpr int kMaxE = 1024, kMaxK = 32, kMaxT = 65536, kMaxH = 65536;   // (kMaxT rows of kMaxH: 2^30 threads)
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kChunks = 8;                               // groups of 64 routes of a wave
constexpr int kWhole = kSortThreads * kChunks;           // routes of a workgroup at most

struct PlanArgs {
    const int32_t* ids;
    int n, E, seg;          // routes, experts, routes of a segment (a multiple of kSortThreads)
    uint32_t* count;        // [segments][E + 1]
    int32_t *offsets, *source, *place;
    uint32_t* status;
};

__device__ __forceinline__ int ex_wave() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

// The bins of the lane's route in each of the wave's kChunks groups of 64, all asked for
// together: its expert, E for none, -1 behind the segment.
__device__ __forceinline__ void ex_bins(const PlanArgs& a, int p0, int p1, int (&b)[kChunks], bool& odd) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) b[i] = p0 + 64 * i < p1 ? a.ids[min(p0 + 64 * i + lane, a.n - 1)] : 0;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        const bool in = p0 + 64 * i + lane < p1;
        odd |= in && (b[i] < -1 || b[i] >= a.E);
        b[i] = !in ? -1 : (uint32_t)b[i] < (uint32_t)a.E ? b[i] : a.E;
    }
}

__global__ __launch_bounds__(kSortThreads) void k_expert_count(PlanArgs a) {
    __shared__ uint32_t s_n[kMaxE + 1];
    const int run = a.seg / kSortWaves, p0 = blockIdx.x * a.seg + ex_wave() * run, p1 = min(a.n, p0 + run);
    int b[kChunks];
    bool odd = false;
    ex_bins(a, p0, p1, b, odd);
    for (int e = threadIdx.x; e <= a.E; e += kSortThreads) s_n[e] = 0u;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
        if (b[i] >= 0) atomicAdd(&s_n[b[i]], 1u);
    __syncthreads();
    for (int e = threadIdx.x; e <= a.E; e += kSortThreads) a.count[(size_t)blockIdx.x * (a.E + 1) + e] = s_n[e];
}

// One segment per workgroup, a contiguous run of it per wave.  Counts per wave and bin in
// LDS (whole numbers, so that the order of the atomics does not matter), prefix sums over
// waves, segments and bins, then every wave places its run 64 routes at a time: a
// route's row is its bin's next one plus the lower lanes with the same bin, found by one
// ballot per bit of the bin.  Bound by latency.
__global__ __launch_bounds__(kSortThreads) void k_expert_place(PlanArgs a) {
    __shared__ uint32_t s_at[kSortWaves * (kMaxE + 1)];   // [waves][E + 1]
    __shared__ uint32_t s_sum[kSortWaves];
    const int lane = threadIdx.x & 63, w = ex_wave(), B = a.E + 1, run = a.seg / kSortWaves;
    const int p0 = blockIdx.x * a.seg + w * run, p1 = min(a.n, p0 + run);
    int bin[kChunks];
    bool odd = false;
    ex_bins(a, p0, p1, bin, odd);
    for (int i = threadIdx.x; i < kSortWaves * B; i += kSortThreads) s_at[i] = 0u;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
        if (bin[i] >= 0) atomicAdd(&s_at[w * B + bin[i]], 1u);
    if (a.status && __any(odd) && lane == 0) atomicOr(a.status, VMI_STATUS_BAD_SLOT);
    __syncthreads();
    // thread b: bin b's routes in all segments, and in those before this one (1025 bins: two turns)
    uint32_t carry = 0;
    for (int b0 = 0; b0 < B; b0 += kSortThreads) {
        const int b = b0 + threadIdx.x;
        uint32_t all = 0, before = 0;
        if (b < B) {
            if (gridDim.x > 1) {
                constexpr int kAhead = 8;
                for (int i0 = 0; i0 < (int)gridDim.x; i0 += kAhead) {
                    uint32_t c[kAhead];
#pragma unroll
                    for (int i = 0; i < kAhead; ++i) c[i] = a.count[(size_t)min(i0 + i, (int)gridDim.x - 1) * B + b];
#pragma unroll
                    for (int i = 0; i < kAhead; ++i) {
                        c[i] = i0 + i < (int)gridDim.x ? c[i] : 0u;
                        before += i0 + i < (int)blockIdx.x ? c[i] : 0u;
                        all += c[i];
                    }
                }
            } else {
                for (int i = 0; i < kSortWaves; ++i) all += s_at[i * B + b];
            }
        }
        // exclusive prefix sum of `all` over the bins
        uint32_t v = all;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t u = (uint32_t)__shfl_up((int)v, d);
            if (lane >= d) v += u;
        }
        if (lane == 63) s_sum[w] = v;
        __syncthreads();
        uint32_t base = carry;
        for (int i = 0; i < kSortWaves; ++i) {
            if (i < w) base += s_sum[i];
            carry += s_sum[i];
        }
        const uint32_t first = base + v - all;
        if (b < B) {
            if (blockIdx.x == 0) a.offsets[b] = (int32_t)first;   // bin E's first: the rows with an expert
            uint32_t at = first + before;
            for (int i = 0; i < kSortWaves; ++i) {
                const uint32_t c = s_at[i * B + b];
                s_at[i * B + b] = at;
                at += c;
            }
        }
        __syncthreads();
    }
    uint32_t* mine = s_at + w * B;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        if (p0 + 64 * i >= p1) break;
        const int p = p0 + 64 * i + lane, b = max(bin[i], 0);
        const bool in = bin[i] >= 0;
        uint64_t same = __ballot(in);
        for (int bit = 0; (B - 1) >> bit; ++bit) {   // wave-uniform
            const uint64_t m = __ballot((b >> bit) & 1);
            same &= (b >> bit) & 1 ? m : ~m;
        }
        if (in) {
            const uint32_t at = mine[b] + __builtin_popcountll(same & ((1ull << lane) - 1));
            const int32_t row = (int32_t)at;
            a.source[row] = p;
            a.place[p] = b < a.E ? row : ~row;
            // (every lane of the bin has read its start before the last of them moves it on: one wave, in order)
            if ((same >> lane) == 1ull) mine[b] = at + 1;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// A place past the routes' rows (none that k_expert_place writes) reads and writes nothing.
struct RowArgs {
    const vmi_u4 *x, *y;      // tokens' rows, routes' rows
    const vmi_u4* residual;
    const int32_t* place;
    const float* scores;
    vmi_u4* out;
    float* dscores;
    int T, k, U, pieces;      // tokens, routes of one, 16-byte units of a row, its pieces of 64
};

// The wave's token and unit: the pieces of a row go to waves side by side, so that a row is
// asked for at once (token by token of one piece, 8192 x 10 rows took 88 us to combine).
__device__ __forceinline__ bool ex_unit(const RowArgs& a, int& t, int& u) {
    const uint32_t w = blockIdx.x * 4 + ex_wave();
    t = (int)(w / (uint32_t)a.pieces);
    u = (int)(w % (uint32_t)a.pieces) * 64 + (threadIdx.x & 63);
    return t < a.T;
}

template <bool F32>
__device__ __forceinline__ void ex_widen(const vmi_u4& u, float (&v)[F32 ? 4 : 8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (F32) {
            v[i] = __uint_as_float(u[i]);
        } else {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
}
template <bool F32>
__device__ __forceinline__ vmi_u4 ex_narrow(const float (&v)[F32 ? 4 : 8]) {
    vmi_u4 u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (F32)
            u[i] = __float_as_uint(v[i]);
        else
            u[i] = vmi_pack_bf16x2(v[2 * i], v[2 * i + 1]);
    }
    return u;
}

// PAST: all routes' rows together are more than the last cache holds (256 MB), and go past it (8192 x 10 rows of 4 KB
// sorted with gradient 147.6 -> 142.6 us, combined with gradients 220 -> 209).
template <bool PAST>
__device__ __forceinline__ void ex_store(const vmi_u4& v, vmi_u4* at) {
    if constexpr (PAST)
        __builtin_nontemporal_store(v, at);
    else
        *at = v;
}
bool past_cache(const RowArgs& a) { return (int64_t)a.T * a.k * a.U * 16 > (int64_t)256 << 20; }

// A wave per token and 64 units of its row: read once, written to its routes' rows; a
// route without an expert gets zeros.
template <bool PAST>
__global__ __launch_bounds__(256) void k_expert_rows(RowArgs a) {
    int t, u;
    if (!ex_unit(a, t, u)) return;
    const bool in = u < a.U;
    vmi_u4 v = {0, 0, 0, 0};
    if (in) v = a.x[(size_t)t * a.U + u];
    for (int j = 0; j < a.k; ++j) {
        const int32_t p = vmi_sload_i32(a.place + (size_t)t * a.k + j), row = p < 0 ? ~p : p;
        if (in && row < a.T * a.k) ex_store<PAST>(p < 0 ? vmi_u4{0, 0, 0, 0} : v, a.out + (size_t)row * a.U + u);
    }
}

// A wave per token and 64 units: the routes' rows in rank order in fp32, then the
// residual, rounded once.  Eight rows are asked for at a time.
template <bool F32>
__global__ __launch_bounds__(256) void k_expert_combine(RowArgs a) {
    constexpr int N = F32 ? 4 : 8, kAhead = 8;
    int t, u;
    if (!ex_unit(a, t, u) || u >= a.U) return;
    float sum[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = 0.0f;
    for (int j0 = 0; j0 < a.k; j0 += kAhead) {
        vmi_u4 r[kAhead];
        float s[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int j = min(j0 + i, a.k - 1);
            int32_t p = j0 + i < a.k ? vmi_sload_i32(a.place + (size_t)t * a.k + j) : -1;
            p = p < a.T * a.k ? p : -1;
            s[i] = p < 0 ? 0.0f : a.scores ? a.scores[(size_t)t * a.k + j] : 1.0f;
            r[i] = vmi_u4{0, 0, 0, 0};
            if (p >= 0) r[i] = __builtin_nontemporal_load(a.y + (size_t)p * a.U + u);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            float v[N];
            ex_widen<F32>(r[i], v);
            if (j0 + i < a.k)
#pragma unroll
                for (int e = 0; e < N; ++e) sum[e] = fmaf(s[i], v[e], sum[e]);
        }
    }
    if (a.residual) {
        float v[N];
        ex_widen<F32>(a.residual[(size_t)t * a.U + u], v);
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += v[e];
    }
    a.out[(size_t)t * a.U + u] = ex_narrow<F32>(sum);
}

// A wave per route: its row's gradient, and the weight's as a sum over the row in a
// fixed order.  Routes without an expert: zeros in both, their rows of y not read.
template <bool F32, bool PAST>
__global__ __launch_bounds__(256) void k_expert_grad(RowArgs a) {
    constexpr int N = F32 ? 4 : 8;
    const int64_t p = (int64_t)blockIdx.x * 4 + ex_wave();
    if (p >= (int64_t)a.T * a.k) return;
    const int lane = threadIdx.x & 63, t = (int)(p / a.k);
    const int32_t at = vmi_sload_i32(a.place + p);
    const int64_t row = at < 0 ? ~at : at;
    if (row >= (int64_t)a.T * a.k) return;
    const float s = at < 0 ? 0.0f : a.scores ? a.scores[p] : 1.0f;
    float dot = 0.0f;
    for (int u = lane; u < a.U; u += 64) {
        float d[N], g[N];
        ex_widen<F32>(a.x[(size_t)t * a.U + u], d);
        if (at >= 0 && a.dscores) {
            float v[N];
            ex_widen<F32>(__builtin_nontemporal_load(a.y + row * a.U + u), v);
#pragma unroll
            for (int e = 0; e < N; ++e) dot = fmaf(d[e], v[e], dot);
        }
        if (a.out) {
#pragma unroll
            for (int e = 0; e < N; ++e) g[e] = at < 0 ? 0.0f : s * d[e];
            ex_store<PAST>(ex_narrow<F32>(g), a.out + row * a.U + u);
        }
    }
    if (a.dscores) {
        dot = vmi_wave_sum_canon(dot);
        if (lane == 0) a.dscores[p] = dot;
    }
}

// Up to kWhole routes one workgroup; above, segments of a quarter of that (40 of them for 8192 x 10) up to 64 segments,
// then whole ones.
int plan_segment(int64_t n) { return n <= kWhole || n > 16 * kWhole ? kWhole : kWhole / 4; }
int plan_segments(int64_t n) { return (int)std::max<int64_t>(1, (n + plan_segment(n) - 1) / plan_segment(n)); }

bool shape_ok(int T, int k) { return T >= 0 && T <= kMaxT && k > 0 && k <= kMaxK; }

// Checks what the row entries share; U: 16-byte units of a row.
int rows_check(const char* what, int dtype, int T, int k, int H, int& U) {
    if (dtype != VMI_F32 && dtype != VMI_BF16) return vmi::fail(VMI_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
    if (!shape_ok(T, k)) return vmi::fail(VMI_ERR_INVALID, "%s: T=%d k=%d (T <= %d, k <= %d)", what, T, k, kMaxT, kMaxK);
    const int per = dtype == VMI_F32 ? 4 : 8;
    if (H <= 0 || H % per || H > kMaxH)
        return vmi::fail(VMI_ERR_UNSUPPORTED, "%s: hidden=%d must be a multiple of %d up to %d", what, H, per, kMaxH);
    U = H / per;
    return VMI_OK;
}
unsigned row_groups(RowArgs& a) {   // of four waves, one a token and piece
    a.pieces = (a.U + 63) / 64;
    return (unsigned)(((int64_t)a.T * a.pieces + 3) / 4);
}
bool aligned(std::initializer_list<const void*> ps) {
    uintptr_t m = 0;
    for (const void* p : ps) m |= reinterpret_cast<uintptr_t>(p);
    return !(m & 15);
}
int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? VMI_OK : vmi::hip_fail(e, what);
}

}  // namespace

extern "C" size_t vmi_expert_plan_workspace_bytes(int T, int k, int num_experts) {
    if (!shape_ok(T, k) || num_experts <= 0 || num_experts > kMaxE) return 0;
    const int nb = plan_segments((int64_t)T * k);
    return vmi::align256(nb == 1 ? 1 : (size_t)nb * (num_experts + 1) * 4);
}

extern "C" int vmi_expert_plan(const int32_t* ids, int T, int k, int num_experts, int32_t* offsets, int32_t* source,
                               int32_t* place, uint32_t* status, void* workspace, size_t workspace_bytes, void* stream) {
    vmi::clear_error();
    if (!shape_ok(T, k)) return vmi::fail(VMI_ERR_INVALID, "T=%d k=%d (T <= %d, k <= %d)", T, k, kMaxT, kMaxK);
    if (num_experts <= 0 || num_experts > kMaxE)
        return vmi::fail(VMI_ERR_UNSUPPORTED, "num_experts=%d must be in [1, %d]", num_experts, kMaxE);
    if (!offsets || (T && (!ids || !source || !place))) return vmi::fail(VMI_ERR_INVALID, "null ids/offsets/source/place");
    const int n = T * k, nb = plan_segments(n);
    const size_t need = vmi_expert_plan_workspace_bytes(T, k, num_experts);
    if (nb > 1 && (!workspace || workspace_bytes < need || !aligned({workspace})))
        return vmi::fail(VMI_ERR_WORKSPACE, "workspace needs %zu bytes, 16-byte aligned (got %zu)", need, workspace_bytes);
    PlanArgs a{ids, n, num_experts, nb == 1 ? (std::max(n, 1) + kSortThreads - 1) / kSortThreads * kSortThreads : plan_segment(n),
               static_cast<uint32_t*>(workspace), offsets, source, place, status};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (nb > 1) hipLaunchKernelGGL(k_expert_count, dim3(nb), dim3(kSortThreads), 0, s, a);
    hipLaunchKernelGGL(k_expert_place, dim3(nb), dim3(kSortThreads), 0, s, a);
    return launched("k_expert_place launch");
}

extern "C" int vmi_expert_rows(const void* x, int dtype, int T, int k, int hidden, const int32_t* place, void* rows,
                               void* stream) {
    vmi::clear_error();
    RowArgs a{};
    if (const int rc = rows_check("vmi_expert_rows", dtype, T, k, hidden, a.U)) return rc;
    if (T == 0) return VMI_OK;
    if (!x || !place || !rows) return vmi::fail(VMI_ERR_INVALID, "null x/place/rows");
    if (!aligned({x, rows})) return vmi::fail(VMI_ERR_INVALID, "x and rows must be 16-byte aligned");
    a.x = static_cast<const vmi_u4*>(x);
    a.place = place;
    a.out = static_cast<vmi_u4*>(rows);
    a.T = T;
    a.k = k;
    const dim3 grid(row_groups(a));
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (past_cache(a))
        hipLaunchKernelGGL(k_expert_rows<true>, grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(k_expert_rows<false>, grid, dim3(256), 0, s, a);
    return launched("k_expert_rows launch");
}

extern "C" int vmi_expert_combine(const void* y, int dtype, int T, int k, int hidden, const int32_t* place,
                                  const float* scores, const void* residual, void* out, void* stream) {
    vmi::clear_error();
    RowArgs a{};
    if (const int rc = rows_check("vmi_expert_combine", dtype, T, k, hidden, a.U)) return rc;
    if (T == 0) return VMI_OK;
    if (!y || !place || !out) return vmi::fail(VMI_ERR_INVALID, "null y/place/out");
    if (!aligned({y, residual, out})) return vmi::fail(VMI_ERR_INVALID, "y, residual and out must be 16-byte aligned");
    a.y = static_cast<const vmi_u4*>(y);
    a.residual = static_cast<const vmi_u4*>(residual);
    a.place = place;
    a.scores = scores;
    a.out = static_cast<vmi_u4*>(out);
    a.T = T;
    a.k = k;
    const dim3 grid(row_groups(a));
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == VMI_F32)
        hipLaunchKernelGGL((k_expert_combine<true>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((k_expert_combine<false>), grid, dim3(256), 0, s, a);
    return launched("k_expert_combine launch");
}

extern "C" int vmi_expert_combine_grad(const void* d_out, const void* y, int dtype, int T, int k, int hidden,
                                       const int32_t* place, const float* scores, void* d_y, float* d_scores,
                                       void* stream) {
    vmi::clear_error();
    RowArgs a{};
    if (const int rc = rows_check("vmi_expert_combine_grad", dtype, T, k, hidden, a.U)) return rc;
    if (T == 0) return VMI_OK;   // (empty outputs are null)
    if (!d_y && !d_scores) return vmi::fail(VMI_ERR_INVALID, "nothing to compute (d_y and d_scores both null)");
    if (!d_out || !place || (d_scores && !y)) return vmi::fail(VMI_ERR_INVALID, "null d_out/place/y");
    if (!aligned({d_out, y, d_y})) return vmi::fail(VMI_ERR_INVALID, "d_out, y and d_y must be 16-byte aligned");
    a.x = static_cast<const vmi_u4*>(d_out);
    a.y = static_cast<const vmi_u4*>(y);
    a.place = place;
    a.scores = scores;
    a.out = static_cast<vmi_u4*>(d_y);
    a.dscores = d_scores;
    a.T = T;
    a.k = k;
    const dim3 grid((unsigned)(((int64_t)T * k + 3) / 4));
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool f32 = dtype == VMI_F32, past = past_cache(a);
    if (f32 && past)
        hipLaunchKernelGGL((k_expert_grad<true, true>), grid, dim3(256), 0, s, a);
    else if (f32)
        hipLaunchKernelGGL((k_expert_grad<true, false>), grid, dim3(256), 0, s, a);
    else if (past)
        hipLaunchKernelGGL((k_expert_grad<false, true>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((k_expert_grad<false, false>), grid, dim3(256), 0, s, a);
    return launched("k_expert_grad launch");
}
