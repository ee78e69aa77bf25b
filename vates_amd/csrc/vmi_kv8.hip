// The 8-bit KV cache of an attention layer: rows quantised as they are
// written, read back, formed from a batch's projections (q and k RMSNorm,
// rotary embedding), and attention over them.
//
// A row (one position's key or value of one kv head, 256 dims) is held as
// codes c in [-127, 127] and one fp32 scale s, and stands for s c:
//   a = max |x|,  s = a / 127,  c = RNE(127 x / a)     (a = 0: s = 0, c = 0)
// The quotient is taken as (x 127 k) / (a k) with one correctly rounded fp32
// division (k = 2^-7 for a > 2^100, else 1: no overflow); for bf16 x the
// numerator is exact and no quotient that is not a tie comes closer to one
// than 2^-8 / 510, more than that division's rounding, so the codes are those
// of exact arithmetic.  A row with an infinity or NaN has s = NaN and reads
// back as NaN.  A scale belongs to one row: a scale shared by several
// positions would change what is held of a position with the ones behind it
// (rejected drafts, a row that is not finite), and an append would round the
// open block again.  It costs 8 bytes beside a position's 512.
//
// Layout: per kv head max_len / 32 records of 16,640 bytes, 32 positions each:
//   [0, 8192)        key codes + 128: position kt, dim d at
//                    ((a*4 + (d>>6))*64 + ((d>>3)&3)*16 + nl)*16 + ((d>>5)&1)*8 + (d&7),
//                    nl = 4*(kt>>3) + (kt&3), a = (kt>>2)&1
//   [8192, 16384)    value codes + 128: ((d>>5)*64 + (kt>>3)*16 + (d&15))*16 + ((d>>4)&1)*8 + (kt&7)
//   [16384, 16512)   key scales, [16512, 16640) value scales, fp32
// the operand order of the matrix instructions that read it: lane l of a wave
// takes the 16 bytes at 16 l of each kilobyte, two operands at once.
//
// Kernels:
//   k_kv8_write    rows [n_kv, n, 256] bf16 into the cache
//   k_kv8_read     rows of the cache as bf16 or fp32
//   k_kv8_heads    q | gate, k and v projections of a batch: q and k normalised
//                  and rotated, q out in bf16, k and v into the cache
//   k_kv8_split    attention of up to 64 query rows per kv head, the keys dealt
//                  to the waves of the whole device
//   k_kv8_flash    attention of more rows, 64 or more to a workgroup
//   k_kv8_merge    joins the parts, times sigmoid(gate)

#include <algorithm>

#include "vmi_attn_device.h"
#include "vmi_internal.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kBlk = VMI_KV_BLOCK;           // positions per record
constexpr int kHalfRec = kKv8Half;           // bytes of a record's keys (or values)
constexpr int kRec = kKv8Record;
static_assert(kRec == 2 * kHalfRec + 2 * kBlk * 4 && kHalfRec == kBlk * kHeadDim, "record");

// One row, dims 4 l .. 4 l + 3 in lane l: the four codes + 128 in a word, the
// row's scale in every lane.
__device__ __forceinline__ uint32_t kv8_quantise(const float (&x)[4], float& scale) {
    const float m = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) bad = bad || !(fabsf(x[j]) < INFINITY);
    const float a = vmi_wave_max(m);
    if (__any(bad)) {
        scale = __builtin_nanf("");
        return 0x80808080u;
    }
    scale = __fdiv_rn(a, 127.0f);
    if (!(a > 0.0f)) return 0x80808080u;
    const float k = a > 0x1p100f ? 0x1p-7f : 1.0f, den = a * k, num = 127.0f * k;
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) w |= (uint32_t)((int)rintf(__fdiv_rn(x[j] * num, den)) + 128) << (8 * j);
    return w;
}

// ------------------------------------------------------------------- store
struct WriteArgs {
    const uint16_t* src[2];       // keys, values
    int64_t head[2], row[2];      // element strides between kv heads and positions
    int n, pos0;
    uint8_t* cache;
    int max_len;
};

// grid (records touched, n_kv): one record per workgroup.  Each wave quantises
// eight positions' keys and values into an image of the record in LDS, which
// then goes out 16 bytes a thread; bytes of positions outside the call are left
// as they are (a key's 16 bytes are one position's; eight positions share a
// value group's 8 bytes, so a group that is not covered goes byte by byte).
// Bound by the bytes of the rows read.
__global__ __launch_bounds__(kThreads) void k_kv8_write(WriteArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t s_rec[kRec];
    const int lane = threadIdx.x & 63, w = at_wave(), g = blockIdx.y;
    const int blk = a.pos0 / kBlk + blockIdx.x;
    const int lo = max(a.pos0 - blk * kBlk, 0), hi = min(a.pos0 + a.n - blk * kBlk, kBlk);  // positions of the record
    uint2 raw[2][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int kt = 8 * w + i;
        const int64_t r = (int64_t)(min(max(kt, lo), hi - 1) + blk * kBlk - a.pos0);
#pragma unroll
        for (int z = 0; z < 2; ++z)
            raw[z][i] = *reinterpret_cast<const uint2*>(a.src[z] + g * a.head[z] + r * a.row[z] + 4 * lane);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int kt = 8 * w + i;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const float x[4] = {__uint_as_float(raw[z][i].x << 16), __uint_as_float(raw[z][i].x & 0xffff0000u),
                                __uint_as_float(raw[z][i].y << 16), __uint_as_float(raw[z][i].y & 0xffff0000u)};
            float s;
            const uint32_t c = kv8_quantise(x, s);
            if (z == 0) {
                *reinterpret_cast<uint32_t*>(s_rec + kv8_k_off(kt, 4 * lane)) = c;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) s_rec[kv8_v_off(kt, 4 * lane + j)] = (uint8_t)(c >> (8 * j));
            }
            if (lane == 0) *reinterpret_cast<float*>(s_rec + kv8_scale_off(kt, z)) = s;
        }
    }
    __syncthreads();
    uint8_t* rec = a.cache + ((size_t)g * (a.max_len / kBlk) + blk) * kRec;
    const bool whole = lo == 0 && hi == kBlk;
    for (int i = threadIdx.x; i < kRec / 16; i += kThreads) {
        const vmi_u4 u = *reinterpret_cast<const vmi_u4*>(s_rec + 16 * i);
        if (whole) {
            *reinterpret_cast<vmi_u4*>(rec + 16 * i) = u;
        } else if (i < kHalfRec / 16) {
            const int nl = i & 15, kt = 8 * (nl >> 2) + 4 * (i >> 8) + (nl & 3);
            if (kt >= lo && kt < hi) *reinterpret_cast<vmi_u4*>(rec + 16 * i) = u;
        } else if (i < 2 * kHalfRec / 16) {
            const int k0 = 8 * ((i >> 4) & 3);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (k0 + e >= lo && k0 + e < hi) {
                    rec[16 * i + e] = s_rec[16 * i + e];
                    rec[16 * i + 8 + e] = s_rec[16 * i + 8 + e];
                }
        } else {
            const int k0 = (4 * i) % kBlk;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (k0 + e >= lo && k0 + e < hi) *reinterpret_cast<uint32_t*>(rec + 16 * i + 4 * e) = u[e];
        }
    }
}

// -------------------------------------------------------------------- load
struct ReadArgs {
    const uint8_t* cache;
    int max_len, pos0, n;
    void* dst[2];   // keys, values: [n_kv, n, 256], either may be null
};

// grid (records touched, n_kv, keys | values): the half record through LDS,
// rows out whole.  Bound by the bytes written.
template <bool F32>
__global__ __launch_bounds__(kThreads) void k_kv8_read(ReadArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t s_half[kHalfRec];
    __shared__ float s_scale[kBlk];
    const int z = blockIdx.z, g = blockIdx.y, blk = a.pos0 / kBlk + blockIdx.x;
    if (!a.dst[z]) return;
    const uint8_t* rec = a.cache + ((size_t)g * (a.max_len / kBlk) + blk) * kRec;
    for (int i = threadIdx.x; i < kHalfRec / 16; i += kThreads)
        *reinterpret_cast<vmi_u4*>(s_half + 16 * i) = *reinterpret_cast<const vmi_u4*>(rec + z * kHalfRec + 16 * i);
    if (threadIdx.x < kBlk) s_scale[threadIdx.x] = *reinterpret_cast<const float*>(rec + kv8_scale_off(threadIdx.x, z));
    __syncthreads();
    const int lane = threadIdx.x & 63, w = at_wave();
    const int lo = max(a.pos0 - blk * kBlk, 0), hi = min(a.pos0 + a.n - blk * kBlk, kBlk);
    for (int kt = lo + w; kt < hi; kt += kWaves) {
        uint32_t c;
        if (z == 0) {
            c = *reinterpret_cast<const uint32_t*>(s_half + kv8_k_off(kt, 4 * lane));
        } else {
            c = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) c |= (uint32_t)s_half[kv8_v_off(kt, 4 * lane + j) - kHalfRec] << (8 * j);
        }
        const float s = s_scale[kt];
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = s * (float)((int)((c >> (8 * j)) & 255u) - 128);
        const size_t at = ((size_t)g * a.n + (blk * kBlk + kt - a.pos0)) * kHeadDim + 4 * lane;
        if constexpr (F32)
            *reinterpret_cast<float4*>(static_cast<float*>(a.dst[z]) + at) = make_float4(x[0], x[1], x[2], x[3]);
        else
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.dst[z]) + at) =
                make_uint2(vmi_pack_bf16x2(x[0], x[1]), vmi_pack_bf16x2(x[2], x[3]));
    }
}

// ------------------------------------------------------------------- heads
using vmi::Kv8Heads;

__device__ __forceinline__ int kv8_pos0(int pos0, const int32_t* pos_dev, int span, int max_len) {
    const int p = pos_dev ? *pos_dev : pos0;
    return min(max(p, 0), max_len - span);
}

// One row, dims 4 l .. in lane l: RMSNorm times the weight, then the rotary
// pairs (i, i + rd/2), in fp32.
__device__ __forceinline__ void kv8_norm_rope(float (&x)[4], const float (&nw)[4], float eps, const float2* cs, int rd,
                                              float* srow) {
    const int lane = threadIdx.x & 63, half = rd / 2;
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) ss = fmaf(x[j], x[j], ss);
    ss = vmi_wave_sum_canon(ss);
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(ss * (1.0f / (float)kHeadDim) + eps));
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (x[j] * inv) * nw[j];
    float pr[4];
    if (rd % 8 == 0) {  // wave-uniform: the partners of a lane's dims are another lane's
        const int src = (4 * lane < half ? lane + half / 4 : lane - half / 4) & 63;
#pragma unroll
        for (int j = 0; j < 4; ++j) pr[j] = __shfl(x[j], src, 64);
    } else {
        *reinterpret_cast<float4*>(srow + 4 * lane) = make_float4(x[0], x[1], x[2], x[3]);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();  // srow is this wave's own
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = 4 * lane + j;
            pr[j] = srow[d < half ? d + half : d < rd ? d - half : d];
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();  // read before the next row is written
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int d = 4 * lane + j;
        if (d < rd) {
            const float2 c = cs[d < half ? d : d - half];
            x[j] = fmaf(x[j], c.x, (d < half ? -pr[j] : pr[j]) * c.y);
        }
    }
}

constexpr int kHeadTok = 8;  // positions of a workgroup: one value group of a record

// grid (groups of eight positions, heads (q, then k, then v), paths): a wave
// takes the group's tokens w and w + 4 of one head.  Keys go out 4 bytes a lane;
// a value group's eight positions are collected in LDS and go out together.
// Bound by the bytes of the projections on a prompt, by latency on a batch.
__global__ __launch_bounds__(kThreads) void k_kv8_heads(Kv8Heads a) {
    __shared__ float2 s_cs[kHeadTok][kHeadDim / 2];
    __shared__ float s_row[kWaves][kHeadDim];
    __shared__ __attribute__((aligned(16))) uint8_t s_v[kHeadDim][kHeadTok];
    const int lane = threadIdx.x & 63, w = at_wave(), path = blockIdx.z;
    const int pos0 = kv8_pos0(a.pos0, a.pos_dev, a.T, a.max_len);
    if (a.pos_dev && a.status && blockIdx.x == 0 && blockIdx.y == 0 && path == 0 && threadIdx.x == 0 && *a.pos_dev != pos0)
        atomicOr(a.status, VMI_STATUS_BAD_POS);
    const int p0 = (pos0 / kHeadTok + blockIdx.x) * kHeadTok;   // the group's first position
    const int lo = max(pos0 - p0, 0), hi = min(pos0 + a.T - p0, kHeadTok);
    if (lo >= hi) return;                                       // whole workgroup
    const int hh = a.h0 + blockIdx.y;
    const bool is_q = hh < a.n_heads, is_v = hh >= a.n_heads + a.n_kv;
    const int stride = (a.n_heads + a.n_kv) * 2 * kHeadDim;
    const int col = is_q ? hh * 2 * kHeadDim : a.n_heads * 2 * kHeadDim + (hh - a.n_heads) * kHeadDim;
    const float* rows = a.qkv + (size_t)path * a.T * stride + col + 4 * lane;
    float x[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int kt = min(max(w + kWaves * i, lo), hi - 1);
        const vmi_f4 v = *reinterpret_cast<const vmi_f4*>(rows + (size_t)(p0 + kt - pos0) * stride);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i][j] = v[j];
    }
    if (!is_v) {
        const uint16_t* nwp = is_q ? a.q_norm : a.k_norm;
        float nw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) nw[j] = vmi_bf16_to_f32(nwp[4 * lane + j]);
        const int half = a.rope_dim / 2;
        for (int i = threadIdx.x; i < kHeadTok * half; i += kThreads) {
            const int kt = i / half, f = i - kt * half;
            if (kt >= lo && kt < hi) s_cs[kt][f] = rotary_cs(p0 + kt, f, a.rope_base);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
            kv8_norm_rope(x[i], nw, a.eps, s_cs[min(max(w + kWaves * i, lo), hi - 1)], a.rope_dim, s_row[w]);
    }
    const int g = is_v ? hh - a.n_heads - a.n_kv : hh - a.n_heads;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int kt = w + kWaves * i, t = p0 + kt - pos0, tb = (p0 + kt) % kBlk;
        const bool mine = kt >= lo && kt < hi;   // wave-uniform
        if (is_q) {
            if (mine)
                *reinterpret_cast<uint2*>(a.q + ((size_t)(path * a.T + t) * a.n_heads + hh) * kHeadDim + 4 * lane) =
                    make_uint2(vmi_pack_bf16x2(x[i][0], x[i][1]), vmi_pack_bf16x2(x[i][2], x[i][3]));
            continue;
        }
        float s;
        const uint32_t c = kv8_quantise(x[i], s);
        if (a.tree) {  // plain rows, one record per token
            if (!mine) continue;
            uint8_t* side = a.tree + ((size_t)(path * a.n_kv + g) * a.T + t) * kKv8TreeRow;
            *reinterpret_cast<uint32_t*>(side + (is_v ? kHeadDim : 0) + 4 * lane) = c;
            if (lane == 0) *reinterpret_cast<float*>(side + 2 * kHeadDim + (is_v ? 4 : 0)) = s;
            continue;
        }
        uint8_t* rec = a.cache + ((size_t)g * (a.max_len / kBlk) + p0 / kBlk) * kRec;
        if (mine && lane == 0) *reinterpret_cast<float*>(rec + kv8_scale_off(tb, is_v)) = s;
        if (!is_v) {
            if (mine) *reinterpret_cast<uint32_t*>(rec + kv8_k_off(tb, 4 * lane)) = c;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) s_v[4 * lane + j][kt] = (uint8_t)(c >> (8 * j));
        }
    }
    if (!is_v || a.tree) return;
    __syncthreads();
    // thread d: dim d of the group's eight positions
    const int d = threadIdx.x;
    uint8_t* dst = a.cache + ((size_t)g * (a.max_len / kBlk) + p0 / kBlk) * kRec + kv8_v_off(p0 % kBlk, d);
    if (lo == 0 && hi == kHeadTok) {
        *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(s_v[d]);
    } else {
        for (int kt = lo; kt < hi; ++kt) dst[kt] = s_v[d][kt];
    }
}

// --------------------------------------------------------------- attention
using vmi::Kv8Attn;

// Eight codes + 128 as fp16 1024 + (c + 128), exactly (0x6400 is 1024 with a
// mantissa step of 1): one byte permute per pair.
__device__ __forceinline__ vmi_u4 kv8_widen(uint32_t w0, uint32_t w1) {
    vmi_u4 r;
    r[0] = __builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u);
    r[1] = __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u);
    r[2] = __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u);
    r[3] = __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u);
    return r;
}
// The codes themselves (1152 taken off again, exact).
__device__ __forceinline__ vmi_u4 kv8_signed(const vmi_u4& u) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    vmi_u4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, (uint32_t)u[i]) + off);
    return r;
}

constexpr float kPScale = 16384.0f;   // probabilities times value scales, in fp16: at most this
constexpr float kMinRef = 1e-30f;

// 16 MS query rows of a wave: lane (nl, q4) belongs to row 16 m + nl.
template <int MS>
struct Kv8Rows {
    vmi_u4 q[MS][8];   // fp16 query times a power of two, dims 32 kk + 8 q4 ..
    float c0[MS];      // -1152 sum(q): what the codes' offset of 1152 adds to a score, taken off
    float cx[MS];      // log2(e) / 16 over the power of two; NaN for a row that is not finite
    int last[MS];      // last visible position
};

// Running softmax of those rows.  o is in units of s / kPScale.
template <int MS>
struct Kv8Sums {
    vmi_f4 o[MS][16];  // dims 16 dt + 4 q4 + r of row nl
    float m[MS];       // maximum score, in powers of two
    float l[MS];       // the lane's share of sum 2^(score - m)
    float s[MS];       // largest value scale seen
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < MS; ++i) {
            m[i] = -3.402823466e38f;
            l[i] = 0.0f;
            s[i] = kMinRef;
#pragma unroll
            for (int d = 0; d < 16; ++d) o[i][d] = vmi_f4{0.f, 0.f, 0.f, 0.f};
        }
    }
};

// The wave's query rows, from row r0 of R (rows behind the last repeat it).
template <int MS>
__device__ __forceinline__ void kv8_load_rows(const Kv8Attn& a, const uint16_t* q, int g, int r0, int R, int pos0,
                                              Kv8Rows<MS>& o) {
    const int lane = threadIdx.x & 63, nl = lane & 15, q4 = lane >> 4, G = a.n_heads / a.n_kv;
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        const int row = min(r0 + 16 * m + nl, R - 1), t = row / G, h = g * G + row % G;
        o.last[m] = pos0 + t;
        const vmi_u4* src = reinterpret_cast<const vmi_u4*>(q + ((size_t)t * a.n_heads + h) * kHeadDim + 8 * q4);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) o.q[m][kk] = src[4 * kk];
    }
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        uint32_t am = 0;   // largest magnitude, as bf16 bits
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i) am = max(am, max(o.q[m][kk][i] & 0x7fffu, (o.q[m][kk][i] >> 16) & 0x7fffu));
        am = max(am, (uint32_t)__shfl_xor((int)am, 16));
        am = max(am, (uint32_t)__shfl_xor((int)am, 32));
        const float amax = __uint_as_float(am << 16);
        // max |q| f in (2^13, 2^14]: the products of a finite row stay finite, and elements
        // down to 2^-28 of the largest keep their eight bits
        const bool fin = amax < INFINITY;
        const float f = vmi_fp16_range_scale(amax);
        float sum = 0.0f;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t u = o.q[m][kk][i];
                const _Float16 lo = (_Float16)(__uint_as_float(u << 16) * f), hi = (_Float16)(__uint_as_float(u & 0xffff0000u) * f);
                sum += (float)lo;
                sum += (float)hi;
                o.q[m][kk][i] = vmi_h2_bits(lo, hi);
            }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        o.c0[m] = -1152.0f * sum;
        o.cx[m] = fin ? 0.09016844005556021f / f : __builtin_nanf("");   // log2(e) / sqrt(256)
    }
}

// One record's 32 keys, the first at position p0.  S^T = K Q^T: a lane holds
// the scores of keys 8 q4 + e of its row, which are, as probabilities, already
// the B operand of O^T = V^T P^T.  A key's scale enters its score, a value's its
// probability; the product goes to fp16 (11 bits) relative to the row's largest
// value scale so far, and whatever raises that or the running maximum rescales
// the sums.  mask (wave-uniform): the record reaches past the visible positions
// of some row; masked scores count as minus infinity and masked scales as zero,
// so that nothing stored behind a row's last position reaches it.
template <int MS>
__device__ __forceinline__ void kv8_step(const uint8_t* rec, const Kv8Rows<MS>& Q, int p0, bool mask, Kv8Sums<MS>& S) {
    const int lane = threadIdx.x & 63, q4 = lane >> 4;
    const vmi_u4* K = reinterpret_cast<const vmi_u4*>(rec);
    const vmi_u4* V = reinterpret_cast<const vmi_u4*>(rec + kHalfRec);
    const vmi_f4* sc = reinterpret_cast<const vmi_f4*>(rec + 2 * kHalfRec + 32 * q4);
    vmi_f4 s[MS][2];
#pragma unroll
    for (int m = 0; m < MS; ++m) s[m][0] = s[m][1] = vmi_f4{Q.c0[m], Q.c0[m], Q.c0[m], Q.c0[m]};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const vmi_u4 u = K[(4 * a + j) * 64 + lane];
            const vmi_u4 k0 = kv8_widen(u[0], u[1]), k1 = kv8_widen(u[2], u[3]);
#pragma unroll
            for (int m = 0; m < MS; ++m) s[m][a] = vmi_mfma_f16(k0, Q.q[m][2 * j], s[m][a]);
#pragma unroll
            for (int m = 0; m < MS; ++m) s[m][a] = vmi_mfma_f16(k1, Q.q[m][2 * j + 1], s[m][a]);
        }
    }
    const vmi_f4 ks[2] = {sc[0], sc[1]}, vs[2] = {sc[8], sc[9]};
    vmi_u4 pb[MS];
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        float x[8], v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = s[m][e >> 2][e & 3] * (ks[e >> 2][e & 3] * Q.cx[m]);
            v[e] = vs[e >> 2][e & 3];
        }
        if (mask) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool seen = p0 + 8 * q4 + e <= Q.last[m];
                x[e] = seen ? x[e] : -INFINITY;
                v[e] = seen ? v[e] : 0.0f;
            }
        }
        float nm = S.m[m], ns = S.s[m];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            nm = fmaxf(nm, x[e]);
            ns = fmaxf(ns, v[e]);
        }
        nm = fmaxf(nm, __shfl_xor(nm, 16));
        ns = fmaxf(ns, __shfl_xor(ns, 16));
        nm = fmaxf(nm, __shfl_xor(nm, 32));
        ns = fmaxf(ns, __shfl_xor(ns, 32));
        if (__any(nm > S.m[m] || ns > S.s[m])) {
            const float f = __builtin_amdgcn_exp2f(S.m[m] - nm);
            S.l[m] *= f;
            const float fo = ns > S.s[m] ? f * (S.s[m] / ns) : f;
#pragma unroll
            for (int d = 0; d < 16; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) S.o[m][d][r] *= fo;
            S.m[m] = nm;
            S.s[m] = ns;
        }
        const float inv = kPScale / ns;
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            p[e] = __builtin_amdgcn_exp2f(x[e] - nm);
            S.l[m] += p[e];
            p[e] *= v[e] * inv;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) pb[m][i] = vmi_h2_bits((_Float16)p[2 * i], (_Float16)p[2 * i + 1]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const vmi_u4 u = V[j * 64 + lane];
        const vmi_u4 v0 = kv8_signed(kv8_widen(u[0], u[1])), v1 = kv8_signed(kv8_widen(u[2], u[3]));
#pragma unroll
        for (int m = 0; m < MS; ++m) S.o[m][2 * j] = vmi_mfma_f16(v0, pb[m], S.o[m][2 * j]);
#pragma unroll
        for (int m = 0; m < MS; ++m) S.o[m][2 * j + 1] = vmi_mfma_f16(v1, pb[m], S.o[m][2 * j + 1]);
    }
}

// A record by DMA into a wave's LDS, 17 operations.
constexpr int kRecOps = 17;
__device__ __forceinline__ void kv8_fetch(const uint8_t* rec, uint8_t* lds) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < 16; ++j) vmi_lds_dma16_opaque_nt(rec + 1024 * j + 16 * lane, lds + 1024 * j);
    vmi_lds_dma4_opaque(rec + 2 * kHalfRec + 4 * lane, lds + 2 * kHalfRec);
}

// Waits for the wave's own LDS reads, before a slot that they read is refilled.
__device__ __forceinline__ void kv8_lds_wait() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt 0
    asm volatile("" ::: "memory");
}

constexpr int kRing = 2;  // records of a wave's ring

// grid (S, n_kv, paths): record b of a kv head belongs to wave (b / S) % 4 of
// workgroup b % S, whatever the length, the batch and the capacity, so that a
// row's sums do not depend on them, a short cache still spreads over the device,
// and a long one keeps every CU reading.  A wave runs its records through its
// own ring in LDS (no barrier until the end); the four waves then join in LDS
// and the workgroup writes one part: maximum, sum and unnormalised output of
// each row, in fp32.  Bound by the bytes of the cache from some ten thousand
// positions on, below by the latency of a record and of the two launches.
template <int MS>
__global__ __launch_bounds__(kThreads, 1) void k_kv8_split(Kv8Attn a) {
    __shared__ __attribute__((aligned(16))) uint8_t s_ring[kWaves][kRing][kRec];
    __shared__ float s_ml[kWaves][16 * MS][2];
    const int lane = threadIdx.x & 63, w = at_wave(), nl = lane & 15, q4 = lane >> 4;
    const int wg = blockIdx.x, S = gridDim.x, g = blockIdx.y, path = blockIdx.z, T = a.span;
    const int pos0 = kv8_pos0(a.pos0, a.pos_dev, T, a.max_len);
    if (a.pos_dev && a.status && wg == 0 && g == 0 && path == 0 && threadIdx.x == 0 && *a.pos_dev != pos0)
        atomicOr(a.status, VMI_STATUS_BAD_POS);
    const int nblk = (pos0 + T + kBlk - 1) / kBlk;
    if (wg >= nblk) return;   // whole workgroup
    const int R = T * (a.n_heads / a.n_kv), step = kWaves * S, first = wg + S * w;
    const uint8_t* head = a.cache + (size_t)g * (a.max_len / kBlk) * kRec;
    Kv8Rows<MS> Q;
    kv8_load_rows<MS>(a, a.q + (size_t)path * T * a.n_heads * kHeadDim, g, 0, R, pos0, Q);
    if (first < nblk) kv8_fetch(head + (size_t)first * kRec, s_ring[w][0]);
    if (first + step < nblk) kv8_fetch(head + (size_t)(first + step) * kRec, s_ring[w][1]);
    Kv8Sums<MS> Y;
    Y.clear();
    int slot = 0;
    for (int b = first; b < nblk; b += step) {
        if (b + step < nblk)
            vmi_vm_wait_c<kRecOps>();   // the next record may be in flight
        else
            vmi_vm_wait_c<0>();
        asm volatile("" ::: "memory");
        uint8_t* rec = s_ring[w][slot];
        if (a.tree && kBlk * b + kBlk > pos0) {
            // a path's own tokens in place of what the cache holds there
            for (int t = max(kBlk * b - pos0, 0); t < min(T, kBlk * b + kBlk - pos0); ++t) {
                const uint8_t* side = a.tree + ((size_t)(path * a.n_kv + g) * T + t) * kKv8TreeRow;
                const int kt = pos0 + t - kBlk * b;
                const uint32_t kc = *reinterpret_cast<const uint32_t*>(side + 4 * lane);
                const uint32_t vc = *reinterpret_cast<const uint32_t*>(side + kHeadDim + 4 * lane);
                *reinterpret_cast<uint32_t*>(rec + kv8_k_off(kt, 4 * lane)) = kc;
#pragma unroll
                for (int j = 0; j < 4; ++j) rec[kv8_v_off(kt, 4 * lane + j)] = (uint8_t)(vc >> (8 * j));
                if (lane < 2)
                    *reinterpret_cast<float*>(rec + kv8_scale_off(kt, lane)) =
                        *reinterpret_cast<const float*>(side + 2 * kHeadDim + 4 * lane);
            }
            kv8_lds_wait();
        }
        kv8_step<MS>(rec, Q, kBlk * b, kBlk * b + kBlk - 1 > pos0, Y);
        kv8_lds_wait();
        if (b + kRing * step < nblk) kv8_fetch(head + (size_t)(b + kRing * step) * kRec, s_ring[w][slot]);
        slot ^= 1;
    }
    // the four waves, in wave order
    float* s_o = reinterpret_cast<float*>(&s_ring[0][0][0]);   // [waves][16][256], one row group at a time
    static_assert(kWaves * 16 * kHeadDim * 4 <= (int)sizeof(s_ring), "row group");
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        float l = Y.l[m];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (q4 == 0) {
            s_ml[w][16 * m + nl][0] = Y.m[m];
            s_ml[w][16 * m + nl][1] = l;
        }
    }
    const size_t part = ((size_t)(g * S + wg) * gridDim.z + path) * a.rp;
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        __syncthreads();   // every wave is done with its ring, or with the group before
        const float u = Y.s[m] * (1.0f / kPScale);
#pragma unroll
        for (int d = 0; d < 16; ++d) {
            const vmi_f4 y = {Y.o[m][d][0] * u, Y.o[m][d][1] * u, Y.o[m][d][2] * u, Y.o[m][d][3] * u};
            *reinterpret_cast<vmi_f4*>(s_o + (w * 16 + nl) * kHeadDim + 4 * ((4 * d + q4) ^ nl)) = y;
        }
        __syncthreads();
        for (int r = w; r < 16; r += kWaves) {   // a wave per row, 4 dims a lane
            const int row = 16 * m + r;
            if (row >= R) break;
            float M = s_ml[0][row][0];
#pragma unroll
            for (int v = 1; v < kWaves; ++v) M = fmaxf(M, s_ml[v][row][0]);
            float l = 0.0f;
            vmi_f4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int v = 0; v < kWaves; ++v) {
                const float f = __builtin_amdgcn_exp2f(s_ml[v][row][0] - M);
                l = fmaf(s_ml[v][row][1], f, l);
                const vmi_f4 z = *reinterpret_cast<const vmi_f4*>(s_o + (v * 16 + r) * kHeadDim + 4 * (lane ^ r));
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = fmaf(z[e], f, y[e]);
            }
            *reinterpret_cast<vmi_f4*>(a.part_o + (part + row) * kHeadDim + 4 * lane) = y;
            if (lane == 0) *reinterpret_cast<float2*>(a.part_ml + (part + row) * 2) = make_float2(M, l);
        }
    }
}

__device__ __forceinline__ uint2 kv8_gated(const vmi_f4& y, float l, const float* gate) {
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = y[e] / l;
    if (gate) {
        const vmi_f4 z = *reinterpret_cast<const vmi_f4*>(gate);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] /= 1.0f + expf(-z[e]);
    }
    return make_uint2(vmi_pack_bf16x2(o[0], o[1]), vmi_pack_bf16x2(o[2], o[3]));
}

// grid (rows of all heads), one wave per part in turn: the parts of a row in
// index order per wave, the four waves in order.  Every row sees position 0, so
// its sum is positive (or NaN, which it hands on).
__global__ __launch_bounds__(kThreads) void k_kv8_merge(Kv8Attn a, int parts, bool by_record) {
    __shared__ float s_m[kWaves], s_l[kWaves];
    __shared__ vmi_f4 s_o[kWaves][64];
    const int lane = threadIdx.x & 63, w = at_wave();
    const int t = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads, G = a.n_heads / a.n_kv, g = h / G;
    const int path = t / a.span, row = (t - path * a.span) * G + h % G;
    const int nblk = (kv8_pos0(a.pos0, a.pos_dev, a.span, a.max_len) + a.span + kBlk - 1) / kBlk;
    const int n = by_record ? min(parts, nblk) : parts;   // k_kv8_split: the workgroups that had a record
    const size_t at = ((size_t)(g * parts) * a.paths + path) * a.rp + row, inc = (size_t)a.paths * a.rp;
    float m = -3.402823466e38f, l = 0.0f;
    vmi_f4 y = {0.f, 0.f, 0.f, 0.f};
    for (int s = w; s < n; s += kWaves) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (at + s * inc) * 2);
        const vmi_f4 z = *reinterpret_cast<const vmi_f4*>(a.part_o + (at + s * inc) * kHeadDim + 4 * lane);
        const float nm = fmaxf(m, ml.x), f = __builtin_amdgcn_exp2f(m - nm), fz = __builtin_amdgcn_exp2f(ml.x - nm);
        m = nm;
        l = fmaf(l, f, ml.y * fz);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = fmaf(y[e], f, z[e] * fz);
    }
    s_o[w][lane] = y;
    if (lane == 0) {
        s_m[w] = m;
        s_l[w] = l;
    }
    __syncthreads();
    if (w) return;
    float M = s_m[0];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) M = fmaxf(M, s_m[v]);
    l = 0.0f;
    y = vmi_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
        const float f = __builtin_amdgcn_exp2f(s_m[v] - M);
        l = fmaf(s_l[v], f, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = fmaf(s_o[v][lane][e], f, y[e]);
    }
    const float* gate = a.gate ? a.gate + t * a.gate_tok + h * a.gate_head + 4 * lane : nullptr;
    *reinterpret_cast<uint2*>(a.o + ((size_t)t * a.n_heads + h) * kHeadDim + 4 * lane) = kv8_gated(y, l, gate);
}

// grid (tiles of 64 M rows, n_kv, key parts): four waves of 16 M rows share
// each record, two slots of LDS by DMA.  Part z of P takes an equal run of the
// tile's records; with P > 1 the parts are written as k_kv8_split's are.
template <int M>
__global__ __launch_bounds__(kThreads, M == 4 ? 1 : 2) void k_kv8_flash(Kv8Attn a) {
    __shared__ __attribute__((aligned(16))) uint8_t s_rec[2][kRec];
    const int lane = threadIdx.x & 63, w = at_wave(), nl = lane & 15, q4 = lane >> 4;
    const int g = blockIdx.y, G = a.n_heads / a.n_kv, R = a.span * G, P = gridDim.z, z = blockIdx.z;
    const int pos0 = kv8_pos0(a.pos0, a.pos_dev, a.span, a.max_len);
    if (a.pos_dev && a.status && blockIdx.x == 0 && g == 0 && z == 0 && threadIdx.x == 0 && *a.pos_dev != pos0)
        atomicOr(a.status, VMI_STATUS_BAD_POS);
    const int tile = (int)gridDim.x - 1 - (int)blockIdx.x;   // late tiles see the most keys: first
    const int r0 = tile * (64 * M) + 16 * M * w, last_row = min(tile * (64 * M) + 64 * M, R) - 1;
    const int nb = (pos0 + last_row / G) / kBlk + 1;
    const int b0 = (int)((long)nb * z / P), b1 = (int)((long)nb * (z + 1) / P);
    const uint8_t* head = a.cache + (size_t)g * (a.max_len / kBlk) * kRec;
    auto issue = [&](int b, int u) {
        const uint8_t* rec = head + (size_t)b * kRec;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            vmi_lds_dma16_opaque(rec + 1024 * (4 * j + w) + 16 * lane, s_rec[u] + 1024 * (4 * j + w));
        vmi_lds_dma4_opaque(rec + 2 * kHalfRec + 4 * lane, s_rec[u] + 2 * kHalfRec);   // every wave the same bytes
    };
    Kv8Rows<M> Q;
    kv8_load_rows<M>(a, a.q, g, r0, R, pos0, Q);
    const int first = pos0 + min(r0, R - 1) / G;
    Kv8Sums<M> Y;
    Y.clear();
    if (b0 < b1) issue(b0, 0);
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
        vmi_vm_wait_c<0>();
        __syncthreads();
        if (b + 1 < b1) issue(b + 1, (b + 1 - b0) & 1);
        kv8_step<M>(s_rec[(b - b0) & 1], Q, kBlk * b, kBlk * b + kBlk - 1 > first, Y);
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
        float l = Y.l[m];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        const int row = r0 + 16 * m + nl;
        if (row >= R) continue;
        const float u = Y.s[m] * (1.0f / kPScale);
        const int t = row / G, h = g * G + row % G;
        if (P > 1) {
            const size_t at = (size_t)(g * P + z) * a.rp + row;
#pragma unroll
            for (int d = 0; d < 16; ++d)
                *reinterpret_cast<vmi_f4*>(a.part_o + at * kHeadDim + 16 * d + 4 * q4) =
                    vmi_f4{Y.o[m][d][0] * u, Y.o[m][d][1] * u, Y.o[m][d][2] * u, Y.o[m][d][3] * u};
            if (q4 == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(Y.m[m], l);
        } else {
            const float* gate = a.gate ? a.gate + t * a.gate_tok + h * a.gate_head + 4 * q4 : nullptr;
            uint16_t* o = a.o + ((size_t)t * a.n_heads + h) * kHeadDim + 4 * q4;
#pragma unroll
            for (int d = 0; d < 16; ++d) {
                const vmi_f4 y = {Y.o[m][d][0] * u, Y.o[m][d][1] * u, Y.o[m][d][2] * u, Y.o[m][d][3] * u};
                *reinterpret_cast<uint2*>(o + 16 * d) = kv8_gated(y, l, gate ? gate + 16 * d : nullptr);
            }
        }
    }
}

// ------------------------------------------------------------------- host
constexpr int kSplitRows = 64;   // rows per kv head of k_kv8_split
constexpr int kMaxTok = 8192;

// Workgroups per kv head that share its records in k_kv8_split: one per CU
// over all kv heads.
int split_groups(int n_kv) { return std::max(1, vmi::device_cus() / n_kv); }

struct FlashPlan {
    int m, tiles, parts;
};

// Tiles of 64 M rows and the parts their keys are split into, from the rows
// and kv heads alone.
FlashPlan flash_plan(int rows, int n_kv) {
    const int ncu = vmi::device_cus();
    FlashPlan p;
    p.m = (rows + 127) / 128 * n_kv >= ncu ? 2 : 1;
    p.tiles = (rows + 64 * p.m - 1) / (64 * p.m);
    p.parts = std::max(1, std::min(2 * ncu / (p.tiles * n_kv), 64));
    return p;
}

}  // namespace

double vmi::kv8_rope_base(float theta, int rope_dim) {
    return rope_dim ? pow((double)theta, -2.0 / (double)rope_dim) : 1.0;
}

bool vmi::kv8_heads_ok(int n_heads, int n_kv) {
    return n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 && n_heads <= 1024;
}

size_t vmi::kv8_attention_parts_bytes(int paths, int span, int n_heads, int n_kv) {
    if (paths < 1 || span < 1 || paths > 16 || span > kMaxTok || !kv8_heads_ok(n_heads, n_kv)) return 0;
    const int R = span * (n_heads / n_kv);
    size_t rows;
    if (R <= kSplitRows) {
        rows = (size_t)n_kv * split_groups(n_kv) * paths * R;
    } else {
        if (paths != 1) return 0;
        const FlashPlan p = flash_plan(R, n_kv);
        rows = p.parts > 1 ? (size_t)n_kv * p.parts * R : 1;
    }
    return align256(rows * kHeadDim * 4) + align256(rows * 2 * 4);
}

hipError_t vmi::launch_kv8_heads(const Kv8Heads& h, int paths, hipStream_t s) {
    const int groups = (h.T + kHeadTok - 2) / kHeadTok + 1;   // at any alignment
    hipLaunchKernelGGL(k_kv8_heads, dim3(groups, h.n_heads + 2 * h.n_kv - h.h0, paths), dim3(kThreads), 0, s, h);
    return hipGetLastError();
}

hipError_t vmi::launch_kv8_attention(Kv8Attn a, void* parts, hipStream_t s) {
    const int R = a.span * (a.n_heads / a.n_kv);
    a.rp = R;
    a.part_o = static_cast<float*>(parts);
    int n;
    size_t rows;
    if (R <= kSplitRows) {
        n = split_groups(a.n_kv);
        rows = (size_t)a.n_kv * n * a.paths * R;
        a.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(parts) + align256(rows * kHeadDim * 4));
        const dim3 grid(n, a.n_kv, a.paths), blk(kThreads);
        switch ((R + 15) / 16) {
            case 1: hipLaunchKernelGGL(k_kv8_split<1>, grid, blk, 0, s, a); break;
            case 2: hipLaunchKernelGGL(k_kv8_split<2>, grid, blk, 0, s, a); break;
            case 3: hipLaunchKernelGGL(k_kv8_split<3>, grid, blk, 0, s, a); break;
            default: hipLaunchKernelGGL(k_kv8_split<4>, grid, blk, 0, s, a); break;
        }
    } else {
        const FlashPlan p = flash_plan(R, a.n_kv);
        n = p.parts;
        rows = n > 1 ? (size_t)a.n_kv * n * R : 1;
        a.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(parts) + align256(rows * kHeadDim * 4));
        const dim3 grid(p.tiles, a.n_kv, p.parts), blk(kThreads);
        if (p.m == 2)
            hipLaunchKernelGGL(k_kv8_flash<2>, grid, blk, 0, s, a);
        else
            hipLaunchKernelGGL(k_kv8_flash<1>, grid, blk, 0, s, a);
        if (n == 1) return hipGetLastError();
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_kv8_merge, dim3(a.paths * a.span * a.n_heads), dim3(kThreads), 0, s, a, n, R <= kSplitRows);
    return hipGetLastError();
}

namespace {

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The checks that every entry point makes of a cache and a range of positions.
int check_cache(const void* cache, int n_kv, int max_len, int pos0, int n, const int32_t* pos_device) {
    if (!cache || !aligned(cache, 16)) return vmi::fail(VMI_ERR_INVALID, "cache null or not 16-byte aligned");
    if (n_kv <= 0 || n_kv > 1024) return vmi::fail(VMI_ERR_INVALID, "n_kv_heads=%d must be in [1, 1024]", n_kv);
    if (max_len <= 0 || max_len % kBlk) return vmi::fail(VMI_ERR_INVALID, "max_len=%d must be a positive multiple of %d", max_len, kBlk);
    if (n <= 0 || n > max_len || (!pos_device && (pos0 < 0 || pos0 > max_len - n)))
        return vmi::fail(VMI_ERR_INVALID, "positions %d.. of %d outside the capacity %d", pos0, n, max_len);
    return VMI_OK;
}

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? VMI_OK : vmi::hip_fail(e, what);
}

}  // namespace

namespace {

constexpr int kMaxSpan = 8, kMaxBatch = 16;   // tokens of a path, of a call (as vmi_attention_layer)

struct LayerWs {
    size_t xn, qkv, q, o, parts, bytes;
};

LayerWs layer_ws(int paths, int span, int H, int n_heads, int n_kv) {
    LayerWs L{};
    const size_t T = (size_t)paths * span, rows = T * kHeadDim;
    size_t off = 0;
    auto take = [&](size_t b) {
        const size_t o = off;
        off += vmi::align256(b);
        return o;
    };
    L.xn = take(T * H * 2);
    L.qkv = take(rows * 2 * (n_heads + n_kv) * 4);
    L.q = take(rows * n_heads * 2);
    L.o = take(rows * n_heads * 2);
    L.parts = take(vmi::kv8_attention_parts_bytes(paths, span, n_heads, n_kv));
    L.bytes = off;
    return L;
}

bool layer_shape_ok(int paths, int span, int hidden, int n_heads, int n_kv) {
    return paths > 0 && span > 0 && span <= kMaxSpan && paths <= kMaxBatch && paths * span <= kMaxBatch && hidden > 0 &&
           hidden % 512 == 0 && hidden <= 4096 && vmi::kv8_heads_ok(n_heads, n_kv) && n_kv <= 1024 &&
           span * (n_heads / n_kv) <= kSplitRows &&
           (size_t)std::min(paths * span, 8) * std::max(hidden, n_heads * kHeadDim) * 2 <= 65536;  // the GEMV's rows
}

// The attention block over `paths` sequences of `span` tokens that share the
// cache below pos0 (one path: a batch, its rows into the cache; several: a draft
// tree, its rows into `tree`).
int layer_impl(const vmi_attn_layer_desc* desc, const uint16_t* x, int paths, int span, int pos0,
               const int32_t* pos_device, uint8_t* cache, int max_len, uint8_t* tree, uint16_t* out, uint32_t* status,
               void* workspace, size_t workspace_bytes, hipStream_t s) {
    if (!desc) return vmi::fail(VMI_ERR_INVALID, "null desc");
    const vmi_attn_layer_desc& D = *desc;
    if (D.head_dim != kHeadDim) return vmi::fail(VMI_ERR_UNSUPPORTED, "head_dim=%d (256 only)", D.head_dim);
    if ((D.bits != 4 && D.bits != 8) || D.group != 64) return vmi::fail(VMI_ERR_UNSUPPORTED, "bits=%d group=%d", D.bits, D.group);
    if (!layer_shape_ok(paths, span, D.hidden, D.n_heads, D.n_kv_heads))
        return vmi::fail(VMI_ERR_UNSUPPORTED, "paths=%d span=%d hidden=%d heads=%d/%d not built", paths, span, D.hidden,
                         D.n_heads, D.n_kv_heads);
    if (D.rope_dim < 0 || D.rope_dim > kHeadDim || D.rope_dim % 2 || !(D.rope_theta > 0.0f))
        return vmi::fail(VMI_ERR_INVALID, "rope_dim=%d rope_theta=%g", D.rope_dim, (double)D.rope_theta);
    const int rc = check_cache(cache, D.n_kv_heads, max_len, pos0, span, pos_device);
    if (rc != VMI_OK) return rc;
    if (!vmi::qmat_ok(D.q_proj) || !vmi::qmat_ok(D.k_proj) || !vmi::qmat_ok(D.v_proj) || !vmi::qmat_ok(D.o_proj))
        return vmi::fail(VMI_ERR_INVALID, "projection weights must be non-null and 16-byte aligned");
    if (!x || !out || !D.input_norm || !D.q_norm || !D.k_norm || !aligned(x, 16) || !aligned(out, 16) ||
        !aligned(D.input_norm, 16))
        return vmi::fail(VMI_ERR_INVALID, "x, out or norm weights null or not 16-byte aligned");
    const int T = paths * span;
    const LayerWs L = layer_ws(paths, span, D.hidden, D.n_heads, D.n_kv_heads);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < L.bytes)
        return vmi::fail(VMI_ERR_WORKSPACE, "workspace needs %zu bytes (got %zu)", L.bytes, workspace_bytes);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    float* qkv = reinterpret_cast<float*>(ws + L.qkv);
    uint16_t* q = reinterpret_cast<uint16_t*>(ws + L.q);
    uint16_t* o = reinterpret_cast<uint16_t*>(ws + L.o);
    const int stride = (D.n_heads + D.n_kv_heads) * 2 * kHeadDim;

    vmi::QgemvCall p{};
    p.x = x; p.T = T; p.K = D.hidden; p.bits = D.bits;
    p.m[0] = D.q_proj; p.m[1] = D.k_proj; p.m[2] = D.v_proj;
    p.rows[0] = D.n_heads * 2 * kHeadDim; p.rows[1] = p.rows[2] = D.n_kv_heads * kHeadDim;
    p.nrows = stride; p.out = qkv; p.out_stride = stride;
    p.norm_w = D.input_norm; p.eps = D.norm_eps;
    hipError_t e;
    if (!vmi::qgemv_fuses_norm(p)) {
        uint16_t* xn = reinterpret_cast<uint16_t*>(ws + L.xn);
        e = vmi::launch_rmsnorm(x, D.input_norm, D.norm_eps, T, D.hidden, xn, s);
        if (e != hipSuccess) return vmi::hip_fail(e, "input norm launch");
        p.x = xn;
        p.norm_w = nullptr;
    }
    e = vmi::launch_qgemv(p, s);
    if (e != hipSuccess) return vmi::hip_fail(e, "qkv projection launch");
    vmi::Kv8Heads h{};
    h.qkv = qkv; h.T = span; h.n_heads = D.n_heads; h.n_kv = D.n_kv_heads;
    h.q_norm = D.q_norm; h.k_norm = D.k_norm; h.eps = D.norm_eps; h.rope_dim = D.rope_dim;
    h.rope_base = vmi::kv8_rope_base(D.rope_theta, D.rope_dim);
    h.pos0 = pos0; h.pos_dev = pos_device; h.max_len = max_len; h.cache = cache; h.tree = tree; h.q = q; h.status = status;
    e = vmi::launch_kv8_heads(h, paths, s);
    if (e != hipSuccess) return vmi::hip_fail(e, "k_kv8_heads launch");
    vmi::Kv8Attn a{};
    a.q = q; a.cache = cache; a.tree = tree; a.n_heads = D.n_heads; a.n_kv = D.n_kv_heads; a.span = span; a.paths = paths;
    a.pos0 = pos0; a.pos_dev = pos_device; a.max_len = max_len;
    a.gate = qkv + kHeadDim; a.gate_tok = stride; a.gate_head = 2 * kHeadDim; a.o = o;
    e = vmi::launch_kv8_attention(a, ws + L.parts, s);
    if (e != hipSuccess) return vmi::hip_fail(e, "attention launch");
    vmi::QgemvCall c{};
    c.x = o; c.T = T; c.K = D.n_heads * kHeadDim; c.bits = D.bits;
    c.m[0] = c.m[1] = c.m[2] = D.o_proj;
    c.rows[0] = c.nrows = D.hidden;
    c.out_stride = D.hidden; c.residual = x; c.out_bf16 = out;
    e = vmi::launch_qgemv(c, s);
    return e == hipSuccess ? VMI_OK : vmi::hip_fail(e, "o_proj launch");
}

}  // namespace

extern "C" size_t vmi_attention_kv8_workspace_bytes(int paths, int span, int hidden, int n_heads, int n_kv_heads) {
    return layer_shape_ok(paths, span, hidden, n_heads, n_kv_heads) ? layer_ws(paths, span, hidden, n_heads, n_kv_heads).bytes : 0;
}

extern "C" int vmi_attention_layer_kv8(const vmi_attn_layer_desc* desc, const uint16_t* x, int T, int pos0,
                                       const int32_t* pos_device, uint8_t* cache, int max_len, uint16_t* out,
                                       uint32_t* status, void* workspace, size_t workspace_bytes, void* stream) {
    vmi::clear_error();
    return layer_impl(desc, x, 1, T, pos0, pos_device, cache, max_len, nullptr, out, status, workspace, workspace_bytes,
                      static_cast<hipStream_t>(stream));
}

extern "C" int vmi_attention_tree_kv8(const vmi_attn_layer_desc* desc, const uint16_t* x, int paths, int span, int pos0,
                                      const int32_t* pos_device, const uint8_t* cache, int max_len, uint8_t* tree,
                                      uint16_t* out, uint32_t* status, void* workspace, size_t workspace_bytes,
                                      void* stream) {
    vmi::clear_error();
    if (!tree || !aligned(tree, 16)) return vmi::fail(VMI_ERR_INVALID, "tree rows null or not 16-byte aligned");
    // the cache is only read: every path's rows go to `tree`
    return layer_impl(desc, x, paths, span, pos0, pos_device, const_cast<uint8_t*>(cache), max_len, tree, out, status,
                      workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" size_t vmi_kv8_bytes(int n_kv_heads, int max_len) {
    if (n_kv_heads <= 0 || n_kv_heads > 1024 || max_len <= 0 || max_len % kBlk) return 0;
    return (size_t)n_kv_heads * (max_len / kBlk) * kRec;
}

extern "C" int vmi_kv8_write(const uint16_t* keys, int64_t key_head, int64_t key_row, const uint16_t* values,
                             int64_t value_head, int64_t value_row, int n_kv_heads, int pos0, int n, uint8_t* cache,
                             int max_len, void* stream) {
    vmi::clear_error();
    const int rc = check_cache(cache, n_kv_heads, max_len, pos0, n, nullptr);
    if (rc != VMI_OK) return rc;
    if (!keys || !values || !aligned(keys, 8) || !aligned(values, 8))
        return vmi::fail(VMI_ERR_INVALID, "keys or values null or not 8-byte aligned");
    if ((key_head | key_row | value_head | value_row) & 3)
        return vmi::fail(VMI_ERR_INVALID, "strides must be multiples of 4 elements");
    WriteArgs a{{keys, values}, {key_head, value_head}, {key_row, value_row}, n, pos0, cache, max_len};
    const int recs = (pos0 + n - 1) / kBlk - pos0 / kBlk + 1;
    hipLaunchKernelGGL(k_kv8_write, dim3(recs, n_kv_heads), dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
    return launched("k_kv8_write launch");
}

extern "C" int vmi_kv8_read(const uint8_t* cache, int n_kv_heads, int max_len, int pos0, int n, void* keys, void* values,
                            int dtype, void* stream) {
    vmi::clear_error();
    const int rc = check_cache(cache, n_kv_heads, max_len, pos0, n, nullptr);
    if (rc != VMI_OK) return rc;
    if (dtype != VMI_F32 && dtype != VMI_BF16) return vmi::fail(VMI_ERR_UNSUPPORTED, "dtype=%d", dtype);
    if ((!keys && !values) || !aligned(keys, 16) || !aligned(values, 16))
        return vmi::fail(VMI_ERR_INVALID, "keys and values null, or not 16-byte aligned");
    ReadArgs a{cache, max_len, pos0, n, {keys, values}};
    const dim3 grid((pos0 + n - 1) / kBlk - pos0 / kBlk + 1, n_kv_heads, 2);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == VMI_F32)
        hipLaunchKernelGGL(k_kv8_read<true>, grid, dim3(kThreads), 0, s, a);
    else
        hipLaunchKernelGGL(k_kv8_read<false>, grid, dim3(kThreads), 0, s, a);
    return launched("k_kv8_read launch");
}

extern "C" int vmi_kv8_append(const float* qkv, int T, int n_heads, int n_kv_heads, const uint16_t* q_norm,
                              const uint16_t* k_norm, float eps, int rope_dim, float rope_theta, int pos0,
                              const int32_t* pos_device, uint8_t* cache, int max_len, uint16_t* q_out, uint32_t* status,
                              void* stream) {
    vmi::clear_error();
    const int rc = check_cache(cache, n_kv_heads, max_len, pos0, T, pos_device);
    if (rc != VMI_OK) return rc;
    if (!vmi::kv8_heads_ok(n_heads, n_kv_heads))
        return vmi::fail(VMI_ERR_INVALID, "n_heads=%d n_kv_heads=%d", n_heads, n_kv_heads);
    if (rope_dim < 0 || rope_dim > kHeadDim || rope_dim % 2 || !(rope_theta > 0.0f))
        return vmi::fail(VMI_ERR_INVALID, "rope_dim=%d rope_theta=%g", rope_dim, (double)rope_theta);
    if (!qkv || !aligned(qkv, 16) || !k_norm || (q_out && !q_norm) || !aligned(q_out, 16))
        return vmi::fail(VMI_ERR_INVALID, "null or misaligned qkv, norm weights or q");
    vmi::Kv8Heads h{};
    h.qkv = qkv; h.T = T; h.n_heads = n_heads; h.n_kv = n_kv_heads; h.h0 = q_out ? 0 : n_heads;
    h.q_norm = q_norm; h.k_norm = k_norm; h.eps = eps; h.rope_dim = rope_dim;
    h.rope_base = vmi::kv8_rope_base(rope_theta, rope_dim);
    h.pos0 = pos0; h.pos_dev = pos_device; h.max_len = max_len; h.cache = cache; h.q = q_out; h.status = status;
    const hipError_t e = vmi::launch_kv8_heads(h, 1, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? VMI_OK : vmi::hip_fail(e, "k_kv8_heads launch");
}

extern "C" size_t vmi_kv8_attention_workspace_bytes(int T, int n_heads, int n_kv_heads) {
    return vmi::kv8_attention_parts_bytes(1, T, n_heads, n_kv_heads);
}

extern "C" int vmi_kv8_attention(const uint16_t* q, int T, int n_heads, int n_kv_heads, int pos0,
                                 const int32_t* pos_device, const uint8_t* cache, int max_len, const float* gate,
                                 int64_t gate_token, int64_t gate_head, uint16_t* out, uint32_t* status, void* workspace,
                                 size_t workspace_bytes, void* stream) {
    vmi::clear_error();
    const int rc = check_cache(cache, n_kv_heads, max_len, pos0, T, pos_device);
    if (rc != VMI_OK) return rc;
    if (!vmi::kv8_heads_ok(n_heads, n_kv_heads))
        return vmi::fail(VMI_ERR_INVALID, "n_heads=%d n_kv_heads=%d", n_heads, n_kv_heads);
    const size_t need = vmi::kv8_attention_parts_bytes(1, T, n_heads, n_kv_heads);
    if (!need) return vmi::fail(VMI_ERR_UNSUPPORTED, "T=%d exceeds %d", T, kMaxTok);
    if (!q || !out || !aligned(q, 16) || !aligned(out, 16)) return vmi::fail(VMI_ERR_INVALID, "q or out null or not 16-byte aligned");
    if (gate && (!aligned(gate, 16) || ((gate_token | gate_head) & 3)))
        return vmi::fail(VMI_ERR_INVALID, "gate rows must be 16-byte aligned");
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < need)
        return vmi::fail(VMI_ERR_WORKSPACE, "workspace needs %zu bytes (got %zu)", need, workspace_bytes);
    vmi::Kv8Attn a{};
    a.q = q; a.cache = cache; a.n_heads = n_heads; a.n_kv = n_kv_heads; a.span = T; a.paths = 1;
    a.pos0 = pos0; a.pos_dev = pos_device; a.max_len = max_len; a.status = status;
    a.gate = gate; a.gate_tok = gate_token; a.gate_head = gate_head; a.o = out;
    const hipError_t e = vmi::launch_kv8_attention(a, workspace, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? VMI_OK : vmi::hip_fail(e, "attention launch");
}
