// The 8-bit KV cache of an attention layer: rows quantised as they are
// written, read back, formed from a batch's projections (q and k RMSNorm,
// rotary embedding), and attention over them.
//
// A row (one position's key or value of one kv head, 256 dims) is held as
// codes c in [-127, 127] and one fp32 scale s, and stands for s c:
//   a = max |x|,  s = a / 127,  c = RNE(127 x / a)     (a = 0: s = 0, c = 0)
// For bf16 x the codes are those of exact arithmetic (kv8_quantise).  A row with an
// infinity or NaN has s = NaN and reads back as NaN.  A scale belongs to one row: a scale
// shared by several positions would change what is held of a position with the ones
// behind it (rejected drafts, a row that is not finite), and an append would round the
// open block again.  It costs 8 bytes beside a position's 512.
//
// Layout: per kv head max_len / 32 records of 16,640 bytes, 32 positions each:
//   [0, 8192)        key codes (int8): position kt, dim d at
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
//   k_kv8_flash, k_kv8_flash_short
//                  attention of more rows, 256 or 128 to a workgroup
//   k_kv8_merge, k_kv8_merge_rows
//                  join the parts, times sigmoid(gate)

#include <algorithm>
#include <type_traits>

#include "vmi_attn_device.h"
#include "vmi_internal.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kBlk = VMI_KV_BLOCK;           // positions per record
constexpr int kHalfRec = kKv8Half;           // bytes of a record's keys (or values)
constexpr int kRec = kKv8Record;
static_assert(kRec == 2 * kHalfRec + 2 * kBlk * 4 && kHalfRec == kBlk * kHeadDim, "record");

constexpr uint32_t kKeySign = 0x80808080u;   // a word's codes + 128 and the codes themselves

// N elements of a row per lane, the row's largest magnitude a and whether the row
// holds an infinity or NaN (alike in every lane of the row): the codes + 128, four to
// a word, and the scale.  127 x / a is taken as x (127 / a), off by at most three parts in
// 2^24, and rounded by adding 2^23 + 2^22 + 128, whose sum's low byte is the code.  BF16:
// x has eight bits, and its quotient is a tie or 2^-17 of itself and more away from
// one (|254 x - (2 n + 1) a| is a multiple of x's last bit): rounded to twenty bits
// first, it goes to the even code exactly where it should (checked for every pair of
// mantissas).  A tie is no rare case, one element in some six hundred: a division where
// a wave has one took twice the instructions, and the store 30 us in place of 20.
template <int N, bool BF16>
__device__ __forceinline__ void kv8_quantise(float (&x)[N], float a, bool bad, uint32_t (&w)[N / 4], float& scale) {
    scale = bad ? __builtin_nanf("") : __fdiv_rn(a, 127.0f);
    if (__any(a < 0x1p-100f && a > 0.0f)) {   // 127 / a would leave fp32
        const float k = a < 0x1p-100f ? 0x1p64f : 1.0f;
        a *= k;
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] *= k;
    }
    const float inv = a > 0.0f && !bad ? __fdiv_rn(127.0f, a) : 0.0f;
    uint32_t t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        constexpr float kMagic = 12582912.0f + 128.0f;
        if constexpr (BF16)
            t[i] = __float_as_uint(__uint_as_float((__float_as_uint(x[i] * inv) + 8u) & ~15u) + kMagic);
        else
            t[i] = __float_as_uint(fmaf(x[i], inv, kMagic));
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const uint32_t lo = __builtin_amdgcn_perm(t[4 * i + 1], t[4 * i], 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(t[4 * i + 3], t[4 * i + 2], 0x04000c0cu);
        w[i] = bad ? 0x80808080u : lo | hi;
    }
}

// ------------------------------------------------------------------- store
struct WriteArgs {
    const uint16_t* src[2];       // keys, values
    int64_t head[2], row[2];      // element strides between kv heads and positions
    int n, pos0;
    uint8_t* cache;
    int max_len;
};

// Sixteen bf16 of a row per lane (two 16-byte pieces), sixteen lanes a row: codes
// and scale.
__device__ __forceinline__ void kv8_row16(const vmi_u4& p0, const vmi_u4& p1, uint32_t (&w)[4], float& scale) {
    typedef uint16_t us2 __attribute__((ext_vector_type(2)));
    us2 pm = {0, 0};   // largest magnitude, as bf16 bits: infinities and NaN above the finite ones
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        pm = __builtin_elementwise_max(pm, __builtin_bit_cast(us2, (uint32_t)p0[i] & 0x7fff7fffu));
        pm = __builtin_elementwise_max(pm, __builtin_bit_cast(us2, (uint32_t)p1[i] & 0x7fff7fffu));
    }
    uint32_t am = max((uint32_t)pm[0], (uint32_t)pm[1]);
    am = max(am, vmi_dpp_u32<VMI_DPP_XOR1>(am));
    am = max(am, vmi_dpp_u32<VMI_DPP_XOR2>(am));
    am = max(am, vmi_dpp_u32<VMI_DPP_HALF_MIRROR>(am));
    am = max(am, vmi_dpp_u32<VMI_DPP_MIRROR>(am));
    float x[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(p0[i] << 16);
        x[2 * i + 1] = __uint_as_float(p0[i] & 0xffff0000u);
        x[8 + 2 * i] = __uint_as_float(p1[i] << 16);
        x[8 + 2 * i + 1] = __uint_as_float(p1[i] & 0xffff0000u);
    }
    kv8_quantise<16, true>(x, __uint_as_float(am << 16), am >= 0x7f80u, w, scale);
}

// Four words of codes, one position each, four dims a word: four words of one dim,
// four positions a word.
__device__ __forceinline__ void kv8_transpose4(const uint32_t (&r)[4], uint32_t (&c)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u), b = __builtin_amdgcn_perm(r[3], r[2], 0x05010400u);
    const uint32_t d = __builtin_amdgcn_perm(r[1], r[0], 0x07030602u), e = __builtin_amdgcn_perm(r[3], r[2], 0x07030602u);
    c[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    c[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    c[2] = __builtin_amdgcn_perm(e, d, 0x05040100u);
    c[3] = __builtin_amdgcn_perm(e, d, 0x07060302u);
}

// Where 16-byte unit u of a record's value codes waits in LDS: the threads write
// units 64 bytes apart, which spreads them over the banks.
__device__ __forceinline__ int kv8_unit(int u) { return u ^ (((u >> 4) & 3) << 2) ^ ((u >> 6) & 3); }

// grid (records touched, n_kv, keys | values): half a record per workgroup, sixteen
// lanes a row.  A key's lane holds the two octets of dims that are stored together, a
// unit of 16 bytes, which goes out as it is; values turn in LDS, where a thread
// collects eight positions of four dims and of the four 16 further on, and go out in
// order, a kilobyte a wave.  Bytes of positions outside the call are left as they are:
// a key's unit is one position's, and a group of eight positions' values that is not
// covered goes byte by byte.  Bound by the bytes of the rows and of the cache: 32768
// positions of two heads, 101 MB, in 19.6 us (5.2 TB/s; a large copy's rate is 5.1), 131072
// in 70.5 (5.7).
template <bool VALUES>
__device__ __forceinline__ void kv8_write_record(const WriteArgs& a, uint8_t* s_mem) {
    constexpr int kPad = kHeadDim + 4;
    vmi_u4* s_unit = reinterpret_cast<vmi_u4*>(s_mem);                 // units in order (kv8_unit)
    uint8_t* s_v = s_mem + kHalfRec;                                   // values [positions][kPad]
    const int lane = threadIdx.x & 63, w = at_wave(), g = blockIdx.y, li = lane & 15, t = threadIdx.x;
    const int blk = a.pos0 / kBlk + blockIdx.x;
    const int lo = max(a.pos0 - blk * kBlk, 0), hi = min(a.pos0 + a.n - blk * kBlk, kBlk);  // positions of the record
    uint8_t* rec = a.cache + ((size_t)g * (a.max_len / kBlk) + blk) * kRec;
    // the wave's positions 8 w + 4 i + (lane >> 4); a key lane's dims 64 j + 8 o .. and 32 further on, a value lane's 16 li ..
    const int j = li >> 2, o = li & 3;
    vmi_u4 r[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int kt = min(max(8 * w + 4 * i + (lane >> 4), lo), hi - 1);
        const uint16_t* src = a.src[VALUES] + g * a.head[VALUES] + (int64_t)(kt + blk * kBlk - a.pos0) * a.row[VALUES] +
                              (VALUES ? 16 * li : 64 * j + 8 * o);
        r[i][0] = *reinterpret_cast<const vmi_u4*>(src);
        r[i][1] = *reinterpret_cast<const vmi_u4*>(src + (VALUES ? 8 : 32));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (8 * w + 4 * i >= hi || 8 * w + 4 * i + 4 <= lo) continue;   // wave-uniform: none of these four
        const int kt = 8 * w + 4 * i + (lane >> 4);
        const bool mine = kt >= lo && kt < hi;
        uint32_t c[4];
        float s;
        kv8_row16(r[i][0], r[i][1], c, s);
        if (VALUES) {
#pragma unroll
            for (int e = 0; e < 4; ++e) *reinterpret_cast<uint32_t*>(s_v + kt * kPad + 16 * li + 4 * e) = c[e];
        } else if (mine) {
            *reinterpret_cast<vmi_u4*>(rec + kv8_k_off(kt, 64 * j + 8 * o)) = vmi_u4{c[0], c[1], c[2], c[3]} ^ kKeySign;
        }
        if (mine && li == 0) *reinterpret_cast<float*>(rec + kv8_scale_off(kt, VALUES)) = s;
    }
    if constexpr (!VALUES) return;
    __syncthreads();
    if (t < kBlk * kHeadDim / 64) {
        // positions 8 q .., dims 32 d + 4 e .. and 16 further on
        const int e = t & 3, d = (t >> 2) & 7, q = t >> 5;
        uint32_t out[4][4];   // per dim: positions 0..3, 4..7 of it, then of the one 16 further on
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                uint32_t p[4], c[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    p[i] = *reinterpret_cast<const uint32_t*>(s_v + (8 * q + 4 * y + i) * kPad + 32 * d + 16 * z + 4 * e);
                kv8_transpose4(p, c);
#pragma unroll
                for (int i = 0; i < 4; ++i) out[i][2 * z + y] = c[i];
            }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            s_unit[kv8_unit(d * 64 + q * 16 + 4 * e + i)] = vmi_u4{out[i][0], out[i][1], out[i][2], out[i][3]};
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kHalfRec / 16 / kThreads; ++i) {
        const int u = t + kThreads * i, kt = 8 * ((u >> 4) & 3);
        const vmi_u4 v = s_unit[kv8_unit(u)];
        uint8_t* dst = rec + kHalfRec + 16 * u;
        if (kt >= lo && kt + 8 <= hi) {
            *reinterpret_cast<vmi_u4*>(dst) = v;
        } else {
#pragma unroll
            for (int y = 0; y < 8; ++y)
                if (kt + y >= lo && kt + y < hi) {
                    dst[y] = (uint8_t)(v[y >> 2] >> (8 * (y & 3)));
                    dst[8 + y] = (uint8_t)(v[2 + (y >> 2)] >> (8 * (y & 3)));
                }
        }
    }
}

__global__ __launch_bounds__(kThreads) void k_kv8_write(WriteArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t s_mem[kHalfRec + kBlk * (kHeadDim + 4)];
    if (blockIdx.z)
        kv8_write_record<true>(a, s_mem);
    else
        kv8_write_record<false>(a, s_mem);
}

// -------------------------------------------------------------------- load
struct ReadArgs {
    const uint8_t* cache;
    int max_len, pos0, n;
    void* dst[2];   // keys, values: [n_kv, n, 256], either may be null
};

// grid (records touched, n_kv, keys | values): the half record through LDS (its
// 16-byte units placed so that the reads spread over the banks); a thread takes eight
// dims of four positions (fp32: four of eight), so that rows go out 16 bytes a lane, side
// by side.  Bound by the bytes written: 32768 positions of two heads, 101 MB, in 18 us
// (5.6 TB/s; four dims a lane 22.7).
template <bool F32>
__global__ __launch_bounds__(kThreads) void k_kv8_read(ReadArgs a) {
    __shared__ vmi_u4 s_unit[kHalfRec / 16];
    const int z = blockIdx.z, g = blockIdx.y, blk = a.pos0 / kBlk + blockIdx.x, t = threadIdx.x;
    if (!a.dst[z]) return;
    const uint8_t* rec = a.cache + ((size_t)g * (a.max_len / kBlk) + blk) * kRec;
    constexpr int kDims = F32 ? 4 : 8, kPos = 32 / kDims;
    const int kt = kPos * (t / (kHeadDim / kDims)), d0 = kDims * (t % (kHeadDim / kDims));
    vmi_f4 scale[kPos / 4];
#pragma unroll
    for (int i = 0; i < kPos / 4; ++i) scale[i] = *reinterpret_cast<const vmi_f4*>(rec + kv8_scale_off(kt + 4 * i, z));
    auto place = [&](int u) { return u ^ (z ? (u >> 6) & 7 : (u >> 4) & 15); };
#pragma unroll
    for (int i = 0; i < kHalfRec / 16 / kThreads; ++i) {
        const int u = t + kThreads * i;
        s_unit[place(u)] = *reinterpret_cast<const vmi_u4*>(rec + z * kHalfRec + 16 * u);
    }
    __syncthreads();
    const uint8_t* half = reinterpret_cast<const uint8_t*>(s_unit);
    uint32_t c[kPos][kDims / 4];   // codes + 128 of position kt + i, dims d0 + 4 y ..
    if (z == 0) {
#pragma unroll
        for (int i = 0; i < kPos; ++i)
#pragma unroll
            for (int y = 0; y < kDims / 4; ++y) {
                const int at = kv8_k_off(kt + i, d0 + 4 * y);
                c[i][y] = *reinterpret_cast<const uint32_t*>(half + 16 * place(at >> 4) + (at & 15)) ^ kKeySign;
            }
    } else {
#pragma unroll
        for (int x = 0; x < kPos / 4; ++x)
#pragma unroll
            for (int y = 0; y < kDims / 4; ++y) {
                uint32_t p[4], q[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = kv8_v_off(kt + 4 * x, d0 + 4 * y + j) - kHalfRec;
                    p[j] = *reinterpret_cast<const uint32_t*>(half + 16 * place(at >> 4) + (at & 15));
                }
                kv8_transpose4(p, q);
#pragma unroll
                for (int i = 0; i < 4; ++i) c[4 * x + i][y] = q[i];
            }
    }
    const int lo = max(a.pos0 - blk * kBlk, 0), hi = min(a.pos0 + a.n - blk * kBlk, kBlk);
#pragma unroll
    for (int i = 0; i < kPos; ++i) {
        if (kt + i < lo || kt + i >= hi) continue;
        float x[kDims];
#pragma unroll
        for (int j = 0; j < kDims; ++j)
            x[j] = scale[i >> 2][i & 3] * ((float)((c[i][j >> 2] >> (8 * (j & 3))) & 255u) - 128.0f);
        const size_t at = ((size_t)g * a.n + (blk * kBlk + kt + i - a.pos0)) * kHeadDim + d0;
        if constexpr (F32)
            *reinterpret_cast<vmi_f4*>(static_cast<float*>(a.dst[z]) + at) = vmi_f4{x[0], x[1], x[2], x[3]};
        else
            *reinterpret_cast<vmi_u4*>(static_cast<uint16_t*>(a.dst[z]) + at) =
                vmi_u4{vmi_pack_bf16x2(x[0], x[1]), vmi_pack_bf16x2(x[2], x[3]), vmi_pack_bf16x2(x[4], x[5]),
                       vmi_pack_bf16x2(x[6], x[7])};
    }
}

// Lane l and lane l ^ 32 (l ^ 16): both lanes' values, the lower lane's first.
__device__ __forceinline__ float2 kv8_pair32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float2 kv8_pair16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float kv8_max32(float v) {
    const float2 p = kv8_pair32(v);
    return fmaxf(p.x, p.y);
}
__device__ __forceinline__ float kv8_max16(float v) {
    const float2 p = kv8_pair16(v);
    return fmaxf(p.x, p.y);
}
__device__ __forceinline__ float kv8_sum32(float v) {
    const float2 p = kv8_pair32(v);
    return p.x + p.y;
}
__device__ __forceinline__ float kv8_sum16(float v) {
    const float2 p = kv8_pair16(v);
    return p.x + p.y;
}

// ------------------------------------------------------------------- heads
using vmi::Kv8Heads;

__device__ __forceinline__ int kv8_pos0(int pos0, const int32_t* pos_dev, int span, int max_len) {
    const int p = pos_dev ? *pos_dev : pos0;
    return min(max(p, 0), max_len - span);
}

// (cos, sin) of pos * base^fi, base = theta^(-2/rd), fi < half: the angle in quarter
// turns in double, to the nearest axis, then Taylor's series over an eighth of a turn (to
// x^9 and x^10: within 2^-28).  The general functions took as many instructions as the
// rest of the heads' kernel, which they bound.
__device__ __forceinline__ float2 kv8_rotary_cs(int pos, int fi, int half, double base) {
    double f = 1.0, b = base;
    for (int k = 0; (half - 1) >> k; ++k) {   // wave-uniform
        f = (fi >> k) & 1 ? f * b : f;
        b *= b;
    }
    const double quarters = (double)pos * (f * 0.6366197723675814);   // 2 / pi
    const double axis = rint(quarters);
    const float x = (float)((quarters - axis) * 1.5707963267948966), z = x * x;
    const int n = (int)axis;
    const float sn = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), x);
    const float cs = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.0f);
    const float c = n & 1 ? sn : cs, d = n & 1 ? cs : sn;
    return make_float2(__uint_as_float(__float_as_uint(c) ^ (uint32_t)((n + 1) & 2) << 30),
                       __uint_as_float(__float_as_uint(d) ^ (uint32_t)(n & 2) << 30));
}

// A row in half a wave, dims 8 l .. in lane l of it: its sum, its largest (as bits of a
// magnitude), alike in every lane.
__device__ __forceinline__ float kv8_row_sum(float v) {
    v += __uint_as_float(vmi_dpp_u32<VMI_DPP_XOR1>(__float_as_uint(v)));
    v += __uint_as_float(vmi_dpp_u32<VMI_DPP_XOR2>(__float_as_uint(v)));
    v += __uint_as_float(vmi_dpp_u32<VMI_DPP_HALF_MIRROR>(__float_as_uint(v)));
    v += __uint_as_float(vmi_dpp_u32<VMI_DPP_MIRROR>(__float_as_uint(v)));
    return kv8_sum16(v);
}
__device__ __forceinline__ uint32_t kv8_row_max(uint32_t v) {
    v = max(v, vmi_dpp_u32<VMI_DPP_XOR1>(v));
    v = max(v, vmi_dpp_u32<VMI_DPP_XOR2>(v));
    v = max(v, vmi_dpp_u32<VMI_DPP_HALF_MIRROR>(v));
    v = max(v, vmi_dpp_u32<VMI_DPP_MIRROR>(v));
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max((uint32_t)r[0], (uint32_t)r[1]);
}

// Such a row: RMSNorm times the weight, then the rotary pairs (i, i + rd/2), in fp32.
// srow: 256 floats of the row's own.
__device__ __forceinline__ void kv8_norm_rope(float (&x)[8], const float (&nw)[8], float eps, const float2* cs, int rd,
                                              float* srow) {
    const int l = threadIdx.x & 31, half = rd / 2;
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
    ss = kv8_row_sum(ss);
    // the hardware's reciprocal square root and one Newton step (a sum past fp32 gives 0)
    const float var = fmaf(ss, 1.0f / (float)kHeadDim, eps), r = __builtin_amdgcn_rsqf(var);
    const float inv = var < INFINITY ? fmaf(0.5f * r, fmaf(-var * r, r, 1.0f), r) : r;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (x[j] * inv) * nw[j];
    float pr[8];
    if (rd % 16 == 0) {  // wave-uniform: the partners of a lane's dims are another lane's
        const int src = (8 * l < half ? l + half / 8 : l - half / 8) & 31;
#pragma unroll
        for (int j = 0; j < 8; ++j) pr[j] = __shfl(x[j], src, 32);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j += 4)
            *reinterpret_cast<float4*>(srow + 8 * l + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int d = 8 * l + j;
            pr[j] = srow[d < half ? d + half : d < rd ? d - half : d];
        }
    }
    if (8 * l < rd) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int d = 8 * l + j;
            if (rd % 16 == 0 || d < rd) {
                const float2 c = cs[d < half ? d : d - half];
                x[j] = fmaf(x[j], c.x, (d < half ? -pr[j] : pr[j]) * c.y);
            }
        }
    }
}

constexpr int kHeadTok = 8;  // positions of a workgroup: one value group of a record

// grid (groups of eight positions, heads (q, then k, then v), paths): half a wave takes
// one of the group's tokens of one head, sixteen bytes a lane in and out.  A value
// group's eight positions are collected in LDS and go out together.  Bound by the
// bytes of the projections on a prompt, by latency on a batch.
__global__ __launch_bounds__(kThreads) void k_kv8_heads(Kv8Heads a) {
    __shared__ float2 s_cs[kHeadTok][kHeadDim / 2];
    __shared__ __attribute__((aligned(16))) float s_row[kHeadTok][kHeadDim];
    __shared__ __attribute__((aligned(16))) uint8_t s_v[kHeadDim][kHeadTok];
    const int l = threadIdx.x & 31, row = threadIdx.x >> 5, path = blockIdx.z;
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
    const int kt = min(max(row, lo), hi - 1);
    const bool mine = kt == row;
    const int t = p0 + kt - pos0, tb = (p0 + kt) % kBlk;
    const float* src = a.qkv + ((size_t)path * a.T + t) * stride + col + 8 * l;
    float x[8];
    {
        const vmi_f4 u = *reinterpret_cast<const vmi_f4*>(src), v = *reinterpret_cast<const vmi_f4*>(src + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] = u[j];
            x[4 + j] = v[j];
        }
    }
    if (!is_v) {
        const uint16_t* nwp = is_q ? a.q_norm : a.k_norm;
        float nw[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) nw[j] = vmi_bf16_to_f32(nwp[8 * l + j]);
        const int half = a.rope_dim / 2;
        if (mine)
            for (int f = l; f < half; f += 32) s_cs[row][f] = kv8_rotary_cs(p0 + row, f, half, a.rope_base);
        __syncthreads();
        kv8_norm_rope(x, nw, a.eps, s_cs[kt], a.rope_dim, s_row[row]);
    }
    if (is_q) {
        if (mine)
            *reinterpret_cast<vmi_u4*>(a.q + ((size_t)(path * a.T + t) * a.n_heads + hh) * kHeadDim + 8 * l) =
                vmi_u4{vmi_pack_bf16x2(x[0], x[1]), vmi_pack_bf16x2(x[2], x[3]), vmi_pack_bf16x2(x[4], x[5]),
                       vmi_pack_bf16x2(x[6], x[7])};
        return;
    }
    const int g = is_v ? hh - a.n_heads - a.n_kv : hh - a.n_heads;
    uint32_t am = 0;   // largest magnitude, as bits: infinities and NaN above the finite ones
#pragma unroll
    for (int j = 0; j < 8; ++j) am = max(am, __float_as_uint(x[j]) & 0x7fffffffu);
    am = kv8_row_max(am);
    float s;
    uint32_t c[2];
    kv8_quantise<8, false>(x, __uint_as_float(am), am >= 0x7f800000u, c, s);
    if (!is_v) {
        c[0] ^= kKeySign;
        c[1] ^= kKeySign;
    }
    if (a.tree) {  // plain rows, one record per token
        if (!mine) return;
        uint8_t* side = a.tree + ((size_t)(path * a.n_kv + g) * a.T + t) * kKv8TreeRow;
        *reinterpret_cast<uint2*>(side + (is_v ? kHeadDim : 0) + 8 * l) = make_uint2(c[0], c[1]);
        if (l == 0) *reinterpret_cast<float*>(side + 2 * kHeadDim + (is_v ? 4 : 0)) = s;
        return;
    }
    uint8_t* rec = a.cache + ((size_t)g * (a.max_len / kBlk) + p0 / kBlk) * kRec;
    if (mine && l == 0) *reinterpret_cast<float*>(rec + kv8_scale_off(tb, is_v)) = s;
    if (!is_v) {
        if (mine) *reinterpret_cast<uint2*>(rec + kv8_k_off(tb, 8 * l)) = make_uint2(c[0], c[1]);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s_v[8 * l + j][row] = (uint8_t)(c[j >> 2] >> (8 * (j & 3)));
    __syncthreads();
    // thread d: dim d of the group's eight positions
    const int d = threadIdx.x;
    uint8_t* dst = rec + kv8_v_off(p0 % kBlk, d);
    if (lo == 0 && hi == kHeadTok) {
        *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(s_v[d]);
    } else {
        for (int i = lo; i < hi; ++i) dst[i] = s_v[d][i];
    }
}

// --------------------------------------------------------------- attention
using vmi::Kv8Attn;

// Eight codes + 128 as fp16 subnormals (c + 128) 2^-24, exactly: one byte
// permute per pair.  The matrix instructions take subnormals as they are.
__device__ __forceinline__ vmi_u4 kv8_widen(uint32_t w0, uint32_t w1) {
    vmi_u4 r;
    r[0] = __builtin_amdgcn_perm(0u, w0, 0x0c010c00u);
    r[1] = __builtin_amdgcn_perm(0u, w0, 0x0c030c02u);
    r[2] = __builtin_amdgcn_perm(0u, w1, 0x0c010c00u);
    r[3] = __builtin_amdgcn_perm(0u, w1, 0x0c030c02u);
    return r;
}
// The codes themselves, c 2^-24 (exact).
__device__ __forceinline__ vmi_u4 kv8_signed(const vmi_u4& u) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 off = {(_Float16)(-0x1p-17f), (_Float16)(-0x1p-17f)};
    vmi_u4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, (uint32_t)u[i]) + off);
    return r;
}
__device__ __forceinline__ uint32_t kv8_pack_f16(float a, float b) {  // one conversion of both, to nearest even
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));
}

// Scores are sums of int8 products, exact in int32: a query row is held as 16-bit
// integers of its largest magnitude over 32512, in two signed bytes each, 256 h + l.
// That is half a step of 2^-16 of the largest element, 256 times finer than a key's
// codes, and a key's bytes go to the matrix instruction as they are stored.
constexpr float kQueryTop = 32512.0f;
constexpr float kScoreUnit = 0.09016844005556021f / kQueryTop;  // log2(e) / sqrt(256) over it
struct Kv8Unit {
    float inv, cx;   // integers per unit of the query; powers of two per unit of score (NaN: a row that is not finite)
};
// am: the row's largest magnitude as bf16 bits.  Rows below 2^-100 keep fewer bits.
__device__ __forceinline__ Kv8Unit kv8_query_unit(uint32_t am) {
    const float top = fmaxf(__uint_as_float(am << 16), 0x1p-100f);
    const bool bad = am >= 0x7f80u;
    return {bad ? 0.0f : __fdiv_rn(kQueryTop, top), bad ? __builtin_nanf("") : kScoreUnit * top};
}
// Four elements' bytes (two words of bf16 pairs), h and l.  The sum's low 16 bits are
// 256 h + l + 128.
__device__ __forceinline__ void kv8_digits(uint32_t p0, uint32_t p1, float inv, uint32_t& h, uint32_t& l) {
    constexpr float kMagic = 12582912.0f + 128.0f;
    const uint32_t a = __float_as_uint(fmaf(__uint_as_float(p0 << 16), inv, kMagic));
    const uint32_t b = __float_as_uint(fmaf(__uint_as_float(p0 & 0xffff0000u), inv, kMagic));
    const uint32_t c = __float_as_uint(fmaf(__uint_as_float(p1 << 16), inv, kMagic));
    const uint32_t d = __float_as_uint(fmaf(__uint_as_float(p1 & 0xffff0000u), inv, kMagic));
    const uint32_t u = __builtin_amdgcn_perm(b, a, 0x05010400u), v = __builtin_amdgcn_perm(d, c, 0x05010400u);
    l = __builtin_amdgcn_perm(v, u, 0x05040100u) ^ kKeySign;
    h = __builtin_amdgcn_perm(v, u, 0x07060302u);
}
__device__ __forceinline__ float kv8_score(int h, int l) { return (float)((int)((uint32_t)h << 8) + l); }

constexpr float kPScale = 16384.0f;            // probabilities times value scales, in fp16: at most this
constexpr float kSumUnit = 0x1p24f / kPScale;  // of their products' sums, codes in units of 2^-24
constexpr float kMinRef = 1e-30f;

// 16 MS query rows of a wave: lane (nl, q4) belongs to row 16 m + nl.
template <int MS>
struct Kv8Rows {
    vmi_u4 q[MS][8];   // h (2 j) and l (2 j + 1) of dims 64 j + 8 q4 .. and 32 further on
    float cx[MS];      // Kv8Unit
};

// The wave's query rows, sixteen from each r0 of R (rows behind the last repeat it).
template <int MS>
__device__ __forceinline__ void kv8_load_rows(const Kv8Attn& a, const uint16_t* q, int g, const int (&r0)[MS], int R,
                                              Kv8Rows<MS>& o) {
    const int lane = threadIdx.x & 63, nl = lane & 15, q4 = lane >> 4, G = a.n_heads / a.n_kv;
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        const int row = min(r0[m] + nl, R - 1), t = row / G, h = g * G + row % G;
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
        const Kv8Unit f = kv8_query_unit(am);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            vmi_u4 h, l;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const vmi_u4& u = o.q[m][2 * j + i / 2];
                uint32_t x, y;
                kv8_digits(u[2 * (i % 2)], u[2 * (i % 2) + 1], f.inv, x, y);
                h[i] = x;
                l[i] = y;
            }
            o.q[m][2 * j] = h;
            o.q[m][2 * j + 1] = l;
        }
        o.cx[m] = f.cx;
    }
}

// A record in a wave's registers: lane (nl, q4) holds the keys 8 (nl>>2) + 4 a +
// (nl&3) and the values of positions 8 q4 .., as they are stored.
struct Kv8Rec {
    vmi_u4 k[8], v[8];   // key operands 2 j, 2 j + 1 of tile a at 4 a + j; value operands 2 j, 2 j + 1 at j
    vmi_f4 ks[2], vs[2]; // scales of positions 8 q4 ..
};

// Record b of a kv head, or nothing where there is none (zeros, and no memory
// read): the loads take no branch, so that every wait counts only what it needs.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t kv8_rsrc(const uint8_t* head, int b, bool present) {
    return vmi_rsrc(head + (size_t)b * kRec, present ? kRec : 0);
}
// ONCE: one workgroup alone reads the record (nontemporal); else another row tile's
// reads it too.
template <bool ONCE>
__device__ __forceinline__ vmi_u4 kv8_bload(__amdgpu_buffer_rsrc_t rs, int at, int base) {
    return ONCE ? vmi_bload_b128_nt(rs, (uint32_t)at, base) : vmi_bload_b128(rs, (uint32_t)at, base);
}
template <bool ONCE>
__device__ __forceinline__ void kv8_load_keys(Kv8Rec& r, __amdgpu_buffer_rsrc_t rs) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < 8; ++j) r.k[j] = kv8_bload<ONCE>(rs, 16 * lane, 1024 * j);
#pragma unroll
    for (int j = 0; j < 2; ++j)
        r.ks[j] = __builtin_bit_cast(vmi_f4, kv8_bload<ONCE>(rs, 2 * kHalfRec + 32 * (lane >> 4) + 16 * j, 0));
}
template <bool ONCE>
__device__ __forceinline__ void kv8_load_value_scales(Kv8Rec& r, __amdgpu_buffer_rsrc_t rs) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < 2; ++j)
        r.vs[j] = __builtin_bit_cast(vmi_f4, kv8_bload<ONCE>(rs, 2 * kHalfRec + 128 + 32 * (lane >> 4) + 16 * j, 0));
}
template <bool ONCE>
__device__ __forceinline__ void kv8_load_value(Kv8Rec& r, __amdgpu_buffer_rsrc_t rs, int j) {
    r.v[j] = kv8_bload<ONCE>(rs, 16 * (threadIdx.x & 63), kHalfRec + 1024 * j);
}

// Position kt of the record from a tree token's row.
__device__ __forceinline__ void kv8_insert(Kv8Rec& r, const uint8_t* row, int kt) {
    const int lane = threadIdx.x & 63, nl = lane & 15, q4 = lane >> 4, e = kt & 7;
    const bool mine = nl == 4 * (kt >> 3) + (kt & 3), at = q4 == kt >> 3;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint2 lo = *reinterpret_cast<const uint2*>(row + 64 * j + 8 * q4);
        const uint2 hi = *reinterpret_cast<const uint2*>(row + 64 * j + 32 + 8 * q4);
        const vmi_u4 u = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
        for (int a = 0; a < 2; ++a)
            if (mine && ((kt >> 2) & 1) == a) r.k[4 * a + j] = u;
    }
    const float2 sc = *reinterpret_cast<const float2*>(row + 2 * kHeadDim);
    const uint32_t keep = ~(0xffu << (8 * (e & 3)));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t lo = (uint32_t)row[kHeadDim + 32 * j + nl] << (8 * (e & 3));
        const uint32_t hi = (uint32_t)row[kHeadDim + 32 * j + 16 + nl] << (8 * (e & 3));
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (at && (e >> 2) == i) {
                r.v[j][i] = (r.v[j][i] & keep) | lo;
                r.v[j][2 + i] = (r.v[j][2 + i] & keep) | hi;
            }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (at && i == e) {
            r.ks[i >> 2][i & 3] = sc.x;
            r.vs[i >> 2][i & 3] = sc.y;
        }
}

// Running softmax of a wave's 16 MS rows.  o is in units of s kSumUnit.
template <int MS>
struct Kv8Sums {
    vmi_f4 o[MS][16];  // dims 16 dt + 4 q4 + r of row 16 m + nl
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

// One record's 32 keys, the first at position p0, against the rows q (kv8_digits,
// in LDS).  S^T = K Q^T: a lane holds the scores of keys 8 q4 + e of its
// row, which are, as probabilities, already the B operand of O^T = V^T P^T.  A
// key's scale enters its score, a value's its probability; the product goes to fp16
// (11 bits) relative to the row's largest value scale so far, and whatever raises
// that or the running maximum rescales the sums.  The codes themselves are multiplied: codes +
// 128, as they are widened, with the 128 taken off at the end, would save half of the
// widening's instructions (1 % of four tokens at 32,764) and leave 2^-24 of a row's
// scale in every dim, also where its code is zero.  mask (wave-uniform): the record
// reaches past the visible positions of some row; masked scores count as minus
// infinity and masked scales as zero, so that nothing stored behind a row's last
// position reaches it.  The next record's keys are asked for once these are used,
// each of its value operands once this record's is.
template <int MS, bool ONCE>
__device__ __forceinline__ void kv8_step(Kv8Rec& rec, const vmi_u4* q, const float (&cx)[MS], const int (&last)[MS], int p0,
                                         bool mask, __amdgpu_buffer_rsrc_t next, Kv8Sums<MS>& S) {
    const int lane = threadIdx.x & 63, q4 = lane >> 4;
    vmi_i4 s[MS][2][2];   // [tile of 16 keys][h, l]
#pragma unroll
    for (int m = 0; m < MS; ++m) s[m][0][0] = s[m][0][1] = s[m][1][0] = s[m][1][1] = vmi_i4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int m = 0; m < MS; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const vmi_u4 qr = q[(8 * m + 2 * j + i) * 64 + lane];
#pragma unroll
                for (int a = 0; a < 2; ++a) s[m][a][i] = vmi_mfma_i8(rec.k[4 * a + j], qr, s[m][a][i]);
            }
    float x[MS][8];
#pragma unroll
    for (int m = 0; m < MS; ++m)
#pragma unroll
        for (int e = 0; e < 8; ++e)
            x[m][e] = kv8_score(s[m][e >> 2][0][e & 3], s[m][e >> 2][1][e & 3]) * (rec.ks[e >> 2][e & 3] * cx[m]);
    kv8_load_keys<ONCE>(rec, next);
    vmi_u4 pb[MS];
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = rec.vs[e >> 2][e & 3];
        if (mask) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool seen = p0 + 8 * q4 + e <= last[m];
                x[m][e] = seen ? x[m][e] : -INFINITY;
                v[e] = seen ? v[e] : 0.0f;
            }
        }
        float nm = S.m[m], ns = S.s[m];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            nm = fmaxf(nm, x[m][e]);
            ns = fmaxf(ns, v[e]);
        }
        nm = kv8_max32(kv8_max16(nm));
        ns = kv8_max32(kv8_max16(ns));
        if (__any(nm > S.m[m] || ns > S.s[m])) {
            const float f = __builtin_amdgcn_exp2f(S.m[m] - nm);
            S.l[m] *= f;
            const float fo = ns > S.s[m] ? f * (S.s[m] * __builtin_amdgcn_rcpf(ns)) : f;
#pragma unroll
            for (int d = 0; d < 16; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) S.o[m][d][r] *= fo;
            S.m[m] = nm;
            S.s[m] = ns;
        }
        const float inv = kPScale * __builtin_amdgcn_rcpf(ns);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[m][e] = __builtin_amdgcn_exp2f(x[m][e] - nm);
            S.l[m] += x[m][e];
            x[m][e] *= v[e] * inv;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) pb[m][i] = kv8_pack_f16(x[m][2 * i], x[m][2 * i + 1]);
    }
    kv8_load_value_scales<ONCE>(rec, next);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const vmi_u4 u = rec.v[j];
        const vmi_u4 v0 = kv8_signed(kv8_widen(u[0], u[1])), v1 = kv8_signed(kv8_widen(u[2], u[3]));
#pragma unroll
        for (int m = 0; m < MS; ++m) S.o[m][2 * j] = vmi_mfma_f16(v0, pb[m], S.o[m][2 * j]);
#pragma unroll
        for (int m = 0; m < MS; ++m) S.o[m][2 * j + 1] = vmi_mfma_f16(v1, pb[m], S.o[m][2 * j + 1]);
        kv8_load_value<ONCE>(rec, next, j);
    }
}

// Waits for the wave's own LDS operations.
__device__ __forceinline__ void kv8_lds_wait() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt 0
    asm volatile("" ::: "memory");
}

// Parts go out nontemporal: left in the XCDs' L2 they would be written back at the
// kernel's end, before the merge can start (four tokens at 4000: 14.1 -> 11.9 us).
__device__ __forceinline__ void kv8_store_part(__amdgpu_buffer_rsrc_t ro, int row, int d, const vmi_f4& y) {
    vmi_bstore_b128_nt(__builtin_bit_cast(vmi_u4, y), ro, (uint32_t)(row * kHeadDim + d) * 4u, 0);
}

constexpr int kSplitWaves = 4, kSplitThreads = 64 * kSplitWaves;

// grid (S, n_kv, paths * row tiles): record b of a kv head belongs to wave
// (b / S) % 4 of workgroup b % S, whatever the length, the batch and the capacity,
// so that a row's sums do not depend on them, a short cache still spreads over the
// device, and a long one keeps every CU reading.  The workgroup forms the rows'
// operands in LDS; a wave then works through its records in registers, up to two
// waves a SIMD (one alone issues an instruction every six cycles), without a barrier
// until the end, where the waves join in LDS and the workgroup writes one part:
// maximum, sum and unnormalised output of each row, in fp32.  Bound by the bytes of
// the cache from some ten thousand positions on (one token of 16 heads on 2 at
// 262,143: 47 us, 5.8 TB/s), below by the latency of a record and of the two launches
// (at 1000: 7.7 us; four tokens at 32,764, two records a wave: 18.2).
template <int MS, bool ONCE>
__global__ __launch_bounds__(kSplitThreads, MS == 1 ? 2 : 1) void k_kv8_split(Kv8Attn a) {
    __shared__ __attribute__((aligned(16))) float s_o[kSplitWaves * 16 * kHeadDim];   // one row group of each wave
    __shared__ vmi_u4 s_q[MS * 8 * 64];
    __shared__ float s_cx[16 * MS], s_ml[kSplitWaves][16 * MS][2];
    const int lane = threadIdx.x & 63, w = at_wave(), nl = lane & 15, q4 = lane >> 4;
    const int wg = blockIdx.x, S = gridDim.x, g = blockIdx.y, path = blockIdx.z % a.paths, T = a.span;
    const int rz = 16 * MS * (blockIdx.z / a.paths);   // the workgroup's first row
    const int pos0 = kv8_pos0(a.pos0, a.pos_dev, T, a.max_len);
    if (a.pos_dev && a.status && wg == 0 && g == 0 && blockIdx.z == 0 && threadIdx.x == 0 && *a.pos_dev != pos0)
        atomicOr(a.status, VMI_STATUS_BAD_POS);
    const int nblk = (pos0 + T + kBlk - 1) / kBlk;
    if (wg >= nblk) return;   // whole workgroup
    const int G = a.n_heads / a.n_kv, R = T * G, step = kSplitWaves * S, first = wg + S * w;
    const uint8_t* head = a.cache + (size_t)g * (a.max_len / kBlk) * kRec;
    // rows 2 NQ w .. of the group, 32 lanes each, then the wave's first record
    constexpr int NQ = 16 * MS / (2 * kSplitWaves);
    vmi_u4 qv[NQ];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        const int row = min(rz + 2 * (NQ * w + i) + (lane >> 5), R - 1), t = row / G;
        qv[i] = *reinterpret_cast<const vmi_u4*>(a.q + ((size_t)(path * T + t) * a.n_heads + g * G + row % G) * kHeadDim +
                                                 8 * (lane & 31));
    }
    asm volatile("" ::: "memory");
    Kv8Rec rec;
    const __amdgpu_buffer_rsrc_t rs0 = kv8_rsrc(head, first, first < nblk);
    kv8_load_keys<ONCE>(rec, rs0);
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        uint32_t am = 0;   // largest magnitude, as bf16 bits
#pragma unroll
        for (int e = 0; e < 4; ++e) am = max(am, max(qv[i][e] & 0x7fffu, (qv[i][e] >> 16) & 0x7fffu));
        am = max(am, vmi_dpp_u32<VMI_DPP_XOR1>(am));
        am = max(am, vmi_dpp_u32<VMI_DPP_XOR2>(am));
        am = max(am, vmi_dpp_u32<VMI_DPP_HALF_MIRROR>(am));
        am = max(am, vmi_dpp_u32<VMI_DPP_MIRROR>(am));
        {
            const auto pr = __builtin_amdgcn_permlane16_swap(am, am, false, false);
            am = max((uint32_t)pr[0], (uint32_t)pr[1]);
        }
        const Kv8Unit f = kv8_query_unit(am);
        uint32_t h[2], l[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) kv8_digits(qv[i][2 * e], qv[i][2 * e + 1], f.inv, h[e], l[e]);
        const int r = 2 * (NQ * w + i) + (lane >> 5), d8 = lane & 31;   // row of the group, dims 8 d8 ..
        uint2* at = reinterpret_cast<uint2*>(s_q + (8 * (r >> 4) + 2 * (d8 >> 3)) * 64 + (d8 & 3) * 16 + (r & 15)) +
                    ((d8 >> 2) & 1);
        at[0] = make_uint2(h[0], h[1]);
        at[2 * 64] = make_uint2(l[0], l[1]);
        if (d8 == 0) s_cx[r] = f.cx;
    }
    asm volatile("" ::: "memory");   // the values behind the forming: a full memory queue would hold it up
    kv8_load_value_scales<ONCE>(rec, rs0);
#pragma unroll
    for (int j = 0; j < 8; ++j) kv8_load_value<ONCE>(rec, rs0, j);
    kv8_lds_wait();
    __builtin_amdgcn_s_barrier();   // (not __syncthreads, which would wait for the records too)
    asm volatile("" ::: "memory");
    float cx[MS];
    int last[MS];
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        cx[m] = s_cx[16 * m + nl];
        last[m] = pos0 + min(rz + 16 * m + nl, R - 1) / G;
    }
    Kv8Sums<MS> Y;
    Y.clear();
#pragma unroll 1
    for (int b = first; b < nblk; b += step) {
        asm volatile("" ::: "memory");   // the rows' operands stay in LDS: they would take the records' registers
        if (a.tree && kBlk * b + kBlk > pos0) {
            // a path's own tokens in place of what the cache holds there
            for (int t = max(kBlk * b - pos0, 0); t < min(T, kBlk * b + kBlk - pos0); ++t)
                kv8_insert(rec, a.tree + ((size_t)(path * a.n_kv + g) * T + t) * kKv8TreeRow, pos0 + t - kBlk * b);
        }
        kv8_step<MS, ONCE>(rec, s_q, cx, last, kBlk * b, kBlk * b + kBlk - 1 > pos0, kv8_rsrc(head, b + step, b + step < nblk), Y);
    }
    const size_t part = ((size_t)(g * S + wg) * a.paths + path) * a.rp;
    const __amdgpu_buffer_rsrc_t ro = vmi_rsrc(a.part_o + part * kHeadDim, (uint32_t)R * kHeadDim * 4);
    float l[MS];
#pragma unroll
    for (int m = 0; m < MS; ++m) l[m] = kv8_sum32(kv8_sum16(Y.l[m]));
    const int active = min(kSplitWaves, (nblk - wg + S - 1) / S);   // waves that had a record
    if (active == 1) {   // the first one's sums are the part
        if (w) return;
#pragma unroll
        for (int m = 0; m < MS; ++m) {
            const int row = rz + 16 * m + nl;
            if (row >= R) continue;
            const float u = Y.s[m] * kSumUnit;
#pragma unroll
            for (int d = 0; d < 16; ++d)
                kv8_store_part(ro, row, 16 * d + 4 * q4,
                               vmi_f4{Y.o[m][d][0] * u, Y.o[m][d][1] * u, Y.o[m][d][2] * u, Y.o[m][d][3] * u});
            if (q4 == 0) *reinterpret_cast<float2*>(a.part_ml + (part + row) * 2) = make_float2(Y.m[m], l[m]);
        }
        return;
    }
    // the waves in order: each brings its sums to the workgroup's maximum, a thread adds four dims of
    // four rows
#pragma unroll
    for (int m = 0; m < MS; ++m)
        if (q4 == 0) {
            s_ml[w][16 * m + nl][0] = Y.m[m];
            s_ml[w][16 * m + nl][1] = l[m];
        }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        if (m) __syncthreads();   // the group before is read
        float M = s_ml[0][16 * m + nl][0];
#pragma unroll
        for (int v = 1; v < kSplitWaves; ++v) M = fmaxf(M, s_ml[v][16 * m + nl][0]);
        if (w < active) {
            const float u = Y.s[m] * kSumUnit * __builtin_amdgcn_exp2f(Y.m[m] - M);
#pragma unroll
            for (int d = 0; d < 16; ++d)
                *reinterpret_cast<vmi_f4*>(s_o + (w * 16 + nl) * kHeadDim + 4 * ((4 * d + q4) ^ nl)) =
                    vmi_f4{Y.o[m][d][0] * u, Y.o[m][d][1] * u, Y.o[m][d][2] * u, Y.o[m][d][3] * u};
        }
        if (w == 0 && q4 == 0 && rz + 16 * m + nl < R) {
            float sum = 0.0f;
#pragma unroll
            for (int v = 0; v < kSplitWaves; ++v)
                sum = fmaf(s_ml[v][16 * m + nl][1], __builtin_amdgcn_exp2f(s_ml[v][16 * m + nl][0] - M), sum);
            *reinterpret_cast<float2*>(a.part_ml + (part + rz + 16 * m + nl) * 2) = make_float2(M, sum);
        }
        __syncthreads();
        vmi_f4 y[16 / kSplitWaves];
#pragma unroll
        for (int i = 0; i < 16 / kSplitWaves; ++i) {
            const int r = w + kSplitWaves * i;
            y[i] = *reinterpret_cast<const vmi_f4*>(s_o + r * kHeadDim + 4 * (lane ^ r));
        }
#pragma unroll
        for (int v = 1; v < kSplitWaves; ++v) {
            if (v >= active) break;
#pragma unroll
            for (int i = 0; i < 16 / kSplitWaves; ++i) {
                const int r = w + kSplitWaves * i;
                const vmi_f4 z = *reinterpret_cast<const vmi_f4*>(s_o + (v * 16 + r) * kHeadDim + 4 * (lane ^ r));
#pragma unroll
                for (int e = 0; e < 4; ++e) y[i][e] += z[e];
            }
        }
#pragma unroll
        for (int i = 0; i < 16 / kSplitWaves; ++i) {
            const int row = rz + 16 * m + w + kSplitWaves * i;
            if (row < R) kv8_store_part(ro, row, 4 * lane, y[i]);
        }
    }
}

// Four outputs y / l, times sigmoid(gate): reciprocals and exp2 of the hardware,
// within 2^-21 of the exact ones.
__device__ __forceinline__ uint2 kv8_gated(const vmi_f4& y, float inv_l, const float* gate) {
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = y[e] * inv_l;
    if (gate) {
        const vmi_f4 z = *reinterpret_cast<const vmi_f4*>(gate);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            o[e] *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z[e] * -1.44269504088896341f));
    }
    return make_uint2(vmi_pack_bf16x2(o[0], o[1]), vmi_pack_bf16x2(o[2], o[3]));
}

// k_kv8_split's parts, many of few rows.  grid (rows of all heads, 4): a quarter of a
// row's dims per workgroup.  Part s is added by slot s % 16 in increasing s, the
// sixteen slots in a fixed order.  Every row sees position 0, so its sum is positive
// (or NaN, which it hands on).
constexpr int kMaxParts = 256;
__global__ __launch_bounds__(kThreads) void k_kv8_merge(Kv8Attn a, int parts) {
    __shared__ float s_f[kMaxParts], s_red[2][kWaves];
    __shared__ vmi_f4 s_num[kWaves][16];
    const int tid = threadIdx.x, lane = tid & 63, w = at_wave();
    const int t = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads, G = a.n_heads / a.n_kv, g = h / G;
    const int path = t / a.span, row = (t - path * a.span) * G + h % G;
    const int nblk = (kv8_pos0(a.pos0, a.pos_dev, a.span, a.max_len) + a.span + kBlk - 1) / kBlk;
    const int n = min(parts, nblk);   // the workgroups that had a record
    const size_t at = ((size_t)(g * parts) * a.paths + path) * a.rp + row, inc = (size_t)a.paths * a.rp;
    const int slot = tid >> 4, d0 = 64 * blockIdx.y + 4 * (tid & 15);
    const float* po = a.part_o + at * kHeadDim + d0;
    // every part's maximum and sum, and the first eight of this slot's outputs
    float2 ml = make_float2(-3.402823466e38f, 0.0f);
    if (tid < n) ml = *reinterpret_cast<const float2*>(a.part_ml + (at + tid * inc) * 2);
    constexpr int kAhead = 8;
    vmi_f4 z[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        const int s = slot + 16 * i;
        z[i] = vmi_f4{0.f, 0.f, 0.f, 0.f};
        if (s < n) z[i] = *reinterpret_cast<const vmi_f4*>(po + s * inc * kHeadDim);
    }
    const float* gp = a.gate ? a.gate + t * a.gate_tok + h * a.gate_head + d0 : nullptr;
    const float wm = vmi_wave_max(ml.x);
    if (lane == 0) s_red[0][w] = wm;
    __syncthreads();
    const float M = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
    const float f = __builtin_amdgcn_exp2f(ml.x - M);
    s_f[tid] = f;
    const float wl = vmi_wave_sum_canon(ml.y * f);
    if (lane == 0) s_red[1][w] = wl;
    __syncthreads();
    const float l = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
    vmi_f4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = fmaf(z[i][e], s_f[slot + 16 * i], y[e]);
    for (int s = slot + 16 * kAhead; s < n; s += 16) {
        const vmi_f4 v = *reinterpret_cast<const vmi_f4*>(po + s * inc * kHeadDim);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = fmaf(v[e], s_f[s], y[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = kv8_sum32(kv8_sum16(y[e]));
    if (lane < 16) s_num[w][lane] = y;
    __syncthreads();
    if (tid >= 16) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (s_num[0][tid][e] + s_num[1][tid][e]) + (s_num[2][tid][e] + s_num[3][tid][e]);
    *reinterpret_cast<uint2*>(a.o + ((size_t)t * a.n_heads + h) * kHeadDim + d0) = kv8_gated(y, __fdiv_rn(1.0f, l), gp);
}

constexpr int kFlashWaves = 8, kFlashThreads = 64 * kFlashWaves, kFlashM = 2, kTileRows = 16 * kFlashWaves;

// Records that a tile of 128 rows of R sees.
__device__ __forceinline__ int kv8_tile_records(int pos0, int tile, int R, int G) {
    return (pos0 + (min((tile + 1) * kTileRows, R) - 1) / G) / kBlk + 1;
}

// The flash kernels' parts, few of many rows: a wave per row, four dims a lane, the parts
// in order.  A part may hold nothing of a row (its maximum is then the lowest).  With
// a.run k_kv8_flash_short's, as many as a row's tile has; rows that have one are out
// already.
__global__ __launch_bounds__(kThreads) void k_kv8_merge_rows(Kv8Attn a, int parts) {
    const int lane = threadIdx.x & 63, r = blockIdx.x * kWaves + at_wave();
    const int t = r / a.n_heads, h = r % a.n_heads, G = a.n_heads / a.n_kv, g = h / G;
    if (t >= a.span) return;
    const int row = t * G + h % G;
    int n = parts;
    if (a.run) {
        const int pos0 = kv8_pos0(a.pos0, a.pos_dev, a.span, a.max_len);
        n = (kv8_tile_records(pos0, row / kTileRows, a.span * G, G) + a.run - 1) / a.run;
        if (n == 1) return;
    }
    const size_t at = (size_t)g * parts * a.rp + row;
    float M = -3.402823466e38f, l = 0.0f;
    for (int s = 0; s < n; ++s) M = fmaxf(M, a.part_ml[(at + (size_t)s * a.rp) * 2]);
    vmi_f4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
        const size_t p = at + (size_t)s * a.rp;
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + p * 2);
        const vmi_f4 z = *reinterpret_cast<const vmi_f4*>(a.part_o + p * kHeadDim + 4 * lane);
        const float f = __builtin_amdgcn_exp2f(ml.x - M);
        l = fmaf(ml.y, f, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = fmaf(z[e], f, y[e]);
    }
    const float* gate = a.gate ? a.gate + t * a.gate_tok + h * a.gate_head + 4 * lane : nullptr;
    *reinterpret_cast<uint2*>(a.o + ((size_t)t * a.n_heads + h) * kHeadDim + 4 * lane) = kv8_gated(y, __fdiv_rn(1.0f, l), gate);
}

// Codes of a value record as fp16 integers, exactly (0x6400 is 1024 with a
// mantissa step of 1), times their positions' factors f.
__device__ __forceinline__ vmi_u4 kv8_scaled(uint32_t w0, uint32_t w1, const vmi_u4& f) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const uint32_t c[4] = {__builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u),
                           __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u)};
    vmi_u4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r[i] = __builtin_bit_cast(uint32_t, (__builtin_bit_cast(h2, c[i]) + off) * __builtin_bit_cast(h2, (uint32_t)f[i]));
    return r;
}

// The larger of three, of results of arithmetic (fmaxf would quiet each first).
__device__ __forceinline__ float kv8_max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// Two probabilities as they are multiplied, in fp16, added to s in fp32.
__device__ __forceinline__ float kv8_sum2(uint32_t p, float s) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, p), h2{(_Float16)1.0f, (_Float16)1.0f}, s, false);
}

// Key scales are held times 2^-18, so that a score stays finite before its row's
// factor.  Value operands are fp16: codes times their scale over 2^(E - kValueBits),
// 2^E the power of two above the largest value scale so far, E at least kMinExp: integers
// times factors of up to 2^kValueBits (eleven bits; a scale below 2^-22 of the largest
// keeps 2^-33 of the largest value).  Probabilities go to fp16 times 2^kProbBits: a
// row's reference lags its largest score by up to 2^kLazyMax.  A record that some row
// of its workgroup does not see to its end has no E that is every row's: its value
// operands are the codes times 2^kValueBits, which is exact, and a position's scale, over
// the 2^E of the scales that the row itself has seen, enters the row's probability, zero
// where the row does not see the position.  (With the record's own E there, a later token's row
// 2^22 times larger took bits from the tokens before it, one 2^34 times larger all.)
// Costs little: 64 tokens from 0, every record such a one, 13.2 -> 13.6 us, 777 34.3 -> 34.5.
constexpr float kKeyUnit = 0x1p-18f;
constexpr int kValueBits = 8, kMinExp = -100, kProbBits = 8;
constexpr float kLazyMax = 6.0f;

// The lane, computed where it is used: a register that a loop need not keep.
__device__ __forceinline__ int kv8_lane() {
    int l = __builtin_amdgcn_mbcnt_lo(~0u, 0u);
    l = __builtin_amdgcn_mbcnt_hi(~0u, l);
    asm volatile("" : "+v"(l));
    return l;
}

// Row `row` of a flash kernel's sums: o times u, maximum and sum, out or as part z.
__device__ __forceinline__ void kv8_finish_rows(const Kv8Attn& a, const vmi_f4 (&o)[16], float top, float sum, float u,
                                                int row, int R, bool out) {
    const int q4 = kv8_lane() >> 4, g = blockIdx.y, G = a.n_heads / a.n_kv, P = gridDim.z;
    if (row >= R) return;
    const int t = row / G, h = g * G + row % G;
    if (!out) {
        const size_t at = (size_t)(g * P + blockIdx.z) * a.rp + row;
#pragma unroll
        for (int d = 0; d < 16; ++d)
            *reinterpret_cast<vmi_f4*>(a.part_o + at * kHeadDim + 16 * d + 4 * q4) =
                vmi_f4{o[d][0] * u, o[d][1] * u, o[d][2] * u, o[d][3] * u};
        if (q4 == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(top, sum);
    } else {
        const float inv = __fdiv_rn(1.0f, sum) * u;
        const float* gate = a.gate ? a.gate + t * a.gate_tok + h * a.gate_head + 4 * q4 : nullptr;
        uint16_t* dst = a.o + ((size_t)t * a.n_heads + h) * kHeadDim + 4 * q4;
#pragma unroll
        for (int d = 0; d < 16; ++d)
            *reinterpret_cast<uint2*>(dst + 16 * d) = kv8_gated(o[d], inv, gate ? gate + 16 * d : nullptr);
    }
}

// The records that every row of a tile of 128 sees to their ends.
__device__ __forceinline__ int kv8_tile_seen(int pos0, int tile, int R, int G) {
    return (pos0 + min(tile * kTileRows, R - 1) / G + 1) / kBlk;
}

// A row's step over a record that it may not see to its end: scores x (before the
// row's factor cx) of the lane's eight keys, of which those up to `seen` are visible, and
// their positions' value scales.  Brings the row's reference top and its exponent ref up,
// the sums o and l with them, and gives the probabilities times their scales, as they
// are multiplied: below 2^(kProbBits + kLazyMax).
__device__ __forceinline__ vmi_u4 kv8_masked_weights(float (&x)[8], const vmi_f4 (&vs)[2], int seen, float cx, float& top,
                                                     int& ref, float& l, vmi_f4 (&o)[16]) {
    float v[8], big = -INFINITY, vm = 0.0f;
#pragma unroll
    for (int y = 0; y < 8; ++y) {
        x[y] = y > seen ? -INFINITY : x[y];
        v[y] = y > seen ? 0.0f : vs[y >> 2][y & 3];
        big = fmaxf(big, x[y]);
        vm = fmaxf(vm, v[y]);
    }
    constexpr float kRaise = kLazyMax + kProbBits;
    if (__any(fmaf(big, cx, -top) > kRaise || (int)(__float_as_uint(vm) >> 23) - 126 > ref)) {
        // each row by its own scores and scales: another row's change nothing of it
        big = kv8_max32(kv8_max16(big));
        const float nt = fmaf(big, cx, -top) > kRaise ? fmaf(big, cx, -(float)kProbBits) : top;
        const int e = max(ref, (int)(__float_as_uint(kv8_max32(kv8_max16(vm))) >> 23) - 126);
        const float f = __builtin_amdgcn_exp2f(top - nt), fo = ldexpf(f, ref - e);
        l *= f;
#pragma unroll
        for (int d = 0; d < 16; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[d][r] *= fo;
        top = nt;
        ref = e;
    }
#pragma unroll
    for (int y = 0; y < 8; ++y) {
        x[y] = __builtin_amdgcn_exp2f(fmaf(x[y], cx, -top));
        l += x[y];
        x[y] *= ldexpf(v[y], -ref);
    }
    vmi_u4 pb;
#pragma unroll
    for (int j = 0; j < 4; ++j) pb[j] = kv8_pack_f16(x[2 * j], x[2 * j + 1]);
    return pb;
}

// grid (pairs of tiles of 128 rows, n_kv, key parts): eight waves share each record, each
// with 16 rows of a tile and 16 of the tile as far from the other end, so that every
// workgroup sees as many keys: the records that both see are taken with 32 rows a wave
// (every operand read from LDS used twice), the rest with 16.  Records come by DMA.
// Keys go to the matrix instructions as they are stored; values are turned into fp16 in
// LDS, an eighth by each wave (in every wave that would cost as much VALU time as the
// softmax), and the scales are prepared by one.  A position whose value scale is not
// finite gets zeros for its value and a NaN for its key's scale: the rows that see it
// end as NaN by their scores, those before it keep theirs.  The sums are rescaled only
// when a score passes its row's reference by 2^kLazyMax or E rises, so that a step has
// no reduction over lanes.
//
// A SIMD's two waves, w and w + 4, are kept half a step apart: while one feeds the
// matrix unit (values of record k - 1, keys of record k), the other is in its softmax;
// a barrier ends each phase.  Waves 0-3 multiply record k in phase 2 k, waves 4-7 in
// phase 2 k + 1.  Record k + 1 and the scales of k + 2 are asked for in phase 2 k and have
// come at the end of 2 k + 1; wave 0 prepares the scales of k + 1 in 2 k (three slots: waves
// 4-7 use those of k - 1 in it); values of k + 1 are turned in 2 k + 2 (by waves 4-7) and
// 2 k + 3 (by waves 0-3).  What is written in a phase was last read in the one before.
// Part z of P takes an equal run of the tile's records; with P > 1 the parts are written
// as k_kv8_split's are.
//
// 4096 tokens behind 8192, 16 heads on 2: 619 to 645 us by the inputs, 1.07 to 1.11 PFLOP/s (a
// large bf16 matrix product reaches 1.23); with every wave in step 915, with the tiles
// unpaired 713; with the mask's branch in every record 626 to 652.  A phase takes some
// 1850 cycles, its 64 matrix instructions 1024 of them: what is left is a single wave's
// instruction issue and the latency of its first LDS reads.  256 registers a lane are
// full; deeper operand prefetch spills.
__global__ __launch_bounds__(kFlashThreads, 2) void k_kv8_flash(Kv8Attn a) {
    __shared__ __attribute__((aligned(16))) uint8_t s_rec[2][2 * kHalfRec];   // keys and values, as stored
    __shared__ float s_scale[2][2 * kBlk];
    __shared__ vmi_u4 s_f16[2][16 * 64];             // values [dt], 64 lanes each
    __shared__ __attribute__((aligned(16))) float s_ks[3][kBlk], s_vs[3][kBlk];
    __shared__ __attribute__((aligned(16))) _Float16 s_vf[3][kBlk];
    __shared__ int s_exp[3];
    constexpr int M = kFlashM, kSchedRead = 0x100, kSchedMfma = 0x8;
    const int w = at_wave(), late = w >> 2;
    const int g = blockIdx.y, G = a.n_heads / a.n_kv, R = a.span * G, P = gridDim.z, z = blockIdx.z;
    const int pos0 = kv8_pos0(a.pos0, a.pos_dev, a.span, a.max_len);
    if (a.pos_dev && a.status && blockIdx.x == 0 && g == 0 && z == 0 && threadIdx.x == 0 && *a.pos_dev != pos0)
        atomicOr(a.status, VMI_STATUS_BAD_POS);
    // tile x and, of the other end, its partner: the first sees the fewest keys
    const int tiles = (R + kTileRows - 1) / kTileRows, part = (int)blockIdx.x, other = tiles - 1 - part;
    const int r0[M] = {other * kTileRows + 16 * w, part * kTileRows + 16 * w};
    const int nb = kv8_tile_records(pos0, other, R, G), b0 = (int)((long)nb * z / P), n = (int)((long)nb * (z + 1) / P) - b0;
    const int nboth = part < other ? min(max(kv8_tile_records(pos0, part, R, G) - b0, 0), n) : 0;   // records that both tiles see
    // of those, and of all, the first that some row does not see to its end
    const int mboth = min(max(kv8_tile_seen(pos0, part, R, G) - b0, 0), nboth);
    const int mone = min(max(kv8_tile_seen(pos0, other, R, G) - b0, nboth), n);
    const uint8_t* head = a.cache + ((size_t)g * (a.max_len / kBlk) + b0) * kRec;
    auto issue_scales = [&](int k) {   // every wave the same bytes
        if (k < n) vmi_lds_dma4_at(head + (size_t)k * kRec + 2 * kHalfRec, 4 * kv8_lane(), s_scale[k & 1]);
    };
    auto issue = [&](int k) {   // and the scales of the next
        if (k >= n) return;
        const uint8_t* rec = head + (size_t)k * kRec;
        uint8_t* dst = s_rec[k & 1];
        const uint32_t at16 = 16 * kv8_lane();
        vmi_lds_dma16_at(rec + 1024 * w, at16, dst + 1024 * w);
        vmi_lds_dma16_at(rec + kHalfRec + 1024 * w, at16, dst + kHalfRec + 1024 * w);
        issue_scales(k + 1);
    };
    // the wave's share of a record's values; and the scales
    auto convert = [&](int k) {
        if (k >= n) return;
        const int lane = kv8_lane();
        const vmi_u4 v = *reinterpret_cast<const vmi_u4*>(s_rec[k & 1] + kHalfRec + 1024 * w + 16 * lane);
        const vmi_u4 f = *reinterpret_cast<const vmi_u4*>(s_vf[k % 3] + 8 * (lane >> 4));
        vmi_u4* dst = s_f16[k & 1] + 2 * w * 64 + lane;
        dst[0] = kv8_scaled(v[0], v[1], f);
        dst[64] = kv8_scaled(v[2], v[3], f);
    };
    int top_exp = kMinExp;   // E, of the wave that prepares the scales
    auto scales = [&](int k) {
        if (k >= n || w != 0) return;
        const int lane = kv8_lane();
        const float ks = s_scale[k & 1][lane & (kBlk - 1)], vs = s_scale[k & 1][kBlk + (lane & (kBlk - 1))];
        const bool ok = vs == vs;
        // (what a masked record raises E by that a row does not see, no unmasked one of that row's follows)
        if (__any(vs >= ldexpf(1.0f, top_exp)))
            top_exp = max(top_exp, (int)(__float_as_uint(vmi_wave_max(ok ? vs : 0.0f)) >> 23) - 126);
        if (lane < kBlk) {
            s_ks[k % 3][lane] = ok ? ks * kKeyUnit : vs;
            s_vs[k % 3][lane] = ok ? vs : 0.0f;
            const bool masked = k < nboth ? k >= mboth : k >= mone;
            s_vf[k % 3][lane] = (_Float16)(masked ? (float)(1 << kValueBits) : ok ? ldexpf(vs, kValueBits - top_exp) : 0.0f);
            s_exp[k % 3] = top_exp;
        }
    };
    auto phase = [&] {
        __builtin_amdgcn_sched_barrier(0);
        kv8_lds_wait();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    issue_scales(0);
    issue(0);
    Kv8Rows<M> Q;
    kv8_load_rows<M>(a, a.q, g, r0, R, Q);
    vmi_f4 o[M][16];     // in units of 2^(ref - kValueBits - kProbBits)
    float top[M];        // the reference score, less kProbBits
    float l[M];          // the lane's share of the probabilities, times 2^kProbBits
    int ref[M];          // E of the sums
#pragma unroll
    for (int i = 0; i < M; ++i) {
        Q.cx[i] *= 1.0f / kKeyUnit;
        top[i] = -3.0e38f;
        ref[i] = kMinExp;
        l[i] = 0.0f;
#pragma unroll
        for (int d = 0; d < 16; ++d) o[i][d] = vmi_f4{0.f, 0.f, 0.f, 0.f};
    }
    vmi_u4 pb[M];
#pragma unroll
    for (int i = 0; i < M; ++i) pb[i] = vmi_u4{0u, 0u, 0u, 0u};
    s_f16[1][threadIdx.x] = s_f16[1][threadIdx.x + kFlashThreads] = vmi_u4{0u, 0u, 0u, 0u};
    auto values = [&](int k, auto mm) {
        constexpr int MM = decltype(mm)::value;
        const vmi_u4* V = s_f16[k & 1] + kv8_lane();
#pragma unroll
        for (int d = 0; d < 16; ++d) {
            const vmi_u4 v = V[d * 64];
#pragma unroll
            for (int i = 0; i < MM; ++i) o[i][d] = vmi_mfma_f16(v, pb[i], o[i][d]);
        }
        // operands kAhead reads ahead of the matrix instructions that take them
        constexpr int kAhead = 5;
        __builtin_amdgcn_sched_group_barrier(kSchedRead, kAhead, 0);
#pragma unroll
        for (int i = 0; i < 16 - kAhead; ++i) {
            __builtin_amdgcn_sched_group_barrier(kSchedMfma, MM, 0);
            __builtin_amdgcn_sched_group_barrier(kSchedRead, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kSchedMfma, MM * kAhead, 0);
    };
    float x[M][8];
    auto scores = [&](int k, auto mm) {
        constexpr int MM = decltype(mm)::value;
        const vmi_u4* K = reinterpret_cast<const vmi_u4*>(s_rec[k & 1] + 16 * kv8_lane());
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            vmi_i4 s[MM][2];   // h, l
#pragma unroll
            for (int i = 0; i < MM; ++i) s[i][0] = s[i][1] = vmi_i4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const vmi_u4 key = K[(4 * t + j) * 64];
#pragma unroll
                for (int i = 0; i < MM; ++i)
#pragma unroll
                    for (int c = 0; c < 2; ++c) s[i][c] = vmi_mfma_i8(key, Q.q[i][2 * j + c], s[i][c]);
            }
#pragma unroll
            for (int i = 0; i < MM; ++i)
#pragma unroll
                for (int y = 0; y < 4; ++y) x[i][4 * t + y] = kv8_score(s[i][0][y], s[i][1][y]);
        }
    };
    auto scaled = [&](int k, int mm) {   // the scores times their keys' scales
        const vmi_f4* ks = reinterpret_cast<const vmi_f4*>(s_ks[k % 3] + 8 * (kv8_lane() >> 4));   // of the lane's keys 8 q4 ..
        const vmi_f4 k0 = ks[0], k1 = ks[1];
#pragma unroll
        for (int i = 0; i < M; ++i)
#pragma unroll
            for (int y = 0; y < 4; ++y)
                if (i < mm) {
                    x[i][y] *= k0[y];
                    x[i][4 + y] *= k1[y];
                }
    };
    // a record that some row may not see to its end
    auto softmax_masked = [&](int k, auto mm) {
        constexpr int MM = decltype(mm)::value;
        scaled(k, MM);
        const vmi_f4* v = reinterpret_cast<const vmi_f4*>(s_vs[k % 3] + 8 * (kv8_lane() >> 4));
        const vmi_f4 vs[2] = {v[0], v[1]};
#pragma unroll
        for (int i = 0; i < MM; ++i) {
            const int lane = kv8_lane();
            const int seen = pos0 + min(r0[i] + (lane & 15), R - 1) / G - 8 * (lane >> 4) - kBlk * (b0 + k);
            pb[i] = kv8_masked_weights(x[i], vs, seen, Q.cx[i], top[i], ref[i], l[i], o[i]);
        }
    };
    auto softmax = [&](int k, auto mm) {
        constexpr int MM = decltype(mm)::value;
        scaled(k, MM);
        const int e = __builtin_amdgcn_readfirstlane(s_exp[k % 3]);
        float big[MM];
        bool raise = false;
        {
#pragma unroll
            for (int i = 0; i < MM; ++i) {
                big[i] = kv8_max3(kv8_max3(x[i][0], x[i][1], x[i][2]), kv8_max3(x[i][3], x[i][4], x[i][5]),
                                  kv8_max3(x[i][6], x[i][7], x[i][7]));
                raise = raise || e != ref[i] || fmaf(big[i], Q.cx[i], -top[i]) > kLazyMax + kProbBits;
            }
        }
        if (__any(raise)) {
#pragma unroll
            for (int i = 0; i < MM; ++i) {
                const float nt = fmaxf(top[i], fmaf(kv8_max32(kv8_max16(big[i])), Q.cx[i], -(float)kProbBits));
                const float f = __builtin_amdgcn_exp2f(top[i] - nt), fo = ldexpf(f, ref[i] - e);
                l[i] *= f;
#pragma unroll
                for (int d = 0; d < 16; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[i][d][r] *= fo;
                top[i] = nt;
                ref[i] = e;
            }
        }
#pragma unroll
        for (int i = 0; i < MM; ++i) {
#pragma unroll
            for (int y = 0; y < 8; ++y) x[i][y] = __builtin_amdgcn_exp2f(fmaf(x[i][y], Q.cx[i], -top[i]));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                pb[i][j] = kv8_pack_f16(x[i][2 * j], x[i][2 * j + 1]);
                l[i] = kv8_sum2(pb[i][j], l[i]);
            }
        }
    };
    constexpr std::integral_constant<int, 2> kBoth{};
    constexpr std::integral_constant<int, 1> kOne{};
    vmi_vm_wait_c<0>();
    phase();
    scales(0);
    phase();
    if (late) {   // phase 0 of the late waves
        convert(0);
        issue(1);
        phase();
    }
    // one record: the values of the one before and its own scores, over mm row groups
    auto step = [&](int k, auto mm, auto masked) {
        if (!late) issue(k + 1);
        values(k - 1, mm);   // (of record -1: zeros)
        scores(k, mm);
        scales(k + 1);
        if (late) vmi_vm_wait_c<0>();
        phase();
        if (late) issue(k + 2);
        if constexpr (masked)
            softmax_masked(k, mm);
        else
            softmax(k, mm);
        convert(k + late);
        if (!late) vmi_vm_wait_c<0>();
        phase();
    };
#pragma unroll 1
    for (int k = 0; k < mboth; ++k) step(k, kBoth, std::false_type{});
#pragma unroll 1
    for (int k = mboth; k < nboth; ++k) step(k, kBoth, std::true_type{});
    if (nboth) {   // the first tile's last values
        const vmi_u4* V = s_f16[(nboth - 1) & 1] + kv8_lane();
#pragma unroll
        for (int d = 0; d < 16; ++d) o[1][d] = vmi_mfma_f16(V[d * 64], pb[1], o[1][d]);
    }
#pragma unroll 1
    for (int k = nboth; k < mone; ++k) step(k, kOne, std::false_type{});
#pragma unroll 1
    for (int k = mone; k < n; ++k) step(k, kOne, std::true_type{});
    values(n - 1, kOne);
    if (!late) phase();   // the late waves' last
#pragma unroll
    for (int i = 0; i < M; ++i)
        if (i == 0 || part < other)
            kv8_finish_rows(a, o[i], top[i] + (float)kProbBits, kv8_sum32(kv8_sum16(l[i])) * (1.0f / (float)(1 << kProbBits)),
                            ldexpf(1.0f, ref[i] - kValueBits - kProbBits), r0[i] + (kv8_lane() & 15), R, P == 1);
}

// grid (tiles of 128 rows, n_kv, key parts): k_kv8_flash for little work (flash_plan),
// where its longer way in and out costs more than its phases give: eight waves of 16
// rows in step, one barrier a record.  It comes by DMA, two ahead; one ahead the waves
// turn its values together, over the largest scale of a record that all rows see.  A
// part takes the same number of records in every tile (a.run), so that the last tiles,
// which see the most, have the most parts; a tile of one part goes out at once.
__global__ __launch_bounds__(kFlashThreads, 2) void k_kv8_flash_short(Kv8Attn a) {
    __shared__ __attribute__((aligned(16))) uint8_t s_key[3][kHalfRec], s_val[2][kHalfRec];   // as stored
    __shared__ __attribute__((aligned(16))) float s_scale[2][2 * kBlk];
    __shared__ vmi_u4 s_v16[2][16 * 64];
    __shared__ __attribute__((aligned(16))) float s_ks[2][kBlk], s_vs[2][kBlk];
    __shared__ int s_exp[2];
    const int lane = threadIdx.x & 63, w = at_wave(), nl = lane & 15, q4 = lane >> 4;
    const int g = blockIdx.y, G = a.n_heads / a.n_kv, R = a.span * G, P = gridDim.z, z = blockIdx.z;
    const int pos0 = kv8_pos0(a.pos0, a.pos_dev, a.span, a.max_len);
    if (a.pos_dev && a.status && blockIdx.x == 0 && g == 0 && z == 0 && threadIdx.x == 0 && *a.pos_dev != pos0)
        atomicOr(a.status, VMI_STATUS_BAD_POS);
    const int tile = (int)gridDim.x - 1 - (int)blockIdx.x;   // late tiles see the most keys: first
    const int r0[1] = {tile * kTileRows + 16 * w};
    const int nb = kv8_tile_records(pos0, tile, R, G);
    const int b0 = z * a.run, b1 = min(b0 + a.run, nb);
    if (b0 >= nb) return;   // whole workgroup: a part that this tile does not have
    const int bm = min(max(kv8_tile_seen(pos0, tile, R, G), b0), b1);   // the first that some row does not see to its end
    const uint8_t* head = a.cache + (size_t)g * (a.max_len / kBlk) * kRec;
    const uint32_t at16 = 16 * lane;
    auto issue = [&](int b, int uk, int u) {
        const uint8_t* rec = head + (size_t)b * kRec;
        vmi_lds_dma16_at(rec + 1024 * w, at16, s_key[uk] + 1024 * w);
        vmi_lds_dma16_at(rec + kHalfRec + 1024 * w, at16, s_val[u] + 1024 * w);
        vmi_lds_dma4_at(rec + 2 * kHalfRec, 4 * lane, s_scale[u]);   // every wave the same bytes
    };
    auto convert = [&](int b, int u) {
        const vmi_u4 v = *reinterpret_cast<const vmi_u4*>(s_val[u] + 1024 * w + at16);
        const vmi_f4* vs = reinterpret_cast<const vmi_f4*>(s_scale[u] + kBlk + 8 * q4);
        int e = kMinExp;
        vmi_u4 f;
        f[0] = f[1] = f[2] = f[3] = kv8_pack_f16((float)(1 << kValueBits), (float)(1 << kValueBits));
        if (b < bm) {
            const vmi_f4 v0 = vs[0], v1 = vs[1];
            float top = fmaxf(fmaxf(fmaxf(v0[0], v0[1]), fmaxf(v0[2], v0[3])), fmaxf(fmaxf(v1[0], v1[1]), fmaxf(v1[2], v1[3])));
            top = fmaxf(kv8_max32(kv8_max16(top)), 0.0f);
            e = max((int)(__float_as_uint(top) >> 23) - 126, kMinExp);
            const float unit = ldexpf(1.0f, kValueBits - e);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = i < 2 ? v0[2 * i] : v1[2 * i - 4], y = i < 2 ? v0[2 * i + 1] : v1[2 * i - 3];
                f[i] = kv8_pack_f16(x == x ? x * unit : 0.0f, y == y ? y * unit : 0.0f);
            }
        }
        s_v16[u][2 * w * 64 + lane] = kv8_scaled(v[0], v[1], f);
        s_v16[u][(2 * w + 1) * 64 + lane] = kv8_scaled(v[2], v[3], f);
        if (w == 0 && lane < kBlk) {
            const float ks = s_scale[u][lane], x = s_scale[u][kBlk + lane];
            s_ks[u][lane] = x == x ? ks * kKeyUnit : x;
            s_vs[u][lane] = x == x ? x : 0.0f;
            if (lane == 0) s_exp[u] = e;
        }
    };
    if (b0 < b1) issue(b0, 0, 0);
    if (b0 + 1 < b1) issue(b0 + 1, 1, 1);
    Kv8Rows<1> Q;
    kv8_load_rows<1>(a, a.q, g, r0, R, Q);
    const float cx = Q.cx[0] * (1.0f / kKeyUnit);
    const int last = pos0 + min(r0[0] + nl, R - 1) / G;
    vmi_f4 o[16];                // in units of 2^(ref - kValueBits - kProbBits)
    float top = -3.0e38f, l = 0.0f;   // the reference score, less kProbBits; probabilities times 2^kProbBits
    int ref = kMinExp;           // exponent of the value scales
#pragma unroll
    for (int d = 0; d < 16; ++d) o[d] = vmi_f4{0.f, 0.f, 0.f, 0.f};
    vmi_vm_wait_c<0>();
    __syncthreads();
    if (b0 < b1) convert(b0, 0);
    int uk = 0;   // of s_key, the record's
    auto step = [&](int b, auto masked) {
        const int u = (b - b0) & 1, uk1 = uk == 2 ? 0 : uk + 1;
        vmi_vm_wait_c<0>();
        __syncthreads();   // record b is in operand order, b + 1 in LDS, and nobody reads what is written below
        if (b + 1 < b1) convert(b + 1, u ^ 1);
        if (b + 2 < b1) issue(b + 2, uk1 == 2 ? 0 : uk1 + 1, u);
        const vmi_u4* K = reinterpret_cast<const vmi_u4*>(s_key[uk]) + lane;
        const vmi_u4* V = s_v16[u] + lane;
        uk = uk1;
        vmi_i4 s[2][2];   // [tile of 16 keys][h, l]
        s[0][0] = s[0][1] = s[1][0] = s[1][1] = vmi_i4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const vmi_u4 key = K[(4 * t + j) * 64];
#pragma unroll
                for (int c = 0; c < 2; ++c) s[t][c] = vmi_mfma_i8(key, Q.q[0][2 * j + c], s[t][c]);
            }
        const vmi_f4* ks = reinterpret_cast<const vmi_f4*>(s_ks[u] + 8 * q4);   // of the lane's keys 8 q4 ..
        float x[8];
        {
            const vmi_f4 k0 = ks[0], k1 = ks[1];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                x[y] = kv8_score(s[0][0][y], s[0][1][y]) * k0[y];
                x[4 + y] = kv8_score(s[1][0][y], s[1][1][y]) * k1[y];
            }
        }
        vmi_u4 pb;
        if constexpr (masked) {
            const vmi_f4* v = reinterpret_cast<const vmi_f4*>(s_vs[u] + 8 * q4);
            const vmi_f4 vs[2] = {v[0], v[1]};
            pb = kv8_masked_weights(x, vs, last - (kBlk * b + 8 * q4), cx, top, ref, l, o);
        } else {
            const int e = max(__builtin_amdgcn_readfirstlane(s_exp[u]), ref);
            const float down = ldexpf(1.0f, __builtin_amdgcn_readfirstlane(s_exp[u]) - e);   // the record's values to E
            const float big = kv8_max3(kv8_max3(x[0], x[1], x[2]), kv8_max3(x[3], x[4], x[5]), kv8_max3(x[6], x[7], x[7]));
            if (e != ref || __any(fmaf(big, cx, -top) > kLazyMax + kProbBits)) {
                const float nt = fmaxf(top, fmaf(kv8_max32(kv8_max16(big)), cx, -(float)kProbBits));
                const float f = __builtin_amdgcn_exp2f(top - nt), fo = ldexpf(f, ref - e);
                l *= f;
#pragma unroll
                for (int d = 0; d < 16; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[d][r] *= fo;
                top = nt;
                ref = e;
            }
#pragma unroll
            for (int y = 0; y < 8; ++y) {
                x[y] = __builtin_amdgcn_exp2f(fmaf(x[y], cx, -top));
                l += x[y];
                x[y] *= down;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) pb[j] = kv8_pack_f16(x[2 * j], x[2 * j + 1]);
        }
#pragma unroll
        for (int d = 0; d < 16; ++d) o[d] = vmi_mfma_f16(V[d * 64], pb, o[d]);
    };
#pragma unroll 1
    for (int b = b0; b < bm; ++b) step(b, std::false_type{});
#pragma unroll 1
    for (int b = bm; b < b1; ++b) step(b, std::true_type{});
    kv8_finish_rows(a, o, top + (float)kProbBits, kv8_sum32(kv8_sum16(l)) * (1.0f / (float)(1 << kProbBits)),
                    ldexpf(1.0f, ref - kValueBits - kProbBits), r0[0] + nl, R, nb <= a.run);
}

// ------------------------------------------------------------------- host
constexpr int kSplitRows = 64;   // rows per kv head of k_kv8_split
constexpr int kMaxTok = 8192, kMaxFlashParts = 64;

// Workgroups per kv head that share its records in k_kv8_split: one per CU
// over all kv heads.
int split_groups(int n_kv) { return std::min(std::max(1, vmi::device_cus() / n_kv), kMaxParts); }

// 16-row groups of a k_kv8_split workgroup.  Two for more than 16 rows over a cache
// that gives a wave three records or more: the groups' workgroups read the cache once
// each, which costs nothing while its records come from L2 (us, one group and two: four
// tokens at 17,000 positions 15.1 and 17.0, at 32,764 18.3 and 18.3; eight 21.1 and 25.7,
// 26.6 and 30.6) and the rate of HBM beyond (four at 64,000 26.8 and 22.9, eight at
// 50,000 38.2 and 36.4).  32 heads on 4: four at 10,000 15.7 and 17.5, at 30,000 26.1 and
// 23.0; 64 on 8: eight at 8000 27.1 and 29.5, at 16,000 48.4 and 40.6.  The results are the same.
int split_row_groups(int rows, int records, int groups) {
    return rows > 16 && records >= 3 * kSplitWaves * groups ? 2 : 1;
}

// Form and grid of more than kSplitRows rows.  k_kv8_flash_short while a CU's share is
// under sixteen records of a 128-row tile (us, that form and k_kv8_flash: 777 tokens from
// position 0 34 and 45, 1024 from 0 42 and 50, 1400 from 0 60 and 60, 200 from 1234 29
// and 38, 64 from 0 13 and 24), k_kv8_flash from there (2048 from 0 95 and 79, 300 from
// 20,000 171 and 122, 4096 from 0 207 and 181, 4096 from 8192 860 and 642).  With more kv
// heads of eight query heads each: on 4, 777 from 0 50 and 52, 1024 from 0 54 and 59, 300 from
// 4000 90 and 72; on 8, 400 from 0 38 and 43, 200 from 2000 72 and 61.  Parts fill the
// device where the tiles do not, of four records or more: a part costs its rows' way out
// and back (100 tokens from 500 in as many parts as records 29, in these 23).
struct FlashPlan {
    bool paired;
    int tiles, parts, run;   // workgroups per kv head and part; records of a part of the short form
};
// The most parts of a form, at any position.
int flash_max_parts(int tiles, int n_kv, bool paired) {
    const int ncu = vmi::device_cus();
    return std::max(1, std::min((paired ? ncu : 2 * ncu) / (tiles * n_kv), kMaxFlashParts));
}
int flash_tiles(int rows, bool paired) {
    const int tiles = (rows + kTileRows - 1) / kTileRows;
    return paired ? (tiles + 1) / 2 : tiles;
}
FlashPlan flash_plan(const Kv8Attn& a, int rows) {
    const int ncu = vmi::device_cus(), pos0 = a.pos_dev ? a.max_len - a.span : a.pos0;   // (on the device: by the capacity)
    const int64_t all = (int64_t)flash_tiles(rows, false) * a.n_kv;   // tiles of all heads
    const int mean = (pos0 + a.span / 2) / kBlk + 1, last = (pos0 + a.span - 1) / kBlk + 1;
    FlashPlan p;
    p.paired = all * mean >= 16 * ncu;
    p.tiles = flash_tiles(rows, p.paired);
    const int most = flash_max_parts(p.tiles, a.n_kv, p.paired);
    int run = 4;   // records of a part
    if (!p.paired) {
        // workgroups: records over run and half a part a tile, of seven eighths of the CUs (the XCDs' shares differ)
        const int64_t room = 7 * ncu / 8 - all / 2;
        run = room > 0 ? (int)std::max<int64_t>(run, (all * mean + room - 1) / room) : last;
        run = std::max(run, (last + most - 1) / most);
    }
    p.parts = std::min((last + run - 1) / run, most);
    p.run = p.paired ? 0 : run;
    return p;
}

}  // namespace

double vmi::kv8_rope_base(float theta, int rope_dim) {
    return rope_dim ? pow((double)theta, -2.0 / (double)rope_dim) : 1.0;
}

// The quarter turns are counted in an int; the fastest pair is the first, or with theta below 1 the last.
bool vmi::kv8_rope_ok(float theta, int rope_dim, int max_len) {
    if (!(theta > 0.0f)) return false;
    return rope_dim == 0 || max_len * std::max(1.0, pow(kv8_rope_base(theta, rope_dim), rope_dim / 2 - 1)) < 0x1p31;
}

bool vmi::kv8_heads_ok(int n_heads, int n_kv) {
    return n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 && n_heads <= 1024;
}

size_t vmi::kv8_attention_parts_bytes(int paths, int span, int n_heads, int n_kv) {
    if (paths < 1 || span < 1 || paths > 16 || span > kMaxTok || !kv8_heads_ok(n_heads, n_kv)) return 0;
    const int R = span * (n_heads / n_kv);
    if (R > kSplitRows && paths != 1) return 0;
    // of this span and of every shorter one: a prompt's blocks share a workspace
    size_t rows = (size_t)n_kv * split_groups(n_kv) * paths * std::min(R, kSplitRows);
    if (R > kSplitRows)
        for (int tiles = 1; (tiles - 1) * kTileRows < R; ++tiles) {
            const int parts = std::max(flash_max_parts(tiles, n_kv, false), flash_max_parts((tiles + 1) / 2, n_kv, true));
            if (parts == 1) break;   // and of more tiles
            rows = std::max(rows, (size_t)n_kv * parts * std::min(tiles * kTileRows, R));
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
    a.run = 0;
    a.part_o = static_cast<float*>(parts);
    int n;
    size_t rows;
    if (R <= kSplitRows) {
        n = split_groups(a.n_kv);
        rows = (size_t)a.n_kv * n * a.paths * R;
        a.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(parts) + align256(rows * kHeadDim * 4));
        const dim3 blk(kSplitThreads);
        // (with the position on the device, by the capacity)
        const int ms = split_row_groups(R, (a.pos_dev ? a.max_len : a.pos0 + a.span) / kBlk, n);
        const int tiles = (R + 16 * ms - 1) / (16 * ms);
        const dim3 grid(n, a.n_kv, a.paths * tiles);
        if (ms == 2)
            if (tiles * a.paths == 1)
                hipLaunchKernelGGL((k_kv8_split<2, true>), grid, blk, 0, s, a);
            else
                hipLaunchKernelGGL((k_kv8_split<2, false>), grid, blk, 0, s, a);
        else if (tiles * a.paths == 1)
            hipLaunchKernelGGL((k_kv8_split<1, true>), grid, blk, 0, s, a);
        else
            hipLaunchKernelGGL((k_kv8_split<1, false>), grid, blk, 0, s, a);
    } else {
        const FlashPlan p = flash_plan(a, R);
        n = p.parts;
        a.run = p.run;
        rows = n > 1 ? (size_t)a.n_kv * n * R : 1;
        a.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(parts) + align256(rows * kHeadDim * 4));
        const dim3 grid(p.tiles, a.n_kv, p.parts), blk(kFlashThreads);
        if (p.paired)
            hipLaunchKernelGGL(k_kv8_flash, grid, blk, 0, s, a);
        else
            hipLaunchKernelGGL(k_kv8_flash_short, grid, blk, 0, s, a);
        if (n == 1) return hipGetLastError();
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int rows_all = a.paths * a.span * a.n_heads;
    if (R <= kSplitRows)
        hipLaunchKernelGGL(k_kv8_merge, dim3(rows_all, 4), dim3(kThreads), 0, s, a, n);
    else
        hipLaunchKernelGGL(k_kv8_merge_rows, dim3((rows_all + kWaves - 1) / kWaves), dim3(kThreads), 0, s, a, n);
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
    if (D.rope_dim < 0 || D.rope_dim > kHeadDim || D.rope_dim % 2 || !vmi::kv8_rope_ok(D.rope_theta, D.rope_dim, max_len))
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
    if (!keys || !values || !aligned(keys, 16) || !aligned(values, 16))
        return vmi::fail(VMI_ERR_INVALID, "keys or values null or not 16-byte aligned");
    if ((key_head | key_row | value_head | value_row) & 7)
        return vmi::fail(VMI_ERR_INVALID, "strides must be multiples of 8 elements");
    WriteArgs a{{keys, values}, {key_head, value_head}, {key_row, value_row}, n, pos0, cache, max_len};
    const int recs = (pos0 + n - 1) / kBlk - pos0 / kBlk + 1;
    hipLaunchKernelGGL(k_kv8_write, dim3(recs, n_kv_heads, 2), dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
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
    if (rope_dim < 0 || rope_dim > kHeadDim || rope_dim % 2 || !vmi::kv8_rope_ok(rope_theta, rope_dim, max_len))
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
