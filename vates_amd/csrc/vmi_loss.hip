// Softmax cross entropy of tokens under a head, and its gradients, without the
// logits in memory.
//
//   z = x . W^T;  lse_t = log sum_v exp z_tv;  loss_t = lse_t - z_t,target
//   g_tv = (dloss_t + dlse_t) exp(z_tv - lse_t) - dloss_t [v = target_t]
//   dx = g W;  dW = g^T x
//
// Tokens left out of the loss are taken out first: the kernels work on the nv
// tokens that are in it (idx: their rows of x), and nothing of the others is read.
//
// All products are one form, D[m][n] = sum_k A[m][k] B[n][k] over tiles of
// 256 x 256 (less where there are few tokens) on 16 x 16 x 32 bf16 matrix
// instructions, 64 of k a step, both operands by DMA into LDS while the step before is
// multiplied:
//   k_loss_score, k_loss_g   m a vocabulary row, n a token, k a hidden value
//   k_loss_dx                m a hidden value,   n a token, k a vocabulary row
//   k_loss_dw                m a hidden value,   n a vocabulary row, k a token
// An operand whose rows run along k lies in LDS as rows of 64 values, 16-byte pieces
// at piece ^ (row & 7); one whose rows run along m or n (W for dx; x and g for dW) as
// it is in memory, 32-byte pieces at piece ^ (k & 7), and ds_read_b64_tr_b16 turns 4 x 16
// values as they are read.  Both placements read without bank conflicts (4.7 and 4.3 cycles an
// instruction, as consecutive addresses do; rows unturned 12.6 and 16).
//
// Kernels beside them:
//   k_loss_rows     the tokens in the loss, and their coefficients
//   k_loss_merge    the strips' maxima and sums of a token joined
//   k_loss_compact  those tokens' rows of x side by side
//   k_loss_dx_out   the split sums of dx joined

#include <algorithm>

#include "vmi_device.h"
#include "vmi_internal.h"

namespace {

constexpr int kThreads = 512, kWaves = 8, kBK = 64;
constexpr int kMaxT = 65536, kMaxH = 8192, kMaxV = 1 << 21;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;

__device__ __forceinline__ int ls_wave() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

// ------------------------------------------------------------------ products
// One workgroup's tile: BM x BN, waves WM x WN.  SLOW operands have k as the slow
// index (rows of BM or BN = 256 values).
template <int BM_, int BN_, int WM_, int WN_, int STAGES_, bool ASLOW_, bool BSLOW_>
struct Tile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_;
    static constexpr bool ASLOW = ASLOW_, BSLOW = BSLOW_;
    static constexpr int MB = BM / WM / 16, NB = BN / WN / 16;
    static constexpr int kA = BM * kBK * 2, kB = BN * kBK * 2, kStage = kA + kB;
    static constexpr int DA = kA / 1024 / kWaves, DB = kB / 1024 / kWaves;   // DMA instructions of a wave a step
    static_assert(WM * WN == kWaves && DA >= 1 && DB >= 1, "shape");
    static_assert((!ASLOW || BM == 256) && (!BSLOW || BN == 256), "slow operands have rows of 512 bytes");
};

// Row and 16-byte piece of a lane in DMA instruction i of D of its wave.
template <int D, bool SLOW>
__device__ __forceinline__ void ls_slot(int i, int& row, int& piece) {
    const int lane = threadIdx.x & 63, u = ls_wave() * D + i;
    if constexpr (SLOW) {   // two rows of 32 pieces
        row = 2 * u + (lane >> 5);
        const int s = lane & 31;
        piece = (((s >> 1) ^ (row & 7)) << 1) | (s & 1);
    } else {                // eight rows of eight
        row = 8 * u + (lane >> 3);
        piece = (lane & 7) ^ (row & 7);
    }
}
template <int D>
__device__ __forceinline__ void ls_dma(const void* base, const uint32_t (&off)[D], uint8_t* lds) {
#pragma unroll
    for (int i = 0; i < D; ++i) vmi_lds_dma16_at(base, off[i], lds + (ls_wave() * D + i) * 1024);
}

// Operand of block b (16 of m or n, from `first` on) and k = 32 kk ..
template <bool SLOW>
__device__ __forceinline__ vmi_u4 ls_operand(const uint8_t* lds, int first, int kk) {
    const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
    if constexpr (SLOW) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef uint32_t u2 __attribute__((ext_vector_type(2)));
        vmi_u4 r;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = 32 * kk + 8 * q + 4 * h + (i >> 2);
            const uint8_t* p = lds + k * 512 + (((first >> 4) ^ (k & 7)) << 5) + 8 * (i & 3);
            const s4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p));
            const u2 w = __builtin_bit_cast(u2, v);
            r[2 * h] = w[0];
            r[2 * h + 1] = w[1];
        }
        return r;
    } else {
        const int row = first + i;
        return *reinterpret_cast<const vmi_u4*>(lds + row * 128 + (((4 * kk + q) ^ (row & 7)) << 4));
    }
}

// acc[m block][n block] += the step in `lds`: lane (i = lane & 15, q = lane >> 4) holds
// D[16 mb + 4 q + r][16 nb + i] of its wave's part.
template <class S>
__device__ __forceinline__ void ls_multiply(const uint8_t* lds, vmi_f4 (&acc)[S::MB][S::NB]) {
    const int w = ls_wave(), m0 = (w / S::WN) * (S::BM / S::WM), n0 = (w % S::WN) * (S::BN / S::WN);
#pragma unroll
    for (int kk = 0; kk < kBK / 32; ++kk) {
        vmi_u4 a[S::MB], b[S::NB];
#pragma unroll
        for (int n = 0; n < S::NB; ++n) b[n] = ls_operand<S::BSLOW>(lds + S::kA, n0 + 16 * n, kk);
#pragma unroll
        for (int m = 0; m < S::MB; ++m) a[m] = ls_operand<S::ASLOW>(lds, m0 + 16 * m, kk);
#pragma unroll
        for (int m = 0; m < S::MB; ++m)
#pragma unroll
            for (int n = 0; n < S::NB; ++n) acc[m][n] = vmi_mfma_bf16(a[m], b[n], acc[m][n]);
    }
}
template <class S>
__device__ __forceinline__ void ls_clear(vmi_f4 (&acc)[S::MB][S::NB]) {
#pragma unroll
    for (int m = 0; m < S::MB; ++m)
#pragma unroll
        for (int n = 0; n < S::NB; ++n) acc[m][n] = vmi_f4{0.f, 0.f, 0.f, 0.f};
}

// The steps 0 .. total - 1 of a workgroup's tiles, one after another: job.issue(lds) asks
// for the next step's operands (behind the last, again for the last's, so that every
// wait counts alike), job.done(acc) ends a step and takes a tile that is complete.
template <class S, class Job>
__device__ __forceinline__ void ls_run(uint8_t* lds, Job& job, int total) {
    vmi_f4 acc[S::MB][S::NB];
    ls_clear<S>(acc);
    for (int s = 0; s < S::STAGES - 1; ++s) job.issue(lds + s * S::kStage);
    int in = S::STAGES - 1, out = 0;
    for (int s = 0; s < total; ++s) {
        vmi_vm_wait_c<(S::STAGES - 2) * (S::DA + S::DB)>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        job.issue(lds + in * S::kStage);
        in = in + 1 == S::STAGES ? 0 : in + 1;
        ls_multiply<S>(lds + out * S::kStage, acc);
        out = out + 1 == S::STAGES ? 0 : out + 1;
        job.done(acc);
    }
    // nothing in flight, and no wave reading, when the next run begins
    vmi_vm_wait_c<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// -------------------------------------------------------------- logits' tiles
// A token's coefficients: g = a exp(z - lse) - b at its target.
struct Coef {
    float a, b, lse;
    int32_t target;
};

struct LogitArgs {
    const uint16_t *x, *w;
    const int32_t *idx, *meta;   // meta[0]: nv
    const Coef* coef;
    int H, V;
    // score
    float2* part;                // [item][BN] maximum, sum
    float* hit;                  // [nv] the target's logit
    // gradient
    int v0, v1;                  // the piece (v1 past V: columns of zeros)
    uint16_t* g;                 // [tokens][ldg]
    int64_t ldg;
};

// The strips that the vocabulary is cut into for nrb blocks of tokens.
__device__ __host__ __forceinline__ int ls_strips(int nrb, int grid) { return 8 * nrb <= grid ? grid / nrb : 8; }

template <class S, bool GRAD>
struct LogitJob {
    const LogitArgs& a;
    int nv, rb, v1;                   // tokens, block, end of the strip
    int tile;                         // first row of the tile being multiplied
    int next, k, nk;                  // first row of the tile being asked for, its step, steps of one
    int kd;                           // step being multiplied
    uint32_t offa[S::DA], offb[S::DB];
    Coef c[S::NB];
    float m[S::NB], l[S::NB];
    int m0, n0;

    __device__ __forceinline__ LogitJob(const LogitArgs& a_, int rb_, int v0_, int v1_) : a(a_), rb(rb_), v1(v1_) {
        nv = vmi_sload_i32(a.meta);
        nk = a.H / kBK;
        tile = v0_;
        next = min(v0_, a.V - 1);   // (a piece's last tile may lie behind the vocabulary: its columns are zeros)
        k = kd = 0;
        const int w = ls_wave(), lane = threadIdx.x & 63;
        m0 = (w / S::WN) * (S::BM / S::WM) + 4 * (lane >> 4);
        n0 = (w % S::WN) * (S::BN / S::WN) + (lane & 15);
#pragma unroll
        for (int i = 0; i < S::DB; ++i) {
            int row, piece;
            ls_slot<S::DB, false>(i, row, piece);
            const int c0 = min(rb * S::BN + row, nv - 1);
            offb[i] = (uint32_t)(a.idx ? a.idx[c0] : c0) * (uint32_t)(2 * a.H) + 16 * piece;
        }
        rows();
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            const int t = rb * S::BN + n0 + 16 * n;
            c[n] = a.coef[min(t, nv - 1)];
            if (t >= nv) c[n] = Coef{0.0f, 0.0f, __builtin_inff(), -1};
            m[n] = kLowest;
            l[n] = 0.0f;
        }
    }
    __device__ __forceinline__ void rows() {
#pragma unroll
        for (int i = 0; i < S::DA; ++i) {
            int row, piece;
            ls_slot<S::DA, false>(i, row, piece);
            offa[i] = (uint32_t)min(row, min(v1, a.V) - 1 - next) * (uint32_t)(2 * a.H) + 16 * piece;
        }
    }
    __device__ __forceinline__ void issue(uint8_t* lds) {
        ls_dma<S::DA>(a.w + (size_t)next * a.H + (size_t)k * kBK, offa, lds);
        ls_dma<S::DB>(a.x + (size_t)k * kBK, offb, lds + S::kA);
        if (++k == nk) {
            if (next + S::BM < min(v1, a.V)) {
                next += S::BM;
                k = 0;
                rows();
            } else {
                k = nk - 1;
            }
        }
    }
    __device__ __forceinline__ void done(vmi_f4 (&acc)[S::MB][S::NB]) {
        if (++kd < nk) return;
        kd = 0;
        if constexpr (GRAD)
            store(acc);
        else
            sum(acc);
        ls_clear<S>(acc);
        tile += S::BM;
    }
    // Running maximum and sum of a lane's own rows of the tiles, joined over lanes at the end only.
    __device__ __forceinline__ void sum(vmi_f4 (&acc)[S::MB][S::NB]) {
        const int last = v1 - 1 - tile - m0;   // rows of the lane up to this one
        if (tile + S::BM > v1) {
#pragma unroll
            for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                for (int n = 0; n < S::NB; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (16 * mb + r > last) acc[mb][n][r] = kLowest;
        }
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            const int d = c[n].target - tile - m0;
            if (__any((uint32_t)d < (uint32_t)(16 * S::MB))) {
#pragma unroll
                for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (d == 16 * mb + r && 16 * mb + r <= last) a.hit[rb * S::BN + n0 + 16 * n] = acc[mb][n][r];
            }
            float top = m[n];
#pragma unroll
            for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, acc[mb][n][r]);
            float s = l[n] * __builtin_amdgcn_exp2f((m[n] - top) * kLog2e);   // (a product's rounding before the difference would
#pragma unroll
            for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                for (int r = 0; r < 4; ++r) s += __builtin_amdgcn_exp2f((acc[mb][n][r] - top) * kLog2e);   // grow with the logits)
            m[n] = top;
            l[n] = s;
        }
    }
    __device__ __forceinline__ void store(vmi_f4 (&acc)[S::MB][S::NB]) {
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            const int t = rb * S::BN + n0 + 16 * n, d = c[n].target - tile - m0;
            uint16_t* dst = a.g + (int64_t)t * a.ldg + (tile - a.v0) + m0;
#pragma unroll
            for (int mb = 0; mb < S::MB; ++mb) {
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    v[r] = c[n].a * __builtin_amdgcn_exp2f((acc[mb][n][r] - c[n].lse) * kLog2e);
                    if (d == 16 * mb + r) v[r] -= c[n].b;
                    if (t >= nv || tile + m0 + 16 * mb + r >= a.V) v[r] = 0.0f;
                }
                *reinterpret_cast<uint2*>(dst + 16 * mb) = make_uint2(vmi_pack_bf16x2(v[0], v[1]), vmi_pack_bf16x2(v[2], v[3]));
            }
        }
    }
};

__device__ __forceinline__ void ls_join(float& m, float& l, float m2, float l2) {
    const float top = fmaxf(m, m2);
    l = l * __builtin_amdgcn_exp2f((m - top) * kLog2e) + l2 * __builtin_amdgcn_exp2f((m2 - top) * kLog2e);
    m = top;
}

// A workgroup takes a block of tokens and a strip of the vocabulary, whose tiles follow
// each other without a pause of the DMA.
template <class S>
__global__ __launch_bounds__(kThreads) void k_loss_score(LogitArgs a) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[S::STAGES * S::kStage];
    const int nv = vmi_sload_i32(a.meta), nrb = (nv + S::BN - 1) / S::BN;
    if (nrb == 0) return;
    const int strips = ls_strips(nrb, gridDim.x), per = ((a.V + strips - 1) / strips + 15) & ~15;
    for (int item = blockIdx.x; item < nrb * strips; item += gridDim.x) {
        const int rb = item % nrb, v0 = (item / nrb) * per, v1 = min(a.V, v0 + per);
        float2* part = a.part + (size_t)item * S::BN;
        if (v0 >= v1) {
            if (threadIdx.x < S::BN) part[threadIdx.x] = make_float2(kLowest, 0.0f);
            continue;
        }
        LogitJob<S, false> job(a, rb, v0, v1);
        ls_run<S>(lds, job, (v1 - v0 + S::BM - 1) / S::BM * job.nk);
        float2* s_ml = reinterpret_cast<float2*>(lds);   // [WM][BN]
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            float m = job.m[n], l = job.l[n];
            ls_join(m, l, __shfl_xor(m, 16), __shfl_xor(l, 16));
            ls_join(m, l, __shfl_xor(m, 32), __shfl_xor(l, 32));
            if ((threadIdx.x & 63) < 16) s_ml[(ls_wave() / S::WN) * S::BN + job.n0 + 16 * n] = make_float2(m, l);
        }
        __syncthreads();
        if (threadIdx.x < S::BN) {
            float2 u = s_ml[threadIdx.x];
            for (int i = 1; i < S::WM; ++i) ls_join(u.x, u.y, s_ml[i * S::BN + threadIdx.x].x, s_ml[i * S::BN + threadIdx.x].y);
            part[threadIdx.x] = u;
        }
        __syncthreads();
    }
}

// The same tiles of one piece of the vocabulary as rows of g.
template <class S>
__global__ __launch_bounds__(kThreads) void k_loss_g(LogitArgs a) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[S::STAGES * S::kStage];
    const int nv = vmi_sload_i32(a.meta), nrb = (nv + S::BN - 1) / S::BN;
    if (nrb == 0) return;
    const int tiles = (a.v1 - a.v0 + S::BM - 1) / S::BM, strips = min(ls_strips(nrb, gridDim.x), tiles);
    const int per = (tiles + strips - 1) / strips * S::BM;
    for (int item = blockIdx.x; item < nrb * strips; item += gridDim.x) {
        const int rb = item % nrb, v0 = a.v0 + (item / nrb) * per, v1 = min(a.v1, v0 + per);
        if (v0 >= v1) continue;
        LogitJob<S, true> job(a, rb, v0, v1);
        ls_run<S>(lds, job, (v1 - v0 + S::BM - 1) / S::BM * job.nk);
    }
}

// ------------------------------------------------------------------------ dx
struct DxArgs {
    const uint16_t *w, *g;
    const int32_t* meta;
    int H, V, v0, cols;      // the piece's first row, its columns of g (a multiple of 64)
    int64_t ldg;
    float* sum;              // [split][token block rows][H]
    int add;                 // a later piece than the first: added to the sums
    int short_steps;         // steps of the shortest piece: no split without columns
};

__device__ __forceinline__ int ls_dx_splits(int nrb, int nht, int grid, int steps) {
    return min(max(grid / (nrb * nht), 1), steps);
}

template <class S>
struct DxJob {
    const DxArgs& a;
    int ht, rb, split, nrb, left;   // left: steps still to be asked for
    int kn;                         // next step's first column of g
    int steps, kd;
    uint32_t offb[S::DB];

    __device__ __forceinline__ DxJob(const DxArgs& a_, int ht_, int rb_, int split_, int nrb_, int k0, int k1)
        : a(a_), ht(ht_), rb(rb_), split(split_), nrb(nrb_), left(k1 - k0), kn(k0 * kBK), steps(k1 - k0), kd(0) {
#pragma unroll
        for (int i = 0; i < S::DB; ++i) {
            int row, piece;
            ls_slot<S::DB, false>(i, row, piece);
            offb[i] = (uint32_t)row * (uint32_t)(2 * a.ldg) + 16 * piece;
        }
    }
    __device__ __forceinline__ void issue(uint8_t* lds) {
        uint32_t offa[S::DA];
        const int rows = a.V - a.v0 - kn;       // rows of W from here on
        const int base = min(kn, a.V - a.v0 - 1);
#pragma unroll
        for (int i = 0; i < S::DA; ++i) {
            int row, piece;
            ls_slot<S::DA, true>(i, row, piece);
            const int col = min(ht * S::BM + 8 * piece, a.H - 8);
            offa[i] = (uint32_t)(max(min(row, rows - 1), 0)) * (uint32_t)(2 * a.H) + 2 * col;
        }
        ls_dma<S::DA>(a.w + (size_t)(a.v0 + base) * a.H, offa, lds);
        ls_dma<S::DB>(a.g + (int64_t)rb * S::BN * a.ldg + kn, offb, lds + S::kA);
        if (--left > 0) kn += kBK;
    }
    __device__ __forceinline__ void done(vmi_f4 (&acc)[S::MB][S::NB]) {
        if (++kd < steps) return;
        const int w = ls_wave(), lane = threadIdx.x & 63;
        const int m0 = ht * S::BM + (w / S::WN) * (S::BM / S::WM) + 4 * (lane >> 4);
        const int n0 = rb * S::BN + (w % S::WN) * (S::BN / S::WN) + (lane & 15);
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            float* row = a.sum + ((size_t)split * nrb * S::BN + n0 + 16 * n) * a.H + m0;
#pragma unroll
            for (int mb = 0; mb < S::MB; ++mb) {
                if (m0 + 16 * mb >= a.H) continue;
                vmi_f4* dst = reinterpret_cast<vmi_f4*>(row + 16 * mb);
                *dst = a.add ? *dst + acc[mb][n] : acc[mb][n];
            }
        }
    }
};

// Tiles of 256 hidden values by a block of tokens; where these leave CUs idle the
// piece's columns are split over several workgroups, each with sums of its own.
template <class S>
__global__ __launch_bounds__(kThreads) void k_loss_dx(DxArgs a) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[S::STAGES * S::kStage];
    const int nv = vmi_sload_i32(a.meta), nrb = (nv + S::BN - 1) / S::BN, nht = (a.H + S::BM - 1) / S::BM, steps = a.cols / kBK;
    if (nrb == 0) return;
    const int splits = ls_dx_splits(nrb, nht, gridDim.x, a.short_steps);
    for (int item = blockIdx.x; item < splits * nht * nrb; item += gridDim.x) {
        const int rb = item % nrb, ht = item / nrb % nht, sp = item / nrb / nht;
        const int k0 = (int)((int64_t)steps * sp / splits), k1 = (int)((int64_t)steps * (sp + 1) / splits);
        DxJob<S> job(a, ht, rb, sp, nrb, k0, k1);
        ls_run<S>(lds, job, k1 - k0);
    }
}

// ------------------------------------------------------------------------ dW
struct DwArgs {
    const uint16_t *x, *g;
    const int32_t* meta;
    int H, V, v0, cols;
    int64_t ldg;
    void* dw;
};

template <class S, bool F32>
struct DwJob {
    const DwArgs& a;
    int nk, nht, step, item, items;      // asked for
    int kd, at;                          // being multiplied
    uint32_t offa[S::DA], offb[S::DB];

    __device__ __forceinline__ DwJob(const DwArgs& a_, int nk_, int nht_, int items_)
        : a(a_), nk(nk_), nht(nht_), step(0), item(blockIdx.x), items(items_), kd(0), at(blockIdx.x) {
        rows();
    }
    __device__ __forceinline__ void rows() {
        const int ht = item % nht, vt = item / nht;
#pragma unroll
        for (int i = 0; i < S::DA; ++i) {
            int row, piece;
            ls_slot<S::DA, true>(i, row, piece);
            offa[i] = (uint32_t)row * (uint32_t)(2 * a.H) + 2 * min(ht * S::BM + 8 * piece, a.H - 8);
        }
#pragma unroll
        for (int i = 0; i < S::DB; ++i) {
            int row, piece;
            ls_slot<S::DB, true>(i, row, piece);
            offb[i] = (uint32_t)row * (uint32_t)(2 * a.ldg) + 2 * (vt * S::BN + 8 * piece);
        }
    }
    __device__ __forceinline__ void issue(uint8_t* lds) {
        ls_dma<S::DA>(a.x + (size_t)step * kBK * a.H, offa, lds);
        ls_dma<S::DB>(a.g + (int64_t)step * kBK * a.ldg, offb, lds + S::kA);
        if (++step == nk) {
            if (item + (int)gridDim.x < items) {
                item += gridDim.x;
                step = 0;
                rows();
            } else {
                step = nk - 1;
            }
        }
    }
    __device__ __forceinline__ void done(vmi_f4 (&acc)[S::MB][S::NB]) {
        if (++kd < nk) return;
        kd = 0;
        write(acc);
        ls_clear<S>(acc);
        at += gridDim.x;
    }
    __device__ __forceinline__ void write(vmi_f4 (&acc)[S::MB][S::NB]) {
        const int w = ls_wave(), lane = threadIdx.x & 63;
        const int m0 = at % nht * S::BM + (w / S::WN) * (S::BM / S::WM) + 4 * (lane >> 4);
        const int n0 = a.v0 + at / nht * S::BN + (w % S::WN) * (S::BN / S::WN) + (lane & 15);
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            if (n0 + 16 * n >= a.V) continue;
            const size_t row = (size_t)(n0 + 16 * n) * a.H + m0;
#pragma unroll
            for (int mb = 0; mb < S::MB; ++mb) {
                if (m0 + 16 * mb >= a.H) continue;
                const vmi_f4 v = acc[mb][n];
                if constexpr (F32)
                    *reinterpret_cast<vmi_f4*>(static_cast<float*>(a.dw) + row + 16 * mb) = v;
                else
                    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.dw) + row + 16 * mb) =
                        make_uint2(vmi_pack_bf16x2(v[0], v[1]), vmi_pack_bf16x2(v[2], v[3]));
            }
        }
    }
};

template <class S, bool F32>
__global__ __launch_bounds__(kThreads) void k_loss_dw(DwArgs a) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[S::STAGES * S::kStage];
    const int nv = vmi_sload_i32(a.meta), nk = (nv + kBK - 1) / kBK, nht = (a.H + S::BM - 1) / S::BM;
    const int items = nht * ((a.cols + S::BN - 1) / S::BN);
    if ((int)blockIdx.x >= items) return;
    DwJob<S, F32> job(a, max(nk, 1), nht, items);
    const int mine = (items - 1 - (int)blockIdx.x) / (int)gridDim.x + 1;
    if (nk == 0) {   // no token in the loss: zeros
        vmi_f4 acc[S::MB][S::NB];
        ls_clear<S>(acc);
        for (int i = 0; i < mine; ++i) {
            job.write(acc);
            job.at += gridDim.x;
        }
        return;
    }
    ls_run<S>(lds, job, mine * nk);
}

// --------------------------------------------------------------- small kernels
struct RowsArgs {
    const int64_t* target;
    int64_t ignore;
    int T, Tp, V;
    int32_t *idx, *pos, *meta;     // tokens in the loss, each token's place among them or -1, their number
    Coef* coef;                    // [Tp]
    float *loss, *lse_out;         // score: written for tokens left out
    uint32_t* status;
    const float *lse, *dloss, *dlse;
};

// One workgroup: a thread takes a run of tokens.  Bound by latency, 3 to 5 us up to 8192 tokens.
__global__ __launch_bounds__(1024) void k_loss_rows(RowsArgs a) {
    __shared__ int s_sum[16];
    const int lane = threadIdx.x & 63, w = ls_wave(), run = (a.T + 1023) / 1024;
    const int t0 = min(a.T, (int)threadIdx.x * run), t1 = min(a.T, t0 + run);
    int n = 0;
    bool bad = false;
    for (int t = t0; t < t1; ++t) {
        const int64_t y = a.target[t];
        const bool in = y >= 0 && y < a.V && y != a.ignore;
        n += in;
        bad |= !in && y != a.ignore;
    }
    if (a.status && __any(bad) && lane == 0) atomicOr(a.status, VMI_STATUS_BAD_TARGET);
    int v = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(v, d);
        if (lane >= d) v += u;
    }
    if (lane == 63) s_sum[w] = v;
    __syncthreads();
    int c = v - n, all = 0;
    for (int i = 0; i < 16; ++i) {
        c += i < w ? s_sum[i] : 0;
        all += s_sum[i];
    }
    for (int t = t0; t < t1; ++t) {
        const int64_t y = a.target[t];
        const bool in = y >= 0 && y < a.V && y != a.ignore;
        a.pos[t] = in ? c : -1;
        if (in) {
            a.idx[c] = t;
            Coef k{0.0f, 0.0f, 0.0f, (int32_t)y};
            if (a.dloss) {
                k.b = a.dloss[t];
                k.a = k.b + (a.dlse ? a.dlse[t] : 0.0f);
                k.lse = a.lse[t];
            }
            a.coef[c++] = k;
        } else if (a.loss) {
            a.loss[t] = a.lse_out[t] = y == a.ignore ? 0.0f : __builtin_nanf("");
        }
    }
    if (threadIdx.x == 0) a.meta[0] = all;
}

// A wave per token: its strips' maxima and sums, in a fixed order.
__global__ __launch_bounds__(256) void k_loss_merge(const int32_t* meta, const int32_t* idx, const float2* part,
                                                    const float* hit, int bn, int grid, float* loss, float* lse) {
    const int c = blockIdx.x * 4 + ls_wave(), lane = threadIdx.x & 63, nv = meta[0];
    if (c >= nv) return;
    const int nrb = (nv + bn - 1) / bn, strips = ls_strips(nrb, grid), rb = c / bn;
    float m = kLowest, l = 0.0f;
    for (int s = lane; s < strips; s += 64) {
        const float2 p = part[((size_t)s * nrb + rb) * bn + c % bn];
        ls_join(m, l, p.x, p.y);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) ls_join(m, l, __shfl_xor(m, d), __shfl_xor(l, d));
    if (lane == 0) {
        const float v = m + logf(l);
        lse[idx[c]] = v;
        loss[idx[c]] = v - hit[c];
    }
}

// Row c of the tokens in the loss, zeros from nv on.
__global__ __launch_bounds__(256) void k_loss_compact(const int32_t* meta, const int32_t* idx, const vmi_u4* x, int U,
                                                      vmi_u4* out) {
    const int c = blockIdx.x;
    const bool in = c < meta[0];
    const size_t src = in ? (size_t)idx[c] * U : 0;
    for (int u = threadIdx.x; u < U; u += 256) out[(size_t)c * U + u] = in ? x[src + u] : vmi_u4{0, 0, 0, 0};
}

// dx of a token: its splits' sums in order, zeros for a token left out.
__global__ __launch_bounds__(256) void k_loss_dx_out(const int32_t* meta, const int32_t* pos, const float* sum, int H, int bn,
                                                     int bm, int grid, int steps, uint16_t* dx) {
    const int t = blockIdx.x, c = pos[t], nrb = (meta[0] + bn - 1) / bn;
    const int splits = nrb ? ls_dx_splits(nrb, (H + bm - 1) / bm, grid, steps) : 0;
    for (int h = 4 * threadIdx.x; h < H; h += 1024) {
        vmi_f4 v = {0.f, 0.f, 0.f, 0.f};
        if (c >= 0)
            for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const vmi_f4*>(sum + ((size_t)s * nrb * bn + c) * H + h);
        *reinterpret_cast<uint2*>(dx + (size_t)t * H + h) = make_uint2(vmi_pack_bf16x2(v[0], v[1]), vmi_pack_bf16x2(v[2], v[3]));
    }
}

// ---------------------------------------------------------------------- host
template <int BN>
struct Shapes;
template <>
struct Shapes<256> {
    using Logit = Tile<256, 256, 2, 4, 2, false, false>;
    using Dx = Tile<256, 256, 2, 4, 2, true, false>;
};
template <>
struct Shapes<64> {
    using Logit = Tile<128, 64, 4, 2, 4, false, false>;
    using Dx = Tile<256, 64, 4, 2, 3, true, false>;
};
using DwTile = Tile<256, 256, 2, 4, 2, true, true>;

// Tokens of a tile.
int token_block(int T) { return T <= 64 ? 64 : 256; }

constexpr int64_t kPieceBytes = (int64_t)256 << 20;

struct Layout {
    int bn, Tp, piece;                // tokens of a block, T in whole blocks, vocabulary rows of a piece
    int64_t ldg;
    size_t idx, pos, meta, coef, part, hit, x, g, sum, bytes;
};

bool form_ok(int T, int H, int V) {
    return T >= 0 && T <= kMaxT && H > 0 && H % kBK == 0 && H <= kMaxH && V > 0 && V <= kMaxV;
}

Layout carve(int T, int H, int V, bool grad) {
    Layout l{};
    l.bn = token_block(T);
    l.Tp = std::max(1, (T + l.bn - 1) / l.bn) * l.bn;
    const int cus = vmi::device_cus();
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t p = at;
        at += vmi::align256(n);
        return p;
    };
    l.meta = take(256);
    l.idx = take((size_t)l.Tp * 4);
    l.pos = take((size_t)l.Tp * 4);
    l.coef = take((size_t)l.Tp * sizeof(Coef));
    if (!grad) {
        const size_t nrb = l.Tp / l.bn;
        l.part = take(std::max<size_t>(cus, 8 * nrb) * l.bn * sizeof(float2));
        l.hit = take((size_t)l.Tp * 4);
    } else {
        const int64_t all = ((int64_t)V + 255) / 256 * 256;
        const int64_t fit = std::max<int64_t>(8192, kPieceBytes / (2 * l.Tp) / 256 * 256);
        l.piece = (int)std::min(all, fit);
        l.ldg = l.piece + 64;         // off a power of two
        l.x = take((size_t)l.Tp * H * 2);
        l.g = take((size_t)l.Tp * l.ldg * 2);
        const int nht = (H + 255) / 256;
        const size_t rows = std::max<size_t>(l.Tp, (size_t)std::max(cus / nht, 1) * l.bn);
        l.sum = take(rows * H * 4);
    }
    l.bytes = at;
    return l;
}

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? VMI_OK : vmi::hip_fail(e, what);
}

int check_form(int T, int H, int V) {
    if (T < 0 || T > kMaxT) return vmi::fail(VMI_ERR_UNSUPPORTED, "T=%d must be in [0, %d]", T, kMaxT);
    if (H <= 0 || H % kBK || H > kMaxH)
        return vmi::fail(VMI_ERR_UNSUPPORTED, "hidden=%d must be a multiple of %d up to %d", H, kBK, kMaxH);
    if (V <= 0 || V > kMaxV) return vmi::fail(VMI_ERR_UNSUPPORTED, "vocab=%d must be in [1, %d]", V, kMaxV);
    return VMI_OK;
}
bool aligned(std::initializer_list<const void*> ps, uintptr_t to) {
    uintptr_t m = 0;
    for (const void* p : ps) m |= reinterpret_cast<uintptr_t>(p);
    return !(m & (to - 1));
}

template <int BN>
void launch_score(const LogitArgs& a, int grid, hipStream_t s) {
    hipLaunchKernelGGL((k_loss_score<typename Shapes<BN>::Logit>), dim3(grid), dim3(kThreads), 0, s, a);
}
template <int BN>
void launch_piece(const LogitArgs& a, const DxArgs* dx, int grid, hipStream_t s) {
    hipLaunchKernelGGL((k_loss_g<typename Shapes<BN>::Logit>), dim3(grid), dim3(kThreads), 0, s, a);
    if (dx) hipLaunchKernelGGL((k_loss_dx<typename Shapes<BN>::Dx>), dim3(grid), dim3(kThreads), 0, s, *dx);
}

}  // namespace

extern "C" size_t vmi_head_loss_workspace_bytes(int T, int hidden, int vocab) {
    return form_ok(T, hidden, vocab) ? carve(T, hidden, vocab, false).bytes : 0;
}

extern "C" int vmi_head_loss(const uint16_t* x, int T, int hidden, const uint16_t* weight, int vocab,
                             const int64_t* targets, int64_t ignore_index, float* loss, float* lse, uint32_t* status,
                             void* workspace, size_t workspace_bytes, void* stream) {
    vmi::clear_error();
    if (const int rc = check_form(T, hidden, vocab)) return rc;
    if (T == 0) return VMI_OK;
    if (!x || !weight || !targets || !loss || !lse) return vmi::fail(VMI_ERR_INVALID, "null x/weight/targets/loss/lse");
    if (!aligned({x, weight}, 16) || !aligned({targets}, 8))
        return vmi::fail(VMI_ERR_INVALID, "x and weight must be 16-byte aligned, targets 8");
    const Layout l = carve(T, hidden, vocab, false);
    if (!workspace || workspace_bytes < l.bytes || !aligned({workspace}, 256))
        return vmi::fail(VMI_ERR_WORKSPACE, "workspace needs %zu bytes, 256-byte aligned (got %zu)", l.bytes, workspace_bytes);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int grid = vmi::device_cus();
    RowsArgs r{};
    r.target = targets;
    r.ignore = ignore_index;
    r.T = T;
    r.Tp = l.Tp;
    r.V = vocab;
    r.idx = reinterpret_cast<int32_t*>(ws + l.idx);
    r.pos = reinterpret_cast<int32_t*>(ws + l.pos);
    r.meta = reinterpret_cast<int32_t*>(ws + l.meta);
    r.coef = reinterpret_cast<Coef*>(ws + l.coef);
    r.loss = loss;
    r.lse_out = lse;
    r.status = status;
    hipLaunchKernelGGL(k_loss_rows, dim3(1), dim3(1024), 0, s, r);
    LogitArgs a{};
    a.x = x;
    a.w = weight;
    a.idx = r.idx;
    a.meta = r.meta;
    a.coef = r.coef;
    a.H = hidden;
    a.V = vocab;
    a.part = reinterpret_cast<float2*>(ws + l.part);
    a.hit = reinterpret_cast<float*>(ws + l.hit);
    if (l.bn == 64)
        launch_score<64>(a, grid, s);
    else
        launch_score<256>(a, grid, s);
    hipLaunchKernelGGL(k_loss_merge, dim3((T + 3) / 4), dim3(256), 0, s, r.meta, r.idx, a.part, a.hit, l.bn, grid, loss, lse);
    return launched("k_loss_merge launch");
}

extern "C" size_t vmi_head_loss_grad_workspace_bytes(int T, int hidden, int vocab) {
    return form_ok(T, hidden, vocab) ? carve(T, hidden, vocab, true).bytes : 0;
}

extern "C" int vmi_head_loss_grad(const uint16_t* x, int T, int hidden, const uint16_t* weight, int vocab,
                                  const int64_t* targets, int64_t ignore_index, const float* lse, const float* d_loss,
                                  const float* d_lse, uint16_t* dx, void* dweight, int dweight_dtype, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    vmi::clear_error();
    if (const int rc = check_form(T, hidden, vocab)) return rc;
    if (!dx && !dweight) return vmi::fail(VMI_ERR_INVALID, "nothing to compute (dx and dweight both null)");
    if (dweight && dweight_dtype != VMI_BF16 && dweight_dtype != VMI_F32)
        return vmi::fail(VMI_ERR_UNSUPPORTED, "dweight_dtype %d", dweight_dtype);
    if (T && (!x || !weight || !targets || !lse || !d_loss))
        return vmi::fail(VMI_ERR_INVALID, "null x/weight/targets/lse/d_loss");
    if (!aligned({x, weight, dx, dweight}, 16) || !aligned({targets}, 8))
        return vmi::fail(VMI_ERR_INVALID, "x, weight, dx and dweight must be 16-byte aligned, targets 8");
    const Layout l = carve(T, hidden, vocab, true);
    if (!workspace || workspace_bytes < l.bytes || !aligned({workspace}, 256))
        return vmi::fail(VMI_ERR_WORKSPACE, "workspace needs %zu bytes, 256-byte aligned (got %zu)", l.bytes, workspace_bytes);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int grid = vmi::device_cus();
    RowsArgs r{};
    r.target = targets;
    r.ignore = ignore_index;
    r.T = T;
    r.Tp = l.Tp;
    r.V = vocab;
    r.idx = reinterpret_cast<int32_t*>(ws + l.idx);
    r.pos = reinterpret_cast<int32_t*>(ws + l.pos);
    r.meta = reinterpret_cast<int32_t*>(ws + l.meta);
    r.coef = reinterpret_cast<Coef*>(ws + l.coef);
    r.lse = lse;
    r.dloss = d_loss;
    r.dlse = d_lse;
    hipLaunchKernelGGL(k_loss_rows, dim3(1), dim3(1024), 0, s, r);
    uint16_t* xc = reinterpret_cast<uint16_t*>(ws + l.x);
    if (T)
        hipLaunchKernelGGL(k_loss_compact, dim3(l.Tp), dim3(256), 0, s, r.meta, r.idx, reinterpret_cast<const vmi_u4*>(x),
                           hidden / 8, reinterpret_cast<vmi_u4*>(xc));
    LogitArgs a{};
    a.x = xc;
    a.w = weight;
    a.meta = r.meta;
    a.coef = r.coef;
    a.H = hidden;
    a.V = vocab;
    a.g = reinterpret_cast<uint16_t*>(ws + l.g);
    a.ldg = l.ldg;
    DxArgs d{};
    d.w = weight;
    d.g = a.g;
    d.meta = r.meta;
    d.H = hidden;
    d.V = vocab;
    d.ldg = l.ldg;
    d.sum = reinterpret_cast<float*>(ws + l.sum);
    DwArgs u{};
    u.x = xc;
    u.g = a.g;
    u.meta = r.meta;
    u.H = hidden;
    u.V = vocab;
    u.ldg = l.ldg;
    u.dw = dweight;
    const int steps = (int)(((int64_t)vocab - 1) % l.piece / 256 + 1) * 256 / kBK;   // of the last piece, the shortest
    for (int v0 = 0; v0 < vocab; v0 += l.piece) {
        const int cols = std::min(l.piece, (vocab - v0 + 255) / 256 * 256);
        a.v0 = v0;
        a.v1 = v0 + cols;
        d.v0 = u.v0 = v0;
        d.cols = u.cols = cols;
        d.add = v0 != 0;
        d.short_steps = steps;
        if (T) {
            if (l.bn == 64)
                launch_piece<64>(a, dx ? &d : nullptr, grid, s);
            else
                launch_piece<256>(a, dx ? &d : nullptr, grid, s);
        }
        if (dweight) {
            if (dweight_dtype == VMI_F32)
                hipLaunchKernelGGL((k_loss_dw<DwTile, true>), dim3(grid), dim3(kThreads), 0, s, u);
            else
                hipLaunchKernelGGL((k_loss_dw<DwTile, false>), dim3(grid), dim3(kThreads), 0, s, u);
        }
    }
    if (dx && T)
        hipLaunchKernelGGL(k_loss_dx_out, dim3(T), dim3(256), 0, s, r.meta, r.pos, d.sum, hidden, l.bn, 256, grid, steps, dx);
    return launched("vmi_head_loss_grad launch");
}
