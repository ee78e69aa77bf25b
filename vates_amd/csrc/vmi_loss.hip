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
//   k_loss_logits   m a vocabulary row, n a token, k a hidden value: maxima and sums, or g
//   k_loss_dx       m a hidden value,   n a token, k a vocabulary row
//   k_loss_dw       m a hidden value,   n a vocabulary row, k a token
// An operand whose rows run along k lies in LDS as rows of 64 values, 16-byte pieces
// at piece ^ (row & 7); one whose rows run along m or n (W for dx, g for dW) as
// it is in memory, 32-byte pieces at piece ^ (k & 7), and ds_read_b64_tr_b16 turns 4 x 16
// values as they are read.  Both placements read without bank conflicts (4.7 and 4.3 cycles an
// instruction, as consecutive addresses do; rows unturned 12.6 and 16).
//
// g is rounded to bf16, the type of the matrix instruction's other operand (W, x): off by 2^-8 of its
// value at most, as much as a bf16 output's own rounding (647 tokens: dx 2.4e-3 from the 64-bit one, 1.7e-3 if only the output
// were rounded; dW in f32 1.7e-3, all of it g's).  Up to 64 tokens, where the head's
// bytes are the bound, what that leaves is multiplied too, in a second bf16.
//
// What bounds it (MI355X, 151,936 x 2048): one token 100 us, 6.7 TB/s of the head's bytes in the kernel
// (a read reaches 7.2); 8192 tokens 3.97 to 4.25 ms over the cards, 1.20 to 1.28 PFLOP/s; a step of 4096 with both gradients 8.8 ms,
// 1.16 PFLOP/s with z formed twice (a library product of these shapes 1.38 to 1.57): the matrix cores are busy 56 % of
// the cycles at 1.9 GHz, the library's 74 % at 1.6 (power).  Tried and slower: 32 of k a step in four or
// five stages (8192 tokens +7 %), 32 x 32 x 16 instructions (+6 %), a SIMD's two waves by turns in four phases a step
// (+10 %), operands read half a step ahead (spills at 256 registers), four waves of 128 x 128 (spills), tiles of 128 or 192
// vocabulary rows with three stages for some hundred tokens (+8 to 15 %), the head's lines of the step after next asked for
// into L2 (8192 tokens +5 %).  Where the rest goes at 8192 tokens, 4.06 ms: 3.77 if every line were in L2, 3.13 without the DMA,
// 3.83 with half the LDS reads; two stages of 64 KB are what LDS holds.
//
// Kernels beside them:
//   k_loss_rows     the tokens in the loss, and their coefficients
//   k_loss_merge    the strips' maxima and sums of a token joined
//   k_loss_turn     those tokens' x turned
//   k_loss_dx_out   the split sums of dx joined

#include <algorithm>
#include <type_traits>

#include "vmi_device.h"
#include "vmi_internal.h"

namespace {

constexpr int kThreads = 512, kWaves = 8, kBK = 64;
constexpr int kMaxT = 65536, kMaxH = 8192, kMaxV = 1 << 21;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;

__device__ __forceinline__ int ls_wave() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

// Two blocks' values, 4 q .. 4 q + 3 of 16 as two words each: eight in a row per lane, as
// rows 0 and 2 (16 lanes each) of the first block's and rows 1 and 3 of the second's.
__device__ __forceinline__ vmi_u4 ls_pair8(uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1) {
    const auto x = __builtin_amdgcn_permlane16_swap(a0, b0, false, false);
    const auto y = __builtin_amdgcn_permlane16_swap(a1, b1, false, false);
    return vmi_u4{x[0], y[0], x[1], y[1]};
}
// Where a lane's eight begin among the two blocks' 32.
__device__ __forceinline__ int ls_pair8_at() { return 16 * ((threadIdx.x >> 4) & 1) + 8 * ((threadIdx.x >> 5) & 1); }

// ------------------------------------------------------------------ products
// One workgroup's tile: BM x BN, waves WM x WN.  SLOW operands have k as the slow
// index (rows of BM or BN = 256 values).  ONCE: A is read by this workgroup alone.
template <int BM_, int BN_, int WM_, int WN_, int STAGES_, bool ASLOW_, bool BSLOW_, bool ONCE_ = false>
struct Tile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_;
    static constexpr bool ASLOW = ASLOW_, BSLOW = BSLOW_, ONCE = ONCE_;
    static constexpr int MB = BM / WM / 16, NB = BN / WN / 16;
    static constexpr int kA = BM * kBK * 2, kB = BN * kBK * 2, kStage = kA + kB;
    // kilobytes, one DMA instruction each, dealt to the waves in turn
    static constexpr int DA = kA / 1024 / kWaves, DB = (kB / 1024 + kWaves - 1) / kWaves, RB = kB / 1024 % kWaves;
    static_assert(WM * WN == kWaves && BM % (16 * WM) == 0 && BN % (16 * WN) == 0 && kA % (1024 * kWaves) == 0, "shape");
    static_assert((!ASLOW || BM == 256) && (!BSLOW || BN == 256), "slow operands have rows of 512 bytes");
};

// This workgroup's item in turn `turn` of n, or -1.  Workgroups go to the eight XCDs in
// turn, and each of these takes a run of consecutive items, which share operands in its L2.
__device__ __forceinline__ int ls_item(int turn, int n) {
    const int grid = gridDim.x, at = turn * grid, count = min(grid, n - at), chunk = (count + 7) / 8;
    const int x = blockIdx.x & 7, j = blockIdx.x >> 3, i = x * chunk + j;
    return j < chunk && i < count ? at + i : -1;
}
// The block of tokens and the strip of item i: eight blocks by all strips after another,
// so that a run of items is some blocks by some strips.
__device__ __forceinline__ void ls_pair(int i, int nrb, int strips, int& rb, int& strip) {
    const int group = i / (8 * strips), wide = min(8, nrb - 8 * group), j = i - group * 8 * strips;
    rb = 8 * group + j % wide;
    strip = j / wide;
}

// Row and 16-byte piece of a lane in the wave's DMA instruction i.
template <bool SLOW>
__device__ __forceinline__ void ls_slot(int i, int& row, int& piece) {
    const int lane = threadIdx.x & 63, u = ls_wave() + kWaves * i;
    if constexpr (SLOW) {   // two rows of 32 pieces
        row = 2 * u + (lane >> 5);
        const int s = lane & 31;
        piece = (((s >> 1) ^ (row & 7)) << 1) | (s & 1);
    } else {                // eight rows of eight
        row = 8 * u + (lane >> 3);
        piece = (lane & 7) ^ (row & 7);
    }
}
// D instructions, the last for the first R waves only (R: 0, all).
template <int D, int R, bool ONCE>
__device__ __forceinline__ void ls_dma(const void* base, const uint32_t (&off)[D], uint8_t* lds) {
    const int w = ls_wave();
#pragma unroll
    for (int i = 0; i < D; ++i) {
        if (R && i == D - 1 && w >= R) continue;
        if constexpr (ONCE)
            vmi_lds_dma16_at_nt(base, off[i], lds + (w + kWaves * i) * 1024);
        else
            vmi_lds_dma16_at(base, off[i], lds + (w + kWaves * i) * 1024);
    }
}
// Until the wave's oldest step is there: STAGES - 1 are in flight, and behind them the
// STORES instructions of the step before, where it ended a tile (vector memory
// operations of a wave end in the order of their issue).
template <class S, int STORES>
__device__ __forceinline__ void ls_wait() {
    constexpr int n = S::STAGES - 2;
    static_assert(n * (S::DA + S::DB) + STORES < 64, "the counter's range");
    if (S::RB == 0 || n == 0 || ls_wave() < S::RB)
        vmi_vm_wait_c<n * (S::DA + S::DB) + STORES>();
    else
        vmi_vm_wait_c<n * (S::DA + S::DB - 1) + STORES>();
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
        // by pairs, each product once both its operands are there
        constexpr int kMost = S::MB > S::NB ? S::MB : S::NB;
#pragma unroll
        for (int i = 0; i < kMost; ++i) {
            if (i < S::MB) a[i] = ls_operand<S::ASLOW>(lds, m0 + 16 * i, kk);
            if (i < S::NB) b[i] = ls_operand<S::BSLOW>(lds + S::kA, n0 + 16 * i, kk);
        }
#pragma unroll
        for (int i = 0; i < kMost; ++i) {
#pragma unroll
            for (int j = 0; j < i; ++j) {
                if (i < S::MB && j < S::NB) acc[i][j] = vmi_mfma_bf16(a[i], b[j], acc[i][j]);
                if (i < S::NB && j < S::MB) acc[j][i] = vmi_mfma_bf16(a[j], b[i], acc[j][i]);
            }
            if (i < S::MB && i < S::NB) acc[i][i] = vmi_mfma_bf16(a[i], b[i], acc[i][i]);
        }
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
// wait counts alike), job.wanted() says whether the wave's part of the tile has any row,
// job.done(acc) ends a step, takes a tile that is complete and says
// whether it has issued its STORES stores (all of them, whatever they cover).
template <class S, class Job>
__device__ __forceinline__ void ls_run(uint8_t* lds, Job& job, int total) {
    vmi_f4 acc[S::MB][S::NB];
    ls_clear<S>(acc);
    for (int s = 0; s < S::STAGES - 1; ++s) job.issue(lds + s * S::kStage);
    int in = S::STAGES - 1, out = 0;
    bool stored = false;
    for (int s = 0; s < total; ++s) {
        if (Job::STORES && stored)
            ls_wait<S, Job::STORES>();
        else
            ls_wait<S, 0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        job.issue(lds + in * S::kStage);
        in = in + 1 == S::STAGES ? 0 : in + 1;
        if (job.wanted()) ls_multiply<S>(lds + out * S::kStage, acc);
        out = out + 1 == S::STAGES ? 0 : out + 1;
        stored = job.done(acc);
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

// What k_loss_rows leaves for the kernels behind it.
struct Meta {
    int32_t nv;          // tokens in the loss
    int32_t bn;          // tokens of a tile
    int32_t strips;      // of the vocabulary, or of a whole piece of it
    int32_t last;        // of the last piece
    int32_t splits;      // sums of dx over the columns of a piece
};
__device__ __forceinline__ Meta ls_meta(const Meta* m) {
    const int32_t* p = &m->nv;
    return {vmi_sload_i32(p), vmi_sload_i32(p + 1), vmi_sload_i32(p + 2), vmi_sload_i32(p + 3), vmi_sload_i32(p + 4)};
}

// Up to 64 tokens every workgroup finds those in the loss by itself: lane t takes token t.
struct Few {
    const int64_t* target;
    int64_t ignore;
    int T, V;
    const float *lse, *dloss, *dlse;   // null for the loss
};
// Their number; the lane's place among them or -1; y: its target.
__device__ __forceinline__ int ls_few(const Few& f, int& place, int64_t& y) {
    const int lane = threadIdx.x & 63;
    y = f.target[min(lane, f.T - 1)];
    const bool in = lane < f.T && y >= 0 && y < f.V && y != f.ignore;
    const uint64_t all = __ballot(in);
    place = in ? __builtin_popcountll(all & ((1ull << lane) - 1)) : -1;
    return __builtin_popcountll(all);
}
// The same, their rows of x and coefficients into LDS (coefficients of `width` places: zeros behind the last).
__device__ __forceinline__ int ls_few(const Few& f, int width, int32_t* idx, Coef* coef) {
    const int lane = threadIdx.x & 63;
    int place;
    int64_t y;
    const int nv = ls_few(f, place, y);
    if (ls_wave() == 0) {
        if (coef && lane >= nv && lane < width) coef[lane] = Coef{0.0f, 0.0f, __builtin_inff(), -1};
        if (place >= 0) {
            idx[place] = lane;
            if (coef) {
                Coef c{0.0f, 0.0f, 0.0f, (int32_t)y};
                if (f.dloss) {
                    c.b = f.dloss[lane];
                    c.a = c.b + (f.dlse ? f.dlse[lane] : 0.0f);
                    c.lse = f.lse[lane];
                }
                coef[place] = c;
            }
        }
    }
    __syncthreads();
    return nv;
}

struct LogitArgs {
    Few few;                     // up to 64 tokens; else meta, idx and coef
    const uint16_t *x, *w;
    const int32_t* idx;
    const Meta* meta;
    const Coef* coef;
    int H, V;
    // score
    float2* part;                // [item][BN] maximum, sum
    float* hit;                  // [nv] the target's logit
    // gradient
    int v0, v1, last;            // the piece (v1 past V: columns of zeros), whether it is the last
    uint16_t* g;                 // [tokens][ldg]
    int64_t ldg;
};

// GRAD: 0 loss, 1 g, 2 g and, BN rows behind it, what its rounding left.
template <class S, int GRAD>
struct LogitJob {
    const LogitArgs& a;
    const Coef* coef;                 // LDS: the block's tokens
    int nv, rb, v1;                   // tokens, block, end of the strip
    int tile;                         // first row of the tile being multiplied
    int next, k, nk;                  // first row of the tile being asked for, its step, steps of one
    int turn;                         // step at which the tiles' rows are begun
    int kd;                           // step being multiplied
    uint32_t offa[S::DA], offb[S::DB];
    float m[S::NB], l[S::NB];
    int m0, n0;

    // idx: rows of x of the tokens in the loss; coef_: filled here from `from`, unless that is null
    __device__ __forceinline__ LogitJob(const LogitArgs& a_, const int32_t* idx, Coef* coef_, const Coef* from, int nv_, int rb_,
                                        int v0_, int v1_)
        : a(a_), coef(coef_), nv(nv_), rb(rb_), v1(v1_) {
        nk = a.H / kBK;
        // Rows of a few KB put the pieces that all workgroups ask for at one time on few memory channels; begun at
        // steps of their own, strips spread over them all (one token 129 -> 109 us, 100 tokens 156 -> 129).
        // Where blocks of tokens share a strip in an XCD's L2, groups of eight do.  Strips against groups, 151,936 x 2048:
        // 100 tokens 116 and 143 us, 300 (two blocks) 221 and 226, 640 (three) 397 and 400, 850 (four) 523 and 505,
        // 1000 591 and 567, 1280 730 and 692, 2048 1143 and 1076, 8192 alike.
        turn = nv <= 2 * S::BN ? v0_ / 16 % nk : (rb >> 3) * 11 % nk;
        tile = v0_;
        next = min(v0_, a.V - 1);   // (a piece's last tile may lie behind the vocabulary: its columns are zeros)
        k = kd = 0;
        const int w = ls_wave(), lane = threadIdx.x & 63;
        m0 = (w / S::WN) * (S::BM / S::WM) + 4 * (lane >> 4);
        n0 = (w % S::WN) * (S::BN / S::WN) + (lane & 15);
#pragma unroll
        for (int i = 0; i < S::DB; ++i) {
            int row, piece;
            ls_slot<false>(i, row, piece);
            const int c = min(rb * S::BN + row, nv - 1);
            offb[i] = (uint32_t)idx[c] * (uint32_t)(2 * a.H) + 16 * piece;
        }
        rows();
        if (from && threadIdx.x < S::BN) {
            const int t = rb * S::BN + threadIdx.x;
            coef_[threadIdx.x] = t < nv ? from[t] : Coef{0.0f, 0.0f, __builtin_inff(), -1};
        }
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            m[n] = kLowest;
            l[n] = 0.0f;
        }
    }
    __device__ __forceinline__ void rows() {
#pragma unroll
        for (int i = 0; i < S::DA; ++i) {
            int row, piece;
            ls_slot<false>(i, row, piece);
            offa[i] = (uint32_t)min(row, min(v1, a.V) - 1 - next) * (uint32_t)(2 * a.H) + 16 * piece;
        }
    }
    __device__ __forceinline__ void issue(uint8_t* lds) {
        const int kk = k + turn >= nk ? k + turn - nk : k + turn;
        // nontemporal where one block of tokens reads a strip (200 tokens 169 -> 165 us; with many 8192 took 4246, not 4058)
        const uint16_t* w = a.w + (size_t)next * a.H + (size_t)kk * kBK;
        if (S::ONCE || nv <= S::BN)
            ls_dma<S::DA, 0, true>(w, offa, lds);
        else
            ls_dma<S::DA, 0, false>(w, offa, lds);
        ls_dma<S::DB, S::RB, false>(a.x + (size_t)kk * kBK, offb, lds + S::kA);
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
    static constexpr int STORES = GRAD * S::MB * S::NB / (S::MB % 2 ? 1 : 2);
    __device__ __forceinline__ bool wanted() const { return tile + (ls_wave() / S::WN) * (S::BM / S::WM) < v1; }
    __device__ __forceinline__ bool done(vmi_f4 (&acc)[S::MB][S::NB]) {
        if (++kd < nk) return false;
        kd = 0;
        if constexpr (GRAD != 0)
            store(acc);
        else
            sum(acc);
        ls_clear<S>(acc);
        tile += S::BM;
        return true;
    }
    // Running maximum and sum of a lane's own rows of the tiles, joined over lanes at the end only.
    __device__ __forceinline__ void sum(vmi_f4 (&acc)[S::MB][S::NB]) {
        const int last = v1 - 1 - tile - m0;   // rows of the lane up to this one
        if (tile + S::BM > v1) {   // (below the maxima's start, so that they add nothing even where every logit is minus infinity)
#pragma unroll
            for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                for (int n = 0; n < S::NB; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (16 * mb + r > last) acc[mb][n][r] = -__builtin_inff();
        }
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            const int d = coef[n0 + 16 * n].target - tile - m0;
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
            // (a product's rounding before the difference would grow with the logits)
            float s = l[n] * __builtin_amdgcn_exp2f((m[n] - top) * kLog2e);
#pragma unroll
            for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                for (int r = 0; r < 4; ++r) s += __builtin_amdgcn_exp2f((acc[mb][n][r] - top) * kLog2e);
            m[n] = top;
            l[n] = s;
        }
    }
    __device__ __forceinline__ void store(vmi_f4 (&acc)[S::MB][S::NB]) {
        constexpr int W = S::MB % 2 ? 1 : 2;      // blocks of a store
        const int q = (threadIdx.x & 63) >> 4;
        // the block's rows of g from the tile's first column on (and, GRAD 2, those of the rest)
        const __amdgpu_buffer_rsrc_t rs = vmi_rsrc(a.g + (int64_t)rb * S::BN * a.ldg + (tile - a.v0), 0x7fffffffu);
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            const Coef c = coef[n0 + 16 * n];
            const int d = c.target - tile - m0;
            const bool in = rb * S::BN + n0 + 16 * n < nv;
            const uint32_t row = (uint32_t)(n0 + 16 * n) * (uint32_t)(2 * a.ldg);
#pragma unroll
            for (int mb = 0; mb < S::MB; mb += W) {
                uint32_t u[W][2], e[W][2];
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    float v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        v[r] = c.a * __builtin_amdgcn_exp2f((acc[mb + j][n][r] - c.lse) * kLog2e);
                        if (d == 16 * (mb + j) + r) v[r] -= c.b;
                        if (!in || tile + m0 + 16 * (mb + j) + r >= a.V) v[r] = 0.0f;
                    }
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        u[j][r] = vmi_pack_bf16x2(v[2 * r], v[2 * r + 1]);
                        e[j][r] = vmi_pack_bf16x2(v[2 * r] - __uint_as_float(u[j][r] << 16),
                                                  v[2 * r + 1] - __uint_as_float(u[j][r] & 0xffff0000u));
                    }
                }
                const int at = W == 2 ? m0 - 4 * q + 16 * mb + ls_pair8_at() : m0 + 16 * mb;
                const uint32_t off = tile + at < v1 ? row + 2 * at : VMI_OOB;   // (else another strip's)
                const uint32_t rest = off == VMI_OOB ? off : off + (uint32_t)S::BN * (uint32_t)(2 * a.ldg);
                if constexpr (W == 2) {
                    vmi_bstore_b128(ls_pair8(u[0][0], u[0][1], u[1][0], u[1][1]), rs, off, 0);
                    if (GRAD == 2) vmi_bstore_b128(ls_pair8(e[0][0], e[0][1], e[1][0], e[1][1]), rs, rest, 0);
                } else {
                    vmi_bstore_b64(make_uint2(u[0][0], u[0][1]), rs, off, 0);
                    if (GRAD == 2) vmi_bstore_b64(make_uint2(e[0][0], e[0][1]), rs, rest, 0);
                }
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
__device__ __forceinline__ void ls_score(const LogitArgs& a, const Meta& me, const int32_t* idx, uint8_t* lds, Coef* coef,
                                         const Coef* from) {
    const int nrb = (me.nv + S::BN - 1) / S::BN, per = ((a.V + me.strips - 1) / me.strips + 15) & ~15;
    for (int turn = 0; turn * (int)gridDim.x < nrb * me.strips; ++turn) {
        const int item = ls_item(turn, nrb * me.strips);
        if (item < 0) break;
        int rb, strip;
        ls_pair(item, nrb, me.strips, rb, strip);
        const int v0 = strip * per, v1 = min(a.V, v0 + per);
        float2* part = a.part + ((size_t)strip * nrb + rb) * S::BN;
        if (v0 >= v1) {
            if (threadIdx.x < S::BN) part[threadIdx.x] = make_float2(kLowest, 0.0f);
            continue;
        }
        LogitJob<S, 0> job(a, idx, coef, from, me.nv, rb, v0, v1);
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
template <class S, int GRAD>
__device__ __forceinline__ void ls_g(const LogitArgs& a, const Meta& me, const int32_t* idx, uint8_t* lds, Coef* coef,
                                     const Coef* from) {
    const int nrb = (me.nv + S::BN - 1) / S::BN, strips = a.last ? me.last : me.strips;
    const int per = ((a.v1 - a.v0 + strips - 1) / strips + 15) & ~15;
    for (int turn = 0; turn * (int)gridDim.x < nrb * strips; ++turn) {
        const int item = ls_item(turn, nrb * strips);
        if (item < 0) break;
        int rb, strip;
        ls_pair(item, nrb, strips, rb, strip);
        const int v0 = a.v0 + strip * per, v1 = min(a.v1, v0 + per);
        if (v0 >= v1) continue;
        LogitJob<S, GRAD> job(a, idx, coef, from, me.nv, rb, v0, v1);
        ls_run<S>(lds, job, (v1 - v0 + S::BM - 1) / S::BM * job.nk);
    }
}

// Tiles by tokens of a block.  Up to 64 tokens the head is read once, by one workgroup each
// part of it, and its bytes bound the call; above, five widths, of which k_loss_rows takes the one with the least work.
constexpr int kFew = 64, kFewest = 32;
using Score32 = Tile<128, 32, 8, 1, 4, false, false, true>;
using Score64 = Tile<128, 64, 4, 2, 4, false, false, true>;
template <int BN>
using ScoreN = Tile<256, BN, 4, 2, BN <= 160 ? 3 : 2, false, false>;
template <class S>
constexpr int kLds = S::STAGES * S::kStage;

// WHICH: 32, 64, or 0 for the widths above.
template <int WHICH, int GRAD>
__global__ __launch_bounds__(kThreads) void k_loss_logits(LogitArgs a) {
    constexpr int kBytes = WHICH == 32 ? kLds<Score32> : WHICH == 64 ? kLds<Score64> : kLds<ScoreN<160>>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kBytes];
    __shared__ Coef coef[WHICH ? WHICH : 256];
    __shared__ int32_t s_idx[WHICH ? WHICH : 1];
    Meta me{0, WHICH, (int)gridDim.x, (int)gridDim.x, 1};   // few: one strip a workgroup, bytes bound it
    if constexpr (WHICH)
        me.nv = ls_few(a.few, WHICH, s_idx, coef);
    else
        me = ls_meta(a.meta);
    if (me.nv == 0) return;
    const int32_t* idx = WHICH ? s_idx : a.idx;
    const Coef* from = WHICH ? nullptr : a.coef;
    auto go = [&](auto s) {
        using S = decltype(s);
        static_assert(kLds<S> <= kBytes, "LDS");
        if constexpr (GRAD)
            ls_g<S, GRAD>(a, me, idx, lds, coef, from);
        else
            ls_score<S>(a, me, idx, lds, coef, from);
    };
    if constexpr (WHICH == 32) {
        go(Score32{});
    } else if constexpr (WHICH == 64) {
        go(Score64{});
    } else {
        switch (me.bn) {
            case 128: go(ScoreN<128>{}); break;
            case 160: go(ScoreN<160>{}); break;
            case 192: go(ScoreN<192>{}); break;
            case 224: go(ScoreN<224>{}); break;
            default: go(ScoreN<256>{}); break;
        }
    }
}

// ------------------------------------------------------------------------ dx
// Splits of dx's sums over the columns: as many workgroups as the grid has, of four steps at least.
__host__ __device__ __forceinline__ int ls_splits(int grid, int blocks, int nht, int steps) {
    const int fill = grid / (blocks * nht), deep = steps / 4, n = fill < deep ? fill : deep;
    return n > 1 ? n : 1;
}

struct DxArgs {
    const uint16_t *w, *g;
    const Meta* meta;
    int H, V, v0, cols;      // the piece's first row, its columns of g (a multiple of 64)
    int64_t ldg;
    float* sum;              // [split][token block rows][H]
    int add;                 // a later piece than the first: added to the sums
    int splits;              // up to 64 tokens (else meta's)
    Few tokens;              // the same: without one in the loss g isn't there
};

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
            ls_slot<false>(i, row, piece);
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
            ls_slot<true>(i, row, piece);
            const int col = min(ht * S::BM + 8 * piece, a.H - 8);
            offa[i] = (uint32_t)(max(min(row, rows - 1), 0)) * (uint32_t)(2 * a.H) + 2 * col;
        }
        ls_dma<S::DA, 0, S::ONCE>(a.w + (size_t)(a.v0 + base) * a.H, offa, lds);
        ls_dma<S::DB, S::RB, false>(a.g + (int64_t)rb * S::BN * a.ldg + kn, offb, lds + S::kA);
        if (--left > 0) kn += kBK;
    }
    static constexpr int STORES = 0;   // (its tiles end the run)
    __device__ __forceinline__ bool wanted() const { return true; }
    __device__ __forceinline__ bool done(vmi_f4 (&acc)[S::MB][S::NB]) {
        if (++kd < steps) return false;
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
        return false;
    }
};

// Tiles of 256 hidden values by a block of tokens; where these leave CUs idle the
// piece's columns are split over several workgroups, each with sums of its own.
template <class S>
__device__ __forceinline__ void ls_dx(const DxArgs& a, int nrb, int splits, uint8_t* lds) {
    const int nht = (a.H + S::BM - 1) / S::BM, steps = a.cols / kBK;
    for (int turn = 0; turn * (int)gridDim.x < splits * nht * nrb; ++turn) {
        const int item = ls_item(turn, splits * nht * nrb);
        if (item < 0) break;
        const int rb = item % nrb, ht = item / nrb % nht, sp = item / nrb / nht;
        const int k0 = (int)((int64_t)steps * sp / splits), k1 = (int)((int64_t)steps * (sp + 1) / splits);
        DxJob<S> job(a, ht, rb, sp, nrb, k0, k1);
        ls_run<S>(lds, job, k1 - k0);
    }
}

// Up to 64 tokens: g and its rest side by side as tokens of one block.
using Dx32 = Tile<256, 64, 4, 2, 3, true, false, true>;
using Dx64 = Tile<256, 128, 4, 2, 3, true, false, true>;
template <int BN>
using DxN = Tile<256, BN, 4, 2, BN <= 160 ? 3 : 2, true, false, true>;

template <int WHICH>
__global__ __launch_bounds__(kThreads) void k_loss_dx(DxArgs a) {
    constexpr int kBytes = WHICH == 32 ? kLds<Dx32> : WHICH == 64 ? kLds<Dx64> : kLds<DxN<160>>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kBytes];
    if constexpr (WHICH) {
        int place;
        int64_t y;
        if (ls_few(a.tokens, place, y) == 0) return;
        ls_dx<std::conditional_t<WHICH == 32, Dx32, Dx64>>(a, 1, a.splits, lds);
    } else {
        const Meta me = ls_meta(a.meta);
        if (me.nv == 0) return;
        auto go = [&](auto s) {
            using S = decltype(s);
            static_assert(kLds<S> <= kBytes, "LDS");
            ls_dx<S>(a, (me.nv + S::BN - 1) / S::BN, me.splits, lds);
        };
        switch (me.bn) {
            case 128: go(DxN<128>{}); break;
            case 160: go(DxN<160>{}); break;
            case 192: go(DxN<192>{}); break;
            case 224: go(DxN<224>{}); break;
            default: go(DxN<256>{}); break;
        }
    }
}

// ------------------------------------------------------------------------ dW
// x as [hidden][token] of the tokens in the loss (ldx values a row), its own rows by idx where there are few.
struct DwArgs {
    const uint16_t *x, *g;
    const Meta* meta;
    int H, V, v0, cols;
    int64_t ldg, ldx;
    void* dw;
    Few tokens;              // where there are few: and g in two parts of `few` tokens each
    int few;
};

template <class S, bool F32>
struct DwJob {
    const DwArgs& a;
    const int32_t* idx;
    int nv, nk, nht, items;
    int turn, item, step;                // asked for
    int kd, done_turn;                   // being multiplied
    uint32_t offa[S::DA], offb[S::DB];

    __device__ __forceinline__ DwJob(const DwArgs& a_, const int32_t* idx_, int nv_, int nk_, int nht_, int items_)
        : a(a_), idx(idx_), nv(nv_), nk(nk_), nht(nht_), items(items_), turn(0), item(ls_item(0, items_)), step(0), kd(0), done_turn(0) {
        rows();
    }
    __device__ __forceinline__ void rows() {
        const int ht = item % nht, vt = item / nht;
#pragma unroll
        for (int i = 0; i < S::DA; ++i) {
            int row, piece;
            ls_slot<S::ASLOW>(i, row, piece);
            if constexpr (S::ASLOW)   // few tokens, by idx (g is zero behind the last)
                offa[i] = (uint32_t)idx[min(row & (a.few - 1), nv - 1)] * (uint32_t)(2 * a.H) +
                          2 * min(ht * S::BM + 8 * piece, a.H - 8);
            else
                offa[i] = (uint32_t)min(ht * S::BM + row, a.H - 1) * (uint32_t)(2 * a.ldx) + 16 * piece;
        }
#pragma unroll
        for (int i = 0; i < S::DB; ++i) {
            int row, piece;
            ls_slot<true>(i, row, piece);
            offb[i] = (uint32_t)row * (uint32_t)(2 * a.ldg) + 2 * (vt * S::BN + 8 * piece);
        }
    }
    __device__ __forceinline__ void issue(uint8_t* lds) {
        ls_dma<S::DA, 0, false>(a.x + (S::ASLOW ? 0 : step * kBK), offa, lds);
        ls_dma<S::DB, S::RB, false>(a.g + (int64_t)step * kBK * a.ldg, offb, lds + S::kA);
        if (++step == nk) {
            const int next = (turn + 1) * (int)gridDim.x < items ? ls_item(turn + 1, items) : -1;
            if (next >= 0) {
                ++turn;
                item = next;
                step = 0;
                rows();
            } else {
                step = nk - 1;
            }
        }
    }
    static constexpr int STORES = S::MB * S::NB / (F32 ? 1 : 2);
    __device__ __forceinline__ bool wanted() const { return true; }
    __device__ __forceinline__ bool done(vmi_f4 (&acc)[S::MB][S::NB]) {
        if (++kd < nk) return false;
        kd = 0;
        write(acc);
        ls_clear<S>(acc);
        return true;
    }
    __device__ __forceinline__ void write(vmi_f4 (&acc)[S::MB][S::NB]) {
        const int w = ls_wave(), lane = threadIdx.x & 63, at = ls_item(done_turn++, items);
        constexpr int e = F32 ? 4 : 2;
        const int m0 = at % nht * S::BM + (w / S::WN) * (S::BM / S::WM) + 4 * (lane >> 4);
        const int first = a.v0 + at / nht * S::BN, n0 = (w % S::WN) * (S::BN / S::WN) + (lane & 15);
        const __amdgpu_buffer_rsrc_t rs = vmi_rsrc(static_cast<uint8_t*>(a.dw) + (size_t)first * a.H * e, 0x7fffffffu);
#pragma unroll
        for (int n = 0; n < S::NB; ++n)
#pragma unroll
            for (int mb = 0; mb < S::MB; mb += F32 ? 1 : 2) {
                const int h = F32 ? m0 + 16 * mb : m0 - 4 * (lane >> 4) + 16 * mb + ls_pair8_at();
                const uint32_t off = first + n0 + 16 * n < a.V && h < a.H ? (uint32_t)((n0 + 16 * n) * a.H + h) * e : VMI_OOB;
                const vmi_f4 v = acc[mb][n], u = acc[mb + (F32 ? 0 : 1)][n];
                if constexpr (F32)
                    vmi_bstore_b128(__builtin_bit_cast(vmi_u4, v), rs, off, 0);
                else
                    vmi_bstore_b128(ls_pair8(vmi_pack_bf16x2(v[0], v[1]), vmi_pack_bf16x2(v[2], v[3]),
                                             vmi_pack_bf16x2(u[0], u[1]), vmi_pack_bf16x2(u[2], u[3])), rs, off, 0);
            }
    }
};

template <bool FEW, bool F32>
__global__ __launch_bounds__(kThreads) void k_loss_dw(DwArgs a) {
    using S = Tile<256, 256, 2, 4, 2, FEW, true>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds<S>];
    __shared__ int32_t s_idx[FEW ? kFew : 1];
    int nv = 0;
    if constexpr (FEW) {
        s_idx[threadIdx.x & (kFew - 1)] = 0;
        __syncthreads();
        if (a.tokens.T) nv = ls_few(a.tokens, 0, s_idx, nullptr);
    } else {
        nv = vmi_sload_i32(&a.meta->nv);
    }
    const int nk = nv ? ((FEW ? 2 * a.few : nv) + kBK - 1) / kBK : 0;
    const int nht = (a.H + S::BM - 1) / S::BM, items = nht * ((a.cols + S::BN - 1) / S::BN);
    if (ls_item(0, items) < 0) return;
    DwJob<S, F32> job(a, s_idx, max(nv, 1), max(nk, 1), nht, items);
    const int whole = items / (int)gridDim.x;    // turns in which every workgroup has an item; the last may leave some out
    const int mine = whole + (whole * (int)gridDim.x < items && ls_item(whole, items) >= 0 ? 1 : 0);
    if (nk == 0) {   // no token in the loss: zeros
        vmi_f4 acc[S::MB][S::NB];
        ls_clear<S>(acc);
        for (int i = 0; i < mine; ++i) job.write(acc);
        return;
    }
    ls_run<S>(lds, job, mine * nk);
}

// --------------------------------------------------------------- small kernels
struct RowsArgs {
    const int64_t* target;
    int64_t ignore;
    int T, V;
    int32_t *idx, *pos;            // tokens in the loss, each token's place among them or -1
    Meta* meta;
    Coef* coef;                    // of the tokens in the loss
    float *loss, *lse_out;         // score: written for tokens left out
    uint32_t* status;
    const float *lse, *dloss, *dlse;
    int grid;                      // workgroups of the products
    int tiles, last, nht, steps;   // vocabulary tiles of a piece and of the last one, hidden tiles, dx's steps of the last piece
};

constexpr int kMaxItems = 4;       // workgroups' turns at most that the strips are cut for

// The least work, in tokens' widths of a tile, of `tiles` cut into s strips by nrb blocks
// of bn tokens: turns of the grid times a turn's tiles in quarters, which the waves behind a strip's end leave out (a tile's own
// cost beside its products about 16 tokens: counted as none, 1200 tokens over 151,936 x 2048 took 746 us for 688, 4096 2390 for
// 2100; as 32 the same as 16.  A turn's, 24: none or 48 changed no size tried by more than 1 %); lane l tries s = l + 1, l + 65, ..  Returns work * 2^16 + s.
__device__ __forceinline__ uint64_t ls_plan(int nrb, int bn, int tiles, int grid) {
    const int most = min(tiles, max(1, kMaxItems * grid / nrb));
    const float per_grid = (float)nrb / (float)grid;
    uint64_t best = ~0ull;
    for (int s = (threadIdx.x & 63) + 1; s <= most; s += 64) {
        // rounded up, whole quotients off by a division's rounding left whole
        const float turns = ceilf((float)s * per_grid - 1e-3f);
        const float deep = 0.25f * ceilf(4.0f * (float)tiles * __builtin_amdgcn_rcpf((float)s) - 1e-3f);
        best = min(best, (uint64_t)(turns * fmaf(deep, (float)(bn + 16), 24.0f)) << 16 | (uint64_t)s);
    }
    return ~vmi_wave_max_u64(~best);
}

// More than 64 tokens.  One workgroup: a wave takes a run of tokens, 64 at a time, eight such groups' loads together.
__global__ __launch_bounds__(1024) void k_loss_rows(RowsArgs a) {
    __shared__ int s_sum[16];
    __shared__ uint64_t s_work[5];
    __shared__ uint32_t s_cut[5];
    const int lane = threadIdx.x & 63, w = ls_wave(), run = (a.T + 1023) / 1024 * 64;
    const int t0 = min(a.T, w * run), t1 = min(a.T, t0 + run);
    constexpr int kAhead = 8;
    int64_t y[kAhead];
    Coef k[kAhead];
    auto load = [&](int t, bool coef) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int at = min(t + 64 * i + lane, a.T - 1);
            y[i] = a.target[at];
            k[i] = Coef{0.0f, 0.0f, 0.0f, 0};
            if (coef && a.dloss) k[i] = Coef{a.dlse ? a.dlse[at] : 0.0f, a.dloss[at], a.lse[at], 0};
        }
    };
    auto in = [&](int i) { return y[i] >= 0 && y[i] < a.V && y[i] != a.ignore; };
    int n = 0;
    bool bad = false;
    // (backward, so that the first groups, all there are up to 8192 tokens, are still held when they are placed)
    for (int t = t0 + (t1 - t0 - 1) / (64 * kAhead) * (64 * kAhead); t >= t0 && t < t1; t -= 64 * kAhead) {
        load(t, t == t0);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const bool here = t + 64 * i + lane < t1;
            n += __builtin_popcountll(__ballot(here && in(i)));
            bad |= here && !in(i) && y[i] != a.ignore;
        }
    }
    if (a.status && __any(bad) && lane == 0) atomicOr(a.status, VMI_STATUS_BAD_TARGET);
    if (lane == 0) s_sum[w] = n;
    __syncthreads();
    int c = 0, nv = 0;
    for (int i = 0; i < 16; ++i) {
        c += i < w ? s_sum[i] : 0;
        nv += s_sum[i];
    }
    for (int t = t0; t < t1; t += 64 * kAhead) {
        if (t != t0) load(t, true);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int at = t + 64 * i + lane;
            const bool here = at < t1;
            const uint64_t all = __ballot(here && in(i));
            const int mine = c + __builtin_popcountll(all & ((1ull << lane) - 1));
            c += __builtin_popcountll(all);
            if (here) a.pos[at] = in(i) ? mine : -1;
            if (here && in(i)) {
                a.idx[mine] = at;
                k[i].a += k[i].b;
                k[i].target = (int32_t)y[i];
                a.coef[mine] = k[i];
            } else if (here && a.loss) {
                a.loss[at] = a.lse_out[at] = y[i] == a.ignore ? 0.0f : __builtin_nanf("");
            }
        }
    }
    // waves 0 to 4 weigh a width each
    if (nv && w < 5) {
        const int bn = 256 - 32 * w, nrb = (nv + bn - 1) / bn;
        const uint64_t p = ls_plan(nrb, bn, a.tiles, a.grid), q = a.last == a.tiles ? p : ls_plan(nrb, bn, a.last, a.grid);
        if (lane == 0) {
            s_work[w] = p >> 16;
            s_cut[w] = (uint32_t)(p & 0xffffu) | (uint32_t)(q & 0xffffu) << 16;
        }
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    Meta me{nv, 256, 1, 1, 1};
    if (nv) {
        int best = 0;
        for (int i = 1; i < 5; ++i) best = s_work[i] < s_work[best] ? i : best;
        me.bn = 256 - 32 * best;
        me.strips = (int)(s_cut[best] & 0xffffu);
        me.last = (int)(s_cut[best] >> 16);
    }
    const int blocks = max((nv + me.bn - 1) / me.bn, 1);
    me.splits = ls_splits(a.grid, blocks, a.nht, a.steps);
    *a.meta = me;
}

// The strips' maxima and sums of a token in the loss, joined by a wave in a fixed order.
__device__ __forceinline__ void ls_merge(const Meta& me, int c, int t, const float2* part, const float* hit, float* loss, float* lse) {
    const int lane = threadIdx.x & 63, nrb = (me.nv + me.bn - 1) / me.bn, rb = c / me.bn;
    float m = kLowest, l = 0.0f;
    for (int s = lane; s < me.strips; s += 64) {
        const float2 p = part[((size_t)s * nrb + rb) * me.bn + c % me.bn];
        ls_join(m, l, p.x, p.y);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) ls_join(m, l, __shfl_xor(m, d), __shfl_xor(l, d));
    if (lane == 0) {
        // (m - z is exact near m, and 0 for a token foreseen: lse - z would round log l to a step of the logits' size first)
        const float v = logf(l);
        lse[t] = m + v;
        loss[t] = m - hit[c] + v;
    }
}
// A wave per token in the loss.
__global__ __launch_bounds__(256) void k_loss_merge(const Meta* meta, const int32_t* idx, const float2* part,
                                                    const float* hit, float* loss, float* lse) {
    const Meta me = ls_meta(meta);
    const int c = blockIdx.x * 4 + ls_wave();
    if (c < me.nv) ls_merge(me, c, idx[c], part, hit, loss, lse);
}
// A wave per token of few, those left out among them.
__global__ __launch_bounds__(256) void k_loss_merge_few(Few f, int few, int strips, const float2* part, const float* hit,
                                                        float* loss, float* lse, uint32_t* status) {
    const int t = blockIdx.x * 4 + ls_wave();
    int place;
    int64_t y;
    const int nv = ls_few(f, place, y);
    if (t >= f.T) return;
    const int c = __builtin_amdgcn_readlane(place, t);
    if (c >= 0) {
        ls_merge(Meta{nv, few, strips, strips, 1}, c, t, part, hit, loss, lse);
    } else if ((int)(threadIdx.x & 63) == t) {
        const bool bad = y != f.ignore;
        loss[t] = lse[t] = bad ? __builtin_nanf("") : 0.0f;
        if (bad && status) atomicOr(status, VMI_STATUS_BAD_TARGET);
    }
}

// x of the tokens in the loss turned, out[h][c], zeros from nv on: the head's gradient then
// reads one operand of its two along memory (both turned as they were read, LDS took longer than the
// products: 4096 tokens 2.5 -> 2.3 ms).  64 tokens by 64 hidden values a workgroup.  Blocks of 160 or 224 tokens may end
// inside the last 64: g's rows behind them, which no piece writes, are zeros too.
__global__ __launch_bounds__(256) void k_loss_turn(const Meta* meta, const int32_t* idx, const uint16_t* x, int H, int64_t ldx,
                                                   uint16_t* out, uint16_t* g, int64_t ldg) {
    __shared__ uint32_t s_x[64][33];
    const Meta me = ls_meta(meta);
    const int nv = me.nv, c0 = blockIdx.x * 64, h0 = blockIdx.y * 64, t = threadIdx.x;
    for (int r = (nv + me.bn - 1) / me.bn * me.bn; r < (nv + kBK - 1) / kBK * kBK; ++r)
        for (int c = 8 * ((blockIdx.y * gridDim.x + blockIdx.x) * 256 + t); c < ldg; c += 8 * 256 * gridDim.x * gridDim.y)
            *reinterpret_cast<vmi_u4*>(g + r * ldg + c) = vmi_u4{0, 0, 0, 0};
    if (c0 >= (nv + kBK - 1) / kBK * kBK) return;
    for (int i = t; i < 64 * 8; i += 256) {
        const int c = i >> 3, u = i & 7;
        vmi_u4 v = {0, 0, 0, 0};
        if (c0 + c < nv) v = *reinterpret_cast<const vmi_u4*>(x + (size_t)idx[c0 + c] * H + h0 + 8 * u);
        for (int j = 0; j < 4; ++j) s_x[c][4 * u + j] = v[j];
    }
    __syncthreads();
    for (int i = t; i < 64 * 8; i += 256) {
        const int h = i >> 3, u = i & 7, sh = 16 * (h & 1);
        vmi_u4 v;
        for (int j = 0; j < 4; ++j)
            v[j] = ((s_x[8 * u + 2 * j][h >> 1] >> sh) & 0xffffu) | ((s_x[8 * u + 2 * j + 1][h >> 1] >> sh) << 16);
        *reinterpret_cast<vmi_u4*>(out + (int64_t)(h0 + h) * ldx + c0 + 8 * u) = v;
    }
}

// dx of a token: the n sums of its row of `rows` in a fixed order (few: those of g's two
// parts, few rows apart), zeros for a token left out.  A wave takes 256 hidden values;
// SPREAD: the workgroup's four waves share one such piece's sums (few tokens of many splits: 22 -> 7 us; with 200 tokens both take 19).
template <bool SPREAD>
__device__ __forceinline__ void ls_dx_out(int t, int c, int n, int rows, int few, const float* sum, int H, uint16_t* dx) {
    __shared__ vmi_f4 s_part[SPREAD ? 3 : 1][64];
    const int lane = threadIdx.x & 63, w = ls_wave(), h = 256 * (SPREAD ? blockIdx.y : 4 * blockIdx.y + w) + 4 * lane;
    vmi_f4 v = {0.f, 0.f, 0.f, 0.f};
    if (c >= 0 && h < H) {
        constexpr int kAhead = 8;
        const int i0 = SPREAD ? n * w / 4 : 0, i1 = SPREAD ? n * (w + 1) / 4 : n;
        for (int i = i0; i < i1; i += kAhead) {
            vmi_f4 u[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int p = min(i + j, i1 - 1), s = few ? p >> 1 : p;
                u[j] = *reinterpret_cast<const vmi_f4*>(sum + ((size_t)s * rows + c + (few && (p & 1) ? few : 0)) * H + h);
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (i + j < i1) v += u[j];
        }
    }
    if constexpr (SPREAD) {
        if (w) s_part[w - 1][lane] = v;
        __syncthreads();
        if (w) return;
        for (int i = 0; i < 3; ++i) v += s_part[i][lane];
    }
    if (h < H)
        *reinterpret_cast<uint2*>(dx + (size_t)t * H + h) = make_uint2(vmi_pack_bf16x2(v[0], v[1]), vmi_pack_bf16x2(v[2], v[3]));
}
__global__ __launch_bounds__(256) void k_loss_dx_out(const Meta* meta, const int32_t* pos, const float* sum, int H, uint16_t* dx) {
    const Meta me = ls_meta(meta);
    const int t = blockIdx.x;
    ls_dx_out<false>(t, pos[t], me.splits, (me.nv + me.bn - 1) / me.bn * me.bn, 0, sum, H, dx);
}
__global__ __launch_bounds__(256) void k_loss_dx_out_few(Few f, int few, int splits, const float* sum, int H, uint16_t* dx) {
    int place;
    int64_t y;
    ls_few(f, place, y);
    const int t = blockIdx.x;
    ls_dx_out<true>(t, __builtin_amdgcn_readlane(place, t), 2 * splits, 2 * few, few, sum, H, dx);
}

// ---------------------------------------------------------------------- host
constexpr int64_t kPieceBytes = (int64_t)512 << 20;

struct Layout {
    int few, rows, piece;             // tokens of the one block where there are few, rows of g, vocabulary rows of a piece
    int64_t ldg, ldx;
    size_t idx, pos, meta, coef, part, hit, x, g, sum, bytes;
};

int workgroups() { return std::max(8, vmi::device_cus() & ~7); }   // one a CU, alike on the eight XCDs

bool form_ok(int T, int H, int V) {
    return T >= 0 && T <= kMaxT && H > 0 && H % kBK == 0 && H <= kMaxH && V > 0 && V <= kMaxV;
}

Layout carve(int T, int H, int V, bool grad) {
    Layout l{};
    l.few = T <= kFewest ? kFewest : T <= kFew ? kFew : 0;
    l.rows = l.few ? 2 * l.few : (T + 255 + 63) / 64 * 64;   // whole blocks of any width end below T + 256
    const int cus = workgroups();
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t p = at;
        at += vmi::align256(n);
        return p;
    };
    l.meta = take(sizeof(Meta));
    l.idx = take((size_t)T * 4);
    l.pos = take((size_t)T * 4);
    l.coef = take((size_t)T * sizeof(Coef));
    if (!grad) {
        // items: a strip for every block at least, kMaxItems turns at most
        const size_t blocks = (T + 127) / 128;
        l.part = take(std::max<size_t>((size_t)kMaxItems * cus, blocks) * (l.few ? l.few : 256) * sizeof(float2));
        l.hit = take((size_t)l.rows * 4);
    } else {
        const int64_t all = ((int64_t)V + 255) / 256 * 256;
        const int64_t fit = std::max<int64_t>(8192, kPieceBytes / (2 * l.rows)), n = (all + fit - 1) / fit;
        l.piece = (int)((all / 256 + n - 1) / n * 256);   // pieces alike
        l.ldg = l.piece + 64;         // off a power of two
        l.ldx = l.rows + 64;
        l.x = take(l.few ? 0 : (size_t)l.ldx * H * 2);
        l.g = take((size_t)l.rows * l.ldg * 2);
        const int nht = (H + 255) / 256;
        l.sum = take(((size_t)l.rows + (size_t)std::max(cus / nht, 1) * (l.few ? 2 * l.few : 256)) * H * 4);
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

RowsArgs rows_args(const int64_t* target, int64_t ignore, int T, int V, const Layout& l, uint8_t* ws, int grid) {
    RowsArgs r{};
    r.target = target;
    r.ignore = ignore;
    r.T = T;
    r.V = V;
    r.idx = reinterpret_cast<int32_t*>(ws + l.idx);
    r.pos = reinterpret_cast<int32_t*>(ws + l.pos);
    r.meta = reinterpret_cast<Meta*>(ws + l.meta);
    r.coef = reinterpret_cast<Coef*>(ws + l.coef);
    r.grid = grid;
    return r;
}
template <int GRAD>
void launch_logits(const LogitArgs& a, int few, int grid, hipStream_t s) {
    constexpr int kSmall = GRAD ? 2 : 0;   // few tokens: g in two parts
    if (few == 32)
        hipLaunchKernelGGL((k_loss_logits<32, kSmall>), dim3(grid), dim3(kThreads), 0, s, a);
    else if (few == 64)
        hipLaunchKernelGGL((k_loss_logits<64, kSmall>), dim3(grid), dim3(kThreads), 0, s, a);
    else
        hipLaunchKernelGGL((k_loss_logits<0, GRAD>), dim3(grid), dim3(kThreads), 0, s, a);
}
void launch_dx(const DxArgs& a, int few, int grid, hipStream_t s) {
    if (few == 32)
        hipLaunchKernelGGL((k_loss_dx<32>), dim3(grid), dim3(kThreads), 0, s, a);
    else if (few == 64)
        hipLaunchKernelGGL((k_loss_dx<64>), dim3(grid), dim3(kThreads), 0, s, a);
    else
        hipLaunchKernelGGL((k_loss_dx<0>), dim3(grid), dim3(kThreads), 0, s, a);
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
    const int grid = workgroups();
    LogitArgs a{};
    a.x = x;
    a.w = weight;
    a.H = hidden;
    a.V = vocab;
    a.part = reinterpret_cast<float2*>(ws + l.part);
    a.hit = reinterpret_cast<float*>(ws + l.hit);
    if (l.few) {
        a.few = Few{targets, ignore_index, T, vocab, nullptr, nullptr, nullptr};
        launch_logits<0>(a, l.few, grid, s);
        hipLaunchKernelGGL(k_loss_merge_few, dim3((T + 3) / 4), dim3(256), 0, s, a.few, l.few, grid, a.part, a.hit, loss, lse, status);
        return launched("k_loss_merge_few launch");
    }
    RowsArgs r = rows_args(targets, ignore_index, T, vocab, l, ws, grid);
    r.loss = loss;
    r.lse_out = lse;
    r.status = status;
    r.tiles = r.last = (vocab + 255) / 256;
    r.nht = r.steps = 1;
    hipLaunchKernelGGL(k_loss_rows, dim3(1), dim3(1024), 0, s, r);
    a.idx = r.idx;
    a.meta = r.meta;
    a.coef = r.coef;
    launch_logits<0>(a, 0, grid, s);
    hipLaunchKernelGGL(k_loss_merge, dim3((T + 3) / 4), dim3(256), 0, s, r.meta, r.idx, a.part, a.hit, loss, lse);
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
    if (T == 0 && !dweight) return VMI_OK;   // (an empty dx is null)
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
    const int grid = workgroups();
    RowsArgs r = rows_args(targets, ignore_index, T, vocab, l, ws, grid);
    r.lse = lse;
    r.dloss = d_loss;
    r.dlse = d_lse;
    r.tiles = l.piece / 256;
    r.last = ((vocab - 1) % l.piece + 256) / 256;
    r.nht = (hidden + 255) / 256;
    r.steps = r.last * 256 / kBK;
    if (!l.few) hipLaunchKernelGGL(k_loss_rows, dim3(1), dim3(1024), 0, s, r);
    const Few few{targets, ignore_index, T, vocab, lse, d_loss, d_lse};
    const int splits = ls_splits(grid, 1, r.nht, r.steps);
    uint16_t* xt = reinterpret_cast<uint16_t*>(ws + l.x);
    if (dweight && !l.few)
        hipLaunchKernelGGL(k_loss_turn, dim3(l.rows / 64, hidden / 64), dim3(256), 0, s, r.meta, r.idx, x, hidden, l.ldx, xt,
                           reinterpret_cast<uint16_t*>(ws + l.g), l.ldg);
    LogitArgs a{};
    a.few = few;
    a.x = x;
    a.w = weight;
    a.idx = r.idx;
    a.meta = r.meta;
    a.coef = r.coef;
    a.H = hidden;
    a.V = vocab;
    a.g = reinterpret_cast<uint16_t*>(ws + l.g);
    a.ldg = l.ldg;
    DxArgs d{};
    d.splits = splits;
    d.tokens = few;
    d.w = weight;
    d.g = a.g;
    d.meta = r.meta;
    d.H = hidden;
    d.V = vocab;
    d.ldg = l.ldg;
    d.sum = reinterpret_cast<float*>(ws + l.sum);
    DwArgs u{};
    u.x = l.few ? x : xt;
    u.ldx = l.ldx;
    u.tokens = few;
    u.few = l.few;
    u.g = a.g;
    u.meta = r.meta;
    u.H = hidden;
    u.V = vocab;
    u.ldg = l.ldg;
    u.dw = dweight;
    for (int v0 = 0; v0 < vocab; v0 += l.piece) {
        const int cols = std::min(l.piece, (vocab - v0 + 255) / 256 * 256);
        a.v0 = v0;
        a.v1 = v0 + cols;
        a.last = v0 + l.piece >= vocab;
        d.v0 = u.v0 = v0;
        d.cols = u.cols = cols;
        d.add = v0 != 0;
        if (T) {
            launch_logits<1>(a, l.few, grid, s);
            if (dx) launch_dx(d, l.few, grid, s);
        }
        if (dweight) {
            const bool f32 = dweight_dtype == VMI_F32;
            if (l.few && f32)
                hipLaunchKernelGGL((k_loss_dw<true, true>), dim3(grid), dim3(kThreads), 0, s, u);
            else if (l.few)
                hipLaunchKernelGGL((k_loss_dw<true, false>), dim3(grid), dim3(kThreads), 0, s, u);
            else if (f32)
                hipLaunchKernelGGL((k_loss_dw<false, true>), dim3(grid), dim3(kThreads), 0, s, u);
            else
                hipLaunchKernelGGL((k_loss_dw<false, false>), dim3(grid), dim3(kThreads), 0, s, u);
        }
    }
    if (dx && T) {
        if (l.few)
            hipLaunchKernelGGL(k_loss_dx_out_few, dim3(T, (hidden + 255) / 256), dim3(256), 0, s, few, l.few, splits, d.sum,
                               hidden, dx);
        else
            hipLaunchKernelGGL(k_loss_dx_out, dim3(T, (hidden + 1023) / 1024), dim3(256), 0, s, r.meta, r.pos, d.sum, hidden, dx);
    }
    return launched("vmi_head_loss_grad launch");
}
