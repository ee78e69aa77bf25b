// Host-side internals shared by the libvmi translation units.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/vmi.h"

namespace vmi {

// Records the thread-local error message and returns `code`.
int fail(int code, const char* fmt, ...);
int hip_fail(hipError_t e, const char* what);
void clear_error();

inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }
int device_cus();  // compute units of the current device

constexpr int kRouteMaxPairs = 160;
constexpr int kRouteMaxT = 16;

// Routing of one verify batch as the down/combine kernel reads it, written by
// one workgroup of the gate/up kernel.
struct RouteInfo {
    int32_t U;                               // distinct valid slots
    int32_t uslot[kRouteMaxPairs];           // slot of distinct index u (first-appearance order)
    float wt[kRouteMaxPairs][kRouteMaxT];    // combine weight of (u, token): sum of its pairs' scores
    int32_t jr[kRouteMaxPairs][kRouteMaxT];  // rank j of the token's first pair on u, -1 if none: the
                                             // token's experts are added in rank order
    int32_t pv[kRouteMaxPairs];              // 1: pair p is its token's first pair on a valid slot
};

// Workspace carve-up of vmi_moe_layer (and its no-allocation variant).
struct MoeWorkspace {
    uint32_t* status;     // device status word (VMI_STATUS_*)
    RouteInfo* route;
    float* logits;        // [T, E]
    float* sg_logit;      // [T]
    uint32_t __attribute__((ext_vector_type(4)))* xop;    // [T, H/8] MFMA operands of the MoE input
    float* xsum;          // [T, H/64] per-group sums of those operands
    float* fscale;        // [T] power-of-two range factor of the operands
    void* groups;         // token groups of a batch of more than eight tokens (RouteGroups, vmi_moe.hip)
    uint16_t* part;       // [T*k + T, I/64, H] weighted bf16 partial rows: pair p's (or the shared
                          // expert's for token t, row T*k + t) down projection of each slice
    size_t bytes;
};

MoeWorkspace carve_workspace(void* base, int T, int k, int hidden, int inter, int num_experts);

// Quantised GEMV over up to three stacked matrices (k_qgemv, vmi_attn.hip):
// out[t][n] = sum_k x[t][k] W[n][k] for T <= 8 tokens, T * K <= 32768.
struct QgemvCall {
    const uint16_t* x;      // [T, K] bf16
    int T, K, bits;
    vmi_qmat m[3];
    int rows[3];            // rows of each matrix
    int nrows;              // total
    float* out;             // [T, out_stride] f32: row n of the stack at column n
    int out_stride;
    const uint16_t* residual;  // optional [T, out_stride] bf16: out_bf16 = bf16(y + residual)
    uint16_t* out_bf16;        // optional
    const uint16_t* norm_w;    // optional [K] bf16: x is first RMS-normalised (canonical order)
    float eps;
};
hipError_t launch_qgemv(const QgemvCall& q, hipStream_t s);
// Whether launch_qgemv can normalise x itself (QgemvCall::norm_w): the MFMA
// kernel with K in {512, 1024, 2048}.
bool qgemv_fuses_norm(const QgemvCall& q);
// bf16 RMSNorm of T rows of width H (H % 512 == 0) into out (stride H).
hipError_t launch_rmsnorm(const uint16_t* x, const uint16_t* w, float eps, int T, int H, uint16_t* out, hipStream_t s);
// Non-null, 16-byte aligned packed weights.
bool qmat_ok(const vmi_qmat& m);

// The 8-bit KV cache (vmi_kv8.hip).
//
// q and k RMSNorm and rotary embedding of a batch's projections, k and v into
// the cache (or a tree's rows into `tree`).  paths sequences of T tokens, all
// from the same position.
struct Kv8Heads {
    const float* qkv;      // [paths * T, 2 n_heads + 2 n_kv, 256]: q | gate per head, then k, then v
    int T, n_heads, n_kv;
    int h0;                // first head formed: 0, or n_heads (keys and values only)
    const uint16_t *q_norm, *k_norm;
    float eps;
    int rope_dim;
    double rope_base;      // kv8_rope_base
    int pos0;
    const int32_t* pos_dev;
    int max_len;
    uint8_t* cache;
    uint8_t* tree;         // or null: [paths][n_kv][T] rows instead of the cache
    uint16_t* q;           // [paths * T, n_heads, 256]
    uint32_t* status;      // or null (VMI_STATUS_BAD_POS)
};
double kv8_rope_base(float theta, int rope_dim);
// Whether the rotation of every position below max_len is formed (rope_dim even, in [0, 256]).
bool kv8_rope_ok(float theta, int rope_dim, int max_len);
hipError_t launch_kv8_heads(const Kv8Heads& h, int paths, hipStream_t s);

// Attention over the cache: paths sequences of span tokens at positions pos0 ..
struct Kv8Attn {
    const uint16_t* q;     // [paths * span, n_heads, 256]
    const uint8_t* cache;
    const uint8_t* tree;   // or null: the paths' own tokens
    int n_heads, n_kv, span, paths, pos0, max_len;
    const int32_t* pos_dev;
    const float* gate;     // or null: f32, element strides gate_tok, gate_head
    int64_t gate_tok, gate_head;
    uint16_t* o;           // [paths * span, n_heads, 256]
    uint32_t* status;      // or null
    int rp, run;           // set by the launch: rows of a part, records of one, and the parts
    float *part_o, *part_ml;
};
bool kv8_heads_ok(int n_heads, int n_kv);
// Bytes of the parts (0: a form that is not built: several paths of more than
// 64 rows, or more than 8192 tokens).
size_t kv8_attention_parts_bytes(int paths, int span, int n_heads, int n_kv);
hipError_t launch_kv8_attention(Kv8Attn a, void* parts, hipStream_t s);

}  // namespace vmi
