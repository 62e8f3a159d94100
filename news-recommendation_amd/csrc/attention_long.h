// internal interface of the attention kernels without a bound on the sequence length (attention_long*.hip)
#pragma once
#include "common.h"
#include "rowops.h"

namespace nr {

// One problem.  Strides are in elements; the innermost axis (head dim) is dense everywhere.  q [N,Sq,H,dh], k / v [N,Sk,G,dh],
// H a multiple of G: query head h reads key head h / (H / G).
struct AttnStrides { int64_t n = 0, s = 0, h = 0; };
struct AttnProblem {
    const void *q = nullptr, *k = nullptr, *v = nullptr;
    const int64_t* key_mask = nullptr;          // [N,Sk], 0 = the key is not there; NULL = every key is
    AttnStrides sq, sk, sv;
    int64_t N = 0;
    int Sq = 0, Sk = 0, H = 0, G = 0, dh = 0;
    bool bf16 = false, causal = false;
    bool additive = false;                      // masked keys get + mask_fill instead of being left out (fp32 only)
    float scale = 1.f;
    DropoutCfg dc;                              // p, seed, site, mask_fill
};
struct AttnOut {                                // what the forward writes
    void* out = nullptr;
    AttnStrides so;
    float *row_max = nullptr, *row_sum = nullptr;      // [N,H,Sq], both or neither; the maximum of bf16 problems in units of log 2
};
struct AttnGrad {                               // what the backward reads besides the problem, and writes
    const void *out = nullptr, *dout = nullptr;
    AttnStrides so, sdo;
    const float *row_max = nullptr, *row_sum = nullptr;
    float* delta = nullptr;                     // scratch: sum_d dout * out per row; element (n, h, i) at n * sd.n + h * sd.h + i * sd.s
    AttnStrides sd;                             // (it may lie in dq: a row's dq is written after its delta was last read)
    void *dq = nullptr, *dk = nullptr, *dv = nullptr;
    AttnStrides sdq, sdk, sdv;
};

size_t attn_long_fwd_ws_bytes(const AttnProblem& p);
int attn_long_fwd(const AttnProblem& p, const AttnOut& o, void* ws, size_t ws_bytes, hipStream_t s);
size_t attn_long_bwd_ws_bytes(const AttnProblem& p);
int attn_long_bwd(const AttnProblem& p, const AttnGrad& g, void* ws, size_t ws_bytes, hipStream_t s);

}  // namespace nr
