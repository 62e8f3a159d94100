// internal interface of the linear attention kernels (linear_attention.hip)
#pragma once
#include "attention_long.h"

namespace nr {

// S_t = e^a S_{t-1} + k_t v_t^T (a = log_decay[h]), o_t = scale * q_t S_t for the first lens[n] tokens of q / k [N,S,H,dk],
// v [N,S,H,dv]; states [N,H,dk,dv] fp32, dense.  Strides in elements, innermost axis dense.
struct LinProblem {
    const void *q = nullptr, *k = nullptr, *v = nullptr;
    const float* log_decay = nullptr;
    const int64_t* lens = nullptr;              // NULL: every sequence has all S tokens
    const float* state = nullptr;               // NULL: zero
    AttnStrides sq, sk, sv;
    int64_t N = 0;
    int S = 0, H = 0, dk = 0, dv = 0;
    bool bf16 = false;
    float scale = 1.f;
};
size_t lin_fwd_ws_bytes(const LinProblem& p);
int lin_fwd(const LinProblem& p, void* out, float* last, void* ws, size_t ws_bytes, hipStream_t s);
size_t lin_bwd_ws_bytes(const LinProblem& p);
int lin_bwd(const LinProblem& p, const void* dout, const float* dlast, void* dq, void* dk, void* dv, float* dstate, void* ws, size_t ws_bytes,
            hipStream_t s);
// one token: q / k [N,H,dk], v [N,H,dv] dense; out_state may be state
int lin_step(const void* q, const void* k, const void* v, const float* log_decay, const float* state, int64_t N, int H, int dk, int dv, bool bf16,
             float scale, void* out, float* out_state, hipStream_t s);

}  // namespace nr
