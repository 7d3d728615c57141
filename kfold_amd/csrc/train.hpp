// Launch interface of the training operators: layer norm, gated feed-forward block, dropout.
#pragma once
#include "kernels.hpp"

namespace kfh {

// ---- layer norm (layernorm.hip) ------------------------------------------------------------
// gamma, beta: fp32 [C] or null; mean, rstd: fp32 [M], both or neither
void launch_ln_forward(const void* x, int io_dtype, const float* gamma, const float* beta, void* y, float* mean,
                       float* rstd, long long M, int C, float eps, hipStream_t stream);
// rows of partial sums a backward call writes: part holds ln_bwd_blocks(M) * 2C fp32
int ln_bwd_blocks(long long M);
// dx, dgamma, dbeta may each be null; part may be null if dgamma and dbeta are
void launch_ln_backward(const void* dy, const void* x, int io_dtype, const float* mean, const float* rstd,
                        const float* gamma, void* dx, float* dgamma, float* dbeta, float* part, long long M, int C,
                        hipStream_t stream);

// ---- dropout (dropout.hip) -----------------------------------------------------------------
struct DropArgs {
    const void* x; const void* residual; void* y;        // [outer, shared, inner]; residual may be null
    long long outer, shared, inner;                       // one mask value covers the shared dimension
    uint32_t t; float scale;                              // keep where 16 random bits >= t
    const unsigned long long* seed_dev;                   // seed in device memory, or null: `seed`
    unsigned long long seed, offset;
};
void launch_dropout(const DropArgs& p, int io_dtype, hipStream_t stream);

// ---- gated feed-forward block (gatedffn.hip) -----------------------------------------------
size_t gated_ffn_ws_bytes(long long M, int C, int F, int backward, int io_dtype);
void launch_gated_ffn_forward(const void* x, const void* w_in, const void* w_out, void* y, char* ws, long long M,
                              int C, int F, int io_dtype, hipStream_t stream);
// dx, dw_in, dw_out may each be null; dw_dtype: element type of dw_in and dw_out
void launch_gated_ffn_backward(const void* dy, const void* x, const void* w_in, const void* w_out, void* dx,
                               void* dw_in, void* dw_out, int dw_dtype, char* ws, long long M, int C, int F,
                               int io_dtype, hipStream_t stream);

}  // namespace kfh
