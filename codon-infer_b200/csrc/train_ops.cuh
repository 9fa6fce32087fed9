// Launchers of the operators on device memory around the encoder's own path: attention with its
// backward pass, LayerNorm with its backward pass, token log probabilities, and the distillation
// loss with its gradient. Element types are ESM_F32 / ESM_F16 / ESM_BF16 (include/esm_b200.h);
// arguments were checked by the C ABI.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace esm {

// Packed sequences: rows cu[b] .. cu[b + 1] of [T, *] matrices belong to sequence b.
struct AttnOp {
  int dtype;               // ESM_F16 or ESM_BF16
  const void* qkv;         // [T, 3 H dh], row stride ld_qkv elements
  int64_t ld_qkv;
  const int32_t* cu;       // [B + 1], device
  int B, T, max_len, H, dh;
  float scale;
  void* out;               // [T, H dh], row stride ld_out (read by the backward pass)
  int64_t ld_out;
  float* lse;              // [H, T] natural-log row sums of exp(scale q k^T); may be null (forward)
  // backward pass
  const void* dout;        // [T, H dh], row stride ld_dout
  int64_t ld_dout;
  void* dqkv;              // [T, 3 H dh], row stride ld_dqkv
  int64_t ld_dqkv;
  float* workspace;
  int num_sms;
  int* err;                // device error word
};
cudaError_t launch_attention_op(const AttnOp& p, cudaStream_t s);
size_t attention_backward_bytes(int B, int T, int H);
cudaError_t launch_attention_backward(const AttnOp& p, cudaStream_t s);

struct LayerNormOp {
  int x_type, y_type;
  const void* x;           // [T, d]
  const float* w;
  const float* b;
  float eps;
  int T, d;
  void* y;                 // forward: [T, d] of y_type
  float* mean;             // [T]
  float* rstd;             // [T]
  // backward pass
  const void* dy;          // [T, d] of y_type
  const void* dres;        // [T, d] of x_type or null: added to dx
  void* dx;                // [T, d] of x_type
  float* dw;
  float* db;
  float* workspace;
  int num_sms;
};
cudaError_t launch_layernorm_op(const LayerNormOp& p, cudaStream_t s);
size_t layernorm_backward_bytes(int T, int d, int num_sms);
cudaError_t launch_layernorm_backward(const LayerNormOp& p, cudaStream_t s);

struct LogitsOp {
  int dtype;
  const void* logits;      // [T, V], row stride ld
  int64_t ld;
  int T, V, k;
  // log probabilities
  const int32_t* targets;  // [T] or null
  float* logp;             // [T] or null
  float* entropy;          // [T] or null
  int32_t* top_ids;        // [T, k]
  float* top_logp;         // [T, k]
  // distillation
  const int32_t* alt_ids;  // [T, k]; an id outside [0, V) is absent
  const float* alt_logits; // [T, k]
  float temperature;
  float* loss;             // [T]
  float* lse;              // [T]
  const float* dloss;      // [T]
  void* dlogits;           // [T, V], row stride ld_grad
  int64_t ld_grad;
};
cudaError_t launch_token_logprobs(const LogitsOp& p, cudaStream_t s);
cudaError_t launch_distill_loss(const LogitsOp& p, cudaStream_t s);
cudaError_t launch_distill_backward(const LogitsOp& p, cudaStream_t s);

}  // namespace esm
