// Attention over packed sequences and its backward pass, for callers that train or distil an
// encoder (the encoder's own attention is attention_tc3.cu).
//
// Per sequence and head, with S = scale Q K^T:
//   lse_i = log sum_j exp(S_ij),  P = exp(S - lse),  O = P V
//   D_i = sum_d dO_id O_id,  dV = P^T dO,  dS = P (dO V^T - D),  dQ = scale dS K,  dK = scale dS^T Q
//
// One warp per query row (forward, dQ) or key row (dK, dV): the lanes take 32 rows of the other
// side at a time, each the dot products of one of them, and then the head's columns.
#include "common.cuh"
#include "train_common.cuh"
#include "train_ops.cuh"

namespace esm {

namespace {

constexpr int kWarps = 8;

// Sequence b of a call, or length 0 where the offsets are not those of packed rows in [0, T].
__device__ __forceinline__ int sequence(const AttnOp& p, int b, int* start) {
  *start = p.cu[b];
  const int len = p.cu[b + 1] - *start;
  if (!packed_rows(*start, len, p.T, p.max_len)) {
    if (threadIdx.x == 0) atomicOr(p.err, kDevBadSeqlens);
    return 0;
  }
  return len;
}

template <typename E>
__device__ __forceinline__ float dot_row(const E* a, const E* b, int dh) {
  float s = 0.0f;
  for (int d = 0; d < dh; ++d) s = fmaf(to_f32(a[d]), to_f32(b[d]), s);
  return s;
}

// D = rowsum(dO O) into the workspace, [H, T].
template <typename E>
__global__ void attention_delta_kernel(const AttnOp p) {
  int start;
  const int len = sequence(p, blockIdx.z, &start), h = blockIdx.y;
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= len) return;
  const E* o = static_cast<const E*>(p.out) + static_cast<size_t>(start + i) * p.ld_out + h * p.dh;
  const E* g = static_cast<const E*>(p.dout) + static_cast<size_t>(start + i) * p.ld_dout + h * p.dh;
  p.workspace[static_cast<size_t>(h) * p.T + start + i] = dot_row(o, g, p.dh);
}

// KEYS: the warp's row is a key (dK and dV); otherwise a query (dQ).
template <typename E, bool KEYS>
__global__ void attention_backward_kernel(const AttnOp p) {
  int start;
  const int len = sequence(p, blockIdx.z, &start), h = blockIdx.y, lane = threadIdx.x & 31;
  const int i = blockIdx.x * kWarps + (threadIdx.x >> 5), dh = p.dh, d = p.H * dh;
  if (i >= len) return;
  const E* q = static_cast<const E*>(p.qkv) + static_cast<size_t>(start) * p.ld_qkv + h * dh;
  const E* k = q + d;
  const E* v = k + d;
  const E* g = static_cast<const E*>(p.dout) + static_cast<size_t>(start) * p.ld_dout + h * dh;
  const float* lse = p.lse + static_cast<size_t>(h) * p.T + start;
  const float* delta = p.workspace + static_cast<size_t>(h) * p.T + start;
  float acc[2] = {0.0f, 0.0f}, acc_v[2] = {0.0f, 0.0f};
  for (int j0 = 0; j0 < len; j0 += 32) {
    const int n = min(32, len - j0), j = j0 + min(lane, n - 1);
    const int qi = KEYS ? j : i, ki = KEYS ? i : j;
    float pr = 0.0f, ds = 0.0f;
    if (lane < n) {
      pr = expf(dot_row(q + qi * p.ld_qkv, k + ki * p.ld_qkv, dh) * p.scale - lse[qi]);
      ds = pr * (dot_row(g + qi * p.ld_dout, v + ki * p.ld_qkv, dh) - delta[qi]) * p.scale;
    }
    for (int r = 0; r < n; ++r) {
      const float dsr = __shfl_sync(0xffffffffu, ds, r), prr = __shfl_sync(0xffffffffu, pr, r);
      const E* other = (KEYS ? q : k) + (j0 + r) * p.ld_qkv;
      for (int c = 0; c < 2; ++c)
        if (lane + 32 * c < dh) {
          acc[c] = fmaf(dsr, to_f32(other[lane + 32 * c]), acc[c]);
          if (KEYS) acc_v[c] = fmaf(prr, to_f32(g[(j0 + r) * p.ld_dout + lane + 32 * c]), acc_v[c]);
        }
    }
  }
  E* out = static_cast<E*>(p.dqkv) + static_cast<size_t>(start + i) * p.ld_dqkv + h * dh + (KEYS ? d : 0);
  for (int c = 0; c < 2; ++c)
    if (lane + 32 * c < dh) {
      out[lane + 32 * c] = from_f32<E>(acc[c]);
      if (KEYS) out[d + lane + 32 * c] = from_f32<E>(acc_v[c]);
    }
}

template <typename E>
cudaError_t backward(const AttnOp& p, cudaStream_t s) {
  const dim3 grid((p.max_len + kWarps - 1) / kWarps, p.H, p.B);
  attention_delta_kernel<E><<<dim3((p.max_len + 127) / 128, p.H, p.B), 128, 0, s>>>(p);
  attention_backward_kernel<E, false><<<grid, kWarps * 32, 0, s>>>(p);
  attention_backward_kernel<E, true><<<grid, kWarps * 32, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

size_t attention_backward_bytes(int B, int T, int H) {
  return static_cast<size_t>(H) * T * 4 + static_cast<size_t>(H) * (T / 64 + B) * 8;
}

cudaError_t launch_attention_backward(const AttnOp& p, cudaStream_t s) {
  return p.dtype == ESM_F16 ? backward<__half>(p, s) : backward<__nv_bfloat16>(p, s);
}

}  // namespace esm
