// Operators on rows of logits x[V]:
//   log probabilities: lse = log sum exp x; logp = x[target] - lse; entropy = lse - sum p x with
//     p = exp(x - lse) (0 where p is 0); the k largest log probabilities, ties to the lowest id;
//   distillation from a teacher's alternatives (id_i, t_i), i < k, at temperature tau: with
//     p = softmax(t / tau) over the present alternatives and q = softmax(x / tau),
//     loss = tau^2 sum_i p_i (log p_i - log q[id_i]) and
//     dx_j = dloss tau (q_j - sum of the p_i with id_i = j).
// One warp per row, which reads the row again for every pass.
#include "train_common.cuh"
#include "train_ops.cuh"

namespace esm {

namespace {

constexpr int kWarps = 4;

// The row's maximum and sum of exp((x - max) * inv_tau); NaN sum where a NaN or +inf is among x.
template <typename E>
__device__ __forceinline__ void row_lse(const E* x, int V, float inv_tau, int lane, float* top, float* sum) {
  float m = -INFINITY;
  for (int j = lane; j < V; j += 32) m = fmaxf(m, to_f32(x[j]));
  m = warp_max(m);
  float s = 0.0f;
  for (int j = lane; j < V; j += 32) s += expf((to_f32(x[j]) - m) * inv_tau);
  *top = m;
  *sum = warp_sum(s);
}

// Keys that order like floats, -0 and +0 alike; larger is better.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <typename E>
__global__ void token_logprobs_kernel(const LogitsOp p) {
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (t >= p.T) return;
  const E* x = static_cast<const E*>(p.logits) + t * p.ld;
  float m, s;
  row_lse(x, p.V, 1.0f, lane, &m, &s);
  const float log_s = logf(s);
  if (p.entropy) {
    float w = 0.0f;
    for (int j = lane; j < p.V; j += 32) {
      const float v = to_f32(x[j]) - m, e = expf(v);
      if (!(e <= 0.0f)) w = fmaf(e, v, w);
    }
    w = warp_sum(w);
    if (lane == 0) p.entropy[t] = log_s - w / s;
  }
  if (p.logp && lane == 0) {
    const int id = p.targets[t];
    p.logp[t] = id >= 0 && id < p.V ? to_f32(x[id]) - m - log_s : 0.0f;
  }
  uint64_t last = ~0ull;  // the best key so far taken; a row without a distribution has no alternatives
  for (int i = 0; i < p.k; ++i) {
    uint64_t best = 0;
    for (int j = lane; j < p.V; j += 32) {
      const uint64_t key = static_cast<uint64_t>(order_key(to_f32(x[j]))) << 32 | ~static_cast<uint32_t>(j);
      if (key < last && key > best) best = key;
    }
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    last = best;
    if (lane == 0) {
      const int id = s == s ? static_cast<int>(~static_cast<uint32_t>(best)) : -1;
      p.top_ids[t * p.k + i] = id;
      p.top_logp[t * p.k + i] = id >= 0 ? to_f32(x[id]) - m - log_s : NAN;
    }
  }
}

// Lane i and 32 + i: the teacher's probabilities of alternatives i and 32 + i (0 where absent).
// Returns false where the row has no alternative.
__device__ __forceinline__ bool teacher(const LogitsOp& p, int64_t t, int lane, int (&id)[2], float (&pr)[2],
                                        float (&logp)[2]) {
  float v[2], m = -INFINITY;
  for (int c = 0; c < 2; ++c) {
    const int i = lane + 32 * c;
    id[c] = i < p.k ? p.alt_ids[t * p.k + i] : -1;
    if (id[c] >= p.V) id[c] = -1;
    v[c] = id[c] >= 0 ? p.alt_logits[t * p.k + i] : -INFINITY;
    m = fmaxf(m, v[c]);
  }
  m = warp_max(m);
  float s = 0.0f;
  for (int c = 0; c < 2; ++c) {
    v[c] = (v[c] - m) / p.temperature;
    pr[c] = id[c] >= 0 ? expf(v[c]) : 0.0f;
    s += pr[c];
  }
  s = warp_sum(s);
  const float log_s = logf(s);
  for (int c = 0; c < 2; ++c) {
    pr[c] /= s;
    logp[c] = v[c] - log_s;
  }
  return m > -INFINITY;
}

template <typename E>
__global__ void distill_loss_kernel(const LogitsOp p) {
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (t >= p.T) return;
  const E* x = static_cast<const E*>(p.logits) + t * p.ld;
  float m, s;
  row_lse(x, p.V, 1.0f / p.temperature, lane, &m, &s);
  const float lse = m / p.temperature + logf(s);
  int id[2];
  float pr[2], logp[2], loss = 0.0f;
  const bool any = teacher(p, t, lane, id, pr, logp);
  for (int c = 0; c < 2; ++c)
    if (pr[c] > 0.0f) loss += pr[c] * (logp[c] - (to_f32(x[id[c]]) / p.temperature - lse));
  loss = warp_sum(loss);
  if (lane == 0) {
    p.loss[t] = any ? p.temperature * p.temperature * loss : 0.0f;
    p.lse[t] = lse;
  }
}

template <typename E>
__global__ void distill_backward_kernel(const LogitsOp p) {
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (t >= p.T) return;
  const E* x = static_cast<const E*>(p.logits) + t * p.ld;
  E* dx = static_cast<E*>(p.dlogits) + t * p.ld_grad;
  int id[2];
  float pr[2], logp[2];
  const bool any = teacher(p, t, lane, id, pr, logp);
  const float g = p.dloss[t] * p.temperature, lse = p.lse[t];
  if (!any || g == 0.0f) {
    for (int j = lane; j < p.V; j += 32) dx[j] = from_f32<E>(0.0f);
    return;
  }
  for (int j = lane; j < p.V; j += 32) {
    float q = expf(to_f32(x[j]) / p.temperature - lse);
    dx[j] = from_f32<E>(g * q);
  }
  __syncwarp();
  // The alternatives' own columns again: the first of equal ids writes, with all their probability.
  for (int c = 0; c < 2; ++c) {
    float sum = 0.0f;
    bool first = id[c] >= 0;
    for (int i = 0; i < p.k; ++i) {
      const int other = __shfl_sync(0xffffffffu, id[i >> 5], i & 31);
      const float o = __shfl_sync(0xffffffffu, pr[i >> 5], i & 31);
      if (other == id[c]) {
        sum += o;
        if (i < lane + 32 * c) first = false;
      }
    }
    if (first) dx[id[c]] = from_f32<E>(g * (expf(to_f32(x[id[c]]) / p.temperature - lse) - sum));
  }
}

unsigned blocks(const LogitsOp& p) { return (static_cast<unsigned>(p.T) + kWarps - 1) / kWarps; }

}  // namespace

#define ESM_BY_TYPE(kernel)                                                      \
  switch (p.dtype) {                                                             \
    case ESM_F32: kernel<float><<<blocks(p), kWarps * 32, 0, s>>>(p); break;     \
    case ESM_F16: kernel<__half><<<blocks(p), kWarps * 32, 0, s>>>(p); break;    \
    default: kernel<__nv_bfloat16><<<blocks(p), kWarps * 32, 0, s>>>(p); break;  \
  }                                                                              \
  return cudaGetLastError()

cudaError_t launch_token_logprobs(const LogitsOp& p, cudaStream_t s) { ESM_BY_TYPE(token_logprobs_kernel); }
cudaError_t launch_distill_loss(const LogitsOp& p, cudaStream_t s) { ESM_BY_TYPE(distill_loss_kernel); }
cudaError_t launch_distill_backward(const LogitsOp& p, cudaStream_t s) { ESM_BY_TYPE(distill_backward_kernel); }

}  // namespace esm
