// LayerNorm over rows with the statistics its backward pass needs, and the backward pass:
//   mean = sum x / d,  rstd = (sum (x - mean)^2 / d + eps)^-1/2,  y = (x - mean) rstd w + b
//   g = dy w,  xh = (x - mean) rstd,  dx = rstd (g - mean(g) - xh mean(g xh)) + dres
//   dw = sum over rows of dy xh,  db = sum over rows of dy
// One block per row; the weight gradients in two passes (row blocks, then their sums in order).
#include "train_common.cuh"
#include "train_ops.cuh"

namespace esm {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float block_sum(float v, float* sm) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.0f;
  for (int i = 0; i < kThreads / 32; ++i) t += sm[i];
  __syncthreads();
  return t;
}

template <typename X, typename Y>
__global__ void layernorm_op_kernel(const LayerNormOp p) {
  __shared__ float sm[kThreads / 32];
  const size_t row = blockIdx.x;
  const X* x = static_cast<const X*>(p.x) + row * p.d;
  float s = 0.0f;
  for (int c = threadIdx.x; c < p.d; c += kThreads) s += to_f32(x[c]);
  const float mean = block_sum(s, sm) / p.d;
  s = 0.0f;
  for (int c = threadIdx.x; c < p.d; c += kThreads) {
    const float v = to_f32(x[c]) - mean;
    s = fmaf(v, v, s);
  }
  const float rstd = 1.0f / sqrtf(block_sum(s, sm) / p.d + p.eps);
  Y* y = static_cast<Y*>(p.y) + row * p.d;
  for (int c = threadIdx.x; c < p.d; c += kThreads)
    y[c] = from_f32<Y>(fmaf((to_f32(x[c]) - mean) * rstd, p.w[c], p.b[c]));
  if (threadIdx.x == 0) {
    if (p.mean) p.mean[row] = mean;
    if (p.rstd) p.rstd[row] = rstd;
  }
}

template <typename X, typename Y>
__global__ void layernorm_dx_kernel(const LayerNormOp p) {
  __shared__ float sm[kThreads / 32];
  const size_t row = blockIdx.x;
  const X* x = static_cast<const X*>(p.x) + row * p.d;
  const Y* dy = static_cast<const Y*>(p.dy) + row * p.d;
  const float mean = p.mean[row], rstd = p.rstd[row];
  float a = 0.0f, b = 0.0f;
  for (int c = threadIdx.x; c < p.d; c += kThreads) {
    const float g = to_f32(dy[c]) * p.w[c];
    a += g;
    b = fmaf(g, (to_f32(x[c]) - mean) * rstd, b);
  }
  a = block_sum(a, sm) / p.d;
  b = block_sum(b, sm) / p.d;
  for (int c = threadIdx.x; c < p.d; c += kThreads) {
    float v = rstd * (to_f32(dy[c]) * p.w[c] - a - (to_f32(x[c]) - mean) * rstd * b);
    if (p.dres) v += to_f32(static_cast<const X*>(p.dres)[row * p.d + c]);
    static_cast<X*>(p.dx)[row * p.d + c] = from_f32<X>(v);
  }
}

constexpr int kRowsPerPart = 64;

template <typename X, typename Y>
__global__ void layernorm_dw_kernel(const LayerNormOp p) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= p.d) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t r = blockIdx.y; r < p.T; r += gridDim.y) {
    const float dy = to_f32(static_cast<const Y*>(p.dy)[r * p.d + c]);
    dw = fmaf(dy, (to_f32(static_cast<const X*>(p.x)[r * p.d + c]) - p.mean[r]) * p.rstd[r], dw);
    db += dy;
  }
  p.workspace[static_cast<size_t>(blockIdx.y) * 2 * p.d + c] = dw;
  p.workspace[static_cast<size_t>(blockIdx.y) * 2 * p.d + p.d + c] = db;
}

__global__ void layernorm_reduce_kernel(const float* part, int n, int d, float* dw, float* db) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= 2 * d) return;
  float s = 0.0f;
  for (int i = 0; i < n; ++i) s += part[static_cast<size_t>(i) * 2 * d + c];
  (c < d ? dw[c] : db[c - d]) = s;
}

int parts(int T, int num_sms) {
  const int n = (T + kRowsPerPart - 1) / kRowsPerPart;
  return n < 1 ? 1 : (n > 4 * num_sms ? 4 * num_sms : n);
}

template <typename X, typename Y>
cudaError_t forward(const LayerNormOp& p, cudaStream_t s) {
  layernorm_op_kernel<X, Y><<<p.T, kThreads, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename X, typename Y>
cudaError_t backward(const LayerNormOp& p, cudaStream_t s) {
  const int n = parts(p.T, p.num_sms);
  if (p.T > 0) layernorm_dx_kernel<X, Y><<<p.T, kThreads, 0, s>>>(p);
  layernorm_dw_kernel<X, Y><<<dim3((p.d + kThreads - 1) / kThreads, n), kThreads, 0, s>>>(p);
  layernorm_reduce_kernel<<<(2 * p.d + kThreads - 1) / kThreads, kThreads, 0, s>>>(p.workspace, n, p.d, p.dw, p.db);
  return cudaGetLastError();
}

template <typename X>
cudaError_t by_y(const LayerNormOp& p, cudaStream_t s, bool back) {
  switch (p.y_type) {
    case ESM_F32: return back ? backward<X, float>(p, s) : forward<X, float>(p, s);
    case ESM_F16: return back ? backward<X, __half>(p, s) : forward<X, __half>(p, s);
    default: return back ? backward<X, __nv_bfloat16>(p, s) : forward<X, __nv_bfloat16>(p, s);
  }
}

cudaError_t by_x(const LayerNormOp& p, cudaStream_t s, bool back) {
  switch (p.x_type) {
    case ESM_F32: return by_y<float>(p, s, back);
    case ESM_F16: return by_y<__half>(p, s, back);
    default: return by_y<__nv_bfloat16>(p, s, back);
  }
}

}  // namespace

cudaError_t launch_layernorm_op(const LayerNormOp& p, cudaStream_t s) { return by_x(p, s, false); }
size_t layernorm_backward_bytes(int T, int d, int num_sms) {
  return static_cast<size_t>(parts(T, num_sms)) * 2 * d * sizeof(float);
}
cudaError_t launch_layernorm_backward(const LayerNormOp& p, cudaStream_t s) { return by_x(p, s, true); }

}  // namespace esm
