// LayerNorm over rows with the statistics its backward pass needs, and the backward pass:
//   mean = sum x / d,  rstd = (sum (x - mean)^2 / d + eps)^-1/2,  y = (x - mean) rstd w + b
//   g = dy w,  xh = (x - mean) rstd,  dx = rstd (g - mean(g) - xh mean(g xh)) + dres
//   dw = sum over rows of dy xh,  db = sum over rows of dy
// Bound by HBM. A block has one row in registers, NV vectors of VEC elements a thread, so x (and dy)
// are read once. In the backward pass blocks stay: each takes every gridDim.x-th row, a thread adds
// up dw and db of its own columns in registers over all of them, and the next row is loaded before
// the current one's sums are exchanged. The blocks' sums go to the workspace and are added there in
// order by layernorm_reduce_kernel, so the gradients do not depend on timing. Rows too wide for the
// registers of a block (kMaxThreads * NV * VEC) take the looping kernels, which read them repeatedly.
#include <algorithm>

#include "train_common.cuh"
#include "train_ops.cuh"

namespace esm {

namespace {

constexpr int kMaxThreads = 512;
constexpr int kMaxParts = 8;  // blocks per SM of the backward pass, at most

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

// The sums of a and b over the block; `sm` has 2 * 16 entries and alternates between two calls.
__device__ __forceinline__ void block_sum2(float& a, float& b, float2* sm) {
  a = warp_sum(a);
  b = warp_sum(b);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  a = b = 0.0f;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) {
    a += sm[i].x;
    b += sm[i].y;
  }
}

template <typename X, typename Y, int VEC, int NV>
__global__ void __launch_bounds__(kMaxThreads) layernorm_row_kernel(const LayerNormOp p) {
  __shared__ float2 sm[2][kMaxThreads / 32];
  const size_t row = blockIdx.x;
  const int n = p.d / VEC;
  const Vec<X, VEC>* x = reinterpret_cast<const Vec<X, VEC>*>(static_cast<const X*>(p.x) + row * p.d);
  const Vec<float, VEC>* w = reinterpret_cast<const Vec<float, VEC>*>(p.w);
  const Vec<float, VEC>* b = reinterpret_cast<const Vec<float, VEC>*>(p.b);
  Vec<X, VEC> raw[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (threadIdx.x + k * blockDim.x < n) raw[k] = x[threadIdx.x + k * blockDim.x];
  float s = 0.0f, s2 = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (threadIdx.x + k * blockDim.x < n)
#pragma unroll
      for (int i = 0; i < VEC; ++i) s += to_f32(raw[k].v[i]);
  block_sum2(s, s2, sm[0]);
  const float mean = s / p.d;
  s = s2 = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (threadIdx.x + k * blockDim.x < n)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float v = to_f32(raw[k].v[i]) - mean;
        s = fmaf(v, v, s);
      }
  block_sum2(s, s2, sm[1]);
  const float rstd = 1.0f / sqrtf(s / p.d + p.eps);
  Vec<Y, VEC>* y = reinterpret_cast<Vec<Y, VEC>*>(static_cast<Y*>(p.y) + row * p.d);
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (threadIdx.x + k * blockDim.x < n) {
      const Vec<float, VEC> wk = w[threadIdx.x + k * blockDim.x], bk = b[threadIdx.x + k * blockDim.x];
      Vec<Y, VEC> o;
#pragma unroll
      for (int i = 0; i < VEC; ++i) o.v[i] = from_f32<Y>(fmaf((to_f32(raw[k].v[i]) - mean) * rstd, wk.v[i], bk.v[i]));
      y[threadIdx.x + k * blockDim.x] = o;
    }
  if (threadIdx.x == 0) {
    if (p.mean) p.mean[row] = mean;
    if (p.rstd) p.rstd[row] = rstd;
  }
}

template <typename X, typename Y, int VEC, int NV, bool RES>
__global__ void __launch_bounds__(kMaxThreads) layernorm_backward_kernel(const LayerNormOp p) {
  __shared__ float2 sm[2][kMaxThreads / 32];
  const int n = p.d / VEC, t = threadIdx.x;
  struct Row {
    Vec<X, VEC> x[NV];
    Vec<Y, VEC> dy[NV];
    Vec<X, VEC> res[RES ? NV : 1];
    float mean, rstd;
  };
  auto load = [&](Row& r, size_t row) {
    const Vec<X, VEC>* x = reinterpret_cast<const Vec<X, VEC>*>(static_cast<const X*>(p.x) + row * p.d);
    const Vec<Y, VEC>* dy = reinterpret_cast<const Vec<Y, VEC>*>(static_cast<const Y*>(p.dy) + row * p.d);
    const Vec<X, VEC>* res = reinterpret_cast<const Vec<X, VEC>*>(static_cast<const X*>(p.dres) + row * p.d);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (t + k * static_cast<int>(blockDim.x) < n) {
        r.x[k] = x[t + k * blockDim.x];
        r.dy[k] = dy[t + k * blockDim.x];
        if constexpr (RES) r.res[k] = res[t + k * blockDim.x];
      }
    r.mean = p.mean[row];
    r.rstd = p.rstd[row];
  };
  Vec<float, VEC> w[NV], dw[NV], db[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (t + k * static_cast<int>(blockDim.x) < n) w[k] = reinterpret_cast<const Vec<float, VEC>*>(p.w)[t + k * blockDim.x];
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[k].v[i] = db[k].v[i] = 0.0f;
  }
  const float inv_d = 1.0f / p.d;
  Row cur, next;
  int turn = 0;
  if (static_cast<int>(blockIdx.x) < p.T) load(cur, blockIdx.x);
  for (int64_t row = blockIdx.x; row < p.T; row += gridDim.x, turn ^= 1) {
    if (row + gridDim.x < p.T) load(next, row + gridDim.x);
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (t + k * static_cast<int>(blockDim.x) < n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float dy = to_f32(cur.dy[k].v[i]), xh = (to_f32(cur.x[k].v[i]) - cur.mean) * cur.rstd, g = dy * w[k].v[i];
          a += g;
          b = fmaf(g, xh, b);
          dw[k].v[i] = fmaf(dy, xh, dw[k].v[i]);
          db[k].v[i] += dy;
        }
    block_sum2(a, b, sm[turn]);
    a *= inv_d;
    b *= inv_d;
    Vec<X, VEC>* dx = reinterpret_cast<Vec<X, VEC>*>(static_cast<X*>(p.dx) + row * p.d);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (t + k * static_cast<int>(blockDim.x) < n) {
        Vec<X, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float xh = (to_f32(cur.x[k].v[i]) - cur.mean) * cur.rstd;
          float v = cur.rstd * (to_f32(cur.dy[k].v[i]) * w[k].v[i] - a - xh * b);
          if constexpr (RES) v += to_f32(cur.res[k].v[i]);
          o.v[i] = from_f32<X>(v);
        }
        dx[t + k * blockDim.x] = o;
      }
    cur = next;
  }
  float* part = p.workspace + static_cast<size_t>(blockIdx.x) * 2 * p.d;
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (t + k * static_cast<int>(blockDim.x) < n)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        part[(t + k * blockDim.x) * VEC + i] = dw[k].v[i];
        part[p.d + (t + k * blockDim.x) * VEC + i] = db[k].v[i];
      }
}

// ---- rows wider than a block's registers -------------------------------------------------------

template <typename X, typename Y>
__global__ void __launch_bounds__(kMaxThreads) layernorm_wide_kernel(const LayerNormOp p) {
  __shared__ float2 sm[2][kMaxThreads / 32];
  const size_t row = blockIdx.x;
  const X* x = static_cast<const X*>(p.x) + row * p.d;
  float s = 0.0f, s2 = 0.0f;
  for (int c = threadIdx.x; c < p.d; c += kMaxThreads) s += to_f32(x[c]);
  block_sum2(s, s2, sm[0]);
  const float mean = s / p.d;
  s = s2 = 0.0f;
  for (int c = threadIdx.x; c < p.d; c += kMaxThreads) {
    const float v = to_f32(x[c]) - mean;
    s = fmaf(v, v, s);
  }
  block_sum2(s, s2, sm[1]);
  const float rstd = 1.0f / sqrtf(s / p.d + p.eps);
  Y* y = static_cast<Y*>(p.y) + row * p.d;
  for (int c = threadIdx.x; c < p.d; c += kMaxThreads)
    y[c] = from_f32<Y>(fmaf((to_f32(x[c]) - mean) * rstd, p.w[c], p.b[c]));
  if (threadIdx.x == 0) {
    if (p.mean) p.mean[row] = mean;
    if (p.rstd) p.rstd[row] = rstd;
  }
}

template <typename X, typename Y>
__global__ void __launch_bounds__(kMaxThreads) layernorm_wide_dx_kernel(const LayerNormOp p) {
  __shared__ float2 sm[kMaxThreads / 32];
  const size_t row = blockIdx.x;
  const X* x = static_cast<const X*>(p.x) + row * p.d;
  const Y* dy = static_cast<const Y*>(p.dy) + row * p.d;
  const float mean = p.mean[row], rstd = p.rstd[row];
  float a = 0.0f, b = 0.0f;
  for (int c = threadIdx.x; c < p.d; c += kMaxThreads) {
    const float g = to_f32(dy[c]) * p.w[c];
    a += g;
    b = fmaf(g, (to_f32(x[c]) - mean) * rstd, b);
  }
  block_sum2(a, b, sm);
  a /= p.d;
  b /= p.d;
  for (int c = threadIdx.x; c < p.d; c += kMaxThreads) {
    float v = rstd * (to_f32(dy[c]) * p.w[c] - a - (to_f32(x[c]) - mean) * rstd * b);
    if (p.dres) v += to_f32(static_cast<const X*>(p.dres)[row * p.d + c]);
    static_cast<X*>(p.dx)[row * p.d + c] = from_f32<X>(v);
  }
}

template <typename X, typename Y>
__global__ void __launch_bounds__(kMaxThreads) layernorm_wide_dw_kernel(const LayerNormOp p) {
  const int c = blockIdx.x * kMaxThreads + threadIdx.x;
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

// ---- sums of the blocks' parts: 32 columns a block, 32 threads a column ---------------------------

__global__ void __launch_bounds__(1024) layernorm_reduce_kernel(const float* part, int n, int d, float* dw, float* db) {
  __shared__ float sm[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (c < 2 * d)
    for (int i = w; i < n; i += 32) s += part[static_cast<size_t>(i) * 2 * d + c];
  sm[w][lane] = s;
  __syncthreads();
  s = warp_sum(sm[lane][w]);
  const int out = blockIdx.x * 32 + w;
  if (lane == 0 && out < 2 * d) (out < d ? dw[out] : db[out - d]) = s;
}

// ---- launches ------------------------------------------------------------------------------------

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Vectors of 4 elements where every row starts on one.
int vector_width(const LayerNormOp& p, size_t ex, size_t ey) {
  const bool ok = p.d % 4 == 0 && aligned(p.x, 4 * ex) && aligned(p.y, 4 * ey) && aligned(p.w, 16) && aligned(p.b, 16) &&
                  aligned(p.dy, 4 * ey) && aligned(p.dres, 4 * ex) && aligned(p.dx, 4 * ex);
  return ok ? 4 : 1;
}

int row_threads(int vectors, int nv) { return ((vectors + nv - 1) / nv + 31) / 32 * 32; }

int parts(int T, int num_sms) { return std::max(1, std::min(T, kMaxParts * num_sms)); }

template <typename X, typename Y>
cudaError_t forward(const LayerNormOp& p, cudaStream_t s) {
  const int vec = vector_width(p, sizeof(X), sizeof(Y)), n = p.d / vec;
  if (n <= 2 * kMaxThreads) {
    if (vec == 4) layernorm_row_kernel<X, Y, 4, 2><<<p.T, row_threads(n, 2), 0, s>>>(p);
    else layernorm_row_kernel<X, Y, 1, 2><<<p.T, row_threads(n, 2), 0, s>>>(p);
  } else if (n <= 4 * kMaxThreads) {
    if (vec == 4) layernorm_row_kernel<X, Y, 4, 4><<<p.T, row_threads(n, 4), 0, s>>>(p);
    else layernorm_row_kernel<X, Y, 1, 4><<<p.T, row_threads(n, 4), 0, s>>>(p);
  } else {
    layernorm_wide_kernel<X, Y><<<p.T, kMaxThreads, 0, s>>>(p);
  }
  return cudaGetLastError();
}

template <typename X, typename Y, int VEC, int NV, bool RES>
int launch_rows(const LayerNormOp& p, int n, cudaStream_t s) {
  const int threads = row_threads(n, NV);
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, layernorm_backward_kernel<X, Y, VEC, NV, RES>, threads, 0) !=
      cudaSuccess)
    return 0;
  const int blocks = std::max(1, std::min(p.T, std::min(per_sm, kMaxParts) * p.num_sms));
  layernorm_backward_kernel<X, Y, VEC, NV, RES><<<blocks, threads, 0, s>>>(p);
  return blocks;
}

template <typename X, typename Y, bool RES>
int backward_rows(const LayerNormOp& p, cudaStream_t s) {
  const int vec = vector_width(p, sizeof(X), sizeof(Y)), n = p.d / vec;
  if (n <= 2 * kMaxThreads)
    return vec == 4 ? launch_rows<X, Y, 4, 2, RES>(p, n, s) : launch_rows<X, Y, 1, 2, RES>(p, n, s);
  if (n <= 4 * kMaxThreads)
    return vec == 4 ? launch_rows<X, Y, 4, 4, RES>(p, n, s) : launch_rows<X, Y, 1, 4, RES>(p, n, s);
  const int blocks = parts(p.T, p.num_sms);
  if (p.T > 0) layernorm_wide_dx_kernel<X, Y><<<p.T, kMaxThreads, 0, s>>>(p);
  layernorm_wide_dw_kernel<X, Y><<<dim3((p.d + kMaxThreads - 1) / kMaxThreads, blocks), kMaxThreads, 0, s>>>(p);
  return blocks;
}

template <typename X, typename Y>
cudaError_t backward(const LayerNormOp& p, cudaStream_t s) {
  const int n = p.dres ? backward_rows<X, Y, true>(p, s) : backward_rows<X, Y, false>(p, s);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || n == 0) return e != cudaSuccess ? e : cudaErrorInvalidConfiguration;
  layernorm_reduce_kernel<<<(2 * p.d + 31) / 32, 1024, 0, s>>>(p.workspace, n, p.d, p.dw, p.db);
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
