// LayerNorm over rows with the statistics its backward pass needs, and the backward pass:
//   mean = sum x / d,  rstd = (sum (x - mean)^2 / d + eps)^-1/2,  y = (x - mean) rstd w + b
//   g = dy w,  xh = (x - mean) rstd,  dx = rstd (g - mean(g) - xh mean(g xh)) + dres
//   dw = sum over rows of dy xh,  db = sum over rows of dy
// Bound by HBM. A block has one row in registers, NV vectors of VEC elements a thread, so x (and dy)
// are read once. Blocks stay and take every gridDim.x-th row. In the backward pass a block loads its next row
// before the current one's sums are exchanged, and a thread adds up dw and db of its own columns in
// registers over all its rows; the blocks' sums go to the workspace and are added there in order by
// layernorm_reduce_kernel, so the gradients do not depend on timing. Few rows, which stay in L2, take
// one launch instead: some blocks compute dx, others read the same rows again for the columns of dw and db.
// Rows too wide for the registers of a block (kMaxThreads * NV * VEC) take the looping kernels, which read
// them repeatedly.
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

// The sum of v over the block.
__device__ __forceinline__ float block_sum(float v, float* sm) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) v += sm[i];
  return v;
}

// 65536 x 1280, fp32 to fp16: 88.6 us in a row of calls, 5.7 TB/s, and 102 us on cold caches; bound by HBM and
// by issue (65 %). The weights come from L1 for every row: in registers
// they cost more blocks per SM than they save (103 us with them and the next row held there; 94 us with
// a block per row).
template <typename X, typename Y, int VEC, int NV>
__global__ void __launch_bounds__(kMaxThreads) layernorm_row_kernel(const LayerNormOp p) {
  __shared__ float sm[2][2][kMaxThreads / 32];
  const int n = p.d / VEC, t = threadIdx.x;
  const float inv_d = 1.0f / p.d;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.T; row += gridDim.x, turn ^= 1) {
    const Vec<X, VEC>* x = reinterpret_cast<const Vec<X, VEC>*>(static_cast<const X*>(p.x) + row * p.d);
    Vec<X, VEC> cur[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (t + k * static_cast<int>(blockDim.x) < n) cur[k] = x[t + k * blockDim.x];
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (t + k * static_cast<int>(blockDim.x) < n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) s += to_f32(cur[k].v[i]);
    const float mean = block_sum(s, sm[turn][0]) * inv_d;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (t + k * static_cast<int>(blockDim.x) < n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float v = to_f32(cur[k].v[i]) - mean;
          s = fmaf(v, v, s);
        }
    const float rstd = 1.0f / sqrtf(block_sum(s, sm[turn][1]) * inv_d + p.eps);
    Vec<Y, VEC>* y = reinterpret_cast<Vec<Y, VEC>*>(static_cast<Y*>(p.y) + row * p.d);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (t + k * static_cast<int>(blockDim.x) < n) {
        const Vec<float, VEC> w = reinterpret_cast<const Vec<float, VEC>*>(p.w)[t + k * blockDim.x];
        const Vec<float, VEC> b = reinterpret_cast<const Vec<float, VEC>*>(p.b)[t + k * blockDim.x];
        Vec<Y, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; ++i) o.v[i] = from_f32<Y>(fmaf((to_f32(cur[k].v[i]) - mean) * rstd, w.v[i], b.v[i]));
        y[t + k * blockDim.x] = o;
      }
    if (t == 0) {
      if (p.mean) p.mean[row] = mean;
      if (p.rstd) p.rstd[row] = rstd;
    }
  }
}

// 65536 x 1280, fp32 with fp16 dy and an fp32 residual gradient: 203 us, 5.8 TB/s, and 8 us for the sums of the
// blocks' parts; bound by HBM. With NV 4 (4096 < d <= 8192) and an fp32 residual gradient the next row's registers
// spill 80 to 232 bytes a thread, 8 to 40 for bf16 rows.
// SMALL: blocks [0, dx_blocks) of the launch compute dx alone, the others 32 columns of dw and db each.
constexpr int kGroups = kMaxThreads / 32;
template <typename X, typename Y>
__device__ void layernorm_columns(const LayerNormOp& p, int block) {
  __shared__ float sw[kGroups][33], sb[kGroups][33];
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5, groups = blockDim.x >> 5, c = block * 32 + lane;
  float dw = 0.0f, db = 0.0f;
  if (c < p.d) {
#pragma unroll 4
    for (int r = group; r < p.T; r += groups) {
      const size_t at = static_cast<size_t>(r) * p.d + c;
      const float dy = to_f32(static_cast<const Y*>(p.dy)[at]);
      dw = fmaf(dy, (to_f32(static_cast<const X*>(p.x)[at]) - p.mean[r]) * p.rstd[r], dw);
      db += dy;
    }
  }
  sw[group][lane] = dw;
  sb[group][lane] = db;
  __syncthreads();
  if (group == 0 && c < p.d) {
    dw = db = 0.0f;
    for (int g = 0; g < groups; ++g) {
      dw += sw[g][lane];
      db += sb[g][lane];
    }
    p.dw[c] = dw;
    p.db[c] = db;
  }
}

template <typename X, typename Y, int VEC, int NV, bool RES, bool SMALL>
__global__ void __launch_bounds__(kMaxThreads) layernorm_backward_kernel(const LayerNormOp p, const int dx_blocks) {
  if (SMALL && static_cast<int>(blockIdx.x) >= dx_blocks) {
    layernorm_columns<X, Y>(p, blockIdx.x - dx_blocks);
    return;
  }
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
  for (int64_t row = blockIdx.x; row < p.T; row += dx_blocks, turn ^= 1) {
    if (row + dx_blocks < p.T) load(next, row + dx_blocks);
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (t + k * static_cast<int>(blockDim.x) < n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float dy = to_f32(cur.dy[k].v[i]), xh = (to_f32(cur.x[k].v[i]) - cur.mean) * cur.rstd, g = dy * w[k].v[i];
          a += g;
          b = fmaf(g, xh, b);
          if constexpr (!SMALL) {
            dw[k].v[i] = fmaf(dy, xh, dw[k].v[i]);
            db[k].v[i] += dy;
          }
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
  if constexpr (SMALL) return;
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
  __shared__ float sm[2][kMaxThreads / 32];
  const size_t row = blockIdx.x;
  const X* x = static_cast<const X*>(p.x) + row * p.d;
  float s = 0.0f;
  for (int c = threadIdx.x; c < p.d; c += kMaxThreads) s += to_f32(x[c]);
  const float mean = block_sum(s, sm[0]) / p.d;
  s = 0.0f;
  for (int c = threadIdx.x; c < p.d; c += kMaxThreads) {
    const float v = to_f32(x[c]) - mean;
    s = fmaf(v, v, s);
  }
  const float rstd = 1.0f / sqrtf(block_sum(s, sm[1]) / p.d + p.eps);
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

// ---- sums of the blocks' parts: 16 columns a block, 32 threads a column ---------------------------

__global__ void __launch_bounds__(512) layernorm_reduce_kernel(const float* part, int n, int d, float* dw, float* db) {
  __shared__ float sm[32][17];
  const int col = threadIdx.x & 15, w = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
  float s = 0.0f;
  if (c < 2 * d) {
#pragma unroll 8
    for (int i = w; i < n; i += 32) s += part[static_cast<size_t>(i) * 2 * d + c];
  }
  sm[w][col] = s;
  __syncthreads();
  const int lane = threadIdx.x & 31, column = threadIdx.x >> 5, out = blockIdx.x * 16 + column;
  s = warp_sum(sm[lane][column]);
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

// Blocks of a row kernel that fit the GPU at once, at most one per row.
template <typename K>
int resident(K kernel, const LayerNormOp& p, int threads, int most) {
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0) != cudaSuccess) return 0;
  return std::max(1, std::min(p.T, std::min(per_sm, most) * p.num_sms));
}

template <typename X, typename Y, int VEC, int NV>
cudaError_t forward_rows(const LayerNormOp& p, int n, cudaStream_t s) {
  const int threads = row_threads(n, NV), blocks = resident(layernorm_row_kernel<X, Y, VEC, NV>, p, threads, 32);
  if (blocks == 0) return cudaErrorInvalidConfiguration;
  layernorm_row_kernel<X, Y, VEC, NV><<<blocks, threads, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename X, typename Y>
cudaError_t forward(const LayerNormOp& p, cudaStream_t s) {
  const int vec = vector_width(p, sizeof(X), sizeof(Y)), n = p.d / vec;
  if (n <= 2 * kMaxThreads) return vec == 4 ? forward_rows<X, Y, 4, 2>(p, n, s) : forward_rows<X, Y, 1, 2>(p, n, s);
  if (n <= 4 * kMaxThreads) return vec == 4 ? forward_rows<X, Y, 4, 4>(p, n, s) : forward_rows<X, Y, 1, 4>(p, n, s);
  layernorm_wide_kernel<X, Y><<<p.T, kMaxThreads, 0, s>>>(p);
  return cudaGetLastError();
}

// Up to this many rows the second launch costs more than reading the rows twice: a block of columns walks
// all of them. One launch against two, d = 640 fp32 with fp16 dy: 128 rows 3.0 and 5.0 us, 384 rows 5.3 and
// 6.1, 512 rows 6.4 and 6.1, 4096 rows 42 and 12; d = 2560: 384 rows 6.6 and 9.0, 1024 rows 13.4 and 11.4.
constexpr int kSmallRows = 384;

template <typename X, typename Y, int VEC, int NV, bool RES>
cudaError_t backward_rows(const LayerNormOp& p, int n, cudaStream_t s) {
  if (p.T > 0 && p.T <= kSmallRows) {
    // At least 256 threads, for the blocks of columns.
    const int threads = std::max(256, row_threads(n, NV));
    layernorm_backward_kernel<X, Y, VEC, NV, RES, true><<<p.T + (p.d + 31) / 32, threads, 0, s>>>(p, p.T);
    return cudaGetLastError();
  }
  const int threads = row_threads(n, NV);
  const int blocks = resident(layernorm_backward_kernel<X, Y, VEC, NV, RES, false>, p, threads, kMaxParts);
  if (blocks == 0) return cudaErrorInvalidConfiguration;
  layernorm_backward_kernel<X, Y, VEC, NV, RES, false><<<blocks, threads, 0, s>>>(p, blocks);
  layernorm_reduce_kernel<<<(2 * p.d + 15) / 16, 512, 0, s>>>(p.workspace, blocks, p.d, p.dw, p.db);
  return cudaGetLastError();
}

template <typename X, typename Y, bool RES>
cudaError_t backward_by_size(const LayerNormOp& p, cudaStream_t s) {
  const int vec = vector_width(p, sizeof(X), sizeof(Y)), n = p.d / vec;
  if (n <= 2 * kMaxThreads)
    return vec == 4 ? backward_rows<X, Y, 4, 2, RES>(p, n, s) : backward_rows<X, Y, 1, 2, RES>(p, n, s);
  if (n <= 4 * kMaxThreads)
    return vec == 4 ? backward_rows<X, Y, 4, 4, RES>(p, n, s) : backward_rows<X, Y, 1, 4, RES>(p, n, s);
  const int blocks = parts(p.T, p.num_sms);
  if (p.T > 0) layernorm_wide_dx_kernel<X, Y><<<p.T, kMaxThreads, 0, s>>>(p);
  layernorm_wide_dw_kernel<X, Y><<<dim3((p.d + kMaxThreads - 1) / kMaxThreads, blocks), kMaxThreads, 0, s>>>(p);
  layernorm_reduce_kernel<<<(2 * p.d + 15) / 16, 512, 0, s>>>(p.workspace, blocks, p.d, p.dw, p.db);
  return cudaGetLastError();
}

template <typename X, typename Y>
cudaError_t backward(const LayerNormOp& p, cudaStream_t s) {
  return p.dres ? backward_by_size<X, Y, true>(p, s) : backward_by_size<X, Y, false>(p, s);
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
