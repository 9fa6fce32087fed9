// Operators on rows of logits x[V]:
//   log probabilities: lse = log sum exp x; logp = x[target] - lse; entropy = lse - sum p x with
//     p = exp(x - lse) (0 where p is 0); the k largest log probabilities, ties to the lowest id;
//   distillation from a teacher's alternatives (id_i, t_i), i < k, at temperature tau: with
//     p = softmax(t / tau) over the present alternatives and q = softmax(x / tau),
//     loss = tau^2 sum_i p_i (log p_i - log q[id_i]) and
//     dx_j = dloss tau (q_j - sum of the p_i with id_i = j).
//
// Two forms of each, both bound by HBM at size and by latency below:
//   V <= kSmallV (the encoder's 33 tokens): one row per thread. A warp copies its 32 rows, which are
//     one contiguous piece of memory when ld = V, into shared memory at an odd pitch, so that reading
//     along a row is free of bank conflicts, and every row's work is serial: no shuffles, and a gradient
//     row is finished in shared memory before it is written.
//   larger V: one block per row and a running maximum and sum, so x is read once for the sums. The
//     top k come from a second pass (out of L2) that collects what reaches a threshold at least k
//     elements are known to reach: see row_top.
#include <algorithm>

#include "common.cuh"
#include "train_common.cuh"
#include "train_ops.cuh"

namespace esm {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSmallV = 64;

// Keys that order like floats, -0 and +0 alike; 0 is below every number.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// ---- one row per thread --------------------------------------------------------------------------

// Calls f(row, column) for the rows x cols elements of a warp's rows, in memory order.
template <typename F>
__device__ __forceinline__ void warp_elements(int rows, int cols, F f) {
  const int lane = threadIdx.x & 31, q = 32 / cols, m = 32 % cols;
  int r = lane / cols, c = lane % cols;
#pragma unroll 4
  for (int i = lane; i < rows * cols; i += 32) {
    f(r, c);
    r += q;
    c += m;
    if (c >= cols) {
      c -= cols;
      ++r;
    }
  }
}

// The 32 rows of a warp and their shared memory: `x` (pitch V | 1), and two arrays of pitch k | 1.
struct WarpRows {
  int64_t r0;
  int rows, lane, px, pk;
  float *x, *a, *b;
  __device__ WarpRows(const LogitsOp& p, float* smem) {
    const int warp = threadIdx.x >> 5;
    lane = threadIdx.x & 31;
    px = p.V | 1;
    pk = p.k | 1;
    r0 = (static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + warp) * 32;
    rows = static_cast<int>(min(static_cast<int64_t>(32), p.T - r0));
    x = smem + static_cast<size_t>(warp) * 32 * (px + 2 * pk);
    a = x + 32 * px;
    b = a + 32 * pk;
  }
};
size_t warp_rows_bytes(const LogitsOp& p) { return 32 * sizeof(float) * ((p.V | 1) + 2 * (p.k | 1)); }

template <typename E>
__global__ void logprobs_small_kernel(const LogitsOp p) {
  extern __shared__ float smem_f[];
  const WarpRows w(p, smem_f);
  if (w.rows <= 0) return;
  const E* x = static_cast<const E*>(p.logits);
  warp_elements(w.rows, p.V, [&](int r, int c) { w.x[r * w.px + c] = to_f32(x[(w.r0 + r) * p.ld + c]); });
  __syncwarp();
  if (w.lane < w.rows) {
    const int64_t t = w.r0 + w.lane;
    float* row = w.x + w.lane * w.px;
    float m = -INFINITY;
    for (int j = 0; j < p.V; ++j) m = fmaxf(m, row[j]);
    float s = 0.0f, u = 0.0f;
#pragma unroll 4
    for (int j = 0; j < p.V; ++j) {
      const float v = row[j] - m, e = fast_exp2(v * kLog2e);
      s += e;
      u += e > 0.0f ? e * v : 0.0f;  // a NaN reaches s
    }
    const float log_s = logf(s);
    if (p.entropy) p.entropy[t] = s == s ? log_s - u / s : s;
    if (p.logp) {
      const int id = p.targets[t];
      p.logp[t] = id >= 0 && id < p.V ? row[id] - m - log_s : 0.0f;
    }
    if (p.k > 0) {
      // k times the best key that is left; the first of equal ones.
      uint32_t* keys = reinterpret_cast<uint32_t*>(row);
      for (int j = 0; j < p.V; ++j) keys[j] = order_key(row[j]);
      for (int i = 0; i < p.k; ++i) {
        uint32_t best = 0;
        int id = 0;
#pragma unroll 4
        for (int j = 0; j < p.V; ++j) {
          const uint32_t key = keys[j];
          if (key > best) {
            best = key;
            id = j;
          }
        }
        keys[id] = 0;
        w.a[w.lane * w.pk + i] = __int_as_float(s == s ? id : -1);
        w.b[w.lane * w.pk + i] = s == s ? key_value(best) - m - log_s : s;
      }
    }
  }
  if (p.k > 0) {
    __syncwarp();
    warp_elements(w.rows, p.k, [&](int r, int c) {
      p.top_ids[(w.r0 + r) * p.k + c] = __float_as_int(w.a[r * w.pk + c]);
      p.top_logp[(w.r0 + r) * p.k + c] = w.b[r * w.pk + c];
    });
  }
}

// The teacher's part of a row: ids in `id` (as bits, -1 where absent), logits in `v`, which become the
// probabilities. Returns whether there are any; *log_scale is what makes (v - top) / tau a log
// probability.
struct Teacher {
  bool any;
  float top, log_s;
};
__device__ __forceinline__ Teacher teacher_row(float* id, float* v, int k, int V, float inv_tau) {
  Teacher t{false, -INFINITY, 0.0f};
  for (int i = 0; i < k; ++i) {
    const int a = __float_as_int(id[i]);
    if (a < 0 || a >= V) {
      id[i] = __int_as_float(-1);
      v[i] = -INFINITY;
    }
    t.top = fmaxf(t.top, v[i]);
  }
  t.any = t.top > -INFINITY;
  float s = 0.0f;
  for (int i = 0; i < k; ++i) s += __float_as_int(id[i]) >= 0 ? fast_exp2((v[i] - t.top) * inv_tau * kLog2e) : 0.0f;
  t.log_s = logf(s);
  return t;
}

// Copies the warp's alternatives into shared memory: ids to w.a, logits to w.b.
__device__ __forceinline__ void load_alternatives(const LogitsOp& p, const WarpRows& w) {
  warp_elements(w.rows, p.k, [&](int r, int c) {
    w.a[r * w.pk + c] = __int_as_float(p.alt_ids[(w.r0 + r) * p.k + c]);
    w.b[r * w.pk + c] = p.alt_logits[(w.r0 + r) * p.k + c];
  });
}

template <typename E>
__global__ void distill_loss_small_kernel(const LogitsOp p) {
  extern __shared__ float smem_f[];
  const WarpRows w(p, smem_f);
  if (w.rows <= 0) return;
  const E* x = static_cast<const E*>(p.logits);
  warp_elements(w.rows, p.V, [&](int r, int c) { w.x[r * w.px + c] = to_f32(x[(w.r0 + r) * p.ld + c]); });
  load_alternatives(p, w);
  __syncwarp();
  if (w.lane >= w.rows) return;
  const int64_t t = w.r0 + w.lane;
  const float inv_tau = 1.0f / p.temperature;
  const float* row = w.x + w.lane * w.px;
  float *id = w.a + w.lane * w.pk, *v = w.b + w.lane * w.pk;
  float m = -INFINITY, s = 0.0f;
  for (int j = 0; j < p.V; ++j) m = fmaxf(m, row[j]);
#pragma unroll 4
  for (int j = 0; j < p.V; ++j) s += fast_exp2((row[j] - m) * inv_tau * kLog2e);
  const float log_s = logf(s);
  const Teacher tr = teacher_row(id, v, p.k, p.V, inv_tau);
  float loss = 0.0f;
  for (int i = 0; i < p.k; ++i) {
    const int a = __float_as_int(id[i]);
    const float logp = (v[i] - tr.top) * inv_tau - tr.log_s, pr = a >= 0 ? fast_exp2(logp * kLog2e) : 0.0f;
    if (!(pr <= 0.0f)) loss += pr * (logp - ((row[a] - m) * inv_tau - log_s));
  }
  p.loss[t] = tr.any ? p.temperature * p.temperature * loss : 0.0f;
  p.lse[t] = m * inv_tau + log_s;
}

template <typename E>
__global__ void distill_backward_small_kernel(const LogitsOp p) {
  extern __shared__ float smem_f[];
  const WarpRows w(p, smem_f);
  if (w.rows <= 0) return;
  const E* x = static_cast<const E*>(p.logits);
  E* dx = static_cast<E*>(p.dlogits);
  warp_elements(w.rows, p.V, [&](int r, int c) { w.x[r * w.px + c] = to_f32(x[(w.r0 + r) * p.ld + c]); });
  load_alternatives(p, w);
  __syncwarp();
  if (w.lane < w.rows) {
    const int64_t t = w.r0 + w.lane;
    const float inv_tau = 1.0f / p.temperature, g = p.dloss[t] * p.temperature, lse = p.lse[t];
    float* row = w.x + w.lane * w.px;
    float *id = w.a + w.lane * w.pk, *v = w.b + w.lane * w.pk;
    const Teacher tr = teacher_row(id, v, p.k, p.V, inv_tau);
    const bool none = !tr.any || g == 0.0f;
#pragma unroll 4
    for (int j = 0; j < p.V; ++j) row[j] = none ? 0.0f : g * fast_exp2((row[j] * inv_tau - lse) * kLog2e);
    for (int i = 0; i < p.k && !none; ++i) {
      const int a = __float_as_int(id[i]);
      if (a >= 0) row[a] -= g * fast_exp2(((v[i] - tr.top) * inv_tau - tr.log_s) * kLog2e);
    }
  }
  __syncwarp();
  warp_elements(w.rows, p.V, [&](int r, int c) { dx[(w.r0 + r) * p.ld_grad + c] = from_f32<E>(w.x[r * w.px + c]); });
}

// ---- one block per row -----------------------------------------------------------------------------

template <typename E>
struct alignas(16) Pack {
  E v[16 / sizeof(E)];
};

// Calls f(first index, values, count) for the row's elements: 16-byte vectors where the row allows, and
// the elements before and after them one at a time. Every thread's indices ascend but for the head,
// whose elements come first.
template <int NT, typename E, typename F>
__device__ __forceinline__ void row_elements(const E* x, int V, F f) {
  constexpr int N = 16 / sizeof(E);
  const int head = min(V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(E)));
  const int packs = (V - head) / N;
  if (static_cast<int>(threadIdx.x) < head) {
    const float v[N] = {to_f32(x[threadIdx.x])};
    f(static_cast<int>(threadIdx.x), v, 1);
  }
  const Pack<E>* body = reinterpret_cast<const Pack<E>*>(x + head);
#pragma unroll 4
  for (int i = threadIdx.x; i < packs; i += NT) {
    const Pack<E> raw = body[i];
    float v[N];
#pragma unroll
    for (int u = 0; u < N; ++u) v[u] = to_f32(raw.v[u]);
    f(head + i * N, v, N);
  }
  const int at = head + packs * N + threadIdx.x;
  if (at < V) {
    const float v[N] = {to_f32(x[at])};
    f(at, v, 1);
  }
}

// Running maximum m, sum of e = exp((x - m) inv_tau) and, with ENTROPY, of e (x - m) inv_tau.
// A NaN or +inf makes s NaN.
struct Online {
  float m = -INFINITY, s = 0.0f, u = 0.0f;
};

template <bool ENTROPY, int N>
__device__ __forceinline__ void online_add(Online& o, const float (&v)[N], int n, float c, float inv_tau) {
  float top = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i)
    if (i < n) top = fmaxf(top, v[i]);
  if (top > o.m) {
    const float d = (o.m - top) * inv_tau, a = fast_exp2(d * kLog2e);
    if (ENTROPY) o.u = a > 0.0f ? a * (o.u + d * o.s) : 0.0f;  // d may be infinite where a is 0
    o.s = a * o.s;  // a is 0 where there was nothing; a NaN stays
    o.m = top;
  }
  if (o.m == -INFINITY) {  // nothing but -inf, or a NaN, so far
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n && v[i] != v[i]) o.s = v[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) {
      const float d = v[i] - o.m, e = fast_exp2(d * c);
      o.s += e;
      if (ENTROPY) o.u += e > 0.0f ? e * d * inv_tau : 0.0f;
    }
}

__device__ __forceinline__ void online_join(Online& o, float m, float s, float u, float inv_tau) {
  const float top = fmaxf(o.m, m);
  if (top == -INFINITY) {
    o.s += s;  // 0, or NaN
    return;
  }
  const float da = (o.m - top) * inv_tau, db = (m - top) * inv_tau;
  const float a = fast_exp2(da * kLog2e), b = fast_exp2(db * kLog2e);
  o.u = (a > 0.0f ? a * (o.u + da * o.s) : 0.0f) + (b > 0.0f ? b * (u + db * s) : 0.0f);
  o.s = a * o.s + b * s;
  o.m = top;
}

// The row's m, s, u in every thread.
template <int NT>
__device__ __forceinline__ Online block_join(Online o, float inv_tau) {
  for (int k = 16; k > 0; k >>= 1) {
    const float m = __shfl_xor_sync(0xffffffffu, o.m, k), s = __shfl_xor_sync(0xffffffffu, o.s, k);
    const float u = __shfl_xor_sync(0xffffffffu, o.u, k);
    online_join(o, m, s, u, inv_tau);
  }
  if constexpr (NT > 32) {
    __shared__ Online sm[NT / 32];
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = o;
    __syncthreads();
    o = Online();
    for (int i = 0; i < NT / 32; ++i) online_join(o, sm[i].m, sm[i].s, sm[i].u, inv_tau);
  } else {  // the lanes joined in different orders
    o.m = __shfl_sync(0xffffffffu, o.m, 0);
    o.s = __shfl_sync(0xffffffffu, o.s, 0);
    o.u = __shfl_sync(0xffffffffu, o.u, 0);
  }
  return o;
}

// The top k of a row. `best` / `at` are the thread's own largest element and its (lowest) index. A
// warp's g-th largest of these, with g = ceil(k / warps), is reached by g elements of that warp, so the
// smallest such value over the warps is reached by k elements of the row. A second pass collects
// what reaches it, with the index as the tie-break, typically a few times k elements, and those are
// ranked against each other. Should more reach it than there is room for (rows in an order that
// favours some threads), the k are taken one by one, each a pass over the row.
constexpr int kCandidates = 1024;
template <int NT, typename E>
__device__ void row_top(const LogitsOp& p, const E* x, int64_t t, float best, int at, const Online& o) {
  constexpr int kWarps = NT / 32;
  __shared__ uint64_t cand[kCandidates];
  __shared__ uint64_t bound[kWarps];
  __shared__ int count;
  const int lane = threadIdx.x & 31;
  const float log_s = logf(o.s);
  if (!(o.s == o.s) || o.m == -INFINITY) {  // no distribution
    for (int i = threadIdx.x; i < p.k; i += NT) {
      p.top_ids[t * p.k + i] = -1;
      p.top_logp[t * p.k + i] = NAN;
    }
    return;
  }
  uint32_t key = at >= 0 ? order_key(best) : 0, last = 0, last_at = 0;
  for (int i = 0; i < (p.k + kWarps - 1) / kWarps; ++i) {
    last = __reduce_max_sync(0xffffffffu, key);
    last_at = __reduce_max_sync(0xffffffffu, key == last ? ~static_cast<uint32_t>(at) : 0u);
    if (key == last && ~static_cast<uint32_t>(at) == last_at) key = 0;
  }
  if (lane == 0) bound[threadIdx.x >> 5] = last ? static_cast<uint64_t>(last) << 32 | last_at : 0;
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  uint64_t least = ~0ull;
  for (int i = 0; i < kWarps; ++i) least = min(least, bound[i]);
  // As a float the bound's value part is a cheap first test; 0 (a warp without elements) lets all pass.
  const float floor_value = least ? key_value(static_cast<uint32_t>(least >> 32)) : -INFINITY;
  row_elements<NT>(x, p.V, [&](int j, const auto& v, int n) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(v) / 4); ++i)
      if (i < n && v[i] >= floor_value) {
        const uint64_t c = static_cast<uint64_t>(order_key(v[i])) << 32 | ~static_cast<uint32_t>(j + i);
        if (c >= least) {
          const int slot = atomicAdd(&count, 1);
          if (slot < kCandidates) cand[slot] = c;
        }
      }
  });
  __syncthreads();
  const int m = count;
  if (m <= kCandidates) {
    for (int i = threadIdx.x; i < m; i += NT) {
      const uint64_t c = cand[i];
      int rank = 0;
      for (int j = 0; j < m; ++j) rank += cand[j] > c;
      if (rank < p.k) {
        p.top_ids[t * p.k + rank] = static_cast<int>(~static_cast<uint32_t>(c));
        p.top_logp[t * p.k + rank] = key_value(static_cast<uint32_t>(c >> 32)) - o.m - log_s;
      }
    }
    return;
  }
  uint64_t taken = ~0ull;
  for (int i = 0; i < p.k; ++i) {
    uint64_t top = 0;
    row_elements<NT>(x, p.V, [&](int j, const auto& v, int n) {
      for (int u = 0; u < n; ++u) {
        const uint64_t c = static_cast<uint64_t>(order_key(v[u])) << 32 | ~static_cast<uint32_t>(j + u);
        if (c < taken && c > top) top = c;
      }
    });
    for (int k = 16; k > 0; k >>= 1) top = max(top, static_cast<uint64_t>(__shfl_xor_sync(0xffffffffu, top, k)));
    __syncthreads();  // bound has been read
    if (lane == 0) bound[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) top = max(top, bound[w]);
    taken = top;
    if (threadIdx.x == 0) {
      p.top_ids[t * p.k + i] = static_cast<int>(~static_cast<uint32_t>(top));
      p.top_logp[t * p.k + i] = key_value(static_cast<uint32_t>(top >> 32)) - o.m - log_s;
    }
  }
}

template <int NT, typename E>
__global__ void __launch_bounds__(NT) logprobs_row_kernel(const LogitsOp p) {
  const int64_t t = blockIdx.x;
  const E* x = static_cast<const E*>(p.logits) + t * p.ld;
  Online o;
  float best = -INFINITY;
  int at = -1;
  row_elements<NT>(x, p.V, [&](int j, const auto& v, int n) {
    online_add<true>(o, v, n, kLog2e, 1.0f);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(v) / 4); ++i)
      if (i < n && (v[i] > best || at < 0)) {
        best = v[i];
        at = j + i;
      }
  });
  o = block_join<NT>(o, 1.0f);
  if (threadIdx.x == 0) {
    const bool none = !(o.s == o.s) || o.m == -INFINITY;
    const float log_s = logf(o.s);
    if (p.entropy) p.entropy[t] = none ? NAN : log_s - o.u / o.s;
    if (p.logp) {
      const int id = p.targets[t];
      p.logp[t] = id >= 0 && id < p.V ? (none ? NAN : to_f32(x[id]) - o.m - log_s) : 0.0f;
    }
  }
  if (p.k > 0) row_top<NT>(p, x, t, best, at, o);
}

// Lane i and 32 + i of a warp: the teacher's alternatives i and 32 + i, probabilities and log
// probabilities (0 where absent). Returns whether the row has any.
__device__ __forceinline__ bool teacher(const LogitsOp& p, int64_t t, int lane, int (&id)[2], float (&pr)[2],
                                        float (&logp)[2]) {
  const float inv_tau = 1.0f / p.temperature;
  float v[2], m = -INFINITY;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int i = lane + 32 * c;
    id[c] = i < p.k ? p.alt_ids[t * p.k + i] : -1;
    if (id[c] >= p.V) id[c] = -1;
    v[c] = id[c] >= 0 ? p.alt_logits[t * p.k + i] : -INFINITY;
    m = fmaxf(m, v[c]);
  }
  m = warp_max(m);
  float s = 0.0f;
#pragma unroll
  for (int c = 0; c < 2; ++c) s += id[c] >= 0 ? fast_exp2((v[c] - m) * inv_tau * kLog2e) : 0.0f;
  const float log_s = logf(warp_sum(s));
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    logp[c] = (v[c] - m) * inv_tau - log_s;
    pr[c] = id[c] >= 0 ? fast_exp2(logp[c] * kLog2e) : 0.0f;
  }
  return m > -INFINITY;
}

template <int NT, typename E>
__global__ void __launch_bounds__(NT) distill_loss_row_kernel(const LogitsOp p) {
  const int64_t t = blockIdx.x;
  const E* x = static_cast<const E*>(p.logits) + t * p.ld;
  const float inv_tau = 1.0f / p.temperature;
  Online o;
  row_elements<NT>(x, p.V, [&](int, const auto& v, int n) { online_add<false>(o, v, n, inv_tau * kLog2e, inv_tau); });
  o = block_join<NT>(o, inv_tau);
  if (threadIdx.x >= 32) return;
  const float log_s = logf(o.m == -INFINITY ? NAN : o.s);
  int id[2];
  float pr[2], logp[2], loss = 0.0f;
  const bool any = teacher(p, t, threadIdx.x, id, pr, logp);
#pragma unroll
  for (int c = 0; c < 2; ++c)
    if (!(pr[c] <= 0.0f)) loss += pr[c] * (logp[c] - ((to_f32(x[id[c]]) - o.m) * inv_tau - log_s));
  loss = warp_sum(loss);
  if (threadIdx.x == 0) {
    p.loss[t] = any ? p.temperature * p.temperature * loss : 0.0f;
    p.lse[t] = o.m * inv_tau + log_s;
  }
}

template <int NT, typename E>
__global__ void __launch_bounds__(NT) distill_backward_row_kernel(const LogitsOp p) {
  __shared__ bool any_sm;
  const int64_t t = blockIdx.x;
  const E* x = static_cast<const E*>(p.logits) + t * p.ld;
  E* dx = static_cast<E*>(p.dlogits) + t * p.ld_grad;
  const float inv_tau = 1.0f / p.temperature, g = p.dloss[t] * p.temperature, lse = p.lse[t];
  int id[2];
  float pr[2], logp[2];
  if (threadIdx.x < 32) {
    const bool any = teacher(p, t, threadIdx.x, id, pr, logp);
    if (threadIdx.x == 0) any_sm = any;
  }
  __syncthreads();
  const bool none = !any_sm || g == 0.0f;
  const float c = inv_tau * kLog2e, d = -lse * kLog2e;
  // 16-byte stores where the gradient's row starts at the same place in a vector as the logits'.
  const bool together = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
  row_elements<NT>(x, p.V, [&](int j, const auto& v, int n) {
    constexpr int N = static_cast<int>(sizeof(v) / 4);
    Pack<E> out;
#pragma unroll
    for (int i = 0; i < N; ++i) out.v[i] = from_f32<E>(none ? 0.0f : g * fast_exp2(fmaf(v[i], c, d)));
    if (n == N && N > 1 && together) {
      *reinterpret_cast<Pack<E>*>(dx + j) = out;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < n) dx[j + i] = out.v[i];
    }
  });
  if (none) return;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  // The alternatives' own columns again: the first of equal ids writes, with all their probability.
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float sum = 0.0f;
    bool first = id[e] >= 0;
    for (int i = 0; i < p.k; ++i) {
      const int other = __shfl_sync(0xffffffffu, i < 32 ? id[0] : id[1], i & 31);
      const float o = __shfl_sync(0xffffffffu, i < 32 ? pr[0] : pr[1], i & 31);
      if (other == id[e]) {
        sum += o;
        if (i < static_cast<int>(threadIdx.x) + 32 * e) first = false;
      }
    }
    if (first) dx[id[e]] = from_f32<E>(g * (fast_exp2(fmaf(to_f32(x[id[e]]), c, d)) - sum));
  }
}

// ---- launches ------------------------------------------------------------------------------------

// Small rows: four warps a block once that fills the GPU, else one.
struct SmallGrid {
  unsigned blocks, threads;
  size_t smem;
  explicit SmallGrid(const LogitsOp& p) {
    const unsigned warps = (static_cast<unsigned>(p.T) + 31) / 32;
    // Up to 48 KB of shared memory a block; more than 24 KB a warp does not occur (V, k <= 64).
    const unsigned per = warps >= 1024 && 4 * warp_rows_bytes(p) <= 48u << 10 ? 4 : 1;
    blocks = (warps + per - 1) / per;
    threads = 32 * per;
    smem = per * warp_rows_bytes(p);
  }
};

template <typename E>
cudaError_t logprobs(const LogitsOp& p, cudaStream_t s) {
  if (p.V <= kSmallV) {
    const SmallGrid g(p);
    logprobs_small_kernel<E><<<g.blocks, g.threads, g.smem, s>>>(p);
  } else if (p.V <= 1024 && p.k <= 16) {  // a warp's 32 maxima bound the top k
    logprobs_row_kernel<32, E><<<p.T, 32, 0, s>>>(p);
  } else if (p.V <= 4096) {
    logprobs_row_kernel<128, E><<<p.T, 128, 0, s>>>(p);
  } else {
    logprobs_row_kernel<512, E><<<p.T, 512, 0, s>>>(p);
  }
  return cudaGetLastError();
}

template <typename E>
cudaError_t loss(const LogitsOp& p, cudaStream_t s) {
  if (p.V <= kSmallV) {
    const SmallGrid g(p);
    distill_loss_small_kernel<E><<<g.blocks, g.threads, g.smem, s>>>(p);
  } else if (p.V <= 1024) {
    distill_loss_row_kernel<32, E><<<p.T, 32, 0, s>>>(p);
  } else if (p.V <= 4096) {
    distill_loss_row_kernel<128, E><<<p.T, 128, 0, s>>>(p);
  } else {
    distill_loss_row_kernel<512, E><<<p.T, 512, 0, s>>>(p);
  }
  return cudaGetLastError();
}

template <typename E>
cudaError_t gradient(const LogitsOp& p, cudaStream_t s) {
  if (p.V <= kSmallV) {
    const SmallGrid g(p);
    distill_backward_small_kernel<E><<<g.blocks, g.threads, g.smem, s>>>(p);
  } else if (p.V <= 1024) {
    distill_backward_row_kernel<32, E><<<p.T, 32, 0, s>>>(p);
  } else if (p.V <= 4096) {
    distill_backward_row_kernel<128, E><<<p.T, 128, 0, s>>>(p);
  } else {
    distill_backward_row_kernel<512, E><<<p.T, 512, 0, s>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace

#define ESM_BY_TYPE(fn)                                   \
  switch (p.dtype) {                                      \
    case ESM_F32: return fn<float>(p, s);                 \
    case ESM_F16: return fn<__half>(p, s);                \
    default: return fn<__nv_bfloat16>(p, s);              \
  }

cudaError_t launch_token_logprobs(const LogitsOp& p, cudaStream_t s) { ESM_BY_TYPE(logprobs) }
cudaError_t launch_distill_loss(const LogitsOp& p, cudaStream_t s) { ESM_BY_TYPE(loss) }
cudaError_t launch_distill_backward(const LogitsOp& p, cudaStream_t s) { ESM_BY_TYPE(gradient) }

}  // namespace esm
