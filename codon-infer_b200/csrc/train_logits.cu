// Operators on rows of logits x[V]:
//   log probabilities: lse = log sum exp x; logp = x[target] - lse; entropy = lse - sum p x with
//     p = exp(x - lse) (0 where p is 0); the k largest log probabilities, ties to the lowest id;
//   distillation from a teacher's alternatives (id_i, t_i), i < k, at temperature tau: with
//     p = softmax(t / tau) over the present alternatives and q = softmax(x / tau),
//     loss = tau^2 sum_i p_i (log p_i - log q[id_i]) and
//     dx_j = dloss tau (q_j - sum of the p_i with id_i = j).
//
// Two forms of each, both bound by HBM at size and by latency below:
//   V <= kSmallV (the encoder's 33 tokens): four lanes per row, which keep its elements in registers, so a
//     row is read once, reductions take two shuffles, and eight rows share a warp's instructions.
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
// The distillation gradient takes q = exp(x / tau - lse) from the loss's lse while that is at most this large: the
// rounding of lse and of x / tau is then at most 2^-17 of q (32 x 2^-24, four times). A row beyond it, for its logits or a low
// temperature, takes its maximum and sum again, and subtracts the maximum first. 1021 x 32003 fp16: 29 us, and
// 38 us with every row beyond it; 65536 x 33 fp32: 8.2 and 9.0.
constexpr float kRoundedLse = 32.0f;

// Keys that order like floats, -0 and +0 alike; 0 is below every number.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// ---- four lanes per row -----------------------------------------------------------------------------

// Lane q of a row's four has elements q, q + 4, .. (N of them, -inf past the end).
template <typename E, int N>
__device__ __forceinline__ void load_quad(const E* x, int V, int q, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = q + 4 * i < V ? to_f32(x[q + 4 * i]) : -INFINITY;
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

// A block of 128 threads has 32 rows; lanes past the last row work on it again and write nothing.
struct QuadRow {
  int64_t t;
  int q;
  bool real;
  __device__ explicit QuadRow(int T) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x >> 2);
    real = r < T;
    t = real ? r : T - 1;
    q = threadIdx.x & 3;
  }
};

// 90600 x 33 fp32, k = 5: 13 us, 16 on cold caches (24 MB: 0.9 and 0.75 TB/s). Bound by the instructions of
// the top k, 66 % of the issue rate; a thread per row took 14 us, a warp per row 111.
template <typename E, int N>
__global__ void __launch_bounds__(128) logprobs_quad_kernel(const LogitsOp p) {
  const QuadRow r(p.T);
  const E* x = static_cast<const E*>(p.logits) + r.t * p.ld;
  float v[N];
  load_quad<E, N>(x, p.V, r.q, v);
  const int target = p.targets ? p.targets[r.t] : -1;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, v[i]);
  m = quad_max(m);
  float s = 0.0f, u = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (r.q + 4 * i < p.V) {
      const float d = v[i] - m, e = fast_exp2(d * kLog2e);
      s += e;
      u += e > 0.0f ? e * d : 0.0f;  // a NaN reaches s
    }
  }
  s = quad_sum(s);
  u = quad_sum(u);
  const bool none = s != s;
  const float log_s = logf(s);
  if (r.real && r.q == 0) {
    if (p.entropy) p.entropy[r.t] = none ? NAN : log_s - u / s;
    if (p.logp) p.logp[r.t] = target >= 0 && target < p.V ? to_f32(x[target]) - m - log_s : 0.0f;
  }
  if (p.k == 0) return;
  // k times the best key that is left, the first of equal ones; taken and missing elements have key 0.
  uint32_t key[N];
#pragma unroll
  for (int i = 0; i < N; ++i) key[i] = r.q + 4 * i < p.V ? order_key(v[i]) : 0u;
  if (p.k > N + N / 4) {  // many: every element's rank, by comparing it with all the others
    int rank[N];
#pragma unroll
    for (int j = 0; j < N; ++j) rank[j] = 0;
#pragma unroll 1
    for (int o = 0; o < 4; ++o) {
      const uint32_t before = o < r.q;  // a lane's elements j are in front of those of later lanes
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t other = __shfl_sync(0xffffffffu, key[i], o, 4);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (i < j) rank[j] += other >= key[j];
          else if (i > j) rank[j] += other > key[j];
          else rank[j] += other > key[j] - before;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (r.real && r.q + 4 * j < p.V && rank[j] < p.k) {
        p.top_ids[r.t * p.k + rank[j]] = none ? -1 : r.q + 4 * j;
        p.top_logp[r.t * p.k + rank[j]] = none ? NAN : v[j] - m - log_s;
      }
    return;
  }
  for (int i = 0; i < p.k; ++i) {
    uint32_t best = 0;
    int id = r.q;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (key[j] > best) {
        best = key[j];
        id = r.q + 4 * j;
      }
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, best, o);
      const int other_id = __shfl_xor_sync(0xffffffffu, id, o);
      if (other > best || (other == best && other_id < id)) {
        best = other;
        id = other_id;
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (r.q + 4 * j == id) key[j] = 0;
    if (r.real && r.q == (i & 3)) {
      p.top_ids[r.t * p.k + i] = none ? -1 : id;
      p.top_logp[r.t * p.k + i] = none ? NAN : key_value(best) - m - log_s;
    }
  }
}

// The teacher's alternatives of a row of four lanes: lane q has i = q, q + 4, ..; ids -1 where absent.
constexpr int kQuadAlts = ESM_MAX_ALTERNATIVES / 4;
template <int K>
struct QuadTeacher {
  int id[K];
  float v[K];  // logits, then log probabilities
  bool any;
  __device__ __forceinline__ void load(const LogitsOp& p, const QuadRow& r) {
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const int i = r.q + 4 * c;
      id[c] = i < p.k ? p.alt_ids[r.t * p.k + i] : -1;
      v[c] = i < p.k ? p.alt_logits[r.t * p.k + i] : -INFINITY;
    }
  }
  __device__ __forceinline__ void normalise(int V, float inv_tau) {
    float top = -INFINITY, s = 0.0f;
    bool there = false;  // a NaN is not dropped by this as by the maximum: it has to show in the loss
#pragma unroll
    for (int c = 0; c < K; ++c) {
      if (id[c] < 0 || id[c] >= V) {
        id[c] = -1;
        v[c] = -INFINITY;
      }
      top = fmaxf(top, v[c]);
      there |= v[c] != -INFINITY;
    }
    top = quad_max(top);
    any = quad_max(there) > 0.0f;
#pragma unroll
    for (int c = 0; c < K; ++c) {
      v[c] = (v[c] - top) * inv_tau;
      s += id[c] >= 0 ? fast_exp2(v[c] * kLog2e) : 0.0f;
    }
    const float log_s = logf(quad_sum(s));
#pragma unroll
    for (int c = 0; c < K; ++c) v[c] -= log_s;
  }
  __device__ __forceinline__ float prob(int c) const { return id[c] >= 0 ? fast_exp2(v[c] * kLog2e) : 0.0f; }
};

// 65536 x 33 fp32, k up to 16: loss 6.4 us, gradient 8.2 (8.7 and 10.9 on cold caches); issue 52 and 64 %.
template <typename E, int N, int K>
__global__ void __launch_bounds__(128) distill_loss_quad_kernel(const LogitsOp p) {
  const QuadRow r(p.T);
  const E* x = static_cast<const E*>(p.logits) + r.t * p.ld;
  const float inv_tau = 1.0f / p.temperature;
  QuadTeacher<K> tr;
  tr.load(p, r);
  float v[N];
  load_quad<E, N>(x, p.V, r.q, v);
  float m = -INFINITY, s = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, v[i]);
  m = quad_max(m);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (r.q + 4 * i < p.V) s += fast_exp2((v[i] - m) * inv_tau * kLog2e);
  const float log_s = logf(quad_sum(s));
  tr.normalise(p.V, inv_tau);
  float loss = 0.0f;
#pragma unroll
  for (int c = 0; c < K; ++c) {
    const float pr = tr.prob(c);
    if (!(pr <= 0.0f)) loss += pr * (tr.v[c] - ((to_f32(x[tr.id[c]]) - m) * inv_tau - log_s));
  }
  loss = quad_sum(loss);
  if (r.real && r.q == 0) {
    p.loss[r.t] = tr.any ? p.temperature * p.temperature * loss : 0.0f;
    p.lse[r.t] = m * inv_tau + log_s;
  }
}

template <typename E, int N, int K>
__global__ void __launch_bounds__(128) distill_backward_quad_kernel(const LogitsOp p) {
  const QuadRow r(p.T);
  const E* x = static_cast<const E*>(p.logits) + r.t * p.ld;
  E* dx = static_cast<E*>(p.dlogits) + r.t * p.ld_grad;
  const float inv_tau = 1.0f / p.temperature, g = p.dloss[r.t] * p.temperature, lse = p.lse[r.t];
  QuadTeacher<K> tr;
  tr.load(p, r);
  float v[N];
  load_quad<E, N>(x, p.V, r.q, v);
  tr.normalise(p.V, inv_tau);
  const bool none = !tr.any || g == 0.0f;
  const bool again = !(fabsf(lse) <= kRoundedLse);
  if (__any_sync(0xffffffffu, again)) {  // each row by its own lse, whatever its neighbours in the warp do
    float m = -INFINITY, s = 0.0f, e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, v[i]);
    m = quad_max(m);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      e[i] = r.q + 4 * i < p.V ? fast_exp2((v[i] - m) * inv_tau * kLog2e) : 0.0f;
      s += e[i];
    }
    const float inv_s = 1.0f / quad_sum(s);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = again ? e[i] * inv_s : fast_exp2((v[i] * inv_tau - lse) * kLog2e);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = fast_exp2((v[i] * inv_tau - lse) * kLog2e);
  }
  // Every alternative to all four lanes; the one that has its column subtracts its probability.
#pragma unroll
  for (int c = 0; c < K; ++c) {
    if (4 * c >= p.k) break;
    const float pr = tr.prob(c);
#pragma unroll
    for (int o = 0; o < 4; ++o) {
      const int id = __shfl_sync(0xffffffffu, tr.id[c], o, 4);
      const float pi = __shfl_sync(0xffffffffu, pr, o, 4);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (id == r.q + 4 * i) v[i] -= pi;
    }
  }
  if (!r.real) return;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (r.q + 4 * i < p.V) dx[r.q + 4 * i] = from_f32<E>(none ? 0.0f : g * v[i]);
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

// TOP: *at is the index of the first element that equals o.m (j that of v[0]).
template <bool TOP, bool ENTROPY, int N>
__device__ __forceinline__ void online_add(Online& o, int* at, int j, const float (&v)[N], int n, float c, float inv_tau) {
  float top = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i)
    if (i < n) top = fmaxf(top, v[i]);
  if (top > o.m) {  // seldom, after the first few elements
    const float d = (o.m - top) * inv_tau, a = fast_exp2(d * kLog2e);
    if (ENTROPY) o.u = a > 0.0f ? a * (o.u + d * o.s) : 0.0f;  // d may be infinite where a is 0
    o.s = a * o.s;  // a is 0 where there was nothing; a NaN stays
    o.m = top;
    if (TOP) {
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
        if (i < n && v[i] == top) *at = j + i;
    }
  }
  if (o.m == -INFINITY) {  // nothing but -inf, or a NaN, so far
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n && v[i] != v[i]) o.s = v[i];
    if (TOP && *at < 0) *at = j;
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) {
      const float d = v[i] - o.m, e = fast_exp2(d * c);
      o.s += e;
      if (ENTROPY) o.u = fmaf(e, fmaxf(d, -1e30f), o.u);  // 0 where e is
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
    o = (threadIdx.x & 31) < NT / 32 ? sm[threadIdx.x & 31] : Online();
    for (int k = NT / 64; k > 0; k >>= 1) {
      const float m = __shfl_xor_sync(0xffffffffu, o.m, k), s = __shfl_xor_sync(0xffffffffu, o.s, k);
      const float u = __shfl_xor_sync(0xffffffffu, o.u, k);
      online_join(o, m, s, u, inv_tau);
    }
  }
  // The lanes joined in different orders: all take the first one's.
  o.m = __shfl_sync(0xffffffffu, o.m, 0);
  o.s = __shfl_sync(0xffffffffu, o.s, 0);
  o.u = __shfl_sync(0xffffffffu, o.u, 0);
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
      if (i < n && v[i] >= floor_value) {  // seldom
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

// 512 x 32768 bf16: 23 us, 27 on cold caches (34 MB read once from HBM, the second pass from L2): issue 73 %.
template <int NT, typename E>
__global__ void __launch_bounds__(NT) logprobs_row_kernel(const LogitsOp p) {
  const int64_t t = blockIdx.x;
  const E* x = static_cast<const E*>(p.logits) + t * p.ld;
  const int target = p.targets ? p.targets[t] : -1;
  Online o;
  int at = -1;
  row_elements<NT>(x, p.V, [&](int j, const auto& v, int n) { online_add<true, true>(o, &at, j, v, n, kLog2e, 1.0f); });
  const float best = o.m;
  o = block_join<NT>(o, 1.0f);
  if (threadIdx.x == 0) {
    const bool none = !(o.s == o.s) || o.m == -INFINITY;
    const float log_s = logf(o.s);
    if (p.entropy) p.entropy[t] = none ? NAN : log_s - o.u / o.s;
    if (p.logp) p.logp[t] = target >= 0 && target < p.V ? (none ? NAN : to_f32(x[target]) - o.m - log_s) : 0.0f;
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
  const bool any = __any_sync(0xffffffffu, v[0] != -INFINITY || v[1] != -INFINITY);  // NaN too: it has to show
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
  return any;
}

// 1021 x 32003 fp16: loss 16 us, gradient 29 (21 and 26 on cold caches: 3.1 and 5.0 TB/s). The loss is bound by its
// exponentials (special-function unit 53 %) and a row's latency, the gradient by the latter.
template <int NT, typename E>
__global__ void __launch_bounds__(NT) distill_loss_row_kernel(const LogitsOp p) {
  const int64_t t = blockIdx.x;
  const E* x = static_cast<const E*>(p.logits) + t * p.ld;
  const float inv_tau = 1.0f / p.temperature;
  int id[2] = {-1, -1};
  float pr[2], logp[2], at[2], loss = 0.0f;
  bool any = false;
  if (threadIdx.x < 32) {  // first, so that its loads' latency is not added to the row's
    any = teacher(p, t, threadIdx.x, id, pr, logp);
#pragma unroll
    for (int c = 0; c < 2; ++c) at[c] = id[c] >= 0 ? to_f32(x[id[c]]) : 0.0f;
  }
  Online o;
  row_elements<NT>(x, p.V, [&](int, const auto& v, int n) { online_add<false, false>(o, nullptr, 0, v, n, inv_tau * kLog2e, inv_tau); });
  o = block_join<NT>(o, inv_tau);
  if (threadIdx.x >= 32) return;
  const float log_s = logf(o.m == -INFINITY ? NAN : o.s);
#pragma unroll
  for (int c = 0; c < 2; ++c)
    if (!(pr[c] <= 0.0f)) loss += pr[c] * (logp[c] - ((at[c] - o.m) * inv_tau - log_s));
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
  const float c = inv_tau * kLog2e;
  float m = 0.0f, d = -lse * kLog2e;  // q = 2^((x - m) c + d)
  if (!none && !(fabsf(lse) <= kRoundedLse)) {
    Online o;
    row_elements<NT>(x, p.V, [&](int, const auto& v, int n) { online_add<false, false>(o, nullptr, 0, v, n, c, inv_tau); });
    o = block_join<NT>(o, inv_tau);
    m = o.m;
    d = -logf(o.m == -INFINITY ? NAN : o.s) * kLog2e;
  }
  // 16-byte stores where the gradient's row starts at the same place in a vector as the logits'.
  const bool together = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
  row_elements<NT>(x, p.V, [&](int j, const auto& v, int n) {
    constexpr int N = static_cast<int>(sizeof(v) / 4);
    Pack<E> out;
#pragma unroll
    for (int i = 0; i < N; ++i) out.v[i] = from_f32<E>(none ? 0.0f : g * fast_exp2(fmaf(v[i] - m, c, d)));
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
    if (first) dx[id[e]] = from_f32<E>(g * (fast_exp2(fmaf(to_f32(x[id[e]]) - m, c, d)) - sum));
  }
}

// ---- launches ------------------------------------------------------------------------------------

unsigned quads(const LogitsOp& p) { return (static_cast<unsigned>(p.T) + 31) / 32; }

// Threads of a row's block, by its length: few rows want many threads, many rows want few. Log probabilities
// without a top k / distillation loss, fp16, us:
//   1024 tokens, 16384 rows: 32 threads 16.8 / 15.2, 128 29.8 / 28.6; 400 rows: 3.9 / 4.2 and 3.3 / 3.8
//   2048 tokens, 8192 rows: 32 threads 14.4 / 12.4, 128 19.7 / 18.4; 400 rows: 5.3 / 5.7 and 3.7 / 4.5
//   6000 tokens, 2796 rows: 128 threads 13.9 / 11.9, 256 16.8 / 14.8; 400 rows: 128 5.4 / 5.3, 512 6.2 / 6.0
//   32768 tokens, 512 rows: 256 threads 12.5 / 11.2, 512 13.5 / 11.8 (gradient 11.5 and 10.9); 1021 x 32003 loss: 256
//   20 us, 512 27. 592 is how many 512-thread blocks fit the GPU at once.
// So 128 threads from 1025 tokens and 256 or 512 from 4097 are up to a third slower with many rows and about as much
// faster, or even, with few. What bounds the long rows is the latency of a row's passes: copying rows to shared
// memory in bulk, or starting from the maximum of a row's first vectors so that the running maximum seldom rises,
// was no faster.
int row_block(const LogitsOp& p) {
  if (p.V <= 1024) return 32;
  if (p.V <= 4096) return 128;
  return p.T > 592 ? 256 : 512;
}

template <typename E>
cudaError_t logprobs(const LogitsOp& p, cudaStream_t s) {
  const int nt = row_block(p);
  if (p.V <= 40) logprobs_quad_kernel<E, 10><<<quads(p), 128, 0, s>>>(p);
  else if (p.V <= kSmallV) logprobs_quad_kernel<E, 16><<<quads(p), 128, 0, s>>>(p);
  // One warp's 32 maxima bound the top 16 well: 32768 x 512 fp16, k = 5: 44 us. With more alternatives, or with 128
  // threads, rows of up to about 900 16-bit or 450 fp32 elements leave a warp without enough maxima, the bound is 0, and
  // every element is ranked against all others: 1395 us with k = 32, and 1386 with k = 5 and 128 threads.
  else if (nt == 32 && p.k <= 16) logprobs_row_kernel<32, E><<<p.T, 32, 0, s>>>(p);
  else if (nt <= 128) logprobs_row_kernel<128, E><<<p.T, 128, 0, s>>>(p);
  else if (nt == 256) logprobs_row_kernel<256, E><<<p.T, 256, 0, s>>>(p);
  else logprobs_row_kernel<512, E><<<p.T, 512, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename E, int N>
void loss_quad(const LogitsOp& p, cudaStream_t s) {
  if (p.k <= 16) distill_loss_quad_kernel<E, N, 4><<<quads(p), 128, 0, s>>>(p);
  else distill_loss_quad_kernel<E, N, kQuadAlts><<<quads(p), 128, 0, s>>>(p);
}

template <typename E>
cudaError_t loss(const LogitsOp& p, cudaStream_t s) {
  const int nt = row_block(p);
  if (p.V <= 40) loss_quad<E, 10>(p, s);
  else if (p.V <= kSmallV) loss_quad<E, 16>(p, s);
  else if (nt == 32) distill_loss_row_kernel<32, E><<<p.T, 32, 0, s>>>(p);
  else if (nt == 128) distill_loss_row_kernel<128, E><<<p.T, 128, 0, s>>>(p);
  else if (nt == 256) distill_loss_row_kernel<256, E><<<p.T, 256, 0, s>>>(p);
  else distill_loss_row_kernel<512, E><<<p.T, 512, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename E, int N>
void gradient_quad(const LogitsOp& p, cudaStream_t s) {
  if (p.k <= 16) distill_backward_quad_kernel<E, N, 4><<<quads(p), 128, 0, s>>>(p);
  else distill_backward_quad_kernel<E, N, kQuadAlts><<<quads(p), 128, 0, s>>>(p);
}

template <typename E>
cudaError_t gradient(const LogitsOp& p, cudaStream_t s) {
  const int nt = row_block(p);
  if (p.V <= 40) gradient_quad<E, 10>(p, s);
  else if (p.V <= kSmallV) gradient_quad<E, 16>(p, s);
  else if (nt == 32) distill_backward_row_kernel<32, E><<<p.T, 32, 0, s>>>(p);
  else if (nt == 128) distill_backward_row_kernel<128, E><<<p.T, 128, 0, s>>>(p);
  else if (nt == 256) distill_backward_row_kernel<256, E><<<p.T, 256, 0, s>>>(p);
  else distill_backward_row_kernel<512, E><<<p.T, 512, 0, s>>>(p);
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
