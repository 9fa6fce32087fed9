// Backward pass of attention over packed sequences, on tcgen05 (the forward operator is
// attention_tc3.cu's kernel). Per sequence and head, with S = scale Q K^T and lse from the forward:
//   P = exp(S - lse),  D_i = sum_d dO_id O_id,  dS = P (dO V^T - D)
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
//
// Two kernels. attention_delta_kernel computes D (and, for fp16, the largest |dO| and |V| of every 64
// rows). attention_backward_kernel has two kinds of blocks: query blocks own 128 query rows, stream
// the sequence's keys and values and accumulate dQ; key blocks own 128 keys, stream queries and dO and
// accumulate dK and dV. So every gradient is summed by one block in a fixed order, without atomics or
// an fp32 copy of dQ; the price is that S and dO V^T are computed twice (7 products instead of 5).
//
// Both kinds are one scheme. A block owns two 128-row operands A1, A2 and streams 64-row tiles B1, B2:
//               A1   A2   B1   B2
//   queries     Q    dO   K    V      S = A1 B1^T, dP = A2 B2^T, acc1 (dQ) += dS B1
//   keys        K    V    Q    dO     S^T = A1 B1^T, dP^T = A2 B2^T, acc1 (dK) += dS^T B1, acc2 (dV) += P^T B2
// Tensor memory (256 columns, so two blocks fit an SM and one's softmax runs under the other's MMAs):
// S in [0, 64), dP in [64, 128), acc1 in [128, 192), acc2 in [192, 256). Eight warps do the
// elementwise work, two per 32-lane quarter, each on 32 of the 64 columns; P and dS go back as 16-bit
// pairs over the first 16 columns of the same warp's 32 and are read from there as the A operand.
//   warps 0..7  elementwise: warp w has lanes 32 (w & 3).. and columns 32 (w >> 2)..
//   warp 8      TMA producer (and, for key blocks, lse and D of the streamed queries)
//   warp 9      tcgen05.mma issuer
// Heads narrower than 32 or 64 columns arrive zero-padded by the 3-D tensor maps. Rows past the
// sequence's end in the last streamed tile are cleared in shared memory (they belong to other
// sequences, and 0 x NaN is not 0); rows past the end of the owned tile stay in their own lanes and
// are not stored.
//
// fp16: P and dS are scaled by powers of two before they are rounded, P by 2^14 in key blocks and dS
// by 2^e with 2^e * 2 dh max|dO| max|V| <= 2^14, which bounds it; the outputs are scaled back in fp32.
#include "common.cuh"
#include "gemm_tc.cuh"
#include "train_common.cuh"
#include "train_ops.cuh"

#include <type_traits>

namespace esm {

namespace {

constexpr int kOwn = 128;      // rows a block owns
constexpr int kStep = 64;      // rows of a streamed tile
constexpr int kStages = 4;
constexpr int kThreads = 320;
constexpr int kDeltaRows = 64;
constexpr uint32_t kTmemCols = 256, kColS = 0, kColDp = 64, kColAcc1 = 128, kColAcc2 = 192;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kPolyEighths = 2;  // exponential pairs of every 8 on the FP32 pipe, as in the forward kernel

template <int DH>
struct Bwd {
  static constexpr int kOwnBytes = kOwn * DH * 2;
  static constexpr int kTileBytes = kStep * DH * 2;
  static constexpr int kOffStream = 2 * kOwnBytes;
  static constexpr int kOffStats = kOffStream + kStages * 2 * kTileBytes;  // per stage: 64 lse terms, 64 D terms
  static constexpr int kOffBar = kOffStats + kStages * 2 * kStep * 4;
  static constexpr int kSmem = kOffBar + 256 + 1024;
  static constexpr uint32_t kDescHi = DH == 64 ? kSw128DescHi : kSw64DescHi;
};

struct BwdParams {
  const void* out;
  const void* dout;
  const void* v;           // values: qkv + 2 H dh
  void* dqkv;
  int64_t ld_out, ld_dout, ld_qkv, ld_dqkv;
  const int32_t* cu;
  const float* lse;        // [H, T]
  float* delta;            // [H, T]
  float* peaks;            // fp16: [2][H][blocks], largest |dO| and |V| of each 64 rows
  int blocks;              // T / 64 + B
  int T, max_len, H, dh;
  float scale;
  int* err;
};

__device__ __forceinline__ bool sequence(const BwdParams& p, int b, int* start, int* len) {
  *start = p.cu[b];
  *len = p.cu[b + 1] - *start;
  if (packed_rows(*start, *len, p.T, p.max_len)) return true;
  if (threadIdx.x == 0) atomicOr(p.err, kDevBadSeqlens);
  return false;
}

// Index of the 64-row block that starts at row 64 i of sequence b, unique over the call.
__device__ __forceinline__ int row_block(int start, int b, int i) { return start / kDeltaRows + b + i; }

// Four threads per row, 16 bytes a load.
template <typename E>
__global__ void __launch_bounds__(256) attention_delta_kernel(const BwdParams p) {
  int start, len;
  if (!sequence(p, blockIdx.z, &start, &len)) return;
  const int h = blockIdx.y, part = threadIdx.x & 3, i = blockIdx.x * kDeltaRows + (threadIdx.x >> 2);
  if (static_cast<int>(blockIdx.x) * kDeltaRows >= len) return;
  constexpr bool kPeaks = std::is_same<E, __half>::value;
  float sum = 0.0f, top_g = 0.0f, top_v = 0.0f;
  if (i < len) {
    const size_t row = start + i;
    const E* o = static_cast<const E*>(p.out) + row * p.ld_out + h * p.dh;
    const E* g = static_cast<const E*>(p.dout) + row * p.ld_dout + h * p.dh;
    const E* v = static_cast<const E*>(p.v) + row * p.ld_qkv + h * p.dh;
    for (int c = 8 * part; c < p.dh; c += 32) {
      uint4 a = *reinterpret_cast<const uint4*>(o + c), b = *reinterpret_cast<const uint4*>(g + c), w{};
      if constexpr (kPeaks) w = *reinterpret_cast<const uint4*>(v + c);
      const E *ae = reinterpret_cast<const E*>(&a), *be = reinterpret_cast<const E*>(&b), *we = reinterpret_cast<const E*>(&w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float x = to_f32(be[k]);
        sum = fmaf(to_f32(ae[k]), x, sum);
        if constexpr (kPeaks) {
          top_g = fmaxf(top_g, fabsf(x));
          top_v = fmaxf(top_v, fabsf(to_f32(we[k])));
        }
      }
    }
  }
  sum += __shfl_xor_sync(0xffffffffu, sum, 1);
  sum += __shfl_xor_sync(0xffffffffu, sum, 2);
  if (part == 0 && i < len) p.delta[static_cast<size_t>(h) * p.T + start + i] = sum;
  if constexpr (kPeaks) {
    __shared__ float sm[2][8];
    top_g = warp_max(top_g);
    top_v = warp_max(top_v);
    if ((threadIdx.x & 31) == 0) {
      sm[0][threadIdx.x >> 5] = top_g;
      sm[1][threadIdx.x >> 5] = top_v;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
      float t = 0.0f;
      for (int w = 0; w < 8; ++w) t = fmaxf(t, sm[threadIdx.x][w]);
      p.peaks[(static_cast<size_t>(threadIdx.x) * p.H + h) * p.blocks + row_block(start, blockIdx.z, blockIdx.x)] = t;
    }
  }
}

// e: dS is rounded as 2^e dS. Called by a whole warp.
template <typename E>
__device__ __forceinline__ int ds_exponent(const BwdParams& p, int start, int len, int b, int h, int lane) {
  if constexpr (!std::is_same<E, __half>::value) return 0;
  const float* g = p.peaks + static_cast<size_t>(h) * p.blocks + row_block(start, b, 0);
  const float* v = g + static_cast<size_t>(p.H) * p.blocks;
  float top_g = 0.0f, top_v = 0.0f;
  for (int i = lane; i < (len + kDeltaRows - 1) / kDeltaRows; i += 32) {
    top_g = fmaxf(top_g, g[i]);
    top_v = fmaxf(top_v, v[i]);
  }
  const float bound = 2.0f * p.dh * warp_max(top_g) * warp_max(top_v);
  if (!(bound > 0.0f)) return 0;
  return min(60, max(-60, 13 - ilogbf(bound)));
}

template <int DH, typename E, bool KEYS>
__device__ __forceinline__ void backward_block(const CUtensorMap& tm_qkv, const CUtensorMap& tm_dout, const BwdParams& p,
                                               const int tile) {
  using G = Bwd<DH>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + G::kOffBar);
  uint64_t* own_full = bars;
  uint64_t* full = own_full + 1;          // [kStages]
  uint64_t* empty = full + kStages;       // [kStages]
  uint64_t* scores = empty + kStages;     // S and dP of a step written
  uint64_t* probs = scores + 1;           // P and dS of a step written
  uint64_t* done = probs + 1;             // every MMA finished
  uint64_t* tail = done + 1;              // the last tile has landed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.y, b = blockIdx.z;
  int start, len;
  if (!sequence(p, b, &start, &len)) return;
  const int r0 = tile * kOwn;
  if (r0 >= len) return;
  const int steps = (len + kStep - 1) / kStep;

  if (threadIdx.x == 0) {
    mbar_init(own_full, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], KEYS ? 2 : 1);  // the copies, and the lse and D terms
      mbar_init(&empty[s], 1);
    }
    mbar_init(scores, 1);
    mbar_init(probs, 8);
    mbar_init(done, 1);
    mbar_init(tail, 1);
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  constexpr bool kScaled = std::is_same<E, __half>::value;
  constexpr float kProbExp = kScaled && KEYS ? 14.0f : 0.0f;  // P is rounded as 2^kProbExp P
  const int ds_exp = ds_exponent<E>(p, start, len, b, h, lane);
  const float f = ldexpf(1.0f, ds_exp - static_cast<int>(kProbExp));  // dS 2^e = (P 2^kProbExp) (dP - D) f

  if (warp == 8) {
    // ---------------- producer ----------------
    const uint64_t pol = l2_policy_evict_normal();
    if (lane == 0) {
      mbar_arrive_expect_tx(own_full, 2 * G::kOwnBytes);
      for (int i = 0; i < 2; ++i) {
        const int row = start + r0 + i * kStep;
        tma_load_3d(smem + i * G::kTileBytes, &tm_qkv, own_full, 0, KEYS ? p.H + h : h, row, pol);
        if (KEYS) tma_load_3d(smem + G::kOwnBytes + i * G::kTileBytes, &tm_qkv, own_full, 0, 2 * p.H + h, row, pol);
        else tma_load_3d(smem + G::kOwnBytes + i * G::kTileBytes, &tm_dout, own_full, 0, h, row, pol);
      }
    }
    const float* lse = p.lse + static_cast<size_t>(h) * p.T + start;
    const float* delta = p.delta + static_cast<size_t>(h) * p.T + start;
    bool ok = true;
    int j = 0;
    for (; j < steps; ++j) {
      const int st = j % kStages, kept = len - j * kStep;  // rows of this tile inside the sequence
      if (!mbar_wait(&empty[st], ((j / kStages) & 1) ^ 1u, p.err, kDevTimeoutProducer)) ok = false;
      if (!__all_sync(0xffffffffu, ok)) break;
      uint8_t* dst = smem + G::kOffStream + st * 2 * G::kTileBytes;
      if (lane == 0) {
        uint64_t* bar = kept < kStep ? tail : &full[st];
        mbar_arrive_expect_tx(bar, 2 * G::kTileBytes);
        const int row = start + j * kStep;
        tma_load_3d(dst, &tm_qkv, bar, 0, KEYS ? h : p.H + h, row, pol);
        if (KEYS) tma_load_3d(dst + G::kTileBytes, &tm_dout, bar, 0, h, row, pol);
        else tma_load_3d(dst + G::kTileBytes, &tm_qkv, bar, 0, 2 * p.H + h, row, pol);
      }
      if constexpr (KEYS) {
        float* stats = reinterpret_cast<float*>(smem + G::kOffStats) + st * 2 * kStep;
#pragma unroll
        for (int c = lane; c < kStep; c += 32) {
          const int row = j * kStep + c;
          stats[c] = row < len ? fmaf(-lse[row], kLog2e, kProbExp) : -INFINITY;  // P = 0 past the end
          stats[kStep + c] = row < len ? -delta[row] * f : 0.0f;
        }
      }
      if (kept < kStep) {
        if (!mbar_wait(tail, 0, p.err, kDevTimeoutProducer)) ok = false;
        if (!__all_sync(0xffffffffu, ok)) break;
        // Rows stay whole under the swizzle.
        constexpr int kRow = DH * 2 / 16;
        for (int i = kept * kRow + lane; i < kStep * kRow; i += 32) {
          reinterpret_cast<uint4*>(dst)[i] = make_uint4(0u, 0u, 0u, 0u);
          reinterpret_cast<uint4*>(dst + G::kTileBytes)[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) {
        if (KEYS) mbar_arrive(&full[st]);
        if (kept < kStep) mbar_arrive(&full[st]);
      }
    }
    if (!ok && lane == 0) {  // let the copies in flight land before the block exits
      mbar_wait(own_full, 0, p.err, kDevTimeoutProducer);
      for (int i = (j - kStages > 0 ? j - kStages : 0); i < j; ++i)
        mbar_wait(&full[i % kStages], (i / kStages) & 1, p.err, kDevTimeoutProducer);
    }
  } else if (warp == 9) {
    // ---------------- MMA issuer ----------------
    if (elect_one_sync()) {
      constexpr uint32_t kOperands = kScaled ? 0u : kIdescBf16;
      constexpr uint32_t idesc_s = umma_idesc_f16(kOwn, kStep) | kOperands;
      constexpr uint32_t idesc_acc = umma_idesc_f16(kOwn, DH) | (1u << 16) | kOperands;  // B is MN-major
      constexpr uint32_t kTileLo = G::kTileBytes >> 4, kRowsLo = (16 * DH * 2) >> 4;
      const uint32_t a1 = umma_sw128_lo(smem_u32(smem)), a2 = a1 + (G::kOwnBytes >> 4);
      const uint32_t stream = umma_sw128_lo(smem_u32(smem + G::kOffStream));
      const uint32_t bar_scores = smem_u32(scores), bar_empty = smem_u32(empty);
      bool ok = mbar_wait_spin(own_full, 0, p.err, kDevTimeoutMma);
      for (int j = 0; j < steps && ok; ++j) {
        const int st = j % kStages;
        if (!mbar_wait_spin(&full[st], (j / kStages) & 1, p.err, kDevTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t b1 = stream + st * 2 * kTileLo, b2 = b1 + kTileLo;
#pragma unroll
        for (int k = 0; k < DH / 16; ++k) umma_f16_lo<G::kDescHi>(tmem + kColS, a1 + 2 * k, b1 + 2 * k, idesc_s, k);
#pragma unroll
        for (int k = 0; k < DH / 16; ++k) umma_f16_lo<G::kDescHi>(tmem + kColDp, a2 + 2 * k, b2 + 2 * k, idesc_s, k);
        umma_commit_addr(bar_scores);
        if (!mbar_wait_spin(probs, j & 1, p.err, kDevTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < kStep / 16; ++k) {
          const uint32_t col = (k >> 1) * 32 + (k & 1) * 8;  // 16 rows of B: 8 columns of pairs
          if constexpr (KEYS)
            umma_f16_ts_lo<G::kDescHi>(tmem + kColAcc2, tmem + kColS + col, b2 + k * kRowsLo, idesc_acc, j > 0 || k > 0);
          umma_f16_ts_lo<G::kDescHi>(tmem + kColAcc1, tmem + kColDp + col, b1 + k * kRowsLo, idesc_acc, j > 0 || k > 0);
        }
        umma_commit_addr(bar_empty + 8 * st);
      }
      umma_commit(done);
      if (!ok) mbar_wait_spin(done, 0, p.err, kDevTimeoutMma);
    }
  } else {
    // ---------------- elementwise: one owned row per thread, 32 of the 64 columns ----------------
    const int quarter = warp & 3, half = warp >> 2;
    const int row = r0 + quarter * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t t_s = lanes + kColS + 32 * half, t_dp = lanes + kColDp + 32 * half;
    const float c = p.scale * kLog2e;
    const uint64_t c2 = f2_pack(c, c), f2 = f2_pack(f, f);
    uint64_t lse2 = 0, delta2 = 0;
    if constexpr (!KEYS) {
      const size_t at = static_cast<size_t>(h) * p.T + start + row;
      const float l = row < len ? -p.lse[at] * kLog2e : 0.0f, d = row < len ? -p.delta[at] * f : 0.0f;
      lse2 = f2_pack(l, l);
      delta2 = f2_pack(d, d);
    }
    bool ok = true;
    for (int j = 0; j < steps; ++j) {
      if (!mbar_wait_spin(scores, j & 1, p.err, kDevTimeoutEpilogue)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int kept = len - j * kStep - 32 * half;  // of this warp's columns
      const float* stats = reinterpret_cast<const float*>(smem + G::kOffStats) + (j % kStages) * 2 * kStep + 32 * half;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t s[16], dp[16], pr[8], ds[8];
        tmem_ld16(t_s + 16 * q, s);
        tmem_ld16(t_dp + 16 * q, dp);
        tmem_ld_wait();
        if (!KEYS && kept < 32) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (16 * q + i >= kept) s[i] = __float_as_uint(-INFINITY);
        }
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          uint64_t l2[2] = {lse2, lse2}, d2[2] = {delta2, delta2};
          if constexpr (KEYS) {
            const ulonglong2 l4 = *reinterpret_cast<const ulonglong2*>(stats + 16 * q + 2 * i);
            const ulonglong2 d4 = *reinterpret_cast<const ulonglong2*>(stats + kStep + 16 * q + 2 * i);
            l2[0] = l4.x, l2[1] = l4.y, d2[0] = d4.x, d2[1] = d4.y;
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int k = i + u;
            float a0, a1, x0, x1;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])), c2, l2[u]), a0, a1);
            const uint64_t e2 = k < kPolyEighths ? poly_exp2_x2(fminf(a0, 126.0f), fminf(a1, 126.0f))
                                                 : f2_pack(fast_exp2(a0), fast_exp2(a1));
            const uint64_t t2 = f2_fma(f2_pack(__uint_as_float(dp[2 * k]), __uint_as_float(dp[2 * k + 1])), f2, d2[u]);
            f2_unpack(f2_mul(e2, t2), x0, x1);
            ds[k] = pack2<E>(x0, x1);
            if constexpr (KEYS) {
              f2_unpack(e2, x0, x1);
              pr[k] = pack2<E>(x0, x1);
            }
          }
        }
        tmem_st8(t_dp + 8 * q, ds);
        if constexpr (KEYS) tmem_st8(t_s + 8 * q, pr);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(probs);
    }
    if (ok && mbar_wait_spin(done, 0, p.err, kDevTimeoutEpilogue)) {
      tc_fence_after();
      // Key blocks: half 0 stores dK, half 1 dV. Query blocks: each half stores half of dQ's columns.
      const float back = KEYS && half == 1 ? ldexpf(1.0f, -static_cast<int>(kProbExp)) : p.scale * ldexpf(1.0f, -ds_exp);
      const int part = KEYS ? 1 + half : 0;
      E* dst = static_cast<E*>(p.dqkv) + static_cast<size_t>(start + row) * p.ld_dqkv + (part * p.H + h) * p.dh;
      constexpr int kCols = KEYS ? DH : DH / 2;
      const int col0 = KEYS ? 0 : half * kCols;
      const uint32_t t_acc = lanes + (KEYS && half == 1 ? kColAcc2 : kColAcc1) + col0;
#pragma unroll
      for (int cc = 0; cc < kCols; cc += 16) {
        uint32_t o[16];
        tmem_ld16(t_acc + cc, o);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int col = col0 + cc + 8 * k;
          if (row < len && col < p.dh) {
            uint32_t v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
              v[u] = pack2<E>(__uint_as_float(o[8 * k + 2 * u]) * back, __uint_as_float(o[8 * k + 2 * u + 1]) * back);
            *reinterpret_cast<uint4*>(dst + col) = *reinterpret_cast<const uint4*>(v);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Even blocks of x own keys, odd ones queries.
template <int DH, typename E>
__global__ void __launch_bounds__(kThreads, 2)
    attention_backward_kernel(const __grid_constant__ CUtensorMap tm_qkv, const __grid_constant__ CUtensorMap tm_dout,
                              const BwdParams p) {
  if (blockIdx.x & 1) backward_block<DH, E, false>(tm_qkv, tm_dout, p, blockIdx.x >> 1);
  else backward_block<DH, E, true>(tm_qkv, tm_dout, p, blockIdx.x >> 1);
}

template <int DH, typename E>
cudaError_t backward(const AttnOp& a, const BwdParams& p, cudaStream_t s) {
  constexpr bool kBf16 = std::is_same<E, __nv_bfloat16>::value;
  CUtensorMap tm_qkv, tm_dout;
  if (!make_tmap_op_heads(&tm_qkv, a.qkv, kBf16, a.T, 3 * a.H, a.dh, a.ld_qkv, kStep) ||
      !make_tmap_op_heads(&tm_dout, a.dout, kBf16, a.T, a.H, a.dh, a.ld_dout, kStep))
    return cudaErrorInvalidValue;
  static std::atomic<unsigned long long> configured{0};
  cudaError_t e = allow_smem(attention_backward_kernel<DH, E>, Bwd<DH>::kSmem, configured);
  if (e != cudaSuccess) return e;
  attention_delta_kernel<E><<<dim3((a.max_len + kDeltaRows - 1) / kDeltaRows, a.H, a.B), 256, 0, s>>>(p);
  attention_backward_kernel<DH, E>
      <<<dim3(2 * ((a.max_len + kOwn - 1) / kOwn), a.H, a.B), kThreads, Bwd<DH>::kSmem, s>>>(tm_qkv, tm_dout, p);
  return cudaGetLastError();
}

}  // namespace

size_t attention_backward_bytes(int B, int T, int H) {
  return static_cast<size_t>(H) * T * 4 + static_cast<size_t>(H) * (T / kDeltaRows + B) * 8;
}

cudaError_t launch_attention_backward(const AttnOp& a, cudaStream_t s) {
  BwdParams p{};
  p.out = a.out;
  p.dout = a.dout;
  p.v = static_cast<const char*>(a.qkv) + static_cast<size_t>(2) * a.H * a.dh * 2;
  p.dqkv = a.dqkv;
  p.ld_out = a.ld_out;
  p.ld_dout = a.ld_dout;
  p.ld_qkv = a.ld_qkv;
  p.ld_dqkv = a.ld_dqkv;
  p.cu = a.cu;
  p.lse = a.lse;
  p.delta = a.workspace;
  p.peaks = a.workspace + static_cast<size_t>(a.H) * a.T;
  p.blocks = a.T / kDeltaRows + a.B;
  p.T = a.T;
  p.max_len = a.max_len;
  p.H = a.H;
  p.dh = a.dh;
  p.scale = a.scale;
  p.err = a.err;
  if (a.dh <= 32) return a.dtype == ESM_F16 ? backward<32, __half>(a, p, s) : backward<32, __nv_bfloat16>(a, p, s);
  return a.dtype == ESM_F16 ? backward<64, __half>(a, p, s) : backward<64, __nv_bfloat16>(a, p, s);
}

}  // namespace esm
