// Backward pass of attention over packed sequences, on tcgen05 (the forward operator is
// attention_tc3.cu's kernel). Per sequence and head, with S = scale Q K^T and lse from the forward:
//   P = exp(S - lse),  D_i = sum_d dO_id O_id,  dS = P (dO V^T - D)
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
//
// Two kernels. attention_delta_kernel computes D (and, for fp16, the largest |dO| and |V| of every 64
// rows). attention_backward_kernel works on items of two kinds: a query item owns 128 query rows,
// streams the sequence's keys and values and accumulates dQ; a key item owns 128 keys, streams queries
// and dO and accumulates dK and dV. So every gradient is summed by one block in a fixed order, without
// atomics or an fp32 copy of dQ; the price is that S and dO V^T are computed twice (7 products, not 5).
//
// Both kinds are one scheme. An item owns two 128-row operands A1, A2 and streams 64-row tiles B1, B2:
//               A1   A2   B1   B2
//   queries     Q    dO   K    V      S = A1 B1^T, dP = A2 B2^T, acc1 (dQ) += dS B1
//   keys        K    V    Q    dO     S^T = A1 B1^T, dP^T = A2 B2^T, acc1 (dK) += dS^T B1, acc2 (dV) += P^T B2
//
// One persistent block per SM takes items from a list (see the producer). Tensor memory (512 columns): three score
// buffers of 128 columns (S in the first 64, dP in the other 64), acc1 and acc2. Step n uses buffer n % 3, so
// the tensor cores compute the next steps' scores and the last one's products while the elementwise warps
// work on a step. P and dS go back over S and dP as 16-bit pairs (each warp over the first half of the 32
// columns it read) and are read from there as the A operand.
//   warps 0..15  elementwise, in two teams of eight that take every other step: a warp has 32 owned rows and 32 of
//                the step's 64 columns
//   warps 16..19 store an item's gradients while the others go on with the next item
//   warp 20      producer: finds items, loads their operands (two slots) and the stream (TMA ring)
//   warp 23      splits lse and D of the streamed queries of key items (below), and clears the rows behind a
//                sequence's end in its last tile
//   warp 21      issues the scores' MMAs: those of step n + 3 once the products of step n have freed its buffer
//   warp 22      issues the products' MMAs
// Steps, buffers and stages are numbered through all items, so an item's first scores are computed while the
// one before it is still finishing.
//
// In key items lse and D belong to the columns of a thread's row. Reading them for every row costs more
// shared-memory bandwidth than all operand reads of the tensor cores (a 16-byte broadcast read is four
// wavefronts), so they are subtracted by the tensor cores: one more K step of 16 with constants in every row of
// A, (2^15, 2^3, 2^-9) for fp16 and ones for bf16, and -lse / scale, or -D, split into three parts of the
// operand type in B. For fp16 that covers magnitudes up to 2^30, to 2^-22 relative or better, or 2^-34.
//
// Heads narrower than 32 or 64 columns arrive zero-padded by the 3-D tensor maps. Rows past the
// sequence's end in the last streamed tile are cleared in shared memory (they belong to other
// sequences, and 0 x NaN is not 0); rows past the end of the owned tile stay in their own lanes and
// are not stored.
//
// fp16: P and dS are scaled by powers of two before they are rounded, P by 2^14 in key items and dS
// by 2^e with 2^e * 2 dh max|dO| max|V| <= 2^14, which bounds it; the outputs are scaled back in fp32.
//
// Measured, in bursts at 1965 MHz: 16 x 1024 tokens of 20 x 64 heads, fp16, 358 us in all, 25 of them
// attention_delta_kernel (126 MB); 2 x 4096 of 40 x 64, bf16, 1.21 ms. Call after call the power cap sets the clock:
// 418 us at 1560 MHz and 1.39 ms at 1665. What bounds it: a step of 64 x 128 takes 1180 cycles. With the elementwise
// arithmetic left out the 358 us become 315, with the MMAs left out 295, with both 259, with the split of lse and D
// left out 355, and with all three 211: the stages are about as long as one another, and none alone is the
// bound. The kernel is at its limit of 80 registers; DH 64 spills 44 (bf16) and 64 bytes (fp16), DH 32 none. Tried
// and slower or no faster: two blocks per SM that are not persistent (518), one issuer for all MMAs (447), 128-row
// streamed tiles (357, but 8 to 16 % more on short sequences), 8 elementwise warps (392), barriers of their own for
// S and dP (375), a second pair of accumulators, exponentials partly on the FP32 pipe, lse and D loaded four steps
// ahead, and for DH 32 16-byte copies by the producer warp instead of TMA (140 -> 167 at 32 x 64..512).
#include "common.cuh"
#include "gemm_tc.cuh"
#include "train_common.cuh"
#include "train_ops.cuh"

#include <algorithm>
#include <type_traits>

namespace esm {

namespace {

constexpr int kOwn = 128;      // rows an item owns
constexpr int kStep = 64;      // rows of a streamed tile
constexpr int kBufs = 3;       // score buffers
constexpr int kElemWarps = 16, kTeams = 2, kTeamWarps = kElemWarps / kTeams;
constexpr int kWarpCols = 4 * kStep / kTeamWarps;  // columns of an elementwise warp
constexpr int kStoreWarp = kElemWarps, kLoadWarp = kStoreWarp + 4;
constexpr int kScoreWarp = kLoadWarp + 1, kProductWarp = kScoreWarp + 1, kSplitWarp = kProductWarp + 1;
constexpr int kThreads = 32 * (kSplitWarp + 1);
constexpr int kInfos = 8;      // item records: the producer writes at most the fifth one after the slowest reader's
constexpr int kDeltaRows = 64;
constexpr uint32_t kTmemCols = 512, kColBuf = 128, kColDp = 64, kColAcc1 = 384, kColAcc2 = 448;
constexpr float kLog2e = 1.4426950408889634f;

struct Item {
  int start, len, r0, h, keys, ds_exp;  // len 0: no more items
};

template <int DH>
struct Bwd {
  static constexpr int kStages = DH == 64 ? 5 : 8;
  static constexpr int kOwnBytes = kOwn * DH * 2;
  static constexpr int kTileBytes = kStep * DH * 2;
  static constexpr int kOffConst = 4 * kOwnBytes;                      // two slots of A1, A2
  static constexpr int kOffStream = kOffConst + kOwnBytes;             // the constants' rows
  static constexpr int kStageBytes = 3 * kTileBytes;                   // B1, B2, and lse and D in parts
  static constexpr int kOffOut = kOffStream + kStages * kStageBytes;   // 32 gradient rows of each storing warp
  static constexpr int kOffInfo = kOffOut + kOwnBytes;
  static constexpr int kOffBar = kOffInfo + kInfos * 32;
  static constexpr int kSmem = kOffBar + 512 + 1024;
  static constexpr uint32_t kDescHi = DH == 64 ? kSw128DescHi : kSw64DescHi;
  static_assert(kSmem <= 232448 && sizeof(Item) <= 32, "shared memory of one block");
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
  unsigned long long* claimed;  // candidates given to blocks; attention_delta_kernel sets it to 0
  int blocks;              // T / 64 + B
  int B, T, max_len, H, dh;
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
  if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) *p.claimed = 0;
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

// e: dS is rounded as 2^e dS.
template <typename E>
__device__ __forceinline__ int ds_exponent(const BwdParams& p, int start, int len, int b, int h) {
  if constexpr (!std::is_same<E, __half>::value) return 0;
  const float* g = p.peaks + static_cast<size_t>(h) * p.blocks + row_block(start, b, 0);
  const float* v = g + static_cast<size_t>(p.H) * p.blocks;
  float top_g = 0.0f, top_v = 0.0f;
#pragma unroll 8
  for (int i = 0; i < (len + kDeltaRows - 1) / kDeltaRows; ++i) {
    top_g = fmaxf(top_g, g[i]);
    top_v = fmaxf(top_v, v[i]);
  }
  const float bound = 2.0f * p.dh * top_g * top_v;
  if (!(bound > 0.0f)) return 0;
  return min(60, max(-60, 13 - ilogbf(bound)));
}

// x as three values of E, times 2^15, 2^3 and 2^-9 for fp16 (whose range the factors extend) and 1
// for bf16, packed into the first 16 bytes of a K step (the other elements are zero). fp16: for |x| <= 2^30 the
// first part is at most 2^15 and leaves at most 2^18, the second is at most 2^15 and leaves at most 2^6, the
// third is at most 2^15; what it leaves is half of its last bit, 2^-34 where that is subnormal. Below 2 the first part
// is subnormal, and the tensor core aligns a sum to the products' exponents before it adds, a subnormal's counted as
// 2^-14: with 2^15 that costs the bits below 2^-24 (42 x 2^-24 of D at 0.01). Below 1/4 it is left out; the
// other two hold x to 2^-22 relative, or 2^-34.
template <typename E>
__device__ __forceinline__ uint4 split_parts(float x) {
  if constexpr (std::is_same<E, __half>::value) {
    const __half h0 = __float2half_rn(fabsf(x) < 0.25f ? 0.0f : x * (1.0f / 32768.0f));
    float r = fmaf(-32768.0f, __half2float(h0), x);
    const __half h1 = __float2half_rn(r * 0.125f);
    r = fmaf(-8.0f, __half2float(h1), r) * 512.0f;
    const __half2 h01 = __halves2half2(h0, h1);
    return make_uint4(*reinterpret_cast<const uint32_t*>(&h01), pack2<E>(r, 0.0f), 0u, 0u);
  } else {  // by truncation: each part is the upper half of what is left
    const uint32_t u0 = __float_as_uint(x);
    float r = x - __uint_as_float(u0 & 0xffff0000u);
    const uint32_t u1 = __float_as_uint(r);
    r -= __uint_as_float(u1 & 0xffff0000u);
    return make_uint4(__byte_perm(u0, u1, 0x7632), __float_as_uint(r) >> 16, 0u, 0u);
  }
}
template <typename E>
__device__ __forceinline__ uint4 split_factors() {
  if constexpr (std::is_same<E, __half>::value) return make_uint4(pack2<E>(32768.0f, 8.0f), pack2<E>(1.0f / 512.0f, 0.0f), 0u, 0u);
  else return make_uint4(pack2<E>(1.0f, 1.0f), pack2<E>(1.0f, 0.0f), 0u, 0u);
}

// Column of the pair of values i, i + 1 of a row of P or dS: every warp packs its columns into the first
// half of their place.
__host__ __device__ constexpr int pair_col(int i) { return i / kWarpCols * kWarpCols + i % kWarpCols / 2; }

// Byte offset of 16-byte chunk `chunk` of row `row` in a tile with rows of DH elements under the
// tensor maps' swizzle (128 bytes for DH 64, 64 bytes for DH 32).
template <int DH>
__device__ __forceinline__ int swizzled(int row, int chunk) {
  if constexpr (DH == 64) return row * 128 + ((chunk ^ (row & 7)) << 4);
  else return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
}

template <int DH, typename E>
__global__ void __launch_bounds__(kThreads, 1)
    attention_backward_kernel(const __grid_constant__ CUtensorMap tm_qkv, const __grid_constant__ CUtensorMap tm_dout,
                              const __grid_constant__ CUtensorMap tm_qkv_own,
                              const __grid_constant__ CUtensorMap tm_dout_own, const BwdParams p) {
  using G = Bwd<DH>;
  constexpr int kStages = G::kStages;
  constexpr bool kScaled = std::is_same<E, __half>::value;
  constexpr int kProbExp = kScaled ? 14 : 0;  // key items round 2^kProbExp P
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  auto info_at = [&](int i) -> Item* { return reinterpret_cast<Item*>(smem + G::kOffInfo + (i % kInfos) * 32); };
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + G::kOffBar);
  uint64_t* info_full = bars;                // [kInfos] an item's record
  uint64_t* own_full = info_full + kInfos;   // [2]
  uint64_t* own_empty = own_full + 2;        // [2]
  uint64_t* full = own_empty + 2;            // [kStages]
  uint64_t* empty = full + kStages;          // [kStages]
  uint64_t* scores = empty + kStages;        // [kBufs] S and dP written
  uint64_t* probs = scores + kBufs;          // [kBufs] P and dS written
  uint64_t* done = probs + kBufs;            // an item's products finished
  uint64_t* acc_free = done + 1;             // its accumulators read
  uint64_t* tail = acc_free + 1;             // [kStages] a sequence's last, partial tile has landed
  uint64_t* drain = tail + kStages;                // [2] everything an issuer issued
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kInfos; ++i) mbar_init(&info_full[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&own_full[i], 1);
      mbar_init(&own_empty[i], 2);  // the item's scores; its record read by the splitting warp
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 2);  // the copies; the parts of lse and D, or for query items the producer again
      mbar_init(&empty[i], 1);
      mbar_init(&tail[i], 1);
    }
    for (int i = 0; i < kBufs; ++i) {
      mbar_init(&scores[i], 1);
      mbar_init(&probs[i], kTeamWarps);
    }
    mbar_init(done, 1);
    mbar_init(acc_free, 4);
    for (int i = 0; i < 2; ++i) mbar_init(&drain[i], 1);
    fence_mbar_init();
  }
  // The constants' rows (K steps 0 and 1), and zeros behind the parts of lse and D.
  for (int i = threadIdx.x; i < kOwn * 4; i += kThreads)
    *reinterpret_cast<uint4*>(smem + G::kOffConst + swizzled<DH>(i >> 2, i & 3)) = (i & 1) ? make_uint4(0u, 0u, 0u, 0u) : split_factors<E>();
  for (int i = threadIdx.x; i < kStages * kStep * 4; i += kThreads) {
    const int st = i / (kStep * 4), c = i % (kStep * 4);
    *reinterpret_cast<uint4*>(smem + G::kOffStream + st * G::kStageBytes + 2 * G::kTileBytes + swizzled<DH>(c >> 2, c & 3)) =
        make_uint4(0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();
  if (warp == kScoreWarp) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == kLoadWarp) {
    // ---------------- producer ----------------
    const uint64_t pol = l2_policy_evict_normal();
    // Candidates are the 128-row blocks of all sequences, for every head (the fastest index: blocks then work on
    // neighbouring memory; with the heads outermost 16 x 1024 took 4 % longer) and kind (key items, which take
    // longer, first). A block takes them in batches, one per lane. Where the sequences are about as long as
    // max_len, each has `tiles` of them and a block takes every gridDim.x-th. Otherwise they are numbered like
    // row_block's (some numbers have no rows), and with every gridDim.x-th the sum of one block's steps was up to
    // a third above the mean: only the first batch, 7/8 of an even share, is given like that, and the rest is
    // claimed from a counter in smaller and smaller batches. 32 x 64..512 tokens, 20 x 24 heads: 117 -> 102 us; 24 x
    // 30..1022 tokens, 20 x 64: 282 -> 249; 64 x 100 tokens by claims 55 -> 72, hence the rule. A claim takes
    // about as long as one or two steps of a short sequence, hence `least`.
    const int tiles = (p.max_len + kOwn - 1) / kOwn;
    const bool even = static_cast<int64_t>(tiles) * p.B <= p.T / kOwn + p.B;
    const int64_t slots = even ? static_cast<int64_t>(tiles) * p.B : p.T / kOwn + p.B, half = slots * p.H, total = 2 * half;
    const int64_t least = 1 + static_cast<int64_t>(512) * p.B / p.T;
    auto share = [&](int64_t left) { return static_cast<int>(min(int64_t(32), max(least, left / gridDim.x))); };
    int batch = even ? 32 : share(total * 7 / 8);
    const int64_t handed = static_cast<int64_t>(batch) * gridDim.x;
    int64_t base = blockIdx.x, stride = gridDim.x;
    bool ok = true;
    int item = 0, n = 0;
    // Loads in flight when a wait gives up must land before the block exits.
    int own_loaded = 0;
    while (base < total && ok) {
      // The next batch is claimed now, so that the counter's latency passes behind this one's items.
      const int next_batch = share((total - max(base, handed)) / 4);
      unsigned long long next = 0;
      if (lane == 0 && !even && handed < total) next = atomicAdd(p.claimed, static_cast<unsigned long long>(next_batch));
      const int64_t at = base + lane * stride;
      Item it{};
      if (lane < batch && at < total) {
        const int64_t r = at < half ? at : at - half;
        const int slot = static_cast<int>(r / p.H);
        it.keys = at < half;
        it.h = static_cast<int>(r % p.H);
        int b = even ? slot / tiles : 0;
        for (int left = even ? 1 : p.B; left > 1;) {  // the last sequence whose first block is not behind the slot
          const int upper = left / 2;
          if (p.cu[b + upper] / kOwn + b + upper <= slot) {
            b += upper;
            left -= upper;
          } else {
            left = upper;
          }
        }
        it.start = p.cu[b];
        it.len = p.cu[b + 1] - it.start;
        const int i = even ? slot % tiles : slot - (it.start / kOwn + b);
        it.r0 = i * kOwn;
        if (!packed_rows(it.start, it.len, p.T, p.max_len) || i < 0 || i >= (it.len + kOwn - 1) / kOwn) it.len = 0;
        if (it.len > 0) it.ds_exp = ds_exponent<E>(p, it.start, it.len, b, it.h);
      }
      for (uint32_t found = __ballot_sync(0xffffffffu, it.len > 0); found != 0 && ok; found &= found - 1) {
        const int src = __ffs(found) - 1;
        Item cur;
        cur.start = __shfl_sync(0xffffffffu, it.start, src);
        cur.len = __shfl_sync(0xffffffffu, it.len, src);
        cur.r0 = __shfl_sync(0xffffffffu, it.r0, src);
        cur.h = __shfl_sync(0xffffffffu, it.h, src);
        cur.keys = __shfl_sync(0xffffffffu, it.keys, src);
        cur.ds_exp = __shfl_sync(0xffffffffu, it.ds_exp, src);
        const int slot = item & 1, h = cur.h, len = cur.len, start = cur.start;
        const bool keys = cur.keys;
        ok = mbar_wait_spin(&own_empty[slot], ((item >> 1) & 1) ^ 1u, p.err, kDevTimeoutProducer);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        // Owned and streamed operands: head h1 of qkv, and head h2 of qkv or dO.
        if (lane == 0) {
          *info_at(item) = cur;
          mbar_arrive(&info_full[item % kInfos]);
          mbar_arrive_expect_tx(&own_full[slot], 2 * G::kOwnBytes);
          uint8_t* dst = smem + slot * 2 * G::kOwnBytes;
          tma_load_3d(dst, &tm_qkv_own, &own_full[slot], 0, keys ? p.H + h : h, start + cur.r0, pol);
          tma_load_3d(dst + G::kOwnBytes, keys ? &tm_qkv_own : &tm_dout_own, &own_full[slot], 0, keys ? 2 * p.H + h : h,
                      start + cur.r0, pol);
          own_loaded = item + 1;
          const int h1 = keys ? h : p.H + h, h2 = keys ? h : 2 * p.H + h;
          const CUtensorMap* map2 = keys ? &tm_dout : &tm_qkv;
          for (int row = 0; row < len; row += kStep) {
            const int st = n % kStages;
            if (!(ok = mbar_wait_spin(&empty[st], ((n / kStages) & 1) ^ 1u, p.err, kDevTimeoutProducer))) break;
            uint8_t* to = smem + G::kOffStream + st * G::kStageBytes;
            uint64_t* bar = len - row < kStep ? &tail[st] : &full[st];
            mbar_arrive_expect_tx(bar, 2 * G::kTileBytes);
            tma_load_3d(to, &tm_qkv, bar, 0, h1, start + row, pol);
            tma_load_3d(to + G::kTileBytes, map2, bar, 0, h2, start + row, pol);
            if (!keys) mbar_arrive(&full[st]);
            ++n;
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        ++item;
      }
      if (even) {
        base += 32 * stride;
        continue;
      }
      if (handed >= total) break;
      base = handed + static_cast<int64_t>(__shfl_sync(0xffffffffu, next, 0));
      batch = next_batch;
      stride = 1;
    }
    if (ok) {
      ok = mbar_wait(&own_empty[item & 1], ((item >> 1) & 1) ^ 1u, p.err, kDevTimeoutProducer);  // the record is free
      if (lane == 0 && ok) {
        info_at(item)->len = 0;
        mbar_arrive(&info_full[item % kInfos]);
      }
    } else if (lane == 0) {
      for (int i = own_loaded > 2 ? own_loaded - 2 : 0; i < own_loaded; ++i)
        mbar_wait(&own_full[i & 1], (i >> 1) & 1, p.err, kDevTimeoutProducer);
      for (int i = n > kStages ? n - kStages : 0; i < n; ++i)  // a partial tile's through the clearing warp
        mbar_wait(&full[i % kStages], (i / kStages) & 1, p.err, kDevTimeoutProducer);
    }
  } else if (warp == kScoreWarp) {
    // ---------------- scores: one thread issues ----------------
    // The two issuers are separate warps because an MMA's operands stay in the issuing warp's registers until
    // the tensor core takes it: a warp stalls there, and what it does next (a commit, a wait, the next
    // addresses) is not hidden. With one issuer for both that cost 490 of 1265 cycles a step.
    if (elect_one_sync()) {
      constexpr uint32_t idesc = umma_idesc_f16(kOwn, kStep) | (kScaled ? 0u : kIdescBf16);
      constexpr uint32_t kTileLo = G::kTileBytes >> 4, kOwnLo = G::kOwnBytes >> 4;
      const uint32_t consts = umma_sw128_lo(smem_u32(smem + G::kOffConst));
      const uint32_t stream = umma_sw128_lo(smem_u32(smem + G::kOffStream));
      bool ok = true;
      int st = 0, phase = 0, buf = 0, n = 0;       // of the step
      int freed_st = 0, freed_phase = 0;           // of step n - kBufs
      uint32_t a = umma_sw128_lo(smem_u32(smem)), b = stream, d = tmem;
      for (int item = 0; ok; ++item) {
        if (!(ok = mbar_wait_spin(&info_full[item % kInfos], (item / kInfos) & 1, p.err, kDevTimeoutMma))) break;
        const int len = info_at(item)->len, keys = info_at(item)->keys;
        if (len == 0) break;
        if (!(ok = mbar_wait_spin(&own_full[item & 1], (item >> 1) & 1, p.err, kDevTimeoutMma))) break;
        for (int left = (len + kStep - 1) / kStep; left > 0; --left, ++n) {
          if (!(ok = mbar_wait_spin(&full[st], phase, p.err, kDevTimeoutMma))) break;
          if (n >= kBufs) {  // the products of step n - kBufs have read the buffer
            if (!(ok = mbar_wait_spin(&empty[freed_st], freed_phase, p.err, kDevTimeoutMma))) break;
            if (++freed_st == kStages) {
              freed_st = 0;
              freed_phase ^= 1;
            }
          }
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < DH / 16; ++k) umma_f16_lo<G::kDescHi>(d, a + 2 * k, b + 2 * k, idesc, k);
          if (keys) umma_f16_lo<G::kDescHi>(d, consts, b + 2 * kTileLo, idesc, 1u);
#pragma unroll
          for (int k = 0; k < DH / 16; ++k) umma_f16_lo<G::kDescHi>(d + kColDp, a + kOwnLo + 2 * k, b + kTileLo + 2 * k, idesc, k);
          if (keys) umma_f16_lo<G::kDescHi>(d + kColDp, consts + 2, b + 2 * kTileLo + 2, idesc, 1u);
          umma_commit(&scores[buf]);
          b += 3 * kTileLo;
          if (++st == kStages) {
            st = 0;
            phase ^= 1;
            b = stream;
          }
          d += kColBuf;
          if (++buf == kBufs) {
            buf = 0;
            d = tmem;
          }
        }
        umma_commit(&own_empty[item & 1]);
        a = (item & 1) ? a - 2 * kOwnLo : a + 2 * kOwnLo;
      }
      umma_commit(&drain[0]);
      mbar_wait_spin(&drain[0], 0, p.err, kDevTimeoutMma);
    }
  } else if (warp == kProductWarp) {
    // ---------------- products: one thread issues ----------------
    if (elect_one_sync()) {
      constexpr uint32_t idesc = umma_idesc_f16(kOwn, DH) | (1u << 16) | (kScaled ? 0u : kIdescBf16);  // B is MN-major
      constexpr uint32_t kTileLo = G::kTileBytes >> 4, kRowsLo = (16 * DH * 2) >> 4;
      const uint32_t stream = umma_sw128_lo(smem_u32(smem + G::kOffStream));
      const uint32_t acc1 = tmem + kColAcc1, acc2 = tmem + kColAcc2;
      bool ok = true;
      int st = 0, buf = 0, phase = 0;
      uint32_t b = stream, d = tmem;
      for (int item = 0; ok; ++item) {
        if (!(ok = mbar_wait_spin(&info_full[item % kInfos], (item / kInfos) & 1, p.err, kDevTimeoutMma))) break;
        const int len = info_at(item)->len, keys = info_at(item)->keys;
        if (len == 0) break;
        if (item > 0 && !(ok = mbar_wait_spin(acc_free, (item - 1) & 1, p.err, kDevTimeoutMma))) break;
        uint32_t add = 0;
        for (int left = (len + kStep - 1) / kStep; left > 0; --left) {
          if (!(ok = mbar_wait_spin(&probs[buf], phase, p.err, kDevTimeoutMma))) break;
          tc_fence_after();
          if (keys) {
#pragma unroll
            for (int k = 0; k < kStep / 16; ++k)  // 16 rows of B: the 8 columns of one warp's pairs
              umma_f16_ts_lo<G::kDescHi>(acc2, d + pair_col(16 * k), b + kTileLo + k * kRowsLo, idesc, k > 0 ? 1u : add);
          }
#pragma unroll
          for (int k = 0; k < kStep / 16; ++k)
            umma_f16_ts_lo<G::kDescHi>(acc1, d + kColDp + pair_col(16 * k), b + k * kRowsLo, idesc, k > 0 ? 1u : add);
          add = 1;
          umma_commit(&empty[st]);
          b += 3 * kTileLo;
          if (++st == kStages) {
            st = 0;
            b = stream;
          }
          d += kColBuf;
          if (++buf == kBufs) {
            buf = 0;
            phase ^= 1;
            d = tmem;
          }
        }
        umma_commit(done);
      }
      umma_commit(&drain[1]);
      mbar_wait_spin(&drain[1], 0, p.err, kDevTimeoutMma);
    }
  } else if (warp == kSplitWarp) {
    // ---------------- parts of lse and D of the streamed queries (key items) ----------------
    const float inv_scale = 1.0f / p.scale;
    bool ok = true;
    int st = 0, phase = 1;      // the stage's turn, and the parity of its release before that
    uint32_t tail_phases = 0;   // bit per stage
    for (int item = 0; ok; ++item) {
      if (!mbar_wait_spin(&info_full[item % kInfos], (item / kInfos) & 1, p.err, kDevTimeoutProducer)) break;
      const Item it = *info_at(item);
      if (it.len == 0) break;
      // Nothing else waits for this warp in query items of whole tiles: the records' ring has to.
      __syncwarp();
      if (lane == 0) mbar_arrive(&own_empty[item & 1]);
      const float* lse = p.lse + static_cast<size_t>(it.h) * p.T + it.start;
      const float* delta = p.delta + static_cast<size_t>(it.h) * p.T + it.start;
      float next_l[2], next_d[2];  // of this lane's two rows of the next tile
      auto stats = [&](int j) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int row = j * kStep + lane + 32 * u;
          next_l[u] = row < it.len ? lse[row] : 0.0f;
          next_d[u] = row < it.len ? delta[row] : 0.0f;
        }
      };
      if (it.keys) stats(0);
      for (int j = 0; j * kStep < it.len; ++j) {
        const int kept = it.len - j * kStep;  // rows of this tile inside the sequence
        uint8_t* tile = smem + G::kOffStream + st * G::kStageBytes;
        if (it.keys) {
          uint4 part_l[2], part_d[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            // P = exp2(c (S - lse / scale)), times 2^kProbExp; 0 past the end, where S is 0 and the first part
            // alone is the constant.
            const float x = lane + 32 * u < kept ? -(next_l[u] - kProbExp * 0.69314718f) * inv_scale : (kScaled ? -57344.0f * 32768.0f : -1e30f);
            part_l[u] = split_parts<E>(x);
            part_d[u] = split_parts<E>(-next_d[u]);
          }
          stats(j + 1);
          ok = __all_sync(0xffffffffu, mbar_wait_spin(&empty[st], phase, p.err, kDevTimeoutProducer));
          if (!ok) break;
          uint8_t* parts = tile + 2 * G::kTileBytes;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            *reinterpret_cast<uint4*>(parts + swizzled<DH>(lane + 32 * u, 0)) = part_l[u];
            *reinterpret_cast<uint4*>(parts + swizzled<DH>(lane + 32 * u, 2)) = part_d[u];
          }
        }
        if (kept < kStep) {
          ok = __all_sync(0xffffffffu, mbar_wait_spin(&tail[st], (tail_phases >> st) & 1, p.err, kDevTimeoutProducer));
          if (!ok) break;
          tail_phases ^= 1u << st;
          // Rows stay whole under the swizzle.
          constexpr int kRow = DH * 2 / 16;
          for (int i = kept * kRow + lane; i < kStep * kRow; i += 32) {
            reinterpret_cast<uint4*>(tile)[i] = make_uint4(0u, 0u, 0u, 0u);
            reinterpret_cast<uint4*>(tile + G::kTileBytes)[i] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        if (it.keys || kept < kStep) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&full[st]);
            if (it.keys && kept < kStep) mbar_arrive(&full[st]);
          }
        }
        if (++st == kStages) {
          st = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp >= kStoreWarp) {
    // ---------------- gradients of finished items: one owned row per thread ----------------
    // Rounded rows go through shared memory, so that whole rows are written by neighbouring lanes.
    const int quarter = warp & 3;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    uint8_t* stage = smem + G::kOffOut + quarter * 32 * DH * 2;
    constexpr int kChunks = DH / 8;  // 16-byte pieces of a row
    for (int item = 0;; ++item) {
      if (!mbar_wait(&info_full[item % kInfos], (item / kInfos) & 1, p.err, kDevTimeoutEpilogue)) break;
      const Item it = *info_at(item);
      if (it.len == 0) break;
      const float back_ds = p.scale * ldexpf(1.0f, -it.ds_exp), back_p = ldexpf(1.0f, -kProbExp);
      if (!mbar_wait_hint(done, item & 1, p.err, kDevTimeoutEpilogue, 64)) break;
      tc_fence_after();
      uint32_t v[DH / 2];
      auto read = [&](uint32_t col, float back) {
#pragma unroll
        for (int cc = 0; cc < DH / 16; ++cc) {
          uint32_t o[16];
          tmem_ld16(lanes + col + 16 * cc, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; ++i)
            v[8 * cc + i] = pack2<E>(__uint_as_float(o[2 * i]) * back, __uint_as_float(o[2 * i + 1]) * back);
        }
      };
      auto release = [&]() {  // the accumulators may be written again
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_free);
      };
      auto put = [&]() {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          *reinterpret_cast<uint4*>(stage + swizzled<DH>(lane, c)) = make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
        __syncwarp();
      };
      auto write = [&](int part) {
        E* dst = static_cast<E*>(p.dqkv) + (static_cast<size_t>(part) * p.H + it.h) * p.dh;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          const int r = (32 / kChunks) * i + lane / kChunks, c = lane % kChunks, row = it.r0 + quarter * 32 + r;
          if (row < it.len && 8 * c < p.dh)
            *reinterpret_cast<uint4*>(dst + static_cast<size_t>(it.start + row) * p.ld_dqkv + 8 * c) =
                *reinterpret_cast<const uint4*>(stage + swizzled<DH>(r, c));
        }
        __syncwarp();
      };
      read(kColAcc1, back_ds);
      if (!it.keys) release();
      put();
      if (it.keys) {
        read(kColAcc2, back_p);
        release();
        write(1);
        put();
        write(2);
      } else {
        write(0);
      }
    }
  } else {
    // ---------------- elementwise: one owned row per thread, 32 of the 64 columns ----------------
    // Eight warps a step, and two teams that take steps in turn: three steps are in flight, and one team's wait for
    // scores, and its reads and writes of tensor memory, pass behind the other's arithmetic. The special-function
    // unit takes 512 cycles a step for the exponentials, less than half of it.
    const int quarter = warp & 3, team = warp / kTeamWarps, cols = kWarpCols * (warp % kTeamWarps >> 2);
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + cols;
    const float c = p.scale * kLog2e;
    const uint64_t c2 = f2_pack(c, c);
    // The record of an item and, for query items, lse and D of this thread's row, which are loaded one step
    // before they are used.
    Item it{};
    float row_l = 0.0f, row_d = 0.0f;
    auto fetch = [&](int item) {
      if (!mbar_wait_spin(&info_full[item % kInfos], (item / kInfos) & 1, p.err, kDevTimeoutEpilogue)) return false;
      it = *info_at(item);
      const int row = it.r0 + quarter * 32 + lane;
      if (it.len > 0 && !it.keys && row < it.len) {
        const size_t at = static_cast<size_t>(it.h) * p.T + it.start + row;
        row_l = p.lse[at];
        row_d = p.delta[at];
      }
      return true;
    };
    bool ok = fetch(0);
    int buf = team % kBufs, phase = 0, skip = team;  // this team's next step: its buffer, and how many steps away
    for (int item = 0; ok && it.len > 0;) {
      const bool keys = it.keys;
      const int len = it.len;
      const float f = __int_as_float((127 + it.ds_exp - (keys ? kProbExp : 0)) << 23);  // 2^e, or 2^(e - kProbExp)
      const uint64_t f2 = f2_pack(f, f);
      const float l = keys ? 0.0f : -row_l * kLog2e, d = keys ? 0.0f : -row_d * f;
      const uint64_t lse2 = f2_pack(l, l), delta2 = f2_pack(d, d);
      int left = (len + kStep - 1) / kStep - skip, kept = len - skip * kStep - cols;  // from this warp's first column on
      ++item;
      if (left <= 0 && !(ok = fetch(item))) break;
      for (; left > 0; left -= kTeams, kept -= kTeams * kStep) {
        if (left <= kTeams && !(ok = fetch(item))) break;
        if (!(ok = mbar_wait_spin(&scores[buf], phase, p.err, kDevTimeoutEpilogue))) break;
        tc_fence_after();
        const uint32_t t_s = lanes + buf * kColBuf, t_dp = t_s + kColDp;
#pragma unroll
        for (int q = 0; q < kWarpCols / 16; ++q) {
          uint32_t s[16], dp[16], pr[8], ds[8];
          tmem_ld16(t_s + 16 * q, s);
          tmem_ld16(t_dp + 16 * q, dp);
          tmem_ld_wait_regs(s, dp);
          if (!keys && kept < 16 * (q + 1)) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (16 * q + i >= kept) s[i] = __float_as_uint(-INFINITY);
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint64_t s2 = f2_pack(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1]));
            const uint64_t d2 = f2_pack(__uint_as_float(dp[2 * k]), __uint_as_float(dp[2 * k + 1]));
            float a0, a1, x0, x1;
            f2_unpack(f2_fma(s2, c2, lse2), a0, a1);
            const uint64_t e2 = f2_pack(fast_exp2(a0), fast_exp2(a1));
            f2_unpack(f2_mul(e2, f2_fma(d2, f2, delta2)), x0, x1);
            ds[k] = pack2<E>(x0, x1);
            f2_unpack(e2, x0, x1);
            pr[k] = pack2<E>(x0, x1);
          }
          if (keys) tmem_st8(t_s + 8 * q, pr);
          tmem_st8(t_dp + 8 * q, ds);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&probs[buf]);
        buf += kTeams;
        if (buf >= kBufs) {
          buf -= kBufs;
          phase ^= 1;
        }
      }
      skip = -left;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kScoreWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <int DH, typename E>
cudaError_t backward(const AttnOp& a, const BwdParams& p, cudaStream_t s) {
  constexpr bool kBf16 = std::is_same<E, __nv_bfloat16>::value;
  CUtensorMap tm_qkv, tm_dout, tm_qkv_own, tm_dout_own;  // boxes of 64 streamed and 128 owned rows
  if (!make_tmap_op_heads(&tm_qkv, a.qkv, kBf16, a.T, 3 * a.H, a.dh, a.ld_qkv, kStep) ||
      !make_tmap_op_heads(&tm_dout, a.dout, kBf16, a.T, a.H, a.dh, a.ld_dout, kStep) ||
      !make_tmap_op_heads(&tm_qkv_own, a.qkv, kBf16, a.T, 3 * a.H, a.dh, a.ld_qkv, kOwn) ||
      !make_tmap_op_heads(&tm_dout_own, a.dout, kBf16, a.T, a.H, a.dh, a.ld_dout, kOwn))
    return cudaErrorInvalidValue;
  static std::atomic<unsigned long long> configured{0};
  cudaError_t e = allow_smem(attention_backward_kernel<DH, E>, Bwd<DH>::kSmem, configured);
  if (e != cudaSuccess) return e;
  attention_delta_kernel<E><<<dim3(std::max(1, (a.max_len + kDeltaRows - 1) / kDeltaRows), a.H, a.B), 256, 0, s>>>(p);
  if (a.max_len == 0) return cudaGetLastError();  // only the offsets were looked at
  const int64_t items = static_cast<int64_t>(2) * (a.T / kOwn + a.B) * a.H;  // at most
  attention_backward_kernel<DH, E>
      <<<static_cast<unsigned>(std::min<int64_t>(items, a.num_sms)), kThreads, Bwd<DH>::kSmem, s>>>(tm_qkv, tm_dout, tm_qkv_own,
                                                                                                   tm_dout_own, p);
  return cudaGetLastError();
}

}  // namespace

size_t attention_backward_bytes(int B, int T, int H) {
  return sizeof(unsigned long long) + static_cast<size_t>(H) * T * 4 + static_cast<size_t>(H) * (T / kDeltaRows + B) * 8;
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
  p.claimed = reinterpret_cast<unsigned long long*>(a.workspace);
  p.delta = a.workspace + 2;
  p.peaks = p.delta + static_cast<size_t>(a.H) * a.T;
  p.blocks = a.T / kDeltaRows + a.B;
  p.B = a.B;
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
