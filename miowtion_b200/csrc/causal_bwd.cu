// Causal attention of packed sequences with grouped heads, backward.
//
// With the forward's log-sum-exp L and D_i = rowsum(dO_i * O_i):
//     P  = exp(S * scale - L)  (S = Q K^T; 0 where the mask hides a pair),
//     dP = dO V^T,  dS = P * (dP - D),
//     dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO,
// dK and dV summed over the query heads of a key head. Query tiles hold all
// heads of a group (causal.cuh), so that sum is one more stretch of the
// product's depth: no atomics, no second pass, and repeats are bit-identical.
//
// Three launches:
//   prep    -D and -L * log2(e) of each query row into the workspace, in tile
//           order [kv_heads][tiles][128], a row without keys or token as
//           -L = -inf, D = 0;
//   dq      a query tile an item, its key tiles one after the other: S and dP
//           (SS products), dS written back over S in tensor memory as bf16,
//           dQ += dS K (TS product);
//   dkdv    a key tile an item, the query tiles that see it: S^T = K Q^T and
//           dP^T = V dO^T, P^T and dS^T written back over them, dV += P^T dO
//           and dK += dS^T Q.
// One CTA per SM, 8 compute warps, a TMA producer warp and a converged MMA
// warp. Tensor memory at D = 128 decides how the two kernels overlap their
// products with the elementwise work. dq has one accumulator, so there is room
// for two S buffers beside dP: while the compute warps turn block b into dS,
// the tensor core has dP of b + 1 (as soon as dP of b is in registers), dQ of
// b - 1 and S of b + 1, all 128 columns wide. dk/dv has two accumulators of D
// columns and, at D = 128, no room: a block's 128 columns run as two halves of
// 64, and the tensor core has one half's products while the compute warps work
// on the other. D = 64 runs the same layout, though it leaves 128 columns
// unused; products 128 wide have not been measured there.
//
// No unit is full. At D = 128 the tensor core is busy 58 % of dq and 57 % of
// dkdv, whose products are 64 columns wide (such a product reads 6 KB of shared
// memory, 48 cycles' worth, for 32 cycles' work: the data path is at 72 %); at
// D = 64 37 and 35 %, the special function unit 50 and 35 %. The rest is
// products and elementwise work waiting for each other. The whole backward of
// 8,192 tokens, 16/4 heads, by step, at D = 128 and 64:
//     dq in halves too, S alone ahead            904 and 736 us
//     dq 128 columns wide                        874 and 743
//     elementwise work on pairs (f32x2), L and D
//     negated so that it is one fma and one add  840 and 709
//     the diagonal's selections in a copy of the
//     loop of their own                          800 and 615-635
// which is 860 and 550 TFLOP/s of the 10 D operations a pair that a backward
// pass is counted with, and 1,200 and 770 of the 14 D that these kernels do.
// 16 compute warps in dkdv, a group of eight a half: 797 against 801 us at D =
// 128, 664 against 617 at D = 64; not kept.
//
// P and dS are rounded to bf16 for their products, which costs the gradients
// as much again as the rounding of the results: dQ and dK are 2.4e-3 off (in
// the 2-norm, relative) where results that are only rounded are 1.7e-3 off.
// (Two bf16 numbers for a dS would be two more products of seven.) D's error
// is the same for all keys of a row and meets a sum that cancels, most of all
// where few keys hold the weight: from out as rounded to bf16 it made dQ
// 2.6e-3 off, and 3.9e-3 and 6.0e-3 with scores 4 and 16 times as large (300, 1
// and 70 tokens of N(0, 1), 4/2 heads, D = 128), so the forward also leaves the
// eight bits behind (causal.cuh), a byte an element: 2.4, 2.7 and 3.1e-3.
//
// Rows behind a sequence's end are cleared in shared memory where they are
// the depth of a product (keys in dq, queries in dkdv); elsewhere they are
// other rows of the result and are not stored, or masked by selection. So
// nothing that stands there, NaN included, reaches this sequence.
//
// The dS of the two kernels is computed twice (7 products a block instead of
// 5) in place of a reduction of dQ over CTAs. All waits are bounded
// (common.cuh).
#include "causal.cuh"

#include <type_traits>

namespace veda {
namespace causal {

namespace {

constexpr int kThreads = 320;
constexpr int kProducer = 8;
constexpr int kMma = 9;
constexpr uint32_t kTmemCols = 512;
constexpr float kLog2e = 1.4426950408889634f;

template <int kD>
struct Bwd {
  static constexpr uint32_t kTileBytes = kTile * kD * 2;
  static constexpr uint32_t kTileUnits = kTileBytes >> 4;
  static constexpr int kSteps = kD / 16;
  static constexpr int kStages = kD == 128 ? 2 : 4;  // pairs of tiles
  // dk/dv: two resident tiles, the stages and their (L, D) vectors.
  static constexpr int kSmem = (2 + 2 * kStages) * kTileBytes +
                               kStages * 1024 + 512 + 1024;
  // dq: Q and dO, rings of K and V.
  static constexpr int kKRing = 3, kVRing = 2;
  static constexpr int kDqSmem =
      (2 + kKRing + kVRing) * kTileBytes + 512 + 1024;
};

struct BwdParams {
  const int32_t* table;
  int entries;
  int kv_heads;
  int group;
  int tokens;           // of a query tile
  int n_tiles;          // query tiles of the pack
  const float* neg_l;   // [kv_heads][n_tiles][128], -L log2(e)
  const float* neg_d;   // [kv_heads][n_tiles][128], -D
  __nv_bfloat16* grad;  // dq or dk
  int64_t grad_st, grad_sh;
  __nv_bfloat16* grad2;  // dv
  int64_t grad2_st, grad2_sh;
  float scale;
  float scale_log2;
  // dk/dv: item of each turn of each CTA, [turns][gridDim.x], -1 behind a
  // CTA's last; null: back and forth.
  const int32_t* order;
  int turns;
  unsigned int* status;
};

// Item number of a CTA's n-th turn; negative behind its last.
__device__ __forceinline__ int64_t key_turn(const BwdParams& p, int n,
                                            int64_t n_items) {
  if (p.order != nullptr)
    return n < p.turns ? __ldg(p.order + static_cast<int64_t>(n) * gridDim.x +
                               blockIdx.x)
                       : -1;
  return static_cast<int64_t>(n) * gridDim.x < n_items ? turn(n) : -1;
}

__device__ __forceinline__ void arrive_warp(uint64_t* bar) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// One box (64-column pieces) of rows row .. of heads h .. into a tile.
template <int kD>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map,
                                          uint64_t* bar, int h, int row) {
#pragma unroll
  for (int c = 0; c < kD / 64; ++c)
    tma_load_3d(dst + c * 16384, map, bar, c * 64, h, row);
}

__device__ __forceinline__ float2 pair_of(const uint32_t* x, int i) {
  return make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
}

// Writes kN bf16 columns of a row (kN / 2 words).
template <int kN>
__device__ __forceinline__ void store_row(__nv_bfloat16* dst,
                                          const uint32_t* w) {
#pragma unroll
  for (int i = 0; i < kN / 16; ++i) store32(dst + 16 * i, w + 8 * i);
}

// Reads kN fp32 TMEM columns of this thread's lane, scales them and packs
// them to bf16 pairs.
template <int kN>
__device__ __forceinline__ void tmem_row_bf16(uint32_t taddr, float scale,
                                              uint32_t* w) {
  uint32_t o[32];
#pragma unroll
  for (int c = 0; c < kN / 32; ++c) {
    tmem_ld32(taddr + c * 32, o);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i)
      w[c * 16 + i] = pack_bf16(__uint_as_float(o[2 * i]) * scale,
                                __uint_as_float(o[2 * i + 1]) * scale);
  }
}

// ---------------------------------------------------------------------------
// prep: a block per (query tile, key head), kD / 8 lanes a row. Bound by
// memory (out, its low bits and dout once): every thread has four rows' loads
// in flight (all eight of D = 128: 122 registers, 19 us against 17 for 8,192
// tokens of 16 heads).
// ---------------------------------------------------------------------------
constexpr int kPrepThreads = 256;

template <int kD>
__global__ void __launch_bounds__(kPrepThreads) causal_bwd_prep_kernel(
    const int32_t* table, int group, int tokens, const __nv_bfloat16* out,
    int64_t o_st, int64_t o_sh, const int8_t* low, const __nv_bfloat16* dout,
    int64_t d_st,
    int64_t d_sh, const float* lse, int64_t l_st, int64_t l_sh, float* neg_l,
    float* neg_d, int n_tiles) {
  constexpr int kLanes = kD / 8;
  constexpr int kStep = kPrepThreads / kLanes;  // rows at a time
  constexpr int kRounds = kTile / kStep;
  constexpr int kBatch = 4;  // rounds whose loads are in flight together
  const int lane = threadIdx.x % kLanes;
  const int h = blockIdx.y;
  const QueryItem it = load_item<QueryItem>(table, blockIdx.x);
  const int64_t at = (static_cast<int64_t>(h) * n_tiles + it.tile) * kTile;
#pragma unroll 1
  for (int first = 0; first < kRounds; first += kBatch) {
    uint4 a[kBatch], b[kBatch];
    uint2 c[kBatch];
    float l[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int r = (first + i) * kStep + threadIdx.x / kLanes;
      const int token = r / group;
      a[i] = b[i] = make_uint4(0, 0, 0, 0);
      c[i] = make_uint2(0, 0);
      l[i] = -INFINITY;
      if (token < it.tokens && token < tokens) {
        const int64_t row = static_cast<int64_t>(it.row) + token;
        const int64_t hq = static_cast<int64_t>(h) * group + r % group;
        a[i] = *reinterpret_cast<const uint4*>(out + row * o_st + hq * o_sh +
                                               lane * 8);
        b[i] = *reinterpret_cast<const uint4*>(dout + row * d_st + hq * d_sh +
                                               lane * 8);
        l[i] = lse[row * l_st + hq * l_sh];
        if (low != nullptr)
          c[i] = *reinterpret_cast<const uint2*>(
              low + (row * gridDim.y * group + hq) * kD + lane * 8);
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const uint32_t x[4] = {a[i].x, a[i].y, a[i].z, a[i].w};
      const uint32_t y[4] = {b[i].x, b[i].y, b[i].z, b[i].w};
      float acc = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t z = (e < 2 ? c[i].x : c[i].y) >> (16 * (e & 1));
        acc = fmaf(with_low<0>(x[e] << 16, z), __uint_as_float(y[e] << 16),
                   acc);
        acc = fmaf(with_low<1>(x[e], z), __uint_as_float(y[e] & 0xFFFF0000u),
                   acc);
      }
#pragma unroll
      for (int s = kLanes / 2; s > 0; s >>= 1)
        acc += __shfl_xor_sync(0xffffffffu, acc, s);
      if (lane == 0) {
        const int r = (first + i) * kStep + threadIdx.x / kLanes;
        // A row without keys or token.
        const bool none = l[i] == -INFINITY;
        neg_d[at + r] = none ? 0.f : -acc;
        neg_l[at + r] = none ? -INFINITY : -(l[i] * kLog2e);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// dq. TMEM: S of block b in [128 (b % 2), ..) (then dS, bf16, over columns 0-31
// and 64-95 of it), dP [256, 384), dQ [384, 384 + kD). Blocks are numbered
// through the CTA's items.
// ---------------------------------------------------------------------------
enum DqBar {
  kQFull = 0,                 // Q of the item landed
  kQEmpty,                    // the item's last S finished
  kDoFull,                    // dO of the item landed
  kDoEmpty,                   // the item's last dP finished
  kSFull,                     // [2] S of the block (by its parity)
  kDpFull = kSFull + 2,       // dP of the block
  kDpFree,                    // dP is in registers (8 warps)
  // dS written (8 warps), [2] by the block's parity: dP of the next block is
  // on its way before the product that waits here, so its dS may be written
  // too, and one barrier could be two phases on.
  kDsFull,
  kDqDone = kDsFull + 2,      // the item's last dQ product finished
  kDqFree,                    // the epilogue has read dQ (8 warps)
  kDqDrain,
  kKFull,                     // [kKRing]
  kKEmpty = kKFull + 3,       // [kKRing]
  kVFull = kKEmpty + 3,       // [kVRing]
  kVEmpty = kVFull + 2,       // [kVRing]
  kDqNumBars = kVEmpty + 2
};

// The query items of a CTA that have key tiles (all with keep_empty).
struct QueryStream {
  int t;  // turns taken
  int h;
  QueryItem it;
  __device__ __forceinline__ bool next(const BwdParams& p, int n_items,
                                       bool keep_empty) {
    while (static_cast<int64_t>(t) * gridDim.x < n_items) {
      const int64_t i = turn(t++);
      if (i >= n_items) continue;
      const int entry = static_cast<int>(i) / p.kv_heads;
      h = static_cast<int>(i) - entry * p.kv_heads;
      it = load_item<QueryItem>(p.table, entry);
      if (it.blocks > 0 || keep_empty) return true;
    }
    return false;
  }
};

// A position in the stream of blocks: block j of the current item.
struct BlockCursor {
  QueryStream st;
  int b, j, items;
  bool valid;
  __device__ __forceinline__ void init(const BwdParams& p, int n_items) {
    st.t = 0;
    b = j = items = 0;
    valid = st.next(p, n_items, false);
  }
  __device__ __forceinline__ bool first() const { return j == 0; }
  __device__ __forceinline__ bool last() const {
    return j == st.it.blocks - 1;
  }
  __device__ __forceinline__ void next(const BwdParams& p, int n_items) {
    ++b;
    if (++j < st.it.blocks) return;
    j = 0;
    ++items;
    valid = st.next(p, n_items, false);
  }
};

template <int kD>
__global__ void __launch_bounds__(kThreads, 1)
    causal_dq_kernel(const __grid_constant__ CUtensorMap map_q,
                     const __grid_constant__ CUtensorMap map_do,
                     const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v,
                     const __grid_constant__ BwdParams p) {
  using C = Bwd<kD>;
  constexpr uint32_t kTileBytes = C::kTileBytes;
  constexpr int kKRing = C::kKRing, kVRing = C::kVRing;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem;
  uint8_t* s_do = smem + kTileBytes;
  uint8_t* s_k = smem + 2 * kTileBytes;  // [kKRing]
  uint8_t* s_v = s_k + kKRing * kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_v + kVRing * kTileBytes);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kDqNumBars);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int tid = threadIdx.x;
  const int warp = tid / 32;
  const int lane = tid % 32;
  const int n_items = p.entries * p.kv_heads;
  if (tid == 0) {
    for (int b = 0; b < kDqNumBars; ++b)
      mbar_init(&bars[b],
                (b == kDpFree || b == kDsFull || b == kDsFull + 1 ||
                 b == kDqFree)
                    ? 8
                    : 1);
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == kMma) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == kProducer) {
    if (lane == 0) {
      prefetch_tensor_map(&map_q);
      prefetch_tensor_map(&map_do);
      prefetch_tensor_map(&map_k);
      prefetch_tensor_map(&map_v);
    }
    const uint32_t q_bytes = p.group * p.tokens * kD * 2;
    int q_loads = 0, do_loads = 0, k_loads = 0, v_loads = 0;
    // Waits for place n of a ring, then loads a tile into it.
    auto ring_load = [&](int& n, int ring, int full, int empty, uint8_t* base,
                         const CUtensorMap* map, int h, int row) -> bool {
      const int slot = n % ring;
      if (n >= ring && !wait_all(&bars[empty + slot], ((n / ring) - 1) & 1,
                                 abort, p.status))
        return false;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars[full + slot], kTileBytes);
        load_tile<kD>(base + slot * kTileBytes, map, &bars[full + slot], h,
                      row);
      }
      __syncwarp();
      ++n;
      return true;
    };
    auto item_load = [&](int& n, int full, int empty, uint8_t* dst,
                         const CUtensorMap* map, int h, int row) -> bool {
      if (n > 0 && !wait_all(&bars[empty], (n - 1) & 1, abort, p.status))
        return false;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars[full], q_bytes);
        load_tile<kD>(dst, map, &bars[full], h, row);
      }
      __syncwarp();
      ++n;
      return true;
    };
    QueryStream st{0};
    bool run = true;
    while (run && st.next(p, n_items, false)) {
      for (int j = 0; run && j < st.it.blocks; ++j) {
        const int row = st.it.k_row + j * kTile;
        run = ring_load(k_loads, kKRing, kKFull, kKEmpty, s_k, &map_k, st.h,
                        row);
        if (run && j == 0)
          run = item_load(q_loads, kQFull, kQEmpty, s_q, &map_q,
                          st.h * p.group, st.it.row);
        if (run)
          run = ring_load(v_loads, kVRing, kVFull, kVEmpty, s_v, &map_v, st.h,
                          row);
        if (run && j == 0)
          run = item_load(do_loads, kDoFull, kDoEmpty, s_do, &map_do,
                          st.h * p.group, st.it.row);
      }
    }
    if (lane == 0 && *abort) {
      // Let the copies in flight land before the CTA retires.
      volatile int never = 0;
      if (q_loads > 0)
        mbar_wait(&bars[kQFull], (q_loads - 1) & 1, &never, nullptr);
      if (do_loads > 0)
        mbar_wait(&bars[kDoFull], (do_loads - 1) & 1, &never, nullptr);
      for (int n = k_loads - kKRing; n < k_loads; ++n)
        if (n >= 0)
          mbar_wait(&bars[kKFull + n % kKRing], (n / kKRing) & 1, &never,
                    nullptr);
      for (int n = v_loads - kVRing; n < v_loads; ++n)
        if (n >= 0)
          mbar_wait(&bars[kVFull + n % kVRing], (n / kVRing) & 1, &never,
                    nullptr);
    }
  } else if (warp == kMma) {
    constexpr uint32_t idesc_sd = idesc_bf16(128, 128, false, false);
    constexpr uint32_t idesc_acc = idesc_bf16(128, kD, false, true);
    const uint32_t q_lo = sw128_desc_lo(smem_u32(s_q), 16);
    const uint32_t do_lo = sw128_desc_lo(smem_u32(s_do), 16);
    const uint32_t k_lo = sw128_desc_lo(smem_u32(s_k), 16);
    const uint32_t v_lo = sw128_desc_lo(smem_u32(s_v), 16);
    const uint32_t kmn_lo = sw128_desc_lo(smem_u32(s_k), 16384);
    bool ok = true;
    auto wait = [&](int bar, int phase) -> bool {
      if (ok && !wait_all(&bars[bar], phase & 1, abort, p.status)) ok = false;
      return ok;
    };
    // S of the block at `c` (waits for its Q and K).
    auto issue_s = [&](const BlockCursor& c) {
      const int slot = c.b % kKRing;
      if (c.first()) wait(kQFull, c.items);
      if (!wait(kKFull + slot, c.b / kKRing)) return;
      // Key rows behind the sequence are the depth of dQ's product.
      const int rows = c.st.it.keys - c.j * kTile;
      if (rows < kTile) clear_rows<kD>(s_k + slot * kTileBytes, rows, lane);
      tc_fence_after();
      const uint32_t bk = k_lo + slot * C::kTileUnits;
      umma_ss_run<C::kSteps>(tmem + (c.b & 1) * 128, q_lo, bk, idesc_sd);
      umma_commit_warp(&bars[kSFull + (c.b & 1)]);
      if (c.last()) umma_commit_warp(&bars[kQEmpty]);
    };
    auto issue_dp = [&](const BlockCursor& c) {
      const int slot = c.b % kVRing;
      if (c.first()) wait(kDoFull, c.items);
      if (!wait(kVFull + slot, c.b / kVRing)) return;
      tc_fence_after();
      const uint32_t bv = v_lo + slot * C::kTileUnits;
      umma_ss_run<C::kSteps>(tmem + 256, do_lo, bv, idesc_sd);
      umma_commit_warp(&bars[kDpFull]);
      umma_commit_warp(&bars[kVEmpty + slot]);
      if (c.last()) umma_commit_warp(&bars[kDoEmpty]);
    };
    // Three places in the stream: dQ of block b, dP of b + 1, S of b + 2.
    BlockCursor at, at_dp, at_s;
    at.init(p, n_items);
    at_dp = at_s = at;
    if (at_s.valid) {
      issue_s(at_s);
      at_s.next(p, n_items);
    }
    if (ok && at_dp.valid) {
      issue_dp(at_dp);
      at_dp.next(p, n_items);
    }
    if (ok && at_s.valid) {
      issue_s(at_s);
      at_s.next(p, n_items);
    }
    while (ok && at.valid) {
      if (!wait(kDpFree, at.b)) break;
      tc_fence_after();
      if (at_dp.valid) {
        issue_dp(at_dp);
        if (!ok) break;
        at_dp.next(p, n_items);
      }
      // The item's first dQ overwrites dQ: the epilogue must have read it.
      if (at.first() && at.items > 0 && !wait(kDqFree, at.items - 1)) break;
      if (!wait(kDsFull + (at.b & 1), at.b >> 1)) break;
      tc_fence_after();
      const int slot = at.b % kKRing;
      const uint32_t bk = kmn_lo + slot * C::kTileUnits;
      const uint32_t ds = tmem + (at.b & 1) * 128;
      umma_ts_run<false>(tmem + 384, ds, bk, idesc_acc, !at.first());
      umma_ts_run<false>(tmem + 384, ds + 64, bk + 512, idesc_acc, 1);
      umma_commit_warp(&bars[kKEmpty + slot]);
      if (at.last()) umma_commit_warp(&bars[kDqDone]);
      if (at_s.valid) {
        issue_s(at_s);
        if (!ok) break;
        at_s.next(p, n_items);
      }
      at.next(p, n_items);
    }
    if (*abort) {
      volatile int never = 0;
      umma_commit_warp(&bars[kDqDrain]);
      mbar_wait(&bars[kDqDrain], 0, &never, nullptr);
    }
  } else {
    // ---------------- compute warps 0-7 ----------------
    const int half = warp / 4;  // keys 64 half .. of each block
    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
    const int quarter = warp % 4;
    const int row = quarter * 32 + lane;
    const int token = row / p.group;
    const int head = row % p.group;
    const bool row_used = row < p.tokens * p.group;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    int blk = 0, items = 0;
    bool ok = true;
    QueryStream st{0};
    while (ok && st.next(p, n_items, true)) {
      const int n = st.it.blocks;
      const bool write = row_used && token < st.it.tokens;
      __nv_bfloat16* dst =
          p.grad + (static_cast<int64_t>(st.it.row) + token) * p.grad_st +
          (static_cast<int64_t>(st.h) * p.group + head) * p.grad_sh +
          half * (kD / 2);
      if (n == 0) {
        uint32_t z[kD / 4] = {0};
        if (write) store_row<kD / 2>(dst, z);
        continue;
      }
      const int64_t at =
          (static_cast<int64_t>(st.h) * p.n_tiles + st.it.tile) * kTile + row;
      const float2 nl = make_float2(p.neg_l[at], p.neg_l[at]);
      const float2 nd = make_float2(p.neg_d[at], p.neg_d[at]);
      const int seen = max(0, min(st.it.keys, st.it.kpos + token + 1));
      for (int j = 0; j < n; ++j, ++blk) {
        const int visible = seen - j * kTile - half * 64;
        const bool masked = __any_sync(0xffffffffu, visible < 64);
        const uint32_t t_s = tmem + (blk & 1) * 128 + half * 64 + lane_base;
        const uint32_t t_dp = tmem + 256 + half * 64 + lane_base;
        if (!wait_all(&bars[kSFull + (blk & 1)], (blk >> 1) & 1, abort,
                      p.status) ||
            !wait_all(&bars[kDpFull], blk & 1, abort, p.status)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t dp[2][32], s[32], w[2][16];
        tmem_ld32(t_dp, dp[0]);
        tmem_ld32(t_dp + 32, dp[1]);
        tmem_ld32(t_s, s);
        tmem_wait_ld();
        arrive_warp(&bars[kDpFree]);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          if (q == 1) {
            tmem_ld32(t_s + 32, s);
            tmem_wait_ld();
          }
          // (On the diagonal apart: a selection costs as much as the rest.)
          auto weigh = [&](auto diagonal) {
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const float2 pr =
                  exp2_pair(__ffma2_rn(pair_of(s, c), scale2, nl));
              float2 ds = __fmul2_rn(pr, __fadd2_rn(pair_of(dp[q], c), nd));
              if (decltype(diagonal)::value) {
                if (q * 32 + 2 * c >= visible) ds.x = 0.f;
                if (q * 32 + 2 * c + 1 >= visible) ds.y = 0.f;
              }
              w[q][c] = pack_bf16(ds.x, ds.y);
            }
          };
          if (masked)
            weigh(std::true_type{});
          else
            weigh(std::false_type{});
        }
        // dS of these 64 keys over the first 32 of this warp's own 64 columns
        // of S (all of them are in registers).
        tmem_st16(t_s, w[0]);
        tmem_st16(t_s + 16, w[1]);
        tmem_wait_st();
        arrive_warp(&bars[kDsFull + (blk & 1)]);
      }
      if (!ok) break;
      if (!wait_all(&bars[kDqDone], items & 1, abort, p.status)) break;
      ++items;
      tc_fence_after();
      uint32_t w[kD / 4];
      tmem_row_bf16<kD / 2>(tmem + 384 + half * (kD / 2) + lane_base, p.scale,
                            w);
      arrive_warp(&bars[kDqFree]);
      if (write) store_row<kD / 2>(dst, w);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// dkdv. TMEM, per half h: S^T [128h, 128h+64) (P^T over its columns 0-15 and
// 32-47), dP^T [128h+64, 128h+128) (dS^T likewise); dV [256, 256 + kD), dK
// [384, 384 + kD).
// ---------------------------------------------------------------------------
enum KvBar {
  kKtFull = 0,                // K and V of the key tile landed
  kKtEmpty,                   // the item's last S^T and dP^T finished
  kStFull,                    // [2 halves] S^T and dP^T of the block's half
  kPdsFull = kStFull + 2,     // [2 halves] P^T and dS^T written (8 warps)
  kKvDone = kPdsFull + 2,     // the item's last dV and dK products finished
  kKvFree,                    // the epilogue has read dV and dK (8 warps)
  kKvDrain,
  kQdFull,                    // [kStages] Q, dO, L and D of the block landed
  kQdEmpty = kQdFull + 4,     // [kStages] the block's products finished
  kKvNumBars = kQdEmpty + 4
};

template <int kD>
__global__ void __launch_bounds__(kThreads, 1)
    causal_dkdv_kernel(const __grid_constant__ CUtensorMap map_q,
                       const __grid_constant__ CUtensorMap map_do,
                       const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v,
                       const __grid_constant__ BwdParams p) {
  using C = Bwd<kD>;
  constexpr int kStages = C::kStages;
  constexpr uint32_t kTileBytes = C::kTileBytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_k = smem;
  uint8_t* s_v = smem + kTileBytes;
  uint8_t* s_qd = smem + 2 * kTileBytes;  // [kStages] x (Q, dO)
  float* s_vec = reinterpret_cast<float*>(
      smem + (2 + 2 * kStages) * kTileBytes);  // [kStages] x (L, D)
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_vec + kStages * 256);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kKvNumBars);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int tid = threadIdx.x;
  const int warp = tid / 32;
  const int lane = tid % 32;
  const int64_t n_items = static_cast<int64_t>(p.entries) * p.kv_heads;
  const int tile_rows = p.tokens * p.group;
  if (tid == 0) {
    for (int b = 0; b < kKvNumBars; ++b)
      mbar_init(&bars[b],
                (b == kPdsFull || b == kPdsFull + 1 || b == kKvFree) ? 8 : 1);
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == kMma) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  // Rows that no box fills (a group that does not divide 128) are the depth
  // of the products: they stay zero.
  if (tile_rows < kTile) {
    for (int i = tid; i < 2 * kStages * static_cast<int>(C::kTileUnits);
         i += kThreads)
      reinterpret_cast<uint4*>(s_qd)[i] = make_uint4(0, 0, 0, 0);
    fence_async_shared();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == kProducer) {
    if (lane == 0) {
      prefetch_tensor_map(&map_q);
      prefetch_tensor_map(&map_do);
      prefetch_tensor_map(&map_k);
      prefetch_tensor_map(&map_v);
    }
    const uint32_t qd_bytes = 2u * tile_rows * kD * 2 + 1024;
    int kt_loads = 0, qd_loads = 0;
    bool run = true;
    for (int t = 0; run; ++t) {
      const int64_t i = key_turn(p, t, n_items);
      if (i < 0) break;
      if (i >= n_items) continue;
      const int h = static_cast<int>(i % p.kv_heads);
      const KeyItem it =
          load_item<KeyItem>(p.table, static_cast<int>(i / p.kv_heads));
      if (it.blocks == 0) continue;
      if (kt_loads > 0 &&
          !wait_all(&bars[kKtEmpty], (kt_loads - 1) & 1, abort, p.status))
        break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars[kKtFull], 2 * kTileBytes);
        load_tile<kD>(s_k, &map_k, &bars[kKtFull], h, it.row);
        load_tile<kD>(s_v, &map_v, &bars[kKtFull], h, it.row);
      }
      __syncwarp();
      ++kt_loads;
      for (int j = 0; j < it.blocks; ++j) {
        const int stage = qd_loads % kStages;
        if (qd_loads >= kStages &&
            !wait_all(&bars[kQdEmpty + stage],
                      ((qd_loads / kStages) - 1) & 1, abort, p.status)) {
          run = false;
          break;
        }
        if (lane == 0) {
          uint8_t* dst = s_qd + stage * 2 * kTileBytes;
          const int64_t base = (static_cast<int64_t>(h) * p.n_tiles +
                                it.tile0 + it.first + j) *
                               kTile;
          const int q_row = it.q_row + (it.first + j) * p.tokens;
          uint64_t* bar = &bars[kQdFull + stage];
          mbar_arrive_expect_tx(bar, qd_bytes);
          load_tile<kD>(dst, &map_q, bar, h * p.group, q_row);
          load_tile<kD>(dst + kTileBytes, &map_do, bar, h * p.group, q_row);
          bulk_load(s_vec + stage * 256, p.neg_l + base, 512, bar);
          bulk_load(s_vec + stage * 256 + 128, p.neg_d + base, 512, bar);
        }
        __syncwarp();
        ++qd_loads;
      }
    }
    if (lane == 0 && *abort) {
      volatile int never = 0;
      if (kt_loads > 0)
        mbar_wait(&bars[kKtFull], (kt_loads - 1) & 1, &never, nullptr);
      for (int b = qd_loads - kStages; b < qd_loads; ++b)
        if (b >= 0)
          mbar_wait(&bars[kQdFull + b % kStages], (b / kStages) & 1, &never,
                    nullptr);
    }
  } else if (warp == kMma) {
    // Per block j, halves a (query rows 0-63) and b (64-127):
    //   S^T_a, dP^T_a, S^T_b, dP^T_b of block 0 of the item, then for each j
    //   dV, dK += half a of j; S^T_a, dP^T_a of j + 1;
    //   dV, dK += half b of j; S^T_b, dP^T_b of j + 1.
    constexpr uint32_t idesc_st = idesc_bf16(128, 64, false, false);
    constexpr uint32_t idesc_acc = idesc_bf16(128, kD, false, true);
    const uint32_t k_lo = sw128_desc_lo(smem_u32(s_k), 16);
    const uint32_t v_lo = sw128_desc_lo(smem_u32(s_v), 16);
    const uint32_t qd_lo = sw128_desc_lo(smem_u32(s_qd), 16);
    const uint32_t qdmn_lo = sw128_desc_lo(smem_u32(s_qd), 16384);
    const uint32_t t_dv = tmem + 256, t_dk = tmem + 384;
    auto issue_st = [&](int stage, int h) {
      const uint32_t q_lo =
          qd_lo + stage * 2 * C::kTileUnits + h * (8192 >> 4);
      const uint32_t do_lo = q_lo + C::kTileUnits;
      const uint32_t t_s = tmem + h * 128, t_dp = t_s + 64;
      umma_ss_run<C::kSteps>(t_s, k_lo, q_lo, idesc_st);
      umma_ss_run<C::kSteps>(t_dp, v_lo, do_lo, idesc_st);
      umma_commit_warp(&bars[kStFull + h]);
    };
    // dV += P^T dO and dK += dS^T Q over half h's 64 query rows.
    auto issue_acc = [&](int stage, int h, bool first) {
      const uint32_t qmn = qdmn_lo + stage * 2 * C::kTileUnits;
      const uint32_t domn = qmn + C::kTileUnits;
      const uint32_t t_p = tmem + h * 128, t_ds = t_p + 64;
      const uint32_t more = (h > 0 || !first) ? 1u : 0u;
      umma_ts_run<true>(t_dv, t_p, domn + h * 512, idesc_acc, more);
      umma_ts_run<true>(t_dk, t_ds, qmn + h * 512, idesc_acc, more);
    };
    int blk = 0, items = 0;
    bool run = true;
    for (int t = 0; run; ++t) {
      const int64_t i = key_turn(p, t, n_items);
      if (i < 0) break;
      if (i >= n_items) continue;
      const KeyItem it =
          load_item<KeyItem>(p.table, static_cast<int>(i / p.kv_heads));
      const int n = it.blocks;
      if (n == 0) continue;
      // Q and dO of block j have landed, and the query rows behind the
      // sequence are clear.
      auto block_ready = [&](int j) -> bool {
        const int b = blk + j;
        if (!wait_all(&bars[kQdFull + b % kStages], (b / kStages) & 1, abort,
                      p.status))
          return false;
        const int left =
            (it.tokens - (it.first + j) * p.tokens) * p.group;
        if (left < tile_rows) {
          uint8_t* dst = s_qd + (b % kStages) * 2 * kTileBytes;
          clear_rows<kD>(dst, left, lane);
          clear_rows<kD>(dst + kTileBytes, left, lane);
        }
        tc_fence_after();
        return true;
      };
      if (!wait_all(&bars[kKtFull], items & 1, abort, p.status) ||
          !block_ready(0))
        break;
      issue_st(blk % kStages, 0);
      issue_st(blk % kStages, 1);
      if (n == 1) umma_commit_warp(&bars[kKtEmpty]);
      for (int j = 0; j < n; ++j) {
        const int b = blk + j;
        const int stage = b % kStages;
        const int next = (b + 1) % kStages;
        const bool first = j == 0, last = j == n - 1;
        // The item's first dV and dK overwrite the accumulators, which the
        // epilogue must have read.
        if (first && items > 0 &&
            !wait_all(&bars[kKvFree], (items - 1) & 1, abort, p.status)) {
          run = false;
          break;
        }
        if (!wait_all(&bars[kPdsFull + 0], b & 1, abort, p.status)) {
          run = false;
          break;
        }
        tc_fence_after();
        issue_acc(stage, 0, first);
        if (!last) {
          if (!block_ready(j + 1)) {
            run = false;
            break;
          }
          issue_st(next, 0);
        }
        if (!wait_all(&bars[kPdsFull + 1], b & 1, abort, p.status)) {
          run = false;
          break;
        }
        tc_fence_after();
        issue_acc(stage, 1, first);
        umma_commit_warp(&bars[kQdEmpty + stage]);
        if (!last) {
          issue_st(next, 1);
          if (j + 1 == n - 1) umma_commit_warp(&bars[kKtEmpty]);
        } else {
          umma_commit_warp(&bars[kKvDone]);
        }
      }
      blk += n;
      ++items;
    }
    if (*abort) {
      volatile int never = 0;
      umma_commit_warp(&bars[kKvDrain]);
      mbar_wait(&bars[kKvDrain], 0, &never, nullptr);
    }
  } else {
    // ---------------- compute warps 0-7 ----------------
    const int wq = warp / 4;  // query rows 32 wq .. of each half
    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
    const int quarter = warp % 4;
    const int row = quarter * 32 + lane;  // key row of the tile
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    int blk = 0, items = 0;
    bool ok = true;
    for (int t = 0; ok; ++t) {
      const int64_t i = key_turn(p, t, n_items);
      if (i < 0) break;
      if (i >= n_items) continue;
      const int h = static_cast<int>(i % p.kv_heads);
      const KeyItem it =
          load_item<KeyItem>(p.table, static_cast<int>(i / p.kv_heads));
      const int n = it.blocks;
      const bool write = row < it.keys;
      const int64_t k_row = static_cast<int64_t>(it.row) + row;
      __nv_bfloat16* dk_dst =
          p.grad + k_row * p.grad_st + h * p.grad_sh + wq * (kD / 2);
      __nv_bfloat16* dv_dst =
          p.grad2 + k_row * p.grad2_st + h * p.grad2_sh + wq * (kD / 2);
      if (n == 0) {
        uint32_t z[kD / 4] = {0};
        if (write) {
          store_row<kD / 2>(dk_dst, z);
          store_row<kD / 2>(dv_dst, z);
        }
        continue;
      }
      for (int j = 0; j < n && ok; ++j, ++blk) {
        const float* vl = s_vec + (blk % kStages) * 256;  // -L log2(e), then -D
        // First query row of the block that sees this key.
        const int64_t from =
            (static_cast<int64_t>(it.shift) + row -
             static_cast<int64_t>(it.first + j) * p.tokens) *
            p.group;
        const bool masked = __any_sync(0xffffffffu, from > 0);
        const int cmin = static_cast<int>(
            from < 0 ? 0 : (from < kTile ? from : kTile));
        // The copy engine wrote L and D: who reads them sees their barrier
        // (which the products, behind it, have long passed).
        if (!wait_all(&bars[kQdFull + blk % kStages], (blk / kStages) & 1,
                      abort, p.status)) {
          ok = false;
          break;
        }
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          if (!wait_all(&bars[kStFull + hh], blk & 1, abort, p.status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const int q0 = hh * 64 + wq * 32;  // query column of the block
          const uint32_t t_s = tmem + hh * 128 + wq * 32 + lane_base;
          const uint32_t t_dp = t_s + 64;
          uint32_t s[32], dp[32];
          tmem_ld32(t_s, s);
          tmem_ld32(t_dp, dp);
          tmem_wait_ld();
          uint32_t wp[16], wd[16];
          auto weigh = [&](auto diagonal) {
#pragma unroll
            for (int c = 0; c < 16; c += 2) {
              const float4 l4 =
                  *reinterpret_cast<const float4*>(vl + q0 + 2 * c);
              const float4 d4 =
                  *reinterpret_cast<const float4*>(vl + 128 + q0 + 2 * c);
              const float2 nl[2] = {make_float2(l4.x, l4.y),
                                    make_float2(l4.z, l4.w)};
              const float2 nd[2] = {make_float2(d4.x, d4.y),
                                    make_float2(d4.z, d4.w)};
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float2 pr =
                    exp2_pair(__ffma2_rn(pair_of(s, c + e), scale2, nl[e]));
                float2 ds =
                    __fmul2_rn(pr, __fadd2_rn(pair_of(dp, c + e), nd[e]));
                if (decltype(diagonal)::value) {
                  const int col = q0 + 2 * (c + e);
                  if (col < cmin) pr.x = ds.x = 0.f;
                  if (col + 1 < cmin) pr.y = ds.y = 0.f;
                }
                wp[c + e] = pack_bf16(pr.x, pr.y);
                wd[c + e] = pack_bf16(ds.x, ds.y);
              }
            }
          };
          if (masked)
            weigh(std::true_type{});
          else
            weigh(std::false_type{});
          // P^T and dS^T of these 32 queries over the first 16 of this
          // warp's own 32 columns of S^T and dP^T.
          tmem_st16(t_s, wp);
          tmem_st16(t_dp, wd);
          tmem_wait_st();
          arrive_warp(&bars[kPdsFull + hh]);
        }
      }
      if (!ok) break;
      if (!wait_all(&bars[kKvDone], items & 1, abort, p.status)) break;
      ++items;
      tc_fence_after();
      uint32_t wv[kD / 4], wk[kD / 4];
      tmem_row_bf16<kD / 2>(tmem + 256 + wq * (kD / 2) + lane_base, 1.0f, wv);
      tmem_row_bf16<kD / 2>(tmem + 384 + wq * (kD / 2) + lane_base, p.scale,
                            wk);
      arrive_warp(&bars[kKvFree]);
      if (write) {
        store_row<kD / 2>(dv_dst, wv);
        store_row<kD / 2>(dk_dst, wk);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

struct Maps {
  CUtensorMap q, dout, k, v;
};

struct PrepArgs {
  const void* out;
  int64_t o_st, o_sh;
  const void* low;
  const void* dout;
  int64_t d_st, d_sh;
  const float* lse;
  int64_t l_st, l_sh;
  float *neg_l, *neg_d;
};

template <int kD>
int launch(const Maps& m, const BwdParams& pq, const BwdParams& pk, int k_ctas,
           const PrepArgs& a, bool want_q, bool want_k, cudaStream_t stream) {
  using C = Bwd<kD>;
  int sms = 0;
  int rc = device_sms(&sms);
  if (rc != VEDA_OK) return rc;
  if (pq.entries > 0) {
    causal_bwd_prep_kernel<kD>
        <<<dim3(pq.entries, pq.kv_heads), kPrepThreads, 0, stream>>>(
            pq.table, pq.group, pq.tokens,
            static_cast<const __nv_bfloat16*>(a.out), a.o_st, a.o_sh,
            static_cast<const int8_t*>(a.low),
            static_cast<const __nv_bfloat16*>(a.dout), a.d_st, a.d_sh, a.lse,
            a.l_st, a.l_sh, a.neg_l, a.neg_d, pq.n_tiles);
    rc = check_launch("causal_bwd_prep_kernel");
    if (rc != VEDA_OK) return rc;
  }
  const int64_t q_items = static_cast<int64_t>(pq.entries) * pq.kv_heads;
  if (want_q && q_items > 0) {
    static std::atomic<uint64_t> allowed{0};
    rc = allow_smem(reinterpret_cast<const void*>(causal_dq_kernel<kD>),
                    C::kDqSmem, &allowed);
    if (rc != VEDA_OK) return rc;
    const int grid = static_cast<int>(q_items < sms ? q_items : sms);
    causal_dq_kernel<kD><<<grid, kThreads, C::kDqSmem, stream>>>(
        m.q, m.dout, m.k, m.v, pq);
    rc = check_launch("causal_dq_kernel");
    if (rc != VEDA_OK) return rc;
  }
  const int64_t k_items = static_cast<int64_t>(pk.entries) * pk.kv_heads;
  if (want_k && k_items > 0) {
    static std::atomic<uint64_t> allowed{0};
    rc = allow_smem(reinterpret_cast<const void*>(causal_dkdv_kernel<kD>),
                    C::kSmem, &allowed);
    if (rc != VEDA_OK) return rc;
    const int grid = pk.order != nullptr
                         ? k_ctas
                         : static_cast<int>(k_items < sms ? k_items : sms);
    causal_dkdv_kernel<kD><<<grid, kThreads, C::kSmem, stream>>>(
        m.q, m.dout, m.k, m.v, pk);
    return check_launch("causal_dkdv_kernel");
  }
  return VEDA_OK;
}

}  // namespace

}  // namespace causal
}  // namespace veda

using namespace veda;

extern "C" int64_t veda_causal_bwd_workspace(int32_t kv_heads,
                                             int64_t n_tiles) {
  if (kv_heads < 1 || n_tiles < 0 || n_tiles >= (int64_t(1) << 31)) return -1;
  // L log2(e) and D of each row of each query tile.
  return 2 * static_cast<int64_t>(kv_heads) * n_tiles * kTile *
         static_cast<int64_t>(sizeof(float));
}

extern "C" int veda_causal_bwd(
    const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k,
    int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
    int64_t v_stride_h, const void* out, int64_t out_stride_t,
    int64_t out_stride_h, const void* out_low, const void* dout,
    int64_t dout_stride_t,
    int64_t dout_stride_h, const float* lse, int64_t lse_stride_t,
    int64_t lse_stride_h, int64_t total_q, int64_t total_k, int32_t n_heads,
    int32_t kv_heads, int32_t head_dim, const int32_t* q_items,
    int64_t n_q_items, const int32_t* k_items, int64_t n_k_items,
    const int32_t* k_order, int32_t k_ctas, int32_t k_turns, int64_t n_tiles,
    void* dq, int64_t dq_stride_t, int64_t dq_stride_h,
    void* dk, int64_t dk_stride_t, int64_t dk_stride_h, void* dv,
    int64_t dv_stride_t, int64_t dv_stride_h, float softmax_scale,
    void* workspace, int64_t workspace_bytes, void* stream) {
  VEDA_REQUIRE(head_dim == 64 || head_dim == 128,
               "head_dim must be 64 or 128");
  VEDA_REQUIRE(kv_heads >= 1 && n_heads >= 1 && n_heads % kv_heads == 0 &&
                   n_heads / kv_heads <= kTile,
               "n_heads must be 1 to 128 times kv_heads");
  VEDA_REQUIRE(total_q >= 0 && total_k >= 0 && total_q < (int64_t(1) << 31) &&
                   total_k < (int64_t(1) << 31) && n_q_items >= 0 &&
                   n_k_items >= 0 && n_tiles >= n_q_items &&
                   kv_heads <= 65535 &&
                   n_tiles * kv_heads < (int64_t(1) << 31) - 65536 &&
                   n_k_items * kv_heads < (int64_t(1) << 31) - 65536,
               "bad sizes");
  VEDA_REQUIRE(softmax_scale > 0.f &&
                   isfinite(softmax_scale * causal::kLog2e),
               "softmax_scale must be positive and finite");
  VEDA_REQUIRE((dk == nullptr) == (dv == nullptr),
               "dk and dv are computed together");
  const int64_t need = veda_causal_bwd_workspace(kv_heads, n_tiles);
  VEDA_REQUIRE(need >= 0 && workspace_bytes >= need &&
                   (need == 0 || workspace != nullptr) &&
                   reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               "workspace too small or not 16-byte aligned "
               "(veda_causal_bwd_workspace)");
  auto aligned = [](const void* ptr, int64_t st, int64_t sh, int elements) {
    return reinterpret_cast<uintptr_t>(ptr) % (2 * elements) == 0 &&
           st % elements == 0 && sh % elements == 0;
  };
  VEDA_REQUIRE(aligned(out, out_stride_t, out_stride_h, 8) &&
                   reinterpret_cast<uintptr_t>(out_low) % 8 == 0 &&
                   aligned(dout, dout_stride_t, dout_stride_h, 8) &&
                   aligned(dq, dq_stride_t, dq_stride_h, 16) &&
                   aligned(dk, dk_stride_t, dk_stride_h, 16) &&
                   aligned(dv, dv_stride_t, dv_stride_h, 16),
               "out and dout must be 16-byte aligned with strides multiple of "
               "8, out_low 8-byte aligned; dq, dk, dv 32-byte aligned with "
               "strides multiple of 16");
  VEDA_REQUIRE(reinterpret_cast<uintptr_t>(q_items) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(k_items) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(k_order) % 4 == 0 &&
                   reinterpret_cast<uintptr_t>(lse) % 4 == 0,
               "q_items and k_items must be 16-byte aligned, k_order and lse "
               "4-byte aligned");
  cudaStream_t s = as_stream(stream);
  const int group = n_heads / kv_heads;
  const int tokens = kTile / group;
  VEDA_REQUIRE(n_q_items == 0 || (q && out && dout && lse && q_items),
               "q, out, dout, lse and q_items are required");
  VEDA_REQUIRE(n_k_items == 0 || (k && v && k_items),
               "k, v and k_items are required");
  VEDA_REQUIRE(k_order == nullptr || (k_ctas >= 1 && k_turns >= 1),
               "k_order needs its CTAs and turns");
  int rc = require_sm100("veda_causal_bwd");
  if (rc != VEDA_OK) return rc;
  causal::Maps m;
  if (total_q > 0) {
    rc = causal::make_rows_map(&m.q, q, total_q, n_heads, head_dim,
                               q_stride_t, q_stride_h, group, tokens, "q");
    if (rc == VEDA_OK)
      rc = causal::make_rows_map(&m.dout, dout, total_q, n_heads, head_dim,
                                 dout_stride_t, dout_stride_h, group, tokens,
                                 "dout");
  }
  if (rc == VEDA_OK && total_k > 0) {
    rc = causal::make_rows_map(&m.k, k, total_k, kv_heads, head_dim,
                               k_stride_t, k_stride_h, 1, kTile, "k");
    if (rc == VEDA_OK)
      rc = causal::make_rows_map(&m.v, v, total_k, kv_heads, head_dim,
                                 v_stride_t, v_stride_h, 1, kTile, "v");
  }
  if (rc != VEDA_OK) return rc;
  // With no rows on one side every item of the other is empty and loads
  // nothing; its maps only have to exist.
  if (total_q == 0) m.q = m.dout = m.k;
  if (total_k == 0) m.k = m.v = m.q;
  causal::BwdParams p{};
  p.kv_heads = kv_heads;
  p.group = group;
  p.tokens = tokens;
  p.n_tiles = static_cast<int>(n_tiles);
  float* neg_l = static_cast<float*>(workspace);
  float* neg_d = neg_l + static_cast<int64_t>(kv_heads) * n_tiles * kTile;
  p.neg_l = neg_l;
  p.neg_d = neg_d;
  p.scale = softmax_scale;
  p.scale_log2 = softmax_scale * causal::kLog2e;
  p.status = device_status_ptr();
  causal::BwdParams pq = p, pk = p;
  pq.table = q_items;
  pq.entries = static_cast<int>(n_q_items);
  pq.grad = static_cast<__nv_bfloat16*>(dq);
  pq.grad_st = dq_stride_t;
  pq.grad_sh = dq_stride_h;
  pk.table = k_items;
  pk.entries = static_cast<int>(n_k_items);
  pk.order = k_order;
  pk.turns = k_turns;
  pk.grad = static_cast<__nv_bfloat16*>(dk);
  pk.grad_st = dk_stride_t;
  pk.grad_sh = dk_stride_h;
  pk.grad2 = static_cast<__nv_bfloat16*>(dv);
  pk.grad2_st = dv_stride_t;
  pk.grad2_sh = dv_stride_h;
  const causal::PrepArgs a{out,     out_stride_t,  out_stride_h,
                           out_low, dout,          dout_stride_t,
                           dout_stride_h, lse,     lse_stride_t,
                           lse_stride_h,  neg_l,   neg_d};
  return head_dim == 128
             ? causal::launch<128>(m, pq, pk, k_ctas, a, dq != nullptr,
                                   dk != nullptr, s)
             : causal::launch<64>(m, pq, pk, k_ctas, a, dq != nullptr,
                                  dk != nullptr, s);
}
