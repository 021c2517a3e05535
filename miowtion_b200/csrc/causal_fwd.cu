// Causal attention of packed sequences with grouped heads, forward.
//
// Token i of a sequence with n queries and c keys sees keys j <= i + c - n:
//     out_i = sum_j softmax_j(scale q_i . k_j) v_j,
//     lse_i = log sum_j exp(scale q_i . k_j);  no keys: out 0, lse -inf.
//
// A persistent kernel, one CTA per SM, on tcgen05. A CTA holds two query
// tiles A and B of one key head (causal.cuh: 128 rows of tokens x heads) and
// streams the key and value tiles of 128 keys once for both. Tensor memory
// (512 columns) holds an accumulator O for each tile and two (D = 128) or three
// (D = 64) buffers of 128 columns for scores, taken in turn by A(0), B(0),
// A(1), B(1), ...
//   warps 0-7   softmax and epilogue: warps 4g .. 4g + 3 own tile g, a query
//               row a thread over all 128 keys, with the running maximum and
//               sum of an online softmax (the maximum moves only when it
//               grows by more than 2^8, then O is rescaled). P goes back over
//               S as bf16, in two halves of 64 keys.
//   warp 8      TMA producer: the two Q tiles of an item, then its K and V
//               tiles through one ring.
//   warp 9      issues every product (and owns the tensor memory), in one
//               order: PV_A(b), QK_A(b + 1), PV_B(b), QK_B(b + 1) with two
//               buffers (the scores take the place of the weights that the
//               product before them read); with three, QK_B(b + 1) follows
//               PV_A(b) and QK_A(b + 2) follows PV_B(b), so that a tile's next
//               scores wait for nothing of its own (644 -> 695-710 TFLOP/s on
//               16,384 tokens, 24/6 heads).
//   warps 10-11 idle; they complete the third warpgroup, whose registers go
//               to the softmax warps (setmaxnreg).
// The tensor core works on one tile while the softmax of the other runs: in
// this order S_A is ready two products after P_A, and S_B two products later,
// so the two softmaxes do not run at the same time and wait at the same time.
// (With an issuer for QK and one for PV, P_A and P_B that became ready
// together led to PV_A, PV_B, QK_A, QK_B, which keeps them together: 1,050
// against 1,250-1,300 TFLOP/s on a causal sequence of 16,384 tokens, 24/6
// heads, D = 128. Measured on it and not kept: a block's first 32 weights
// computed against the reference so far while the other scores come in, 1,191;
// an eighth, a quarter, half of the exponentials as polynomials, 1,223, 1,177
// to 1,210 and 1,117 against 1,245; at D = 64 678 and 658 against 708.) The
// blocks of consecutive items form one stream, so the next item's first scores
// are computed while this item's epilogue runs. One issuer also makes barriers
// superfluous: the warps that write P of an item's first block have read the
// previous item's O, and with two buffers the scores of block b arrive after
// the product of block b - 1.
// Rows past a sequence's end belong to the next sequence (or to nothing):
// their scores are set to -inf by selection and the value rows are cleared in
// shared memory, so what stands there, NaN included, reaches no row of this
// sequence.
//
// All waits are bounded (common.cuh).
#include "causal.cuh"

namespace veda {
namespace causal {

namespace {

constexpr int kWarps = 12;
constexpr int kProducer = 8, kMma = 9;
constexpr uint32_t kTmemCols = 512;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;

template <int kD>
struct Fwd {
  static constexpr uint32_t kTileBytes = kTile * kD * 2;
  static constexpr int kRing = kD == 128 ? 4 : 8;
  // S buffers, taken in turn by A(0), B(0), A(1), B(1), ..., and the columns of
  // O_A and O_B behind them.
  static constexpr int kSBufs = kD == 128 ? 2 : 3;
  static constexpr uint32_t kO = kSBufs * 128;
  // With three the scores run a block ahead: V behind the next block's K.
  static constexpr bool kAhead = kSBufs == 3;
  // Q tiles, ring, then 4 KB a softmax warp to stage its output in.
  static constexpr int kSmem = (2 + kRing) * kTileBytes + 8 * 4096 + 512 + 1024;
  static constexpr int kSteps = kD / 16;  // K-steps of Q K^T
};

enum Bar {
  kQFull = 0,             // [2] Q of the tile landed
  kQEmpty = kQFull + 2,   // [2] the tile's last S product finished
  kSFull = kQEmpty + 2,   // [kSBufs] the scores in the buffer are finished
  // P of keys 0-63 and of keys 64-127 written (4 warps), [block % 2][2]: with
  // three buffers a tile's scores come a block ahead of its product, so its P
  // may too, and one barrier could be two phases on, which a wait by parity
  // takes for none.
  kPHalfA = kSFull + 3,
  kPHalfB = kPHalfA + 4,
  kODone = kPHalfB + 4,   // [2] the tile's last product of the item finished
  kPvDone = kODone + 2,   // [2] the tile's product of the block (3 buffers)
  kDrain = kPvDone + 2,
  kFull,                  // [kRing]
  kEmpty = kFull + 8,     // [kRing]
  kNumBars = kEmpty + 8
};

struct FwdParams {
  const int32_t* table;
  int entries;
  int kv_heads;
  int group;
  int tokens;    // of a query tile: 128 / group
  int warp_boxes;  // a warp's 32 rows are whole tokens: TMA stores them
  __nv_bfloat16* out;
  int64_t out_st, out_sh;
  int8_t* low;   // [tokens][heads][kD], out's low bits, or null
  float* lse;    // or null
  int64_t lse_st, lse_sh;
  float scale_log2;
  // Parts: [kv_heads][n_parts][2 tiles][128 rows][kD] accumulators, then
  // [...][128 rows][2] maxima and sums.
  float* part_o;
  float2* part_ml;
  int n_parts;
  const int32_t* joins;
  unsigned int* status;
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ float row_max32(const float* s) {
  float m[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) m[i] = max3(s[i], s[8 + i], s[16 + i]);
#pragma unroll
  for (int i = 0; i < 8; ++i) m[i] = fmaxf(m[i], s[24 + i]);
  return max3(max3(m[0], m[1], m[2]), max3(m[3], m[4], m[5]),
              fmaxf(m[6], m[7]));
}

// exp2(s * scale - m) of 32 scores, as bf16 pairs into r; returns their sum.
__device__ __forceinline__ float weights32(uint32_t* r, const float* s,
                                           float2 scale2, float2 neg_m2) {
  float2 sum_a = make_float2(0.f, 0.f), sum_b = make_float2(0.f, 0.f);
#pragma unroll
  for (int c = 0; c < 32; c += 4) {
    const float2 x0 = __ffma2_rn(make_float2(s[c], s[c + 1]), scale2, neg_m2);
    const float2 x1 =
        __ffma2_rn(make_float2(s[c + 2], s[c + 3]), scale2, neg_m2);
    const float2 e0 = make_float2(ex2_approx(x0.x), ex2_approx(x0.y));
    const float2 e1 = make_float2(ex2_approx(x1.x), ex2_approx(x1.y));
    sum_a = __fadd2_rn(sum_a, e0);
    sum_b = __fadd2_rn(sum_b, e1);
    r[c / 2] = pack_bf16(e0.x, e0.y);
    r[c / 2 + 1] = pack_bf16(e1.x, e1.y);
  }
  sum_a = __fadd2_rn(sum_a, sum_b);
  return sum_a.x + sum_a.y;
}

__device__ __forceinline__ void rescale16(uint32_t t_row, float alpha) {
  uint32_t o[16];
  tmem_ld16(t_row, o);
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 16; ++i)
    o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
  tmem_st16(t_row, o);
  tmem_wait_st();
}

// The items of a CTA that have key tiles (every role walks the same ones).
struct Stream {
  int t;  // turns taken
  int h;
  ForwardItem it;
  // The next item with blocks (kEmpty: any); false at the end.
  __device__ __forceinline__ bool next(const FwdParams& p, int64_t n_items,
                                       bool keep_empty) {
    while (static_cast<int64_t>(t) * gridDim.x < n_items) {
      const int64_t i = turn(t++);
      if (i >= n_items) continue;
      const int entry = static_cast<int>(
          static_cast<uint32_t>(i) / static_cast<uint32_t>(p.kv_heads));
      h = static_cast<int>(i) - entry * p.kv_heads;
      it = load_item<ForwardItem>(p.table, entry);
      if (it.blocks > 0 || keep_empty) return true;
    }
    return false;
  }
};

// A place in the stream of blocks of a CTA's items: block j of the current
// item, block b of the stream.
struct Cursor {
  Stream st;
  int b, j, items;
  bool valid;
  __device__ __forceinline__ void init(const FwdParams& p, int64_t n_items) {
    st.t = 0;
    b = j = items = 0;
    valid = st.next(p, n_items, false);
  }
  __device__ __forceinline__ bool last() const {
    return j == st.it.blocks - 1;
  }
  __device__ __forceinline__ void next(const FwdParams& p, int64_t n_items) {
    ++b;
    if (++j < st.it.blocks) return;
    j = 0;
    ++items;
    valid = st.next(p, n_items, false);
  }
};

template <int kD>
__global__ void __launch_bounds__(32 * kWarps, 1)
    causal_fwd_kernel(const __grid_constant__ CUtensorMap map_q,
                      const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ CUtensorMap map_out,
                      const __grid_constant__ FwdParams p) {
  using C = Fwd<kD>;
  constexpr int kRing = C::kRing;
  constexpr uint32_t kTileBytes = C::kTileBytes;
  constexpr uint32_t kTileUnits = kTileBytes >> 4;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem;                     // [2] tiles
  uint8_t* s_ring = smem + 2 * kTileBytes;  // [kRing] tiles
  uint64_t* bars =
      reinterpret_cast<uint64_t*>(smem + (2 + kRing) * kTileBytes + 8 * 4096);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kNumBars);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int tid = threadIdx.x;
  const int warp = tid / 32;
  const int lane = tid % 32;
  const int64_t n_items = static_cast<int64_t>(p.entries) * p.kv_heads;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (tid == 0) {
    for (int b = 0; b < kNumBars; ++b) {
      uint32_t count = 1;
      if (b >= kPHalfA && b < kODone) count = 4;
      mbar_init(&bars[b], count);
    }
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

  if (warp >= kProducer) {
    // 3 warpgroups x 128 threads x 168 registers = 2 x 128 x 216 + 128 x 72.
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == kProducer) {
      // ---------------- TMA producer ----------------
      if (lane == 0) {
        prefetch_tensor_map(&map_q);
        prefetch_tensor_map(&map_k);
        prefetch_tensor_map(&map_v);
      }
      const uint32_t q_bytes = p.group * p.tokens * kD * 2;  // of a tile
      int n_ring = 0;
      int q_issued[2] = {0, 0};
      bool run = true;
      // One K or V tile (rows k_row ..) into the ring's next place.
      auto load = [&](const CUtensorMap* map, int h, int row) -> bool {
        const int slot = n_ring % kRing;
        if (n_ring >= kRing && !wait_all(&bars[kEmpty + slot],
                                         ((n_ring / kRing) - 1) & 1, abort,
                                         p.status))
          return false;
        if (lane == 0) {
          uint8_t* dst = s_ring + slot * kTileBytes;
          mbar_arrive_expect_tx(&bars[kFull + slot], kTileBytes);
#pragma unroll
          for (int c = 0; c < kD / 64; ++c)
            tma_load_3d(dst + c * 16384, map, &bars[kFull + slot], c * 64, h,
                        row);
        }
        __syncwarp();
        ++n_ring;
        return true;
      };
      // K0, V0, K1, V1, ..., or K0, K1, V0, K2, V1, ... (kAhead).
      Cursor c;
      c.init(p, n_items);
      [[maybe_unused]] int v_row = 0, v_head = 0;
      while (run && c.valid) {
        const int row = c.st.it.k_row + (c.st.it.first + c.j) * kTile;
        const int h = c.st.h;
        run = load(&map_k, h, row);
        // Q behind the item's first K tile: it has to wait for the last scores
        // of the item before.
        for (int g = 0; run && c.j == 0 && g < 2; ++g) {
          if (c.items > 0 && !wait_all(&bars[kQEmpty + g], (c.items - 1) & 1,
                                       abort, p.status)) {
            run = false;
            break;
          }
          if (lane == 0) {
            mbar_arrive_expect_tx(&bars[kQFull + g], q_bytes);
#pragma unroll
            for (int x = 0; x < kD / 64; ++x)
              tma_load_3d(s_q + g * kTileBytes + x * 16384, &map_q,
                          &bars[kQFull + g], x * 64, h * p.group,
                          c.st.it.row + g * p.tokens);
            q_issued[g] = c.items + 1;
          }
          __syncwarp();
        }
        if constexpr (C::kAhead) {
          if (run && c.b > 0) run = load(&map_v, v_head, v_row);
          v_row = row;
          v_head = h;
        } else {
          if (run) run = load(&map_v, h, row);
        }
        c.next(p, n_items);
      }
      if (C::kAhead && run && c.b > 0) run = load(&map_v, v_head, v_row);
      if (lane == 0 && *abort) {
        // Let the copies in flight land before the CTA retires.
        volatile int never = 0;
        for (int g = 0; g < 2; ++g)
          if (q_issued[g] > 0)
            mbar_wait(&bars[kQFull + g], (q_issued[g] - 1) & 1, &never,
                      nullptr);
        for (int k = n_ring - kRing; k < n_ring; ++k)
          if (k >= 0)
            mbar_wait(&bars[kFull + k % kRing], (k / kRing) & 1, &never,
                      nullptr);
      }
    } else if (warp == kMma) {
      // ---------------- the products ----------------
      constexpr uint32_t idesc_qk = idesc_bf16(128, 128, false, false);
      constexpr uint32_t idesc_pv = idesc_bf16(128, kD, false, true);
      const uint32_t q_lo = sw128_desc_lo(smem_u32(s_q), 16);
      const uint32_t k_lo = sw128_desc_lo(smem_u32(s_ring), 16);
      const uint32_t v_lo = sw128_desc_lo(smem_u32(s_ring), 16384);
      // K of block b lies at place 2b of the ring's sequence and V at 2b + 1;
      // with kAhead K at 2b - 1 (0 of the first) and V at 2b + 2 (2b + 1 of
      // the last).
      auto landed = [&](int place) -> bool {
        return wait_all(&bars[kFull + place % kRing], (place / kRing) & 1,
                        abort, p.status);
      };
      bool ok = true;
      if constexpr (C::kAhead) {
        // Scores of tile `qg` of the block at `qk`, then on to the next.
        Cursor pv;
        pv.init(p, n_items);
        Cursor qk = pv;
        int qg = 0;
        auto issue_qk = [&]() {
          if (!ok || !qk.valid) return;
          const int place =
              2 * qk.b - (qk.b > 0 ? 1 : 0);
          if (qg == 0) ok = landed(place);
          if (ok && qk.j == 0)
            ok = wait_all(&bars[kQFull + qg], qk.items & 1, abort, p.status);
          if (!ok) return;
          tc_fence_after();
          const int buf = (2 * qk.b + qg) % C::kSBufs;
          umma_ss_run<C::kSteps>(tmem + buf * 128, q_lo + qg * kTileUnits,
                                 k_lo + (place % kRing) * kTileUnits, idesc_qk);
          umma_commit_warp(&bars[kSFull + buf]);
          if (qk.last()) umma_commit_warp(&bars[kQEmpty + qg]);
          if (qg == 1) {
            umma_commit_warp(&bars[kEmpty + place % kRing]);
            qk.next(p, n_items);
          }
          qg ^= 1;
        };
#pragma unroll
        for (int i = 0; i < C::kSBufs; ++i) issue_qk();
        while (ok && pv.valid) {
          // (The scores are ahead of the products: is this the last block?)
          const bool end = !qk.valid && qk.b == pv.b + 1;
          const int place = 2 * pv.b + (end ? 1 : 2);
          const int slot = place % kRing;
          if (!landed(place)) {
            ok = false;
            break;
          }
          // Rows behind the sequence's last key take no part: a weight of 0
          // would not keep a NaN out.
          const int rows = pv.st.it.keys - (pv.st.it.first + pv.j) * kTile;
          if (rows < kTile)
            clear_rows<kD>(s_ring + slot * kTileBytes, rows, lane);
          const uint32_t bv = v_lo + slot * kTileUnits;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const uint32_t t_p = tmem + (2 * pv.b + g) % C::kSBufs * 128;
            const uint32_t t_o = tmem + C::kO + g * kD;
            const int p_bar = 2 * (pv.b & 1) + g;
            if (!wait_all(&bars[kPHalfA + p_bar], (pv.b >> 1) & 1, abort,
                          p.status)) {
              ok = false;
              break;
            }
            tc_fence_after();
            umma_ts_run<false>(t_o, t_p, bv, idesc_pv, pv.j > 0);
            if (!wait_all(&bars[kPHalfB + p_bar], (pv.b >> 1) & 1, abort,
                          p.status)) {
              ok = false;
              break;
            }
            tc_fence_after();
            umma_ts_run<false>(t_o, t_p + 32, bv + 512, idesc_pv, 1);
            if (pv.last()) umma_commit_warp(&bars[kODone + g]);
            umma_commit_warp(&bars[kPvDone + g]);
            issue_qk();
          }
          if (!ok) break;
          umma_commit_warp(&bars[kEmpty + slot]);
          pv.next(p, n_items);
        }
      } else {
        // (last: the item's last block.)
        auto issue_qk = [&](int b, int g, bool last) {
          const uint32_t a = q_lo + g * kTileUnits;
          const uint32_t bk = k_lo + ((2 * b) % kRing) * kTileUnits;
          umma_ss_run<C::kSteps>(tmem + g * 128, a, bk, idesc_qk);
          umma_commit_warp(&bars[kSFull + g]);
          if (last) umma_commit_warp(&bars[kQEmpty + g]);
          if (g == 1) umma_commit_warp(&bars[kEmpty + (2 * b) % kRing]);
        };
        Stream st{0};
        bool more = st.next(p, n_items, false);
        int b = 0, items = 0;
        if (more) {
          ok = landed(0);
          for (int g = 0; ok && g < 2; ++g) {
            ok = wait_all(&bars[kQFull + g], 0, abort, p.status);
            if (ok) {
              tc_fence_after();
              issue_qk(0, g, st.it.blocks == 1);
            }
          }
        }
        while (ok && more) {
          const int n = st.it.blocks;
          const int keys = st.it.keys - st.it.first * kTile;
          more = st.next(p, n_items, false);
          for (int j = 0; j < n; ++j, ++b) {
            const bool last = j == n - 1;
            const bool ahead = !last || more;
            const int slot = (2 * b + 1) % kRing;
            if (!landed(2 * b + 1)) {
              ok = false;
              break;
            }
            // Rows behind the sequence's last key take no part: a weight of 0
            // would not keep a NaN out.
            const int rows = keys - j * kTile;
            if (rows < kTile)
              clear_rows<kD>(s_ring + slot * kTileBytes, rows, lane);
            const uint32_t bv = v_lo + slot * kTileUnits;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const int p_bar = 2 * (b & 1) + g;
              if (!wait_all(&bars[kPHalfA + p_bar], (b >> 1) & 1, abort,
                            p.status)) {
                ok = false;
                break;
              }
              tc_fence_after();
              umma_ts_run<false>(tmem + C::kO + g * kD, tmem + g * 128, bv,
                                 idesc_pv, j > 0);
              if (!wait_all(&bars[kPHalfB + p_bar], (b >> 1) & 1, abort,
                            p.status)) {
                ok = false;
                break;
              }
              tc_fence_after();
              umma_ts_run<false>(tmem + C::kO + g * kD, tmem + g * 128 + 32,
                                 bv + 512, idesc_pv, 1);
              if (last) umma_commit_warp(&bars[kODone + g]);
              if (ahead) {
                if ((g == 0 && !landed(2 * b + 2)) ||
                    (last && !wait_all(&bars[kQFull + g], (items + 1) & 1,
                                       abort, p.status))) {
                  ok = false;
                  break;
                }
                tc_fence_after();
                issue_qk(b + 1, g, last ? st.it.blocks == 1 : j + 1 == n - 1);
              }
            }
            if (!ok) break;
            umma_commit_warp(&bars[kEmpty + slot]);
          }
          ++items;
        }
      }
      if (*abort) {
        volatile int never = 0;
        umma_commit_warp(&bars[kDrain]);
        mbar_wait(&bars[kDrain], 0, &never, nullptr);
      }
    }
  } else {
    // ---------------- softmax and epilogue (warps 0-7) ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int grp = warp / 4;
    const int quarter = warp % 4;
    const int row = quarter * 32 + lane;
    const int token = grp * p.tokens + row / p.group;  // of the item
    const int head = row % p.group;
    const bool row_used = row < p.tokens * p.group;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_o = tmem + C::kO + grp * kD + lane_base;
    uint8_t* s_stage = smem + (2 + kRing) * kTileBytes + warp * 4096;
    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
    uint32_t b = 0;
    int items = 0;
    bool ok = true;
    Stream st{0};
    while (ok && st.next(p, n_items, true)) {
      const int h = st.h;
      const ForwardItem it = st.it;
      const int n = it.blocks;
      // Keys of this row, from the item's first key tile on.
      const int seen = max(0, min(it.keys, it.kpos + token + 1)) -
                       it.first * kTile;
      float m_ref = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j, ++b) {
        const int visible = seen - j * kTile;
        const bool masked = __any_sync(0xffffffffu, visible < kTile);
        const uint32_t turn_s = 2 * b + grp;  // of the S buffers
        const uint32_t t_s =
            tmem + turn_s % C::kSBufs * 128 + lane_base;
        if (!wait_all(&bars[kSFull + turn_s % C::kSBufs],
                      (turn_s / C::kSBufs) & 1, abort, p.status)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t x[4][32];
        auto scores = [&](int q) { return reinterpret_cast<float*>(x[q]); };
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(t_s + q * 32, x[q]);
        tmem_wait_ld();
        if (masked) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int k = visible - q * 32;
            const uint32_t word =
                k >= 32 ? ~0u : (k <= 0 ? 0u : (1u << k) - 1u);
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (!((word >> c) & 1u)) scores(q)[c] = -INFINITY;
          }
        }
        float mx = row_max32(scores(0));
#pragma unroll
        for (int q = 1; q < 4; ++q) mx = fmaxf(mx, row_max32(scores(q)));
        const float mb = mx * p.scale_log2;
        const bool grow = mb > m_ref + 8.0f;
        if (j == 0) {
          m_ref = mb;
        } else if (__any_sync(0xffffffffu, grow)) {
          const float m_new = grow ? mb : m_ref;
          // A row without a key so far has an O of zeros.
          const float alpha =
              m_ref == -INFINITY ? 0.f : ex2_approx(m_ref - m_new);
          m_ref = m_new;
          // The previous blocks' products are in O: with two buffers they
          // were issued before this block's scores. This block's waits for P.
          if constexpr (C::kSBufs == 3) {
            if (!wait_all(&bars[kPvDone + grp], (b - 1) & 1, abort,
                          p.status)) {
              ok = false;
              break;
            }
            tc_fence_after();
          }
#pragma unroll 1
          for (int q16 = 0; q16 < kD / 16; ++q16)
            rescale16(t_o + q16 * 16, alpha);
          l *= alpha;
        }
        const float neg = m_ref == -INFINITY ? 0.f : -m_ref;
        const float2 negm2 = make_float2(neg, neg);
        float sum = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          sum += weights32(x[q], scores(q), scale2, negm2);
          tmem_st16(t_s + q * 16, x[q]);
          if (q & 1) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
              mbar_arrive(&bars[(q == 1 ? kPHalfA : kPHalfB) + 2 * (b & 1) +
                                grp]);
          }
        }
        l += sum;
      }
      if (!ok) break;
      // ---------------- epilogue ----------------
      const bool write = row_used && token < it.tokens;
      const int64_t out_row = static_cast<int64_t>(it.row) + token;
      const int64_t out_head = static_cast<int64_t>(h) * p.group + head;
      __nv_bfloat16* dst = p.out + out_row * p.out_st + out_head * p.out_sh;
      const float inv_l = l == 0.f ? 0.f : 1.0f / l;
      if (n > 0) {
        if (!wait_all(&bars[kODone + grp], items & 1, abort, p.status)) {
          ok = false;
          break;
        }
        tc_fence_after();
        ++items;
      }
      if (it.part >= 0) {
        // A part leaves its accumulator, maximum and sum to the join.
        const int64_t at =
            ((static_cast<int64_t>(h) * p.n_parts + it.part) * 2 + grp) *
                kTile +
            row;
        if (write) p.part_ml[at] = make_float2(m_ref, l);
#pragma unroll 1
        for (int c = 0; c < kD / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(t_o + c * 32, o);
          tmem_wait_ld();
          if (write) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              store32(p.part_o + at * kD + c * 32 + e * 8, o + e * 8);
          }
        }
      } else {
      // A warp whose rows all have tokens stages 64 columns at a time and
      // stores them by TMA; others store from registers, 32 rows at a time.
      const bool boxed =
          p.warp_boxes && __all_sync(0xffffffffu, write) && n > 0;
#pragma unroll 1
      for (int c = 0; c < kD / 64; ++c) {
        if (boxed) {
          if (lane == 0) bulk_wait_read();
          __syncwarp();
        }
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) {
          uint32_t o[32];
          if (n > 0) {
            tmem_ld32(t_o + c * 64 + c2 * 32, o);
            tmem_wait_ld();
          }
          if (l == 0.f) {  // no key
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0u;
          }
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e)
            w[e] = pack_bf16(__uint_as_float(o[2 * e]) * inv_l,
                             __uint_as_float(o[2 * e + 1]) * inv_l);
          if (boxed) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<uint4*>(
                  s_stage + lane * 128 +
                  (((c2 * 4 + e) ^ (lane & 7)) << 4)) =
                  make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2],
                             w[4 * e + 3]);
          } else if (write) {
            store32(dst + c * 64 + c2 * 32, w);
            store32(dst + c * 64 + c2 * 32 + 16, w + 8);
          }
          if (p.low != nullptr && write) {
            uint32_t low[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              uint32_t two[2];
#pragma unroll
              for (int i = 0; i < 2; ++i)
                two[i] = low_bits(__uint_as_float(o[4 * e + 2 * i]) * inv_l,
                                  __uint_as_float(o[4 * e + 2 * i + 1]) *
                                      inv_l,
                                  w[2 * e + i]);
              low[e] = __byte_perm(two[0], two[1], 0x6420);
            }
            store32(p.low + (out_row * p.kv_heads * p.group + out_head) * kD +
                        c * 64 + c2 * 32,
                    low);
          }
        }
        if (boxed) {
          fence_async_shared();
          __syncwarp();
          if (lane == 0)
            tma_store_3d(&map_out, s_stage, c * 64,
                         static_cast<int>(out_head), static_cast<int>(out_row));
        }
      }
      }
      tc_fence_before();  // O is read before P of the next item is released
      if (write && it.part < 0 && p.lse != nullptr)
        p.lse[out_row * p.lse_st + out_head * p.lse_sh] =
            l == 0.f ? -INFINITY : (m_ref + log2f(l)) * kLn2;
    }
    if (lane == 0) bulk_wait_read();  // the stores have read the stage
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Puts the parts of cut items together, in the order of the keys: a block per
// cut item, key head and 32 of the 256 rows, a warp a row, four parts' loads in
// flight.
constexpr int kJoinThreads = 512;
constexpr int kJoinRows = 32;

template <int kD>
__global__ void __launch_bounds__(kJoinThreads)
    causal_join_kernel(const __grid_constant__ FwdParams p) {
  constexpr int kPer = kD / 32;  // elements a lane
  constexpr int kBatch = 4;
  const JoinItem it = load_item<JoinItem>(p.joins, blockIdx.x);
  const int h = blockIdx.y, lane = threadIdx.x % 32;
  // The parts are written by the kernel that this one follows.
  asm volatile("griddepcontrol.wait;" ::: "memory");
#pragma unroll
  for (int i = 0; i < kJoinRows / (kJoinThreads / 32); ++i) {
    const int r = blockIdx.z * kJoinRows + i * (kJoinThreads / 32) +
                  threadIdx.x / 32;
    const int grp = r / kTile, row = r % kTile;
    const int token = grp * p.tokens + row / p.group;
    if (row >= p.tokens * p.group || token >= it.tokens) continue;
    const int64_t at0 =
        ((static_cast<int64_t>(h) * p.n_parts + it.part) * 2 + grp) * kTile +
        row;
    float m = -INFINITY, l = 0.f, o[kPer] = {};
    for (int base = 0; base < it.parts; base += kBatch) {
      float2 ml[kBatch];
      float x[kBatch][kPer];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        // (Past the last part: the last one again, with no weight.)
        const int part = min(base + b, it.parts - 1);
        const int64_t at = at0 + static_cast<int64_t>(part) * 2 * kTile;
        ml[b] = p.part_ml[at];
        const float* src = p.part_o + at * kD + lane * kPer;
#pragma unroll
        for (int e = 0; e < kPer; e += 2) {
          const float2 v = *reinterpret_cast<const float2*>(src + e);
          x[b][e] = v.x;
          x[b][e + 1] = v.y;
        }
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        // A part that the row sees nothing of has no weight either (and an
        // accumulator of zeros).
        if (base + b >= it.parts || ml[b].x == -INFINITY) continue;
        const float next = fmaxf(m, ml[b].x);
        const float f = ex2_approx(m - next), g = ex2_approx(ml[b].x - next);
        m = next;
        l = l * f + ml[b].y * g;
#pragma unroll
        for (int e = 0; e < kPer; ++e) o[e] = o[e] * f + x[b][e] * g;
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t out_row = static_cast<int64_t>(it.row) + token;
    const int64_t out_head =
        static_cast<int64_t>(h) * p.group + row % p.group;
    uint32_t* dst = reinterpret_cast<uint32_t*>(
        p.out + out_row * p.out_st + out_head * p.out_sh + lane * kPer);
    int8_t* low = p.low == nullptr
                      ? nullptr
                      : p.low + (out_row * p.kv_heads * p.group + out_head) *
                                    kD + lane * kPer;
#pragma unroll
    for (int e = 0; e < kPer / 2; ++e) {
      const float a = o[2 * e] * inv, b = o[2 * e + 1] * inv;
      dst[e] = pack_bf16(a, b);
      if (low != nullptr)
        reinterpret_cast<uint16_t*>(low)[e] = static_cast<uint16_t>(
            __byte_perm(low_bits(a, b, dst[e]), 0, 0x4420));
    }
    if (lane == 0 && p.lse != nullptr)
      p.lse[out_row * p.lse_st + out_head * p.lse_sh] =
          l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
  }
}

template <int kD>
int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
           const CUtensorMap& mo, const FwdParams& p, int64_t n_joins,
           cudaStream_t stream) {
  int sms = 0;
  int rc = device_sms(&sms);
  if (rc != VEDA_OK) return rc;
  static std::atomic<uint64_t> allowed{0};
  rc = allow_smem(reinterpret_cast<const void*>(causal_fwd_kernel<kD>),
                  Fwd<kD>::kSmem, &allowed);
  if (rc != VEDA_OK) return rc;
  const int cap = sms - sm_reserve() > 0 ? sms - sm_reserve() : 1;
  const int64_t items = static_cast<int64_t>(p.entries) * p.kv_heads;
  const int grid = static_cast<int>(items < cap ? items : cap);
  causal_fwd_kernel<kD><<<grid, 32 * kWarps, Fwd<kD>::kSmem, stream>>>(
      mq, mk, mv, mo, p);
  rc = check_launch("causal_fwd_kernel");
  if (rc != VEDA_OK || n_joins == 0) return rc;
  // The join starts while the last CTAs run (griddepcontrol).
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(n_joins), p.kv_heads,
                        2 * kTile / kJoinRows);
  config.blockDim = dim3(kJoinThreads);
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  VEDA_CUDA(cudaLaunchKernelEx(&config, causal_join_kernel<kD>, p));
  return check_launch("causal_join_kernel");
}

}  // namespace

}  // namespace causal
}  // namespace veda

using namespace veda;

extern "C" int64_t veda_causal_fwd_workspace(int32_t kv_heads,
                                             int32_t head_dim,
                                             int64_t n_parts) {
  if (kv_heads < 1 || (head_dim != 64 && head_dim != 128) || n_parts < 0 ||
      n_parts >= (int64_t(1) << 31))
    return -1;
  return static_cast<int64_t>(kv_heads) * n_parts * 2 * kTile *
         (head_dim + 2) * static_cast<int64_t>(sizeof(float));
}

extern "C" int veda_causal_fwd(
    const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k,
    int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
    int64_t v_stride_h, int64_t total_q, int64_t total_k, int32_t n_heads,
    int32_t kv_heads, int32_t head_dim, const int32_t* items, int64_t n_items,
    const int32_t* joins, int64_t n_joins, int64_t n_parts, void* out,
    int64_t out_stride_t, int64_t out_stride_h, void* out_low, float* lse,
    int64_t lse_stride_t, int64_t lse_stride_h, float softmax_scale,
    void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = require_sm100("veda_causal_fwd");
  if (rc != VEDA_OK) return rc;
  VEDA_REQUIRE(head_dim == 64 || head_dim == 128,
               "head_dim must be 64 or 128");
  VEDA_REQUIRE(kv_heads >= 1 && n_heads >= 1 && n_heads % kv_heads == 0 &&
                   n_heads / kv_heads <= kTile,
               "n_heads must be 1 to 128 times kv_heads");
  VEDA_REQUIRE(total_q >= 0 && total_k >= 0 && total_q < (int64_t(1) << 31) &&
                   total_k < (int64_t(1) << 31) && n_items >= 0 &&
                   n_items * kv_heads < (int64_t(1) << 31) - 65536,
               "bad sizes");
  VEDA_REQUIRE(softmax_scale > 0.f &&
                   isfinite(softmax_scale * causal::kLog2e),
               "softmax_scale must be positive and finite");
  if (total_q == 0 || n_items == 0) return VEDA_OK;
  VEDA_REQUIRE(q && out && items, "q, out and items are required");
  VEDA_REQUIRE(reinterpret_cast<uintptr_t>(out) % 32 == 0 &&
                   out_stride_t % 16 == 0 && out_stride_h % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(out_low) % 32 == 0 &&
                   reinterpret_cast<uintptr_t>(items) % 16 == 0,
               "out must be 32-byte aligned with strides multiple of 16, "
               "out_low 32-byte aligned, items 16-byte aligned");
  VEDA_REQUIRE(n_joins >= 0 && n_joins <= n_items && n_parts >= n_joins &&
                   n_parts <= n_items && kv_heads <= 65535 &&
                   (n_joins == 0) == (n_parts == 0) &&
                   (n_joins == 0 || joins != nullptr) &&
                   reinterpret_cast<uintptr_t>(joins) % 16 == 0,
               "the joins do not match the parts");
  const int64_t need = veda_causal_fwd_workspace(kv_heads, head_dim, n_parts);
  VEDA_REQUIRE(need >= 0 && workspace_bytes >= need &&
                   (need == 0 || workspace != nullptr) &&
                   reinterpret_cast<uintptr_t>(workspace) % 32 == 0,
               "workspace too small or not 32-byte aligned "
               "(veda_causal_fwd_workspace)");
  const int group = n_heads / kv_heads;
  const int tokens = kTile / group;
  CUtensorMap mq, mk, mv, mo;
  rc = causal::make_rows_map(&mq, q, total_q, n_heads, head_dim, q_stride_t,
                             q_stride_h, group, tokens, "q");
  const bool warp_boxes = 32 % group == 0;
  if (rc == VEDA_OK)
    rc = causal::make_rows_map(&mo, out, total_q, n_heads, head_dim,
                               out_stride_t, out_stride_h, group,
                               warp_boxes ? 32 / group : 1, "out");
  // Without keys no item loads any; the maps then only have to exist.
  if (total_k == 0) {
    mk = mv = mq;
  } else {
    VEDA_REQUIRE(k && v, "k and v are required");
    if (rc == VEDA_OK)
      rc = causal::make_rows_map(&mk, k, total_k, kv_heads, head_dim,
                                 k_stride_t, k_stride_h, 1, kTile, "k");
    if (rc == VEDA_OK)
      rc = causal::make_rows_map(&mv, v, total_k, kv_heads, head_dim,
                                 v_stride_t, v_stride_h, 1, kTile, "v");
  }
  if (rc != VEDA_OK) return rc;
  causal::FwdParams p{};
  p.table = items;
  p.entries = static_cast<int>(n_items);
  p.kv_heads = kv_heads;
  p.group = group;
  p.tokens = tokens;
  p.warp_boxes = warp_boxes;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_st = out_stride_t;
  p.out_sh = out_stride_h;
  p.low = static_cast<int8_t*>(out_low);
  p.lse = lse;
  p.lse_st = lse_stride_t;
  p.lse_sh = lse_stride_h;
  p.scale_log2 = softmax_scale * causal::kLog2e;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(
      p.part_o + static_cast<int64_t>(kv_heads) * n_parts * 2 * kTile *
                     head_dim);
  p.n_parts = static_cast<int>(n_parts);
  p.joins = joins;
  p.status = device_status_ptr();
  cudaStream_t s = as_stream(stream);
  return head_dim == 128 ? causal::launch<128>(mq, mk, mv, mo, p, n_joins, s)
                         : causal::launch<64>(mq, mk, mv, mo, p, n_joins, s);
}
