// Attention of one new token per sequence over the paged key-value cache,
// split over the cache's length and joined.
//
// For head h of a sequence with cached rows j < length, kv head h / group:
//     s_j = scale q_h . k_j,  out_h = sum_j softmax(s)_j v_j,
//     lse_h = log sum_j exp(s_j);  no rows: out 0, lse -inf.
//
// The cache is read once and each of its bytes meets all heads of a group,
// so the kernel is bound by memory. The heads of a group are the rows of
// m16n8k16 tensor-core products (a group of 16 or fewer is one tile, larger
// ones take several and find the rows in L2): tcgen05's 128 rows would leave
// seven eighths or more of them empty, and at the cache's rate the legacy
// products take a fraction of the time of its loads.
//
// The contexts of a call are cut into chunks of 16 keys of one kv head
// (a page holds a multiple of 16 rows, so a chunk is one contiguous piece),
// numbered sequence by sequence and head by head, and warp i of all W warps
// of the grid takes the i-th of W equal runs of the numbers, whatever the
// lengths: the split needs the lengths on the device only. A warp streams its
// run through a ring of its own with cp.async (rows past the length are
// filled with zeros, not read), a chunk a step (two with 8-bit pages at D =
// 64), with its own running maximum, sum and accumulator, and never waits for
// another warp. A
// (sequence, head) that lies inside the run is written out; the run's first
// and last may be parts, which the CTA adds up in shared memory at its end and,
// where they go on in another CTA, leaves in the workspace for
// decode_join_kernel, which starts while the last CTAs run. (The last CTA to
// arrive doing that, by a counter, took the smallest calls longer, 18 against
// 14 us on the device, and no less on the host.) Parts are added in the order
// of the keys, with no atomics: repeats are bit-identical.
//
// int8 and e4m3 codes become fp16 exactly, in registers. In the scores an int8
// code is the fp16 number (code + 128) 2^-24 (a subnormal: its bits are the
// byte), which takes an instruction and a half a pair, and 128 sum(q) comes out
// again: the sum is over D products, and what fp32 loses of it is lost once.
// The values' sums go over a whole run of keys, where the product's fp32
// additions, which do not round to nearest, lost bits of an ever larger sum of
// code + 128 at every step (64 contexts of 32,768 equally weighted rows, 8
// heads: 2.4e-2 of the result; of 8,192 rows: 2.8e-3). So a value's code is
// taken as 1024 + (code + 128), less 1152, an instruction more a pair (64 x
// 8,192 rows, 8 heads, D = 128: 222 us against 215). The order of d
// inside the first product and of the columns of the second is free, and is
// the one that the bytes of a word have. A key's scale multiplies its scores. A
// value row's scale multiplies its weights, and these products are taken
// relative to the largest of the head so far, so that they stay inside fp16 and
// what a row adds to the result, not its size, decides which bits it keeps
// (relative to the largest scale, a large row that nothing attends to cost all
// others theirs; 2 % of the time). q is brought to [1, 2) per head by a
// power of two, so it loses nothing in fp16 but elements 2^-14 below the
// head's largest. Scores, maxima, sums and accumulators are fp32; weights are
// rounded to the 16-bit type of the products (bf16 pages: bf16), as everywhere
// in this library.
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <math.h>

#include <type_traits>

#include "kvcache.cuh"

namespace veda {

namespace {

constexpr int kChunk = 16;  // keys
constexpr int kRows = 16;   // heads of a tile
constexpr int kJoinThreads = 512;
constexpr float kWeight = 64.f;  // factor of the fp16 weights
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;

struct DecodeParams {
  CacheView c;
  const __nv_bfloat16* q;
  int64_t q_sb, q_sh;
  const int32_t* lengths;
  int group;   // query heads of a kv head
  int tiles;   // tiles of kRows heads in a group
  __nv_bfloat16* out;  // [n_seqs, heads, D]
  float* lse;          // [n_seqs, heads] or null
  float* partial;      // [n_ctas][2][kRows][D + 2]
  int n_ctas;
  int warps;      // of a CTA
  float scale_log2;
  unsigned int* status;
};

// Rows of sequence b: its length, held inside what its table row addresses.
__device__ __forceinline__ int context(const DecodeParams& p, int b) {
  const int n = p.lengths[b];
  const int cap = p.c.max_pages << p.c.page_shift;
  return n < 0 ? 0 : (n > cap ? cap : n);
}

__device__ __forceinline__ int chunks_of(int length) {
  return (length + kChunk - 1) / kChunk;
}

// a / b for b >= 1, by the 32-bit quotient where that does (a 64-bit one is
// a few hundred cycles, and these are on the way to the first load).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 31) == 0)
    return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// [0, total) chunks in runs for the grid's warps: the first `extra` warps
// take size + 1, the others size. With more warps than chunks one for each
// chunk takes part, so that no run is empty.
struct Split {
  int64_t size;
  int extra;
  int warps;
  __device__ __forceinline__ Split(const DecodeParams& p, int64_t total) {
    const int all = p.n_ctas * p.warps;
    warps = total < all ? static_cast<int>(total) : all;
    size = warps > 0 ? quotient(total, warps) : 0;
    extra = static_cast<int>(total - size * warps);
  }
  __device__ __forceinline__ int64_t begin(int warp) const {
    return size * warp + min(warp, extra);
  }
  __device__ __forceinline__ int warp_of(int64_t chunk) const {
    const int64_t big = (size + 1) * extra;
    return static_cast<int>(chunk < big
                                ? quotient(chunk, size + 1)
                                : extra + quotient(chunk - big, size));
  }
};

// Exclusive prefix of x over the block's threads; *sum receives the total.
template <int kBlock>
__device__ __forceinline__ int64_t block_scan(int64_t* warp_sum, int64_t x,
                                              int64_t* sum) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int64_t inc = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  __syncthreads();
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  int64_t pre = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kBlock / 32; ++w) {
    const int64_t y = warp_sum[w];
    if (w < warp) pre += y;
    all += y;
  }
  *sum = all;
  return pre + inc - x;
}

// Where this warp's run begins: chunk numbers [*lo, *hi), the sequence of the
// first and the chunks before that sequence. `ends` holds kThreads numbers.
// Returns false for a warp without a run. All threads of the block call it.
template <int kThreads>
__device__ __forceinline__ bool find_run(const DecodeParams& p, int heads,
                                         int64_t* warp_sum, int64_t* ends,
                                         int64_t* lo, int64_t* hi, int* seq,
                                         int64_t* before) {
  const int n = p.c.n_seqs;
  const int tid = threadIdx.x, lane = tid % 32;
  const bool one_pass = n <= kThreads;
  int64_t mine = 0;
  for (int b = tid; b < n; b += kThreads) mine += chunks_of(context(p, b));
  mine *= heads;
  int64_t sum;
  int64_t pre = block_scan<kThreads>(warp_sum, mine, &sum);
  const Split split(p, sum);
  const int w = blockIdx.x * (kThreads / 32) + tid / 32;
  const bool run = w < split.warps;
  *lo = run ? split.begin(w) : 0;
  *hi = run ? split.begin(w + 1) : 0;
  *seq = -1;
  int64_t base = 0;
  for (int b0 = 0; b0 < n; b0 += kThreads) {
    if (!one_pass) {
      const int b = b0 + tid;
      mine = b < n ? chunks_of(context(p, b)) * static_cast<int64_t>(heads)
                   : int64_t(0);
      pre = base + block_scan<kThreads>(warp_sum, mine, &sum);
    }
    __syncthreads();
    ends[tid] = pre + mine;
    __syncthreads();
    if (run && *seq < 0 && *lo < ends[kThreads - 1]) {
      // The first sequence of the block that ends behind lo.
      for (int i = 0; i < kThreads; i += 32) {
        const unsigned hit =
            __ballot_sync(0xffffffffu, ends[i + lane] > *lo);
        if (hit != 0) {
          const int at = i + __ffs(hit) - 1;
          *seq = b0 + at;
          *before = at > 0 ? ends[at - 1] : base;
          break;
        }
      }
    }
    base += sum;
  }
  return run && *seq >= 0;
}

// The pieces of a warp's run: sequence, head tile, chunks [c0, c1).
struct Pieces {
  int b, vh, c0, c1, n;  // n: chunks of the whole (sequence, head)
  int length;
  int64_t left;  // chunks of the run from c0 on
  int heads;     // kv heads x tiles
  __device__ void bound() {
    const int64_t room = n - c0;
    c1 = c0 + static_cast<int>(left < room ? left : room);
  }
  __device__ bool valid() const { return left > 0; }
  __device__ void next(const DecodeParams& p) {
    left -= c1 - c0;
    c0 = 0;
    if (left <= 0) return;
    if (++vh == heads) {
      vh = 0;
      length = 0;
      while (length == 0 && ++b < p.c.n_seqs) length = context(p, b);
      n = chunks_of(length);
      if (n == 0) {  // not reached while the lengths stay as they are
        left = 0;
        return;
      }
    }
    bound();
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src,
                                           bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst),
               "l"(src), "r"(take ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src)
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src)
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src,
                                          bool take) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst),
               "l"(src), "r"(take ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int kLeft>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile(
      "ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t* r) {
  asm volatile(
      "ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(addr)
      : "memory");
}

__device__ __forceinline__ float2 lds64(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(addr)
               : "memory");
  return v;
}

// c[4] += A (16 x 16) . B (16 x 8), bf16 or fp16 in, fp32 accumulate.
template <bool kHalf>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a,
                                         uint32_t b0, uint32_t b1) {
  if constexpr (kHalf)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, "
        "%3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four int8 codes (bytes 0 .. 3 of a word) as two fp16 pairs of (code + 128)
// 2^-24: bytes 0 and 2, and bytes 1 and 3.
__device__ __forceinline__ void int8_offset_pairs(uint32_t w, uint32_t* even,
                                                  uint32_t* odd) {
  *even = (w ^ 0x00800080u) & 0x00ff00ffu;
  *odd = __byte_perm(w, 0, 0x4341) ^ 0x00800080u;
}

// Four codes as two fp16 pairs, exactly: bytes 0 and 2, and bytes 1 and 3.
template <int kStore>
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t* even,
                                              uint32_t* odd) {
  if constexpr (kStore == kStoreInt8) {
    const uint32_t x = (w & 0x00ff00ffu) ^ 0x64806480u;
    const uint32_t y = __byte_perm(w, 0x64646464u, 0x4341) ^ 0x00800080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480),
                                        __ushort_as_half(0x6480));  // 1152
    const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&x), bias);
    const __half2 b = __hsub2(*reinterpret_cast<const __half2*>(&y), bias);
    *even = *reinterpret_cast<const uint32_t*>(&a);
    *odd = *reinterpret_cast<const uint32_t*>(&b);
  } else {
    w = __byte_perm(w, 0, 0x3120);
    const __half2_raw x = __nv_cvt_fp8x2_to_halfraw2(
        static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3);
    const __half2_raw y = __nv_cvt_fp8x2_to_halfraw2(
        static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
    *even = static_cast<uint32_t>(x.x) | (static_cast<uint32_t>(x.y) << 16);
    *odd = static_cast<uint32_t>(y.x) | (static_cast<uint32_t>(y.y) << 16);
  }
}

// Bytes 0, 1 and bytes 2, 3 of a word of e4m3 codes (the K operand; no
// regrouping).
__device__ __forceinline__ void e4m3_pairs(uint32_t w, uint32_t* lo,
                                           uint32_t* hi) {
  const __half2_raw x = __nv_cvt_fp8x2_to_halfraw2(
      static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3);
  const __half2_raw y = __nv_cvt_fp8x2_to_halfraw2(
      static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
  *lo = static_cast<uint32_t>(x.x) | (static_cast<uint32_t>(x.y) << 16);
  *hi = static_cast<uint32_t>(y.x) | (static_cast<uint32_t>(y.y) << 16);
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <int kD, int kStore>
struct Shape {
  static constexpr bool kHalf = kStore != kStoreBf16;
  // Warps of a CTA (one a SM). Twelve warps of one chunk a step take less time
  // than eight of two with 8-bit pages at D = 128 (64 x 8,192 rows, 8 key
  // heads, groups of 4: int8 225 and 231 us, e4m3 240 and 258): converting
  // codes is what bounds both, at 76 and 71 % of the copy rate (bf16 pages:
  // 100 %).
  static constexpr int kWarps = kHalf && kD == 128 ? 12 : 8;
  static constexpr int kRowBytes = kHalf ? kD : 2 * kD;
  static constexpr int kTileBytes = kChunk * kRowBytes;  // k or v of a chunk
  // k, v, and (8-bit) 16 k scales and 16 v scales.
  static constexpr int kStageBytes = 2 * kTileBytes + (kHalf ? 128 : 0);
  static constexpr int kPieces = kRowBytes / 16;  // 16-byte pieces of a row
  // Chunks a step: two share the maxima and the loop's overhead.
  static constexpr int kPair = kHalf && kWarps == 8 ? 2 : 1;
  static constexpr int kJoinFloats = kD + 4;      // a row of the join buffer
};

// Byte offset of 16-byte piece `c` of row `r` of a k or v tile: the pieces
// are permuted within groups of eight rows so that ldmatrix, which reads the
// same piece of eight rows, meets all banks.
template <int kPieces>
__device__ __forceinline__ uint32_t piece_at(int r, int c) {
  if constexpr (kPieces >= 8)
    return (r * kPieces + (c ^ (r & 7))) * 16;
  else  // 64-byte rows: two rows make up 128 bytes
    return (r * kPieces + (c ^ ((r >> 1) & 3))) * 16;
}

// A part of a (sequence, head tile) that a warp leaves for its CTA.
struct Part {
  int b, vh;    // -1: none
  int starts;   // it holds the first chunk
  int ends;     // it holds the last chunk
};

// Shared memory behind the rings: every warp's first part (a last part lies
// in the warp's own ring, which is free by then).
template <int kD, int kStore>
__host__ __device__ constexpr int part_floats(int pitch) {
  return pitch * Shape<kD, kStore>::kJoinFloats;
}

template <int kD, int kStore, int kStages>
__global__ void __launch_bounds__(32 * Shape<kD, kStore>::kWarps, 1)
    decode_kernel(const __grid_constant__ DecodeParams p) {
  using S = Shape<kD, kStore>;
  constexpr bool kHalf = S::kHalf;
  constexpr int kWarps = S::kWarps;
  constexpr int kThreads = 32 * kWarps;
  constexpr int kSteps = kD / 16;
  constexpr int kRingBytes = kStages * S::kStageBytes;
  static_assert(kRingBytes >= kRows * S::kJoinFloats * 4,
                "a last part fits the ring");
  static_assert(kWarps * kRingBytes >= kThreads * 8, "find_run's numbers fit");
  static_assert(kStages <= 32, "a bit a stage");
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int64_t s_sums[kWarps];
  __shared__ Part s_parts[kWarps][2];
  __shared__ int s_list[2 * kWarps], s_open[2 * kWarps + 1], s_groups;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int quad = lane % 4, row_lo = lane / 4;  // fragment coordinates
  const int pitch = min(p.group, kRows);

  uint8_t* ring = smem + warp * kRingBytes;
  float* firsts = reinterpret_cast<float*>(smem + kWarps * kRingBytes);
  auto part_at = [&](int w, int slot) -> float* {
    return slot == 0 ? firsts + w * part_floats<kD, kStore>(pitch)
                     : reinterpret_cast<float*>(smem + w * kRingBytes);
  };

  // The join kernel may start; it waits for this grid's end before it reads.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int heads = p.c.kv_heads * p.tiles;
  if (blockIdx.x == 0) {
    // A length that its table row cannot hold is reported.
    const int64_t cap = static_cast<int64_t>(p.c.max_pages)
                        << p.c.page_shift;
    for (int b = threadIdx.x; b < p.c.n_seqs; b += kThreads)
      if (p.lengths[b] < 0 || p.lengths[b] > cap)
        raise_status(p.status, VEDA_ERR_INVALID);
  }
  if (lane < 2) s_parts[warp][lane].b = -1;
  int64_t lo, hi, before = 0;
  Pieces seg;
  seg.left = 0;
  if (find_run<kThreads>(p, heads, s_sums, reinterpret_cast<int64_t*>(smem),
                         &lo, &hi, &seg.b, &before)) {
    seg.length = context(p, seg.b);
    seg.n = chunks_of(seg.length);
    seg.heads = heads;
    if (seg.n > 0) {
      seg.vh = static_cast<int>(quotient(lo - before, seg.n));
      seg.c0 = static_cast<int>(lo - before -
                                static_cast<int64_t>(seg.vh) * seg.n);
      seg.left = hi - lo;
      seg.bound();
    }
  }
  __syncthreads();  // find_run's numbers lie in the rings

  // ---- loads: the run's chunks, piece after piece ----
  Pieces ld = seg;
  int ld_chunk = ld.c0;
  // The page of the next chunk is looked up one load ahead of its use.
  int next_page = -1;
  auto look_up = [&]() {
    if (ld.valid() && ld_chunk >= ld.c1) {
      ld.next(p);
      ld_chunk = ld.c0;
    }
    if (ld.valid())
      next_page = p.c.table[ld.b * p.c.table_ld +
                            ((ld_chunk * kChunk) >> p.c.page_shift)];
  };
  if (ld.valid()) look_up();
  int ld_stage = 0;
  // Stages of the ring whose chunk lies in a page that does not exist (a bit
  // each): its keys are absent, which only the scores' mask can tell from rows
  // of zeros.
  unsigned absent = 0;
  // This lane's 16-byte pieces of a tile are 512 bytes apart; where pieces move
  // with the row, every other one lies at the other side of bit 6.
  const uint32_t ring_at = smem_u32(ring);
  const uint32_t put = piece_at<S::kPieces>(lane / S::kPieces,
                                            lane % S::kPieces);
  auto put_at = [&](int i) -> uint32_t {
    const int r = i * (32 / S::kPieces);  // the rows' step
    if constexpr (S::kPieces >= 8)
      return (put ^ ((r & 7) * 16)) + i * 512;
    else
      return (put ^ (((r >> 1) & 3) * 16)) + i * 512;
  };
  auto load_next = [&]() {
    if (ld.valid()) {
      const int key0 = ld_chunk * kChunk;
      const bool ok = next_page >= 0 && next_page < p.c.n_pages;
      if (!ok && lane == 0) raise_status(p.status, VEDA_ERR_INVALID);
      absent = (absent & ~(1u << ld_stage)) |
               (static_cast<unsigned>(!ok) << ld_stage);
      // Rows of the chunk to load; the others become zeros.
      const int live = ok ? ld.length - key0 : 0;
      const int64_t row0 =
          ok ? (((static_cast<int64_t>(next_page) * p.c.kv_heads +
                  ld.vh / p.tiles)
                 << p.c.page_shift) +
                (key0 & ((1 << p.c.page_shift) - 1)))
             : 0;
      const uint32_t dst = ring_at + ld_stage * S::kStageBytes;
      const uint8_t* ksrc = p.c.k + row0 * S::kRowBytes + lane * 16;
      const uint8_t* vsrc = p.c.v + row0 * S::kRowBytes + lane * 16;
      const float* scales = nullptr;
      if constexpr (kHalf)
        scales = (lane < 16 ? p.c.k_scale : p.c.v_scale) + row0 + lane % 16;
      if (live >= kChunk) {
#pragma unroll
        for (int i = 0; i < kChunk * S::kPieces / 32; ++i) {
          cp_async16(dst + put_at(i), ksrc + i * 512);
          cp_async16(dst + S::kTileBytes + put_at(i), vsrc + i * 512);
        }
        if constexpr (kHalf)
          cp_async4(dst + 2 * S::kTileBytes + lane * 4, scales);
      } else {
#pragma unroll
        for (int i = 0; i < kChunk * S::kPieces / 32; ++i) {
          const int r = (i * 32 + lane) / S::kPieces;
          cp_async16(dst + put_at(i), ksrc + i * 512, r < live);
          cp_async16(dst + S::kTileBytes + put_at(i), vsrc + i * 512,
                     r < live);
        }
        if constexpr (kHalf)
          cp_async4(dst + 2 * S::kTileBytes + lane * 4, scales,
                    lane % 16 < live);
      }
      ++ld_chunk;
      look_up();
    }
    cp_async_commit();
    ld_stage = ld_stage + 1 == kStages ? 0 : ld_stage + 1;
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) load_next();

  int stage = 0;
  for (; seg.valid(); seg.next(p)) {
    const int kvh = seg.vh / p.tiles, tile = seg.vh % p.tiles;
    const int n_rows = min(kRows, p.group - tile * kRows);
    const int head0 = kvh * p.group + tile * kRows;
    // ---- q fragments of the piece's heads ----
    uint32_t qf[kSteps][4];
    float row_scale[2] = {p.scale_log2, p.scale_log2};
    [[maybe_unused]] float row_bias[2] = {0.f, 0.f};  // int8: the 128s'
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = row_lo + 8 * half;
      const __nv_bfloat16* src =
          p.q + seg.b * p.q_sb + (head0 + (r < n_rows ? r : 0)) * p.q_sh;
      if constexpr (!kHalf) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          qf[s][half] =
              *reinterpret_cast<const uint32_t*>(src + s * 16 + quad * 2);
          qf[s][half + 2] =
              *reinterpret_cast<const uint32_t*>(src + s * 16 + 8 + quad * 2);
        }
      } else {
        // The products' depth index runs over d in the order that a thread's
        // four consecutive code bytes give: int8 takes bytes 0, 2 and 1, 3
        // together, e4m3 bytes 0, 1 and 2, 3.
        float x[kSteps][4];
        float top = 0.f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const uint2 w =
              *reinterpret_cast<const uint2*>(src + s * 16 + quad * 4);
          x[s][0] = __uint_as_float(w.x << 16);
          x[s][1] = __uint_as_float(w.x & 0xFFFF0000u);
          x[s][2] = __uint_as_float(w.y << 16);
          x[s][3] = __uint_as_float(w.y & 0xFFFF0000u);
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(x[s][i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^e <= top < 2^(e+1), e held to [-126, 126] so that its inverse
        // exists.
        int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
        e = max(-126, min(126, e));
        const float inv =
            __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        row_scale[half] =
            p.scale_log2 *
            __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        if constexpr (kStore == kStoreInt8) {
          float sum = 0.f;
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            qf[s][half] = pack_half(x[s][0] * inv, x[s][2] * inv);
            qf[s][half + 2] = pack_half(x[s][1] * inv, x[s][3] * inv);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t w = qf[s][half + 2 * i];
              const float2 f =
                  __half22float2(*reinterpret_cast<const __half2*>(&w));
              sum += f.x + f.y;
            }
          }
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          row_bias[half] = -128.f * sum * row_scale[half];
          row_scale[half] *= 0x1p24f;
        } else {
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            qf[s][half] = pack_half(x[s][0] * inv, x[s][1] * inv);
            qf[s][half + 2] = pack_half(x[s][2] * inv, x[s][3] * inv);
          }
        }
      }
    }

    // ---- the piece's chunks, kPair a step ----
    // m: the rows' references (-inf before the first key), m_ref: the same or
    // 0. 8-bit pages: c_ref, the reference of weight times value scale (0
    // before the first key), and c_inv, kWeight over it; o is held in units of
    // c_ref / kWeight.
    float m[2] = {-INFINITY, -INFINITY}, m_ref[2] = {0.f, 0.f};
    float l[2] = {0.f, 0.f};
    [[maybe_unused]] float c_ref[2] = {0.f, 0.f}, c_inv[2] = {0.f, 0.f};
    float o[kD / 8][4];
#pragma unroll
    for (int i = 0; i < kD / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    // This lane's rows of the tiles that ldmatrix reads: in k, 16-byte pieces
    // lane / 8 + 0 .. 3 of key lane % 8; in v, piece lane / 16 of key lane %
    // 16. Further pieces differ in bits that only the exclusive or meets.
    const uint32_t k_get = piece_at<S::kPieces>(lane & 7, lane / 8);
    const uint32_t v_get =
        piece_at<S::kPieces>((lane & 7) + ((lane >> 3) & 1) * 8, lane / 16);
    constexpr uint32_t kEight = 8 * S::kRowBytes;  // eight keys on
    // kN chunks (1 or kPair) from `chunk` on.
    auto step = [&](auto count, int chunk) {
      constexpr int kN = decltype(count)::value;
      cp_async_wait<kStages - 1 - kN>();
      __syncwarp();
      uint32_t base[kN];
      int live[kN];  // keys of each chunk that exist (16 and more: all)
      bool whole = true;
#pragma unroll
      for (int u = 0; u < kN; ++u) {
        base[u] = ring_at + stage * S::kStageBytes;
        live[u] = (absent >> stage) & 1u
                      ? 0
                      : seg.length - (chunk + u) * kChunk;
        whole &= live[u] >= kChunk;
        stage = stage + 1 == kStages ? 0 : stage + 1;
      }
      // The chunks have landed, and the whole warp has read the stages before
      // them: the first of those takes the next load.
      load_next();

      // Scores: [16 heads] x [2 kN x 8 keys].
      float s[2 * kN][4] = {};
#pragma unroll
      for (int nt = 0; nt < 2 * kN; ++nt) {
        const uint32_t at = base[nt / 2] + k_get;
#pragma unroll
        for (int pc = 0; pc < S::kPieces; pc += 4) {
          uint32_t b[4];
          ldsm4((at ^ (pc * 16)) + (nt & 1) * kEight, b);
          if constexpr (!kHalf) {
            mma16816<false>(s[nt], qf[pc / 2], b[0], b[1]);
            mma16816<false>(s[nt], qf[pc / 2 + 1], b[2], b[3]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t b0, b1;
              if constexpr (kStore == kStoreInt8)
                int8_offset_pairs(b[i], &b0, &b1);
              else
                e4m3_pairs(b[i], &b0, &b1);
              mma16816<true>(s[nt], qf[pc + i], b0, b1);
            }
          }
        }
      }
      // Columns of this thread: keys 2 quad + {0, 1} of each tile of 8.
      float top[2] = {-INFINITY, -INFINITY};
      [[maybe_unused]] float v_top = 0.f;
      [[maybe_unused]] float2 vs[2 * kN];
#pragma unroll
      for (int nt = 0; nt < 2 * kN; ++nt) {
        float2 ks = make_float2(1.f, 1.f);
        if constexpr (kHalf) {
          const uint32_t at = base[nt / 2] + 2 * S::kTileBytes +
                              (nt & 1) * 32 + quad * 8;
          ks = lds64(at);
          vs[nt] = lds64(at + 64);
          v_top = fmaxf(v_top, fmaxf(fabsf(vs[nt].x), fabsf(vs[nt].y)));
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float& a = s[nt][2 * half];
          float& b = s[nt][2 * half + 1];
          if constexpr (kStore == kStoreInt8) {
            a = fmaf(a, row_scale[half], row_bias[half]) * ks.x;
            b = fmaf(b, row_scale[half], row_bias[half]) * ks.y;
          } else if constexpr (kHalf) {
            a *= row_scale[half] * ks.x;
            b *= row_scale[half] * ks.y;
          } else {
            a *= row_scale[half];
            b *= row_scale[half];
          }
        }
        if (!whole) {
          const int key = (nt & 1) * 8 + quad * 2;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (key >= live[nt / 2]) s[nt][2 * half] = -INFINITY;
            if (key + 1 >= live[nt / 2]) s[nt][2 * half + 1] = -INFINITY;
          }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
          top[half] = fmaxf(top[half],
                            fmaxf(s[nt][2 * half], s[nt][2 * half + 1]));
      }
      // The references move only when they must. That of the weights: when a
      // score is more than 2^8 above it (bf16), or above it at all (8-bit,
      // where it is put 2^8 above the maximum, so that a weight times any value
      // scale is finite). That of weights times scales: when one may be more
      // than 2^9 above it, so that the fp16 weights, with a factor 2^6
      // (kWeight), stay below 2^15; those down to 2^-20 of it keep all of
      // fp16's bits. (Maxima over a row's four threads, and of the products
      // themselves, are taken only then.)
      constexpr float kAbove = kHalf ? 8.f : 0.f;
      constexpr float kSlack = 8.f - kAbove;
      bool grow = top[0] > m[0] + kSlack || top[1] > m[1] + kSlack;
      if constexpr (kHalf)
        grow = grow ||
               ex2_approx(top[0] - m_ref[0]) * v_top > 512.f * c_ref[0] ||
               ex2_approx(top[1] - m_ref[1]) * v_top > 512.f * c_ref[1];
      if (__any_sync(0xffffffffu, grow)) {
        float f[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float x = top[half];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
          if (kHalf && !(x > m[half])) {
            f[half] = 1.f;
          } else {
            const float next = fmaxf(m[half], x + kAbove);
            f[half] = m[half] == -INFINITY ? 0.f : ex2_approx(m[half] - next);
            m[half] = next;
            // m is -inf where no key of the row has existed so far.
            m_ref[half] = next == -INFINITY ? 0.f : next;
            l[half] *= f[half];
          }
          if constexpr (kHalf) {
            // What o holds keeps its unit, which shrinks with the weights, and
            // goes over to the new one.
            float c = 0.f;
#pragma unroll
            for (int nt = 0; nt < 2 * kN; ++nt)
              c = fmaxf(c, fmaxf(ex2_approx(s[nt][2 * half] - m_ref[half]) *
                                     fabsf(vs[nt].x),
                                 ex2_approx(s[nt][2 * half + 1] -
                                            m_ref[half]) *
                                     fabsf(vs[nt].y)));
            c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, 1));
            c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, 2));
            const float held = c_ref[half] * f[half];
            // (Above 2^-100: its inverse exists.)
            c_ref[half] = fmaxf(fmaxf(held, c), 0x1p-100f);
            c_inv[half] = kWeight / c_ref[half];
            f[half] = held / c_ref[half];
          }
        }
#pragma unroll
        for (int i = 0; i < kD / 8; ++i) {
          o[i][0] *= f[0];
          o[i][1] *= f[0];
          o[i][2] *= f[1];
          o[i][3] *= f[1];
        }
      }
      // Weights, as the A operand of the second product.
      uint32_t a[kN][4];
#pragma unroll
      for (int nt = 0; nt < 2 * kN; ++nt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float p0 = ex2_approx(s[nt][2 * half] - m_ref[half]);
          const float p1 = ex2_approx(s[nt][2 * half + 1] - m_ref[half]);
          l[half] += p0 + p1;
          if constexpr (kHalf)
            a[nt / 2][(nt & 1) * 2 + half] =
                pack_half(p0 * vs[nt].x * c_inv[half],
                          p1 * vs[nt].y * c_inv[half]);
          else
            a[nt / 2][(nt & 1) * 2 + half] = pack_bf16(p0, p1);
        }
      // O += P V.
#pragma unroll
      for (int u = 0; u < kN; ++u) {
        const uint32_t at = base[u] + S::kTileBytes + v_get;
#pragma unroll
        for (int pc = 0; pc < S::kPieces; pc += 2) {
          uint32_t b[4];
          ldsm4_trans(at ^ (pc * 16), b);
          if constexpr (!kHalf) {
            mma16816<false>(o[pc], a[u], b[0], b[1]);
            mma16816<false>(o[pc + 1], a[u], b[2], b[3]);
          } else {
            // A 16-byte piece of a row is 16 d: column n of the even tile is
            // d = 2 n, of the odd tile 2 n + 1.
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t even0, odd0, even1, odd1;
              codes_to_half<kStore>(b[2 * i], &even0, &odd0);
              codes_to_half<kStore>(b[2 * i + 1], &even1, &odd1);
              mma16816<true>(o[2 * (pc + i)], a[u], even0, even1);
              mma16816<true>(o[2 * (pc + i) + 1], a[u], odd0, odd1);
            }
          }
        }
      }
      // The other stages of this step are free once the warp has read them.
      if constexpr (kN > 1) {
        __syncwarp();
#pragma unroll
        for (int u = 1; u < kN; ++u) load_next();
      }
    };
    int chunk = seg.c0;
    if constexpr (S::kPair == 2)
      for (; chunk + 2 <= seg.c1; chunk += 2)
        step(std::integral_constant<int, 2>{}, chunk);
    for (; chunk < seg.c1; ++chunk)
      step(std::integral_constant<int, 1>{}, chunk);

    // ---- the piece's end ----
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
      l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
    }
    const float unit[2] = {kHalf ? c_ref[0] * (1.f / kWeight) : 1.f,
                           kHalf ? c_ref[1] * (1.f / kWeight) : 1.f};
    const bool starts = seg.c0 == 0, ends = seg.c1 == seg.n;
    const int slot = starts ? 1 : 0;
    if (!(starts && ends)) {
      if (slot == 1) {
        // The run's last piece: the ring is empty, but another lane may still
        // read it.
        cp_async_wait<0>();
        __syncwarp();
      }
      if (lane == 0) s_parts[warp][slot] = Part{seg.b, seg.vh, starts, ends};
    }
    float* part = part_at(warp, slot);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = row_lo + 8 * half;
      if (r >= n_rows) continue;
      const int64_t at =
          static_cast<int64_t>(seg.b) * (p.c.kv_heads * p.group) + head0 + r;
      if (starts && ends) {
        const float inv = l[half] == 0.f ? 0.f : unit[half] / l[half];
        __nv_bfloat16* dst = p.out + at * kD;
#pragma unroll
        for (int dt = 0; dt < kD / 8; dt += 2) {
          const float a0 = o[dt][2 * half] * inv;
          const float a1 = o[dt][2 * half + 1] * inv;
          const float b0 = o[dt + 1][2 * half] * inv;
          const float b1 = o[dt + 1][2 * half + 1] * inv;
          if constexpr (!kHalf) {
            *reinterpret_cast<uint32_t*>(dst + dt * 8 + quad * 2) =
                pack_bf16(a0, a1);
            *reinterpret_cast<uint32_t*>(dst + dt * 8 + 8 + quad * 2) =
                pack_bf16(b0, b1);
          } else {
            *reinterpret_cast<uint2*>(dst + dt * 8 + quad * 4) =
                make_uint2(pack_bf16(a0, b0), pack_bf16(a1, b1));
          }
        }
        if (quad == 0 && p.lse != nullptr)
          p.lse[at] = (m[half] + log2f(l[half])) * kLn2;
      } else {
        float* dst = part + r * S::kJoinFloats;
        if (quad == 0) {
          dst[kD] = m[half];
          dst[kD + 1] = l[half];
        }
#pragma unroll
        for (int dt = 0; dt < kD / 8; dt += 2) {
          const float a0 = o[dt][2 * half] * unit[half];
          const float a1 = o[dt][2 * half + 1] * unit[half];
          const float b0 = o[dt + 1][2 * half] * unit[half];
          const float b1 = o[dt + 1][2 * half + 1] * unit[half];
          if constexpr (!kHalf) {
            *reinterpret_cast<float2*>(dst + dt * 8 + quad * 2) =
                make_float2(a0, a1);
            *reinterpret_cast<float2*>(dst + dt * 8 + 8 + quad * 2) =
                make_float2(b0, b1);
          } else {
            *reinterpret_cast<float4*>(dst + dt * 8 + quad * 4) =
                make_float4(a0, b0, a1, b1);
          }
        }
      }
    }
  }

  // ---- add up the CTA's parts in the order of the keys ----
  // Warp 0 lists the parts that there are (part number 2 * warp + slot) and
  // where each (sequence, head tile)'s begin in the list.
  __syncthreads();
  if (warp == 0) {
    Part x = Part{-1, 0, 0, 0};
    if (lane < 2 * kWarps) x = s_parts[lane / 2][lane % 2];
    const unsigned there = __ballot_sync(0xffffffffu, x.b >= 0);
    const unsigned below = there & ((1u << lane) - 1);
    const int prev = below != 0 ? 31 - __clz(below) : lane;
    const int pb = __shfl_sync(0xffffffffu, x.b, prev);
    const int pv = __shfl_sync(0xffffffffu, x.vh, prev);
    const bool opens =
        x.b >= 0 && (below == 0 || pb != x.b || pv != x.vh);
    const unsigned open = __ballot_sync(0xffffffffu, opens);
    if (x.b >= 0) s_list[__popc(below)] = lane;
    if (opens)
      s_open[__popc(open & ((1u << lane) - 1))] = __popc(below);
    if (lane == 0) {
      s_open[__popc(open)] = __popc(there);
      s_groups = __popc(open);
    }
  }
  __syncthreads();
  const int per_group = pitch * (kD / 2);
  for (int i = threadIdx.x; i < s_groups * per_group; i += kThreads) {
    const int g = i / per_group, r = i % per_group / (kD / 2);
    const int d = i % (kD / 2) * 2;
    const int first = s_open[g], end = s_open[g + 1];
    const int f0 = s_list[first], f1 = s_list[end - 1];
    const Part head = s_parts[f0 / 2][f0 % 2];
    const int kvh = head.vh / p.tiles, tile = head.vh % p.tiles;
    if (r >= min(kRows, p.group - tile * kRows)) continue;
    float top = -INFINITY;
    for (int w = first; w < end; ++w) {
      const int at = s_list[w];
      top = fmaxf(top, part_at(at / 2, at % 2)[r * S::kJoinFloats + kD]);
    }
    const float ref = top == -INFINITY ? 0.f : top;
    float x = 0.f, y = 0.f, sum = 0.f;
#pragma unroll 4
    for (int w = first; w < end; ++w) {
      const int at = s_list[w];
      const float* src = part_at(at / 2, at % 2) + r * S::kJoinFloats;
      const float f = ex2_approx(src[kD] - ref);
      const float2 ow = *reinterpret_cast<const float2*>(src + d);
      x = fmaf(f, ow.x, x);
      y = fmaf(f, ow.y, y);
      sum = fmaf(f, src[kD + 1], sum);
    }
    if (head.starts && s_parts[f1 / 2][f1 % 2].ends) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int64_t at =
          static_cast<int64_t>(head.b) * (p.c.kv_heads * p.group) +
          kvh * p.group + tile * kRows + r;
      *reinterpret_cast<uint32_t*>(p.out + at * kD + d) =
          pack_bf16(x * inv, y * inv);
      if (d == 0 && p.lse != nullptr)
        p.lse[at] = (top + log2f(sum)) * kLn2;
    } else {
      // One that an earlier CTA began (slot 0), or one that this CTA begins
      // (slot 1): at most one of each goes on elsewhere.
      float* dst = p.partial +
                   ((static_cast<int64_t>(blockIdx.x) * 2 + head.starts) *
                        kRows +
                    r) *
                       (kD + 2);
      *reinterpret_cast<float2*>(dst + d) = make_float2(x, y);
      if (d == 0) {
        dst[kD] = top;
        dst[kD + 1] = sum;
      }
    }
  }
}

// Adds up the parts of the (sequence, head tile)s that several CTAs share, in
// the order of the keys, and writes the rows of empty sequences. Block i takes
// the head tile, if there is one, that goes on from CTA i (where it begins) to
// CTA i + 1.
template <int kD>
__global__ void __launch_bounds__(kJoinThreads)
    decode_join_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int kPer = kD / 32;  // elements a lane
  __shared__ int64_t sums[kJoinThreads / 32];
  __shared__ float tops[kJoinThreads / 32], totals[kJoinThreads / 32];
  __shared__ float rows[kJoinThreads / 32][kD];
  __shared__ int s_seq;
  __shared__ int64_t s_before;
  const int heads = p.c.kv_heads * p.tiles;
  const int all_heads = p.c.kv_heads * p.group;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int64_t total = 0;
  for (int i = threadIdx.x; i < p.c.n_seqs; i += kJoinThreads)
    total += chunks_of(context(p, i));
  {
    int64_t sum;
    block_scan<kJoinThreads>(sums, total * heads, &sum);
    total = sum;
  }
  const Split split(p, total);
  // The first chunk of CTA i + 1, and the sequence it lies in.
  const int next_warp = (static_cast<int>(blockIdx.x) + 1) * p.warps;
  const int64_t at = next_warp < split.warps ? split.begin(next_warp) : total;
  if (threadIdx.x == 0) s_seq = -1;
  int64_t base = 0;
  for (int b0 = 0; b0 < p.c.n_seqs; b0 += kJoinThreads) {
    const int b = b0 + threadIdx.x;
    const int64_t n =
        b < p.c.n_seqs ? chunks_of(context(p, b)) * static_cast<int64_t>(heads)
                       : int64_t(0);
    int64_t sum;
    const int64_t pre = base + block_scan<kJoinThreads>(sums, n, &sum);
    if (pre <= at && at < pre + n) {
      s_seq = b;
      s_before = pre;
    }
    base += sum;
  }
  __syncthreads();
  // Every block waits, so that this grid ends after the one it follows.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // Rows of empty sequences, a sequence a block at a time.
  for (int b = blockIdx.x; b < p.c.n_seqs; b += gridDim.x) {
    if (context(p, b) > 0) continue;
    const int64_t first = static_cast<int64_t>(b) * all_heads;
    for (int i = threadIdx.x; i < all_heads * (kD / 2); i += kJoinThreads)
      reinterpret_cast<uint32_t*>(p.out + first * kD)[i] = 0u;
    if (p.lse != nullptr)
      for (int i = threadIdx.x; i < all_heads; i += kJoinThreads)
        p.lse[first + i] = -INFINITY;
  }
  const int b = s_seq;
  if (b < 0) return;  // CTA i + 1 has no chunks
  const int n = chunks_of(context(p, b));
  const int vh = static_cast<int>(quotient(at - s_before, n));
  const int64_t first = s_before + static_cast<int64_t>(vh) * n;
  const int c0 = split.warp_of(first) / p.warps;
  const int c1 = split.warp_of(first + n - 1) / p.warps;
  // It begins at CTA i + 1 itself, or began before CTA i.
  if (c0 != static_cast<int>(blockIdx.x)) return;
  const int kvh = vh / p.tiles, tile = vh % p.tiles;
  const int n_rows = min(kRows, p.group - tile * kRows);
  const int64_t at0 = static_cast<int64_t>(b) * all_heads + kvh * p.group +
                      tile * kRows;
  // `ways` warps a row, every ways-th part each, then added up.
  constexpr int kBatch = 4;
  const int ways = min(kJoinThreads / 32 / n_rows, c1 - c0 + 1);
  const int r = warp % n_rows, way = warp / n_rows;
  float top = -INFINITY, sum = 0.f, acc[kPer] = {};
  if (way < ways) {
    for (int base = c0 + way; base <= c1; base += ways * kBatch) {
      float m[kBatch], l[kBatch], x[kBatch][kPer];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int c = base + i * ways;
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[i][e] = 0.f;
        if (c > c1) continue;
        const float* src =
            p.partial + ((static_cast<int64_t>(c) * 2 + (c == c0 ? 1 : 0)) *
                             kRows +
                         r) *
                            (kD + 2);
        m[i] = src[kD];
        l[i] = src[kD + 1];
#pragma unroll
        for (int e = 0; e < kPer; e += 2) {
          const float2 v =
              *reinterpret_cast<const float2*>(src + lane * kPer + e);
          x[i][e] = v.x;
          x[i][e + 1] = v.y;
        }
      }
      float next = top;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) next = fmaxf(next, m[i]);
      const float ref = next == -INFINITY ? 0.f : next;
      const float f = ex2_approx(top - ref);
      top = next;
      sum *= f;
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] *= f;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float g = ex2_approx(m[i] - ref);
        sum = fmaf(g, l[i], sum);
#pragma unroll
        for (int e = 0; e < kPer; ++e) acc[e] = fmaf(g, x[i][e], acc[e]);
      }
    }
    if (lane == 0) {
      tops[warp] = top;
      totals[warp] = sum;
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) rows[warp][lane * kPer + e] = acc[e];
  }
  __syncthreads();
  if (way != 0) return;
  float all = -INFINITY;
  for (int w = 0; w < ways; ++w) all = fmaxf(all, tops[r + w * n_rows]);
  const float ref = all == -INFINITY ? 0.f : all;
  sum = 0.f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
  for (int w = 0; w < ways; ++w) {
    const int at = r + w * n_rows;
    const float g = ex2_approx(tops[at] - ref);
    sum = fmaf(g, totals[at], sum);
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      acc[e] = fmaf(g, rows[at][lane * kPer + e], acc[e]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint32_t* dst =
      reinterpret_cast<uint32_t*>(p.out + (at0 + r) * kD + lane * kPer);
#pragma unroll
  for (int e = 0; e < kPer / 2; ++e)
    dst[e] = pack_bf16(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  if (lane == 0 && p.lse != nullptr)
    p.lse[at0 + r] = (all + log2f(sum)) * kLn2;
}

// kPitch: the heads of a tile, at most.
template <int kD, int kStore, int kStages, int kPitch>
int launch(DecodeParams p, cudaStream_t stream) {
  using S = Shape<kD, kStore>;
  constexpr int kSmem = S::kWarps * (kStages * S::kStageBytes +
                                     part_floats<kD, kStore>(kPitch) * 4);
  static_assert(kSmem <= 226 * 1024, "beside the static part");
  p.warps = S::kWarps;
  static std::atomic<uint64_t> allowed{0};
  int rc = allow_smem(
      reinterpret_cast<const void*>(decode_kernel<kD, kStore, kStages>),
      kSmem, &allowed);
  if (rc != VEDA_OK) return rc;
  decode_kernel<kD, kStore, kStages>
      <<<p.n_ctas, 32 * S::kWarps, kSmem, stream>>>(p);
  rc = check_launch("decode_kernel");
  if (rc != VEDA_OK) return rc;
  // The join starts while the last CTAs run (griddepcontrol).
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(p.n_ctas));
  config.blockDim = dim3(kJoinThreads);
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  VEDA_CUDA(cudaLaunchKernelEx(&config, decode_join_kernel<kD>, p));
  return check_launch("decode_join_kernel");
}

// Depth of the ring, beside the buffer of parts, whose rows are the group's
// heads (16 at most). D = 64 and 8-bit pages: as deep as shared memory allows,
// which at D = 128 are three stages with parts of 8 rows and two with parts of
// 16. The buffer is therefore cut to the group where that gives the third stage
// (64 x 8,192 rows, 8 key heads, D = 128; three stages against two: int8 232 us
// against 239-246 for groups of 8 and the same for 4, e4m3 240 against 244 for
// 4). bf16 pages at D = 128 need two (321 us against 329 with three for
// groups of 4, 328 and 334 for 8; 128 x 300 rows 43 and 42).
template <int kD, int kStore>
int launch_stages(const DecodeParams& p, cudaStream_t stream) {
  if constexpr (kD == 64) {
    return launch<kD, kStore, kStore == kStoreBf16 ? 5 : 8, kRows>(p, stream);
  } else if constexpr (kStore == kStoreBf16) {
    return launch<kD, kStore, 2, kRows>(p, stream);
  } else {
    return p.group <= 8 ? launch<kD, kStore, 3, 8>(p, stream)
                        : launch<kD, kStore, 2, kRows>(p, stream);
  }
}

}  // namespace

}  // namespace veda

using namespace veda;

extern "C" int64_t veda_decode_workspace(int32_t head_dim) {
  if (head_dim != 64 && head_dim != 128) return -1;
  int sms = 0;
  if (device_sms(&sms) != VEDA_OK) return -1;
  return static_cast<int64_t>(sms) * 2 * kRows * (head_dim + 2) *
         static_cast<int64_t>(sizeof(float));
}

extern "C" int veda_decode(
    const void* k_pages, const void* v_pages, const float* k_scale,
    const float* v_scale, int64_t n_pages, int32_t page_size, int32_t kv_heads,
    int32_t head_dim, int32_t storage, const int32_t* table, int64_t table_ld,
    int64_t max_pages, int64_t n_seqs, const int32_t* lengths, const void* q,
    int64_t q_stride_b, int64_t q_stride_h, int32_t n_heads, void* out,
    float* lse, float softmax_scale, void* workspace, int64_t workspace_bytes,
    void* stream) {
  int rc = require_sm100("veda_decode");
  if (rc != VEDA_OK) return rc;
  DecodeParams p{};
  rc = make_cache_view(&p.c, const_cast<void*>(k_pages),
                       const_cast<void*>(v_pages),
                       const_cast<float*>(k_scale),
                       const_cast<float*>(v_scale), n_pages, page_size,
                       kv_heads, head_dim, storage, table, table_ld, max_pages,
                       n_seqs);
  if (rc != VEDA_OK) return rc;
  VEDA_REQUIRE(lengths && q && out && workspace,
               "lengths, q, out and workspace are required");
  VEDA_REQUIRE(n_heads >= 1 && n_heads % kv_heads == 0,
               "n_heads must be a multiple of kv_heads");
  VEDA_REQUIRE(n_seqs * n_heads < (int64_t(1) << 31), "too many rows");
  VEDA_REQUIRE(softmax_scale > 0.f && isfinite(softmax_scale * kLog2e),
               "softmax_scale must be positive and finite");
  VEDA_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 &&
                   q_stride_b % 8 == 0 && q_stride_h % 8 == 0 &&
                   reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               "q, out and workspace must be 16-byte aligned, q's strides "
               "multiples of 8");
  const int64_t need = veda_decode_workspace(head_dim);
  VEDA_REQUIRE(need > 0 && workspace_bytes >= need,
               "workspace too small (veda_decode_workspace)");
  rc = device_sms(&p.n_ctas);
  if (rc != VEDA_OK) return rc;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_sb = q_stride_b;
  p.q_sh = q_stride_h;
  p.lengths = lengths;
  p.group = n_heads / kv_heads;
  p.tiles = (p.group + kRows - 1) / kRows;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.partial = static_cast<float*>(workspace);
  p.scale_log2 = softmax_scale * kLog2e;
  p.status = device_status_ptr();
  cudaStream_t s = as_stream(stream);
  if (head_dim == 128) {
    if (storage == kStoreBf16) return launch_stages<128, kStoreBf16>(p, s);
    if (storage == kStoreInt8) return launch_stages<128, kStoreInt8>(p, s);
    return launch_stages<128, kStoreE4m3>(p, s);
  }
  if (storage == kStoreBf16) return launch_stages<64, kStoreBf16>(p, s);
  if (storage == kStoreInt8) return launch_stages<64, kStoreInt8>(p, s);
  return launch_stages<64, kStoreE4m3>(p, s);
}
