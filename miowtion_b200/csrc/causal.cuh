// Causal attention of packed sequences: the work items and helpers shared by
// the forward (causal_fwd.cu) and the backward (causal_bwd.cu).
//
// Grouped heads are folded into the rows of a query tile: with g query heads
// per key head a tile is floor(128 / g) tokens of one sequence times the g
// heads of one key head, token-major, so that a TMA box (64 columns, g heads,
// tokens) lands in shared memory as the tile's rows and every key and value
// tile read meets all g heads. The diagonal of a tile then covers 128 / g
// tokens instead of 128, and short sequences fill their tiles g times
// better. For a g that does not divide 128 the last rows of a tile stay
// empty (g * floor(128 / g) of 128 are used: 126 for 3, 125 for 5).
//
// Work items (eight int32 each) are built on the host from the lengths,
// longest first, without the key heads: item i of a kernel is table entry
// i / kv_heads of key head i % kv_heads. CTA c takes items c, 2G - 1 - c,
// 2G + c, ... of G CTAs (back and forth), which pairs long with short; the key
// gradient's items may come dealt (sequences.py, deal_items).
#pragma once

#include <math.h>

#include "common.cuh"

namespace veda {
namespace causal {

// Forward: two query tiles of one sequence and the key tiles that the second
// reaches, or a part of them (sequences.py cuts items along the keys where
// there are few).
struct alignas(16) ForwardItem {
  int row;     // packed row of the first token
  int tokens;  // tokens of the two tiles
  int k_row;   // packed row of the sequence's first key
  int kpos;    // the first token sees keys 0 .. kpos (negative: none)
  int keys;    // keys of the sequence
  int blocks;  // key tiles
  int first;   // the first of them
  int part;    // number of the part; -1: the whole
};

// The parts of a forward item: part .. part + parts - 1 (in the order of the
// keys).
struct alignas(16) JoinItem {
  int row;
  int tokens;
  int part;
  int parts;
  int pad[4];
};

// Query gradient: a query tile of one sequence.
struct alignas(16) QueryItem {
  int row;     // packed row of the first token
  int tokens;  // tokens of the tile
  int k_row;   // packed row of the sequence's first key
  int kpos;    // the first token sees keys 0 .. kpos (negative: none)
  int keys;    // keys of the sequence
  int blocks;  // key tiles that the last token reaches
  int tile;    // number of the query tile, over the whole pack
  int pad;
};

// A key tile of one sequence.
struct alignas(16) KeyItem {
  int row;     // packed row of the first key
  int keys;    // keys of the tile
  int q_row;   // packed row of the sequence's first token
  int tokens;  // tokens of the sequence
  int shift;   // token t sees key r of the tile if t >= shift + r
  int first;   // first query tile of the sequence that sees the tile
  int blocks;  // query tiles from there to the sequence's end
  int tile0;   // number of the sequence's first query tile
};

template <typename Item>
__device__ __forceinline__ Item load_item(const int32_t* table, int entry) {
  static_assert(sizeof(Item) == 32, "eight int32");
  union {
    int4 v[2];
    Item it;
  } u;
  const int4* src = reinterpret_cast<const int4*>(table) + 2 * entry;
  u.v[0] = __ldg(src);
  u.v[1] = __ldg(src + 1);
  return u.it;
}

// Item number of a CTA's n-th turn (may lie past the last item).
__device__ __forceinline__ int64_t turn(int n) {
  const int64_t base = static_cast<int64_t>(n) * gridDim.x;
  return base + ((n & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity,
                                         volatile int* abort,
                                         unsigned int* status) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, status));
}

// 2^x of a pair, free to be scheduled among other work.
__device__ __forceinline__ float2 exp2_pair(float2 x) {
  float2 y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(x.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(x.y));
  return y;
}

// Orders this thread's shared memory accesses before later accesses of the
// asynchronous proxy (TMA, tcgen05).
__device__ __forceinline__ void fence_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Writes 32 bytes (aligned): the rows of a tile are the lanes of a
// warp, so a store meets 32 lines however narrow it is, and the widest takes
// the fewest passes through them.
__device__ __forceinline__ void store32(void* dst, const uint32_t* w) {
  asm volatile(
      "st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst),
      "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
      "r"(w[6]), "r"(w[7])
      : "memory");
}

// An fp32 number keeps, beside its rounding to bf16, the eight bits behind
// bf16's: value = the float whose bits are (bf16 bits << 16) + (low << 8), low
// in [-128, 127], to 2^-16 of it, or to 2^-15 where 128 is held at 127 (a
// number that lies half way between two of bf16, or nearly). (The bits of a float's magnitude are in the
// order of the numbers, so the sum carries into the exponent where it has to.)
//
// The low bits of two numbers whose bf16 pair is w: in bits 0-7 and 16-23.
__device__ __forceinline__ uint32_t low_bits(float a, float b, uint32_t w) {
  const int x = (__float_as_int(a) - static_cast<int>(w << 16) + 128) >> 8;
  const int y =
      (__float_as_int(b) - static_cast<int>(w & 0xFFFF0000u) + 128) >> 8;
  return __byte_perm(max(-128, min(127, x)), max(-128, min(127, y)), 0x5410);
}

// The float of bf16 bits (in the high half of `high`) and byte kByte of low
// bits.
template <int kByte>
__device__ __forceinline__ float with_low(uint32_t high, uint32_t low) {
  const int sign_extended = static_cast<int>(low << (24 - 8 * kByte)) >> 16;
  return __uint_as_float((high & 0xFFFF0000u) +
                         (static_cast<uint32_t>(sign_extended) & ~0xffu));
}

// TMA: stores a box from shared memory (written by this warp, ordered by
// fence_async_shared); one lane issues it and later waits until the boxes it
// stored have been read from shared memory.
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map,
                                             const void* src, int c0, int c1,
                                             int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, "
      "%4}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
      "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

// Clears rows [first, 128) of a 128 x kD bf16 tile (64-column halves of 128
// bytes a row; the swizzle moves pieces inside a row only). One warp.
template <int kD>
__device__ __forceinline__ void clear_rows(uint8_t* tile, int first,
                                           int lane) {
#pragma unroll
  for (int half = 0; half < kD / 64; ++half)
    for (int i = first * 8 + lane; i < kTile * 8; i += 32)
      reinterpret_cast<uint4*>(tile + half * 16384)[i] = make_uint4(0, 0, 0, 0);
  fence_async_shared();
  __syncwarp();
}

// A run of MMAs issued by one elected lane of a converged warp. One election
// and one conversion of the operands' addresses for the whole run: issued one
// by one (umma_ss_warp) an MMA costs the issuing warp some 70 cycles, more
// than a product of 64 columns takes.
//
// D[tmem] (+)= A . B over kSteps steps of 16 along the depth, A and B K-major
// tiles of 64-column halves (16 KB apart). Descriptors as low halves.
#define VEDA_SS_STEP(N, OFF)                                            \
  "add.u32 al, %1, " OFF "; add.u32 bl, %2, " OFF ";"                   \
  "mov.b64 da, {al, %5}; mov.b64 db, {bl, %5};"                         \
  "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, " N ";"
template <int kSteps>
__device__ __forceinline__ void umma_ss_run(uint32_t d_tmem, uint32_t a_lo,
                                            uint32_t b_lo, uint32_t idesc) {
  static_assert(kSteps == 4 || kSteps == 8, "64 or 128 columns");
  if constexpr (kSteps == 8)
    asm volatile(
        "{ .reg .pred z, o, e; .reg .b64 da, db; .reg .b32 rx, al, bl;"
        "elect.sync rx|e, 0xFFFFFFFF; setp.ne.b32 z, %4, 0; "
        "setp.eq.b32 o, %4, 0;"
        VEDA_SS_STEP("z", "0") VEDA_SS_STEP("o", "2") VEDA_SS_STEP("o", "4")
        VEDA_SS_STEP("o", "6") VEDA_SS_STEP("o", "1024")
        VEDA_SS_STEP("o", "1026") VEDA_SS_STEP("o", "1028")
        VEDA_SS_STEP("o", "1030") "}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(0u), "r"(kSw128DescHi)
        : "memory");
  else
    asm volatile(
        "{ .reg .pred z, o, e; .reg .b64 da, db; .reg .b32 rx, al, bl;"
        "elect.sync rx|e, 0xFFFFFFFF; setp.ne.b32 z, %4, 0; "
        "setp.eq.b32 o, %4, 0;"
        VEDA_SS_STEP("z", "0") VEDA_SS_STEP("o", "2") VEDA_SS_STEP("o", "4")
        VEDA_SS_STEP("o", "6") "}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(0u), "r"(kSw128DescHi)
        : "memory");
}
#undef VEDA_SS_STEP

// D[tmem] (+)= A[tmem] . B over 64 of the depth: A's steps at columns 0, 8,
// 16, 24 (kGap: 0, 8, 32, 40) from a_tmem, B MN-major, 2 KB a step. The first
// step overwrites D unless `accumulate`.
#define VEDA_TS_STEP(N, COL, OFF)                                       \
  "add.u32 al, %1, " COL "; add.u32 bl, %2, " OFF ";"                   \
  "mov.b64 db, {bl, %5};"                                               \
  "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [al], db, %3, " N ";"
template <bool kGap>
__device__ __forceinline__ void umma_ts_run(uint32_t d_tmem, uint32_t a_tmem,
                                            uint32_t b_lo, uint32_t idesc,
                                            uint32_t accumulate) {
  if constexpr (kGap)
    asm volatile(
        "{ .reg .pred z, o, e; .reg .b64 db; .reg .b32 rx, al, bl;"
        "elect.sync rx|e, 0xFFFFFFFF; setp.ne.b32 z, %4, 0; "
        "setp.ne.b32 o, %5, 0;"
        VEDA_TS_STEP("z", "0", "0") VEDA_TS_STEP("o", "8", "128")
        VEDA_TS_STEP("o", "32", "256") VEDA_TS_STEP("o", "40", "384")
        "}" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate),
        "r"(kSw128DescHi)
        : "memory");
  else
    asm volatile(
        "{ .reg .pred z, o, e; .reg .b64 db; .reg .b32 rx, al, bl;"
        "elect.sync rx|e, 0xFFFFFFFF; setp.ne.b32 z, %4, 0; "
        "setp.ne.b32 o, %5, 0;"
        VEDA_TS_STEP("z", "0", "0") VEDA_TS_STEP("o", "8", "128")
        VEDA_TS_STEP("o", "16", "256") VEDA_TS_STEP("o", "24", "384")
        "}" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate),
        "r"(kSw128DescHi)
        : "memory");
}
#undef VEDA_TS_STEP

// 3D bf16 tensor map over rows x heads x kD with a (64, heads_box, rows_box)
// box and 128-byte swizzle.
int make_rows_map(CUtensorMap* map, const void* base, int64_t rows,
                  int64_t heads, int head_dim, int64_t stride_row,
                  int64_t stride_head, int heads_box, int rows_box,
                  const char* name);

}  // namespace causal
}  // namespace veda
