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
// 2G + c, ... of G CTAs (back and forth), which pairs long with short.
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

// 3D bf16 tensor map over rows x heads x kD with a (64, heads_box, rows_box)
// box and 128-byte swizzle.
int make_rows_map(CUtensorMap* map, const void* base, int64_t rows,
                  int64_t heads, int head_dim, int64_t stride_row,
                  int64_t stride_head, int heads_box, int rows_box,
                  const char* name);

}  // namespace causal
}  // namespace veda
