// The paged key-value cache: rows quantised as they are written, contexts
// read back as packed bf16 rows.
//
// A row x (one token, one head) is stored as codes and one scale:
//     int8   scale = max|x| / 127, code = round(127 x / max|x|)
//     e4m3   scale = 2^e with the smallest integer e >= -120 for which
//            max|x| <= 448 2^e; code = x / scale rounded to e4m3
//     bf16   the row itself, no scale
// rounding to nearest, ties to even. A power-of-two scale costs a
// floating-point code nothing (but at its subnormals) and makes both the
// division before the rounding and the product on reading exact, so the one
// rounding is that to e4m3. For int8 the quotient is taken as the correctly
// rounded fp32 quotient of 127 x (exact: 8 + 7 bits) and max|x|: an exact
// half is representable and stays one, and a quotient that is not a half
// differs from it by more than the quotient's rounding error (bf16 operands),
// so the codes are those of real arithmetic. It is computed as the product with
// the reciprocal of max|x|, corrected once by the exact remainder (Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor",
// 1990): a product that is off by a relative e leaves a remainder that brings
// it to within e^2, which the last rounding takes to the quotient where that is
// representable. (With a division for each value 55,504 tokens of 8 heads, D =
// 128, took 131 us.) A row with a value that is not finite gets the scale NaN,
// and reads back as NaN throughout; an all-zero row has scale 0.
//
// Both kernels are bound by memory: a group of D / 8 lanes holds a row of k
// and the row of v at the same place, 16 bytes of bf16 a lane each, and the
// maximum crosses the group with shuffles, so a row is read once and written
// once.
#include "kvcache.cuh"

#include <cuda_fp8.h>

#include <type_traits>

namespace veda {

namespace {

constexpr int kThreads = 256;

// The sequence that packed row t belongs to: offsets[b] <= t < offsets[b+1];
// some sequence for a row outside all of them.
__device__ __forceinline__ int find_sequence(const int32_t* offsets, int n,
                                             int64_t t) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (offsets[mid] <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// Two bf16 as floats.
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  return make_float2(__uint_as_float(w << 16),
                     __uint_as_float(w & 0xFFFF0000u));
}

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// The larger of the eight magnitudes of a lane, as bf16 bits. Magnitudes of
// bf16 order as their bits do, infinity behind the numbers and NaN behind
// infinity, so nothing is lost in the maximum.
__device__ __forceinline__ uint32_t top8(const uint4& w) {
  constexpr uint32_t kAbs = 0x7fff7fffu;
  const uint32_t high = __vmaxu2(__vmaxu2(w.x & kAbs, w.y & kAbs),
                                 __vmaxu2(w.z & kAbs, w.w & kAbs));
  return max(high >> 16, high & 0xffffu);
}

// max|x| of a row of k (low half) and of the row of v at its place (high
// half), which kGroup lanes hold.
template <int kGroup>
__device__ __forceinline__ uint32_t row_tops(const uint4& k, const uint4& v) {
  uint32_t high = top8(k) | (top8(v) << 16);
#pragma unroll
  for (int s = kGroup / 2; s > 0; s >>= 1)
    high = __vmaxu2(high, __shfl_xor_sync(0xffffffffu, high, s));
  return high;
}

// Codes of a lane's 8 values of a row whose largest magnitude has the bits
// `high`, and the row's scale.
template <int kStore>
__device__ __forceinline__ uint2 encode8(const uint4& w, uint32_t high,
                                         float* scale) {
  const float top = __uint_as_float(high << 16);
  uint32_t word[2] = {0u, 0u};
  if (high >= 0x7f80u) {
    *scale = __int_as_float(0x7fffffff);
    return make_uint2(0u, 0u);
  }
  if (high == 0u) {
    *scale = 0.f;
    return make_uint2(0u, 0u);
  }
  const float2 x[4] = {unpack2(w.x), unpack2(w.y), unpack2(w.z), unpack2(w.w)};
  if constexpr (kStore == kStoreInt8) {
    // top / 127, corrected the same way (the correctly rounded quotient for
    // each of the 32,639 finite magnitudes: checked one by one).
    const float unit = 1.f / 127.f;
    float sc = top * unit;
    sc = fmaf(fmaf(-sc, 127.f, top), unit, sc);
    *scale = sc;
    // By a power of two 127 x stays finite in large rows, and max|x| normal in
    // small ones.
    const float pre = top > 1.f ? 0x1p-8f : 0x1p24f;
    const float den = top * pre, num = 127.f * pre;
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(den));
    // Adding 1.5 2^23 rounds to an integer (ties to even) and leaves it in
    // the low bits.
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 n = __fmul2_rn(x[i], both(num));
      float2 quot = __fmul2_rn(n, both(inv));
      quot = __ffma2_rn(__ffma2_rn(quot, both(-den), n), both(inv), quot);
      quot = __fadd2_rn(quot, both(12582912.f));
      c[2 * i] = __float_as_uint(quot.x);
      c[2 * i + 1] = __float_as_uint(quot.y);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      word[i] = __byte_perm(__byte_perm(c[4 * i], c[4 * i + 1], 0x0040),
                            __byte_perm(c[4 * i + 2], c[4 * i + 3], 0x0040),
                            0x5410);
  } else {
    // top = 1.f 2^x: 448 = 1.75 2^8. Subnormal tops end at the clamp.
    const uint32_t bits = __float_as_uint(top);
    int e = static_cast<int>(bits >> 23) - 127 - 8 +
            ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    if (e < -120) e = -120;
    *scale = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
    const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_fp8x2_storage_t c = __nv_cvt_float2_to_fp8x2(
          __fmul2_rn(x[i], both(inv)), __NV_SATFINITE, __NV_E4M3);
      word[i >> 1] |= static_cast<uint32_t>(c) << (16 * (i & 1));
    }
  }
  return make_uint2(word[0], word[1]);
}

// Eight codes times their scale, rounded once to bf16.
template <int kStore>
__device__ __forceinline__ uint4 decode8(const uint2& w, float scale) {
  const uint32_t u[2] = {w.x, w.y};
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 x;
    if constexpr (kStore == kStoreInt8) {
      // 2^23 + (code + 128), less 2^23 + 128.
      const uint32_t biased = u[i >> 1] ^ 0x80808080u;
      x.x = __uint_as_float(
          __byte_perm(biased, 0x4B000000u, 0x7540 | 2 * (i & 1)));
      x.y = __uint_as_float(
          __byte_perm(biased, 0x4B000000u, 0x7541 | 2 * (i & 1)));
      x = __fadd2_rn(x, both(-8388736.f));
    } else {
      const uint32_t pair = u[i >> 1] >> (16 * (i & 1));
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
          static_cast<__nv_fp8x2_storage_t>(pair & 0xffffu), __NV_E4M3);
      x = __half22float2(__half2(h));
    }
    x = __fmul2_rn(x, both(scale));
    out[i] = pack_bf16(x.x, x.y);
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

// Rows of k and v a group of lanes takes at a time. Finding a row's place is a
// chain of four dependent loads and more: each lane of a warp finds one row's,
// and the data of all of them is in flight meanwhile. 55,504 tokens of 8
// heads, D = 128, int8: written in 79 us against 104 with every lane finding
// its rows' places, 66 with the encoding on pairs of values (e4m3 61, bf16 73);
// read in 58 against 68 with a row at a time (e4m3 the same, bf16 74), which is
// the copy rate. Two rows at a time write 15 % slower, eight at once 20 %
// (registers); two batches of four behind one search for places write int8 in
// 62 but a single token in 4.0 us against 2.75.
constexpr int kBatch = 4;

template <int kStore, int kD>
__global__ void __launch_bounds__(kThreads)
    cache_write_kernel(CacheView c, const __nv_bfloat16* k, int64_t k_st,
                       int64_t k_sh, const __nv_bfloat16* v, int64_t v_st,
                       int64_t v_sh, const int32_t* offsets,
                       const int32_t* starts, int n_rows,
                       unsigned int* status) {
  constexpr int kGroup = kD / 8;
  constexpr int kGroups = kThreads / kGroup;
  const int lane = threadIdx.x % kGroup;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kGroups * kBatch +
                       threadIdx.x / kGroup;
  // Lane i * kWide + g finds the place of row i of group g of the warp; the
  // groups then take theirs from it.
  constexpr int kWide = 32 / kGroup;  // groups of a warp
  const int64_t warp_row = row0 - (threadIdx.x % 32) / kGroup;
  const int wl = threadIdx.x % 32;
  int my_t = 0, my_h = 0;
  int64_t my_at = -1;
  {
    const int64_t row = warp_row + (wl / kWide % kBatch) * kGroups + wl % kWide;
    // Past the end: the last row's values, stored nowhere.
    const int r = row < n_rows ? static_cast<int>(row) : n_rows - 1;
    my_t = r / c.kv_heads;
    my_h = r - my_t * c.kv_heads;
    if (row < n_rows && wl < kWide * kBatch) {
      const int b = find_sequence(offsets, c.n_seqs, my_t);
      const int first = offsets[b];
      // (A row before the first sequence or behind the last is stored nowhere.)
      if (my_t >= first && my_t < offsets[b + 1]) {
        my_at = cache_row(c, b, my_h,
                          static_cast<int64_t>(starts[b]) + (my_t - first));
        if (my_at < 0) raise_status(status, VEDA_ERR_INVALID);
      }
    }
  }
  uint4 kw[kBatch], vw[kBatch];
  int64_t at[kBatch];
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    const int from = i * kWide + wl / kGroup;
    const int t = __shfl_sync(0xffffffffu, my_t, from);
    const int h = __shfl_sync(0xffffffffu, my_h, from);
    kw[i] = *reinterpret_cast<const uint4*>(k + t * k_st + h * k_sh +
                                            lane * 8);
    vw[i] = *reinterpret_cast<const uint4*>(v + t * v_st + h * v_sh +
                                            lane * 8);
  }
#pragma unroll
  for (int i = 0; i < kBatch; ++i)
    at[i] = __shfl_sync(0xffffffffu, my_at, i * kWide + wl / kGroup);
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    if constexpr (kStore == kStoreBf16) {
      if (at[i] >= 0) {
        reinterpret_cast<uint4*>(c.k)[at[i] * kGroup + lane] = kw[i];
        reinterpret_cast<uint4*>(c.v)[at[i] * kGroup + lane] = vw[i];
      }
    } else {
      float ks, vs;
      const uint32_t tops = row_tops<kGroup>(kw[i], vw[i]);
      const uint2 kc = encode8<kStore>(kw[i], tops & 0xffffu, &ks);
      const uint2 vc = encode8<kStore>(vw[i], tops >> 16, &vs);
      if (at[i] >= 0) {
        reinterpret_cast<uint2*>(c.k)[at[i] * kGroup + lane] = kc;
        reinterpret_cast<uint2*>(c.v)[at[i] * kGroup + lane] = vc;
        if (lane == 0) {
          c.k_scale[at[i]] = ks;
          c.v_scale[at[i]] = vs;
        }
      }
    }
  }
}

template <int kStore, int kD>
__global__ void __launch_bounds__(kThreads)
    cache_read_kernel(CacheView c, const int32_t* offsets, int64_t n_rows,
                      __nv_bfloat16* k, __nv_bfloat16* v,
                      unsigned int* status) {
  constexpr int kGroup = kD / 8;
  constexpr int kGroups = kThreads / kGroup;
  constexpr int kWide = 32 / kGroup;
  const int lane = threadIdx.x % kGroup, wl = threadIdx.x % 32;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kGroups * kBatch +
                       threadIdx.x / kGroup;
  // As in the other kernel, a lane a row. (kNoRow: a row before the first
  // sequence or behind the last, which is not written.)
  constexpr int64_t kNoRow = -2;
  int64_t my_at = kNoRow;
  {
    const int64_t row = row0 - wl / kGroup +
                        (wl / kWide % kBatch) * kGroups + wl % kWide;
    if (row < n_rows && wl < kWide * kBatch) {
      const int t = static_cast<int>(row) / c.kv_heads;
      const int h = static_cast<int>(row) - t * c.kv_heads;
      const int b = find_sequence(offsets, c.n_seqs, t);
      const int first = offsets[b];
      if (t >= first && t < offsets[b + 1]) {
        my_at = cache_row(c, b, h, t - first);
        if (my_at < 0) raise_status(status, VEDA_ERR_INVALID);
      }
    }
  }
  // Rows that are nowhere read as zeros (and load the cache's first row: with
  // a branch around the loads the compiler puts a row's conversion behind its
  // load, inside the branch, and the rows wait for one another).
  using Word = typename std::conditional<kStore == kStoreBf16, uint4,
                                         uint2>::type;
  Word kw[kBatch], vw[kBatch];
  float ks[kBatch], vs[kBatch];
  bool there[kBatch], taken[kBatch];
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    int64_t at = __shfl_sync(0xffffffffu, my_at, i * kWide + wl / kGroup);
    there[i] = at >= 0;
    taken[i] = at != kNoRow;
    if (at < 0) at = 0;
    kw[i] = reinterpret_cast<const Word*>(c.k)[at * kGroup + lane];
    vw[i] = reinterpret_cast<const Word*>(c.v)[at * kGroup + lane];
    if constexpr (kStore != kStoreBf16) {
      ks[i] = c.k_scale[at];
      vs[i] = c.v_scale[at];
    }
  }
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    // Packed outputs [rows, kv_heads, D]: row-major in (token, head).
    const int64_t row = row0 + i * kGroups;
    if (!taken[i]) continue;
    uint4 ko, vo;
    if constexpr (kStore == kStoreBf16) {
      ko = kw[i];
      vo = vw[i];
    } else {
      ko = decode8<kStore>(kw[i], ks[i]);
      vo = decode8<kStore>(vw[i], vs[i]);
    }
    if (!there[i]) ko = vo = make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4*>(k)[row * kGroup + lane] = ko;
    reinterpret_cast<uint4*>(v)[row * kGroup + lane] = vo;
  }
}

// Calls fn.template operator()<kStore, kD>() for the runtime pair.
template <typename Fn>
int dispatch(int storage, int head_dim, Fn fn) {
  if (head_dim == 128) {
    if (storage == kStoreBf16) return fn.template operator()<kStoreBf16, 128>();
    if (storage == kStoreInt8) return fn.template operator()<kStoreInt8, 128>();
    return fn.template operator()<kStoreE4m3, 128>();
  }
  if (storage == kStoreBf16) return fn.template operator()<kStoreBf16, 64>();
  if (storage == kStoreInt8) return fn.template operator()<kStoreInt8, 64>();
  return fn.template operator()<kStoreE4m3, 64>();
}

struct WriteLaunch {
  CacheView c;
  const __nv_bfloat16 *k, *v;
  int64_t k_st, k_sh, v_st, v_sh;
  const int32_t *offsets, *starts;
  int64_t rows;
  unsigned int* status;
  cudaStream_t stream;
  template <int kStore, int kD>
  int operator()() const {
    constexpr int kRows = kThreads / (kD / 8) * kBatch;  // of a block
    const int64_t blocks = (rows + kRows - 1) / kRows;
    cache_write_kernel<kStore, kD>
        <<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(
            c, k, k_st, k_sh, v, v_st, v_sh, offsets, starts,
            static_cast<int>(rows), status);
    return check_launch("cache_write_kernel");
  }
};

struct ReadLaunch {
  CacheView c;
  const int32_t* offsets;
  int64_t rows;
  __nv_bfloat16 *k, *v;
  unsigned int* status;
  cudaStream_t stream;
  template <int kStore, int kD>
  int operator()() const {
    constexpr int kRows = kThreads / (kD / 8) * kBatch;  // of a block
    const int64_t blocks = (rows + kRows - 1) / kRows;
    cache_read_kernel<kStore, kD>
        <<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(
            c, offsets, rows, k, v, status);
    return check_launch("cache_read_kernel");
  }
};

}  // namespace

int make_cache_view(CacheView* view, void* k, void* v, float* k_scale,
                    float* v_scale, int64_t n_pages, int32_t page_size,
                    int32_t kv_heads, int32_t head_dim, int32_t storage,
                    const int32_t* table, int64_t table_ld, int64_t max_pages,
                    int64_t n_seqs) {
  VEDA_REQUIRE(storage == kStoreBf16 || storage == kStoreInt8 ||
                   storage == kStoreE4m3,
               "storage must be 0 (bf16), 1 (int8) or 2 (e4m3)");
  VEDA_REQUIRE(head_dim == 64 || head_dim == 128,
               "head_dim must be 64 or 128");
  int shift = 0;
  while (shift < 9 && (1 << shift) < page_size) ++shift;
  VEDA_REQUIRE(page_size >= 16 && page_size <= 256 &&
                   (1 << shift) == page_size,
               "page_size must be 16, 32, 64, 128 or 256");
  VEDA_REQUIRE(kv_heads >= 1 && kv_heads <= 65535, "bad kv_heads");
  VEDA_REQUIRE(n_pages >= 1 && n_pages < (int64_t(1) << 31), "bad n_pages");
  VEDA_REQUIRE(n_seqs >= 1 && n_seqs < (int64_t(1) << 24), "bad n_seqs");
  VEDA_REQUIRE(max_pages >= 1 && max_pages * page_size < (int64_t(1) << 31) &&
                   table_ld >= max_pages,
               "a table row must hold 1 page or more and address fewer than "
               "2^31 rows");
  VEDA_REQUIRE(k && v && table, "k, v and table are required");
  VEDA_REQUIRE(reinterpret_cast<uintptr_t>(k) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(v) % 16 == 0,
               "the pages must be 16-byte aligned");
  VEDA_REQUIRE(storage == kStoreBf16 ? (!k_scale && !v_scale)
                                     : (k_scale && v_scale),
               "int8 and e4m3 pages have scales, bf16 pages have none");
  VEDA_REQUIRE(storage == kStoreBf16 ||
                   (reinterpret_cast<uintptr_t>(k_scale) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(v_scale) % 16 == 0),
               "the scales must be 16-byte aligned");
  view->k = static_cast<uint8_t*>(k);
  view->v = static_cast<uint8_t*>(v);
  view->k_scale = k_scale;
  view->v_scale = v_scale;
  view->n_pages = static_cast<int>(n_pages);
  view->page_shift = shift;
  view->kv_heads = kv_heads;
  view->table = table;
  view->table_ld = table_ld;
  view->max_pages = static_cast<int>(max_pages);
  view->n_seqs = static_cast<int>(n_seqs);
  return VEDA_OK;
}

}  // namespace veda

using namespace veda;

extern "C" int veda_cache_write(
    void* k_pages, void* v_pages, float* k_scale, float* v_scale,
    int64_t n_pages, int32_t page_size, int32_t kv_heads, int32_t head_dim,
    int32_t storage, const int32_t* table, int64_t table_ld, int64_t max_pages,
    int64_t n_seqs, const void* k, int64_t k_stride_t, int64_t k_stride_h,
    const void* v, int64_t v_stride_t, int64_t v_stride_h, int64_t n_tokens,
    const int32_t* offsets, const int32_t* starts, void* stream) {
  int rc = require_sm100("veda_cache_write");
  if (rc != VEDA_OK) return rc;
  CacheView c;
  rc = make_cache_view(&c, k_pages, v_pages, k_scale, v_scale, n_pages,
                       page_size, kv_heads, head_dim, storage, table, table_ld,
                       max_pages, n_seqs);
  if (rc != VEDA_OK) return rc;
  VEDA_REQUIRE(n_tokens >= 0 && n_tokens * kv_heads < (int64_t(1) << 31),
               "n_tokens * kv_heads must lie in [0, 2^31)");
  VEDA_REQUIRE(offsets && starts, "offsets and starts are required");
  if (n_tokens == 0) return VEDA_OK;
  VEDA_REQUIRE(k && v, "k and v are required");
  auto aligned = [](const void* p, int64_t st, int64_t sh) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && st % 8 == 0 &&
           sh % 8 == 0;
  };
  VEDA_REQUIRE(aligned(k, k_stride_t, k_stride_h) &&
                   aligned(v, v_stride_t, v_stride_h),
               "k and v must be 16-byte aligned with strides multiple of 8");
  WriteLaunch launch{c,
                     static_cast<const __nv_bfloat16*>(k),
                     static_cast<const __nv_bfloat16*>(v),
                     k_stride_t,
                     k_stride_h,
                     v_stride_t,
                     v_stride_h,
                     offsets,
                     starts,
                     n_tokens * kv_heads,
                     device_status_ptr(),
                     as_stream(stream)};
  return dispatch(storage, head_dim, launch);
}

extern "C" int veda_cache_read(
    const void* k_pages, const void* v_pages, const float* k_scale,
    const float* v_scale, int64_t n_pages, int32_t page_size, int32_t kv_heads,
    int32_t head_dim, int32_t storage, const int32_t* table, int64_t table_ld,
    int64_t max_pages, int64_t n_seqs, const int32_t* offsets,
    int64_t n_tokens, void* k, void* v, void* stream) {
  int rc = require_sm100("veda_cache_read");
  if (rc != VEDA_OK) return rc;
  CacheView c;
  rc = make_cache_view(&c, const_cast<void*>(k_pages),
                       const_cast<void*>(v_pages),
                       const_cast<float*>(k_scale),
                       const_cast<float*>(v_scale), n_pages, page_size,
                       kv_heads, head_dim, storage, table, table_ld, max_pages,
                       n_seqs);
  if (rc != VEDA_OK) return rc;
  VEDA_REQUIRE(n_tokens >= 0 && n_tokens * kv_heads < (int64_t(1) << 31),
               "n_tokens * kv_heads must lie in [0, 2^31)");
  VEDA_REQUIRE(offsets != nullptr, "offsets are required");
  if (n_tokens == 0) return VEDA_OK;
  VEDA_REQUIRE(k && v && reinterpret_cast<uintptr_t>(k) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(v) % 16 == 0,
               "k and v are required, 16-byte aligned");
  ReadLaunch launch{c,
                    offsets,
                    n_tokens * kv_heads,
                    static_cast<__nv_bfloat16*>(k),
                    static_cast<__nv_bfloat16*>(v),
                    device_status_ptr(),
                    as_stream(stream)};
  return dispatch(storage, head_dim, launch);
}
