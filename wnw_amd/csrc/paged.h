// The paged K/V cache: what its append and its attention kernels share.
#pragma once

#include <type_traits>

#include "wnw_common.h"

namespace wnw {

static constexpr float kPgLog2e = 1.4426950408889634f;
static constexpr float kPgLowest = -3.402823466e38f;  // running maxima start below every score

// wnw_paged_cache with what its checks have established: 32-bit counts,
// page_rows = 1 << shift, strides in bytes.
struct PagedCache {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  const int32_t* table;
  int64_t k_stride, v_stride;  // bytes from one page to the next
  int64_t table_stride;        // entries from one segment's row of the table to the next
  int32_t n_seg, n_pages, max_blocks, shift, capacity;  // capacity: rows a table row can name
};

// Checks a cache description and fills *out; WNW_OK or the status of the
// refusal (wnw_last_error set).
int paged_cache_of(const wnw_paged_cache* c, PagedCache* out);

// A token sequence of samples: cu_tokens, or one token per sample.
struct PagedTokens {
  const int32_t* cu;  // [samples + 1] or null: sample b's only token is b
  int32_t total, hkv, most;  // tokens in all, KV heads, most tokens of one sample (as the caller says)
};

// First token and token count of segment s's sample; false (and count 0)
// where cu_tokens is not what it has to be.
__device__ __forceinline__ bool paged_tokens_of(const PagedTokens& t, int s, int* first, int* count) {
  const int b = s / t.hkv;
  if (!t.cu) {
    *first = b;
    *count = 1;
    return true;
  }
  const int a = t.cu[b], e = t.cu[b + 1];
  *first = a;
  *count = e - a;
  if (a < 0 || e < a || e > t.total || e - a > t.most) {
    *first = *count = 0;
    return false;
  }
  return true;
}

// x, as a value that the compiler does not know: what follows from it is worked
// out here and not, ahead of the loops around, held in registers all along
template <typename I>
__device__ __forceinline__ I here(I x) {
  asm volatile("" : "+v"(x));
  return x;
}

template <typename T>
struct HalfOps;
template <>
struct HalfOps<bf16_t> {
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  typedef __bf16 v4 __attribute__((ext_vector_type(4)));
  __device__ static f32x4 mma16(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  // columns of 4 rows: lane i of 16 gets column i of the rows its 16 lanes point at
  __device__ static uint64_t read_tr(const uint8_t* lds) {
    return __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) v4*)lds));
  }
  // the values of two e4m3 codes of w (its upper or lower half): exact
  template <bool HI>
  __device__ static uint32_t e4m3x2(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  }
  // two values, round to nearest even
  __device__ static uint32_t pack2(float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, v2));
  }
};
template <>
struct HalfOps<f16_t> {
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  typedef __fp16 v4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
  __device__ static f32x4 mma16(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  __device__ static uint64_t read_tr(const uint8_t* lds) {
    return __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) v4*)lds));
  }
  template <bool HI>
  __device__ static uint32_t e4m3x2(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
  }
  __device__ static uint32_t pack2(float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, v2));
  }
};

// Infinities and NaN among V's elements.  Where a product's columns do not all
// see a row, its weight 0 does not take them out (0 times either is NaN): there
// they are staged as zeros, and added to the sums of the columns that see them at
// the end.  E: the page's element, uint8_t for e4m3 codes.
//
// All ones in the elements of w that are infinite or NaN
template <typename E>
__device__ __forceinline__ uint32_t odd_elems(uint32_t w) {
  constexpr bool kCodes = std::is_same<E, uint8_t>::value;
  constexpr uint32_t kMost = kCodes ? 0x7f7f7f7fu : std::is_same<E, bf16_t>::value ? 0x7f807f80u : 0x7c007c00u;
  constexpr uint32_t kOne = kMost & ~(kMost << 1);  // the lowest bit of each field
  const uint32_t top = ((w & kMost) + kOne) & (kCodes ? 0x80808080u : 0x80008000u);
  return kCodes ? (top >> 7) * 0xffu : (top >> 15) * 0xffffu;
}
// Takes them out of x; whether there were any
template <typename E>
__device__ __forceinline__ bool take_odd(u32x4& x) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t m = odd_elems<E>(x[i]);
    any |= m;
    x[i] &= ~m;
  }
  return any != 0;
}
// Elements d .. d + 3 of a row in its page: those that are infinite or NaN, else zeros
template <typename E>
__device__ __forceinline__ f32x4 odd_quad(const uint8_t* row, int d) {
  f32x4 y;
  if constexpr (std::is_same<E, uint8_t>::value) {
    const uint32_t m = odd_elems<E>(*gptr<uint32_t>(row + d));
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = m >> (8 * e) & 1 ? __builtin_nanf("") : 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t w = gptr<uint32_t>(row + 2 * d)[i], x = w & odd_elems<E>(w);
      y[2 * i] = std::is_same<E, bf16_t>::value ? bf16_lo(x) : f16_bits_to_f32(x & 0xffffu);
      y[2 * i + 1] = std::is_same<E, bf16_t>::value ? bf16_hi(x) : f16_bits_to_f32(x >> 16);
    }
  }
  return y;
}
// Row `row` of segment seg in V's pages; null where no page holds it
__device__ __forceinline__ const uint8_t* paged_v_row(const PagedCache& c, int seg, int row, int row_bytes) {
  const int page = c.table[seg * c.table_stride + (row >> c.shift)];
  return (uint32_t)page < (uint32_t)c.n_pages ? c.v + page * c.v_stride + (row & ((1 << c.shift) - 1)) * row_bytes : nullptr;
}

// 8 codes (two words) as 8 elements of T
template <typename T>
__device__ __forceinline__ u32x4 e4m3x8(uint32_t lo, uint32_t hi) {
  using Ops = HalfOps<T>;
  return u32x4{Ops::template e4m3x2<false>(lo), Ops::template e4m3x2<true>(lo), Ops::template e4m3x2<false>(hi),
               Ops::template e4m3x2<true>(hi)};
}

}  // namespace wnw
