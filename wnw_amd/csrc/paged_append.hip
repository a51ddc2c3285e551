// Append to the paged cache with the rotation of q and K on the way (gfx950).
//
// Mathematics.  Pair j of a head (j < rot / 2; elements (j, j + rot / 2), or
// (2 j, 2 j + 1) interleaved) at position x of its axis turns by the angle
// x * inv_freq[j]: (a, b) -> (a cos - b sin, b cos + a sin).  The angle is a
// product in 64 bits, in quarter turns, and the whole ones are taken off there:
// at position 10^5 a 32-bit product is off by 2^-8 of a radian.  Sine and cosine
// of what is left are their Taylor series in 32 bits (|x| <= pi / 4; the terms
// left out, x^11 / 11! and x^12 / 12!, are below 2 * 10^-9 and 2 * 10^-10).  All
// else is 32-bit, rounded once where a value is stored.
//
// What bounds it: memory.  A prompt of 4,564 tokens (40 q and K / V heads of 128
// into 8 bits, 103 MB) takes 21.8 us, 4.7 TB/s, a large copy 5.1.  One token
// takes 4.3 us, most of it the launch and one chain of dependent loads: length,
// table entry, position, row.
//
// 8-bit pages hold e4m3 codes under one scale per page, the least power of two
// 2^e (e >= -64) with |x| <= 448 * 2^e for all its rows.  e4m3 has the same
// relative step in every binade, so a finer scale would gain nothing, and a
// power of two makes x / scale exact: each code is x rounded once.  When
// a row raises the scale of a page that holds rows already, their codes are
// divided by the same power of two (exact but for codes that become
// subnormal).  Infinities and NaN become NaN codes and do not count for the scale.
#include <algorithm>
#include <type_traits>

#include "paged.h"

namespace wnw {

struct PagedAppendParams {
  PagedCache c;
  PagedTokens t;
  const int32_t* seg_len;  // [n_seg] rows before
  int32_t* new_len;        // [n_seg] rows after
  const void *q, *k, *v;   // q null: none
  void* q_out;             // [tokens, Hkv * G, D]
  int64_t qt, qh, kt, kh, vt, vh;  // strides in elements
  const void* pos;         // [axes, tokens] int64 or int32; null: no rotation
  const void* inv_freq;    // [rot / 2] double or float
  int64_t pos_axis;        // elements from one axis to the next
  int32_t pos64, freq64, interleaved, rot, G, units, unit_shift;
  int32_t sec1, sec2, sec3;  // first pair of the second, third and fourth axis
  int32_t* err;
};

// sin and cos of u quarter turns, |u| < 2^51
__device__ __forceinline__ void turn_of(double u, float* sn, float* cs) {
  // adding 1.5 * 2^52 leaves the nearest whole number in the low bits
  const double t = u + 6755399441055744.0;
  const int quarter = (int)__builtin_bit_cast(uint64_t, t);
  const float y = (float)(u - (t - 6755399441055744.0)) * 1.57079633f;  // [-pi / 4, pi / 4]
  const float z = y * y;
  float s = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  s = fmaf(z, s, 8.3333333e-3f);
  s = fmaf(z, s, -1.6666667e-1f);
  s = fmaf(z * y, s, y);
  float c = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  c = fmaf(z, c, -1.3888889e-3f);
  c = fmaf(z, c, 4.1666667e-2f);
  c = fmaf(z, c, -0.5f);
  c = fmaf(z, c, 1.0f);
  const float a = quarter & 1 ? c : s, b = quarter & 1 ? s : c;
  *sn = __uint_as_float(__float_as_uint(a) ^ (uint32_t)(quarter & 2) << 30);
  *cs = __uint_as_float(__float_as_uint(b) ^ (uint32_t)((quarter + 1) & 2) << 30);
}

// PP consecutive 16-bit elements (2 or 8): as they lie, as floats, and back
template <int PP>
using Run = typename std::conditional<PP == 8, u32x4, uint32_t>::type;
template <typename T, int PP>
__device__ __forceinline__ Run<PP> load_run(const T* p) {
  return *gptr<Run<PP>>(p);
}
template <typename T, int PP>
__device__ __forceinline__ void elems_of(const Run<PP>& w, float (&x)[PP]) {
  if constexpr (PP == 8) {
    unpack8(w, x, (T*)nullptr);
  } else if constexpr (std::is_same<T, bf16_t>::value) {
    x[0] = bf16_lo(w);
    x[1] = bf16_hi(w);
  } else {
    x[0] = f16_bits_to_f32(w & 0xffffu);
    x[1] = f16_bits_to_f32(w >> 16);
  }
}
template <typename T, int PP>
__device__ __forceinline__ void store_elems(T* p, const float (&x)[PP]) {
  if constexpr (PP == 8) {
    *gptr_w<u32x4>(p) = u32x4{HalfOps<T>::pack2(x[0], x[1]), HalfOps<T>::pack2(x[2], x[3]),
                                                HalfOps<T>::pack2(x[4], x[5]), HalfOps<T>::pack2(x[6], x[7])};
  } else {
    *gptr_w<uint32_t>(p) = HalfOps<T>::pack2(x[0], x[1]);
  }
}
template <int PP>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&x)[PP], float inv) {
  uint32_t w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
  if constexpr (PP == 2) {
    *gptr_w<uint16_t>(p) = (uint16_t)w;
  } else {
    typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
    w = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, w, true);
    uint32_t y = __builtin_amdgcn_cvt_pk_fp8_f32(x[4] * inv, x[5] * inv, 0, false);
    y = __builtin_amdgcn_cvt_pk_fp8_f32(x[6] * inv, x[7] * inv, y, true);
    *gptr_w<u32x2_t>(p) = u32x2_t{w, y};
  }
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;  // false for NaN too
}

// log2 of the scale that holds magnitudes up to amax
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);  // 448 = 1.75 * 2^8
  return max(e, -64);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// A workgroup takes one unit: the rows of one append that fall into one page of
// one segment, so that the page's largest magnitude is known before a code is
// written.  With 16-bit pages it is 4,096 elements of one (a long prompt into
// pages of 256 rows of 128: 24.2 us by 32 rows, 26.1 by 16, 25.9 by 64, 32.1 whole;
// of 256 elements: 22.0 by 32 rows, 18.5 by 16, 25.1 by 64).  A thread holds PP
// pairs of a row (2 PP elements in two runs of PP) and up to NIT rows.  V's loads
// go out first and a q head's before the one ahead of it is stored.
//   PP = 8 (chunks of prompts): 16-byte loads; the unit does K, V and the
//       group's q heads, so a row's sines are worked out once for all of them;
//       with few units the q heads are shared out over blockIdx.y.
//   PP = 2 (a few tokens): K, V and each q head in workgroups of their own
//       (blockIdx.y), a quarter of the sines in each thread: with one token the
//       time is one chain of loads, sines and stores.
template <typename T, int PP, bool Q8, int NT, int NIT>
__global__ __launch_bounds__(NT) void paged_append_kernel(PagedAppendParams p, int D) {
  __shared__ float red[2][NT / 64];
  const int tid = threadIdx.x;
  const int s = blockIdx.x / p.units, unit = blockIdx.x - s * p.units;
  // PP = 2: 0 K, 1 V, 2 + g q head g.  PP = 8: -1 K, V and the first share of the q heads, 2 another share
  const int what = PP == 2 ? (int)blockIdx.y : blockIdx.y == 0 ? -1 : 2;
  const int h = s % p.t.hkv;
  int first, count;
  const bool told = paged_tokens_of(p.t, s, &first, &count);
  const int len0 = p.seg_len[s];
  const bool good_len = len0 >= 0 && (int64_t)len0 + count <= p.c.capacity;
  const int len = len0 >= 0 && len0 <= (1 << 30) ? len0 : 0;
  if (unit == 0 && tid == 0 && what <= 0) {
    p.new_len[s] = (int32_t)((uint32_t)len0 + (uint32_t)count);
    if (!told) raise_device_error(p.err, WNW_DEVERR_BOUNDS);
    if (!good_len) raise_device_error(p.err, WNW_DEVERR_CAPACITY);
  }
  const int R = 1 << p.c.shift, us = p.unit_shift;
  const int at = (len >> us) + unit;
  const int row0 = max(at << us, len), row1 = min((at + 1) << us, len + count);  // rows of the segment
  if (row0 >= row1) return;
  // where they go: rows past the table, or in no page, are not stored
  int page = -1;
  const int block = row0 >> p.c.shift;
  if (good_len && block < p.c.max_blocks) {
    page = p.c.table[s * p.c.table_stride + block];
    if (page < 0 || page >= p.c.n_pages) {
      if (tid == 0) raise_device_error(p.err, WNW_DEVERR_BOUNDS);
      page = -1;
    }
  }
  const int fill = row0 & (R - 1);  // rows that the page held before
  // the thread's place in a row
  const int tpr = D / (2 * PP), rpp = NT / tpr, turning = p.pos ? p.rot / (2 * PP) : 0;
  const int cth = tid % tpr, rth = tid / tpr;
  const bool turns = cth < turning;
  int e0, e1;
  if (turns && !p.interleaved) {
    e0 = cth * PP;
    e1 = p.rot / 2 + cth * PP;
  } else {
    e0 = cth * 2 * PP;
    e1 = e0 + PP;
  }
  const int n = row1 - row0, t0 = first + row0 - len;

  // what a position is worth in quarter turns, pair by pair, and the pairs' axes
  double fq[PP];
  const int64_t axis0 = ((cth * PP >= p.sec1) + (cth * PP >= p.sec2) + (cth * PP >= p.sec3)) * p.pos_axis;
  const int last = cth * PP + PP - 1;
  const bool one_axis = axis0 == ((last >= p.sec1) + (last >= p.sec2) + (last >= p.sec3)) * p.pos_axis;
  if (turns && what != 1) {
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      const int j = cth * PP + i;
      fq[i] = (p.freq64 ? gptr<double>(p.inv_freq)[j] : (double)gptr<float>(p.inv_freq)[j]) * 0.63661977236758134;
    }
  }
  auto position = [&](int64_t at) {
    return p.pos64 ? (double)gptr<int64_t>(p.pos)[at] : (double)gptr<int32_t>(p.pos)[at];
  };
  auto sines = [&](int row, float (&sn)[PP], float (&cs)[PP]) {
    if (one_axis) {
      const double x = position(axis0 + t0 + row);
#pragma unroll
      for (int i = 0; i < PP; ++i) turn_of(x * fq[i], &sn[i], &cs[i]);
    } else {
#pragma unroll
      for (int i = 0; i < PP; ++i) {
        const int j = cth * PP + i;
        turn_of(position(((j >= p.sec1) + (j >= p.sec2) + (j >= p.sec3)) * p.pos_axis + t0 + row) * fq[i], &sn[i], &cs[i]);
      }
    }
  };
  auto turned = [&](float (&a)[PP], float (&b)[PP], const float (&sn)[PP], const float (&cs)[PP]) {
    if (!turns) return;
    if (p.interleaved) {  // pair i: elements 2 i and 2 i + 1 of the 2 PP
      float x[2 * PP];
#pragma unroll
      for (int i = 0; i < PP; ++i) {
        const float u = i < PP / 2 ? a[2 * i] : b[2 * i - PP], w = i < PP / 2 ? a[2 * i + 1] : b[2 * i + 1 - PP];
        x[2 * i] = u * cs[i] - w * sn[i];
        x[2 * i + 1] = w * cs[i] + u * sn[i];
      }
#pragma unroll
      for (int i = 0; i < PP; ++i) {
        a[i] = x[i];
        b[i] = x[PP + i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < PP; ++i) {
        const float u = a[i], w = b[i];
        a[i] = u * cs[i] - w * sn[i];
        b[i] = w * cs[i] + u * sn[i];
      }
    }
  };
  // the unit's K or V rows, held by its threads, into the page
  auto put = [&](const float (&x)[NIT][2][PP], uint8_t* pages, int64_t stride, float* scales, float* slot) {
    uint8_t* dst = pages + (int64_t)max(page, 0) * stride;
    if constexpr (!Q8) {
#pragma unroll
      for (int it = 0; it < NIT; ++it) {
        const int r = it * rpp + rth;
        if (r >= n || page < 0) continue;
        T* row = (T*)dst + (int64_t)(fill + r) * D;
        store_elems<T, PP>(row + e0, x[it][0]);
        store_elems<T, PP>(row + e1, x[it][1]);
      }
    } else {
      float amax = 0.f;
#pragma unroll
      for (int it = 0; it < NIT; ++it)
        if (it * rpp + rth < n)
#pragma unroll
          for (int i = 0; i < PP; ++i) amax = fmaxf(amax, fmaxf(finite_abs(x[it][0][i]), finite_abs(x[it][1][i])));
      amax = wave_max(amax);
      if (NT > 64) {
        if ((tid & 63) == 0) slot[tid >> 6] = amax;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) amax = fmaxf(amax, slot[i]);
      }
      if (page < 0) return;
      int e = scale_exponent(amax);
      float was = 0.f;
      if (fill > 0) was = scales[page];
      const float need = pow2(e), now = was > need ? was : need;  // a scale that is not a number counts for nothing
      if (fill > 0 && now > was) {
        const float ratio = was / now;
        const int words = fill * D / 4;
        for (int i = tid; i < words; i += NT) {
          WNW_GLOBAL uint32_t* at = gptr_w<uint32_t>(dst) + i;
          const uint32_t w = *at;
          typedef float f2 __attribute__((ext_vector_type(2)));
          const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
          uint32_t y = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * ratio, a[1] * ratio, 0, false);
          *at = __builtin_amdgcn_cvt_pk_fp8_f32(b[0] * ratio, b[1] * ratio, y, true);
        }
      }
      const float inv = 1.0f / now;
#pragma unroll
      for (int it = 0; it < NIT; ++it) {
        const int r = it * rpp + rth;
        if (r >= n) continue;
        uint8_t* row = dst + (int64_t)(fill + r) * D;
        store_codes<PP>(row + e0, x[it][0], inv);
        store_codes<PP>(row + e1, x[it][1], inv);
      }
      __syncthreads();  // every thread has read the scale
      if (tid == 0) scales[page] = now;
    }
  };

  // V's loads first, where there are registers for them
  constexpr bool kEarly = NIT <= 2;
  Run<PP> vr[NIT][2];
  auto load_v = [&]() {
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      // rows past the unit's repeat its last
      const T* row = (const T*)p.v + (int64_t)(t0 + min(it * rpp + rth, n - 1)) * p.vt + h * p.vh;
      vr[it][0] = load_run<T, PP>(row + e0);
      vr[it][1] = load_run<T, PP>(row + e1);
    }
  };
  if (kEarly && (what == -1 || what == 1)) load_v();
  float x[NIT][2][PP];
  if (what != 1) {
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int r = it * rpp + rth;
#pragma unroll
      for (int i = 0; i < PP; ++i) x[it][0][i] = x[it][1][i] = 0.f;
      if (r >= n) continue;
      Run<PP> ka, kb, qa, qb;
      if (what <= 0) {
        const T* row = (const T*)p.k + (int64_t)(t0 + r) * p.kt + h * p.kh;
        ka = load_run<T, PP>(row + e0);
        kb = load_run<T, PP>(row + e1);
      }
      const int g0 = PP == 2 ? what - 2 : p.G * (int)blockIdx.y / (int)gridDim.y;
      const int g1 = PP == 2 ? what - 1 : p.G * ((int)blockIdx.y + 1) / (int)gridDim.y;
      const T* qp = (const T*)p.q + (int64_t)(t0 + r) * p.qt + (h * p.G + g0) * p.qh;
      if (p.q && what != 0 && g0 < g1) {
        qa = load_run<T, PP>(qp + e0);
        qb = load_run<T, PP>(qp + e1);
      }
      float sn[PP], cs[PP];
      if (turns) sines(r, sn, cs);
      if (what <= 0) {
        elems_of<T, PP>(ka, x[it][0]);
        elems_of<T, PP>(kb, x[it][1]);
        turned(x[it][0], x[it][1], sn, cs);
      }
      if (p.q && what != 0) {
        T* dst = (T*)p.q_out + ((int64_t)(t0 + r) * (p.t.hkv * p.G) + h * p.G + g0) * D;
        for (int g = g0; g < g1; ++g) {
          float a[PP], b[PP];
          elems_of<T, PP>(qa, a);
          elems_of<T, PP>(qb, b);
          if (g + 1 < g1) {
            qp += p.qh;
            qa = load_run<T, PP>(qp + e0);
            qb = load_run<T, PP>(qp + e1);
          }
          turned(a, b, sn, cs);
          store_elems<T, PP>(dst + e0, a);
          store_elems<T, PP>(dst + e1, b);
          dst += D;
        }
      }
    }
    if (what <= 0) put(x, p.c.k, p.c.k_stride, p.c.k_scale, red[0]);
  }
  if (what == -1 || what == 1) {
    if (!kEarly) load_v();
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      elems_of<T, PP>(vr[it][0], x[it][0]);
      elems_of<T, PP>(vr[it][1], x[it][1]);
    }
    put(x, p.c.v, p.c.v_stride, p.c.v_scale, red[1]);
  }
}

// Workgroups that shares of the q heads are made for: 584 of a 4,564-token prompt
// take 22.0 us in one share, 21.8 in two and 28.1 in four (the sines again in each),
// 552 of ragged chunks 10.8, 9.5 and 9.0.
static constexpr int64_t kPaWgs = 1536;

template <typename T, bool Q8>
static hipError_t launch_append(const PagedAppendParams& p, int D, int64_t most, hipStream_t st) {
  // Rows of a unit and threads for them, measured on both sides (us):
  //   PP = 2 up to 1,024 elements (one token 4.4, with PP = 8 6.6; 7 tokens of 8
  //   samples 4.7 and 6.8; but units of 16 rows of a long prompt 58.8 and 23.4);
  //   then the most workgroups that hide each other's loads: pages of 4,096
  //   elements 20.9 with 256 threads and one row each, 22.1 with 128; 8,192:
  //   22.3 (two rows), with 512 threads 22.9, 128 22.2 but 13.9 for 10.7 with few
  //   units; 16,384: 27.3 (256, four rows), 512 34.0; 32,768: 30.5 (512), 1,024
  //   41.2; 65,536: 30.6 (512, eight rows), 1,024 39.2.
  const int64_t rows = std::min<int64_t>(1 << p.unit_shift, most);
  const dim3 grid((unsigned)((int64_t)p.c.n_seg * p.units));
  const dim3 heads(grid.x, p.q ? 2 + p.G : 2);
  const dim3 shares(grid.x, p.q ? (unsigned)std::max<int64_t>(1, std::min<int64_t>(p.G, kPaWgs / grid.x)) : 1u);
  if (rows * D <= 4 * 64)
    hipLaunchKernelGGL((paged_append_kernel<T, 2, Q8, 64, 1>), heads, dim3(64), 0, st, p, D);
  else if (rows * D <= 4 * 256)
    hipLaunchKernelGGL((paged_append_kernel<T, 2, Q8, 256, 1>), heads, dim3(256), 0, st, p, D);
  else if (rows * D <= 16 * 128)
    hipLaunchKernelGGL((paged_append_kernel<T, 8, Q8, 128, 1>), shares, dim3(128), 0, st, p, D);
  else if (rows * D <= 4096 || !Q8)
    hipLaunchKernelGGL((paged_append_kernel<T, 8, Q8, 256, 1>), shares, dim3(256), 0, st, p, D);
  if constexpr (Q8) {  // a page that is one unit, however large
    if (rows * D <= 4096) return hipGetLastError();
    if (rows * D <= 2 * 4096)
      hipLaunchKernelGGL((paged_append_kernel<T, 8, Q8, 256, 2>), shares, dim3(256), 0, st, p, D);
    else if (rows * D <= 4 * 4096)
      hipLaunchKernelGGL((paged_append_kernel<T, 8, Q8, 256, 4>), shares, dim3(256), 0, st, p, D);
    else if (rows * D <= 8 * 4096)
      hipLaunchKernelGGL((paged_append_kernel<T, 8, Q8, 512, 4>), shares, dim3(512), 0, st, p, D);
    else
      hipLaunchKernelGGL((paged_append_kernel<T, 8, Q8, 512, 8>), shares, dim3(512), 0, st, p, D);
  }
  return hipGetLastError();
}

int paged_cache_of(const wnw_paged_cache* c, PagedCache* out) {
  WNW_CHECK_ARG(c != nullptr, "the cache description is null");
  WNW_CHECK_ARG(c->page_dtype == WNW_BF16 || c->page_dtype == WNW_F16 || c->page_dtype == WNW_E4M3, "bad page type %d",
                c->page_dtype);
  WNW_CHECK_ARG(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, "head_dim must be 64, 128 or 256");
  int shift = 4;
  while (shift < 8 && (1 << shift) != c->page_rows) ++shift;
  WNW_CHECK_ARG((1 << shift) == c->page_rows, "page_rows must be 16, 32, 64, 128 or 256");
  const int64_t elem = c->page_dtype == WNW_E4M3 ? 1 : 2;
  WNW_CHECK_ARG(c->n_seg >= 0 && c->n_seg < (1 << 24) && c->n_pages >= 0 && c->n_pages < (1ll << 31) && c->max_blocks >= 0 &&
                    c->table_stride >= c->max_blocks,
                "bad sizes of the page table");
  WNW_CHECK_ARG(c->max_blocks <= (1 << 30) / c->page_rows, "a table row names at most 2^30 rows");
  WNW_CHECK_ARG(c->table_stride < (1ll << 31), "bad stride of the page table");
  const int64_t page = c->page_rows * c->head_dim;
  WNW_CHECK_ARG(c->k_stride >= page && c->v_stride >= page && c->k_stride * elem % 16 == 0 && c->v_stride * elem % 16 == 0 &&
                    c->k_stride < (1ll << 40) && c->v_stride < (1ll << 40),
                "pages must lie a multiple of 16 bytes apart, without overlap");
  WNW_CHECK_ARG(c->n_seg == 0 || c->max_blocks == 0 || c->page_table, "the page table is null");
  WNW_CHECK_ARG(c->n_pages == 0 || (c->k_pages && c->v_pages), "the pages are null");
  WNW_CHECK_ARG((uintptr_t)c->k_pages % 16 == 0 && (uintptr_t)c->v_pages % 16 == 0, "pages must be 16-byte aligned");
  if (c->page_dtype == WNW_E4M3)
    WNW_CHECK_ARG(c->n_pages == 0 || (c->k_scale && c->v_scale), "8-bit pages need k_scale and v_scale");
  else
    WNW_CHECK_ARG(!c->k_scale && !c->v_scale, "16-bit pages have no scales");
  out->k = (uint8_t*)c->k_pages;
  out->v = (uint8_t*)c->v_pages;
  out->k_scale = c->k_scale;
  out->v_scale = c->v_scale;
  out->table = c->page_table;
  out->k_stride = c->k_stride * elem;
  out->v_stride = c->v_stride * elem;
  out->table_stride = c->table_stride;
  out->n_seg = (int32_t)c->n_seg;
  out->n_pages = (int32_t)c->n_pages;
  out->max_blocks = (int32_t)c->max_blocks;
  out->shift = shift;
  out->capacity = (int32_t)(c->max_blocks * c->page_rows);
  return WNW_OK;
}

}  // namespace wnw

using namespace wnw;

extern "C" int wnw_paged_append(const wnw_paged_cache* cache, const int32_t* seg_len, int32_t* new_len, const void* q,
                                const void* k, const void* v, void* q_out, const int64_t* strides, int64_t n_tokens,
                                int64_t n_samples, int64_t group, const int32_t* cu_tokens, int64_t max_tokens,
                                const void* positions, int pos_bits, int64_t pos_stride, const void* inv_freq, int freq_bits,
                                int64_t rot, const int32_t* sections, int n_sections, int interleaved, int dtype,
                                void* stream) {
  PagedAppendParams p = {};
  if (int rc = paged_cache_of(cache, &p.c)) return rc;
  const int64_t D = cache->head_dim, N = cache->n_seg;
  WNW_CHECK_ARG(dtype == WNW_BF16 || dtype == WNW_F16, "q, k and v must be bf16 or f16");
  WNW_CHECK_ARG(cache->page_dtype == WNW_E4M3 || cache->page_dtype == dtype, "16-bit pages must have the type of k and v");
  WNW_CHECK_ARG(n_samples >= 0 && (n_samples > 0 ? N % n_samples == 0 : N == 0), "segments must be samples x KV heads");
  WNW_CHECK_ARG(n_tokens >= 0 && n_tokens < (1 << 30) && max_tokens >= 0 && (cu_tokens || n_tokens == n_samples),
                "without cu_tokens every sample has one token");
  WNW_CHECK_ARG(group >= 1 && group <= 1024, "bad group");
  if (N == 0) return WNW_OK;
  WNW_CHECK_ARG(seg_len && new_len && strides, "null pointer argument");
  WNW_CHECK_ARG(n_tokens == 0 || (k && v), "k or v is null");
  WNW_CHECK_ARG(seg_len + N <= new_len || new_len + N <= seg_len, "new_len must not overlap seg_len");
  WNW_CHECK_ARG(cache->n_pages == 0 || (cache->k_pages != cache->v_pages && (!cache->k_scale || cache->k_scale != cache->v_scale)),
                "K and V need pages and scales of their own");
  WNW_CHECK_ARG((q == nullptr) == (q_out == nullptr), "q and q_out come together");
  for (int i = 0; i < 6; ++i)
    WNW_CHECK_ARG(strides[i] >= 0 && strides[i] % 8 == 0 && strides[i] < (1ll << 40), "strides must be multiples of 8 elements");
  WNW_CHECK_ARG((uintptr_t)q % 16 == 0 && (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (uintptr_t)q_out % 16 == 0,
                "rows must be 16-byte aligned");
  const int64_t hkv = N / n_samples;
  p.sec1 = p.sec2 = p.sec3 = 1 << 30;
  if (positions) {
    WNW_CHECK_ARG(inv_freq && sections, "positions need inv_freq and sections");
    WNW_CHECK_ARG((pos_bits == 64 || pos_bits == 32) && (freq_bits == 64 || freq_bits == 32), "bad type of positions or inv_freq");
    WNW_CHECK_ARG(rot >= 16 && rot <= D && rot % 16 == 0, "the rotated part must be a multiple of 16 elements within head_dim");
    WNW_CHECK_ARG(n_sections >= 1 && n_sections <= 4, "one to four axes");
    int64_t at = 0;
    for (int i = 0; i < n_sections; ++i) {
      WNW_CHECK_ARG(sections[i] >= 0 && sections[i] <= rot / 2, "bad section");
      if (i == 1) p.sec1 = (int32_t)at;
      if (i == 2) p.sec2 = (int32_t)at;
      if (i == 3) p.sec3 = (int32_t)at;
      at += sections[i];
    }
    WNW_CHECK_ARG(at == rot / 2, "the sections must add up to half of the rotated part");
    WNW_CHECK_ARG(n_sections == 1 || pos_stride >= n_tokens, "positions must be [axes, tokens]");
  }
  const int64_t most = cu_tokens ? std::min(max_tokens, n_tokens) : 1;
  const bool q8 = cache->page_dtype == WNW_E4M3;
  const int64_t unit_rows = q8 ? cache->page_rows : std::min(cache->page_rows, 4096 / D);
  const int64_t units = (std::max<int64_t>(most, 1) + unit_rows - 2) / unit_rows + 1;
  WNW_CHECK_ARG(N * units < (1ll << 23), "too many segments and tokens for one call");
  p.t = PagedTokens{cu_tokens, (int32_t)n_tokens, (int32_t)hkv, (int32_t)most};
  p.seg_len = seg_len;
  p.new_len = new_len;
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_out = q_out;
  p.qt = strides[0], p.qh = strides[1], p.kt = strides[2], p.kh = strides[3], p.vt = strides[4], p.vh = strides[5];
  p.pos = positions;
  p.inv_freq = inv_freq;
  p.pos_axis = pos_stride;
  p.pos64 = pos_bits == 64;
  p.freq64 = freq_bits == 64;
  p.interleaved = interleaved != 0;
  p.rot = (int32_t)rot;
  p.G = (int32_t)group;
  p.units = (int32_t)units;
  p.err = device_error_word();
  p.unit_shift = __builtin_ctzll(unit_rows);
  const int64_t rows = std::max<int64_t>(most, 1);
  hipStream_t st = (hipStream_t)stream;
  const hipError_t e = dtype == WNW_BF16 ? (q8 ? launch_append<bf16_t, true>(p, (int)D, rows, st)
                                               : launch_append<bf16_t, false>(p, (int)D, rows, st))
                                         : (q8 ? launch_append<f16_t, true>(p, (int)D, rows, st)
                                               : launch_append<f16_t, false>(p, (int)D, rows, st));
  WNW_CHECK_HIP(e, "paged_append launch");
  return WNW_OK;
}
