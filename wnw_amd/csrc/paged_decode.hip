// Decode attention over the paged cache (gfx950): up to 16 query rows per
// segment (a group's heads, times the few tokens a sample may bring).
//
// Mathematics: per segment o = sum_t w_t v_t / sum_t w_t, w_t = 2^(s_t - m),
// s_t = scale log2(e) q . k_t, in one pass over the rows with the running
// maximum m; partial sums (m, l, o) of disjoint rows add up after a factor
// 2^(m' - m) each, so any split of the rows gives the same sums.
//
// Work split: the segments' rows in steps of 32 (no step crosses a segment),
// all steps cut evenly over the workgroups, and a workgroup's steps dealt to its
// waves by pieces: a piece (its steps of one segment) has as many waves as its
// share, whole waves, so that no wave holds the sums of two pieces at once and
// short segments run side by side.  A piece of one wave ends in its registers,
// one of several in LDS; a segment cut between workgroups in memory, added up by
// the last of them to arrive.  The lengths are read on the device, so a captured
// launch stays right as segments grow.
//
// A step: S^T (rows x queries) = K Q^T with the rows' 16-byte chunks straight
// from memory as matrix operands (any order of the elements of a dot will do,
// if q has the same), V through LDS for its transpose (each wave its own part,
// no barrier), O^T += V^T P^T, whose P^T operand is S^T's own layout when V's
// rows follow its order.  The next step's rows are loaded while a step is used.
// 8-bit codes become 16-bit elements in registers (exact); K's scale
// multiplies the scores, V's scale the weights.  Weights go through two 16-bit
// parts, the upper cut off, not rounded: 16 bits of each, beside 32-bit sums.
//
// What bounds it: with many rows memory (256 segments of up to 5,003 16-bit rows,
// 224 MB: 48.0 us, 4.7 TB/s, a large copy 5.1; loads that leave the caches alone,
// as each byte is used once: 51.3 us without); with few, the launch and one chain of
// dependent round trips: lengths, table, pages, partial sums, counter (8 segments
// of at most 813 rows: 11.3 us).
#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "paged.h"

namespace wnw {

struct PagedDecodeParams {
  PagedCache c;
  PagedTokens t;
  const int32_t* seg_len;
  const void* q;
  void* out;
  int64_t qt, qh, ot, oh;  // strides in elements
  float* part_acc;         // [2 grid, cols, D]
  float* part_ml;          // [2 grid, cols, 2]
  int32_t* counters;       // [n_seg], zero between launches
  float scale_log2;
  int32_t G, cols;         // cols: query rows of a segment at most
  int32_t* err;
};

static constexpr int kPdStep = 32;  // rows of a step
// Where segments are cut.  More workgroups have fewer steps each, but whoever adds
// up a segment's pieces reads as many partial sums, one round trip to memory for 8.
// A workgroup has kPdMin steps at least (8 sequences of 2 x 7,564 and 6 x 512 rows:
// 18.7 us; with 4: 18.9, 12: 20.0, 16: 20.9), a segment about kPdPieces pieces at
// most, or half as many of 2,048 sums or more (30,000 rows of 2 heads: 4 query
// heads 20.9 us with 117 pieces, 19.1 with 58, 20.2 with 39; 16 query heads 31.4,
// 24.3, 22.5), and segments of up to kPdWhole steps stay whole (26 steps: 11.2 us,
// cut 12.4).
static constexpr int kPdMin = 8;
static constexpr int kPdPieces = 64;
static constexpr int kPdWhole = 40;

template <int D, bool Q8>
struct PagedDecodeGeom {
  static constexpr int RB = D * (Q8 ? 1 : 2);      // bytes of a row
  static constexpr int KC = RB / 64;               // 16-byte chunks of a K row per lane
  static constexpr int VI = kPdStep * RB / 1024;   // loads of a step's V per lane
  // Bytes in flight and registers: a step is 4 to 32 KB of loads per wave, and
  // 128 KB a CU keep the memory busy.  Two workgroups of 8 waves a CU, where the
  // registers allow it, take 18.7 us where one of 16 takes 20.7.
  static constexpr int kWaves = RB >= 512 ? 4 : 8;  // of a workgroup
  static constexpr int kWgs = RB >= 256 ? 1 : 2;    // workgroups per CU
  static constexpr int kStage = kPdStep * RB;       // LDS of a wave's V
  static constexpr int kQ = D * 32;                 // of its q
  static constexpr int kState = 16 * (D + 4) * 4;   // of its sums, in the place of both
  static constexpr int kPart = kStage + kQ > kState ? kStage + kQ : kState;
};

// A step's V in LDS: row r's 16-byte chunk c lies at r * RB + 16 * (c ^ x(r)).
// The transposed reads take 8 rows of one chunk (8 bits: rows 4 q .. + 3 and 16 +
// 4 q .. + 3) or 4 rows of two chunks (16 bits) at a time; x keeps both, and the
// writes of whole rows, free of bank conflicts.  x(r) is a lane's part and a
// load's part that do not overlap, so an address is a lane's constant XOR a
// number known at compile time.
template <int D, bool Q8>
struct PagedDecodeV {
  static constexpr int RB = PagedDecodeGeom<D, Q8>::RB, VI = PagedDecodeGeom<D, Q8>::VI, CH = RB / 16;
  // load i writes rows i * 64 / CH + lane / CH
  __device__ static uint32_t write_base(int lane) {
    const int r = lane / CH, c = lane % CH;
    const int x = !Q8 ? 2 * (r & 3) : CH == 4 ? r >> 1 & 1 : r & 3;
    return r * RB + 16 * (c ^ x);
  }
  static constexpr uint32_t write_x(int i) {
    return !Q8 ? (D == 256 ? 64 * (i & 1) : 0) : i >= VI / 2 ? (CH == 4 ? 32 : 64) : 0;
  }
  // 16 columns i * 16 .. of the lane's rows
  __device__ static uint32_t read_base(int lq, int lc) {
    if (!Q8) return (4 * lq + (lc >> 2)) * RB + 16 * (((lc & 3) >> 1) ^ (2 * (lc >> 2))) + 8 * (lc & 1);
    return (4 * lq + (lc >> 1 & 3) + 16 * (lc >> 3)) * RB + 16 * (CH == 4 ? lc >> 2 : lc >> 1) + 8 * (lc & 1);
  }
  static constexpr uint32_t read_x(int i) { return (Q8 ? 16 : 32) * i; }
};

// Two weights as two pairs of 16-bit parts.  The lower parts of weights that are not 0 are not 0
// either: an infinity of V times such a part would be NaN.  bf16's are 2^-24 of the upper at least
// (a weight has 16 bits here), f16's, short of exponents, its least number, 2^-36 of the
// largest weight; what has no weight adds nothing, however large.
template <typename T>
__device__ __forceinline__ void two_parts(float a, float b, uint32_t* hi, uint32_t* lo) {
  if constexpr (std::is_same<T, bf16_t>::value) {
    const uint32_t ua = __float_as_uint(a) & 0xffff0000u, ub = __float_as_uint(b) & 0xffff0000u;
    *hi = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
    const float ha = __uint_as_float(ua), hb = __uint_as_float(ub);
    const float la = fmaxf(a - ha, ha * 0x1p-24f), lb = fmaxf(b - hb, hb * 0x1p-24f);
    *lo = __builtin_amdgcn_perm(__float_as_uint(lb), __float_as_uint(la), 0x07060302u);
  } else {
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    *hi = __builtin_bit_cast(uint32_t, h);
    const float ha = (float)h[0], hb = (float)h[1];
    const float la = fmaxf(a - ha, fminf(ha, 0x1p-24f)), lb = fmaxf(b - hb, fminf(hb, 0x1p-24f));
    *lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(la, lb));
  }
}

__device__ __forceinline__ void store_agent(float* p, float a, float b) {
  __hip_atomic_store((uint64_t*)p, (uint64_t)__float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void load_agent(const float* p, float* a, float* b) {
  const uint64_t x = __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  *a = __uint_as_float((uint32_t)x);
  *b = __uint_as_float((uint32_t)(x >> 32));
}

// What a segment's query rows are.  The divisions are branched around where
// they are by one: code that a launch meets for the first time costs more
// than its instructions (a cold line of the instruction cache is a memory round
// trip), which is why what follows a piece is kept short and rolled.
struct DecodeRows {
  int first, count, h, n, cols;  // tokens, KV head, rows of the segment, query rows
};
__device__ __forceinline__ DecodeRows decode_rows(const PagedDecodeParams& p, int seg, int n) {
  DecodeRows r;
  if (p.t.hkv == 1 && !p.t.cu) {
    r.first = seg;
    r.count = 1;
    r.h = 0;
  } else {
    paged_tokens_of(p.t, seg, &r.first, &r.count);
    r.h = seg % p.t.hkv;
  }
  r.n = n;
  r.cols = min(r.count * p.G, p.cols);
  return r;
}
__device__ __forceinline__ int token_of(const PagedDecodeParams& p, const DecodeRows& r, int col) {
  return r.count > 1 ? col / p.G : 0;
}
// Where query row col's result goes
template <typename T>
__device__ __forceinline__ T* out_row(const PagedDecodeParams& p, const DecodeRows& r, int col, int ti) {
  return (T*)p.out + (int64_t)(r.first + ti) * p.ot + (int64_t)(r.h * p.G + col - ti * p.G) * p.oh;
}
// Elements d .. d + 3 of a result, from its sums
template <typename T>
__device__ __forceinline__ void paged_decode_out(const PagedDecodeParams& p, const DecodeRows& r, int col, int d, const f32x4& o,
                                                 float L) {
  const int ti = token_of(p, r, col);
  const bool sees = r.n - r.count + ti + 1 > 0;  // else a row without keys
  const float inv = __builtin_amdgcn_rcpf(L);
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = sees ? o[i] * inv : 0.f;
  store_quad<T>(out_row<T>(p, r, col, ti), d, y);
}

// The partials of workgroups [w0, w1] (the first in slot 2 w0 + late, the
// others each in its first slot) added up, in as many runs as there are threads
// for, 8 at a time; the runs by way of lds.
template <typename T, int D, int NT>
__device__ __forceinline__ void paged_decode_gather(const PagedDecodeParams& p, const DecodeRows& r, int tid, int late, int w0,
                                                    int w1, float* lds) {
  constexpr int kSc1 = 16;  // buffer cache policy: coherent over the device
  tid = here(tid);
  const int items = r.cols * (D / 4), np = w1 - w0 + 1;
  int runs = 1;
  while (runs < 8 && 2 * runs * items <= NT && 2 * runs < np) runs *= 2;
  const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(p.part_acc, 0, 0x7fffffff, 0x00027000);
  const __amdgpu_buffer_rsrc_t rm = __builtin_amdgcn_make_buffer_rsrc(p.part_ml, 0, 0x7fffffff, 0x00027000);
  __syncthreads();
  for (int e = tid; e < items * runs; e += NT) {
    const int run = runs > 1 ? e / items : 0, item = e - run * items, col = item / (D / 4);
    float M = kPgLowest, L = 0.f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k0 = run; k0 < np; k0 += 8 * runs) {
      f32x4 po[8];
      float pm[8], pl[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = min(k0 + i * runs, np - 1);  // past the last: the last again, not added
        const int slot = (2 * (w0 + k) + (k == 0 ? late : 0)) * p.cols;
        po[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(ra, slot * (D * 4) + item * 16, 0, kSc1));
        const auto ml = __builtin_amdgcn_raw_buffer_load_b64(rm, (slot + col) * 8, 0, kSc1);
        pm[i] = __uint_as_float(ml[0]);
        pl[i] = __uint_as_float(ml[1]);
      }
      float now = M;
#pragma unroll
      for (int i = 0; i < 8; ++i) now = fmaxf(now, pm[i]);
      const float f0 = __builtin_amdgcn_exp2f(M - now);
      L *= f0;
      o *= f0;
      M = now;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = k0 + i * runs < np;  // a weight of 0 would not do: the last one may hold an infinity
        const float f = in ? __builtin_amdgcn_exp2f(pm[i] - M) : 0.f;
        L += f * pl[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += f * (in ? po[i][j] : 0.f);
      }
    }
    if (runs == 1) {
      paged_decode_out<T>(p, r, col, 4 * (item % (D / 4)), o, L);
    } else {
      float* to = lds + e * 8;
      *(f32x4*)to = o;
      to[4] = M;
      to[5] = L;
    }
  }
  if (runs == 1) return;
  __syncthreads();
  if (tid < items) {
    float M = kPgLowest, L = 0.f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int i = 0; i < runs; ++i) {
      const float* at = lds + (i * items + tid) * 8;
      const float now = fmaxf(M, at[4]), f = __builtin_amdgcn_exp2f(M - now), g = __builtin_amdgcn_exp2f(at[4] - now);
      L = L * f + g * at[5];
      o = o * f + g * *(const f32x4*)at;
      M = now;
    }
    paged_decode_out<T>(p, r, tid / (D / 4), 4 * (tid % (D / 4)), o, L);
  }
}

template <typename T, int D, bool Q8>
__global__ __launch_bounds__((64 * PagedDecodeGeom<D, Q8>::kWaves),
                             (PagedDecodeGeom<D, Q8>::kWaves * PagedDecodeGeom<D, Q8>::kWgs / 4)) void
paged_decode_kernel(PagedDecodeParams p) {
  using Ge = PagedDecodeGeom<D, Q8>;
  using VT = typename std::conditional<Q8, bf16_t, T>::type;  // the value product's type: any scale fits bf16
  using PE = typename std::conditional<Q8, uint8_t, T>::type;  // the pages' elements
  using QO = HalfOps<T>;
  using VO = HalfOps<VT>;
  using Vl = PagedDecodeV<D, Q8>;
  constexpr int W = Ge::kWaves, NT = 64 * W;
  constexpr int RB = Ge::RB, KC = Ge::KC, VI = Ge::VI, DT = D / 16, KK = D / 32;
  // weights of f16 are held times 2^12: their lower parts reach 2^-36 of the
  // largest; of bf16 times 2^-16: 2^16 times the type's largest value is a sum yet
  constexpr float kBias = std::is_same<VT, f16_t>::value ? 12.f : -16.f;
  __shared__ __attribute__((aligned(16))) uint8_t lds[W * Ge::kPart];
  __shared__ float st[W][16][2];
  __shared__ int32_t sh[2 * W];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int N = p.c.n_seg, wg = blockIdx.x;

  auto steps_of = [&](int n) { return n >= 0 && n <= p.c.capacity ? (n + kPdStep - 1) / kPdStep : 0; };
  auto scan = [&](int x) {  // inclusive, over the wave
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o);
      if (lane >= o) x += y;
    }
    return x;
  };
  // All steps and the most of a segment, this workgroup's [x0, x1), and the
  // window of 64 segments from its first one on: lane j has segment win + j, of
  // `len` rows, whose `num` steps come after `at` others.
  int win = 0, len = 0, num = 0, at = 0, S, longest;
  int mine = 0, incl = 0, before = 0;
  const int per = (N + NT - 1) / NT, sa = min(tid * per, N), sb = min(sa + per, N);
  if (N <= 64) {
    len = lane < N ? p.seg_len[lane] : 0;
    num = steps_of(len);
    at = scan(num);
    S = __builtin_amdgcn_readlane(at, 63);
    at -= num;
    longest = (int)wave_max((float)num);  // as good as exact: it is compared with kPdWhole
  } else {
    int most = 0;
    for (int s = sa; s < sb; ++s) {
      const int n = steps_of(p.seg_len[s]);
      mine += n;
      most = max(most, n);
    }
    incl = scan(mine);
    most = (int)wave_max((float)most);
    if (lane == 63) {
      sh[w] = incl;
      sh[W + w] = most;
    }
    __syncthreads();
    S = longest = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (i < w) before += sh[i];
      S += sh[i];
      longest = max(longest, sh[W + i]);
    }
    S = __builtin_amdgcn_readfirstlane(S);
    __syncthreads();
  }
  longest = __builtin_amdgcn_readfirstlane(longest);
  // Short segments are not cut (a workgroup takes whole ones), others not into pieces
  // of less than `least` steps.
  const bool uncut = longest <= kPdWhole;
  const int least = max(kPdMin, longest / (p.cols * D >= 2048 ? kPdPieces / 2 : kPdPieces));
  const int total = uncut ? N : S, P = min((int)gridDim.x, uncut ? N : max(S / least, 1));
  const int share = total / P, more = total - share * P;  // the first `more` workgroups take one more
  auto start_of = [&](int i) { return i * share + min(i, more); };
  auto owner_of = [&](int x) {  // the workgroup that has step x
    const int big = more * (share + 1);
    return x < big ? x / (share + 1) : more + (x - big) / max(share, 1);
  };
  int x0 = wg < P ? start_of(wg) : 0, x1 = wg < P ? start_of(wg + 1) : 0;
  if (x0 < x1) {
    const int s0 = x0, s1 = x1;  // segments, if uncut
    if (N <= 64) {
      if (uncut) {
        x0 = __builtin_amdgcn_readlane(at, s0);
        x1 = s1 < N ? __builtin_amdgcn_readlane(at, s1) : S;
      }
    } else {
      int e = before + incl - mine;  // steps before the thread's segments
      for (int s = sa; s < sb; ++s) {
        const int n = steps_of(p.seg_len[s]);
        if (uncut ? s == s0 : e <= x0 && x0 < e + n) {
          sh[0] = s;
          sh[1] = e;
        }
        if (uncut && s == s1) sh[2] = e;
        e += n;
      }
      __syncthreads();
      win = __builtin_amdgcn_readfirstlane(sh[0]);
      at = __builtin_amdgcn_readfirstlane(sh[1]);
      if (uncut) {
        x0 = at;
        x1 = s1 < N ? __builtin_amdgcn_readfirstlane(sh[2]) : S;
      }
    }
  }

  for (int x = x0; x < x1 && win < N;) {
    if (N > 64) {
      len = win + lane < N ? p.seg_len[win + lane] : 0;
      num = steps_of(len);
      at += scan(num) - num;
    }
    // the pieces of this window, and the waves [wf, wt) of each; a piece that
    // has none (wf == wt) is done by a wave beside its own
    const int xe = min(x1, __builtin_amdgcn_readlane(at + num, 63));
    const int pa = max(at, x), pb = min(at + num, xe), all = xe - x;
    const bool some = pa < pb;
    const int wf = some ? (2 * W * (pa - x) + all) / (2 * all) : 0, wt = some ? (2 * W * (pb - x) + all) / (2 * all) : 0;
    const uint64_t several = __ballot(some && wt - wf > 1), cut = __ballot(some && (pa != at || pb != at + num));
    const int waves = wf | wt << 8;
    // segment win + j: its steps before the piece and up to its end
    auto piece = [&](int j, int* a, int* b) {
      const int e = __builtin_amdgcn_readlane(at, j);
      *a = max(x - e, 0);
      *b = min(xe - e, __builtin_amdgcn_readlane(num, j));
      return e;
    };
    // those beside its own first: its own sums stay in its LDS
    uint64_t beside = __ballot(some && wf == wt && min(wf, W - 1) == w), own = __ballot(some && wf <= w && w < wt);
    while (beside | own) {
      const int j = __builtin_ctzll(beside ? beside : own), ln = here(lane), lq = ln >> 4, lc = ln & 15;
      const int seg = win + j, n = __builtin_amdgcn_readlane(len, j);
      const int f = __builtin_amdgcn_readlane(waves, j) & 255, t = __builtin_amdgcn_readlane(waves, j) >> 8;
      const int nw = max(t - f, 1), iw = t > f ? w - f : 0;
      int a, b;  // the wave's steps of the segment: a, a + nw, ... below b
      const int first_step = piece(j, &a, &b);
      a += iw;
      const int mysteps = (b - a + nw - 1) / nw;
      const DecodeRows r = decode_rows(p, seg, n);
      const int cols = r.cols;
      const int c = min(lc, max(cols - 1, 0)), ti = token_of(p, r, c);
      const int limit = n - r.count + ti + 1;  // rows that the lane's column sees
      const int all_see = n - r.count + 1;     // rows that every column sees
      f32x4 acc[DT];
#pragma unroll
      for (int i = 0; i < DT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      float m = kPgLowest, l = 0.f;
      uint8_t* stage = lds + w * Ge::kPart;
      const uint32_t klane = lc * RB + lq * 16, vlane = ln * 16;
      uint32_t vput = Vl::write_base(ln), vget = Vl::read_base(lq, lc);
      u32x4* qs = (u32x4*)(stage + Ge::kStage) + lane;

      // a window of 32 steps' pages: lane l has the page of half l & 1 of step l / 2
      int pid = -1;
      float ks = 1.f, vs = 1.f;
      auto window = [&](int k0) {
        const int step = a + nw * (k0 + (lane >> 1));
        const int row = step * kPdStep + 16 * (lane & 1);
        pid = -1;
        if (step < b && row < n) {
          pid = p.c.table[seg * p.c.table_stride + (row >> p.c.shift)];
          if (pid < 0 || pid >= p.c.n_pages) {
            raise_device_error(p.err, WNW_DEVERR_BOUNDS);
            pid = -1;
          }
        }
        if (Q8) {  // a half in no page has weights of 0, or rows of zeros: page 0's scale, whatever it is, is not theirs
          const float k_of = p.c.k_scale[max(pid, 0)], v_of = p.c.v_scale[max(pid, 0)];
          ks = pid < 0 ? 1.f : k_of;
          vs = pid < 0 ? 1.f : v_of;
        }
      };
      u32x4 kr[2][KC], vr[VI];
      int odd = 0;  // V had infinities or NaN where not every column sees its row
      int bad = 0;  // halves of the loaded step that no page holds
      auto load = [&](int k) {
        const int from = 2 * (k & 31);
        const int step = a + nw * k;
        const int p0 = __builtin_amdgcn_readlane(pid, from), p1 = __builtin_amdgcn_readlane(pid, from + 1);
        bad = (p0 < 0 ? 1 : 0) | (p1 < 0 ? 2 : 0);
        const int in = (step * kPdStep) & ((1 << p.c.shift) - 1);  // first row in its page
        const int in1 = (step * kPdStep + 16) & ((1 << p.c.shift) - 1);
        const int r0 = p0 < 0 ? max(p1, 0) : p0, r1 = p1 < 0 ? r0 : p1;  // a half in no page reads the other's
        const WNW_GLOBAL uint8_t* k0 = gptr<uint8_t>(p.c.k) + (int64_t)r0 * p.c.k_stride + (p0 < 0 ? 0 : in) * RB;
        const WNW_GLOBAL uint8_t* k1 = gptr<uint8_t>(p.c.k) + (int64_t)r1 * p.c.k_stride + (p1 < 0 ? 0 : in1) * RB;
        const WNW_GLOBAL uint8_t* v0 = gptr<uint8_t>(p.c.v) + (int64_t)r0 * p.c.v_stride + (p0 < 0 ? 0 : in) * RB;
        const WNW_GLOBAL uint8_t* v1 = gptr<uint8_t>(p.c.v) + (int64_t)r1 * p.c.v_stride + (p1 < 0 ? 0 : in1) * RB;
        const uint32_t kl = here(klane), vl = here(vlane);
#pragma unroll
        for (int i = 0; i < KC; ++i) {
          kr[0][i] = __builtin_nontemporal_load((const WNW_GLOBAL u32x4*)(k0 + (kl + 64 * i)));
          kr[1][i] = __builtin_nontemporal_load((const WNW_GLOBAL u32x4*)(k1 + (kl + 64 * i)));
        }
#pragma unroll
        for (int i = 0; i < VI; ++i) vr[i] = __builtin_nontemporal_load((const WNW_GLOBAL u32x4*)((i < VI / 2 ? v0 : v1) + (vl + (i % (VI / 2)) * 1024)));
      };
      // q, in the order of K's chunks
      u32x4 qf[KK];
      {
        const T* qp = (const T*)p.q + (int64_t)(r.first + ti) * p.qt + (int64_t)(r.h * p.G + c - ti * p.G) * p.qh;
#pragma unroll
        for (int i = 0; i < KK; ++i)
          qf[i] = cols > 0 ? *gptr<u32x4>(qp + (Q8 ? 16 * (lq + 4 * (i >> 1)) + 8 * (i & 1) : 8 * (lq + 4 * i)))
                                : u32x4{0, 0, 0, 0};
      }
      window(0);
      load(0);
#pragma unroll
      for (int i = 0; i < KK; ++i) qs[64 * i] = qf[i];
      for (int k = 0; k < mysteps; ++k) {
        const int row0 = (a + nw * k) * kPdStep;
        const bool edge = row0 + kPdStep > all_see || bad;
        const int bad_now = bad, from = 2 * (k & 31);
        // the 8 to 16 addresses made of these are worked out where they are used: held, they would cost registers
        asm volatile("" : "+v"(vput), "+v"(vget));
        // scores of the step's rows: lane holds rows 16 t + 4 lq + i of column lc
        float y[2][4];
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
          f32x4 z = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < KK; ++i) {
            if constexpr (Q8)
              z = QO::mma16(e4m3x8<T>(kr[t2][i >> 1][2 * (i & 1)], kr[t2][i >> 1][2 * (i & 1) + 1]), qs[64 * i], z);
            else
              z = QO::mma16(kr[t2][i], qs[64 * i], z);
          }
          const float sc = Q8 ? p.scale_log2 * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks), from + t2))
                              : p.scale_log2;
#pragma unroll
          for (int i = 0; i < 4; ++i) y[t2][i] = z[i] * sc;
        }
        __builtin_amdgcn_sched_barrier(0);
        // V into LDS; rows that are not the segment's become zero
        if (edge) {
#pragma unroll
          for (int i = 0; i < VI; ++i) {
            const int rr = (i * 1024 + lane * 16) / RB;
            if (row0 + rr >= n || (bad_now >> (rr >> 4) & 1)) vr[i] = u32x4{0, 0, 0, 0};
          }
          if (row0 + kPdStep > all_see && r.count > 1) {
            bool any = false;
#pragma unroll
            for (int i = 0; i < VI; ++i)
              if (row0 + (i * 1024 + lane * 16) / RB >= all_see) any |= take_odd<PE>(vr[i]);
            if (__ballot(any)) odd = 1;
          }
#pragma unroll
          for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (bad_now >> t2 & 1) y[t2][i] = 0.f;
              if (row0 + 16 * t2 + 4 * lq + i >= limit) y[t2][i] = -INFINITY;
            }
        }
#pragma unroll
        for (int i = 0; i < VI; ++i) *(u32x4*)(stage + ((vput ^ Vl::write_x(i)) + i * 1024)) = vr[i];
        const float w0 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), from));
        const float w1 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), from + 1));
        if (k + 1 < mysteps) {
          if (((k + 1) & 31) == 0) window(k + 1);
          load(k + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        float mx = m;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, y[t2][i]);
        mx = max_x32(max_x16(mx));
        if (__ballot(mx > m)) {
          const float fall = __builtin_amdgcn_exp2f(m - mx);
          l *= fall;
#pragma unroll
          for (int i = 0; i < DT; ++i) acc[i] *= fall;
          m = mx;
        }
        u32x4 hi, lo;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[t2][i] = __builtin_amdgcn_exp2f(y[t2][i] - m + kBias);
            l += y[t2][i];
            if (Q8) y[t2][i] *= t2 ? w1 : w0;
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t uh, ul;
            two_parts<VT>(y[t2][2 * i], y[t2][2 * i + 1], &uh, &ul);
            hi[2 * t2 + i] = uh;
            lo[2 * t2 + i] = ul;
          }
        }
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);
          u32x4 v;
          if constexpr (Q8) {
            typedef int i2 __attribute__((ext_vector_type(2)));
            const i2 z = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                (__attribute__((address_space(3))) i2*)(stage + (vget ^ Vl::read_x(i))));
            v = e4m3x8<VT>(z[0], z[1]);
          } else {
            const uint64_t z0 = VO::read_tr(stage + (vget ^ Vl::read_x(i)));
            const uint64_t z1 = VO::read_tr(stage + ((vget ^ Vl::read_x(i)) + 16 * RB));
            v = u32x4{(uint32_t)z0, (uint32_t)(z0 >> 32), (uint32_t)z1, (uint32_t)(z1 >> 32)};
          }
          acc[i] = VO::mma16(v, hi, acc[i]);
          acc[i] = VO::mma16(v, lo, acc[i]);
        }
        __builtin_amdgcn_wave_barrier();
      }
      if (odd) {
#pragma unroll 1
        for (int row = max(all_see, 0); row < n; ++row) {
          const int step = row / kPdStep - a;  // nw apart in the wave
          const uint8_t* from = step >= 0 && step % nw == 0 && row / kPdStep < b ? paged_v_row(p.c, seg, row, RB) : nullptr;
          if (!from || row >= limit) continue;
#pragma unroll
          for (int i = 0; i < DT; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            acc[i] += odd_quad<PE>(from, 16 * i + 4 * lq);
          }
        }
      }
      l = sum_x32(sum_x16(l));
      const int oq = here(lane) >> 4, oc = here(lane) & 15;
      if (oc < cols) {
        if (nw > 1) {  // the sums to LDS
          float* state = (float*)stage + oc * (D + 4) + 4 * oq;
#pragma unroll
          for (int i = 0; i < DT; ++i) *(f32x4*)(state + 16 * i) = acc[i];
          if (oq == 0) {
            st[w][oc][0] = m;
            st[w][oc][1] = l;
          }
        } else if (!(cut >> j & 1)) {  // the whole segment
#pragma unroll
          for (int i = 0; i < DT; ++i) paged_decode_out<T>(p, r, oc, 16 * i + 4 * oq, acc[i], l);
        } else {
          const int64_t slot = (int64_t)(2 * wg + (first_step + a == x0 ? 0 : 1)) * p.cols + oc;
#pragma unroll
          for (int i = 0; i < DT; ++i) {
            float* to = p.part_acc + slot * D + 16 * i + 4 * oq;
            store_agent(to, acc[i][0], acc[i][1]);
            store_agent(to + 2, acc[i][2], acc[i][3]);
          }
          if (oq == 0) store_agent(p.part_ml + slot * 2, m, l);
        }
      }
      __builtin_amdgcn_wave_barrier();
      if (beside)
        beside &= beside - 1;
      else
        own = 0;  // a wave has one at most
    }

    // pieces of several waves: their sums added up
    if (several) {
      __syncthreads();
      for (uint64_t todo = several; todo; todo &= todo - 1) {
        const int j = __builtin_ctzll(todo);
        const int f = __builtin_amdgcn_readlane(waves, j) & 255, t = __builtin_amdgcn_readlane(waves, j) >> 8;
        const DecodeRows r = decode_rows(p, win + j, __builtin_amdgcn_readlane(len, j));
        int a, b;
        const int slot = (2 * wg + (piece(j, &a, &b) + a == x0 ? 0 : 1)) * p.cols;
        for (int e = here(tid); e < r.cols * (D / 4); e += NT) {
          const int col = e / (D / 4), d = 4 * (e % (D / 4));
          float M = kPgLowest, L = 0.f;
          f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
          for (int i = f; i < t; ++i) {
            const float mi = st[i][col][0], now = fmaxf(M, mi);
            const float u = __builtin_amdgcn_exp2f(M - now), v = __builtin_amdgcn_exp2f(mi - now);
            L = L * u + v * st[i][col][1];
            o = o * u + v * *(const f32x4*)((const float*)(lds + i * Ge::kPart) + col * (D + 4) + d);
            M = now;
          }
          if (!(cut >> j & 1)) {
            paged_decode_out<T>(p, r, col, d, o, L);
          } else {
            float* to = p.part_acc + (slot + col) * D + d;
            store_agent(to, o[0], o[1]);
            store_agent(to + 2, o[2], o[3]);
            if (d == 0) store_agent(p.part_ml + (slot + col) * 2, M, L);
          }
        }
      }
    }
    // segments cut between workgroups: the last one to arrive adds up the pieces, in their order
    if (cut) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      const int j0 = __builtin_ctzll(cut), j1 = 63 - __builtin_clzll(cut);  // at most the first and the last piece
      int a, b;
      piece(j0, &a, &b);
      const int mine0 = b - a, all0 = __builtin_amdgcn_readlane(num, j0);
      piece(j1, &a, &b);
      const int mine1 = b - a, all1 = __builtin_amdgcn_readlane(num, j1);
      if (tid < 2 && (tid == 0 || j1 != j0)) {
        // the counter has the steps that are done
        int* counter = p.counters + win + (tid ? j1 : j0);
        const int add = tid ? mine1 : mine0;
        const int seen = __hip_atomic_fetch_add(counter, add, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool last = seen + add == (tid ? all1 : all0);
        if (last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sh[tid] = last;
      }
      __syncthreads();
#pragma unroll 1
      for (int i = 0; i < (j1 != j0 ? 2 : 1); ++i) {
        if (!sh[i]) continue;
        const int j = i ? j1 : j0, b0 = __builtin_amdgcn_readlane(at, j), w0 = owner_of(b0);
        paged_decode_gather<T, D, NT>(p, decode_rows(p, win + j, __builtin_amdgcn_readlane(len, j)), tid, b0 > start_of(w0), w0,
                                      owner_of(b0 + __builtin_amdgcn_readlane(num, j) - 1), (float*)lds);
      }
    }
    if (N <= 64) break;
    x = xe;
    at = __builtin_amdgcn_readlane(at + num, 63);
    win += 64;
    __syncthreads();  // the next window's waves write the LDS that this one's sums lie in
  }
  // segments without rows, or that cannot be read: zeros
  for (int s = wg; s < N; s += gridDim.x) {
    const int n = p.seg_len[s];
    if (tid == 0) {
      int first, count;
      if (!paged_tokens_of(p.t, s, &first, &count) || n < 0 || n > p.c.capacity) raise_device_error(p.err, WNW_DEVERR_BOUNDS);
    }
    if (steps_of(n) > 0) continue;
    const DecodeRows r = decode_rows(p, s, 0);
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    for (int e = here(tid); e < r.cols * (D / 4); e += NT) {
      const int col = e / (D / 4);
      store_quad<T>(out_row<T>(p, r, col, token_of(p, r, col)), 4 * (e % (D / 4)), zero);
    }
  }
}

// The counters' part of a workspace: the same for any number of segments up to
// 4,096, so that calls of different sizes can share one that was cleared once.
static int64_t counter_bytes(int64_t n_seg) { return (n_seg + 4095) / 4096 * 4096 * 4; }

struct PagedDecodeLayout {
  int64_t ml, acc, total;  // bytes: counters first
};
static int decode_grid(int D, bool q8) { return device_cus() * (D * (q8 ? 1 : 2) >= 256 ? 1 : 2); }
static PagedDecodeLayout decode_layout(int64_t n_seg, int64_t cols, int64_t D) {
  const int64_t slots = 2ll * 2 * device_cus();
  PagedDecodeLayout y;
  y.ml = counter_bytes(n_seg);
  y.acc = y.ml + (slots * cols * 8 + 255) / 256 * 256;
  y.total = y.acc + slots * cols * D * 4;
  return y;
}

template <typename T, int D>
static void launch_decode(const PagedDecodeParams& p, bool q8, int grid, hipStream_t st) {
  if (q8)
    hipLaunchKernelGGL((paged_decode_kernel<T, D, true>), dim3(grid), dim3(64 * PagedDecodeGeom<D, true>::kWaves), 0, st, p);
  else
    hipLaunchKernelGGL((paged_decode_kernel<T, D, false>), dim3(grid), dim3(64 * PagedDecodeGeom<D, false>::kWaves), 0, st, p);
}

// Shared with the prompt attention's entry point, which hands it the calls of a few tokens.
int paged_decode_launch(const wnw_paged_cache* cache, const int32_t* seg_len, const void* q, void* out, const int64_t* strides,
                        const PagedTokens& t, int64_t group, float scale, int dtype, void* workspace, int64_t bytes,
                        void* stream) {
  PagedDecodeParams p = {};
  if (int rc = paged_cache_of(cache, &p.c)) return rc;
  const int64_t N = cache->n_seg, D = cache->head_dim, cols = group * t.most;
  const PagedDecodeLayout y = decode_layout(N, cols, D);
  WNW_CHECK_ARG(workspace && bytes >= y.total, "workspace too small: %lld bytes, %lld needed", (long long)bytes,
                (long long)y.total);
  WNW_CHECK_ARG((uintptr_t)workspace % 256 == 0, "the workspace must be 256-byte aligned");
  const int64_t steps = N * ((p.c.capacity + kPdStep - 1) / kPdStep);
  WNW_CHECK_ARG(steps < (1ll << 31), "the page table names too many rows for one call");
  const bool q8 = cache->page_dtype == WNW_E4M3;
  p.t = t;
  p.seg_len = seg_len;
  p.q = q;
  p.out = out;
  p.qt = strides[0], p.qh = strides[1], p.ot = strides[2], p.oh = strides[3];
  p.counters = (int32_t*)workspace;
  p.part_ml = (float*)((uint8_t*)workspace + y.ml);
  p.part_acc = (float*)((uint8_t*)workspace + y.acc);
  p.scale_log2 = scale * kPgLog2e;
  p.G = (int32_t)group;
  p.cols = (int32_t)cols;
  p.err = device_error_word();
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(decode_grid((int)D, q8), steps / kPdMin + 1));
  hipStream_t st = (hipStream_t)stream;
  const bool bf = dtype == WNW_BF16;
  if (D == 64)
    bf ? launch_decode<bf16_t, 64>(p, q8, grid, st) : launch_decode<f16_t, 64>(p, q8, grid, st);
  else if (D == 128)
    bf ? launch_decode<bf16_t, 128>(p, q8, grid, st) : launch_decode<f16_t, 128>(p, q8, grid, st);
  else
    bf ? launch_decode<bf16_t, 256>(p, q8, grid, st) : launch_decode<f16_t, 256>(p, q8, grid, st);
  WNW_CHECK_HIP(hipGetLastError(), "paged attention launch");
  return WNW_OK;
}

// Whether out's rows [tokens, heads, D] overlap q's without being q itself, whose rows other workgroups may yet read.
bool paged_out_over_q(const void* q, const void* out, const int64_t* strides, int64_t tokens, int64_t heads, int64_t D) {
  const int64_t qt = tokens > 1 ? strides[0] : 0, qh = heads > 1 ? strides[1] : 0;
  const int64_t ot = tokens > 1 ? strides[2] : 0, oh = heads > 1 ? strides[3] : 0;
  const int64_t apart = ((intptr_t)out - (intptr_t)q) / 2;  // elements
  const bool alike = qt == ot && qh == oh;
  if (apart >= (tokens - 1) * qt + (heads - 1) * qh + D || -apart >= (tokens - 1) * ot + (heads - 1) * oh + D) return false;
  if (!alike || apart == 0) return !alike;
  for (int64_t h = 1 - heads; h < heads; ++h) {  // the nearest rows h heads apart
    const int64_t x = apart - h * qh, t = qt ? x / qt : 0;
    for (int64_t i = t - 1; i <= t + 1; ++i)
      if (i > -tokens && i < tokens && std::abs(x - i * qt) < D) return true;
  }
  return false;
}

// Checks of an attention call that the cache's own do not cover.
int paged_attn_check(const wnw_paged_cache* cache, const int32_t* seg_len, const void* q, const void* out,
                     const int64_t* strides, int64_t group, float scale, int dtype) {
  WNW_CHECK_ARG(dtype == WNW_BF16 || dtype == WNW_F16, "q must be bf16 or f16");
  WNW_CHECK_ARG(cache->page_dtype == WNW_E4M3 || cache->page_dtype == dtype, "16-bit pages must have the type of q");
  WNW_CHECK_ARG(seg_len && q && out && strides, "null pointer argument");
  WNW_CHECK_ARG(cache->n_pages > 0 || cache->max_blocks == 0, "a page table without pages");
  WNW_CHECK_ARG(group >= 1 && group <= 1024, "bad group");
  WNW_CHECK_ARG(scale > 0 && scale < INFINITY, "the scale must be positive");
  for (int i = 0; i < 4; ++i)
    WNW_CHECK_ARG(strides[i] >= 0 && strides[i] % 8 == 0 && strides[i] < (1ll << 40), "strides must be multiples of 8 elements");
  WNW_CHECK_ARG((uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0, "rows must be 16-byte aligned");
  return WNW_OK;
}

}  // namespace wnw

using namespace wnw;

extern "C" int64_t wnw_paged_counter_bytes(int64_t n_seg) {
  return n_seg < 0 || n_seg >= (1 << 24) ? -1 : counter_bytes(n_seg);
}

extern "C" int64_t wnw_paged_decode_workspace_bytes(int64_t n_seg, int64_t rows, int64_t head_dim) {
  if (n_seg < 0 || n_seg >= (1 << 24) || rows < 1 || rows > 16 || head_dim < 1 || head_dim > 256) return -1;
  return decode_layout(n_seg, rows, head_dim).total;
}

extern "C" int wnw_paged_decode_attn(const wnw_paged_cache* cache, const int32_t* seg_len, const void* q, void* out,
                                     int64_t group, float scale, int dtype, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
  WNW_CHECK_ARG(cache != nullptr, "the cache description is null");
  if (cache->n_seg == 0) return WNW_OK;
  const int64_t D = cache->head_dim;
  const int64_t strides[4] = {group * D, D, group * D, D};
  if (int rc = paged_attn_check(cache, seg_len, q, out, strides, group, scale, dtype)) return rc;
  WNW_CHECK_ARG(group <= 16, "at most 16 query heads per KV head (%lld)", (long long)group);
  WNW_CHECK_ARG(!paged_out_over_q(q, out, strides, cache->n_seg, group, D), "out covers a part of q");
  // every segment as a sample with one KV head and one token
  const PagedTokens t{nullptr, (int32_t)cache->n_seg, 1, 1};
  return paged_decode_launch(cache, seg_len, q, out, strides, t, group, scale, dtype, workspace, workspace_bytes, stream);
}
