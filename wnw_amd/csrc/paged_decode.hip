// Decode attention over the paged cache (gfx950): up to 16 query rows per
// segment (a group's heads, times the few tokens a sample may bring).
//
// Mathematics: per segment o = sum_t w_t v_t / sum_t w_t, w_t = 2^(s_t - m),
// s_t = scale log2(e) q . k_t, in one pass over the rows with the running
// maximum m; partial sums (m, l, o) of disjoint rows add up after a factor
// 2^(m' - m) each, so any split of the rows gives the same sums.
//
// Work split: the segments' rows in steps of 32 (no step crosses a segment),
// all steps cut evenly over the workgroups; a workgroup's steps of one segment
// are dealt to its four waves in turn.  The lengths are read on the device, so a
// captured launch stays right as segments grow.
//
// A step: S^T (rows x queries) = K Q^T with the rows' 16-byte chunks straight
// from memory as matrix operands (any order of the elements of a dot will do,
// if q has the same), V through LDS for its transpose (each wave its own part,
// no barrier), O^T += V^T P^T, whose P^T operand is S^T's own layout when V's
// rows follow its order.  The next step's rows are loaded while a step is used.
// 8-bit codes become 16-bit elements in registers (exact); K's scale
// multiplies the scores, V's scale the weights.  Weights go through two 16-bit
// parts (the upper cut off, not rounded, and neither ever zero, so that an
// infinity in V stays one): 16 bits of each, beside 32-bit sums.
#include <algorithm>
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
static constexpr int kPdWaves = 4;
static constexpr int kPdMin = 4;    // steps of a workgroup at least

template <int D, bool Q8>
struct PagedDecodeGeom {
  static constexpr int RB = D * (Q8 ? 1 : 2);  // bytes of a row
  static constexpr int KC = RB / 64;           // 16-byte chunks of a K row per lane
  static constexpr int VI = kPdStep * RB / 1024;  // loads of a step's V per lane
  static constexpr int kStage = kPdStep * RB;     // LDS of a wave's V
  static constexpr int kState = 16 * (D + 4) * 4; // LDS of a wave's sums
  static constexpr int kLds = kPdWaves * (kStage > kState ? kStage : kState);
  // workgroups per CU
  static constexpr int kWgs = D == 256 ? 2 : Q8 || D == 64 ? 4 : 3;
};

// Row r's 16-byte chunk c of a step's V in LDS.  The transposed reads take 8
// rows of one chunk (8 bits: rows 4 q .. + 3 and 16 + 4 q .. + 3) or 4 rows of
// two chunks (16 bits) at a time: both without bank conflicts.
template <int D, bool Q8>
__device__ __forceinline__ int v_at(int r, int c) {
  constexpr int RB = PagedDecodeGeom<D, Q8>::RB;
  if constexpr (!Q8) return r * RB + ((c ^ (2 * (r & 3))) * 16);
  const int f = (r & 3) | ((r >> 4) & 1) << 2;
  return r * RB + ((c ^ (RB == 64 ? f >> 1 : f)) * 16);
}

// Two positive values as two pairs of 16-bit parts
template <typename T>
__device__ __forceinline__ void two_parts(float a, float b, uint32_t* hi, uint32_t* lo) {
  if constexpr (std::is_same<T, bf16_t>::value) {
    const uint32_t ua = __float_as_uint(a) & 0xffff0000u, ub = __float_as_uint(b) & 0xffff0000u;
    *hi = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
    const float la = fmaxf(a - __uint_as_float(ua), 7.888609e-31f), lb = fmaxf(b - __uint_as_float(ub), 7.888609e-31f);
    *lo = __builtin_amdgcn_perm(__float_as_uint(lb), __float_as_uint(la), 0x07060302u);
  } else {
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    *hi = __builtin_bit_cast(uint32_t, h);
    const float la = fmaxf(a - (float)h[0], 5.9604645e-8f), lb = fmaxf(b - (float)h[1], 5.9604645e-8f);
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

template <typename T, int D, bool Q8>
__global__ __launch_bounds__(256, (PagedDecodeGeom<D, Q8>::kWgs)) void paged_decode_kernel(PagedDecodeParams p) {
  using Ge = PagedDecodeGeom<D, Q8>;
  using VT = typename std::conditional<Q8, bf16_t, T>::type;  // the value product's type: any scale fits bf16
  using QO = HalfOps<T>;
  using VO = HalfOps<VT>;
  constexpr int RB = Ge::RB, KC = Ge::KC, VI = Ge::VI, DT = D / 16, KK = D / 32;
  // weights of f16 are held times 2^12: their lower parts reach 2^-36 of the largest
  constexpr float kBias = std::is_same<VT, f16_t>::value ? 12.f : 0.f;
  __shared__ __attribute__((aligned(16))) uint8_t lds[Ge::kLds];
  __shared__ float st[kPdWaves][16][2];
  __shared__ int32_t sh[8];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lq = lane >> 4, lc = lane & 15;
  const int N = p.c.n_seg, wg = blockIdx.x;

  auto steps_of = [&](int s) {
    const int n = p.seg_len[s];
    return n >= 0 && n <= p.c.capacity ? (n + kPdStep - 1) / kPdStep : 0;
  };
  // all steps, and where this workgroup's begin
  const int per = (N + 255) / 256;
  const int sa = min(tid * per, N), sb = min(sa + per, N);
  int mine = 0;
  for (int s = sa; s < sb; ++s) mine += steps_of(s);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 63) sh[w] = incl;
  __syncthreads();
  int before = 0, S = 0;
#pragma unroll
  for (int i = 0; i < kPdWaves; ++i) {
    if (i < w) before += sh[i];
    S += sh[i];
  }
  S = __builtin_amdgcn_readfirstlane(S);
  const int P = min((int)gridDim.x, max(S / kPdMin, 1));
  const int share = S / P, more = S - share * P;  // the first `more` workgroups take one step more
  auto start_of = [&](int i) { return i * share + min(i, more); };
  auto owner_of = [&](int x) {  // the workgroup that has step x
    const int big = more * (share + 1);
    return x < big ? x / (share + 1) : more + (x - big) / max(share, 1);
  };
  const int x0 = wg < P ? start_of(wg) : 0, x1 = wg < P ? start_of(wg + 1) : 0;
  if (x0 < x1) {
    int e = before + incl - mine;  // steps before the thread's segments
    if (e <= x0 && x0 < e + mine) {
      int s = sa;
      for (int n; e + (n = steps_of(s)) <= x0; ++s) e += n;
      sh[4] = s;
      sh[5] = e;
    }
  }
  __syncthreads();
  int seg = __builtin_amdgcn_readfirstlane(sh[4]), base = __builtin_amdgcn_readfirstlane(sh[5]);

  for (int x = x0; x < x1 && seg < N; ++seg) {
    const int len = p.seg_len[seg], ns = steps_of(seg);
    if (ns == 0) continue;
    const int a = x - base, b = min(ns, x1 - base);  // the piece: steps [a, b) of the segment
    int first, count;
    paged_tokens_of(p.t, seg, &first, &count);
    const int h = seg % p.t.hkv;
    const int cols = min(count * p.G, p.cols);
    const int c = min(lc, max(cols - 1, 0)), ti = c / p.G, g = c - ti * p.G;
    const int limit = len - count + ti + 1;           // rows that the lane's column sees
    const int all_see = len - count + 1;              // rows that every column sees
    // q, in the order of K's chunks
    u32x4 qf[KK];
    {
      const T* qp = (const T*)p.q + (int64_t)(first + ti) * p.qt + (int64_t)(h * p.G + g) * p.qh;
#pragma unroll
      for (int i = 0; i < KK; ++i) {
        const int d = Q8 ? 16 * (lq + 4 * (i >> 1)) + 8 * (i & 1) : 8 * (lq + 4 * i);
        qf[i] = cols > 0 ? *gptr<u32x4>(qp + d) : u32x4{0, 0, 0, 0};
      }
    }
    f32x4 acc[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = kPgLowest, l = 0.f;
    const int mysteps = (b - a - w + kPdWaves - 1) / kPdWaves;  // this wave's: a + w + 4 k
    uint8_t* stage = lds + w * (Ge::kLds / kPdWaves);

    // a window of 32 steps' pages: lane l has the page of half l & 1 of step l / 2
    int pid = -1;
    float ks = 1.f, vs = 1.f;
    auto window = [&](int k0) {
      const int step = a + w + kPdWaves * (k0 + (lane >> 1));
      const int row = step * kPdStep + 16 * (lane & 1);
      pid = -1;
      if (step < b && row < len) {
        pid = p.c.table[seg * p.c.table_stride + (row >> p.c.shift)];
        if (pid < 0 || pid >= p.c.n_pages) {
          raise_device_error(p.err, WNW_DEVERR_BOUNDS);
          pid = -1;
        }
        if (Q8 && pid >= 0) {
          ks = p.c.k_scale[pid];
          vs = p.c.v_scale[pid];
        }
      }
    };
    u32x4 kr[2][KC], vr[VI];
    float ks0, ks1, vs0, vs1;  // of the step whose rows are in kr and vr
    int bad = 0;               // halves of that step that no page holds
    auto load = [&](int k) {
      const int at = 2 * (k & 31);
      const int step = a + w + kPdWaves * k;
      const int p0 = __builtin_amdgcn_readlane(pid, at), p1 = __builtin_amdgcn_readlane(pid, at + 1);
      if (Q8) {
        ks0 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks), at));
        ks1 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks), at + 1));
        vs0 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), at));
        vs1 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), at + 1));
      }
      bad = (p0 < 0 ? 1 : 0) | (p1 < 0 ? 2 : 0);
      const int in = (step * kPdStep) & ((1 << p.c.shift) - 1);             // first row in its page
      const int in1 = (step * kPdStep + 16) & ((1 << p.c.shift) - 1);
      const int r0 = p0 < 0 ? (p1 < 0 ? 0 : p1) : p0, r1 = p1 < 0 ? r0 : p1;  // a half in no page reads the other's
      const uint8_t* k0 = p.c.k + (int64_t)r0 * p.c.k_stride + (p0 < 0 ? 0 : in) * RB;
      const uint8_t* k1 = p.c.k + (int64_t)r1 * p.c.k_stride + (p1 < 0 ? 0 : in1) * RB;
      const uint8_t* v0 = p.c.v + (int64_t)r0 * p.c.v_stride + (p0 < 0 ? 0 : in) * RB;
      const uint8_t* v1 = p.c.v + (int64_t)r1 * p.c.v_stride + (p1 < 0 ? 0 : in1) * RB;
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        kr[0][i] = *gptr<u32x4>(k0 + lc * RB + (lq + 4 * i) * 16);
        kr[1][i] = *gptr<u32x4>(k1 + lc * RB + (lq + 4 * i) * 16);
      }
#pragma unroll
      for (int i = 0; i < VI; ++i) vr[i] = *gptr<u32x4>((i < VI / 2 ? v0 : v1) + (i % (VI / 2)) * 1024 + lane * 16);
    };
    if (mysteps > 0) {
      window(0);
      load(0);
    }
    for (int k = 0; k < mysteps; ++k) {
      const int row0 = (a + w + kPdWaves * k) * kPdStep;
      const bool edge = row0 + kPdStep > all_see || bad;
      const int bad_now = bad;
      // scores of the step's rows: lane holds rows 16 t + 4 lq + i of column lc
      float x[2][4];
      {
        const float s0 = Q8 ? p.scale_log2 * ks0 : p.scale_log2, s1 = Q8 ? p.scale_log2 * ks1 : p.scale_log2;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x4 y = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < KK; ++i) {
            if constexpr (Q8)
              y = QO::mma16(e4m3x8<T>(kr[t][i >> 1][2 * (i & 1)], kr[t][i >> 1][2 * (i & 1) + 1]), qf[i], y);
            else
              y = QO::mma16(kr[t][i], qf[i], y);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) x[t][i] = y[i] * (t ? s1 : s0);
        }
      }
      // V into LDS; rows that are not the segment's become zero
      if (edge) {
#pragma unroll
        for (int i = 0; i < VI; ++i) {
          const int r = (i * 1024 + lane * 16) / RB;
          if (row0 + r >= len || (bad_now >> (r >> 4) & 1)) vr[i] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (bad_now >> t & 1) x[t][i] = 0.f;
            if (row0 + 16 * t + 4 * lq + i >= limit) x[t][i] = -INFINITY;
          }
      }
#pragma unroll
      for (int i = 0; i < VI; ++i) {
        const int at = i * 1024 + lane * 16;
        *(u32x4*)(stage + v_at<D, Q8>(at / RB, at % RB / 16)) = vr[i];
      }
      const float w0 = vs0, w1 = vs1;
      if (k + 1 < mysteps) {
        if (((k + 1) & 31) == 0) window(k + 1);
        load(k + 1);
      }
      float mx = m;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, x[t][i]);
      mx = max_x32(max_x16(mx));
      if (__ballot(mx > m)) {
        const float f = __builtin_amdgcn_exp2f(m - mx);
        l *= f;
#pragma unroll
        for (int i = 0; i < DT; ++i) acc[i] *= f;
        m = mx;
      }
      u32x4 hi, lo;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[i] = __builtin_amdgcn_exp2f(x[t][i] - m + kBias);
          l += y[i];
          if (Q8) y[i] *= t ? w1 : w0;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t uh, ul;
          two_parts<VT>(y[2 * i], y[2 * i + 1], &uh, &ul);
          hi[2 * t + i] = uh;
          lo[2 * t + i] = ul;
        }
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        u32x4 v;
        if constexpr (Q8) {
          typedef int i2 __attribute__((ext_vector_type(2)));
          const int r = 4 * lq + (lc >> 1 & 3) + (lc >> 3) * 16;
          const i2 y = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
              (__attribute__((address_space(3))) i2*)(stage + v_at<D, true>(r, i) + (lc & 1) * 8));
          v = e4m3x8<VT>(y[0], y[1]);
        } else {
          const int r = 4 * lq + (lc >> 2), ch = 2 * i + ((lc & 3) >> 1);
          const uint64_t y0 = VO::read_tr(stage + v_at<D, false>(r, ch) + (lc & 1) * 8);
          const uint64_t y1 = VO::read_tr(stage + v_at<D, false>(r + 16, ch) + (lc & 1) * 8);
          v = u32x4{(uint32_t)y0, (uint32_t)(y0 >> 32), (uint32_t)y1, (uint32_t)(y1 >> 32)};
        }
        acc[i] = VO::mma16(v, hi, acc[i]);
        acc[i] = VO::mma16(v, lo, acc[i]);
      }
      __builtin_amdgcn_wave_barrier();
    }
    // the waves' sums through LDS
    l = sum_x32(sum_x16(l));
    __syncthreads();
    {
      float* state = (float*)stage + lc * (D + 4) + 4 * lq;
      if (lc < cols) {
#pragma unroll
        for (int i = 0; i < DT; ++i) *(f32x4*)(state + 16 * i) = acc[i];
        if (lq == 0) {
          st[w][lc][0] = m;
          st[w][lc][1] = l;
        }
      }
    }
    __syncthreads();
    const bool whole = a == 0 && b == ns;
    const int slot = 2 * wg + (a > 0 || x == x0 ? 0 : 1);  // the first or the last piece of the workgroup
    auto finish = [&](int col, int d, float* o, float L) {
      const int t2 = col / p.G;
      const bool none = len - count + t2 + 1 <= 0;  // a row that sees no key
      const float inv = 1.f / L;
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = none ? 0.f : o[i] * inv;
      T* op = (T*)p.out + (int64_t)(first + t2) * p.ot + (int64_t)(h * p.G + col - t2 * p.G) * p.oh;
      store_quad<T>(op, d, y);
    };
    for (int e = tid; e < cols * (D / 4); e += 256) {
      const int col = e / (D / 4), d = 4 * (e % (D / 4));
      float M = kPgLowest, L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kPdWaves; ++i) M = fmaxf(M, st[i][col][0]);
#pragma unroll
      for (int i = 0; i < kPdWaves; ++i) {
        const float f = __builtin_amdgcn_exp2f(st[i][col][0] - M);
        const f32x4 y = *(const f32x4*)((const float*)(lds + i * (Ge::kLds / kPdWaves)) + col * (D + 4) + d);
        L += f * st[i][col][1];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += f * y[j];
      }
      if (whole) {
        finish(col, d, o, L);
      } else {
        float* pa = p.part_acc + ((int64_t)slot * p.cols + col) * D + d;
        store_agent(pa, o[0], o[1]);
        store_agent(pa + 2, o[2], o[3]);
        if (d == 0) store_agent(p.part_ml + ((int64_t)slot * p.cols + col) * 2, M, L);
      }
    }
    if (!whole) {
      // the last workgroup to arrive at a segment adds up its pieces, in their order
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      const int w0 = owner_of(base), w1 = owner_of(base + ns - 1);
      if (tid == 0) {
        const int seen = __hip_atomic_fetch_add(p.counters + seg, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sh[6] = seen == w1 - w0;
        if (seen == w1 - w0) __hip_atomic_store(p.counters + seg, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
      if (sh[6]) {
        for (int e = tid; e < cols * (D / 4); e += 256) {
          const int col = e / (D / 4), d = 4 * (e % (D / 4));
          float M = kPgLowest, L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
          for (int i0 = w0; i0 <= w1; i0 += 8) {
            float pm[8], pl[8], po[8][4];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int from = min(i0 + i, w1);
              const int64_t sl = (int64_t)(2 * from + (base > start_of(from) ? 1 : 0)) * p.cols + col;
              load_agent(p.part_ml + sl * 2, &pm[i], &pl[i]);
              load_agent(p.part_acc + sl * D + d, &po[i][0], &po[i][1]);
              load_agent(p.part_acc + sl * D + d + 2, &po[i][2], &po[i][3]);
            }
            float now = M;
#pragma unroll
            for (int i = 0; i < 8; ++i) now = fmaxf(now, pm[i]);
            const float f0 = __builtin_amdgcn_exp2f(M - now);
            L *= f0;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] *= f0;
            M = now;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (i0 + i > w1) continue;
              const float f = __builtin_amdgcn_exp2f(pm[i] - M);
              L += f * pl[i];
#pragma unroll
              for (int j = 0; j < 4; ++j) o[j] += f * po[i][j];
            }
          }
          finish(col, d, o, L);
        }
      }
    }
    __syncthreads();  // the next piece writes the LDS that this one's sums lie in
    x += b - a;
    base += ns;
  }
  // segments without rows, or that cannot be read: zeros
  for (int s = wg; s < N; s += gridDim.x) {
    const int len = p.seg_len[s];
    int first, count;
    const bool told = paged_tokens_of(p.t, s, &first, &count);
    if (tid == 0 && (!told || len < 0 || len > p.c.capacity)) raise_device_error(p.err, WNW_DEVERR_BOUNDS);
    if (steps_of(s) > 0) continue;
    const int h = s % p.t.hkv, cols = min(count * p.G, p.cols);
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    for (int e = tid; e < cols * (D / 4); e += 256) {
      const int col = e / (D / 4), t2 = col / p.G;
      store_quad<T>((T*)p.out + (int64_t)(first + t2) * p.ot + (int64_t)(h * p.G + col - t2 * p.G) * p.oh, 4 * (e % (D / 4)),
                    zero);
    }
  }
}

// The counters' part of a workspace: the same for any number of segments up to
// 4,096, so that calls of different sizes can share one that was cleared once.
static int64_t counter_bytes(int64_t n_seg) { return (n_seg + 4095) / 4096 * 4096 * 4; }

struct PagedDecodeLayout {
  int64_t ml, acc, total;  // bytes: counters first
};
static int decode_grid(int D, bool q8) {
  const int per = D == 256 ? 2 : q8 || D == 64 ? 4 : 3;
  return device_cus() * per;
}
static PagedDecodeLayout decode_layout(int64_t n_seg, int64_t cols, int64_t D) {
  const int64_t slots = 2ll * 4 * device_cus();
  PagedDecodeLayout y;
  y.ml = counter_bytes(n_seg);
  y.acc = y.ml + (slots * cols * 8 + 255) / 256 * 256;
  y.total = y.acc + slots * cols * D * 4;
  return y;
}

template <typename T, int D>
static void launch_decode(const PagedDecodeParams& p, bool q8, int grid, hipStream_t st) {
  if (q8)
    hipLaunchKernelGGL((paged_decode_kernel<T, D, true>), dim3(grid), dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((paged_decode_kernel<T, D, false>), dim3(grid), dim3(256), 0, st, p);
}

// Shared with the prompt attention's entry point, which hands it the calls of a few tokens.
int paged_decode_launch(const wnw_paged_cache* cache, const int32_t* seg_len, const void* q, void* out, const int64_t* strides,
                        const PagedTokens& t, int64_t group, float scale, int dtype, void* workspace, int64_t bytes,
                        void* stream) {
  PagedDecodeParams p = {};
  if (int rc = paged_cache_of(cache, false, &p.c)) return rc;
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
  // every segment as a sample with one KV head and one token
  const PagedTokens t{nullptr, (int32_t)cache->n_seg, 1, 1};
  return paged_decode_launch(cache, seg_len, q, out, strides, t, group, scale, dtype, workspace, workspace_bytes, stream);
}
