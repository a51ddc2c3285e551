// Prompt attention over the paged cache (gfx950): the tokens of a prompt or of
// a chunk of one, each against the rows up to its own.
//
// Mathematics: as decode attention, causal: token i of a sample's n sees the
// segment's first len - n + i + 1 rows.
//
// A workgroup takes 128 or 256 query rows of one segment, a row being (token,
// head of the group): the group shares the keys.  A wave has 32 of them and
// walks the 64-key tiles up to its last row's:
//   S^T (64 keys x 32 queries) = K Q^T, Q in registers, K from LDS;
//   O^T (D x 32) += V^T P^T, the weights in 16 bits (f16's held times 2^8), their
//       sum in 32, V^T by transposed LDS reads in S^T's own order.
// The weights are relative to the running maximum itself: one that trails it by
// a bounded factor saved the rescaling of O (2 %), but its weights above 1 cost a
// quarter more of the 16-bit rounding.
// The tiles go through registers into LDS, where 8-bit codes become 16-bit
// elements once for all waves; one barrier per tile, the next tile written among
// the products of S and the one after it loaded then (head_dim 256: one buffer,
// two barriers).  K's page scale multiplies the exponent, V's is added to it as
// its logarithm (a part of 2^x either way), so that scales cost a few
// instructions per 16 keys.  Such weights are held in bf16, whose exponents reach
// from the append's least scale, 2^-64, to its largest, 2^120: no page but a
// query's own has a say in how its weights are held.  f16 queries, whose weights
// have 11 bits over 16-bit pages, have two parts of 8 here (2,048 tokens at
// head_dim 64 and 128: 46.8 and 71.2 us, bf16 queries 40.7 and 60.2).
//
// Few query rows and many keys: the tiles of each block of rows are cut into
// splits, whose sums a second launch adds up.
//
// What bounds it: the instructions.  Per tile and wave at head_dim 128 the products
// take 1,024 cycles of the matrix unit, 32 exponentials 512 and about 230 other
// vector instructions 920, and on one SIMD these add up: 4,564 tokens take 442,000
// cycles, for 37 % of which matrix instructions run and for 51 % vector ones.  That
// is 196 to 211 us a pass (by the card) where passes have pauses between them, 0.8
// to 0.87 PFLOP/s (plain bf16 products of size 8,192: 1.2), and 233 us in a row of
// 24, over which the clock falls to 2.1 GHz or less.
// Without gain: half of the waves a phase behind the others, so that one's
// products meet the other's exponentials (8 % slower in one loop); the next tile's
// scores among the exponentials (2 to 5 % slower); loads two tiles ahead; raised
// wave priority in the products.
#include <algorithm>
#include <type_traits>

#include "paged.h"

namespace wnw {

typedef float f32x16 __attribute__((ext_vector_type(16)));

int paged_decode_launch(const wnw_paged_cache* cache, const int32_t* seg_len, const void* q, void* out, const int64_t* strides,
                        const PagedTokens& t, int64_t group, float scale, int dtype, void* workspace, int64_t bytes,
                        void* stream);
int paged_attn_check(const wnw_paged_cache* cache, const int32_t* seg_len, const void* q, const void* out,
                     const int64_t* strides, int64_t group, float scale, int dtype);
bool paged_out_over_q(const void* q, const void* out, const int64_t* strides, int64_t tokens, int64_t heads, int64_t D);

struct PagedPromptParams {
  PagedCache c;
  PagedTokens t;
  const int32_t* seg_len;
  const void* q;
  void* out;
  int64_t qt, qh, ot, oh;  // strides in elements
  float* part;             // [blocks, splits, waves]: D / 32 x 16 sums a lane, then max, sum
  float scale_log2;
  int32_t G, nqb, splits;
  int32_t* err;
};

static constexpr int kPpKeys = 64;  // keys of a tile

template <typename T>
__device__ __forceinline__ f32x16 mma32(const u32x4& a, const u32x4& b, const f32x16& c) {
  if constexpr (std::is_same<T, bf16_t>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// What a workgroup's rows are.
struct PromptRows {
  int first, count, len, rows;  // the sample's tokens, the segment's rows, query rows
};
__device__ __forceinline__ PromptRows prompt_rows(const PagedPromptParams& p, int seg, bool tell) {
  PromptRows r;
  const bool told = paged_tokens_of(p.t, seg, &r.first, &r.count);
  r.len = p.seg_len[seg];
  const bool good = r.len >= 0 && r.len <= p.c.capacity;
  if (tell && (!told || !good)) raise_device_error(p.err, WNW_DEVERR_BOUNDS);
  if (!good) r.len = 0;
  r.rows = r.count * p.G;
  return r;
}

// Into how many splits a block's tiles are cut, of the most that the launch has: by
// the block's own tiles, as the table that the launch was planned for may be far
// wider than the segments are long (100 tokens in a table of 25,000 rows: 14 us, cut
// by the table 26; 64 tokens after 500 rows 19 and 26, with pieces of 4 tiles or
// more 21).
__device__ __forceinline__ int splits_of(int tiles, int most) { return max(min(tiles / 2, most), 1); }
// Tiles that a block of query rows walks
template <int W>
__device__ __forceinline__ int tiles_of(const PagedPromptParams& p, const PromptRows& r, int qblk) {
  const int last = r.len - r.count + 1 + min(32 * W * (qblk + 1) - 1, r.rows - 1) / p.G;  // rows that its last one sees
  return max((last + kPpKeys - 1) / kPpKeys, 0);
}

// The wave's rows out, 32-element parts dt0 .. dt0 + NT - 1: lane (hi, n) has
// elements 32 i + 8 j + 4 hi + 0..3 of row n
template <typename T, int NT>
__device__ __forceinline__ void prompt_store(const PagedPromptParams& p, const PromptRows& r, int row, int h, int hi, int dt0,
                                             const f32x16* o, float l) {
  if (row >= r.rows) return;
  const int i = row / p.G, g = row - i * p.G;
  T* op = (T*)p.out + (int64_t)(r.first + i) * p.ot + (int64_t)(h * p.G + g) * p.oh;
  const bool none = r.len - r.count + i + 1 <= 0;
  const float inv = 1.0f / l;
#pragma unroll
  for (int dt = 0; dt < NT; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = none ? 0.f : o[dt][4 * j + e] * inv;
      store_quad<T>(op, 32 * (dt0 + dt) + 8 * j + 4 * hi, y);
    }
}

// Registers for at most 3 waves per SIMD: made to fit 4, head_dim 64 over 8 bits takes 43.5 us for 40.7 (2,048 tokens).
template <typename T, int D, bool Q8, int W>
__global__ __launch_bounds__((64 * W)) __attribute__((amdgpu_waves_per_eu((D == 256 && !Q8 ? 1 : 2), (D == 256 && !Q8 ? 1 : 3)))) void
paged_prompt_kernel(PagedPromptParams p) {
  using VT = typename std::conditional<Q8, bf16_t, T>::type;   // the value product's type
  using VO = HalfOps<VT>;
  using PE = typename std::conditional<Q8, uint8_t, T>::type;  // the pages' elements
  constexpr int kPpQ = 32 * W;
  constexpr int RB = D * 2, CH = RB / 16, TB = kPpKeys * RB;  // a tile in LDS: 16-bit elements
  constexpr int GB = D * (Q8 ? 1 : 2);                        // bytes of a row in its page
  constexpr int NI = kPpKeys * GB / (1024 * W);                     // 16-byte loads per thread and tensor
  constexpr int KK = D / 16, DT = D / 32;
  constexpr int NB = D == 256 ? 1 : 2;  // tiles in LDS
  constexpr bool kAhead = D != 256 || !Q8;  // the next tile's loads are on their way during the products
  // f16 weights are held times 2^8: normal numbers down to 2^-22 of the largest;
  // bf16 ones times 2^-16: 2^16 times the type's largest value is a sum yet
  constexpr float kBias = std::is_same<VT, f16_t>::value ? 8.f : -16.f;
  constexpr bool kTwo = Q8 && std::is_same<T, f16_t>::value;  // weights of two parts
  __shared__ __attribute__((aligned(16))) uint8_t lds[NB * 2 * TB];  // [NB][K, V]
  __shared__ int odd;  // V had infinities or NaN in such a tile
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hi = lane >> 5, n = lane & 31;
  const int N = p.c.n_seg;
  // the blocks with the most tiles first; workgroups of one segment N apart (8 segments: each in one L2)
  const int seg = blockIdx.x % N, rank = blockIdx.x / N;
  const int block = rank / p.splits, split = rank - block * p.splits, qblk = p.nqb - 1 - block;
  const PromptRows r = prompt_rows(p, seg, tid == 0 && qblk == 0 && split == 0);
  if (qblk * kPpQ >= r.rows) return;
  const int h = seg % p.t.hkv;
  const int base = r.len - r.count + 1;  // token i sees base + i rows
  const int row = qblk * kPpQ + 32 * w + n;
  const int ri = min(row, r.rows - 1) / p.G, rg = min(row, r.rows - 1) - ri * p.G;
  const int limit = base + ri;
  // rows that the wave's first and last query see
  const int wfirst = base + min(qblk * kPpQ + 32 * w, r.rows - 1) / p.G;
  const int wlast = base + min(qblk * kPpQ + 32 * w + 31, r.rows - 1) / p.G;
  const int first = base + qblk * kPpQ / p.G;  // and the workgroup's first
  const int tiles = tiles_of<W>(p, r, qblk), splits = splits_of(tiles, p.splits);
  if (split >= splits) return;
  const int t0 = (int)((int64_t)tiles * split / splits), t1 = (int)((int64_t)tiles * (split + 1) / splits);
  const bool busy = qblk * kPpQ + 32 * w < r.rows;  // a wave without rows only moves tiles
  const int mine = busy ? min(t1, (wlast + kPpKeys - 1) / kPpKeys) : t0;  // the wave's tiles end here
  u32x4 qr[KK];
  {
    const T* qp = (const T*)p.q + (int64_t)(r.first + ri) * p.qt + (int64_t)(h * p.G + rg) * p.qh + 8 * hi;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qr[kk] = *gptr<u32x4>(qp + 16 * kk);
  }
  // Staging: a wave's load is 16 bytes of each of 64 / CG (2 to 16) rows that
  // lie in one page, so a load's page and its address are scalars.  They come
  // from a window of 64 x 16 keys (16 tiles) that a wave keeps in registers: lane j
  // has the page, and K's and V's scale, of keys 16 j ...  The next window's
  // pages are loaded when a window is entered, its scales half way through.
  constexpr int CG = GB / 16;     // 16-byte chunks of a row in its page
  constexpr int RPL = 64 * W / CG;   // rows per load of the workgroup
  constexpr int kWin = 16;        // tiles of a window
  const int srow = tid / CG, sch = tid % CG;
  // 8 bits: a lane has 8 codes of either half of a row, so that what it writes,
  // a 16-byte chunk of 16-bit elements each, meets every LDS bank once per row
  uint32_t soff = (uint32_t)((lane / CG) * GB + sch * (Q8 ? 8 : 16));
  // the lane's place in a tile's K and V in LDS (load u: u * RPL rows on); K's
  // second half has the chunk's top bit turned, V's lies half a row on
  constexpr uint32_t kHalf = RB / 2;
  static_assert(RPL % 4 == 0 && (RPL % CH == 0 || CH % RPL == 0), "rows of a load: whole turns of the swizzle, or a part of one");
  uint32_t kput = srow * RB + ((sch ^ (srow % CH)) * 16), vput = srow * RB + ((sch ^ (2 * (srow & 3))) * 16);
  const int32_t* table = p.c.table + seg * p.c.table_stride;
  int pid = 0, pid_next = 0;  // of the window that fetch() is in, and of the next
  float ks = 1.f, vs = 1.f, ks_next = 1.f, vs_next = 1.f;
  bool wrong = false;
  // Rows past the segment's take its last page; an entry that is no page page
  // 0, with its sign bit set.
  auto find = [&](int window) {
    const int id = table[min((window * 64 + lane) * 16, r.len - 1) >> p.c.shift];
    const bool is = (uint32_t)id < (uint32_t)p.c.n_pages;
    wrong |= !is;
    pid_next = is ? id : (int)0x80000000;
  };
  auto find_scales = [&]() {
    if constexpr (Q8) {
      const int id = pid_next & 0x7fffffff;
      ks_next = pid_next < 0 ? 1.f : p.c.k_scale[id];
      vs_next = pid_next < 0 ? 1.f : p.c.v_scale[id];
    }
  };
  auto enter = [&](int window) {
    pid = pid_next;
    ks = ks_next;
    vs = vs_next;
    find(window + 1);
  };
  u32x4 kr[NI], vr[NI];
  int gone[NI];  // rows of kr and vr in no page: negative
  auto fetch = [&](int tile) {
    if (tile % kWin == 0)
      enter(tile / kWin);
    else if (tile % kWin == kWin / 2)
      find_scales();
    const int in = (1 << p.c.shift) - 1;
    typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
    soff = here(soff);
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      const int row = tile * kPpKeys + u * RPL + w * (64 / CG);
      const int id = __builtin_amdgcn_readlane(pid, (row >> 4) & 63);
      const int64_t page = id & 0x7fffffff;
      const WNW_GLOBAL uint8_t* kp = gptr<uint8_t>(p.c.k) + (page * p.c.k_stride + (row & in) * GB);
      const WNW_GLOBAL uint8_t* vp = gptr<uint8_t>(p.c.v) + (page * p.c.v_stride + (row & in) * GB);
      if constexpr (Q8) {
        const u32x2_t k0 = *(const WNW_GLOBAL u32x2_t*)(kp + soff), k1 = *(const WNW_GLOBAL u32x2_t*)(kp + (soff + GB / 2));
        const u32x2_t v0 = *(const WNW_GLOBAL u32x2_t*)(vp + soff), v1 = *(const WNW_GLOBAL u32x2_t*)(vp + (soff + GB / 2));
        kr[u] = u32x4{k0[0], k0[1], k1[0], k1[1]};
        vr[u] = u32x4{v0[0], v0[1], v1[0], v1[1]};
      } else {
        kr[u] = *(const WNW_GLOBAL u32x4*)(kp + soff);
        vr[u] = *(const WNW_GLOBAL u32x4*)(vp + soff);
      }
      gone[u] = id;
    }
  };
  auto clear = [&](int tile) {  // rows of kr and vr that are not the segment's
    int any = (tile + 1) * kPpKeys > r.len;
#pragma unroll
    for (int u = 0; u < NI; ++u) any |= gone[u] < 0;
    if (!any) return;
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      if (gone[u] < 0) kr[u] = u32x4{0, 0, 0, 0};
      if (gone[u] < 0 || tile * kPpKeys + u * RPL + srow >= r.len) vr[u] = u32x4{0, 0, 0, 0};
    }
  };
  // takes infinities and NaN out of the V of a tile that not every row of the workgroup sees whole
  auto even = [&](int tile) {
    if ((tile + 1) * kPpKeys <= first) return;
    bool any = false;
#pragma unroll
    for (int u = 0; u < NI; ++u) any |= take_odd<PE>(vr[u]);
    if (any) odd = 1;
  };
  auto put = [&](int tile) {
    uint8_t* kt = lds + (NB == 2 ? (tile & 1) * 2 * TB : 0);
    uint8_t* vt = kt + TB;
    kput = here(kput);
    vput = here(vput);
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      // load u's rows lie u * RPL further; where that changes the row's place in the swizzle, so do the chunks
      constexpr int kRot = RPL % CH;
      const uint32_t kx = kRot ? ((u * kRot) % CH) * 16 : 0;
      uint8_t* const kd = kt + u * RPL * RB;
      uint8_t* const vd = vt + u * RPL * RB;
      if constexpr (Q8) {
        *(u32x4*)(kd + (kput ^ kx)) = e4m3x8<T>(kr[u][0], kr[u][1]);
        *(u32x4*)(kd + (kput ^ kx ^ kHalf)) = e4m3x8<T>(kr[u][2], kr[u][3]);
        *(u32x4*)(vd + vput) = e4m3x8<VT>(vr[u][0], vr[u][1]);
        *(u32x4*)(vd + (vput ^ kHalf)) = e4m3x8<VT>(vr[u][2], vr[u][3]);
      } else {
        *(u32x4*)(kd + (kput ^ kx)) = kr[u];
        *(u32x4*)(vd + vput) = vr[u];
      }
    }
  };
  // The lane's operands inside a tile: K's chunks 2 kk + hi of row n, V's chunks
  // 4 dt .. + 3; the swizzle leaves kk and dt to a XOR, which head_dim 256, short
  // of registers, does at each read.
  uint32_t kget = n * RB + ((hi ^ (n % CH)) * 16), vget;
  {
    const int lc = lane & 15, dsub = (lane >> 4) & 1;
    vget = (4 * hi + (lc >> 2)) * RB + (((2 * dsub + ((lc & 3) >> 1)) ^ (2 * (lc >> 2))) * 16) + (lc & 1) * 8;
  }
  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16{};
  float m = kPgLowest, l = 0.f;
  // Q8, per 16 keys of the window that the products are in: what a score is
  // worth in the exponent, the logarithm of V's scale, and what undoes it.  V's
  // scales below 2^-80 (one of 0 too) count as that.
  float wk = 0.f, wl = 0.f, wu = 0.f;
  auto enter_scales = [&]() {
    wk = fmaxf(ks, 7.888609e-31f) * p.scale_log2;  // a scale of 0 would make a masked score NaN
    wl = fminf(fmaxf(__builtin_amdgcn_logf(vs), -80.f), 127.f);
    wu = __builtin_amdgcn_exp2f(-wl);
  };
  auto tile = [&](int i, auto masked) {
    const uint8_t* kt = lds + (NB == 2 ? (i & 1) * 2 * TB : 0);
    const uint8_t* vt = kt + TB;
    if (D == 256) {
      kget = here(kget);
      vget = here(vget);
    }
    f32x16 s[2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) s[mt] = f32x16{};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) s[mt] = mma32<T>(*(const u32x4*)(kt + (kget ^ 32 * kk) + mt * 32 * RB), qr[kk], s[mt]);
    if constexpr (NB == 2) {  // among the products: the next tile into the other buffer, the one after it on its way
      put(i + 1);
      fetch(i + 2);
    }
    float ck[4], lv[4], un[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      auto at = [&](float x) {
        return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), (4 * i + b) & 63));
      };
      ck[b] = Q8 ? at(wk) : p.scale_log2;
      lv[b] = Q8 ? at(wl) : 0.f;
      un[b] = Q8 ? at(wu) : 1.f;
    }
    if constexpr (decltype(masked)::value) {
      const int lim = limit - i * kPpKeys - 4 * hi;  // keys 32 mt + 8 j + c (+ 4 hi) below it
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (32 * mt + 8 * (e >> 2) + (e & 3) >= lim) s[mt][e] = -INFINITY;
    }
    float mx = m;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      float y = s[b >> 1][8 * (b & 1)];
#pragma unroll
      for (int e = 1; e < 8; ++e) y = fmaxf(y, s[b >> 1][8 * (b & 1) + e]);
      mx = fmaxf(mx, y * ck[b]);
    }
    mx = max_x32(mx);
    if (__ballot(mx > m)) {
      const float f = __builtin_amdgcn_exp2f(m - mx);
      l *= f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= f;
      m = mx;
    }
    u32x4 pb[4], pc[kTwo ? 4 : 1];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const float off = lv[b] - m + kBias;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y0 = __builtin_amdgcn_exp2f(fmaf(s[b >> 1][8 * (b & 1) + 2 * j], ck[b], off));
        const float y1 = __builtin_amdgcn_exp2f(fmaf(s[b >> 1][8 * (b & 1) + 2 * j + 1], ck[b], off));
        sum += y0 + y1;
        if constexpr (kTwo) {
          const uint32_t u0 = __float_as_uint(y0), u1 = __float_as_uint(y1);
          pb[b][j] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);  // the upper part cut off, what is left rounded
          pc[b][j] = VO::pack2(y0 - __uint_as_float(u0 & 0xffff0000u), y1 - __uint_as_float(u1 & 0xffff0000u));
        } else {
          pb[b][j] = VO::pack2(y0, y1);
        }
      }
      l = Q8 ? fmaf(sum, un[b], l) : l + sum;
    }
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const uint64_t v0 = VO::read_tr(vt + (vget ^ 64 * dt) + 16 * b * RB);
        const uint64_t v1 = VO::read_tr(vt + (vget ^ 64 * dt) + (16 * b + 8) * RB);
        const u32x4 v{(uint32_t)v0, (uint32_t)(v0 >> 32), (uint32_t)v1, (uint32_t)(v1 >> 32)};
        o[dt] = mma32<VT>(v, pb[b], o[dt]);
        if constexpr (kTwo) o[dt] = mma32<VT>(v, pc[b], o[dt]);
      }
  };
  if (t0 < t1) {
    if (tid == 0) odd = 0;
    __syncthreads();
    find(t0 / kWin);
    find_scales();
    if (t0 % kWin != 0) enter(t0 / kWin);
    if (kAhead) fetch(t0);
    if (t0 % kWin >= kWin / 2) find_scales();
    if constexpr (NB == 2) {
      clear(t0);
      even(t0);
      put(t0);
    }
    if (Q8 && kAhead) enter_scales();
    if constexpr (NB == 2) fetch(t0 + 1);
    // (the tile after next is fetched while a tile is used, or the next one with
    // one buffer: the window of the products follows that of fetch() by as much)
    auto turn = [&](int i) {
      if (!kAhead) fetch(i);
      if (Q8 && (kAhead ? i % kWin == 0 && i > t0 : i % kWin == 0 || i == t0)) enter_scales();
      __syncthreads();  // everyone is done with tile i - 1; with two buffers tile i is in LDS
      if constexpr (NB == 2) {
        clear(i + 1);
        even(i + 1);
      } else {
        clear(i);
        even(i);
        put(i);
        if (kAhead) fetch(i + 1);
        __syncthreads();
      }
    };
    // the tiles that every row of the wave sees whole, the others, the turns of the workgroup's later waves
    int i = t0;
    for (const int full = min(wfirst / kPpKeys, mine); i < full; ++i) {
      turn(i);
      tile(i, std::false_type());
    }
    for (; i < mine; ++i) {
      turn(i);
      tile(i, std::true_type());
    }
    for (; i < t1; ++i) {
      turn(i);
      if constexpr (NB == 2) {
        put(i + 1);
        fetch(i + 2);
      }
    }
    if (wrong) raise_device_error(p.err, WNW_DEVERR_BOUNDS);
    if (odd) {  // what even() took out, to the rows that see it (the wave's tiles are behind a barrier)
      const int from = max(t0, max(first, 0) / kPpKeys) * kPpKeys, to = min(t1 * kPpKeys, wlast);
#pragma unroll 1
      for (int key = from; key < to; ++key) {
        const uint8_t* at = paged_v_row(p.c, seg, key, GB);
        if (!at || key >= limit) continue;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            __builtin_amdgcn_sched_barrier(0);
            const f32x4 x = odd_quad<PE>(at, 32 * dt + 8 * j + 4 * hi);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[dt][4 * j + e] += x[e];
          }
      }
    }
  }
  l = sum_x32(l);
  if (splits == 1) {
    prompt_store<T, DT>(p, r, row, h, hi, 0, o, l);
  } else if (busy) {
    float* part = p.part + ((((int64_t)block * N + seg) * p.splits + split) * W + w) * (DT * 16 + 2) * 64;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *(WNW_GLOBAL f32x4*)gptr_w<float>(part + ((dt * 4 + j) * 64 + lane) * 4) =
            f32x4{o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]};
    part += DT * 16 * 64;
    part[lane] = m;
    part[64 + lane] = l;
  }
}

// The splits' sums added up: a workgroup for 32 query rows and 32 elements of
// them, its four waves a quarter of the splits each, joined through LDS.
template <typename T, int D, int W>
__global__ __launch_bounds__(256) void paged_prompt_join_kernel(PagedPromptParams p) {
  constexpr int DT = D / 32, kPpQ = 32 * W;
  __shared__ float sums[4][18][64];
  const int lane = threadIdx.x & 63, k = threadIdx.x >> 6, hi = lane >> 5, n = lane & 31;
  const int N = p.c.n_seg, block = blockIdx.x / (W * DT), w = blockIdx.x / DT % W, dt = blockIdx.x % DT;
  const int seg = block % N, qblk = p.nqb - 1 - block / N;
  const PromptRows r = prompt_rows(p, seg, false);
  if (qblk * kPpQ + 32 * w >= r.rows) return;
  const int splits = splits_of(tiles_of<W>(p, r, qblk), p.splits);
  if (splits == 1) return;
  constexpr int64_t kPart = (DT * 16 + 2) * 64;
  const float* part = p.part + ((int64_t)block * p.splits * W + w) * kPart;
  f32x16 o = f32x16{};
  float m = kPgLowest, l = 0.f;
  auto add = [&](float pm, float pl, const f32x16& y) {
    const float mx = fmaxf(m, pm);
    const float f = __builtin_amdgcn_exp2f(m - mx), g = __builtin_amdgcn_exp2f(pm - mx);
    l = l * f + pl * g;
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = o[e] * f + y[e] * g;
    m = mx;
  };
#pragma unroll 2
  for (int s = k; s < splits; s += 4) {
    const float* at = part + s * W * kPart;
    f32x16 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4 z = *gptr<f32x4>(at + ((dt * 4 + j) * 64 + lane) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[4 * j + e] = z[e];
    }
    at += DT * 16 * 64 + lane;
    add(gptr<float>(at)[0], gptr<float>(at)[64], y);
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) sums[k][e][lane] = o[e];
  sums[k][16][lane] = m;
  sums[k][17][lane] = l;
  __syncthreads();
  if (k != 0) return;
#pragma unroll 1
  for (int i = 1; i < 4; ++i) {
    f32x16 y;
#pragma unroll
    for (int e = 0; e < 16; ++e) y[e] = sums[i][e][lane];
    add(sums[i][16][lane], sums[i][17][lane], y);
  }
  prompt_store<T, 1>(p, r, qblk * kPpQ + 32 * w + n, seg % p.t.hkv, hi, dt, &o, l);
}

// How a call is cut, from what the host knows of it (us measured on one GPU, bf16
// queries in 8 KV heads of 4, 8-bit pages).
//
// Waves of a workgroup, 32 query rows each.  head_dim 128 takes 8: K and V go
// through LDS once for 256 rows (1,024 tokens after 4,000 rows: 108 us, with 4
// waves 112; 3,500 tokens: 128 and 136).  But where such workgroups would be one
// per CU at most and the rows mainly the call's own tokens, so that the last
// tokens' workgroup sets the time, smaller ones are shorter (2,048 tokens: 79 us,
// with 4 waves 67; 1,500: 56 and 49; 300: 19 and 16).  head_dim 64 and 256 keep 4:
// registers and LDS for two or more workgroups per CU.
//
// Splits of a block's tiles: as many workgroups as the CUs hold, of at least 4
// tiles each (64 tokens after 8,000 rows, 126 tiles: 32 us; with 8 tiles 38, with 32 tiles 91), where that
// takes away 8 tiles or more: the second launch costs as much as 5 to 8 (700
// tokens, 11 tiles: 25 us, cut in two 31).
struct PromptPlan {
  int64_t waves, nqb, splits, bytes;
};
static PromptPlan prompt_plan(int64_t n_seg, int64_t group, int64_t max_tokens, int64_t capacity, int64_t D) {
  PromptPlan y;
  const int64_t rows = max_tokens * group, cus = device_cus(), tiles = (capacity + kPpKeys - 1) / kPpKeys;
  const bool own = n_seg * ((rows + 255) / 256) <= cus && 2 * max_tokens >= capacity;
  y.waves = D == 128 && !own ? 8 : 4;
  y.nqb = (rows + 32 * y.waves - 1) / (32 * y.waves);
  const int64_t wgs = std::max<int64_t>(n_seg * y.nqb, 1), want = (y.waves == 8 ? 1 : 2) * cus;
  y.splits = std::max<int64_t>(1, std::min({want / wgs, tiles / 4, (int64_t)64}));
  if (tiles - tiles / y.splits < 8) y.splits = 1;
  y.bytes = y.splits == 1 ? 0 : wgs * y.splits * y.waves * (D / 2 + 2) * 64 * 4;
  return y;
}

template <typename T, int D, bool Q8, int W>
static hipError_t launch_prompt_q(const PagedPromptParams& p, hipStream_t st) {
  const unsigned blocks = (unsigned)(p.c.n_seg * (int64_t)p.nqb);
  hipLaunchKernelGGL((paged_prompt_kernel<T, D, Q8, W>), dim3(blocks * p.splits), dim3(64 * W), 0, st, p);
  if (p.splits > 1) hipLaunchKernelGGL((paged_prompt_join_kernel<T, D, W>), dim3(blocks * W * (D / 32)), dim3(256), 0, st, p);
  return hipGetLastError();
}
template <typename T>
static hipError_t launch_prompt(const PagedPromptParams& p, int64_t D, bool q8, int64_t waves, hipStream_t st) {
  if (D == 64) return q8 ? launch_prompt_q<T, 64, true, 4>(p, st) : launch_prompt_q<T, 64, false, 4>(p, st);
  if (D == 256) return q8 ? launch_prompt_q<T, 256, true, 4>(p, st) : launch_prompt_q<T, 256, false, 4>(p, st);
  if (waves == 8) return q8 ? launch_prompt_q<T, 128, true, 8>(p, st) : launch_prompt_q<T, 128, false, 8>(p, st);
  return q8 ? launch_prompt_q<T, 128, true, 4>(p, st) : launch_prompt_q<T, 128, false, 4>(p, st);
}

// Query rows of a segment that decode attention takes: four tokens of 8 samples after
// 7,560 rows, 4 heads a group, 41 us, as tiles of 32 rows 59; of one sample 23 and 22.
static constexpr int kFewRows = 16;

}  // namespace wnw

using namespace wnw;

extern "C" int64_t wnw_paged_prompt_workspace_bytes(const wnw_paged_cache* cache, int64_t group, int64_t max_tokens) {
  PagedCache c;
  if (!cache || group < 1 || group > 1024 || max_tokens < 0 || max_tokens >= (1 << 24)) return -1;
  if (paged_cache_of(cache, &c)) return -1;
  if (max_tokens == 0) return 0;
  if (max_tokens * group <= kFewRows) return wnw_paged_decode_workspace_bytes(cache->n_seg, max_tokens * group, cache->head_dim);
  return prompt_plan(cache->n_seg, group, max_tokens, c.capacity, cache->head_dim).bytes;
}

extern "C" int wnw_paged_prompt_attn(const wnw_paged_cache* cache, const int32_t* seg_len, const void* q, void* out,
                                     const int64_t* strides, int64_t n_tokens, int64_t n_samples, int64_t group,
                                     const int32_t* cu_tokens, int64_t max_tokens, float scale, int dtype, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
  PagedPromptParams p = {};
  if (int rc = paged_cache_of(cache, &p.c)) return rc;
  const int64_t N = cache->n_seg, D = cache->head_dim;
  WNW_CHECK_ARG(n_samples >= 0 && (n_samples > 0 ? N % n_samples == 0 : N == 0), "segments must be samples x KV heads");
  WNW_CHECK_ARG(n_tokens >= 0 && n_tokens < (1 << 24) && max_tokens >= 0 && max_tokens < (1 << 24), "bad token counts");
  if (N == 0 || n_tokens == 0) return WNW_OK;
  WNW_CHECK_ARG(cu_tokens, "cu_tokens is null");
  if (int rc = paged_attn_check(cache, seg_len, q, out, strides, group, scale, dtype)) return rc;
  {
    const int64_t heads = N / n_samples * group, t = strides[2], h = strides[3];
    const bool apart = t >= h ? (heads == 1 || h >= D) && (n_tokens == 1 || t >= h * (heads - 1) + D)
                              : (n_tokens == 1 || t >= D) && (heads == 1 || h >= t * (n_tokens - 1) + D);
    WNW_CHECK_ARG(apart, "the rows of out overlap");
    WNW_CHECK_ARG(!paged_out_over_q(q, out, strides, n_tokens, heads, D), "out covers a part of q");
  }
  const int64_t most = max_tokens;  // as the workspace's size was asked for
  WNW_CHECK_ARG(most > 0, "max_tokens is zero");
  p.t = PagedTokens{cu_tokens, (int32_t)n_tokens, (int32_t)(N / n_samples), (int32_t)most};
  if (most * group <= kFewRows)
    return paged_decode_launch(cache, seg_len, q, out, strides, p.t, group, scale, dtype, workspace, workspace_bytes, stream);
  WNW_CHECK_ARG(most * group < (1ll << 30), "too many query rows");
  const PromptPlan y = prompt_plan(N, group, most, p.c.capacity, D);
  WNW_CHECK_ARG(N * y.nqb < (1ll << 23), "too many segments and tokens for one call");
  WNW_CHECK_ARG(y.bytes == 0 || (workspace && workspace_bytes >= y.bytes), "workspace too small: %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)y.bytes);
  WNW_CHECK_ARG((uintptr_t)workspace % 256 == 0, "the workspace must be 256-byte aligned");
  p.seg_len = seg_len;
  p.q = q;
  p.out = out;
  p.qt = strides[0], p.qh = strides[1], p.ot = strides[2], p.oh = strides[3];
  p.part = (float*)workspace;
  p.scale_log2 = scale * kPgLog2e;
  p.G = (int32_t)group;
  p.nqb = (int32_t)y.nqb;
  p.splits = (int32_t)y.splits;
  p.err = device_error_word();
  const hipError_t e = dtype == WNW_BF16 ? launch_prompt<bf16_t>(p, D, cache->page_dtype == WNW_E4M3, y.waves, (hipStream_t)stream)
                                         : launch_prompt<f16_t>(p, D, cache->page_dtype == WNW_E4M3, y.waves, (hipStream_t)stream);
  WNW_CHECK_HIP(e, "paged prompt attention launch");
  return WNW_OK;
}
