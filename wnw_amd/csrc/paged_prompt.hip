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
// to 0.87 PFLOP/s (plain bf16 products of size 8,192: 1.2 to 1.4), and 233 us in a row of
// 24, over which the clock falls to 2.1 GHz or less.
// Without gain: half of the waves a phase behind the others, so that one's
// products meet the other's exponentials (8 % slower in one loop); the next tile's
// scores among the exponentials (2 to 5 % slower); loads two tiles ahead; raised
// wave priority in the products.
//
// Through a window (WIN): what none of a block's rows sees is left out, in groups of 16
// keys, and the rest put together to tiles (PromptTiles): tiles of 64 keys in their own
// places walked a tile more at each border (ragged f16 prompts through 301 rows 72 us,
// in groups 66).  Masks at both ends of the window only; tiles between take none.
// Few blocks are cut into shares by the tiles that each has (prompt_share).  8-bit
// pages at head_dim 128 have the products of one tile beside the vector work of the
// next (kSideBySide); 16-bit pages go straight into LDS (kDirect).
//
// What bounds it: 4,564 tokens through 1,024 rows take 101 to 107 us (0.66 PFLOP/s; up to
// 117 in a row of 24, by the card), 512 tokens after 22,116 rows, 2 of 8 heads unwindowed,
// 92 (8.9 of them the join).  Over 2,048 to 6,144 tokens the time is a line, 16.5 us and
// 5.1 ns a tile of 128 rows, within 3 us wherever the workgroups fill the CUs a whole
// number of times or not.  The 16.5 are the launch, the first tiles' round trips, the rows out and the
// last workgroups; the 5.1, 1.3 us of a CU, are 2,700 to 3,150 cycles (2.06 to 2.4 GHz) of
// its SIMDs for a wave's tile, whose matrix and vector instructions one after the other
// are 2,450: beside the instructions, which overlap in part, it is the barrier of each tile
// and its waits for LDS, not measured one by one.  The ragged prompts, 57 us, have short
// blocks: a workgroup's lengths, pages and q, its first tiles' round trips and its rows
// out are a third of its time, and two are on a CU.
#include <algorithm>
#include <type_traits>

#include "paged.h"

namespace wnw {

typedef float f32x16 __attribute__((ext_vector_type(16)));

int paged_decode_launch(const wnw_paged_cache* cache, const int32_t* seg_len, const void* q, void* out, const int64_t* strides,
                        const PagedTokens& t, const PagedView* view, int64_t group, float scale, int dtype, void* workspace,
                        int64_t bytes, void* stream);
bool paged_view_host(const int32_t* window, int64_t window_all, const int32_t* sinks, int64_t sinks_all, PagedView* out);
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
  float* part;             // [blocks, splits, waves] (WIN: [shares, waves]): D / 32 x 16 sums a lane, then max, sum
  float scale_log2;
  int32_t G, nqb, splits;
  int32_t* err;
  PagedView view;          // WIN: the windows, the workgroups of the launch if blocks are shared out
  int32_t wgs;             // (else 0), and each block's first share and shares
  int32_t* shares;
};

static constexpr int kPpKeys = 64;  // keys of a tile
static constexpr int kPpLeast = 4;  // tiles of a share at least (as pieces without a window, below)

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
  int window, sinks;            // WIN: no larger than the segment
  bool blind;                   // WIN: a window of no rows, and no sinks
};
template <bool WIN>
__device__ __forceinline__ PromptRows prompt_rows(const PagedPromptParams& p, int seg, bool tell) {
  PromptRows r;
  const bool told = paged_tokens_of(p.t, seg, &r.first, &r.count);
  r.len = p.seg_len[seg];
  bool good = r.len >= 0 && r.len <= p.c.capacity;
  if constexpr (WIN) {
    good &= paged_view_of(p.view, seg, r.len, &r.window, &r.sinks);
    r.blind = (r.window | r.sinks) == 0;
  }
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
// Tiles that a block of query rows walks.  Through a window, the groups of 16 keys that
// none of its rows sees are left out: `gap` of them behind the `head` that hold the
// sinks, and what is left is put together, four groups a tile (a page has whole
// groups).  Places in that walk, not keys, are what the loops, the splits, the LDS
// buffers and the pages held in registers count.
struct PromptTiles {
  int n, head, gap;
  int lo, last_lo;  // rows from here on are in the window of the block's first row (none with a window of 0), of its last
  __device__ __forceinline__ int group(int place) const { return place < head ? place : place + gap; }
  // the place of the first group at or past row x
  __device__ __forceinline__ int place_of(int x) const {
    const int g = (max(x, 0) + 15) >> 4;
    return g < head ? g : max(g - gap, head);
  }
};
template <int W, bool WIN>
__device__ __forceinline__ PromptTiles tiles_of(const PagedPromptParams& p, const PromptRows& r, int qblk) {
  const int base = r.len - r.count + 1;
  const int last = base + min(32 * W * (qblk + 1) - 1, r.rows - 1) / p.G;  // rows that its last one sees
  PromptTiles y = {max((last + kPpKeys - 1) / kPpKeys, 0), 0, 0, 0, 0};
  if constexpr (WIN) {
    const int groups = max((last + 15) >> 4, 0);
    y.lo = r.window > 0 ? max(base + 32 * W * qblk / p.G - r.window, 0) : 0x7fffffff;
    y.last_lo = last - r.window;
    y.head = min((r.sinks + 15) >> 4, groups);
    y.gap = max(min(y.lo >> 4, groups) - y.head, 0);
    y.n = (groups - y.gap + 3) >> 2;
  }
  return y;
}

// Through windows of different lengths the blocks' tiles differ (512 tokens after
// 22,116 rows: 354 where a head sees everything, 36 through 2,048), so where there are few
// blocks each is cut by its own: all of them into shares of at most `most` tiles, the
// least number with which the launch's workgroups have a share each.  Every workgroup
// finds that out for itself, a wave over at most 512 blocks, from numbers that
// are on the device.
static constexpr int kPpShared = 512;  // blocks at most: 8 a lane, as many as workgroups of 4 waves at a time
struct PromptShare {
  int block, split, splits;  // block -1: none
};
__device__ __forceinline__ int div_up(int x, int y, float inv) {  // inv = 1 / y, y >= 4
  x += y - 1;
  int q = (int)((float)x * inv);
  const int rest = x - q * y;
  q += rest >= y ? 1 : 0;
  return q - (rest < 0 ? 1 : 0);
}
template <int W>
__device__ __forceinline__ PromptShare prompt_share(const PagedPromptParams& p, int id, int lane, bool tell) {
  constexpr int L = kPpShared / 64;
  const int blocks = p.c.n_seg * p.nqb;
  int tiles[L], longest = 0;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int b = i * 64 + lane;
    tiles[i] = 0;
    if (i * 64 < blocks && b < blocks) {
      const int qblk = p.nqb - 1 - b / p.c.n_seg;
      const PromptRows r = prompt_rows<true>(p, b % p.c.n_seg, tell && qblk == 0);
      if (qblk * 32 * W < r.rows) tiles[i] = max(tiles_of<W, true>(p, r, qblk).n, 1);  // (rows that see none are written too)
    }
    sum += (float)tiles[i];
    longest = max(longest, tiles[i]);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) longest = max(longest, __shfl_xor(longest, o));
  sum = wave_sum(sum);
  auto shares_of = [&](int most, int* mine) {
    const float inv = 1.0f / (float)most;
    int all = 0;
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (i * 64 < blocks) {
        mine[i] = min(div_up(tiles[i], most, inv), p.wgs + 1);
        all += mine[i];
      } else {
        mine[i] = 0;
      }
    return all;
  };
  int mine[L];
  int lo = max((int)(0.999f * sum / (float)p.wgs), kPpLeast), hi = max(longest, lo);
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    int all = shares_of(mid, mine);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) all += __shfl_xor(all, o);
    if (all <= p.wgs)
      hi = mid;
    else
      lo = mid + 1;
  }
  const int own = shares_of(lo, mine);
  int incl = own;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(incl, o);
    if (lane >= o) incl += y;
  }
  PromptShare y = {-1, 0, 1};
  int at = incl - own;
#pragma unroll
  for (int i = 0; i < L; ++i) {
    if (id >= at && id < at + mine[i]) y = PromptShare{i * 64 + lane, id - at, mine[i]};
    at += mine[i];
  }
  const uint64_t who = __ballot(y.block >= 0);
  if (!who) return PromptShare{-1, 0, 1};
  const int from = __builtin_ctzll(who);
  return PromptShare{__builtin_amdgcn_readlane(y.block, from), __builtin_amdgcn_readlane(y.split, from),
                     __builtin_amdgcn_readlane(y.splits, from)};
}

// The wave's rows out, 32-element parts dt0 .. dt0 + NT - 1: lane (hi, n) has
// elements 32 i + 8 j + 4 hi + 0..3 of row n
template <typename T, int NT, bool WIN>
__device__ __forceinline__ void prompt_store(const PagedPromptParams& p, const PromptRows& r, int row, int h, int hi, int dt0,
                                             const f32x16* o, float l) {
  if (row >= r.rows) return;
  const int i = row / p.G, g = row - i * p.G;
  T* op = (T*)p.out + (int64_t)(r.first + i) * p.ot + (int64_t)(h * p.G + g) * p.oh;
  bool none = r.len - r.count + i + 1 <= 0;
  if constexpr (WIN) none |= r.blind;
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

// Waves per SIMD that the registers are for, at least and at most: 3 at most, as made to
// fit 4, head_dim 64 over 8 bits takes 43.5 us for 40.7 (2,048 tokens).  Windows over 16-bit
// pages, whose tiles do not go through registers, take 4 at head_dim 64 and 2 at 256.
constexpr int prompt_waves(int d, bool q8, bool win, bool most) {
  if (win && !q8 && d != 128) return d == 64 ? 4 : 2;
  return d == 256 && !q8 ? 1 : most ? 3 : 2;
}
template <typename T, int D, bool Q8, int W, bool WIN>
__global__ __launch_bounds__((64 * W)) __attribute__((amdgpu_waves_per_eu(prompt_waves(D, Q8, WIN, false), prompt_waves(D, Q8, WIN, true)))) void
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
  // Windows over 16-bit pages: the tiles go straight into LDS, by loads that need no
  // registers (through 301 rows, ragged f16 prompts at head_dim 128 67 us for 72, 4,564
  // tokens through 1,024 rows 113 for 119, at head_dim 64 61 for 67, at 256, whose
  // registers then are enough for a second workgroup on a CU, 206 for 296; but 23 -> 25 for
  // 300 tokens, where each has a CU of its own).
  constexpr bool kDirect = WIN && !Q8;
  constexpr bool kAhead = D != 256 || !Q8;  // the next tile's loads are on their way during the products
  // f16 weights are held times 2^8: normal numbers down to 2^-22 of the largest;
  // bf16 ones times 2^-16: 2^16 times the type's largest value is a sum yet
  constexpr float kBias = std::is_same<VT, f16_t>::value ? 8.f : -16.f;
  // How a window's tiles run over 8-bit pages at head_dim 128: 4,564 tokens, window 1,024,
  // 105 us for 114 one after the other (in a row of such calls, the clock falling, 109 for
  // 111).  16-bit pages, which have no codes to convert, lose by it (a ragged batch 69 for
  // 66), and so does head_dim 64, whose products are short (window 500: 53 for 48).
  constexpr bool kSideBySide = WIN && Q8 && D == 128;
  constexpr bool kTwo = Q8 && std::is_same<T, f16_t>::value;  // weights of two parts
  __shared__ __attribute__((aligned(16))) uint8_t lds[NB * 2 * TB];  // [NB][K, V]; kDirect: [NB] K, [NB] V
  __shared__ int odd;  // V had infinities or NaN in such a tile
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hi = lane >> 5, n = lane & 31;
  const int N = p.c.n_seg;
  // the blocks with the most tiles first; workgroups of one segment N apart (8 segments: each in one L2)
  int seg, block, split, shared = 1;
  if (WIN && p.wgs > 0) {
    const PromptShare mine = prompt_share<W>(p, blockIdx.x, lane, blockIdx.x == 0 && w == 0);
    if (mine.block < 0) return;
    seg = mine.block % N;
    block = mine.block / N;
    split = mine.split;
    shared = mine.splits;
    if (split == 0 && tid == 0) {
      p.shares[2 * mine.block] = blockIdx.x;
      p.shares[2 * mine.block + 1] = shared;
    }
  } else {
    const int rank = blockIdx.x / N;
    seg = blockIdx.x % N;
    block = rank / p.splits;
    split = rank - block * p.splits;
  }
  const int qblk = p.nqb - 1 - block;
  const PromptRows r = prompt_rows<WIN>(p, seg, tid == 0 && qblk == 0 && split == 0);
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
  const PromptTiles walk = tiles_of<W, WIN>(p, r, qblk);
  const int tiles = walk.n, splits = WIN ? shared : splits_of(tiles, p.splits);
  // the first key of group b of a tile
  auto key_of = [&](int tile, int b) { return WIN ? walk.group(4 * tile + b) * 16 : tile * kPpKeys + 16 * b; };
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
    const int key = (WIN ? walk.group(window * 64 + lane) : window * 64 + lane) * 16;
    const int id = table[min(key, r.len - 1) >> p.c.shift];
    const bool is = (uint32_t)id < (uint32_t)p.c.n_pages;
    wrong |= !is && (!WIN || key < r.sinks || key + 16 > walk.lo);  // others may have been given back
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
    if (!WIN || (window + 1) * kWin <= t1 + 1) find(window + 1);  // (short walks end before: no round trip for nothing)
  };
  // kDirect: a lane's 16 bytes of a load go to its place in the load's rows, so it fetches the
  // chunk that the swizzle puts there.  What is in no page, or not seen by all, is taken out in LDS.
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)lds);
  const uint32_t ksrc = (lane / CG) * GB + (((lane % CG) ^ (srow % CH)) * 16);
  const uint32_t vsrc = (lane / CG) * GB + (((lane % CG) ^ (2 * (srow & 3))) * 16);
  uint32_t knone = 0, vnone = 0;  // loads of the tile's K, of its V, whose rows are in no page: a bit each
  auto issue = [&](int tile, bool v, uint32_t to) __attribute__((always_inline)) {
    const int in = (1 << p.c.shift) - 1;
    uint32_t none = 0;
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      const int in_tile = u * RPL + w * (64 / CG);
      const int row = key_of(tile, in_tile >> 4) + (in_tile & 15);
      const int id = __builtin_amdgcn_readlane(pid, ((tile * kPpKeys + in_tile) >> 4) & 63);
      const uint8_t* from = (v ? p.c.v : p.c.k) + ((int64_t)(id & 0x7fffffff) * (v ? p.c.v_stride : p.c.k_stride) + (row & in) * GB);
      constexpr uint32_t kRot = RPL % CH;  // load u's rows lie u * RPL further: as in put()
      lds_copy16(uniform_ptr(from), v ? vsrc : ksrc ^ (u * kRot % CH * 16), to + in_tile * RB);
      none |= id < 0 ? 1u << u : 0;
    }
    return none;
  };
  auto issue_k = [&](int tile) __attribute__((always_inline)) {
    if (tile % kWin == 0) enter(tile / kWin);
    knone = issue(tile, false, lds0 + (tile & (NB - 1)) * TB);
  };
  auto issue_v = [&](int tile) __attribute__((always_inline)) { vnone = issue(tile, true, lds0 + (NB + (tile & (NB - 1))) * TB); };
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
      const int in_tile = u * RPL + w * (64 / CG);
      const int row = WIN ? key_of(tile, in_tile >> 4) + (in_tile & 15) : tile * kPpKeys + in_tile;
      const int id = __builtin_amdgcn_readlane(pid, ((tile * kPpKeys + in_tile) >> 4) & 63);
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
    int any = WIN ? key_of(tile, 3) + 16 > r.len : (tile + 1) * kPpKeys > r.len;
#pragma unroll
    for (int u = 0; u < NI; ++u) any |= gone[u] < 0;
    if (!any) return;
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      if (gone[u] < 0) kr[u] = u32x4{0, 0, 0, 0};
      const int at = u * RPL + srow;
      const int row = WIN ? key_of(tile, (u * RPL + w * (64 / CG)) >> 4) + (at & 15) : tile * kPpKeys + at;
      if (gone[u] < 0 || row >= r.len) vr[u] = u32x4{0, 0, 0, 0};
    }
  };
  // Whether rows see the whole of a tile, the first of them `seen` rows and the last from the group at place `late` on:
  // every group before it is of sinks alone.
  auto all_see = [&](int tile, int seen, int late) {
    if constexpr (!WIN) return (tile + 1) * kPpKeys <= seen;
    const int early = r.sinks >> 4;
    return key_of(tile, 3) + 16 <= seen && (4 * tile >= late || 4 * tile + 4 <= early || early >= late);
  };
  const int late = WIN ? walk.place_of(walk.last_lo) : 0;
  auto whole = [&](int tile) { return all_see(tile, first, late); };  // every row of the workgroup
  // takes infinities and NaN out of the V of one that not every row does
  auto even = [&](int tile) {
    if (whole(tile)) return;
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
  // Scores of keys that a row does not see, in the tile's groups that not all of the wave's rows see whole (as all_see)
  auto hide = [&](int i, int wlate, f32x16* s) {
    const int early = r.sinks >> 4;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int place = 4 * i + b, key = walk.group(place) * 16;
      if (key + 16 <= wfirst && (place >= wlate || place < early)) continue;
      const int lo = limit - r.window - key - 4 * hi, sink = min(r.sinks, limit) - key - 4 * hi;
      const bool sinks = place < walk.head;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = 8 * (e >> 2) + (e & 3);  // of the group's keys (+ 4 hi)
        const bool sees = (uint32_t)(k - lo) < (uint32_t)r.window || (sinks && k < sink);
        s[b >> 1][8 * (b & 1) + e] = sees ? s[b >> 1][8 * (b & 1) + e] : -INFINITY;
      }
    }
  };
  // kDirect: takes out of a tile's V, which has landed, what some of the rows do not see
  auto only_seen = [&](int i) __attribute__((always_inline)) {
    const bool all = whole(i);
    if (all && !vnone) return;
    bool any = false;
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      const int in_tile = u * RPL + w * (64 / CG);
      const int row = key_of(i, in_tile >> 4) + ((in_tile + lane / CG) & 15);
      u32x4* at = (u32x4*)(lds + (NB + (i & (NB - 1))) * TB + in_tile * RB + lane * 16);
      u32x4 x = *at;
      if ((vnone >> u & 1) || row >= r.len) x = u32x4{0, 0, 0, 0};
      if (!all) any |= take_odd<PE>(x);
      *at = x;
    }
    if (any) odd = 1;
  };
  // kDirect, one buffer: V is loaded during the scores, the next K during V's products
  auto landed = [&](int i) __attribute__((always_inline)) {
    if constexpr (NB == 1) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      only_seen(i);
      __syncthreads();
      if (i + 1 < t1) issue_k(i + 1);
    }
  };
  auto tile = [&](int i, auto masked) __attribute__((always_inline)) {
    const uint8_t* kt = lds + (kDirect ? (i & (NB - 1)) * TB : NB == 2 ? (i & 1) * 2 * TB : 0);
    const uint8_t* vt = kDirect ? lds + (NB + (i & (NB - 1))) * TB : kt + TB;
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
    if constexpr (NB == 2 && !kDirect) {  // among the products: the next tile into the other buffer, the one after it on its way
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
    if (masked) {
      if constexpr (WIN) {
        hide(i, walk.place_of(wlast - r.window), s);
      } else {
        const int lim = limit - i * kPpKeys - 4 * hi;  // keys 32 mt + 8 j + c (+ 4 hi) below it
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (32 * mt + 8 * (e >> 2) + (e & 3) >= lim) s[mt][e] = -INFINITY;
      }
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
    if constexpr (kDirect) landed(i);
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
  auto finish = [&]() {  // (the wave's tiles are behind a barrier)
    if (wrong) raise_device_error(p.err, WNW_DEVERR_BOUNDS);
    if (odd) {  // what even() took out, to the rows that see it
      auto give = [&](int from, int to) {
#pragma unroll 1
        for (int key = from; key < to; ++key) {
          const uint8_t* at = paged_v_row(p.c, seg, key, GB);
          if (!at || key >= limit || (WIN && key >= r.sinks && key < limit - r.window)) continue;
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
      };
      if constexpr (WIN) {
#pragma unroll 1
        for (int i = t0; i < t1; ++i)
          for (int b = 0; b < 4 && !whole(i); ++b) give(key_of(i, b), min(key_of(i, b) + 16, wlast));
      } else {
        give(max(t0, max(first, 0) / kPpKeys) * kPpKeys, min(t1 * kPpKeys, wlast));
      }
    }
  };
  if constexpr (kSideBySide) {
    // A tile's products and vector instructions run side by side where they are of
    // different tiles: the next tile's scores among this one's exponentials, this one's
    // values among the next one's maximum and the staging.  So K is staged a tile ahead of
    // V: when tile i is used, K of i + 1 and V of i are in LDS, K of i + 2 and V of i + 1 in
    // registers on their way there, K of i + 3 and V of i + 2 on their way from memory.
    // What a group's page and scales are lies in LDS, kRef tiles from tile ref0 on.
    static_assert(Q8, "16-bit pages go straight into LDS");
    if (t0 < t1) {
      if (tid == 0) odd = 0;
      constexpr int kRef = 64;
      struct Refs {
        int32_t id[4 * kRef];
        float k[4 * kRef], l[4 * kRef], u[4 * kRef];
      };
      __shared__ __attribute__((aligned(16))) Refs refs;
      int ref0 = t0;
      auto refer_pages = [&](int tile) {  // the thread's group's page, or -1
        ref0 = tile;
        int id = -1;
        if (tid < 4 * kRef) {
          const int key = walk.group(4 * tile + tid) * 16;
          id = table[min(key, r.len - 1) >> p.c.shift];
          const bool is = (uint32_t)id < (uint32_t)p.c.n_pages;
          wrong |= !is && (key < r.sinks || key + 16 > walk.lo);  // others may have been given back
          id = is ? id : -1;
          refs.id[tid] = is ? id : (int)0x80000000;
        }
        return id;
      };
      auto refer_scales = [&](int id) {
        if (tid < 4 * kRef) {
          const float k_of = p.c.k_scale[max(id, 0)], v_of = p.c.v_scale[max(id, 0)];
          refs.k[tid] = fmaxf(id >= 0 ? k_of : 1.f, 7.888609e-31f) * p.scale_log2;  // a scale of 0 would make a masked score NaN
          const float log_v = fminf(fmaxf(__builtin_amdgcn_logf(id >= 0 ? v_of : 1.f), -80.f), 127.f);
          refs.l[tid] = log_v;
          refs.u[tid] = __builtin_amdgcn_exp2f(-log_v);
        }
      };
      auto load = [&](int tile, const uint8_t* pages, int64_t stride, u32x4* to, int* none) {
        const int in = (1 << p.c.shift) - 1;
        typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
        soff = here(soff);
#pragma unroll
        for (int u = 0; u < NI; ++u) {
          const int in_tile = u * RPL + w * (64 / CG);
          const int row = key_of(tile, in_tile >> 4) + (in_tile & 15);
          const int id = __builtin_amdgcn_readfirstlane(refs.id[4 * (tile - ref0) + (in_tile >> 4)]);
          const WNW_GLOBAL uint8_t* at = gptr<uint8_t>(pages) + ((int64_t)(id & 0x7fffffff) * stride + (row & in) * GB);
          const u32x2_t x0 = *(const WNW_GLOBAL u32x2_t*)(at + soff), x1 = *(const WNW_GLOBAL u32x2_t*)(at + (soff + GB / 2));
          to[u] = u32x4{x0[0], x0[1], x1[0], x1[1]};
          none[u] = id;
        }
      };
      int vgone[NI];
      auto load_k = [&](int tile) { load(tile, p.c.k, p.c.k_stride, kr, gone); };
      auto load_v = [&](int tile) { load(tile, p.c.v, p.c.v_stride, vr, vgone); };
      auto clear_k = [&]() {
#pragma unroll
        for (int u = 0; u < NI; ++u)
          if (gone[u] < 0) kr[u] = u32x4{0, 0, 0, 0};
      };
      auto clear_v = [&](int tile) {
        int any = key_of(tile, 3) + 16 > r.len;
#pragma unroll
        for (int u = 0; u < NI; ++u) any |= vgone[u] < 0;
        if (any) {
#pragma unroll
          for (int u = 0; u < NI; ++u) {
            const int row = key_of(tile, (u * RPL + w * (64 / CG)) >> 4) + ((u * RPL + srow) & 15);
            if (vgone[u] < 0 || row >= r.len) vr[u] = u32x4{0, 0, 0, 0};
          }
        }
        even(tile);
      };
      constexpr int kAheadK = 2, kAheadV = 3;  // steps that K's and V's operands are read ahead of their products
      // what the staging of K's tile and of V's writes to LDS, in kPut pieces each
      constexpr int kPut = NI * 2;
      auto put_k = [&](int tile, int piece) {
        const int u = piece / 2;
        constexpr int kRot = RPL % CH;
        const uint32_t kx = kRot ? ((u * kRot) % CH) * 16 : 0;
        uint8_t* kd = lds + (tile & 1) * 2 * TB + u * RPL * RB;
        if (piece % 2 == 0)
          *(u32x4*)(kd + (kput ^ kx)) = e4m3x8<T>(kr[u][0], kr[u][1]);
        else
          *(u32x4*)(kd + (kput ^ kx ^ kHalf)) = e4m3x8<T>(kr[u][2], kr[u][3]);
      };
      auto put_v = [&](int tile, int piece) {
        const int u = piece / 2;
        uint8_t* vd = lds + (tile & 1) * 2 * TB + TB + u * RPL * RB;
        if (piece % 2 == 0)
          *(u32x4*)(vd + vput) = e4m3x8<VT>(vr[u][0], vr[u][1]);
        else
          *(u32x4*)(vd + (vput ^ kHalf)) = e4m3x8<VT>(vr[u][2], vr[u][3]);
      };
      auto put_all = [&](auto put, int tile) {
#pragma unroll
        for (int piece = 0; piece < kPut; ++piece) put(tile, piece);
      };
      {
        const int id = refer_pages(t0);
        __syncthreads();
        u32x4 first_k[NI];
        int first_gone[NI];
        load(t0, p.c.k, p.c.k_stride, first_k, first_gone);
        load_v(t0);
        load_k(t0 + 1);
        refer_scales(id);
#pragma unroll
        for (int u = 0; u < NI; ++u) {  // K of t0 by way of kr
          const u32x4 x = kr[u];
          const int none = gone[u];
          kr[u] = first_k[u];
          gone[u] = first_gone[u];
          first_k[u] = x;
          first_gone[u] = none;
        }
        clear_k();
        put_all(put_k, t0);
        clear_v(t0);
        put_all(put_v, t0);
        load_v(t0 + 1);
#pragma unroll
        for (int u = 0; u < NI; ++u) {
          kr[u] = first_k[u];
          gone[u] = first_gone[u];
        }
        clear_k();
        put_all(put_k, t0 + 1);
        load_k(t0 + 2);
      }
      __syncthreads();
      // the score's worth in the exponent, V's scale and what undoes it, of a tile's groups
      f32x4 ck, lv, un;
      auto numbers = [&](int i) {
        const int at = 4 * (i - ref0);
        ck = *(const f32x4*)(refs.k + at);
        lv = *(const f32x4*)(refs.l + at);
        un = *(const f32x4*)(refs.u + at);
      };
      auto scores = [&](int i, f32x16* s) {
        const uint8_t* kt = lds + (i & 1) * 2 * TB;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) s[mt] = f32x16{};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) s[mt] = mma32<T>(*(const u32x4*)(kt + (kget ^ 32 * kk) + mt * 32 * RB), qr[kk], s[mt]);
      };
      auto most = [&](const f32x16* s) {
        float mx = m;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          float y = s[b >> 1][8 * (b & 1)];
#pragma unroll
          for (int e = 1; e < 8; ++e) y = fmaxf(y, s[b >> 1][8 * (b & 1) + e]);
          mx = fmaxf(mx, y * ck[b]);
        }
        return mx;
      };
      const int wlate = walk.place_of(wlast - r.window);
      float mx = m;
      // tile i, whose scores s are there; next: the next one's
      auto turn = [&](int i) {
        __syncthreads();
        if (i + 3 >= ref0 + kRef) {
          refer_scales(refer_pages(i));
          __syncthreads();
        }
      };
      auto use = [&](int i, f32x16* s, f32x16* next) {
          turn(i);
          const float f = __builtin_amdgcn_exp2f(m - mx);
          const bool grown = __ballot(mx > m) != 0;
          m = mx;
          l *= f;
          // Each step below is a product or two and the vector instructions that run in their
          // shadow; operands from LDS are read a step ahead.
          __builtin_amdgcn_sched_barrier(0);
          u32x4 pb[4], pc[kTwo ? 4 : 1];
          const uint8_t* vt = lds + (i & 1) * 2 * TB + TB;
          constexpr int kSteps = 4 * DT, kHalfway = kSteps / 2;
          u32x4 va[kAheadV + 1];
          auto read_v = [&](int t) {
            const int b = t / DT, dt = t % DT;
            const uint64_t v0 = VO::read_tr(vt + (vget ^ 64 * dt) + 16 * b * RB);
            const uint64_t v1 = VO::read_tr(vt + (vget ^ 64 * dt) + (16 * b + 8) * RB);
            va[t % (kAheadV + 1)] = u32x4{(uint32_t)v0, (uint32_t)(v0 >> 32), (uint32_t)v1, (uint32_t)(v1 >> 32)};
          };
          {
            const uint8_t* kt = lds + ((i + 1) & 1) * 2 * TB;
            u32x4 ka[kAheadK + 1][2];
            auto read = [&](int kk) {
#pragma unroll
              for (int mt = 0; mt < 2; ++mt) ka[kk % (kAheadK + 1)][mt] = *(const u32x4*)(kt + (kget ^ 32 * kk) + mt * 32 * RB);
            };
#pragma unroll
            for (int kk = 0; kk < kAheadK; ++kk) read(kk);
            constexpr int kEach = 32 / KK;  // of the lane's weights to a step
            float sum = 0.f;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
              if (kk + kAheadK < KK) read(kk + kAheadK);
              if (kk == KK - 1) {
#pragma unroll
                for (int t = 0; t < kAheadV; ++t) read_v(t);
              }
#pragma unroll
              for (int mt = 0; mt < 2; ++mt) next[mt] = mma32<T>(ka[kk % (kAheadK + 1)][mt], qr[kk], kk == 0 ? f32x16{} : next[mt]);
              const int b = kk * kEach / 8;
              const float off = lv[b] - m + kBias;
#pragma unroll
              for (int j = kk * kEach % 8 / 2; j < (kk * kEach % 8 + kEach) / 2; ++j) {
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
              if ((kk + 1) * kEach % 8 == 0) {
                l = fmaf(sum, un[b], l);
                sum = 0.f;
                asm volatile("" : "+v"(pb[b]), "+v"(l));  // here, not where they are used
                if constexpr (kTwo) asm volatile("" : "+v"(pc[b]));
              }
              __builtin_amdgcn_sched_barrier(0);
            }
          }
          if (grown) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] *= f;
          }
          numbers(i + 1);
          if (!all_see(i + 1, wfirst, wlate)) hide(i + 1, wlate, next);
          kput = here(kput);
          vput = here(vput);
          float y = 0.f;
          mx = m;
          auto value = [&](int t) {
            const int b = t / DT, dt = t % DT;
            if (t + kAheadV < kSteps) read_v(t + kAheadV);
            o[dt] = mma32<VT>(va[t % (kAheadV + 1)], pb[b], o[dt]);
            if constexpr (kTwo) o[dt] = mma32<VT>(va[t % (kAheadV + 1)], pc[b], o[dt]);
          };
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int t = 0; t < kHalfway; ++t) {
            value(t);
            constexpr int kEach = 32 / kHalfway;
#pragma unroll
            for (int e = t * kEach; e < (t + 1) * kEach; ++e) {
              const float x = next[e >> 4][e & 15];
              y = e % 8 == 0 ? x : fmaxf(y, x);
              if (e % 8 == 7) mx = fmaxf(mx, y * ck[e / 8]);
            }
            asm volatile("" : "+v"(y), "+v"(mx));
            __builtin_amdgcn_sched_barrier(0);
          }
          clear_k();
          clear_v(i + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int t = kHalfway; t < kSteps; ++t) {
            value(t);
#pragma unroll
            for (int piece = 0; piece < 2 * kPut; ++piece)
              if (piece * kHalfway / (2 * kPut) == t - kHalfway) {
                if (piece < kPut)
                  put_v(i + 1, piece);
                else
                  put_k(i + 2, piece - kPut);
              }
            __builtin_amdgcn_sched_barrier(0);
          }
          mx = i + 1 < t1 ? max_x32(mx) : m;
          load_v(i + 2);
          load_k(i + 3);
      };
      if (busy) {
        f32x16 s[2], next[2];
        numbers(t0);
        scores(t0, s);
        if (!all_see(t0, wfirst, wlate)) hide(t0, wlate, s);
        mx = max_x32(most(s));
        int i = t0;
        for (; i + 1 < t1; i += 2) {
          use(i, s, next);
          use(i + 1, next, s);
        }
        if (i < t1) use(i, s, next);
      } else {
        for (int i = t0; i < t1; ++i) {
          turn(i);
          clear_k();
          clear_v(i + 1);
          put_all(put_k, i + 2);
          put_all(put_v, i + 1);
          load_v(i + 2);
          load_k(i + 3);
        }
      }
      finish();
    }
  } else if (t0 < t1) {
    if (tid == 0) odd = 0;
    __syncthreads();
    find(t0 / kWin);
    find_scales();
    if (t0 % kWin != 0) enter(t0 / kWin);
    if (kDirect) {
      issue_k(t0);
      issue_v(t0);
    } else if (kAhead) {
      fetch(t0);
    }
    if (t0 % kWin >= kWin / 2) find_scales();
    if constexpr (NB == 2 && !kDirect) {
      clear(t0);
      even(t0);
      put(t0);
    }
    if (Q8 && kAhead) enter_scales();
    if constexpr (NB == 2 && !kDirect) fetch(t0 + 1);
    // (the tile after next is fetched while a tile is used, or the next one with
    // one buffer: the window of the products follows that of fetch() by as much)
    auto turn = [&](int i) {
      if constexpr (kDirect) {  // the loads of a tile are on their way while the one before it is used
        if (NB == 1 && i == t0)
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NI) : "memory");  // V behind K
        else
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (knone) {
#pragma unroll
          for (int u = 0; u < NI; ++u)
            if (knone >> u & 1)
              *(u32x4*)(lds + (i & (NB - 1)) * TB + (u * RPL + w * (64 / CG)) * RB + lane * 16) = u32x4{0, 0, 0, 0};
        }
        if constexpr (NB == 2) only_seen(i);
        __syncthreads();  // tile i, K of it at least, is in LDS; everyone is done with tile i - 1
        if (NB == 1 && i > t0) issue_v(i);
        if (NB == 2 && i + 1 < t1) {
          issue_k(i + 1);
          issue_v(i + 1);
        }
        return;
      }
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
    auto pass = [&](int i) {  // a tile that none of the wave's rows sees
      if constexpr (kDirect) {
        landed(i);
      } else if constexpr (NB == 2) {
        put(i + 1);
        fetch(i + 2);
      }
    };
    if constexpr (WIN) {
      // places of the first group that the wave's first row sees past the sinks, and of the first that its last row sees whole
      const int from = walk.place_of(wfirst - r.window - 15), wlate = walk.place_of(wlast - r.window);
      for (int i = t0; i < t1; ++i) {
        turn(i);
        if (!busy || key_of(i, 0) >= wlast || (4 * i >= walk.head && 4 * i + 4 <= from))
          pass(i);
        else
          tile(i, !all_see(i, wfirst, wlate));
      }
    } else {
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
        pass(i);
      }
    }
    finish();
  }
  l = sum_x32(l);
  if (splits == 1) {
    if constexpr (WIN) {  // whole rows, by way of LDS: a window of 300 rows 64.4 us for 68.5 (4,564 tokens, 8-bit pages)
      static_assert(W * 32 * RB <= (int)sizeof(lds), "the waves' rows");
      __syncthreads();  // everyone is done with the tiles
      uint8_t* const rows = lds + w * 32 * RB;
      const bool none = limit <= 0 || r.blind;
      const float inv = 1.0f / l;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = none ? 0.f : o[dt][4 * j + e] * inv;
          *(uint64_t*)(rows + n * RB + (((4 * dt + j) ^ (n % CH)) * 16) + hi * 8) =
              (uint64_t)HalfOps<T>::pack2(y[2], y[3]) << 32 | HalfOps<T>::pack2(y[0], y[1]);
        }
      __builtin_amdgcn_wave_barrier();
#pragma unroll 2
      for (int at = lane / CH; at < 32; at += 64 / CH) {
        const int to = qblk * kPpQ + 32 * w + at;
        if (to >= r.rows) break;
        const int i = to / p.G;
        T* const op = (T*)p.out + (int64_t)(r.first + i) * p.ot + (int64_t)(h * p.G + to - i * p.G) * p.oh;
        *gptr_w<u32x4>(op + 8 * ((lane % CH) ^ (at % CH))) = *(const u32x4*)(rows + at * RB + (lane % CH) * 16);
      }
    } else {
      prompt_store<T, DT, WIN>(p, r, row, h, hi, 0, o, l);
    }
  } else if (busy) {
    const int64_t place = WIN ? blockIdx.x : ((int64_t)block * N + seg) * p.splits + split;
    float* part = p.part + (place * W + w) * (DT * 16 + 2) * 64;
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
template <typename T, int D, int W, bool WIN>
__global__ __launch_bounds__(256) void paged_prompt_join_kernel(PagedPromptParams p) {
  constexpr int DT = D / 32, kPpQ = 32 * W;
  __shared__ float sums[4][18][64];
  const int lane = threadIdx.x & 63, k = threadIdx.x >> 6, hi = lane >> 5, n = lane & 31;
  const int N = p.c.n_seg, block = blockIdx.x / (W * DT), w = blockIdx.x / DT % W, dt = blockIdx.x % DT;
  const int seg = block % N, qblk = p.nqb - 1 - block / N;
  const PromptRows r = prompt_rows<WIN>(p, seg, false);
  if (qblk * kPpQ + 32 * w >= r.rows) return;
  const int splits = WIN ? p.shares[2 * block + 1] : splits_of(tiles_of<W, WIN>(p, r, qblk).n, p.splits);
  if (splits == 1) return;
  constexpr int64_t kPart = (DT * 16 + 2) * 64;
  const int64_t place = WIN ? p.shares[2 * block] : (int64_t)block * p.splits;
  const float* part = p.part + (place * W + w) * kPart;
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
  prompt_store<T, 1, WIN>(p, r, qblk * kPpQ + 32 * w + n, seg % p.t.hkv, hi, dt, &o, l);
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
  int64_t wgs = 0, part = 0;  // through windows: the workgroups that blocks are shared out to, bytes ahead of the partial sums
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

// Through windows: a block's tiles are at most those of its rows' windows, where these are
// known (on the device they may be anything, and differ).
//
// Few blocks, of tiles that may differ or be cut with a gain as above, are shared out to
// as many workgroups as the CUs hold, of 8 waves at head_dim 128 (512 tokens after
// 22,116 rows, two of eight heads unwindowed: 93 us, with 4 waves 97).  Others have about
// the same walk each, and smaller workgroups walk less beyond their own rows, two at a
// time on a CU (8-bit pages, 4,564 tokens, window 300: 61 us, with 8 waves 71; 500 73 and
// 88; 1,024 105 and 107; 1,400 129 and 125; 2,000 153 and 158; the whole prompt 211 and
// 208; 9,000 tokens, window 1,024 206 and 224, the whole prompt 722 and 703).
static PromptPlan window_plan(int64_t n_seg, int64_t group, int64_t max_tokens, int64_t capacity, int64_t D, const PagedView& view) {
  const bool alike = !view.window && !view.sinks;
  const int64_t rows = max_tokens * group, cus = device_cus();
  int64_t tiles = (capacity + kPpKeys - 1) / kPpKeys;
  if (alike) tiles = std::min(tiles, ((int64_t)view.window_all + view.sinks_all + 256 / group) / kPpKeys + 2);
  PromptPlan y;
  auto blocks = [&](int64_t waves) {
    y.waves = waves;
    y.nqb = (rows + 32 * waves - 1) / (32 * waves);
    return std::max<int64_t>(n_seg * y.nqb, 1);
  };
  y.splits = 1;
  y.bytes = 0;
  const int64_t wgs = blocks(D == 128 ? 8 : 4), want = (y.waves == 8 ? 1 : 2) * cus;
  const int64_t most = alike ? std::min(want / wgs, tiles / 4) : wgs <= std::min<int64_t>(want, kPpShared) ? 4 : 1;
  if (most > 1 && tiles - tiles / most >= 8) {
    y.wgs = want;
    y.part = (wgs * 8 + 255) / 256 * 256;
    y.bytes = y.part + want * y.waves * (D / 2 + 2) * 64 * 4;
  } else {
    blocks(4);
  }
  return y;
}

template <typename T, int D, bool Q8, int W, bool WIN>
static hipError_t launch_prompt_q(const PagedPromptParams& p, hipStream_t st) {
  const unsigned blocks = (unsigned)(p.c.n_seg * (int64_t)p.nqb);
  hipLaunchKernelGGL((paged_prompt_kernel<T, D, Q8, W, WIN>), dim3(WIN && p.wgs ? p.wgs : blocks * p.splits), dim3(64 * W), 0, st, p);
  if (p.splits > 1 || (WIN && p.wgs > 0))
    hipLaunchKernelGGL((paged_prompt_join_kernel<T, D, W, WIN>), dim3(blocks * W * (D / 32)), dim3(256), 0, st, p);
  return hipGetLastError();
}
template <typename T, bool WIN>
static hipError_t launch_prompt_view(const PagedPromptParams& p, int64_t D, bool q8, int64_t waves, hipStream_t st) {
  if (D == 64) return q8 ? launch_prompt_q<T, 64, true, 4, WIN>(p, st) : launch_prompt_q<T, 64, false, 4, WIN>(p, st);
  if (D == 256) return q8 ? launch_prompt_q<T, 256, true, 4, WIN>(p, st) : launch_prompt_q<T, 256, false, 4, WIN>(p, st);
  if (waves == 8) return q8 ? launch_prompt_q<T, 128, true, 8, WIN>(p, st) : launch_prompt_q<T, 128, false, 8, WIN>(p, st);
  return q8 ? launch_prompt_q<T, 128, true, 4, WIN>(p, st) : launch_prompt_q<T, 128, false, 4, WIN>(p, st);
}
template <typename T>
static hipError_t launch_prompt(const PagedPromptParams& p, int64_t D, bool q8, int64_t waves, bool view, hipStream_t st) {
  return view ? launch_prompt_view<T, true>(p, D, q8, waves, st) : launch_prompt_view<T, false>(p, D, q8, waves, st);
}

// Query rows of a segment that decode attention takes: four tokens of 8 samples after
// 7,560 rows, 4 heads a group, 41 us, as tiles of 32 rows 59; of one sample 23 and 22.
static constexpr int kFewRows = 16;

}  // namespace wnw

using namespace wnw;

static int64_t prompt_workspace(const wnw_paged_cache* cache, int64_t group, int64_t max_tokens, const PagedView* view) {
  PagedCache c;
  if (!cache || group < 1 || group > 1024 || max_tokens < 0 || max_tokens >= (1 << 24)) return -1;
  if (paged_cache_of(cache, &c)) return -1;
  if (max_tokens == 0) return 0;
  if (max_tokens * group <= kFewRows) return wnw_paged_decode_workspace_bytes(cache->n_seg, max_tokens * group, cache->head_dim);
  const int64_t N = cache->n_seg, D = cache->head_dim;
  return (view ? window_plan(N, group, max_tokens, c.capacity, D, *view) : prompt_plan(N, group, max_tokens, c.capacity, D)).bytes;
}

static int prompt_attn(const wnw_paged_cache* cache, const int32_t* seg_len, const void* q, void* out, const int64_t* strides,
                       int64_t n_tokens, int64_t n_samples, int64_t group, const int32_t* cu_tokens, int64_t max_tokens,
                       const PagedView* view, float scale, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
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
    return paged_decode_launch(cache, seg_len, q, out, strides, p.t, view, group, scale, dtype, workspace, workspace_bytes, stream);
  WNW_CHECK_ARG(most * group < (1ll << 30), "too many query rows");
  const PromptPlan y = view ? window_plan(N, group, most, p.c.capacity, D, *view) : prompt_plan(N, group, most, p.c.capacity, D);
  WNW_CHECK_ARG(N * y.nqb * y.waves < (1ll << 26), "too many segments and tokens for one call");  // 2^32 threads
  WNW_CHECK_ARG(y.bytes == 0 || (workspace && workspace_bytes >= y.bytes), "workspace too small: %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)y.bytes);
  WNW_CHECK_ARG((uintptr_t)workspace % 256 == 0, "the workspace must be 256-byte aligned");
  p.seg_len = seg_len;
  p.q = q;
  p.out = out;
  p.qt = strides[0], p.qh = strides[1], p.ot = strides[2], p.oh = strides[3];
  p.part = (float*)((uint8_t*)workspace + y.part);
  p.shares = (int32_t*)workspace;
  p.wgs = (int32_t)y.wgs;
  p.scale_log2 = scale * kPgLog2e;
  p.G = (int32_t)group;
  p.nqb = (int32_t)y.nqb;
  p.splits = (int32_t)y.splits;
  p.err = device_error_word();
  if (view) p.view = *view;
  const bool q8 = cache->page_dtype == WNW_E4M3;
  const hipError_t e = dtype == WNW_BF16 ? launch_prompt<bf16_t>(p, D, q8, y.waves, view, (hipStream_t)stream)
                                         : launch_prompt<f16_t>(p, D, q8, y.waves, view, (hipStream_t)stream);
  WNW_CHECK_HIP(e, "paged prompt attention launch");
  return WNW_OK;
}

extern "C" int64_t wnw_paged_prompt_workspace_bytes(const wnw_paged_cache* cache, int64_t group, int64_t max_tokens) {
  return prompt_workspace(cache, group, max_tokens, nullptr);
}

extern "C" int wnw_paged_prompt_attn(const wnw_paged_cache* cache, const int32_t* seg_len, const void* q, void* out,
                                     const int64_t* strides, int64_t n_tokens, int64_t n_samples, int64_t group,
                                     const int32_t* cu_tokens, int64_t max_tokens, float scale, int dtype, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
  return prompt_attn(cache, seg_len, q, out, strides, n_tokens, n_samples, group, cu_tokens, max_tokens, nullptr, scale, dtype,
                     workspace, workspace_bytes, stream);
}

extern "C" int64_t wnw_paged_prompt_window_workspace_bytes(const wnw_paged_cache* cache, int64_t group, int64_t max_tokens,
                                                           const int32_t* window, int64_t window_all, const int32_t* sinks,
                                                           int64_t sinks_all) {
  PagedView view;
  if (!paged_view_host(window, window_all, sinks, sinks_all, &view)) return -1;
  return prompt_workspace(cache, group, max_tokens, &view);
}

extern "C" int wnw_paged_prompt_attn_window(const wnw_paged_cache* cache, const int32_t* seg_len, const void* q, void* out,
                                            const int64_t* strides, int64_t n_tokens, int64_t n_samples, int64_t group,
                                            const int32_t* cu_tokens, int64_t max_tokens, const int32_t* window,
                                            int64_t window_all, const int32_t* sinks, int64_t sinks_all, float scale, int dtype,
                                            void* workspace, int64_t workspace_bytes, void* stream) {
  PagedView view;
  if (!paged_view_host(window, window_all, sinks, sinks_all, &view)) return WNW_EINVAL;
  return prompt_attn(cache, seg_len, q, out, strides, n_tokens, n_samples, group, cu_tokens, max_tokens, &view, scale, dtype,
                     workspace, workspace_bytes, stream);
}
