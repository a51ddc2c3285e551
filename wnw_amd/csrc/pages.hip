// The paged cache's pages (gfx950): samples forked and reordered, pages reserved
// for the next rows and given back behind a window, a pool's used pages moved to
// its front, rows copied from page to page.
//
// Which pages are used is counted: refs[p] table entries name page p, 0: it is free.  With
// U used pages, need_s fresh pages of segment s and the free pages f_0 < f_1 < ..., segment s
// gets f_i, i from sum_{s' < s} need_s' on; a compaction moves the i-th used page
// at or above U to the i-th free one below.  All of it is prefix sums.
//
// A fork or a reservation is planned by one workgroup, which alone can hand pages out
// in order, and reads counts only until it has found as many free ones as are
// needed; others copy the counts meanwhile.  A second launch carries it out, a workgroup
// a segment: rows of the table, counts by integer atomics, whose order does not
// show.  The plan says whether the call can be done; the second launch leaves
// everything as it was where it cannot.  A compaction needs the whole pool's counts:
// up to 64 workgroups each sum all of them, from their L2, and rank their own pages
// (13,653 pages and their copies: 30 us a pass, planned by one workgroup 41).
//
// What bounds it: the launches and the plan's chain of loads; the bytes are few.
// Forking 256 segments (6,060 pages) 5.7 us for the plan, 3.7 for the rest, and 3.2 for the
// copies; reserving a row for 256 segments of up to 313 blocks (30,677 pages) 5.0 and 3.6;
// compacting 13,653 pages 5.5 and 3.4.  The page copy is bound by memory: up to 4,096
// workgroups for K and for V, a page at a time by 256 threads with four 16-byte loads in
// flight (3,277 pages of 8 KB, 107 MB read and written with K and V: 21.4 us, 5.0 TB/s).
// Reserving for prompts the plan is bound by its waves, each of which looks 16 segments'
// blocks over one after the other: 256 segments of 500 to 2,000 new rows 24 us a pass with
// pages of 64 (5,132 of them), 34 with pages of 16 (21,920); a row each 9.4.
#include <algorithm>

#include "paged.h"

namespace wnw {

static constexpr int kPlanThreads = 1024;
static constexpr int kPlanWaves = kPlanThreads / 64;
static constexpr int kPlanPer = 16;          // pages of a thread at a time: four 16-byte loads, 16,384 pages a round
static constexpr int kPlanCopy = 4096;       // counts that another workgroup of the plan copies: four a thread
static constexpr int kMaxSamples = 8192;     // of a fork: two words of LDS each

// A workspace, in 32-bit words: the head, then lists.
enum { kOk = 0, kUsed = 1, kMoves = 2, kHead = 64 };

struct PagesParams {
  const int32_t* table;
  int32_t* new_table;
  int64_t stride, new_stride;
  const int32_t* seg_len;
  const int32_t* refs;
  int32_t* new_refs;
  int32_t* ws;
  int32_t* err;
  int32_t n_seg, max_blocks, n_pages, shift;
};
struct ForkParams {
  PagesParams g;
  const int32_t* parents;
  int32_t* new_len;
  int32_t* copies;
  int32_t n_old, n_new, heads;
};
struct ReserveParams {
  PagesParams g;
  PagedView view;
  const int32_t* cu;
  int32_t tokens, heads, windowed, wide;
};
struct CompactParams {
  PagesParams g;
  int32_t* moves;
  int32_t* used;
  int32_t range;
};

// Where the lists of a workspace begin
__device__ __forceinline__ int32_t* ws_fresh(const PagesParams& g) { return g.ws + kHead; }  // [n_pages] at most
__device__ __forceinline__ int32_t* ws_place(const PagesParams& g) { return ws_fresh(g) + g.n_pages; }  // [segments] or [n_pages]

struct PlanShared {
  int wave[kPlanWaves], second[kPlanWaves];
};
// x summed over the threads before, *all over all of them
__device__ __forceinline__ int plan_scan(PlanShared& sh, int x, int* all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int incl = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(incl, o);
    if (lane >= o) incl += y;
  }
  __syncthreads();
  if (lane == 63) sh.wave[w] = incl;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < kPlanWaves; ++i) {
    const int y = sh.wave[i];
    if (i < w) before += y;
    sum += y;
  }
  *all = sum;
  return before + incl - x;
}

// Sum over the wave's lanes
template <int kCtrl>
__device__ __forceinline__ int lane_add(int x) {
  return x + __builtin_amdgcn_mov_dpp(x, kCtrl, 0xf, 0xf, false);
}
__device__ __forceinline__ int lane_sum(int x) {
  x = lane_add<0xB1>(x);   // quad_perm [1, 0, 3, 2]
  x = lane_add<0x4E>(x);   // quad_perm [2, 3, 0, 1]
  x = lane_add<0x141>(x);  // row_half_mirror
  x = lane_add<0x140>(x);  // row_mirror
  const auto y = __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false);
  x = (int)(y[0] + y[1]);
  const auto z = __builtin_amdgcn_permlane32_swap((uint32_t)x, (uint32_t)x, false, false);
  return (int)(z[0] + z[1]);
}
// Sums of two numbers over all threads
__device__ __forceinline__ void plan_sums(PlanShared& sh, int* a, int* b) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  *a = lane_sum(*a);
  *b = lane_sum(*b);
  __syncthreads();
  if (lane == 0) {
    sh.wave[w] = *a;
    sh.second[w] = *b;
  }
  __syncthreads();
  *a = *b = 0;
#pragma unroll
  for (int i = 0; i < kPlanWaves; ++i) {
    *a += sh.wave[i];
    *b += sh.second[i];
  }
}

// The counts of 16 pages from `at` on; -1 past the pool
struct Counts {
  int32_t n[kPlanPer];
};
__device__ __forceinline__ Counts plan_counts(const PagesParams& g, int at) {
  Counts c;
  if (at + kPlanPer <= g.n_pages) {
    struct __attribute__((packed, aligned(4))) Any {
      u32x4 x;
    };
#pragma unroll
    for (int i = 0; i < kPlanPer / 4; ++i) {
      const u32x4 x = ((const WNW_GLOBAL Any*)(uintptr_t)(g.refs + at + 4 * i))->x;
#pragma unroll
      for (int j = 0; j < 4; ++j) c.n[4 * i + j] = (int32_t)x[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) c.n[i] = at + i < g.n_pages ? g.refs[at + i] : -1;
  }
  return c;
}

// The first `need` free pages into the fresh list; whether there are as many.  c: the
// thread's counts of the pool's first pages, on their way since before the need was known.
__device__ __forceinline__ bool plan_fresh(const PagesParams& g, PlanShared& sh, int need, Counts c) {
  int have = 0;
  for (int base = 0; base < g.n_pages && have < need; base += kPlanThreads * kPlanPer) {
    const int at = base + (int)threadIdx.x * kPlanPer;
    int mine = 0;
    if (at < g.n_pages) {
      if (base > 0) c = plan_counts(g, at);
#pragma unroll
      for (int i = 0; i < kPlanPer; ++i) mine += c.n[i] == 0;
    }
    int all;
    int rank = have + plan_scan(sh, mine, &all);
    if (mine > 0) {
#pragma unroll
      for (int i = 0; i < kPlanPer; ++i)
        if (c.n[i] == 0) {
          if (rank < need) ws_fresh(g)[rank] = at + i;
          ++rank;
        }
    }
    have += all;
  }
  return have >= need;
}

// The plan's other workgroups copy the counts
__device__ __forceinline__ void plan_copy(const PagesParams& g) {
  constexpr int N = kPlanCopy / kPlanThreads;
  const int from = ((int)blockIdx.x - 1) * kPlanCopy + (int)threadIdx.x;
  int32_t x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = g.refs[min(from + i * kPlanThreads, g.n_pages - 1)];
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (from + i * kPlanThreads < g.n_pages) g.new_refs[from + i * kPlanThreads] = x[i];
}
// A table entry: the page, or -1
__device__ __forceinline__ int entry_of(const PagesParams& g, int e, bool tell) {
  if ((uint32_t)e < (uint32_t)g.n_pages) return e;
  if (e != -1 && tell) raise_device_error(g.err, WNW_DEVERR_BOUNDS);
  return -1;
}
__device__ __forceinline__ void plan_end(const PagesParams& g, bool good, bool room) {
  if (threadIdx.x != 0) return;
  g.ws[kOk] = good && room;
  if (!good)
    raise_device_error(g.err, WNW_DEVERR_BOUNDS);
  else if (!room)
    raise_device_error(g.err, WNW_DEVERR_CAPACITY);
}

// ---------------------------------------------------------------------------
// fork
// ---------------------------------------------------------------------------
__device__ __forceinline__ int32_t* fork_first(const ForkParams& p) { return ws_place(p.g) + (int64_t)p.n_new * p.heads; }

__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(ForkParams p) {
  __shared__ PlanShared sh;
  __shared__ int first[kMaxSamples], count[kMaxSamples];  // of each parent: its first child, its children
  const PagesParams& g = p.g;
  if (blockIdx.x > 0) {
    plan_copy(g);
    return;
  }
  const int tid = threadIdx.x, rows = g.max_blocks << g.shift;
  const Counts counts = plan_counts(g, tid * kPlanPer);
  bool good = true;
  for (int i = tid; i < p.n_old; i += kPlanThreads) {
    first[i] = 0x7fffffff;
    count[i] = 0;
  }
  __syncthreads();
  for (int i = tid; i < p.n_new; i += kPlanThreads) {
    const int a = p.parents[i];
    if (a >= 0 && a < p.n_old) {
      atomicMin(&first[a], i);
      atomicAdd(&count[a], 1);
    } else {
      good &= a == -1;
    }
  }
  for (int s = tid; s < g.n_seg; s += kPlanThreads) {
    const int n = g.seg_len[s];
    good &= n >= 0 && n <= rows;
  }
  good = __syncthreads_and(good);
  bool room = true;
  if (good) {
    int need = 0;
    const int segs = p.n_new * p.heads;
    for (int base = 0; base < segs; base += kPlanThreads) {
      const int s = base + tid;
      bool mine = false;
      if (s < segs) {
        const int i = s / p.heads, a = p.parents[i];
        if (a >= 0 && first[a] != i) {
          const int from = a * p.heads + s - i * p.heads, n = g.seg_len[from];
          mine = (n & ((1 << g.shift) - 1)) != 0 && entry_of(g, g.table[from * g.stride + (n >> g.shift)], false) >= 0;
        }
      }
      int all;
      const int at = need + plan_scan(sh, mine, &all);
      if (s < segs) ws_place(g)[s] = mine ? at : -1;
      need += all;
    }
    room = plan_fresh(g, sh, need, counts);
    for (int i = tid; i < p.n_old; i += kPlanThreads) {
      fork_first(p)[i] = first[i];
      fork_first(p)[p.n_old + i] = count[i];
    }
  }
  plan_end(g, good, room);
}

// A workgroup for each new segment, then one for each old one (whose counts change)
__global__ __launch_bounds__(256) void fork_kernel(ForkParams p) {
  const PagesParams& g = p.g;
  const int tid = threadIdx.x, segs = p.n_new * p.heads;
  const bool ok = g.ws[kOk] != 0;
  if ((int)blockIdx.x < segs) {
    const int s = blockIdx.x, i = s / p.heads, a = ok ? p.parents[i] : -1;
    const int from = max(a, 0) * p.heads + s - i * p.heads;
    const int n = a >= 0 ? g.seg_len[from] : 0, full = n >> g.shift, part = n & ((1 << g.shift) - 1);
    const bool more = a >= 0 && fork_first(p)[a] != i;
    const int place = more ? ws_place(g)[s] : -1;
    const int fresh = place >= 0 ? ws_fresh(g)[place] : -1;
    for (int j = tid; j < g.max_blocks; j += 256) {
      int e = -1;
      if (a >= 0 && (!more || j < full || (j == full && fresh >= 0))) e = entry_of(g, g.table[from * g.stride + j], true);
      if (more && j == full && fresh >= 0) {
        p.copies[3 * s] = e;
        e = fresh;
      }
      g.new_table[s * g.new_stride + j] = e;
    }
    if (tid == 0) {
      p.new_len[s] = n;
      if (fresh >= 0) {
        atomicAdd(&g.new_refs[fresh], 1);
      } else {
        p.copies[3 * s] = -1;
      }
      p.copies[3 * s + 1] = fresh;
      p.copies[3 * s + 2] = fresh >= 0 ? part : 0;
    }
  } else if (ok) {
    const int s = blockIdx.x - segs, children = fork_first(p)[p.n_old + s / p.heads], full = g.seg_len[s] >> g.shift;
    if (children == 1) return;
    for (int j = tid; j < (children ? full : g.max_blocks); j += 256) {
      const int e = entry_of(g, g.table[s * g.stride + j], false);
      if (e >= 0) atomicAdd(&g.new_refs[e], children - 1);
    }
  }
}

// ---------------------------------------------------------------------------
// reserve
// ---------------------------------------------------------------------------
// A segment's rows before and after, and what of it goes: blocks from `sinks` rows
// on that end at or below row `low`.
struct ReserveSeg {
  int n, end, sinks, low;
  bool good;
};
__device__ __forceinline__ ReserveSeg reserve_seg(const ReserveParams& p, int s) {
  ReserveSeg r;
  const int rows = p.g.max_blocks << p.g.shift;
  r.n = p.g.seg_len[s];
  int t = p.tokens;
  r.good = r.n >= 0 && r.n <= rows;
  if (p.cu) {
    const int b = s / p.heads, from = p.cu[b], to = p.cu[b + 1];
    t = to - from;
    r.good &= from >= 0 && to >= from;
  }
  r.end = (int)min((int64_t)r.n + t, (int64_t)0x7fffffff);
  r.sinks = r.low = 0;
  if (p.windowed) {
    int w;
    r.good &= paged_view_of(p.view, s, r.n + 1, &w, &r.sinks);
    r.low = r.n + 1 - max(w, 1);
  }
  return r;
}
__device__ __forceinline__ bool reserve_needs(const ReserveParams& p, const ReserveSeg& r, int j, int e) {
  return e < 0 && j >= r.n >> p.g.shift && (int64_t)j << p.g.shift < r.end;
}

__global__ __launch_bounds__(kPlanThreads) void reserve_plan_kernel(ReserveParams p) {
  __shared__ PlanShared sh;
  __shared__ unsigned long long total;
  const PagesParams& g = p.g;
  if (blockIdx.x > 0) {
    plan_copy(g);
    return;
  }
  const int tid = threadIdx.x, rows = g.max_blocks << g.shift;
  const Counts counts = plan_counts(g, tid * kPlanPer);
  bool good = true, room = true;
  if (tid == 0) total = 0;
  __syncthreads();
  // a segment's needs: of one thread where they are a block or two, of a wave otherwise
  if (!p.wide && g.n_seg <= kPlanThreads) {  // (a decode step's call: nothing goes through memory)
    __shared__ int bad;
    if (tid == 0) bad = 0;
    __syncthreads();
    int mine = 0;
    if (tid < g.n_seg) {
      const ReserveSeg r = reserve_seg(p, tid);
      const int b0 = r.n >> g.shift;
      if (!r.good || r.end > rows) {
        atomicOr(&bad, r.good ? 2 : 1);
      } else if (r.end > r.n) {
        const int e0 = g.table[tid * g.stride + b0], e1 = g.table[tid * g.stride + min(b0 + 1, g.max_blocks - 1)];
        mine = (entry_of(g, e0, false) < 0) + ((b0 + 1) << g.shift < r.end && entry_of(g, e1, false) < 0);
      }
    }
    int need;
    const int before = plan_scan(sh, mine, &need);
    good = !(bad & 1);
    room = !(bad & 2) && need <= g.n_pages;
    if (good && room) {
      if (tid < g.n_seg) ws_place(g)[tid] = before;
      room = plan_fresh(g, sh, need, counts);
    }
    plan_end(g, good, room);
    return;
  }
  if (p.wide) {
    const int lane = tid & 63;
    for (int s = tid >> 6; s < g.n_seg; s += kPlanWaves) {
      const ReserveSeg r = reserve_seg(p, s);
      int mine = 0;
      good &= r.good;
      room &= r.end <= rows;
      if (r.good && r.end <= rows)
        for (int j = (r.n >> g.shift) + lane; (int64_t)j << g.shift < r.end; j += 64)
          mine += entry_of(g, g.table[s * g.stride + j], false) < 0;
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) mine += __shfl_xor(mine, o);
      if (lane == 0) {
        ws_place(g)[s] = mine;
        atomicAdd(&total, (unsigned long long)mine);
      }
    }
  } else {
    for (int s = tid; s < g.n_seg; s += kPlanThreads) {
      const ReserveSeg r = reserve_seg(p, s);
      int mine = 0;
      good &= r.good;
      room &= r.end <= rows;
      if (r.good && r.end <= rows)
        for (int j = r.n >> g.shift; (int64_t)j << g.shift < r.end; ++j) mine += entry_of(g, g.table[s * g.stride + j], false) < 0;
      ws_place(g)[s] = mine;
      if (mine) atomicAdd(&total, (unsigned long long)mine);
    }
  }
  good = __syncthreads_and(good);
  room = __syncthreads_and(room);
  room &= total <= (unsigned long long)g.n_pages;  // below 2^30
  if (good && room) {
    int need = 0;
    for (int base = 0; base < g.n_seg; base += kPlanThreads) {
      const int s = base + tid, mine = s < g.n_seg ? ws_place(g)[s] : 0;
      int all;
      const int before = plan_scan(sh, mine, &all);
      if (s < g.n_seg) ws_place(g)[s] = need + before;
      need += all;
    }
    room = plan_fresh(g, sh, need, counts);
  }
  plan_end(g, good, room);
}

// A workgroup for each segment
__global__ __launch_bounds__(256) void reserve_kernel(ReserveParams p) {
  __shared__ int sums[4];
  const PagesParams& g = p.g;
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int32_t* from = g.table + s * g.stride;
  int32_t* to = g.new_table + s * g.new_stride;
  if (!g.ws[kOk]) {
    if (from != to)
      for (int j = tid; j < g.max_blocks; j += 256) to[j] = from[j];
    return;
  }
  const ReserveSeg r = reserve_seg(p, s);
  int at = ws_place(g)[s];
  for (int base = 0; base < g.max_blocks; base += 256) {
    const int j = base + tid;
    int e = j < g.max_blocks ? entry_of(g, from[j], true) : -1;
    const bool need = j < g.max_blocks && reserve_needs(p, r, j, e);
    if (base + 256 > r.n >> g.shift && (int64_t)base << g.shift < r.end) {  // some of these may
      const uint64_t all = __ballot(need);
      __syncthreads();
      if (lane == 0) sums[w] = __popcll(all);
      __syncthreads();
      int rank = at + __popcll(all & ((1ull << lane) - 1));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i < w) rank += sums[i];
        at += sums[i];
      }
      if (need) {
        e = ws_fresh(g)[rank];
        atomicAdd(&g.new_refs[e], 1);
      }
    }
    if (!need && e >= 0 && p.windowed && (int64_t)j << g.shift >= r.sinks && (int64_t)(j + 1) << g.shift <= r.low) {
      atomicAdd(&g.new_refs[e], -1);
      e = -1;
    }
    if (j < g.max_blocks) to[j] = e;
  }
}

// ---------------------------------------------------------------------------
// compact
// ---------------------------------------------------------------------------
// The lists: of a used page at U or above, or a free one below, its rank among such
// (place; -1 of the others); by rank, the free ones (fresh), and the used ones above and
// their counts.
__device__ __forceinline__ int32_t* compact_page(const PagesParams& g) { return ws_place(g) + g.n_pages; }
__device__ __forceinline__ int32_t* compact_refs(const PagesParams& g) { return compact_page(g) + g.n_pages / 2 + 1; }

// A workgroup for `range` pages, which counts the used ones of the whole pool for itself:
// how many there are, U, how many below its pages, and (where these lie past U) below U.
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(CompactParams p) {
  __shared__ PlanShared sh;
  const PagesParams& g = p.g;
  const int tid = threadIdx.x, from = (int)blockIdx.x * p.range, to = min(from + p.range, g.n_pages);
  const Counts head = plan_counts(g, tid * kPlanPer);
  const int own0 = from + tid < to ? g.refs[from + tid] : 0;
  auto count = [&](int x, int* below) {  // used pages, and those below page x
    int all = 0, low = 0;
    for (int at = tid * kPlanPer; at < g.n_pages; at += kPlanThreads * kPlanPer) {
      const Counts c = at < kPlanThreads * kPlanPer ? head : plan_counts(g, at);
#pragma unroll
      for (int i = 0; i < kPlanPer; ++i) {
        all += c.n[i] != 0;
        low += c.n[i] != 0 && at + i < x;
      }
      all -= max(at + kPlanPer - g.n_pages, 0);  // those past the pool
    }
    plan_sums(sh, &all, &low);
    *below = low;
    return all;
  };
  int before, under;
  const int used = count(from, &before);
  if (from > used)
    count(used, &under);
  else
    under = -1;  // found on the way
  int at_u = under;
  // its pages, 1,024 at a time
  int seen = before;  // used ones below the thread's
  for (int base = from; base < to; base += kPlanThreads) {
    const int i = base + tid, c = base == from ? own0 : i < to ? g.refs[i] : 0;
    int all;
    const int mine = seen + plan_scan(sh, c != 0, &all);
    if (at_u < 0 && base <= used && used < base + kPlanThreads) {  // uniform
      __shared__ int found;
      if (i == used) found = mine;
      __syncthreads();
      at_u = found;
    }
    if (i < to) {
      if (i < used) {
        if (c == 0) ws_fresh(g)[i - mine] = i;
        ws_place(g)[i] = c == 0 ? i - mine : -1;
      } else {
        const int rank = mine - at_u;
        if (c != 0) {
          compact_page(g)[rank] = i;
          compact_refs(g)[rank] = c;
        }
        ws_place(g)[i] = c != 0 ? rank : -1;
      }
    }
    seen += all;
  }
  if (blockIdx.x == gridDim.x - 1 && tid == 0) {
    g.ws[kUsed] = used;
    g.ws[kMoves] = at_u < 0 ? 0 : used - at_u;
  }
}

// Workgroups of the segments, then of 256 pages each
__global__ __launch_bounds__(256) void compact_kernel(CompactParams p) {
  const PagesParams& g = p.g;
  const int tid = threadIdx.x, used = g.ws[kUsed], movers = g.ws[kMoves];
  if ((int)blockIdx.x < g.n_seg) {
    const int s = blockIdx.x;
    for (int j = tid; j < g.max_blocks; j += 256) {
      int e = entry_of(g, g.table[s * g.stride + j], true);
      if (e >= 0) {
        const int rank = ws_place(g)[e];
        if (e < used ? rank >= 0 : rank < 0) {  // the counts call it free: another page may land in it
          raise_device_error(g.err, WNW_DEVERR_BOUNDS);
          e = -1;
        } else if (e >= used) {
          e = ws_fresh(g)[rank];
        }
      }
      g.new_table[s * g.new_stride + j] = e;
    }
    return;
  }
  const int i = ((int)blockIdx.x - g.n_seg) * 256 + tid;
  if (i == 0) *p.used = used;
  if (i < g.n_pages) {
    if (i < g.n_pages / 2) {
      const bool is = i < movers;
      p.moves[3 * i] = is ? compact_page(g)[i] : -1;
      p.moves[3 * i + 1] = is ? ws_fresh(g)[i] : -1;
      p.moves[3 * i + 2] = is ? 1 << g.shift : 0;
    }
    const int c = g.refs[i];
    g.new_refs[i] = i >= used ? 0 : c != 0 ? c : compact_refs(g)[ws_place(g)[i]];
  }
}

// ---------------------------------------------------------------------------
// copy
// ---------------------------------------------------------------------------
struct PagedCopyParams {
  PagedCache c;
  const int32_t* copies;
  int64_t n;
  int32_t row_bytes;
  int32_t* err;
};
// blockIdx.y: K or V
__global__ __launch_bounds__(256) void paged_copy_kernel(PagedCopyParams p) {
  const bool v = blockIdx.y != 0;
  const int64_t stride = v ? p.c.v_stride : p.c.k_stride;
  uint8_t* const pages = v ? p.c.v : p.c.k;
  float* const scales = v ? p.c.v_scale : p.c.k_scale;
  for (int64_t i = blockIdx.x; i < p.n; i += gridDim.x) {
    const int src = p.copies[3 * i], dst = p.copies[3 * i + 1], rows = p.copies[3 * i + 2];
    if (src < 0) continue;
    if (src >= p.c.n_pages || (uint32_t)dst >= (uint32_t)p.c.n_pages || src == dst || rows < 0 || rows > 1 << p.c.shift) {
      if (threadIdx.x == 0 && !v) raise_device_error(p.err, WNW_DEVERR_BOUNDS);
      continue;
    }
    const WNW_GLOBAL u32x4* from = gptr<u32x4>(pages + src * stride);
    WNW_GLOBAL u32x4* to = gptr_w<u32x4>(pages + dst * stride);
    const int chunks = rows * p.row_bytes / 16;
    for (int c = threadIdx.x; c < chunks; c += 4 * 256) {
      u32x4 x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c + u * 256 < chunks) x[u] = from[c + u * 256];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c + u * 256 < chunks) to[c + u * 256] = x[u];
    }
    if (scales && threadIdx.x == 0) scales[dst] = scales[src];
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
bool paged_view_host(const int32_t* window, int64_t window_all, const int32_t* sinks, int64_t sinks_all, PagedView* out);

static bool apart(const void* a, int64_t n, const void* b, int64_t m) {  // bytes
  return n == 0 || m == 0 || (const uint8_t*)a + n <= (const uint8_t*)b || (const uint8_t*)b + m <= (const uint8_t*)a;
}
static int64_t table_bytes(int64_t n_seg, int64_t stride, int64_t blocks) { return n_seg ? ((n_seg - 1) * stride + blocks) * 4 : 0; }
static int64_t pages_workspace(int64_t n_seg, int64_t n_samples, int64_t n_pages) {
  return (kHead + 3 * n_pages + 2 + n_seg + 2 * n_samples + 63) / 64 * 256;
}

static int pages_of(const int32_t* table, int64_t stride, const int32_t* seg_len, const int32_t* page_refs, int64_t n_seg, int64_t max_blocks,
                    int64_t n_pages, int64_t page_rows, int32_t* new_table, int64_t new_stride, int32_t* new_refs,
                    int64_t new_seg, int64_t n_samples, bool in_place, void* workspace, int64_t bytes, PagesParams* g) {
  int shift = 4;
  while (shift < 8 && (1 << shift) != page_rows) ++shift;
  WNW_CHECK_ARG((1 << shift) == page_rows, "page_rows must be 16, 32, 64, 128 or 256");
  WNW_CHECK_ARG(n_seg >= 0 && n_seg < (1 << 23) && new_seg < (1 << 23) && n_pages >= 0 && n_pages < (1 << 30) && max_blocks >= 0 &&
                    max_blocks <= (1 << 30) / page_rows && stride >= max_blocks && new_stride >= max_blocks &&
                    stride < (1ll << 31) && new_stride < (1ll << 31),
                "bad sizes of the page table");
  const bool entries = n_seg > 0 && max_blocks > 0, new_entries = new_seg > 0 && max_blocks > 0;
  WNW_CHECK_ARG((!entries || table) && (!new_entries || new_table) && (n_pages == 0 || (page_refs && new_refs)),
                "null pointer argument");
  const int64_t old_bytes = entries ? table_bytes(n_seg, stride, max_blocks) : 0;
  const int64_t new_bytes = new_entries ? table_bytes(new_seg, new_stride, max_blocks) : 0;
  WNW_CHECK_ARG(apart(table, old_bytes, new_table, new_bytes) || (in_place && table == new_table && stride == new_stride),
                "new_table overlaps page_table");
  WNW_CHECK_ARG(apart(page_refs, 4 * n_pages, new_refs, 4 * n_pages) || (in_place && page_refs == new_refs),
                "new_refs overlaps page_refs");
  WNW_CHECK_ARG(apart(new_table, new_bytes, new_refs, 4 * n_pages) && apart(new_table, new_bytes, page_refs, 4 * n_pages) &&
                    apart(new_refs, 4 * n_pages, table, old_bytes) && apart(new_table, new_bytes, seg_len, seg_len ? 4 * n_seg : 0) &&
                    apart(new_refs, 4 * n_pages, seg_len, seg_len ? 4 * n_seg : 0),
                "an output overlaps another array");
  WNW_CHECK_ARG(workspace && bytes >= pages_workspace(std::max(n_seg, new_seg), n_samples, n_pages),
                "workspace too small: %lld bytes", (long long)bytes);
  WNW_CHECK_ARG((uintptr_t)workspace % 256 == 0, "the workspace must be 256-byte aligned");
  *g = PagesParams{table, new_table, stride, new_stride, seg_len, page_refs, new_refs, (int32_t*)workspace, device_error_word(),
                   (int32_t)n_seg, (int32_t)max_blocks, (int32_t)n_pages, shift};
  return WNW_OK;
}
static unsigned plan_blocks(const PagesParams& g) {  // the plan's own, and those that copy the counts
  return 1 + (g.refs == g.new_refs ? 0 : (unsigned)((g.n_pages + kPlanCopy - 1) / kPlanCopy));
}

}  // namespace wnw

using namespace wnw;

extern "C" int64_t wnw_pages_workspace_bytes(int64_t n_seg, int64_t n_samples, int64_t n_pages) {
  if (n_seg < 0 || n_seg >= (1 << 23) || n_samples < 0 || n_samples > (1 << 23) || n_pages < 0 || n_pages >= (1 << 30)) return -1;
  return pages_workspace(n_seg, n_samples, n_pages);
}

extern "C" int wnw_paged_fork(const int32_t* page_table, int64_t table_stride, const int32_t* seg_len, const int32_t* page_refs,
                              const int32_t* parents, int64_t n_old, int64_t n_new, int64_t kv_heads, int64_t max_blocks,
                              int64_t n_pages, int64_t page_rows, int32_t* new_table, int64_t new_stride, int32_t* new_len,
                              int32_t* new_refs, int32_t* copies, void* workspace, int64_t workspace_bytes, void* stream) {
  ForkParams p = {};
  WNW_CHECK_ARG(n_old >= 0 && n_old <= kMaxSamples && n_new >= 0 && n_new <= kMaxSamples && kv_heads >= 1 && kv_heads <= 1024,
                "at most %d samples before and after, and 1,024 KV heads", kMaxSamples);
  const int64_t N = n_old * kv_heads, M = n_new * kv_heads;
  if (int rc = pages_of(page_table, table_stride, seg_len, page_refs, N, max_blocks, n_pages, page_rows, new_table, new_stride, new_refs, M,
                        n_old, false, workspace, workspace_bytes, &p.g))
    return rc;
  WNW_CHECK_ARG((N == 0 || seg_len) && (M == 0 || (parents && new_len && copies)), "null pointer argument");
  WNW_CHECK_ARG(N == 0 || M == 0 || apart(seg_len, 4 * N, new_len, 4 * M), "new_len overlaps seg_len");
  p.parents = parents;
  p.new_len = new_len;
  p.copies = copies;
  p.n_old = (int32_t)n_old;
  p.n_new = (int32_t)n_new;
  p.heads = (int32_t)kv_heads;
  hipLaunchKernelGGL(fork_plan_kernel, dim3(plan_blocks(p.g)), dim3(kPlanThreads), 0, (hipStream_t)stream, p);
  if (N + M > 0) hipLaunchKernelGGL(fork_kernel, dim3((unsigned)(N + M)), dim3(256), 0, (hipStream_t)stream, p);
  WNW_CHECK_HIP(hipGetLastError(), "fork launch");
  return WNW_OK;
}

extern "C" int wnw_paged_reserve(const int32_t* page_table, int64_t table_stride, const int32_t* seg_len, const int32_t* page_refs,
                                 int64_t n_seg, int64_t n_samples, int64_t max_blocks, int64_t n_pages, int64_t page_rows,
                                 const int32_t* cu_tokens, int64_t tokens, const int32_t* window, int64_t window_all,
                                 const int32_t* sinks, int64_t sinks_all, int32_t* new_table, int64_t new_stride,
                                 int32_t* new_refs, void* workspace, int64_t workspace_bytes, void* stream) {
  ReserveParams p = {};
  WNW_CHECK_ARG(n_samples >= 0 && (n_samples > 0 ? n_seg % n_samples == 0 : n_seg == 0), "segments must be samples x KV heads");
  WNW_CHECK_ARG(cu_tokens || (tokens >= 0 && tokens <= (1 << 30)), "bad token count");
  if (int rc = pages_of(page_table, table_stride, seg_len, page_refs, n_seg, max_blocks, n_pages, page_rows, new_table, new_stride,
                        new_refs, n_seg, n_samples, true, workspace, workspace_bytes, &p.g))
    return rc;
  WNW_CHECK_ARG(n_seg == 0 || seg_len, "null pointer argument");
  p.windowed = window || window_all >= 0;
  if (p.windowed && !paged_view_host(window, window_all, sinks, sinks_all, &p.view)) return WNW_EINVAL;
  p.cu = cu_tokens;
  p.tokens = cu_tokens ? 0 : (int32_t)tokens;
  p.heads = n_samples ? (int32_t)(n_seg / n_samples) : 1;
  p.wide = cu_tokens || tokens > page_rows;
  hipLaunchKernelGGL(reserve_plan_kernel, dim3(plan_blocks(p.g)), dim3(kPlanThreads), 0, (hipStream_t)stream, p);
  if (n_seg > 0) hipLaunchKernelGGL(reserve_kernel, dim3((unsigned)n_seg), dim3(256), 0, (hipStream_t)stream, p);
  WNW_CHECK_HIP(hipGetLastError(), "reserve launch");
  return WNW_OK;
}

extern "C" int wnw_paged_compact(const int32_t* page_table, int64_t table_stride, const int32_t* page_refs, int64_t n_seg,
                                 int64_t max_blocks, int64_t n_pages, int64_t page_rows, int32_t* new_table, int64_t new_stride,
                                 int32_t* new_refs, int32_t* moves, int32_t* used, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  CompactParams p = {};
  if (int rc = pages_of(page_table, table_stride, nullptr, page_refs, n_seg, max_blocks, n_pages, page_rows, new_table, new_stride,
                        new_refs, n_seg, 0, true, workspace, workspace_bytes, &p.g))
    return rc;
  WNW_CHECK_ARG(used && (n_pages < 2 || moves), "null pointer argument");
  p.moves = moves;
  p.used = used;
  // each of at most 64 workgroups reads all counts: from its L2
  p.range = (int32_t)(((n_pages + 63) / 64 + kPlanThreads - 1) / kPlanThreads * kPlanThreads);
  const unsigned plan = n_pages ? (unsigned)((n_pages + p.range - 1) / p.range) : 1;
  hipLaunchKernelGGL(compact_plan_kernel, dim3(plan), dim3(kPlanThreads), 0, (hipStream_t)stream, p);
  const unsigned blocks = (unsigned)(n_seg + std::max<int64_t>((n_pages + 255) / 256, 1));
  hipLaunchKernelGGL(compact_kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, p);
  WNW_CHECK_HIP(hipGetLastError(), "compact launch");
  return WNW_OK;
}

extern "C" int wnw_paged_copy(const wnw_paged_cache* cache, const int32_t* copies, int64_t n_copies, void* stream) {
  PagedCopyParams p = {};
  WNW_CHECK_ARG(cache != nullptr, "the cache description is null");
  wnw_paged_cache pages = *cache;  // the table is not looked at
  pages.n_seg = pages.max_blocks = pages.table_stride = 0;
  pages.page_table = nullptr;
  if (int rc = paged_cache_of(&pages, &p.c)) return rc;
  WNW_CHECK_ARG(n_copies >= 0 && (n_copies == 0 || copies), "bad copies");
  if (n_copies == 0 || cache->n_pages == 0) return WNW_OK;
  p.copies = copies;
  p.n = n_copies;
  p.row_bytes = (int32_t)(cache->head_dim * (cache->page_dtype == WNW_E4M3 ? 1 : 2));
  p.err = device_error_word();
  hipLaunchKernelGGL(paged_copy_kernel, dim3((unsigned)std::min<int64_t>(n_copies, 4096), 2), dim3(256), 0, (hipStream_t)stream, p);
  WNW_CHECK_HIP(hipGetLastError(), "page copy launch");
  return WNW_OK;
}
