// Selection of a beam search's next beams (gfx950): the k best continuations of
// each sample, over all of its beams and the vocabulary.
//
// Mathematics: candidate (w, v) has total(w, v) = score_w + (x_wv - lse_w), lse_w =
// log sum_v exp x_wv; the k largest totals, equal ones by the lower (w, v).  Totals are
// formed and compared in 64 bits.  Within a beam they go with the logits, so a beam need
// not be sorted, and its order is exact.  Between beams it is up to what lse is off:
// exponentials, their arguments and sums of 4 or 8 of them are in 32 bits (an exponential
// is one instruction, in 64 bits a polynomial), what follows in 64.  An argument d = x - max,
// |d| log2 e, is off by 2.3 * 2^-24 of its size, its exponential by twice 2^-24 more, a sum
// of 8 by 7 times; the same for the factor that joins tasks, and for each 64 tasks past the
// first 64 of a row once more 2 * 2^-24.  The mean of |d| under a softmax of n terms is at
// most 11 for n = 2^20 (t - 1 with t = 1 + n exp(-t)): in all 2.3 * 11 + 2 + 7 + 2 + 14 = 50
// times 2^-24, below 2^-18, up to 2^20 tokens.
//
// Two launches.  The first reads the logits once: a wave takes 2,048 of a row and
// leaves their maximum, sum exp(x - max) and the maximum of each group of 128.  In
// the second, a workgroup a sample puts the sums together, finds the k best groups
// by their maxima (the k best elements lie in those: each other group is behind k
// maxima), reads these alone again, and ranks what is not below the k-th group's
// maximum.
//
// What bounds it: memory for many rows (512 of 51,865 f16 logits, a fifth of the beams
// finished, 43 MB: 12.9 us for the first launch, 3.3 TB/s; 7.7 for the second), else the
// launches and a chain of dependent loads (5 rows of 32,000: 3.5 and 6.7; 32 of
// 131,072 f32: 6.6 and 8.0).  One launch, whose last workgroup of a sample to arrive does
// the second's work: 10.5, 14.5 and 35.0 us in all, for 10.6, 13.8 and 19.2: what is left
// for another workgroup has to pass by the caches.
#include "wnw_common.h"

namespace wnw {

static constexpr int kBeamTask = 2048;    // logits of a wave: four to eight loads in flight
static constexpr int kBeamThreads = 1024; // of a sample's workgroup
static constexpr int kBeamMax = 64;       // beams, and candidates to select
static constexpr int kBeamList = 512;     // candidates that are ranked against each other; more go in k rounds of a maximum
static constexpr float kBeamLog2e = 1.4426950408889634f;
static constexpr float kBeamLowest = -3.402823466e38f;  // running maxima start here

struct BeamParams {
  const void* logits;
  const float* scores;  // [B, W]
  const uint8_t* done;  // [B, W] or null
  double* part_sum;     // [rows, tasks]
  float* part_max;      // [rows, tasks]
  float* group_max;     // [rows, tasks, kBeamGroups]
  float* out_scores;    // [B, k]
  int32_t* out_parents;
  int64_t* out_tokens;
  int32_t* err;
  int64_t stride_b, stride_w;  // in elements
  int32_t B, W, V, k, tasks, end;
};

static constexpr int kBeamGroup = 128;                     // logits of a group
static constexpr int kBeamGroups = kBeamTask / kBeamGroup;  // of a task
static constexpr int kBeamWaves = kBeamThreads / 64;
static constexpr int kBeamHeld = 8;  // chunks of 64 groups whose maxima a wave of the pick holds

template <typename T>
struct BeamGeom {
  static constexpr int kVec = 16 / Elem<T>::kBytes;        // elements of a load
  static constexpr int kLoads = kBeamTask / (64 * kVec);   // of a lane in a task
  static constexpr int kEach = kBeamGroup / 16;            // elements of a thread of the 16 that read a group again
};

// Elements e .. e + kVec - 1 of a row of V, those past its end -inf.  Rows may
// start at any element: a load near the end is taken from the row's last kVec.
template <typename T>
__device__ __forceinline__ void beam_load(const T* row, int e, int V, u32x4* raw, int* from) {
  constexpr int N = BeamGeom<T>::kVec;
  struct __attribute__((packed, aligned(Elem<T>::kBytes))) Any {
    u32x4 x;
  };
  *from = max(min(e, V - N), 0);
  if (V >= N) {
    *raw = ((const WNW_GLOBAL Any*)(uintptr_t)(row + *from))->x;
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
    for (int i = 0; i < V; ++i) {
      if constexpr (Elem<T>::kBytes == 4)
        w[i] = ((const uint32_t*)row)[i];
      else
        w[i >> 1] |= (uint32_t)((const uint16_t*)row)[i] << (16 * (i & 1));
    }
    *raw = u32x4{w[0], w[1], w[2], w[3]};
  }
}
template <typename T>
__device__ __forceinline__ void beam_values(const u32x4& raw, int e, int from, int V, float* x) {
  constexpr int N = BeamGeom<T>::kVec;
  if constexpr (Elem<T>::kBytes == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __uint_as_float(raw[i]);
  } else {
    unpack8(raw, x, (T*)nullptr);
  }
  if (from != e || e + N > V) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (from + i < e || from + i >= V) x[i] = -INFINITY;
  }
}

template <int kCtrl>
__device__ __forceinline__ float dpp_max(float x) {
  return fmaxf(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), kCtrl, 0xf, 0xf, false)));
}
// Maximum over the 16 lanes of a row
__device__ __forceinline__ float max_row16(float x) {
  x = dpp_max<0xB1>(x);   // quad_perm [1, 0, 3, 2]
  x = dpp_max<0x4E>(x);   // quad_perm [2, 3, 0, 1]
  x = dpp_max<0x141>(x);  // row_half_mirror
  return dpp_max<0x140>(x);
}
// Maximum and sum over the wave, without LDS
__device__ __forceinline__ float beam_max(float x) { return max_x32(max_x16(max_row16(x))); }
__device__ __forceinline__ double f64_of(uint32_t lo, uint32_t hi) {
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int kCtrl>
__device__ __forceinline__ double dpp_sum64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return x + f64_of(__builtin_amdgcn_mov_dpp((int)(uint32_t)u, kCtrl, 0xf, 0xf, false),
                    __builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), kCtrl, 0xf, 0xf, false));
}
__device__ __forceinline__ double beam_sum64(double x) {
  x = dpp_sum64<0xB1>(x);
  x = dpp_sum64<0x4E>(x);
  x = dpp_sum64<0x141>(x);
  x = dpp_sum64<0x140>(x);
  {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)u, (uint32_t)u, false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
    x = f64_of(lo[0], hi[0]) + f64_of(lo[1], hi[1]);
  }
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const auto lo = __builtin_amdgcn_permlane32_swap((uint32_t)u, (uint32_t)u, false, false);
  const auto hi = __builtin_amdgcn_permlane32_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
  return f64_of(lo[0], hi[0]) + f64_of(lo[1], hi[1]);
}

template <typename T>
__global__ __launch_bounds__(256) void beam_rows_kernel(BeamParams p) {
  using Ge = BeamGeom<T>;
  constexpr int N = Ge::kVec, U = Ge::kLoads;
  static_assert(U <= 16, "a lane of 16 for each load's maximum");
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t at = (int64_t)blockIdx.x * 4 + w;  // the task
  if (at >= (int64_t)p.B * p.W * p.tasks) return;
  const int row = (int)(at / p.tasks), task = (int)(at - (int64_t)row * p.tasks);
  if (p.done && p.done[row]) return;  // its logits are not looked at
  const T* x0 = (const T*)p.logits + (int64_t)(row / p.W) * p.stride_b + (int64_t)(row % p.W) * p.stride_w;
  const int first = task * kBeamTask + lane * N;
  u32x4 raw[U];
  int from[U];
#pragma unroll
  for (int u = 0; u < U; ++u) beam_load<T>(x0, first + u * 64 * N, p.V, &raw[u], &from[u]);
  float x[U][N], most[U];
  float m = kBeamLowest;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    beam_values<T>(raw[u], first + u * 64 * N, from[u], p.V, x[u]);
    float y = x[u][0];
#pragma unroll
    for (int i = 1; i < N; ++i) y = fmaxf(y, x[u][i]);
    most[u] = max_row16(y);
    m = fmaxf(m, most[u]);
  }
  m = max_x32(max_x16(m));
  // (a logit of NaN or +inf leaves NaN in the sum: the pick refuses the beam)
  double sum = 0.0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += __builtin_amdgcn_exp2f((x[u][i] - m) * kBeamLog2e);
    sum += (double)s;
  }
  sum = beam_sum64(sum);
  if (lane == 0) {
    p.part_max[at] = m;
    p.part_sum[at] = sum;
  }
  // a group is a row of 16 lanes' load, or two rows' with 4 elements a load
  if constexpr (N == 4) {
#pragma unroll
    for (int u = 0; u < U; ++u) most[u] = max_x16(most[u]);
  }
  constexpr int R = N == 8 ? 4 : 2;  // groups of a load
  float mine = most[0];
#pragma unroll
  for (int u = 1; u < U; ++u) mine = (lane & 15) == u ? most[u] : mine;
  if ((lane & 15) < U && (N == 8 || !(lane & 16)))
    p.group_max[at * kBeamGroups + (lane & 15) * R + (lane >> (N == 8 ? 4 : 5))] = mine;
}

// A candidate's place in the order: its total as an ordered integer, and (w, v).
struct BeamKey {
  uint64_t total;
  uint32_t id;
};
__device__ __forceinline__ uint64_t ordered(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);  // -0 is 0
  return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double unordered(uint64_t u) {
  return __builtin_bit_cast(double, u >> 63 ? u & ~(1ull << 63) : ~u);
}
static constexpr BeamKey kBeamNone = {0, 0xffffffffu};  // behind every candidate
__device__ __forceinline__ bool ahead(const BeamKey& a, const BeamKey& b) {
  return a.total > b.total || (a.total == b.total && a.id < b.id);
}
__device__ __forceinline__ BeamKey ahead_of(const BeamKey& a, const BeamKey& b) { return ahead(a, b) ? a : b; }
__device__ __forceinline__ BeamKey wave_first(BeamKey x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const BeamKey y = {(uint64_t)__shfl_xor((unsigned long long)x.total, o), (uint32_t)__shfl_xor((int)x.id, o)};
    x = ahead_of(x, y);
  }
  return x;
}

struct BeamShared {
  double lse[kBeamMax];
  float score[kBeamMax];
  int state[kBeamMax];  // 1: continues, 2: finished, 0: neither
  BeamKey list[kBeamList];
  BeamKey best[kBeamMax];
  BeamKey wave[kBeamWaves];
  uint32_t high[64];
  int count, found;
};

// The k first candidates, one after the other: next(last) gives a thread's first one behind `last`.
template <typename F>
__device__ __forceinline__ void beam_rounds(BeamShared& sh, int k, F next) {
  BeamKey last = {~0ull, 0};
  int r = 0;
  for (; r < k; ++r) {
    const BeamKey mine = wave_first(next(last));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = mine;
    __syncthreads();
    BeamKey x = sh.wave[0];
    for (int i = 1; i < kBeamWaves; ++i) x = ahead_of(x, sh.wave[i]);
    if (x.id == kBeamNone.id) break;
    if (threadIdx.x == 0) sh.best[r] = x;
    last = x;
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.found = r;
  __syncthreads();
}
template <int kCtrl>
__device__ __forceinline__ int dpp_add(int x) {
  return x + __builtin_amdgcn_mov_dpp(x, kCtrl, 0xf, 0xf, false);
}
// The k first of the list's n, by their ranks: 16 threads count those ahead of one.
__device__ __forceinline__ void beam_ranks(BeamShared& sh, int k, int n) {
  for (int base = 0; base < n; base += kBeamThreads / 16) {
    const int i = base + (int)(threadIdx.x >> 4);
    const BeamKey x = sh.list[min(i, n - 1)];
    int rank = 0;
    for (int j = threadIdx.x & 15; j < n; j += 16) rank += ahead(sh.list[j], x);
    rank = dpp_add<0xB1>(rank);
    rank = dpp_add<0x4E>(rank);
    rank = dpp_add<0x141>(rank);
    rank = dpp_add<0x140>(rank);
    if (i < n && rank < k && (threadIdx.x & 15) == 0) sh.best[rank] = x;
  }
  if (threadIdx.x == 0) sh.found = min(n, k);
  __syncthreads();
}

// A group of a sample: its beam, and its place among the beam's.
struct BeamPlace {
  int w, group;
};

template <typename T>
__global__ __launch_bounds__(kBeamThreads) void beam_pick_kernel(BeamParams p) {
  using Ge = BeamGeom<T>;
  constexpr int N = Ge::kVec, E = Ge::kEach;
  __shared__ BeamShared sh;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int W = p.W, k = p.k, groups = p.tasks * kBeamGroups, chunks = (groups + 63) / 64;
  // Chunk c of the sample's: 64 groups of beam c / chunks.  A wave takes every 16th, and
  // has the first of them on their way before anything else.
  struct Chunk {
    int w, c;  // the beam, and the chunk of its own
  };
  const int more_w = kBeamWaves / chunks, more_c = kBeamWaves % chunks;
  const Chunk chunk0 = {wave / chunks, wave % chunks};
  auto next_of = [&](Chunk x) {
    x.w += more_w;
    x.c += more_c;
    if (x.c >= chunks) {
      x.c -= chunks;
      ++x.w;
    }
    return x;
  };
  auto place_of = [&](const Chunk& x) { return BeamPlace{x.w, x.c * 64 + lane}; };
  auto max_of = [&](const BeamPlace& x) {
    return x.group < groups ? p.group_max[((int64_t)b * W + x.w) * groups + x.group] : -INFINITY;
  };
  float held[kBeamHeld];
  Chunk rest = chunk0;  // the first that is not held
#pragma unroll
  for (int i = 0; i < kBeamHeld; ++i) {
    held[i] = rest.w < W ? max_of(place_of(rest)) : -INFINITY;
    rest = next_of(rest);
  }
  // the rows' sums
  for (int w = wave; w < W; w += kBeamWaves) {
    const int row = b * W + w;
    const float* pm = p.part_max + (int64_t)row * p.tasks;
    const double* ps = p.part_sum + (int64_t)row * p.tasks;
    const bool in = lane < p.tasks;
    float m = in ? pm[lane] : kBeamLowest;
    double s = in ? ps[lane] : 0.0;
    const float score = p.scores[row];
    int state = p.done && p.done[row] ? 2 : 1;
    bool bad = !(score < INFINITY);
    double lse = 0.0;
    if (state == 1) {
      for (int i = lane + 64; i < p.tasks; i += 64) {  // (a vocabulary past 131,072)
        const float y = pm[i], now = fmaxf(m, y);
        s = s * (double)__builtin_amdgcn_exp2f((m - now) * kBeamLog2e) +
            ps[i] * (double)__builtin_amdgcn_exp2f((y - now) * kBeamLog2e);
        m = now;
      }
      const float most = beam_max(m);
      s = beam_sum64(s * (double)__builtin_amdgcn_exp2f((m - most) * kBeamLog2e));
      lse = (double)most + log(s);
      bad |= !(s < (double)INFINITY);
      if (s == 0.0) state = 0;
    }
    if (bad || score == -INFINITY) state = 0;
    if (lane == 0) {
      sh.lse[w] = lse;
      sh.score[w] = score;
      sh.state[w] = state;
      if (bad) raise_device_error(p.err, WNW_DEVERR_VALUES);
    }
  }
  if (tid == 0) sh.count = 0;
  __syncthreads();
  auto total_of = [&](int w, float x) { return (double)sh.score[w] + ((double)x - sh.lse[w]); };
  auto key_of = [&](const BeamPlace& at, float x) {
    return sh.state[at.w] == 1 && x > -INFINITY
               ? BeamKey{ordered(total_of(at.w, x)), (uint32_t)(at.w * groups + at.group)}
               : kBeamNone;
  };

  // The k best groups.  First what they are not behind: the k-th largest of 16 waves'
  // maxima, or of 64 rows' of 16 lanes, by the totals' upper words, of which 20 bits are enough.
  BeamKey keys[kBeamHeld];
  uint32_t high = 0;
  Chunk x = chunk0;
#pragma unroll
  for (int i = 0; i < kBeamHeld; ++i) {
    keys[i] = kBeamNone;
    if (x.w < W) keys[i] = key_of(place_of(x), held[i]);
    high = max(high, (uint32_t)(keys[i].total >> 32));
    x = next_of(x);
  }
  for (x = rest; x.w < W; x = next_of(x)) {
    const BeamPlace at = place_of(x);
    high = max(high, (uint32_t)(key_of(at, max_of(at)).total >> 32));
  }
  high = max(high, (uint32_t)__builtin_amdgcn_mov_dpp((int)high, 0xB1, 0xf, 0xf, false));
  high = max(high, (uint32_t)__builtin_amdgcn_mov_dpp((int)high, 0x4E, 0xf, 0xf, false));
  high = max(high, (uint32_t)__builtin_amdgcn_mov_dpp((int)high, 0x141, 0xf, 0xf, false));
  high = max(high, (uint32_t)__builtin_amdgcn_mov_dpp((int)high, 0x140, 0xf, 0xf, false));
  if ((lane & 15) == 0) sh.high[tid >> 4] = high;
  __syncthreads();
  uint32_t least = 0;
  {
    uint32_t y = sh.high[lane];
    if (k <= kBeamWaves) {  // one a wave: the other rows' lanes count nothing
      y = max(y, (uint32_t)__builtin_amdgcn_mov_dpp((int)y, 0xB1, 0xf, 0xf, false));
      y = max(y, (uint32_t)__builtin_amdgcn_mov_dpp((int)y, 0x4E, 0xf, 0xf, false));
      if (lane & 3) y = 0;
    }
#pragma unroll
    for (int bit = 31; bit >= 12; --bit) {
      const uint32_t up = least | 1u << bit;
      if (__popcll(__ballot(y >= up)) >= k) least = up;
    }
  }
  auto put = [&](const BeamKey& x) {
    const int slot = atomicAdd(&sh.count, 1);
    if (slot < kBeamList) sh.list[slot] = x;
  };
  auto offer = [&](const BeamKey& x) {
    if (x.id != kBeamNone.id && (uint32_t)(x.total >> 32) >= least) put(x);
  };
#pragma unroll
  for (int i = 0; i < kBeamHeld; ++i) offer(keys[i]);
  for (x = rest; x.w < W; x = next_of(x)) {
    const BeamPlace at = place_of(x);
    offer(key_of(at, max_of(at)));
  }
  __syncthreads();
  const int near = sh.count;
  if (near <= kBeamList)
    beam_ranks(sh, k, near);
  else
    beam_rounds(sh, k, [&](const BeamKey& last) {
      BeamKey first = kBeamNone;
      for (Chunk x = chunk0; x.w < W; x = next_of(x)) {
        const BeamPlace at = place_of(x);
        const BeamKey key = key_of(at, max_of(at));
        if (ahead(last, key)) first = ahead_of(key, first);
      }
      return first;
    });

  // their elements, 16 threads a group, and the finished beams
  const int found = sh.found, mine = tid >> 4;
  const uint64_t floor_total = found == k ? sh.best[k - 1].total : 0;
  if (tid == 0) sh.count = 0;  // (behind the barrier that ended the ranks)
  BeamKey each[E], lone = kBeamNone;
#pragma unroll
  for (int i = 0; i < E; ++i) each[i] = kBeamNone;
  if (mine < found) {
    const int g = (int)sh.best[mine].id, w = g / groups, e = (g - w * groups) * kBeamGroup + (tid & 15) * N;
    const T* row = (const T*)p.logits + (int64_t)b * p.stride_b + (int64_t)w * p.stride_w;
    u32x4 raw[E / N];
    int from[E / N];
    float x[E];
#pragma unroll
    for (int u = 0; u < E / N; ++u) beam_load<T>(row, e + 16 * N * u, p.V, &raw[u], &from[u]);
#pragma unroll
    for (int u = 0; u < E / N; ++u) {
      beam_values<T>(raw[u], e + 16 * N * u, from[u], p.V, x + N * u);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint64_t t = ordered(total_of(w, x[N * u + i]));
        if (x[N * u + i] > -INFINITY && t >= floor_total)
          each[N * u + i] = BeamKey{t, (uint32_t)w * (uint32_t)p.V + (uint32_t)(from[u] + i)};
      }
    }
  }
  if (tid < W && sh.state[tid] == 2)
    lone = BeamKey{ordered((double)sh.score[tid]), (uint32_t)tid * (uint32_t)p.V + (uint32_t)p.end};
  __syncthreads();
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (each[i].id != kBeamNone.id) put(each[i]);
  if (lone.id != kBeamNone.id && lone.total >= floor_total) put(lone);
  __syncthreads();
  const int last_few = sh.count;
  if (last_few <= kBeamList)
    beam_ranks(sh, k, last_few);
  else
    beam_rounds(sh, k, [&](const BeamKey& last) {
      BeamKey first = ahead(last, lone) ? lone : kBeamNone;
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (ahead(last, each[i])) first = ahead_of(each[i], first);
      return first;
    });
  if (tid < k) {
    const bool is = tid < sh.found;
    const BeamKey x = is ? sh.best[tid] : kBeamNone;
    const int w = is ? (int)(x.id / (uint32_t)p.V) : 0;
    const int64_t at = (int64_t)b * k + tid;
    p.out_scores[at] = is ? (float)unordered(x.total) : -INFINITY;
    p.out_parents[at] = b * W + w;
    p.out_tokens[at] = is ? (int64_t)(x.id - (uint32_t)w * (uint32_t)p.V) : (int64_t)p.end;
  }
}

struct BeamLayout {
  int64_t tasks, max, groups, total;  // bytes, the sums first
};
static BeamLayout beam_layout(int64_t rows, int64_t vocab) {
  BeamLayout y;
  y.tasks = (vocab + kBeamTask - 1) / kBeamTask;
  y.max = (rows * y.tasks * 8 + 255) / 256 * 256;
  y.groups = y.max + (rows * y.tasks * 4 + 255) / 256 * 256;
  y.total = y.groups + rows * y.tasks * kBeamGroups * 4;
  return y;
}
static bool beam_sizes(int64_t batch, int64_t beams, int64_t vocab, int dtype) {
  return batch >= 0 && batch < (1 << 20) && beams >= 1 && beams <= kBeamMax && vocab >= 1 && vocab < (1 << 25) &&
         (dtype == WNW_F32 || dtype == WNW_F16 || dtype == WNW_BF16);
}

template <typename T>
static void launch_beam(const BeamParams& p, hipStream_t st) {
  const int64_t tasks = (int64_t)p.B * p.W * p.tasks;
  hipLaunchKernelGGL((beam_rows_kernel<T>), dim3((unsigned)((tasks + 3) / 4)), dim3(256), 0, st, p);
  hipLaunchKernelGGL((beam_pick_kernel<T>), dim3((unsigned)p.B), dim3(kBeamThreads), 0, st, p);
}

}  // namespace wnw

using namespace wnw;

extern "C" int64_t wnw_beam_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab, int dtype) {
  return beam_sizes(batch, beams, vocab, dtype) ? beam_layout(batch * beams, vocab).total : -1;
}

extern "C" int wnw_beam_select(const void* logits, const int64_t* strides, int64_t batch, int64_t beams, int64_t vocab,
                               const float* scores, const uint8_t* done, int64_t end, int64_t k, int dtype, float* out_scores,
                               int32_t* out_parents, int64_t* out_tokens, void* workspace, int64_t workspace_bytes, void* stream) {
  WNW_CHECK_ARG(dtype == WNW_F32 || dtype == WNW_F16 || dtype == WNW_BF16, "logits must be f32, f16 or bf16");
  WNW_CHECK_ARG(beam_sizes(batch, beams, vocab, dtype), "bad sizes: %lld samples of %lld beams (at most %d), vocabulary %lld",
                (long long)batch, (long long)beams, kBeamMax, (long long)vocab);
  WNW_CHECK_ARG(k >= 1 && k <= kBeamMax, "k must be 1 to %d", kBeamMax);
  WNW_CHECK_ARG(end >= 0 && end < vocab, "end must be a token of the vocabulary");
  if (batch == 0) return WNW_OK;
  WNW_CHECK_ARG(logits && strides && scores && out_scores && out_parents && out_tokens, "null pointer argument");
  const int64_t elem = elem_bytes(dtype);
  WNW_CHECK_ARG(strides[0] >= 0 && strides[1] >= 0 && strides[0] < (1ll << 40) && strides[1] < (1ll << 40), "bad strides");
  WNW_CHECK_ARG((uintptr_t)logits % elem == 0, "the logits are not aligned to their type");
  const BeamLayout y = beam_layout(batch * beams, vocab);
  WNW_CHECK_ARG((batch * beams * y.tasks + 3) / 4 < (1ll << 24), "too many logits for one call");
  WNW_CHECK_ARG(workspace && workspace_bytes >= y.total, "workspace too small: %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)y.total);
  WNW_CHECK_ARG((uintptr_t)workspace % 256 == 0, "the workspace must be 256-byte aligned");
  BeamParams p;
  p.logits = logits;
  p.scores = scores;
  p.done = done;
  p.part_sum = (double*)workspace;
  p.part_max = (float*)((uint8_t*)workspace + y.max);
  p.group_max = (float*)((uint8_t*)workspace + y.groups);
  p.out_scores = out_scores;
  p.out_parents = out_parents;
  p.out_tokens = out_tokens;
  p.err = device_error_word();
  p.stride_b = strides[0];
  p.stride_w = strides[1];
  p.B = (int32_t)batch;
  p.W = (int32_t)beams;
  p.V = (int32_t)vocab;
  p.k = (int32_t)k;
  p.tasks = (int32_t)y.tasks;
  p.end = (int32_t)end;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == WNW_F32)
    launch_beam<float>(p, st);
  else if (dtype == WNW_F16)
    launch_beam<f16_t>(p, st);
  else
    launch_beam<bf16_t>(p, st);
  WNW_CHECK_HIP(hipGetLastError(), "beam selection launch");
  return WNW_OK;
}
