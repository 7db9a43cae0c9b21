// Scaled table lookup and its gradient (include/istnet_vocab.h).  gfx950 only, wave64, no matrix work: both directions move bytes.
//
//   out_i = s * w_id(i)                       reads the touched rows and n indices, writes n rows
//   dw_v  = s * sum_{i: id(i) = v} g_i        reads n rows and n indices, writes ALL v rows (zeros where no index points)
//
// The gradient is a sum over the tokens of each index in the order of the tokens, so it is the same bits on every run: the tokens
// are sorted by index (stable, least significant digit first), every table row then owns a run of the sorted list and one team of
// lanes adds it up in registers -- no atomics, dw written once.  A run longer than L tokens would leave one team with a long chain
// of loads; it is cut where the sorted list is cut into pieces of L, the pieces are summed side by side and joined in order.
//
// 32768 tokens of a table of 65536 x 1024 bfloat16: lookup 25 us (67 MB written, 20 to 40 MB of rows read: 4 TB/s), gradient 85 us of
// which the sums take 45 us (67 MB read, 134 MB written: 4.5 TB/s) and the sort 40 us: six launches of 4 to 11 us that wait for memory
// and for each other, whatever the width of the rows.
#include <algorithm>

#include "vocab_common.h"

namespace {

constexpr int kSmallSort = 8192;      // tokens that one workgroup sorts in LDS
constexpr int kSmallThreads = 1024;
constexpr int kSmallDigit = 6;        // bits of a digit there: 64 digits x 16 waves = one counter per thread
constexpr int kDigit = 9;             // most bits of a digit of the sort over many workgroups
constexpr int kSortThreads = 256;
constexpr int kFewBlocks = 64;        // workgroups up to which the scatter adds up the digit counts of all of them (saves a launch)
// tokens per thread of that sort, up to 2^20 tokens (lookup and gradient of 2^18: 90 us with 4, 120 us with 16) and above (2^23: 840 and 790 us)
constexpr int kFewItems = 4, kSortItems = 16;

__device__ __forceinline__ uint32_t key_of(const void* ids, long long i, int idx64, int v, long long padding) {
  const long long id = load_index(ids, i, idx64);
  return (id < 0 || id >= v || id == padding) ? (uint32_t)v : (uint32_t)id;      // key v: nobody's gradient, sorted last
}

// lanes of the wave that are active and hold the same digit
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, bool active) {
  uint64_t m = __ballot(active);
  for (int b = 0; b < bits; ++b) {
    const bool one = (digit >> b) & 1u;
    const uint64_t has = __ballot(one);
    m &= one ? has : ~has;
  }
  return m;
}
__device__ __forceinline__ int lanes_below(uint64_t m) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
}
// position of this lane's key among the keys of its digit that the wave has seen so far; counts the wave's keys in cnt[digit]
__device__ __forceinline__ int rank_and_count(uint32_t digit, int bits, bool active, int* cnt, int lane) {
  const uint64_t m = same_digit(digit, bits, active);
  const int lead = active ? __builtin_ctzll(m) : lane;
  int base = 0;
  if (active && lane == lead) base = atomicAdd(&cnt[digit], (int)__popcll(m));
  base = __shfl(base, lead);
  return base + lanes_below(m);
}

// exclusive scan of one int per thread over the workgroup; tmp: one int per wave
template <int THREADS> __device__ __forceinline__ int block_exclusive(int x, int* tmp, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(s, o);
    if (lane >= o) s += y;
  }
  if (lane == 63) tmp[wave] = s;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    const int t = tmp[w];
    if (w < wave) before += t;
    all += t;
  }
  __syncthreads();
  *total = all;
  return before + s - x;
}

// up to kSmallSort tokens: every pass in LDS, one launch
__global__ __launch_bounds__(kSmallThreads) void embed_sort_small_kernel(int n, int v, const void* __restrict__ ids, int idx64,
                                                                         long long padding, int bits, int passes,
                                                                         uint32_t* __restrict__ keys, uint32_t* __restrict__ perm) {
  constexpr int WAVES = kSmallThreads / 64, ROUNDS = kSmallSort / kSmallThreads;
  __shared__ uint32_t skey[2][kSmallSort];
  __shared__ uint16_t sperm[2][kSmallSort];
  __shared__ int cnt[1 << kSmallDigit][WAVES];      // digit-major: the scan order is the sort order
  __shared__ int wcnt[WAVES][1 << kSmallDigit];
  __shared__ int tmp[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int rounds = (n + kSmallThreads - 1) / kSmallThreads, first = wave * rounds * 64;
  for (int r = 0; r < rounds; ++r) {
    const int i = first + r * 64 + lane;
    if (i < n) {
      skey[0][i] = key_of(ids, i, idx64, v, padding);
      sperm[0][i] = (uint16_t)i;
    }
  }
  const int radix = 1 << bits;
  for (int p = 0; p < passes; ++p) {
    const int from = p & 1, shift = p * bits;
    for (int d = lane; d < radix; d += 64) wcnt[wave][d] = 0;
    __syncthreads();
    int rank[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      if (r < rounds) {
        const int i = first + r * 64 + lane;
        const bool active = i < n;
        const uint32_t digit = active ? (skey[from][i] >> shift) & (uint32_t)(radix - 1) : 0u;
        rank[r] = rank_and_count(digit, bits, active, wcnt[wave], lane);
      }
    }
    for (int d = lane; d < radix; d += 64) cnt[d][wave] = wcnt[wave][d];
    __syncthreads();
    int all;
    int* flat = &cnt[0][0];
    const int mine = tid < radix * WAVES ? flat[tid] : 0;
    const int before = block_exclusive<kSmallThreads>(mine, tmp, &all);
    if (tid < radix * WAVES) flat[tid] = before;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const int i = first + r * 64 + lane;
      if (r < rounds && i < n) {
        const uint32_t k = skey[from][i];
        const int pos = cnt[(k >> shift) & (uint32_t)(radix - 1)][wave] + rank[r];
        skey[from ^ 1][pos] = k;
        sperm[from ^ 1][pos] = sperm[from][i];
      }
    }
    __syncthreads();
  }
  for (int i = tid; i < n; i += kSmallThreads) {
    keys[i] = skey[passes & 1][i];
    perm[i] = sperm[passes & 1][i];
  }
}

// One pass of the sort over many workgroups: digit counts per workgroup, scan of the counts digit by digit, stable scatter.
// Wave w of workgroup b owns tokens [b * tile + w * 64 * items, ...): the order of (workgroup, wave, round, lane) is token order.
__global__ __launch_bounds__(kSortThreads) void embed_hist_kernel(int n, int v, const void* __restrict__ ids, int idx64,
                                                                  long long padding, const uint32_t* __restrict__ keys_in, int shift,
                                                                  int bits, int items, int nb, int* __restrict__ hist) {
  __shared__ int cnt[1 << kDigit];
  const int radix = 1 << bits, b = blockIdx.x;
  for (int d = threadIdx.x; d < radix; d += kSortThreads) cnt[d] = 0;
  __syncthreads();
  const long long base = (long long)b * kSortThreads * items;
#pragma unroll 4
  for (int r = 0; r < items; ++r) {
    const long long i = base + r * kSortThreads + threadIdx.x;
    if (i < n) {
      const uint32_t k = keys_in ? keys_in[i] : key_of(ids, i, idx64, v, padding);
      atomicAdd(&cnt[(k >> shift) & (uint32_t)(radix - 1)], 1);
    }
  }
  __syncthreads();
  // few workgroups: counts of one workgroup side by side, added up by the scatter itself; many: digit by digit, for the scan
  for (int d = threadIdx.x; d < radix; d += kSortThreads) hist[nb <= kFewBlocks ? (long long)b * radix + d : (long long)d * nb + b] = cnt[d];
}

// many workgroups: workgroup d scans its digit's counts over the workgroups of the sort; the digits' totals follow behind all counts
// (64 M tokens: one workgroup over all counts was the longest kernel of the sort)
__global__ __launch_bounds__(256) void embed_scan_kernel(int nb, int* __restrict__ hist) {
  __shared__ int tmp[4];
  int* mine = hist + (long long)blockIdx.x * nb;
  int carry = 0;
  for (int base = 0; base < nb; base += 1024) {
    const int i = base + 4 * threadIdx.x;
    int x[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = i + j < nb ? mine[i + j] : 0;
      sum += x[j];
    }
    int all;
    int at = carry + block_exclusive<256>(sum, tmp, &all);
    carry += all;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (i + j < nb) mine[i + j] = at;
      at += x[j];
    }
  }
  if (threadIdx.x == 0) hist[(long long)gridDim.x * nb + blockIdx.x] = carry;
}

template <int ITEMS>
__global__ __launch_bounds__(kSortThreads) void embed_scatter_kernel(int n, int v, const void* __restrict__ ids, int idx64,
                                                                     long long padding, const uint32_t* __restrict__ keys_in,
                                                                     const uint32_t* __restrict__ perm_in, int shift, int bits, int nb,
                                                                     const int* __restrict__ hist, uint32_t* __restrict__ keys_out,
                                                                     uint32_t* __restrict__ perm_out) {
  constexpr int WAVES = kSortThreads / 64;
  __shared__ int cnt[WAVES][1 << kDigit];
  __shared__ int tmp[WAVES];
  const int radix = 1 << bits, b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int d = lane; d < radix; d += 64) cnt[wave][d] = 0;
  __syncthreads();
  const long long first = ((long long)b * WAVES + wave) * 64 * ITEMS;
  int rank[ITEMS];
  uint32_t key[ITEMS], from_token[ITEMS];
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {      // all loads on their way before the first is counted
    const long long i = first + r * 64 + lane;
    const bool active = i < n;
    key[r] = active ? (keys_in ? keys_in[i] : key_of(ids, i, idx64, v, padding)) : 0u;
    from_token[r] = active && perm_in ? perm_in[i] : (uint32_t)i;
  }
#pragma unroll
  for (int r = 0; r < ITEMS; ++r)
    rank[r] = rank_and_count((key[r] >> shift) & (uint32_t)(radix - 1), bits, first + r * 64 + lane < n, cnt[wave], lane);
  __syncthreads();
  constexpr int PER = (1 << kDigit) / kSortThreads;      // digits of a thread: PER consecutive ones
  static_assert(PER == 2, "the counts of a thread's digits are one load");
  int at[PER], before[PER] = {}, total[PER] = {};
  const int d0 = threadIdx.x * PER;
  if (d0 < radix) {      // radix is even
    if (nb <= kFewBlocks) {
#pragma unroll 16
      for (int o = 0; o < nb; ++o) {
        const int2 c = *reinterpret_cast<const int2*>(hist + (long long)o * radix + d0);
        total[0] += c.x;
        total[1] += c.y;
        before[0] += o < b ? c.x : 0;
        before[1] += o < b ? c.y : 0;
      }
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        total[j] = hist[(long long)radix * nb + d0 + j];
        before[j] = hist[(long long)(d0 + j) * nb + b];
      }
    }
  }
  int mine = 0, all;
#pragma unroll
  for (int j = 0; j < PER; ++j) mine += total[j];
  int from = block_exclusive<kSortThreads>(mine, tmp, &all);
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    at[j] = from + before[j];
    from += total[j];
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int d = threadIdx.x * PER + j;
    if (d < radix) {
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const int c = cnt[w][d];
        cnt[w][d] = at[j];
        at[j] += c;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const long long i = first + r * 64 + lane;
    if (i < n) {
      const int pos = cnt[wave][(key[r] >> shift) & (uint32_t)(radix - 1)] + rank[r];
      keys_out[pos] = key[r];
      perm_out[pos] = from_token[r];
    }
  }
}

// start[t] = number of sorted keys below t, t = 0 .. v
__global__ __launch_bounds__(256) void embed_starts_kernel(int n, int v, const uint32_t* __restrict__ keys, int* __restrict__ start) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t > v) return;
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = lo + ((hi - lo) >> 1);
    if (keys[mid] < (uint32_t)t) lo = mid + 1; else hi = mid;
  }
  start[t] = lo;
}

// sum of the gradient rows of sorted tokens [a, e), elements [col, col + left), added in order: four loads in flight, two where the run ends
// (most runs are short; eight and one: 120 us for lookup and gradient of 32768 tokens of 65536 x 1024 bfloat16, this 110 us)
template <typename T>
__device__ __forceinline__ void sum_run(const T* __restrict__ grad, long long ldg, const uint32_t* __restrict__ perm, int a, int e,
                                        int col, int left, float (&acc)[kVec<T>]) {
  constexpr int U = 4;
  int p = a;
  if (left >= kVec<T>) {
    for (; p + U <= e; p += U) {
      u32x4 raw[U];
#pragma unroll
      for (int j = 0; j < U; ++j) raw[j] = load16(grad + (long long)perm[p + j] * ldg + col);
#pragma unroll
      for (int j = 0; j < U; ++j) {
        float f[kVec<T>];
        unpack<T>(raw[j], f);
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) acc[i] += f[i];
      }
    }
  }
  if (left >= kVec<T>) {
    for (; p < e; p += 2) {
      u32x4 raw[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) raw[j] = load16(grad + (long long)perm[min(p + j, e - 1)] * ldg + col);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float f[kVec<T>];
        unpack<T>(raw[j], f);
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) acc[i] = p + j < e ? acc[i] + f[i] : acc[i];
      }
    }
    return;
  }
  for (; p < e; ++p) {
    float f[kVec<T>];
    load_part(grad + (long long)perm[p] * ldg + col, left, f);
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) acc[i] += f[i];
  }
}

constexpr int kTeamRows = 4;      // table rows per team of lanes

// The rows of a team are far apart: frequent indices are often neighbours, and one team would have to add up several of them.
template <typename T>
__device__ __forceinline__ void sum_rows(long long wg, long long wgs, int v, int d, int lanes_log, int longest,
                                         const T* __restrict__ grad, long long ldg, const uint32_t* __restrict__ perm,
                                         const int* __restrict__ start, float scale, T* __restrict__ dw) {
  const int lanes = 1 << lanes_log, at = threadIdx.x & (lanes - 1);
  const long long teams = wgs << (8 - lanes_log);
  for (long long row0 = (wg << (8 - lanes_log)) + (threadIdx.x >> lanes_log); row0 < v; row0 += teams * kTeamRows) {
    int s[kTeamRows], e[kTeamRows];
#pragma unroll
    for (int r = 0; r < kTeamRows; ++r) {
      const long long row = row0 + r * teams;
      s[r] = start[row < v ? row : v];
      e[r] = start[row < v ? row + 1 : v];
    }
    for (int col = at * kVec<T>; col < d; col += lanes * kVec<T>) {
#pragma unroll
      for (int r = 0; r < kTeamRows; ++r) {
        const long long row = row0 + r * teams;
        if (row < v && e[r] - s[r] <= longest) {
          float acc[kVec<T>] = {};
          sum_run(grad, ldg, perm, s[r], e[r], col, d - col, acc);
#pragma unroll
          for (int i = 0; i < kVec<T>; ++i) acc[i] *= scale;
          store_part(dw + row * d + col, d - col, acc);
        }
      }
    }
  }
}

// the teams of a workgroup hold partial sums of the same columns: team 0 gets them added in team order
template <typename T>
__device__ __forceinline__ void join_teams(float (&acc)[kVec<T>], float* lds, int lanes_log, int teams) {
  const int at = threadIdx.x & ((1 << lanes_log) - 1), team = threadIdx.x >> lanes_log;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) lds[(i << 8) + threadIdx.x] = acc[i];
  __syncthreads();
  if (team == 0) {
    for (int t = 1; t < teams; ++t)
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) acc[i] += lds[(i << 8) + (t << lanes_log) + at];
  }
  __syncthreads();
}

// Piece p holds sorted tokens [p L, (p + 1) L).  At most two runs longer than L touch it: the one of its first token (slot 0) and
// the one of its last (slot 1, if that is another one).
template <typename T>
__device__ __forceinline__ void sum_piece(float* lds, int n, int v, int d, int lanes_log, int longest, const T* __restrict__ grad,
                                          long long ldg, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ perm,
                                          const int* __restrict__ start, float* __restrict__ part) {
  const int lanes = 1 << lanes_log, teams = 256 >> lanes_log, at = threadIdx.x & (lanes - 1), team = threadIdx.x >> lanes_log;
  const int p0 = blockIdx.x * longest, p1 = min(n, p0 + longest);
  const uint32_t ka = keys[p0], kb = keys[p1 - 1];
  for (int slot = 0; slot < 2; ++slot) {
    const uint32_t k = slot ? kb : ka;
    if (k >= (uint32_t)v || (slot && kb == ka)) continue;
    const int s = start[k], e = start[k + 1];
    if (e - s <= longest) continue;
    const int a0 = max(s, p0), a1 = min(e, p1), per = (a1 - a0 + teams - 1) / teams;
    const int a = min(a1, a0 + team * per), b = min(a1, a + per);
    for (int c0 = 0; c0 < d; c0 += lanes * kVec<T>) {
      const int col = c0 + at * kVec<T>;
      float acc[kVec<T>] = {};
      if (col < d) sum_run(grad, ldg, perm, a, b, col, d - col, acc);
      join_teams<T>(acc, lds, lanes_log, teams);
      if (team == 0 && col < d) {
        float* o = part + ((long long)blockIdx.x * 2 + slot) * ((d + 7) / 8 * 8) + col;
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) o[i] = acc[i];
      }
    }
  }
}

// Short runs and the pieces of long ones do not meet: one launch, the pieces first because one takes longer.  (32768 tokens of a table of
// 65536 x 1024 bfloat16: 45 us for both, with 15 us more for the pieces in a launch of their own.)
template <typename T>
__global__ __launch_bounds__(256) void embed_sums_kernel(int n, int v, int d, int lanes_log, int longest, int pieces,
                                                         const T* __restrict__ grad, long long ldg, const uint32_t* __restrict__ keys,
                                                         const uint32_t* __restrict__ perm, const int* __restrict__ start, float scale,
                                                         float* __restrict__ part, T* __restrict__ dw) {
  __shared__ float lds[256 * kVec<T>];
  if ((int)blockIdx.x < pieces)
    sum_piece(lds, n, v, d, lanes_log, longest, grad, ldg, keys, perm, start, part);
  else
    sum_rows<T>(blockIdx.x - pieces, gridDim.x - pieces, v, d, lanes_log, longest, grad, ldg, perm, start, scale, dw);
}

// the run longer than L that STARTS in piece p (there is at most one, that of the piece's last token): its partial sums in order
template <typename T>
__global__ __launch_bounds__(256) void embed_join_kernel(int n, int v, int d, int lanes_log, int longest,
                                                         const uint32_t* __restrict__ keys, const int* __restrict__ start,
                                                         const float* __restrict__ part, float scale, T* __restrict__ dw) {
  __shared__ float lds[256 * kVec<T>];
  const int lanes = 1 << lanes_log, teams = 256 >> lanes_log, at = threadIdx.x & (lanes - 1), team = threadIdx.x >> lanes_log;
  const int p0 = blockIdx.x * longest, p1 = min(n, p0 + longest);
  const uint32_t k = keys[p1 - 1];
  if (k >= (uint32_t)v) return;
  const int s = start[k], e = start[k + 1];
  if (e - s <= longest || s < p0) return;
  const int q0 = blockIdx.x, q1 = (e - 1) / longest + 1, per = (q1 - q0 + teams - 1) / teams;
  const int a = min(q1, q0 + team * per), b = min(q1, a + per);
  for (int c0 = 0; c0 < d; c0 += lanes * kVec<T>) {
    const int col = c0 + at * kVec<T>;
    float acc[kVec<T>] = {};
    if (col < d) {
#pragma unroll 8
      for (int q = a; q < b; ++q) {
        const float* o = part + ((long long)q * 2 + (s > q * longest ? 1 : 0)) * ((d + 7) / 8 * 8) + col;
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) acc[i] += o[i];
      }
    }
    join_teams<T>(acc, lds, lanes_log, teams);
    if (team == 0 && col < d) {
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) acc[i] *= scale;
      store_part(dw + (long long)k * d + col, d - col, acc);
    }
  }
}

// Few tokens: one launch.  A workgroup owns `rows` (<= 64) consecutive table rows, picks their tokens out of all n in order, sorts them
// by row in LDS and adds them up; a run longer than kShortRun is shared by its teams.  (77 x 99 into 1000 rows: 5 launches of 2 to 5 us
// each became one of 6 us, and what they cost the host is gone: 20 us.  2048 tokens into 1000 rows: lookup and gradient 38 us in a graph,
// 29 us with the sort, 4096: 56 and 34 us; launched one by one both wait for the host up to some 60 us.)
constexpr int kFewTokens = 2048, kFewRows = 64, kShortRun = 32;
template <typename T>
__global__ __launch_bounds__(256) void embed_few_kernel(int n, int v, int d, int rows, int lanes_log, const T* __restrict__ grad,
                                                        long long ldg, const void* __restrict__ ids, int idx64, long long padding,
                                                        float scale, T* __restrict__ dw) {
  __shared__ float lds[256 * kVec<T>];
  __shared__ uint32_t list[kFewTokens], sorted[kFewTokens];
  __shared__ int start[kFewRows + 1], cnt[kFewRows], waves[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long row0 = (long long)blockIdx.x * rows;
  int m = 0;
  for (int base = 0; base < n; base += 256) {
    const int i = base + tid;
    const uint32_t key = i < n ? key_of(ids, i, idx64, v, padding) : (uint32_t)v;
    const bool mine = key < (uint32_t)v && key >= (uint32_t)row0 && key < (uint32_t)(row0 + rows);
    const uint64_t has = __ballot(mine);
    if (lane == 0) waves[wave] = __popcll(has);
    __syncthreads();
    int at = m + lanes_below(has);
    for (int w = 0; w < 4; ++w) {
      at += w < wave ? waves[w] : 0;
      m += waves[w];
    }
    if (mine) list[at] = (uint32_t)(key - (uint32_t)row0) << 16 | (uint32_t)i;
    __syncthreads();
  }
  if (tid < kFewRows) cnt[tid] = 0;
  __syncthreads();
  for (int j = tid; j < m; j += 256) atomicAdd(&cnt[list[j] >> 16], 1);
  __syncthreads();
  if (wave == 0) {
    int s = cnt[lane];
    const int own = s;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(s, o);
      if (lane >= o) s += y;
    }
    start[lane] = s - own;
    if (lane == 63) start[64] = s;
    cnt[lane] = s - own;      // from here on: where the row's next token goes
    for (int j = 0; j < m; j += 64) {
      const bool active = j + lane < m;
      const uint32_t e = active ? list[j + lane] : 0u;
      const int to = rank_and_count(e >> 16, 6, active, cnt, lane);
      if (active) sorted[to] = e & 0xffffu;
    }
  }
  __syncthreads();
  const int lanes = 1 << lanes_log, teams = 256 >> lanes_log, at = tid & (lanes - 1), team = tid >> lanes_log;
  const int last = (int)(v - row0 < rows ? v - row0 : rows);
  for (int c0 = 0; c0 < d; c0 += lanes * kVec<T>) {
    const int col = c0 + at * kVec<T>;
    for (int r = 0; r < last; ++r) {      // long runs: every team a part
      const int a0 = start[r], a1 = start[r + 1];
      if (a1 - a0 <= kShortRun) continue;
      const int per = (a1 - a0 + teams - 1) / teams, a = min(a1, a0 + team * per), b = min(a1, a + per);
      float acc[kVec<T>] = {};
      if (col < d) sum_run(grad, ldg, sorted, a, b, col, d - col, acc);
      join_teams<T>(acc, lds, lanes_log, teams);
      if (team == 0 && col < d) {
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) acc[i] *= scale;
        store_part(dw + (row0 + r) * d + col, d - col, acc);
      }
    }
    for (int r = team; r < last && col < d; r += teams) {
      const int a0 = start[r], a1 = start[r + 1];
      if (a1 - a0 > kShortRun) continue;
      float acc[kVec<T>] = {};
      sum_run(grad, ldg, sorted, a0, a1, col, d - col, acc);
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) acc[i] *= scale;
      store_part(dw + (row0 + r) * d + col, d - col, acc);
    }
  }
}

constexpr int kLookupRows = 4;      // rows per team of lanes: their loads are in flight together

template <typename T>
__global__ __launch_bounds__(256) void embed_lookup_kernel(long long n, int v, int d, int lanes_log, int idx64,
                                                           const T* __restrict__ weight, long long ldw, const void* __restrict__ ids,
                                                           float scale, T* __restrict__ out) {
  const int lanes = 1 << lanes_log, at = threadIdx.x & (lanes - 1);
  const long long step = (long long)gridDim.x * kLookupRows << (8 - lanes_log);
  for (long long row0 = (((long long)blockIdx.x << (8 - lanes_log)) + (threadIdx.x >> lanes_log)) * kLookupRows; row0 < n; row0 += step) {
    long long id[kLookupRows];
#pragma unroll
    for (int r = 0; r < kLookupRows; ++r) {
      const long long i = row0 + r < n ? load_index(ids, row0 + r, idx64) : -1;
      id[r] = (i < 0 || i >= v) ? -1 : i;
    }
    for (int col = at * kVec<T>; col < d; col += lanes * kVec<T>) {
      float f[kLookupRows][kVec<T>];
#pragma unroll
      for (int r = 0; r < kLookupRows; ++r) {
        if (id[r] >= 0) {
          load_part(weight + id[r] * ldw + col, d - col, f[r]);
#pragma unroll
          for (int i = 0; i < kVec<T>; ++i) f[r][i] *= scale;
        } else {
#pragma unroll
          for (int i = 0; i < kVec<T>; ++i) f[r][i] = __uint_as_float(0x7fc00000u);
        }
      }
#pragma unroll
      for (int r = 0; r < kLookupRows; ++r)
        if (row0 + r < n) store_part(out + (row0 + r) * d + col, d - col, f[r]);
    }
  }
}

constexpr long long kMaxGrid = 1 << 22;      // a launch holds fewer than 2^32 threads; the kernels over rows stride beyond it

inline int log2_ceil(long long x) {
  int l = 0;
  while ((1ll << l) < x) ++l;
  return l;
}
// lanes that share a row: enough for sixteen bytes each, a workgroup at most
inline int lanes_log_of(int d, int dtype) {
  const int vec = dtype == ISTNET_VOCAB_F32 ? 4 : 8, l = log2_ceil((d + vec - 1) / vec);
  return l > 8 ? 8 : l;
}
inline bool embed_ok(long long n, int v, int d, int dtype) {
  return n >= 1 && n <= (1ll << 30) && v >= 1 && v < 0x7fffffff - 256 && d >= 1 && dtype >= 0 && dtype <= 2;
}

// a table of more rows takes more workgroups of embed_few_kernel than one launch may hold
inline bool embed_few(long long n, int v) { return n <= kFewTokens && v <= (1 << 28); }

struct EmbedPlan {
  int bits, passes, items, nb, longest, pieces;
  long long keys[2], perm[2], hist, start, part, bytes;      // offsets into the scratch memory
};
inline EmbedPlan embed_plan(long long n, int v, int d) {
  EmbedPlan p = {};
  const int key_bits = log2_ceil((long long)v + 1), most = n <= kSmallSort ? kSmallDigit : kDigit;
  p.passes = (key_bits + most - 1) / most;
  p.bits = (key_bits + p.passes - 1) / p.passes;
  p.items = n <= 1024 * 1024 ? kFewItems : kSortItems;
  p.nb = (int)((n + kSortThreads * p.items - 1) / (kSortThreads * p.items));
  // pieces short enough that one is a few rounds of loads, long enough that the partial sums of one row do not become many
  p.longest = std::max(32, (1 << ((log2_ceil(n) + 1) / 2)) / 8);
  p.pieces = n > p.longest ? (int)((n + p.longest - 1) / p.longest) : 0;
  long long at = 0;
  auto take = [&](long long bytes) { const long long o = at; at += (bytes + 255) / 256 * 256; return o; };
  const bool small = n <= kSmallSort;
  for (int i = 0; i < (small ? 1 : 2); ++i) { p.keys[i] = take(4 * n); p.perm[i] = take(4 * n); }
  p.hist = small ? 0 : take(4ll * (p.nb + 1) << p.bits);
  p.start = take(4ll * (v + 1ll));
  p.part = p.pieces ? take(8ll * p.pieces * ((d + 7) / 8 * 8)) : 0;
  p.bytes = at;
  return p;
}

}  // namespace

extern "C" int istnet_embed_forward(long long n, int v, int d, int dtype, int idx64, const void* weight, long long ldw,
                                    const void* ids, float scale, void* out, void* stream) {
  if (!embed_ok(n, v, d, dtype) || !weight || !ids || !out || ldw < d) return ISTNET_PN2_EINVAL;
  const int ll = lanes_log_of(d, dtype);
  const long long rows = (256 >> ll) * (long long)kLookupRows, grid = std::min((n + rows - 1) / rows, kMaxGrid);
  VOCAB_DISPATCH(dtype, T, hipLaunchKernelGGL(HIP_KERNEL_NAME(embed_lookup_kernel<T>), dim3((unsigned)grid), dim3(256), 0,
                                              (hipStream_t)stream, n, v, d, ll, idx64, (const T*)weight, ldw, ids, scale, (T*)out));
  return launch_status();
}

extern "C" int istnet_embed_scratch_kib(long long n, int v, int d) {
  if (!embed_ok(n, v, d, 0)) return -1;
  if (embed_few(n, v)) return 0;
  return (int)((embed_plan(n, v, d).bytes + 1023) / 1024);
}

extern "C" int istnet_embed_backward(long long n, int v, int d, int dtype, int idx64, const void* grad, long long ldg,
                                     const void* ids, long long padding, float scale, void* ws, void* dw, void* stream) {
  if (!embed_ok(n, v, d, dtype) || !grad || !ids || (!ws && !embed_few(n, v)) || !dw || ldg < d) return ISTNET_PN2_EINVAL;
  const hipStream_t st = (hipStream_t)stream;
  const int ll = lanes_log_of(d, dtype);
  if (embed_few(n, v)) {
    // rows per workgroup: enough workgroups for the chip, few enough that reading all indices in each of them stays cheap (1000 tokens,
    // table of 65536 x 256: 30 us with 16, 43 us with 64; 2000 tokens, 2^20 x 16: 230 and 108 us)
    const int rows = v <= 65536 ? 16 : kFewRows;
    VOCAB_DISPATCH(dtype, T, hipLaunchKernelGGL(HIP_KERNEL_NAME(embed_few_kernel<T>), dim3((unsigned)((v + rows - 1ll) / rows)), dim3(256),
                                                0, st, (int)n, v, d, rows, ll, (const T*)grad, ldg, ids, idx64, padding, scale, (T*)dw));
    return launch_status();
  }
  const EmbedPlan p = embed_plan(n, v, d);
  char* base = (char*)ws;
  uint32_t *keys[2], *perm[2];
  for (int i = 0; i < 2; ++i) { keys[i] = (uint32_t*)(base + p.keys[i]); perm[i] = (uint32_t*)(base + p.perm[i]); }
  int* start = (int*)(base + p.start);
  float* part = (float*)(base + p.part);
  int last = 0;
  if (n <= kSmallSort) {
    hipLaunchKernelGGL(embed_sort_small_kernel, dim3(1), dim3(kSmallThreads), 0, st, (int)n, v, ids, idx64, padding, p.bits,
                       p.passes, keys[0], perm[0]);
  } else {
    int* hist = (int*)(base + p.hist);
    for (int i = 0; i < p.passes; ++i) {
      const uint32_t* kin = i ? keys[last] : nullptr;
      const uint32_t* pin = i ? perm[last] : nullptr;
      const int to = i ? last ^ 1 : 0;
      hipLaunchKernelGGL(embed_hist_kernel, dim3(p.nb), dim3(kSortThreads), 0, st, (int)n, v, ids, idx64, padding, kin, i * p.bits,
                         p.bits, p.items, p.nb, hist);
      if (p.nb > kFewBlocks)
        hipLaunchKernelGGL(embed_scan_kernel, dim3(1u << p.bits), dim3(256), 0, st, p.nb, hist);
      const auto scatter = p.items == kFewItems ? embed_scatter_kernel<kFewItems> : embed_scatter_kernel<kSortItems>;
      hipLaunchKernelGGL(scatter, dim3(p.nb), dim3(kSortThreads), 0, st, (int)n, v, ids, idx64, padding, kin, pin, i * p.bits, p.bits,
                         p.nb, hist, keys[to], perm[to]);
      last = to;
    }
  }
  hipLaunchKernelGGL(embed_starts_kernel, dim3((unsigned)(v / 256 + 1)), dim3(256), 0, st, (int)n, v, keys[last], start);
  const long long rows = (256 >> ll) * (long long)kTeamRows, grid = std::min((v + rows - 1) / rows, kMaxGrid);
  VOCAB_DISPATCH(dtype, T, {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(embed_sums_kernel<T>), dim3((unsigned)(p.pieces + grid)), dim3(256), 0, st, (int)n, v, d, ll,
                       p.longest, p.pieces, (const T*)grad, ldg, keys[last], perm[last], start, scale, part, (T*)dw);
    if (p.pieces)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(embed_join_kernel<T>), dim3(p.pieces), dim3(256), 0, st, (int)n, v, d, ll, p.longest,
                         keys[last], start, part, scale, (T*)dw);
  });
  return launch_status();
}
