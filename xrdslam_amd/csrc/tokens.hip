// Tokens: a stable sort of ids by counting digits (xrd_token_plan) and the
// scaled lookup of table rows with its gradients (xrd_lookup_*).
//
//   plan    order = stable argsort(ids), starts[g] = first position of group g
//   lookup  y_i = s sum_k w_ik E[id_ik]
//   grads   dE_v = s sum_{tokens t of v, in order} w_t dy_{t/K}
//           dw_ik = s <E[id_ik], dy_i>
//
// An id outside [0, rows) is "no row": it adds nothing and gets no gradient.
// Sums are f32 in a fixed order (no atomics): equal inputs give equal bits.
#include "element.h"

namespace xrd {
namespace {

// ------------------------------------------------------------------- plan
// Digits of up to 9 bits, lowest first; the groups' bits are dealt evenly over
// the passes (100000 groups: 9 + 8 bits, two passes).
constexpr int kMaxBits = 9;
constexpr int kMaxBins = 1 << kMaxBits;
constexpr int kSmall = 8192;       // tokens that one block sorts in its LDS
constexpr int kSmallThreads = 1024;
constexpr int kSmallWaves = kSmallThreads / 64;

// ids -> keys: an id outside the groups sorts behind them
template <typename I>
__device__ __forceinline__ uint32_t key_of(I id, int64_t n_groups) {
  return (id >= 0 && (int64_t)id < n_groups) ? (uint32_t)id
                                             : (uint32_t)n_groups;
}

// keys of pass 0 come from the ids themselves, later ones from the buffer
template <typename I>
__device__ __forceinline__ uint32_t load_key(const I* __restrict__ ids,
                                             const uint32_t* __restrict__ keys,
                                             int64_t n_groups, int64_t i) {
  return ids != nullptr ? key_of(ids[i], n_groups) : keys[i];
}

// exclusive prefix of v over the block, total -> sum.  wsum: one word a wave.
template <int WAVES>
__device__ __forceinline__ int block_scan(int v, int* wsum, int& sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 63) wsum[wave] = inc;
  __syncthreads();
  int woff = 0;
  sum = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) woff += wsum[w];
    sum += wsum[w];
  }
  __syncthreads();
  return woff + inc - v;
}

// rank[j] of this lane's key j among the wave's keys of its digit, those of the
// items before j first, then the lanes below: equal keys keep their order.  cnt:
// the wave's counts so far, left increased.  A lane's peers are found bit by bit,
// all items side by side; the first lane of a digit adds the peers' number to
// cnt and hands what was there to them.  (A wave's LDS operations are carried
// out in order, so the items' additions need no wait between them: 8 million
// keys of 100000 groups take 253 us, 268 with a read, a wait and a write each.)
template <int ITEMS>
__device__ __forceinline__ void wave_ranks(int* cnt,
                                           const uint32_t (&digit)[ITEMS],
                                           const bool (&live)[ITEMS], int bits,
                                           int (&rank)[ITEMS]) {
  uint32_t lo[ITEMS] = {}, hi[ITEMS] = {};      // lanes of another digit
  for (int b = 0; b < bits; ++b)
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const uint32_t mine = 0u - (digit[j] >> b & 1u);
      const uint64_t v = __builtin_amdgcn_ballot_w64(mine != 0);
      lo[j] |= (uint32_t)v ^ mine;
      hi[j] |= (uint32_t)(v >> 32) ^ mine;
    }
  const int lane = threadIdx.x & 63;
  int before[ITEMS], first[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const uint64_t peers = ~((uint64_t)hi[j] << 32 | lo[j]) &
                           __builtin_amdgcn_ballot_w64(live[j]);
    first[j] = __ffsll((unsigned long long)peers) - 1;
    rank[j] = __popcll(peers & ((1ull << lane) - 1ull));
    before[j] = 0;
    if (live[j] && first[j] == lane)
      before[j] = atomicAdd(&cnt[digit[j]], __popcll(peers));
    __builtin_amdgcn_wave_barrier();
  }
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) rank[j] += __shfl(before[j], first[j] & 63);
  wave_lds_sync();
}

// starts[g] = number of keys below g, by halving
__device__ __forceinline__ int64_t keys_below(const uint32_t* keys, int64_t n,
                                              int64_t g) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if ((int64_t)keys[mid] < g) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// All passes of a short list in one block: keys and token numbers live in LDS,
// a thread holds ITEMS keys in registers (a wave ITEMS * 64 consecutive ones).
// With few groups it also writes the starts, else the sorted keys.  2000 tokens
// in 16 groups take 5 us as this one launch and 15.5 us as four.
template <typename I, int ITEMS>
__global__ __launch_bounds__(kSmallThreads) void plan_small_kernel(
    int n, int64_t n_groups, const I* __restrict__ ids, int bits, int passes,
    int* __restrict__ order, int* __restrict__ starts, int* __restrict__ rank,
    uint32_t* __restrict__ keys_out) {
  __shared__ uint32_t keys[ITEMS * kSmallThreads];
  __shared__ int tok[ITEMS * kSmallThreads];
  __shared__ int cnt[kSmallWaves][kMaxBins];
  __shared__ int wsum[kSmallWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int base = wave * ITEMS * 64 + lane;
  uint32_t key[ITEMS];
  int t[ITEMS], r[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const int i = base + j * 64;
    t[j] = i;
    key[j] = i < n ? key_of(ids[i], n_groups) : 0u;
  }
  const int bins = 1 << bits;
  for (int p = 0; p < passes; ++p) {
    for (int d = threadIdx.x; d < kSmallWaves * kMaxBins; d += kSmallThreads)
      (&cnt[0][0])[d] = 0;
    __syncthreads();
    uint32_t digit[ITEMS];
    bool live[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      digit[j] = (key[j] >> (p * bits)) & (bins - 1);
      live[j] = base + j * 64 < n;
    }
    wave_ranks<ITEMS>(cnt[wave], digit, live, bits, r);
    __syncthreads();
    int mine = 0, sum;
    if (threadIdx.x < bins)
      for (int w = 0; w < kSmallWaves; ++w) mine += cnt[w][threadIdx.x];
    int run = block_scan<kSmallWaves>(mine, wsum, sum);
    if (threadIdx.x < bins)
      for (int w = 0; w < kSmallWaves; ++w) {
        const int c = cnt[w][threadIdx.x];
        cnt[w][threadIdx.x] = run;
        run += c;
      }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (base + j * 64 < n) {
        const int pos = cnt[wave][digit[j]] + r[j];
        keys[pos] = key[j];
        tok[pos] = t[j];
      }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (base + j * 64 < n) {
        key[j] = keys[base + j * 64];
        t[j] = tok[base + j * 64];
      }
  }
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const int i = base + j * 64;
    if (i < n) {
      order[i] = t[j];
      if (rank != nullptr) rank[t[j]] = i;
    }
  }
  if (keys_out != nullptr) {
    for (int i = threadIdx.x; i < n; i += kSmallThreads) keys_out[i] = keys[i];
    return;
  }
  for (int64_t g = threadIdx.x; g <= n_groups; g += kSmallThreads)
    starts[g] = (int)keys_below(keys, n, g);
}

// Longer lists: tiles of keys, a block each, two launches a digit - count and
// scatter - up to 256 tiles, whose counts every scattering block adds up itself;
// beyond that a launch in between scans them.  A block's work is a chain of
// latencies, so tiles are 2048 keys while that makes at most 256 of them (393216
// tokens of 20000 groups: 34.8 us; 39.0 with 4096; 40.8 with 1024) and 4096
// beyond (600000 of 100000: 47.5, 51.4 with 2048).
constexpr int kShortTile = 2048, kLongTile = 4096;
constexpr int kSelfTiles = 256, kSelfThreads = 1024;

// counts[block][d] of a block's keys with digit d
template <typename I, int THREADS, int TILE>
__global__ __launch_bounds__(THREADS) void plan_count_kernel(
    int64_t n, int64_t n_groups, const I* __restrict__ ids,
    const uint32_t* __restrict__ keys, int shift, int bits,
    int* __restrict__ counts) {
  __shared__ int bins[kMaxBins];
  const int n_bins = 1 << bits;
  for (int d = threadIdx.x; d < n_bins; d += THREADS) bins[d] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * TILE;
#pragma unroll
  for (int j = 0; j < TILE / THREADS; ++j) {
    const int64_t i = base + j * THREADS + threadIdx.x;
    if (i < n)
      atomicAdd(
          &bins[(load_key(ids, keys, n_groups, i) >> shift) & (n_bins - 1)], 1);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < n_bins; d += THREADS)
    counts[((int64_t)blockIdx.x << bits) + d] = bins[d];
}

// a block a digit: exclusive scan of its counts over the blocks, their total
// -> totals[d].  (Its reads are scattered so that those of the two kernels
// around it, a block's counts of all digits, are not.)
__global__ __launch_bounds__(256) void plan_scan_kernel(
    int n_blocks, int bits, int* __restrict__ counts,
    int* __restrict__ totals) {
  __shared__ int wsum[4];
  int carry = 0;
  for (int base = 0; base < n_blocks; base += 256) {
    const int i = base + threadIdx.x;
    const int64_t at = ((int64_t)i << bits) + blockIdx.x;
    const int v = i < n_blocks ? counts[at] : 0;
    int sum;
    const int ex = block_scan<4>(v, wsum, sum);
    if (i < n_blocks) counts[at] = carry + ex;
    carry += sum;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// A wave takes consecutive keys of the tile, 64 at a time.  SELF: counts are
// the blocks' own (added up here, four digits a thread), else scanned, with
// their totals.
template <typename I, int THREADS, int TILE, bool SELF>
__global__ __launch_bounds__(THREADS) void plan_scatter_kernel(
    int64_t n, int64_t n_groups, const I* __restrict__ ids,
    const uint32_t* __restrict__ keys, const int* __restrict__ payload,
    int shift, int bits, const int* __restrict__ counts,
    const int* __restrict__ totals, uint32_t* __restrict__ keys_out,
    int* __restrict__ payload_out, int* __restrict__ rank_out) {
  constexpr int WAVES = THREADS / 64, ITEMS = TILE / THREADS;
  static_assert(!SELF || THREADS >= kMaxBins, "a thread a digit");
  __shared__ __attribute__((aligned(16))) int cnt[WAVES][kMaxBins];
  __shared__ int first[kMaxBins];        // where the block's keys of a digit go
  __shared__ int wsum[WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n_bins = 1 << bits;
  const int64_t base =
      (int64_t)blockIdx.x * TILE + wave * ITEMS * 64 + lane;
  uint32_t key[ITEMS];
  int pay[ITEMS], rank[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const int64_t i = base + j * 64;
    key[j] = i < n ? load_key(ids, keys, n_groups, i) : 0u;
    pay[j] = i < n && payload != nullptr ? payload[i] : (int)i;
  }
  // the scan of the digits' totals, and this block's place among the blocks
  constexpr int PER = SELF ? 1 : (kMaxBins + THREADS - 1) / THREADS;
  int total[PER], mine[PER], sum = 0, all;
  if constexpr (SELF) {
    // a thread adds four digits over every 8th (16th) block; cnt takes the parts
    const int quads = n_bins >> 2, q = threadIdx.x & (quads - 1);
    const int g = threadIdx.x >> (bits - 2);
    const int parts = (THREADS * 4 / kMaxBins) << (bits != kMaxBits);
    int* part_t = &cnt[0][0];
    int* part_m = part_t + (WAVES * kMaxBins) / 2;
    if (g < parts) {
      const int4* __restrict__ rows = reinterpret_cast<const int4*>(counts);
      const int nb = (int)gridDim.x;
      int4 t = {0, 0, 0, 0}, m = {0, 0, 0, 0};
#pragma unroll 8
      for (int b = g; b < nb; b += parts) {
        const int4 c = rows[b * quads + q];
        const int own = b < (int)blockIdx.x ? -1 : 0;
        t.x += c.x, t.y += c.y, t.z += c.z, t.w += c.w;
        m.x += c.x & own, m.y += c.y & own, m.z += c.z & own, m.w += c.w & own;
      }
      *reinterpret_cast<int4*>(part_t + g * n_bins + 4 * q) = t;
      *reinterpret_cast<int4*>(part_m + g * n_bins + 4 * q) = m;
    }
    __syncthreads();
    const int d = threadIdx.x;
    total[0] = mine[0] = 0;
    if (d < n_bins)
      for (int p = 0; p < parts; ++p) {
        total[0] += part_t[p * n_bins + d];
        mine[0] += part_m[p * n_bins + d];
      }
    sum = total[0];
  } else {
#pragma unroll
    for (int c = 0; c < PER; ++c) {
      const int d = threadIdx.x * PER + c;
      total[c] = d < n_bins ? totals[d] : 0;
      mine[c] =
          d < n_bins ? counts[((int64_t)blockIdx.x << bits) + d] : 0;
      sum += total[c];
    }
  }
  int run = block_scan<WAVES>(sum, wsum, all);
#pragma unroll
  for (int c = 0; c < PER; ++c) {
    const int d = threadIdx.x * PER + c;
    if (d < kMaxBins) first[d] = run + mine[c];
    run += total[c];
  }
  // (the scan's barrier is behind the last read of the parts)
  for (int d = lane; d < kMaxBins; d += 64) cnt[wave][d] = 0;
  wave_lds_sync();
  uint32_t digit[ITEMS];
  bool live[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    digit[j] = (key[j] >> shift) & (n_bins - 1);
    live[j] = base + j * 64 < n;
  }
  wave_ranks<ITEMS>(cnt[wave], digit, live, bits, rank);
  __syncthreads();
  for (int d = threadIdx.x; d < n_bins; d += THREADS) {
    int at = first[d];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const int k = cnt[w][d];
      cnt[w][d] = at;
      at += k;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ITEMS; ++j)
    if (live[j]) {
      const int pos = cnt[wave][digit[j]] + rank[j];
      keys_out[pos] = key[j];
      payload_out[pos] = pay[j];
      if (rank_out != nullptr) rank_out[pay[j]] = pos;
    }
}

// position i fills the groups behind key i - 1 up to key i (position n: up to
// n_groups), a gap of more than a few groups with its wave's help.  For lists
// of a token a group and more: 1.9 us for 393216 tokens of 20000 groups, where
// the search takes 6; but 20 us for 8192 tokens spread over 32000, 5 by search.
constexpr int kThreadGap = 8;
__global__ __launch_bounds__(256) void plan_fill_kernel(
    int64_t n, int64_t n_groups, const uint32_t* __restrict__ keys,
    int* __restrict__ starts) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int64_t from = 0, to = -1;
  if (i <= n) {
    from = i == 0 ? 0 : (int64_t)keys[i - 1] + 1;
    to = i == n ? n_groups : (int64_t)keys[i];
  }
  const bool wide = to - from >= kThreadGap;
  if (!wide)
    for (int64_t g = from; g <= to; ++g) starts[g] = (int)i;
  const int lane = threadIdx.x & 63;
  for (unsigned long long left = __ballot(wide); left != 0; left &= left - 1) {
    const int who = __ffsll(left) - 1;
    const int64_t f = __shfl(from, who), t = __shfl(to, who);
    const int value = (int)(i - lane + who);
    for (int64_t g = f + lane; g <= t; g += 64) starts[g] = value;
  }
}
__global__ __launch_bounds__(256) void plan_search_kernel(
    int64_t n, int64_t n_groups, const uint32_t* __restrict__ keys,
    int* __restrict__ starts) {
  const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (g <= n_groups) starts[g] = (int)keys_below(keys, n, g);
}

int launch_starts(int64_t n, int64_t n_groups, const uint32_t* keys,
                  int* starts, hipStream_t st) {
  if (n >= n_groups)
    hipLaunchKernelGGL(plan_fill_kernel, dim3((unsigned)ceil_div(n + 1, 256)),
                       dim3(256), 0, st, n, n_groups, keys, starts);
  else
    hipLaunchKernelGGL(plan_search_kernel,
                       dim3((unsigned)ceil_div(n_groups + 1, 256)), dim3(256),
                       0, st, n, n_groups, keys, starts);
  return check_launch("xrd_token_plan");
}

struct Passes {
  int count, bits;
};
Passes plan_passes(int64_t n_groups) {
  int bits = 0;
  while ((n_groups >> bits) != 0) ++bits;      // keys 0 .. n_groups
  if (bits < 2) bits = 2;                      // the scatter reads four counts
  const int count = (bits + kMaxBits - 1) / kMaxBits;
  return Passes{count, (bits + count - 1) / count};
}
int plan_tile(int64_t n) {
  return n <= (int64_t)kSelfTiles * kShortTile ? kShortTile : kLongTile;
}
int64_t plan_blocks(int64_t n) { return ceil_div(n, plan_tile(n)); }

template <typename I, int TILE>
void launch_self_pass(int64_t n, int64_t n_groups, const I* ids,
                      const uint32_t* kin, const int* pin, int shift, int bits,
                      int* counts, uint32_t* kout, int* pout, int* rank,
                      hipStream_t st) {
  const dim3 grid((unsigned)plan_blocks(n)), block(kSelfThreads);
  hipLaunchKernelGGL((plan_count_kernel<I, kSelfThreads, TILE>), grid, block, 0,
                     st, n, n_groups, ids, kin, shift, bits, counts);
  hipLaunchKernelGGL((plan_scatter_kernel<I, kSelfThreads, TILE, true>), grid,
                     block, 0, st, n, n_groups, ids, kin, pin, shift, bits,
                     counts, (const int*)nullptr, kout, pout, rank);
}
template <typename I>
void launch_pass(int64_t n, int64_t n_groups, const I* ids,
                 const uint32_t* kin, const int* pin, int shift, int bits,
                 int* counts, int* totals, uint32_t* kout, int* pout,
                 int* rank, hipStream_t st) {
  const int nb = (int)plan_blocks(n);
  if (plan_tile(n) == kShortTile)
    return launch_self_pass<I, kShortTile>(n, n_groups, ids, kin, pin, shift,
                                           bits, counts, kout, pout, rank, st);
  if (nb <= kSelfTiles)
    return launch_self_pass<I, kLongTile>(n, n_groups, ids, kin, pin, shift,
                                          bits, counts, kout, pout, rank, st);
  hipLaunchKernelGGL((plan_count_kernel<I, 256, kLongTile>), dim3(nb), dim3(256),
                     0, st, n, n_groups, ids, kin, shift, bits, counts);
  hipLaunchKernelGGL(plan_scan_kernel, dim3(1 << bits), dim3(256), 0, st, nb,
                     bits, counts, totals);
  hipLaunchKernelGGL((plan_scatter_kernel<I, 256, kLongTile, false>), dim3(nb),
                     dim3(256), 0, st, n, n_groups, ids, kin, pin, shift, bits,
                     counts, totals, kout, pout, rank);
}

template <typename I, int ITEMS>
void launch_small(int64_t n, int64_t n_groups, const I* ids, Passes ps,
                  int* order, int* starts, int* rank, uint32_t* keys_out,
                  hipStream_t st) {
  hipLaunchKernelGGL((plan_small_kernel<I, ITEMS>), dim3(1),
                     dim3(kSmallThreads), 0, st, (int)n, n_groups, ids,
                     ps.bits, ps.count, order, starts, rank, keys_out);
}

constexpr int64_t kSmallGroups = 4096;   // searched by the sorting block itself
template <typename I>
int launch_plan(int64_t n, int64_t n_groups, const I* ids, int32_t* order,
                int32_t* starts, int32_t* rank, int32_t* ws, hipStream_t st) {
  const Passes ps = plan_passes(n_groups);
  if (n <= kSmall) {
    uint32_t* kout = n_groups > kSmallGroups ? (uint32_t*)ws : nullptr;
    if (n <= kSmallThreads)
      launch_small<I, 1>(n, n_groups, ids, ps, order, starts, rank, kout, st);
    else if (n <= 2 * kSmallThreads)
      launch_small<I, 2>(n, n_groups, ids, ps, order, starts, rank, kout, st);
    else if (n <= 4 * kSmallThreads)
      launch_small<I, 4>(n, n_groups, ids, ps, order, starts, rank, kout, st);
    else
      launch_small<I, 8>(n, n_groups, ids, ps, order, starts, rank, kout, st);
    if (kout != nullptr) return launch_starts(n, n_groups, kout, starts, st);
    return check_launch("xrd_token_plan");
  }
  uint32_t* keys[2] = {(uint32_t*)ws, (uint32_t*)ws + n};
  int* spare = ws + 2 * n;
  int* totals = ws + 3 * n;
  int* counts = (int*)(((uintptr_t)(totals + kMaxBins) + 15) & ~(uintptr_t)15);
  for (int p = 0; p < ps.count && n > 0; ++p) {
    const I* from_ids = p == 0 ? ids : nullptr;
    const uint32_t* kin = p == 0 ? nullptr : keys[(p + 1) & 1];
    // the payload alternates between order and the spare buffer, ending in
    // order
    int* pout = ((ps.count - 1 - p) & 1) ? spare : order;
    const int* pin = p == 0 ? nullptr : pout == order ? spare : order;
    int* rank_out = p == ps.count - 1 ? rank : nullptr;
    launch_pass(n, n_groups, from_ids, kin, pin, p * ps.bits, ps.bits, counts,
                totals, keys[p & 1], pout, rank_out, st);
  }
  return launch_starts(n, n_groups, keys[(ps.count - 1) & 1], starts, st);
}

// ------------------------------------------------------------------ lookup
// N consecutive columns of a row as f32
template <typename T, int N>
__device__ __forceinline__ void load_cols(const T* __restrict__ p,
                                          float (&v)[N]) {
  const Vec<T, N> r = *reinterpret_cast<const Vec<T, N>*>(p);
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = to_f32(r.v[e]);
}
template <typename T, int N, bool PAST = false>
__device__ __forceinline__ void store_cols(T* __restrict__ p,
                                           const float (&v)[N]) {
  Vec<T, N> r;
#pragma unroll
  for (int e = 0; e < N; ++e) r.v[e] = from_f32<T>(v[e]);
  if constexpr (sizeof(r) == 16)
    store16<PAST>(reinterpret_cast<Vec<T, N>*>(p), r);
  else
    *reinterpret_cast<Vec<T, N>*>(p) = r;
}

// The kernels below give a row of `cols` chunks of N columns to 1 << LG lanes
// (the power of two at or above cols, at most a block): no division by cols.
// Up to BATCH tokens of a row are loaded before any of them is used, so that
// their latencies overlap: ids, then rows and weights.
constexpr int kBatch = 8;

// weights and rows of tokens t0 .. t0 + kBatch - 1 (those below `end`) added to
// acc: row_of(t) gives the row's address, or NULL for a token that adds nothing
template <typename T, int N, typename R, typename W>
__device__ __forceinline__ void add_batch(int64_t t0, int64_t end, int c,
                                          R row_of, W weight_of,
                                          float (&acc)[N]) {
  const T* row[kBatch];
  float w[kBatch];
  Vec<T, N> v[kBatch];
#pragma unroll
  for (int b = 0; b < kBatch; ++b)
    row[b] = t0 + b < end ? row_of(t0 + b, w[b]) : nullptr;
#pragma unroll
  for (int b = 0; b < kBatch; ++b) {
    v[b] = row[b] != nullptr ? *reinterpret_cast<const Vec<T, N>*>(row[b] + c)
                             : Vec<T, N>{};
    w[b] = row[b] != nullptr ? weight_of(t0 + b, w[b]) : 0.f;
  }
#pragma unroll
  for (int b = 0; b < kBatch; ++b)
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = fmaf(w[b], to_f32(v[b].v[e]), acc[e]);
}

// out row = scale * (weight of) one table row: a load and a store a lane
template <typename T, typename I, int N>
__global__ __launch_bounds__(256) void lookup_one_kernel(
    int64_t n, int64_t n_rows, int cols, int lg, const T* __restrict__ table,
    int64_t table_stride, const I* __restrict__ ids,
    const float* __restrict__ weights, float scale, T* __restrict__ out) {
  const int64_t i = ((int64_t)blockIdx.x << (8 - lg)) + (threadIdx.x >> lg);
  if (i >= n) return;
  const int64_t id = (int64_t)ids[i];
  const bool hit = id >= 0 && id < n_rows;
  const float w = hit && weights != nullptr ? weights[i] : 1.f;
  for (int c = threadIdx.x & ((1 << lg) - 1); c < cols; c += 1 << lg) {
    float v[N] = {};
    if (hit) {
      load_cols<T, N>(table + id * table_stride + c * N, v);
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = v[e] * w * scale;
    }
    store_cols<T, N>(out + (i * cols + c) * N, v);
  }
}

// 1 << lg lanes an output row
template <typename T, typename I, int N>
__global__ __launch_bounds__(256) void lookup_fwd_kernel(
    int64_t n, int k, int64_t n_rows, int cols, int lg,
    const T* __restrict__ table, int64_t table_stride,
    const I* __restrict__ ids, const float* __restrict__ weights, float scale,
    T* __restrict__ out) {
  const int64_t i = ((int64_t)blockIdx.x << (8 - lg)) + (threadIdx.x >> lg);
  if (i >= n) return;
  for (int c = threadIdx.x & ((1 << lg) - 1); c < cols; c += 1 << lg) {
    float acc[N] = {};
    for (int64_t t = i * k; t < (i + 1) * k; t += kBatch)
      add_batch<T, N>(
          t, (i + 1) * k, c * N,
          [&](int64_t u, float&) -> const T* {
            const int64_t id = (int64_t)ids[u];
            return id >= 0 && id < n_rows ? table + id * table_stride
                                          : nullptr;
          },
          [&](int64_t u, float) {
            return weights != nullptr ? weights[u] : 1.f;
          },
          acc);
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] *= scale;
    store_cols<T, N>(out + (i * cols + c) * N, acc);
  }
}

// Gradient of the table.  A row of up to kLong tokens is summed by one group of
// lanes.  The tokens of longer rows are cut at multiples of kLong of the sorted
// list: a chunk holds at most the end of one long row (its part 0) and the
// start of another (part 1), so two partial sums a chunk have room for all; a
// second launch adds the parts of each long row.  (A batch in which one row
// owns 550 of 8192 tokens, 2048 columns: 219 us summed row by row.)  Both
// launches, us, with 8, 16, 32, 64: 8192 tokens of 2048 bf16 columns 43, 41, 48,
// 81; 393216 of 16 f32 columns 25.5, 24.8, 29.2, -.
constexpr int kLong = 16;
// rows a group of lanes takes where there are more rows than the chip holds (the
// 8192 tokens above, a table of 32000 rows: 58, 45, 41, 57 us with 1, 2, 4, 8)
constexpr int kRows = 4;

// The plan's arrays come from the caller.  Whatever they hold, nothing outside the
// list of `total` tokens is read: starts are cut to 0 .. total (one median
// instruction), token numbers to 0 .. total - 1 (one unsigned minimum), and in a
// row's sum a token outside adds nothing.  Several are loaded first and cut then:
// under a load's own condition the cut would make every load wait for the one
// before.
__device__ __forceinline__ int cut_start(int s, int total) {
  return max(0, min(s, total));
}
__device__ __forceinline__ int cut_token(int t, int total) {
  return (int)min((unsigned)t, (unsigned)total - 1u);
}

// the tokens [s, e) of the sorted list for columns c ..
template <typename T, int N>
__device__ __forceinline__ void sum_tokens(
    int64_t s, int64_t e, int total, int k, int c, const T* __restrict__ dout,
    int64_t dout_stride, const int* __restrict__ order,
    const float* __restrict__ weights, float (&acc)[N]) {
  for (int64_t t = s; t < e; t += kBatch) {
    int tok[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) tok[b] = t + b < e ? order[t + b] : 0;
    add_batch<T, N>(
        0, e - t, c,
        [&](int64_t u, float&) -> const T* {
          const int64_t i = k == 1 ? tok[u] : tok[u] / k;
          return (unsigned)tok[u] < (unsigned)total ? dout + i * dout_stride
                                                    : nullptr;
        },
        [&](int64_t u, float) {
          return weights != nullptr ? weights[tok[u]] : 1.f;
        },
        acc);
  }
}

template <typename T, typename I, int N, bool PAST>
__device__ __forceinline__ void table_block(
    int64_t block, int64_t n_rows, int total, int k, int cols, int lg,
    int rows_each, int64_t row_blocks, const T* __restrict__ dout, int64_t dout_stride,
    const I* __restrict__ ids, const int* __restrict__ order,
    const int* __restrict__ starts, const float* __restrict__ weights,
    float scale, T* __restrict__ dtable, float* __restrict__ parts) {
  const int c0 = threadIdx.x & ((1 << lg) - 1), g = threadIdx.x >> lg;
  if (block < row_blocks) {
    const int64_t row0 = ((block << (8 - lg)) + g) * rows_each;
    int at[kRows + 1];
#pragma unroll
    for (int r = 0; r <= kRows; ++r)
      at[r] = r <= rows_each && row0 + r <= n_rows ? starts[row0 + r] : 0;
#pragma unroll
    for (int r = 0; r <= kRows; ++r) at[r] = cut_start(at[r], total);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (r >= rows_each || row0 + r >= n_rows) return;
      if (at[r + 1] - at[r] > kLong) continue;
      for (int c = c0; c < cols; c += 1 << lg) {
        float acc[N] = {};
        sum_tokens<T, N>(at[r], at[r + 1], total, k, c * N, dout, dout_stride,
                         order, weights, acc);
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] *= scale;
        store_cols<T, N, PAST>(dtable + ((row0 + r) * cols + c) * N, acc);
      }
    }
    return;
  }
  const int64_t chunk =
      ((block - row_blocks) << (8 - lg)) + g;
  const int64_t live = cut_start(starts[n_rows], total);
  const int64_t lo = chunk * kLong;
  const int64_t hi = lo + kLong < live ? lo + kLong : live;
  if (lo >= hi) return;
  const int64_t v0 = (int64_t)ids[cut_token(order[lo], total)];
  const int64_t v1 = (int64_t)ids[cut_token(order[hi - 1], total)];
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const int64_t v = part == 0 ? v0 : v1;
    if (part == 1 && v1 == v0) return;
    if (v < 0 || v >= n_rows) continue;      // (the plan of other ids)
    const int64_t s = cut_start(starts[v], total);
    const int64_t e = cut_start(starts[v + 1], total);
    if (e - s <= kLong) continue;
    const int64_t from = s > lo ? s : lo, to = e < hi ? e : hi;
    float* out = parts + (2 * chunk + part) * (int64_t)cols * N;
    for (int c = c0; c < cols; c += 1 << lg) {
      float acc[N] = {};
      sum_tokens<T, N>(from, to, total, k, c * N, dout, dout_stride, order,
                       weights, acc);
      store_cols<float, N>(out + c * N, acc);
    }
  }
}

// A block looks at as many chunks as it has groups of lanes (64 at most) for
// long rows that start in them.  A row of up to
// kParts parts is summed by one group of lanes; longer ones by all groups of
// the block side by side (chunk numbers apart by their number), whose sums meet
// in LDS.
constexpr int kJoin = 64, kParts = 32;
template <typename T, typename I, int N>
__global__ __launch_bounds__(256) void lookup_join_kernel(
    int64_t n_rows, int total, int cols, int lg, int each,
    const I* __restrict__ ids, const int* __restrict__ order,
    const int* __restrict__ starts, float scale,
    T* __restrict__ dtable, const float* __restrict__ parts) {
  struct Row {
    int64_t v, chunk, last;
    int part;            // of the first chunk
  };
  __shared__ float sums[256][N];
  __shared__ Row rows[kJoin];
  __shared__ int found;
  if (threadIdx.x == 0) found = 0;
  __syncthreads();
  if (threadIdx.x < each) {
    const int64_t chunk = (int64_t)blockIdx.x * each + threadIdx.x;
    const int64_t lo = chunk * kLong, live = cut_start(starts[n_rows], total);
    const int64_t hi = lo + kLong < live ? lo + kLong : live;
    if (lo < hi) {
      // a long row that starts here reaches the chunk's end
      const int64_t v0 = (int64_t)ids[cut_token(order[lo], total)];
      const int64_t v = (int64_t)ids[cut_token(order[hi - 1], total)];
      if (v >= 0 && v < n_rows) {              // (else the plan of other ids)
        const int64_t s = cut_start(starts[v], total);
        const int64_t e = cut_start(starts[v + 1], total);
        if (e - s > kLong && s >= lo)
          rows[atomicAdd(&found, 1)] =
              Row{v, chunk, (e - 1) / kLong, v != v0 ? 1 : 0};
      }
    }
  }
  __syncthreads();
  const int c0 = threadIdx.x & ((1 << lg) - 1), g = threadIdx.x >> lg;
  const int groups = 256 >> lg;
  const int64_t dim = (int64_t)cols * N;
  const auto add = [&](const Row& r, int64_t q, int c, float (&acc)[N]) {
    float w[N];
    const int part = q == r.chunk ? r.part : 0;
    load_cols<float, N>(parts + (2 * q + part) * dim + c * N, w);
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] += w[j];
  };
  const auto put = [&](const Row& r, int c, float (&acc)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] *= scale;
    store_cols<T, N>(dtable + r.v * dim + c * N, acc);
  };
  for (int k = g; k < found; k += groups) {
    const Row r = rows[k];
    if (r.last - r.chunk >= kParts) continue;
    for (int c = c0; c < cols; c += 1 << lg) {
      float acc[N] = {};
#pragma unroll 4
      for (int64_t q = r.chunk; q <= r.last; ++q) add(r, q, c, acc);
      put(r, c, acc);
    }
  }
  for (int k = 0; k < found; ++k) {
    const Row r = rows[k];
    if (r.last - r.chunk < kParts) continue;
    for (int c = c0; c - c0 < cols; c += 1 << lg) {
      float acc[N] = {};
      if (c < cols)
#pragma unroll 4
        for (int64_t q = r.chunk + g; q <= r.last; q += groups)
          add(r, q, c, acc);
      for (int half = groups >> 1; half > 0; half >>= 1) {
        __syncthreads();
        if (g >= half && g < 2 * half)
#pragma unroll
          for (int j = 0; j < N; ++j)
            sums[threadIdx.x - (half << lg)][j] = acc[j];
        __syncthreads();
        if (g < half)
#pragma unroll
          for (int j = 0; j < N; ++j) acc[j] += sums[threadIdx.x][j];
      }
      if (g == 0 && c < cols) put(r, c, acc);
    }
  }
}

// dw_ij = scale * <row of token ij, dout_i>: 1 << lg lanes (at most a wave) take
// one i and kBatch of its k tokens at once (`turn` numbers the batches), so
// dout_i is read once for them and their rows are in flight together.
template <typename T, typename I, int N>
__device__ __forceinline__ void weights_block(
    int64_t block, int turn, int64_t n, int k, int64_t n_rows, int cols, int lg,
    const T* __restrict__ table, int64_t table_stride,
    const I* __restrict__ ids, const T* __restrict__ dout, int64_t dout_stride,
    float scale, float* __restrict__ dw) {
  const int l = threadIdx.x & ((1 << lg) - 1);
  const int64_t i = (block << (8 - lg)) + (threadIdx.x >> lg);
  if (i >= n) return;
  const int j0 = turn * kBatch;
  const T* row[kBatch];
  float acc[kBatch] = {};
#pragma unroll
  for (int b = 0; b < kBatch; ++b) {
    const int64_t id = j0 + b < k ? (int64_t)ids[i * k + j0 + b] : -1;
    row[b] = id >= 0 && id < n_rows ? table + id * table_stride : nullptr;
  }
  const T* g = dout + i * dout_stride;
  for (int c = l; c < cols; c += 1 << lg) {
    const Vec<T, N> y = *reinterpret_cast<const Vec<T, N>*>(g + c * N);
    Vec<T, N> v[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (row[b] != nullptr)
        v[b] = *reinterpret_cast<const Vec<T, N>*>(row[b] + c * N);
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (row[b] != nullptr)
#pragma unroll
        for (int e = 0; e < N; ++e)
          acc[b] = fmaf(to_f32(v[b].v[e]), to_f32(y.v[e]), acc[b]);
  }
#pragma unroll
  for (int b = 0; b < kBatch; ++b) {
    for (int o = 1 << lg >> 1; o > 0; o >>= 1)
      acc[b] += __shfl_xor(acc[b], o);
    if (l == 0 && j0 + b < k) dw[i * k + j0 + b] = acc[b] * scale;
  }
}

// Both gradients in one launch (they do not need each other, and each alone
// leaves most of the chip waiting for memory): first the blocks of the table's,
// then those of the weights'.  PAST: see store16.
template <typename T>
struct LookupGrad {
  const T *table, *dout;
  int64_t table_stride, dout_stride, n, n_rows;
  const void* ids;
  const int *order, *starts;
  const float* weights;
  T* dtable;
  float *dw, *parts;
  int64_t row_blocks;
  unsigned table_blocks, weight_blocks;
  int k, cols, lg_table, lg_weights, rows_each;
  float scale;
};
template <typename T, typename I, int N, bool PAST>
__global__ __launch_bounds__(256) void lookup_bwd_kernel(LookupGrad<T> a) {
  if (blockIdx.x < a.table_blocks) {
    table_block<T, I, N, PAST>(
        blockIdx.x, a.n_rows, (int)(a.n * a.k), a.k, a.cols, a.lg_table, a.rows_each,
        a.row_blocks, a.dout, a.dout_stride, (const I*)a.ids, a.order, a.starts,
        a.weights, a.scale, a.dtable, a.parts);
  } else {
    const unsigned w = blockIdx.x - a.table_blocks;
    weights_block<T, I, N>(w % a.weight_blocks, w / a.weight_blocks, a.n, a.k,
                           a.n_rows, a.cols, a.lg_weights, a.table,
                           a.table_stride, (const I*)a.ids, a.dout,
                           a.dout_stride, a.scale, a.dw);
  }
}

// log2 of the lanes that share a row of cols chunks
int lanes_log(int64_t cols, int most) {
  int lg = 0;
  while (lg < most && (1ll << lg) < cols) ++lg;
  return lg;
}
constexpr int64_t kMaxBlocks = (1ll << 24) - 1;   // 2^32 threads a launch

// columns a lane loads at once: 16 bytes where every row is 16-byte aligned
template <typename T>
bool wide_rows(int dim, std::initializer_list<const void*> bases,
               std::initializer_list<int64_t> strides) {
  constexpr int N = 16 / (int)sizeof(T);
  if (dim % N) return false;
  for (const void* b : bases)
    if (!aligned16(b)) return false;
  for (int64_t s : strides)
    if (s % N) return false;
  return true;
}

bool bad_ids(int id_bytes) { return id_bytes != 4 && id_bytes != 8; }
constexpr int64_t kMaxTokens = (1ll << 31) - 1 - 65536;

}  // namespace
}  // namespace xrd

using namespace xrd;

extern "C" {

int64_t xrd_token_plan_ws_ints(int64_t n, int64_t n_groups) {
  if (n < 0 || n > kMaxTokens || n_groups < 1 || n_groups > kMaxTokens)
    return -1;
  return 3 * n + kMaxBins + 4 + plan_blocks(n) * kMaxBins;
}

int xrd_token_plan(int64_t n, int64_t n_groups, const void* ids, int id_bytes,
                   int32_t* order, int32_t* starts, int32_t* rank, int32_t* ws,
                   void* stream) {
  if (n < 0 || n_groups < 1 || starts == nullptr || bad_ids(id_bytes))
    return XRD_ERR_ARG;
  if (n > 0 && (ids == nullptr || order == nullptr || ws == nullptr))
    return XRD_ERR_ARG;
  if (xrd_token_plan_ws_ints(n, n_groups) < 0) return XRD_ERR_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  return id_bytes == 4
             ? launch_plan(n, n_groups, (const int32_t*)ids, order, starts,
                           rank, ws, st)
             : launch_plan(n, n_groups, (const int64_t*)ids, order, starts,
                           rank, ws, st);
}

int xrd_lookup_fwd(int dtype, int64_t n, int k, int64_t n_rows, int dim,
                   const void* table, int64_t table_stride, const void* ids,
                   int id_bytes, const float* weights, float scale, void* out,
                   void* stream) {
  if (n < 0 || k < 1 || n_rows < 0 || dim < 1 || table_stride < 0 ||
      element_size(dtype) == 0 || bad_ids(id_bytes))
    return XRD_ERR_ARG;
  if (n == 0) return XRD_OK;
  if ((table == nullptr && n_rows > 0) || ids == nullptr || out == nullptr)
    return XRD_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
#define XRD_FWD(I, N)                                                     \
  do {                                                                    \
    const int lg = lanes_log(dim / (N), 8);                               \
    const int64_t blocks = ceil_div(n, 256 >> lg);                        \
    if (blocks > kMaxBlocks) return XRD_ERR_UNSUPPORTED;                  \
    if (k == 1)                                                           \
      hipLaunchKernelGGL((lookup_one_kernel<T, I, N>),                    \
                         dim3((unsigned)blocks), dim3(256), 0, st, n,     \
                         n_rows, dim / (N), lg, (const T*)table,          \
                         table_stride, (const I*)ids, weights, scale,     \
                         (T*)out);                                        \
    else                                                                  \
      hipLaunchKernelGGL((lookup_fwd_kernel<T, I, N>),                    \
                         dim3((unsigned)blocks), dim3(256), 0, st, n, k,  \
                         n_rows, dim / (N), lg, (const T*)table,          \
                         table_stride, (const I*)ids, weights, scale,     \
                         (T*)out);                                        \
  } while (0)
  XRD_BY_DTYPE(dtype, {
    constexpr int W = 16 / (int)sizeof(T);
    if (wide_rows<T>(dim, {table, out}, {table_stride})) {
      if (id_bytes == 4) XRD_FWD(int32_t, W);
      else XRD_FWD(int64_t, W);
    } else {
      if (id_bytes == 4) XRD_FWD(int32_t, 1);
      else XRD_FWD(int64_t, 1);
    }
  });
#undef XRD_FWD
  return check_launch("xrd_lookup_fwd");
}

int64_t xrd_lookup_bwd_ws_floats(int64_t n, int k, int dim) {
  if (n < 0 || k < 1 || dim < 1 || n > kMaxTokens / k) return -1;
  return 2 * ceil_div(n * k, kLong) * dim;
}

int xrd_lookup_bwd(int dtype, int64_t n, int k, int64_t n_rows, int dim,
                   const void* table, int64_t table_stride, const void* ids,
                   int id_bytes, const float* weights, const void* dout,
                   int64_t dout_stride, const int32_t* order,
                   const int32_t* starts, float scale, void* dtable, float* dw,
                   float* ws, void* stream) {
  if (n < 0 || k < 1 || n_rows < 0 || dim < 1 || table_stride < 0 ||
      dout_stride < 0 || element_size(dtype) == 0 || bad_ids(id_bytes) ||
      (dtable == nullptr && dw == nullptr && n > 0 && n_rows > 0))
    return XRD_ERR_ARG;
  const bool to_table = dtable != nullptr && n_rows > 0;
  const bool to_weights = dw != nullptr && n > 0;
  if (n > 0 && (dout == nullptr || ids == nullptr)) return XRD_ERR_ARG;
  if (to_table &&
      (starts == nullptr || (n > 0 && (order == nullptr || ws == nullptr))))
    return XRD_ERR_ARG;
  if (to_weights && table == nullptr && n_rows > 0) return XRD_ERR_ARG;
  if (n > kMaxTokens / k) return XRD_ERR_UNSUPPORTED;
  if (!to_table && !to_weights) return XRD_OK;
  hipStream_t st = (hipStream_t)stream;
#define XRD_BWD(I, N)                                                        \
  do {                                                                       \
    LookupGrad<T> a;                                                         \
    a.table = (const T*)table, a.dout = (const T*)dout, a.ids = ids;         \
    a.table_stride = table_stride, a.dout_stride = dout_stride;              \
    a.n = n, a.n_rows = n_rows, a.k = k, a.cols = dim / (N);                 \
    a.order = order, a.starts = starts, a.weights = weights;                 \
    a.dtable = (T*)dtable, a.dw = dw, a.parts = ws, a.scale = scale;         \
    a.lg_table = lanes_log(a.cols, 8), a.lg_weights = lanes_log(a.cols, 6);  \
    const int per = 256 >> a.lg_table;                                       \
    const int64_t chunks = ceil_div(n * k, kLong);                           \
    a.rows_each = ceil_div(n_rows, per) > 8192 ? kRows : 1;                  \
    a.row_blocks = ceil_div(n_rows, (int64_t)per * a.rows_each);             \
    const int64_t tb =                                                       \
        to_table ? a.row_blocks + ceil_div(chunks, per) : 0;                 \
    const int64_t wb = to_weights ? ceil_div(n, 256 >> a.lg_weights) : 0;    \
    const int64_t blocks = tb + wb * ceil_div(k, kBatch);                    \
    if (blocks > kMaxBlocks) return XRD_ERR_UNSUPPORTED;                     \
    a.table_blocks = (unsigned)tb, a.weight_blocks = (unsigned)wb;           \
    const bool past = n_rows * dim * (int64_t)sizeof(T) > kCachedBytes;      \
    const dim3 grid((unsigned)blocks);                                       \
    if (past)                                                                \
      hipLaunchKernelGGL((lookup_bwd_kernel<T, I, N, (N > 1)>), grid,        \
                         dim3(256), 0, st, a);                               \
    else                                                                     \
      hipLaunchKernelGGL((lookup_bwd_kernel<T, I, N, false>), grid,          \
                         dim3(256), 0, st, a);                               \
    const int look = per < kJoin ? per : kJoin;                              \
    if (to_table && chunks > 1)                                              \
      hipLaunchKernelGGL((lookup_join_kernel<T, I, N>),                      \
                         dim3((unsigned)ceil_div(chunks, look)), dim3(256),  \
                         0, st, n_rows, (int)(n * k), a.cols, a.lg_table,    \
                         look,                                               \
                         (const I*)ids, order, starts, scale, (T*)dtable,    \
                         ws);                                                \
  } while (0)
  XRD_BY_DTYPE(dtype, {
    constexpr int W = 16 / (int)sizeof(T);
    if (wide_rows<T>(dim, {table, dout, dtable, ws},
                     {table_stride, dout_stride})) {
      if (id_bytes == 4) XRD_BWD(int32_t, W);
      else XRD_BWD(int64_t, W);
    } else {
      if (id_bytes == 4) XRD_BWD(int32_t, 1);
      else XRD_BWD(int64_t, 1);
    }
  });
#undef XRD_BWD
  return check_launch("xrd_lookup_bwd");
}

}  // extern "C"
