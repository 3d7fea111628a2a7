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
constexpr int kSortThreads = 256;
constexpr int kSortItems = 16;                           // keys a thread
constexpr int kSortTile = kSortThreads * kSortItems;     // keys a block
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kDigitBits = 8;
constexpr int kBins = 1 << kDigitBits;

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

template <typename I>
__global__ __launch_bounds__(kSortThreads) void plan_count_kernel(
    int64_t n, int64_t n_groups, const I* __restrict__ ids,
    const uint32_t* __restrict__ keys, int shift, int n_blocks,
    int* __restrict__ counts) {
  __shared__ int bins[kBins];
  for (int d = threadIdx.x; d < kBins; d += kSortThreads) bins[d] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kSortTile;
  for (int j = 0; j < kSortItems; ++j) {
    const int64_t i = base + j * kSortThreads + threadIdx.x;
    if (i < n)
      atomicAdd(&bins[(load_key(ids, keys, n_groups, i) >> shift) & (kBins - 1)],
                1);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < kBins; d += kSortThreads)
    counts[(int64_t)d * n_blocks + blockIdx.x] = bins[d];
}

// exclusive scan in place, one block
__global__ __launch_bounds__(1024) void plan_scan_kernel(int64_t n,
                                                         int* __restrict__ a) {
  __shared__ int wsum[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int carry = 0;
  for (int64_t base = 0; base < n; base += 1024) {
    const int64_t i = base + threadIdx.x;
    const int v = i < n ? a[i] : 0;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 63) wsum[wave] = inc;
    __syncthreads();
    int woff = 0, total = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) woff += wsum[w];
      total += wsum[w];
    }
    if (i < n) a[i] = carry + woff + inc - v;
    carry += total;
    __syncthreads();
  }
}

// the lanes of a wave whose digit equals this lane's
__device__ __forceinline__ unsigned long long same_digit(uint32_t d, bool live) {
  unsigned long long m = __ballot(live);
#pragma unroll
  for (int b = 0; b < kDigitBits; ++b) {
    const unsigned long long v = __ballot((d >> b) & 1u);
    m &= ((d >> b) & 1u) ? v : ~v;
  }
  return m;
}

// A wave takes kSortItems * 64 consecutive keys, 64 at a time: a key's rank is
// the wave's count of its digit so far plus the equal lanes below it, so equal
// keys keep their order.
template <typename I>
__global__ __launch_bounds__(kSortThreads) void plan_scatter_kernel(
    int64_t n, int64_t n_groups, const I* __restrict__ ids,
    const uint32_t* __restrict__ keys, const int* __restrict__ payload,
    int shift, int n_blocks, const int* __restrict__ offsets,
    uint32_t* __restrict__ keys_out, int* __restrict__ payload_out,
    int* __restrict__ rank_out) {
  __shared__ int cnt[kSortWaves][kBins];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int d = threadIdx.x; d < kSortWaves * kBins; d += kSortThreads)
    (&cnt[0][0])[d] = 0;
  __syncthreads();
  const int64_t base =
      (int64_t)blockIdx.x * kSortTile + (int64_t)wave * kSortItems * 64;
  uint32_t key[kSortItems];
  int rank[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int64_t i = base + j * 64 + lane;
    key[j] = i < n ? load_key(ids, keys, n_groups, i) : 0u;
  }
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const bool live = base + j * 64 + lane < n;
    const uint32_t d = (key[j] >> shift) & (kBins - 1);
    const unsigned long long m = same_digit(d, live);
    const int below = __popcll(m & ((1ull << lane) - 1ull));
    int before = 0;
    if (live) before = cnt[wave][d];
    wave_lds_sync();
    if (live && below == 0) cnt[wave][d] = before + __popcll(m);
    wave_lds_sync();
    rank[j] = before + below;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < kBins; d += kSortThreads) {
    int run = offsets[(int64_t)d * n_blocks + blockIdx.x];
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = cnt[w][d];
      cnt[w][d] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int64_t i = base + j * 64 + lane;
    if (i < n) {
      const uint32_t d = (key[j] >> shift) & (kBins - 1);
      const int pos = cnt[wave][d] + rank[j];
      const int p = payload != nullptr ? payload[i] : (int)i;
      keys_out[pos] = key[j];
      payload_out[pos] = p;
      if (rank_out != nullptr) rank_out[p] = pos;
    }
  }
}

// starts[g] = number of sorted keys below g
__global__ __launch_bounds__(256) void plan_starts_kernel(
    int64_t n, int64_t n_groups, const uint32_t* __restrict__ keys,
    int* __restrict__ starts) {
  const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (g > n_groups) return;
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if ((int64_t)keys[mid] < g) lo = mid + 1;
    else hi = mid;
  }
  starts[g] = (int)lo;
}

int plan_passes(int64_t n_groups) {
  int bits = 0;
  while ((n_groups >> bits) != 0) ++bits;      // keys 0 .. n_groups
  return (bits + kDigitBits - 1) / kDigitBits;
}

template <typename I>
int launch_plan(int64_t n, int64_t n_groups, const I* ids, int32_t* order,
                int32_t* starts, int32_t* rank, int32_t* ws, hipStream_t st) {
  const int passes = plan_passes(n_groups);
  const int n_blocks = (int)ceil_div(n, kSortTile);
  uint32_t* keys[2] = {(uint32_t*)ws, (uint32_t*)ws + n};
  int* spare = ws + 2 * n;
  int* counts = ws + 3 * n;
  for (int p = 0; p < passes && n > 0; ++p) {
    const I* from_ids = p == 0 ? ids : nullptr;
    const uint32_t* kin = p == 0 ? nullptr : keys[(p + 1) & 1];
    // the payload alternates between order and the spare buffer, ending in
    // order
    int* pout = ((passes - 1 - p) & 1) ? spare : order;
    const int* pin = p == 0 ? nullptr : pout == order ? spare : order;
    hipLaunchKernelGGL(plan_count_kernel<I>, dim3(n_blocks),
                       dim3(kSortThreads), 0, st, n, n_groups, from_ids, kin,
                       p * kDigitBits, n_blocks, counts);
    hipLaunchKernelGGL(plan_scan_kernel, dim3(1), dim3(1024), 0, st,
                       (int64_t)n_blocks * kBins, counts);
    hipLaunchKernelGGL(plan_scatter_kernel<I>, dim3(n_blocks),
                       dim3(kSortThreads), 0, st, n, n_groups, from_ids, kin,
                       pin, p * kDigitBits, n_blocks, counts, keys[p & 1],
                       pout, p == passes - 1 ? rank : nullptr);
  }
  hipLaunchKernelGGL(plan_starts_kernel,
                     dim3((unsigned)ceil_div(n_groups + 1, 256)), dim3(256), 0,
                     st, n, n_groups, keys[(passes - 1) & 1], starts);
  return check_launch("xrd_token_plan");
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
template <typename T, int N>
__device__ __forceinline__ void store_cols(T* __restrict__ p,
                                           const float (&v)[N]) {
  Vec<T, N> r;
#pragma unroll
  for (int e = 0; e < N; ++e) r.v[e] = from_f32<T>(v[e]);
  *reinterpret_cast<Vec<T, N>*>(p) = r;
}

// one thread = N columns of one output row
template <typename T, typename I, int N>
__global__ __launch_bounds__(256) void lookup_fwd_kernel(
    int64_t n, int k, int64_t n_rows, int cols, const T* __restrict__ table,
    int64_t table_stride, const I* __restrict__ ids,
    const float* __restrict__ weights, float scale, T* __restrict__ out) {
  const int64_t total = n * cols;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total;
       t += (int64_t)gridDim.x * 256) {
    const int64_t i = t / cols;
    const int c = (int)(t - i * cols) * N;
    float acc[N] = {};
    for (int j = 0; j < k; ++j) {
      const int64_t id = (int64_t)ids[i * k + j];
      if (id < 0 || id >= n_rows) continue;
      const float w = weights != nullptr ? weights[i * k + j] : 1.f;
      float v[N];
      load_cols<T, N>(table + id * table_stride + c, v);
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = fmaf(w, v[e], acc[e]);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] *= scale;
    store_cols<T, N>(out + (i * cols) * N + c, acc);
  }
}

// one thread = N columns of one table row: the row's tokens in order
template <typename T, int N>
__global__ __launch_bounds__(256) void lookup_bwd_table_kernel(
    int64_t n_rows, int k, int cols, const T* __restrict__ dout,
    int64_t dout_stride, const int* __restrict__ order,
    const int* __restrict__ starts, const float* __restrict__ weights,
    float scale, T* __restrict__ dtable) {
  const int64_t total = n_rows * cols;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total;
       t += (int64_t)gridDim.x * 256) {
    const int64_t row = t / cols;
    const int c = (int)(t - row * cols) * N;
    const int end = starts[row + 1];
    float acc[N] = {};
    for (int s = starts[row]; s < end; ++s) {
      const int tok = order[s];
      const float w = weights != nullptr ? weights[tok] : 1.f;
      float v[N];
      load_cols<T, N>(dout + (int64_t)(tok / k) * dout_stride + c, v);
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = fmaf(w, v[e], acc[e]);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] *= scale;
    store_cols<T, N>(dtable + (row * cols) * N + c, acc);
  }
}

// `lanes` (a power of two) lanes share one token: dot product over the columns
template <typename T, typename I, int N>
__global__ __launch_bounds__(256) void lookup_bwd_weights_kernel(
    int64_t n, int k, int64_t n_rows, int cols, int lanes,
    const T* __restrict__ table, int64_t table_stride,
    const I* __restrict__ ids, const T* __restrict__ dout, int64_t dout_stride,
    float scale, float* __restrict__ dw) {
  const int per_block = 256 / lanes;
  const int l = threadIdx.x & (lanes - 1);
  for (int64_t t = (int64_t)blockIdx.x * per_block + threadIdx.x / lanes;
       t < n * k; t += (int64_t)gridDim.x * per_block) {
    const int64_t id = (int64_t)ids[t];
    float acc = 0.f;
    if (id >= 0 && id < n_rows) {
      const T* row = table + id * table_stride;
      const T* g = dout + (t / k) * dout_stride;
      for (int c = l; c < cols; c += lanes) {
        float a[N], b[N];
        load_cols<T, N>(row + c * N, a);
        load_cols<T, N>(g + c * N, b);
#pragma unroll
        for (int e = 0; e < N; ++e) acc = fmaf(a[e], b[e], acc);
      }
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) acc += __shfl_xor(acc, o);
    if (l == 0) dw[t] = acc * scale;
  }
}

unsigned grid_for(int64_t work) {
  const int64_t b = ceil_div(work, 256);
  return (unsigned)(b > (1 << 20) ? (1 << 20) : b < 1 ? 1 : b);
}

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
constexpr int64_t kMaxTokens = (1ll << 31) - 1 - kSortTile;

}  // namespace
}  // namespace xrd

using namespace xrd;

extern "C" {

int64_t xrd_token_plan_ws_ints(int64_t n, int64_t n_groups) {
  if (n < 0 || n > kMaxTokens || n_groups < 1 || n_groups >= (1ll << 31) - 1)
    return -1;
  return 3 * n + ceil_div(n, kSortTile) * kBins + 1;
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
#define XRD_FWD(I, N)                                                        \
  hipLaunchKernelGGL((lookup_fwd_kernel<T, I, N>),                           \
                     dim3(grid_for(n * (dim / (N)))), dim3(256), 0, st, n, k, \
                     n_rows, dim / (N), (const T*)table, table_stride,       \
                     (const I*)ids, weights, scale, (T*)out)
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

int xrd_lookup_bwd_table(int dtype, int64_t n, int k, int64_t n_rows, int dim,
                         const void* dout, int64_t dout_stride,
                         const int32_t* order, const int32_t* starts,
                         const float* weights, float scale, void* dtable,
                         void* stream) {
  if (n < 0 || k < 1 || n_rows < 0 || dim < 1 || dout_stride < 0 ||
      element_size(dtype) == 0)
    return XRD_ERR_ARG;
  if (n_rows == 0) return XRD_OK;
  if (starts == nullptr || dtable == nullptr ||
      (n > 0 && (dout == nullptr || order == nullptr)))
    return XRD_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
#define XRD_BWD(N)                                                           \
  hipLaunchKernelGGL((lookup_bwd_table_kernel<T, N>),                        \
                     dim3(grid_for(n_rows * (dim / (N)))), dim3(256), 0, st, \
                     n_rows, k, dim / (N), (const T*)dout, dout_stride,      \
                     order, starts, weights, scale, (T*)dtable)
  XRD_BY_DTYPE(dtype, {
    constexpr int W = 16 / (int)sizeof(T);
    if (wide_rows<T>(dim, {dout, dtable}, {dout_stride})) XRD_BWD(W);
    else XRD_BWD(1);
  });
#undef XRD_BWD
  return check_launch("xrd_lookup_bwd_table");
}

int xrd_lookup_bwd_weights(int dtype, int64_t n, int k, int64_t n_rows,
                           int dim, const void* table, int64_t table_stride,
                           const void* ids, int id_bytes, const void* dout,
                           int64_t dout_stride, float scale, float* dw,
                           void* stream) {
  if (n < 0 || k < 1 || n_rows < 0 || dim < 1 || table_stride < 0 ||
      dout_stride < 0 || element_size(dtype) == 0 || bad_ids(id_bytes))
    return XRD_ERR_ARG;
  if (n == 0) return XRD_OK;
  if ((table == nullptr && n_rows > 0) || ids == nullptr || dout == nullptr ||
      dw == nullptr)
    return XRD_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
#define XRD_DW(I, N)                                                          \
  hipLaunchKernelGGL((lookup_bwd_weights_kernel<T, I, N>),                    \
                     dim3(grid_for(n * k * lanes)), dim3(256), 0,             \
                     st, n, k, n_rows, dim / (N), lanes, (const T*)table,     \
                     table_stride, (const I*)ids, (const T*)dout,             \
                     dout_stride, scale, dw)
  XRD_BY_DTYPE(dtype, {
    constexpr int W = 16 / (int)sizeof(T);
    const bool wide =
        wide_rows<T>(dim, {table, dout}, {table_stride, dout_stride});
    int lanes = 1;
    while (lanes < 64 && lanes < (wide ? dim / W : dim)) lanes *= 2;
    if (wide) {
      if (id_bytes == 4) XRD_DW(int32_t, W);
      else XRD_DW(int64_t, W);
    } else {
      if (id_bytes == 4) XRD_DW(int32_t, 1);
      else XRD_DW(int64_t, 1);
    }
  });
#undef XRD_DW
  return check_launch("xrd_lookup_bwd_weights");
}

}  // extern "C"
