// Products of ragged row groups with a matrix per group (xrd_grouped_*).
// Rows are sorted by group, group e owns rows [starts[e], starts[e+1]):
//
//   fwd    y_r  = act(W_e x_r + b_e)                 W_e [out, in]
//   bwd_x  dx_r = W_e^T dz_r
//   bwd_w  dW_e = sum_r dz_r x_r^T, db_e = sum_r dz_r
//
// Rows of no group (behind the last one, before the first) read 0 in y and dx.
// starts lives on the device: a block finds its group and row range itself
// (find_item), so nothing waits for the host.  Sums are f32 in a fixed order.
#include "element.h"

namespace xrd {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// One fragment = 16 bytes a lane: row l & 15, 16 bytes (l >> 4) of a 64-byte
// row piece: 32 16-bit or 16 f32 contraction steps.  C: register r of lane l
// is row 4 (l >> 4) + r, column l & 15.
__device__ __forceinline__ void mma(const Pack16<__bf16>& a,
                                    const Pack16<__bf16>& b, f32x4& c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
      __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ void mma(const Pack16<_Float16>& a,
                                    const Pack16<_Float16>& b, f32x4& c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_f16(
      __builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// step j takes element j of the four lane groups: the contraction index runs
// in another order than in memory, the same one for both operands
__device__ __forceinline__ void mma(const Pack16<float>& a,
                                    const Pack16<float>& b, f32x4& c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = XRD_MFMA4(a.v[j], b.v[j], c);
}

struct Item {
  int group;     // < n_groups; n_groups: rows of no group; -1: none left
  int64_t r0, r1;  // rows of this item
  int part;      // its number within the group
};

// rows of group g, made safe against any content of starts; the rows behind
// the last group and before the first one count as two more groups
__device__ __forceinline__ void group_rows(const int* __restrict__ starts,
                                           int n_groups, int64_t m, int g,
                                           int64_t& s, int64_t& t) {
  s = g <= n_groups ? (int64_t)starts[g] : 0;
  t = g < n_groups ? (int64_t)starts[g + 1]
                   : g == n_groups ? m : (int64_t)starts[0];
  s = s < 0 ? 0 : s > m ? m : s;
  t = t < s ? s : t > m ? m : t;
}

// item `want` of the list: every group cut into pieces of `rows` rows (at
// least `least` pieces a group).  64 groups at a time: piece counts, a wave
// scan, the lane whose range holds `want`.  All waves do the same.
__device__ __forceinline__ Item find_item(const int* __restrict__ starts,
                                          int n_groups, int64_t m, int rows,
                                          int least, bool loose_rows,
                                          int64_t want) {
  const int lane = threadIdx.x & 63;
  const int n = loose_rows ? n_groups + 2 : n_groups;
  int64_t base = 0;
  for (int g0 = 0; g0 < n; g0 += 64) {
    const int g = g0 + lane;
    int64_t s = 0, t = 0;
    int pieces = 0;
    if (g < n) {
      group_rows(starts, n_groups, m, g, s, t);
      pieces = (int)((t - s + rows - 1) / rows);
      if (g < n_groups && pieces < least) pieces = least;
    }
    int inc = pieces;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(inc, o);
      if (lane >= o) inc += u;
    }
    const unsigned long long past = __ballot(base + inc > want);
    if (past != 0) {
      const int at = __ffsll(past) - 1;
      const int before = __shfl(inc - pieces, at);
      Item it;
      it.part = (int)(want - base) - before;
      const int64_t gs = (int64_t)__shfl((int)s, at);
      const int64_t gt = (int64_t)__shfl((int)t, at);
      it.group = g0 + at < n_groups ? g0 + at : n_groups;
      it.r0 = gs + (int64_t)it.part * rows;
      it.r0 = it.r0 < gs ? gs : it.r0 > gt ? gt : it.r0;
      it.r1 = it.r0 + rows < gt ? it.r0 + rows : gt;
      return it;
    }
    base += __shfl(inc, 63);
  }
  return Item{-1, 0, 0, 0};
}

// ------------------------------------------------------------ plain tiles
// 64 x 64 of C a block of four waves (32 x 32 each), 64 bytes of the
// contraction a step, both operands stored contraction-contiguous in LDS.
constexpr int kTile = 64;

// element (i, k) of an operand: rows of the matrix (SWAP false) or its columns
// (SWAP true); zero outside
template <typename T, bool SWAP>
struct Operand {
  const T* p;
  int64_t stride;
  int64_t n_i, n_k;      // valid extents
  __device__ __forceinline__ T at(int64_t i, int64_t k) const {
    if (i >= n_i || k >= n_k) return (T)0.f;
    return SWAP ? p[k * stride + i] : p[i * stride + k];
  }
};

template <typename T, bool SA, bool SB>
__device__ __forceinline__ void tile_product(const Operand<T, SA>& a,
                                             const Operand<T, SB>& b,
                                             int64_t i0, int64_t j0,
                                             f32x4 (&acc)[2][2]) {
  constexpr int BK = 64 / (int)sizeof(T);
  constexpr int LD = BK + 16 / (int)sizeof(T);
  __shared__ __align__(16) T sa[kTile * LD];
  __shared__ __align__(16) T sb[kTile * LD];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
  const int64_t n_k = a.n_k;
  for (int64_t k0 = 0; k0 < n_k; k0 += BK) {
    __syncthreads();
    for (int e = tid; e < kTile * BK; e += 256) {
      // consecutive threads along the contiguous direction of the operand
      const int ia = SA ? e % kTile : e / BK, ka = SA ? e / kTile : e % BK;
      sa[ia * LD + ka] = a.at(i0 + ia, k0 + ka);
      const int ib = SB ? e % kTile : e / BK, kb = SB ? e / kTile : e % BK;
      sb[ib * LD + kb] = b.at(j0 + ib, k0 + kb);
    }
    __syncthreads();
    Pack16<T> fa[2], fb[2];
    const int at = (lane >> 4) * Pack16<T>::N;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      fa[u] = *reinterpret_cast<const Pack16<T>*>(
          &sa[(wi + 16 * u + (lane & 15)) * LD + at]);
      fb[u] = *reinterpret_cast<const Pack16<T>*>(
          &sb[(wj + 16 * u + (lane & 15)) * LD + at]);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int v = 0; v < 2; ++v) mma(fa[u], fb[v], acc[u][v]);
  }
}

// f(i, j, value) for every element of the block's tile this lane holds
template <typename F>
__device__ __forceinline__ void each_element(const f32x4 (&acc)[2][2], F f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        f(wi + 16 * u + 4 * (lane >> 4) + r, wj + 16 * v + (lane & 15),
          acc[u][v][r]);
}

// y = x W^T + b (SB false) or dx = dz W (SB true)
template <typename T, bool SB>
__global__ __launch_bounds__(256) void grouped_rows_kernel(
    int64_t m, int n_groups, int n_k, int n_j, const T* __restrict__ x,
    int64_t x_stride, const T* __restrict__ w, const T* __restrict__ bias,
    const int* __restrict__ starts, int relu, int j_tiles, T* __restrict__ y) {
  const int64_t it_no = blockIdx.x / j_tiles;
  const int64_t j0 = (int64_t)(blockIdx.x % j_tiles) * kTile;
  const Item it = find_item(starts, n_groups, m, kTile, 0, true, it_no);
  if (it.group < 0) return;
  f32x4 acc[2][2] = {};
  const bool live = it.group < n_groups;
  if (live) {
    const Operand<T, false> a{x, x_stride, it.r1, n_k};
    const Operand<T, SB> b{w + (int64_t)it.group * n_k * n_j,
                           SB ? (int64_t)n_j : (int64_t)n_k, n_j, n_k};
    tile_product(a, b, it.r0, j0, acc);
  }
  each_element(acc, [&](int i, int j, float v) {
    const int64_t row = it.r0 + i, col = j0 + j;
    if (row >= it.r1 || col >= n_j) return;
    if (live && bias != nullptr)
      v += to_f32(bias[(int64_t)it.group * n_j + col]);
    if (relu && v <= 0.f) v = 0.f;
    y[row * n_j + col] = from_f32<T>(v);
  });
}

template <typename T>
__global__ __launch_bounds__(256) void grouped_weights_kernel(
    int64_t m, int n_groups, int n_in, int n_out, const T* __restrict__ x,
    int64_t x_stride, const T* __restrict__ dz, int64_t dz_stride,
    const int* __restrict__ starts, int in_tiles, int out_tiles,
    T* __restrict__ dw) {
  const int j = blockIdx.x % in_tiles;
  const int i = (blockIdx.x / in_tiles) % out_tiles;
  const int e = blockIdx.x / (in_tiles * out_tiles);
  int64_t s, t;
  group_rows(starts, n_groups, m, e, s, t);
  f32x4 acc[2][2] = {};
  const Operand<T, true> a{dz + s * dz_stride, dz_stride, n_out, t - s};
  const Operand<T, true> b{x + s * x_stride, x_stride, n_in, t - s};
  tile_product(a, b, (int64_t)i * kTile, (int64_t)j * kTile, acc);
  each_element(acc, [&](int ti, int tj, float v) {
    const int64_t row = (int64_t)i * kTile + ti, col = (int64_t)j * kTile + tj;
    if (row < n_out && col < n_in)
      dw[((int64_t)e * n_out + row) * n_in + col] = from_f32<T>(v);
  });
}

// 64 columns a block, rows dealt over its four waves
template <typename T>
__global__ __launch_bounds__(256) void grouped_bias_kernel(
    int64_t m, int n_groups, int n_out, const T* __restrict__ dz,
    int64_t dz_stride, const int* __restrict__ starts, int tiles,
    T* __restrict__ db) {
  __shared__ float part[4][64];
  const int e = blockIdx.x / tiles;
  const int64_t col = (int64_t)(blockIdx.x % tiles) * 64 + (threadIdx.x & 63);
  const int wave = threadIdx.x >> 6;
  int64_t s, t;
  group_rows(starts, n_groups, m, e, s, t);
  float acc = 0.f;
  if (col < n_out)
    for (int64_t r = s + wave; r < t; r += 4)
      acc += to_f32(dz[r * dz_stride + col]);
  part[wave][threadIdx.x & 63] = acc;
  __syncthreads();
  if (wave == 0 && col < n_out) {
    const int l = threadIdx.x;
    db[(int64_t)e * n_out + col] =
        from_f32<T>((part[0][l] + part[1][l]) + (part[2][l] + part[3][l]));
  }
}

// dz = dy where the ReLU let the value pass (a NaN passes, as it did forward)
template <typename T>
__global__ __launch_bounds__(256) void grouped_relu_grad_kernel(
    int64_t m, int n, const T* __restrict__ y, const T* __restrict__ dy,
    int64_t dy_stride, T* __restrict__ dz) {
  const int64_t total = m * n;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total;
       t += (int64_t)gridDim.x * 256) {
    const int64_t r = t / n;
    const T g = dy[r * dy_stride + (t - r * n)];
    dz[t] = to_f32(y[t]) <= 0.f ? (T)0.f : g;
  }
}

constexpr int64_t kMaxBlocks = (1ll << 24) - 1;   // 2^32 threads a launch

bool bad_shape(int dtype, int64_t m, int n_groups, int n_in, int n_out) {
  return element_size(dtype) == 0 || m < 0 || n_groups < 1 || n_in < 1 ||
         n_out < 1;
}
bool too_large(int64_t m, int n_groups, int n_in, int n_out) {
  return m > (1ll << 31) - 1024 || n_groups > (1 << 20) || n_in > (1 << 20) ||
         n_out > (1 << 20);
}

template <typename T, bool SB>
int launch_rows(int64_t m, int n_groups, int n_k, int n_j, const void* x,
                int64_t x_stride, const void* w, const void* bias,
                const int32_t* starts, int relu, void* y, hipStream_t st) {
  const int64_t j_tiles = ceil_div(n_j, kTile);
  const int64_t blocks = (ceil_div(m, kTile) + n_groups + 2) * j_tiles;
  if (blocks > kMaxBlocks) return XRD_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((grouped_rows_kernel<T, SB>), dim3((unsigned)blocks),
                     dim3(256), 0, st, m, n_groups, n_k, n_j, (const T*)x,
                     x_stride, (const T*)w, (const T*)bias, starts, relu,
                     (int)j_tiles, (T*)y);
  return check_launch("xrd_grouped");
}

}  // namespace
}  // namespace xrd

using namespace xrd;

extern "C" {

int xrd_grouped_fwd(int dtype, int64_t m, int n_groups, int n_in, int n_out,
                    const void* x, int64_t x_stride, const void* weight,
                    const void* bias, const int32_t* starts, int relu, void* y,
                    void* stream) {
  if (bad_shape(dtype, m, n_groups, n_in, n_out) || x_stride < 0 ||
      starts == nullptr || weight == nullptr)
    return XRD_ERR_ARG;
  if (too_large(m, n_groups, n_in, n_out)) return XRD_ERR_UNSUPPORTED;
  if (m == 0) return XRD_OK;
  if (x == nullptr || y == nullptr) return XRD_ERR_ARG;
  XRD_BY_DTYPE(dtype, return (launch_rows<T, false>(
                          m, n_groups, n_in, n_out, x, x_stride, weight, bias,
                          starts, relu, y, (hipStream_t)stream)));
}

int xrd_grouped_bwd_x(int dtype, int64_t m, int n_groups, int n_in, int n_out,
                      const void* dz, int64_t dz_stride, const void* weight,
                      const int32_t* starts, void* dx, void* stream) {
  if (bad_shape(dtype, m, n_groups, n_in, n_out) || dz_stride < 0 ||
      starts == nullptr || weight == nullptr)
    return XRD_ERR_ARG;
  if (too_large(m, n_groups, n_in, n_out)) return XRD_ERR_UNSUPPORTED;
  if (m == 0) return XRD_OK;
  if (dz == nullptr || dx == nullptr) return XRD_ERR_ARG;
  XRD_BY_DTYPE(dtype, return (launch_rows<T, true>(
                          m, n_groups, n_out, n_in, dz, dz_stride, weight,
                          nullptr, starts, 0, dx, (hipStream_t)stream)));
}

int xrd_grouped_bwd_w(int dtype, int64_t m, int n_groups, int n_in, int n_out,
                      const void* x, int64_t x_stride, const void* dz,
                      int64_t dz_stride, const int32_t* starts, void* dweight,
                      void* dbias, void* stream) {
  if (bad_shape(dtype, m, n_groups, n_in, n_out) || x_stride < 0 ||
      dz_stride < 0 || starts == nullptr ||
      (dweight == nullptr && dbias == nullptr) ||
      (m > 0 && (dz == nullptr || (x == nullptr && dweight != nullptr))))
    return XRD_ERR_ARG;
  if (too_large(m, n_groups, n_in, n_out)) return XRD_ERR_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  if (dweight != nullptr) {
    const int64_t it = ceil_div(n_in, kTile), ot = ceil_div(n_out, kTile);
    if (it * ot * n_groups > kMaxBlocks) return XRD_ERR_UNSUPPORTED;
    XRD_BY_DTYPE(dtype, hipLaunchKernelGGL(
                            (grouped_weights_kernel<T>),
                            dim3((unsigned)(it * ot * n_groups)), dim3(256), 0,
                            st, m, n_groups, n_in, n_out, (const T*)x,
                            x_stride, (const T*)dz, dz_stride, starts, (int)it,
                            (int)ot, (T*)dweight));
  }
  if (dbias != nullptr) {
    const int64_t tiles = ceil_div(n_out, 64);
    if (tiles * n_groups > kMaxBlocks) return XRD_ERR_UNSUPPORTED;
    XRD_BY_DTYPE(dtype, hipLaunchKernelGGL(
                            (grouped_bias_kernel<T>),
                            dim3((unsigned)(tiles * n_groups)), dim3(256), 0,
                            st, m, n_groups, n_out, (const T*)dz, dz_stride,
                            starts, (int)tiles, (T*)dbias));
  }
  return check_launch("xrd_grouped_bwd_w");
}

int xrd_grouped_relu_grad(int dtype, int64_t m, int n_out, const void* y,
                          const void* dy, int64_t dy_stride, void* dz,
                          void* stream) {
  if (bad_shape(dtype, m, 1, 1, n_out) || dy_stride < 0) return XRD_ERR_ARG;
  if (m == 0) return XRD_OK;
  if (y == nullptr || dy == nullptr || dz == nullptr) return XRD_ERR_ARG;
  int64_t blocks = ceil_div(m * n_out, 256);
  if (blocks > (1 << 16)) blocks = 1 << 16;
  XRD_BY_DTYPE(dtype, hipLaunchKernelGGL((grouped_relu_grad_kernel<T>),
                                         dim3((unsigned)blocks), dim3(256), 0,
                                         (hipStream_t)stream, m, n_out,
                                         (const T*)y, (const T*)dy, dy_stride,
                                         (T*)dz));
  return check_launch("xrd_grouped_relu_grad");
}

}  // extern "C"
