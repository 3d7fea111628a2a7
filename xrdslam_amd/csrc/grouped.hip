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
#include "grouped_tile.h"

namespace xrd {
namespace {

struct Item {
  int group;     // < n_groups; n_groups: rows of no group; -1: none
  int64_t r0, r1;  // rows of this piece
  int pieces;    // of the group
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

// pieces of at most `rows` rows of group g (at least `least` of an own group)
__device__ __forceinline__ int pieces_of(int64_t s, int64_t t, int rows,
                                         bool own, int least) {
  const int p = (int)((t - s + rows - 1) / rows);
  return own && p < least ? least : p;
}

// number of pieces of all groups (LOOSE: and of the rows of no group).  All
// waves do the same: 64 groups at a time, one a lane.
template <bool LOOSE>
__device__ __forceinline__ int64_t count_items(const int* __restrict__ starts,
                                               int n_groups, int64_t m,
                                               int rows, int least) {
  const int lane = threadIdx.x & 63;
  const int n = LOOSE ? n_groups + 2 : n_groups;
  int64_t total = 0;
  for (int g0 = 0; g0 < n; g0 += 64) {
    const int g = g0 + lane;
    int v = 0;
    if (g < n) {
      int64_t s, t;
      group_rows(starts, n_groups, m, g, s, t);
      v = pieces_of(s, t, rows, g < n_groups, least);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    total += v;
  }
  return total;
}

// piece `want` of that list: a scan over the lanes' piece counts, the lane
// whose range holds `want`
template <bool LOOSE>
__device__ __forceinline__ Item find_item(const int* __restrict__ starts,
                                          int n_groups, int64_t m, int rows,
                                          int least, int64_t want) {
  const int lane = threadIdx.x & 63;
  const int n = LOOSE ? n_groups + 2 : n_groups;
  int64_t base = 0;
  for (int g0 = 0; g0 < n; g0 += 64) {
    const int g = g0 + lane;
    int64_t s = 0, t = 0;
    int pieces = 0;
    if (g < n) {
      group_rows(starts, n_groups, m, g, s, t);
      pieces = pieces_of(s, t, rows, g < n_groups, least);
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
      const int64_t gs = (int64_t)__shfl((int)s, at);
      const int64_t gt = (int64_t)__shfl((int)t, at);
      it.pieces = __shfl(pieces, at);
      it.group = g0 + at < n_groups ? g0 + at : n_groups;
      it.r0 = gs + (want - base - before) * rows;
      // (whatever starts holds, rows outside [gs, gt) are never touched)
      it.r0 = it.r0 < gs ? gs : it.r0 > gt ? gt : it.r0;
      it.r1 = it.r0 + rows < gt ? it.r0 + rows : gt;
      return it;
    }
    base += __shfl(inc, 63);
  }
  return Item{-1, 0, 0, 0};
}

// Blocks are dealt to the eight XCDs in turn; each XCD gets a contiguous part
// of the work list, so that the tiles that share rows or a weight panel meet in
// one L2.  -> position in the list of `total`, or -1
__device__ __forceinline__ int64_t xcd_position(int64_t block, int64_t total) {
  const int64_t x = block & 7, per = total >> 3, extra = total & 7;
  const int64_t mine = per + (x < extra);
  if ((block >> 3) >= mine) return -1;
  return x * per + (x < extra ? x : extra) + (block >> 3);
}

// four consecutive columns of a row from column j on, of n_j
template <typename T>
__device__ __forceinline__ void store4(T* __restrict__ p, int64_t j,
                                       int64_t n_j, bool whole,
                                       const f32x4& v) {
  if (whole) {
    Vec<T, 4> o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.v[e] = from_f32<T>(v[e]);
    if (j < n_j) *reinterpret_cast<Vec<T, 4>*>(p + j) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (j + e < n_j) p[j + e] = from_f32<T>(v[e]);
  }
}

// rows of y: y = x W^T + b (SB false) or dx = dz W (SB true)
template <class Tile, bool SB>
__global__ __launch_bounds__(Tile::THREADS) void grouped_rows_kernel(
    int64_t m, int n_groups, int n_k, int n_j,
    const typename Tile::T* __restrict__ x, int64_t x_stride,
    const typename Tile::T* __restrict__ w,
    const typename Tile::T* __restrict__ bias, const int* __restrict__ starts,
    int relu, int j_tiles, typename Tile::T* __restrict__ y) {
  using T = typename Tile::T;
  extern __shared__ __align__(16) char smem[];
  const int64_t total =
      count_items<true>(starts, n_groups, m, Tile::BI, 0) * j_tiles;
  const int64_t at = xcd_position(blockIdx.x, total);
  if (at < 0) return;
  const int64_t j0 = (at % j_tiles) * Tile::BJ;
  const Item it =
      find_item<true>(starts, n_groups, m, Tile::BI, 0, at / j_tiles);
  if (it.group < 0 || it.r0 >= it.r1) return;
  const bool live = it.group < n_groups;
  const bool whole = (n_j & 3) == 0 && ((uintptr_t)y & (4 * sizeof(T) - 1)) == 0;
  Tile tile;
  const T* wg = w + (int64_t)(live ? it.group : 0) * n_k * n_j;
  tile.run(smem, x, x_stride, it.r0, it.r1, wg, SB ? n_j : n_k, j0, n_j,
           live ? n_k : 0, false);
  const T* bg = live && bias != nullptr ? bias + (int64_t)it.group * n_j
                                        : nullptr;
  tile.each4([&](int i, int j, f32x4 v) {
    const int64_t row = it.r0 + i, col = j0 + j;
    if (row >= it.r1) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (bg != nullptr && col + e < n_j) v[e] += to_f32(bg[col + e]);
      if (relu && v[e] <= 0.f) v[e] = 0.f;
    }
    store4(y + row * n_j, col, n_j, whole, v);
  });
}

// A piece of a group's rows, one tile of dW (and its part of db): written
// right away when the group is one piece, else as f32 partial sums
// part_w [piece][n_out][n_in], part_b [piece][n_out] for grouped_join_kernel.
template <class Tile>
__global__ __launch_bounds__(Tile::THREADS) void grouped_weights_kernel(
    int64_t m, int n_groups, int n_in, int n_out, int piece_rows,
    int64_t piece_room, const typename Tile::T* __restrict__ x, int64_t x_stride,
    const typename Tile::T* __restrict__ dz, int64_t dz_stride,
    const int* __restrict__ starts, int in_tiles, int out_tiles,
    typename Tile::T* __restrict__ dw, typename Tile::T* __restrict__ db,
    float* __restrict__ part_w, float* __restrict__ part_b) {
  using T = typename Tile::T;
  extern __shared__ __align__(16) char smem[];
  const int tiles = in_tiles * out_tiles;
  const int64_t total =
      count_items<false>(starts, n_groups, m, piece_rows, 1) * tiles;
  const int64_t at = xcd_position(blockIdx.x, total);
  if (at < 0) return;
  const int64_t piece = at / tiles;
  const int64_t j0 = (at % in_tiles) * Tile::BJ;
  const int64_t i0 = (at / in_tiles % out_tiles) * Tile::BI;
  const Item it =
      find_item<false>(starts, n_groups, m, piece_rows, 1, piece);
  if (it.group < 0) return;
  // (more pieces than the workspace holds: starts that are not ascending)
  if (it.pieces > 1 && piece >= piece_room) return;
  const bool sums = db != nullptr && j0 == 0;
  Tile tile;
  tile.run(smem, dz + it.r0 * dz_stride, dz_stride, i0, n_out,
           x + it.r0 * x_stride, x_stride, j0, n_in, it.r1 - it.r0, sums);
  const bool alone = it.pieces == 1;
  if (alone) {
    T* out = dw + (int64_t)it.group * n_out * n_in;
    const bool whole =
        (n_in & 3) == 0 && ((uintptr_t)dw & (4 * sizeof(T) - 1)) == 0;
    tile.each4([&](int i, int j, f32x4 v) {
      if (i0 + i < n_out)
        store4(out + (i0 + i) * n_in, j0 + j, n_in, whole, v);
    });
  } else {
    float* out = part_w + piece * n_out * n_in;
    const bool whole = (n_in & 3) == 0;
    tile.each4([&](int i, int j, f32x4 v) {
      if (i0 + i < n_out)
        store4(out + (i0 + i) * n_in, j0 + j, n_in, whole, v);
    });
  }
  if (sums)
    tile.each_sum([&](int i, float v) {
      if (i0 + i >= n_out) return;
      if (alone) db[(int64_t)it.group * n_out + i0 + i] = from_f32<T>(v);
      else part_b[piece * n_out + i0 + i] = v;
    });
}

// sums of the pieces of every group that has several, in their order
template <typename T>
__global__ __launch_bounds__(256) void grouped_join_kernel(
    int64_t m, int n_groups, int64_t n_w, int n_out, int piece_rows,
    int64_t piece_room, int blocks_a_group, const int* __restrict__ starts, T* __restrict__ dw,
    T* __restrict__ db, const float* __restrict__ part_w,
    const float* __restrict__ part_b) {
  const int g = blockIdx.x / blocks_a_group;
  int64_t s, t;
  group_rows(starts, n_groups, m, g, s, t);
  const int pieces = pieces_of(s, t, piece_rows, true, 1);
  if (pieces == 1) return;
  const int64_t first =
      count_items<false>(starts, g, m, piece_rows, 1);
  if (first + pieces > piece_room) return;
  const int64_t e = (int64_t)(blockIdx.x % blocks_a_group) * 256 + threadIdx.x;
  if (e < n_w) {
    float acc = 0.f;
    for (int p = 0; p < pieces; ++p) acc += part_w[(first + p) * n_w + e];
    dw[g * n_w + e] = from_f32<T>(acc);
  } else if (db != nullptr && e < n_w + n_out) {
    const int64_t c = e - n_w;
    float acc = 0.f;
    for (int p = 0; p < pieces; ++p) acc += part_b[(first + p) * n_out + c];
    db[(int64_t)g * n_out + c] = from_f32<T>(acc);
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

// 16-byte chunks: every row starts on 16 bytes and is made of whole chunks
template <typename T>
bool chunked(const void* p, int64_t stride, int n) {
  constexpr int N = 16 / (int)sizeof(T);
  return aligned16(p) && stride % N == 0 && n % N == 0;
}

template <class Tile, bool SB>
int launch_rows_tile(int64_t m, int n_groups, int n_k, int n_j, const void* x,
                     int64_t x_stride, const void* w, const void* bias,
                     const int32_t* starts, int relu, void* y,
                     hipStream_t st) {
  using T = typename Tile::T;
  const int64_t j_tiles = ceil_div(n_j, Tile::BJ);
  // a group's last piece may be short, and so may the two runs of other rows
  const int64_t blocks =
      ceil_div((m / Tile::BI + n_groups + 2) * j_tiles, 8) * 8;
  if (blocks > kMaxBlocks) return XRD_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((grouped_rows_kernel<Tile, SB>), dim3((unsigned)blocks),
                     dim3(Tile::THREADS), Tile::LDS, st, m, n_groups, n_k, n_j,
                     (const T*)x, x_stride, (const T*)w, (const T*)bias,
                     starts, relu, (int)j_tiles, (T*)y);
  return check_launch("xrd_grouped");
}

template <typename T, bool SB>
int launch_rows(int64_t m, int n_groups, int n_k, int n_j, const void* x,
                int64_t x_stride, const void* w, const void* bias,
                const int32_t* starts, int relu, void* y, hipStream_t st) {
  const bool whole =
      chunked<T>(x, x_stride, n_k) && chunked<T>(w, 0, SB ? n_j : n_k);
  if (whole)
    return launch_rows_tile<MatrixTile<T, false, SB, false, 128, 128, 2, 2,
                                       false>, SB>(
        m, n_groups, n_k, n_j, x, x_stride, w, bias, starts, relu, y, st);
  return launch_rows_tile<MatrixTile<T, false, SB, true, 128, 128, 2, 2,
                                     false>, SB>(
      m, n_groups, n_k, n_j, x, x_stride, w, bias, starts, relu, y, st);
}

// Rows a piece of the weight gradient holds.  One piece a group where groups
// and tiles alone fill the chip (no partial sums to write and read back), else
// as many pieces as make about four blocks a CU, of 256 rows or more.
constexpr int kWeightTile = 128;
int piece_rows_of(int64_t m, int n_groups, int n_in, int n_out) {
  const int64_t tiles = ceil_div(n_in, kWeightTile) *
                        ceil_div(n_out, kWeightTile);
  if (tiles * n_groups >= 512) return 1 << 30;
  const int64_t pieces = ceil_div(1024, tiles);
  int64_t rows = ceil_div(ceil_div(m, pieces), 64) * 64;
  if (rows < 256) rows = 256;
  return (int)(rows > (1 << 30) ? (1 << 30) : rows);
}
// pieces of all groups at most (0: every group is one piece)
int64_t piece_bound(int64_t m, int n_groups, int n_in, int n_out) {
  const int rows = piece_rows_of(m, n_groups, n_in, n_out);
  return m <= rows ? 0 : m / rows + n_groups;
}

template <class Tile>
int launch_weights(int64_t m, int n_groups, int n_in, int n_out, const void* x,
                   int64_t x_stride, const void* dz, int64_t dz_stride,
                   const int32_t* starts, void* dw, void* db, float* ws,
                   hipStream_t st) {
  using T = typename Tile::T;
  const int64_t it = ceil_div(n_in, Tile::BJ), ot = ceil_div(n_out, Tile::BI);
  const int rows = piece_rows_of(m, n_groups, n_in, n_out);
  const int64_t bound = piece_bound(m, n_groups, n_in, n_out);
  const int64_t blocks =
      ceil_div((m / rows + n_groups) * it * ot, 8) * 8;
  if (blocks > kMaxBlocks) return XRD_ERR_UNSUPPORTED;
  const int64_t n_w = (int64_t)n_out * n_in;
  float* part_b = ws + bound * n_w;
  hipLaunchKernelGGL((grouped_weights_kernel<Tile>), dim3((unsigned)blocks),
                     dim3(Tile::THREADS), Tile::LDS, st, m, n_groups, n_in,
                     n_out, rows, bound, (const T*)x, x_stride, (const T*)dz,
                     dz_stride, starts, (int)it, (int)ot, (T*)dw, (T*)db, ws,
                     part_b);
  if (bound > 0) {
    const int64_t per = ceil_div(n_w + (db != nullptr ? n_out : 0), 256);
    if (per * n_groups > kMaxBlocks) return XRD_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((grouped_join_kernel<T>), dim3((unsigned)(per * n_groups)),
                       dim3(256), 0, st, m, n_groups, n_w, n_out, rows,
                       bound, (int)per, starts, (T*)dw, (T*)db, ws, part_b);
  }
  return check_launch("xrd_grouped_bwd_w");
}

template <typename T, bool ONES>
int launch_weights_of(int64_t m, int n_groups, int n_in, int n_out,
                      const void* x, int64_t x_stride, const void* dz,
                      int64_t dz_stride, const int32_t* starts, void* dw,
                      void* db, float* ws, hipStream_t st) {
  if (chunked<T>(x, x_stride, n_in) && chunked<T>(dz, dz_stride, n_out))
    return launch_weights<MatrixTile<T, true, true, false, kWeightTile,
                                     kWeightTile, 2, 2, ONES>>(
        m, n_groups, n_in, n_out, x, x_stride, dz, dz_stride, starts, dw, db,
        ws, st);
  return launch_weights<MatrixTile<T, true, true, true, kWeightTile,
                                   kWeightTile, 2, 2, ONES>>(
      m, n_groups, n_in, n_out, x, x_stride, dz, dz_stride, starts, dw, db, ws,
      st);
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

int64_t xrd_grouped_ws_floats(int64_t m, int n_groups, int n_in, int n_out) {
  if (bad_shape(XRD_F32, m, n_groups, n_in, n_out) ||
      too_large(m, n_groups, n_in, n_out))
    return -1;
  return piece_bound(m, n_groups, n_in, n_out) *
         ((int64_t)n_out * n_in + n_out);
}

int xrd_grouped_bwd_w(int dtype, int64_t m, int n_groups, int n_in, int n_out,
                      const void* x, int64_t x_stride, const void* dz,
                      int64_t dz_stride, const int32_t* starts, void* dweight,
                      void* dbias, float* ws, void* stream) {
  if (bad_shape(dtype, m, n_groups, n_in, n_out) || x_stride < 0 ||
      dz_stride < 0 || starts == nullptr || dweight == nullptr ||
      (m > 0 && (dz == nullptr || x == nullptr)))
    return XRD_ERR_ARG;
  const int64_t need = xrd_grouped_ws_floats(m, n_groups, n_in, n_out);
  if (need < 0) return XRD_ERR_UNSUPPORTED;
  if (need > 0 && ws == nullptr) return XRD_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  XRD_BY_DTYPE(dtype, {
    if (dbias != nullptr)
      return (launch_weights_of<T, true>(m, n_groups, n_in, n_out, x, x_stride,
                                         dz, dz_stride, starts, dweight, dbias,
                                         ws, st));
    return (launch_weights_of<T, false>(m, n_groups, n_in, n_out, x, x_stride,
                                        dz, dz_stride, starts, dweight,
                                        nullptr, ws, st));
  });
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
