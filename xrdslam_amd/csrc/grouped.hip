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

// Rows and pieces are counted in 32 bits (there are fewer than 2^31 rows): 64-bit
// divisions are a hundred instructions each, in front of every tile.
struct Item {
  int group;     // < n_groups; n_groups: rows of no group; -1: none
  int r0, r1;    // rows of this piece
  int pieces;    // of the group
};

// rows of group g, made safe against any content of starts; the rows behind
// the last group and before the first one count as two more groups
__device__ __forceinline__ void group_rows(const int* __restrict__ starts,
                                           int n_groups, int m, int g, int& s,
                                           int& t) {
  s = g <= n_groups ? starts[g] : 0;
  t = g < n_groups ? starts[g + 1] : g == n_groups ? m : starts[0];
  s = s < 0 ? 0 : s > m ? m : s;
  t = t < s ? s : t > m ? m : t;
}

// pieces of at most `rows` rows of group g (at least `least` of an own group)
__device__ __forceinline__ int pieces_of(int s, int t, int rows, bool own,
                                         int least) {
  const int n = t - s;
  const int p = (int)((unsigned)n / (unsigned)rows) + (n % rows != 0);
  return own && p < least ? least : p;
}

// inclusive sum over the lanes up to this one (row shifts, then row broadcasts)
__device__ __forceinline__ int wave_scan(int v) {
#define XRD_SCAN(CTRL, ROWS) \
  v += __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, true)
  XRD_SCAN(0x111, 0xf);   // row_shr:1
  XRD_SCAN(0x112, 0xf);   // row_shr:2
  XRD_SCAN(0x114, 0xf);   // row_shr:4
  XRD_SCAN(0x118, 0xf);   // row_shr:8
#undef XRD_SCAN
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // bcast:31
  return v;
}

// The list of pieces, 64 groups at a time, one a lane (all waves do the same).
// LOOSE: the rows of no group are listed too.  A list of at most 64 groups is
// read from memory once.
template <bool LOOSE>
struct PieceList {
  const int* starts;
  int n_groups, m, rows, least;
  int s, t;           // this lane's group of the chunk read last
  int pieces, upto;   // its pieces, and those of the lanes up to it

  __device__ __forceinline__ PieceList(const int* starts_, int n_groups_,
                                       int64_t m_, int rows_, int least_)
      : starts(starts_), n_groups(n_groups_), m((int)m_), rows(rows_),
        least(least_) {}
  __device__ __forceinline__ int length() const {
    return LOOSE ? n_groups + 2 : n_groups;
  }
  // reads groups g0 .. g0 + 63 (below `end`) -> their pieces
  __device__ __forceinline__ int read(int g0, int end) {
    const int lane = threadIdx.x & 63, g = g0 + lane;
    s = t = 0;
    pieces = 0;
    if (g < end) {
      group_rows(starts, n_groups, m, g, s, t);
      pieces = pieces_of(s, t, rows, g < n_groups, least);
    }
    upto = wave_scan(pieces);
    return __builtin_amdgcn_readlane(upto, 63);
  }
  // pieces of the groups below `end`
  __device__ __forceinline__ int64_t count(int end) {
    int64_t total = 0;
    for (int g0 = 0; g0 < end; g0 += 64) total += read(g0, end);
    return total;
  }
  // piece `want`; have: the list was counted and has one chunk
  __device__ __forceinline__ Item find(int64_t want, bool have) {
    int64_t base = 0;
    for (int g0 = 0; g0 < length(); g0 += 64) {
      const int sum =
          have ? __builtin_amdgcn_readlane(upto, 63) : read(g0, length());
      const unsigned long long past = __ballot(base + upto > want);
      if (past != 0) {
        const int at = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
        const int before = __builtin_amdgcn_readlane(upto - pieces, at);
        const int gs = __builtin_amdgcn_readlane(s, at);
        const int gt = __builtin_amdgcn_readlane(t, at);
        Item it;
        it.pieces = __builtin_amdgcn_readlane(pieces, at);
        it.group = g0 + at < n_groups ? g0 + at : n_groups;
        const int64_t r0 = gs + (want - base - before) * rows;
        // (whatever starts holds, rows outside [gs, gt) are never touched)
        it.r0 = (int)(r0 < gs ? gs : r0 > gt ? gt : r0);
        it.r1 = gt - it.r0 > rows ? it.r0 + rows : gt;
        return it;
      }
      base += sum;
    }
    return Item{-1, 0, 0, 0};
  }
};

// Blocks are dealt to the eight XCDs in turn; each XCD gets a contiguous part
// of the work list, so that the tiles that share rows or a weight panel meet in
// one L2.  -> position in the list of `total`, or -1.  (A list longer than the
// 2^24 blocks of a launch comes from starts that are not ascending.)
__device__ __forceinline__ int xcd_position(int block, int64_t total64) {
  const unsigned total = total64 < (1 << 30) ? (unsigned)total64 : 1u << 30;
  const unsigned x = block & 7, per = total >> 3, extra = total & 7;
  const unsigned mine = per + (x < extra);
  if ((unsigned)block >> 3 >= mine) return -1;
  return (int)(x * per + (x < extra ? x : extra) + ((unsigned)block >> 3));
}

// 16 bytes of a row from column j on, of n_j columns; whole: rows are whole
// aligned chunks; past: see store16
template <typename O>
__device__ __forceinline__ void store_chunk(O* __restrict__ p, int64_t j,
                                            int64_t n_j, bool whole, bool past,
                                            const Pack16<O>& v) {
  if (whole) {
    if (j >= n_j) return;
    Pack16<O>* to = reinterpret_cast<Pack16<O>*>(p + j);
    if (past) store16<true>(to, v);
    else store16<false>(to, v);
  } else {
#pragma unroll
    for (int e = 0; e < Pack16<O>::N; ++e)
      if (j + e < n_j) p[j + e] = v.v[e];
  }
}
template <typename O>
__device__ __forceinline__ bool whole_rows(const O* p, int64_t n_j) {
  return n_j % Pack16<O>::N == 0 && ((uintptr_t)p & 15) == 0;
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
  __shared__ __align__(16) char smem[Tile::LDS];
  PieceList<true> list(starts, n_groups, m, Tile::BI, 0);
  const int64_t total = list.count(list.length()) * j_tiles;
  const int at = xcd_position(blockIdx.x, total);
  if (at < 0) return;
  const int64_t j0 = (int64_t)(at % j_tiles) * Tile::BJ;
  const Item it = list.find(at / j_tiles, list.length() <= 64);
  if (it.group < 0 || it.r0 >= it.r1) return;
  const bool live = it.group < n_groups;
  const bool whole = whole_rows(y, n_j);
  const bool past = m * n_j * (int64_t)sizeof(T) > kCachedBytes;
  const int64_t mine = j0 + threadIdx.x;
  const float add = live && bias != nullptr && threadIdx.x < Tile::BJ &&
                            mine < n_j
                        ? to_f32(bias[(int64_t)it.group * n_j + mine])
                        : 0.f;
  Tile tile;
  const T* wg = w + (int64_t)(live ? it.group : 0) * n_k * n_j;
  tile.run(smem, x, x_stride, it.r0, it.r1, wg, SB ? n_j : n_k, j0, n_j,
           live ? n_k : 0, false);
  tile.template emit<T>(
      smem, add,
      [&](f32x4 v, f32x4 b) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] += b[e];
          if (relu && v[e] <= 0.f) v[e] = 0.f;
        }
        return v;
      },
      [&](int i, int j, const Pack16<T>& v) {
        const int row = it.r0 + i;
        if (row < it.r1)
          store_chunk(y + (int64_t)row * n_j, j0 + j, n_j, whole, past, v);
      });
}

// One 16 x 16 product of fragments of 16 bytes a lane: index l & 15, the
// 16-byte piece l >> 4 of 64.  C: register r of lane l is j = 4 (l >> 4) + r,
// i = l & 15.
__device__ __forceinline__ void mma16(const Pack16<__bf16>& b,
                                      const Pack16<__bf16>& a, f32x4& c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
      __builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), c, 0, 0, 0);
}
__device__ __forceinline__ void mma16(const Pack16<_Float16>& b,
                                      const Pack16<_Float16>& a, f32x4& c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_f16(
      __builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), c, 0, 0, 0);
}
__device__ __forceinline__ void mma16(const Pack16<float>& b,
                                      const Pack16<float>& a, f32x4& c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = XRD_MFMA4(b.v[e], a.v[e], c);
}

// y for groups of few rows, where reading the weights is all there is: 16 rows
// x 16 columns a block, no staging - a weight is used once, so its fragments go
// from memory to registers (64 bytes of 16 weight rows an instruction), DEPTH
// of them in flight.  The four waves take every fourth 128 bytes of the
// contraction; their sums meet in LDS.
constexpr int kFew = 16;
template <typename T>
__global__ __launch_bounds__(256) void grouped_few_kernel(
    int64_t m, int n_groups, int n_k, int n_j, const T* __restrict__ x,
    int64_t x_stride, const T* __restrict__ w, const T* __restrict__ bias,
    const int* __restrict__ starts, int relu, int j_tiles,
    T* __restrict__ y) {
  constexpr int PER = Pack16<T>::N, LINE = 8 * PER;    // 128 bytes
  constexpr int LINES = 2, DEPTH = 2 * LINES;          // a wave and turn
  __shared__ f32x4 part[3][64];
  const int64_t j0 = (int64_t)(blockIdx.x % j_tiles) * kFew;
  PieceList<true> list(starts, n_groups, m, kFew, 0);
  const Item it = list.find(blockIdx.x / j_tiles, false);
  if (it.group < 0 || it.r0 >= it.r1) return;
  const bool live = it.group < n_groups;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int q = lane >> 4;
  const int row = it.r0 + (lane & 15);
  const T* px = x + (int64_t)(row < it.r1 ? row : it.r1 - 1) * x_stride;
  const int64_t col = j0 + (lane & 15);
  const T* pw = w + ((int64_t)(live ? it.group : 0) * n_j +
                     (col < n_j ? col : n_j - 1)) * n_k;
  f32x4 add = {};
  if (live && bias != nullptr && wave == 0)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (j0 + 4 * q + e < n_j)
        add[e] = to_f32(bias[(int64_t)it.group * n_j + j0 + 4 * q + e]);
  f32x4 acc = {};
  if (live)
    for (int64_t k0 = (int64_t)wave * LINE; k0 < n_k; k0 += 4 * LINES * LINE) {
      Pack16<T> fa[DEPTH], fb[DEPTH];
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        const int64_t k = k0 + (d / 2) * 4 * LINE + (d % 2 * 4 + q) * PER;
        const bool in = k < n_k;
        fb[d] = in ? *reinterpret_cast<const Pack16<T>*>(pw + k) : Pack16<T>{};
        fa[d] = in ? *reinterpret_cast<const Pack16<T>*>(px + k) : Pack16<T>{};
      }
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) mma16(fb[d], fa[d], acc);
    }
  if (wave > 0) part[wave - 1][lane] = acc;
  __syncthreads();
  if (wave > 0 || row >= it.r1) return;
  acc = ((acc + part[0][lane]) + (part[1][lane] + part[2][lane])) + add;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t j = j0 + 4 * q + e;
    if (relu && acc[e] <= 0.f) acc[e] = 0.f;
    if (j < n_j) y[(int64_t)row * n_j + j] = from_f32<T>(acc[e]);
  }
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
  __shared__ __align__(16) char smem[Tile::LDS];
  // pieces differ in length, so every XCD gets an eighth of each piece's tiles
  // (neighbours, which share operand panels); pieces of fewer tiles go round
  const int tiles = in_tiles * out_tiles;
  const int per = (tiles + 7) / 8;
  int piece, t;
  if (tiles >= 8) {
    const int turn = blockIdx.x >> 3;
    piece = turn / per;
    t = (int)(blockIdx.x & 7) * per + turn % per;
    if (t >= tiles) return;
  } else {
    piece = blockIdx.x / tiles;
    t = blockIdx.x % tiles;
  }
  const int64_t j0 = (int64_t)(t % in_tiles) * Tile::BJ;
  const int64_t i0 = (int64_t)(t / in_tiles) * Tile::BI;
  PieceList<false> list(starts, n_groups, m, piece_rows, 1);
  const Item it = list.find(piece, false);
  if (it.group < 0) return;
  // (more pieces than the workspace holds: starts that are not ascending)
  if (it.pieces > 1 && piece >= piece_room) return;
  const bool sums = db != nullptr && j0 == 0;
  Tile tile;
  tile.run(smem, dz + (int64_t)it.r0 * dz_stride, dz_stride, i0, n_out,
           x + (int64_t)it.r0 * x_stride, x_stride, j0, n_in, it.r1 - it.r0, sums);
  const bool alone = it.pieces == 1;
  const auto as_is = [](f32x4 v, f32x4) { return v; };
  if (alone) {
    T* out = dw + (int64_t)it.group * n_out * n_in;
    const bool whole = whole_rows(dw, n_in);
    const bool past = (int64_t)n_groups * n_out * n_in * (int64_t)sizeof(T) >
                      kCachedBytes;
    tile.template emit<T>(smem, 0.f, as_is, [&](int i, int j, const Pack16<T>& v) {
      if (i0 + i < n_out)
        store_chunk(out + (i0 + i) * n_in, j0 + j, n_in, whole, past, v);
    });
  } else {
    float* out = part_w + (int64_t)piece * n_out * n_in;
    const bool whole = whole_rows(out, n_in);
    tile.template emit<float>(
        smem, 0.f, as_is, [&](int i, int j, const Pack16<float>& v) {
          if (i0 + i < n_out)
            store_chunk(out + (i0 + i) * n_in, j0 + j, n_in, whole, false, v);
        });
  }
  if (sums)
    tile.each_sum([&](int i, float v) {
      if (i0 + i >= n_out) return;
      if (alone) db[(int64_t)it.group * n_out + i0 + i] = from_f32<T>(v);
      else part_b[(int64_t)piece * n_out + i0 + i] = v;
    });
}

// Sums of the pieces of every group that has several: a block takes 64 chunks
// of four columns, its four waves a quarter of the pieces each; the quarters
// meet in LDS.  The order is fixed.  rows: n_w / 4 chunks of dW, then db.
template <typename T>
__global__ __launch_bounds__(256) void grouped_join_kernel(
    int64_t m, int n_groups, int64_t n_w, int n_out, int piece_rows,
    int64_t piece_room, int blocks_a_group, const int* __restrict__ starts,
    T* __restrict__ dw, T* __restrict__ db, const float* __restrict__ part_w,
    const float* __restrict__ part_b) {
  __shared__ f32x4 quarter[3][64];
  const int g = blockIdx.x / blocks_a_group;
  int s, t;
  group_rows(starts, n_groups, (int)m, g, s, t);
  const int pieces = pieces_of(s, t, piece_rows, true, 1);
  if (pieces == 1) return;
  PieceList<false> list(starts, n_groups, m, piece_rows, 1);
  const int64_t first = list.count(g);
  if (first + pieces > piece_room) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t w_blocks = (n_w + 255) / 256;
  const int64_t blk = blockIdx.x % blocks_a_group;
  const bool is_b = blk >= w_blocks;
  const int64_t n = is_b ? n_out : n_w;
  const float* part = (is_b ? part_b : part_w) + first * n;
  T* out = (is_b ? db : dw) + g * n;
  const int64_t e = ((is_b ? blk - w_blocks : blk) * 64 + lane) * 4;
  const int per = (pieces + 3) / 4;
  const int p0 = wave * per, p1 = p0 + per < pieces ? p0 + per : pieces;
  f32x4 acc = {};
  if (e + 4 <= n && n % 4 == 0) {
#pragma unroll 8
    for (int p = p0; p < p1; ++p)
      acc += *reinterpret_cast<const f32x4*>(part + p * n + e);
  } else {
    for (int p = p0; p < p1; ++p)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (e + c < n) acc[c] += part[p * n + e + c];
  }
  if (wave > 0) quarter[wave - 1][lane] = acc;
  __syncthreads();
  if (wave > 0) return;
  acc = (acc + quarter[0][lane]) + (quarter[1][lane] + quarter[2][lane]);
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (e + c < n) out[e + c] = from_f32<T>(acc[c]);
}

// dz = dy where the ReLU let the value pass (a NaN passes, as it did forward).
// One thread N columns of one row; a block 256 of them, row by row.
template <typename T, int N>
__global__ __launch_bounds__(256) void grouped_relu_grad_kernel(
    int64_t m, int cols, int row_blocks, const T* __restrict__ y,
    const T* __restrict__ dy, int64_t dy_stride, T* __restrict__ dz) {
  const int c = (int)(blockIdx.x % row_blocks) * 256 + threadIdx.x;
  if (c >= cols) return;
  for (int64_t r = blockIdx.x / row_blocks; r < m;
       r += gridDim.x / row_blocks) {
    const Vec<T, N> v =
        *reinterpret_cast<const Vec<T, N>*>(y + (r * cols + c) * N);
    Vec<T, N> g =
        *reinterpret_cast<const Vec<T, N>*>(dy + r * dy_stride + c * N);
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (to_f32(v.v[e]) <= 0.f) g.v[e] = (T)0.f;
    *reinterpret_cast<Vec<T, N>*>(dz + (r * cols + c) * N) = g;
  }
}

constexpr int64_t kMaxBlocks = (1ll << 24) - 1;   // 2^32 threads a launch

// distances between rows that the tiles' 32-bit offsets do not hold
bool far_rows(int64_t m, int64_t stride) {
  return m > 1 && stride > kMaxStride;
}
bool bad_shape(int dtype, int64_t m, int n_groups, int n_in, int n_out) {
  return element_size(dtype) == 0 || m < 0 || n_groups < 1 || n_in < 1 ||
         n_out < 1;
}
// (every block scans the list of groups, 64 at a time, so the groups' number
// counts twice; 65536 are half a millisecond a block)
bool too_large(int64_t m, int n_groups, int n_in, int n_out) {
  return m > (1ll << 31) - 1024 || n_groups > (1 << 16) || n_in > (1 << 20) ||
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
                     dim3(Tile::THREADS), 0, st, m, n_groups, n_k, n_j,
                     (const T*)x, x_stride, (const T*)w, (const T*)bias,
                     starts, relu, (int)j_tiles, (T*)y);
  return check_launch("xrd_grouped");
}

template <typename T>
int launch_few(int64_t m, int n_groups, int n_k, int n_j, const void* x,
               int64_t x_stride, const void* w, const void* bias,
               const int32_t* starts, int relu, void* y, hipStream_t st) {
  const int64_t j_tiles = ceil_div(n_j, kFew);
  const int64_t blocks = (m / kFew + n_groups + 2) * j_tiles;
  if (blocks > kMaxBlocks) return XRD_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((grouped_few_kernel<T>), dim3((unsigned)blocks),
                     dim3(256), 0, st, m, n_groups, n_k, n_j, (const T*)x,
                     x_stride, (const T*)w, (const T*)bias, starts, relu,
                     (int)j_tiles, (T*)y);
  return check_launch("xrd_grouped_fwd");
}

// Tiles: measured on gfx950 (m rows, groups, in x out; us forward).
//   f32    64 x 64: more blocks and less padding than 128 x 128, and the matrix
//          unit is as busy (32768, 8, 512 x 512: 155 and 183; 49152, 8,
//          128 x 128: 25 and 31; 20011, 5, 144 x 129: 19 and 36)
//   16-bit 64 x 64 for up to 96 rows a group (4096, 64, 1024 x 1024: 36; 40 with
//          64 x 128); from 1024 tiles of 128 x 128 on the large tiles, else 64 x
//          128 (8192, 8, 1024 x 1024: 31; 39 with 128 x 256).  Large tiles are
//          128 x 256 with three buffers for the product (16384, 16, 2048 x 2048,
//          weights cold: 175; 187 with 128 x 128, 187 with 256 x 256, 229 with
//          64 x 128) and 128 x 128, two blocks a CU, for the input gradient,
//          whose right operand is turned as it is read (warm: 156; 162 with 128 x 256)
//   few rows a group: grouped_few_kernel (8, 16, 1024 x 2048: 9; 13 with 64 x 64;
//          f32 256, 16, 512 x 512: 13 and 19; bf16 128, 16, 1024 x 2048: 19, 18)
template <typename T, bool SB>
int launch_rows(int64_t m, int n_groups, int n_k, int n_j, const void* x,
                int64_t x_stride, const void* w, const void* bias,
                const int32_t* starts, int relu, void* y, hipStream_t st) {
  const bool wx = chunked<T>(x, x_stride, n_k);
  const bool ww = chunked<T>(w, 0, SB ? n_j : n_k);
  const int64_t mean = m / n_groups;     // rows a group, were all used
#define XRD_ROWS(...)                                                       \
  return launch_rows_tile<MatrixTile<T, false, SB, __VA_ARGS__, false>, SB>( \
      m, n_groups, n_k, n_j, x, x_stride, w, bias, starts, relu, y, st)
  if constexpr (!SB)
    if (wx && ww && mean <= (sizeof(T) == 4 ? 16 : 4) &&
        (m / kFew + n_groups + 2) * ceil_div(n_j, kFew) <= kMaxBlocks)
      return launch_few<T>(m, n_groups, n_k, n_j, x, x_stride, w, bias, starts,
                           relu, y, st);
  if constexpr (sizeof(T) == 4) {
    if (wx && ww) XRD_ROWS(16, 16, 64, 64, 2, 2, 64, 2);
    if (wx) XRD_ROWS(16, 4, 64, 64, 2, 2, 64, 2);
    if (ww) XRD_ROWS(4, 16, 64, 64, 2, 2, 64, 2);
    XRD_ROWS(4, 4, 64, 64, 2, 2, 64, 2);
  } else {
    if (!wx || !ww) XRD_ROWS(0, 0, 64, 64, 2, 2, 128, 2);
    if (mean <= 96) XRD_ROWS(16, 16, 64, 64, 2, 2, 128, 2);
    if ((m / 128 + n_groups) * ceil_div(n_j, 128) >= 1024)
      XRD_ROWS(16, 16, 128, SB ? 128 : 256, 2, SB ? 2 : 4, 128, SB ? 2 : 3);
    XRD_ROWS(16, 16, 64, 128, 2, 2, 128, 2);
  }
#undef XRD_ROWS
}

// Rows a piece of the weight gradient holds.  One piece a group where groups
// and tiles alone fill the chip (no partial sums to write and read back), else
// as many pieces as make two blocks a CU (f32) or four (16-bit, whose blocks are
// shorter), of at least 128 (256) rows.  f32, 20011 rows of 5 groups, 144 x 129:
// 37 us with 512 blocks, 43 with 1024; 49152 of 8, 128 x 128: 33, 32 (256: 40).
int weight_tile(int dtype, int64_t m, int n_groups, int n_in, int n_out) {
  if (dtype == XRD_F32)
    return m / n_groups >= 1024 && n_in > 128 && n_out > 128 ? 128 : 64;
  return ceil_div(n_in, 256) * ceil_div(n_out, 256) * n_groups >= 512 ? 256
                                                                      : 128;
}
int piece_rows_of(int dtype, int64_t m, int n_groups, int n_in, int n_out) {
  const int tile = weight_tile(dtype, m, n_groups, n_in, n_out);
  const int64_t tiles = ceil_div(n_in, tile) * ceil_div(n_out, tile);
  if (tiles * n_groups >= 512) return 1 << 30;
  const bool f32 = dtype == XRD_F32;
  const int64_t pieces = ceil_div(f32 ? 512 : 1024, tiles);
  int64_t rows = ceil_div(ceil_div(m, pieces), 64) * 64;
  if (rows < (f32 ? 128 : 256)) rows = f32 ? 128 : 256;
  return (int)(rows > (1 << 30) ? (1 << 30) : rows);
}
// pieces of all groups at most (0: every group is one piece)
int64_t piece_bound(int dtype, int64_t m, int n_groups, int n_in, int n_out) {
  const int rows = piece_rows_of(dtype, m, n_groups, n_in, n_out);
  return m <= rows ? 0 : m / rows + n_groups;
}

template <class Tile>
int launch_weights(int dtype, int64_t m, int n_groups, int n_in, int n_out, const void* x,
                   int64_t x_stride, const void* dz, int64_t dz_stride,
                   const int32_t* starts, void* dw, void* db, float* ws,
                   hipStream_t st) {
  using T = typename Tile::T;
  const int64_t it = ceil_div(n_in, Tile::BJ), ot = ceil_div(n_out, Tile::BI);
  const int rows = piece_rows_of(dtype, m, n_groups, n_in, n_out);
  const int64_t bound = piece_bound(dtype, m, n_groups, n_in, n_out);
  const int64_t tiles = it * ot;
  const int64_t blocks = (m / rows + n_groups) *
                         (tiles >= 8 ? ceil_div(tiles, 8) * 8 : tiles);
  if (blocks > kMaxBlocks) return XRD_ERR_UNSUPPORTED;
  const int64_t n_w = (int64_t)n_out * n_in;
  float* part_b = ws + bound * n_w;
  hipLaunchKernelGGL((grouped_weights_kernel<Tile>), dim3((unsigned)blocks),
                     dim3(Tile::THREADS), 0, st, m, n_groups, n_in,
                     n_out, rows, bound, (const T*)x, x_stride, (const T*)dz,
                     dz_stride, starts, (int)it, (int)ot, (T*)dw, (T*)db, ws,
                     part_b);
  if (bound > 0) {
    const int64_t per =
        ceil_div(n_w, 256) + (db != nullptr ? ceil_div(n_out, 256) : 0);
    if (per * n_groups > kMaxBlocks) return XRD_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((grouped_join_kernel<T>), dim3((unsigned)(per * n_groups)),
                       dim3(256), 0, st, m, n_groups, n_w, n_out, rows,
                       bound, (int)per, starts, (T*)dw, (T*)db, ws, part_b);
  }
  return check_launch("xrd_grouped_bwd_w");
}

template <typename T, bool ONES>
int launch_weights_of(int dtype, int64_t m, int n_groups, int n_in, int n_out,
                      const void* x, int64_t x_stride, const void* dz,
                      int64_t dz_stride, const int32_t* starts, void* dw,
                      void* db, float* ws, hipStream_t st) {
  const bool wx = chunked<T>(x, x_stride, n_in);
  const bool wz = chunked<T>(dz, dz_stride, n_out);
#define XRD_WEIGHTS(...)                                                      \
  return launch_weights<MatrixTile<T, true, true, __VA_ARGS__, ONES>>(        \
      dtype, m, n_groups, n_in, n_out, x, x_stride, dz, dz_stride, starts, dw, \
      db, ws, st)
  const int tile = weight_tile(dtype, m, n_groups, n_in, n_out);
  if constexpr (sizeof(T) == 4) {
    if (wx && wz && tile == 128) XRD_WEIGHTS(16, 16, 128, 128, 2, 2, 128, 2);
    if (wx && wz) XRD_WEIGHTS(16, 16, 64, 64, 2, 2, 64, 2);
    if (wx) XRD_WEIGHTS(4, 16, 64, 64, 2, 2, 64, 2);
    if (wz) XRD_WEIGHTS(16, 4, 64, 64, 2, 2, 64, 2);
    XRD_WEIGHTS(4, 4, 64, 64, 2, 2, 64, 2);
  } else {
    if (!wx || !wz) XRD_WEIGHTS(0, 0, 64, 64, 2, 2, 128, 2);
    // (with the bias sums beside its 128 accumulators a lane would spill)
    if constexpr (!ONES)
      if (tile == 256) XRD_WEIGHTS(16, 16, 256, 256, 2, 4, 128, 2);
    XRD_WEIGHTS(16, 16, 128, 128, 2, 2, 128, 2);
  }
#undef XRD_WEIGHTS
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
  if (too_large(m, n_groups, n_in, n_out) || far_rows(m, x_stride))
    return XRD_ERR_UNSUPPORTED;
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
  if (too_large(m, n_groups, n_in, n_out) || far_rows(m, dz_stride))
    return XRD_ERR_UNSUPPORTED;
  if (m == 0) return XRD_OK;
  if (dz == nullptr || dx == nullptr) return XRD_ERR_ARG;
  XRD_BY_DTYPE(dtype, return (launch_rows<T, true>(
                          m, n_groups, n_out, n_in, dz, dz_stride, weight,
                          nullptr, starts, 0, dx, (hipStream_t)stream)));
}

int64_t xrd_grouped_ws_floats(int dtype, int64_t m, int n_groups, int n_in,
                              int n_out) {
  if (bad_shape(dtype, m, n_groups, n_in, n_out) ||
      too_large(m, n_groups, n_in, n_out))
    return -1;
  return piece_bound(dtype, m, n_groups, n_in, n_out) *
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
  const int64_t need = xrd_grouped_ws_floats(dtype, m, n_groups, n_in, n_out);
  if (need < 0 || far_rows(m, x_stride) || far_rows(m, dz_stride))
    return XRD_ERR_UNSUPPORTED;
  if (need > 0 && ws == nullptr) return XRD_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  XRD_BY_DTYPE(dtype, {
    if (dbias != nullptr)
      return (launch_weights_of<T, true>(dtype, m, n_groups, n_in, n_out, x,
                                         x_stride, dz, dz_stride, starts,
                                         dweight, dbias, ws, st));
    return (launch_weights_of<T, false>(dtype, m, n_groups, n_in, n_out, x,
                                        x_stride, dz, dz_stride, starts,
                                        dweight, nullptr, ws, st));
  });
}

int xrd_grouped_relu_grad(int dtype, int64_t m, int n_out, const void* y,
                          const void* dy, int64_t dy_stride, void* dz,
                          void* stream) {
  if (bad_shape(dtype, m, 1, 1, n_out) || dy_stride < 0) return XRD_ERR_ARG;
  if (m == 0) return XRD_OK;
  if (y == nullptr || dy == nullptr || dz == nullptr) return XRD_ERR_ARG;
#define XRD_RELU(N, ROW, ROWS, STRIDE)                                      \
  do {                                                                      \
    const int64_t wide = ceil_div((ROW) / (N), 256);                        \
    const int64_t most = ceil_div(1 << 16, wide);                           \
    const int64_t blocks = wide * ((ROWS) < most ? (ROWS) : most);          \
    hipLaunchKernelGGL((grouped_relu_grad_kernel<T, N>),                    \
                       dim3((unsigned)blocks), dim3(256), 0,                \
                       (hipStream_t)stream, ROWS, (int)((ROW) / (N)),       \
                       (int)wide, (const T*)y, (const T*)dy, STRIDE, (T*)dz); \
  } while (0)
  XRD_BY_DTYPE(dtype, {
    constexpr int W = 16 / (int)sizeof(T);
    const bool whole = chunked<T>(dy, dy_stride, n_out) && aligned16(y) &&
                       aligned16(dz);
    // rows one behind the other make one row, cut into lines of 2048 chunks
    const int64_t all = m * n_out;
    const int64_t line = 2048 * W;
    if (whole && dy_stride == n_out && all % line == 0)
      XRD_RELU(W, line, all / line, line);
    else if (whole)
      XRD_RELU(W, n_out, m, dy_stride);
    else
      XRD_RELU(1, n_out, m, dy_stride);
  });
#undef XRD_RELU
  return check_launch("xrd_grouped_relu_grad");
}

}  // extern "C"
