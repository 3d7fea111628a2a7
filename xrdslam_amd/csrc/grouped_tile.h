// One C tile of a ragged product on the matrix unit (used by grouped.hip):
// C[i][j] = sum_k A(i, k) B(j, k), both operands streamed through LDS.
//
// Geometry is in bytes, so one code serves 16- and 32-bit elements: a step of
// the contraction is STEP = 64 or 128 bytes of an index; a tile of 128 or 256
// indices is staged by loads that go from memory to LDS directly
// (global_load_lds_dwordx4: 1 KB a wave instruction, lane l's 16 bytes land at
// base + 16 l), up to NBUF steps ahead of the one that is computed on.
//
// The landing place is fixed by the lane, so the bank swizzle is applied to
// the address a lane fetches from:
//   contraction-contiguous operand: rows of STEP bytes, chunk c of row i lies at
//     c ^ (i >> 1 & 7) (128-byte rows) or c ^ (i >> 2 & 3) (64): the 16 lanes
//     that read 16 bytes each in a cycle (rows i .. i + 15) then fall into 16
//     different places of the 64 banks;
//   index-contiguous operand ([k][i] in memory): rows of one k, for 16-bit
//     elements chunk c of row k at c ^ 4 (k & 3) (c ^ 4 (k >> 1 & 1) in tiles of
//     64 indices, whose rows fill half the banks), read transposed four rows at
//     a time (ds_read_b64_tr_b16): the four rows of a lane group fall into
//     different banks.
//
// The matrix instruction's row operand is B, its column operand A: a lane then
// holds four consecutive j of one i and stores them at once.
#pragma once
#include <type_traits>

#include "element.h"

namespace xrd {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// what a lane at the end of the contraction fetches in place of data
__device__ __attribute__((aligned(16))) uint32_t g_zero16[4];

// UNIT (16 or 4) bytes a lane -> LDS base + UNIT lane, from a wave-uniform base
// plus the lane's 32-bit offset: the base is advanced by scalar additions, so a
// step's fetches cost no vector instruction (f32 products share the vector
// lanes).  The wait state between the write of m0 and its use is the one the
// ISA asks for.
template <int UNIT>
__device__ __forceinline__ void lds_fetch(const void* base, uint32_t off,
                                          uint32_t lds_base) {
  const uint32_t at = __builtin_amdgcn_readfirstlane(lds_base);
  if constexpr (UNIT == 16)
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
        :
        : "s"(at), "v"(off), "s"(base)
        : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                 :
                 : "s"(at), "v"(off), "s"(base)
                 : "memory");
}
// the same with an address of its own for every lane
template <int UNIT>
__device__ __forceinline__ void lds_fetch_at(const void* p,
                                             uint32_t lds_base) {
  const uint32_t at = __builtin_amdgcn_readfirstlane(lds_base);
  if constexpr (UNIT == 16)
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
        :
        : "s"(at), "v"(p)
        : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
                 :
                 : "s"(at), "v"(p)
                 : "memory");
}
// a pointer that is the same in all lanes, in scalar registers.  (readfirstlane
// gives an int: without the casts a low word of 2^31 and more would spill its
// sign into the high one.)
template <typename P>
__device__ __forceinline__ P* uniform(P* p) {
  const uint64_t v = (uint64_t)p;
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32));
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
  return (P*)((uint64_t)hi << 32 | lo);
}
// rows of a tile are at most this many elements apart: 256 of them stay within
// the 32-bit offsets
constexpr int64_t kMaxStride = 1 << 20;

template <int PENDING>
__device__ __forceinline__ void fetched() {
  static_assert(PENDING < 64, "six bits");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PENDING) : "memory");
}

// acc += B-fragment x A-fragment, 16 bytes a lane each: index l & 31, the
// 16-byte piece l >> 5 of 32.  C: register r of lane l is
// j = (r & 3) + 8 (r >> 2) + 4 (l >> 5), i = l & 31.
__device__ __forceinline__ void mma32(const Pack16<__bf16>& b,
                                      const Pack16<__bf16>& a, f32x16& c) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
      __builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), c, 0, 0, 0);
}
__device__ __forceinline__ void mma32(const Pack16<_Float16>& b,
                                      const Pack16<_Float16>& a, f32x16& c) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_f16(
      __builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), c, 0, 0, 0);
}
// step e takes element e of both halves: k runs in another order than in
// memory, the same one for both operands
__device__ __forceinline__ void mma32(const Pack16<float>& b,
                                      const Pack16<float>& a, f32x16& c) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(b.v[e], a.v[e], c, 0, 0, 0);
}

// where chunk c of row i of a contraction-contiguous tile lies in its row
template <int STEP>
__device__ __forceinline__ constexpr int place_of(int i, int c) {
  return STEP == 128 ? c ^ (i >> 1 & 7) : c ^ (i >> 2 & 3);
}

// what chunk numbers of row k of an index-contiguous tile are xored with
template <typename T, int EXT>
__device__ __forceinline__ constexpr int swap_of(int k) {
  return sizeof(T) != 2 ? 0 : EXT == 64 ? 4 * (k >> 1 & 1) : 4 * (k & 3);
}

// EXT indices of one operand, fetched by NW waves, UNIT bytes a lane: 16 where
// rows are whole aligned 16-byte chunks, 4 for f32 rows of any alignment.
template <typename T, bool SWAP, int EXT, int NW, int STEP, int UNIT>
struct TileStage {
  static constexpr int KS = STEP / (int)sizeof(T);           // steps of k
  static constexpr int SPAN = 64 * UNIT;                     // bytes a fetch
  static constexpr int N = EXT * STEP / SPAN / NW;           // fetches a wave
  static constexpr int PER = UNIT / (int)sizeof(T);          // elements a lane
  // lanes along a row of the tile (an index's step, SWAP: a step's indices)
  static constexpr int ROWB = SWAP ? EXT * (int)sizeof(T) : STEP;
  static constexpr int ACROSS = ROWB / UNIT;
  static_assert(N * SPAN * NW == EXT * STEP && N >= 1, "whole fetches");
  static_assert(ROWB % SPAN == 0 || SPAN % ROWB == 0, "rows and fetches");
  const T* base;         // wave-uniform: index 0, k of the next step
  uint32_t off[N];       // bytes of this lane's element from there
  int64_t step;
  int lane_, wave_;

  // byte of the tile that fetch t of this lane fills
  __device__ __forceinline__ int place(int t) const {
    return (wave_ * N + t) * SPAN + lane_ * UNIT;
  }
  // element this lane fetches: row of the tile and column in it
  __device__ __forceinline__ int row(int t) const { return place(t) / ROWB; }
  __device__ __forceinline__ int col(int t) const {
    const int r = row(t), b = place(t) % ROWB;
    const int c = SWAP ? b / 16 ^ swap_of<T, EXT>(r)
                       : place_of<STEP>(r, b / 16);
    return (c * 16 + b % 16) / (int)sizeof(T);
  }
  // indices i0.. of the operand (those past n_i fetch a valid one instead)
  __device__ __forceinline__ void start(const T* p, int64_t stride,
                                        int64_t i0, int64_t n_i, int wave,
                                        int lane) {
    lane_ = lane, wave_ = wave;
    step = SWAP ? KS * stride : KS;
    base = uniform(SWAP ? p + i0 : p + i0 * stride);
    const uint32_t st = (uint32_t)stride;
    const int left = (int)(n_i - i0 < EXT ? n_i - i0 : EXT);   // >= 1
#pragma unroll
    for (int t = 0; t < N; ++t) {
      int i = SWAP ? col(t) : row(t);
      i = i < left ? i : SWAP ? 0 : left - 1;
      const uint32_t k = SWAP ? row(t) : col(t);
      off[t] = (SWAP ? k * st + i : i * st + k) * (uint32_t)sizeof(T);
    }
  }
  // the next step of the contraction, at k0, into LDS at `lds`
  __device__ __forceinline__ void fetch(uint32_t lds, int k0, int n_k) {
    const uint32_t at = lds + (uint32_t)(wave_ * N) * SPAN;
    if (k0 + KS <= n_k) {
#pragma unroll
      for (int t = 0; t < N; ++t) lds_fetch<UNIT>(base, off[t], at + t * SPAN);
    } else {
#pragma unroll
      for (int t = 0; t < N; ++t) {
        const int k = k0 + (SWAP ? row(t) : col(t));
        const void* q = k < n_k ? (const void*)((const char*)base + off[t])
                                : (const void*)g_zero16;
        lds_fetch_at<UNIT>(q, at + t * SPAN);
      }
    }
    base += step;
  }
};

// The same tile layout filled through registers, element by element: 16-bit
// operands whose rows are not made of whole aligned 16-byte chunks.  load() brings the
// next step into registers while the current one is computed on, store() puts
// it into the other buffer.
template <typename T, bool SWAP, int EXT, int NW, int STEP>
struct TileStageAny {
  static constexpr int PER = Pack16<T>::N;
  static constexpr int CHUNKS = EXT * (int)sizeof(T) / 16;
  static constexpr int C = STEP / 16;
  static constexpr int N = EXT * C / (64 * NW);     // chunks a lane
  const T* base;
  int64_t stride, i0, n_i;
  Pack16<T> r[N];

  __device__ __forceinline__ void start(const T* b, int64_t s, int64_t first,
                                        int64_t end) {
    base = b, stride = s, i0 = first, n_i = end;
  }
  // chunk number of lane-wide chunk t: its place in the tile is 16 times that
  __device__ __forceinline__ int place(int t) const {
    return t * 64 * NW + (int)threadIdx.x;
  }
  __device__ __forceinline__ void load(int k0, int n_k) {
#pragma unroll
    for (int t = 0; t < N; ++t) {
      const int at = place(t);
      if constexpr (!SWAP) {
        const int row = at / C, c = place_of<STEP>(row, at % C);
        int64_t i = i0 + row;
        i = i < n_i ? i : n_i - 1;
        const int k = k0 + c * PER;
        const T* q = base + i * stride + k;
#pragma unroll
        for (int e = 0; e < PER; ++e)
          r[t].v[e] = k + e < n_k ? q[e] : (T)0.f;
      } else {
        const int row = at / CHUNKS;
        const int c = at % CHUNKS ^ swap_of<T, EXT>(row);
        const int k = k0 + row;
        const int64_t i = i0 + c * PER;
        const T* q = base + (int64_t)k * stride + i;
#pragma unroll
        for (int e = 0; e < PER; ++e)
          r[t].v[e] = k < n_k && i + e < n_i ? q[e] : (T)0.f;
      }
    }
  }
  __device__ __forceinline__ void store(char* tile) const {
#pragma unroll
    for (int t = 0; t < N; ++t)
      *reinterpret_cast<Pack16<T>*>(tile + place(t) * 16) = r[t];
  }
};

// fragment of 32 indices i.., piece kk (32 bytes) of the step
template <typename T, bool SWAP, int EXT, int STEP>
__device__ __forceinline__ Pack16<T> fragment(const char* tile, int i, int kk,
                                              int lane) {
  const int q = lane >> 5;
  if constexpr (!SWAP) {
    return *reinterpret_cast<const Pack16<T>*>(
        tile + (i + (lane & 31)) * STEP +
        (place_of<STEP>(lane & 31, kk * 2 + q) << 4));
  } else if constexpr (sizeof(T) == 2) {
    const int t = lane & 15;
    const int col = (i + (lane & 16)) * 2 + (t & 3) * 8;      // bytes
    const char* row = tile + (kk * 16 + q * 8 + (t >> 2)) * (EXT * 2) +
                      (col ^ (swap_of<T, EXT>(t >> 2) << 4));
    struct Two {
      s16x4 v[2];
    } r;
    r.v[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(row));
    r.v[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(row + 4 * EXT * 2));
    return __builtin_bit_cast(Pack16<T>, r);
  } else {
    Pack16<T> r;
    const char* row =
        tile + (kk * 8 + q * 4) * (EXT * 4) + (i + (lane & 31)) * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      r.v[e] = *reinterpret_cast<const T*>(row + e * (EXT * 4));
    return r;
  }
}

// A tile of BI x BJ by WI x WJ waves.  UA, UB: 16 or 4 bytes a fetch and lane of
// either operand (see TileStage), both 0: through registers.  ONES: also the sums of A over the
// contraction: for 16-bit elements a product with a column of ones, for f32,
// whose products take 16 times as long as the four additions, additions.
template <typename T_, bool SA, bool SB, int UA, int UB, int BI_, int BJ_,
          int WI, int WJ, int STEP, int NBUF, bool ONES>
struct MatrixTile {
  using T = T_;
  static constexpr int BI = BI_, BJ = BJ_;
  static constexpr int NW = WI * WJ, THREADS = 64 * NW;
  static constexpr int TI = BI / WI / 32, TJ = BJ / WJ / 32;
  static constexpr int BUF = (BI + BJ) * STEP;
  static constexpr int EMIT = NW * 32 * (BJ / WJ * 4 + 16) + BJ * 4;
  static constexpr int LDS = NBUF * BUF > EMIT ? NBUF * BUF : EMIT;
  static constexpr int PIECES = STEP / 32;
  static_assert((UA == 0) == (UB == 0), "both or none through registers");
  static_assert(UA != 0 || NBUF == 2, "through registers: one step ahead");
  f32x16 acc[TI][TJ];
  static constexpr bool ADDS = sizeof(T) == 4;
  typename std::conditional<ADDS, float, f32x16>::type sum[ONES ? TI : 1];

  // fragments of a piece: two sets, one read while the other is multiplied
  Pack16<T> fa[2][TI], fb[2][TJ];

  __device__ __forceinline__ void multiply(int set, bool ones) {
#pragma unroll
    for (int u = 0; u < TI; ++u)
#pragma unroll
      for (int v = 0; v < TJ; ++v) mma32(fb[set][v], fa[set][u], acc[u][v]);
    if (ONES && ones) {
      if constexpr (ADDS) {
#pragma unroll
        for (int u = 0; u < TI; ++u) {
          const Pack16<T>& f = fa[set][u];
          sum[u] += (f.v[0] + f.v[1]) + (f.v[2] + f.v[3]);
        }
      } else {
        Pack16<T> one;
#pragma unroll
        for (int e = 0; e < Pack16<T>::N; ++e) one.v[e] = (T)1.f;
#pragma unroll
        for (int u = 0; u < TI; ++u) mma32(one, fa[set][u], sum[u]);
      }
    }
  }

  // piece kk of the step staged at ta -> set kk & 1
  __device__ __forceinline__ void read(const char* ta, int kk, int lane, int wi,
                                       int wj) {
    const char* tb = ta + BI * STEP;
#pragma unroll
    for (int u = 0; u < TI; ++u)
      fa[kk & 1][u] = fragment<T, SA, BI, STEP>(ta, wi + 32 * u, kk, lane);
#pragma unroll
    for (int v = 0; v < TJ; ++v)
      fb[kk & 1][v] = fragment<T, SB, BJ, STEP>(tb, wj + 32 * v, kk, lane);
  }

  // a: base, stride, first index, end of the indices; b alike; n_k: length of
  // the contraction (0 leaves zeros); ones: fill `sum` (first wave column)
  __device__ __forceinline__ void run(char* smem, const T* a, int64_t a_stride,
                                      int64_t i0, int64_t n_i, const T* b,
                                      int64_t b_stride, int64_t j0,
                                      int64_t n_j, int n_k, bool ones) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);
#pragma unroll
    for (int u = 0; u < TI; ++u) {
#pragma unroll
      for (int v = 0; v < TJ; ++v) acc[u][v] = f32x16{};
      if (ONES) sum[u] = {};
    }
    if (n_k <= 0) return;
    constexpr int KS = STEP / (int)sizeof(T);
    const int steps = (n_k + KS - 1) / KS;
    int buf = 0;
    if constexpr (UA == 0) {
      TileStageAny<T, SA, BI, NW, STEP> sa;
      TileStageAny<T, SB, BJ, NW, STEP> sb;
      sa.start(a, a_stride, i0, n_i);
      sb.start(b, b_stride, j0, n_j);
      sa.load(0, n_k);
      sb.load(0, n_k);
      for (int s = 0; s < steps; ++s, buf ^= 1) {
        char* ta = smem + buf * BUF;
        sa.store(ta);
        sb.store(ta + BI * STEP);
        __syncthreads();
        if (s + 1 < steps) {
          sa.load((s + 1) * KS, n_k);
          sb.load((s + 1) * KS, n_k);
        }
        read(ta, 0, lane, wi, wj);
#pragma unroll
        for (int kk = 0; kk < PIECES; ++kk) {
          if (kk + 1 < PIECES) read(ta, kk + 1, lane, wi, wj);
          multiply(kk & 1, ones);
        }
      }
    } else {
      TileStage<T, SA, BI, NW, STEP, UA> sa;
      TileStage<T, SB, BJ, NW, STEP, UB> sb;
      constexpr int F = sa.N + sb.N;        // fetches a step
      sa.start(a, a_stride, i0, n_i, wave, lane);
      sb.start(b, b_stride, j0, n_j, wave, lane);
      const uint32_t lds = lds_addr((const float*)smem);
      const auto fetch = [&](int s, int to) {
        sa.fetch(lds + to * BUF, s * KS, n_k);
        sb.fetch(lds + to * BUF + BI * STEP, s * KS, n_k);
      };
#pragma unroll
      for (int s = 0; s < NBUF; ++s)
        if (s < steps) fetch(s, s);
      // fetches land in order: when no more are outstanding than were made
      // after a step's, this wave's part of that step is there; behind the
      // barrier every wave's is
      if (steps >= NBUF) fetched<(NBUF - 1) * F>();
      else fetched<0>();
      __syncthreads();
      read(smem, 0, lane, wi, wj);
      for (int s = 0; s < steps; ++s) {
        const int next = buf + 1 == NBUF ? 0 : buf + 1;
#pragma unroll
        for (int kk = 0; kk < PIECES; ++kk) {
          if (kk + 1 < PIECES) {
            read(smem + buf * BUF, kk + 1, lane, wi, wj);
          } else if (s + 1 < steps) {
            // The last piece of the step is in registers, in all waves: its
            // buffer is free for the fetches NBUF steps ahead, and the first
            // piece of the next step is read behind this one's products, so no
            // wave starts a step by waiting for the LDS.
            // (The wait is an asm with a memory clobber, which no read of the
            // LDS moves past; the builtin would let them.)
            lds_landed<0>();
            if (s + NBUF <= steps) fetched<(NBUF - 2) * F>();
            else fetched<0>();
            __syncthreads();
            read(smem + next * BUF, 0, lane, wi, wj);
            if (s + NBUF < steps) fetch(s + NBUF, buf);
          }
          multiply(kk & 1, ones);
        }
        buf = next;
      }
    }
  }

  // The tile as elements of O, row by row: prep(q, b) finishes four
  // consecutive columns in f32 (b: their columns of the row of additions that
  // thread j holds `add` of; read before the contraction, so that nothing waits
  // for it here), put(i, j, chunk) gets 16 bytes of a row.  A lane holds four
  // columns of 32 different rows, which would be stores of 8 or 16 bytes a row;
  // each wave turns 32 rows at a time round in its own corner of the LDS and
  // stores whole lines (a forward pass of 16384 x 2048 x 2048 in bf16 spends
  // 33 us around its contraction instead of 45).
  template <typename O, typename P, typename F>
  __device__ __forceinline__ void emit(char* smem, float add, P prep,
                                       F put) const {
    constexpr int COLS = BJ / WJ, ROWB = COLS * (int)sizeof(O);
    constexpr int LINE = ROWB + 16;       // rows on different banks
    constexpr int CHUNKS = ROWB / 16, PER = Pack16<O>::N;
    static_assert(NW * 32 * LINE + BJ * 4 <= LDS, "the waves' corners");
    static_assert(BJ <= THREADS, "a column a thread");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);
    char* mine = smem + wave * 32 * LINE;
    float* row = reinterpret_cast<float*>(smem + NW * 32 * LINE);
    __syncthreads();                      // the tiles have been read
    if (threadIdx.x < BJ) row[threadIdx.x] = add;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < TI; ++u) {
#pragma unroll
      for (int v = 0; v < TJ; ++v)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = 32 * v + 8 * r + 4 * (lane >> 5);
          f32x4 q;
#pragma unroll
          for (int e = 0; e < 4; ++e) q[e] = acc[u][v][4 * r + e];
          q = prep(q, *reinterpret_cast<const f32x4*>(row + wj + j));
          Vec<O, 4> o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o.v[e] = from_f32<O>(q[e]);
          *reinterpret_cast<Vec<O, 4>*>(mine + (lane & 31) * LINE +
                                        j * (int)sizeof(O)) = o;
        }
      wave_lds_sync();
#pragma unroll
      for (int t = 0; t < CHUNKS / 2; ++t) {
        const int at = t * 64 + lane;
        const int i = at / CHUNKS, c = at % CHUNKS;
        put(wi + 32 * u + i, wj + c * PER,
            *reinterpret_cast<const Pack16<O>*>(mine + i * LINE + c * 16));
      }
      wave_lds_sync();
    }
  }
  // f(i, sum) once for every i of the tile
  template <typename F>
  __device__ __forceinline__ void each_sum(F f) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (wave % WJ != 0) return;
#pragma unroll
    for (int u = 0; u < TI; ++u) {
      float v;
      if constexpr (ADDS) v = sum[u] + __shfl_xor(sum[u], 32);
      else v = sum[u][0];
      if (lane < 32) f((wave / WJ) * (BI / WI) + 32 * u + lane, v);
    }
  }
};

}  // namespace xrd
