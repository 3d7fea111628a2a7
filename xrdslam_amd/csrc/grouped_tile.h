// One C tile of a ragged product on the matrix unit (used by grouped.hip):
// C[i][j] = sum_k A(i, k) B(j, k), both operands streamed through LDS.
//
// Geometry is in bytes, so one code serves 16- and 32-bit elements: a step of
// the contraction is 128 bytes (64 or 32 elements), a tile of 64, 128 or 256
// indices is staged by loads that go from memory to LDS directly
// (global_load_lds_dwordx4: 1 KB a wave instruction, lane l's 16 bytes land at
// base + 16 l), into one of two buffers while the other one is computed on.
//
// The landing place is fixed by the lane, so the bank swizzle is applied to
// the address a lane fetches from:
//   contraction-contiguous operand: rows of 128 bytes, chunk c of row i lies at
//     c ^ (i & 7); a fragment read (16 bytes of 32 rows) touches every bank
//     group evenly;
//   index-contiguous operand ([k][i] in memory): rows of one k, for 16-bit
//     elements chunk c of row k at c ^ 4 (k & 3), read transposed four rows at
//     a time (ds_read_b64_tr_b16): the four rows of a lane group fall into
//     different banks.
//
// The matrix instruction's row operand is B, its column operand A: a lane then
// holds four consecutive j of one i and stores them at once.
#pragma once
#include "element.h"

namespace xrd {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// what a lane at the end of the contraction fetches in place of data
__device__ __attribute__((aligned(16))) uint32_t g_zero16[4];

// 16 bytes a lane -> LDS base + 16 lane; every lane with its own address.  The
// wait state between the write of m0 and its use is the one the ISA asks for.
__device__ __forceinline__ void lds_fetch16(const void* p, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(lds_base), "v"(p)
               : "memory");
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

template <typename T>
constexpr int kStepK = 128 / (int)sizeof(T);

// EXT indices of one operand, fetched by NW waves
template <typename T, bool SWAP, int EXT, int NW>
struct TileStage {
  static constexpr int BYTES = EXT * 128;
  static constexpr int N = BYTES / 1024 / NW;           // fetches a wave
  static constexpr int PER = Pack16<T>::N;
  static constexpr int CHUNKS = EXT * (int)sizeof(T) / 16;   // SWAP: a k row
  static constexpr int LINES = 64 / CHUNKS;                  // SWAP: a fetch
  static_assert(N * 1024 * NW == BYTES, "whole fetches");
  static_assert(!SWAP || (CHUNKS <= 64 && CHUNKS >= 16), "k rows in a fetch");
  const T* p[N];
  int64_t step;
  int k_of;           // first k of this lane's chunk (SWAP: of fetch 0)

  // indices i0.. of the operand (those past n_i fetch a valid one instead)
  __device__ __forceinline__ void start(const T* base, int64_t stride,
                                        int64_t i0, int64_t n_i, int wave,
                                        int lane) {
    if constexpr (!SWAP) {
      const int c = (lane & 7) ^ (lane >> 3);
      k_of = c * PER;
      step = kStepK<T>;
#pragma unroll
      for (int t = 0; t < N; ++t) {
        int64_t i = i0 + (wave * N + t) * 8 + (lane >> 3);
        i = i < n_i ? i : n_i - 1;
        p[t] = base + i * stride + k_of;
      }
    } else {
      k_of = wave * N * LINES + lane / CHUNKS;
      step = kStepK<T> * stride;
#pragma unroll
      for (int t = 0; t < N; ++t) {
        const int k = k_of + t * LINES;
        int c = lane % CHUNKS;
        if (sizeof(T) == 2) c ^= 4 * (k & 3);
        int64_t i = i0 + c * PER;
        i = i < n_i ? i : 0;
        p[t] = base + k * stride + i;
      }
    }
  }
  // the next step of the contraction (k0 .. k0 + kStepK) into LDS at `lds`
  __device__ __forceinline__ void fetch(uint32_t lds, int wave, int64_t k0,
                                        int64_t n_k) {
    const uint32_t at = lds + (uint32_t)(wave * N) * 1024u;
    if (k0 + kStepK<T> <= n_k) {
#pragma unroll
      for (int t = 0; t < N; ++t) lds_fetch16(p[t], at + t * 1024u);
    } else {
#pragma unroll
      for (int t = 0; t < N; ++t) {
        const int64_t k = k0 + k_of + (SWAP ? t * LINES : 0);
        const void* q = k < n_k ? (const void*)p[t] : (const void*)g_zero16;
        lds_fetch16(q, at + t * 1024u);
      }
    }
#pragma unroll
    for (int t = 0; t < N; ++t) p[t] += step;
  }
};

// The same tile layout filled through registers, element by element: operands
// whose rows are not made of whole aligned 16-byte chunks.  load() brings the
// next step into registers while the current one is computed on, store() puts
// it into the other buffer.
template <typename T, bool SWAP, int EXT, int NW>
struct TileStageAny {
  static constexpr int PER = Pack16<T>::N;
  static constexpr int CHUNKS = EXT * (int)sizeof(T) / 16;
  static constexpr int N = EXT * 8 / (64 * NW);     // chunks a lane
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
  __device__ __forceinline__ void load(int64_t k0, int64_t n_k) {
#pragma unroll
    for (int t = 0; t < N; ++t) {
      const int at = place(t);
      if constexpr (!SWAP) {
        const int row = at >> 3, c = (at & 7) ^ (row & 7);
        int64_t i = i0 + row;
        i = i < n_i ? i : n_i - 1;
        const int64_t k = k0 + c * PER;
        const T* q = base + i * stride + k;
#pragma unroll
        for (int e = 0; e < PER; ++e)
          r[t].v[e] = k + e < n_k ? q[e] : (T)0.f;
      } else {
        const int row = at / CHUNKS;
        int c = at % CHUNKS;
        if (sizeof(T) == 2) c ^= 4 * (row & 3);
        const int64_t k = k0 + row, i = i0 + c * PER;
        const T* q = base + k * stride + i;
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

// fragment of 32 indices i.., quarter kk of the step
template <typename T, bool SWAP, int EXT>
__device__ __forceinline__ Pack16<T> fragment(const char* tile, int i, int kk,
                                              int lane) {
  const int q = lane >> 5;
  if constexpr (!SWAP) {
    return *reinterpret_cast<const Pack16<T>*>(
        tile + (i + (lane & 31)) * 128 + (((kk * 2 + q) ^ (lane & 7)) << 4));
  } else if constexpr (sizeof(T) == 2) {
    const int t = lane & 15;
    const int col = (i + (lane & 16)) * 2 + (t & 3) * 8;      // bytes
    const char* row = tile + (kk * 16 + q * 8 + (t >> 2)) * (EXT * 2) +
                      (col ^ ((t >> 2) << 6));
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

// A tile of BI x BJ by WI x WJ waves.  ANY: rows of any alignment.  ONES: also
// the sums of A over the contraction (a product with a column of ones).
template <typename T_, bool SA, bool SB, bool ANY, int BI_, int BJ_, int WI,
          int WJ, bool ONES>
struct MatrixTile {
  using T = T_;
  static constexpr int BI = BI_, BJ = BJ_;
  static constexpr int NW = WI * WJ, THREADS = 64 * NW;
  static constexpr int TI = BI / WI / 32, TJ = BJ / WJ / 32;
  static constexpr int BUF = (BI + BJ) * 128;
  static constexpr int LDS = 2 * BUF;
  f32x16 acc[TI][TJ];
  f32x16 sum[ONES ? TI : 1];

  __device__ __forceinline__ void step(const char* ta, int lane, int wi,
                                       int wj, bool ones) {
    const char* tb = ta + BI * 128;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      Pack16<T> fa[TI], fb[TJ];
#pragma unroll
      for (int u = 0; u < TI; ++u)
        fa[u] = fragment<T, SA, BI>(ta, wi + 32 * u, kk, lane);
#pragma unroll
      for (int v = 0; v < TJ; ++v)
        fb[v] = fragment<T, SB, BJ>(tb, wj + 32 * v, kk, lane);
#pragma unroll
      for (int u = 0; u < TI; ++u)
#pragma unroll
        for (int v = 0; v < TJ; ++v) mma32(fb[v], fa[u], acc[u][v]);
      if (ONES && ones) {
        Pack16<T> one;
#pragma unroll
        for (int e = 0; e < Pack16<T>::N; ++e) one.v[e] = (T)1.f;
#pragma unroll
        for (int u = 0; u < TI; ++u) mma32(one, fa[u], sum[u]);
      }
    }
  }

  // a: base, stride, first index, end of the indices; b alike; n_k: length of
  // the contraction (0 leaves zeros); ones: fill `sum` (first wave column)
  __device__ __forceinline__ void run(char* smem, const T* a, int64_t a_stride,
                                      int64_t i0, int64_t n_i, const T* b,
                                      int64_t b_stride, int64_t j0,
                                      int64_t n_j, int64_t n_k, bool ones) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);
#pragma unroll
    for (int u = 0; u < TI; ++u) {
#pragma unroll
      for (int v = 0; v < TJ; ++v) acc[u][v] = f32x16{};
      if (ONES) sum[u] = f32x16{};
    }
    if (n_k <= 0) return;
    constexpr int KS = kStepK<T>;
    int buf = 0;
    if constexpr (ANY) {
      TileStageAny<T, SA, BI, NW> sa;
      TileStageAny<T, SB, BJ, NW> sb;
      sa.start(a, a_stride, i0, n_i);
      sb.start(b, b_stride, j0, n_j);
      sa.load(0, n_k);
      sb.load(0, n_k);
      for (int64_t k0 = 0; k0 < n_k; k0 += KS, buf ^= 1) {
        char* ta = smem + buf * BUF;
        sa.store(ta);
        sb.store(ta + BI * 128);
        __syncthreads();
        if (k0 + KS < n_k) {
          sa.load(k0 + KS, n_k);
          sb.load(k0 + KS, n_k);
        }
        step(ta, lane, wi, wj, ones);
      }
    } else {
      TileStage<T, SA, BI, NW> sa;
      TileStage<T, SB, BJ, NW> sb;
      sa.start(a, a_stride, i0, n_i, wave, lane);
      sb.start(b, b_stride, j0, n_j, wave, lane);
      const uint32_t lds = lds_addr((const float*)smem);
      sa.fetch(lds, wave, 0, n_k);
      sb.fetch(lds + BI * 128, wave, 0, n_k);
      for (int64_t k0 = 0; k0 < n_k; k0 += KS, buf ^= 1) {
        // this wave's part of the step has landed; behind the barrier every
        // wave's has, and all are done with the other buffer
        lds_dma_landed();
        __syncthreads();
        if (k0 + KS < n_k) {
          const uint32_t to = lds + (uint32_t)((buf ^ 1) * BUF);
          sa.fetch(to, wave, k0 + KS, n_k);
          sb.fetch(to + BI * 128, wave, k0 + KS, n_k);
        }
        step(smem + buf * BUF, lane, wi, wj, ones);
      }
    }
  }

  // f(i, j, four values of consecutive j), offsets within the tile
  template <typename F>
  __device__ __forceinline__ void each4(F f) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);
#pragma unroll
    for (int u = 0; u < TI; ++u)
#pragma unroll
      for (int v = 0; v < TJ; ++v)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          f32x4 q;
#pragma unroll
          for (int e = 0; e < 4; ++e) q[e] = acc[u][v][4 * r + e];
          f(wi + 32 * u + (lane & 31), wj + 32 * v + 8 * r + 4 * (lane >> 5),
            q);
        }
  }
  // f(i, sum) once for every i of the tile
  template <typename F>
  __device__ __forceinline__ void each_sum(F f) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (wave % WJ != 0 || lane >= 32) return;
#pragma unroll
    for (int u = 0; u < TI; ++u)
      f((wave / WJ) * (BI / WI) + 32 * u + lane, sum[u][0]);
  }
};

}  // namespace xrd
