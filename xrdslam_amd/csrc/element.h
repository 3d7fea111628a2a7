// Element types of the token and grouped-product kernels: storage type T, all
// arithmetic in f32, one round-to-nearest-even at the store.
#pragma once
#include "common.h"

namespace xrd {

// 16 bytes of T, the widest load a lane makes
template <typename T>
struct alignas(16) Pack16 {
  static constexpr int N = 16 / (int)sizeof(T);
  T v[N];
};
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__bf16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return (float)x; }
template <typename T>
__device__ __forceinline__ T from_f32(float x) {
  return (T)x;
}

// Results larger than the chip's L2s (eight of 4 MB) are stored past them: their
// lines would be evicted anyhow, and until then push out what is read.  Smaller
// ones are kept for the kernel that reads them next.  Table gradient of 131 MB, both
// launches: 40 us past the caches, 50 through them; bf16 16384 x 2048 x 2048 twice in
// a row (67 MB): 313 and 318; 8192 x 1024 x 1024 twice (17 MB): 66 and 60.
constexpr int64_t kCachedBytes = 32 << 20;
template <bool PAST, typename V>
__device__ __forceinline__ void store16(V* p, const V& v) {
  static_assert(sizeof(V) == 16, "one store");
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  if constexpr (PAST)
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v),
                                reinterpret_cast<u32x4*>(p));
  else
    *p = v;
}

inline int element_size(int dtype) {
  return dtype == XRD_F32 ? 4 : dtype == XRD_BF16 || dtype == XRD_F16 ? 2 : 0;
}
// F(T{}) with the storage type of dtype (checked by the caller)
#define XRD_BY_DTYPE(dtype, CALL)              \
  do {                                         \
    if ((dtype) == XRD_F32) {                  \
      using T = float;                         \
      CALL;                                    \
    } else if ((dtype) == XRD_BF16) {          \
      using T = __bf16;                        \
      CALL;                                    \
    } else {                                   \
      using T = _Float16;                      \
      CALL;                                    \
    }                                          \
  } while (0)

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace xrd
