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
