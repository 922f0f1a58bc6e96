// What the kernels of libfedtrain share: element types, and the host's checks.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/fedtrain.h"

namespace fedtrain {

typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

// 16-bit types convert from f32 to the nearest value, ties to even
template <int D> struct Elem;
template <> struct Elem<FEDTRAIN_F32> {
  using type = float;
  static __device__ float up(float x) { return x; }
  static __device__ float down(float x) { return x; }
};
template <> struct Elem<FEDTRAIN_BF16> {
  using type = __bf16;
  static __device__ float up(__bf16 x) { return static_cast<float>(x); }
  static __device__ __bf16 down(float x) { return static_cast<__bf16>(x); }
};
template <> struct Elem<FEDTRAIN_F16> {
  using type = _Float16;
  static __device__ float up(_Float16 x) { return static_cast<float>(x); }
  static __device__ _Float16 down(float x) { return static_cast<_Float16>(x); }
};

inline bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// workgroups of 256 in a launch: its threads are counted in 32 bits
constexpr int64_t kMostGroups = UINT32_MAX / 256;

// the status of the launches so far, without leaving an error behind
inline int launched() { return static_cast<int>(hipGetLastError()); }

}  // namespace fedtrain
