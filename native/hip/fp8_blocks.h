// Shared pieces of the 8-bit block-scaled operators (fp8_blocks.hip, fp8_matmul.hip).
//
// A block matrix holds R x K values in e4m3 and one scale for each 1 x 128 block (activations)
// or 128 x 128 block (weights). K is padded with zeros to Kp, the next multiple of 128, so every
// row of bytes starts on a 128-byte line and no product has a tail along K.
//   values  [R][Kp] bytes
//   scales  1 x 128:   [Kp/128][R up to a multiple of 8]   block by block: the rows of a tile are neighbours
//           128 x 128: [ceil(R/128)][Kp/128 up to a multiple of 4]
// A scale is a float32 (largest magnitude / 448) or an e8m0 byte b that stands for 2^(b-127).
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

namespace yoda_fp8 {

constexpr int kBlockK = 128;

// types of a tensor's elements, as ops/fp8.py passes them
enum Type : int { kBf16 = 0, kFp16 = 1, kFp32 = 2 };

inline bool valid_type(int t) { return t >= kBf16 && t <= kFp32; }

// The device of a call, made current for its length (a caller's tensors may live on another
// device than the thread's current one).
struct DeviceScope {
  int before = -1;
  hipError_t err;
  explicit DeviceScope(int device) {
    err = hipGetDevice(&before);
    if (err == hipSuccess && before != device) err = hipSetDevice(device);
    else before = -1;
  }
  ~DeviceScope() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float to_f32(uint16_t v, __hip_bfloat16*) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ float to_f32(uint16_t v, __half*) { return __half2float(__ushort_as_half(v)); }

template <typename T>
struct Bits {   // the storage of one element of T
  using type = uint16_t;
};
template <>
struct Bits<float> {
  using type = uint32_t;
};

template <typename T>
__device__ __forceinline__ float load_f32(typename Bits<T>::type v) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(v);
  else return to_f32(v, (T*)nullptr);
}

// float32 to the storage of T, to nearest, ties to even
template <typename T>
__device__ __forceinline__ typename Bits<T>::type store_bits(float v) {
  if constexpr (sizeof(T) == 4) return __float_as_uint(v);
  else if constexpr (__is_same(T, __half)) return __half_as_ushort(__float2half_rn(v));
  else {
    typedef __bf16 bf16_t;
    const bf16_t b = (bf16_t)v;
    return __builtin_bit_cast(uint16_t, b);
  }
}

// Two float32 to two neighbours of a 16-bit type, to nearest, ties to even.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (__is_same(T, __half)) {
    return (uint32_t)store_bits<__half>(a) | (uint32_t)store_bits<__half>(b) << 16;
  } else {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
  }
}

// 16 bytes at any element of 2 or 4 bytes: one access, whatever the row's pitch. (A packed struct of
// elements would be taken apart into one access an element.)
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
template <int SIZE>
struct Wide {
  using type = u32x4_at2;
  static __device__ __forceinline__ u32x4 load(const void* p) { return *(const type*)p; }
  static __device__ __forceinline__ void store(void* p, u32x4 v) { *(type*)p = v; }
};
template <>
struct Wide<4> {
  using type = u32x4_at4;
  static __device__ __forceinline__ u32x4 load(const void* p) { return *(const type*)p; }
  static __device__ __forceinline__ void store(void* p, u32x4 v) { *(type*)p = v; }
};

}  // namespace yoda_fp8
