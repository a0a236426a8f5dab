// The element types of the decode-step operators (MB_F32, MB_F16, MB_BF16): widening, rounding, vectors.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace elem {

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

// To nearest even.
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <int BYTES> struct Raw;
template <> struct Raw<2> { typedef uint16_t type; };
template <> struct Raw<4> { typedef uint32_t type; };
template <> struct Raw<8> { typedef uint2 type; };
template <> struct Raw<16> { typedef uint4 type; };

// N elements moved as one word; the address is a multiple of its size.
template <typename T, int N>
struct Vec {
  typedef typename Raw<N * sizeof(T)>::type Word;
  union {
    Word word;
    T v[N];
  };
  __device__ __forceinline__ Vec() {}
  __device__ __forceinline__ void load(const T *p) { word = *reinterpret_cast<const Word *>(p); }
  __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<Word *>(p) = word; }
};

}  // namespace elem

// Runs `...` with T the element type that `dtype` names (one that the caller has checked).
#define MB_FOR_ELEMENT(dtype, ...)                                  \
  do {                                                              \
    if ((dtype) == MB_F32) {                                        \
      typedef float T;                                              \
      __VA_ARGS__;                                                  \
    } else if ((dtype) == MB_F16) {                                 \
      typedef __half T;                                             \
      __VA_ARGS__;                                                  \
    } else {                                                        \
      typedef __nv_bfloat16 T;                                      \
      __VA_ARGS__;                                                  \
    }                                                               \
  } while (0)

// A kernel met an index in device memory outside its range: mb_stream_sync says so.
__device__ __forceinline__ void mb_report_bad_index(int *status) { *static_cast<volatile int *>(status) = MB_DEV_BAD_INDEX; }
