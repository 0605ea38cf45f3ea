// What the operators' kernels share: element types, loads that need no more
// alignment than an element, reductions over a workgroup.
#include "mlc_cdna4.h"

namespace mlc {

typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

// Codes that kernels leave in the invalid-input word.
enum { INVALID_CACHE_RANGE = 2 };

template <class T> struct element;
template <> struct element<float> {
  static __device__ __forceinline__ float widen(float x) { return x; }
  static __device__ __forceinline__ float narrow(float x) { return x; }
};
template <> struct element<f16> {
  static __device__ __forceinline__ float widen(f16 x) { return (float)x; }
  static __device__ __forceinline__ f16 narrow(float x) { return (f16)x; }
};
template <> struct element<__bf16> {
  static __device__ __forceinline__ float widen(__bf16 x) { return bf16_to_f32(__builtin_bit_cast(uint16_t, x)); }
  static __device__ __forceinline__ __bf16 narrow(float x) { return (__bf16)x; }
};

// N elements from an address that is aligned to ``A`` bytes: the hardware
// takes wide accesses at any address, the type says so to the compiler.
template <class T, int N, int A> struct __attribute__((packed, aligned(A))) piece { T x[N]; };
template <int A, int N, class T> __device__ __forceinline__ void load_n(T (&x)[N], const T* p) {
  const auto w = *reinterpret_cast<const piece<T, N, A>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = w.x[i];
}
template <int A, int N, class T> __device__ __forceinline__ void store_n(T* p, const T (&x)[N]) {
  piece<T, N, A> w;
#pragma unroll
  for (int i = 0; i < N; ++i) w.x[i] = x[i];
  *reinterpret_cast<piece<T, N, A>*>(p) = w;
}

template <class T> __device__ __forceinline__ const T* at(const void* p, int64_t bytes) {
  return reinterpret_cast<const T*>(reinterpret_cast<const char*>(p) + bytes);
}

}  // namespace mlc
