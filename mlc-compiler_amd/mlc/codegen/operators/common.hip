// What the operators' kernels share: element types, loads that need no more
// alignment than an element, reductions over a workgroup.
#include "mlc_cdna4.h"

namespace mlc {

typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

// Codes that kernels leave in the invalid-input word.
enum { INVALID_CACHE_RANGE = 2 };

// The weights of values from the 8-bit cache are fp16, the largest 2^14 or 2^15, and a value
// with its scale may be as large as fp32 holds: O and the sum of the weights are kept 2^-46
// times themselves, so that O stays finite over 2^30 keys. Values below 2^-100 lose digits.
constexpr float SCALE_ROOM = 0x1p-46f;

template <bool B> struct bool_constant { static constexpr bool value = B; };

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

// Two e4m3 codes of a word, the low or the high pair, as two 16-bit values: exact.
template <class T> struct codes;
template <> struct codes<f16> {
  typedef half8 v8;
  static __device__ __forceinline__ uint32_t widen(uint32_t w, int hi) {
    return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
  }
};
template <> struct codes<__bf16> {
  typedef bf16x8 v8;
  static __device__ __forceinline__ uint32_t widen(uint32_t w, int hi) {
    return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
  }
};

// One row of O out of the parts that workgroups made of it: ``of`` of them, ``step`` floats
// apart, each dim values not normalised, then the reference of their exponentials in log2
// units and the sum of their weights. For one workgroup of WAVES: groups of 16, 32 or 64
// lanes (4 values a lane, dim <= 256) take parts in turn, four loads on their way at a
// time, since latency is all that this costs, and meet in LDS.
template <int WAVES, class T>
__device__ __forceinline__ void join_parts(const float* part, int64_t step, int of, int dim, T* out) {
  constexpr int THREADS = 64 * WAVES;
  __shared__ __attribute__((aligned(16))) float4v lx[THREADS];
  __shared__ float2v ls[THREADS];
  const int width = dim <= 64 ? 16 : dim <= 128 ? 32 : 64, groups = THREADS / width;
  const int group = threadIdx.x / width, d = threadIdx.x % width * 4;
  float4v x = {0.0f, 0.0f, 0.0f, 0.0f};
  float sum = 0.0f, top = -__builtin_inff();
  // (top, sum, x) and a part or another group's: to their common reference
  auto meet = [&](float2v ml, float4v v) {
    const float next = ml.x > top ? ml.x : top;
    const float ref = next == -__builtin_inff() ? 0.0f : next;
    const float f = __builtin_amdgcn_exp2f(top - ref), g = __builtin_amdgcn_exp2f(ml.x - ref);
    top = next;
    sum = __builtin_fmaf(ml.y, g, sum * f);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(v[e], g, x[e] * f);
  };
  for (int i0 = group; i0 < of; i0 += 4 * groups) {
    float4v v[4];
    float2v ml[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j * groups;
      v[j] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
      ml[j] = float2v{-__builtin_inff(), 0.0f};
      if (i < of) {
        ml[j] = *reinterpret_cast<const float2v*>(part + i * step + dim);
        if (d < dim) v[j] = *reinterpret_cast<const float4v*>(part + i * step + d);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) meet(ml[j], v[j]);
  }
  lx[threadIdx.x] = x;
  ls[threadIdx.x] = float2v{top, sum};
  __syncthreads();
  if (group > 0 || d >= dim) return;
  for (int g = 1; g < groups; ++g) meet(ls[threadIdx.x + g * width], lx[threadIdx.x + g * width]);
  const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
  T v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = element<T>::narrow(x[e] * inverse);
  store_n<8>(out + d, v);
}

}  // namespace mlc
