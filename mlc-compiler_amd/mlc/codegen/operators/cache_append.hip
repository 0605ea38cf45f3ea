// New keys and values into the 8-bit cache: code = e4m3(x / scale), one power of
// two as the scale of a (block of tokens, head), the smallest that brings the
// block's largest finite magnitude to 448 or less.
//
// A power of two makes the quotient exact, so a code is the value rounded once,
// whatever the scale, and a block whose scale grows keeps its older values but
// for those that leave e4m3's normal range (2^-9 * 448 below the largest).
// Running it again on the same arguments changes nothing.
//
// Bound by memory (a value read, a byte written). One workgroup for each block
// that new tokens can touch, each of its rows read once and kept in registers
// between the search for the largest and the rounding: 4 x 2000 tokens, 8 heads of 128,
// fp16, 11.4 us, 3.5 TB/s, in fp32 16.3, 5.0; one token of 32 sequences 3.8 us, a launch's
// latency, where one wave a block is enough.

namespace mlc {

struct AppendArgs {
  void* cache[2];  // keys, values
  void* scale[2];
  const void* fresh[2];
  const void* start;
  const void* count;  // null: every new token is real
  int* error;
  int64_t cache_off[2], scale_off[2], fresh_off[2], start_off, count_off;  // bytes
  int64_t fb[2], ft[2], fh[2], ss, sc;                                     // elements
  int32_t tokens, heads, dim, capacity, block, touched;  // touched: blocks of a row, at most
};

__device__ __forceinline__ float power_of_two(int e) {  // -126 <= e <= 127
  return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}

// Exponent of the smallest power of two, a normal number, that brings ``amax``
// (finite, not negative) to 448 = 1.75 * 2^8 or less.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, amax);
  const int e = (int)(bits >> 23) - 127;
  const int need = (bits & 0x7fffffu) <= 0x600000u ? e - 8 : e - 7;
  return need < -126 ? -126 : need;
}

// Four values to e4m3, to nearest even; NaN and infinity become its NaN.
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
__device__ __forceinline__ uint32_t rescaled(uint32_t w, float by) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return to_e4m3(lo[0] * by, lo[1] * by, hi[0] * by, hi[1] * by);
}

// N items of 8 values for each of 64 * WAVES threads hold the block's new rows.
template <class T, int A, int N, int WAVES>
__device__ __forceinline__ void cache_append(const AppendArgs& a) {
  constexpr int THREADS = 64 * WAVES;
  // heads inside blocks: workgroups next to each other read the same tokens
  uint32_t w = blockIdx.x;
  const int h = (int)(w % (uint32_t)a.heads);
  w /= (uint32_t)a.heads;
  const int which = (int)(w & 1);
  w >>= 1;
  const int nth = (int)(w % (uint32_t)a.touched), b = (int)(w / (uint32_t)a.touched);

  const int64_t start = at<int32_t>(a.start, a.start_off)[b * a.ss];
  const int64_t count = a.count ? at<int32_t>(a.count, a.count_off)[b * a.sc] : a.tokens;
  if (start < 0 || count < 0 || count > a.tokens || start + count > a.capacity) {
    if (threadIdx.x == 0) *a.error = INVALID_CACHE_RANGE;
    return;
  }
  const int64_t block = start / a.block + nth, base = block * a.block;
  const int lo = start > base ? (int)(start - base) : 0;  // rows of the block
  const int hi = start + count < base + a.block ? (int)(start + count - base) : a.block;
  if (lo >= hi) return;

  const int units = a.dim / 8;
  const T* src = at<T>(a.fresh[which], a.fresh_off[which]) + b * a.fb[which] + h * a.fh[which] +
                 (base + lo - start) * a.ft[which];
  const int items = (hi - lo) * units;
  T x[N][8];
  float top = 0.0f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int i = threadIdx.x + n * THREADS;
    if (i < items) load_n<A>(x[n], src + (int64_t)(i / units) * a.ft[which] + i % units * 8);
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (threadIdx.x + n * THREADS < items) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float m = __builtin_fabsf(element<T>::widen(x[n][j]));
        top = m < __builtin_inff() ? __builtin_fmaxf(top, m) : top;
      }
    }
  }
  __shared__ float part[WAVES];
  top = row_reduce<THREADS, OpMax>(top, part);

  const int64_t tile = ((int64_t)b * a.heads + h) * (a.capacity / a.block) + block;
  float* const scale_at = const_cast<float*>(at<float>(a.scale[which], a.scale_off[which])) + tile;
  uint8_t* const codes = const_cast<uint8_t*>(at<uint8_t>(a.cache[which], a.cache_off[which])) +
                         tile * a.block * a.dim;
  const int e = scale_exponent(top);
  float scale = power_of_two(e), inverse = power_of_two(-e);
  if (lo > 0) {
    const float before = *scale_at;
    if (before >= scale) {
      scale = before;
      inverse = 1.0f / before;
    } else {
      const float by = before / scale;
      for (int i = threadIdx.x; i < lo * units; i += THREADS) {
        uint2v* p = reinterpret_cast<uint2v*>(codes) + i;
        const uint2v old = *p;
        *p = uint2v{rescaled(old.x, by), rescaled(old.y, by)};
      }
    }
    if constexpr (WAVES > 1) __syncthreads();  // everyone has read the scale
  }
  if (threadIdx.x == 0) *scale_at = scale;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int i = threadIdx.x + n * THREADS;
    if (i < items) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = element<T>::widen(x[n][j]);
        y[j] = __builtin_fabsf(v) < __builtin_inff() ? v * inverse : __builtin_nanf("");
      }
      reinterpret_cast<uint2v*>(codes + (int64_t)lo * a.dim)[i] =
          uint2v{to_e4m3(y[0], y[1], y[2], y[3]), to_e4m3(y[4], y[5], y[6], y[7])};
    }
  }
}

}  // namespace mlc

#define CACHE_APPEND(NAME, T, A, N, WAVES)                                                  \
  extern "C" __global__ void __launch_bounds__(64 * WAVES) NAME(mlc::AppendArgs a) {        \
    mlc::cache_append<T, A, N, WAVES>(a);                                                   \
  }
