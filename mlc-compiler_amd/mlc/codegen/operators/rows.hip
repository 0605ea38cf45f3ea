// Rows on their way into products: the root-mean-square norm, with the residual's addition in
// front of it, and rows as 8-bit codes with a scale for each 128 values, from the norm, from a
// row as it is, or from one times silu of its gate.
//
//   h = x + residual;  y = h / sqrt(mean(h^2) + eps) * weight
//   scale = max(amax / 448, 2^-126) of a block's finite values;  code = e4m3(y / scale)
//
// Sums, the root and y are taken in 64 bits, whose additions and products cost what fp32's do
// here: squares of any fp32 value fit, and y is rounded to fp32 once. Infinities and NaN become
// codes of NaN and do not count for a scale.

namespace mlc {

struct RowsArgs {
  const void* x;
  const void* other;  // the residual, or the gate; null: none
  const void* weight;
  void* out;
  float* scales;
  void* sum;                    // of x and the residual
  int64_t x_off, o_off, w_off;  // bytes
  int64_t xb, xt, ob, ot;       // elements
  int32_t rows, seq, dim, wide_weight;
  double eps;
};

__device__ __forceinline__ double add_over_wave(double x) {
#pragma unroll
  for (int by = 1; by < 64; by *= 2) x += __shfl_xor(x, by);
  return x;
}

// Four values to e4m3, to nearest even; NaN becomes its NaN.
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// The codes of a block of 128 values, 8 in each of 16 neighbouring lanes, of which the first
// writes the scale. Lanes past the row's end have zeros and ``in`` false.
__device__ __forceinline__ void store_block(const float (&y)[8], bool in, uint8_t* codes, float* scale_at,
                                            bool first) {
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float m = __builtin_fabsf(y[j]);
    top = m < __builtin_inff() ? __builtin_fmaxf(top, m) : top;
  }
  top = group_reduce<16, OpMax>(top);
  const float scale = __builtin_fmaxf(top / 448.0f, 0x1p-126f);
  // In 64 bits a quotient in the middle of two codes is there exactly, and goes to the even one:
  // among 16-bit values, whose largest has few digits too, many are.
  const double by = __builtin_fmin(448.0 / (double)top, 0x1p126);
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)  // infinity is a NaN
    q[j] = __builtin_fabsf(y[j]) < __builtin_inff() ? (float)((double)y[j] * by) : __builtin_nanf("");
  if (in) {
    *reinterpret_cast<uint2v*>(codes) = uint2v{to_e4m3(q[0], q[1], q[2], q[3]), to_e4m3(q[4], q[5], q[6], q[7])};
    if (first) *scale_at = scale;
  }
}

// 8 values of a row from d on, which end at ``dim``. A: bytes that packs lie on.
template <int A, class T> __device__ __forceinline__ void load_pack_of(T (&v)[8], const T* p, int d, int dim) {
  if (d + 8 <= dim) {
    load_n<A>(v, p + d);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (d + j < dim) v[j] = p[d + j];
  }
}
template <int A, class T> __device__ __forceinline__ void store_pack_of(T* p, const float (&x)[8], int d, int dim) {
  T v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = element<T>::narrow(x[j]);
  if (d + 8 <= dim) {
    store_n<A>(p + d, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (d + j < dim) p[d + j] = v[j];
  }
}

// One row in WAVES waves, N packs of 8 values for each lane.
template <class T, int A, int WAVES, int N, bool EIGHT>
__device__ __forceinline__ void rms_norm(const RowsArgs& a) {
  constexpr int LANES = 64 * WAVES, ROWS = WAVES < 4 ? 4 / WAVES : 1;
  const int lane = threadIdx.x % LANES, dim = a.dim;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
  if (WAVES == 1 && row >= a.rows) return;  // a whole wave, and no barrier follows
  const int64_t b = row / a.seq, t = row % a.seq;
  const T* const x = at<T>(a.x, a.x_off) + b * a.xb + t * a.xt;
  const T* const r = at<T>(a.other, a.o_off) + b * a.ob + t * a.ot;
  T v[N][8], u[N][8];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int d = (lane + n * LANES) * 8;
    if (d < dim) {
      load_pack_of<A>(v[n], x, d, dim);
      if (a.other) load_pack_of<A>(u[n], r, d, dim);
    }
  }
  float h[N][8];
  double sum = 0.0;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int d = (lane + n * LANES) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float f = 0.0f;
      if (d + j < dim) {
        f = element<T>::widen(v[n][j]);
        if (a.other) f += element<T>::widen(u[n][j]);
      }
      h[n][j] = f;
      sum = __builtin_fma((double)f, (double)f, sum);
    }
  }
  if (a.sum) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int d = (lane + n * LANES) * 8;
      if (d < dim) store_pack_of<A>(reinterpret_cast<T*>(a.sum) + row * dim, h[n], d, dim);
    }
  }
  sum = add_over_wave(sum);
  if constexpr (WAVES > 1) {
    __shared__ double parts[WAVES];
    if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += parts[w];
  }
  const double by = 1.0 / __builtin_sqrt(sum / (double)dim + a.eps);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int d = (lane + n * LANES) * 8;
    const bool in = d < dim;
    float w[8] = {}, y[8];
    if (in) {
      if (a.wide_weight) {
        load_pack_of<4>(w, at<float>(a.weight, a.w_off), d, dim);
      } else {
        T z[8] = {};
        load_pack_of<(int)sizeof(T)>(z, at<T>(a.weight, a.w_off), d, dim);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = element<T>::widen(z[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = (float)((double)h[n][j] * by * (double)w[j]);
    if constexpr (EIGHT) {
      store_block(y, in, reinterpret_cast<uint8_t*>(a.out) + row * dim + d,
                  a.scales + row * ((dim + 127) / 128) + d / 128, lane % 16 == 0);
    } else if (in) {
      store_pack_of<A>(reinterpret_cast<T*>(a.out) + row * dim, y, d, dim);
    }
  }
}

// g / (1 + e^-g). e^-g is 2^h with h the rounded product, corrected by what the rounding left
// (as exp_nonpos does); where it is infinite the quotient is a zero, as in fp32's own formula.
__device__ __forceinline__ float silu(float g) {
  const float x = __builtin_fmaxf(-g, -104.0f), h = x * 0x1.715476p+0f;
  float r = __builtin_fmaf(-h, 0x1.62e430p-1f, x);
  r = __builtin_fmaf(-h, -0x1.05c610p-29f, r);
  const float e = __builtin_amdgcn_exp2f(h);
  const float s = 1.0f + (e < __builtin_inff() ? __builtin_fmaf(e, r, e) : e);
  const float f = s > 0x1p64f ? 0x1p-64f : 1.0f;  // no reciprocal below the normal numbers
  const float z = s * f, q = __builtin_amdgcn_rcpf(z);
  const float n = __builtin_fmaf(-z, q, 1.0f);  // one step of Newton's; z may be infinite
  return g * f * (s < __builtin_inff() ? __builtin_fmaf(n, q, q) : q);
}

constexpr int QUANTIZE_BLOCK = 256, QUANTIZE_PACKS = 2;  // of 8 values, for each thread

template <class T, int A, bool GATED> __device__ __forceinline__ void quantize(const RowsArgs& a) {
  constexpr int N = QUANTIZE_PACKS;
  const uint32_t blocks = (a.dim + 127) / 128, packs = blocks * 16;
  const uint64_t first = (uint64_t)blockIdx.x * (QUANTIZE_BLOCK * N);
  const uint32_t row0 = (uint32_t)(first / packs), rest = (uint32_t)(first % packs);
  T v[N][8], u[N][8];
  uint32_t rows[N], ds[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const uint32_t i = rest + threadIdx.x + n * QUANTIZE_BLOCK;
    const uint32_t row = row0 + i / packs, d = i % packs * 8;
    rows[n] = row;
    ds[n] = d;
    if (row < (uint32_t)a.rows && d < (uint32_t)a.dim) {
      const int64_t b = row / (uint32_t)a.seq, t = row % (uint32_t)a.seq;
      load_n<A>(v[n], at<T>(a.x, a.x_off) + b * a.xb + t * a.xt + d);
      if constexpr (GATED) load_n<A>(u[n], at<T>(a.other, a.o_off) + b * a.ob + t * a.ot + d);
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const bool in = rows[n] < (uint32_t)a.rows && ds[n] < (uint32_t)a.dim;
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      y[j] = in ? element<T>::widen(v[n][j]) : 0.0f;
      if constexpr (GATED) y[j] *= silu(in ? element<T>::widen(u[n][j]) : 0.0f);
    }
    store_block(y, in, reinterpret_cast<uint8_t*>(a.out) + (int64_t)rows[n] * a.dim + ds[n],
                a.scales + (int64_t)rows[n] * blocks + ds[n] / 128, threadIdx.x % 16 == 0);
  }
}

}  // namespace mlc

#define RMS_NORM(NAME, T, A, WAVES, N, EIGHT)                                                        \
  extern "C" __global__ void __launch_bounds__(WAVES < 4 ? 256 : 64 * WAVES) NAME(mlc::RowsArgs a) { \
    mlc::rms_norm<T, A, WAVES, N, EIGHT>(a);                                                         \
  }
#define QUANTIZE(NAME, T, A, GATED)                                                           \
  extern "C" __global__ void __launch_bounds__(mlc::QUANTIZE_BLOCK) NAME(mlc::RowsArgs a) {   \
    mlc::quantize<T, A, GATED>(a);                                                            \
  }
