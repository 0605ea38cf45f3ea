// Rows on their way into products: the root-mean-square norm, with the residual's addition in
// front of it, and rows as 8-bit codes with a scale for each 128 values, from the norm, from a
// row as it is, or from one times silu of its gate.
//
//   h = x + residual;  y = h / sqrt(mean(h^2) + eps) * weight
//   scale = max(amax / 448, 2^-126) of a block's finite values;  code = e4m3(y / scale)
//
// Memory bounds both: a row is read once into registers, so that nothing is read again, and all of
// its loads, the weight's too, are on their way before the first is used. What else is to be watched are the
// instructions for each value: a wave's double takes one and its conversions take more.
// fp32's sums, root, y and quotients are taken in 64 bits, and a norm's y is rounded once; 16-bit values'
// in fp32, but for the sums of eight squares, whose range is any value's, and for what fp32 does not tell.
// Infinities and NaN become codes of NaN and do not count for a scale.
//
// 8192 rows of 4096 in bf16 with a residual, to codes: 49.8 us, 4.7 TB/s, with 55 % of the time in vector
// instructions (in 64 bits all through 54.8); with 8 waves of one pack instead of 4 of two 51.1. 6063 rows
// of 12288 in bf16, gated: 75 us, 5.0 TB/s. A
// single row: 3 us.

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
  double eps, part;  // part: 1 / dim
};

// x of a lane below this one by DPP, 0 where there is none.
template <int CONTROL, int ROWS> __device__ __forceinline__ double lower(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CONTROL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CONTROL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double add_over_wave(double x) {
  x += lower<0x111, 0xf>(x);  // by 1, 2, 4 and 8 lanes of 16, then the last of 16 and of 32
  x += lower<0x112, 0xf>(x);
  x += lower<0x114, 0xf>(x);
  x += lower<0x118, 0xf>(x);
  x += lower<0x142, 0xa>(x);
  x += lower<0x143, 0xc>(x);
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)u, 63), hi = __builtin_amdgcn_readlane((uint32_t)(u >> 32), 63);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Four values to e4m3, to nearest even; NaN becomes its NaN.
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// What y is: of T's digits, or rounded to fp32 from more, or that of fp32 values.
enum { GIVEN, ROUNDED, FULL };

// The codes of a block of 128 values, 8 in each of 16 neighbouring lanes, of which the first
// writes the scale. Lanes past the row's end have zeros and ``in`` false.
//
// Values that are given have quotients in the middle of two codes, which go to the even one, so these have to
// be exact. y * 448 and the middle times the largest are whole numbers of 14 and 16 bits where y has 11: the
// quotient is in the middle or at least 2^-16 beside it. So one in fp32, off by 2^-22, is rounded to 18
// digits, which puts it there or leaves it on its side. Of fp32 values it is taken in 64 bits.
//
// Of values rounded to fp32 a quotient is rounded once more, by a factor of two floats, so that few codes are
// others than the real quotients'. What all values have in common, ``factor``, is left to the scale: codes do
// not depend on it.
template <int KIND>
__device__ __forceinline__ void store_block(const float (&y)[8], float factor, bool in, uint8_t* codes,
                                            float* scale_at, bool first) {
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = __builtin_elementwise_maximum(top, __builtin_fabsf(y[j]));
  top = group_reduce<16, OpMax>(top);
  const bool finite = top < __builtin_inff();
  if (!finite) {
    top = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float m = __builtin_fabsf(y[j]);
      top = m < __builtin_inff() ? __builtin_fmaxf(top, m) : top;
    }
    top = group_reduce<16, OpMax>(top);
  }
  float q[8];
  if constexpr (KIND == GIVEN) {
    // 448 / top, whose reciprocal is a normal number: two roundings and the reciprocal's unit of a quotient
    const float by = __builtin_fminf(1.75f * __builtin_amdgcn_rcpf(top * 0x1p-8f), 0x1p126f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      q[j] = y[j] * by;
      q[j] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, q[j]) + 0x20) & 0xffffffc0u);
    }
  } else {
    const double r = __builtin_amdgcn_rcp((double)top);
    double by = 448.0 * __builtin_fma(__builtin_fma(-(double)top, r, 1.0), r, r);  // NaN for zeros alone
    by = factor == factor ? __builtin_fmin(by, (double)factor * 0x1p126) : (double)factor;
    const float hi = (float)by, lo = (float)(by - (double)hi);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      q[j] = KIND == FULL ? (float)((double)y[j] * by) : __builtin_fmaf(y[j], hi, y[j] * lo);
  }
  if (!finite) {
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = __builtin_fabsf(y[j]) < __builtin_inff() ? q[j] : __builtin_nanf("");
  }
  if (in) {
    *reinterpret_cast<uint2v*>(codes) = uint2v{to_e4m3(q[0], q[1], q[2], q[3]), to_e4m3(q[4], q[5], q[6], q[7])};
    if (first) *scale_at = __builtin_fmaxf(top * (1.0f / 448.0f) * factor, 0x1p-126f);
  }
}

// store_block of gated 16-bit values in fp32, where that tells every code. A value is within (7.5 + 1.25 g) 2^-24 of
// itself, with ``far`` this lane's largest g = -gate (``gated``). So is the largest, with that of the lanes that may have
// it, and a quotient by four roundings more: 19 + 1.25 (g + g) units of 2^-23 of its power of two. Three digits behind
// that power e4m3 ends, or below 2^-6 at 2^-9, where a value with 2^-6 added has its middles in the same place. Where
// a quotient is so near to one nothing is stored and the result is true, for the whole block, which is then taken in 64
// bits: 1 of 160 blocks, 6063 rows of 12288 75 us, as without that, all of them 110. So are infinities and NaN, gates
// below -80, and blocks so small that fp32 loses digits.
__device__ __forceinline__ bool store_rough_block(const float (&y)[8], float far, bool in, uint8_t* codes,
                                                  float* scale_at, bool first) {
  float own = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) own = __builtin_elementwise_maximum(own, __builtin_fabsf(y[j]));
  const float top = group_reduce<16, OpMax>(own);
  const float top_far = group_reduce<16, OpMax>(own < top * 0.9999f ? 0.0f : far);
  const bool fine = far <= 80.0f && top < __builtin_inff() && (top >= 0x1p-60f || top == 0.0f);
  const uint32_t near = (uint32_t)__builtin_fmaf(far + top_far, 1.25f, 21.0f) << 12, base = near - 0x80000000u;
  const float by = 1.75f * __builtin_amdgcn_rcpf(__builtin_fmaxf(top, 0x1p-60f) * 0x1p-8f);
  float q[8];
  uint32_t least = ~0u;  // of what lies behind three digits, from ``near`` below the middle on
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    q[j] = y[j] * by;
    const float m = __builtin_fabsf(q[j]);
    const uint32_t behind = (__builtin_bit_cast(uint32_t, m + (m < 0x1p-6f ? 0x1p-6f : 0.0f)) << 12) + base;
    least = behind < least ? behind : least;
  }
  if (__ballot(least < 2 * near || !fine) >> (threadIdx.x & 48) & 0xffff) return true;
  if (in) {
    *reinterpret_cast<uint2v*>(codes) = uint2v{to_e4m3(q[0], q[1], q[2], q[3]), to_e4m3(q[4], q[5], q[6], q[7])};
    if (first) *scale_at = __builtin_fmaxf(top * (1.0f / 448.0f), 0x1p-126f);
  }
  return false;
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
  static_assert(WAVES == 1 || WAVES >= 4, "the grid is made for 4 rows or one");
  constexpr int LANES = 64 * WAVES, ROWS = WAVES == 1 ? 4 : 1;
  const int lane = threadIdx.x % LANES, dim = a.dim;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
  if (WAVES == 1 && row >= a.rows) return;  // a whole wave, and no barrier follows
  const int64_t b = row / a.seq, t = row % a.seq;
  const T* const x = at<T>(a.x, a.x_off) + b * a.xb + t * a.xt;
  const T* const r = at<T>(a.other, a.o_off) + b * a.ob + t * a.ot;
  T v[N][8] = {}, u[N][8] = {};
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
#pragma unroll
    for (int j = 0; j < 8; ++j) h[n][j] = element<T>::widen(v[n][j]) + element<T>::widen(u[n][j]);
    float eight = 0.0f;
    if constexpr (sizeof(T) < 4) {
#pragma unroll
      for (int j = 0; j < 8; ++j) eight = __builtin_fmaf(h[n][j], h[n][j], eight);
    }
    if (sizeof(T) < 4 && eight > 0x1p-80f && eight < 0x1p100f) {
      sum += (double)eight;
    } else {  // fp32, zeros, or squares that leave its range
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = __builtin_fma((double)h[n][j], (double)h[n][j], sum);
    }
  }
  if (a.sum) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int d = (lane + n * LANES) * 8;
      if (d < dim) store_pack_of<A>(reinterpret_cast<T*>(a.sum) + row * dim, h[n], d, dim);
    }
  }
  T z[N][8] = {};
  float wide[N][8] = {};
  auto load_weight = [&](int n) {
    const int d = (lane + n * LANES) * 8;
    if (d < dim) {
      if (sizeof(T) < 4 && a.wide_weight) load_pack_of<4>(wide[n], at<float>(a.weight, a.w_off), d, dim);
      else load_pack_of<(int)sizeof(T)>(z[n], at<T>(a.weight, a.w_off), d, dim);
    }
  };
  constexpr bool EARLY = WAVES * N < 64;  // or there are no registers for it
  if constexpr (EARLY) {
#pragma unroll
    for (int n = 0; n < N; ++n) load_weight(n);
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
  const double mean = __builtin_fma(sum, a.part, a.eps);
  auto weight = [&](int n, int j) { return sizeof(T) < 4 && a.wide_weight ? wide[n][j] : element<T>::widen(z[n][j]); };
  float factor = 1.0f;
  if constexpr (sizeof(T) < 4) {
    // A power of two near the root goes into h, so that the reciprocal is a normal number whatever the root: from 1 to 2,
    // so that h times the weight is not beyond fp32 where the norm is not.
    const int power = (__builtin_amdgcn_frexp_exp(mean) + 1) >> 1;
    const float by = __builtin_amdgcn_rsqf((float)__builtin_amdgcn_ldexp(mean, -2 * power));
    factor = by;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!EARLY) load_weight(n);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[n][j] = __builtin_amdgcn_ldexpf(h[n][j], -power) * (EIGHT ? 1.0f : by) * weight(n, j);
    }
  } else {
    const double by = 1.0 / __builtin_sqrt(mean);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!EARLY) load_weight(n);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[n][j] = (float)((double)h[n][j] * by * (double)weight(n, j));
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int d = (lane + n * LANES) * 8;
    if constexpr (EIGHT) {
      store_block<sizeof(T) < 4 ? ROUNDED : FULL>(h[n], factor, d < dim, reinterpret_cast<uint8_t*>(a.out) + row * dim + d,
                                                  a.scales + row * ((dim + 127) / 128) + d / 128, lane % 16 == 0);
    } else if (d < dim) {
      store_pack_of<A>(reinterpret_cast<T*>(a.out) + row * dim, h[n], d, dim);
    }
  }
}

// 1 / (1 + e^-g): 2^h from h's whole part and a polynomial of the rest, up to 1/2 to both sides, which is 2^-28 of
// itself off (a least squares fit of degree 6, weighted for that).
__device__ __forceinline__ double sigmoid(float g) {
  const double h = __builtin_fmax(__builtin_fmin((double)g * -0x1.71547652b82fep+0, 1000.0), -1000.0);
  const double n = __builtin_rint(h), f = h - n;
  double p = 0x1.41c82d5786988p-13;
  p = __builtin_fma(p, f, 0x1.5f69753d724cbp-10);
  p = __builtin_fma(p, f, 0x1.3b2e341c3f47ep-7);
  p = __builtin_fma(p, f, 0x1.c6ae81545310dp-5);
  p = __builtin_fma(p, f, 0x1.ebfbd9497c82ap-3);
  p = __builtin_fma(p, f, 0x1.62e431121ea6dp-1);
  p = __builtin_fma(p, f, 0x1.00000003b033bp+0);
  const double z = 1.0 + __builtin_amdgcn_ldexp(p, (int)n), q = __builtin_amdgcn_rcp(z);
  return __builtin_fma(__builtin_fma(-z, q, 1.0), q, q);  // one step of Newton's
}

// x of a lane of the same 16 by DPP, BY lanes on.
template <int BY> __device__ __forceinline__ double turned(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, 0x120 + BY, 0xf, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), 0x120 + BY, 0xf, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// store_block of values in 64 bits. What fp32 does not hold is an infinity.
__device__ __forceinline__ void store_wide_block(const double (&y)[8], bool in, uint8_t* codes, float* scale_at,
                                                 bool first) {
  constexpr double MOST = 0x1.fffffep127;
  double top = 0.0, zero = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    top = __builtin_fmax(top, __builtin_fabs(y[j]));
    zero = __builtin_fma(y[j], 0.0, zero);  // or NaN
  }
  const bool odd = zero != 0.0 || top > MOST;
  if (odd) {
    top = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = __builtin_fabs(y[j]) <= MOST ? __builtin_fmax(top, __builtin_fabs(y[j])) : top;
  }
  top = __builtin_fmax(top, turned<8>(top));
  top = __builtin_fmax(top, turned<4>(top));
  top = __builtin_fmax(top, turned<2>(top));
  top = __builtin_fmax(top, turned<1>(top));
  const double r = __builtin_amdgcn_rcp(top);
  const double by = __builtin_fmin(448.0 * __builtin_fma(__builtin_fma(-top, r, 1.0), r, r), 0x1p126);
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = (float)(y[j] * by);
  if (odd) {
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = __builtin_fabs(y[j]) <= MOST ? q[j] : __builtin_nanf("");
  }
  if (in) {
    *reinterpret_cast<uint2v*>(codes) = uint2v{to_e4m3(q[0], q[1], q[2], q[3]), to_e4m3(q[4], q[5], q[6], q[7])};
    if (first) *scale_at = __builtin_fmaxf((float)(top * (1.0 / 448.0)), 0x1p-126f);
  }
}

// x g times that in fp32, for 16-bit values and gates from -80 on. The exponent's roundings are 1.22 |g| 2^-24 of
// e^-g, and of the result where that is large; its unit, a sum, a reciprocal's unit and two products are 7 more. Only x g
// can leave fp32's range before the result does: upwards it is then infinite.
__device__ __forceinline__ float gated(float x, float g) {
  return x * g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -0x1.715476p+0f));
}

constexpr int QUANTIZE_BLOCK = 256, QUANTIZE_PACKS = 2;  // of 8 values, for each thread

template <class T, int A, bool GATED> __device__ __forceinline__ void quantize(const RowsArgs& a) {
  constexpr int N = QUANTIZE_PACKS;
  const uint32_t blocks = (a.dim + 127) / 128, packs = blocks * 16;
  const uint64_t first = (uint64_t)blockIdx.x * (QUANTIZE_BLOCK * N);
  uint32_t row0, rest;  // divided in 64 bits only where that is needed
  if (first >> 32) {
    row0 = (uint32_t)(first / packs);
    rest = (uint32_t)(first % packs);
  } else {
    row0 = (uint32_t)first / packs;
    rest = (uint32_t)first % packs;
  }
  const uint32_t b0 = row0 / (uint32_t)a.seq, t0 = row0 % (uint32_t)a.seq;
  const float share = __builtin_amdgcn_rcpf((float)packs);
  T v[N][8] = {}, u[N][8] = {};
  uint32_t rows[N], ds[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const uint32_t i = rest + threadIdx.x + n * QUANTIZE_BLOCK;
    uint32_t more = (uint32_t)((float)i * share);  // i / packs, or one beside it
    more -= more * packs > i;
    more += (more + 1) * packs <= i;
    rows[n] = row0 + more;
    ds[n] = (i - more * packs) * 8;
    if (rows[n] < (uint32_t)a.rows && ds[n] < (uint32_t)a.dim) {
      uint32_t b = b0, t = t0 + more;
      if (t >= (uint32_t)a.seq) {
        b += t / (uint32_t)a.seq;
        t %= (uint32_t)a.seq;
      }
      load_n<A>(v[n], at<T>(a.x, a.x_off) + (int64_t)b * a.xb + (int64_t)t * a.xt + ds[n]);
      if constexpr (GATED) load_n<A>(u[n], at<T>(a.other, a.o_off) + (int64_t)b * a.ob + (int64_t)t * a.ot + ds[n]);
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const bool in = rows[n] < (uint32_t)a.rows && ds[n] < (uint32_t)a.dim;
    uint8_t* const codes = reinterpret_cast<uint8_t*>(a.out) + (int64_t)rows[n] * a.dim + ds[n];
    float* const scale = a.scales + (int64_t)rows[n] * blocks + ds[n] / 128;
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = element<T>::widen(v[n][j]);
    if constexpr (GATED) {
      float g[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = element<T>::widen(u[n][j]);
      if constexpr (sizeof(T) < 4) {
        float y[8], far = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          y[j] = gated(x[j], g[j]);
          far = __builtin_fmaxf(far, -g[j]);
        }
        if (!store_rough_block(y, far, in, codes, scale, threadIdx.x % 16 == 0)) continue;
      }
      double y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = (double)x[j] * (double)g[j] * sigmoid(g[j]);
      store_wide_block(y, in, codes, scale, threadIdx.x % 16 == 0);
    } else {
      store_block<sizeof(T) == 4 ? FULL : GIVEN>(x, 1.0f, in, codes, scale, threadIdx.x % 16 == 0);
    }
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
