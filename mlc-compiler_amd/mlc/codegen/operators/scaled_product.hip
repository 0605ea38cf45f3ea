// Products of 8-bit rows whose scales change every 128 values of the sum:
//
//   out[m, n] = sum over blocks i of  sa[m, i] * sb[n / 128, i] * (a[m, i] . b[n, i])  + bias[n]
//
// A block's dot products come from matrix instructions begun at zero; their fp32 result is added
// to the sum with the block's two scales as its factor.
//
// The 8-bit instruction (16x16x128) takes neighbouring products by eights and cuts them at
// 2^-13 of the power of two of a group's largest: a sum of random values is 1.5e-5 of itself off, which is
// a tenth of what a result's rounding to fp16 takes and a hundredth of bf16's. Many rows with
// such results use it. Results in fp32, and few rows, where the weight's way from memory is all that
// counts, use the fp16 one on widened codes, which is exact: 2e-8.
//
// The weight's rows are the instruction's rows and the activations' its columns, so that a lane
// holds four neighbouring outputs of one row m, whose scale is one number for all of them.
// Which of a block's values lie in which of the instruction's places is free as long as both
// operands agree: lane (r, g) holds bytes 16 g .. + 15 and 64 + 16 g .. + 15 of row r.

namespace mlc {

typedef int int4v __attribute__((ext_vector_type(4)));
typedef int int8v __attribute__((ext_vector_type(8)));

struct ScaledProductArgs {
  const void* a;
  const void* a_scales;
  const void* b;
  const void* b_scales;
  const void* bias;  // null: none
  void* out;
  float* part;                                  // where blocks are split: [split][m][n]
  int64_t a_off, as_off, b_off, bs_off, c_off;  // bytes
  int64_t ab, at, asb, ast, ass, br, bsr, bss;  // elements: a's rows, its scales', b's, theirs
  int32_t rows, seq, n, k, splits, row_tiles, wide_bias;
  int32_t regular;  // rows of a have one stride, and seq is all of them
};

// A lane's 32 codes of a row's block, as they are or widened to fp16.
template <bool EXACT> struct Codes;
template <> struct Codes<false> {
  int8v x;
  __device__ __forceinline__ Codes() {}
  __device__ __forceinline__ Codes(int4v lo, int4v hi) : x(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)) {}
};
template <> struct Codes<true> {
  half8 x[4];
  __device__ __forceinline__ Codes() {}
  __device__ __forceinline__ Codes(int4v lo, int4v hi) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = (uint32_t)(i < 2 ? lo[2 * i] : hi[2 * i - 4]), b = (uint32_t)(i < 2 ? lo[2 * i + 1] : hi[2 * i - 3]);
      x[i] = __builtin_bit_cast(half8, uint4v{codes<f16>::widen(a, 0), codes<f16>::widen(a, 1),
                                              codes<f16>::widen(b, 0), codes<f16>::widen(b, 1)});
    }
  }
};

// 16x16 dot products of 128 values.
__device__ __forceinline__ float4v dots(const Codes<false>& a, const Codes<false>& b) {
  // zeros: without the instruction's own scales
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.x, b.x, float4v{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ float4v dots(const Codes<true>& a, const Codes<true>& b) {
  float4v c = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 4; ++i) c = mfma_16x16x32(a.x[i], b.x[i], c);
  return c;
}

// The operand of one row's block: bytes 16 g and 64 + 16 g on, zeros from ``left`` on.
__device__ __forceinline__ Codes<true> operand(const uint8_t* p, int g, int left) {
  int4v lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
  if (16 * g < left) lo = *reinterpret_cast<const int4v*>(p + 16 * g);
  if (64 + 16 * g < left) hi = *reinterpret_cast<const int4v*>(p + 64 + 16 * g);
  return Codes<true>(lo, hi);
}

template <class T> __device__ __forceinline__ float bias_of(const ScaledProductArgs& a, int n) {
  return a.wide_bias ? at<float>(a.bias, a.c_off)[n] : element<T>::widen(at<T>(a.bias, a.c_off)[n]);
}

// Few rows: the weight is read once and is all that counts. A workgroup has 16 of its rows and
// up to 16 * MT rows of a; its waves take blocks of the sum in turn and meet in LDS.
template <class T, int MT, int WAVES>
__device__ __forceinline__ void scaled_product_rows(const ScaledProductArgs& a) {
  __shared__ __attribute__((aligned(16))) float4v parts[WAVES][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4, n0 = blockIdx.x * 16;
  const int nr = n0 + r < a.n ? n0 + r : a.n - 1;
  const uint8_t* const b = at<uint8_t>(a.b, a.b_off) + (int64_t)nr * a.br;
  const float* const bs = at<float>(a.b_scales, a.bs_off) + (int64_t)(n0 / 128) * a.bsr;
  const uint8_t* x[MT];
  const float* xs[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = 16 * i + r < a.rows ? 16 * i + r : a.rows - 1;
    x[i] = at<uint8_t>(a.a, a.a_off) + m / a.seq * a.ab + m % a.seq * a.at;
    xs[i] = at<float>(a.a_scales, a.as_off) + m / a.seq * a.asb + m % a.seq * a.ast;
  }
  float4v sum[MT] = {};
  const int blocks = (a.k + 127) / 128;
  for (int i = wave; i < blocks; i += WAVES) {
    const int left = a.k - 128 * i;
    const auto w = operand(b + 128 * i, g, left);
    const float s = bs[i * a.bss];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const float4v p = dots(w, operand(x[j] + 128 * i, g, left));
      const float f = xs[j][i * a.ass] * s;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[j][e] = __builtin_fmaf(p[e], f, sum[j][e]);
    }
  }
#pragma unroll
  for (int j = 0; j < MT; ++j) parts[wave][j][lane] = sum[j];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 64; i += 64 * WAVES) {
    const int j = i / 64, l = i % 64, m = 16 * j + (l & 15), n = n0 + 4 * (l >> 4);
    float4v s = parts[0][j][l];
#pragma unroll
    for (int w = 1; w < WAVES; ++w)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += parts[w][j][l][e];
    if (m >= a.rows) continue;
    T* const out = reinterpret_cast<T*>(a.out) + (int64_t)m * a.n + n;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.n) out[e] = element<T>::narrow(s[e] + (a.bias ? bias_of<T>(a, n + e) : 0.0f));
  }
}

// Many rows: tiles of BM rows of a and BN of the weight, WM x WN waves. Blocks of both pass
// through LDS, STAGES - 1 of them on their way while one is in use. A row is 8 pieces of 16 bytes, piece
// c of row r in slot c ^ (r / 2 % 8): the same piece of 16 rows lies in 64 distinct banks.
// A buffer's offsets of 32 bits reach a tile of rows with one stride from its first, and others from
// the tensor's; what lies past the last row or value has an offset past the buffer's end, and is zeros.
constexpr uint32_t OUTSIDE = 0x80000000u;

template <class T, int BM, int BN, int WM, int WN, int STAGES>
__device__ __forceinline__ void scaled_product_tiles(const ScaledProductArgs& a) {
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int WAVES = WM * WN, THREADS = 64 * WAVES, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int LA = BM * 8 / THREADS, LB = BN * 8 / THREADS, STEP = THREADS / 8;
  constexpr int TILE = (BM + BN) * 128, STAGE = TILE + BM * 4;
  static_assert(STEP % 16 == 0 && LA >= 1 && LB >= 1 && BN / WN <= 128 && BM % 64 == 0, "staging");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * STAGE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int col_tiles = (a.n + BN - 1) / BN;
  // neighbouring workgroups go to the 8 XCDs in turn: each XCD gets a run of tiles
  int w = blockIdx.x;
  const int split = w % a.splits;
  w /= a.splits;
  const int all = a.row_tiles * col_tiles;
  {
    const int per = all / 8, more = all % 8, x = w % 8, y = w / 8;
    w = x * per + (x < more ? x : more) + y;
  }
  // in bands of 8 row tiles
  int mt, nt;
  {
    constexpr int BAND = 8;
    const int band = w / (BAND * col_tiles), first = band * BAND;
    const int high = a.row_tiles - first < BAND ? a.row_tiles - first : BAND;
    const int in = w - first * col_tiles;
    mt = first + in % high;
    nt = in / high;
  }
  const int m0 = mt * BM, n0 = nt * BN;
  const int wm = wave % WM, wn = wave / WM;
  const int blocks = (a.k + 127) / 128;
  const int begin = (int)((int64_t)blocks * split / a.splits), end = (int)((int64_t)blocks * (split + 1) / a.splits);

  const int own = threadIdx.x / 8, chunk = (threadIdx.x & 7) ^ (own >> 1 & 7);
  const int base = a.regular ? m0 : 0;
  auto offset = [&](int m, int64_t batch, int64_t token) {
    m += m0 - base;
    return a.regular ? m * (uint32_t)token : m / a.seq * (uint32_t)batch + m % a.seq * (uint32_t)token;
  };
  const auto ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(at<uint8_t>(a.a, a.a_off) + base * a.at), 0, OUTSIDE, 0x27000);
  const auto rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(at<uint8_t>(a.b, a.b_off) + n0 * a.br), 0, OUTSIDE, 0x27000);
  const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(at<float>(a.a_scales, a.as_off) + base * a.ast), 0, OUTSIDE, 0x27000);
  uint32_t va[LA], vb[LB];
#pragma unroll
  for (int i = 0; i < LA; ++i) {
    const int m = own + i * STEP;
    va[i] = m0 + m < a.rows ? offset(m, a.ab, a.at) : OUTSIDE;
  }
#pragma unroll
  for (int i = 0; i < LB; ++i) {
    const int n = own + i * STEP;
    vb[i] = n0 + n < a.n ? n * (uint32_t)a.br : OUTSIDE;
  }
  const int sr = (wave * 64 + lane) % BM;
  const uint32_t vs = m0 + sr < a.rows ? offset(sr, a.asb, a.ast) * 4 : OUTSIDE;
  const int nb = (n0 + wn * (BN / WN)) / 128;
  const float* const bs = at<float>(a.b_scales, a.bs_off) + (nb < (a.n + 127) / 128 ? nb : 0) * a.bsr;
  // the weight's scales of 64 steps, one a lane: a load in every step would wait for the tiles on
  // their way (a vector's) or for the reads of LDS (a scalar's)
  float held = 0.0f;

  auto load = [&](int i, int into) __attribute__((always_inline)) {
    const uint32_t piece = 128 * i + 16 * chunk < a.k ? 16 * chunk : OUTSIDE;
    uint8_t* const to = lds + into * STAGE + wave * 1024;
#pragma unroll
    for (int l = 0; l < LA; ++l)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (__attribute__((address_space(3))) void*)(to + l * THREADS * 16), 16, va[l] | piece, i * 128, 0, 0);
#pragma unroll
    for (int l = 0; l < LB; ++l)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (__attribute__((address_space(3))) void*)(to + BM * 128 + l * THREADS * 16), 16, vb[l] | piece, i * 128, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(lds + into * STAGE + TILE + wave * 64 % BM * 4), 4, vs, i * (int)a.ass * 4, 0, 0);
  };
  float4v sum[TN][TM] = {};
  const int swizzle = r >> 1 & 7;
  const uint32_t a_at = (wm * TM * 16 + r) * 128, b_at = BM * 128 + (wn * TN * 16 + r) * 128;
  const uint32_t lo = (g ^ swizzle) * 16, hi = ((4 + g) ^ swizzle) * 16, s_at = TILE + (wm * TM * 16 + r) * 4;
  auto compute = [&](int i, int stage) __attribute__((always_inline)) {
    const uint8_t* const from = lds + stage * STAGE;
    auto read = [&](uint32_t row) __attribute__((always_inline)) {
      return Codes<EXACT>(*reinterpret_cast<const int4v*>(from + row + lo), *reinterpret_cast<const int4v*>(from + row + hi));
    };
    const float by = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, held), (i - begin) & 63));
    Codes<EXACT> x[TM], y = read(b_at), z;
    float s[TM];
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      s[j] = *reinterpret_cast<const float*>(from + s_at + j * 64) * by;
      x[j] = read(a_at + j * 2048);
    }
    float4v p[2][TM];
#pragma unroll
    for (int l = 0; l <= TN; ++l) {
      if (l + 1 < TN) z = read(b_at + (l + 1) * 2048);
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        if (l < TN) p[l & 1][j] = dots(y, x[j]);
        if (l > 0)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[l - 1][j][e] = __builtin_fmaf(p[l - 1 & 1][j][e], s[j], sum[l - 1][j][e]);
      }
      y = z;
      // a product, then the four additions of one before, whose result is there by then
      if (!EXACT && l > 0 && l < TN) {
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // no reads further ahead: registers
    }
  };
  constexpr int LOADS = LA + LB + 1;
  const int steps = end - begin;
#pragma unroll
  for (int p = 0; p < STAGES - 1; ++p)
    if (p < steps) load(begin + p, p);
  int stage = 0;
  for (int i = 0; i < steps; ++i) {
    if ((i & 63) == 0) held = bs[(begin + i + lane < end ? begin + i + lane : end - 1) * a.bss];
    // all but the loads of the steps after this one
    if (STAGES > 2 && i + STAGES - 1 <= steps)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(LOADS * (STAGES - 2)) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    if (i + STAGES - 1 < steps) load(begin + i + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
    compute(begin + i, stage);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
#pragma unroll
  for (int l = 0; l < TN; ++l)
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int m = m0 + (wm * TM + j) * 16 + r, n = n0 + (wn * TN + l) * 16 + 4 * g;
      if (m >= a.rows) continue;
      if (a.splits > 1) {
        float* const part = a.part + ((int64_t)split * a.rows + m) * a.n + n;
        if (n + 4 <= a.n) {
          const float y[4] = {sum[l][j][0], sum[l][j][1], sum[l][j][2], sum[l][j][3]};
          store_n<4>(part, y);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < a.n) part[e] = sum[l][j][e];
        }
      } else {
        T* const out = reinterpret_cast<T*>(a.out) + (int64_t)m * a.n + n;
        T y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          y[e] = element<T>::narrow(sum[l][j][e] + (a.bias && n + e < a.n ? bias_of<T>(a, n + e) : 0.0f));
        if (n + 4 <= a.n) {
          store_n<(int)sizeof(T)>(out, y);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < a.n) out[e] = y[e];
        }
      }
    }
}

// The sum of the parts that splits of the blocks have left.
constexpr int JOIN_BLOCK = 256;
template <class T> __device__ __forceinline__ void scaled_product_join(const ScaledProductArgs& a) {
  const int64_t i = (int64_t)blockIdx.x * JOIN_BLOCK + threadIdx.x, all = (int64_t)a.rows * a.n;
  if (i >= all) return;
  float s = 0.0f;
  for (int p = 0; p < a.splits; ++p) s += a.part[p * all + i];
  if (a.bias) s += bias_of<T>(a, (int)(i % a.n));
  reinterpret_cast<T*>(a.out)[i] = element<T>::narrow(s);
}

}  // namespace mlc

#define SCALED_PRODUCT_TILES(NAME, T, BM, BN, WM, WN, STAGES)                                  \
  extern "C" __global__ void __launch_bounds__(64 * WM * WN) NAME(mlc::ScaledProductArgs a) {  \
    mlc::scaled_product_tiles<T, BM, BN, WM, WN, STAGES>(a);                                   \
  }
#define SCALED_PRODUCT_JOIN(NAME, T)                                                                \
  extern "C" __global__ void __launch_bounds__(mlc::JOIN_BLOCK) NAME(mlc::ScaledProductArgs a) {    \
    mlc::scaled_product_join<T>(a);                                                                 \
  }
#define SCALED_PRODUCT_ROWS(NAME, T, MT, WAVES)                                                 \
  extern "C" __global__ void __launch_bounds__(64 * WAVES) NAME(mlc::ScaledProductArgs a) {     \
    mlc::scaled_product_rows<T, MT, WAVES>(a);                                                  \
  }
