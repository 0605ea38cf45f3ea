// Products of 8-bit rows whose scales change every 128 values of the sum:
//
//   out[m, n] = sum over blocks i of  sa[m, i] * sb[n / 128, i] * (a[m, i] . b[n, i])  + bias[n]
//
// A block's dot products come from matrix instructions begun at zero; their fp32 result is added
// to the sum with the block's two scales as its factor.
//
// The 8-bit instruction (16x16x128) takes neighbouring products by eights and cuts them at
// 2^-13 of the power of two of a group's largest: a sum of random values is 1.3e-5 to 3e-5 of itself off, which is
// a tenth of what a result's rounding to fp16 takes and a hundredth of bf16's; where large terms cancel it is that much
// of them. Many rows with such results use it. Results in fp32, and few rows, where the weight's way from memory is all
// that counts, use the fp16 one on widened codes, which is exact: 2e-8 to 5e-8.
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
      const uint32_t a = (uint32_t)(i < 2 ? lo[2 * i] : hi[2 * i - 4]);
      const uint32_t b = (uint32_t)(i < 2 ? lo[2 * i + 1] : hi[2 * i - 3]);
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

// The first ``count`` of N values, or all.
template <int A, int N, class T> __device__ __forceinline__ void store_some(T* p, const T (&x)[N], int count) {
  if (count >= N) {
    store_n<A>(p, x);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < count) p[e] = x[e];
  }
}

template <class T> __device__ __forceinline__ float bias_of(const ScaledProductArgs& a, int n) {
  return a.wide_bias ? at<float>(a.bias, a.c_off)[n] : element<T>::widen(at<T>(a.bias, a.c_off)[n]);
}

// Up to 16 rows: the weight is read once and is all that counts. A workgroup has 16 of its rows and
// all of a's; its waves take U blocks of the sum in turn, whose operands they ask for at once, and
// meet in LDS. 1 row, 4096 -> 6144 8.6 us, 12288 -> 4096 10.9, 4.6 TB/s.
template <class T, int U, int WAVES> __device__ __forceinline__ void scaled_product_rows(const ScaledProductArgs& a) {
  __shared__ __attribute__((aligned(16))) float4v parts[WAVES][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4, n0 = blockIdx.x * 16;
  const int nr = n0 + r < a.n ? n0 + r : a.n - 1, mr = r < a.rows ? r : a.rows - 1;
  const uint8_t* const b = at<uint8_t>(a.b, a.b_off) + nr * a.br + 16 * g;
  const float* const bs = at<float>(a.b_scales, a.bs_off) + n0 / 128 * a.bsr;
  const uint8_t* const x = at<uint8_t>(a.a, a.a_off) + mr / a.seq * a.ab + mr % a.seq * a.at + 16 * g;
  const float* const xs = at<float>(a.a_scales, a.as_off) + mr / a.seq * a.asb + mr % a.seq * a.ast;
  float4v sum = {0.0f, 0.0f, 0.0f, 0.0f};
  const int blocks = (a.k + 127) / 128;
  // a row's block: bytes 16 g and 64 + 16 g on, zeros past the row's end
  auto take = [&](const uint8_t* p, int i, int4v (&v)[2]) __attribute__((always_inline)) {
    const int left = a.k - 128 * i - 16 * g;
    v[0] = v[1] = int4v{0, 0, 0, 0};
    if (left > 0) v[0] = *reinterpret_cast<const int4v*>(p + 128 * (int64_t)i);
    if (left > 64) v[1] = *reinterpret_cast<const int4v*>(p + 128 * (int64_t)i + 64);
  };
  for (int i0 = wave * U; i0 < blocks; i0 += WAVES * U) {
    int4v w[U][2], c[U][2];
    float scale[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int in = i0 + u < blocks ? i0 + u : blocks - 1;
      take(b, i0 + u, w[u]);
      take(x, i0 + u, c[u]);
      scale[u] = xs[in * a.ass] * bs[in * a.bss];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u >= blocks) break;  // scales of a block that is not there may be infinite
      const float4v p = dots(Codes<true>(w[u][0], w[u][1]), Codes<true>(c[u][0], c[u][1]));
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(p[e], scale[u], sum[e]);
    }
  }
  parts[wave][lane] = sum;
  __syncthreads();
  const int m = r, n = n0 + 4 * g;
  if (wave > 0 || m >= a.rows) return;
#pragma unroll
  for (int w = 1; w < WAVES; ++w)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += parts[w][lane][e];
  T v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = element<T>::narrow(sum[e] + (a.bias && n + e < a.n ? bias_of<T>(a, n + e) : 0.0f));
  store_some<(int)sizeof(T)>(reinterpret_cast<T*>(a.out) + (int64_t)m * a.n + n, v, a.n - n);
}

// Many rows: tiles of BM rows of a and BN of the weight, WM x WN waves. Two blocks of both are in LDS
// or on their way there. A row is 8 pieces of 16 bytes, piece c of row r in slot c ^ (r / 2 % 8): the
// same piece of 16 rows lies in 64 distinct banks.
//
// A wave keeps its rows of a in registers for a block and takes the weight's 16 by 16; each such row
// of products begins when the one before is added. The weight's rows come in LB parts, each
// with a barrier of its own: what has been read is free, and is asked for again for the block after
// the next, nearly two blocks ahead (one ahead, with a barrier a block, 8192 rows, 12288 -> 4096 take 405 us and
// with these 350). No branch lies between the rows: additions would be moved behind it, and their products
// would not fit the registers.
//
// A buffer's offsets of 32 bits reach a tile of rows with one stride from its first, and others from
// the tensor's; what lies past the last row or value has an offset past the buffer's end, and is zeros.
constexpr uint32_t OUTSIDE = 0x80000000u;

template <class T, int BM, int BN, int WM, int WN>
__device__ __forceinline__ void scaled_product_tiles(const ScaledProductArgs& a) {
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int WAVES = WM * WN, THREADS = 64 * WAVES, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int LA = BM * 8 / THREADS, LB = BN * 8 / THREADS, STEP = THREADS / 8;  // loads, and rows of one
  constexpr int R = TN / LB;                                                       // rows of products of a part
  constexpr int STAGE = (BM + BN) * 128, GROUP = 8, SCALES = BM * GROUP * 4;       // scales of 8 blocks
  static_assert(LA >= 1 && LB >= 2 && R * LB == TN && R * 16 * WN == STEP && BN / WN <= 128, "staging");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * STAGE + 2 * SCALES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int col_tiles = (a.n + BN - 1) / BN;
  int w = blockIdx.x;
  const int split = w % a.splits;
  w /= a.splits;
  const int all = a.row_tiles * col_tiles;
  {  // neighbouring workgroups go to the 8 XCDs in turn: each XCD gets a run of tiles
    const int per = all / 8, more = all % 8, x = w % 8, y = w / 8;
    w = x * per + (x < more ? x : more) + y;
  }
  int mt, nt;
  {  // in bands of 4 row tiles
    constexpr int BAND = 4;
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
  const int steps = end - begin;

  const int base = a.regular ? m0 : 0;
  auto offset = [&](int m, int64_t batch, int64_t token) {
    m += m0 - base;
    return a.regular ? m * (uint32_t)token : m / a.seq * (uint32_t)batch + m % a.seq * (uint32_t)token;
  };
  auto buffer_at = [](const void* p) __attribute__((always_inline)) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, OUTSIDE, 0x27000);
  };
  const auto ra = buffer_at(at<uint8_t>(a.a, a.a_off) + base * a.at);
  const auto rb = buffer_at(at<uint8_t>(a.b, a.b_off) + n0 * a.br);
  const auto rs = buffer_at(at<float>(a.a_scales, a.as_off) + base * a.ast);
  const int own = threadIdx.x / 8, chunk = (threadIdx.x & 7) ^ (own >> 1 & 7);
  uint32_t va[LA], vb[LB];
#pragma unroll
  for (int i = 0; i < LA; ++i) {
    const int m = own + i * STEP;
    va[i] = m0 + m < a.rows ? offset(m, a.ab, a.at) + 16 * chunk : OUTSIDE;
  }
#pragma unroll
  for (int i = 0; i < LB; ++i) {  // a part has R * 16 rows of each column of waves
    const int n = own / (R * 16) * (TN * 16) + i * R * 16 + own % (R * 16);
    vb[i] = n0 + n < a.n ? n * (uint32_t)a.br + 16 * chunk : OUTSIDE;
  }
  typedef __attribute__((address_space(3))) void* lds_ptr;
  auto past = [&](int i) { return i < end && 128 * i + 16 * chunk < a.k ? 0u : OUTSIDE; };
  auto load_a = [&](int i) __attribute__((always_inline)) {
    uint8_t* const to = lds + (i - begin & 1) * STAGE + wave * 1024;
#pragma unroll
    for (int l = 0; l < LA; ++l)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr)(to + l * THREADS * 16), 16, va[l] | past(i), i * 128, 0, 0);
  };
  auto load_b = [&](int i, int l) __attribute__((always_inline)) {
    uint8_t* const to = lds + (i - begin & 1) * STAGE + wave * 1024 + BM * 128;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_ptr)(to + l * THREADS * 16), 16, vb[l] | past(i), i * 128, 0, 0);
  };
  // Scales of a's rows for 8 blocks: row by row they lie far apart, and a load for each block would
  // take as many requests as the codes. In pieces of 4 where no piece crosses a row's end.
  const bool fours = a.ass == 1 && (blocks - begin & 3) == 0;
  auto load_scales = [&](int i) __attribute__((always_inline)) {
    uint8_t* const to = lds + 2 * STAGE + (i - begin & GROUP ? SCALES : 0);
#pragma unroll
    for (int at_row = wave * 32; at_row < BM; at_row += WAVES * 32) {  // 1024 bytes at a time
      if (fours) {
        const int m = at_row + lane / 2, block = i + lane % 2 * 4;
        const uint32_t v = m0 + m < a.rows && block < blocks ? offset(m, a.asb, a.ast) * 4 + block * 4 : OUTSIDE;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(to + at_row * GROUP * 4), 16, v, 0, 0, 0);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int m = at_row + q * 8 + lane / 8, block = i + lane % 8;
          const uint32_t far = (offset(m, a.asb, a.ast) + block * (uint32_t)a.ass) * 4;
          const uint32_t v = m0 + m < a.rows && block < blocks ? far : OUTSIDE;
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(to + (at_row + q * 8) * GROUP * 4), 4, v, 0, 0, 0);
        }
      }
    }
  };
  // the weight's scales of 64 blocks, one a lane
  const int nb = (n0 + wn * (BN / WN)) / 128;
  const float* const bs = at<float>(a.b_scales, a.bs_off) + (nb < (a.n + 127) / 128 ? nb : 0) * a.bsr;
  float held = 0.0f;

  float4v sum[TN][TM] = {}, p[TM] = {};
  const int swizzle = r >> 1 & 7;
  const uint32_t lo = (g ^ swizzle) * 16, hi = ((4 + g) ^ swizzle) * 16;
  const uint32_t a_at = (wm * TM * 16 + r) * 128, b_at = BM * 128 + (wn * R * 16 + r) * 128;
  auto read = [&](const uint8_t* from) __attribute__((always_inline)) {
    return Codes<EXACT>(*reinterpret_cast<const int4v*>(from + lo), *reinterpret_cast<const int4v*>(from + hi));
  };
  auto part_of = [&](int l) { return b_at + (l / R * STEP + l % R * 16) * 128; };
  // Part s of step i is there for everyone, and what lies in front of it has been read: its place
  // is filled again. Loads end in order; the counts are of those that were asked for later.
  auto arrive = [&](int i, int s) __attribute__((always_inline)) {
    if (s < 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(LA + 2 * LB - 2) : "memory");
    else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(2 * LA + 2 * LB - 2) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    if (s == 0) {
      load_b(i + 1, LB - 1);
    } else {
      if (s == 1) load_a(i + 2);
      load_b(i + 2, s - 1);
    }
  };
  load_scales(begin);
  load_a(begin);
#pragma unroll
  for (int l = 0; l < LB; ++l) load_b(begin, l);
  load_a(begin + 1);
#pragma unroll
  for (int l = 0; l < LB - 1; ++l) load_b(begin + 1, l);
  arrive(begin, 0);
  Codes<EXACT> x[TM], y, z;
#pragma unroll
  for (int j = 0; j < TM; ++j) x[j] = read(lds + a_at + j * 2048);
  y = read(lds + part_of(0));
  float before[TM] = {};  // the scales of the step before
  for (int i = 0; i < steps; ++i) {
    if (i % GROUP == 0) load_scales(begin + i + GROUP);
    if (i % 64 == 0) {
      held = bs[(begin + i + lane < end ? begin + i + lane : end - 1) * a.bss];
      asm volatile("" : "+v"(held));  // waits here, and in no other step
    }
    const float by = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, held), i % 64));
    const uint8_t* const from = lds + (i & 1) * STAGE;
    const uint8_t* const next = lds + (~i & 1) * STAGE;
    const float* const scales = reinterpret_cast<const float*>(lds + 2 * STAGE + (i & GROUP ? SCALES : 0)) + i % GROUP;
    float s[TM];
#pragma unroll
    for (int j = 0; j < TM; ++j) s[j] = scales[((wm * TM + j) * 16 + r) * GROUP] * by;
#pragma unroll
    for (int l = 0; l < TN; ++l) {
      if (l % R < R - 1) {
        z = read(from + part_of(l + 1));
      } else if (l + 1 < TN) {
        arrive(begin + i, l / R + 1);
        z = read(from + part_of(l + 1));
      } else {
        arrive(begin + i + 1, 0);
        z = read(next + part_of(0));
      }
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const float by_row = l > 0 ? s[j] : before[j];
        float4v& to = sum[l > 0 ? l - 1 : TN - 1][j];
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = __builtin_fmaf(p[j][e], by_row, to[e]);
        p[j] = dots(y, x[j]);
        if (l + 1 == TN) x[j] = read(next + a_at + j * 2048);  // as this step's goes
      }
      y = z;
      if (!EXACT && l > 0 && l + 1 < TN) {
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // no reads further ahead: registers
    }
#pragma unroll
    for (int j = 0; j < TM; ++j) before[j] = s[j];
  }
#pragma unroll
  for (int j = 0; j < TM; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[TN - 1][j][e] = __builtin_fmaf(p[j][e], before[j], sum[TN - 1][j][e]);
  asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // the zeros behind the last step are in LDS too
  const int first_m = m0 + wm * TM * 16, first_n = n0 + wn * TN * 16;
  auto bias_from = [&](int n, float (&add)[4]) __attribute__((always_inline)) {
    if (a.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < a.n) add[e] = bias_of<T>(a, n + e);
    }
  };
  if (EXACT || a.splits > 1) {  // four fp32 values are a piece
    const bool parts = a.splits > 1;
    float* const out = parts ? a.part + (int64_t)split * a.rows * a.n : reinterpret_cast<float*>(a.out);
#pragma unroll
    for (int l = 0; l < TN; ++l) {
      const int n = first_n + l * 16 + 4 * g;
      float add[4] = {};
      if (!parts) bias_from(n, add);
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const int m = first_m + j * 16 + r;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = sum[l][j][e] + add[e];
        if (m < a.rows) store_some<4>(out + (int64_t)m * a.n + n, v, a.n - n);
      }
    }
    return;
  }
  // A wave's results go through LDS, so that rows are written in 16-byte pieces side by side: lanes
  // hold four values of 16 rows, and stores of 8 bytes took 24 us a tile of 256 x 256. Pieces
  // of a row are xor-ed with its number, as the tiles'.
  constexpr int SIZE = sizeof(T), PIECES = TN * SIZE, EACH = 16 / SIZE;
  static_assert(EXACT || WAVES * TM * 16 * PIECES * 16 <= 2 * STAGE, "results in LDS");
  __syncthreads();
  uint8_t* const own_lds = lds + wave * (TM * 16 * PIECES * 16);
  auto slot = [&](int row, int piece) __attribute__((always_inline)) {
    return (row * PIECES + (piece ^ (PIECES >= 16 ? row & 15 : PIECES == 8 ? row >> 1 & 7 : row >> 2 & 3))) * 16;
  };
#pragma unroll
  for (int l = 0; l < TN; ++l) {
    float add[4] = {};
    bias_from(first_n + l * 16 + 4 * g, add);
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      T v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = element<T>::narrow(sum[l][j][e] + add[e]);
      const int at_byte = (l * 16 + 4 * g) * SIZE;
      store_n<4 * SIZE>(reinterpret_cast<T*>(own_lds + slot(j * 16 + r, at_byte / 16) + at_byte % 16), v);
    }
  }
  // a wave's own part of LDS: its writes are in order before its reads
#pragma unroll
  for (int i = lane; i < TM * 16 * PIECES; i += 64) {
    const int row = i / PIECES, piece = i % PIECES, m = first_m + row, n = first_n + piece * EACH;
    T v[EACH];
    load_n<16>(v, reinterpret_cast<const T*>(own_lds + slot(row, piece)));
    if (m < a.rows) store_some<SIZE>(reinterpret_cast<T*>(a.out) + (int64_t)m * a.n + n, v, a.n - n);
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

#define SCALED_PRODUCT_TILES(NAME, T, BM, BN, WM, WN)                                          \
  extern "C" __global__ void __launch_bounds__(64 * WM * WN) NAME(mlc::ScaledProductArgs a) {  \
    mlc::scaled_product_tiles<T, BM, BN, WM, WN>(a);                                           \
  }
#define SCALED_PRODUCT_JOIN(NAME, T)                                                                \
  extern "C" __global__ void __launch_bounds__(mlc::JOIN_BLOCK) NAME(mlc::ScaledProductArgs a) {    \
    mlc::scaled_product_join<T>(a);                                                                 \
  }
#define SCALED_PRODUCT_ROWS(NAME, T, U, WAVES)                                                  \
  extern "C" __global__ void __launch_bounds__(64 * WAVES) NAME(mlc::ScaledProductArgs a) {     \
    mlc::scaled_product_rows<T, U, WAVES>(a);                                                   \
  }
