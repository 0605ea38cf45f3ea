// Attention of queries over keys and values in 16 bits, with the masks made from
// indices instead of read: out = softmax(mask(bias(cap(scale q k^T)))) v, fp32
// softmax, a row with nothing visible all zeros.
//
// Rows are (token, head of a group) pairs: all heads that share keys and values
// go through one workgroup, which so reads them once. A workgroup of 4 waves has
// 128 rows, a wave 32 of them, one row in lanes c and c + 32. Keys pass in tiles
// of 64 through LDS. Where there are few rows its waves have the same 32 instead, and a
// quarter of the tiles each (APART).
//  * S^T = K Q^T on 32x32x16 products: lane (c, h) ends with row c's scores. The
//    rows of K are taken in the order that makes them tokens 16 i + 8 h .. + 7,
//    the B operand of O^T = V^T P^T: probabilities never leave their lane.
//  * V^T's operand is read transposed from V's rows (ds_read_b64_tr_b16).
//  * The softmax is online: a running maximum, the sum and O scaled when it grows.
//
// Long rows are bound by the softmax's vector work beside the products, and by the clock,
// which falls under them and differs from card to card: 8192 tokens, 32 heads over 8 of 128,
// bf16, causal 550 to 570 us, 970 TFLOP/s, without a mask 1100 us, 1000 TFLOP/s (a library's
// product of 8192^3 reaches 1214); a cap adds two transcendentals to a score's one, 660 to 715
// us, 800 TFLOP/s. Short ones are bound by a chain of loads and products that few waves hide:
// 32 x 512 tokens, 12 heads of 64, fp16, causal 34 us, with a bias and prefixes 38 to 40 (19 to
// move the bytes), vector units 55 % and matrix units 15 % of the time busy; 128 tokens, 12 heads
// 5.3. 4 x 2048 tokens, 8 heads of 256, causal 107 us for 57 of products: tiles of 32 keys, each
// behind a wait and a barrier, two waves a SIMD.
//
// Tried and slower: 8 waves a workgroup and 4 buffers (916 against 960 TFLOP/s then), the
// scores of a tile before the softmax of the one before (registers spill), the sums as one
// more product.

namespace mlc {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));

struct AttentionArgs {
  const void* q;
  const void* k;
  const void* v;
  const void* slopes;     // null: no bias by distance
  const void* documents;  // null: one document
  const void* prefix;     // null: none
  void* out;
  float* part;  // where keys are split: [split][pair][row][dim + 4], see join_parts
  const void* k_scale;  // and what follows: of an 8-bit cache
  const void* v_scale;
  const void* start;
  const void* count;  // null: every token is real
  int* error;
  int64_t q_off, k_off, v_off, s_off, d_off, p_off;      // bytes
  int64_t ks_off, vs_off, start_off, count_off;
  int64_t qb, qt, qh, kb, kt, kh, vb, vt, vh, ss, db, dt, ps, start_s, count_s;  // elements
  int32_t batch, queries, keys, kv_heads, group, dim, causal, tiles;  // tiles of rows
  int32_t splits, block_shift;  // of keys; tokens of a scale
  float scale, cap;  // scale times log2 e where cap is 0, else 1/cap of it and cap log2 e
};

// Keys of a tile: with heads of 256, rows of 64 scores would not fit the registers beside O
// and Q, and O would move between vector and accumulation registers twice a tile (2048 causal
// tokens, 4 x 8 heads of 256: 136 us; 32 keys 116). A tile of the cache has one scale.
// Where waves take keys apart, four tiles of 32 rows of 128 values have room in LDS.
template <int DP, int SOURCE, bool APART>
constexpr int tile_keys = DP == 256 || SOURCE == 2 || (APART && DP > 64) ? 32 : 64;

template <class T> struct vec8;
template <> struct vec8<f16> {
  typedef half8 type;
  static constexpr uint32_t exponent = 0x7c00u;
  static constexpr float lift = 7.0f;  // see LIFT
  static constexpr float least = 0x1p-24f;
};
template <> struct vec8<__bf16> {
  typedef bf16x8 type;
  static constexpr uint32_t exponent = 0x7f80u;
  static constexpr float lift = -40.0f;
  static constexpr float least = 0x1p-126f;
};

__device__ __forceinline__ float16v mfma_32x32x16(half8 a, half8 b, float16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float16v mfma_32x32x16(bf16x8 a, bf16x8 b, float16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// 16-byte slot of chunk ``c`` of row ``r``: a row is PC slots of 256 (DP 64: 128)
// bytes and its slots are xor-ed with its number, so that 16 rows of one chunk,
// and 4 rows of 4 chunks, each lie in 64 distinct banks.
template <int PC> __device__ __forceinline__ int slot(int r, int c) {
  if constexpr (PC == 8) return r * 8 + (c ^ ((((r >> 1) & 1) << 2) | ((r >> 2) & 3)));
  return r * PC + (c ^ (((r & 3) << 2) | ((r >> 2) & 3)));
}

// Four tokens of 16 values, one a lane: lane i of 16 gives the address of values
// 4 (i % 4) .. + 3 of token i / 4 and gets value i of the four tokens.
__device__ __forceinline__ h4 read_transposed(const void* p) {
  return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) short4v*)p));
}

// Zeros in the place of what is infinite or NaN (all of exponent E set) among 8
// values of 16 bits; whether there was any.
template <uint32_t E> __device__ __forceinline__ bool drop_not_finite(uint4v& x) {
  bool found = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool lo = (x[i] & E) == E, hi = (x[i] & (E << 16)) == (E << 16);
    found |= lo || hi;
    x[i] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
  }
  return found;
}

template <bool B, class X, class Y> struct choose { typedef X type; };
template <class X, class Y> struct choose<false, X, Y> { typedef Y type; };

// 16 bytes of a lane from ``g`` straight to LDS at ``lds`` + 16 * lane.
__device__ __forceinline__ void to_lds(const void* g, void* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// SOURCE of keys and values:
//  DIRECT: rows of 16-byte aligned pieces, dim == DP: tiles go from memory to LDS without
//    passing registers, the next one while one is in use;
//  COPIED: through registers, with zeros past dim;
//  CODES: the 8-bit cache of cache_attention, for many rows: codes are widened on their way
//    to LDS, K's in the queries' type and V's, with P, in fp16, both exact; a scale of K goes
//    into the factor of its scores, one of V multiplies its keys' part of O.
enum { COPIED, DIRECT, CODES };

// APART: the waves of a workgroup have the same 32 rows and take tiles of keys in turn, each
// with LDS of its own and no barrier until their parts of O are joined there. Few workgroups
// wait for a row's tiles one behind the other: 128 tokens, 12 heads of 64 5.6 us for 7.2 in
// workgroups of 128 rows, 1000 tokens 12.3 for 19.3.
// SCORES that are more than products: PLAIN none, BIASED a cap or a bias, DOCUMENTS both and
// documents. Apart, since what a kernel does not use still takes its registers: 32 x 512 tokens,
// 12 heads of 64 with a bias 45 us in a kernel that looks for documents too, 39 without.
enum { PLAIN, BIASED, DOCUMENTS };
// Waves that a SIMD has to have registers for. More hide more, where nothing spills: with a
// cap and documents, 6 x 999 tokens, 8 heads of 256 56 us for one and 66 for two, plain 2048
// tokens of them 133 and 121; 8 x 512, 12 heads of 64 with documents 19.2 for two, 20.6 three.
constexpr int waves_a_simd(int dp, int scores, bool apart) {
  return dp == 256 && scores != PLAIN ? 1 : dp == 64 && scores != DOCUMENTS && !apart ? 3 : 2;
}

template <class T, int DP, int WAVES, int SOURCE, int SCORES, bool APART>
__device__ __forceinline__ void attention(const AttentionArgs& a) {
  typedef typename vec8<T>::type v8;
  typedef typename choose<SOURCE == CODES, f16, T>::type PT;  // of P and V
  typedef typename vec8<PT>::type p8;
  constexpr bool IS_DIRECT = SOURCE == DIRECT, CACHE = SOURCE == CODES;
  constexpr bool GENERAL = SCORES != PLAIN, DOCS = SCORES == DOCUMENTS;
  constexpr int PC = DP == 64 ? 8 : DP <= 128 ? 16 : 32;  // 16-byte slots of an LDS row
  constexpr int CH = DP / 8;                               // of which hold values
  constexpr int TEAMS = APART ? WAVES : 1, TEAM = WAVES / TEAMS;  // waves that share tiles of keys
  constexpr int THREADS = 64 * TEAM, ROWS = 32 * TEAM;
  constexpr int BUFFERS = 2;
  constexpr float V_FACTOR = CACHE ? SCALE_ROOM : 1.0f;
  constexpr int KEYS = tile_keys<DP, SOURCE, APART>, U = KEYS / 32;
  constexpr int EACH = CACHE ? 16 : 8, ROW = DP / EACH;    // values of a piece, pieces of a row
  constexpr int N = (KEYS * ROW + THREADS - 1) / THREADS;  // pieces of a tile for a thread
  constexpr int NL = KEYS * PC / THREADS;                  // slots of a tile for a thread
  static_assert(!IS_DIRECT || KEYS * PC % THREADS == 0, "staging");
  constexpr int TILE = KEYS * PC * 16;                 // bytes of LDS, a power of two
  // keys, then values
  __shared__ __attribute__((aligned(BUFFERS * TILE))) char all_lds[TEAMS][2 * BUFFERS * TILE];
  __shared__ __attribute__((aligned(16))) int ldoc[DOCS ? BUFFERS : 1][DOCS ? WAVES : 1][64];
  __shared__ uint64_t lbits[WAVES];
  __shared__ int lrange[3][WAVES];
  __shared__ __attribute__((aligned(16))) PT lp[WAVES][32][16];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, h = lane >> 5;
  const int team = APART ? wave : 0, mate = APART ? 0 : wave;  // and which of its waves
  const int thread = APART ? lane : (int)threadIdx.x;          // of the team
  char* const lds = all_lds[team];
  auto sync = [] {
    if constexpr (APART) {
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
      __builtin_amdgcn_wave_barrier();
    } else {
      __syncthreads();
    }
  };
  const int rows = a.queries * a.group;
  // Workgroups go to the 8 XCDs in turn: a unit (batch, key head, split of the keys) stays on
  // one where there are enough of them, and long tiles come first
  const int units = a.batch * a.kv_heads * a.splits;
  int unit, tile;
  if (units % 8 == 0) {
    const int i = blockIdx.x / 8;
    unit = i % (units / 8) * 8 + blockIdx.x % 8;
    tile = a.tiles - 1 - i / (units / 8);
  } else {
    unit = blockIdx.x % units;
    tile = a.tiles - 1 - blockIdx.x / units;
  }
  const int pair = unit / a.splits, split = unit % a.splits * TEAMS + team, splits = a.splits * TEAMS;
  const int b = pair / a.kv_heads, hk = pair % a.kv_heads;

  int keys = a.keys, shift = a.keys - a.queries;  // position of query 0
  int real = a.queries;                            // queries that are not padding
  if constexpr (CACHE) {
    const int start = at<int32_t>(a.start, a.start_off)[b * a.start_s];
    const int count = a.count ? at<int32_t>(a.count, a.count_off)[b * a.count_s] : a.queries;
    const bool ok = start >= 0 && count >= 0 && count <= a.queries && (int64_t)start + count <= a.keys;
    if (!ok && threadIdx.x == 0) *a.error = INVALID_CACHE_RANGE;
    shift = start;
    real = ok ? count : 0;
    keys = real > 0 ? start + real : 0;
  }
  int prefix = a.prefix ? at<int32_t>(a.prefix, a.p_off)[b * a.ps] : 0;
  prefix = prefix < 0 ? 0 : prefix;
  // last key that query ``t`` may see
  auto last = [&](int t) {
    int lim = keys - 1;
    if (CACHE || a.causal) {
      const int own = t + shift > prefix - 1 ? t + shift : prefix - 1;
      lim = own < lim ? own : lim;
    }
    return lim;
  };
  const int first_row = tile * ROWS, wave_row = first_row + mate * 32;
  const int row = wave_row + c;
  const int r = row < rows ? row : rows - 1;  // rows past the end repeat the last, and are not stored
  const int t = r / a.group, head = hk * a.group + r % a.group;
  const int32_t* const doc = at<int32_t>(a.documents, a.d_off) + b * a.db;
  const int mine = DOCS && a.documents ? doc[(t + shift) * a.dt] : 0;
  const int lim = mine < 0 ? -1 : last(t);
  const int end_row = first_row + ROWS < rows ? first_row + ROWS : rows;
  const int lim_wg = last((end_row - 1) / a.group);
  const int lim_wave = wave_row < rows ? last((wave_row + 31 < rows ? wave_row + 31 : rows - 1) / a.group) : -1;
  // Tiles of keys before ``tiles`` are seen. A split takes every splits-th of them: those that
  // are read at one time then lie side by side.
  const int tiles = lim_wg < 0 ? 0 : lim_wg / KEYS + 1;

  v8 q[DP / 16];
  {
    const T* p = at<T>(a.q, a.q_off) + b * a.qb + (int64_t)t * a.qt + head * a.qh;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      T x[8] = {};
      if (16 * s + 8 * h < a.dim) load_n<2>(x, p + 16 * s + 8 * h);
#pragma unroll
      for (int i = 0; i < 8; ++i) q[s][i] = x[i];
    }
  }
  float slope = 0.0f;
  if (GENERAL && a.slopes) slope = at<float>(a.slopes, a.s_off)[head * a.ss] * 0x1.715476p+0f;

  typedef typename choose<CACHE, uint8_t, T>::type stored;
  const stored* const kp = at<stored>(a.k, a.k_off) + b * a.kb + hk * a.kh;
  const stored* const vp = at<stored>(a.v, a.v_off) + b * a.vb + hk * a.vh;
  const int64_t scales_at = CACHE ? ((int64_t)pair * a.keys) >> a.block_shift : 0;
  const float* const ks = at<float>(a.k_scale, a.ks_off) + scales_at;
  const float* const vs = at<float>(a.v_scale, a.vs_off) + scales_at;
  // slot i = thread + n * THREADS of a tile is chunk (i % PC) ^ swizzle of row i / PC; rows of
  // one thread are STEP apart, and the swizzle comes again after 16 rows
  constexpr int STEP = THREADS / PC, KINDS = STEP >= 16 || !IS_DIRECT ? 1 : 16 / STEP < NL ? 16 / STEP : NL;
  uint32_t kv[KINDS], vv[KINDS];
  auto chunk_of = [&](int kr) { return (slot<PC>(kr, thread % PC) % PC) % CH; };
#pragma unroll
  for (int i = 0; i < KINDS; ++i) {
    const int kr = thread / PC, chunk = chunk_of(kr + i * STEP);
    kv[i] = (kr * (uint32_t)a.kt + chunk * 8) * (uint32_t)sizeof(T);
    vv[i] = (kr * (uint32_t)a.vt + chunk * 8) * (uint32_t)sizeof(T);
  }
  // 8 values of 16 bits, or 16 codes, a piece
  uint4v rk[IS_DIRECT ? 1 : N], rv[IS_DIRECT ? 1 : N];
  int rdoc = 0;
  // with documents, a tile that needs a mask is its number and this
  constexpr int MASK = 1 << 28;
  auto place = [](int kt) { return DOCS ? kt & (MASK - 1) : kt; };
  auto load = [&](int kt, int into) {
    const int base = place(kt) * KEYS;
    if constexpr (IS_DIRECT) {
      char* const to = lds + into * TILE + mate * 1024;
      if (base + KEYS <= keys) {
        const char* const kb = reinterpret_cast<const char*>(kp + base * a.kt);
        const char* const vb = reinterpret_cast<const char*>(vp + base * a.vt);
#pragma unroll
        for (int n = 0; n < NL; ++n) {
          to_lds(kb + n * STEP * a.kt * sizeof(T) + kv[n % KINDS], to + n * THREADS * 16);
          to_lds(vb + n * STEP * a.vt * sizeof(T) + vv[n % KINDS], to + BUFFERS * TILE + n * THREADS * 16);
        }
      } else {  // past the last key the last one again
#pragma unroll
        for (int n = 0; n < NL; ++n) {
          const int kr = thread / PC + n * STEP, key = base + kr < keys ? base + kr : keys - 1;
          const int chunk = chunk_of(kr);
          to_lds(kp + key * a.kt + chunk * 8, to + n * THREADS * 16);
          to_lds(vp + key * a.vt + chunk * 8, to + BUFFERS * TILE + n * THREADS * 16);
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int i = thread + n * THREADS, key = base + i / ROW, d = i % ROW * EACH;
        rk[n] = rv[n] = uint4v{0, 0, 0, 0};
        if (key < keys && d < a.dim && i < KEYS * ROW) {
          if constexpr (CACHE) {
            rk[n] = *reinterpret_cast<const uint4v*>(kp + key * a.kt + d);
            rv[n] = *reinterpret_cast<const uint4v*>(vp + key * a.vt + d);
          } else {
            T x[8];
            load_n<2>(x, kp + key * a.kt + d);
            rk[n] = __builtin_bit_cast(uint4v, x);
            load_n<2>(x, vp + key * a.vt + d);
            rv[n] = __builtin_bit_cast(uint4v, x);
          }
        }
      }
    }
    if (DOCS && a.documents) {
      // every wave its own copy, so that all have as many loads on their way; what lies
      // behind the last key is masked by its index
      const int key = base + lane % KEYS < keys ? base + lane % KEYS : keys - 1;
      if constexpr (IS_DIRECT)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(doc + key * a.dt),
                                         (__attribute__((address_space(3))) void*)ldoc[into][wave], 4, 0, 0);
      else
        rdoc = doc[key * a.dt];
    }
  };

  float16v o[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
  float m = -__builtin_inff(), l = 0.0f;
  // token of a 32-token half tile that row c of the score product is
  const int token = ((c >> 4) << 4) | (((c >> 2) & 1) << 3) | (((c >> 3) & 1) << 2) | (c & 3);
  // where this lane reads K, and V^T (token 8 h + group / 4 of 16 and value 16 (lane / 16 % 2)
  // + 4 (lane % 4) of 32): the other pieces of a tile are an xor or a constant away, since a
  // slot's number is, and the other buffer too
  const int vk = 8 * h + ((lane & 15) >> 2), vd = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  uint32_t k_at = slot<PC>(token, h) * 16, v_at = slot<PC>(vk, vd >> 3) * 16 + (vd & 7) * 2;
  constexpr int PITCH = PC * 16;

  int it = 0;       // the buffer of the tile in use
  int behind = 0;   // the tile that is on its way: to the other buffer, or to registers
  // registers to buffer ``into``
  auto store = [&](int into) {
    uint4v* const lk = reinterpret_cast<uint4v*>(lds + into * TILE);
    uint4v* const lv = reinterpret_cast<uint4v*>(lds + (BUFFERS + into) * TILE);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = thread + n * THREADS, r0 = i / ROW, c0 = i % ROW;
      if (KEYS * ROW % THREADS != 0 && i >= KEYS * ROW) continue;
      if constexpr (CACHE) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t k0 = rk[n][2 * y], k1 = rk[n][2 * y + 1], v0 = rv[n][2 * y], v1 = rv[n][2 * y + 1];
          lk[slot<PC>(r0, 2 * c0 + y)] = uint4v{codes<T>::widen(k0, 0), codes<T>::widen(k0, 1),
                                                codes<T>::widen(k1, 0), codes<T>::widen(k1, 1)};
          lv[slot<PC>(r0, 2 * c0 + y)] = uint4v{codes<PT>::widen(v0, 0), codes<PT>::widen(v0, 1),
                                                codes<PT>::widen(v1, 0), codes<PT>::widen(v1, 1)};
        }
      } else {
        lk[slot<PC>(r0, c0)] = rk[n];
        lv[slot<PC>(r0, c0)] = rv[n];
      }
    }
    if (DOCS && a.documents) ldoc[into][wave][lane] = rdoc;
  };
  // the first tile on its way; ``after`` says which follows one
  auto begin = [&](int kt, auto after) {
    if (place(kt) < tiles) load(kt, it);
    behind = kt;
    if constexpr (!IS_DIRECT) {
      if (place(kt) < tiles) {
        store(it);
        behind = after(kt);
        if (place(behind) < tiles) load(behind, 0);
      }
    }
    return kt;
  };
  // Waits for tile ``kt``, and for this wave's reads of the one before, whose buffer is the
  // next to be filled, and starts on the tile after it; which that is.
  auto arrive = [&](int kt, auto after) {
    if constexpr (IS_DIRECT) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
      if constexpr (APART) __builtin_amdgcn_wave_barrier();
      else __builtin_amdgcn_s_barrier();
      asm volatile("" : : : "memory");
      const int next = after(kt);
      if (place(next) < tiles) load(next, it ^ 1);
      return next;
    } else {
      sync();
      const int next = behind;
      if (place(next) < tiles) {
        store(it ^ 1);
        behind = after(next);
        if (place(behind) < tiles) load(behind, 0);
      }
      return next;
    }
  };
  auto compute = [&](int kt, auto is_masked, auto is_safe) {
    constexpr bool MASKED = decltype(is_masked)::value, SAFE = decltype(is_safe)::value;
    const int base = place(kt) * KEYS;

    float16v s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < 16; ++j) s[u][j] = 0.0f;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
        s[u] = mfma_32x32x16(*reinterpret_cast<const v8*>(lds + (k_at ^ (i << 5)) + u * 32 * PITCH), q[i], s[u]);
    }
    float scale = a.scale, v_scale = 1.0f;
    if constexpr (CACHE) {
      const float k_scale = ks[base >> a.block_shift];
      scale *= __builtin_fmaf(k_scale, 0.0f, k_scale);  // keys of infinity: NaN, not a mask's -infinity
      v_scale = vs[base >> a.block_shift] * V_FACTOR;
      // scales that are not finite, of keys that this row does not see
      if (SAFE && base > lim) scale = 1.0f, v_scale = 0.0f;
    }
    if constexpr (GENERAL) {
      // in log2 units: the cap, then the bias
      if (a.cap != 0.0f) {
        // cap tanh y = cap - 2 cap / (e^2y + 1)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            s[u][j] = __builtin_fmaf(-2.0f * a.cap,
                                     __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[u][j] * (scale * (2.0f * 0x1.715476p+0f))) + 1.0f), a.cap);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < 16; ++j) s[u][j] *= scale;
      }
      scale = 1.0f;
      if (a.slopes) {
        const float away = (float)(base + 8 * h - (t + shift));
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            s[u][j] = __builtin_fmaf(-slope, __builtin_fabsf(away + (float)(32 * u + 16 * (j >> 3) + (j & 7))), s[u][j]);
      }
    }
    if constexpr (MASKED) {
      if constexpr (CACHE) {
        // before the mask: the scale of a key block may be zero, and a mask's -infinity times it NaN
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < 16; ++j) s[u][j] *= scale;
        scale = 1.0f;
      }
      const int own = lim - base - 8 * h;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int k = 32 * u + 16 * (j >> 3) + (j & 7);
          bool seen = k <= own;
          if (DOCS && a.documents) seen = seen && ldoc[it][wave][k + 8 * h] == mine;
          s[u][j] = seen ? s[u][j] : -__builtin_inff();
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 16; ++j) top = __builtin_fmaxf(top, s[u][j]);
    top = xor32<OpMax>(top * scale);
    // The reference of the exponentials is not the maximum itself: O is scaled only when a
    // maximum is 2^8 above the one that set it, and the largest weight is then 2^LIFT. In
    // fp16 that keeps weights down to 2^-21 of it normal numbers, up to 2^15; bf16 has
    // exponents to spare, and weights of 2^-40 leave fp32 room for any value it holds.
    constexpr float LIFT = vec8<PT>::lift;
    if (__any(top > m + (LIFT + 8.0f))) {
      const float next = top - LIFT > m ? top - LIFT : m;
      const float alpha = next == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - next);
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][j] *= alpha;
      l *= alpha;
      m = next;
    }
    const float ref = m == -__builtin_inff() ? 0.0f : m;
    // Weights are rounded to 16 bits, as a product of 16-bit values takes them; the sum is of what
    // they were. Against 64 bits results are so off by 2.0e-3 to 2.2e-3 (bf16, root of the mean
    // square) and 2.2e-4 to 2.4e-4 (fp16), where the result's own rounding makes 1.6e-3 and
    // 2.0e-4. With the sum of the rounded weights 1.9e-3 to 2.1e-3, in 2 to 7 % more time.
    p8 p[2 * U];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][j], scale, -ref));
        l += e;
        p[2 * u + (j >> 3)][j & 7] = (PT)e;
        // a weight that is too small for its type still makes an infinity or a NaN count
        if (SAFE && s[u][j] > -__builtin_inff() && e < vec8<PT>::least)
          p[2 * u + (j >> 3)][j & 7] = (PT)vec8<PT>::least;
      }
    auto values = [&](int i, int u) {
      const char* const at = lds + BUFFERS * TILE + u * 16 * PITCH;
      const h4 lo = read_transposed(at + (v_at ^ (i << 6)));
      const h4 hi = read_transposed(at + (v_at ^ (i << 6) ^ 16) + 4 * PITCH);
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    bool spoiled = false;
    if constexpr (CACHE) {
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        float16v add;
#pragma unroll
        for (int j = 0; j < 16; ++j) add[j] = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint4v w = __builtin_bit_cast(uint4v, values(i, u));
          if constexpr (SAFE) spoiled |= drop_not_finite<vec8<PT>::exponent>(w);
          add = mfma_32x32x16(__builtin_bit_cast(p8, w), p[u], add);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][j] = __builtin_fmaf(add[j], v_scale, o[i][j]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int u = 0; u < 2 * U; ++u) {
          uint4v w = __builtin_bit_cast(uint4v, values(i, u));
          if constexpr (SAFE) spoiled |= drop_not_finite<vec8<PT>::exponent>(w);
          o[i] = mfma_32x32x16(__builtin_bit_cast(p8, w), p[u], o[i]);
        }
    }
    if constexpr (SAFE) {
      if (__any(spoiled)) {
        const PT* const value = reinterpret_cast<const PT*>(lds + (BUFFERS + it) * TILE);
#pragma unroll 1
        for (int u = 0; u < 2 * U; ++u) {
          // p by a constant index only: it stays in registers
          const p8 pu = u == 0 ? p[0] : u == 1 ? p[1] : u == 2 ? p[2 * U - 2] : p[2 * U - 1];
          *reinterpret_cast<p8*>(&lp[wave][c][8 * h]) = pu;
          __builtin_amdgcn_wave_barrier();
#pragma unroll 1
          for (int j = 0; j < 16; ++j) {
            const float x = element<PT>::widen(lp[wave][c][j]);
            const int k = 16 * u + j;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i)
#pragma unroll
              for (int z = 0; z < 16; ++z) {
                const int d = 32 * i + 8 * (z >> 2) + 4 * h + (z & 3);
                const float y = element<PT>::widen(value[slot<PC>(k, d >> 3) * 8 + (d & 7)]);
                if (x != 0.0f && !(__builtin_fabsf(y) < __builtin_inff())) o[i][z] += x * y;
              }
          }
          __builtin_amdgcn_wave_barrier();
        }
      }
    }
  };

  auto turn = [&] {  // to the other buffer
    k_at ^= TILE;
    v_at ^= TILE;
    it ^= 1;
  };
  // tiles that every row sees whole
  int whole = (last(first_row / a.group) + 1) / KEYS;
  whole = whole < tiles ? whole : tiles;
  auto every = [&](int kt) { return kt + splits; };
  if (!(DOCS && a.documents)) {
    // those first, then the ones that need a mask
    int kt = begin(split, every);
    while (kt < whole) {
      const int next = arrive(kt, every);
      compute(kt, bool_constant<false>{}, bool_constant<false>{});
      turn();
      kt = next;
    }
    while (kt < tiles) {
      const int next = arrive(kt, every);
      if (kt * KEYS <= lim_wave) compute(kt, bool_constant<true>{}, bool_constant<false>{});
      turn();
      kt = next;
    }
  }
  if constexpr (DOCS) {
    if (a.documents) {
      // The documents of the workgroup's rows, least and largest, and whether a row has none.
      // A tile whose documents lie outside is left out, one that is of the rows' only
      // document needs no mask: tiles are looked through SPAN at a time, 8 keys a lane, or, by
      // a wave apart, a tile. That takes 2 us a span, a tile without a mask 2 and with one 3:
      // 3 x 2021 tokens, 16 heads over 4 of 96, bf16, causal, 8 documents a row 39 to 45 us, 64
      // 29 us, one 67 to 75 (55 to 63 without). Latency bounds it: vector units are 25 %, matrix
      // units 6 % of the time busy.
      constexpr int LANES = APART ? 1 : KEYS / 8, PER_WAVE = 64 / LANES, SPAN = PER_WAVE * TEAM;
      static_assert(SPAN <= 64, "bits");
      auto least = [](int x, int y) { return x < y ? x : y; };
      auto largest = [](int x, int y) { return x > y ? x : y; };
      // One or two tiles are not worth a look: all with a mask (9 tokens 10.7 us with it, 9.0).
      const bool few = tiles <= 2 * splits && tiles <= SPAN;
      int lo = mine < 0 ? 0x7fffffff : mine, hi = mine, none = mine < 0;
      if (!few) {
        for (int d = 1; d < 32; d <<= 1) {
          lo = least(lo, __shfl_xor(lo, d, 64));
          hi = largest(hi, __shfl_xor(hi, d, 64));
          none |= __shfl_xor(none, d, 64);
        }
        if constexpr (TEAM > 1) {
          if (lane == 0) lrange[0][wave] = lo, lrange[1][wave] = hi, lrange[2][wave] = none;
          sync();
          for (int i = 0; i < TEAM; ++i) {
            lo = least(lo, lrange[0][i]);
            hi = largest(hi, lrange[1][i]);
            none |= lrange[2][i];
          }
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        hi = __builtin_amdgcn_readfirstlane(hi);
      }
      const bool one = __builtin_amdgcn_readfirstlane(none) == 0 && lo == hi;
      for (int span = 0; span * SPAN < tiles; ++span) {
        // this split's tiles of the span that rows see some of, and all of
        uint64_t open = 0, full = 0;
        if (few) {
          for (int kt = split; kt < tiles; kt += splits) open |= 1ull << kt;
        } else {
          const int tile = span * SPAN + mate * PER_WAVE + lane / LANES;
          int dl = 0x7fffffff, dh = -1;
          bool gap = false;  // a token of no document
#pragma unroll
          for (int j = 0; j < KEYS / LANES; ++j) {
            const int key = tile * KEYS + lane % LANES * (KEYS / LANES) + j;
            const int x = key < keys ? doc[key * a.dt] : -1;
            gap |= x < 0;
            dl = x < 0 ? dl : least(dl, x);
            dh = largest(dh, x);
          }
          int holes = gap;
          for (int d = 1; d < LANES; d <<= 1) {
            dl = least(dl, __shfl_xor(dl, d, 64));
            dh = largest(dh, __shfl_xor(dh, d, 64));
            holes |= __shfl_xor(holes, d, 64);
          }
          const bool first = lane % LANES == 0 && tile < tiles && tile % splits == split;
          const uint64_t some = __ballot(first && dh >= lo && dl <= hi);
          const uint64_t all = __ballot(first && one && !holes && dl == lo && dh == lo && tile < whole);
          open = some;
          full = all;
          if constexpr (LANES > 1) {
            uint64_t bits = 0;
            for (int i = 0; i < PER_WAVE; ++i) {
              bits |= ((some >> (i * LANES)) & 1) << i;
              bits |= ((all >> (i * LANES)) & 1) << (i + 32);
            }
            open = full = 0;
            if constexpr (TEAM > 1) {
              sync();  // everyone is done with the span before
              if (lane == 0) lbits[wave] = bits;
              sync();
            }
            for (int i = 0; i < TEAM; ++i) {
              const uint64_t w = TEAM > 1 ? lbits[i] : bits;
              open |= (w & 0xffffffffu) << (i * PER_WAVE);
              full |= (w >> 32) << (i * PER_WAVE);
            }
          }
        }
        auto uniform = [](uint64_t x) {
          return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 |
                 (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
        };
        full = uniform(full);
        open = uniform(open) & ~full;
        // those that need no mask, then those that do
        auto take = [&](uint64_t& from, int flag) {
          const int at = __builtin_ctzll(from);
          from &= from - 1;
          return (span * SPAN + at) | flag;
        };
        auto after = [&](int) { return full ? take(full, 0) : open ? take(open, MASK) : tiles; };
        int kt = begin(after(0), after);
        while (kt < tiles) {
          const int next = arrive(kt, after);
          compute(kt, bool_constant<false>{}, bool_constant<false>{});
          turn();
          kt = next;
        }
        while (kt & MASK) {
          const int next = arrive(kt, after);
          if (place(kt) * KEYS <= lim_wave) compute(kt, bool_constant<true>{}, bool_constant<false>{});
          turn();
          kt = next;
        }
      }
    }
  }
  // 0 times an infinity or NaN of a key that a row does not see is NaN in the products.
  // Where something came out not finite, all is done again with such values left out
  // of the products and added key by key to the rows that see them.
  float check = 0.0f;
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) check = __builtin_fmaf(o[i][j], 0.0f, check);
  if (APART ? __any(check != 0.0f) : __syncthreads_or(check != 0.0f)) {
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
    m = -__builtin_inff();
    l = 0.0f;
    begin(split, every);
    for (int kt = split; kt < tiles; kt += splits) {
      arrive(kt, every);
      if (kt * KEYS <= lim_wave) compute(kt, bool_constant<true>{}, bool_constant<true>{});
      turn();
    }
  }
  l = xor32<OpSum>(l) * V_FACTOR;
  if (CACHE && t >= real) {  // padding
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
    m = -__builtin_inff();
    l = 0.0f;
  }
  // four values of a row: to the parts, or as they are
  auto put = [&](int row, int d, float4v x, float m, float l) {
    if (a.splits > 1) {
      float* const part = a.part + (((int64_t)(unit % a.splits) * a.batch * a.kv_heads + pair) * rows + row) * (a.dim + 4);
      *reinterpret_cast<float4v*>(part + d) = x;
      if (d == 0) *reinterpret_cast<float4v*>(part + a.dim) = float4v{m, l, 0.0f, 0.0f};
      return;
    }
    const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
    const int t = row / a.group, head = hk * a.group + row % a.group;
    T y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = element<T>::narrow(x[j] * inverse);
    store_n<8>(reinterpret_cast<T*>(a.out) +
               (((int64_t)b * a.queries + t) * a.kv_heads * a.group + head) * a.dim + d, y);
  };
  if constexpr (APART) {
    // the waves' parts, each in its own LDS, whose tiles it is done with
    constexpr int PITCH = DP + 4;
    static_assert(32 * PITCH * 4 <= 2 * BUFFERS * TILE, "parts");
    __shared__ float lm[WAVES][32], ll[WAVES][32];
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
    float* const mine = reinterpret_cast<float*>(lds) + c * PITCH;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int z = 0; z < 4; ++z)
        *reinterpret_cast<float4v*>(mine + 32 * i + 8 * z + 4 * h) =
            float4v{o[i][4 * z], o[i][4 * z + 1], o[i][4 * z + 2], o[i][4 * z + 3]};
    if (h == 0) lm[wave][c] = m, ll[wave][c] = l;
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * (DP / 4); i += 64 * WAVES) {
      const int y = i / (DP / 4), d = i % (DP / 4) * 4;
      if (first_row + y >= rows || d >= a.dim) continue;
      float top = lm[0][y];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) top = __builtin_fmaxf(top, lm[w][y]);
      const float ref = top == -__builtin_inff() ? 0.0f : top;
      float4v x = float4v{0.0f, 0.0f, 0.0f, 0.0f};
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float f = __builtin_amdgcn_exp2f(lm[w][y] - ref);
        sum = __builtin_fmaf(ll[w][y], f, sum);
        const float4v v = *reinterpret_cast<const float4v*>(reinterpret_cast<const float*>(all_lds[w]) + y * PITCH + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(v[e], f, x[e]);
      }
      put(first_row + y, d, x, top, sum);
    }
  } else {
    if (row >= rows) return;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const int d = 32 * i + 8 * z + 4 * h;
        if (d < a.dim)
          put(row, d, float4v{o[i][4 * z], o[i][4 * z + 1], o[i][4 * z + 2], o[i][4 * z + 3]}, m, l);
      }
  }
}

// One workgroup for each (sequence, token, head).
template <class T, int WAVES>
__device__ __forceinline__ void attention_join(const AttentionArgs& a) {
  const int heads = a.kv_heads * a.group, head = (int)(blockIdx.x % (uint32_t)heads);
  const uint32_t w = blockIdx.x / (uint32_t)heads;
  const int t = (int)(w % (uint32_t)a.queries), b = (int)(w / (uint32_t)a.queries);
  const int64_t rows = (int64_t)a.queries * a.group;
  const int64_t row = ((int64_t)b * a.kv_heads + head / a.group) * rows + (int64_t)t * a.group + head % a.group;
  join_parts<WAVES>(a.part + row * (a.dim + 4), a.batch * a.kv_heads * rows * (a.dim + 4), a.splits, a.dim,
             reinterpret_cast<T*>(a.out) + (((int64_t)b * a.queries + t) * heads + head) * a.dim);
}

}  // namespace mlc

#define ATTENTION(NAME, T, DP, WAVES, SOURCE, SCORES, APART)                                      \
  extern "C" __global__ void __launch_bounds__(64 * WAVES, mlc::waves_a_simd(DP, mlc::SCORES, APART)) \
  NAME(mlc::AttentionArgs a) {                                                                    \
    mlc::attention<T, DP, WAVES, mlc::SOURCE, mlc::SCORES, APART>(a);                             \
  }
#define ATTENTION_JOIN(NAME, T, WAVES)                                                   \
  extern "C" __global__ void __launch_bounds__(64 * WAVES) NAME(mlc::AttentionArgs a) {                  \
    mlc::attention_join<T, WAVES>(a);                                                   \
  }
