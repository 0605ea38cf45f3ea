// Attention of the newest tokens over the 8-bit cache: token i of a sequence stands
// at position start + i and sees the keys up to its own. Rows are (token, head of
// a group) pairs, 16 to a workgroup, so keys and values are read once for all
// heads that share them.
//
// Bound by memory where rows are few: the cache is read once, 2 (dim + 4 / block)
// bytes a key and head. A sequence's keys are cut into items; how long an item is
// follows from the lengths that the sequences have on the device, so that no
// workgroup has much more to read than an even share. Each wave of an item
// takes its own keys straight into registers:
//  * S^T = K Q^T on 16x16x32 products; the order of K's rows makes lane (c, g) end
//    with row c's scores of keys 8 g .. 8 g + 7 of every 32, the B operand of
//  * O^T = V^T P^T, whose V^T operand is made of V's rows by byte permutes. P is
//    fp16 whatever the queries are: e4m3 is exact in it, and P, 2^14 where a score is the
//    largest, is a normal number down to 2^-28 of that.
//  * A key block's scales are powers of two outside the products: K's goes into the
//    factor of its scores, V's multiplies the block's part of O.
// The waves of a workgroup are joined in LDS, the items of a sequence by a second
// kernel (cache_attention_join).
//
// One token, 32 heads over 8 of 128, bf16: 32 sequences of up to 8192 keys 63 to 67 us a call,
// 4.6 TB/s, one of 131072 55 to 57 us, 4.8 TB/s (a read reaches 6.2; the join is 4 us of each);
// over the same cache again and again, some of it in the last-level cache, 57 and 48 us. 12 heads
// of 64 over 1024 keys 6.3 us, the latency of one workgroup's steps. Tens of rows are bound by
// latency too: 2 x 61 tokens, 16 heads over 2, 4096 keys 24 us for 3.2 of products, with vector
// units a third and matrix units 6 % of the time busy. A wave has two steps between looking for
// its item, the first loads and the join in LDS, and a second launch follows; the last step's
// loads are made once more for nothing; every 16 rows widen the codes again. Tiles of 128 rows
// (attention.hip) widen them once and take 28.

namespace mlc {

struct CacheAttentionArgs {
  const void* q;
  const void* cache[2];
  const void* scale[2];
  const void* slopes;  // null: no bias by distance
  const void* start;
  const void* count;  // null: every token is real
  void* out;
  float* part;  // {first item, items} of each sequence, then [item][kv head][row][dim + 4]
  int* error;
  int64_t q_off, cache_off[2], scale_off[2], sl_off, start_off, count_off;  // bytes
  int64_t qb, qt, qh, sls, ss, sc;                                          // elements
  int32_t batch, tokens, kv_heads, group, dim, capacity, block_shift, row_tiles;
  int32_t items, shortest;  // items wanted of all sequences, 0: each is one; keys of the shortest
  float factor, cap;
};

// Keys of a sequence that its tokens may see; 0 for one that is refused.
__device__ __forceinline__ int held(const CacheAttentionArgs& a, int b, int& start, int& count) {
  start = at<int32_t>(a.start, a.start_off)[b * a.ss];
  count = a.count ? at<int32_t>(a.count, a.count_off)[b * a.sc] : a.tokens;
  const bool ok = start >= 0 && count >= 0 && count <= a.tokens &&
                  (int64_t)start + count <= a.capacity;
  if (!ok) count = -1;
  return count > 0 ? start + count : 0;
}

typedef int int2v __attribute__((ext_vector_type(2)));

// Where the parts begin: behind two words a sequence.
__device__ __forceinline__ int64_t parts_at(const CacheAttentionArgs& a) { return ((int64_t)a.batch + 1) / 2 * 4; }

struct Item {
  int b, nth, of, keys;  // the nth of the items of a sequence of so many keys
};

// How the sequences' keys are cut: every wave finds it again from the lengths. Items are
// ``length`` keys long at most, as few as are wanted of all sequences together.
__device__ __forceinline__ bool find_item(const CacheAttentionArgs& a, int want, Item& found, int& first) {
  const int lane = threadIdx.x & 63;
  int start, count;
  if (a.items == 0) {  // none is cut
    found.b = want;
    found.nth = first = 0;
    found.of = 1;
    found.keys = held(a, found.b, start, count);
    return true;
  }
  auto cut = [](int keys, int length) { return keys == 0 ? 1 : (keys + length - 1) / length; };
  int mine = lane < a.batch ? held(a, lane, start, count) : 0;  // of the first 64 sequences
  auto keys_of = [&](int b) { return b < 64 ? mine : b < a.batch ? held(a, b, start, count) : 0; };
  float total = 0.0f;  // exact, or near enough: all waves come to the same
  for (int b0 = 0; b0 < a.batch; b0 += 64) total += (float)keys_of(b0 + lane);
  total = group_reduce<64, OpSum>(total);
  // Each sequence's last item is short: longer items until there are no more than wanted, but at
  // most twice an even share. Every sequence is an item at least, so without that limit many
  // short ones keep a long one whole: 65536 keys and 255 sequences of 200, 8 heads of 128, 192 us
  // and 68 with it; 5 of 32768 and 95 of 500 105 and 82; 64 of 819 to 8190, which it leaves as
  // they are, 114.
  int length = a.shortest, longest = 0x7fffffff;
  for (int i = 0; i < 3; ++i) {
    float n = 0.0f;
    if (i > 0) {
      for (int b0 = 0; b0 < a.batch; b0 += 64)
        if (b0 + lane < a.batch) n += (float)cut(keys_of(b0 + lane), length);
      n = group_reduce<64, OpSum>(n);
      if (n <= (float)a.items) break;
    }
    const float longer = i == 0 ? total / (float)a.items : (float)length * n / (float)a.items;
    int next = longer < (float)a.capacity ? ((int)longer + 64) / 64 * 64 : (a.capacity + 63) / 64 * 64;
    next = next < longest ? next : longest;
    length = next > length ? next : length;
    if (i == 0) longest = length < 0x3fffffff ? 2 * length : length;
  }
  first = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int b = b0 + lane, keys = keys_of(b);
    const int n = b < a.batch ? cut(keys, length) : 0;
    int sum = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int other = __shfl_up(sum, d, 64);
      sum += lane >= d ? other : 0;
    }
    const uint64_t past = __ballot(first + sum > want);
    if (past) {
      const int at_lane = __builtin_ctzll(past);
      found.b = b0 + at_lane;
      found.of = __shfl(n, at_lane, 64);
      found.keys = __shfl(keys, at_lane, 64);
      first += __shfl(sum, at_lane, 64) - found.of;
      found.nth = want - first;
      return true;
    }
    first += __shfl(sum, 63, 64);
  }
  return false;
}

template <int W> struct words { uint32_t x[W]; };

template <class T, int DP, int TOK, int WAVES, bool GENERAL>
__device__ __forceinline__ void cache_attention(const CacheAttentionArgs& a) {
  typedef typename codes<T>::v8 v8;
  constexpr int KP = DP / 64;   // 16-byte pieces of a key's row per lane
  constexpr int VB = DP / 16;   // bytes of a value's row per lane
  constexpr int VW = VB / 4;    // and words
  constexpr int CH = TOK / 32;  // chunks of 32 keys a step
  __shared__ __attribute__((aligned(16))) float lo[WAVES][16][DP + 4];
  __shared__ float lm[WAVES][16], ll[WAVES][16];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  uint32_t w = blockIdx.x;
  const int hk = (int)(w % (uint32_t)a.kv_heads);
  w /= (uint32_t)a.kv_heads;
  const int row_tile = (int)(w % (uint32_t)a.row_tiles);
  w /= (uint32_t)a.row_tiles;
  Item item;
  int first;
  if (!find_item(a, (int)w, item, first)) return;
  const int b = __builtin_amdgcn_readfirstlane(item.b);
  int start, count;
  held(a, b, start, count);
  if (count < 0 && threadIdx.x == 0) *a.error = INVALID_CACHE_RANGE;
  // an item's waves take every so-manieth step of the keys: what is read at one time lies
  // side by side
  const int hi_key = __builtin_amdgcn_readfirstlane(item.keys);
  const int nth = __builtin_amdgcn_readfirstlane(item.nth), of = __builtin_amdgcn_readfirstlane(item.of);
  if (a.items > 0 && nth == 0 && row_tile == 0 && hk == 0 && threadIdx.x == 0)
    reinterpret_cast<int2v*>(a.part)[b] = int2v{first, of};

  const int rows = a.tokens * a.group;
  const int own = row_tile * 16 + c, r = own < rows ? own : rows - 1;
  const int t = r / a.group, head = hk * a.group + r % a.group;
  const int pos = start + t, lim = t < count ? pos : -1;
  v8 q[2 * KP];
  float slope = GENERAL && a.slopes ? at<float>(a.slopes, a.sl_off)[head * a.sls] * 0x1.715476p+0f : 0.0f;
  const T* p = at<T>(a.q, a.q_off) + b * a.qb + t * a.qt + head * a.qh;
#pragma unroll
  for (int s = 0; s < 2 * KP; ++s) {
    const int d = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
    T x[8] = {};
    if (d < a.dim) load_n<2>(x, p + d);
#pragma unroll
    for (int i = 0; i < 8; ++i) q[s][i] = x[i];
  }
  // the least of the rows' last keys: steps below it need no mask
  int lim_min = lim;
  for (int d = 1; d < 16; d <<= 1) {
    const int other = __shfl_xor(lim_min, d, 64);
    lim_min = other < lim_min ? other : lim_min;
  }
  lim_min = __builtin_amdgcn_readfirstlane(lim_min);

  const int64_t head_at = ((int64_t)b * a.kv_heads + hk) * a.capacity;
  const uint8_t* const kc = at<uint8_t>(a.cache[0], a.cache_off[0]) + head_at * a.dim;
  const uint8_t* const vc = at<uint8_t>(a.cache[1], a.cache_off[1]) + head_at * a.dim;
  const float* const ks = at<float>(a.scale[0], a.scale_off[0]) + (head_at >> a.block_shift);
  const float* const vs = at<float>(a.scale[1], a.scale_off[1]) + (head_at >> a.block_shift);

  float m = -__builtin_inff(), l = 0.0f;
  float4v o[VB];
#pragma unroll
  for (int j = 0; j < VB; ++j) o[j] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
  const int krow = 8 * (c >> 2) + (c & 3);
  // What lies past the last key or past dim is read as the last key or the row's start:
  // such scores are masked, such values meet zeros of Q or columns that nobody stores.
  const uint32_t v_at = c * VB < a.dim ? c * VB : 0;
  uint32_t k_at[KP];
#pragma unroll
  for (int s = 0; s < KP; ++s) k_at[s] = 64 * s + 16 * g < a.dim ? 64 * s + 16 * g : 0;
  uint4v kr[CH][2][KP];
  words<VW> vr[CH][8];
  float kscale_next, vscale_next;
  auto load_keys = [&](int tb) {
    const uint8_t* const base = kc + (int64_t)tb * a.dim;
    auto rows_at = [&](auto place) {
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int s = 0; s < KP; ++s)
            kr[ch][u][s] = *reinterpret_cast<const uint4v*>(place(32 * ch + 4 * u) + k_at[s]);
    };
    if (tb + TOK <= hi_key) {
      const uint32_t own = krow * (uint32_t)a.dim;
      rows_at([&](int row) { return base + row * a.dim + own; });
    } else {
      rows_at([&](int row) {
        const int key = row + krow < hi_key - tb ? row + krow : hi_key - tb - 1;
        return base + key * (uint32_t)a.dim;
      });
    }
    kscale_next = ks[tb >> a.block_shift];
  };
  auto load_values = [&](int tb) {
    const uint8_t* const base = vc + (int64_t)tb * a.dim;
    auto rows_at = [&](auto place) {
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int i = 0; i < 8; ++i) vr[ch][i] = *reinterpret_cast<const words<VW>*>(place(32 * ch + i) + v_at);
    };
    if (tb + TOK <= hi_key) {
      const uint32_t own = 8 * g * (uint32_t)a.dim;
      rows_at([&](int row) { return base + row * a.dim + own; });
    } else {
      rows_at([&](int row) {
        const int key = row + 8 * g < hi_key - tb ? row + 8 * g : hi_key - tb - 1;
        return base + key * (uint32_t)a.dim;
      });
    }
    vscale_next = vs[tb >> a.block_shift];
  };

  // The next step's keys are asked for when this one's are in the products, the next
  // values likewise: half of the registers' loads are always on their way.
  const int step = of * WAVES * TOK, begin = (nth * WAVES + wave) * TOK;
  auto pass = [&](auto is_safe) {
    constexpr bool SAFE = decltype(is_safe)::value;
    if (begin < hi_key) {
      load_keys(begin);
      load_values(begin);
    }
    for (int tb = begin; tb < hi_key; tb += step) {
      const float kscale = __builtin_fmaf(kscale_next, 0.0f, kscale_next);  // infinity: NaN, not a mask's
      float vscale = vscale_next * SCALE_ROOM;
      // a scale that is not finite, of keys that this row does not see
      if (SAFE && tb > lim) vscale = 0.0f;
      const int next = tb + step < hi_key ? tb + step : tb;  // past the end: once more, for nothing
      const bool masked = tb + TOK - 1 > lim_min;

      float4v s[CH][2];
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 2 * KP; ++i) {
            uint4v k;
            const uint32_t w0 = kr[ch][u][i >> 1][(i & 1) * 2], w1 = kr[ch][u][i >> 1][(i & 1) * 2 + 1];
            k.x = codes<T>::widen(w0, 0);
            k.y = codes<T>::widen(w0, 1);
            k.z = codes<T>::widen(w1, 0);
            k.w = codes<T>::widen(w1, 1);
            if (i == 0) s[ch][u] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
            s[ch][u] = mfma_16x16x32(__builtin_bit_cast(v8, k), q[i], s[ch][u]);
          }
      load_keys(next);
      half8 p[CH];
      const float factor = a.factor * kscale;
      auto each = [&](auto of_score) {
#pragma unroll
        for (int ch = 0; ch < CH; ++ch)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            s[ch][e >> 2][e & 3] = of_score(s[ch][e >> 2][e & 3], 32 * ch + e);
      };
      if (GENERAL && a.cap != 0.0f) {
        // cap tanh y = cap - 2 cap / (e^2y + 1)
        const float by = factor * (2.0f * 0x1.715476p+0f);
        each([&](float x, int) {
          return __builtin_fmaf(-2.0f * a.cap, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * by) + 1.0f), a.cap);
        });
      } else {
        each([&](float x, int) { return x * factor; });
      }
      if (GENERAL && a.slopes) {
        const float away = (float)(tb + 8 * g - pos);
        each([&](float x, int k) { return __builtin_fmaf(-slope, __builtin_fabsf(away + (float)k), x); });
      }
      if (masked) {
        const int left = lim - tb - 8 * g;
        each([&](float x, int k) { return k <= left ? x : -__builtin_inff(); });
      }
      float top = s[0][0][0];
      each([&](float x, int) {
        top = __builtin_fmaxf(top, x);
        return x;
      });
      top = xor32<OpMax>(xor16<OpMax>(top));
      const float now = top > m ? top : m;
      const float ref = now == -__builtin_inff() ? 0.0f : now;
      const float low = ref - 14.0f, alpha = __builtin_amdgcn_exp2f(m - ref);
      m = now;
      l *= alpha;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = __builtin_amdgcn_exp2f(s[ch][e >> 2][e & 3] - low);
          l += x;
          p[ch][e] = (f16)x;
        }
      float4v add[VB];
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int z = 0; z < VW; ++z) {
          uint32_t f[4][4];  // [byte][pair of tokens]
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t t0 = vr[ch][2 * i].x[z], t1 = vr[ch][2 * i + 1].x[z];
            const uint32_t even = __builtin_amdgcn_perm(t1, t0, 0x05010400u);
            const uint32_t odd = __builtin_amdgcn_perm(t1, t0, 0x07030602u);
            f[0][i] = codes<f16>::widen(even, 0);
            f[1][i] = codes<f16>::widen(even, 1);
            f[2][i] = codes<f16>::widen(odd, 0);
            f[3][i] = codes<f16>::widen(odd, 1);
          }
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            half8 v = __builtin_bit_cast(half8, uint4v{f[y][0], f[y][1], f[y][2], f[y][3]});
            const int j = 4 * z + y;
            if (ch == 0) add[j] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (SAFE) {
              // rows that see one of the values that are NaN get a NaN, others a zero of it
              half8 nan, sees;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                nan[e] = v[e] != v[e] ? (f16)1.0f : (f16)0.0f;
                v[e] = v[e] != v[e] ? (f16)0.0f : v[e];
                sees[e] = tb + 32 * ch + 8 * g + e <= lim ? (f16)1.0f : (f16)0.0f;
              }
              const float4v hits = mfma_16x16x32(nan, sees, float4v{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (hits[i] > 0.0f) add[j][i] = __builtin_nanf("");
            }
            add[j] = mfma_16x16x32(v, p[ch], add[j]);
          }
        }
      load_values(next);
#pragma unroll
      for (int j = 0; j < VB; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          o[j][i] = __builtin_fmaf(add[j][i], vscale, o[j][i] * alpha);
    }

  };
  pass(bool_constant<false>{});
  // 0 times a NaN of a key that a row does not see is NaN in the products. Where something
  // came out not finite, the wave goes through its keys again with such values apart.
  float check = 0.0f;
#pragma unroll
  for (int j = 0; j < VB; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) check = __builtin_fmaf(o[j][i], 0.0f, check);
  if (__any(check != 0.0f)) {
    m = -__builtin_inff();
    l = 0.0f;
#pragma unroll
    for (int j = 0; j < VB; ++j) o[j] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    pass(bool_constant<true>{});
  }

  // the waves' rows together; thread (row of 16, 4 values) at a time
  l = xor32<OpSum>(xor16<OpSum>(l)) * SCALE_ROOM;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < VB; j += 4)
      *reinterpret_cast<float4v*>(&lo[wave][c][VB * (4 * g + i) + j]) =
          float4v{o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]};
  if (g == 0) {
    lm[wave][c] = m;
    ll[wave][c] = l;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * (DP / 4); i += 64 * WAVES) {
    const int y = i / (DP / 4), d = i % (DP / 4) * 4;
    const int row = row_tile * 16 + y;
    if (row >= rows || d >= a.dim) continue;
    float top = lm[0][y];
#pragma unroll
    for (int z = 1; z < WAVES; ++z) top = __builtin_fmaxf(top, lm[z][y]);
    const float ref = top == -__builtin_inff() ? 0.0f : top;
    float4v x = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    float sum = 0.0f;
#pragma unroll
    for (int z = 0; z < WAVES; ++z) {
      const float f = __builtin_amdgcn_exp2f(lm[z][y] - ref);
      sum = __builtin_fmaf(ll[z][y], f, sum);
      const float4v v = *reinterpret_cast<const float4v*>(&lo[z][y][d]);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(v[e], f, x[e]);
    }
    if (of == 1) {
      const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
      const int t = row / a.group, head = hk * a.group + row % a.group;
      T v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = element<T>::narrow(x[e] * inverse);
      store_n<8>(reinterpret_cast<T*>(a.out) +
                 (((int64_t)b * a.tokens + t) * a.kv_heads * a.group + head) * a.dim + d, v);
    } else {
      float* const part = a.part + parts_at(a) + (((int64_t)w * a.kv_heads + hk) * rows + row) * (a.dim + 4);
      *reinterpret_cast<float4v*>(part + d) = x;
      if (d == 0) *reinterpret_cast<float4v*>(part + a.dim) = float4v{top, sum, 0.0f, 0.0f};
    }
  }
}

// One workgroup for each (sequence, token, head): its items' parts as one.
template <class T, int WAVES>
__device__ __forceinline__ void cache_attention_join(const CacheAttentionArgs& a) {
  const int heads = a.kv_heads * a.group;
  const int head = (int)(blockIdx.x % (uint32_t)heads);
  const uint32_t w = blockIdx.x / (uint32_t)heads;
  const int t = (int)(w % (uint32_t)a.tokens), b = (int)(w / (uint32_t)a.tokens);
  const int2v items = reinterpret_cast<const int2v*>(a.part)[b];
  if (items.y == 1) return;  // whole, and done
  const int hk = head / a.group, rows = a.tokens * a.group, row = t * a.group + head % a.group;
  const int64_t step = (int64_t)a.kv_heads * rows * (a.dim + 4);
  const float* const part = a.part + parts_at(a) + (((int64_t)items.x * a.kv_heads + hk) * rows + row) * (a.dim + 4);
  join_parts<WAVES>(part, step, items.y, a.dim,
             reinterpret_cast<T*>(a.out) + (((int64_t)b * a.tokens + t) * heads + head) * a.dim);
}

}  // namespace mlc

#define CACHE_ATTENTION(NAME, T, DP, TOK, WAVES, GENERAL)                                         \
  extern "C" __global__ void __launch_bounds__(64 * WAVES) NAME(mlc::CacheAttentionArgs a) {      \
    mlc::cache_attention<T, DP, TOK, WAVES, GENERAL>(a);                                          \
  }
#define CACHE_ATTENTION_JOIN(NAME, T, WAVES)                                             \
  extern "C" __global__ void __launch_bounds__(64 * WAVES) NAME(mlc::CacheAttentionArgs a) {             \
    mlc::cache_attention_join<T, WAVES>(a);                                             \
  }
