// One token of each row of logits, from a random number that is given. With T the row's
// temperature and m its largest logit, a token's weight is w = e^((x - m) / T). In the order of
// falling logits, and of indexes where they are equal, a token is kept that is
//  * among the first top_k, if top_k is above zero,
//  * of those, one before which less than top_p of their weight lies (the first always),
//  * and of a weight of min_p or more.
// All three end at a border in that order, (logit, index), so what is kept is what lies in front
// of the nearest one. The token is the first, in the vocabulary's order, up to which more than
// ``uniform`` of the kept weight lies.
//
// Sums are of whole numbers of 2^-40, so they are exact whatever their order: results do not depend
// on the order of atomics. What is rounded to one is a token's weight where tokens lie in a list, and in passes over a
// row the weight of eight neighbouring tokens, added in fp32: beside a weight of 1 one of 2^-25 counts as nothing
// there, and sums are up to 2^-21 of themselves off. With each token's own, in 64 bits, 256 rows of 131072 with top_p take
// 61 us instead of 54, without options 29 instead of 26.
//
// A workgroup has a row: no word passes between workgroups, one launch does it, and 256 rows fill the card. Only
// the first pass, for the largest logit, is bound by memory; then caches hold the row, and each instruction of
// a token takes 0.85 us in 131072 of them, on one unit. What runs once is bound by its own way from
// memory, 64 bytes of code at a time. So loops are short and passes few:
//  * What can be kept is gathered where a bound for it is at hand (the top_k-th of the threads' own
//    largest, or min_p) and fits a list: sorted, it says everything.
//  * Else tokens are counted by their distance to the largest, which says in which bins the borders
//    are. The tokens of those are gathered, the weight in front of them is summed up, exactly.
//  * The token comes from the kept weight of ever smaller segments of the row.
//  * Where a list is too short (equal logits), borders are found digit by digit.
//
// 131072 bf16 logits, in us, 1 row / 256 rows: no options 17.6 / 26.4, top_k = 50 15.7 / 23.4, top_p = 0.9
// 39 / 54, min_p = 0.05 9.5 / 40.5; 1 row of 50257: 11.1, 12.9, 24.7 and 6.5. 256 rows are read in 13 us.

namespace mlc {

enum { INVALID_SAMPLE = 3 };

struct SampleArgs {
  const void* logits;
  const void* uniform;
  const void* temperature;  // null: 1, and below: none
  const void* top_k;
  const void* top_p;
  const void* min_p;
  int64_t* out;
  int* error;
  int64_t l_off, u_off, t_off, k_off, p_off, m_off;  // bytes
  int64_t lb, us, ts, ks, ps, ms;                    // elements
  int32_t batch, size;
};

typedef unsigned long long u64;
constexpr int SAMPLE_THREADS = 1024, SAMPLE_WAVES = SAMPLE_THREADS / 64, SAMPLE_BINS = 2048, SAMPLE_COUNTS = 16384;
constexpr int SAMPLE_LIST = 1024, SAMPLE_EACH = 512;  // tokens that are sorted, a thread for each, and gathered by a wave
constexpr int SAMPLE_FEW = 512;                          // top_k whose tokens are gathered
constexpr float LEAST_TEMPERATURE = 0x1p-100f, MOST_TEMPERATURE = 0x1p100f;  // below the least the likeliest token

// A number that orders as floats do, -0 as 0, and back.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_order(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct SampleLds {
  alignas(16) char tail[64];  // the row's last pack, and one of -infinity
  union {
    u64 bins[SAMPLE_BINS];  // and a list's weights
    uint32_t counts[SAMPLE_COUNTS + 64];
  };
  u64 gathered[SAMPLE_WAVES][SAMPLE_EACH], list[SAMPLE_LIST], sorted[SAMPLE_LIST];
  u64 sums[SAMPLE_WAVES];
  u64 found[2];
  float tops[SAMPLE_WAVES];
  uint32_t least[SAMPLE_WAVES];
  int counts_of[SAMPLE_WAVES], digits[6];
};

// x of a lane below this one by DPP, 0 where there is none.
template <int CONTROL, int ROWS> __device__ __forceinline__ u64 moved(u64 x) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CONTROL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CONTROL, ROWS, 0xf, false);
  return (u64)hi << 32 | lo;
}

// The sum of x over the workgroup; ``below``: of the threads before this one.
__device__ __forceinline__ u64 sum_over_threads(u64 x, SampleLds& l, u64& below) {
  u64 run = x;
  run += moved<0x111, 0xf>(run);  // by 1, 2, 4 and 8 lanes of 16, then the last of 16 and of 32
  run += moved<0x112, 0xf>(run);
  run += moved<0x114, 0xf>(run);
  run += moved<0x118, 0xf>(run);
  run += moved<0x142, 0xa>(run);
  run += moved<0x143, 0xc>(run);
  __syncthreads();  // sums of the time before have been read
  if ((threadIdx.x & 63) == 63) l.sums[threadIdx.x >> 6] = run;
  __syncthreads();
  u64 all = 0, before = 0;
#pragma unroll
  for (int w = 0; w < SAMPLE_WAVES; ++w) {
    if (w < (int)(threadIdx.x >> 6)) before += l.sums[w];
    all += l.sums[w];
  }
  below = before + run - x;
  return all;
}

// The n (up to SAMPLE_LIST) different numbers of l.list in rising order, number t to thread t, the
// others' are the largest there is.
__device__ __forceinline__ u64 sort_list(int n, SampleLds& l) {
  const int tid = threadIdx.x;
  constexpr u64 LAST = ~(u64)0;
  if (n <= 256) {  // by counting the ones below, 16 at a time
    if (tid >= n && tid < n + 15) l.list[tid] = LAST;
    __syncthreads();
    if (tid < n) {
      const u64 own = l.list[tid];
      int rank = 0;
      for (int i = 0; i < n; i += 16) {
#pragma unroll
        for (int j = 0; j < 16; ++j) rank += l.list[i + j] < own;
      }
      l.sorted[rank] = own;
    }
    __syncthreads();
    return tid < n ? l.sorted[tid] : LAST;
  }
  const int size = n <= 512 ? 512 : 1024;
  u64 own = tid < n ? l.list[tid] : LAST;
  for (int run = 2; run <= size; run *= 2)
    for (int by = run / 2; by > 0; by /= 2) {
      u64 other;
      if (by >= 64) {
        __syncthreads();
        l.sorted[tid] = own;
        __syncthreads();
        other = l.sorted[tid ^ by];
      } else {
        other = __shfl_xor(own, by);
      }
      const bool least = ((tid & by) == 0) == ((tid & run) == 0);
      if (least ? other < own : other > own) own = other;
    }
  return own;
}

// e^((x - m) / T): 2^t goes to the hardware, with log2 e / T as two floats. t is rounded once. Weights do not rise
// where logits fall (looked at for every t from 0 to -128), so that what min_p keeps is in front of the rest.
struct Weigh {
  float m, hi, lo, least;  // the distance, finite for a masked token too, from which on a weight is 0
  __device__ __forceinline__ Weigh(float m, float temperature) : m(m) {
    const double c = 1.4426950408889634074 / (double)temperature;
    hi = (float)c;
    lo = (float)(c - (double)hi);
    least = -256.0f / hi;
  }
  __device__ __forceinline__ float operator()(float x) const {
    const float d = __builtin_fmaxf(x - m, least);
    return __builtin_amdgcn_exp2f(__builtin_fmaf(d, hi, d * lo));
  }
};
// In units of 2^-40, rounded: a whole number, as which a double adds them exactly up to 2^53.
__device__ __forceinline__ double whole(float w) { return __builtin_fma((double)w, 0x1p40, 0x1p52) - 0x1p52; }
__device__ __forceinline__ u64 units(float w) {
  return __builtin_bit_cast(u64, __builtin_fma((double)w, 0x1p40, 0x1p52)) & 0xfffffffffffffull;
}

// A border of the order: kept are logits above x, and those that are x up to index ``last``.
struct Border {
  float x;
  int last;
  __device__ __forceinline__ bool keeps(float y, int i) const { return (y > x) | ((y == x) & (i <= last)); }
};

template <class T> __device__ __forceinline__ void sample(const SampleArgs& a) {
  __shared__ __attribute__((aligned(16))) SampleLds l;
  const int b = blockIdx.x, tid = threadIdx.x, size = a.size;
  const T* const row = at<T>(a.logits, a.l_off) + b * a.lb;
  const float uniform = at<float>(a.uniform, a.u_off)[b * a.us];
  const float temperature = a.temperature ? at<float>(a.temperature, a.t_off)[b * a.ts] : 1.0f;
  int top_k = a.top_k ? at<int32_t>(a.top_k, a.k_off)[b * a.ks] : 0;
  const float top_p = a.top_p ? at<float>(a.top_p, a.p_off)[b * a.ps] : 1.0f;
  const float min_p = a.min_p ? at<float>(a.min_p, a.m_off)[b * a.ms] : 0.0f;
  constexpr float NONE = -__builtin_inff();

  // the row's last pack, with -infinity behind its end, and a whole pack of that
  T* const tail = reinterpret_cast<T*>(l.tail);
  if (tid < 16) tail[tid] = size / 8 * 8 + tid < size ? row[size / 8 * 8 + tid] : element<T>::narrow(NONE);
  __syncthreads();
  // f(8 logits, index of the first) of the packs of this thread from lo up to hi, a multiple of 8 from
  // lo or the row's end. One pack is on its way while one is in use.
  auto over = [&](int lo, int hi, int thread, int threads, auto f) __attribute__((always_inline)) {
    const int whole = hi < size / 8 * 8 ? hi : size / 8 * 8;
    int i = lo + thread * 8;
    T next[8];
    if (i < whole) load_n<(int)sizeof(T)>(next, row + i);
#pragma unroll 1
    for (; i < hi; i += threads * 8) {
      if (i >= whole) load_n<16>(next, tail);
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = element<T>::widen(next[j]);
      if (i + threads * 8 < whole) load_n<(int)sizeof(T)>(next, row + i + threads * 8);
      f(x, i);
    }
  };

  float own_top = NONE;
#pragma unroll 1
  for (int i = tid * 8; i < size; i += SAMPLE_THREADS * 32) {  // four packs on their way: from memory
    T x[4][8];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = i + u * SAMPLE_THREADS * 8;
      if (at + 8 <= size) load_n<(int)sizeof(T)>(x[u], row + at);
      else load_n<16>(x[u], at < size ? tail : tail + 8);  // the last one is one thread's, as in ``over``
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) own_top = __builtin_elementwise_maximum(own_top, element<T>::widen(x[u][j]));
  }
  float top = group_reduce<64, OpMax>(own_top);  // NaN where there is one
  if ((tid & 63) == 0) l.tops[tid >> 6] = top;
  __syncthreads();
  top = group_reduce<SAMPLE_WAVES, OpMax>(l.tops[tid & (SAMPLE_WAVES - 1)]);
  const bool fine = uniform >= 0.0f && uniform < 1.0f && temperature >= 0.0f && temperature <= MOST_TEMPERATURE &&
                    top_p >= 0.0f && top_p <= 1.0f && min_p >= 0.0f && min_p <= 1.0f && top < __builtin_inff();
  if (!fine || top == NONE) {
    if (tid == 0) {
      a.out[b] = -1;
      if (!fine) *a.error = INVALID_SAMPLE;
    }
    return;
  }
  if (temperature < LEAST_TEMPERATURE || top_k == 1) {
    uint32_t first = 0xffffffffu;
    if (own_top == top)  // few threads have it
      over(0, size, tid, SAMPLE_THREADS, [&](const float (&x)[8], int i) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 7; j >= 0; --j) first = x[j] == top && (uint32_t)(i + j) < first ? i + j : first;
      });
    for (int by = 1; by < 64; by *= 2) {
      const uint32_t y = __shfl_xor(first, by);
      first = y < first ? y : first;
    }
    if ((tid & 63) == 0) l.least[tid >> 6] = first;
    __syncthreads();
    for (int w = 0; w < SAMPLE_WAVES; ++w) first = l.least[w] < first ? l.least[w] : first;
    if (tid == 0) a.out[b] = first;
    return;
  }
  const Weigh weigh(top, temperature);
  if (top_k <= 0 || top_k >= size) top_k = 0;
  // logits below this have less than min_p's weight; which of the others have is for their weight to say
  const float least = min_p > 0.0f ? top + (__builtin_amdgcn_logf(min_p) - 0.01f) / weigh.hi : NONE;

  auto clear_bins = [&] {
    __syncthreads();
    l.bins[tid] = l.bins[tid + SAMPLE_THREADS] = 0;
    __syncthreads();
  };
  // Numbers that rise along the order. Each wave gathers its own, without atomics: ``held`` says how
  // many it has, which may be more than fit.
  const int wave = tid >> 6;
  auto x_of = [](u64 key) { return of_order(~(uint32_t)(key >> 32)); };
  int held = 0;
  // Of each lane the tokens from i on that ``bits`` names, as indexes first.
  auto put = [&](uint32_t bits, int i) __attribute__((always_inline)) {
#pragma unroll 1
    for (u64 mask = __ballot(bits != 0); mask && held <= SAMPLE_EACH; mask = __ballot(bits != 0)) {
      const int at = held + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
      if (bits && at < SAMPLE_EACH) l.gathered[wave][at] = (uint32_t)(i + __builtin_ctz(bits));
      bits &= bits - 1;
      held += __popcll(mask);
    }
  };
  auto settle = [&] {
    held = __builtin_amdgcn_readfirstlane(held);  // the first lane has seen all of the wave's
    __syncthreads();
#pragma unroll 1
    for (int n = tid & 63; n < held && n < SAMPLE_EACH; n += 64) {
      const uint32_t i = (uint32_t)l.gathered[wave][n];
      l.gathered[wave][n] = (u64)~order_of(element<T>::widen(row[i])) << 32 | i;
    }
  };
  // How many all waves have, and those of them that f says in one list, or more than fit it.
  auto collect = [&](auto f) __attribute__((always_inline)) {
    const bool fits = held <= SAMPLE_EACH;
    int own = 0;
    __syncthreads();  // gathered, and the list has been read
    if (fits)
#pragma unroll 1
      for (int i = tid & 63; i < held; i += 64) own += f(l.gathered[wave][i]);
    u64 below;
    const int n = (int)sum_over_threads(fits ? own : SAMPLE_LIST + 1, l, below);
    int at = (int)below;
    if (n <= SAMPLE_LIST)
#pragma unroll 1
      for (int i = tid & 63; i < held; i += 64) {
        const u64 key = l.gathered[wave][i];
        if (f(key)) l.list[at++] = key;
      }
    __syncthreads();
    return n;
  };
  auto any_of = [](u64) { return true; };
  auto gather = [&](auto f) __attribute__((always_inline)) {
    held = 0;
    over(0, size, tid, SAMPLE_THREADS, [&](const float (&x)[8], int i) __attribute__((always_inline)) {
      bool any = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) any |= f(x[j], i + j);
      if (__any(any)) {
        uint32_t bits = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) bits |= (f(x[j], i + j) & (i + j < size)) ? 1u << j : 0u;
        put(bits, i);
      }
    });
    settle();
    return collect(any_of);
  };
  // what of ``all`` lies in front of the token that is drawn
  auto target_of = [](double part, u64 all) {
    const u64 target = (u64)(part * (double)all);
    return target < all ? target : all - 1;
  };

  bool gathers = size <= SAMPLE_LIST;
  float from = NONE;
  if (!gathers && top_k && top_k <= SAMPLE_FEW) {
    // As many threads as top_k have a token at or above the end of the bin, a 64th, of their top_k-th: each one of
    // its own packs, so that as many tokens are gathered.
    l.bins[tid] = 0;  // two counts
    __syncthreads();
    atomicAdd(&l.counts[(int)__builtin_fminf((top - own_top) * 64.0f, (float)(SAMPLE_BINS - 1))], 1u);
    __syncthreads();
    const u64 first = l.counts[2 * tid], second = l.counts[2 * tid + 1];
    u64 below;
    sum_over_threads(first + second, l, below);
    if (below < (u64)top_k && below + first + second >= (u64)top_k) l.digits[0] = 2 * tid + 1;
    __syncthreads();
    const int bin = l.digits[0];
    gathers = bin < SAMPLE_BINS - 1;
    from = top - (float)(bin + 2) * 0x1p-6f;  // one more for roundings
  }
  if (top_p >= 1.0f && min_p > 0.0f) {
    gathers = true;
    from = least > from ? least : from;
  }
  if (gathers) {
    int n;
    if (tid == 0) l.digits[1] = l.digits[2] = 0;
    const int seers = __syncthreads_count(own_top >= from);
    // a place behind the ``counter`` for each lane of ``mask``
    auto place = [&](u64 mask, int* counter) __attribute__((always_inline)) {
      const int lane = __builtin_ctzll(mask);
      int first = 0;
      if ((tid & 63) == lane) first = atomicAdd(counter, __popcll(mask));
      return __builtin_amdgcn_readlane(first, lane) +
             (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
    };
    if (seers <= 512) {
      // few threads have one: all look through what those have seen, two tokens of theirs on their way
      const u64 some = __ballot(own_top >= from);
      if (some) {
        const int at = place(some, &l.digits[2]);
        if (own_top >= from) l.sorted[at] = tid;
      }
      __syncthreads();
      const int per = (size + SAMPLE_THREADS * 8 - 1) / (SAMPLE_THREADS * 8) * 8, all = seers * per;
      const float share = 1.0f / (float)per;
#pragma unroll 1
      for (int begin = 0; begin < all; begin += 2 * SAMPLE_THREADS) {
        int i[2];
        float x[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int at = begin + u * SAMPLE_THREADS + tid;
          const int nth = (int)(((float)at + 0.5f) * share), e = at - nth * per;  // at / per: below 2^21
          i[u] = at < all ? (int)l.sorted[nth] * 8 + e / 8 * (SAMPLE_THREADS * 8) + e % 8 : size;
          x[u] = i[u] < size ? element<T>::widen(row[i[u]]) : NONE;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const bool in = i[u] < size && x[u] >= from;
          const u64 mask = __ballot(in);
          if (mask) {
            const int at = place(mask, &l.digits[1]);
            if (in && at < SAMPLE_LIST) l.list[at] = (u64)~order_of(x[u]) << 32 | (uint32_t)i[u];
          }
        }
      }
      __syncthreads();
      n = l.digits[1];
    } else {
      n = gather([&](float x, int) __attribute__((always_inline)) { return x >= from; });
    }
    if (n <= SAMPLE_LIST) {
      // min_p alone asks for no order
      const bool orders = top_k || top_p < 1.0f;
      const u64 key = orders ? sort_list(n, l) : tid < n ? l.list[tid] : ~(u64)0;
      const bool in = tid < n && (top_k == 0 || tid < top_k);
      const float own = in ? weigh(x_of(key)) : 0.0f;
      bool kept = in && own >= min_p;
      u64 w = units(own), below;
      if (top_p < 1.0f) {
        const u64 all = sum_over_threads(w, l, below);
        kept = kept && (double)below < (double)top_p * (double)all;
      }
      kept |= tid == 0 && orders;
      w = kept ? w : 0;
      // of the first m, in the order of their indexes
      const int m = orders ? __syncthreads_count(kept) : n;
      u64 unused;
      if (m <= 256) {  // the weight of the kept ones in front, 8 at a time
        if (tid < m + 7) {
          l.list[tid] = tid < m ? (uint32_t)key : ~(u64)0;
          l.bins[tid] = w;
        }
        const u64 target = target_of(uniform, sum_over_threads(w, l, unused));
        below = 0;
        if (tid < m)
          for (int i = 0; i < m; i += 8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) below += l.list[i + j] < (uint32_t)key ? l.bins[i + j] : 0;
          }
        if (below <= target && target < below + w) a.out[b] = (uint32_t)key;
        return;
      }
      // the weight of every range of indexes, then of the tokens of one
      const int index = (int)(uint32_t)key, range = (size + SAMPLE_BINS - 1) / SAMPLE_BINS;
      clear_bins();
      if (w) atomicAdd(&l.bins[index / range], w);
      if (tid == 0) l.digits[1] = 0;
      __syncthreads();
      const u64 first = l.bins[2 * tid], second = l.bins[2 * tid + 1];
      const u64 target = target_of(uniform, sum_over_threads(first + second, l, below));
      if (below <= target && target < below + first + second) {
        l.digits[0] = 2 * tid + (below + first <= target);
        l.found[0] = below + first <= target ? below + first : below;
      }
      __syncthreads();
      const bool close = w && index / range == l.digits[0];
      if (close) {
        const int at = atomicAdd(&l.digits[1], 1);
        l.list[at] = index;
        l.bins[at] = w;
      }
      __syncthreads();
      if (close) {
        const int some = l.digits[1];
        below = l.found[0];
        for (int i = 0; i < some; ++i) below += l.list[i] < (u64)index ? l.bins[i] : 0;
        if (below <= target && target < below + w) a.out[b] = index;
      }
      return;
    }
  }

  // Border of the first tokens, among those in front of ``before``, whose ``mass`` reaches ``want``, a number
  // or, where that is 0, ``share`` of all: by 11, 11 and 10 bits of the logit, 11 and 11 of the index.
  auto find = [&](const Border& before, u64 want, double share, auto mass) __attribute__((always_inline)) {
    uint32_t k = 0, i = 0;  // what is known of the border's logit and index, and which bits that are
    uint32_t k_mask = 0, i_mask = 0;
#pragma unroll 1
    for (int level = 0; level < 5; ++level) {
      const bool of_index = level > 2;
      const int shift = level == 0 ? 21 : level == 1 ? 10 : level == 3 ? 11 : 0;
      const uint32_t digits = level == 2 ? 1023 : 2047;
      clear_bins();
      over(0, size, tid, SAMPLE_THREADS, [&](const float (&x)[8], int first) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t at = first + j, key = ~order_of(x[j]);
          const bool in = ((((key ^ k) & k_mask) | ((at ^ i) & i_mask)) == 0) & (at < (uint32_t)size) &
                          before.keeps(x[j], at);
          const u64 some = __ballot(in);
          if (some == 0) continue;
          // equal logits, the reason to be here, at once: atomics on one word go one after the other
          const int digit = ((of_index ? at : key) >> shift) & digits, lane = __builtin_ctzll(some);
          const bool same = in & (key == (uint32_t)__builtin_amdgcn_readlane(key, lane)) &
                            (digit == __builtin_amdgcn_readlane(digit, lane));
          const int n = __popcll(__ballot(same));
          if (in & (!same | ((tid & 63) == lane))) atomicAdd(&l.bins[digit], mass(x[j]) * (same ? n : 1));
        }
      });
      __syncthreads();
      const u64 one = l.bins[2 * tid], two = l.bins[2 * tid + 1];
      u64 below;
      const u64 all = sum_over_threads(one + two, l, below);
      if (want == 0) {
        want = (u64)__builtin_ceil(share * (double)all);
        want = want ? want : 1;
      }
      if (below < want && below + one + two >= want) {
        l.digits[0] = 2 * tid + (below + one < want);
        l.found[1] = below + one < want ? below + one : below;
      }
      __syncthreads();
      want -= l.found[1];
      (of_index ? i : k) |= (uint32_t)l.digits[0] << shift;
      (of_index ? i_mask : k_mask) |= digits << shift;
      __syncthreads();
    }
    return Border{of_order(~k), (int)i};
  };

  // Segments of the row: a sixteenth each for the 16 waves, and of the one that the token is in again,
  // until a wave sees all of it at once. ``part``: of a segment's kept weight what lies in front of the token.
  auto segment = [](int length) { return ((length + SAMPLE_WAVES - 1) / SAMPLE_WAVES + 511) / 512 * 512; };
  int lo = 0, hi = size, each = segment(size);
  double part = uniform;
  auto enter = [&](u64 own) __attribute__((always_inline)) {  // each lane's kept weight of its wave's segment
#pragma unroll
    for (int by = 1; by < 64; by *= 2) own += __shfl_xor(own, by);
    __syncthreads();
    if ((tid & 63) == 0) l.sums[wave] = own;
    __syncthreads();
    u64 before = 0, all = 0;
    for (int w = 0; w < SAMPLE_WAVES; ++w) {
      const u64 x = l.sums[w];
      before += w < wave ? x : 0;
      all += x;
    }
    const u64 target = target_of(part, all);
    if ((tid & 63) == 0 && before <= target && target < before + own) {
      l.digits[0] = wave;
      const double rest = (part * (double)all - (double)before) / (double)own;
      l.found[0] = __builtin_bit_cast(u64, __builtin_fmin(__builtin_fmax(rest, 0.0), 0x1.fffffffffffffp-1));
    }
    __syncthreads();
    lo += l.digits[0] * each;
    hi = lo + each < hi ? lo + each : hi;
    part = __builtin_bit_cast(double, l.found[0]);
    each = segment(hi - lo);
    __syncthreads();
  };

  Border kept = {NONE, 0x7fffffff};
  if (top_k || top_p < 1.0f) {
    // tokens in each 512th of a power of two of the weight
    const float per = 512.0f * weigh.hi;
    constexpr int COUNTS = SAMPLE_COUNTS, EACH = COUNTS / SAMPLE_THREADS;
    auto count_of = [&](float x) __attribute__((always_inline)) {
      return (int)__builtin_fminf((top - x) * per, (float)COUNTS);
    };
    // What is further away, or behind the row's end, is counted for each lane: the atomics of 64 on one
    // word take as long as on 64 words one after the other.
    const float far = (float)(COUNTS + (tid & 63));
    auto count = [&](float x) __attribute__((always_inline)) {
      atomicAdd(&l.counts[(int)__builtin_fminf((top - x) * per, far)], 1u);
    };
    auto clear_counts = [&] {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < EACH; j += 4)
        *reinterpret_cast<uint4v*>(&l.counts[j * SAMPLE_THREADS + tid * 4]) = uint4v{0, 0, 0, 0};
      __syncthreads();
    };
    clear_counts();
    over(0, size, tid, SAMPLE_THREADS, [&](const float (&x)[8], int) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) count(x[j]);
    });
    __syncthreads();
    if (top_k) {
      u64 own = 0, below;
#pragma unroll 4
      for (int j = 0; j < EACH; ++j) own += l.counts[tid * EACH + j];
      const u64 near = sum_over_threads(own, l, below);
      if (tid == 0 && near < (u64)top_k) {
        l.digits[0] = COUNTS;
        l.found[1] = near;
      }
      if (below < (u64)top_k && below + own >= (u64)top_k) {
        int bin = tid * EACH;
        while (below + l.counts[bin] < (u64)top_k) below += l.counts[bin++];
        l.digits[0] = bin;
        l.found[1] = below;
      }
      __syncthreads();
      const int bin = l.digits[0];
      const u64 more = top_k - l.found[1];  // of the bin
      const int n = gather([&](float x, int) __attribute__((always_inline)) { return (count_of(x) == bin) & (x > NONE); });
      if (n <= SAMPLE_LIST && (u64)n < more) {
        // all that has a weight is kept
      } else if (n <= SAMPLE_LIST) {
        const u64 key = sort_list(n, l);
        if ((u64)tid + 1 == more) l.found[0] = key;
        __syncthreads();
        kept = Border{x_of(l.found[0]), (int)(uint32_t)l.found[0]};
        // and are the only ones that count for top_p
#pragma unroll 4
        for (int j = 0; j < EACH; ++j)
          if (tid * EACH + j >= bin) l.counts[tid * EACH + j] = tid * EACH + j == bin ? (uint32_t)more : 0;
      } else {
        kept = find(kept, top_k, 0.0, [](float) { return (u64)1; });
        if (top_p < 1.0f) {
          clear_counts();
          over(0, size, tid, SAMPLE_THREADS, [&](const float (&x)[8], int i) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (kept.keeps(x[j], i + j)) count(x[j]);
          });
        }
      }
      __syncthreads();
    }
    if (top_p < 1.0f) {
      // If all bins' tokens had the most weight that their bin allows, up to where would the border be, and if
      // they had the least, RATIO of it (nothing of those far away)? It lies where the one is
      // large enough for the other's share, or before. A little apart, for roundings.
      constexpr double RATIO = 0x1.ffp-1;  // below 2^(-1/512 - 1/2048)
      const Border before = kept;
      const u64 limit = (u64)~order_of(before.x) << 32 | (uint32_t)before.last;
      const bool some = top_k != 0;
      const int start = wave * each, end = start + each < size ? start + each : size;
      int from_bin = 0, first_bin, last_bin;
      float early = 0.0f, late = 0.0f;
      double front_own;
      u64 all, in_front, want;
      // Behind that the weight in front of those bins is known. If they have more tokens than can be gathered, it
      // says which few of them the border is in (145384 logits with top_p = 0.99 76 us, and digit by digit 214).
#pragma unroll 1
      for (int turn = 0; turn < 2; ++turn) {
        float up_to[EACH], own = 0.0f, most = __builtin_amdgcn_exp2f((float)(tid * EACH) * -0x1p-9f + 0x1p-12f);
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
          own += (float)l.counts[tid * EACH + j] * most;
          up_to[j] = own;
          most *= 0x1.ff4eacp-1f;  // 2^(-1/512)
        }
        if (tid == 0) {
          l.digits[0] = l.digits[1] = COUNTS;
          l.digits[3] = 0;
        }
        u64 below;
        const double near = (double)sum_over_threads((u64)((double)own * 0x1p40), l, below) * 0x1p-40;
        if (turn == 0) {
          early = (float)(top_p * RATIO * near);
          late = (float)(top_p / RATIO * (near + size * 0x1p-32));
        }
        const float under = (float)below * 0x1p-40f;
        int first_of = EACH, last_of = EACH;
#pragma unroll
        for (int j = EACH - 1; j >= 0; --j) {
          first_of = under + up_to[j] >= early ? j : first_of;
          last_of = under + up_to[j] > late ? j : last_of;
        }
        // the first threads that have one, and perhaps one after them
        if (first_of < EACH && under <= early * 1.0001f) atomicMin(&l.digits[0], tid * EACH + first_of);
        if (last_of < EACH && under <= late * 1.0001f) atomicMin(&l.digits[1], tid * EACH + last_of);
        __syncthreads();
        // logits above ``high`` are in front of the first of those bins, below ``low`` behind the last
        first_bin = l.digits[0] > from_bin ? l.digits[0] : from_bin;
        last_bin = l.digits[1];
        const float high = first_bin == 0 ? __builtin_inff() : top - ((float)first_bin - 0.25f) / per;
        // nor is one where a border is already, or -infinity: the row's end
        const float low = __builtin_fmaxf(last_bin == COUNTS ? NONE : top - ((float)last_bin + 1.25f) / per,
                                          __builtin_fmaxf(before.x, -0x1.fffffep127f));
        double all_own = 0.0;
        front_own = 0.0;
        held = 0;
        over(start, end, tid & 63, 64, [&](const float (&x)[8], int i) __attribute__((always_inline)) {
          float w[8], sum = 0.0f, front = 0.0f;
          bool in[8], any = false;
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = weigh(x[j]);
          if (some) {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = before.keeps(x[j], i + j) ? w[j] : 0.0f;
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            sum += w[j];
            front += x[j] > high ? w[j] : 0.0f;
            in[j] = (x[j] >= low) & (x[j] <= high);
            any |= in[j];
          }
          all_own += whole(sum);
          front_own += whole(front);
          if (__any(any)) {
            uint32_t bits = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) bits |= in[j] ? 1u << j : 0u;
            put(bits, i);
          }
        });
        settle();
        if ((tid & 63) == 0) atomicAdd(&l.digits[3], held);
        u64 unused;
        all = sum_over_threads((u64)all_own, l, unused);
        in_front = sum_over_threads((u64)front_own, l, unused);
        const double share = __builtin_ceil((double)top_p * (double)all);
        want = share < 1.0 ? 1 : (u64)share;
        if (want <= in_front || !__syncthreads_or(held > SAMPLE_EACH)) break;
        // the last quarter of the bin in front of the first is not yet among what lies in front
        const float rest = (float)(want - in_front) * 0x1p-40f;
        const int front_bin = first_bin > 0 ? first_bin - 1 : 0;
        const float quarter = (float)l.counts[front_bin] * __builtin_amdgcn_exp2f((float)front_bin * -0x1p-9f + 0x1p-12f);
        early = first_bin == 0 ? 0.0f : __builtin_fmaxf(rest - quarter, 0.0f);
        late = rest / (float)RATIO;
        from_bin = first_bin;
        __syncthreads();
#pragma unroll 1
        for (int bin = tid * EACH; bin < (tid + 1) * EACH && bin < from_bin; ++bin) l.counts[bin] = 0;
      }
      bool done = false;
      if (want > in_front && !__syncthreads_or(held > SAMPLE_EACH)) {
        want -= in_front;
        int m = 0;
        if (l.digits[3] <= 256) {
          m = collect([&](u64 key) { return key <= limit; });
        } else {
          // not all of the window, but one of fine bins that it is taken apart into
          const float wide = (float)SAMPLE_BINS / (float)(last_bin - first_bin + 2);
          auto fine_bin = [&](u64 key) {
            const float at = ((top - x_of(key)) * per - ((float)first_bin - 0.5f)) * wide;
            return (int)__builtin_fminf(__builtin_fmaxf(at, 0.0f), (float)(SAMPLE_BINS - 1));
          };
          clear_bins();
#pragma unroll 1
          for (int i = tid & 63; i < held; i += 64) {
            const u64 key = l.gathered[wave][i];
            if (key <= limit) atomicAdd(&l.bins[fine_bin(key)], units(weigh(x_of(key))));
          }
          if (tid == 0) l.found[0] = ~(u64)0;
          __syncthreads();
          const u64 first = l.bins[2 * tid], second = l.bins[2 * tid + 1];
          u64 below;
          sum_over_threads(first + second, l, below);
          if (below < want && below + first + second >= want) {
            l.digits[0] = 2 * tid + (below + first < want);
            l.found[0] = below + first < want ? below + first : below;
          }
          __syncthreads();
          m = SAMPLE_LIST + 1;
          if (l.found[0] != ~(u64)0) {
            const int bin = l.digits[0];
            want -= l.found[0];
            m = collect([&](u64 key) { return key <= limit && fine_bin(key) == bin; });
          }
        }
        if (m <= SAMPLE_LIST) {
          const u64 key = sort_list(m, l);
          const u64 w = tid < m ? units(weigh(x_of(key))) : 0;
          if (tid == 0) l.found[0] = ~(u64)0;
          u64 below;
          sum_over_threads(w, l, below);
          if (below < want && below + w >= want) l.found[0] = key;
          __syncthreads();
          const u64 last = l.found[0];
          if (last != ~(u64)0) {
            kept = Border{x_of(last), (int)(uint32_t)last};
            done = true;
            if (weigh(kept.x) >= min_p) {
              // each wave's segment: what lies in front of the window, and what is kept of it
#pragma unroll 1
              for (int i = tid & 63; i < held; i += 64) {
                const u64 key = l.gathered[wave][i];
                if (key <= last) front_own += whole(weigh(x_of(key)));
              }
              enter((u64)front_own);
            }
          }
        }
      }
      if (!done)
        kept = find(before, 0, (double)top_p, [&](float x) __attribute__((always_inline)) { return units(weigh(x)); });
    }
  }

  // The kept weight of a pack is its weights' sum in fp32.
  const float least_weight = min_p;
  const bool plain = kept.x == NONE && min_p == 0.0f;
  const float above = kept.x == NONE ? NONE : of_order(order_of(kept.x) + 1);  // the next logit
  for (;;) {
    const int start = lo + wave * each, end = start + each < hi ? start + each : hi;
    auto weight_of = [&](float x, int i) __attribute__((always_inline)) {
      const float w = weigh(x);
      return ((x >= (i <= kept.last ? kept.x : above)) & (w >= least_weight)) ? w : 0.0f;
    };
    double own = 0.0;
    if (plain)
      over(start, end, tid & 63, 64, [&](const float (&x)[8], int) __attribute__((always_inline)) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += weigh(x[j]);
        own += whole(sum);
      });
    else
      over(start, end, tid & 63, 64, [&](const float (&x)[8], int i) __attribute__((always_inline)) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += weight_of(x[j], i + j);
        own += whole(sum);
      });
    if (each > 512) {
      enter((u64)own);
      continue;
    }
    // a lane has one pack
    u64 below;
    const u64 all = sum_over_threads((u64)own, l, below), target = target_of(part, all);
    if (below <= target && target < below + (u64)own)
      over(start, end, tid & 63, 64, [&](const float (&x)[8], int i) __attribute__((always_inline)) {
        float sum = 0.0f;
        int token = -1;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sum += weight_of(x[j], i + j);
          if (token < 0 && below + units(sum) > target) token = i + j;
        }
        a.out[b] = token;
      });
    return;
  }
}

}  // namespace mlc

#define SAMPLE(NAME, T)                                                                         \
  extern "C" __global__ void __launch_bounds__(mlc::SAMPLE_THREADS) NAME(mlc::SampleArgs a) {   \
    mlc::sample<T>(a);                                                                          \
  }
