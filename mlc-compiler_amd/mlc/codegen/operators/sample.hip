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
// on how a row is divided or on the order of atomics.
//
// A workgroup has a row, which its caches hold after the first pass, for the largest logit, the
// only one that memory bounds. A pass over 131072 tokens on one unit then costs 0.85 us for each
// instruction of a token. So what can be kept is gathered first where a bound for it is at
// hand (the top_k-th of the threads' own largest, or min_p) and fits a list: sorted in LDS, it
// says everything. Otherwise borders come from a histogram of distances to the largest, whose
// border bin fits the list, and the token from the kept weight of ever smaller segments.

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
constexpr int SAMPLE_THREADS = 1024, SAMPLE_WAVES = SAMPLE_THREADS / 64, SAMPLE_BINS = 2048;
constexpr int SAMPLE_LIST = 1024;                                          // a thread for each
constexpr int SAMPLE_FEW = 512;                                            // top_k whose tokens are gathered
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
  u64 bins[SAMPLE_BINS];  // and a list's weights
  u64 list[SAMPLE_LIST], sorted[SAMPLE_LIST];
  u64 sums[SAMPLE_WAVES];
  u64 found[2];
  float tops[SAMPLE_WAVES];
  uint32_t least[SAMPLE_WAVES];
  int count, digits[6];
};

// The sum of x over the workgroup; ``below``: of the threads before this one.
__device__ __forceinline__ u64 sum_over_threads(u64 x, SampleLds& l, u64& below) {
  u64 run = x;
#pragma unroll
  for (int by = 1; by < 64; by *= 2) {
    const u64 y = __shfl_up(run, by);
    if ((threadIdx.x & 63) >= by) run += y;
  }
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
  if (n <= 256) {  // by counting the ones below
    __syncthreads();
    if (tid < n) {
      const u64 own = l.list[tid];
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += l.list[i] < own;
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

// e^((x - m) / T): 2^t goes to the hardware, with log2 e / T as two floats. t is rounded once.
struct Weigh {
  float m, hi, lo, least;  // the distance from which on a weight is 2^-64
  __device__ __forceinline__ Weigh(float m, float temperature) : m(m) {
    const double c = 1.4426950408889634074 / (double)temperature;
    hi = (float)c;
    lo = (float)(c - (double)hi);
    least = -64.0f / hi;
  }
  __device__ __forceinline__ float operator()(float x) const {
    const float d = __builtin_fmaxf(x - m, least);
    return __builtin_amdgcn_exp2f(__builtin_fmaf(d, hi, d * lo));
  }
};
// In units of 2^-40, rounded; up to 8.
__device__ __forceinline__ u64 units(float w) {
  return __builtin_bit_cast(u64, __builtin_fma((double)w, 0x1p40, 0x1p52)) & 0xfffffffffffffull;
}

// A border of the order: kept are logits above x, and those that are x up to index ``last``.
struct Border {
  float x;
  int last;
  __device__ __forceinline__ bool keeps(float y, int i) const { return y > x || (y == x && i <= last); }
};

template <class T> __device__ __forceinline__ void sample(const SampleArgs& a) {
  __shared__ SampleLds l;
  const int b = blockIdx.x, tid = threadIdx.x, size = a.size;
  const T* const row = at<T>(a.logits, a.l_off) + b * a.lb;
  const float uniform = at<float>(a.uniform, a.u_off)[b * a.us];
  const float temperature = a.temperature ? at<float>(a.temperature, a.t_off)[b * a.ts] : 1.0f;
  int top_k = a.top_k ? at<int32_t>(a.top_k, a.k_off)[b * a.ks] : 0;
  const float top_p = a.top_p ? at<float>(a.top_p, a.p_off)[b * a.ps] : 1.0f;
  const float min_p = a.min_p ? at<float>(a.min_p, a.m_off)[b * a.ms] : 0.0f;

  // f(8 logits, index of the first) of the tokens of this thread from lo up to hi, which is a
  // multiple of 8 from lo or the row's end; -infinity past that. Four packs are on their way at a time.
  auto over = [&](int lo, int hi, int thread, int threads, auto f) __attribute__((always_inline)) {
    for (int i = lo + thread * 8; i < hi; i += threads * 32) {
      T x[4][8];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int at = i + u * threads * 8;
        if (at + 8 <= size && at < hi) load_n<(int)sizeof(T)>(x[u], row + at);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int at = i + u * threads * 8;
        if (at >= hi) break;
        float y[8];
        if (at + 8 <= size) {
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = element<T>::widen(x[u][j]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = at + j < size ? element<T>::widen(row[at + j]) : -__builtin_inff();
        }
        f(y, at);
      }
    }
  };

  float own_top = -__builtin_inff();
  over(0, size, tid, SAMPLE_THREADS, [&](const float (&x)[8], int) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) own_top = __builtin_elementwise_maximum(own_top, x[j]);
  });
  float top = own_top;
  for (int by = 1; by < 64; by *= 2) top = __builtin_elementwise_maximum(top, __shfl_xor(top, by));
  if ((tid & 63) == 0) l.tops[tid >> 6] = top;
  if (tid == 0) l.count = 0;
  __syncthreads();
  for (int w = 0; w < SAMPLE_WAVES; ++w) top = __builtin_elementwise_maximum(top, l.tops[w]);
  const bool fine = uniform >= 0.0f && uniform < 1.0f && temperature >= 0.0f && temperature <= MOST_TEMPERATURE &&
                    top_p >= 0.0f && top_p <= 1.0f && min_p >= 0.0f && min_p <= 1.0f && top < __builtin_inff();
  if (!fine || top == -__builtin_inff()) {
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
  float least = -__builtin_inff();  // the least logit of min_p's weight or more
  if (min_p > 0.0f) {
    const double x = (double)top + (double)temperature * log((double)min_p);
    least = (float)x;
    if ((double)least < x)  // the next float
      least = least == 0.0f ? 0x1p-149f : __builtin_bit_cast(float, __builtin_bit_cast(int, least) + (least > 0.0f ? 1 : -1));
  }

  auto clear_bins = [&] {
    __syncthreads();
    for (int i = tid; i < SAMPLE_BINS; i += SAMPLE_THREADS) l.bins[i] = 0;
    __syncthreads();
  };
  // The bin up to which the bins' sum reaches ``want``, and the sum in front of it
  auto find_bin = [&](u64 want, u64& before) {
    const u64 first = l.bins[2 * tid], second = l.bins[2 * tid + 1];
    u64 below;
    sum_over_threads(first + second, l, below);
    if (below < want && below + first >= want) {
      l.found[0] = 2 * tid;
      l.found[1] = below;
    } else if (below + first < want && below + first + second >= want) {
      l.found[0] = 2 * tid + 1;
      l.found[1] = below + first;
    }
    __syncthreads();
    before = l.found[1];
    return (int)l.found[0];
  };
  // the distance to the largest in 1 / per
  auto bin_of = [&](float x, float per) __attribute__((always_inline)) {
    return (int)__builtin_fminf((top - x) * per, (float)(SAMPLE_BINS - 1));
  };
  // Numbers that rise along the order, of the tokens that f says, into the list; how many there are,
  // which may be more than fit.
  auto gather = [&](auto f) __attribute__((always_inline)) {
    over(0, size, tid, SAMPLE_THREADS, [&](const float (&x)[8], int i) __attribute__((always_inline)) {
      bool any = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) any |= f(x[j], i + j);
      if (any) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (f(x[j], i + j) && i + j < size) {
            const int at = atomicAdd(&l.count, 1);
            if (at < SAMPLE_LIST) l.list[at] = (u64)~order_of(x[j]) << 32 | (uint32_t)(i + j);
          }
      }
    });
    __syncthreads();
    const int n = l.count;
    __syncthreads();
    if (tid == 0) l.count = 0;
    return n;
  };

  bool gathers = size <= SAMPLE_LIST;
  float from = -__builtin_inff();
  if (!gathers && top_k && top_k <= SAMPLE_FEW) {
    // as many threads as top_k have a token at or above the bin's end
    clear_bins();
    atomicAdd(&l.bins[bin_of(own_top, 64.0f)], (u64)1);
    __syncthreads();
    u64 before;
    const int bin = find_bin(top_k, before);
    gathers = bin < SAMPLE_BINS - 1;
    from = top - (float)(bin + 2) * 0x1p-6f;  // one more for roundings
  }
  if (top_p >= 1.0f && min_p > 0.0f) {
    gathers = true;
    from = least > from ? least : from;
  }
  if (gathers) {
    const int n = gather([&](float x, int) __attribute__((always_inline)) { return x >= from; });
    if (n <= SAMPLE_LIST) {
      const u64 key = sort_list(n, l);
      const float x = of_order(~(uint32_t)(key >> 32));
      const bool in = tid < n && (top_k == 0 || tid < top_k);
      u64 w = in ? units(weigh(x)) : 0, below, all = sum_over_threads(w, l, below);
      const bool kept = in && x >= least && (tid == 0 || top_p >= 1.0f || (double)below < (double)top_p * (double)all);
      // and once more by their indexes
      u64 rank;
      const int m = (int)sum_over_threads(kept, l, rank);  // the first m
      if (tid < m) {
        l.bins[tid] = w;
        l.list[tid] = key << 32 | tid;
      }
      const u64 again = sort_list(m, l);
      w = tid < m ? l.bins[(int)(again & (SAMPLE_LIST - 1))] : 0;
      all = sum_over_threads(w, l, below);
      const double wanted = (double)uniform * (double)all;  // below all: uniform is below 1
      if (w && (double)below <= wanted && (double)(below + w) > wanted) a.out[b] = (int64_t)(again >> 32);
      return;
    }
  }

  // Border of the first tokens, among those in front of ``before``, whose ``mass`` reaches ``want``, a number
  // or, where that is 0, ``share`` of all. By the distance's bin, and by the list, or
  // where that is too short by 11, 11 and 10 bits of the logit, 11 and 11 of the index.
  auto find = [&](const Border& before, u64 want, double share, float per, auto mass) __attribute__((always_inline)) {
    auto digit = [&](int level, float x, int i) __attribute__((always_inline)) -> int {
      if (level == 0) return bin_of(x, per);
      const uint32_t k = ~order_of(x);
      return level == 1 ? (int)(k >> 21) : level == 2 ? (int)(k >> 10 & 2047) : level == 3 ? (int)(k & 1023)
             : level == 4 ? i >> 11 : i & 2047;
    };
#pragma unroll 1
    for (int level = 0; level < 6; ++level) {
      clear_bins();
      over(0, size, tid, SAMPLE_THREADS, [&](const float (&x)[8], int i) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          bool in = before.keeps(x[j], i + j) && i + j < size;
          if (level > 0)
            for (int n = 0; n < level; ++n) in = in && digit(n, x[j], i + j) == l.digits[n];
          if (in) atomicAdd(&l.bins[digit(level, x[j], i + j)], mass(x[j]));
        }
      });
      __syncthreads();
      if (want == 0) {
        u64 below;
        const double part = share * (double)sum_over_threads(l.bins[2 * tid] + l.bins[2 * tid + 1], l, below);
        want = (u64)__builtin_ceil(part);
        want = want ? want : 1;
      }
      u64 front;
      const int bin = find_bin(want, front);
      if (tid == 0) l.digits[level] = bin;
      want -= front;
      if (level == 0) {
        const int n = gather([&](float x, int i) __attribute__((always_inline)) { return bin_of(x, per) == bin && before.keeps(x, i); });
        if (n <= SAMPLE_LIST) {
          const u64 key = sort_list(n, l);
          const u64 w = tid < n ? mass(of_order(~(uint32_t)(key >> 32))) : 0;
          u64 below;
          sum_over_threads(w, l, below);
          if (below < want && below + w >= want) l.found[0] = key;
          __syncthreads();
          const u64 last = l.found[0];
          return Border{of_order(~(uint32_t)(last >> 32)), (int)(uint32_t)last};
        }
      }
    }
    __syncthreads();
    return Border{of_order(~((uint32_t)l.digits[1] << 21 | (uint32_t)l.digits[2] << 10 | (uint32_t)l.digits[3])),
                  l.digits[4] << 11 | l.digits[5]};
  };

  Border kept = {-__builtin_inff(), 0x7fffffff};
  if (top_k) kept = find(kept, top_k, 0.0, 64.0f, [](float) { return (u64)1; });
  if (top_p < 1.0f)
    kept = find(kept, 0, (double)top_p, 64.0f * weigh.hi, [&](float x) __attribute__((always_inline)) { return units(weigh(x)); });
  if (least > kept.x) kept = Border{least, 0x7fffffff};

  // Segments of the row: a sixteenth each for the 16 waves, and of the one that the token is in
  // again, until a wave sees all of it at once. The kept weight of a pack is its weights' sum in fp32.
  int lo = 0, hi = size;
  u64 target = 0;
  double wanted = -1.0;
  for (;;) {
    const int each = ((hi - lo + SAMPLE_WAVES - 1) / SAMPLE_WAVES + 511) / 512 * 512;
    const int wave = tid >> 6, start = lo + wave * each, end = start + each < hi ? start + each : hi;
    u64 own = 0;
    over(start, end, tid & 63, 64, [&](const float (&x)[8], int i) __attribute__((always_inline)) {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += kept.keeps(x[j], i + j) ? weigh(x[j]) : 0.0f;
      own += units(sum);
    });
    u64 below;
    const u64 all = sum_over_threads(own, l, below);
    if (wanted < 0.0) wanted = (double)uniform * (double)all;
    if (each <= 512) {  // a lane has one pack
      const u64 first = target + below;
      if (own && (double)first <= wanted && (double)(first + own) > wanted) {
        float sum = 0.0f;
        int token = -1;
        over(start, end, tid & 63, 64, [&](const float (&x)[8], int i) __attribute__((always_inline)) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            sum += kept.keeps(x[j], i + j) ? weigh(x[j]) : 0.0f;
            if (token < 0 && (double)(first + units(sum)) > wanted) token = i + j;
          }
        });
        a.out[b] = token;
      }
      return;
    }
    u64 front = target;
    for (int w = 0; w < wave; ++w) front += l.sums[w];
    if ((tid & 63) == 0 && (double)front <= wanted && (double)(front + l.sums[wave]) > wanted) {
      l.found[0] = wave;
      l.found[1] = front;
    }
    __syncthreads();
    lo += (int)l.found[0] * each;
    hi = lo + each < hi ? lo + each : hi;
    target = l.found[1];
    __syncthreads();
  }
}

}  // namespace mlc

#define SAMPLE(NAME, T)                                                                         \
  extern "C" __global__ void __launch_bounds__(mlc::SAMPLE_THREADS) NAME(mlc::SampleArgs a) {   \
    mlc::sample<T>(a);                                                                          \
  }
