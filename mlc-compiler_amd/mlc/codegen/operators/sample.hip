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
// Weights are whole numbers of 2^-40, so sums are exact whatever their order: results do not
// depend on how a row is divided or on the order of atomics. Borders are found by histograms of the
// order's digits, (a logit's distance to the largest, its 32 bits, the index), each over what
// the digits before have left.

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
constexpr int SAMPLE_THREADS = 1024, SAMPLE_BINS = 2048;
constexpr float LEAST_TEMPERATURE = 0x1p-100f, MOST_TEMPERATURE = 0x1p100f;  // below the least the likeliest token

// A number that orders as floats do, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct SampleLds {
  u64 bins[SAMPLE_BINS];
  u64 sums[16];
  u64 found[2];
  float tops[16];
  uint32_t least[16];
};

// The sum of x over the workgroup; ``below``: of the threads before this one.
__device__ __forceinline__ u64 sum_over_threads(u64 x, SampleLds& l, u64* below = nullptr) {
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
  for (int w = 0; w < SAMPLE_THREADS / 64; ++w) {
    if (w < (int)(threadIdx.x >> 6)) before += l.sums[w];
    all += l.sums[w];
  }
  if (below) *below = before + run - x;
  return all;
}

// e^((x - m) / T) in units of 2^-40, rounded. 2^t goes to the hardware with t rounded, and what
// the rounding left (with the factor's own) comes back to first order: 2^-23 of a weight is off.
struct Weigh {
  float m, hi, lo, least;  // log2 e / T as two floats; the distance from which on a weight is 2^-64
  __device__ __forceinline__ Weigh(float m, float temperature) : m(m) {
    const double c = 1.4426950408889634074 / (double)temperature;
    hi = (float)c;
    lo = (float)(c - (double)hi);
    least = -64.0f / hi;
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    const float d = __builtin_fmaxf(x - m, least), t = d * hi;
    const float e = __builtin_fmaf(d, lo, __builtin_fmaf(d, hi, -t));
    const float p = __builtin_amdgcn_exp2f(t);
    const double w = (double)__builtin_fmaf(p, e * 0x1.62e430p-1f, p);
    return __builtin_bit_cast(u64, __builtin_fma(w, 0x1p40, 0x1p52)) & 0xfffffffffffffull;
  }
};

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

  // f(logit, index) of every token of this thread from lo up to hi, a multiple of 8 from lo
  auto over = [&](int lo, int hi, int thread, int threads, auto f) __attribute__((always_inline)) {
    for (int i = lo + thread * 8; i < hi; i += threads * 8) {
      T x[8];
      if (i + 8 <= size) {
        load_n<(int)sizeof(T)>(x, row + i);
#pragma unroll
        for (int j = 0; j < 8; ++j) f(element<T>::widen(x[j]), i + j);
      } else {
        for (int j = 0; j < 8 && i + j < size; ++j) f(element<T>::widen(row[i + j]), i + j);
      }
    }
  };

  float top = -__builtin_inff();
  over(0, size, tid, SAMPLE_THREADS, [&](float x, int) { top = __builtin_elementwise_maximum(top, x); });
  for (int by = 1; by < 64; by *= 2) top = __builtin_elementwise_maximum(top, __shfl_xor(top, by));
  if ((tid & 63) == 0) l.tops[tid >> 6] = top;
  __syncthreads();
  for (int w = 0; w < SAMPLE_THREADS / 64; ++w) top = __builtin_elementwise_maximum(top, l.tops[w]);
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
    over(0, size, tid, SAMPLE_THREADS, [&](float x, int i) { first = x == top && (uint32_t)i < first ? i : first; });
    for (int by = 1; by < 64; by *= 2) {
      const uint32_t y = __shfl_xor(first, by);
      first = y < first ? y : first;
    }
    if ((tid & 63) == 0) l.least[tid >> 6] = first;
    __syncthreads();
    for (int w = 0; w < SAMPLE_THREADS / 64; ++w) first = l.least[w] < first ? l.least[w] : first;
    if (tid == 0) a.out[b] = first;
    return;
  }
  const Weigh weigh(top, temperature);
  if (top_k <= 0 || top_k >= size) top_k = 0;

  // Border of the first tokens, among those in front of ``before``, whose ``mass`` reaches ``want``
  // (1 or more, and not more than all of them have). Digits: the distance in 64ths of
  // a unit of ``per``, 11, 11 and 10 bits of the logit, 11 and 11 of the index.
  auto find = [&](const Border& before, u64 want, float per, auto mass) __attribute__((always_inline)) {
    auto digit = [&](int level, float x, int i) __attribute__((always_inline)) -> int {
      if (level == 0) return (int)__builtin_fminf((top - x) * per, (float)(SAMPLE_BINS - 1));
      const uint32_t k = ~order_of(x);
      return level == 1 ? (int)(k >> 21) : level == 2 ? (int)(k >> 10 & 2047) : level == 3 ? (int)(k & 1023)
             : level == 4 ? i >> 11 : i & 2047;
    };
    int digits[6];
    for (int level = 0; level < 6; ++level) {
      for (int i = tid; i < SAMPLE_BINS; i += SAMPLE_THREADS) l.bins[i] = 0;
      __syncthreads();
      over(0, size, tid, SAMPLE_THREADS, [&](float x, int i) {
        if (!before.keeps(x, i)) return;
        for (int n = 0; n < level; ++n)
          if (digit(n, x, i) != digits[n]) return;
        atomicAdd(&l.bins[digit(level, x, i)], mass(x));
      });
      __syncthreads();
      const u64 first = l.bins[2 * tid], second = l.bins[2 * tid + 1];
      u64 below;
      sum_over_threads(first + second, l, &below);
      if (below < want && below + first >= want) {
        l.found[0] = 2 * tid;
        l.found[1] = below;
      } else if (below + first < want && below + first + second >= want) {
        l.found[0] = 2 * tid + 1;
        l.found[1] = below + first;
      }
      __syncthreads();
      digits[level] = (int)l.found[0];
      want -= l.found[1];
      __syncthreads();
    }
    const uint32_t k = ~((uint32_t)digits[1] << 21 | (uint32_t)digits[2] << 10 | (uint32_t)digits[3]);
    return Border{__builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k), digits[4] << 11 | digits[5]};
  };

  Border kept = {-__builtin_inff(), 0x7fffffff};
  if (top_k) kept = find(kept, top_k, 64.0f, [](float) { return (u64)1; });
  if (top_p < 1.0f) {
    u64 own = 0;
    over(0, size, tid, SAMPLE_THREADS, [&](float x, int i) { own += kept.keeps(x, i) ? weigh(x) : 0; });
    const double share = (double)top_p * (double)sum_over_threads(own, l);
    const u64 want = (u64)__builtin_ceil(share);
    kept = find(kept, want ? want : 1, 64.0f * weigh.hi, [&](float x) { return weigh(x); });
  }
  if (min_p > 0.0f) {
    // the least logit of that weight or more
    const double least = (double)top + (double)temperature * log((double)min_p);
    float x = (float)least;
    if ((double)x < least)  // the next float
      x = x == 0.0f ? 0x1p-149f : __builtin_bit_cast(float, __builtin_bit_cast(int, x) + (x > 0.0f ? 1 : -1));
    if (x > kept.x) kept = Border{x, 0x7fffffff};
  }

  // Segments of the row: a sixteenth each for the 16 waves, and of the one that the token is in
  // again, until a wave sees all of it at once.
  int lo = 0, hi = size;
  u64 target = 0;
  double wanted = -1.0;
  for (;;) {
    const int each = ((hi - lo + SAMPLE_THREADS / 64 - 1) / (SAMPLE_THREADS / 64) + 511) / 512 * 512;
    const int wave = tid >> 6, from = lo + wave * each, to = from + each < hi ? from + each : hi;
    u64 own = 0;
    over(from, to, tid & 63, 64, [&](float x, int i) { own += kept.keeps(x, i) ? weigh(x) : 0; });
    u64 below;
    const u64 all = sum_over_threads(own, l, &below);
    if (wanted < 0.0) wanted = (double)uniform * (double)all;  // below all: uniform is below 1
    // the sum up to and with a token is above ``wanted``
    const u64 mine = l.sums[wave];
    u64 start = target;
    for (int w = 0; w < wave; ++w) start += l.sums[w];
    const bool here = (double)start <= wanted && (double)(start + mine) > wanted;
    if (each <= 512) {
      // lanes have 8 neighbouring tokens each
      const u64 at_lane = target + below;
      if ((double)at_lane <= wanted && (double)(at_lane + own) > wanted) {
        u64 run = at_lane;
        int token = -1;
        over(from, to, tid & 63, 64, [&](float x, int i) {
          run += kept.keeps(x, i) ? weigh(x) : 0;
          if (token < 0 && (double)run > wanted) token = i;
        });
        a.out[b] = token;
      }
      return;
    }
    if (here && (tid & 63) == 0) {
      l.found[0] = wave;
      l.found[1] = start;
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
