// Rotary positions. Pair (a, b) of a head's first ``turned`` values at position p
// becomes (a cos t - b sin t, a sin t + b cos t) * magnitude, t = p * frequency;
// a pair is (2i, 2i + 1) or (i, i + turned/2). The values behind are copied.
//
// Bound by memory: every value is read once and written once. The angle is
// taken in 64 bits (a position of 10^6 leaves an fp32 angle 0.06 off), as turns
// minus whole turns, and evaluated once for each (token, pair): a workgroup
// fills LDS with the cosines and sines of its tokens, then streams all heads of
// queries and keys past them in 16-byte packs.

namespace mlc {

struct RotaryArgs {
  const void* q;
  const void* k;
  const void* positions;
  const void* frequencies;
  void* qo;
  void* ko;
  int64_t q_off, k_off, p_off, f_off;         // bytes
  int64_t qb, qt, qh, kb, kt, kh, pb, pt, fs;  // elements
  int32_t tokens, seq, heads, kv_heads, dim, turned, group, wide_positions;
  float magnitude;
  int32_t pad;
};

constexpr int ROTARY_BLOCK = 256;
constexpr int ROTARY_PAIRS = 1024;  // pairs of LDS: group * turned / 2 at most

template <class T, int V, bool INTERLEAVED>
__device__ __forceinline__ void rotary(const RotaryArgs& a) {
  constexpr int A = V > 1 ? 16 : (int)sizeof(T);
  __shared__ __attribute__((aligned(16))) float cs[ROTARY_PAIRS], sn[ROTARY_PAIRS];
  const int half = a.turned / 2;
  const T* q = at<T>(a.q, a.q_off);
  const T* k = at<T>(a.k, a.k_off);
  const double* f = at<double>(a.frequencies, a.f_off);
  T* const qo = reinterpret_cast<T*>(a.qo);
  T* const ko = reinterpret_cast<T*>(a.ko);
  const int heads = a.heads + a.kv_heads;
  // items of one head: packs of pairs, then packs that are copied
  const int turns = INTERLEAVED ? a.turned / V : half / V;
  const int per_head = turns + (a.dim - a.turned) / V;
  const int per_token = heads * per_head;
  for (int64_t first = (int64_t)blockIdx.x * a.group; first < a.tokens;
       first += (int64_t)gridDim.x * a.group) {
    const int n = a.tokens - first < a.group ? (int)(a.tokens - first) : a.group;
    for (int i = threadIdx.x; i < n * half; i += ROTARY_BLOCK) {
      const int64_t token = first + i / half;
      const int64_t b = token / a.seq, t = token % a.seq;
      const int64_t at_p = b * a.pb + t * a.pt;
      const double p = a.wide_positions ? (double)at<int64_t>(a.positions, a.p_off)[at_p]
                                        : (double)at<int32_t>(a.positions, a.p_off)[at_p];
      // quarter turns: the nearest whole number of them goes to the quadrant
      const double w = p * f[(i % half) * a.fs] * 0.63661977236758134308;
      const double whole = __builtin_rint(w);
      const int quadrant = (int)(whole - 4.0 * __builtin_floor(whole * 0.25));
      float s, c;
      sincosf((float)((w - whole) * 1.57079632679489661923), &s, &c);
      float x = quadrant & 1 ? s : c, y = quadrant & 1 ? c : s;
      x = quadrant == 1 || quadrant == 2 ? -x : x;
      y = quadrant >= 2 ? -y : y;
      cs[i] = x * a.magnitude;
      sn[i] = y * a.magnitude;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * per_token; i += ROTARY_BLOCK) {
      const int g = i / per_token, rest = i % per_token;
      const int h = rest / per_head, item = rest % per_head;
      const int64_t token = first + g;
      const int64_t b = token / a.seq, t = token % a.seq;
      const bool is_q = h < a.heads;
      const int kh = h - a.heads;
      const T* src = is_q ? q + b * a.qb + t * a.qt + h * a.qh : k + b * a.kb + t * a.kt + kh * a.kh;
      T* dst = is_q ? qo + (token * a.heads + h) * a.dim : ko + (token * a.kv_heads + kh) * a.dim;
      T x[V], y[V];
      if (item >= turns) {
        const int d = a.turned + (item - turns) * V;
        load_n<A>(x, src + d);
        store_n<A>(dst + d, x);
        continue;
      }
      if constexpr (INTERLEAVED) {
        // V == 1: one pair of two values
        constexpr int N = V > 1 ? V : 2;
        const int d = item * V;
        if constexpr (V == 1) {
          if (d & 1) continue;  // the even value's item turns both
        }
        T z[N];
        load_n<A>(z, src + d);
        const float* c = cs + g * half + d / 2;
        const float* s = sn + g * half + d / 2;
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
          const float u = element<T>::widen(z[2 * j]), v = element<T>::widen(z[2 * j + 1]);
          z[2 * j] = element<T>::narrow(u * c[j] - v * s[j]);
          z[2 * j + 1] = element<T>::narrow(u * s[j] + v * c[j]);
        }
        store_n<A>(dst + d, z);
      } else {
        const int d = item * V;
        load_n<A>(x, src + d);
        load_n<A>(y, src + half + d);
        const float* c = cs + g * half + d;
        const float* s = sn + g * half + d;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float u = element<T>::widen(x[j]), v = element<T>::widen(y[j]);
          x[j] = element<T>::narrow(u * c[j] - v * s[j]);
          y[j] = element<T>::narrow(u * s[j] + v * c[j]);
        }
        store_n<A>(dst + d, x);
        store_n<A>(dst + half + d, y);
      }
    }
    __syncthreads();
  }
}

}  // namespace mlc

#define ROTARY(NAME, T, V, INTERLEAVED)                                                    \
  extern "C" __global__ void __launch_bounds__(mlc::ROTARY_BLOCK) NAME(mlc::RotaryArgs a) { \
    mlc::rotary<T, V, INTERLEAVED>(a);                                                     \
  }
