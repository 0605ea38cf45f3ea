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
constexpr int ROTARY_TOKENS = 64;   // and group

// V values (a pack) at a time: the largest power of two up to 16 bytes that divides sizes,
// strides and addresses. 4 x 4096 tokens, 32 + 8 heads of 128, bf16: 69 us, 4.9 TB/s (a copy
// reaches 5.2); 2 x 4096 tokens in fp32, pairs side by side: 63 us.
template <class T, int V, bool INTERLEAVED>
__device__ __forceinline__ void rotary(const RotaryArgs& a) {
  constexpr int A = V * (int)sizeof(T);
  __shared__ __attribute__((aligned(16))) float cs[ROTARY_PAIRS], sn[ROTARY_PAIRS];
  __shared__ int64_t q_row[ROTARY_TOKENS], k_row[ROTARY_TOKENS];
  const uint32_t half = a.turned / 2, heads = a.heads + a.kv_heads;
  const T* const q = at<T>(a.q, a.q_off);
  const T* const k = at<T>(a.k, a.k_off);
  const double* const f = at<double>(a.frequencies, a.f_off);
  T* const qo = reinterpret_cast<T*>(a.qo);
  T* const ko = reinterpret_cast<T*>(a.ko);
  // items of one head: packs of pairs, then packs that are copied
  const uint32_t turns = (INTERLEAVED ? (uint32_t)a.turned : half) / V;
  const uint32_t items = turns + (a.dim - a.turned) / V;
  // a thread keeps its item and goes through (token, head) rows, ``abreast`` at a time
  const uint32_t lanes = items < ROTARY_BLOCK ? items : ROTARY_BLOCK, abreast = ROTARY_BLOCK / lanes;
  const uint32_t own_row = threadIdx.x / lanes, own_item = threadIdx.x % lanes;
  const float per_head = 1.0f / (float)heads;

  for (uint32_t first = blockIdx.x * (uint32_t)a.group; first < (uint32_t)a.tokens;
       first += gridDim.x * (uint32_t)a.group) {
    const uint32_t n = a.tokens - first < (uint32_t)a.group ? a.tokens - first : a.group;
    for (uint32_t i = threadIdx.x; i < n; i += ROTARY_BLOCK) {
      const uint32_t b = (first + i) / (uint32_t)a.seq, t = (first + i) % (uint32_t)a.seq;
      q_row[i] = b * a.qb + t * a.qt;
      k_row[i] = b * a.kb + t * a.kt;
    }
    for (uint32_t i = threadIdx.x; i < n * half; i += ROTARY_BLOCK) {
      const uint32_t token = first + i / half;
      const int64_t at_p = token / (uint32_t)a.seq * a.pb + token % (uint32_t)a.seq * a.pt;
      const double p = a.wide_positions ? (double)at<int64_t>(a.positions, a.p_off)[at_p]
                                        : (double)at<int32_t>(a.positions, a.p_off)[at_p];
      // quarter turns: the nearest whole number of them goes to the quadrant
      const double w = p * f[i % half * a.fs] * 0.63661977236758134308;
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
    const uint32_t rows = n * heads;
    for (uint32_t r = own_row < abreast ? own_row : rows; r < rows; r += abreast) {
      const uint32_t g = (uint32_t)(((float)r + 0.5f) * per_head);  // r / heads: r stays below 2^20
      const uint32_t h = r - g * heads;
      const bool is_q = h < (uint32_t)a.heads;
      const uint32_t kh = h - a.heads;
      const T* const src = is_q ? q + q_row[g] + h * a.qh : k + k_row[g] + kh * a.kh;
      const int64_t token = first + g;
      T* const dst = is_q ? qo + (token * a.heads + h) * a.dim : ko + (token * a.kv_heads + kh) * a.dim;
      for (uint32_t item = own_item; item < items; item += ROTARY_BLOCK) {
        T x[V], y[V];
        if (item >= turns) {
          const uint32_t d = a.turned + (item - turns) * V;
          load_n<A>(x, src + d);
          store_n<A>(dst + d, x);
          continue;
        }
        if constexpr (INTERLEAVED && V == 1) {
          const uint32_t d = item;
          if (d & 1) continue;  // the even value's item turns both
          const float u = element<T>::widen(src[d]), v = element<T>::widen(src[d + 1]);
          const float c = cs[g * half + d / 2], s = sn[g * half + d / 2];
          dst[d] = element<T>::narrow(u * c - v * s);
          dst[d + 1] = element<T>::narrow(u * s + v * c);
        } else if constexpr (INTERLEAVED) {
          const uint32_t d = item * V;
          load_n<A>(x, src + d);
          float c[V / 2], s[V / 2];
          load_n<V * 2>(c, cs + g * half + d / 2);
          load_n<V * 2>(s, sn + g * half + d / 2);
#pragma unroll
          for (int j = 0; j < V / 2; ++j) {
            const float u = element<T>::widen(x[2 * j]), v = element<T>::widen(x[2 * j + 1]);
            y[2 * j] = element<T>::narrow(u * c[j] - v * s[j]);
            y[2 * j + 1] = element<T>::narrow(u * s[j] + v * c[j]);
          }
          store_n<A>(dst + d, y);
        } else {
          const uint32_t d = item * V;
          load_n<A>(x, src + d);
          load_n<A>(y, src + half + d);
          float c[V], s[V];
          load_n<4 * (V < 4 ? V : 4)>(c, cs + g * half + d);
          load_n<4 * (V < 4 ? V : 4)>(s, sn + g * half + d);
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
    }
    __syncthreads();
  }
}

}  // namespace mlc

#define ROTARY(NAME, T, V, INTERLEAVED)                                                    \
  extern "C" __global__ void __launch_bounds__(mlc::ROTARY_BLOCK) NAME(mlc::RotaryArgs a) { \
    mlc::rotary<T, V, INTERLEAVED>(a);                                                     \
  }
