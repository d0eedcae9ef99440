// The probability of given tokens under rows of logits, and the losses and
// gradients made of it.
//
//   logp = x_y - m - log S,   m = max_k x_k,  S = sum_k exp(x_k - m)
//   d loss / d x_k = c (1[k = y] - exp(x_k - m) / S),  c = d loss / d logp
//
// A row of weight 0 is not read: its logp is 0 and its gradient row is zeros.
// A token outside [0, K) in a row that counts makes its logp NaN, and with it
// the row's gradient, unless c is 0: nothing depends on the row then.
// The sums of a row and what follows them (log, ratio, comparison with the
// clip's borders, sums over tokens) are in 64 bits: an error of 1e-7 there could
// move a token across a border, and a gain adds up those of hundreds of tokens.
#include <hip/hip_runtime.h>

#include "opcommon.h"

namespace {

using namespace wap;

struct Rows {
  const int64_t* y;   // [N]
  const float* w;     // [N] weights, or null: all one
  long sb, st;        // strides of logits over sequence and time
  long N, T;          // rows, rows of one sequence
  int K;
};

// What the policy loss takes for a row.
struct Policy {
  const float *old_logp, *adv, *ref;  // ref may be null
  long ab, at;                        // strides of adv
  double lo, hi, beta;
};

__device__ __forceinline__ float weight(const Rows& r, long row) {
  return r.w ? r.w[row] : 1.f;
}

// Rows and sequences are below 2^31: their quotients are 32-bit work.
__device__ __forceinline__ long row_at(const Rows& r, uint32_t row) {
  return (long)(row / (uint32_t)r.T) * r.sb + (long)(row % (uint32_t)r.T) * r.st;
}

// 16 bytes of a row, which may begin at any element.
template <typename T>
struct Wide {
  static constexpr int V = 16 / sizeof(T);
  typedef typename VecOf<T, V, sizeof(T)>::type type;
};

// A row as `whole` vectors of 16 bytes from its first element on, wherever that
// lies (rows of 50001 f32 tokens read at 5.6 TB/s, rows of 50000 at 5.7; and a
// sum does not depend on the place), and the `rest` behind them, one a lane.
template <typename T>
struct Cut {
  int whole, rest;

  __device__ __forceinline__ explicit Cut(int K) {
    whole = K / Wide<T>::V;
    rest = K - whole * Wide<T>::V;
  }
  // token of vector i, and of a lane of the rest
  __device__ __forceinline__ long vec_at(int i) const {
    return (long)i * Wide<T>::V;
  }
  __device__ __forceinline__ int rest_at(int lane) const {
    return whole * Wide<T>::V + lane;
  }
};

constexpr float LOG2E = 1.44269502162933349609f;
// log2 e = LOG2E (1 + LOST)
constexpr double LOST = 1.92596299112661746887e-8 / 1.44269502162933349609;

// log2 of exp(x - m).  x - m first: it is exact where it matters, and lowest
// values stay finite.
__device__ __forceinline__ float log2_from(float x, float m) {
  return (x - m) * LOG2E;
}

__device__ __forceinline__ float exp_from(float x, float m) {
  return __builtin_amdgcn_exp2f(log2_from(x, m));
}

// Exponentials of a row, added up.  The sum is 64-bit: a row's largest
// exponential is 1, and an f32 sum beside it would round every other one to
// 2^-24, which a gain over hundreds of tokens adds up.  What e = exp2(u) lacks
// goes into `t`, to first order, and is a millionth of the sum: f32.
// - f32 logits: u's own rounding and LOG2E's, from two products more.
// - 16-bit logits, whose differences have few bits: LOG2E's alone, which makes
//   every e too large by u LOST ln 2 (5e-8 of the sum).
template <typename T>
struct Sum {
  static constexpr bool FINE = sizeof(T) == 4;
  double s = 0.0;
  float t = 0.f;

  // e, and its share of t
  __device__ __forceinline__ float take(float x, float m) {
    // 2^-150 is nothing beside the maximum's 1, and what it is multiplied with
    // stays finite
    const float d = __builtin_elementwise_maximum(x - m, -104.f);
    const float u = d * LOG2E;
    const float e = __builtin_amdgcn_exp2f(u);
    if constexpr (FINE)
      t = fmaf(e, fmaf(d, (float)(LOST * LOG2E), fmaf(d, LOG2E, -u)), t);
    else
      t = fmaf(e, u, t);
    return e;
  }
  __device__ __forceinline__ void add(float x, float m) {
    s += (double)take(x, m);
  }
  __device__ __forceinline__ void add(const Sum& o) {
    s += o.s;
    t += o.t;
  }
  // to another maximum
  __device__ __forceinline__ void scale(double f) {
    s *= f;
    t *= (float)f;
  }
  __device__ __forceinline__ double value() const {
    constexpr double ln2 = 0.693147180559945309417;
    return s + (double)t * (FINE ? ln2 : LOST * ln2);
  }
};

// The hardware's exp2 is too small by this share on average (all fractions
// alike, arguments in [-30, 0]: 3.4e-9 in each octave below -1/2), exp2(0) is
// exact: a sum `v` of which `exact` is the largest's, with that put right.
__device__ __forceinline__ double with_mean(double v, double exact) {
  return v + 3.4e-9 * (v - exact);
}

// Over the workgroup, on every thread; `red`: one value a wave.
// The sum of the threads' parts is in 64 bits, for the logarithm.
template <int NT>
__device__ __forceinline__ double group_sum(double v, double* red) {
  v = lanes_sum(v);
  if constexpr (NT == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) s += red[i];
  return s;
}

template <int NT>
__device__ __forceinline__ float group_max(float v, float* red) {
  v = lanes_max(v);
  if constexpr (NT == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = red[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) s = fmaxf(s, red[i]);
  return s;
}

// logp of a row from its token's logit, maximum and sum.
__device__ __forceinline__ double row_logp(float xy, float m, double sum) {
  return (double)xy - (double)m - log(sum);
}

// What a row of the policy loss is given, read while the row is on its way.
struct Given {
  float adv = 0.f, old_logp = 0.f, ref = 0.f;

  Given() = default;
  __device__ __forceinline__ Given(const Policy& p, uint32_t row, uint32_t T)
      : adv(p.adv[(long)(row / T) * p.ab + (long)(row % T) * p.at]),
        old_logp(p.old_logp[row]),
        ref(p.ref ? p.ref[row] : 0.f) {}
};

// Loss of one token and its derivative by logp, both without the 1 / sum of
// weights.  At a border of the clip the unclipped side counts.
__device__ __forceinline__ void policy_row(const Policy& p, const Given& g,
                                           double logp, double* loss,
                                           double* slope) {
  const double adv = g.adv;
  const double ratio = exp(logp - (double)g.old_logp);
  const double kept = fmin(fmax(ratio, 1.0 - p.lo), 1.0 + p.hi);
  // an advantage of 0 is worth nothing, however far the ratio is off; a NaN
  // stays one
  const double free_ = adv == 0.0 && ratio == ratio ? 0.0 : ratio * adv;
  const double clipped = kept * adv;
  const bool on = !(free_ > clipped);  // NaN passes through
  *loss = -(on ? free_ : clipped);
  *slope = -(on ? free_ : 0.0);
  if (p.ref) {
    const double gap = (double)g.ref - logp, e = exp(gap);
    // (far out the rest is lost beside e, and infinity less itself is none)
    *loss += p.beta * (gap > 64.0 ? e : e - gap - 1.0);
    *slope += p.beta * (1.0 - e);
  }
}

// Stores past the caches where `cold`: a gradient larger than the 256 MB of
// the last cache would only push out what is still to be read (8192 x 32768
// bf16 policy: 191 us, 205 with plain stores); a smaller one is read from there next.
template <bool COLD, typename V>
__device__ __forceinline__ void put(V* p, const V& v) {
  if constexpr (COLD)
    __builtin_nontemporal_store(v, p);
  else
    *p = v;
}

// Where a row's results go.
struct Out {
  float* logp;       // or null
  double* wide;      // logp in 64 bits, or null
  float2* stats;     // maximum and sum, or null
  double* loss;      // share of the loss (policy)
  float *coef, *held;  // the row's c, the factor that its gradient holds
};

// A row's gradient from the values at hand: 16 bytes beginning at token k.
template <typename T>
__device__ __forceinline__ typename Wide<T>::type grad_of(
    const typename Wide<T>::type& x, long k, long y, float m, float scale,
    float c) {
  constexpr int V = Wide<T>::V;
  float v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = scale * exp_from((float)x[i], m);
  if (y >= k && y < k + V) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (k + i == y) v[i] += c;
  }
  typename Wide<T>::type d;
#pragma unroll
  for (int i = 0; i < V; ++i) d[i] = (T)v[i];
  return d;
}

// The gradient of a row's vectors begin + lane, + step, .. below end; the
// part that begins at 0 has the rest of the row.
template <bool COLD, typename T>
__device__ __forceinline__ void grad_span(const T* x, T* d, int K, int begin,
                                          int end, int lane, int step, long y,
                                          float m, float scale, float c) {
  typedef typename Wide<T>::type vec;
  const Cut<T> cut(K);
  for (int i = begin + lane; i < end && i < cut.whole; i += step) {
    const long k = cut.vec_at(i);
    put<COLD>(
        reinterpret_cast<vec*>(d + k),
        grad_of<T>(*reinterpret_cast<const vec*>(x + k), k, y, m, scale, c));
  }
  if (begin == 0 && lane < cut.rest) {
    const int k = cut.rest_at(lane);
    d[k] = (T)(scale * exp_from((float)x[k], m) + (k == y ? c : 0.f));
  }
}

template <bool COLD, typename T>
__device__ __forceinline__ void zero_span(T* d, int K, int begin, int end,
                                          int lane, int step) {
  typedef typename Wide<T>::type vec;
  constexpr int V = Wide<T>::V;
  const Cut<T> cut(K);
  for (int i = begin + lane; i < end && i < cut.whole; i += step) {
    vec z;
#pragma unroll
    for (int j = 0; j < V; ++j) z[j] = (T)0.f;
    put<COLD>(reinterpret_cast<vec*>(d + cut.vec_at(i)), z);
  }
  if (begin == 0 && lane < cut.rest) d[cut.rest_at(lane)] = (T)0.f;
}

// Rows of logits to logp, and with POLICY to the loss and, if `dlogits`, its
// gradient, in the same launch: a row's c needs nothing but the row and the
// sum of the weights, so logits are read once and the gradient is written
// once, where a pass of its own would read the logits again.
//
// NT threads a row.  E > 0: the row waits in registers, E 16-byte vectors a
// thread, packed as they came.  E = 0: rows too long for that are read once
// for the sums (a running maximum and sum a thread) and again for the
// gradient.  Bound by memory: the vector work stays behind it, that of the
// 64-bit sums too (8192 x 32768 bf16 policy 189 us, 4096 x 131072 bf16 logprob
// 133, 4206 x 50001 f32 preference 413; with f32 sums 189, 132, 413).
template <typename T, int NT, int E, bool POLICY, bool COLD>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void rows_kernel(
    const T* __restrict__ logits, Rows r, Policy p,
    const double* __restrict__ count, Out o, T* __restrict__ dlogits) {
  typedef typename Wide<T>::type vec;
  constexpr int V = Wide<T>::V;
  __shared__ float red_max[NT / 64];
  __shared__ double red_sum[NT / 64];
  __shared__ float row_c;
  const int tid = NT == 64 ? threadIdx.x & 63 : threadIdx.x;
  // NT = 64: four rows a workgroup, one a wave, no barriers
  const long row = NT == 64 ? (long)blockIdx.x * 4 +
                                  __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)
                            : (long)blockIdx.x;
  if (row >= r.N) return;
  const float w = weight(r, row);
  if (w == 0.f) {
    if (tid == 0) {
      if (o.logp) o.logp[row] = 0.f;
      if (o.wide) o.wide[row] = 0.0;
      if (o.stats) o.stats[row] = make_float2(0.f, 1.f);
      if (POLICY) {
        o.loss[row] = 0.0;
        if (dlogits) o.coef[row] = 0.f, o.held[row] = 1.f;
      }
    }
    if (POLICY && dlogits)
      zero_span<COLD>(dlogits + row * r.K, r.K, 0, r.K, tid, NT);
    return;
  }
  const T* x = logits + row_at(r, row);
  const long y = r.y[row];
  Given given = POLICY ? Given(p, row, r.T) : Given();
  const bool inside = y >= 0 && y < r.K;
  const float xy = inside ? (float)x[y] : NAN;
  const Cut<T> cut(r.K);
  const int whole = cut.whole, rest = cut.rest;
  float tail = tid < rest ? (float)x[cut.rest_at(tid)] : -INFINITY;
  constexpr int HELD = E > 0 ? E : 1;
  vec raw[HELD];
  float m = tail;
  double mine;  // this thread's part of the sum
  if constexpr (E > 0) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e * NT + tid < whole)
        raw[e] = *reinterpret_cast<const vec*>(x + cut.vec_at(e * NT + tid));
  }
  // Up to 1024 rows every row adds up the weights by itself, which
  // spares a launch.
  double weights = 0.0;
  if (POLICY && (NT == 64 || threadIdx.x < 64)) {
    if (count) {
      weights = *count;
    } else {
      double part[4] = {0.0, 0.0, 0.0, 0.0};
      for (int i = tid; i < r.N; i += 4 * 64)
#pragma unroll
        for (int u = 0; u < 4; ++u)  // on their way at once
          if (i + u * 64 < r.N) part[u] += (double)weight(r, i + u * 64);
      weights = lanes_sum((part[0] + part[1]) + (part[2] + part[3]));
    }
  }
  if constexpr (E > 0) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e * NT + tid < whole) {
#pragma unroll
        for (int i = 0; i < V; ++i) m = fmaxf(m, (float)raw[e][i]);
      }
    m = group_max<NT>(m, red_max);
    Sum<T> part[2];  // two chains of additions
    if (tid < rest) part[0].add(tail, m);
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e * NT + tid < whole) {
#pragma unroll
        for (int i = 0; i < V; ++i) part[i & 1].add((float)raw[e][i], m);
      }
    part[0].add(part[1]);
    mine = part[0].value();
  } else {
    // A thread's own maximum, and its sum from an earlier one, `m`: the sum
    // moves only where exponentials would pass e^8.  Neither ever holds a NaN;
    // the sum keeps one.
    float top = fmaxf(m, -INFINITY);
    m = top;
    Sum<T> part[2];
    if (tid < rest) part[0].s = tail != tail ? (double)NAN : tail > -INFINITY ? 1.0 : 0.0;
    constexpr int U = 4;
    for (int i0 = tid; i0 < whole; i0 += U * NT) {
      vec q[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * NT < whole)
          q[u] = *reinterpret_cast<const vec*>(x + cut.vec_at(i0 + u * NT));
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * NT < whole) {
#pragma unroll
          for (int i = 0; i < V; ++i) top = fmaxf(top, (float)q[u][i]);
        }
      if (top > m + 8.f) {
        // (all minus infinity so far: nothing to move)
        if (m > -INFINITY) {
          part[0].add(part[1]);
          part[0].scale(exp((double)m - (double)top));
          part[1] = Sum<T>();
        }
        m = top;
      }
      const float at = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * NT < whole) {
#pragma unroll
          for (int i = 0; i < V; ++i) part[i & 1].add((float)q[u][i], at);
        }
    }
    part[0].add(part[1]);
    const float all = group_max<NT>(top, red_max);
    mine = 0.0;
    if (m > -INFINITY) {
      Sum<T> one;
      one.add(top, m);
      const double v = part[0].value(), largest = one.value();
      mine = with_mean(v, largest);
      // the row's largest is 1 exactly, not what exp2 made of it
      const bool holds = top == all;
      if (holds) mine -= largest;
      mine *= exp((double)m - (double)all);
      if (holds) mine += 1.0;
    } else if (part[0].s != part[0].s) {
      mine = NAN;
    }
    m = all;
  }
  double total_exp = group_sum<NT>(mine, red_sum);
  if (E > 0) total_exp = with_mean(total_exp, 1.0);
  const float s = (float)total_exp;
  float c = 0.f;
  if (NT == 64 || threadIdx.x < 64) {
    const double logp = inside ? row_logp(xy, m, total_exp) : (double)NAN;
    if (tid == 0) {
      if (o.logp) o.logp[row] = (float)logp;
      if (o.wide) o.wide[row] = logp;
      if (o.stats) o.stats[row] = make_float2(m, s);
    }
    if constexpr (POLICY) {
      double loss, slope;
      policy_row(p, given, logp, &loss, &slope);
      const double share = (double)w / fmax(weights, 1.0);
      c = (float)(share * slope);
      if (tid == 0) {
        o.loss[row] = share * loss;
        if (dlogits) o.coef[row] = c, o.held[row] = 1.f;
      }
    }
  }
  if constexpr (POLICY) {
    if (!dlogits) return;
    if constexpr (NT > 64) {
      if (threadIdx.x == 0) row_c = c;
      __syncthreads();
      c = row_c;
    }
    const float scale = -c / s;
    T* d = dlogits + row * r.K;
    if constexpr (E > 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = e * NT + tid;
        if (i < whole)
          put<COLD>(reinterpret_cast<vec*>(d + cut.vec_at(i)),
                    grad_of<T>(raw[e], cut.vec_at(i), y, m, scale, c));
      }
      if (tid < rest) {
        const int k = cut.rest_at(tid);
        d[k] = (T)(scale * exp_from(tail, m) + (k == y ? c : 0.f));
      }
    } else {
      grad_span<COLD>(x, d, r.K, 0, r.K, tid, NT, y, m, scale, c);
    }
  }
}

// c of a row whose statistics are known: the product of what is given, `coef`
// a row, `seq` a sequence, its weight (if `weighted`), `up` for all.
struct Factors {
  const float *coef, *seq, *up;
  bool weighted;
};

__device__ __forceinline__ float factor(const Factors& f, const Rows& r,
                                        uint32_t row, float w) {
  float c = f.up ? *f.up : 1.f;
  if (f.coef) c *= f.coef[row];
  if (f.seq) c *= f.seq[row / (uint32_t)r.T];
  return f.weighted ? c * w : c;
}

template <bool COLD, typename T>
__device__ __forceinline__ void grad_row(const T* logits, const Rows& r,
                                         const float2* stats, const Factors& f,
                                         long row, int begin, int end,
                                         int lane, int step, T* dlogits) {
  const float w = weight(r, row);
  T* d = dlogits + row * r.K;
  if (w == 0.f) return zero_span<COLD>(d, r.K, begin, end, lane, step);
  const long y = r.y[row];
  float c = factor(f, r, row, w);
  // of a token that is none: what depends on its NaN is NaN
  if (c != 0.f && (y < 0 || y >= r.K)) c = NAN;
  const float2 q = stats[row];
  grad_span<COLD>(logits + row_at(r, row), d, r.K, begin, end, lane, step, y,
                  q.x, -c / q.y, c);
}

// Gradient of rows with known statistics: `lanes` threads and a part of the
// row each (blockIdx.y), `span` vectors a part.
template <typename T, bool COLD>
__global__ __launch_bounds__(256) void rows_grad_kernel(
    const T* __restrict__ logits, Rows r, const float2* __restrict__ stats,
    Factors f, int lanes, int span, T* __restrict__ dlogits) {
  const int sub = threadIdx.x / lanes;
  const long row = (long)blockIdx.x * (256 / lanes) + sub;
  if (row >= r.N) return;
  const int begin = blockIdx.y * span;
  grad_row<COLD>(logits, r, stats, f, row, begin, begin + span,
           (int)threadIdx.x - sub * lanes, lanes, dlogits);
}

// The same for rows of which some hold this gradient already (`held` is the
// upstream gradient that a row was made with): those are left as they are.  A
// workgroup looks at `per` rows at once.
template <typename T>
__global__ __launch_bounds__(256) void rows_again_kernel(
    const T* __restrict__ logits, Rows r, const float2* __restrict__ stats,
    Factors f, int per, float* __restrict__ held, T* __restrict__ dlogits) {
  __shared__ int other[64];
  const long first = (long)blockIdx.x * per;
  const float up = *f.up;
  int any = 0;
  if ((int)threadIdx.x < per) {
    const long row = first + threadIdx.x;
    any = row < r.N && !(held[row] == up);
    other[threadIdx.x] = any;
  }
  if (!__syncthreads_or(any)) return;
  for (int i = 0; i < per; ++i)
    if (other[i])
      grad_row<false>(logits, r, stats, f, first + i, 0, r.K, (int)threadIdx.x, 256,
               dlogits);
  if (any) held[first + threadIdx.x] = up;
}

// Sum of n values in a fixed order, in 64 bits: one workgroup of 1024.
__device__ __forceinline__ double wide_sum(double v, double* red) {
  v = lanes_sum(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < (int)blockDim.x / 64; ++i) s += red[i];
  __syncthreads();
  return s;
}

template <typename V, typename O>
__global__ __launch_bounds__(1024) void sum_kernel(const V* __restrict__ v, long n,
                           O* __restrict__ out) {
  __shared__ double red[16];
  // four loads on their way at once: the time is all latency
  double part[4] = {0.0, 0.0, 0.0, 0.0};
  for (long i = threadIdx.x; i < n; i += 4 * 1024)
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * 1024 < n) part[u] += (double)v[i + u * 1024];
  const double s = wide_sum((part[0] + part[1]) + (part[2] + part[3]), red);
  if (threadIdx.x == 0) *out = (O)s;
}

// gain_b = sum_t w (logp - ref) of every sequence, one workgroup each.
__global__ void gain_kernel(const double* __restrict__ logp,
                            const float* __restrict__ ref, Rows r,
                            double* __restrict__ gain) {
  __shared__ double red[16];
  const long at = (long)blockIdx.x * r.T;
  double s = 0.0;
  for (long t = threadIdx.x; t < r.T; t += blockDim.x) {
    const float w = weight(r, at + t);
    if (w != 0.f) s += (double)w * (logp[at + t] - (double)ref[at + t]);
  }
  s = wide_sum(s, red);
  if (threadIdx.x == 0) gain[blockIdx.x] = s;
}

// loss = mean_i (1 - eps) softplus(-margin_i) + eps softplus(margin_i), and
// every sequence's d loss / d gain, by one workgroup.
__device__ __forceinline__ void pairs_loss(const double* gain, long P,
                                           double beta, double eps,
                                           float* loss, float* margin,
                                           float* seq, double* red) {
  double s = 0.0;
  for (long i = threadIdx.x; i < P; i += blockDim.x) {
    const double m = beta * (gain[i] - gain[P + i]);
    const double e = exp(-fabs(m)), soft = log1p(e), big = 1.0 / (1.0 + e);
    // a term of coefficient 0 is none, not 0 times an infinite one: the margin
    // is infinite where a token has been ruled out
    if (eps < 1.0) s += (1.0 - eps) * (soft + fmax(-m, 0.0));
    if (eps > 0.0) s += eps * (soft + fmax(m, 0.0));
    // sigmoid(m), sigmoid(-m) from the one exponential
    const double up = m >= 0.0 ? big : e * big, down = m >= 0.0 ? e * big : big;
    const double d = beta * (eps * up - (1.0 - eps) * down) / (double)P;
    margin[i] = (float)m;
    seq[i] = (float)d;
    seq[P + i] = (float)-d;
  }
  s = wide_sum(s, red);
  if (threadIdx.x == 0) *loss = (float)(s / (double)P);
}

__global__ void pairs_kernel(const double* __restrict__ gain, long P,
                             double beta, double eps, float* __restrict__ loss,
                             float* __restrict__ margin,
                             float* __restrict__ seq) {
  __shared__ double red[16];
  pairs_loss(gain, P, beta, eps, loss, margin, seq, red);
}

// Both at once for few tokens, up to FEW_SEQS sequences: `each` of the 16 waves
// share one, four tokens of a lane on their way at once.
constexpr int FEW_SEQS = 256;

__global__ __launch_bounds__(1024) void gain_pairs_kernel(
    const double* __restrict__ logp, const float* __restrict__ ref, Rows r,
    long P, int each, double beta, double eps, float* __restrict__ loss,
    float* __restrict__ margin, float* __restrict__ seq) {
  __shared__ double red[16];
  __shared__ double gain[FEW_SEQS], shares[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int part = wave % each, step = 64 * each, T = (int)r.T;
  for (int b = wave / each; b < 2 * P; b += 16 / each) {
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    for (int t = part * 64 + lane; t < T; t += 4 * step) {
      float w[4];
      double d[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        w[u] = 0.f, d[u] = 0.0;
        if (t + u * step < T) {
          const long i = (long)b * T + t + u * step;
          w[u] = weight(r, i);
          d[u] = logp[i] - (double)ref[i];
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (w[u] != 0.f) s[u] += (double)w[u] * d[u];
    }
    const double all = lanes_sum((s[0] + s[1]) + (s[2] + s[3]));
    if (lane == 0) {
      if (each == 1)
        gain[b] = all;
      else
        shares[wave] = all;  // 2 P * each <= 16: one turn
    }
  }
  __syncthreads();
  if (each > 1) {
    if ((int)threadIdx.x < 2 * P) {
      double s = 0.0;
      for (int i = 0; i < each; ++i) s += shares[threadIdx.x * each + i];
      gain[threadIdx.x] = s;
    }
    __syncthreads();
  }
  pairs_loss(gain, P, beta, eps, loss, margin, seq, red);
}

Rows rows_of(const torch::Tensor& logits, const torch::Tensor& y,
             const c10::optional<torch::Tensor>& w, const char* what) {
  TORCH_CHECK(logits.is_cuda(), what, ": logits must be on the GPU");
  TORCH_CHECK(logits.dim() == 3 && logits.numel() > 0 &&
                  (logits.stride(2) == 1 || logits.size(2) == 1),
              what, ": logits must be [B, T, K] with a dense last axis");
  TORCH_CHECK(logits.size(2) < (1 << 28), what, ": too many tokens");
  TORCH_CHECK(logits.size(0) * logits.size(1) < (1L << 31), what,
              ": too many rows");
  TORCH_CHECK(y.scalar_type() == at::kLong && y.is_contiguous() &&
                  y.device() == logits.device() &&
                  y.numel() == logits.size(0) * logits.size(1),
              what, ": y must be contiguous int64 [B, T] on the same device");
  if (w.has_value()) {
    WAP_F32(*w, logits, "token weights");
    TORCH_CHECK(w->numel() == y.numel(), what, ": mask must be [B, T]");
  }
  Rows r;
  r.y = data<int64_t>(y);
  r.w = data_or_null<float>(w);
  r.sb = logits.stride(0);
  r.st = logits.stride(1);
  r.N = y.numel();
  r.T = logits.size(1);
  r.K = logits.size(2);
  return r;
}

// f(true) for gradients that are stored past the caches.
template <typename F>
void by_size(const torch::Tensor& logits, F&& f) {
  if (logits.numel() * logits.element_size() > (256L << 20))
    f(std::true_type());
  else
    f(std::false_type());
}

// f(threads a row, vectors a thread) as constants.  A wave for short rows;
// then as few threads as hold the row in 64 registers each, for more rows at
// once (8192 x 32768 bf16 policy: 191 us with 256 or 512 threads a row, 193
// with 1024); 0 vectors: too long to be held, or nothing to hold it for (4096 x
// 131072 bf16 logprob, 2616 rows that count: 134 us with 512, 139 with 256).
template <typename T, bool HOLD, typename F>
void by_length(int K, F&& f) {
  constexpr int V = Wide<T>::V;
  const int v = (K + V - 1) / V;
  auto at = [&](auto nt, auto e) { f(nt, e); };
  if (v <= 64) return at(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
  if (v <= 256) return at(std::integral_constant<int, 64>(), std::integral_constant<int, 4>());
  if (v <= 1024) return at(std::integral_constant<int, 256>(), std::integral_constant<int, 4>());
  if constexpr (HOLD) {
    if (v <= 2048) return at(std::integral_constant<int, 256>(), std::integral_constant<int, 8>());
    if (v <= 4096) return at(std::integral_constant<int, 256>(), std::integral_constant<int, 16>());
    if (v <= 8192) return at(std::integral_constant<int, 512>(), std::integral_constant<int, 16>());
    if (v <= 16384) return at(std::integral_constant<int, 1024>(), std::integral_constant<int, 16>());
  }
  at(std::integral_constant<int, 512>(), std::integral_constant<int, 0>());
}

template <bool POLICY>
void launch_rows(const torch::Tensor& logits, const Rows& r, const Policy& p,
                 const double* count, const Out& o, void* dlogits) {
  by_type(logits, "seqloss", [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    by_length<T, POLICY>(r.K, [&](auto nt, auto e) {
      constexpr int NT = decltype(nt)::value, E = decltype(e)::value;
      const long groups = NT == 64 ? (r.N + 3) / 4 : r.N;
      auto go = [&](auto cold) {
        hipLaunchKernelGGL(
            (rows_kernel<T, NT, E, POLICY, decltype(cold)::value>),
            dim3(groups), dim3(NT < 256 ? 256 : NT), 0, stream_of(logits),
            data<T>(logits), r, p, count, o, (T*)dlogits);
      };
      if constexpr (POLICY)
        by_size(logits, go);
      else
        go(std::false_type());
    });
  });
  launched("seqloss");
}

void launch_grad(const torch::Tensor& logits, const Rows& r,
                 const float2* stats, const Factors& f,
                 torch::Tensor& dlogits) {
  by_type(logits, "seqloss", [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const int v = r.K / Wide<T>::V + 1;  // with the rest of the row
    int lanes = 16;
    while (lanes < 256 && lanes < v) lanes *= 2;
    const int span = 256 * 8;
    const long groups = (r.N * lanes + 255) / 256;
    by_size(logits, [&](auto cold) {
      hipLaunchKernelGGL((rows_grad_kernel<T, decltype(cold)::value>),
                         dim3(groups, (v + span - 1) / span), dim3(256), 0,
                         stream_of(logits), data<T>(logits), r,
                         stats, f, lanes, span,
                         data<T>(dlogits));
    });
  });
  launched("seqloss gradient");
}

}  // namespace

// -> logp [B, T] and the rows' (maximum, sum).
std::vector<torch::Tensor> token_logprob_fwd(
    torch::Tensor logits, torch::Tensor y, c10::optional<torch::Tensor> w) {
  const Rows r = rows_of(logits, y, w, "token_logprob");
  c10::DeviceGuard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat);
  auto logp = torch::empty({logits.size(0), logits.size(1)}, f32);
  auto stats = torch::empty({r.N, 2}, f32);
  launch_rows<false>(logits, r, Policy{}, nullptr,
                     Out{data<float>(logp), nullptr, data<float2>(stats)},
                     nullptr);
  return {logp, stats};
}

// d logits from d logp (weighted = false: logp is the log-probability itself,
// where the row counts at all).
torch::Tensor token_logprob_bwd(
    torch::Tensor logits, torch::Tensor y, c10::optional<torch::Tensor> w,
    torch::Tensor stats, torch::Tensor dlogp) {
  const Rows r = rows_of(logits, y, w, "token_logprob");
  WAP_F32(dlogp, logits, "token_logprob");
  WAP_F32(stats, logits, "token_logprob");
  TORCH_CHECK(dlogp.numel() == r.N && stats.numel() == 2 * r.N);
  c10::DeviceGuard guard(logits.device());
  auto d = torch::empty(logits.sizes(), logits.options());
  launch_grad(logits, r, data<float2>(stats), Factors{data<float>(dlogp)}, d);
  return d;
}

// Which capture the current stream of `like`'s device belongs to; 0: none.
int64_t capture_of(const torch::Tensor& like) {
  hipStreamCaptureStatus status;
  unsigned long long id = 0;
  const hipError_t err = hipStreamGetCaptureInfo(stream_of(like), &status, &id);
  if (err != hipSuccess) {
    (void)hipGetLastError();  // told here, not by the next launch
    TORCH_CHECK(false, "policy_loss: ", hipGetErrorString(err));
  }
  return status == hipStreamCaptureStatusNone ? 0 : (int64_t)id + 1;
}

// -> loss, logp and, with `grad`: d logits for an upstream gradient of one, and
// of every row its statistics [N, 2], its c [N], and the upstream gradient that
// its part of d logits holds [N], in one tensor.
std::vector<torch::Tensor> policy_loss_fwd(
    torch::Tensor logits, torch::Tensor y, torch::Tensor w,
    torch::Tensor old_logp, torch::Tensor adv,
    c10::optional<torch::Tensor> ref, double lo, double hi, double beta,
    bool grad) {
  const Rows r = rows_of(logits, y, w, "policy_loss");
  WAP_F32(old_logp, logits, "policy_loss");
  TORCH_CHECK(old_logp.numel() == r.N, "policy_loss: old_logp must be [B, T]");
  TORCH_CHECK(adv.scalar_type() == at::kFloat &&
                  adv.device() == logits.device() && adv.dim() == 2 &&
                  adv.size(0) == logits.size(0) &&
                  adv.size(1) == logits.size(1),
              "policy_loss: advantage must be f32 [B, T]");
  if (ref.has_value()) {
    WAP_F32(*ref, logits, "policy_loss");
    TORCH_CHECK(ref->numel() == r.N, "policy_loss: ref_logp must be [B, T]");
  }
  c10::DeviceGuard guard(logits.device());
  const Policy p{data<float>(old_logp), data<float>(adv),
                 data_or_null<float>(ref), adv.stride(0), adv.stride(1),
                 lo, hi, beta};
  const auto f32 = logits.options().dtype(at::kFloat);
  auto loss = torch::empty({}, f32);
  auto logp = torch::empty({logits.size(0), logits.size(1)}, f32);
  auto wide = torch::empty({r.N + 1}, f32.dtype(at::kDouble));
  double* row_loss = data<double>(wide);
  double* count = row_loss + r.N;
  torch::Tensor dlogits, rows;
  Out o{data<float>(logp), nullptr, nullptr, row_loss, nullptr, nullptr};
  if (grad) {
    dlogits = torch::empty(logits.sizes(), logits.options());
    rows = torch::empty({4 * r.N}, f32);
    o.stats = data<float2>(rows);
    o.coef = data<float>(rows) + 2 * r.N;
    o.held = o.coef + r.N;
  }
  const bool few = r.N <= 1024;
  if (!few)
    hipLaunchKernelGGL((sum_kernel<float, double>), dim3(1), dim3(1024), 0,
                       stream_of(logits), r.w, r.N, count);
  launch_rows<true>(logits, r, p, few ? nullptr : count, o,
                    grad ? dlogits.data_ptr() : nullptr);
  hipLaunchKernelGGL((sum_kernel<double, float>), dim3(1), dim3(1024), 0,
                     stream_of(logits), row_loss, r.N, data<float>(loss));
  launched("policy_loss");
  if (!grad) return {loss, logp};
  return {loss, logp, dlogits, rows};
}

// Brings `dlogits` to the upstream gradient `up`: with `again` rows that hold
// it already stay as they are, without it every row is made.
void policy_loss_bwd(
    torch::Tensor logits, torch::Tensor y, torch::Tensor w, torch::Tensor rows,
    bool again, torch::Tensor up, torch::Tensor dlogits) {
  const Rows r = rows_of(logits, y, w, "policy_loss");
  WAP_F32(rows, logits, "policy_loss");
  WAP_F32(up, logits, "policy_loss");
  TORCH_CHECK(up.numel() == 1 && rows.numel() == 4 * r.N &&
              dlogits.is_contiguous() && dlogits.sizes() == logits.sizes() &&
              dlogits.scalar_type() == logits.scalar_type() &&
              dlogits.device() == logits.device());
  c10::DeviceGuard guard(logits.device());
  const float2* stats = data<float2>(rows);
  float* coef = data<float>(rows) + 2 * r.N;
  const Factors f{coef, nullptr, data<float>(up), false};
  if (!again) return launch_grad(logits, r, stats, f, dlogits);
  const int per = std::min((r.N + 2047) / 2048, 64L);
  by_type(logits, "policy_loss", [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL(rows_again_kernel<T>, dim3((r.N + per - 1) / per),
                       dim3(256), 0, stream_of(logits), data<T>(logits), r,
                       stats, f, per, coef + r.N, data<T>(dlogits));
  });
  launched("policy_loss gradient");
}

// -> loss, margins [P], and for the backward pass the rows' statistics [N, 2]
// and the sequences' d loss / d gain [2P] in one tensor.
std::vector<torch::Tensor> preference_loss_fwd(
    torch::Tensor logits, torch::Tensor y, torch::Tensor w, torch::Tensor ref,
    double beta, double eps) {
  const Rows r = rows_of(logits, y, w, "preference_loss");
  const long B = logits.size(0);
  TORCH_CHECK(B % 2 == 0, "preference_loss: sequences come in pairs");
  WAP_F32(ref, logits, "preference_loss");
  TORCH_CHECK(ref.numel() == r.N, "preference_loss: ref_logp must be [B, T]");
  c10::DeviceGuard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat);
  auto loss = torch::empty({}, f32);
  auto margin = torch::empty({B / 2}, f32);
  // 64-bit: a gain is a small difference of long sums
  auto logp = torch::empty({r.N}, f32.dtype(at::kDouble));
  auto rows = torch::empty({2 * r.N + B}, f32);
  float* seq = data<float>(rows) + 2 * r.N;
  launch_rows<false>(logits, r, Policy{}, nullptr,
                     Out{nullptr, data<double>(logp), data<float2>(rows)},
                     nullptr);
  // a second launch takes about 5 us; one workgroup reads 16384 tokens in that
  if (r.N <= 16384 && B <= FEW_SEQS) {
    int each = 1;  // a power of two: 16 waves in whole shares
    while (2 * each * B <= 16) each *= 2;
    hipLaunchKernelGGL(gain_pairs_kernel, dim3(1), dim3(1024), 0,
                       stream_of(logits), data<double>(logp), data<float>(ref),
                       r, B / 2, each, beta, eps, data<float>(loss),
                       data<float>(margin), seq);
  } else {
    auto gain = torch::empty({B}, logp.options());
    hipLaunchKernelGGL(gain_kernel, dim3(B), dim3(256), 0, stream_of(logits),
                       data<double>(logp), data<float>(ref), r,
                       data<double>(gain));
    hipLaunchKernelGGL(pairs_kernel, dim3(1), dim3(256), 0, stream_of(logits),
                       data<double>(gain), B / 2, beta, eps, data<float>(loss),
                       data<float>(margin), seq);
  }
  launched("preference_loss");
  return {loss, margin, rows};
}

torch::Tensor preference_loss_bwd(
    torch::Tensor logits, torch::Tensor y, torch::Tensor w, torch::Tensor rows,
    torch::Tensor up) {
  const Rows r = rows_of(logits, y, w, "preference_loss");
  WAP_F32(rows, logits, "preference_loss");
  WAP_F32(up, logits, "preference_loss");
  TORCH_CHECK(up.numel() == 1 && rows.numel() == 2 * r.N + logits.size(0));
  c10::DeviceGuard guard(logits.device());
  auto d = torch::empty(logits.sizes(), logits.options());
  launch_grad(logits, r, data<float2>(rows),
              Factors{nullptr, data<float>(rows) + 2 * r.N, data<float>(up),
                      true},
              d);
  return d;
}
