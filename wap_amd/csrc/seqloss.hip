// The probability of given tokens under rows of logits, and the losses and
// gradients made of it.
//
//   logp = x_y - m - log S,   m = max_k x_k,  S = sum_k exp(x_k - m)
//   d loss / d x_k = c (1[k = y] - exp(x_k - m) / S),  c = d loss / d logp
//
// A row of weight 0 is not read: its logp is 0 and its gradient row is zeros.
// A token outside [0, K) in a row that counts makes its logp NaN.
// What follows the sums of a row (log, ratio, comparison with the clip's
// borders, sums over tokens) is in 64 bits: it is one thread's work a row, and
// an error of 1e-7 there could move a token across a border.
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

__device__ __forceinline__ long row_at(const Rows& r, long row) {
  return row / r.T * r.sb + row % r.T * r.st;
}

// Sum / max over the workgroup, on every thread. `red`: one value a wave.
template <int NT>
__device__ __forceinline__ float group_sum(float v, float* red) {
  v = lanes_sum(v);
  if constexpr (NT == 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) s += red[i];
  return s;
}

template <int NT>
__device__ __forceinline__ float group_max(float v, float* red) {
  v = lanes_max(v);
  if constexpr (NT == 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = red[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) s = fmaxf(s, red[i]);
  return s;
}

// logp of a row from its token's logit, maximum and sum.
__device__ __forceinline__ double row_logp(float xy, float m, float sum) {
  return (double)xy - (double)m - log((double)sum);
}

// Loss of one token and its derivative by logp, both without the 1 / sum of
// weights.  At a border of the clip the unclipped side counts.
__device__ __forceinline__ void policy_row(
    const Policy& p, long row, long T, double logp, double* loss,
    double* slope) {
  const double adv = p.adv[row / T * p.ab + row % T * p.at];
  const double ratio = exp(logp - (double)p.old_logp[row]);
  const double kept = fmin(fmax(ratio, 1.0 - p.lo), 1.0 + p.hi);
  const double free_ = adv == 0.0 ? 0.0 : ratio * adv, clipped = kept * adv;
  const bool on = !(free_ > clipped);  // NaN passes through
  *loss = -(on ? free_ : clipped);
  *slope = -(on ? free_ : 0.0);
  if (p.ref) {
    const double gap = (double)p.ref[row] - logp, e = exp(gap);
    *loss += p.beta * (e - gap - 1.0);
    *slope += p.beta * (1.0 - e);
  }
}

// One workgroup per row, three passes over it.  POLICY: loss and gradient in
// the same launch.
template <typename T, int NT, bool POLICY>
__global__ void rows_kernel(
    const T* __restrict__ logits, Rows r, Policy p,
    const double* __restrict__ count, float* __restrict__ logp_out,
    double* __restrict__ wide_out, float2* __restrict__ stats, double* __restrict__ row_loss,
    float* __restrict__ coef, float* __restrict__ held,
    T* __restrict__ dlogits) {
  __shared__ float red[NT / 64];
  const long row = blockIdx.x;
  const float w = weight(r, row);
  if (w == 0.f) {
    if (threadIdx.x == 0) {
      if (logp_out) logp_out[row] = 0.f;
      if (wide_out) wide_out[row] = 0.0;
      if (stats) stats[row] = make_float2(0.f, 1.f);
      if (POLICY) {
        row_loss[row] = 0.0;
        if (dlogits) coef[row] = 0.f, held[row] = 1.f;
      }
    }
    if (POLICY && dlogits)
      for (int k = threadIdx.x; k < r.K; k += NT)
        dlogits[row * r.K + k] = (T)0.f;
    return;
  }
  const T* x = logits + row_at(r, row);
  float m = -INFINITY, s = 0.f;
  for (int k = threadIdx.x; k < r.K; k += NT) m = fmaxf(m, (float)x[k]);
  m = group_max<NT>(m, red);
  for (int k = threadIdx.x; k < r.K; k += NT) s += expf((float)x[k] - m);
  s = group_sum<NT>(s, red);
  const long y = r.y[row];
  const bool inside = y >= 0 && y < r.K;
  const double logp = inside ? row_logp((float)x[y], m, s) : (double)NAN;
  if (threadIdx.x == 0) {
    if (logp_out) logp_out[row] = (float)logp;
    if (wide_out) wide_out[row] = logp;
    if (stats) stats[row] = make_float2(m, s);
  }
  if constexpr (POLICY) {
    double loss, slope;
    policy_row(p, row, r.T, logp, &loss, &slope);
    const double share = (double)w / fmax(*count, 1.0);
    if (threadIdx.x == 0) row_loss[row] = share * loss;
    if (dlogits) {
      const float c = (float)(share * slope);
      if (threadIdx.x == 0) coef[row] = c, held[row] = 1.f;
      const float scale = c / s;
      for (int k = threadIdx.x; k < r.K; k += NT) {
        float v = -scale * expf((float)x[k] - m);
        if (k == y) v += c;
        dlogits[row * r.K + k] = (T)v;
      }
    }
  }
}

// Gradient of rows whose statistics are known.  The row's c is the product of
// what is given: `coef` a row, `seq` a sequence, its weight (if `weighted`),
// `up` for all.  held: the factor that the row already holds; such a row is
// left as it is.
template <typename T>
__global__ void rows_grad_kernel(
    const T* __restrict__ logits, Rows r, const float2* __restrict__ stats,
    const float* __restrict__ coef, const float* __restrict__ seq,
    bool weighted, const float* __restrict__ up, float* __restrict__ held,
    T* __restrict__ dlogits) {
  for (long row = blockIdx.x; row < r.N; row += gridDim.x) {
    const float w = weight(r, row);
    const float u = up ? *up : 1.f;
    if (held && held[row] == u) continue;
    float c = u;
    if (coef) c *= coef[row];
    if (seq) c *= seq[row / r.T];
    if (weighted) c *= w;
    T* d = dlogits + row * r.K;
    if (w == 0.f) {
      for (int k = threadIdx.x; k < r.K; k += blockDim.x) d[k] = (T)0.f;
    } else {
      const T* x = logits + row_at(r, row);
      const long y = r.y[row];
      const float2 q = stats[row];
      const float scale = c / q.y;
      for (int k = threadIdx.x; k < r.K; k += blockDim.x) {
        float v = -scale * expf((float)x[k] - q.x);
        if (k == y) v += c;
        d[k] = (T)v;
      }
    }
    __syncthreads();
    if (held && threadIdx.x == 0) held[row] = u;
  }
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
__global__ void sum_kernel(const V* __restrict__ v, long n,
                           O* __restrict__ out) {
  __shared__ double red[16];
  double s = 0.0;
  for (long i = threadIdx.x; i < n; i += blockDim.x) s += (double)v[i];
  s = wide_sum(s, red);
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
// every sequence's d loss / d gain.
__global__ void pairs_kernel(const double* __restrict__ gain, long P,
                             double beta, double eps, float* __restrict__ loss,
                             float* __restrict__ margin,
                             float* __restrict__ seq) {
  __shared__ double red[16];
  double s = 0.0;
  for (long i = threadIdx.x; i < P; i += blockDim.x) {
    const double m = beta * (gain[i] - gain[P + i]);
    const double soft = log1p(exp(-fabs(m)));
    s += (1.0 - eps) * (soft + fmax(-m, 0.0)) + eps * (soft + fmax(m, 0.0));
    const double up = 1.0 / (1.0 + exp(-m)), down = 1.0 / (1.0 + exp(m));
    const double d = beta * (eps * up - (1.0 - eps) * down) / (double)P;
    margin[i] = (float)m;
    seq[i] = (float)d;
    seq[P + i] = (float)-d;
  }
  s = wide_sum(s, red);
  if (threadIdx.x == 0) *loss = (float)(s / (double)P);
}

Rows rows_of(const torch::Tensor& logits, const torch::Tensor& y,
             const c10::optional<torch::Tensor>& w, const char* what) {
  TORCH_CHECK(logits.is_cuda(), what, ": logits must be on the GPU");
  TORCH_CHECK(logits.dim() == 3 && logits.numel() > 0 &&
                  (logits.stride(2) == 1 || logits.size(2) == 1),
              what, ": logits must be [B, T, K] with a dense last axis");
  TORCH_CHECK(logits.size(2) < (1 << 30), what, ": too many tokens");
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

template <bool POLICY>
void launch_rows(const torch::Tensor& logits, const Rows& r, const Policy& p,
                 const double* count, float* logp, double* wide,
                 float2* stats, double* row_loss, float* coef, float* held, void* dlogits) {
  by_type(logits, "seqloss", [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL((rows_kernel<T, 256, POLICY>), dim3(r.N), dim3(256), 0,
                       stream_of(logits), data<T>(logits), r, p, count, logp,
                       wide, stats, row_loss, coef, held, (T*)dlogits);
  });
  launched("seqloss");
}

void launch_grad(const torch::Tensor& logits, const Rows& r,
                 const torch::Tensor& stats, const float* coef,
                 const float* seq, bool weighted, const float* up, float* held,
                 torch::Tensor& dlogits) {
  by_type(logits, "seqloss", [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL(rows_grad_kernel<T>, dim3(std::min(r.N, 4096L)),
                       dim3(256), 0, stream_of(logits), data<T>(logits), r,
                       data<float2>(stats), coef, seq, weighted, up, held,
                       data<T>(dlogits));
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
  launch_rows<false>(logits, r, Policy{}, nullptr, data<float>(logp), nullptr,
                     data<float2>(stats), nullptr, nullptr, nullptr, nullptr);
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
  launch_grad(logits, r, stats, data<float>(dlogp), nullptr, false, nullptr,
              nullptr, d);
  return d;
}

// -> loss, logp and, with `grad`: d logits for an upstream gradient of one,
// stats, the rows' c, and the factor that each row of d logits holds.
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
  torch::Tensor dlogits, stats, coef, held;
  if (grad) {
    dlogits = torch::empty(logits.sizes(), logits.options());
    stats = torch::empty({r.N, 2}, f32);
    coef = torch::empty({r.N}, f32);
    held = torch::empty({r.N}, f32);
  }
  hipLaunchKernelGGL((sum_kernel<float, double>), dim3(1), dim3(1024), 0,
                     stream_of(logits), r.w, r.N, count);
  launch_rows<true>(logits, r, p, count, data<float>(logp), nullptr,
                    grad ? data<float2>(stats) : nullptr, row_loss,
                    grad ? data<float>(coef) : nullptr,
                    grad ? data<float>(held) : nullptr,
                    grad ? dlogits.data_ptr() : nullptr);
  hipLaunchKernelGGL((sum_kernel<double, float>), dim3(1), dim3(1024), 0,
                     stream_of(logits), row_loss, r.N, data<float>(loss));
  launched("policy_loss");
  if (!grad) return {loss, logp};
  return {loss, logp, dlogits, stats, coef, held};
}

// Brings `dlogits` to the upstream gradient `up`: rows that hold it already
// (`held`) stay.  Without `held` every row is made.
void policy_loss_bwd(
    torch::Tensor logits, torch::Tensor y, torch::Tensor w,
    torch::Tensor stats, torch::Tensor coef, c10::optional<torch::Tensor> held,
    torch::Tensor up, torch::Tensor dlogits) {
  const Rows r = rows_of(logits, y, w, "policy_loss");
  WAP_F32(stats, logits, "policy_loss");
  WAP_F32(coef, logits, "policy_loss");
  WAP_F32(up, logits, "policy_loss");
  TORCH_CHECK(up.numel() == 1 && stats.numel() == 2 * r.N &&
              coef.numel() == r.N && dlogits.is_contiguous() &&
              dlogits.sizes() == logits.sizes() &&
              dlogits.scalar_type() == logits.scalar_type() &&
              dlogits.device() == logits.device());
  if (held.has_value()) {
    WAP_F32(*held, logits, "policy_loss");
    TORCH_CHECK(held->numel() == r.N);
  }
  c10::DeviceGuard guard(logits.device());
  launch_grad(logits, r, stats, data<float>(coef), nullptr, false,
              data<float>(up), data_or_null<float>(held), dlogits);
}

// -> loss, margins [P], and for the backward pass: stats, d loss / d gain [2P].
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
  auto stats = torch::empty({r.N, 2}, f32);
  auto gain = torch::empty({B}, f32.dtype(at::kDouble));
  auto seq = torch::empty({B}, f32);
  launch_rows<false>(logits, r, Policy{}, nullptr, nullptr, data<double>(logp),
                     data<float2>(stats), nullptr, nullptr, nullptr, nullptr);
  hipLaunchKernelGGL(gain_kernel, dim3(B), dim3(256), 0, stream_of(logits),
                     data<double>(logp), data<float>(ref), r,
                     data<double>(gain));
  hipLaunchKernelGGL(pairs_kernel, dim3(1), dim3(256), 0, stream_of(logits),
                     data<double>(gain), B / 2, beta, eps, data<float>(loss),
                     data<float>(margin), data<float>(seq));
  launched("preference_loss");
  return {loss, margin, stats, seq};
}

torch::Tensor preference_loss_bwd(
    torch::Tensor logits, torch::Tensor y, torch::Tensor w,
    torch::Tensor stats, torch::Tensor seq, torch::Tensor up) {
  const Rows r = rows_of(logits, y, w, "preference_loss");
  WAP_F32(stats, logits, "preference_loss");
  WAP_F32(seq, logits, "preference_loss");
  WAP_F32(up, logits, "preference_loss");
  TORCH_CHECK(up.numel() == 1 && stats.numel() == 2 * r.N &&
              seq.numel() == logits.size(0));
  c10::DeviceGuard guard(logits.device());
  auto d = torch::empty(logits.sizes(), logits.options());
  launch_grad(logits, r, stats, nullptr, data<float>(seq), true,
              data<float>(up), nullptr, d);
  return d;
}
