// Gated linear recurrence over a sequence, forward, backward and one step.
//
//   z_t = sigmoid(gz_t), n_t = tanh(gn_t)          gates packed [z|n]
//   h_t = (1 - z_t) n_t + z_t h_{t-1}              masked step: h_t = h_{t-1}
//
// The blend is the GRU's; its gates do not see the state, so h is linear in
// the state before and the time axis can be cut.  The state, the gates and
// all sums are f32; h is rounded once, where it is stored.
#include <hip/hip_runtime.h>

#include "opcommon.h"

namespace {

using namespace wap;

struct Gates {
  float z, zc, n;  // z, 1 - z (from its own exponential: no cancellation), n
};

__device__ __forceinline__ Gates gates(float gz, float gn) {
  const float e = expf(-fabsf(gz));
  const float big = 1.f / (1.f + e), small = e * big;
  Gates r;
  r.z = gz >= 0.f ? big : small;
  r.zc = gz >= 0.f ? small : big;
  if (gz != gz) r.z = r.zc = gz;
  r.n = tanhf(gn);
  return r;
}

// One thread per (sequence, channel), serial over time.
template <typename T>
__global__ void gscan_fwd_kernel(
    const T* __restrict__ g, long gsb, long gst, const float* __restrict__ h0,
    const float* __restrict__ mask, T* __restrict__ out,
    float* __restrict__ last, int B, long L, int D) {
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (long)B * D) return;
  const long b = i / D, d = i % D;
  float h = h0 ? h0[i] : 0.f;
  for (long t = 0; t < L; ++t) {
    if (!mask || mask[b * L + t] > 0.f) {
      const T* p = g + b * gsb + t * gst + d;
      const Gates q = gates((float)p[0], (float)p[D]);
      h = fmaf(q.z, h, q.zc * q.n);
    }
    out[(b * L + t) * D + d] = (T)h;
  }
  last[i] = h;
}

// delta_t = dh_t + z_{t+1} delta_{t+1}; the states come from a second forward
// walk whose results wait in `hs` (f32).
template <typename T>
__global__ void gscan_bwd_kernel(
    const T* __restrict__ g, long gsb, long gst, const float* __restrict__ h0,
    const float* __restrict__ mask, const T* __restrict__ dh, long dsb,
    long dst, const float* __restrict__ dlast, float* __restrict__ hs,
    T* __restrict__ dg, float* __restrict__ dh0, int B, long L, int D) {
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (long)B * D) return;
  const long b = i / D, d = i % D;
  float h = h0 ? h0[i] : 0.f;
  for (long t = 0; t < L; ++t) {
    hs[(b * L + t) * D + d] = h;
    if (!mask || mask[b * L + t] > 0.f) {
      const T* p = g + b * gsb + t * gst + d;
      const Gates q = gates((float)p[0], (float)p[D]);
      h = fmaf(q.z, h, q.zc * q.n);
    }
  }
  float c = dlast ? dlast[i] : 0.f;
  for (long t = L - 1; t >= 0; --t) {
    if (dh) c += (float)dh[b * dsb + t * dst + d];
    T* o = dg + (b * L + t) * 2 * D + d;
    if (mask && !(mask[b * L + t] > 0.f)) {
      o[0] = (T)0.f;
      o[D] = (T)0.f;
      continue;
    }
    const T* p = g + b * gsb + t * gst + d;
    const Gates q = gates((float)p[0], (float)p[D]);
    o[0] = (T)(c * (hs[(b * L + t) * D + d] - q.n) * (q.z * q.zc));
    o[D] = (T)(c * q.zc * (1.f - q.n * q.n));
    c *= q.z;
  }
  if (dh0) dh0[i] = c;
}

template <typename T>
__global__ void gstep_kernel(
    const T* __restrict__ g, long gsb, const float* __restrict__ h,
    T* __restrict__ out, float* __restrict__ h_new, long total, int D) {
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= total) return;
  const long b = i / D, d = i % D;
  const T* p = g + b * gsb + d;
  const Gates q = gates((float)p[0], (float)p[D]);
  const float v = fmaf(q.z, h[i], q.zc * q.n);
  h_new[i] = v;
  out[i] = (T)v;
}

void check_gates(const torch::Tensor& g, int dim) {
  TORCH_CHECK(g.is_cuda(), "gated_scan: g must be on the GPU");
  TORCH_CHECK(g.dim() == dim && g.size(-1) % 2 == 0 && g.stride(-1) == 1,
              "gated_scan: g must end in a dense axis of 2 D");
  TORCH_CHECK(g.size(-1) / 2 < (1 << 30) && g.numel() > 0,
              "gated_scan: empty or too wide");
}

void check_state(const c10::optional<torch::Tensor>& h,
                 const torch::Tensor& g) {
  if (!h.has_value()) return;
  WAP_F32(*h, g, "gated_scan");
  TORCH_CHECK(h->dim() == 2 && h->size(0) == g.size(0) &&
                  h->size(1) == g.size(-1) / 2,
              "gated_scan: a state must be [B, D]");
}

void check_mask(const c10::optional<torch::Tensor>& mask,
                const torch::Tensor& g) {
  if (!mask.has_value()) return;
  WAP_F32(*mask, g, "gated_scan");
  TORCH_CHECK(mask->dim() == 2 && mask->size(0) == g.size(0) &&
                  mask->size(1) == g.size(1),
              "gated_scan: mask must be [B, T]");
}

}  // namespace

std::vector<torch::Tensor> gated_scan_fwd(
    torch::Tensor g, c10::optional<torch::Tensor> h0,
    c10::optional<torch::Tensor> mask) {
  check_gates(g, 3);
  check_state(h0, g);
  check_mask(mask, g);
  c10::DeviceGuard guard(g.device());
  const int B = g.size(0), D = g.size(2) / 2;
  const long L = g.size(1);
  auto out = torch::empty({B, L, D}, g.options());
  auto last = torch::empty({B, D}, g.options().dtype(at::kFloat));
  const long blocks = ((long)B * D + 63) / 64;
  by_type(g, "gated_scan", [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL(gscan_fwd_kernel<T>, dim3(blocks), dim3(64), 0,
                       stream_of(g), data<T>(g), g.stride(0), g.stride(1),
                       data_or_null<float>(h0), data_or_null<float>(mask),
                       data<T>(out), data<float>(last), B, L, D);
  });
  launched("gated_scan");
  return {out, last};
}

std::vector<torch::Tensor> gated_scan_bwd(
    torch::Tensor g, c10::optional<torch::Tensor> h0,
    c10::optional<torch::Tensor> mask, c10::optional<torch::Tensor> dh,
    c10::optional<torch::Tensor> dlast) {
  check_gates(g, 3);
  check_state(h0, g);
  check_state(dlast, g);
  check_mask(mask, g);
  const int B = g.size(0), D = g.size(2) / 2;
  const long L = g.size(1);
  if (dh.has_value())
    TORCH_CHECK(dh->scalar_type() == g.scalar_type() &&
                    dh->device() == g.device() && dh->dim() == 3 &&
                    dh->size(0) == B && dh->size(1) == L &&
                    dh->size(2) == D && dh->stride(2) == 1,
                "gated_scan: dh must be [B, T, D] in g's type");
  c10::DeviceGuard guard(g.device());
  auto dg = torch::empty({B, L, 2 * (long)D}, g.options());
  auto dh0 = torch::empty({B, D}, g.options().dtype(at::kFloat));
  auto hs = torch::empty({B, L, D}, g.options().dtype(at::kFloat));
  const long blocks = ((long)B * D + 63) / 64;
  by_type(g, "gated_scan", [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL(gscan_bwd_kernel<T>, dim3(blocks), dim3(64), 0,
                       stream_of(g), data<T>(g), g.stride(0), g.stride(1),
                       data_or_null<float>(h0), data_or_null<float>(mask),
                       data_or_null<T>(dh), dh.has_value() ? dh->stride(0) : 0,
                       dh.has_value() ? dh->stride(1) : 0,
                       data_or_null<float>(dlast), data<float>(hs),
                       data<T>(dg), data<float>(dh0), B, L, D);
  });
  launched("gated_scan backward");
  return {dg, dh0};
}

std::vector<torch::Tensor> gated_step(torch::Tensor g, torch::Tensor h) {
  check_gates(g, 2);
  check_state(h, g);
  c10::DeviceGuard guard(g.device());
  const long total = h.numel();
  const int D = h.size(1);
  auto out = torch::empty_like(h, g.options());
  auto h_new = torch::empty_like(h);
  by_type(g, "gated_step", [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL(gstep_kernel<T>, dim3((total + 255) / 256), dim3(256),
                       0, stream_of(g), data<T>(g), g.stride(0),
                       data<float>(h), data<T>(out), data<float>(h_new), total,
                       D);
  });
  launched("gated_step");
  return {out, h_new};
}
