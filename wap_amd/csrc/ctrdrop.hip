// Dropout whose mask is a function of (seed, step, stream, place).
//
// The draws come from the counter-based generator Philox4x32 of Salmon,
// Moraes, Dror and Shaw ("Parallel random numbers: as easy as 1, 2, 3",
// SC 2011) with seven rounds, the fewest that pass their whole battery of
// tests: key = seed, counter = (group, stream and group's high bits, step).
// One call gives 128 bits = eight draws of 16 bits, for the eight elements of
// a group; an element is kept where its draw is >= round(p 2^16), and scaled
// by the inverse of the exact share that is kept, so the mean is not moved by
// the rounding of p.  The backward pass makes the same draws again: the mask
// is never stored.
#include <hip/hip_runtime.h>

#include "opcommon.h"

namespace {

using namespace wap;

struct Draws {
  uint32_t w[4];
};

__device__ __forceinline__ Draws draws(
    uint64_t group, uint32_t stream, uint64_t seed, uint64_t step) {
  uint32_t c0 = (uint32_t)group;
  uint32_t c1 = (stream << 8) | (uint32_t)(group >> 32);
  uint32_t c2 = (uint32_t)step, c3 = (uint32_t)(step >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t p = (uint64_t)c0 * 0xD2511F53u;
    const uint64_t q = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(q >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)q;
    c2 = (uint32_t)(p >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// One thread per group of eight elements, 16 or 2 x 16 bytes a load.  Bound by
// memory: a draw of eight is 7 rounds of two 32x32->64-bit products and four
// xors, about 12 slots an element, half of what reading and writing 16-bit
// values takes.  16384 x 4096 fp16 on an MI355X, a call among others: 40 us (6.7
// TB/s), with a residual 69 us (5.8 TB/s), where a copy reaches 5.1; two or four
// groups a thread are slower (43, 47 us): the chip is full of waves as it is.
constexpr int THREADS = 256;

template <typename T, bool RES>
__global__ __launch_bounds__(THREADS) void ctr_dropout_kernel(
    const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y,
    long n, const int64_t* __restrict__ rng, uint64_t seed, uint64_t step,
    uint32_t stream, uint32_t limit, float scale, int64_t* __restrict__ used) {
  // any place in memory: views begin at any element
  typedef typename VecOf<T, 8, sizeof(T)>::type vec;
  const long grp = (long)blockIdx.x * THREADS + threadIdx.x;
  if (rng) {
    seed = (uint64_t)rng[0];
    step = (uint64_t)rng[1];
  }
  if (used && grp == 0) {
    used[0] = (int64_t)seed;
    used[1] = (int64_t)step;
  }
  if (grp * 8 >= n) return;
  const bool whole = grp * 8 + 8 <= n;
  vec a, b;
  if (whole) {
    a = *reinterpret_cast<const vec*>(x + grp * 8);
    if constexpr (RES) b = *reinterpret_cast<const vec*>(res + grp * 8);
  }
  const Draws u = draws((uint64_t)grp, stream, seed, step);
  if (whole) {
    vec o;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t v = (j & 1) ? u.w[j >> 1] >> 16 : u.w[j >> 1] & 0xffffu;
      float f = v >= limit ? (float)a[j] * scale : 0.f;
      if constexpr (RES) f += (float)b[j];
      o[j] = (T)f;
    }
    *reinterpret_cast<vec*>(y + grp * 8) = o;
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j) {
      const long i = grp * 8 + j;
      if (i < n) {
        const uint32_t v = (j & 1) ? u.w[j >> 1] >> 16 : u.w[j >> 1] & 0xffffu;
        float f = v >= limit ? (float)x[i] * scale : 0.f;
        if constexpr (RES) f += (float)res[i];
        y[i] = (T)f;
      }
    }
  }
}

}  // namespace

// x (and residual) contiguous; rng: [seed, step] on the
// device, or the two numbers.  Returns y and, where rng is a tensor, the seed
// and step that were used: the backward pass draws from that copy, whatever
// the caller has done to rng since.
std::vector<torch::Tensor> counter_dropout_run(
    torch::Tensor x, c10::optional<torch::Tensor> residual, double p,
    c10::optional<torch::Tensor> rng, int64_t seed, int64_t step,
    int64_t stream, bool keep_used) {
  TORCH_CHECK(x.is_cuda(), "counter_dropout: x must be on the GPU");
  TORCH_CHECK(x.is_contiguous(), "counter_dropout: x must be contiguous");
  TORCH_CHECK(p >= 0.0 && p <= 1.0, "counter_dropout: p in [0, 1]");
  TORCH_CHECK(stream >= 0 && stream < (1 << 24),
              "counter_dropout: stream in [0, 2^24)");
  if (residual.has_value())
    TORCH_CHECK(residual->sizes() == x.sizes() &&
                    residual->is_contiguous() &&
                    residual->scalar_type() == x.scalar_type() &&
                    residual->device() == x.device(),
                "counter_dropout: residual must match x");
  if (rng.has_value())
    TORCH_CHECK(rng->scalar_type() == at::kLong && rng->numel() == 2 &&
                    rng->is_contiguous() && rng->device() == x.device(),
                "counter_dropout: rng must be int64 [2] on x's device");
  const long n = x.numel();
  TORCH_CHECK(n < (1L << 42), "counter_dropout: too many elements");
  c10::DeviceGuard guard(x.device());
  auto y = torch::empty_like(x);
  torch::Tensor used;
  if (keep_used && rng.has_value()) used = torch::empty_like(*rng);
  const uint32_t limit = (uint32_t)std::floor(p * 65536.0 + 0.5);
  const float scale =
      limit == 65536u ? 0.f : (float)(65536.0 / (65536.0 - limit));
  if (n > 0) {
    const long groups = (n + 7) / 8;
    by_type(x, "counter_dropout", [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      auto go = [&](auto with) {
        hipLaunchKernelGGL(
            (ctr_dropout_kernel<T, decltype(with)::value>),
            dim3((groups + THREADS - 1) / THREADS), dim3(THREADS), 0,
            stream_of(x), data<T>(x), data_or_null<T>(residual), data<T>(y), n,
            data_or_null<int64_t>(rng), (uint64_t)seed, (uint64_t)step,
            (uint32_t)stream, limit, scale,
            used.defined() ? data<int64_t>(used) : nullptr);
      };
      if (residual.has_value())
        go(std::true_type());
      else
        go(std::false_type());
    });
    launched("counter_dropout");
  }
  if (used.defined()) return {y, used};
  return {y};
}
