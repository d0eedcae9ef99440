// Shared by the operator files that take f32, bf16 and fp16: element types,
// conversions, wave reductions, host-side dispatch and checks.
#pragma once

#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <vector>

namespace wap {

// N elements of T as the compiler's own vector, aligned to `A` bytes: rows of
// an odd width start at any element, and the hardware takes wide loads there.
template <typename T, int N, int A>
struct VecOf {
  typedef T type __attribute__((ext_vector_type(N), aligned(A)));
};

// Sum / maximum over the 64 lanes, the result on every lane.
template <typename F>
__device__ __forceinline__ F lanes_sum(F v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// fmaxf drops NaN; a NaN that is lost here comes back in the sum of the
// exponentials, which sees every element again.
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  return v;
}

// ------------------------------------------------------------------ host

inline hipStream_t stream_of(const torch::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

inline void launched(const char* what) {
  const hipError_t err = hipGetLastError();
  TORCH_CHECK(err == hipSuccess, what, ": HIP kernel launch failed: ",
              hipGetErrorString(err));
}

template <typename T>
T* data_or_null(const c10::optional<torch::Tensor>& t) {
  return t.has_value() ? reinterpret_cast<T*>(t->data_ptr()) : nullptr;
}

template <typename T>
T* data(const torch::Tensor& t) {
  return reinterpret_cast<T*>(t.data_ptr());
}

#define WAP_F32(t, like, what)                                          \
  TORCH_CHECK((t).scalar_type() == at::kFloat && (t).is_contiguous() && \
                  (t).device() == (like).device(),                      \
              what ": " #t " must be contiguous f32 on the same device")

// Calls f with a null pointer of the element type.
template <typename F>
void by_type(const torch::Tensor& t, const char* what, F&& f) {
  switch (t.scalar_type()) {
    case at::kFloat: f((float*)nullptr); break;
    case at::kBFloat16: f((__bf16*)nullptr); break;
    case at::kHalf: f((_Float16*)nullptr); break;
    default:
      TORCH_CHECK(false, what, ": f32, bf16 or fp16, not ", t.scalar_type());
  }
}

}  // namespace wap
