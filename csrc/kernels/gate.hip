// The element-wise half of a gated feed-forward block for products that were computed in float32: h = act(g) * u and its
// gradients from g | u [M, 2 H].  (bf16 and fp16 do this in the epilogues of the two matrix products, gemm_bf16.hip; the float32 product
// kernel has no such epilogue, and with 16 times less matrix rate the extra pass is a few percent of it.)
// No counterpart in the reference, whose model has no activation (reference min_DDP.py:41-49).
#include <type_traits>

#include "device_utils.h"
#include "kernels.h"

namespace dpa {
namespace kernels {

namespace {

// One thread per element; rows of H are short against the grid and every access of a wave is contiguous.
template <typename TR, int ACT>
__global__ __launch_bounds__(256) void gate_fwd_kernel(const typename TR::T* __restrict__ gu, typename TR::T* __restrict__ h, long long n, long long H) {
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * 256) {
    const long long row = i / H, at = row * 2 * H + (i - row * H);
    h[i] = TR::from_f32(gate_value<ACT>(TR::to_f32(gu[at])) * TR::to_f32(gu[at + H]));
  }
}

template <typename TR, int ACT>
__global__ __launch_bounds__(256) void gate_bwd_kernel(const typename TR::T* __restrict__ dh, const typename TR::T* __restrict__ gu,
                                                       typename TR::T* __restrict__ dgu, long long n, long long H) {
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * 256) {
    const long long row = i / H, at = row * 2 * H + (i - row * H);
    float value, slope;
    gate_value_and_slope<ACT>(TR::to_f32(gu[at]), value, slope);
    const float d = TR::to_f32(dh[i]);
    dgu[at] = TR::from_f32(d * TR::to_f32(gu[at + H]) * slope);
    dgu[at + H] = TR::from_f32(d * value);
  }
}

template <typename F>
void with_act(int act, F&& f) {
  if (act == kActSilu) f(std::integral_constant<int, kActSilu>{});
  else if (act == kActGelu) f(std::integral_constant<int, kActGelu>{});
  else f(std::integral_constant<int, kActRelu>{});
}

unsigned blocks_for(long long n) {
  const long long b = (n + 255) / 256;
  return static_cast<unsigned>(b < 16384 ? b : 16384);
}

}  // namespace

void launch_gate_fwd(const void* gu, void* h, long long M, long long H, int dtype, int act, hipStream_t stream) {
  if (M * H <= 0) return;
  with_act(act, [&](auto act_c) {
    dispatch_dtype(dtype, [&](auto tr) {
      using TR = decltype(tr);
      using T = typename TR::T;
      hipLaunchKernelGGL((gate_fwd_kernel<TR, decltype(act_c)::value>), dim3(blocks_for(M * H)), dim3(256), 0, stream, static_cast<const T*>(gu),
                         static_cast<T*>(h), M * H, H);
    });
  });
}

void launch_gate_bwd(const void* dh, const void* gu, void* dgu, long long M, long long H, int dtype, int act, hipStream_t stream) {
  if (M * H <= 0) return;
  with_act(act, [&](auto act_c) {
    dispatch_dtype(dtype, [&](auto tr) {
      using TR = decltype(tr);
      using T = typename TR::T;
      hipLaunchKernelGGL((gate_bwd_kernel<TR, decltype(act_c)::value>), dim3(blocks_for(M * H)), dim3(256), 0, stream, static_cast<const T*>(dh),
                         static_cast<const T*>(gu), static_cast<T*>(dgu), M * H, H);
    });
  });
}

}  // namespace kernels
}  // namespace dpa
