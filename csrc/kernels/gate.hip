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
template <int ACT>
__global__ __launch_bounds__(256) void gate_fwd_kernel(const float* __restrict__ gu, float* __restrict__ h, long long n, long long H) {
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * 256) {
    const long long row = i / H, at = row * 2 * H + (i - row * H);
    h[i] = gate_value<ACT>(gu[at]) * gu[at + H];
  }
}

template <int ACT>
__global__ __launch_bounds__(256) void gate_bwd_kernel(const float* __restrict__ dh, const float* __restrict__ gu, float* __restrict__ dgu, long long n,
                                                       long long H) {
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * 256) {
    const long long row = i / H, at = row * 2 * H + (i - row * H);
    float value, slope;
    gate_value_and_slope<ACT>(gu[at], value, slope);
    const float d = dh[i];
    dgu[at] = d * gu[at + H] * slope;
    dgu[at + H] = d * value;
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

void launch_gate_fwd(const float* gu, float* h, long long M, long long H, int act, hipStream_t stream) {
  if (M * H <= 0) return;
  with_act(act, [&](auto act_c) { hipLaunchKernelGGL((gate_fwd_kernel<decltype(act_c)::value>), dim3(blocks_for(M * H)), dim3(256), 0, stream, gu, h, M * H, H); });
}

void launch_gate_bwd(const float* dh, const float* gu, float* dgu, long long M, long long H, int act, hipStream_t stream) {
  if (M * H <= 0) return;
  with_act(act, [&](auto act_c) { hipLaunchKernelGGL((gate_bwd_kernel<decltype(act_c)::value>), dim3(blocks_for(M * H)), dim3(256), 0, stream, dh, gu, dgu, M * H, H); });
}

}  // namespace kernels
}  // namespace dpa
