// y = x W^T + b for a few rows of x (one token to 64), and the gated pair of projections h = act(x W_g^T) * (x W_u^T) likewise: what a
// feed-forward block does for single tokens.
//
// Not a shape of the reference's training loop (reference min_DDP.py:95-103).  Bound by reading W once, not by arithmetic: the tiled
// kernels put 128 x 128 outputs on a workgroup and walk the contraction alone, 6 workgroups for W [768, 2048] (29 us for one token).  Here a
// workgroup owns 16 outputs (16 of either half of a gated pair), its eight waves take the contraction 64 at a time in turns, each
// loading 128 consecutive bytes of 16 weight rows straight into matrix operands -- W is never staged, no element of it is used twice -- and
// the waves' sums meet in LDS.  One token through W [4096, 768] as a gated pair: 4.8 us, through W [768, 2048]: 5.7 us, most of either a launch and two
// trips to memory.  v_mfma_f32_16x16x32 takes the weight rows as A and 16 rows of x as B, so a lane ends up with
// four consecutive outputs of one row of x.
#include <type_traits>

#include "device_utils.h"
#include "kernels.h"

namespace dpa {
namespace kernels {

namespace {

constexpr int kWaves = 8;

template <typename TR>
__device__ __forceinline__ f32x4 mfma(const u16x8& a, const u16x8& b, const f32x4& c) {
  if constexpr (std::is_same<TR, F16>::value) {
    typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else {
    typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
}

// Elements k .. k + 7 of a row of K that may start anywhere; zero beyond its end.
__device__ __forceinline__ u16x8 load8(const u16* row, long long k, long long K) {
  if (k + 8 <= K) return *reinterpret_cast<const u16x8_any*>(row + k);
  u16x8 v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = k + j < K ? row[k + j] : static_cast<u16>(0);
  return v;
}

// MT: 16-row tiles of x.  GACT: activation of a gated pair, kActNone for a plain product.
template <typename TR, int MT, int GACT>
__global__ __launch_bounds__(64 * kWaves) void few_rows_kernel(GemmArgs p) {
  constexpr int P = GACT == kActNone ? 1 : 2;  // weight rows per output
  __shared__ f32x4 sums[kWaves][MT][P][64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, g = lane >> 4, li = lane & 15;
  const long long N = GACT == kActNone ? p.N : p.gate_H, n0 = static_cast<long long>(blockIdx.x) * 16;
  const long long n = n0 + li < N ? n0 + li : N - 1;  // rows past the edge repeat the last one and are not stored
  const u16* W = static_cast<const u16*>(p.B) + n * p.ldb;
  const u16* X[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) X[t] = static_cast<const u16*>(p.A) + (16 * t + li < p.M ? 16 * t + li : p.M - 1) * p.lda;
  f32x4 acc[MT][P];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int q = 0; q < P; ++q) acc[t][q] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (long long k0 = 64 * wid; k0 < p.K; k0 += 64 * kWaves) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const long long k = k0 + 32 * s + 8 * g;
      u16x8 w[P], x[MT];
#pragma unroll
      for (int q = 0; q < P; ++q) w[q] = load8(W + q * N * p.ldb, k, p.K);
#pragma unroll
      for (int t = 0; t < MT; ++t) x[t] = load8(X[t], k, p.K);
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int q = 0; q < P; ++q) acc[t][q] = mfma<TR>(w[q], x[t], acc[t][q]);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int q = 0; q < P; ++q) sums[wid][t][q][lane] = acc[t][q];
  __syncthreads();
  if (wid >= MT) return;
  const int t = wid;
  const long long row = 16 * t + li, col = n0 + 4 * g;
  f32x4 r[P];
#pragma unroll
  for (int q = 0; q < P; ++q) {
    r[q] = sums[0][t][q][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) r[q] += sums[w][t][q][lane];
  }
  if (row >= p.M) return;
  const u16* bias = static_cast<const u16*>(p.bias);
  u16* C = static_cast<u16*>(p.C) + row * p.ldc;
  u16* GU = p.pre_act ? static_cast<u16*>(p.pre_act) + row * 2 * N : nullptr;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (col + e >= N) break;
    float a = r[0][e] + (bias ? TR::to_f32(bias[col + e]) : 0.f);
    if constexpr (GACT != kActNone) {
      const float u = r[P - 1][e] + (bias ? TR::to_f32(bias[N + col + e]) : 0.f);
      if (GU) {
        GU[col + e] = TR::from_f32(a);
        GU[N + col + e] = TR::from_f32(u);
      }
      a = gate_value<GACT>(a) * u;
    }
    C[col + e] = TR::from_f32(a);
  }
}

}  // namespace

bool few_rows_supported(const GemmArgs& a, int dtype) {
  return (dtype == kBF16 || dtype == kF16) && a.a_kmajor && a.b_kmajor && a.M >= 1 && a.M <= kFewRows && a.N >= 1 && a.K >= 1 &&
         a.N < (1ll << 27) /* a launch counts its threads in 32 bits */ && a.beta == 0.f && a.alpha == 1.f && (a.gate == 1 || (a.gate == 0 && a.act == kActNone && a.pre_act == nullptr));
}

void launch_few_rows(const GemmArgs& a, int dtype, hipStream_t stream) {
  const long long N = a.gate ? a.gate_H : a.N;
  const dim3 grid(static_cast<unsigned>((N + 15) / 16));
  auto typed = [&](auto tr) {
    using TR = decltype(tr);
    auto sized = [&](auto act_c) {
      constexpr int GACT = decltype(act_c)::value;
      if (a.M <= 16) hipLaunchKernelGGL((few_rows_kernel<TR, 1, GACT>), grid, dim3(64 * kWaves), 0, stream, a);
      else if (a.M <= 32) hipLaunchKernelGGL((few_rows_kernel<TR, 2, GACT>), grid, dim3(64 * kWaves), 0, stream, a);
      else hipLaunchKernelGGL((few_rows_kernel<TR, 4, GACT>), grid, dim3(64 * kWaves), 0, stream, a);
    };
    if (a.gate == 0) sized(std::integral_constant<int, kActNone>{});
    else if (a.act == kActSilu) sized(std::integral_constant<int, kActSilu>{});
    else if (a.act == kActGelu) sized(std::integral_constant<int, kActGelu>{});
    else sized(std::integral_constant<int, kActRelu>{});
  };
  if (dtype == kF16) typed(F16{});
  else typed(BF16{});
}

}  // namespace kernels
}  // namespace dpa
