// Distillation from a teacher's top logits for gfx950: loss and logits gradient of a student's row against K stored
// (class, logit) pairs of a teacher, mixed with the cross-entropy of a hard label.
//
// No counterpart in the reference, whose only criterion is nn.CrossEntropyLoss (reference min_DDP.py:75,100); it stands
// beside the fused cross-entropy of softmax_xent.hip.  Per row, with z the C student logits and t the K teacher logits:
//   p_k  = softmax(t / tau) over the K entries that are there (id in [0, C), t > -inf)
//   q    = softmax(z / tau),  q1 = softmax(z)                                     over the C classes
//   loss = (1 - a) tau^2 sum_k p_k (log p_k - log q[id_k])  -  a log q1[y]
//   dz_j = w { (1 - a) tau ( q_j - sum_{k: id_k = j} p_k )  +  a ( q1_j - [j = y] ) },   w = upstream gradient / #rows
//
// One workgroup per row.  The row is read once: every thread keeps its 16-byte vectors packed in registers through the
// maximum, the two sums of exponentials and the gradient, so a fused call moves exactly one read and one write of the
// logits.  Rows too wide for the registers are read twice, the second time out of the 256 MB cache: maximum and sums are then taken in one pass.
// With one temperature in play (tau = 1, a = 0 or a = 1) there is one exponential per element and pass; otherwise the one at temperature 1 is a power of the other where tau is 2 or 4,
// and a second exponential for other tau (an exponential takes four issue slots, a power one or two).
// The K teacher entries (and the label, as one more) are a scatter into the row.  A vector that is about to be stored has to know its entries: LDS
// holds one bit per vector (a wave's 64 vectors are one 64-bit word, so most waves skip the look-up on a scalar
// branch) and a chained hash from vector to entries.  Entries of one class are summed beforehand in index order by the
// first of them, which makes the result independent of the order in which the chains were built.
// Bound by memory with one temperature: 8192 x 50304 bf16, 32 entries, every row counted, forward and gradient in 345 us (4.8 TB/s, the rate of a
// copy); 2049 x 50257 fp32 with a second exponential 228 us (3.6 TB/s).  With both temperatures and powers 24576 x 50304 float32 logits and their
// bf16 gradient take 1.75 ms (4.2 TB/s of one reading and the gradient).
// Everything is fp32 but the logits and their gradient; in fp16 the gradient is only ever rounded with the upstream gradient in it.
// Rows need no alignment: element j of a row sits in vector (j + shift) / V of the 16-byte grid, the vectors at both ends are stored
// element by element.
#include <type_traits>

#include "device_utils.h"
#include "kernels.h"

namespace dpa {
namespace kernels {

namespace {

constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kNone = 0x7fffffff;
// An exponent below those of all logits that count (2^24 in size after the division by tau), where nothing has been added up yet.  Not lower: relative to itself
// a logit of -1e30 or the type's lowest value, as masks have, would be off by the rounding of its exponent, which is then beyond any float's.
constexpr float kLowest = -1e8f;
constexpr long long kRowsPerLaunch = 1 << 21;  // a launch counts its threads (1024 a row at most) in 32 bits
enum Mode : int { kForward = 0, kBackward = 1, kFused = 2 };

// Sum / maximum over the threads of a workgroup, in a fixed order.
template <int NW>
__device__ __forceinline__ float sum_of_waves(const float* s) {
  float v = s[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) v += s[w];
  return v;
}

__device__ __forceinline__ float teacher_at(const DistillArgs& a, long long i) {
  if (a.teacher_dtype == kF32) return static_cast<const float*>(a.teacher)[i];
  const u16 raw = static_cast<const u16*>(a.teacher)[i];
  return a.teacher_dtype == kBF16 ? BF16::to_f32(raw) : F16::to_f32(raw);
}

// THREADS x KEEP 16-byte vectors are held in registers (KEEP = 0: none, every pass reads memory).  SECOND: how the exponentials at
// temperature 1 come about when both temperatures are needed -- 0: they are not, 1: by an exponential of their own, 2 / 4: as the square /
// fourth power of those at temperature 2 / 4.  TO: type of the gradient, TR's own or, of float32 logits on rows that start on 16-byte boundaries, a
// 16-bit one.
template <typename TR, typename TO, int THREADS, int KEEP, int MODE, int SECOND, int WAVES_PER_SIMD>
__global__ __launch_bounds__(THREADS, WAVES_PER_SIMD) void distill_kernel(DistillArgs a) {
  using T = typename TR::T;
  using O = typename TO::T;
  constexpr int V = TR::kVec, NW = THREADS / 64;
  constexpr bool GRAD = MODE != kForward;
  static_assert(KEEP == 0 || MODE != kBackward, "the backward reads every vector once");
  extern __shared__ int s_dyn[];  // ids[K + 1] | p[K + 1] | x[K + 1] | next[K + 1] | head[hash] | bits[2 * words]
  __shared__ float s_m[NW], s_s[NW], s_s1[NW], s_b, s_xy;
  __shared__ int s_arg[NW], s_some, s_first;
  const int entries = a.K + 1;  // the hard label is the last entry
  int* const s_id = s_dyn;
  float* const s_p = reinterpret_cast<float*>(s_dyn + entries);
  float* const s_x = s_p + entries;
  int* const s_next = s_dyn + 3 * entries;
  int* const s_head = s_next + entries;
  unsigned* const s_bits = reinterpret_cast<unsigned*>(s_head + a.hash);

  const long long r = a.row0 + blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int C = static_cast<int>(a.C), ld = static_cast<int>(a.out_ld);
  const T* row = static_cast<const T*>(a.logits) + r * a.ld;
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const char* grid_in = reinterpret_cast<const char*>(row) - shift * sizeof(T);                       // the row's first 16-byte vector
  char* grid_out = GRAD ? reinterpret_cast<char*>(static_cast<O*>(a.dlogits) + r * a.out_ld - shift) : nullptr;  // (its alignment: checked by the host)
  const int nvec = (shift + C + V - 1) / V, nvec_ld = (shift + ld + V - 1) / V;
  const long long target = a.targets ? a.targets[r] : -1;
  const bool ignored = a.targets && (target == a.ignore_index || target < 0 || target >= C);

  auto store_vec = [&](int k, const float (&d)[V]) __attribute__((always_inline)) {
    const int j0 = k * V - shift;
    O* out = reinterpret_cast<O*>(grid_out + static_cast<unsigned>(V * sizeof(O)) * static_cast<unsigned>(k));
    if (j0 >= 0 && j0 + V <= ld) {
      if constexpr (V == TO::kVec) {
        store_from_f32<TO, V, true>(out, d);
      } else {
        u16x4 v;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = TO::from_f32(d[j]);
        __builtin_nontemporal_store(v, reinterpret_cast<u16x4_any*>(out));
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j0 + j >= 0 && j0 + j < ld) out[j] = TO::from_f32(d[j]);
    }
  };
  if (ignored) {
    if (GRAD) {
      const float z[V] = {};
      for (int k = tid; k < nvec_ld; k += THREADS) store_vec(k, z);
    }
    if (MODE != kBackward && tid == 0) {
      a.row_loss[r] = 0.f;
      a.correct[r] = 0;
      if (MODE == kForward)
        for (int i = 0; i < 3; ++i) a.row_stats[3 * r + i] = 0.f;
    }
    return;
  }

  raw16 kept[KEEP > 0 ? KEEP : 1];
  auto load_vec = [&](int k) { return __builtin_nontemporal_load(reinterpret_cast<const raw16*>(grid_in + 16u * static_cast<unsigned>(k))); };
  if constexpr (KEEP > 0) {
#pragma unroll
    for (int q = 0; q < KEEP; ++q) {
      const int k = tid + q * THREADS;
      if (k < nvec) kept[q] = load_vec(k);
    }
  }
  // One pass over the row's vectors: f(k, packed vector).  WHOLE tells vectors of nothing but classes from those at the row's ends.
  auto each_vec = [&](auto&& f) __attribute__((always_inline)) {
    auto one = [&](int k, const raw16& v) __attribute__((always_inline)) {
      const int j0 = k * V - shift;
      if (j0 >= 0 && j0 + V <= C) f(k, v, std::true_type{});
      else f(k, v, std::false_type{});
    };
    if constexpr (KEEP > 0) {
#pragma unroll
      for (int q = 0; q < KEEP; ++q) {
        const int k = tid + q * THREADS;
        if (k < nvec) one(k, kept[q]);
        __builtin_amdgcn_sched_barrier(0);  // one vector at a time: interleaved, the expansions of all of them would be live at once
      }
      // opaque between the passes, or the compiler keeps the fp32 expansions of one pass for the next and spills
#pragma unroll
      for (int q = 0; q < KEEP; ++q) keep_packed(kept[q]);
    } else {
      constexpr int AHEAD = 4;  // vectors on their way at a time
      for (int k0 = tid; k0 < nvec; k0 += AHEAD * THREADS) {
        raw16 v[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q)
          if (k0 + q * THREADS < nvec) v[q] = *reinterpret_cast<const raw16*>(grid_in + 16u * static_cast<unsigned>(k0 + q * THREADS));
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
          if (k0 + q * THREADS < nvec) one(k0 + q * THREADS, v[q]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  };
  // Element j of a vector outside the classes?
  auto outside = [&](int k, int j) { const int at = k * V - shift + j; return at < 0 || at >= C; };

  // ---- the teacher's entries: ids, scaled logits, the student's logits at those classes; the label behind them
  if (GRAD) {
    for (int i = tid; i < a.hash; i += THREADS) s_head[i] = -1;
    for (int i = tid; i < a.words * 2; i += THREADS) s_bits[i] = 0u;
  }
  for (int k = tid; k < a.K; k += THREADS) {
    const long long at = r * a.K + k;
    const long long id = a.ids_64 ? static_cast<const long long*>(a.ids)[at] : static_cast<const int*>(a.ids)[at];
    const bool in = id >= 0 && id < C;
    const float t = in ? teacher_at(a, at) : kNegInf;  // (divided by tau as a difference to the largest: the type's lowest value is an entry too)
    const bool there = in && t != kNegInf && a.soft_weight != 0.f;  // without a soft term the teacher's values do not matter at all
    s_id[k] = there ? static_cast<int>(id) : -1;
    s_p[k] = t;
    if (MODE != kBackward) s_x[k] = there ? TR::to_f32(row[id]) : 0.f;
  }
  if (tid == 0) {
    s_id[a.K] = a.hard_weight != 0.f ? static_cast<int>(target) : -1;
    if (MODE != kBackward) s_xy = a.targets ? TR::to_f32(row[target]) : 0.f;
  }
  __syncthreads();
  if (GRAD) {
    for (int k = tid; k < entries; k += THREADS) {
      const int id = s_id[k];
      if (id < 0) continue;
      const int vec = (id + shift) / V;
      s_next[k] = atomicExch(&s_head[vec & (a.hash - 1)], k);
      atomicOr(&s_bits[vec >> 5], 1u << (vec & 31));
    }
  }

  auto power = [](float e) __attribute__((always_inline)) {  // of an exponential at temperature 2 / 4, the one at temperature 1
    const float e2 = e * e;
    return SECOND == 2 ? e2 : e2 * e2;
  };

  // ---- row maximum: of whole vectors, three values an instruction; which element it is, only its owners look up
  const float c = a.exp_scale;  // log2(e) / temperature of the first exponential
  float m, mt = kNegInf, S = 0.f, S1 = 0.f;
  float s = 0.f, s1 = 0.f, at = kLowest, at1 = kLowest;  // (rows read again: sums so far, relative to this thread's largest exponents so far)
  int best = kNone;
  if (MODE == kBackward) {
    m = a.row_stats[3 * r];
    S = a.row_stats[3 * r + 1];
    S1 = a.row_stats[3 * r + 2];
  } else {
    each_vec([&](int k, const raw16& v, auto whole) __attribute__((always_inline)) {
      float x[V];
      raw_to_f32<TR, V>(v, x);
      float vm = kNegInf;
#pragma unroll
      for (int j = 0; j < V; ++j) vm = fmaxf(vm, decltype(whole)::value || !outside(k, j) ? x[j] : kNegInf);
      if (vm > mt) { mt = vm; best = k; }
      if constexpr (KEEP == 0) {
        // A row that is not kept would have to be read once more for the sums: they are taken along, and follow the maximum.
        const float to = fmaxf(at, vm * c), f = __builtin_amdgcn_exp2f(at - to);
        at = to;
        s *= f;
        if (SECOND == 1) {
          const float to1 = fmaxf(at1, vm * kLog2e);
          s1 *= __builtin_amdgcn_exp2f(at1 - to1);
          at1 = to1;
        } else if (SECOND) {
          s1 *= power(f);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (!decltype(whole)::value && outside(k, j)) x[j] = kNegInf;
          const float e = __builtin_amdgcn_exp2f(fmaf(x[j], c, -at));
          s += e;
          if (SECOND == 1) s1 += __builtin_amdgcn_exp2f(fmaf(x[j], kLog2e, -at1));
          else if (SECOND) s1 += power(e);
        }
      }
    });
    m = mt;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    if (lane == 0) s_m[wid] = m;
    __syncthreads();
    m = s_m[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = fmaxf(m, s_m[w]);
  }
  // Exponents are fma(x, c, -mc): the rounding of mc is the same in every term and in the sums, so it cancels wherever the same mc is used.
  const float mc = m * c, mc1 = m * kLog2e;
  auto second = [&](float x, float e) __attribute__((always_inline)) {
    if (SECOND == 1) return __builtin_amdgcn_exp2f(fmaf(x, kLog2e, -mc1));
    return power(e);
  };
  if (MODE != kBackward) {
    int arg = kNone;
    if (__any(mt == m)) {
      if (mt == m) {
        raw16 v = raw16{0u, 0u, 0u, 0u};
        if constexpr (KEEP > 0) {
#pragma unroll
          for (int q = 0; q < KEEP; ++q)
            if (best == tid + q * THREADS) v = kept[q];
        } else {
          if (best != kNone) v = *reinterpret_cast<const raw16*>(grid_in + 16u * static_cast<unsigned>(best));
        }
        float x[V];
        raw_to_f32<TR, V>(v, x);
#pragma unroll
        for (int j = V - 1; j >= 0; --j)
          if (best != kNone && x[j] == m && !outside(best, j)) arg = best * V - shift + j;
      }
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) {
        const int oa = __shfl_xor(arg, off, 64);
        arg = oa < arg ? oa : arg;
      }
    }
    if (lane == 0) s_arg[wid] = arg;

    // ---- sums of exponentials at both temperatures
    if constexpr (KEEP == 0) {
      const float f = __builtin_amdgcn_exp2f(at - mc);
      s *= f;
      if (SECOND == 1) s1 *= __builtin_amdgcn_exp2f(at1 - mc1);
      else if (SECOND) s1 *= power(f);
    }
    else each_vec([&](int k, const raw16& v, auto whole) __attribute__((always_inline)) {
      float x[V];
      raw_to_f32<TR, V>(v, x);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (!decltype(whole)::value && outside(k, j)) x[j] = kNegInf;
        const float e = __builtin_amdgcn_exp2f(fmaf(x[j], c, -mc));
        s += e;
        if (SECOND) s1 += second(x[j], e);
      }
    });
    s = wave_sum(s);
    if (SECOND) s1 = wave_sum(s1);
    if (lane == 0) { s_s[wid] = s; s_s1[wid] = s1; }
  }
  if (MODE == kBackward) __syncthreads();  // the chains are complete

  // ---- one wave turns the teacher's logits into probabilities
  if (wid == 0) {
    float tm = kNegInf;
    int first = kNone;  // first entry with the largest logit
    for (int k = lane; k < a.K; k += 64)
      if (s_id[k] >= 0 && !(s_p[k] <= tm)) { tm = s_p[k]; first = k; }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const float om = __shfl_xor(tm, off, 64);
      const int ob = __shfl_xor(first, off, 64);
      if (om > tm || (om == tm && ob < first)) { tm = om; first = ob; }
    }
    float z = 0.f;
    for (int k = lane; k < a.K; k += 64)
      if (s_id[k] >= 0) z += __builtin_amdgcn_exp2f((s_p[k] - tm) * a.inv_tau * kLog2e);
    z = wave_sum(z);
    const float log_z = logf(z), inv_z = 1.f / z;
    float b = 0.f;  // sum_k p_k (log p_k - log(exponential of x_k)); with log(sum) added it is the divergence
    for (int k = lane; k < a.K; k += 64) {
      if (s_id[k] < 0) continue;
      const float t = (s_p[k] - tm) * a.inv_tau;
      const float p = __builtin_amdgcn_exp2f(t * kLog2e) * inv_z;
      if (MODE != kBackward && !(p == 0.f)) b += p * ((t - log_z) - fmaf(s_x[k], c, -mc) * kLn2);
      s_p[k] = p * (a.soft_weight * a.tau);  // its share of the gradient
    }
    if (lane == 0) s_p[a.K] = a.hard_weight;
    b = wave_sum(b);
    if (GRAD) {
      // shares of the entries of one class, added up by the first of them: s_x[k]
      for (int k = lane; k < entries; k += 64) {
        const int id = s_id[k];
        if (id < 0) continue;
        bool leads = true, alone = true;
        for (int e = s_head[((id + shift) / V) & (a.hash - 1)]; e >= 0; e = s_next[e])
          if (e != k && s_id[e] == id) {
            alone = false;
            leads = leads && k < e;
          }
        float p = s_p[k];
        if (!alone && leads)
          for (int e = k + 1; e < entries; ++e) p += s_id[e] == id ? s_p[e] : 0.f;
        s_x[k] = leads ? p : 0.f;
      }
    }
    if (lane == 0) {
      s_some = first != kNone;
      s_first = first != kNone ? s_id[first] : -1;
      s_b = b;
    }
  }
  __syncthreads();
  const bool some = s_some != 0;
  if (MODE != kBackward) {
    S = sum_of_waves<NW>(s_s);
    if (SECOND) S1 = sum_of_waves<NW>(s_s1);
    if (tid == 0) {
      int arg = s_arg[0];
#pragma unroll
      for (int w = 1; w < NW; ++w) arg = s_arg[w] < arg ? s_arg[w] : arg;
      const float soft = some && a.soft_weight != 0.f ? (s_b + logf(S)) * a.tau * a.tau * a.soft_weight : 0.f;
      const float hard =
          a.hard_weight != 0.f ? (logf(SECOND ? S1 : S) - (SECOND ? fmaf(s_xy, kLog2e, -mc1) : fmaf(s_xy, c, -mc)) * kLn2) * a.hard_weight : 0.f;
      a.row_loss[r] = soft + hard;
      // without targets: agreement with the teacher's first choice
      a.correct[r] = arg == (a.targets ? static_cast<int>(target) : s_first) ? 1 : 0;
      if (MODE == kForward) {
        a.row_stats[3 * r] = m;
        a.row_stats[3 * r + 1] = S;
        a.row_stats[3 * r + 2] = S1;
      }
    }
  }
  if (!GRAD) return;

  // ---- gradient
  float w = 1.f;
  if (a.scale) {
    w = a.scale[0];
  } else if (a.mean) {  // few rows: every wave counts them itself
    int n = static_cast<int>(a.N);
    if (a.targets) {
      n = 0;
      for (int i = lane; i < a.N; i += 64) n += a.targets[i] != a.ignore_index ? 1 : 0;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, 64);
    }
    w = 1.f / fmaxf(static_cast<float>(n), 1.f);
  }
  if (MODE == kBackward) w *= a.grad_out[a.grad_out_rows ? r : 0];
  const float cs = some ? w * a.soft_weight * a.tau : 0.f, ch = w * a.hard_weight;
  // coefficients of the exponentials: with one temperature both terms share it (tau = 1) or one of them is absent
  const float c0 = (SECOND ? cs : cs + ch) / S, c1 = SECOND ? ch / S1 : 0.f;
  each_vec([&](int k, const raw16& v, auto whole) __attribute__((always_inline)) {
    float x[V], d[V];
    raw_to_f32<TR, V>(v, x);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float e = __builtin_amdgcn_exp2f(fmaf(x[j], c, -mc));
      d[j] = c0 * e;
      if (SECOND) d[j] = fmaf(c1, second(x[j], e), d[j]);
      if (!decltype(whole)::value && outside(k, j)) d[j] = 0.f;
    }
    // a wave's vectors are 64 consecutive ones: one word of bits, the same for all its lanes
    const unsigned* bits = s_bits + 2 * (k >> 6);
    const unsigned mine = bits[lane >> 5];
    if (__any(mine != 0u) && (mine >> (k & 31) & 1u)) {
      const int j0 = k * V - shift;
      for (int e = s_head[k & (a.hash - 1)]; e >= 0; e = s_next[e]) {
        const int at = s_id[e] - j0;
        if (at < 0 || at >= V) continue;
        const float p = w * s_x[e];
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] -= j == at ? p : 0.f;
      }
    }
    store_vec(k, d);
  });
  const float zero[V] = {};
  for (int k = nvec + tid; k < nvec_ld; k += THREADS) store_vec(k, zero);
}

// metrics = {loss sum, correct, counted rows, loss sum / counted rows}; loss[0] = the requested reduction.  One workgroup,
// fixed order.
__global__ __launch_bounds__(1024) void distill_reduce_kernel(const float* __restrict__ row_loss, const unsigned char* __restrict__ correct,
                                                              const long long* __restrict__ targets, long long N, long long ignore_index,
                                                              int mean, float* __restrict__ metrics, float* __restrict__ loss) {
  __shared__ float scratch[16];
  float l = 0.f, c = 0.f, n = 0.f;
#pragma unroll 4
  for (long long i = threadIdx.x; i < N; i += 1024) {
    l += row_loss[i];
    c += correct[i] ? 1.f : 0.f;
    n += !targets || targets[i] != ignore_index ? 1.f : 0.f;
  }
  l = block_sum<16>(l, scratch);
  c = block_sum<16>(c, scratch);
  n = block_sum<16>(n, scratch);
  if (threadIdx.x == 0) {
    metrics[0] = l;
    metrics[1] = c;
    metrics[2] = n;
    metrics[3] = l / fmaxf(n, 1.f);
    loss[0] = mean ? l / fmaxf(n, 1.f) : l;
  }
}

// scale[0] = 1 / max(#rows that count, 1) for a mean, 1 for a sum.
__global__ __launch_bounds__(1024) void distill_scale_kernel(const long long* __restrict__ targets, long long N, long long ignore_index, int mean,
                                                             float* __restrict__ scale) {
  __shared__ float scratch[16];
  float n = 0.f;
  if (mean && targets) {
#pragma unroll 4
    for (long long i = threadIdx.x; i < N; i += 1024) n += targets[i] != ignore_index ? 1.f : 0.f;
    n = block_sum<16>(n, scratch);
  } else {
    n = static_cast<float>(N);
  }
  if (threadIdx.x == 0) scale[0] = mean ? 1.f / fmaxf(n, 1.f) : 1.f;
}

// x *= g[0] unless g[0] is 1 (the usual loss.backward()), in which case nothing is read or written.
template <typename TR>
__global__ __launch_bounds__(256) void distill_apply_upstream_kernel(typename TR::T* x, long long n, const float* __restrict__ g) {
  const float s = g[0];
  if (s == 1.f) return;
  constexpr int V = TR::kVec;
  const long long nv = (reinterpret_cast<uintptr_t>(x) & 15) == 0 ? n / V : 0, step = static_cast<long long>(gridDim.x) * 256;
  const long long first = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  for (long long i = first; i < nv; i += step) {
    float v[V];
    load_as_f32<TR, V>(x + i * V, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] *= s;
    store_from_f32<TR, V>(x + i * V, v);
  }
  for (long long i = nv * V + first; i < n; i += step) x[i] = TR::from_f32(TR::to_f32(x[i]) * s);
}

}  // namespace

bool distill_supported(long long C, long long ld, long long K) {
  return C >= 1 && C <= ld && ld <= kDistillMaxWidth && K >= 1 && K <= kDistillMaxEntries;
}

void launch_distill(const DistillArgs& args, int dtype, int out_dtype, int mode, hipStream_t stream) {
  if (args.N <= 0) return;
  DistillArgs a = args;
  if (mode == kForward || dtype == out_dtype) a.out_ld = a.ld;
  const bool dual = a.tau != 1.f && a.soft_weight != 0.f && a.hard_weight != 0.f;
  // one exponential: at the temperature of the term that is there (tau = 1: of both)
  a.exp_scale = (a.soft_weight != 0.f ? a.inv_tau : 1.f) * kLog2e;
  a.hash = 64;
  while (a.hash <= a.K) a.hash *= 2;
  auto typed = [&](auto tr, auto to) {
    using TR = decltype(tr);
    using TO = decltype(to);
    constexpr int V = TR::kVec;
    const long long nvec = (a.ld + 2 * V - 2) / V;  // worst alignment
    a.words = static_cast<int>((nvec + 63) / 64);
    const size_t lds = (static_cast<size_t>(4) * (a.K + 1) + a.hash + 2 * static_cast<size_t>(a.words)) * 4;
    auto go = [&](auto threads_c, auto keep_c, auto mode_c, auto waves_c) {
      constexpr int THREADS = decltype(threads_c)::value, KEEP = decltype(keep_c)::value, MODE = decltype(mode_c)::value;
      constexpr int WAVES = decltype(waves_c)::value;
      const dim3 grid(static_cast<unsigned>(args.N - a.row0 < kRowsPerLaunch ? args.N - a.row0 : kRowsPerLaunch));
      if (!dual) hipLaunchKernelGGL((distill_kernel<TR, TO, THREADS, KEEP, MODE, 0, WAVES>), grid, dim3(THREADS), lds, stream, a);
      else if (a.tau == 2.f) hipLaunchKernelGGL((distill_kernel<TR, TO, THREADS, KEEP, MODE, 2, WAVES>), grid, dim3(THREADS), lds, stream, a);
      else if (a.tau == 4.f) hipLaunchKernelGGL((distill_kernel<TR, TO, THREADS, KEEP, MODE, 4, WAVES>), grid, dim3(THREADS), lds, stream, a);
      else hipLaunchKernelGGL((distill_kernel<TR, TO, THREADS, KEEP, MODE, 1, WAVES>), grid, dim3(THREADS), lds, stream, a);
    };
    static_assert(((4 * (kDistillMaxEntries + 1) + 2 * kDistillMaxEntries + 2 * ((kDistillMaxWidth / 4 + 64) / 64)) * 4) <= 60 * 1024,
                  "a workgroup's tables fit the 64 KiB that a launch may have without asking");
    using std::integral_constant;
    auto by_size = [&](auto mode_c) {
      constexpr int MODE = decltype(mode_c)::value;
      constexpr integral_constant<int, MODE> m{};
      constexpr integral_constant<int, 4> w4{};
      constexpr integral_constant<int, 8> w8{};
      constexpr integral_constant<int, 64> t64{};
      constexpr integral_constant<int, 256> t256{};
      [[maybe_unused]] constexpr integral_constant<int, 512> t512{};
      constexpr integral_constant<int, 1024> t1024{};
      constexpr integral_constant<int, 0> none{};
      if constexpr (MODE == kBackward) {
        if (nvec <= 64 * 4) go(t64, none, m, w4);
        else if (nvec <= 256 * 7) go(t256, none, m, w4);
        else go(t1024, none, m, w8);
      } else {
        if (nvec <= 64 * 4) go(t64, integral_constant<int, 4>{}, m, w4);
        else if (nvec <= 256 * 7) go(t256, integral_constant<int, 7>{}, m, w4);
        else if (nvec <= 1024 * 7) go(t1024, integral_constant<int, 7>{}, m, w8);
        else if constexpr (std::is_same<TR, TO>::value) {
          if (nvec <= 1024 * 16) go(t1024, integral_constant<int, 16>{}, m, w4);
          else go(t1024, none, m, w8);
        } else {
          // Float32 logits of a projection, twice the bytes of their gradient: held, a row takes a whole compute unit's registers and is fetched, computed
          // and stored by itself (24576 x 50304: 2.25 ms); read twice, four rows share one and the second reading comes out of the 256 MB cache (1.75 ms;
          // with two rows of 1024 threads 1.91, with eight of 256, whose 400 MB do not stay there, 2.24).
          go(t512, none, m, w8);
        }
      }
    };
    for (a.row0 = 0; a.row0 < args.N; a.row0 += kRowsPerLaunch) {
      if constexpr (std::is_same<TR, TO>::value) {
        if (mode == kForward) by_size(integral_constant<int, kForward>{});
        else if (mode == kBackward) by_size(integral_constant<int, kBackward>{});
        else if constexpr (!std::is_same<TR, F16>::value) by_size(integral_constant<int, kFused>{});  // (fp16 gradients wait for the upstream one)
      } else if constexpr (std::is_same<TO, BF16>::value) {
        by_size(integral_constant<int, kFused>{});  // (bf16 gradients of float32 logits are only asked for with the loss, ...
      } else {
        by_size(integral_constant<int, kBackward>{});  // ... fp16 ones only with the upstream gradient)
      }
    }
  };
  if (mode == kForward || dtype == out_dtype) dispatch_dtype(dtype, [&](auto tr) { typed(tr, tr); });
  else if (out_dtype == kBF16) typed(F32{}, BF16{});
  else typed(F32{}, F16{});
}


void launch_distill_scale(const long long* targets, long long N, long long ignore_index, int mean, float* scale, hipStream_t stream) {
  hipLaunchKernelGGL(distill_scale_kernel, dim3(1), dim3(1024), 0, stream, targets, N, ignore_index, mean, scale);
}

void launch_distill_reduce(const float* row_loss, const unsigned char* correct, const long long* targets, long long N, long long ignore_index,
                           int mean, float* metrics, float* loss, hipStream_t stream) {
  hipLaunchKernelGGL(distill_reduce_kernel, dim3(1), dim3(1024), 0, stream, row_loss, correct, targets, N, ignore_index, mean, metrics, loss);
}

void launch_distill_apply_upstream(void* x, int dtype, long long n, const float* g, hipStream_t stream) {
  if (n <= 0) return;
  dispatch_dtype(dtype, [&](auto tr) {
    using TR = decltype(tr);
    const long long blocks = (n / TR::kVec + 255) / 256;
    hipLaunchKernelGGL((distill_apply_upstream_kernel<TR>), dim3(static_cast<unsigned>(blocks < 1 ? 1 : blocks > 2048 ? 2048 : blocks)), dim3(256), 0,
                       stream, static_cast<typename TR::T*>(x), n, g);
  });
}

}  // namespace kernels
}  // namespace dpa
