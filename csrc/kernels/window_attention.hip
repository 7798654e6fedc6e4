// Causal attention with a sliding window and sinks for gfx950, forward and backward: bf16 / fp16, head size 64 or 128,
// key / value heads shared by groups of query heads, any sequence length, padded batches.
//
// Not an op of the reference (its model is two linear layers, reference min_DDP.py:41-49); it stands beside the causal
// attention of attention.hip.  Query i of a sequence of `len` positions sees key j when
//     j <= i  and  (i - j < window  or  j < sinks)
//   s_ij = c q_i k_j,  p_ij = exp(s_ij - lse_i),  o_i = sum_j p_ij v_j
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i v_j - delta_i),  delta_i = do_i o_i,  dq_i = c sum_j ds_ij k_j,  dk_j = c sum_i ds_ij q_i
// (dk, dv summed over the query heads of a group).
//
// Layout of the work: a workgroup is four waves of 32 rows each -- queries in the forward and dQ kernels, keys in the
// dK/dV kernel -- and walks only the 64-row tiles of the other operand that the window or the sinks can reach; a wave
// skips the tiles that miss its own 32 rows, and only tiles that straddle a border of the mask pay for the comparisons.  The
// products run transposed (S^T = K Q^T), so a query's softmax statistics are scalars of its lane and the probabilities leave the
// accumulators as the operand of the next product without changing lanes; the other operand of that product comes
// from the row-major tile through the transposing LDS read.  Probabilities and score gradients are rounded to the 16-bit type there, as operands
// of a matrix instruction have to be; scores, statistics, delta (of the output as it is stored) and all sums are fp32, and the row sums add up the rounded probabilities, so that
// a row's weights sum to 1.  Tiles travel global -> LDS by DMA, requested one tile (two in the dK/dV kernel at head size 128) ahead.  The tile image is one for both kinds of reads: 16-byte chunk c of row r sits at chunk c ^ swz(r).  The 16 lanes that a row-wise
// read serves at once (rows 0-3 and 12-15 at one chunk, rows 4-11 at the next) then fall on 16 different 16-byte bank groups, and the 8
// rows of a transposing read on 8 different 32-byte groups.
// Rows at and beyond a sequence's length are never read: source rows are clamped to the last valid one, what they
// would contribute is masked, and their outputs and gradients are written as zero.
//
// dK/dV: blocks of 128 keys cost unlike amounts -- a block with sinks meets every later query of every head of its group, the
// others only a window of them -- so the list of (key block, head, query tile) units is cut into pieces of about equal length, one per
// workgroup slot of the chip.  A block inside one piece is written directly; a block that is cut leaves fp32 partial
// sums, which a last kernel adds up in order: no atomics, the same result every time.
//
// Measured (bf16), window 256 / sinks 4 over 64 x 1024 positions, 12 heads of 64: forward 128 us (3.1 TB/s of its inputs and outputs), dQ 174 us
// (3.5 TB/s), dK/dV 215 us (2.8 TB/s).  Neither memory nor the matrix pipes (21 - 35 % busy) are what bounds them: by the counters a square of 32 x 32 scores
// takes 160 vector and 106 scalar instructions in the forward (166 and 103 in dQ, 174 and 126 in dK/dV) beside its 18 to 32 products -- 10 vector
// instructions a score, of which the softmax needs about 4; the others are the mask's comparisons, addresses, and prologues and epilogues over the fewer than
// nine squares that a wave has here -- and the waves wait for the rest (the forward at head size 64 spills 2 registers, dK/dV 9).  Window 1024 / sinks 4 over 16384 positions, 8 heads of 128 on 2: forward 105 us (636 TFLOP/s of
// the visible pairs), dQ 127 us (784), dK/dV 257 us (520; one workgroup a compute unit: its stages and strips are 131 of 160 KiB
// of LDS, and a wave a SIMD, at 304 of 512 registers, has nothing to run while it waits, 48 % of its cycles), join 17 us.
#include <type_traits>

#include "device_utils.h"
#include "kernels.h"

namespace dpa {
namespace kernels {

namespace {

constexpr int kRows = 128;     // rows per workgroup
constexpr int kTile = 64;      // rows per LDS tile
constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_huge_valf();

typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;
using lptr_t = __attribute__((address_space(3))) void*;

template <typename TR>
__device__ __forceinline__ f32x4 mfma(const s16x8& a, const s16x8& b, const f32x4& c) {
  if constexpr (std::is_same<TR, F16>::value) {
    typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else {
    typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
}

template <typename TR>
__device__ __forceinline__ s16x8 pack8(const f32x4& a, const f32x4& b) {
  u16x8 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    r[e] = TR::from_f32(a[e]);
    r[4 + e] = TR::from_f32(b[e]);
  }
  return __builtin_bit_cast(s16x8, r);
}

// Byte offset of 16-byte chunk c of row r in a tile image of [rows][D] 16-bit elements.
template <int D>
__device__ __forceinline__ int swz(int r) {
  return D == 64 ? ((r >> 1) & 3) << 1 : (r & 7) << 1;
}
template <int D>
__device__ __forceinline__ int tile_off(int r, int c) { return r * (2 * D) + ((c ^ swz<D>(r)) << 4); }

// Matrix operand fragment out of a tile: lane holds row 16 t + (lane & 15), d = 32 kk + 8 (lane >> 4) ..
template <int D>
__device__ __forceinline__ s16x8 row_frag(const char* tile, int t, int kk, int lane) {
  return *reinterpret_cast<const s16x8*>(tile + tile_off<D>(16 * t + (lane & 15), 4 * kk + (lane >> 4)));
}
// Transposed fragment: lane holds d = 16 td + (lane & 15); its eight k-slots are rows base + 4 g + 0..3 and base + 16 + 4 g + 0..3
// (g = lane >> 4), the rows that a 16x16 accumulator pair keeps in that lane group's registers.
template <int D>
__device__ __forceinline__ s16x8 tr_frag(const char* tile, int base, int td, int lane) {
  const int g = lane >> 4, i = lane & 15, qq = i >> 2, pp = i & 3;
  const int c = 2 * td + (pp >> 1), sub = (pp & 1) << 3, r = base + 4 * g + qq;
  using lds_ptr = __attribute__((address_space(3))) s16x4*;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(tile + tile_off<D>(r, c) + sub));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(tile + tile_off<D>(r + 16, c) + sub));
  return s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

__device__ __forceinline__ float groups_max(float x) {  // over the four 16-lane groups of a wave
  const unsigned xi = __float_as_uint(x);
  const u32x2 a = __builtin_amdgcn_permlane32_swap(xi, xi, false, false);
  const float m = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const unsigned mi = __float_as_uint(m);
  const u32x2 b = __builtin_amdgcn_permlane16_swap(mi, mi, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float groups_sum(float x) {
  const unsigned xi = __float_as_uint(x);
  const u32x2 a = __builtin_amdgcn_permlane32_swap(xi, xi, false, false);
  const float s = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const unsigned si = __float_as_uint(s);
  const u32x2 b = __builtin_amdgcn_permlane16_swap(si, si, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// At most N of this wave's vector-memory operations (DMA included) outstanding, visible to the compiler's own bookkeeping.
template <int N>
__device__ __forceinline__ void wait_vmem_at_most() {
  static_assert(N >= 0 && N < 64, "vmcnt is a 6-bit counter");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}
__device__ __forceinline__ const char* uniform_ptr(const void* p) {
  const unsigned long long v = reinterpret_cast<unsigned long long>(p);
  const unsigned lo = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(v));
  const unsigned hi = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(v >> 32));
  return reinterpret_cast<const char*>((static_cast<unsigned long long>(hi) << 32) | lo);
}
// 64 x 16 (64 x 4) bytes global -> LDS: lane l's piece lands at lds + 16 l (4 l).  As assembly, because the compiler would put
// every transposing read behind ALL the DMA it knows of; the kernels order DMA and reads by counted waits and barriers.
__device__ __forceinline__ void dma_16B(const char* base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "s"(lds) : "memory");
}
__device__ __forceinline__ void dma_4B(const char* base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dword %0, %1" : : "v"(off), "s"(base), "s"(lds) : "memory");
}
__device__ __forceinline__ unsigned lds_address(const char* p) {
  return __builtin_amdgcn_readfirstlane(static_cast<unsigned>(reinterpret_cast<uintptr_t>((lptr_t)p)));
}

// One wave's share of a tile's requests: D / 16 pieces of 1 KiB of one operand, starting at piece `piece0`.
template <int D>
struct TileSource {
  static constexpr int kPieces = D / 16;
  static constexpr int kPieceRows = 512 / D;   // rows of 2 D bytes per 1 KiB
  static constexpr int kLanesPerRow = 64 / kPieceRows;
  unsigned off[kPieces];
  unsigned pitch;   // bytes between rows
  int row0;         // this lane's row of the first piece
  static __device__ __forceinline__ unsigned chunk_of(int row, int lane) {
    return static_cast<unsigned>(((lane % kLanesPerRow) ^ swz<D>(row)) * 16);
  }
  __device__ __forceinline__ void init(long long stride, int piece0, int lane) {
    pitch = static_cast<unsigned>(stride) * 2u;
    row0 = piece0 * kPieceRows + lane / kLanesPerRow;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) off[i] = static_cast<unsigned>(row0 + i * kPieceRows) * pitch + chunk_of(row0 + i * kPieceRows, lane);
  }
  // `first`: the tile's first row; only `valid` (>= 1) of its rows may be read, the others repeat the last of those.
  __device__ __forceinline__ void request(const u16* first, int valid, unsigned lds) const {
    const char* base = uniform_ptr(first);
    if (valid >= kTile) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) dma_16B(base, off[i], lds + i * 1024);
    } else {
      const int lane = threadIdx.x & 63;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int row = row0 + i * kPieceRows, r = row < valid ? row : valid - 1;
        dma_16B(base, static_cast<unsigned>(r) * pitch + chunk_of(row, lane), lds + i * 1024);
      }
    }
  }
};

template <int D>
constexpr int kTileBytes = kTile * D * 2;
template <int D>
constexpr int kStripPitch = 2 * D + 16;
template <int D>
constexpr int kStripBytes = 32 * kStripPitch<D>;

// The wave's 32 rows leave through an LDS strip of its own, whole rows per store instruction.  acc[st][td]: row 16 st + (lane & 15), d = 16 td + 4 g + e.
// Rows at or beyond `len` become zero, rows at or beyond `T` are not written.  row0: the wave's first row.
template <typename TR, int D>
__device__ __forceinline__ void store_rows(char* strip, const f32x4 (&acc)[2][D / 16], const float (&scale)[2], u16* out, long long stride, int row0, int len,
                                           int T, int lane) {
  const int g = lane >> 4, li = lane & 15;
#pragma unroll
  for (int st = 0; st < 2; ++st) {
    const bool live = row0 + 16 * st + li < len;
#pragma unroll
    for (int td = 0; td < D / 16; ++td) {
      u16x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = live ? TR::from_f32(acc[st][td][e] * scale[st]) : static_cast<u16>(0);
      *reinterpret_cast<u16x4*>(strip + (16 * st + li) * kStripPitch<D> + (16 * td + 4 * g) * 2) = w;
    }
  }
  // a wave reads back only its own writes; the LDS serves one wave's requests in order
  constexpr int kPerRow = D / 8, kRowsPerStore = 64 / kPerRow;
#pragma unroll
  for (int it = 0; it < 32 / kRowsPerStore; ++it) {
    const int r = it * kRowsPerStore + lane / kPerRow, ch = lane % kPerRow;
    const u32x4 v = *reinterpret_cast<const u32x4*>(strip + r * kStripPitch<D> + ch * 16);
    if (row0 + r < T) __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(out + static_cast<long long>(row0 + r) * stride + ch * 8));
  }
}

template <int D>
__device__ __forceinline__ void zero_rows(u16* out, long long stride, int row0, int T) {
  constexpr int kPerRow = D / 8;
  for (int i = threadIdx.x; i < kRows * kPerRow; i += kThreads) {
    const int r = row0 + i / kPerRow;
    if (r < T) *reinterpret_cast<u32x4*>(out + static_cast<long long>(r) * stride + (i % kPerRow) * 8) = u32x4{0u, 0u, 0u, 0u};
  }
}

// Workgroup id -> position in an order whose neighbours share an XCD (and so its L2).
__device__ __forceinline__ int xcd_order(int id, int n) {
  const int q = n >> 3, r = n & 7, x = id & 7;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (id >> 3);
}

__device__ __forceinline__ int length_of(const WindowAttnArgs& p, int b) {
  if (!p.lens) return p.T;
  const int n = p.lens[b];
  return n < 0 ? 0 : n > p.T ? p.T : n;
}

// Key tiles that a block of queries q0 .. q0 + 127 can see: the first `sink_tiles` tiles, then tiles first .. last.
struct KeyTiles {
  int sink_tiles, first, count;
  __device__ __forceinline__ KeyTiles(const WindowAttnArgs& p, int q0, int len) {
    const int lo = q0 - p.window + 1, hi = q0 + kRows - 1 < len - 1 ? q0 + kRows - 1 : len - 1;
    first = (lo > 0 ? lo : 0) / kTile;
    const int s = (p.sinks + kTile - 1) / kTile;
    sink_tiles = s < first ? s : first;
    count = sink_tiles + hi / kTile - first + 1;
  }
  __device__ __forceinline__ int key0(int it) const { return (it < sink_tiles ? it : first + it - sink_tiles) * kTile; }
  // Rows of the tile that the block may see at all: the tiles in front of the window hold sinks only.
  __device__ __forceinline__ int valid(const WindowAttnArgs& p, int it, int len) const {
    return (it < sink_tiles && p.sinks < len ? p.sinks : len) - key0(it);
  }
};

// What a wave of 32 queries from qw has to do with the 32 keys from k0.  A border of the mask crosses few of these squares, and most of
// those are crossed by one border only: the comparisons are instantiated for the border (two instructions a score) and only squares
// with several take all of them.
enum Border : int { kClear = 0, kCausal = 1, kWindow = 2, kSinks = 3, kSeveral = 4, kUnseen = 5 };
__device__ __forceinline__ int border_of(const WindowAttnArgs& p, int qw, int k0) {
  if (k0 > qw + 31) return kUnseen;
  const bool future = k0 + 31 > qw, past = k0 <= qw + 31 - p.window && k0 + 31 >= p.sinks;
  if (!past) return future ? kCausal : kClear;
  if (k0 + 31 <= qw - p.window) return k0 < p.sinks ? kSinks : kUnseen;  // behind every query's window: sinks or nothing
  return future || k0 < p.sinks ? kSeveral : kWindow;
}
// Hides key index j of a lane whose query is at index `rel`; sinks end at index `sink`.
template <int BORDER>
__device__ __forceinline__ bool hidden(const WindowAttnArgs& p, int j, int rel, int sink) {
  if (BORDER == kCausal) return j > rel;
  if (BORDER == kWindow) return j <= rel - p.window;
  if (BORDER == kSinks) return j >= sink;
  if (BORDER == kSeveral) return j > rel || (j <= rel - p.window && j >= sink);
  return false;
}
// f(std::integral_constant<int, border>) for a border other than kClear and kUnseen.
template <typename F>
__device__ __forceinline__ void with_border(int border, F&& f) {
  if (border == kCausal) f(std::integral_constant<int, kCausal>{});
  else if (border == kWindow) f(std::integral_constant<int, kWindow>{});
  else if (border == kSinks) f(std::integral_constant<int, kSinks>{});
  else f(std::integral_constant<int, kSeveral>{});
}
// Scores of hidden pairs become -inf: their probabilities are then exactly 0, and with them all they contribute.  Register (t, e) of s[st] is query
// qw + 16 st + (lane & 15) and key k0 + 16 t + 4 (lane >> 4) + e.  (Only this step depends on the border.  With the whole square instantiated for each,
// the five copies' accumulators met in 42 moves a square.)
__device__ __forceinline__ void hide_keys(const WindowAttnArgs& p, f32x4 (&s)[2][2], int qw, int k0, int border, int lane) {
  if (border == kClear) return;
  with_border(border, [&](auto b_c) __attribute__((always_inline)) {
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const int rel = qw + 16 * st + (lane & 15) - k0 - 4 * (lane >> 4), sink = p.sinks - k0 - 4 * (lane >> 4);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (hidden<decltype(b_c)::value>(p, 16 * (i >> 2) + (i & 3), rel, sink)) s[st][i >> 2][i & 3] = kNegInf;
    }
  });
}

// ---------------------------------------------------------------------------------------------------- forward
// Online softmax over raw scores with the scale in the exponent's FMA; the running maximum (log2 domain) only moves when a score
// exceeds it by more than kDefer, so probabilities stay below 2^kDefer and the rescale of the output is rare.  Row sums come out of
// the matrix pipe (ones times P), of exactly the rounded values that multiply V.
constexpr float kDefer = 8.f;
constexpr float kLowest = -1e30f;  // a start below every score that keeps exp2(-inf - m) at zero where a query sees nothing yet

// The 32 keys in rows 32 half .. of a tile, key k0 first.
template <typename TR, int D>
__device__ __forceinline__ void fwd_half(const WindowAttnArgs& p, const char* ks, const char* vs, const s16x8 (&qf)[2][D / 32], f32x4 (&o)[2][D / 16],
                                         float (&m)[2], f32x4 (&lsum)[2], int half, int k0, int qw, int border, int lane) {
  const float c = p.scale_log2;
  f32x4 s[2][2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int st = 0; st < 2; ++st) s[st][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) {
      const s16x8 kf = row_frag<D>(ks, 2 * half + t, kk, lane);
#pragma unroll
      for (int st = 0; st < 2; ++st) s[st][t] = mfma<TR>(kf, qf[st][kk], s[st][t]);
    }
  }
  hide_keys(p, s, qw, k0, border, lane);
  float mx[2];
#pragma unroll
  for (int st = 0; st < 2; ++st) {
    mx[st] = s[st][0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mx[st] = fmaxf(mx[st], s[st][i >> 2][i & 3]);
    mx[st] *= c;  // c > 0
  }
  if (__any(mx[0] > m[0] + kDefer || mx[1] > m[1] + kDefer)) {
    // Rare.  The rescale is done in place, as assembly: as plain products the accumulators would get new registers here, and every pass that
    // does NOT come this way would pay 42 moves a strip to reconcile the two.  The assembly waits out the matrix pipe itself.
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const float mg = groups_max(mx[st]);
      const float m_new = mg > m[st] + kDefer ? mg : m[st];
      const float alpha = __builtin_amdgcn_exp2f(m[st] - m_new);
      m[st] = m_new;
#pragma unroll
      for (int td = 0; td < D / 16; ++td)
#pragma unroll
        for (int e = 0; e < 4; ++e) asm volatile("v_mul_f32 %0, %0, %1" : "+v"(o[st][td][e]) : "v"(alpha));
#pragma unroll
      for (int e = 0; e < 4; ++e) asm volatile("v_mul_f32 %0, %0, %1" : "+v"(lsum[st][e]) : "v"(alpha));
    }
    asm volatile("s_nop 4" ::: "memory");  // and the products leave the vector pipe before a matrix instruction reads them
  }
  s16x8 pf[2];
#pragma unroll
  for (int st = 0; st < 2; ++st) {
    const float nm = -m[st];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[st][i >> 2][i & 3] = __builtin_amdgcn_exp2f(fmaf(s[st][i >> 2][i & 3], c, nm));
    pf[st] = pack8<TR>(s[st][0], s[st][1]);
  }
  const short one = std::is_same<TR, F16>::value ? 0x3C00 : 0x3F80;
  const s16x8 ones = {one, one, one, one, one, one, one, one};
#pragma unroll
  for (int st = 0; st < 2; ++st) lsum[st] = mfma<TR>(ones, pf[st], lsum[st]);
#pragma unroll
  for (int td = 0; td < D / 16; ++td) {
    const s16x8 vf = tr_frag<D>(vs, 32 * half, td, lane);
#pragma unroll
    for (int st = 0; st < 2; ++st) o[st][td] = mfma<TR>(vf, pf[st], o[st][td]);
  }
}

// Workgroup -> (batch, query head, query block): the heads of a group next to each other, then the blocks, the long ones first.
__device__ __forceinline__ void query_item(const WindowAttnArgs& p, int& b, int& h, int& qb) {
  const int G = p.H / p.KV, nqb = (p.T + kRows - 1) / kRows;
  const int v = xcd_order(blockIdx.x, gridDim.x);
  const int per_kv = nqb * G, bk = v / per_kv, rest = v - bk * per_kv;
  b = bk / p.KV;
  h = (bk - b * p.KV) * G + rest % G;
  qb = nqb - 1 - rest / G;
}

template <typename TR, int D>
__global__ __launch_bounds__(kThreads, D == 64 ? 4 : 2) void window_fwd_kernel(WindowAttnArgs p) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];  // [stages][K | V], then the output strips
  constexpr int TB = kTileBytes<D>, NP = TileSource<D>::kPieces;
  int b, h, qb;
  query_item(p, b, h, qb);
  const int q0 = qb * kRows, len = length_of(p, b);
  const long long o_stride = static_cast<long long>(p.H) * D;
  u16* out = static_cast<u16*>(p.o) + static_cast<long long>(b) * p.T * o_stride + static_cast<long long>(h) * D;
  if (q0 >= len) {
    zero_rows<D>(out, o_stride, q0, p.T);
    return;
  }
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, li = lane & 15, qw = q0 + wid * 32;
  const u16* base = static_cast<const u16*>(p.qkv) + static_cast<long long>(b) * p.batch_stride;
  const u16* Q = base + static_cast<long long>(h) * D;
  const int kv = h / (p.H / p.KV);
  const bool moves_v = wid >= 2;
  const u16* src = base + static_cast<long long>(p.H + kv + (moves_v ? p.KV : 0)) * D;
  const KeyTiles tiles(p, q0, len);
  TileSource<D> ts;
  ts.init(p.row_stride, (wid & 1) * NP, lane);
  const unsigned dst = lds_address(smem) + (moves_v ? TB : 0) + (wid & 1) * NP * 1024;
  auto request = [&](int it, int stage) {
    const int k0 = tiles.key0(it);
    ts.request(src + static_cast<long long>(k0) * p.row_stride, tiles.valid(p, it, len), dst + stage * 2 * TB);
  };
  request(0, 0);
  s16x8 qf[2][D / 32];
#pragma unroll
  for (int st = 0; st < 2; ++st) {
    const int qi = qw + 16 * st + li < len ? qw + 16 * st + li : len - 1;
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) qf[st][kk] = *reinterpret_cast<const s16x8*>(Q + static_cast<long long>(qi) * p.row_stride + 32 * kk + 8 * g);
  }
  f32x4 o[2][D / 16], lsum[2];
  float m[2] = {kLowest, kLowest};
#pragma unroll
  for (int st = 0; st < 2; ++st) {
    lsum[st] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int td = 0; td < D / 16; ++td) o[st][td] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  wait_vmem_at_most<0>();
  int stage = 0;
  for (int it = 0; it < tiles.count; ++it) {
    wait_vmem_at_most<0>();  // this wave's pieces of the tile have landed
    __syncthreads();         // everybody's have; nobody still reads the other stage
    if (it + 1 < tiles.count) request(it + 1, stage ^ 1);
    const char* ks = smem + stage * 2 * TB;
    const int key0 = tiles.key0(it);
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      const int k0 = key0 + 32 * half, border = border_of(p, qw, k0);
      if (border != kUnseen) fwd_half<TR, D>(p, ks, ks + TB, qf, o, m, lsum, half, k0, qw, border, lane);
    }
    stage ^= 1;
  }
  float inv[2];
#pragma unroll
  for (int st = 0; st < 2; ++st) {
    const float l = lsum[st][0];  // every accumulator row holds the sum for this lane's query
    inv[st] = 1.f / l;
    const int qi = qw + 16 * st + li;
    if (p.lse2 && g == 0 && qi < len) p.lse2[(static_cast<long long>(b) * p.H + h) * p.T + qi] = m[st] + log2f(l);
  }
  __syncthreads();  // tile stages -> output strips
  store_rows<TR, D>(smem + wid * kStripBytes<D>, o, inv, out, o_stride, qw, len, p.T, lane);
}

// ---------------------------------------------------------------------------------------------------- backward: dQ
template <typename TR, int D>
__device__ __forceinline__ void dq_half(const WindowAttnArgs& p, const char* ks, const char* vs, const s16x8 (&qf)[2][D / 32], const s16x8 (&dof)[2][D / 32],
                                        f32x4 (&dq)[2][D / 16], const float (&lse2)[2], const f32x4 (&minus_delta)[2], int half, int k0, int qw, int border, int lane) {
  const float c = p.scale_log2;
  f32x4 s[2][2], dp[2][2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      s[st][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      dp[st][t] = minus_delta[st];  // dp - delta without a subtraction per score
    }
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) {
      const s16x8 kf = row_frag<D>(ks, 2 * half + t, kk, lane), vf = row_frag<D>(vs, 2 * half + t, kk, lane);
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        s[st][t] = mfma<TR>(kf, qf[st][kk], s[st][t]);
        dp[st][t] = mfma<TR>(vf, dof[st][kk], dp[st][t]);
      }
    }
  }
  hide_keys(p, s, qw, k0, border, lane);
  s16x8 dsf[2];
#pragma unroll
  for (int st = 0; st < 2; ++st) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = i >> 2, e = i & 3;
      const float pe = __builtin_amdgcn_exp2f(fmaf(s[st][t][e], c, -lse2[st]));
      s[st][t][e] = pe * dp[st][t][e];  // the softmax scale is applied once, to the finished rows
    }
    dsf[st] = pack8<TR>(s[st][0], s[st][1]);
  }
#pragma unroll
  for (int td = 0; td < D / 16; ++td) {
    const s16x8 kt = tr_frag<D>(ks, 32 * half, td, lane);
#pragma unroll
    for (int st = 0; st < 2; ++st) dq[st][td] = mfma<TR>(kt, dsf[st], dq[st][td]);
  }
}

template <typename TR, int D>
__global__ __launch_bounds__(kThreads, D == 64 ? 3 : 2) void window_dq_kernel(WindowAttnArgs p) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  constexpr int TB = kTileBytes<D>, NP = TileSource<D>::kPieces;
  int b, h, qb;
  query_item(p, b, h, qb);
  const int q0 = qb * kRows, len = length_of(p, b);
  const long long g_stride = static_cast<long long>(p.H + 2 * p.KV) * D, o_stride = static_cast<long long>(p.H) * D;
  u16* out = static_cast<u16*>(p.dqkv) + static_cast<long long>(b) * p.T * g_stride + static_cast<long long>(h) * D;
  if (q0 >= len) {
    zero_rows<D>(out, g_stride, q0, p.T);
    return;
  }
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, li = lane & 15, qw = q0 + wid * 32;
  const u16* base = static_cast<const u16*>(p.qkv) + static_cast<long long>(b) * p.batch_stride;
  const u16* Q = base + static_cast<long long>(h) * D;
  const int kv = h / (p.H / p.KV);
  const bool moves_v = wid >= 2;
  const u16* src = base + static_cast<long long>(p.H + kv + (moves_v ? p.KV : 0)) * D;
  const KeyTiles tiles(p, q0, len);
  TileSource<D> ts;
  ts.init(p.row_stride, (wid & 1) * NP, lane);
  const unsigned dst = lds_address(smem) + (moves_v ? TB : 0) + (wid & 1) * NP * 1024;
  auto request = [&](int it, int stage) {
    const int k0 = tiles.key0(it);
    ts.request(src + static_cast<long long>(k0) * p.row_stride, tiles.valid(p, it, len), dst + stage * 2 * TB);
  };
  request(0, 0);
  const long long ho = static_cast<long long>(b) * p.T * o_stride + static_cast<long long>(h) * D;
  const u16* O = static_cast<const u16*>(p.o) + ho;
  const u16* DO = static_cast<const u16*>(p.d_o) + ho;
  const long long stat = (static_cast<long long>(b) * p.H + h) * p.T;
  s16x8 qf[2][D / 32], dof[2][D / 32];
  float lse2[2];
  f32x4 minus_delta[2];
#pragma unroll
  for (int st = 0; st < 2; ++st) {
    const bool live = qw + 16 * st + li < len;
    const long long qi = live ? qw + 16 * st + li : len - 1;
    float part = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) {
      qf[st][kk] = *reinterpret_cast<const s16x8*>(Q + qi * p.row_stride + 32 * kk + 8 * g);
      dof[st][kk] = *reinterpret_cast<const s16x8*>(DO + qi * o_stride + 32 * kk + 8 * g);
      const s16x8 of = *reinterpret_cast<const s16x8*>(O + qi * o_stride + 32 * kk + 8 * g);
#pragma unroll
      for (int j = 0; j < 8; ++j) part = fmaf(TR::to_f32(static_cast<u16>(dof[st][kk][j])), TR::to_f32(static_cast<u16>(of[j])), part);
    }
    lse2[st] = p.lse2[stat + qi];
    const float delta = groups_sum(part);  // the four lane groups hold D / 4 values each
    minus_delta[st] = f32x4{-delta, -delta, -delta, -delta};
    if (g == 0 && live) p.delta[stat + qi] = -delta;  // as the dK/dV kernel wants it
  }
  f32x4 dq[2][D / 16];
#pragma unroll
  for (int st = 0; st < 2; ++st)
#pragma unroll
    for (int td = 0; td < D / 16; ++td) dq[st][td] = f32x4{0.f, 0.f, 0.f, 0.f};
  wait_vmem_at_most<0>();
  int stage = 0;
  for (int it = 0; it < tiles.count; ++it) {
    wait_vmem_at_most<0>();
    __syncthreads();
    if (it + 1 < tiles.count) request(it + 1, stage ^ 1);
    const char* ks = smem + stage * 2 * TB;
    const int key0 = tiles.key0(it);
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      const int k0 = key0 + 32 * half, border = border_of(p, qw, k0);
      if (border != kUnseen) dq_half<TR, D>(p, ks, ks + TB, qf, dof, dq, lse2, minus_delta, half, k0, qw, border, lane);
    }
    stage ^= 1;
  }
  __syncthreads();
  const float by_scale[2] = {p.scale, p.scale};
  store_rows<TR, D>(smem + wid * kStripBytes<D>, dq, by_scale, out, g_stride, qw, len, p.T, lane);
}

// ---------------------------------------------------------------------------------------------------- backward: dK, dV
// Units of one (batch, key / value head): key block kb (128 keys) meets the query tiles (64 queries) 2 kb .. 2 kb + tiles(kb) - 1 of each
// of the G heads of its group; its units are numbered head by head.
struct Units {
  int T, window, sinks, G, n_tiles, n_blocks;
  int by_window;   // query tiles that a window reaches from a block, its own two among them
  int sink_blocks;
  __host__ __device__ Units(int T_, int window_, int sinks_, int G_) : T(T_), window(window_), sinks(sinks_), G(G_) {
    n_tiles = (T + kTile - 1) / kTile;
    n_blocks = (T + kRows - 1) / kRows;
    by_window = static_cast<int>((static_cast<long long>(kRows) + window - 2) / kTile) + 1;
    sink_blocks = (sinks + kRows - 1) / kRows;
    if (sink_blocks > n_blocks) sink_blocks = n_blocks;
  }
  __host__ __device__ int tiles(int kb) const {
    const int left = n_tiles - 2 * kb;
    return kb < sink_blocks || left < by_window ? left : by_window;
  }
  __host__ __device__ long long before(int kb) const {  // units of the blocks in front of kb
    const long long s = kb < sink_blocks ? kb : sink_blocks, w = kb - s;
    long long n = s * n_tiles - s * (s - 1);
    if (w > 0) {
      // blocks s .. kb - 1: by_window tiles each until fewer are left, from block `cut` on
      long long cut = n_tiles - by_window >= 0 ? (n_tiles - by_window) / 2 + 1 : 0;
      cut = cut < s ? s : cut > kb ? kb : cut;
      n += (cut - s) * by_window;
      n += (kb - cut) * n_tiles - (static_cast<long long>(kb) * (kb - 1) - cut * (cut - 1));
    }
    return n * G;
  }
  __host__ __device__ long long all() const { return before(n_blocks); }
  __host__ __device__ int block_of(long long u) const {  // the block that unit u belongs to
    int lo = 0, hi = n_blocks - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (before(mid) <= u) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }
};

template <int D>
constexpr int kDkdvStageBytes = 2 * kTileBytes<D> + 2 * kTile * 4;  // Q | dO | lse2 | delta
template <int D>
constexpr int kDkdvStages = D == 64 ? 2 : 3;

template <typename TR, int D>
__device__ __forceinline__ void dkdv_half(const WindowAttnArgs& p, const char* qs_, const char* dos_, const char* stats, const s16x8 (&kf)[2][D / 32],
                                          const s16x8 (&vf)[2][D / 32], f32x4 (&dk)[2][D / 16], f32x4 (&dv)[2][D / 16], int half, int q0, int kw,
                                          int len, int border, int lane) {
  // the 32 queries from q0, rows 32 half .. of the stage's tiles, against the wave's 32 keys from kw
  const int g = lane >> 4;
  const float c = p.scale_log2;
  // D = 64: probabilities first, then dP -- the two products' operands and statistics are then not live together, which lets three waves share a
  // SIMD (257 -> 211 us at 64 x 1024 x 12 heads).  D = 128 has one wave a SIMD either way and overlaps the two products instead (275 -> 241 us).
  constexpr bool TOGETHER = D == 128;
  f32x4 s[2][2], dp[2][2];  // register (qs, e): query q0 + 16 qs + 4 g + e
  auto start_dp = [&](int qs) __attribute__((always_inline)) {
    const f32x4 minus_delta = *reinterpret_cast<const f32x4*>(stats + (kTile + 32 * half + 16 * qs + 4 * g) * 4);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) dp[kt][qs] = minus_delta;  // dp - delta without a subtraction per score
  };
  auto step_dp = [&](int qs, int kk) __attribute__((always_inline)) {
    const s16x8 dr = row_frag<D>(dos_, 2 * half + qs, kk, lane);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) dp[kt][qs] = mfma<TR>(dr, vf[kt][kk], dp[kt][qs]);
  };
#pragma unroll
  for (int qs = 0; qs < 2; ++qs) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) s[kt][qs] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (TOGETHER) start_dp(qs);
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) {
      const s16x8 qr = row_frag<D>(qs_, 2 * half + qs, kk, lane);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) s[kt][qs] = mfma<TR>(qr, kf[kt][kk], s[kt][qs]);
      if (TOGETHER) step_dp(qs, kk);
    }
  }
  if (border != kClear) {
    with_border(border, [&](auto b_c) __attribute__((always_inline)) {
      constexpr int BORDER = decltype(b_c)::value;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const int key = kw + 16 * kt + (lane & 15), rel = key - q0 - 4 * g;  // register (qs, e) is query index 16 qs + e against rel
        const bool sink = key < p.sinks;
        const int far = BORDER == kSeveral && sink ? 0x7fffffff : rel + p.window;  // first index beyond the window
        const int end = len - q0 - 4 * g;                                            // first index beyond the sequence
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int i = 16 * (j >> 2) + (j & 3);
          const bool hide = BORDER == kCausal   ? i < rel
                            : BORDER == kWindow ? i >= far
                            : BORDER == kSinks  ? !sink
                                                : i < rel || i >= far || i >= end;
          if (hide) s[kt][j >> 2][j & 3] = kNegInf;
        }
      }
    });
  }
  s16x8 pB[2], dsB[2];
#pragma unroll
  for (int qs = 0; qs < 2; ++qs) {
    const f32x4 l2 = *reinterpret_cast<const f32x4*>(stats + (32 * half + 16 * qs + 4 * g) * 4);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[kt][qs][e] = __builtin_amdgcn_exp2f(fmaf(s[kt][qs][e], c, -l2[e]));
  }
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) pB[kt] = pack8<TR>(s[kt][0], s[kt][1]);
  if (!TOGETHER) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int qs = 0; qs < 2; ++qs) {
      start_dp(qs);
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk) step_dp(qs, kk);
    }
  }
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
    for (int qs = 0; qs < 2; ++qs)
#pragma unroll
      for (int e = 0; e < 4; ++e) dp[kt][qs][e] *= s[kt][qs][e];
    dsB[kt] = pack8<TR>(dp[kt][0], dp[kt][1]);
  }
  if (!TOGETHER) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int td = 0; td < D / 16; ++td) {
    const s16x8 dot = tr_frag<D>(dos_, 32 * half, td, lane), qt = tr_frag<D>(qs_, 32 * half, td, lane);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      dv[kt][td] = mfma<TR>(dot, pB[kt], dv[kt][td]);
      dk[kt][td] = mfma<TR>(qt, dsB[kt], dk[kt][td]);
    }
  }
}

// fp32 partial sums of a cut block: [slot][wave][dk | dv][kt][td][lane] of four values.
template <int D>
constexpr long long kPartialFloats = 2LL * kRows * D;

// Where piece w of the unit list begins.  Equal pieces, but a boundary inside a short block moves to the block's nearer end: a cut costs 128 KiB (D = 64) of
// partial sums written and read, the time of about eight units, and the move at most half a block.  Blocks longer than kShort units -- sinks, wide
// windows, large groups -- and than a quarter of a piece are cut.
constexpr int kShort = 16;
__device__ __forceinline__ long long even_start(const WindowAttnArgs& p, int w) {
  return p.piece_units * w + (w < p.piece_rest ? w : p.piece_rest);
}
__host__ __device__ __forceinline__ bool is_short(const WindowAttnArgs& p, long long units) { return units <= kShort || 4 * units <= p.piece_units; }
struct UnitPlace {  // a unit's (batch, key / value head) and key block
  long long bk, start;
  int kb, units;
  __device__ __forceinline__ UnitPlace(const WindowAttnArgs& p, const Units& u, long long s) {
    bk = s < (1ll << 32) && p.units_per_head < (1ll << 32) ? static_cast<unsigned>(s) / static_cast<unsigned>(p.units_per_head) : s / p.units_per_head;
    kb = u.block_of(s - bk * p.units_per_head);
    start = bk * p.units_per_head + u.before(kb);
    units = u.tiles(kb) * u.G;
  }
};
__device__ __forceinline__ long long piece_start(const WindowAttnArgs& p, const Units& u, int w) {
  const long long s = even_start(p, w);
  if (w == 0 || w == p.pieces) return s;
  const UnitPlace at(p, u, s);
  if (!is_short(p, at.units)) return s;
  return 2 * (s - at.start) < at.units ? at.start : at.start + at.units;
}

// A key block of the unit list and the part of it that belongs to a piece.
struct Part {
  int b, kv, kb;
  long long start, stop;  // the block's units
  int len, n, ne;         // sequence length; query tiles per head at full length, and those that hold anything
  int ua, left;           // the part's first unit in the block; how many of its units are walked (those with a tile index below ne)
  __device__ __forceinline__ void open(const WindowAttnArgs& p, const Units& units, long long u0, long long u1) {
    len = length_of(p, b);
    n = units.tiles(kb);
    stop = start + static_cast<long long>(n) * units.G;
    ne = (len + kTile - 1) / kTile - 2 * kb;
    ne = ne < 0 ? 0 : ne < n ? ne : n;
    ua = u0 > start ? static_cast<int>(u0 - start) : 0;
    const int ub = stop <= u1 ? n * units.G : static_cast<int>(u1 - start);
    left = walked(ub, units.G) - walked(ua, units.G);
  }
  __device__ __forceinline__ int walked(int x, int G) const {
    if (x == 0) return 0;
    if (x == n * G) return ne * G;
    const int q = x / n, r = x - q * n;
    return q * ne + (r < ne ? r : ne);
  }
  __device__ __forceinline__ void next(const WindowAttnArgs& p, const Units& units, long long u0, long long u1) {
    start = stop;
    if (++kb == units.n_blocks) {
      kb = 0;
      if (++kv == p.KV) {
        kv = 0;
        ++b;
      }
    }
    open(p, units, u0, u1);
  }
};

// A piece is walked as one stream: the requests run one unit (two at head size 128) ahead of the products, across the end of a block into the next one, and the
// next block's K and V rows are fetched while the finished one is stored (18 KiB of LDS of its own for that), so only a piece's first
// block waits for memory.  (Starting every block by itself -- unit arithmetic with 64-bit divisions, requests, K / V, two trips to memory --
// cost about as much as 4 of its 6 units at a window of 256.)
template <typename TR, int D>
__global__ __launch_bounds__(kThreads, D == 64 ? 3 : 1) void window_dkdv_kernel(WindowAttnArgs p) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];  // [stages][Q | dO | lse2 | delta] | output strips
  constexpr int S = kDkdvStages<D>, TB = kTileBytes<D>, SB = kDkdvStageBytes<D>, NP = TileSource<D>::kPieces;
  const int G = p.H / p.KV;
  const Units units(p.T, p.window, p.sinks, G);
  const int piece = xcd_order(blockIdx.x, p.pieces);
  const long long u0 = piece_start(p, units, piece), u1 = piece_start(p, units, piece + 1);
  if (u0 >= u1) return;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, li = lane & 15;
  const long long o_stride = static_cast<long long>(p.H) * D, g_stride = static_cast<long long>(p.H + 2 * p.KV) * D;
  const bool moves_do = wid >= 2, moves_stat = (wid & 1) == 0;
  TileSource<D> ts;
  ts.init(moves_do ? o_stride : p.row_stride, (wid & 1) * NP, lane);
  const unsigned lds0 = lds_address(smem);
  const unsigned dst = lds0 + (moves_do ? TB : 0) + (wid & 1) * NP * 1024;
  const unsigned stat_dst = lds0 + 2 * TB + (moves_do ? kTile * 4 : 0);
  char* const strip = smem + S * SB + wid * kStripBytes<D>;

  Part cp;  // the part being multiplied
  {
    const UnitPlace at(p, units, u0);
    cp.b = static_cast<int>(at.bk / p.KV);
    cp.kv = static_cast<int>(at.bk - static_cast<long long>(cp.b) * p.KV);
    cp.kb = at.kb;
    cp.start = at.start;
    cp.open(p, units, u0, u1);
  }
  Part rp = cp;  // the part being requested, with the head of the group and the tile that come next
  int rg = rp.ua / rp.n, rt = rp.ua - rg * rp.n;
  auto tile_in_part = [](const Part& q, int& head, int& tile) {  // a unit beyond the sequence: the next head's first
    if (tile >= q.ne) {
      tile = 0;
      ++head;
    }
  };
  tile_in_part(rp, rg, rt);
  int ahead = 0, fill = 0;  // units requested and not multiplied yet; stage that is filled next
  auto request = [&]() __attribute__((always_inline)) {
    while (rp.left == 0) {
      if (rp.stop >= u1) return;
      rp.next(p, units, u0, u1);
      rg = rt = 0;
    }
    const int row = (2 * rp.kb + rt) * kTile, h = rp.kv * G + rg;
    const u16* src = moves_do ? static_cast<const u16*>(p.d_o) + (static_cast<long long>(rp.b) * p.T + row) * o_stride + static_cast<long long>(h) * D
                              : static_cast<const u16*>(p.qkv) + static_cast<long long>(rp.b) * p.batch_stride +
                                    static_cast<long long>(row) * p.row_stride + static_cast<long long>(h) * D;
    ts.request(src, rp.len - row, dst + fill * SB);
    if (moves_stat) {
      const float* st = (moves_do ? p.delta : p.lse2) + (static_cast<long long>(rp.b) * p.H + h) * p.T + row;
      const int i = lane < rp.len - row ? lane : rp.len - row - 1;
      dma_4B(uniform_ptr(st), static_cast<unsigned>(i) * 4u, stat_dst + fill * SB);
    }
    if (++rt == rp.ne) {
      rt = 0;
      ++rg;
    }
    --rp.left;
    ++ahead;
    fill = fill + 1 == S ? 0 : fill + 1;
  };
  s16x8 kf[2][D / 32], vf[2][D / 32];
  auto load_kv = [&](const Part& q) __attribute__((always_inline)) {
    const u16* K = static_cast<const u16*>(p.qkv) + static_cast<long long>(q.b) * p.batch_stride + static_cast<long long>(p.H + q.kv) * D;
    const u16* V = K + static_cast<long long>(p.KV) * D;
    const int kw = q.kb * kRows + wid * 32;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const long long key = kw + 16 * kt + li < q.len ? kw + 16 * kt + li : (q.len > 0 ? q.len - 1 : 0);
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk) {
        kf[kt][kk] = *reinterpret_cast<const s16x8*>(K + key * p.row_stride + 32 * kk + 8 * g);
        vf[kt][kk] = *reinterpret_cast<const s16x8*>(V + key * p.row_stride + 32 * kk + 8 * g);
      }
    }
  };
  for (int i = 0; i < S - 1; ++i) request();
  load_kv(cp);
  int stage = 0;
  bool stored_whole = false;  // the last part left exactly kStores stores per wave behind its K / V loads
  constexpr int kStores = 2 * 32 / (64 / (D / 8));

  while (true) {
    const int kw = cp.kb * kRows + wid * 32, len = cp.len;
    f32x4 dk[2][D / 16], dv[2][D / 16];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int td = 0; td < D / 16; ++td) dk[kt][td] = dv[kt][td] = f32x4{0.f, 0.f, 0.f, 0.f};
    int ct = cp.ua - (cp.ua / cp.n) * cp.n;  // tile being multiplied
    if (ct >= cp.ne) ct = 0;
    for (int it = 0; it < cp.left; ++it) {
      // This wave's pieces of the unit have landed.  A part's first unit is older than its K / V loads; behind those only the stores of the part before.
      if (it == 0) {
        if (stored_whole) wait_vmem_at_most<kStores>();
        else wait_vmem_at_most<0>();
      } else if (ahead > 1) {
        if (moves_stat) wait_vmem_at_most<NP + 1>();
        else wait_vmem_at_most<NP>();
      } else {
        wait_vmem_at_most<0>();
      }
      __syncthreads();  // everybody's have; nobody still reads the stage that is filled next
      --ahead;
      request();
      const char* qs = smem + stage * SB;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int q0 = (2 * cp.kb + ct) * kTile + 32 * half;
        // as border_of, with the 32 queries and the wave's keys in each other's place, and the end of the sequence as one more border
        const bool past = q0 + 31 >= kw + p.window && kw + 31 >= p.sinks, gone = q0 >= kw + 31 + p.window;
        if (q0 + 31 < kw || (past && gone && kw >= p.sinks) || q0 >= len) continue;
        const bool future = q0 < kw + 31, ends = q0 + 31 >= len;
        const int border = ends ? kSeveral : !past ? (future ? kCausal : kClear) : gone ? kSinks : future || kw < p.sinks ? kSeveral : kWindow;
        dkdv_half<TR, D>(p, qs, qs + TB, qs + 2 * TB, kf, vf, dk, dv, half, q0, kw, len, border, lane);
      }
      if (++ct == cp.ne) ct = 0;
      stage = stage + 1 == S ? 0 : stage + 1;
    }
    const Part done = cp;
    const bool last = cp.stop >= u1;
    if (!last) {
      cp.next(p, units, u0, u1);
      load_kv(cp);
    }
    stored_whole = false;
    if (done.ua == 0 && done.stop <= u1) {
      u16* out = static_cast<u16*>(p.dqkv) + static_cast<long long>(done.b) * p.T * g_stride + static_cast<long long>(p.H + done.kv) * D;
      const float by_scale[2] = {p.scale, p.scale}, one[2] = {1.f, 1.f};
      store_rows<TR, D>(strip, dk, by_scale, out, g_stride, kw, len, p.T, lane);
      store_rows<TR, D>(strip, dv, one, out + static_cast<long long>(p.KV) * D, g_stride, kw, len, p.T, lane);
      stored_whole = kw + 32 <= p.T;
    } else {
      // slot 0: the block began in an earlier piece; slot 1: it began here
      f32x4* ws = reinterpret_cast<f32x4*>(p.partial + (2LL * piece + (done.ua == 0 ? 1 : 0)) * kPartialFloats<D>) + wid * (4 * (D / 16) * 64) + lane;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int td = 0; td < D / 16; ++td) {
          ws[(kt * (D / 16) + td) * 64] = dk[kt][td];
          ws[((2 + kt) * (D / 16) + td) * 64] = dv[kt][td];
        }
    }
    if (last) return;
  }
}

// Adds up the partial sums of a long block, if it was cut: blockIdx.x numbers the long blocks (the first p.cuts of every head).  blockIdx.y: the
// part of the block that was wave y / 2's, dK (y even) or dV; a wave here takes a quarter of the columns.
template <typename TR, int D>
__global__ __launch_bounds__(kThreads) void window_join_kernel(WindowAttnArgs p) {
  const Units units(p.T, p.window, p.sinks, p.H / p.KV);
  const int bk = blockIdx.x / p.cuts, kb = blockIdx.x - bk * p.cuts, b = bk / p.KV, kv = bk - b * p.KV;
  const long long start = bk * p.units_per_head + units.before(kb), stop = start + static_cast<long long>(units.tiles(kb)) * units.G;
  // the first piece that begins behind the block's first unit
  int w = static_cast<int>(start / (p.piece_units + 1));
  while (even_start(p, w) <= start) ++w;
  if (even_start(p, w) >= stop) return;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, g = lane >> 4, li = lane & 15;
  const int owner = blockIdx.y >> 1, is_dv = blockIdx.y & 1;
  const int len = length_of(p, b), kw = kb * kRows + owner * 32;
  constexpr int Q = D / 64;  // 16-column tiles per wave
  f32x4 sum[2][Q];
  auto add = [&](int piece, int slot, bool first) {
    const f32x4* ws = reinterpret_cast<const f32x4*>(p.partial + (2LL * piece + slot) * kPartialFloats<D>) + owner * (4 * (D / 16) * 64) + lane;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const f32x4 a = ws[((2 * is_dv + kt) * (D / 16) + wid * Q + q) * 64];
        sum[kt][q] = first ? a : sum[kt][q] + a;
      }
  };
  add(w - 1, 1, true);
#pragma unroll 4
  for (int piece = w; piece < p.pieces && even_start(p, piece) < stop; ++piece) add(piece, 0, false);
  const long long g_stride = static_cast<long long>(p.H + 2 * p.KV) * D;
  u16* out = static_cast<u16*>(p.dqkv) + static_cast<long long>(b) * p.T * g_stride + static_cast<long long>(p.H + kv + is_dv * p.KV) * D;
  const float scale = is_dv ? 1.f : p.scale;
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const int key = kw + 16 * kt + li;
    if (key >= p.T) continue;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      u16x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = key < len ? TR::from_f32(sum[kt][q][e] * scale) : static_cast<u16>(0);
      *reinterpret_cast<u16x4*>(out + key * g_stride + 16 * (wid * Q + q) + 4 * g) = v;
    }
  }
}

// More than 64 KiB of dynamic LDS has to be asked for.
template <typename Kernel>
void allow_lds(Kernel k, int bytes) {
  if (bytes > 65536) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <int D>
constexpr int kQueryLds = 4 * kTileBytes<D>;  // [2 stages][K | V]
static_assert(4 * kStripBytes<64> <= kQueryLds<64> && 4 * kStripBytes<128> <= kQueryLds<128>, "the output strips reuse the tiles' memory");
template <int D>
constexpr int kDkdvLds = kDkdvStages<D> * kDkdvStageBytes<D> + 4 * kStripBytes<D>;

template <typename F>
void dispatch(int dtype, int D, F&& f) {
  if (dtype == kBF16) {
    if (D == 64) f(BF16{}, std::integral_constant<int, 64>{});
    else f(BF16{}, std::integral_constant<int, 128>{});
  } else {
    if (D == 64) f(F16{}, std::integral_constant<int, 64>{});
    else f(F16{}, std::integral_constant<int, 128>{});
  }
}

long long query_items(const WindowAttnArgs& a) { return static_cast<long long>(a.B) * a.H * ((a.T + kRows - 1) / kRows); }

}  // namespace

bool window_attention_supported(long long B, long long T, long long H, long long KV, long long D, long long row_stride, int dtype) {
  if (!(dtype == kBF16 || dtype == kF16) || !(D == 64 || D == 128)) return false;
  if (B < 0 || T < 0 || H < 1 || KV < 1 || H % KV != 0) return false;
  if (T > (1ll << 30) || row_stride % 8 != 0 || row_stride >= (1ll << 24) || (H + 2 * KV) * D >= (1ll << 24)) return false;  // a tile's byte offsets are 32-bit
  return B * H * ((T + kRows - 1) / kRows) < (1ll << 24);  // a launch counts its threads in 32 bits
}

// One piece per workgroup that the chip holds at once; at least a unit each, or four where blocks are long enough to be cut.
void window_attention_plan(WindowAttnArgs& a) {
  const Units units(a.T, a.window, a.sinks, a.H / a.KV);
  a.units_per_head = units.all();
  const long long total = a.units_per_head * a.KV * a.B;
  long long n = a.compute_units * (a.D == 64 ? 3 : 1);
  const long long most = units.tiles(0) * units.G <= kShort ? total : total / 4;  // (no block is longer than the first)
  if (n > most) n = most;
  a.pieces = static_cast<int>(n < 1 ? 1 : n);
  a.piece_units = total / a.pieces;
  a.piece_rest = static_cast<int>(total % a.pieces);
  a.cuts = 0;  // blocks get no longer from first to last
  while (a.pieces > 1 && a.cuts < units.n_blocks && !is_short(a, static_cast<long long>(units.tiles(a.cuts)) * units.G)) ++a.cuts;
}
long long window_attention_partial_floats(const WindowAttnArgs& a) { return a.cuts ? 2LL * a.pieces * 2 * kRows * a.D : 0; }

void launch_window_attention_fwd(const WindowAttnArgs& args, int dtype, hipStream_t stream) {
  WindowAttnArgs a = args;
  if (a.B == 0 || a.T == 0) return;
  a.scale_log2 = a.scale * kLog2e;
  const dim3 grid(static_cast<unsigned>(query_items(a)));
  dispatch(dtype, a.D, [&](auto tr, auto d) {
    constexpr int D = decltype(d)::value;
    auto k = window_fwd_kernel<decltype(tr), D>;
    allow_lds(k, kQueryLds<D>);
    hipLaunchKernelGGL(k, grid, dim3(kThreads), kQueryLds<D>, stream, a);
  });
}

void launch_window_attention_bwd(const WindowAttnArgs& args, int dtype, hipStream_t stream) {
  WindowAttnArgs a = args;
  if (a.B == 0 || a.T == 0) return;
  a.scale_log2 = a.scale * kLog2e;
  const dim3 grid(static_cast<unsigned>(query_items(a)));
  dispatch(dtype, a.D, [&](auto tr, auto d) {
    constexpr int D = decltype(d)::value;
    using TR = decltype(tr);
    auto dq = window_dq_kernel<TR, D>;
    auto dkdv = window_dkdv_kernel<TR, D>;
    auto join = window_join_kernel<TR, D>;
    allow_lds(dq, kQueryLds<D>);
    allow_lds(dkdv, kDkdvLds<D>);
    hipLaunchKernelGGL(dq, grid, dim3(kThreads), kQueryLds<D>, stream, a);
    hipLaunchKernelGGL(dkdv, dim3(static_cast<unsigned>(a.pieces)), dim3(kThreads), kDkdvLds<D>, stream, a);
    if (a.cuts) hipLaunchKernelGGL(join, dim3(static_cast<unsigned>(a.B) * a.KV * a.cuts, 8), dim3(kThreads), 0, stream, a);
  });
}

}  // namespace kernels
}  // namespace dpa
