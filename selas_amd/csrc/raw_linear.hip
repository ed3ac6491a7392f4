// Linear with an unquantized weight and the block's epilogue, on gfx950:
//   y[b, l, n] = residual[b, l, n] + gate[b, n] * act(sum_k x[b, l, k] w[n, k] + bias[n])
// with act(..) clamped to the fp16 range where the fp16 guard is on.
//
// UnitView.linear for raw weights (selas/store.py:289-293) together with what follows
// it in a block: the GELU or SiLU (flux.py:150-151, 194-195) and the gated residual add
// (flux.py:169-171). The sum, the activation, the gate and the residual stay in fp32 and
// are rounded once, to the output's type.
//
// 2 M N K operations against the operands and the output moved once (eo bytes per output): products of 32 or fewer rows or 64
// or fewer columns are bound by HBM and run in kernels that stream the large operand (raw_stream_kernel, raw_few_kernel);
// the others are tiles of MFMAs (raw_tile_kernel), with K in ranges where the tiles leave CUs idle (raw_merge_kernel adds
// them), and with operands off the DMA's alignment copied first (raw_pack_kernel). Every route adds in a fixed order.
//
// Times below: a large copy reaches 5.1 TB/s on the card, a library product of 8192^3 in bf16 1,590 TFLOP/s.
#include <atomic>

#include "common.h"

namespace selas {
namespace {

// One problem as the kernels see it: rows m = b * L + l in [0, M).
struct RawProblem {
  const void *x, *w, *bias, *gate, *residual;
  void *y;
  int64_t x_sb, x_sl, ldw, gate_sb, r_sb, r_sl, y_sb, y_sl;
  int M, L, N, K;
  FastDiv by_l;
  int act;
  bool bias_f32, gate_f32, residual_f32, y_f32;
  // N is a multiple of 8, bias, gate, residual and y take 16-byte accesses at every 8th column, and the rows of y and
  // of the residual are equally spaced over the batches, a tile of them within 31 bits of bytes.
  bool vec;
  bool one_gate;  // one gate row for all batches
  bool guard;     // the fp16 guard
};

// Four dwords, and the same at the address of any 16-bit element (global accesses may start there).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));

// v_mfma_f32_16x16x32 of two 16-bit fragments: D(16x16) += A(16x32) B(32x16). Lane l supplies A[l % 16][8 (l / 16) ..
// +8] and B[8 (l / 16) .. +8][l % 16] and holds D[4 (l / 16) + r][l % 16] in register r.
template <int DT>
__device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
  if constexpr (DT == SELAS_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

// The same, accumulated in place in accumulation registers. The builtin leaves the compiler free to give the sum
// other registers than the addend; with 256 accumulators it then moves and spills them inside the K loop. The hazards of
// an instruction that the compiler does not know: a is not read by anything but later calls until settle_mfma(), and the
// same a comes again 16 calls (4 in the 128 x 128 tile) later at the earliest.
template <int DT>
__device__ __forceinline__ void mfma16_inplace(uint4 a, uint4 b, f32x4 &c) {
  const u32x4 av = {a.x, a.y, a.z, a.w}, bv = {b.x, b.y, b.z, b.w};
  if constexpr (DT == SELAS_BF16) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(av), "v"(bv));
  else asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(av), "v"(bv));
}
// The products in flight reach their registers.
__device__ __forceinline__ void settle_mfma() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// x / (1 + e^-x) by the hardware base-2 exponential and reciprocal, like gelu_tanh_fast.
__device__ __forceinline__ float silu_fast(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}

__device__ __forceinline__ float activate(float v, int act) {
  return act == SELAS_ACT_GELU ? gelu_tanh_fast(v) : act == SELAS_ACT_SILU ? silu_fast(v) : v;
}

// The activation and the fp16 guard. The sums are fp32, but fp16 inputs may be infinite (a hidden value stored past 65504),
// and an infinite sum would stay in the residual stream.
__device__ __forceinline__ float activate(float v, int act, bool guard) {
  v = activate(v, act);
  return guard ? clamp_guard(v) : v;
}

template <int A, int B>
__device__ __forceinline__ void activate_all(float (&v)[A][B], int act, bool guard) {  // one branch for all
  if (act == SELAS_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < A; ++i)
#pragma unroll
      for (int j = 0; j < B; ++j) v[i][j] = gelu_tanh_fast(v[i][j]);
  } else if (act == SELAS_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < A; ++i)
#pragma unroll
      for (int j = 0; j < B; ++j) v[i][j] = silu_fast(v[i][j]);
  }
  if (guard) {
#pragma unroll
    for (int i = 0; i < A; ++i)
#pragma unroll
      for (int j = 0; j < B; ++j) v[i][j] = clamp_guard(v[i][j]);
  }
}

template <int DT>
__device__ __forceinline__ float load_either(const void *p, int64_t i, bool f32) {
  return f32 ? static_cast<const float *>(p)[i] : load_f<DT>(p, i);
}

// One output from its sum: the epilogue and the store.
template <int DT>
__device__ __forceinline__ void finish_one(const RawProblem &P, int b, int l, int n, float v) {
  if (P.bias) v += load_either<DT>(P.bias, n, P.bias_f32);
  v = activate(v, P.act, P.guard);
  if (P.gate) v *= load_either<DT>(P.gate, b * P.gate_sb + n, P.gate_f32);
  if (P.residual) v = load_either<DT>(P.residual, b * P.r_sb + l * P.r_sl + n, P.residual_f32) + v;
  const int64_t o = b * P.y_sb + l * P.y_sl + n;
  if (P.y_f32) static_cast<float *>(P.y)[o] = v;
  else store_f<DT>(P.y, o, v);
}

// f(integral_constant<int, 0>), ..., f(integral_constant<int, N - 1>): a loop over register arrays that cannot stay rolled.
template <int N, int I = 0, typename F>
__device__ __forceinline__ void for_each_index(F &&f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    for_each_index<N, I + 1>(f);
  }
}

// W consecutive columns of a row as fp32, from 16-byte aligned addresses (8-byte for four 16-bit ones).
template <int DT, int W>
__device__ __forceinline__ void load_cols(const void *p, int64_t i, bool f32, float (&v)[W]) {
  if (f32) {
#pragma unroll
    for (int j = 0; j < W; j += 4) {
      const float4 u = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i + j);
      v[j] = u.x; v[j + 1] = u.y; v[j + 2] = u.z; v[j + 3] = u.w;
    }
  } else {
    uint32_t w[W / 2];
    const uint16_t *q = static_cast<const uint16_t *>(p) + i;
    if constexpr (W == 8) {
      const uint4 u = *reinterpret_cast<const uint4 *>(q);
      w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2 *>(q);
      w[0] = u.x; w[1] = u.y;
    }
#pragma unroll
    for (int t = 0; t < W / 2; ++t) {
      if constexpr (DT == SELAS_BF16) {
        v[2 * t] = __uint_as_float(w[t] << 16);
        v[2 * t + 1] = __uint_as_float(w[t] & 0xffff0000u);
      } else {
        v[2 * t] = f16_bits_to_f32(w[t] & 0xffffu);
        v[2 * t + 1] = f16_bits_to_f32(w[t] >> 16);
      }
    }
  }
}

// W consecutive columns of U rows, row u from element at[u] on, of which the first `live` exist (0 or fewer: none; the
// others repeat the last). Whether all exist is asked for a whole wave and the type for all rows, so that every row's loads
// are in flight before the first one's values are used: asked per row, each row waited for the one before.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
template <int DT, int U, int W>
__device__ __forceinline__ void load_rows_any(const void *p, const int64_t (&at)[U], bool f32, bool whole, int live,
                                              float (&v)[U][W]) {
  const float *const pf = static_cast<const float *>(p);
  const uint16_t *const ph = static_cast<const uint16_t *>(p);
  if (whole && f32) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < W; j += 4) {
        const f32x4 q = *reinterpret_cast<const f32x4_any *>(pf + at[u] + j);
        v[u][j] = q[0]; v[u][j + 1] = q[1]; v[u][j + 2] = q[2]; v[u][j + 3] = q[3];
      }
  } else if (whole) {
    uint32_t w[U][W / 2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < W; j += 4) {
        const auto q = *reinterpret_cast<const u32x2_any *>(ph + at[u] + j);
        w[u][j / 2] = q[0]; w[u][j / 2 + 1] = q[1];
      }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < W / 2; ++t) {
        if constexpr (DT == SELAS_BF16) {
          v[u][2 * t] = __uint_as_float(w[u][t] << 16);
          v[u][2 * t + 1] = __uint_as_float(w[u][t] & 0xffff0000u);
        } else {
          v[u][2 * t] = f16_bits_to_f32(w[u][t] & 0xffffu);
          v[u][2 * t + 1] = f16_bits_to_f32(w[u][t] >> 16);
        }
      }
  } else if (f32) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < W; ++j) v[u][j] = pf[at[u] + min(j, live - 1)];
  } else {
    uint16_t w[U][W];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < W; ++j) w[u][j] = ph[at[u] + min(j, live - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < W; ++j) {
        if constexpr (DT == SELAS_BF16) v[u][j] = __uint_as_float(static_cast<uint32_t>(w[u][j]) << 16);
        else v[u][j] = f16_bits_to_f32(w[u][j]);
      }
  }
}

// W == 4: fp32 outputs; W == 8: 16-bit ones.
template <int DT, int W>
__device__ __forceinline__ void store_cols_any(void *y, int64_t i, int live, const float (&v)[W]) {
  if (live < W) {
#pragma unroll
    for (int j = 0; j < W; ++j)
      if (j < live) {
        if constexpr (W == 4) static_cast<float *>(y)[i + j] = v[j];
        else store_f<DT>(y, i + j, v[j]);
      }
  } else if constexpr (W == 4) {
    *reinterpret_cast<f32x4_any *>(static_cast<float *>(y) + i) = f32x4{v[0], v[1], v[2], v[3]};
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == SELAS_BF16) w[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
      else w[j] = f16_bits_rne(v[2 * j]) | (static_cast<uint32_t>(f16_bits_rne(v[2 * j + 1])) << 16);
    }
    *reinterpret_cast<u32x4_any *>(static_cast<uint16_t *>(y) + i) = u32x4{w[0], w[1], w[2], w[3]};
  }
}

// Four outputs of row (b, l) from column n on, from their sums.
template <int DT>
__device__ __forceinline__ void finish_four(const RawProblem &P, int b, int l, int n, f32x4 s) {
  if (!P.vec) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < P.N) finish_one<DT>(P, b, l, n + j, s[j]);
    return;
  }
  if (n >= P.N) return;
  float v[4] = {s[0], s[1], s[2], s[3]}, u[4];
  if (P.bias) {
    load_cols<DT, 4>(P.bias, n, P.bias_f32, u);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += u[j];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = activate(v[j], P.act, P.guard);
  if (P.gate) {
    load_cols<DT, 4>(P.gate, b * P.gate_sb + n, P.gate_f32, u);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= u[j];
  }
  if (P.residual) {
    load_cols<DT, 4>(P.residual, b * P.r_sb + l * P.r_sl + n, P.residual_f32, u);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = u[j] + v[j];
  }
  const int64_t o = b * P.y_sb + l * P.y_sl + n;
  if (P.y_f32) {
    *reinterpret_cast<float4 *>(static_cast<float *>(P.y) + o) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint2 w;
    if constexpr (DT == SELAS_BF16) {
      w.x = pack_bf16x2(v[0], v[1]);
      w.y = pack_bf16x2(v[2], v[3]);
    } else {
      w.x = f16_bits_rne(v[0]) | (static_cast<uint32_t>(f16_bits_rne(v[1])) << 16);
      w.y = f16_bits_rne(v[2]) | (static_cast<uint32_t>(f16_bits_rne(v[3])) << 16);
    }
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(P.y) + o) = w;
  }
}

// The problem whose outputs are the plain fp32 sums, [M, N] contiguous at `part`: one range of K of a split launch.
__device__ __forceinline__ void to_partial(RawProblem &P, float *part) {
  P.bias = P.gate = P.residual = nullptr;
  P.act = SELAS_ACT_NONE;
  P.guard = false;
  P.y = part;
  P.y_sl = P.N;
  P.y_sb = static_cast<int64_t>(P.L) * P.N;
  P.y_f32 = true;
  P.vec = P.N % 8 == 0;
}

// y = epilogue(sum over the K ranges, in their order): four columns per thread. Bound by the partial sums' reads, from the
// Infinity Cache: 512 x 3072 of 8 ranges with an fp32 residual 11.6 us (63 MB, 5.4 TB/s). A pass of its own, on all CUs.
// Not tried: the last workgroup of a tile to count itself in adds the ranges, in the same order and without anyone waiting.
// That saves the launch; the sums of these 24 tiles would be read by 24 CUs.
template <int DT>
__global__ __launch_bounds__(256) void raw_merge_kernel(RawProblem P, const float *__restrict__ part, int split) {
  const int groups = (P.N + 3) / 4;
  const int64_t size = static_cast<int64_t>(P.M) * P.N;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= static_cast<int64_t>(P.M) * groups) return;
  const int m = static_cast<int>(i / groups), n = static_cast<int>(i - static_cast<int64_t>(m) * groups) * 4;
  const float *src = part + static_cast<int64_t>(m) * P.N + n;
  f32x4 v = {};
  if (P.N % 4 == 0) {
    for (int s = 0; s < split; ++s) v += *reinterpret_cast<const f32x4 *>(src + s * size);
  } else {
    for (int s = 0; s < split; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < P.N) v[j] += src[s * size + j];
  }
  const int b = static_cast<int>(div31(static_cast<uint32_t>(m), P.by_l));
  finish_four<DT>(P, b, m - b * P.L, n, v);
}

// Eight elements of a row from k on, zeros from K on. The address need not be aligned: global loads may start at any
// element.
__device__ __forceinline__ uint4 load_any(const uint16_t *p) {
  return __builtin_bit_cast(uint4, static_cast<u32x4>(*reinterpret_cast<const u32x4_any *>(p)));
}
__device__ __forceinline__ uint4 load_chunk(const uint16_t *row, int k, int K) {
  if (k + 8 <= K) return load_any(row + k);
  uint32_t w[4] = {};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (k + j < K) w[j / 2] |= static_cast<uint32_t>(row[k + j]) << (16 * (j & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// ------------------------------------------------------------------ operands off alignment
//
// The tiled kernel's DMA takes whole 16-byte chunks. An operand whose rows are not made of them (K not a multiple of 8, an
// odd stride or address) or span too much is copied first, to rows of K rounded up to 64 that end in zeros, a thread per
// 16-byte chunk. The copy of 1386 x 667 and 1431 x 667 is 6.3 us (7.6 MB: a launch, and one load's latency), the tiles after
// it 16.3 us with GELU, gate and residual; tiles of 64 x 64 that load such rows through registers took 26 us without it, and
// 4001 x 5999 x 5003 ran at 500 TFLOP/s there against 1,060 (the copy included).
template <int DT>
__global__ __launch_bounds__(256) void raw_pack_kernel(RawProblem P, uint16_t *xp, uint16_t *wp, int kp) {
  const int per_row = kp / 8;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, row = i / per_row;
  const int k = static_cast<int>(i - row * per_row) * 8;
  const int64_t xrows = xp ? P.M : 0;
  if (row >= xrows + (wp ? P.N : 0)) return;
  const uint16_t *src;
  uint16_t *dst;
  if (row < xrows) {
    const int m = static_cast<int>(row), b = static_cast<int>(div31(static_cast<uint32_t>(m), P.by_l));
    src = static_cast<const uint16_t *>(P.x) + b * P.x_sb + (m - b * P.L) * P.x_sl;
    dst = xp + row * kp;
  } else {
    src = static_cast<const uint16_t *>(P.w) + (row - xrows) * P.ldw;
    dst = wp + (row - xrows) * kp;
  }
  *reinterpret_cast<uint4 *>(dst + k) = load_chunk(src, k, P.K);
}

// ------------------------------------------------------------------ few rows
//
// One operand of at most 64 rows (x of a modulation or an embedding; the weight of the final layer): HBM-bound by the
// other, the streamed one. A workgroup takes NT x 16 of its rows; its 8 waves share K in ranges, each lane loading 16
// bytes of row lane % 16 straight into the fragments of v_mfma_f32_16x16x32 (two loads cover a 128-byte line), and the
// few rows' fragments from the caches. The waves' sums are added in LDS, in wave order.
// SWAP: x is the streamed operand.
//
// A workgroup reads the few rows again for its 16 or 32 streamed ones (28 x 18432 x 3072: 576 workgroups, 99 MB from the
// caches beside the weight's 113 MB), and 16 adjacent lanes load from 16 rows: rows that the DMA could read take 36 us here,
// rows of the weight that start at odd elements 81.
constexpr int kFewWaves = 8;

// The epilogue of the kernels for few rows: the waves' sums red[wave][few row][streamed row] are added in wave order, a
// thread per four adjacent columns n of a row m.
template <int DT, int NT, int MT, bool SWAP, int WAVES>
__device__ __forceinline__ void finish_few(const RawProblem &P, int r0, const float *red) {
  constexpr int BIG = NT * 16, FEW = MT * 16, LD = BIG + 4;
  constexpr int ROWS = SWAP ? BIG : FEW, COLS = SWAP ? FEW : BIG;
  for (int i = threadIdx.x; i < ROWS * COLS / 4; i += 64 * WAVES) {
    const int rm = i / (COLS / 4), cn = i % (COLS / 4) * 4;
    const int m = (SWAP ? r0 : 0) + rm, n = (SWAP ? 0 : r0) + cn;
    if (m >= P.M || n >= P.N) continue;
    f32x4 v = {};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float *p = red + w * FEW * LD;
      if constexpr (SWAP) v += f32x4{p[cn * LD + rm], p[(cn + 1) * LD + rm], p[(cn + 2) * LD + rm], p[(cn + 3) * LD + rm]};
      else v += *reinterpret_cast<const f32x4 *>(p + rm * LD + cn);
    }
    const int b = static_cast<int>(div31(static_cast<uint32_t>(m), P.by_l));
    finish_four<DT>(P, b, m - b * P.L, n, v);
  }
}

template <int DT, int NT, int MT, bool SWAP>
__global__ __launch_bounds__(64 * kFewWaves) void raw_few_kernel(RawProblem P, float *part, int split) {
  constexpr int BIG = NT * 16, FEW = MT * 16, LD = BIG + 4, U = 4;
  __shared__ float red[kFewWaves][FEW][LD];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r0 = blockIdx.x * BIG, c = lane & 15, g = lane >> 4;
  // Steps of 32 columns, dealt in contiguous ranges to the launch's splits and to the waves.
  const int steps = (P.K + 31) / 32, ways = split * kFewWaves, way = blockIdx.y * kFewWaves + wave;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * way / ways);
  const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (way + 1) / ways);
  auto x_row = [&](int m) {
    m = min(m, P.M - 1);
    const int b = static_cast<int>(div31(static_cast<uint32_t>(m), P.by_l));
    return static_cast<const uint16_t *>(P.x) + b * P.x_sb + (m - b * P.L) * P.x_sl;
  };
  auto w_row = [&](int n) { return static_cast<const uint16_t *>(P.w) + min(n, P.N - 1) * P.ldw; };
  const uint16_t *big[NT], *few[MT];
#pragma unroll
  for (int i = 0; i < NT; ++i) big[i] = (SWAP ? x_row(r0 + 16 * i + c) : w_row(r0 + 16 * i + c)) + 8 * g;
#pragma unroll
  for (int j = 0; j < MT; ++j) few[j] = (SWAP ? w_row(16 * j + c) : x_row(16 * j + c)) + 8 * g;
  f32x4 acc[NT][MT] = {};
  int s = s0;
  for (; s + U <= s1 && 32 * (s + U) <= P.K; s += U) {  // no column of these steps is past K
    uint4 a[U][NT], b[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < NT; ++i) a[u][i] = load_any(big[i] + 32 * (s + u));
#pragma unroll
      for (int j = 0; j < MT; ++j) b[u][j] = load_any(few[j] + 32 * (s + u));
    }
    __builtin_amdgcn_sched_barrier(0);  // all loads ahead of the products: the compiler would pair them up again
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = mfma16<DT>(a[u][i], b[u][j], acc[i][j]);
  }
  for (; s < s1; ++s) {
    uint4 a[NT], b[MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) a[i] = load_chunk(big[i], 32 * s, P.K - 8 * g);
#pragma unroll
    for (int j = 0; j < MT; ++j) b[j] = load_chunk(few[j], 32 * s, P.K - 8 * g);
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[i][j] = mfma16<DT>(a[i], b[j], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
      *reinterpret_cast<f32x4 *>(&red[wave][16 * j + c][16 * i + 4 * g]) = acc[i][j];
  __syncthreads();
  if (split > 1) to_partial(P, part + static_cast<int64_t>(blockIdx.y) * P.M * P.N);
  finish_few<DT, NT, MT, SWAP, kFewWaves>(P, r0, &red[0][0][0]);
}

// The same for operands whose rows the DMA can read (dma_ok_x, dma_ok_w): the fragments' lane order takes each of 16 adjacent
// lanes to another row, 64 cache lines looked up per load, which held the loads above at 16 bytes per clock and CU (28 x
// 18432 x 3072 36 us). Here each wave copies its range of K to LDS of its own by DMA, 8 rows of 128 bytes per
// instruction, ST steps of 64 columns ahead, and reads the fragments there; no barrier until the sums are added. 28 x 18432 x
// 3072 26.7 us (the floor is 22.5): 231 workgroups of five blocks (80 rows) on 256 CUs, 4.24 TB/s of weight, and the few
// rows' 40 MB from the caches beside it. 1 x 3072 x 768 4.5 us and 4096 x 64 x 3072 10.8 us, where a launch, one chain of loads
// per wave and the sum over the waves are what is left.
constexpr int kStreamWaves = 4;
constexpr int stream_stages(int blocks) { return blocks <= 2 ? 4 : blocks == 3 ? 3 : 2; }

template <int DT, int NT, int MT, bool SWAP>
__global__ __launch_bounds__(64 * kStreamWaves) void raw_stream_kernel(RawProblem P, float *part, int split) {
  constexpr int NB = NT + MT, ST = stream_stages(NB), SB = NB * 2048;  // blocks of 16 rows, stages, bytes of one
  constexpr int D = 2 * NB;                                            // DMAs per stage
  constexpr int BIG = NT * 16, FEW = MT * 16, LD = BIG + 4;
  constexpr int RED = kStreamWaves * FEW * LD * 4, ALL = kStreamWaves * SB;
  static_assert(RED <= ALL, "the sums take the place of a stage");
  __shared__ __attribute__((aligned(1024))) uint8_t st0[ALL], st1[ALL], st2[ST > 2 ? ALL : 16], st3[ST > 3 ? ALL : 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r0 = blockIdx.x * BIG;
  const int steps = (P.K + 63) / 64, ways = split * kStreamWaves, way = blockIdx.y * kStreamWaves + wave;
  const int lo = static_cast<int>(static_cast<int64_t>(steps) * way / ways);
  const int hi = static_cast<int>(static_cast<int64_t>(steps) * (way + 1) / ways);
  // Row offsets from the lowest row's address (as in the tiled kernel); rows past the end load zeros.
  constexpr uint32_t kOut = 0x80000000u;
  const int xm0 = SWAP ? r0 : 0, b0 = static_cast<int>(div31(static_cast<uint32_t>(xm0), P.by_l)), l0 = xm0 - b0 * P.L;
  int64_t x_base = b0 * P.x_sb + l0 * P.x_sl;
  if (l0 + min(SWAP ? BIG : FEW, P.M - xm0) > P.L) x_base = min(x_base, (b0 + 1) * P.x_sb);
  const int64_t w_base = SWAP ? 0 : r0 * P.ldw;
  auto x_off = [&](int m) {
    const int b = static_cast<int>(div31(static_cast<uint32_t>(m), P.by_l));
    return m < P.M ? static_cast<uint32_t>((b * P.x_sb + (m - b * P.L) * P.x_sl - x_base) * 2) : kOut;
  };
  auto w_off = [&](int n) { return n < P.N ? static_cast<uint32_t>((n * P.ldw - w_base) * 2) : kOut; };
  uint32_t off[D];
  int kc[2];
#pragma unroll
  for (int j = 0; j < D; ++j) {
    const int r = 8 * j + (lane >> 3);  // streamed rows, then the few
    const int c = (lane & 7) ^ (4 * (j & 1) + (lane >> 4));
    uint32_t o;
    if (j < 2 * NT) o = SWAP ? x_off(r0 + r) : w_off(r0 + r);
    else o = SWAP ? w_off(r - BIG) : x_off(r - BIG);
    off[j] = o == kOut ? kOut : o + 16 * c;
    kc[j & 1] = 8 * c;
  }
  const uint16_t *const xb = static_cast<const uint16_t *>(P.x) + x_base, *const wb = static_cast<const uint16_t *>(P.w) + w_base;
  auto issue = [&](uint8_t *stage, int step) __attribute__((always_inline)) {
    const uint32_t range = step < hi ? 0x7fffffffu : 0u;
    const __amdgpu_buffer_rsrc_t big = make_rsrc(SWAP ? xb : wb, range), few = make_rsrc(SWAP ? wb : xb, range);
#pragma unroll
    for (int j = 0; j < D; ++j)
      load_lds16(j < 2 * NT ? big : few, stage + wave * SB + j * 1024, kc[j & 1] + 64 * step < P.K ? off[j] : kOut, 128u * step);
  };
  f32x4 acc[NT][MT] = {};
  auto step = [&](uint8_t *stage, int s) __attribute__((always_inline)) {
    wait_vmcnt<(ST - 1) * D>();
    uint4 f[NB][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < NB; ++i)
        f[i][h] = *reinterpret_cast<const uint4 *>(stage + wave * SB + i * 2048 + (lane & 15) * 128 +
                                                   (((4 * h + (lane >> 4)) ^ ((lane & 15) >> 1)) << 4));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the next DMA writes there
    issue(stage, s + ST);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = mfma16<DT>(f[i][h], f[NT + j][h], acc[i][j]);
  };
  issue(st0, lo);
  issue(st1, lo + 1);
  if constexpr (ST > 2) issue(st2, lo + 2);
  if constexpr (ST > 3) issue(st3, lo + 3);
  for (int s = lo; s < hi; s += ST) {  // steps past hi multiply zeros
    step(st0, s);
    step(st1, s + 1);
    if constexpr (ST > 2) step(st2, s + 2);
    if constexpr (ST > 3) step(st3, s + 3);
  }
  wait_vmcnt<0>();
  __syncthreads();
  float *const red = reinterpret_cast<float *>(st0);
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
      *reinterpret_cast<f32x4 *>(red + (wave * FEW + 16 * j + (lane & 15)) * LD + 16 * i + 4 * (lane >> 4)) = acc[i][j];
  __syncthreads();
  if (split > 1) to_partial(P, part + static_cast<int64_t>(blockIdx.y) * P.M * P.N);
  finish_few<DT, NT, MT, SWAP, kStreamWaves>(P, r0, red);
}

// ------------------------------------------------------------------ tiled

constexpr int kMaxProblems = SELAS_MAX_BATCHED_LINEARS;

// The problems of one launch; problem i's tiles are [tile0[i], tile0[i + 1]) of all.
struct RawBatch {
  RawProblem p[kMaxProblems];
  int tiles_m[kMaxProblems], tiles_n[kMaxProblems], tile0[kMaxProblems];
  float *part[kMaxProblems];
  int count, tiles, per_xcd;
  int split;  // K ranges per tile: item r * tiles + t is range r of tile t
};

__device__ __forceinline__ void wait_lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// 4 waves (WM x WN), each with MB x NB blocks of 16 x 16 outputs: tiles of TM rows of x by TN rows of w, K in steps of 64.
//
// LDS holds two steps, each operand in halves: half h of x is the first or second half of every wave's rows. A step runs
// as four phases, one quarter of each wave's outputs each, (x0, w0), (x0, w1), (x1, w1), (x1, w0), in odd steps with w0
// and w1 exchanged, so that every phase needs one operand half in registers that the phase before did not, and one
// half's registers are free for it. Phase p:
//   waits until the fragments read in phase p - 1 are in registers and the half that it reads now has landed, barrier;
//   reads the fragments of phase p + 1 from LDS, issues the DMA of the half that phase p - 1 read (which no wave needs
//   any more), and multiplies.
// A half is read 7 phases after its DMA was issued, so 6 newer halves' loads may be pending at each wait. Past the end
// of K the loads are out of range: they bring zeros and no traffic, and the counts stay the same.
//
// Why so: 256 x 256 is the largest tile whose sums (256 registers a lane) and fragments fit one wave per SIMD, and the
// fewest LDS bytes per product (one fragment read for 8 MFMAs). A half's 16 KB per DMA wave and the XOR of chunk and row
// (row / 2) % 8 leave no bank conflict (counted: 0). Two barriers a step instead of four, and the reads and DMAs pinned
// between the products, took the MFMAs from 72 to 83 % busy at 8192^3 (708-787 us back to back on several cards, the
// library's product 710-735).
// Of the block's linears, 4096 x 12288 x 3072 with GELU is 227-244 us where other kernels run in between and 244-268 back
// to back (1,154-1,362 TFLOP/s, floor 194; the library's product with its bias 220-261 back to back): three rounds of 256
// tiles whose prologue and epilogue, 11 us each, nothing overlaps at one workgroup per CU. 4608 x 3072 x 15360 with an
// fp32 residual is 316-333 and 325-354 us (1,228-1,376 TFLOP/s, floor 273; the library's product 526): 216 tiles for 256
// CUs, and all residual traffic at the end. MFMAs 65 and 66 % busy. HBM traffic is 1.0 of the output written, and of the
// operands read 2.3 and 1.7 times (the XCDs' L2s each load what their tiles share).
template <int DT, int WM, int WN, int MB, int NB, int OCC, bool TAIL>
__global__ __launch_bounds__(64 * WM * WN, OCC) void raw_tile_kernel(RawBatch batch) {
  constexpr int TM = WM * MB * 16, TN = WN * NB * 16, HM = MB / 2, HN = NB / 2, NW = WM * WN;
  constexpr int XB = TM / 2 * 128, WB = TN / 2 * 128;      // bytes of one half of x and of w
  constexpr int DX = XB / (1024 * NW), DW = WB / (1024 * NW);  // DMAs of a wave per half
  constexpr int ER = 32;                                   // rows that the epilogue stages at once
  constexpr int EB = ER * NB * 16 * 4;                     // bytes of them
  static_assert(NW == 4 && DX >= 1 && DW >= 1 && XB <= 16384 && WB <= 16384 && XB >= EB, "tile");
  __shared__ __attribute__((aligned(1024))) uint8_t x00[XB], x01[XB], x10[XB], x11[XB], w00[WB], w01[WB], w10[WB], w11[WB];

  const int item = (blockIdx.x & 7) * batch.per_xcd + (blockIdx.x >> 3);
  if (item >= batch.tiles * batch.split) return;
  const int range = item / batch.tiles, t = item - range * batch.tiles;
  // The tile's problem (uniform: scalar selects over the kernel arguments).
  RawProblem P = batch.p[0];
  int tile0 = 0, tn = batch.tiles_n[0], tm = batch.tiles_m[0];
  float *part = batch.part[0];
#pragma unroll
  for (int i = 1; i < kMaxProblems; ++i)
    if (i < batch.count && t >= batch.tile0[i]) {
      P = batch.p[i];
      tile0 = batch.tile0[i];
      tn = batch.tiles_n[i];
      tm = batch.tiles_m[i];
      part = batch.part[i];
    }
  if (batch.split > 1) {
    const int steps = (P.K + 63) / 64;
    const int lo = steps * range / batch.split * 64, hi = steps * (range + 1) / batch.split * 64;
    P.x = static_cast<const uint16_t *>(P.x) + lo;
    P.w = static_cast<const uint16_t *>(P.w) + lo;
    P.K = min(P.K, hi) - lo;
    to_partial(P, part + static_cast<int64_t>(range) * P.M * P.N);
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM, wn = wave / WM;
  int m0, n0;
  {
    // Groups of 4 row slabs, the row fastest: the tiles that an XCD runs at once share both operands in its L2.
    const int lt = t - tile0;
    const int group = lt / (4 * tn), gm = min(4, tm - 4 * group), in = lt - group * 4 * tn;
    m0 = (4 * group + in % gm) * TM;
    n0 = (in / gm) * TN;
  }
  const int M = P.M, N = P.N, K = P.K;

  // Operand bases: the tile's lowest row, so that the rows' offsets fit the buffer's 31 bits (checked on the host).
  const int b0 = static_cast<int>(div31(static_cast<uint32_t>(m0), P.by_l)), l0 = m0 - b0 * P.L;
  int64_t x_base = b0 * P.x_sb + l0 * P.x_sl;
  if (l0 + min(TM, M - m0) > P.L) x_base = min(x_base, (b0 + 1) * P.x_sb);
  const uint16_t *const xb = static_cast<const uint16_t *>(P.x) + x_base;
  const uint16_t *const wb = static_cast<const uint16_t *>(P.w) + static_cast<int64_t>(n0) * P.ldw;
  constexpr uint32_t kOut = 0x80000000u;  // past every range

  // DMA j of a half writes its LDS rows 8 j .. 8 j + 7: lane i row 8 j + i / 8, physical chunk i % 8, which holds logical
  // chunk (i % 8) ^ (row / 2) % 8, (row / 2) % 8 = 4 (j % 2) + i / 16.
  uint32_t xo[2][DX], wo[2][DW];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int j = 0; j < DX; ++j) {
      const int lr = 8 * (wave * DX + j) + (lane >> 3);
      const int m = m0 + (lr / (8 * MB)) * (16 * MB) + h * (8 * MB) + lr % (8 * MB);
      const int b = static_cast<int>(div31(static_cast<uint32_t>(m), P.by_l)), l = m - b * P.L;
      const uint32_t c = (lane & 7) ^ (4 * ((wave * DX + j) & 1) + (lane >> 4));
      xo[h][j] = m < M ? static_cast<uint32_t>((b * P.x_sb + l * P.x_sl - x_base) * 2) + 16 * c : kOut;
    }
#pragma unroll
    for (int j = 0; j < DW; ++j) {
      const int lr = 8 * (wave * DW + j) + (lane >> 3);
      const int r = (lr / (8 * NB)) * (16 * NB) + h * (8 * NB) + lr % (8 * NB);
      const uint32_t c = (lane & 7) ^ (4 * ((wave * DW + j) & 1) + (lane >> 4));
      wo[h][j] = n0 + r < N ? static_cast<uint32_t>(r * P.ldw * 2) + 16 * c : kOut;
    }
  }
  // Steps past the end of K load through an empty range. A last step of fewer than 64 columns (TAIL) compares, per lane,
  // the column that its chunks of even and odd DMAs start at.
  const int kc[2] = {8 * static_cast<int>((lane & 7) ^ (lane >> 4)), 8 * static_cast<int>((lane & 7) ^ (4 + (lane >> 4)))};
  auto load_step = [&](__amdgpu_buffer_rsrc_t r, uint8_t *dst, uint32_t off, int par, int step) __attribute__((always_inline)) {
    if constexpr (TAIL) off = kc[par] + 64 * step < K ? off : kOut;
    load_lds16(r, dst, off, 128u * step);
  };
  auto dma_x = [&](uint8_t *dst, int h, int step, int j) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(xb, TAIL || 64 * step < K ? 0x7fffffffu : 0u);
    load_step(r, dst + (wave * DX + j) * 1024, xo[h][j], (wave * DX + j) & 1, step);
  };
  auto dma_w = [&](uint8_t *dst, int h, int step, int j) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(wb, TAIL || 64 * step < K ? 0x7fffffffu : 0u);
    load_step(r, dst + (wave * DW + j) * 1024, wo[h][j], (wave * DW + j) & 1, step);
  };

  // Fragment i (16 rows) of k half s: row 16 i + lane % 16 of the wave's rows, chunk 4 s + lane / 16.
  uint32_t rd[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) rd[s] = (lane & 15) * 128 + (((4 * s + (lane >> 4)) ^ ((lane & 15) >> 1)) << 4);
  const uint32_t xrow = wm * HM * 2048, wrow = wn * HN * 2048;
  uint4 x0[HM][2], x1[HM][2], w0[HN][2], w1[HN][2];
  f32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{};
  // One phase: products of quarter (HX, HW) from (xf, wf); between them, in this order, the reads of the next fragments
  // (`read` i of R) and the DMAs (`dma` j of D), one after each product. Reads come first: they have the rest of the
  // phase to arrive.
  auto phase = [&](auto hx, auto hw, const uint4 (&xf)[HM][2], const uint4 (&wf)[HN][2], auto reads, auto &&read, auto dmas,
                   auto &&dma) __attribute__((always_inline)) {
    constexpr int HX = decltype(hx)::value, HW = decltype(hw)::value, R = decltype(reads)::value, D = decltype(dmas)::value;
    constexpr int F = HM * HN * 2, SPAN = F * 7 / 8;
    for_each_index<F>([&](auto index) __attribute__((always_inline)) {
      constexpr int q = decltype(index)::value, s = q / (HM * HN), i = q / HN % HM, j = q % HN;
      mfma16_inplace<DT>(wf[j][s], xf[i][s], acc[HX * HM + i][HW * HN + j]);
      for_each_index<R>([&](auto slot) __attribute__((always_inline)) {
        if constexpr (decltype(slot)::value * SPAN / R == q) read(slot);
      });
      for_each_index<D>([&](auto slot) __attribute__((always_inline)) {
        constexpr int u = decltype(slot)::value;
        if constexpr (((2 * u + 1) * F / (2 * D)) == q) dma(u);
      });
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  auto read_x = [&](uint4 (&f)[HM][2], const uint8_t *src, int u) {
    f[u % HM][u / HM] = *reinterpret_cast<const uint4 *>(src + xrow + (u % HM) * 2048 + rd[u / HM]);
  };
  auto read_w = [&](uint4 (&f)[HN][2], const uint8_t *src, int u) {
    f[u % HN][u / HN] = *reinterpret_cast<const uint4 *>(src + wrow + (u % HN) * 2048 + rd[u / HN]);
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using RX = std::integral_constant<int, 2 * HM>;
  using RW = std::integral_constant<int, 2 * HN>;
  using CX = std::integral_constant<int, DX>;
  using CW = std::integral_constant<int, DW>;

  const int steps = ((K + 63) / 64 + 1) & ~1;
  auto all_x = [&](uint8_t *dst, int h, int step) {
#pragma unroll
    for (int j = 0; j < DX; ++j) dma_x(dst, h, step, j);
  };
  auto all_w = [&](uint8_t *dst, int h, int step) {
#pragma unroll
    for (int j = 0; j < DW; ++j) dma_w(dst, h, step, j);
  };
  all_x(x00, 0, 0); all_w(w00, 0, 0); all_w(w01, 1, 0); all_x(x01, 1, 0);
  all_x(x10, 0, 1); all_w(w11, 1, 1); all_w(w10, 0, 1); all_x(x11, 1, 1);
  __builtin_amdgcn_sched_barrier(0);
  wait_vmcnt<3 * DW + 3 * DX>();
  wait_lds_barrier();
#pragma unroll
  for (int u = 0; u < 2 * HM; ++u) read_x(x0, x00, u);
#pragma unroll
  for (int u = 0; u < 2 * HN; ++u) read_w(w0, w00, u);
  __builtin_amdgcn_sched_barrier(0);
  for (int k = 0; k < steps; k += 2) {
    // Arrays: operand, step % 2, half.
    wait_vmcnt<2 * DW + 2 * DX>();
    wait_lds_barrier();
    phase(I0{}, I0{}, x0, w0, RW{}, [&](auto u) { read_w(w1, w01, decltype(u)::value); },
          CX{}, [&](int j) { dma_x(x00, 0, k + 2, j); });
    phase(I0{}, I1{}, x0, w1, RX{}, [&](auto u) { read_x(x1, x01, decltype(u)::value); },
          CW{}, [&](int j) { dma_w(w00, 0, k + 2, j); });
    wait_vmcnt<2 * DW + 2 * DX>();
    wait_lds_barrier();
    phase(I1{}, I1{}, x1, w1, RX{}, [&](auto u) { read_x(x0, x10, decltype(u)::value); },
          CW{}, [&](int j) { dma_w(w01, 1, k + 2, j); });
    phase(I1{}, I0{}, x1, w0, RW{}, [&](auto u) { read_w(w1, w11, decltype(u)::value); },
          CX{}, [&](int j) { dma_x(x01, 1, k + 2, j); });
    wait_vmcnt<2 * DW + 2 * DX>();
    wait_lds_barrier();
    phase(I0{}, I1{}, x0, w1, RW{}, [&](auto u) { read_w(w0, w10, decltype(u)::value); },
          CX{}, [&](int j) { dma_x(x10, 0, k + 3, j); });
    phase(I0{}, I0{}, x0, w0, RX{}, [&](auto u) { read_x(x1, x11, decltype(u)::value); },
          CW{}, [&](int j) { dma_w(w11, 1, k + 3, j); });
    wait_vmcnt<2 * DW + 2 * DX>();
    wait_lds_barrier();
    phase(I1{}, I0{}, x1, w0, RX{}, [&](auto u) { read_x(x0, x00, decltype(u)::value); },
          CW{}, [&](int j) { dma_w(w10, 0, k + 3, j); });
    phase(I1{}, I1{}, x1, w1, RW{}, [&](auto u) { read_w(w0, w00, decltype(u)::value); },
          CX{}, [&](int j) { dma_x(x11, 1, k + 3, j); });
  }
  settle_mfma();
  // No DMA may land in LDS that the epilogue (or a later workgroup) uses.
  wait_vmcnt<0>();
  wait_lds_barrier();

  // Epilogue: each wave passes its outputs, 32 rows at a time, through its own part of LDS, so that a lane owns W
  // adjacent columns and a row leaves in whole lines.
  uint8_t *const st = wave == 0 ? x00 : wave == 1 ? x01 : wave == 2 ? x10 : x11;
  const int nw = n0 + wn * NB * 16;  // first column of this wave
  auto stage = [&](int e) __attribute__((always_inline)) {
    for_each_index<MB / 2>([&](auto part) __attribute__((always_inline)) {
      constexpr int E = decltype(part)::value;
      if (e != E) return;
      // Each case keeps its code: merged into one, the accumulators would be indexed at run time, in scratch memory.
      asm volatile("; rows %0" ::"i"(E) : "memory");
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          const int r = 16 * i + (lane & 15), c = 4 * j + (lane >> 4);  // row, 16-byte chunk of it
          f32x4 q = acc[2 * E + i][j];
          asm volatile("" : "+a"(q));
          *reinterpret_cast<f32x4 *>(st + r * (NB * 64) + ((c ^ (r & 15)) << 4)) = q;
        }
      asm volatile("; rows %0 done" ::"i"(E) : "memory");
    });
  };
  // The wave's outputs by way of LDS, 32 rows (a part) at a time, W columns per lane. One wave reads what it wrote: no
  // barrier. Addresses are a lane's offset plus a scalar for the rows, out of range for rows past M and columns past N.
  // The residual of a part is loaded while the part before is stored.
  auto finish = [&](auto width) __attribute__((always_inline)) {
    constexpr int W = decltype(width)::value;
    constexpr int LPR = NB * 16 / W, RPI = 64 / LPR, G = ER / RPI;  // lanes per row, rows per instruction, groups of them
    const int n = nw + (lane % LPR) * W, row = lane / LPR;
    const int mw = m0 + wm * MB * 16, rows = M - mw;  // first row of the wave, rows there are
    const int ye = P.y_f32 ? 4 : 2, re = P.residual_f32 ? 4 : 2;
    const __amdgpu_buffer_rsrc_t yr =
        make_rsrc(static_cast<uint8_t *>(P.y) + (mw * P.y_sl + nw) * ye, 0x7fffffffu);
    const __amdgpu_buffer_rsrc_t rr =
        make_rsrc(static_cast<const uint8_t *>(P.residual) + (mw * P.r_sl + nw) * re, 0x7fffffffu);
    const uint32_t ys = static_cast<uint32_t>(P.y_sl) * ye, rs = static_cast<uint32_t>(P.r_sl) * re;
    const uint32_t yv = row * ys + (n - nw) * ye, rv = row * rs + (n - nw) * re;
    float bias[W] = {}, gate[W];
    if (P.bias && n < N) load_cols<DT, W>(P.bias, n, P.bias_f32, bias);
    if (P.gate && P.one_gate && n < N) load_cols<DT, W>(P.gate, n, P.gate_f32, gate);
    uint4 res[G][W / 4] = {};
    auto load_res = [&](int e) __attribute__((always_inline)) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint32_t at = e * ER + g * RPI + row < rows && n < N ? rv : kOut, so = (e * ER + g * RPI) * rs;
        if (P.residual_f32) {
#pragma unroll
          for (int q = 0; q < W / 4; ++q) res[g][q] = load_b128(rr, at + 16 * q, so);
        } else if constexpr (W == 8) {
          res[g][0] = load_b128(rr, at, so);
        } else {
          const auto u = __builtin_amdgcn_raw_buffer_load_b64(rr, at, so, 0);
          res[g][0].x = u[0], res[g][0].y = u[1];
        }
      }
    };
    if (P.residual) load_res(0);
#pragma unroll 1
    for (int e = 0; e < MB / 2; ++e) {
      stage(e);
      float v[G][W];
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int q = 0; q < W / 4; ++q) {
          const int r = g * RPI + row, c = (lane % LPR) * (W / 4) + q;
          const f32x4 f = *reinterpret_cast<const f32x4 *>(st + r * (NB * 64) + ((c ^ (r & 15)) << 4));
#pragma unroll
          for (int j = 0; j < 4; ++j) v[g][4 * q + j] = f[j] + bias[4 * q + j];
        }
      activate_all(v, P.act, P.guard);
      if (P.gate) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          if (!P.one_gate) {
            const int m = min(mw + e * ER + g * RPI + row, M - 1);
            const int64_t at = static_cast<int64_t>(div31(static_cast<uint32_t>(m), P.by_l)) * P.gate_sb + n;
            if (n < N) load_cols<DT, W>(P.gate, at, P.gate_f32, gate);
          }
#pragma unroll
          for (int j = 0; j < W; ++j) v[g][j] *= gate[j];
        }
      }
      if (P.residual) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          if (P.residual_f32) {
#pragma unroll
            for (int q = 0; q < W / 4; ++q) {
              const uint4 u = res[g][q];
              v[g][4 * q] = __uint_as_float(u.x) + v[g][4 * q];
              v[g][4 * q + 1] = __uint_as_float(u.y) + v[g][4 * q + 1];
              v[g][4 * q + 2] = __uint_as_float(u.z) + v[g][4 * q + 2];
              v[g][4 * q + 3] = __uint_as_float(u.w) + v[g][4 * q + 3];
            }
          } else {
            const uint32_t w[4] = {res[g][0].x, res[g][0].y, res[g][0].z, res[g][0].w};
#pragma unroll
            for (int t = 0; t < W / 2; ++t) {
              if constexpr (DT == SELAS_BF16) {
                v[g][2 * t] = __uint_as_float(w[t] << 16) + v[g][2 * t];
                v[g][2 * t + 1] = __uint_as_float(w[t] & 0xffff0000u) + v[g][2 * t + 1];
              } else {
                v[g][2 * t] = f16_bits_to_f32(w[t] & 0xffffu) + v[g][2 * t];
                v[g][2 * t + 1] = f16_bits_to_f32(w[t] >> 16) + v[g][2 * t + 1];
              }
            }
          }
        }
        if (e + 1 < MB / 2) load_res(e + 1);
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint32_t at = e * ER + g * RPI + row < rows && n < N ? yv : kOut, so = (e * ER + g * RPI) * ys;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (W == 4) w[j] = __float_as_uint(v[g][j]);
          else if constexpr (DT == SELAS_BF16) w[j] = pack_bf16x2(v[g][2 * j], v[g][2 * j + 1]);
          else w[j] = f16_bits_rne(v[g][2 * j]) | (static_cast<uint32_t>(f16_bits_rne(v[g][2 * j + 1])) << 16);
        }
        __builtin_amdgcn_raw_buffer_store_b128(u32x4{w[0], w[1], w[2], w[3]}, yr, at, so, 0);
      }
    }
  };
  // The same for outputs off alignment, N not a multiple of 8 or batches with spacing of their own: addresses per row, and
  // vector accesses that may start at any element, except in the columns that N cuts. Columns past N and rows past M read
  // the last one (live - 1 is then negative: the column N - 1). Two rows at once in the tile of two workgroups per CU, whose
  // registers do not hold four (1386 x 1431 x 667 with GELU and residual 21.5 us; four 24.1, one after another 25.5).
  auto finish_any = [&](auto width) __attribute__((always_inline)) {
    constexpr int W = decltype(width)::value, LPR = NB * 16 / W, RPI = 64 / LPR, U = OCC == 1 ? 4 : 2;
    const int n = nw + (lane % LPR) * W, row = lane / LPR, live = N - n;
    const int mw = m0 + wm * MB * 16;
    const bool whole = nw + NB * 16 <= N;
    float bias[1][W] = {}, gate[1][W] = {};
    const int64_t only[1] = {n};
    if (P.bias) load_rows_any<DT, 1, W>(P.bias, only, P.bias_f32, whole, live, bias);
    if (P.gate && P.one_gate) load_rows_any<DT, 1, W>(P.gate, only, P.gate_f32, whole, live, gate);
#pragma unroll 1
    for (int e = 0; e < MB / 2; ++e) {
      stage(e);
#pragma unroll 1
      for (int g = 0; g < ER / RPI; g += U) {
        float v[U][W], res[U][W];
        int64_t ga[U], ra[U], ya[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int m = min(mw + e * ER + (g + u) * RPI + row, M - 1);
          const int b = static_cast<int>(div31(static_cast<uint32_t>(m), P.by_l)), l = m - b * P.L;
          ga[u] = b * P.gate_sb + n;
          ra[u] = b * P.r_sb + l * P.r_sl + n;
          ya[u] = b * P.y_sb + l * P.y_sl + n;
        }
        if (P.residual) load_rows_any<DT, U, W>(P.residual, ra, P.residual_f32, whole, live, res);
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int q = 0; q < W / 4; ++q) {
            const int r = (g + u) * RPI + row, c = (lane % LPR) * (W / 4) + q;
            const f32x4 f = *reinterpret_cast<const f32x4 *>(st + r * (NB * 64) + ((c ^ (r & 15)) << 4));
#pragma unroll
            for (int j = 0; j < 4; ++j) v[u][4 * q + j] = f[j] + bias[0][4 * q + j];
          }
        }
        activate_all(v, P.act, P.guard);
        if (P.gate && P.one_gate) {
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < W; ++j) v[u][j] *= gate[0][j];
        } else if (P.gate) {
          float gates[U][W];
          load_rows_any<DT, U, W>(P.gate, ga, P.gate_f32, whole, live, gates);
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < W; ++j) v[u][j] *= gates[u][j];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (P.residual) {
#pragma unroll
            for (int j = 0; j < W; ++j) v[u][j] = res[u][j] + v[u][j];
          }
          if (mw + e * ER + (g + u) * RPI + row < M) store_cols_any<DT, W>(P.y, ya[u], live, v[u]);
        }
      }
    }
  };
  if (P.vec && P.y_f32) finish(std::integral_constant<int, 4>{});
  else if (P.vec) finish(std::integral_constant<int, 8>{});
  else if (P.y_f32) finish_any(std::integral_constant<int, 4>{});
  else finish_any(std::integral_constant<int, 8>{});
}

// ------------------------------------------------------------------ host side

bool float_or(int dt, int dtype) { return dt == SELAS_F32 || dt == dtype; }

int check_problem(const selas_raw_linear_problem &p, int64_t i, int dtype) {
  const long long at = i;
  if (p.B < 0 || p.L < 0 || p.N < 0 || p.K < 0)
    return set_error(SELAS_EINVAL, "raw_linear[%lld]: bad shape B=%lld L=%lld N=%lld K=%lld", at, (long long)p.B,
                     (long long)p.L, (long long)p.N, (long long)p.K);
  if (p.act < SELAS_ACT_NONE || p.act > SELAS_ACT_SILU)
    return set_error(SELAS_EINVAL, "raw_linear[%lld]: unknown activation %d", at, p.act);
  if (!float_or(p.y_dtype, dtype) || (p.bias && !float_or(p.bias_dtype, dtype)) ||
      (p.gate && !float_or(p.gate_dtype, dtype)) || (p.residual && !float_or(p.residual_dtype, dtype)))
    return set_error(SELAS_EINVAL, "raw_linear[%lld]: bias, gate, residual and y are f32 or %s", at, dtype_name(dtype));
  if (p.x_sb < 0 || p.x_sl < 0 || p.ldw < 0 || p.gate_sb < 0 || p.r_sb < 0 || p.r_sl < 0 || p.y_sb < 0 || p.y_sl < 0)
    return set_error(SELAS_EINVAL, "raw_linear[%lld]: negative stride", at);
  if (p.B >= (1ll << 31) || p.L >= (1ll << 31) || p.B * p.L >= (1ll << 31) - 256 || p.N >= (1ll << 31) - 256 ||
      p.K >= (1ll << 31) - 256)
    return set_error(SELAS_EUNSUPPORTED, "raw_linear[%lld]: rows, columns or K above 2^31", at);
  return SELAS_OK;
}

// Whether rows of p (stride s, batch stride sb, in elements of `size` bytes) take 16-byte accesses at every 8th element.
bool rows_ok(const void *p, int64_t sb, int64_t s, int size) {
  return aligned(p, 16) && sb * size % 16 == 0 && s * size % 16 == 0;
}

bool epilogue_vec(const selas_raw_linear_problem &p) {
  auto size = [](int dt) { return dt == SELAS_F32 ? 4 : 2; };
  auto even = [&](int64_t sb, int64_t sl) { return (p.B == 1 || sb == p.L * sl) && sl < (1ll << 20); };
  return p.N % 8 == 0 && rows_ok(p.y, p.y_sb, p.y_sl, size(p.y_dtype)) && even(p.y_sb, p.y_sl) &&
         (!p.bias || aligned(p.bias, 16)) && (!p.gate || rows_ok(p.gate, p.gate_sb, 0, size(p.gate_dtype))) &&
         (!p.residual || (rows_ok(p.residual, p.r_sb, p.r_sl, size(p.residual_dtype)) && even(p.r_sb, p.r_sl)));
}

RawProblem make_problem(const selas_raw_linear_problem &p) {
  RawProblem r{};
  r.x = p.x; r.w = p.w; r.bias = p.bias; r.gate = p.gate; r.residual = p.residual; r.y = p.y;
  r.x_sb = p.x_sb; r.x_sl = p.x_sl; r.ldw = p.ldw; r.gate_sb = p.gate_sb;
  r.r_sb = p.r_sb; r.r_sl = p.r_sl; r.y_sb = p.y_sb; r.y_sl = p.y_sl;
  r.M = static_cast<int>(p.B * p.L); r.L = static_cast<int>(p.L);
  r.N = static_cast<int>(p.N); r.K = static_cast<int>(p.K);
  r.by_l = fast_div(static_cast<uint32_t>(p.L));
  r.act = p.act;
  r.guard = p.guard != 0;
  r.bias_f32 = p.bias_dtype == SELAS_F32; r.gate_f32 = p.gate_dtype == SELAS_F32;
  r.residual_f32 = p.residual_dtype == SELAS_F32; r.y_f32 = p.y_dtype == SELAS_F32;
  r.vec = epilogue_vec(p);
  r.one_gate = p.B == 1 || p.gate_sb == 0;
  return r;
}

// Whether the kernels' DMA can read an operand where it is: whole 16-byte chunks, and the rows of a tile within 31 bits
// of bytes.
bool dma_ok_w(const selas_raw_linear_problem &p) {
  return p.K % 8 == 0 && rows_ok(p.w, 0, p.ldw, 2) && p.ldw < (1ll << 40) && (256 * p.ldw + p.K) * 2 < (1ll << 31) - 4096;
}
bool dma_ok_x(const selas_raw_linear_problem &p) {
  if (p.K % 8 || !rows_ok(p.x, p.x_sb, p.x_sl, 2) || p.x_sl >= (1ll << 40) || p.x_sb >= (1ll << 40)) return false;
  const int64_t rows = 256, gap = p.x_sb - (p.L - 1) * p.x_sl, crossings = p.B > 1 ? rows / p.L + 1 : 0;
  const int64_t span = gap >= 0 || p.B == 1 ? rows * p.x_sl + crossings * gap : p.L * p.x_sl + crossings * p.x_sb;
  return (span + p.K) * 2 < (1ll << 31) - 4096;
}

// Whether the rows of a tile of a copied operand of `rows` rows (raw_pack_kernel) span less than 31 bits of bytes.
bool pack_ok(int64_t rows, int64_t K) { return (rows < 256 ? rows : 256) * cdiv(K, 64) * 128 < (1ll << 31) - 4096; }

// The current device's CU count (asked once per device).
int cu_count() {
  constexpr int kDevices = 64;
  static std::atomic<int> counts[kDevices];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) {
    (void)hipGetLastError();
    return 256;
  }
  const int slot = dev >= 0 && dev < kDevices ? dev : 0;
  int v = counts[slot].load(std::memory_order_relaxed);
  if (v > 0) return v;
  if (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || v <= 0) {
    (void)hipGetLastError();
    v = 256;
  }
  counts[slot].store(v, std::memory_order_relaxed);
  return v;
}

// How a problem runs. kFew and kStream are launches of their own; the tiled problems of a call share one.
enum class Route { kEmpty, kFew, kStream, kTiled };

// Rows of x and of w per tile, K ranges per tile.
struct TileChoice {
  int tm, tn, split;
};

struct Plan {
  Route route[kMaxProblems];
  int few_split[kMaxProblems];  // K ranges of a kFew or kStream problem
  TileChoice tile;              // of the tiled launch
  // The workspace, in 16-byte units: each problem's partial sums, then its packed x and w (0: none).
  int64_t part[kMaxProblems], pack_x[kMaxProblems], pack_w[kMaxProblems];
  int64_t units;
};

// Few rows: 32 of x (33 to 64 run faster as tiles: 60 x 9216 x 3072 25 us against 29), 64 of the weight (1024 x 64 x
// 3072 9.6 us against 12). Each of these problems is a launch of its own.
constexpr int kFewX = 32, kFewW = 64;

// Blocks of 16 streamed rows per workgroup. Streamed weights: as many as make one round of one workgroup per CU, up to six,
// for fewer reads of the few rows and no second round (us against two blocks: 28 x 18432 x 3072, five, 26.7 against 29.9;
// 28 x 9216 x 3072, three, 16.8 against 20.2; 28 x 21504 x 3072, six, 30.3 against 32.1). Two instead of four are one round of two
// workgroups per CU (4 x 16384 x 4096 25.2 against 28.7; with 17 to 32 rows, 27.0, four were not measured), and two past six
// (28 x 40000 x 1024 22.7 us, five 24.6).
// Streamed x, and rows off the DMA's alignment: two blocks where that gives every CU two workgroups, else one.
int few_blocks(int64_t big, bool weights) {
  const int64_t blocks = cdiv(cdiv(big, 16), cu_count());  // per CU
  if (!weights) return blocks > 2 ? 2 : 1;
  return blocks == 4 || blocks > 6 ? 2 : static_cast<int>(blocks);
}

// K ranges of a few-row launch: doubled while its workgroups leave CUs idle and a wave keeps 3 steps of 64 (1024 x 64 x
// 3072 11.0 us whole, 9.6 us in four; with 192 workgroups, 28 x 3072 x 3072, two ranges cost 9.5 -> 13 us).
int few_split(int64_t big, int64_t K) {
  const int64_t units = cdiv(big, 16), steps = cdiv(K, 64);
  int split = 1;
  while (units * split * 2 <= cu_count() && steps / (kStreamWaves * split * 2) >= 3) split *= 2;
  return split;
}

// Tile and K ranges of the tiled launch: the fastest by this model of a launch in us, fitted to 275 shapes (40 to 4608
// rows, 256 to 21504 columns, K 256 to 12288, weights from HBM; every tile and split timed). Its choices are within 1 %
// of the fastest in the mean and 18 % at worst (384 x 12288 x 3072: 40 us in tiles of 256 x 128, 54 of 128 x 128; 1024 x
// 12288 x 3072: 67 us of 256 x 256, 84 of 128 x 128; tiles of 128 x 256 were ahead in 13 shapes, by 0.3 % over all, and
// are left out). Other ranges than the seven were not timed. A round is one tile on every CU; a step of K costs the more
// the more CUs are busy; a split launch pays for its second kernel and for writing and reading the partial sums.
struct TileCost {
  int tm, tn;
  double start, step, busy, round;
};
constexpr TileCost kTiles[] = {{256, 256, 10.6, 0.682, 0.263, 4.7},
                               {256, 128, 9.7, 0.440, 0.185, 2.3},
                               {128, 128, 6.5, 0.315, 0.138, 0.56}};

TileChoice pick_tile(const selas_raw_linear_problem *problems, const Plan &plan, int64_t count) {
  const int cus = cu_count();
  TileChoice best{256, 256, 1};
  double best_us = 1e30;
  for (const TileCost &t : kTiles)
    for (int split : {1, 2, 3, 4, 6, 8, 12}) {
      int64_t tiles = 0, steps = 0, sums = 0, merges = 0;
      for (int64_t i = 0; i < count; ++i) {
        if (plan.route[i] != Route::kTiled) continue;
        const selas_raw_linear_problem &p = problems[i];
        tiles += cdiv(p.B * p.L, t.tm) * cdiv(p.N, t.tn);
        steps = steps > cdiv(p.K, 64) ? steps : cdiv(p.K, 64);
        sums += p.B * p.L * p.N;
        ++merges;
      }
      const int64_t items = tiles * split, rounds = cdiv(items, cus);
      if (split > 1 && (steps < 3 * split || items > 2 * cus)) continue;
      const double busy = items < cus ? static_cast<double>(items) / cus : 1.0;
      double us = t.start + (t.step + t.busy * busy) * cdiv(steps, split) * rounds + t.round * (rounds - 1);
      if (split > 1) us += 3.7 * merges + 0.81e-6 * split * sums;
      if (us < best_us) {
        best_us = us;
        best = TileChoice{t.tm, t.tn, split};
      }
    }
  return best;
}

Plan make_plan(const selas_raw_linear_problem *problems, int64_t count) {
  Plan plan{};
  bool tiled = false;
  for (int64_t i = 0; i < count; ++i) {
    const selas_raw_linear_problem &p = problems[i];
    const int64_t M = p.B * p.L;
    plan.few_split[i] = 1;
    if (M == 0 || p.N == 0) {
      plan.route[i] = Route::kEmpty;
    } else if (M <= kFewX || p.N <= kFewW) {
      plan.route[i] = dma_ok_x(p) && dma_ok_w(p) ? Route::kStream : Route::kFew;
      plan.few_split[i] = few_split(M <= kFewX ? p.N : M, p.K);
    } else {
      plan.route[i] = Route::kTiled;
      tiled = true;
      const int64_t chunks = cdiv(p.K, 64) * 8;
      if (!dma_ok_x(p)) plan.pack_x[i] = M * chunks;
      if (!dma_ok_w(p)) plan.pack_w[i] = p.N * chunks;
    }
  }
  if (tiled) plan.tile = pick_tile(problems, plan, count);
  for (int64_t i = 0; i < count; ++i) {
    const int split = plan.route[i] == Route::kTiled ? plan.tile.split : plan.few_split[i];
    plan.part[i] = split > 1 ? cdiv(split * problems[i].B * problems[i].L * problems[i].N, 4) : 0;
    plan.units += plan.part[i] + plan.pack_x[i] + plan.pack_w[i];
  }
  return plan;
}

template <int DT>
int launch_merge(const RawProblem &P, const float *part, int split, hipStream_t s) {
  const int64_t groups = static_cast<int64_t>(P.M) * ((P.N + 3) / 4);
  raw_merge_kernel<DT><<<dim3(static_cast<uint32_t>(cdiv(groups, 256))), dim3(256), 0, s>>>(P, part, split);
  return check_launch("raw_linear");
}

template <int DT>
int launch_few(const RawProblem &P, bool stream, float *part, int split, hipStream_t s) {
  const bool swap = P.M > kFewX;
  const int few = swap ? P.N : P.M, big = swap ? P.M : P.N;
  const int nt = few_blocks(big, stream && !swap), mt = few <= 16 ? 1 : few <= 32 ? 2 : 4;
  const dim3 grid(static_cast<uint32_t>(cdiv(big, 16 * nt)), static_cast<uint32_t>(split)), blk(64 * kFewWaves), sblk(64 * kStreamWaves);
#define SELAS_FEW(NT, MT, SWAP)                                                                  \
  do {                                                                                           \
    if (stream) raw_stream_kernel<DT, NT, MT, SWAP><<<grid, sblk, 0, s>>>(P, part, split);       \
    else raw_few_kernel<DT, NT, MT, SWAP><<<grid, blk, 0, s>>>(P, part, split);                  \
  } while (0)
#define SELAS_FEW_NT(MT, SWAP)            \
  do {                                    \
    if (nt == 2) SELAS_FEW(2, MT, SWAP);  \
    else SELAS_FEW(1, MT, SWAP);          \
  } while (0)
#define SELAS_WIDE(NT)                                                                                     \
  else if (nt == NT && mt == 2) raw_stream_kernel<DT, NT, 2, false><<<grid, sblk, 0, s>>>(P, part, split); \
  else if (nt == NT) raw_stream_kernel<DT, NT, 1, false><<<grid, sblk, 0, s>>>(P, part, split);
  if (swap && mt == 4) SELAS_FEW_NT(4, true);
  else if (swap && mt == 2) SELAS_FEW_NT(2, true);
  else if (swap) SELAS_FEW_NT(1, true);
  SELAS_WIDE(3) SELAS_WIDE(5) SELAS_WIDE(6)
  else if (mt == 2) SELAS_FEW_NT(2, false);
  else SELAS_FEW_NT(1, false);
#undef SELAS_WIDE
#undef SELAS_FEW_NT
#undef SELAS_FEW
  if (int e = check_launch("raw_linear")) return e;
  return split > 1 ? launch_merge<DT>(P, part, split, s) : ok();
}

template <int DT>
int launch_tiled(RawBatch &batch, const Plan &plan, hipStream_t s) {
  batch.tiles = 0;
  batch.split = plan.tile.split;
  bool tail = false;
  for (int i = 0; i < batch.count; ++i) {
    const RawProblem &P = batch.p[i];
    batch.tiles_m[i] = static_cast<int>(cdiv(P.M, plan.tile.tm));
    batch.tiles_n[i] = static_cast<int>(cdiv(P.N, plan.tile.tn));
    batch.tile0[i] = batch.tiles;
    if (static_cast<int64_t>(batch.tiles_m[i]) * batch.tiles_n[i] >= (1ll << 24) - batch.tiles)
      return set_error(SELAS_EUNSUPPORTED, "raw_linear: too many tiles");
    batch.tiles += batch.tiles_m[i] * batch.tiles_n[i];
    tail = tail || P.K % 64;
  }
  batch.per_xcd = static_cast<int>(cdiv(batch.tiles * batch.split, 8));
  const dim3 grid(static_cast<uint32_t>(batch.per_xcd * 8)), blk(256);
#define SELAS_TILE(MB, NB, OCC)                                                         \
  do {                                                                                  \
    if (tail) raw_tile_kernel<DT, 2, 2, MB, NB, OCC, true><<<grid, blk, 0, s>>>(batch); \
    else raw_tile_kernel<DT, 2, 2, MB, NB, OCC, false><<<grid, blk, 0, s>>>(batch);     \
  } while (0)
  if (plan.tile.tm == 256 && plan.tile.tn == 256) SELAS_TILE(8, 8, 1);
  else if (plan.tile.tm == 256) SELAS_TILE(8, 4, 1);
  else SELAS_TILE(4, 4, 2);
#undef SELAS_TILE
  if (int e = check_launch("raw_linear")) return e;
  if (batch.split > 1)
    for (int i = 0; i < batch.count; ++i)
      if (int e = launch_merge<DT>(batch.p[i], batch.part[i], batch.split, s)) return e;
  return ok();
}

template <int DT>
int launch_pack(RawProblem &P, uint4 *xp, uint4 *wp, hipStream_t s) {
  const int kp = static_cast<int>(cdiv(P.K, 64)) * 64;
  const int64_t chunks = (static_cast<int64_t>(xp ? P.M : 0) + (wp ? P.N : 0)) * (kp / 8);
  if (chunks == 0) return ok();
  if (cdiv(chunks, 256) >= (1ll << 31)) return set_error(SELAS_EUNSUPPORTED, "raw_linear: operands too large to copy");
  raw_pack_kernel<DT><<<dim3(static_cast<uint32_t>(cdiv(chunks, 256))), dim3(256), 0, s>>>(
      P, reinterpret_cast<uint16_t *>(xp), reinterpret_cast<uint16_t *>(wp), kp);
  if (xp) {
    P.x = xp;
    P.x_sl = kp;
    P.x_sb = static_cast<int64_t>(P.L) * kp;
  }
  if (wp) {
    P.w = wp;
    P.ldw = kp;
  }
  // An operand that stays where it is has no columns past K, so K grows only where both were copied.
  if (xp && wp) P.K = kp;
  return check_launch("raw_linear");
}

template <int DT>
int launch_plan(const selas_raw_linear_problem *problems, int64_t count, const Plan &plan, uint4 *ws, hipStream_t s) {
  RawBatch batch{};
  for (int64_t i = 0; i < count; ++i) {
    if (plan.route[i] == Route::kEmpty) continue;
    RawProblem P = make_problem(problems[i]);
    float *const part = plan.part[i] ? reinterpret_cast<float *>(ws) : nullptr;
    uint4 *const xp = plan.pack_x[i] ? ws + plan.part[i] : nullptr;
    uint4 *const wp = plan.pack_w[i] ? ws + plan.part[i] + plan.pack_x[i] : nullptr;
    ws += plan.part[i] + plan.pack_x[i] + plan.pack_w[i];
    if (plan.route[i] == Route::kTiled) {
      if (int e = launch_pack<DT>(P, xp, wp, s)) return e;
      batch.part[batch.count] = part;
      batch.p[batch.count++] = P;
    } else if (int e = launch_few<DT>(P, plan.route[i] == Route::kStream, part, plan.few_split[i], s)) {
      return e;
    }
  }
  return batch.count ? launch_tiled<DT>(batch, plan, s) : ok();
}

int check_call(const selas_raw_linear_problem *problems, int64_t count, int dtype) {
  if (count < 0 || count > SELAS_MAX_BATCHED_LINEARS || (count && !problems))
    return set_error(SELAS_EINVAL, "raw_linear: takes up to %d problems, got %lld", SELAS_MAX_BATCHED_LINEARS,
                     (long long)count);
  if (!valid_dtype(dtype)) return set_error(SELAS_EINVAL, "raw_linear: bad dtype %d", dtype);
  if (dtype == SELAS_F32) return set_error(SELAS_EUNSUPPORTED, "raw_linear: takes bf16 or fp16 weights");
  for (int64_t i = 0; i < count; ++i) {
    const selas_raw_linear_problem &p = problems[i];
    if (int e = check_problem(p, i, dtype)) return e;
    const int64_t M = p.B * p.L;
    if (M > kFewX && p.N > kFewW && ((!dma_ok_x(p) && !pack_ok(M, p.K)) || (!dma_ok_w(p) && !pack_ok(p.N, p.K))))
      return set_error(SELAS_EUNSUPPORTED, "raw_linear[%lld]: K = %lld: the rows of a tile span 2^31 bytes", (long long)i,
                       (long long)p.K);
  }
  return SELAS_OK;
}

}  // namespace
}  // namespace selas

using namespace selas;

extern "C" int selas_raw_linear_workspace_bytes(const selas_raw_linear_problem *problems, int64_t count, int dtype,
                                                int64_t *bytes) {
  if (!bytes) return set_error(SELAS_EINVAL, "raw_linear: null result");
  *bytes = 0;
  if (int e = check_call(problems, count, dtype)) return e;
  *bytes = make_plan(problems, count).units * 16;
  return ok();
}

extern "C" int selas_raw_linear_tile(const selas_raw_linear_problem *problems, int64_t count, int dtype, int64_t *rows,
                                     int64_t *cols, int64_t *ranges) {
  if (!rows || !cols || !ranges) return set_error(SELAS_EINVAL, "raw_linear: null result");
  *rows = *cols = *ranges = 0;
  if (int e = check_call(problems, count, dtype)) return e;
  const Plan plan = make_plan(problems, count);
  *rows = plan.tile.tm;
  *cols = plan.tile.tn;
  *ranges = plan.tile.split;
  return ok();
}

extern "C" int selas_raw_linear(const selas_raw_linear_problem *problems, int64_t count, int dtype, void *workspace,
                                int64_t workspace_bytes, void *stream) {
  if (int e = check_call(problems, count, dtype)) return e;
  for (int64_t i = 0; i < count; ++i) {
    const selas_raw_linear_problem &p = problems[i];
    if (p.B * p.L == 0 || p.N == 0) continue;
    if (!p.y || (p.K && (!p.x || !p.w))) return set_error(SELAS_EINVAL, "raw_linear[%lld]: null pointer", (long long)i);
  }
  const Plan plan = make_plan(problems, count);
  if (plan.units && (!workspace || workspace_bytes < plan.units * 16 || !aligned(workspace, 16)))
    return set_error(SELAS_EINVAL, "raw_linear: needs a 16-byte aligned workspace of %lld bytes",
                     (long long)(plan.units * 16));
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint4 *ws = static_cast<uint4 *>(workspace);
  return dtype == SELAS_BF16 ? launch_plan<SELAS_BF16>(problems, count, plan, ws, s)
                             : launch_plan<SELAS_F16>(problems, count, plan, ws, s);
}
