// Linear with an unquantized weight and the block's epilogue, on gfx950:
//   y[b, l, n] = residual[b, l, n] + gate[b, n] * act(sum_k x[b, l, k] w[n, k] + bias[n])
//
// UnitView.linear for raw weights (selas/store.py:289-293) together with what follows
// it in a block: the GELU or SiLU (flux.py:150-151, 194-195) and the gated residual add
// (flux.py:169-171). The sum, the activation, the gate and the residual stay in fp32 and
// are rounded once, to the output's type.
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
};

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

// x / (1 + e^-x) by the hardware base-2 exponential and reciprocal, like gelu_tanh_fast.
__device__ __forceinline__ float silu_fast(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}

__device__ __forceinline__ float activate(float v, int act) {
  return act == SELAS_ACT_GELU ? gelu_tanh_fast(v) : act == SELAS_ACT_SILU ? silu_fast(v) : v;
}

template <int DT>
__device__ __forceinline__ float load_either(const void *p, int64_t i, bool f32) {
  return f32 ? static_cast<const float *>(p)[i] : load_f<DT>(p, i);
}

// Eight elements of a row from k on, zeros from K on. The address need not be aligned: global loads may start at any
// element.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
__device__ __forceinline__ uint4 load_chunk(const uint16_t *row, int k, int K) {
  if (k + 8 <= K) return __builtin_bit_cast(uint4, static_cast<u32x4>(*reinterpret_cast<const u32x4_any *>(row + k)));
  uint32_t w[4] = {};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (k + j < K) w[j / 2] |= static_cast<uint32_t>(row[k + j]) << (16 * (j & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// ------------------------------------------------------------------ any layout
//
// 4 waves, 64 x 64 outputs, 64 columns of K per step, staged through registers (the next step's loads are in flight
// during this step's products). Rows of 128 bytes in LDS, their 16-byte chunks XOR-swizzled by (row / 2) % 8 so that the
// 16 rows of a fragment read lie in distinct groups of the 64 banks.
constexpr int kAnyT = 64;

template <int DT>
__global__ __launch_bounds__(256) void raw_any_kernel(RawProblem P) {
  __shared__ uint4 xs[kAnyT * 8], ws[kAnyT * 8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int m0 = blockIdx.y * kAnyT, n0 = blockIdx.x * kAnyT;
  // Thread t loads chunks t % 8 of rows t / 8 and t / 8 + 32 of each operand.
  const int c = tid & 7;
  const uint16_t *xr[2], *wr[2];
  int dst[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = (tid >> 3) + 32 * i;
    const int m = m0 + r, n = n0 + r;
    const int b = static_cast<int>(div31(static_cast<uint32_t>(min(m, P.M - 1)), P.by_l));
    const int l = min(m, P.M - 1) - b * P.L;
    xr[i] = static_cast<const uint16_t *>(P.x) + b * P.x_sb + l * P.x_sl;
    wr[i] = static_cast<const uint16_t *>(P.w) + static_cast<int64_t>(min(n, P.N - 1)) * P.ldw;
    dst[i] = r * 8 + (c ^ ((r >> 1) & 7));
  }
  uint4 xv[2], wv[2];
  auto load = [&](int k) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      xv[i] = load_chunk(xr[i], k + 8 * c, P.K);
      wv[i] = load_chunk(wr[i], k + 8 * c, P.K);
    }
  };
  f32x4 acc[2][2] = {};
  const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
  auto frag = [&](const uint4 *s, int r, int kc) { return s[r * 8 + (kc ^ ((r >> 1) & 7))]; };
  if (P.K > 0) load(0);
  for (int k = 0; k < P.K; k += 64) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) xs[dst[i]] = xv[i], ws[dst[i]] = wv[i];
    __syncthreads();
    if (k + 64 < P.K) load(k + 64);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      uint4 a[2], b[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        a[i] = frag(ws, wn + 16 * i + (lane & 15), 4 * s + (lane >> 4));
        b[i] = frag(xs, wm + 16 * i + (lane & 15), 4 * s + (lane >> 4));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma16<DT>(a[i], b[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int m = m0 + wm + 16 * j + (lane & 15);
    if (m >= P.M) continue;
    const int b = static_cast<int>(div31(static_cast<uint32_t>(m), P.by_l)), l = m - b * P.L;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = n0 + wn + 16 * i + 4 * (lane >> 4) + r;
        if (n >= P.N) continue;
        float v = acc[i][j][r];
        if (P.bias) v += load_either<DT>(P.bias, n, P.bias_f32);
        v = activate(v, P.act);
        if (P.gate) v *= load_either<DT>(P.gate, b * P.gate_sb + n, P.gate_f32);
        if (P.residual) v += load_either<DT>(P.residual, b * P.r_sb + l * P.r_sl + n, P.residual_f32);
        const int64_t o = b * P.y_sb + l * P.y_sl + n;
        if (P.y_f32) static_cast<float *>(P.y)[o] = v;
        else store_f<DT>(P.y, o, v);
      }
  }
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

RawProblem make_problem(const selas_raw_linear_problem &p) {
  RawProblem r{};
  r.x = p.x; r.w = p.w; r.bias = p.bias; r.gate = p.gate; r.residual = p.residual; r.y = p.y;
  r.x_sb = p.x_sb; r.x_sl = p.x_sl; r.ldw = p.ldw; r.gate_sb = p.gate_sb;
  r.r_sb = p.r_sb; r.r_sl = p.r_sl; r.y_sb = p.y_sb; r.y_sl = p.y_sl;
  r.M = static_cast<int>(p.B * p.L); r.L = static_cast<int>(p.L);
  r.N = static_cast<int>(p.N); r.K = static_cast<int>(p.K);
  r.by_l = fast_div(static_cast<uint32_t>(p.L));
  r.act = p.act;
  r.bias_f32 = p.bias_dtype == SELAS_F32; r.gate_f32 = p.gate_dtype == SELAS_F32;
  r.residual_f32 = p.residual_dtype == SELAS_F32; r.y_f32 = p.y_dtype == SELAS_F32;
  return r;
}

template <int DT>
int launch_any(const RawProblem &P, hipStream_t s) {
  const int64_t tn = cdiv(P.N, kAnyT), tm = cdiv(P.M, kAnyT);
  if (tm > 65535) return set_error(SELAS_EUNSUPPORTED, "raw_linear: too many rows (%d)", P.M);
  raw_any_kernel<DT><<<dim3(static_cast<uint32_t>(tn), static_cast<uint32_t>(tm)), dim3(256), 0, s>>>(P);
  return check_launch("raw_linear");
}

int check_call(const selas_raw_linear_problem *problems, int64_t count, int dtype) {
  if (count < 0 || count > SELAS_MAX_BATCHED_LINEARS || (count && !problems))
    return set_error(SELAS_EINVAL, "raw_linear: takes up to %d problems, got %lld", SELAS_MAX_BATCHED_LINEARS,
                     (long long)count);
  if (!valid_dtype(dtype)) return set_error(SELAS_EINVAL, "raw_linear: bad dtype %d", dtype);
  if (dtype == SELAS_F32) return set_error(SELAS_EUNSUPPORTED, "raw_linear: takes bf16 or fp16 weights");
  for (int64_t i = 0; i < count; ++i)
    if (int e = check_problem(problems[i], i, dtype)) return e;
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
  (void)workspace, (void)workspace_bytes;
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (int64_t i = 0; i < count; ++i) {
    const selas_raw_linear_problem &p = problems[i];
    if (p.B * p.L == 0 || p.N == 0) continue;
    const RawProblem P = make_problem(p);
    if (int e = dtype == SELAS_BF16 ? launch_any<SELAS_BF16>(P, s) : launch_any<SELAS_F16>(P, s)) return e;
  }
  return ok();
}
