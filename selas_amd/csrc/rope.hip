// Rotary positions with several axes (time, row, column), on gfx950.
//
// Restates qk_rms, rope_tables and apply_rope of selas/models/flux.py:106-126
// from the positions themselves instead of cos/sin tables: every image of a batch
// may stand at its own positions, a head may leave channels unrotated, and the
// pairs may be adjacent channels or the two halves of the rotated ones.
//
// HBM-bound: q and k (and v, when it is laid out on the way) are read and written
// once. A thread takes one unit of a token, two vectors of V channels that hold
// V whole pairs, forms the V angles once and applies them to its share of the
// heads, the next head's vectors in flight while one is turned; no table is read.
// The G adjacent lanes of a token (its units, rounded up to a power of two) hold a
// whole head, so the RMS sum is a short cross-lane reduction.
//
// Measured (bytes read and written at the 5.1 TB/s of a large copy: the floor): q and
// k of two clips of 20280 tokens, 24 heads of 128, fp16: 197 us (195.5, 5.06 TB/s);
// q, k and v of 4608 tokens with norms 41 us (33); one token 5.1 us. What lies between is
// the 5 to 8 us of a launch, the positions' loads and the angles ahead of the first store.
//
// Angles: pos * theta^(-2j/d) / 2 pi in fp64 (exact to 1e-11 turns at a position of
// 10^5), reduced to the nearest quarter turn there; the remainder, at most 1/8 turn,
// goes to fp32, where sin and cos are their Taylor sums up to x^11 and x^12: on |x| <=
// pi / 4 the next terms are below 2^-36.
#include <cmath>

#include "common.h"

namespace selas {
namespace {

constexpr int kMaxPairs = 128;  // Dh <= 256
constexpr float kRmsEps = 1e-6f;

// theta^(-2j / axis_dim) / (2 pi) of every pair.
struct Turns {
  double per_pos[kMaxPairs];
};

struct RopeArgs {
  selas_rope_part part[SELAS_ROPE_MAX_PARTS];
  int count, heads;  // heads: of all parts
  int tokens, L, Dh;
  FastDiv by_l;
  int pairs;         // rotated pairs, R / 2
  int axes;
  int axis_end[SELAS_ROPE_MAX_AXES];  // the pair after each axis's last
  int units, group;  // units of a token, and the lanes that hold them
  int heads_per_block;
  const void *ids;
  int64_t ids_sb, ids_sl;
  int ids_dtype;
  int inverse;
};

// sin and cos of 2 pi t.
__device__ __forceinline__ void sincos_turns(double t, float &s, float &c) {
  const double f = t - rint(t);  // [-1/2, 1/2] turns; NaN for positions that are not finite
  const double q = rint(4.0 * f);
  const float x = static_cast<float>((f - 0.25 * q) * 6.283185307179586);  // |x| <= pi / 4
  const float y = x * x;
  float ps = -1.0f / 39916800.0f, pc = 1.0f / 479001600.0f;
  ps = __builtin_fmaf(ps, y, 1.0f / 362880.0f);
  ps = __builtin_fmaf(ps, y, -1.0f / 5040.0f);
  ps = __builtin_fmaf(ps, y, 1.0f / 120.0f);
  ps = __builtin_fmaf(ps, y, -1.0f / 6.0f);
  ps = __builtin_fmaf(ps * y, x, x);
  pc = __builtin_fmaf(pc, y, -1.0f / 3628800.0f);
  pc = __builtin_fmaf(pc, y, 1.0f / 40320.0f);
  pc = __builtin_fmaf(pc, y, -1.0f / 720.0f);
  pc = __builtin_fmaf(pc, y, 1.0f / 24.0f);
  pc = __builtin_fmaf(pc, y, -0.5f);
  pc = __builtin_fmaf(pc, y, 1.0f);
  const int k = static_cast<int>(q) & 3;  // quarter turns
  const float a = (k & 1) ? pc : ps, b = (k & 1) ? ps : pc;
  s = (k & 2) ? -a : a;
  c = (k == 1 || k == 2) ? -b : b;
}

// Sum over the `group` lanes (a power of two) of a token: swaps inside quads, then mirrors of 8 and 16 lanes (each half's
// lanes are equal by then), all on the vector unit; only wider groups go through the cross-lane network.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float group_sum(float v, int group) {
  if (group > 1) v = dpp_add<0xB1>(v);    // quad_perm 1 0 3 2
  if (group > 2) v = dpp_add<0x4E>(v);    // quad_perm 2 3 0 1
  if (group > 4) v = dpp_add<0x141>(v);   // row_half_mirror
  if (group > 8) v = dpp_add<0x140>(v);   // row_mirror
  if (group > 16) v += __shfl_xor(v, 16, 64);
  if (group > 32) v += __shfl_xor(v, 32, 64);
  return v;
}

template <int DT, int V>
__device__ __forceinline__ void load_vec(const void *p, int64_t i, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = load_f<DT>(p, i);
  } else if constexpr (DT == SELAS_F32) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const float4 u = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i + j);
      v[j] = u.x; v[j + 1] = u.y; v[j + 2] = u.z; v[j + 3] = u.w;
    }
  } else {
    uint32_t w[V / 2];
    if constexpr (V == 8) {
      const uint4 u = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i);
      w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + i);
      w[0] = u.x; w[1] = u.y;
    }
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      if constexpr (DT == SELAS_BF16) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      } else {
        v[2 * j] = f16_bits_to_f32(w[j] & 0xffffu);
        v[2 * j + 1] = f16_bits_to_f32(w[j] >> 16);
      }
    }
  }
}

template <int DT, int V>
__device__ __forceinline__ void store_vec(void *p, int64_t i, const float (&v)[V]) {
  if constexpr (V == 1) {
    store_f<DT>(p, i, v[0]);
  } else if constexpr (DT == SELAS_F32) {
#pragma unroll
    for (int j = 0; j < V; j += 4)
      *reinterpret_cast<float4 *>(static_cast<float *>(p) + i + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
  } else {
    uint32_t w[V / 2];
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      if constexpr (DT == SELAS_BF16) w[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
      else w[j] = f16_bits_rne(v[2 * j]) | (static_cast<uint32_t>(f16_bits_rne(v[2 * j + 1])) << 16);
    }
    if constexpr (V == 8)
      *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
    else
      *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p) + i) = make_uint2(w[0], w[1]);
  }
}

// V channels per vector: 8 (16-bit types) or 4 where everything is aligned to that, else 1. With V = 1 a unit is
// one pair; otherwise the first vector of a rotated unit u of U starts at channel u V, the second at (U + u) V, which are
// halves of the same pairs (V divides R/2 = U V) or, for adjacent pairs, V/2 pairs each; where R / V is odd the last
// unit's second is the first unrotated vector. The others follow in pairs of vectors, the last without its second where
// one is left over.
template <int DT, int V, bool HALVES>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a, Turns turns) {
  const int group = a.group;
  const int u = threadIdx.x & (group - 1);
  const uint32_t token = blockIdx.x * (256 / group) + threadIdx.x / group;
  const bool live = token < static_cast<uint32_t>(a.tokens) && u < a.units;
  const int b = live ? static_cast<int>(div31(token, a.by_l)) : 0, l = live ? static_cast<int>(token) - b * a.L : 0;
  const int R = 2 * a.pairs, rot_units = (R + 2 * V - 1) / (2 * V);
  const bool rotated = live && u < rot_units;
  int c0, c1;
  if (u < rot_units) {
    c0 = (V == 1 && !HALVES) ? 2 * u : u * V;
    c1 = (V == 1 && !HALVES) ? 2 * u + 1 : (rot_units + u) * V;
  } else {
    c0 = 2 * u * V;
    c1 = c0 + V;
  }
  const bool two = live && c1 < a.Dh, rotated1 = rotated && c1 < R;

  float sn[V], cs[V];
  if (rotated) {
    // All of the token's positions at once: an axis looked up first would put two loads in a row.
    double pos[SELAS_ROPE_MAX_AXES] = {};
    const int64_t at = b * a.ids_sb + l * a.ids_sl;
#pragma unroll
    for (int i = 0; i < SELAS_ROPE_MAX_AXES; ++i)
      if (i < a.axes)
        pos[i] = a.ids_dtype == SELAS_F32   ? static_cast<double>(static_cast<const float *>(a.ids)[at + i])
                 : a.ids_dtype == SELAS_I32 ? static_cast<double>(static_cast<const int32_t *>(a.ids)[at + i])
                                            : static_cast<double>(static_cast<const int64_t *>(a.ids)[at + i]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      // Pair j of this unit: of its two vectors' adjacent pairs, or of its halves.
      const int i = (V == 1 || HALVES) ? u * V + j : (j < V / 2 ? c0 / 2 + j : min(c1 / 2 + j - V / 2, a.pairs - 1));
      double p = pos[0];
#pragma unroll
      for (int e = 1; e < SELAS_ROPE_MAX_AXES; ++e) p = i >= a.axis_end[e - 1] ? pos[e] : p;
      sincos_turns(p * turns.per_pos[i], sn[j], cs[j]);
      if (a.inverse) sn[j] = -sn[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) sn[j] = 0.0f, cs[j] = 1.0f;
  }

  const float inv_dh = 1.0f / static_cast<float>(a.Dh);
  const int h_lo = blockIdx.y * a.heads_per_block, h_hi = min(a.heads, h_lo + a.heads_per_block);
  int first = 0;  // of the part, in the heads of all parts
  for (int p = 0; p < a.count; ++p) {
    const selas_rope_part &part = a.part[p];
    const int heads = static_cast<int>(part.heads);
    const int lo = max(h_lo, first) - first, hi = min(h_hi, first + heads) - first;
    first += heads;
    if (lo >= hi) continue;
    const int64_t xo = b * part.x_sb + l * part.x_sl, yo = b * part.y_sb + l * part.y_sl;
    const bool turn = part.rotate != 0;
    float s0[V] = {}, s1[V] = {};
    if (part.scale) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (live) s0[j] = part.scale[c0 + j];
        if (two) s1[j] = part.scale[c1 + j];
      }
    }
    // The next head's vectors are in flight while one is turned and stored.
    float n0[V] = {}, n1[V] = {};
    auto load = [&](int h) {
      if (live) load_vec<DT, V>(part.x, xo + h * part.x_sh + c0, n0);
      if (two) load_vec<DT, V>(part.x, xo + h * part.x_sh + c1, n1);
    };
    load(lo);
    for (int h = lo; h < hi; ++h) {
      float v0[V], v1[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v0[j] = n0[j], v1[j] = n1[j];
      if (h + 1 < hi) load(h + 1);
      if (part.scale) {
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) ss += v0[j] * v0[j] + v1[j] * v1[j];
        const float r = __builtin_amdgcn_rsqf(group_sum(ss, group) * inv_dh + kRmsEps);  // within 1 ulp
#pragma unroll
        for (int j = 0; j < V; ++j) v0[j] = (v0[j] * r) * s0[j], v1[j] = (v1[j] * r) * s1[j];
      }
      if (turn && rotated) {
        if constexpr (V == 1 || HALVES) {  // rotated1 holds
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float e = v0[j], o = v1[j];
            v0[j] = e * cs[j] - o * sn[j];
            v1[j] = e * sn[j] + o * cs[j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < V / 2; ++j) {
            const float e = v0[2 * j], o = v0[2 * j + 1];
            v0[2 * j] = e * cs[j] - o * sn[j];
            v0[2 * j + 1] = e * sn[j] + o * cs[j];
          }
          if (rotated1) {
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
              const float e = v1[2 * j], o = v1[2 * j + 1];
              v1[2 * j] = e * cs[V / 2 + j] - o * sn[V / 2 + j];
              v1[2 * j + 1] = e * sn[V / 2 + j] + o * cs[V / 2 + j];
            }
          }
        }
      }
      if (live) store_vec<DT, V>(part.y, yo + h * part.y_sh + c0, v0);
      if (two) store_vec<DT, V>(part.y, yo + h * part.y_sh + c1, v1);
    }
  }
}

// Whether every vector of `bytes` bytes (V elements) that the kernel would access is aligned, and the rotated channels are
// whole vectors: two for each unit with halves, and with vectors of 8 (where that fails for 8, it holds for 4). Against
// single elements, q and k of 4608 tokens, 24 heads, bf16, adjacent pairs: 72 channels of which 36 turn 46 -> 21 us, 128 of
// which 124 turn 47 -> 24.
bool rope_vec_ok(const RopeArgs &a, int V, int esize, bool halves) {
  if (a.Dh % V || (halves || V == 8 ? a.pairs : 2 * a.pairs) % V) return false;
  const uintptr_t bytes = static_cast<uintptr_t>(V) * esize > 16 ? 16 : static_cast<uintptr_t>(V) * esize;
  for (int i = 0; i < a.count; ++i) {
    const selas_rope_part &p = a.part[i];
    if (!aligned(p.x, bytes) || !aligned(p.y, bytes) || p.x_sb % V || p.x_sh % V || p.x_sl % V || p.y_sb % V ||
        p.y_sh % V || p.y_sl % V)
      return false;
  }
  return true;
}

}  // namespace
}  // namespace selas

using namespace selas;

extern "C" int selas_rope(const selas_rope_part *parts, int64_t count, int64_t B, int64_t L, int64_t Dh,
                          const void *ids, int ids_dtype, int64_t ids_sb, int64_t ids_sl, int64_t axes,
                          const int64_t *axis_dim, double theta, int halves, int inverse, int dtype, void *stream) {
  if (count < 1 || count > SELAS_ROPE_MAX_PARTS || !parts)
    return set_error(SELAS_EINVAL, "rope: takes 1 to %d tensors, got %lld", SELAS_ROPE_MAX_PARTS, (long long)count);
  if (axes < 1 || axes > SELAS_ROPE_MAX_AXES || !axis_dim)
    return set_error(SELAS_EINVAL, "rope: takes 1 to %d axes, got %lld", SELAS_ROPE_MAX_AXES, (long long)axes);
  if (B < 0 || L < 0 || Dh <= 0) return set_error(SELAS_EINVAL, "rope: bad shape B=%lld L=%lld Dh=%lld", (long long)B,
                                                  (long long)L, (long long)Dh);
  if (!valid_dtype(dtype)) return set_error(SELAS_EINVAL, "rope: bad dtype %d", dtype);
  if (ids_dtype != SELAS_F32 && ids_dtype != SELAS_I32 && ids_dtype != SELAS_I64)
    return set_error(SELAS_EINVAL, "rope: positions are fp32, int32 or int64 (dtype %d)", ids_dtype);
  if (!(theta > 0.0) || std::isinf(theta)) return set_error(SELAS_EINVAL, "rope: theta must be positive");
  int64_t R = 0;
  for (int64_t i = 0; i < axes; ++i) {
    if (axis_dim[i] < 0 || axis_dim[i] % 2 || axis_dim[i] > Dh)
      return set_error(SELAS_EINVAL, "rope: axis %lld has %lld channels (even, at most the head's %lld)", (long long)i,
                       (long long)axis_dim[i], (long long)Dh);
    R += axis_dim[i];
  }
  if (R > Dh) return set_error(SELAS_EINVAL, "rope: the axes have %lld channels, the heads %lld", (long long)R,
                               (long long)Dh);
  RopeArgs a{};
  a.count = static_cast<int>(count);
  int64_t heads = 0;
  for (int64_t i = 0; i < count; ++i) {
    const selas_rope_part &p = parts[i];
    if (p.heads < 0 || p.x_sb < 0 || p.x_sh < 0 || p.x_sl < 0 || p.y_sb < 0 || p.y_sh < 0 || p.y_sl < 0)
      return set_error(SELAS_EINVAL, "rope: negative heads or strides");
    if (inverse && p.scale) return set_error(SELAS_EINVAL, "rope: the inverse rotation takes no norm");
    if (p.heads && B && L && (!p.x || !p.y)) return set_error(SELAS_EINVAL, "rope: null tensor");
    a.part[i] = p;
    heads += p.heads;
  }
  if (B == 0 || L == 0 || heads == 0) return ok();
  if (R && (!ids || ids_sb < 0 || ids_sl < 0)) return set_error(SELAS_EINVAL, "rope: positions missing");
  if (Dh > 2 * kMaxPairs) return set_error(SELAS_EUNSUPPORTED, "rope: head_dim %lld is above %d", (long long)Dh,
                                           2 * kMaxPairs);
  if (B >= (1ll << 31) || L >= (1ll << 31) || B * L >= (1ll << 31) || heads >= (1ll << 16))
    return set_error(SELAS_EUNSUPPORTED, "rope: too many tokens or heads");
  a.heads = static_cast<int>(heads);
  a.tokens = static_cast<int>(B * L);
  a.L = static_cast<int>(L);
  a.by_l = fast_div(static_cast<uint32_t>(L));
  a.Dh = static_cast<int>(Dh);
  a.pairs = static_cast<int>(R / 2);
  a.ids = ids;
  a.ids_sb = ids_sb;
  a.ids_sl = ids_sl;
  a.ids_dtype = ids_dtype;
  a.inverse = inverse != 0;
  Turns turns{};
  a.axes = static_cast<int>(axes);
  int pairs = 0;
  for (int i = 0; i < SELAS_ROPE_MAX_AXES; ++i) {
    // The power of theta of pair j: pow where j is a power of two, otherwise the product of j's lowest bit's and the
    // rest's, at most six roundings of 64 bits from it (a call of pow per pair took 2 us of a launch).
    double *const t = turns.per_pos + pairs;
    const int n = i < axes ? static_cast<int>(axis_dim[i] / 2) : 0;
    for (int j = 0; j < n; ++j) {
      const int low = j & -j;
      t[j] = j == 0 ? 1.0 : j == low ? std::pow(theta, -2.0 * j / static_cast<double>(axis_dim[i])) : t[j - low] * t[low];
    }
    for (int j = 0; j < n; ++j) t[j] /= 6.283185307179586;
    pairs += n;
    a.axis_end[i] = pairs;
  }
  const int esize = dtype == SELAS_F32 ? 4 : 2;
  const int V = dtype != SELAS_F32 && rope_vec_ok(a, 8, esize, halves != 0) ? 8 : rope_vec_ok(a, 4, esize, halves != 0) ? 4 : 1;
  a.units = static_cast<int>(cdiv(Dh, 2 * V));
  a.group = 1;
  while (a.group < a.units) a.group *= 2;
  if (a.group > 64)
    return set_error(SELAS_EUNSUPPORTED, "rope: heads of %lld channels off 4-element alignment (%lld rotated%s)", (long long)Dh,
                     (long long)R, halves ? " in halves" : "");
  // Heads per thread: the fewest that leave no more than 4 workgroups per CU of 256, which are resident at once (90
  // registers allow 5). A thread's positions, angles and scales then serve as many heads as possible, and no second round
  // pays for them again (image of 4608 tokens, us: 41.3 with 1152 workgroups, 46 with 1728, 50 with 1296 of which 16 wait).
  const int64_t blocks = cdiv(B * L, 256 / a.group);
  int64_t hpb = 1;
  while (hpb < heads && blocks * cdiv(heads, hpb) > 4 * 256) ++hpb;
  a.heads_per_block = static_cast<int>(hpb);
  const dim3 grid(static_cast<uint32_t>(blocks), static_cast<uint32_t>(cdiv(heads, hpb))), blk(256);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define SELAS_ROPE(DT, VV)                                               \
  do {                                                                   \
    if (halves) rope_kernel<DT, VV, true><<<grid, blk, 0, s>>>(a, turns); \
    else rope_kernel<DT, VV, false><<<grid, blk, 0, s>>>(a, turns);       \
  } while (0)
#define SELAS_ROPE_16(DT)                  \
  do {                                     \
    if (V == 8) SELAS_ROPE(DT, 8);         \
    else if (V == 4) SELAS_ROPE(DT, 4);    \
    else SELAS_ROPE(DT, 1);                \
  } while (0)
  if (dtype == SELAS_BF16) SELAS_ROPE_16(SELAS_BF16);
  else if (dtype == SELAS_F16) SELAS_ROPE_16(SELAS_F16);
  else if (V == 4) SELAS_ROPE(SELAS_F32, 4);
  else SELAS_ROPE(SELAS_F32, 1);
#undef SELAS_ROPE_16
#undef SELAS_ROPE
  return check_launch("rope");
}
