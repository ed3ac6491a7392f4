// Attention of the text side, forward, for gfx950: keys of another length than the queries, shared key heads, images whose
// keys end early or are masked, a causal mask, and a learned bias by buckets of the distance. Per image b, head h and key
// head g = h / (H / Hk):
//   s_ij = scale q_i . k_j + table[bucket(j - (start_b + i)), h],   out_i = sum_j softmax_j(s_ij) v_j
// over the keys that row i sees; a row that sees none gives zeros. Scores, maxima and sums are fp32; the running maximum and
// sum make it one pass over the keys.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "text_attention.h"

namespace selas {
namespace textattn {
namespace {

// ------------------------------------------------------------------ few rows

// Rows (query head in the group, query) that share one key head: R of them at most, `rows` = group * Lq. A row is
// r = g * Lq + i.
//
// Bounded by the stream of k and v: 4 bytes a key and channel for 2 R multiply-adds, so plain vector instructions are
// enough (MFMAs would fill 1 to 8 of their 32 columns). A lane holds 8 channels; D / 8 lanes make a key, 64 / (D / 8) key
// slots a wave; each slot keeps a softmax of its own over the keys it meets, joined once at the end. k and v go from memory
// to registers, the next unit's loads ahead of this one's arithmetic: units of 8 keys a slot hold 16 KiB a wave in flight.
// From 3 rows on the registers of a softmax per row and key leave room for units of 2: us with 2 / 4 / 8, 64 x 8 key heads of 64
// and 4 rows over 2048 keys 56 / 90 / 220, 16 x 8 key heads of 128 and 4 rows 36 / 55 / 148, 16 x 4 of 64 and 8 rows over up to
// 2048 keys 23 / 28 / 69; where 4 key heads alone leave a workgroup or two to a CU 4 are ahead (32,768 keys, 4 rows: 81 / 59 /
// 95). 64 x 32 heads of 64, one row over 2048 keys: 215 us, 5.0 TB/s; 16 x 32: 57.
template <int D, int R>
struct Few {
  static constexpr int kLanes = D / 8, kSlots = 64 / kLanes;
  static constexpr int kU = R <= 2 ? 8 : 2;  // keys of a slot per unit
  static constexpr int kUnit = kU * kSlots;        // keys per wave and step (at most 64)
  static constexpr int kFloats = R * (D + 2);      // a part's result: R x D outputs, maxima, sums
};

// Sum over the D / 8 neighbouring lanes of a key.
template <int LANES>
__device__ __forceinline__ float key_sum(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  v += dpp(v, std::integral_constant<int, 0xB1>{});   // quad_perm 1 0 3 2
  v += dpp(v, std::integral_constant<int, 0x4E>{});   // quad_perm 2 3 0 1
  v += dpp(v, std::integral_constant<int, 0x141>{});  // row_half_mirror: the other four of 8
  if constexpr (LANES == 16) v += dpp(v, std::integral_constant<int, 0x140>{});  // row_mirror: the other eight of 16
  return v;
}

// Eight products, two an instruction, summed in fp32.
template <bool BF>
__device__ __forceinline__ float dot8(uint4 a, uint4 b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF)
      s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x[i]), __builtin_bit_cast(bf16x2, y[i]), s, false);
    else
      s = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, x[i]), __builtin_bit_cast(f16x2, y[i]), s, false);
  }
  return s;
}

template <bool BF, int D, int R, int NW, bool BIAS>
__global__ __launch_bounds__(64 * NW, R == 4 ? 4 : 2) void few_kernel(Args a, int parts, float *__restrict__ partial) {
  using F = Few<D, R>;
  constexpr int kSlots = F::kSlots, kU = F::kU, kUnit = F::kUnit;
  extern __shared__ __attribute__((aligned(16))) float table[];  // [group][2 reach + 1], by distance
  __shared__ float red[NW][F::kFloats];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int part = blockIdx.x % parts, item = blockIdx.x / parts, b = item / a.Hk, hk = item - b * a.Hk;
  const int rows = a.group * a.Lq;
  const int keys = keys_of(a, b), start = start_of(a, b);
  const int slot = lane / F::kLanes, ch = (lane % F::kLanes) * 8;
  const bool given = ch < a.dh;

  const int reach = a.bias.reach, span = 2 * reach + 1;
  if constexpr (BIAS) {
    for (int i = threadIdx.x; i < a.group * span; i += 64 * NW) {
      const int g = i / span;
      table[i] = bias_at(a.bias, hk * a.group + g, i - g * span - reach, kLog2e);
    }
    __syncthreads();
  }

  uint4 qf[R];
  int at[R], head[R];  // position, head in the group
#pragma unroll
  for (int r = 0; r < R; ++r) {
    head[r] = r < rows ? r / a.Lq : 0;
    const int i = r < rows ? r - head[r] * a.Lq : 0;
    at[r] = start + i;
    const uint16_t *p = a.q.p + b * a.q.sb + (hk * a.group + head[r]) * a.q.sh + i * a.q.sl + ch;
    qf[r] = given && r < rows ? *reinterpret_cast<const uint4 *>(p) : make_uint4(0, 0, 0, 0);
  }

  const uint16_t *kp = a.k.p + b * a.k.sb + hk * a.k.sh, *vp = a.v.p + b * a.v.sb + hk * a.v.sh;
  const uint8_t *mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
  const uint32_t koff = given ? slot * static_cast<uint32_t>(2 * a.k.sl) + 2 * ch : kPast;
  const uint32_t voff = given ? slot * static_cast<uint32_t>(2 * a.v.sl) + 2 * ch : kPast;
  auto bytes_of = [&](int64_t sl, int n) {
    n = min(n, kUnit);
    return n > 0 ? 2 * ((n - 1) * static_cast<uint32_t>(sl) + a.dh) : 0u;
  };
  uint4 kf[kU], vf[kU];
  auto load_k = [&](int unit) {
    const int64_t key0 = static_cast<int64_t>(unit) * kUnit;
    const __amdgpu_buffer_rsrc_t r = make_rsrc(kp + key0 * a.k.sl, bytes_of(a.k.sl, keys - static_cast<int>(key0)));
#pragma unroll
    for (int u = 0; u < kU; ++u) kf[u] = load_b128(r, koff, u * kSlots * static_cast<uint32_t>(2 * a.k.sl));
  };
  auto load_v = [&](int unit, uint64_t bits) {  // masked values read as zeros: what they hold must not reach a product
    const int64_t key0 = static_cast<int64_t>(unit) * kUnit;
    const __amdgpu_buffer_rsrc_t r = make_rsrc(vp + key0 * a.v.sl, bytes_of(a.v.sl, keys - static_cast<int>(key0)));
#pragma unroll
    for (int u = 0; u < kU; ++u)
      vf[u] = load_b128(r, (bits >> (u * kSlots + slot)) & 1 ? voff : kPast, u * kSlots * static_cast<uint32_t>(2 * a.v.sl));
  };
  auto load_byte = [&](int unit) {
    const int64_t key = static_cast<int64_t>(unit) * kUnit + lane;
    return mask && lane < kUnit && key < keys ? mask[key] : 0;
  };
  auto word = [&](int unit, int byte) {
    if (mask) return __builtin_amdgcn_ballot_w64(byte != 0);
    return up_to(keys - unit * kUnit - 1);
  };

  // This part's units, dealt to the waves in turn.
  int n = (keys + kUnit - 1) / kUnit;
  if (a.causal) n = min(n, max(start + a.Lq + kUnit - 1, 0) / kUnit);
  const int per = (n + parts - 1) / parts, end = min(n, (part + 1) * per);
  int unit = uniform(part * per + wave);

  float m[R], l[R], o[R][8];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = kLowest;
    l[r] = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[r][e] = 0.0f;
  }

  uint64_t bits = 0, bits_next = 0;
  int byte = 0;
  if (unit < end) {
    bits = word(unit, load_byte(unit));
    load_k(unit);
    load_v(unit, bits);
    byte = load_byte(unit + NW);
  }
  for (; unit < end; unit += NW) {
    const int next = unit + NW;
    bits_next = word(next, byte);
    float s[kU][R];
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int r = 0; r < R; ++r) s[u][r] = key_sum<F::kLanes>(dot8<BF>(kf[u], qf[r]));
    if (next < end) load_k(next);
    byte = load_byte(next + NW);
    float p[kU][R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float mx = m[r];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int key = unit * kUnit + u * kSlots + slot, d = key - at[r];
        float x = s[u][r] * a.c2;
        if constexpr (BIAS) x += table[head[r] * span + min(max(d, -reach), reach) + reach];
        const bool seen = ((bits >> (u * kSlots + slot)) & 1) && !(a.causal && d > 0);
        s[u][r] = seen ? x : -__builtin_inff();
        mx = fmaxf(mx, s[u][r]);
      }
      const float alpha = __builtin_amdgcn_exp2f(m[r] - mx);
      m[r] = mx;
      l[r] *= alpha;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[r][e] *= alpha;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        p[u][r] = __builtin_amdgcn_exp2f(s[u][r] - mx);
        l[r] += p[u][r];
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const uint32_t w[4] = {vf[u].x, vf[u].y, vf[u].z, vf[u].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float lo = lo_of<BF>(w[e]), hi = hi_of<BF>(w[e]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          o[r][2 * e] = __builtin_fmaf(p[u][r], lo, o[r][2 * e]);
          o[r][2 * e + 1] = __builtin_fmaf(p[u][r], hi, o[r][2 * e + 1]);
        }
      }
    }
    bits = bits_next;
    if (next < end) load_v(next, bits);
  }

  // The slots of a wave, then the waves.
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int x = F::kLanes; x < 64; x <<= 1) {
      const float om = __shfl_xor(m[r], x, 64), ol = __shfl_xor(l[r], x, 64), mx = fmaxf(m[r], om);
      const float f = __builtin_amdgcn_exp2f(m[r] - mx), g = __builtin_amdgcn_exp2f(om - mx);
      l[r] = l[r] * f + ol * g;
      m[r] = mx;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[r][e] = o[r][e] * f + __shfl_xor(o[r][e], x, 64) * g;
    }
    if (slot == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) red[wave][r * D + ch + e] = o[r][e];
      if (ch == 0) {
        red[wave][R * D + r] = m[r];
        red[wave][R * D + R + r] = l[r];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * D; i += 64 * NW) {
    const int r = i / D, c = i - r * D;
    if (r >= rows) continue;
    float mx = kLowest, sum = 0.0f, x = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, red[w][R * D + r]);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(red[w][R * D + r] - mx);
      sum += red[w][R * D + R + r] * f;
      x += red[w][i] * f;
    }
    if (parts > 1) {
      float *out = partial + static_cast<int64_t>(blockIdx.x) * F::kFloats;
      out[i] = x;
      if (c == 0) {
        out[R * D + r] = mx;
        out[R * D + R + r] = sum;
      }
      continue;
    }
    const int g = r / a.Lq, q = r - g * a.Lq, h = hk * a.group + g;
    if (c < a.dh)
      store_f<BF ? SELAS_BF16 : SELAS_F16>(a.out + b * a.out_sb + q * a.out_sl + h * a.dh, c, sum == 0.0f ? 0.0f : x / sum);
    if (a.lse && c == 0) a.lse[(static_cast<int64_t>(b) * a.H + h) * a.Lq + q] = (mx + __builtin_log2f(sum)) * kLn2;
  }
}

// The parts of few_kernel, joined in their order: a workgroup per (image, key head, row).
template <bool BF>
__global__ __launch_bounds__(128) void few_merge_kernel(Args a, int parts, int D, int R, const float *__restrict__ partial) {
  const int rows = a.group * a.Lq, item = blockIdx.x / rows, r = blockIdx.x - item * rows, c = threadIdx.x;
  const int b = item / a.Hk, hk = item - b * a.Hk, step = R * (D + 2);
  const float *w = partial + static_cast<int64_t>(item) * parts * step;
  if (c >= a.dh) return;
  float mx = kLowest, sum = 0.0f, x = 0.0f;
  for (int p = 0; p < parts; ++p) mx = fmaxf(mx, w[p * step + R * D + r]);
  for (int p = 0; p < parts; ++p) {
    const float f = __builtin_amdgcn_exp2f(w[p * step + R * D + r] - mx);
    sum += w[p * step + R * D + R + r] * f;
    x += w[p * step + r * D + c] * f;
  }
  const int g = r / a.Lq, q = r - g * a.Lq, h = hk * a.group + g;
  store_f<BF ? SELAS_BF16 : SELAS_F16>(a.out + b * a.out_sb + q * a.out_sl + h * a.dh, c, sum == 0.0f ? 0.0f : x / sum);
  if (a.lse && c == 0) a.lse[(static_cast<int64_t>(b) * a.H + h) * a.Lq + q] = (mx + __builtin_log2f(sum)) * kLn2;
}

// ------------------------------------------------------------------ tiles

// A call cut into work items of NW blocks of 32 rows: the blocks of one query head, or (pack) of all the heads of a group one
// after another, so that few queries of several heads share their key head's tiles. Parts of the keys are outside the blocks
// and the heads of a group, so that what reads the same keys runs at the same time behind the same L2.
struct Cut {
  int qblocks;  // of 32 queries, per head
  int tiles;    // items per head, or per group (pack)
  int parts, pack;
  Deal deal;
  FastDiv by_tiles, by_group, by_parts, by_hk, by_qblocks;
  float *partial;
};
constexpr int partial_floats(int D) { return 64 * (D / 2) + 2 * 64; }  // per wave: outputs in register order, maxima, sums

// What a workgroup has to know of an item. Uniform but for the wave's share.
struct Item {
  int b, hk, head;  // head: of this wave
  int row0;         // this wave's first query (Lq: no rows)
  int keys, start, kt, end;
  const uint16_t *kp, *vp;
};

__device__ __forceinline__ Item item_at(const Args &a, const Cut &cut, int t, int nw, int wave) {
  Item x;
  int rest, g = 0;
  const int tile0 = split(t, cut.by_tiles, cut.tiles, rest);
  if (!cut.pack) g = split(rest, cut.by_group, a.group, rest);
  const int part = split(rest, cut.by_parts, cut.parts, rest);
  x.hk = split(rest, cut.by_hk, a.Hk, x.b);
  const int tile = a.causal ? cut.tiles - 1 - tile0 : tile0;  // the longest first
  int block = tile * nw + wave;
  if (cut.pack) block = split(block, cut.by_qblocks, cut.qblocks, g);
  x.row0 = g < a.group ? min(32 * block, a.Lq) : a.Lq;
  x.head = x.hk * a.group + min(g, a.group - 1);
  x.keys = keys_of(a, x.b);
  x.start = start_of(a, x.b);
  int n = (x.keys + kRows - 1) / kRows;
  if (a.causal) n = min(n, max(x.start + min((tile + 1) * nw * 32, a.Lq) + kRows - 1, 0) / kRows);
  const int per = static_cast<int>(div31(n + cut.parts - 1, cut.by_parts));
  x.kt = part * per;
  x.end = max(min(n, x.kt + per), x.kt + 1);  // without keys: one tile of which nothing is seen
  x.kp = a.k.p + x.b * a.k.sb + x.hk * a.k.sh;
  x.vp = a.v.p + x.b * a.v.sb + x.hk * a.v.sh;
  return x;
}

// One workgroup = NW waves = NW blocks of 32 queries. The keys stream through LDS in double-buffered tiles of 64 that all
// waves share. Per tile: S^T = K Q^T (K row-wise from LDS, Q held), the softmax on the scores in registers, O^T += V^T P^T
// (V transposed by the LDS reads, the probabilities straight from the score registers: the K rows of a block are read with
// bits 2 and 3 of the row exchanged, so that register r of a lane holds key 16 (r / 8) + 8 h + r % 8 of it, as the second
// product's operand wants them). Three workgroups a CU; with 128 channels and a bias 4 registers spill for that.
template <bool BF, int D, int NW, bool BIAS>
__global__ __launch_bounds__(64 * NW, NW >= 4 ? 3 : 1) void fwd_kernel(Args a, Cut cut) {
  using T = TileOf<D>;
  constexpr int KJ = T::kLoads / NW;
  static_assert(KJ * NW == T::kLoads, "loads per wave");
  constexpr bool kTwo = D == 64;  // two stages of the values as well
  __shared__ __attribute__((aligned(16))) uint8_t keys0[T::kBytes], keys1[T::kBytes], values0[T::kBytes];
  __shared__ __attribute__((aligned(16))) uint8_t values1[kTwo ? T::kBytes : 16];
  extern __shared__ __attribute__((aligned(16))) float table[];  // the head's bias by distance
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5, c = lane & 31;
  const int t = item_of(cut.deal);
  if (t >= cut.deal.total) return;
  const Item x = item_at(a, cut, t, NW, wave);
  const KeyBits keybits(a, x.b, x.keys, lane);
  const typename T::template Loader<KJ> kl(wave, lane, a.k.sl, a.dh), vl(wave, lane, a.v.sl, a.dh);
  const typename T::RowReader rows(lane);
  const typename T::ColReader cols(lane);
  const int reach = a.bias.reach, pitch = bias_pitch(reach);

  auto issue_keys = [&](int stage, int kt, uint64_t bits) __attribute__((always_inline)) {
    uint8_t *to = stage ? keys1 : keys0;
    const uint16_t *p = x.kp + static_cast<int64_t>(kt) * kRows * a.k.sl;
    const int left = x.keys - kt * kRows;
    if (a.mask) kl.template issue<true>(to, p, a.k.sl, a.dh, left, bits);
    else kl.template issue<false>(to, p, a.k.sl, a.dh, left, bits);
  };
  auto issue_values = [&](int stage, int kt, uint64_t bits) __attribute__((always_inline)) {
    uint8_t *to = kTwo && stage ? values1 : values0;
    const uint16_t *p = x.vp + static_cast<int64_t>(kt) * kRows * a.v.sl;
    const int left = x.keys - kt * kRows;
    if (a.mask) vl.template issue<true>(to, p, a.v.sl, a.dh, left, bits);
    else vl.template issue<false>(to, p, a.v.sl, a.dh, left, bits);
  };
  int kt = x.kt;
  uint64_t bits = keybits.word(kt, keybits.load(kt));
  int byte = keybits.load(kt + 1);  // mask bytes a tile ahead of the loads that they are for
  Held<D> q;
  issue_keys(0, kt, bits);
  if (kTwo) issue_values(0, kt, bits);
  q.load(a.q.p + x.b * a.q.sb + x.head * a.q.sh + x.row0 * a.q.sl, a.q.sl, a.dh, a.Lq - x.row0, lane);
  if constexpr (BIAS) build_bias(table, a.bias, x.head, 64 * NW, false);

  f32x16 o[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) o[db] = f32x16{};
  float m_run = kLowest, l_run = 0.0f;
  constexpr float kRoom = headroom<BF>();

  // The probabilities of a tile. near: the bias differs among its scores (otherwise it is `bc`, times log2(e), for all); part:
  // some are not seen.
  uint4 pb[2][2];
  auto scores = [&](int stage, float bc, bool near, bool part) __attribute__((always_inline)) {
    const uint8_t *ks = stage ? keys1 : keys0;
    const int pos = x.start + x.row0 + c;
    f32x16 sc[2] = {f32x16{}, f32x16{}};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < D / 16; ++i) sc[kb] = mfma<BF>(rows.read(ks, kb, i), q.f[i], sc[kb]);
    if (BIAS && near) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
          float bv[8];
          bias_run(table, pitch, reach, kt * kRows + 32 * kb + 16 * t2 + 8 * h - pos, bv);
#pragma unroll
          for (int e = 0; e < 8; ++e) sc[kb][8 * t2 + e] += bv[e];
        }
    }
    if (part) {
      const uint64_t seen = (a.causal ? bits & up_to(pos - kt * kRows) : bits) >> (8 * h);
      const uint32_t w[2] = {static_cast<uint32_t>(seen), static_cast<uint32_t>(seen >> 32)};
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          sc[kb][r] = (w[kb] >> (16 * (r >> 3) + (r & 7))) & 1 ? sc[kb][r] : -__builtin_inff();
    }
    float mx = sc[0][0];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[kb][r]);
    mx = __builtin_fmaf(pair_max(mx), a.c2, bc);
    const bool raise = mx - kRoom > m_run + 8.0f;
    if (__builtin_amdgcn_ballot_w64(raise)) {
      const float to = mx - kRoom, alpha = raise ? __builtin_amdgcn_exp2f(m_run - to) : 1.0f;
#pragma unroll
      for (int db = 0; db < D / 32; ++db) o[db] *= alpha;
      l_run *= alpha;
      m_run = raise ? to : m_run;
    }
    const float sub = m_run - bc;
    float ls = 0.0f;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          auto prob = [&](float s) {
            return materialize(__builtin_amdgcn_exp2f(__builtin_fmaf(s, a.c2, -sub)));
          };
          const float p0 = prob(sc[kb][8 * t2 + 2 * e]), p1 = prob(sc[kb][8 * t2 + 2 * e + 1]);
          ls += p0 + p1;
          w[e] = pack<BF>(p0, p1);
        }
        pb[kb][t2] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    l_run += ls;
  };
  auto products = [&](int stage) __attribute__((always_inline)) {
    uint8_t *vs = kTwo && stage ? values1 : values0;
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
      o[i / 4] = mfma<BF>(cols.read(vs, i / 4, (i / 2) % 2, i % 2), pb[(i / 2) % 2][i % 2], o[i / 4]);
  };

  auto step = [&](int stage) __attribute__((always_inline)) {
    const bool more = kt + 1 < x.end;
    uint64_t bits_next = 0;
    if (more) {
      bits_next = keybits.word(kt + 1, byte);
      issue_keys(stage ^ 1, kt + 1, bits_next);
      if (kTwo) issue_values(stage ^ 1, kt + 1, bits_next);
      byte = keybits.load(kt + 2);
    }
    const int key0 = kt * kRows, first = x.start + x.row0;
    const bool any = bits && !(a.causal && key0 > first + 31);
    if (any) {
      const bool all = bits == ~0ull && !(a.causal && key0 + kRows - 1 > first);
      bool near = BIAS;
      float bc = 0.0f;
      if constexpr (BIAS) {
          const bool behind = key0 + kRows - 1 - first <= -reach, ahead = key0 - first - 31 >= (a.bias.ahead ? reach : 0);
        near = !behind && !ahead;
        if (!near) bc = table[behind ? 0 : 2 * reach + 16] * a.c2;
      }
      scores(stage, bc, near, !all);
    }
    if (!kTwo) {
      // This tile's values have landed: only the next keys, loaded after them, may be on their way.
      if (more) wait_vmcnt<KJ>();
      else wait_vmcnt<0>();
      __syncthreads();
    }
    if (any) products(stage);
    bits = bits_next;
    wait_vmcnt<0>();
    __syncthreads();  // the next tile has landed for every wave, and no wave reads this one any more
    if (!kTwo && more) {
      issue_values(0, kt + 1, bits);
      asm volatile("" ::: "memory");  // counted by the wait above: no load moves across
    }
  };
  wait_vmcnt<0>();
  __syncthreads();
  if (!kTwo) {
    issue_values(0, kt, bits);
    asm volatile("" ::: "memory");
  }
  while (true) {
    step(0);
    if (++kt >= x.end) break;
    step(1);
    if (++kt >= x.end) break;
  }

  // The result: divided by the sums, or as it is where the keys are in parts.
  const Args &e = args_here();
  const float l_all = pair_sum(l_run);
  const int row = x.row0 + c;
  if (cut.parts > 1) {
    float *w = cut.partial + (static_cast<int64_t>(t) * NW + wave) * partial_floats(D);
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
      *reinterpret_cast<float4 *>(w + (i * 64 + lane) * 4) =
          make_float4(o[i >> 2][4 * (i & 3)], o[i >> 2][4 * (i & 3) + 1], o[i >> 2][4 * (i & 3) + 2], o[i >> 2][4 * (i & 3) + 3]);
    *reinterpret_cast<float2 *>(w + 32 * D + 2 * lane) = make_float2(m_run, l_all);
  } else {
    const float inv = l_all == 0.0f ? 0.0f : 1.0f / l_all;  // no key seen: zeros
    if (e.lse && h == 0 && row < e.Lq)
      e.lse[(static_cast<int64_t>(x.b) * e.H + x.head) * e.Lq + row] = (m_run + __builtin_log2f(l_all)) * kLn2;
    const int rows = min(e.Lq - x.row0, 32);
    const __amdgpu_buffer_rsrc_t r = make_rsrc(e.out + x.b * e.out_sb + x.row0 * e.out_sl + x.head * e.dh,
                                               rows > 0 ? 2 * ((rows - 1) * static_cast<uint32_t>(e.out_sl) + e.dh) : 0);
    const uint32_t at = static_cast<uint32_t>(lane & 31) * static_cast<uint32_t>(2 * e.out_sl);
    // Lanes c and c + 32 hold the halves of 8 channels: they exchange halves, and each stores 8 channels of row c.
    // What does not exist is steered out of the buffer's range.
#pragma unroll
    for (int i = 0; i < D / 8; i += 2) {
      uint32_t w[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const f32x16 &z = o[i >> 2];
        const int y = 4 * (i & 3) + 2 * u;
        const uint32_t lo = pack<BF>(materialize(z[y] * inv), materialize(z[y + 1] * inv));
        const uint32_t hi = pack<BF>(materialize(z[y + 4] * inv), materialize(z[y + 5] * inv));
        const auto p = __builtin_amdgcn_permlane32_swap(lo, hi, false, false);
        w[0][u] = p[0];
        w[1][u] = p[1];
      }
      typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
      const int ch = 8 * (i + h);
      __builtin_amdgcn_raw_buffer_store_b128(u32x4{w[0][0], w[0][1], w[1][0], w[1][1]}, r,
                                             ch < e.dh && row < e.Lq ? at + 2 * ch : kPast, 0, 0);
    }
  }
}

// The parts of fwd_kernel, joined: a workgroup per 32 queries and 32 channels, whose four waves take parts in turn, in the lane
// order of that kernel.
template <bool BF, int D>
__global__ __launch_bounds__(256) void merge_kernel(Args a, Cut cut, int nw) {
  __shared__ float4 so[4][4][64];
  __shared__ float2 sm[4][64];
  const int lane = threadIdx.x & 63, sub = threadIdx.x >> 6, db = blockIdx.x % (D / 32);
  int rest = blockIdx.x / (D / 32);
  const int qb = rest % cut.qblocks;
  rest /= cut.qblocks;
  const int head = rest % a.H, b = rest / a.H, hk = head / a.group, g = head - hk * a.group;
  const int block = cut.pack ? g * cut.qblocks + qb : qb, tile = block / nw, wave = block - tile * nw;
  const int tile0 = a.causal ? cut.tiles - 1 - tile : tile;
  const int heads = cut.pack ? 1 : a.group;
  const int64_t bhk = static_cast<int64_t>(b) * a.Hk + hk;
  const int64_t item = cut.pack ? bhk * cut.parts * cut.tiles + tile0 : (bhk * cut.parts * a.group + g) * cut.tiles + tile0;
  const int64_t step = static_cast<int64_t>(heads) * cut.tiles * nw * partial_floats(D);  // from one part to the next
  const float *w = cut.partial + (item * nw + wave) * partial_floats(D);
  float m = kLowest, l = 0.0f;
  for (int p = sub; p < cut.parts; p += 4) m = fmaxf(m, w[p * step + 32 * D + 2 * lane]);
  float4 o[4] = {};
#pragma unroll 2
  for (int p = sub; p < cut.parts; p += 4) {
    const float2 ml = *reinterpret_cast<const float2 *>(w + p * step + 32 * D + 2 * lane);
    const float f = __builtin_amdgcn_exp2f(ml.x - m);
    l += f * ml.y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 x = *reinterpret_cast<const float4 *>(w + p * step + ((4 * db + i) * 64 + lane) * 4);
      o[i].x += f * x.x;
      o[i].y += f * x.y;
      o[i].z += f * x.z;
      o[i].w += f * x.w;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) so[sub][i][lane] = o[i];
  sm[sub][lane] = make_float2(m, l);
  __syncthreads();
  // Wave `sub` joins the channels 8 sub .. + 8.
  float2 ml[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) ml[j] = sm[j][lane];
  m = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
  l = 0.0f;
  float4 x = {};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float f = __builtin_amdgcn_exp2f(ml[j].x - m);
    const float4 z = so[j][sub][lane];
    l += f * ml[j].y;
    x.x += f * z.x;
    x.y += f * z.y;
    x.z += f * z.z;
    x.w += f * z.w;
  }
  const int row = 32 * qb + (lane & 31), ch = 32 * db + 8 * sub;
  if (row >= a.Lq) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (ch < a.dh)
    *reinterpret_cast<uint2 *>(a.out + b * a.out_sb + row * a.out_sl + head * a.dh + ch + 4 * (lane >> 5)) =
        make_uint2(pack<BF>(materialize(x.x * inv), materialize(x.y * inv)), pack<BF>(materialize(x.z * inv), materialize(x.w * inv)));
  if (a.lse && db == 0 && sub == 0 && lane < 32)
    a.lse[(static_cast<int64_t>(b) * a.H + head) * a.Lq + row] = (m + __builtin_log2f(l)) * kLn2;
}

}  // namespace
}  // namespace textattn
}  // namespace selas

// ------------------------------------------------------------------ host side

namespace selas {
namespace textattn {

int cu_count() {
  static std::atomic<int> counts[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) {
    (void)hipGetLastError();
    dev = 0;
  }
  int v = counts[dev].load(std::memory_order_relaxed);
  if (v > 0) return v;
  if (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || v <= 0) {
    (void)hipGetLastError();
    v = 256;
  }
  counts[dev].store(v, std::memory_order_relaxed);
  return v;
}

namespace {

// Whole numbers of up to 40 words, for the borders of the buckets.
struct Big {
  uint32_t w[40] = {1};
  int n = 1;
  bool mul(uint32_t m) {
    uint64_t carry = 0;
    for (int i = 0; i < n; ++i) {
      carry += static_cast<uint64_t>(w[i]) * m;
      w[i] = static_cast<uint32_t>(carry);
      carry >>= 32;
    }
    if (carry) {
      if (n == 40) return false;
      w[n++] = static_cast<uint32_t>(carry);
    }
    return true;
  }
  void pow(uint32_t m, int e) {
    for (int i = 0; i < e; ++i) mul(m);
  }
  bool at_least(const Big &o) const {
    if (n != o.n) return n > o.n;
    for (int i = n - 1; i >= 0; --i)
      if (w[i] != o.w[i]) return w[i] > o.w[i];
    return true;
  }
};

// Whether (a / e)^k >= (m / e)^t, that is a^k e^t >= m^t e^k: at most 10 bits times 64 + 63, 40 words hold it.
bool past_border(int a, int e, int m, int k, int t) {
  Big x, y;
  x.pow(a, k);
  x.pow(e, t);
  y.pow(m, t);
  y.pow(e, k);
  return x.at_least(y);
}

int fill_buckets(const char *what, int64_t buckets, int64_t max_distance, int bidirectional, int32_t *edge, int &n) {
  if (bidirectional && buckets % 2)
    return set_error(SELAS_EINVAL, "%s: %lld buckets do not halve into two directions", what, (long long)buckets);
  const int64_t side = bidirectional ? buckets / 2 : buckets;
  if (side < 2) return set_error(SELAS_EINVAL, "%s: needs two buckets a direction, got %lld", what, (long long)side);
  if (max_distance <= side / 2)
    return set_error(SELAS_EINVAL, "%s: max_distance %lld is not above the %lld exact distances", what, (long long)max_distance,
                     (long long)(side / 2));
  if (side > kMaxSide || max_distance > kMaxDistance)
    return set_error(SELAS_EUNSUPPORTED, "%s: takes up to %d buckets a direction and distances up to %d", what, kMaxSide,
                     kMaxDistance);
  n = static_cast<int>(side);
  const int e = n / 2, m = static_cast<int>(max_distance), k = n - e;
  for (int t = 0; t <= e; ++t) edge[t] = t;
  for (int t = 1; t < k; ++t) {
    // The real border, and the distance at or after it: whole numbers decide where rounding could.
    int a = std::max(static_cast<int>(e * pow(static_cast<double>(m) / e, static_cast<double>(t) / k)) - 1, e);
    while (!past_border(a, e, m, k, t)) ++a;
    edge[e + t] = a;
  }
  for (int t = n; t < kMaxSide; ++t) edge[t] = INT32_MAX;
  return SELAS_OK;
}

int check_side(const char *what, const char *name, const void *p, int64_t sb, int64_t sh, int64_t sl, const Args &a, int heads,
               int rows, Side &side) {
  if (!p) return set_error(SELAS_EINVAL, "%s: null pointer (%s)", what, name);
  if (sb < 0 || sh < 0 || sl < 0) return set_error(SELAS_EINVAL, "%s: %s has a negative stride", what, name);
  sb = stride_of(a.B, sb, 0);
  sh = stride_of(heads, sh, 0);
  sl = stride_of(rows, sl, a.dh);
  if (!aligned(p, 16) || sb % 8 || sh % 8 || sl % 8)
    return set_error(SELAS_EUNSUPPORTED, "%s: %s must be 16-byte aligned with strides of whole 16 bytes", what, name);
  if (sl > (1 << 23)) return set_error(SELAS_EUNSUPPORTED, "%s: %s has a row stride above 2^23 elements", what, name);
  side = {static_cast<const uint16_t *>(p), sb, sh, sl};
  return SELAS_OK;
}

}  // namespace

int check_args(const char *what, const selas_text_attention_problem *p, int dtype, bool pointers, Args &a) {
  if (!p) return set_error(SELAS_EINVAL, "%s: null problem", what);
  if (p->B < 0 || p->H < 0 || p->Hk < 0 || p->Lq < 0 || p->Lk < 0 || p->Dh <= 0)
    return set_error(SELAS_EINVAL, "%s: bad shape B=%lld H=%lld Hk=%lld Lq=%lld Lk=%lld Dh=%lld", what, (long long)p->B,
                     (long long)p->H, (long long)p->Hk, (long long)p->Lq, (long long)p->Lk, (long long)p->Dh);
  if (p->Hk == 0 ? p->H != 0 : p->H % p->Hk != 0)
    return set_error(SELAS_EINVAL, "%s: %lld heads do not share %lld key heads evenly", what, (long long)p->H, (long long)p->Hk);
  if (!valid_dtype(dtype)) return set_error(SELAS_EINVAL, "%s: bad dtype %d", what, dtype);
  if (p->reserved != 0) return set_error(SELAS_EINVAL, "%s: reserved must be 0", what);
  if (!(p->scale >= 1e-10 && p->scale <= 1e10))
    return set_error(SELAS_EINVAL, "%s: scale %g is outside 1e-10 .. 1e10", what, p->scale);
  if (p->table && !valid_dtype(p->table_dtype)) return set_error(SELAS_EINVAL, "%s: bad table dtype %d", what, p->table_dtype);
  if (dtype == SELAS_F32 || p->Dh % 8 || p->Dh > 128)
    return set_error(SELAS_EUNSUPPORTED, "%s: takes bf16 or fp16 and head dims of whole 8 up to 128 (got %s, %lld)", what,
                     dtype_name(dtype), (long long)p->Dh);
  if (p->Lq >= (1 << 28) || p->Lk >= (1 << 28) || p->B >= (1 << 28) || p->H >= (1 << 28) ||
      p->B * p->H * cdiv(std::max<int64_t>(std::max(p->Lq, p->Lk), 1), 32) >= (1ll << 26))
    return set_error(SELAS_EUNSUPPORTED, "%s: more than 2^26 blocks of 32 rows", what);
  a = Args{};
  a.bias.dtype = p->table_dtype;
  if (p->table) {
    if (int e = fill_buckets(what, p->buckets, p->max_distance, p->bidirectional, a.bias.edge, a.bias.n)) return e;
    a.bias.ahead = p->bidirectional ? a.bias.n : 0;
    a.bias.reach = a.bias.edge[a.bias.n - 1];
    a.bias.row = p->table_sl;
    a.bias.table = p->table;
    a.bias.inv_scale = static_cast<float>(1.0 / p->scale);
    if (p->table_sl < 0) return set_error(SELAS_EINVAL, "%s: the table has a negative stride", what);
  }
  a.B = static_cast<int>(p->B);
  a.H = static_cast<int>(p->H);
  a.Hk = static_cast<int>(p->Hk);
  a.group = p->Hk ? static_cast<int>(p->H / p->Hk) : 0;
  a.Lq = static_cast<int>(p->Lq);
  a.Lk = static_cast<int>(p->Lk);
  a.dh = static_cast<int>(p->Dh);
  a.causal = p->causal != 0;
  a.c2 = static_cast<float>(p->scale * 1.4426950408889634);
  a.lse = p->lse;
  a.lengths = p->lengths;
  a.mask = p->mask;
  a.mask_sb = p->mask_sb;
  a.start = p->start;
  a.start0 = static_cast<int>(std::min<int64_t>(std::max<int64_t>(p->start0, -(1 << 29)), 1 << 29));
  if (!pointers || p->B == 0 || p->H == 0 || p->Lq == 0) return SELAS_OK;
  if (int e = check_side(what, "q", p->q, p->q_sb, p->q_sh, p->q_sl, a, a.H, a.Lq, a.q)) return e;
  if (p->Lk) {  // without keys there may be no memory
    if (int e = check_side(what, "k", p->k, p->k_sb, p->k_sh, p->k_sl, a, a.Hk, a.Lk, a.k)) return e;
    if (int e = check_side(what, "v", p->v, p->v_sb, p->v_sh, p->v_sl, a, a.Hk, a.Lk, a.v)) return e;
  }
  if (!p->out) return set_error(SELAS_EINVAL, "%s: null pointer (out)", what);
  if (p->o_sb < 0 || p->o_sl < 0 || p->mask_sb < 0) return set_error(SELAS_EINVAL, "%s: negative stride", what);
  a.out = static_cast<uint16_t *>(p->out);
  a.out_sb = stride_of(a.B, p->o_sb, 0);
  a.out_sl = stride_of(a.Lq, p->o_sl, a.dh);
  if (!aligned(p->out, 8) || a.out_sb % 4 || a.out_sl % 4)
    return set_error(SELAS_EUNSUPPORTED, "%s: out must be 8-byte aligned with strides of whole 8 bytes", what);
  if (a.out_sl > (1 << 23)) return set_error(SELAS_EUNSUPPORTED, "%s: out has a row stride above 2^23 elements", what);
  return SELAS_OK;
}

namespace {

struct Plan {
  int few = 0;  // rows held by the few-row kernel, 0: tiles
  int D, nw;
  Cut cut{};
  int few_parts;
  int64_t bytes = 0;  // workspace
  Threads threads;
};

Plan plan_of(const Args &a) {
  Plan p{};
  p.D = width_of(a.dh);
  const int64_t cu = cu_count();
  const int64_t rows = static_cast<int64_t>(a.group) * a.Lq, items = static_cast<int64_t>(a.B) * a.Hk;
  if (rows <= 8) {
    p.few = rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : 8;
    p.nw = 8;
    p.D = a.dh <= 64 ? 64 : 128;
    const int unit = (p.few <= 2 ? 8 : 2) * (512 / p.D);
    const int64_t units = cdiv(a.Lk, unit);
    // Parts for two workgroups a CU, of four units a wave at least.
    p.few_parts = static_cast<int>(std::max<int64_t>(1, std::min(2 * cu / std::max<int64_t>(items, 1), units / (4 * p.nw))));
    if (p.few_parts > 1) p.bytes = items * p.few_parts * p.few * (p.D + 2) * 4;
    p.threads.add(items * p.few_parts, 512);
    if (p.few_parts > 1) p.threads.add(items * rows, 128);
    return p;
  }
  Cut &c = p.cut;
  c.qblocks = static_cast<int>(cdiv(a.Lq, 32));
  c.pack = a.group > 1 && !a.causal && !a.bias.table;
  const int64_t blocks = c.pack ? static_cast<int64_t>(a.group) * c.qblocks : c.qblocks;
  p.nw = blocks <= 1 ? 1 : blocks <= 2 ? 2 : 4;
  c.tiles = static_cast<int>(cdiv(blocks, p.nw));
  const int64_t whole = items * (c.pack ? 1 : a.group) * c.tiles, tiles = cdiv(a.Lk, kRows);
  // Parts where items are too few for two to a CU, of eight tiles at least: a part's output is written and read again, and the
  // merge is a launch of its own. us, parts of four tiles / eight: 64 heads of 512 with a bias 25.8 / 20.0, 4 heads of 256 rows
  // over 20,280 keys 36.9 / 34.6. Parts for one to a CU instead: 32.0 there, but 24 heads of 1024 rows over 2048 keys 46.8 ->
  // 51.8.
  c.parts = static_cast<int>(std::max<int64_t>(1, std::min(2 * cu / std::max<int64_t>(whole, 1), tiles / 8)));
  c.deal = deal(whole * c.parts, static_cast<int64_t>(c.pack ? 1 : a.group) * c.tiles, a.lengths || a.mask);
  c.by_tiles = fast_div(c.tiles);
  c.by_group = fast_div(a.group);
  c.by_parts = fast_div(c.parts);
  c.by_hk = fast_div(a.Hk);
  c.by_qblocks = fast_div(c.qblocks);
  if (c.parts > 1) p.bytes = static_cast<int64_t>(c.deal.total) * p.nw * partial_floats(p.D) * 4;
  p.threads.add(c.deal.blocks, 64 * p.nw);
  if (c.parts > 1) p.threads.add(static_cast<int64_t>(a.B) * a.H * c.qblocks * (p.D / 32), 256);
  return p;
}

template <bool BF, int D, int R, bool BIAS>
void launch_few(const Args &a, const Plan &p, float *ws, hipStream_t st) {
  const int items = a.B * a.Hk, parts = p.few_parts;
  const size_t lds = BIAS ? static_cast<size_t>(a.group) * (2 * a.bias.reach + 1) * 4 : 0;
  few_kernel<BF, D, R, 8, BIAS><<<dim3(items * parts), dim3(512), lds, st>>>(a, parts, ws);
  if (parts > 1) few_merge_kernel<BF><<<dim3(items * a.group * a.Lq), dim3(128), 0, st>>>(a, parts, D, R, ws);
}

template <bool BF, int D, int NW, bool BIAS>
void launch_tiles(const Args &a, const Plan &p, float *ws, hipStream_t st) {
  Cut cut = p.cut;
  cut.partial = ws;
  fwd_kernel<BF, D, NW, BIAS><<<dim3(cut.deal.blocks), dim3(64 * NW), BIAS ? bias_bytes(a.bias.reach) : 0, st>>>(a, cut);
  if (cut.parts > 1)
    merge_kernel<BF, D><<<dim3(a.B * a.H * cut.qblocks * (D / 32)), dim3(256), 0, st>>>(a, cut, NW);
}

template <bool BF, int D, bool BIAS>
void launch(const Args &a, const Plan &p, float *ws, hipStream_t st) {
  if constexpr (D != 96) {
    switch (p.few) {
      case 1: return launch_few<BF, D, 1, BIAS>(a, p, ws, st);
      case 2: return launch_few<BF, D, 2, BIAS>(a, p, ws, st);
      case 4: return launch_few<BF, D, 4, BIAS>(a, p, ws, st);
      case 8: return launch_few<BF, D, 8, BIAS>(a, p, ws, st);
    }
  }
  switch (p.nw) {
    case 1: return launch_tiles<BF, D, 1, BIAS>(a, p, ws, st);
    case 2: return launch_tiles<BF, D, 2, BIAS>(a, p, ws, st);
    default: return launch_tiles<BF, D, 4, BIAS>(a, p, ws, st);
  }
}

}  // namespace
}  // namespace textattn
}  // namespace selas

using namespace selas;
using namespace selas::textattn;

extern "C" int selas_relative_buckets(int64_t buckets, int64_t max_distance, int bidirectional, int32_t *edges,
                                      int64_t *count) {
  if (!edges || !count) return set_error(SELAS_EINVAL, "relative_buckets: null pointer");
  int32_t edge[kMaxSide];
  int n = 0;
  if (int e = fill_buckets("relative_buckets", buckets, max_distance, bidirectional, edge, n)) return e;
  for (int t = 0; t < n; ++t) edges[t] = edge[t];
  *count = n;
  return ok();
}

extern "C" int selas_text_attention_workspace_bytes(const selas_text_attention_problem *problem, int dtype, int64_t *bytes) {
  if (!bytes) return set_error(SELAS_EINVAL, "text_attention_workspace_bytes: null pointer");
  *bytes = 0;
  Args a;
  if (int e = check_args("text_attention_workspace_bytes", problem, dtype, false, a)) return e;
  if (!a.B || !a.H || !a.Lq) return ok();
  const Plan p = plan_of(a);
  if (int e = p.threads.check("text_attention_workspace_bytes")) return e;
  *bytes = p.bytes;
  return ok();
}

extern "C" int selas_text_attention(const selas_text_attention_problem *problem, int dtype, void *workspace,
                                    int64_t workspace_bytes, void *stream) {
  Args a;
  if (int e = check_args("text_attention", problem, dtype, true, a)) return e;
  if (!a.B || !a.H || !a.Lq) return ok();
  const Plan p = plan_of(a);
  if (int e = p.threads.check("text_attention")) return e;
  if (p.bytes && (workspace_bytes < p.bytes || !workspace || !aligned(workspace, 16)))
    return set_error(SELAS_EINVAL, "text_attention: needs a 16-byte aligned workspace of %lld bytes", (long long)p.bytes);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  float *ws = static_cast<float *>(workspace);
  auto go = [&](auto bf, auto d) {
    constexpr bool kBf = decltype(bf)::value;
    constexpr int kD = decltype(d)::value;
    if (a.bias.table) launch<kBf, kD, true>(a, p, ws, st);
    else launch<kBf, kD, false>(a, p, ws, st);
  };
  using I64 = std::integral_constant<int, 64>;
  using I96 = std::integral_constant<int, 96>;
  using I128 = std::integral_constant<int, 128>;
  auto width = [&](auto bf) { p.D == 64 ? go(bf, I64{}) : p.D == 96 ? go(bf, I96{}) : go(bf, I128{}); };
  if (dtype == SELAS_BF16) width(std::true_type{});
  else width(std::false_type{});
  return check_launch("text_attention");
}
