// The gradients of selas_text_attention, for gfx950. With dO the gradient of out and p the probabilities:
//   D_i = dO_i . out_i,  dP_ij = dO_i . v_j,  dS_ij = p_ij (dP_ij - D_i)
//   dv_j = sum_i p_ij dO_i,  dk_j = scale sum_i dS_ij q_i,  dq_i = scale sum_j dS_ij k_j,  dtable[r, h] = sum of dS_ij over
//   the pairs in bucket r; dk and dv sum over the query heads that share the key head.
// p is formed again from q, k and the forward pass's lse. Two kernels: query_kernel has the queries as owners and streams keys
// past them (dq, dtable; it also leaves lse and D per row), then key_kernel has the keys as owners and streams queries (dk,
// dv). S and dP are formed in both: 7 products where one kernel would need 5 and floating-point atomics, whose order would
// change the bits from call to call.
#include <algorithm>
#include <type_traits>

#include "text_attention.h"

namespace selas {
namespace textattn {
namespace {

// fp16 operands of the second products. p <= 1 is stored times 2^15, and dS times a power of two (per image and key head)
// that puts its bound, 2 max|dO| max|v|, at or below 2^15: nothing overflows, and what falls below fp16's normal numbers is
// under 2^-29 of that bound. bf16 has fp32's range and needs neither.
constexpr float kProbShift = 15.0f;
template <bool BF>
__device__ constexpr float prob_shift() {
  return BF ? 0.0f : kProbShift;
}

struct Grads {
  Side g;  // dO as [B, H, Lq, dh]
  uint16_t *dq, *dk, *dv;  // contiguous [B, heads, L, dh]
  float *neg_lse, *dot;    // [B, H, Lqp]: -lse log2(e) (-inf for rows that see nothing and rows past Lq), D (0 there)
  int Lqp, qblocks, kblocks;  // rows padded to whole tiles; tiles of queries, of keys
  float *g_norm, *v_norm;  // fp16: largest squared norms of the rows of dO and v, per tile
  float *dtable_part;      // [B, H, qtiles * parts, buckets]
  void *dtable;
};

// A kernel's work items: `parts` ranges of the streamed axis; sums of a part go to `partial` (fp32) where parts > 1.
struct Cut {
  int tiles, parts;
  Deal deal;
  FastDiv by_tiles, by_parts, by_group, by_hk;
  float *partial;
  float2 *missing;  // query_kernel with parts: [parts][B, H, Lqp], the sums of dS and of |dS|
  int again;        // its second launch
};

// fp16: the largest squared norm among 64 rows of dO, or (blocks past the queries') of 64 values; 4 lanes to a row. What
// queries that see no key or masked values hold is left out.
__global__ __launch_bounds__(256) void norm_kernel(Args a, Grads w) {
  __shared__ float red[4];
  const int lane = threadIdx.x & 63, r = threadIdx.x >> 2, part = threadIdx.x & 3;
  const int queries = a.B * a.H * w.qblocks;
  int t = blockIdx.x;
  const uint16_t *p = nullptr;
  float *out;
  if (t < queries) {
    const int qt = t % w.qblocks, bh = t / w.qblocks, b = bh / a.H, row = qt * kRows + r;
    out = w.g_norm + t;
    if (row < a.Lq && a.lse[static_cast<int64_t>(bh) * a.Lq + row] != -__builtin_inff())
      p = w.g.p + b * w.g.sb + (bh - b * a.H) * w.g.sh + row * w.g.sl;
  } else {
    t -= queries;
    const int kt = t % w.kblocks, bh = t / w.kblocks, b = bh / a.Hk, row = kt * kRows + r;
    out = w.v_norm + t;
    if (row < keys_of(a, b) && (!a.mask || a.mask[b * a.mask_sb + row]))
      p = a.v.p + b * a.v.sb + (bh - b * a.Hk) * a.v.sh + row * a.v.sl;
  }
  float norm = 0.0f;
  if (p)
    for (int ch = 8 * part; ch < a.dh; ch += 32) {
      const uint4 x = *reinterpret_cast<const uint4 *>(p + ch);
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float lo = lo_of<false>(xs[e]), hi = hi_of<false>(xs[e]);
        norm = __builtin_fmaf(lo, lo, norm);
        norm = __builtin_fmaf(hi, hi, norm);
      }
    }
  norm += __shfl_xor(norm, 1, 64);
  norm += __shfl_xor(norm, 2, 64);
#pragma unroll
  for (int o = 4; o < 64; o <<= 1) norm = fmaxf(norm, __shfl_xor(norm, o, 64));
  if (lane == 0) red[threadIdx.x >> 6] = norm;
  __syncthreads();
  if (threadIdx.x == 0) *out = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// log2 of the factor that dS of image b and key head hk is stored with.
template <bool BF>
__device__ __forceinline__ float ds_shift(const Args &a, const Grads &w, int b, int hk, int lane) {
  if constexpr (BF) return 0.0f;
  float g = 0.0f, v = 0.0f;
  const float *gn = w.g_norm + static_cast<int64_t>(b * a.H + hk * a.group) * w.qblocks;
  const float *vn = w.v_norm + static_cast<int64_t>(b * a.Hk + hk) * w.kblocks;
  for (int i = lane; i < a.group * w.qblocks; i += 64) g = fmaxf(g, gn[i]);
  for (int i = lane; i < w.kblocks; i += 64) v = fmaxf(v, vn[i]);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    g = fmaxf(g, __shfl_xor(g, o, 64));
    v = fmaxf(v, __shfl_xor(v, o, 64));
  }
  // 0.5 log2(g v): of each, a product of squares might overflow. A step of 1 / 16 covers the logarithms' rounding.
  const float bound = 0.5f * (__builtin_log2f(g) + __builtin_log2f(v)) + 1.0625f;
  const float e = floorf(15.0f - bound);
  return e >= -120.0f && e <= 120.0f ? e : 0.0f;  // zeros, infinities and NaN: as they are
}

// ------------------------------------------------------------------ dk, dv

// One workgroup = NW waves = 32 NW keys of one (image, key head); wave w owns keys 32 w .. + 32 and holds their k and v.
// Tiles of 64 queries (q and dO rows, lse and D), of all the heads of the group in turn, stream through LDS. Per block of 32
// queries: S = Q K^T and dP = dO V^T with the query rows read row-wise, so that a lane's registers hold 16 queries of one
// key, in runs of 8; then dV^T += dO^T P and dK^T += Q^T dS with the same tiles read transposed and P, dS straight from the
// registers. A key's column depends on nothing of the other keys, so masked keys need no select: their results are zeroed at
// the end. A query that sees no key has p = 0, but what it and its dO hold, NaN included, meets that in a product: where an
// image may have such a query and others (a causal mask with masked keys or a negative start) its rows are cleared in LDS.
//
// Bounded by LDS reads (an MFMA reads 1 KiB) and by waiting: dk and dv of 32 keys take D registers a lane and k and v D / 2
// more, which leaves three workgroups a CU at D = 64 and two at D = 128, where 4 to 8 registers spill but for bf16 without a
// bias (MFMA 30 % busy at 4 x 64 heads of 512 tokens, 58 us; 24 heads of 128, 4096 queries over 512 keys 66 us, 780 TFLOP/s).
// With each 16 rows' products right behind their packing one pair of packed operands is live instead of two (178 -> 164
// registers); a lone workgroup a CU at D = 128 took 100 us there.
template <bool BF, int D, int NW, bool BIAS>
__global__ __launch_bounds__(64 * NW, 2) void key_kernel(Args a, Grads w, Cut cut) {
  using T = TileOf<D>;
  constexpr int KJ = T::kLoads / NW, kStats = 2 * kRows * 4;
  __shared__ __attribute__((aligned(16))) uint8_t smem0[2 * T::kBytes + kStats], smem1[2 * T::kBytes + kStats];
  extern __shared__ __attribute__((aligned(16))) float tables[];  // two heads' bias by distance
  const int t = item_of(cut.deal);
  if (t >= cut.deal.total) return;
  int rest, bhk, b;
  const int tile = split(t, cut.by_tiles, cut.tiles, rest), part = split(rest, cut.by_parts, cut.parts, bhk);
  const int hk = split(bhk, cut.by_hk, a.Hk, b);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5, c = lane & 31;
  const int keys = keys_of(a, b), start = start_of(a, b);
  const int wg_key = tile * NW * 32, key0 = wg_key + wave * 32, key = key0 + c;

  // The tiles of queries that see a key of this workgroup, for each head; this part's range of them all.
  int qt0 = a.causal ? max(wg_key - start, 0) / kRows : 0;
  const int each = wg_key < keys ? max(w.qblocks - qt0, 0) : 0, n = each * a.group;
  const int per = (n + cut.parts - 1) / cut.parts;
  int i = part * per;
  const int end = min(n, i + per);
  int g = each ? i / each : 0, qt = qt0 + (each ? i % each : 0);

  bool valid = key < keys;
  if (valid && a.mask) valid = a.mask[b * a.mask_sb + key] != 0;
  Held<D> k, v;
  k.load(a.k.p + b * a.k.sb + hk * a.k.sh + key0 * a.k.sl, a.k.sl, a.dh, keys - key0, lane, valid);
  v.load(a.v.p + b * a.v.sb + hk * a.v.sh + key0 * a.v.sl, a.v.sl, a.dh, keys - key0, lane, valid);
  const typename T::template Loader<KJ> ql(wave, lane, a.q.sl, a.dh), gl(wave, lane, w.g.sl, a.dh);
  const typename T::RowReader rows(lane);
  const typename T::ColReader cols(lane);
  auto issue = [&](int stage, int g, int qt) {
    uint8_t *base = stage ? smem1 : smem0;
    const int head = hk * a.group + g, left = a.Lq - qt * kRows;
    const int64_t row = static_cast<int64_t>(qt) * kRows;
    ql.template issue<false>(base, a.q.p + b * a.q.sb + head * a.q.sh + row * a.q.sl, a.q.sl, a.dh, left, 0);
    gl.template issue<false>(base + T::kBytes, w.g.p + b * w.g.sb + head * w.g.sh + row * w.g.sl, w.g.sl, a.dh, left, 0);
    if (wave < 2) {  // 64 floats each
      const float *p = (wave ? w.dot : w.neg_lse) + (static_cast<int64_t>(b) * a.H + head) * w.Lqp + row;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          make_rsrc(p, kRows * 4), (__attribute__((address_space(3))) void *)(base + 2 * T::kBytes + wave * kRows * 4), 4,
          4 * lane, 0, 0, 0);
    }
  };
  const int reach = a.bias.reach, pitch = bias_pitch(reach);
  auto table_of = [&](int g) { return tables + (g & 1) * 4 * pitch; };  // the heads of the group take the two in turn
  auto next_table = [&](int g) __attribute__((always_inline)) {
    const Args &a = args_here();
    build_bias(table_of(g), a.bias, hk * a.group + g, 64 * NW, true);
  };
  const float shift = ds_shift<BF>(a, w, b, hk, lane);
  const float ds_mul = BF ? 1.0f : __builtin_exp2f(shift - kProbShift);

  f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) dk[db] = dv[db] = f32x16{};

  // One tile; near and part as in the forward pass.
  auto compute = [&](int stage, int qt, const float *table, float bc, bool near, bool part) __attribute__((always_inline)) {
    uint8_t *qs = stage ? smem1 : smem0, *gs = qs + T::kBytes;
    const float *stats = reinterpret_cast<const float *>(qs + 2 * T::kBytes);
    const int pos0 = start + qt * kRows;  // of the tile's first query
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
      for (int x = 0; x < D / 16; ++x) s = mfma<BF>(rows.read(qs, qb, x), k.f[x], s);
#pragma unroll
      for (int x = 0; x < D / 16; ++x) dp = mfma<BF>(rows.read(gs, qb, x), v.f[x], dp);
      if (BIAS && near) {
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
          float bv[8];
          bias_run(table, pitch, reach, pos0 + 32 * qb + 16 * t2 + 8 * h - key, bv);
#pragma unroll
          for (int e = 0; e < 8; ++e) s[8 * t2 + e] += bv[e];
        }
      }
      if (part) {
        const uint32_t seen = static_cast<uint32_t>(~up_to(key - pos0 - 32 * qb - 8 * h - 1));  // queries at or after the key
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = (seen >> (16 * (r >> 3) + (r & 7))) & 1 ? s[r] : -__builtin_inff();
      }
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        const int at = 32 * qb + 16 * t2 + 8 * h;  // the first of this lane's 8 queries
        float p[8], ds[8];
#pragma unroll
        for (int e4 = 0; e4 < 2; ++e4) {
          const f32x4 nl = *reinterpret_cast<const f32x4 *>(stats + at + 4 * e4);
          const f32x4 dd = *reinterpret_cast<const f32x4 *>(stats + kRows + at + 4 * e4);
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int e = 4 * e4 + y, r = 8 * t2 + e;
            const float x = __builtin_fmaf(s[r], a.c2, BIAS || !BF ? nl[y] + bc : nl[y]);
            p[e] = materialize(__builtin_amdgcn_exp2f(x));
            ds[e] = materialize(p[e] * (dp[r] - dd[y]) * ds_mul);
          }
        }
        const uint4 pb = pack8<BF>(p), sb = pack8<BF>(ds);
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
          dv[db] = mfma<BF>(cols.read(gs, db, qb, t2), pb, dv[db]);
          dk[db] = mfma<BF>(cols.read(qs, db, qb, t2), sb, dk[db]);
        }
      }
    }
  };

  if (i < end) {
    if constexpr (BIAS) next_table(g);
    issue(0, g, qt);
  }
  const bool blind = a.causal && (a.mask || start < 0);  // some queries may see no key
  auto step = [&](int stage) __attribute__((always_inline)) {
    wait_vmcnt<0>();
    __syncthreads();  // this tile has landed for every wave, and no wave reads the other stage any more
    const int at = qt;
    if (blind) {
      static_assert(NW == 4, "four threads a row");
      uint8_t *base = stage ? smem1 : smem0;
      const float nl = reinterpret_cast<const float *>(base + 2 * T::kBytes)[lane];
      const uint64_t rows = __builtin_amdgcn_ballot_w64(nl == -__builtin_inff()) & up_to(a.Lq - 1 - at * kRows);
      if (rows) {
        int thread = threadIdx.x;
        asm volatile("" : "+v"(thread));  // addresses of this rare branch hold no registers in the loop
        const int r = thread >> 2;
        if ((rows >> r) & 1)
          for (int i = thread & 3; i < T::kChunks; i += 4) {
            uint8_t *to = base + T::at(r) + r % T::kGroupRows * T::kRow + 16 * i;
            *reinterpret_cast<uint4 *>(to) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4 *>(to + T::kBytes) = make_uint4(0, 0, 0, 0);
          }
        __syncthreads();
      }
    }
    const float *table = table_of(g);
    if (++qt == w.qblocks) {
      qt = qt0;
      ++g;
    }
    if (i + 1 < end) {
      if constexpr (BIAS)
        if (qt == qt0) next_table(g);
      issue(stage ^ 1, g, qt);
    }
    const int pos0 = start + at * kRows;
    if (key0 < keys && !(a.causal && pos0 + kRows - 1 < key0)) {
      bool near = BIAS;
      float bc = prob_shift<BF>();
      if constexpr (BIAS) {
        const bool behind = key0 + 31 - pos0 <= -reach, ahead = key0 - (pos0 + kRows - 1) >= (a.bias.ahead ? reach : 0);
        near = !behind && !ahead;
        if (!near) bc += table[behind ? 2 * reach + 16 : 0] * a.c2;
      }
      compute(stage, at, table, bc, near, a.causal && pos0 < key0 + 31);
    }
  };
  while (i < end) {
    step(0);
    if (++i >= end) break;
    step(1);
    ++i;
  }

  const Args &e = args_here();
  if (key >= e.Lk) return;
  const float k_mul = e.c2 * kLn2 * (BF ? 1.0f : __builtin_exp2f(-shift)), v_mul = BF ? 1.0f : __builtin_exp2f(-kProbShift);
  const int64_t at = (static_cast<int64_t>(bhk) * e.Lk + key) * e.dh, all = static_cast<int64_t>(e.B) * e.Hk * e.Lk * e.dh;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int ch = 32 * db + 8 * y + 4 * h;
      if (32 * db + 8 * y >= e.dh) continue;
      float x[4], z[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = materialize(valid ? dk[db][4 * y + i] * k_mul : 0.0f);
        z[i] = materialize(valid ? dv[db][4 * y + i] * v_mul : 0.0f);
      }
      if (cut.parts > 1) {
        float *p = cut.partial + 2 * part * all + at + ch;
        *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4 *>(p + all) = make_float4(z[0], z[1], z[2], z[3]);
      } else {
        *reinterpret_cast<uint2 *>(w.dk + at + ch) = make_uint2(pack<BF>(x[0], x[1]), pack<BF>(x[2], x[3]));
        *reinterpret_cast<uint2 *>(w.dv + at + ch) = make_uint2(pack<BF>(z[0], z[1]), pack<BF>(z[2], z[3]));
      }
    }
}

// ------------------------------------------------------------------ dq, dtable

// One workgroup = NW waves = 32 NW queries of one (image, head), the keys in tiles of 64 as in the forward pass; q and dO are
// held. S^T = K Q^T and dP^T = V dO^T leave a lane's registers with keys of one query, in runs of 8; dQ^T += K^T dS^T reads
// the same K tile transposed.
//
// Bounded as key_kernel: 3 products of 7, 153 to 168 registers at D = 64 (75 us at 4 x 64 heads of 512 with a bias), 223 at
// D = 128 (72 us at 4096 queries over 512 keys).
//
// dtable: tiles that hold only one value of the bias add dS up in a register. In the others dS is summed along the diagonals
// (one distance each): a lane's run of 8 keys moves a lane per key through the 16 lanes of its row (Diagonals), and what is
// left, a value per lane and 16 distances, is added to a histogram by distance in LDS, one for each half of each wave. It
// covers every distance that such a tile can hold (kSpill past `reach` on either side). At the end the histograms are summed
// by bucket, and by dtable_kernel over workgroups. LDS float additions of every element instead took 120 cycles an
// instruction: all gradients of 16 x 64 heads of 512 with a bias 1160 us, this way 567 at the time.
//
// D is first the product of dO and out in the order of the matrix unit, as dP is: where a row sees one key, out is that key's
// value and dS is exactly 0. But out was rounded, and where a few keys carry a row, or all values are alike, dP - D is small
// beside dP and D, and D's share of that rounding is many times those of dS and of the result. The sum of dS over a row's keys
// is 0 but for that share, so it says what D lacks. Workgroups of up to kRefine tiles of keys take that sum in a pass over them
// ahead of the others (77 keys: 14.4 -> 20.9 us). Longer ones take it, and the sum of |dS|, as they go; where in any of their
// rows it is above off_limit of the latter, three quarters of half a step of dS, they add it to D and begin again. Where
// the keys are in parts, a second launch does both, of which most workgroups end at once.
// Errors of dq against 64 bits in the 2-norm, in halves of a step, out's rounding left in / this way (0.6 is two roundings):
// 600 causal keys with 0.97 of the weight on a row's own 6.9 / 0.59; 3 seen keys of 300 0.93 / 0.60; 600 keys and scores of
// deviation 3 0.92 / 0.61; scores of deviation 1 0.61 / 0.61. It costs 2 % (the two sums; 24 heads of 128, 4096 queries over 512
// keys, all of forward and backward 174 -> 177 us), 4 % where a few rows of most heads are that far off (4 x 64 heads of 512
// with a random bias: 151 -> 157; at half instead of three quarters 160, with nothing gained), 8 % in parts (64 queries over
// 20,280 keys: 101 -> 109). Two launches in every case instead: 180 and 195 for the first two.
constexpr int kSpill = 112, kRefine = 4;
template <bool BF>
__device__ constexpr float off_limit() {
  return BF ? 0x1.8p-9f : 0x1.8p-12f;
}
__host__ __device__ inline int hist_floats(int reach) { return 2 * reach + 2 * kSpill + 1; }

// Sums along the diagonals of a wave's 32 keys x 32 queries. v[e] of lane q belongs to distance o + e - q. With
// t_e[p] = v[e][p] + t_{e+1}[p + 1], the lanes' indices modulo 16, t_0[p] holds distance o - p and, from the lanes below e
// that wrapped, o + 16 - p. Each is summed apart (subtracting the latter from the sum of both would leave its rounding in the
// other's bucket); the latter belong to the next 16 keys' first part.
struct Diagonals {
  float u[3] = {};  // u[m] of lane q: distance d0 + 16 m of that lane
  __device__ __forceinline__ static float next_lane(float v) {  // row_ror:15
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x12F, 0xF, 0xF, false));
  }
  __device__ __forceinline__ void add(int m, const f32x16 &v, int lane) {  // the m-th 8 of v
    const int p = lane & 15;
    float high = 0.0f, low = 0.0f;
#pragma unroll
    for (int e = 7; e >= 0; --e) {
      const float x = v[8 * m + e];
      if (e < 7) {
        high = next_lane(high);
        low = next_lane(low);
      }
      high += p >= e ? x : 0.0f;
      if (e) low += p < e ? x : 0.0f;
    }
    u[m] += high;
    u[m + 1] += low;
  }
  // u[m + 1] of the lanes 16 .. 31 meets u[m] of the lanes 0 .. 15: first the even ones, then the odd one. LDS instructions
  // of a wave are in order.
  __device__ __forceinline__ void store(float *at) const {
    const float x = at[0], y = at[32];
    at[0] = x + u[0];
    at[32] = y + u[2];
    asm volatile("" ::: "memory");
    at[16] += u[1];
    asm volatile("" ::: "memory");
  }
};

template <bool BF, int D, int NW, bool BIAS>
__global__ __launch_bounds__(64 * NW, D == 64 ? 3 : 2) void query_kernel(Args a, Grads w, Cut cut) {
  using T = TileOf<D>;
  constexpr int KJ = T::kLoads / NW;
  __shared__ __attribute__((aligned(16))) uint8_t smem0[2 * T::kBytes], smem1[2 * T::kBytes];
  __shared__ int off[NW];
  extern __shared__ __attribute__((aligned(16))) float table[];
  const int t = item_of(cut.deal);
  if (t >= cut.deal.total) return;
  int rest, b;
  const int qt0 = split(t, cut.by_tiles, cut.tiles, rest), g = split(rest, cut.by_group, a.group, rest);
  const int part = split(rest, cut.by_parts, cut.parts, rest), hk = split(rest, cut.by_hk, a.Hk, b), head = hk * a.group + g;
  const int qt = a.causal ? cut.tiles - 1 - qt0 : qt0;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5, c = lane & 31;
  const int keys = keys_of(a, b), start = start_of(a, b);
  const int row0 = (qt * NW + wave) * 32, first = start + row0, pos = first + c;
  int ntiles = (keys + kRows - 1) / kRows;
  if (a.causal) ntiles = min(ntiles, max(start + min((qt + 1) * NW * 32, a.Lq) + kRows - 1, 0) / kRows);
  const int per = (ntiles + cut.parts - 1) / cut.parts;
  int kt = part * per;
  const int end = min(ntiles, kt + per);

  // Whether D of any of the workgroup's rows is off by more than it may, where dS sums to `sum` and |dS| to `size`.
  auto any_off = [&](float sum, float size) __attribute__((always_inline)) {
    const uint64_t found = __builtin_amdgcn_ballot_w64(fabsf(sum) > off_limit<BF>() * size);
    if (lane == 0) off[wave] = found != 0;
    __syncthreads();
    int any = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) any |= off[i];
    return any != 0;
  };
  const int64_t stat = (static_cast<int64_t>(b) * a.H + head) * w.Lqp + row0 + c;
  float missing = 0.0f, size = 0.0f;  // of this lane's keys: the sums of dS and of |dS|, which is infinite once D is right
  if (cut.again) {
    if (row0 + c < w.Lqp)
      for (int i = h; i < cut.parts; i += 2) {
        const float2 x = cut.missing[i * (static_cast<int64_t>(a.B) * a.H * w.Lqp) + stat];
        missing += x.x;
        size += x.y;
      }
    missing = pair_sum(missing);
    if (!any_off(missing, pair_sum(size))) return;
    size = __builtin_inff();
  }

  Held<D> q, dO;
  q.load(a.q.p + b * a.q.sb + head * a.q.sh + row0 * a.q.sl, a.q.sl, a.dh, a.Lq - row0, lane);
  dO.load(w.g.p + b * w.g.sb + head * w.g.sh + row0 * w.g.sl, w.g.sl, a.dh, a.Lq - row0, lane);
  float nl = -__builtin_inff(), dd;
  if (row0 + c < a.Lq) {
    nl = a.lse[(static_cast<int64_t>(b) * a.H + head) * a.Lq + row0 + c];
    nl = nl == -__builtin_inff() ? nl : -nl * kLog2e;
  }
  {
    Held<D> out;
    out.load(a.out + b * a.out_sb + row0 * a.out_sl + head * a.dh, a.out_sl, a.dh, a.Lq - row0, lane);
    f32x16 x = f32x16{};
#pragma unroll
    for (int s = 0; s < D / 16; ++s) x = mfma<BF>(out.f[s], dO.f[s], x);
    // Row c of column c: register 4 (c / 8) + c % 4 of the lanes of half (c / 4) % 2.
    float d = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) d = r == 4 * (c >> 3) + (c & 3) ? x[r] : d;
    dd = pair_sum(h == ((c >> 2) & 1) ? d : 0.0f);
    dd += missing;  // 0 but in the second launch
    if (nl == -__builtin_inff()) {  // a row that sees no key: what its dO holds must not meet p = 0
      dd = 0.0f;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) dO.f[s] = make_uint4(0, 0, 0, 0);
    }
  }
  const uint16_t *kp = a.k.p + b * a.k.sb + hk * a.k.sh, *vp = a.v.p + b * a.v.sb + hk * a.v.sh;
  const typename T::template Loader<KJ> kl(wave, lane, a.k.sl, a.dh), vl(wave, lane, a.v.sl, a.dh);
  const typename T::RowReader rows(lane);
  const typename T::ColReader cols(lane);
  const KeyBits keybits(a, b, keys, lane);
  auto issue = [&](int stage, int kt, uint64_t bits) {
    uint8_t *base = stage ? smem1 : smem0;
    const int64_t key0 = static_cast<int64_t>(kt) * kRows;
    const int left = keys - kt * kRows;
    if (keybits.mask) {
      kl.template issue<true>(base, kp + key0 * a.k.sl, a.k.sl, a.dh, left, bits);
      vl.template issue<true>(base + T::kBytes, vp + key0 * a.v.sl, a.v.sl, a.dh, left, bits);
    } else {
      kl.template issue<false>(base, kp + key0 * a.k.sl, a.k.sl, a.dh, left, bits);
      vl.template issue<false>(base + T::kBytes, vp + key0 * a.v.sl, a.v.sl, a.dh, left, bits);
    }
  };

  const int reach = a.bias.reach, pitch = bias_pitch(reach), span = hist_floats(reach);
  float *hist = table + 4 * pitch;  // [2 NW][span]; after that [NW][2] sums
  float *mine = hist + (2 * wave + h) * span;
  float sum_behind = 0.0f, sum_ahead = 0.0f, far_behind = 0.0f, far_ahead = 0.0f;
  auto clear_hist = [&]() __attribute__((always_inline)) {
    for (int i = threadIdx.x; i < 2 * NW * span; i += 64 * NW) hist[i] = 0.0f;
  };
  if constexpr (BIAS) {
    build_bias(table, a.bias, head, 64 * NW, false);
    clear_hist();
  }
  const float shift = ds_shift<BF>(a, w, b, hk, lane), ds_mul = BF ? 1.0f : __builtin_exp2f(shift);

  f32x16 dq[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) dq[db] = f32x16{};
  uint64_t bits = 0;
  int byte = 0;
  // What is known of a tile ahead of its scores: whether any are needed, whether some are not seen, where the bias is one value.
  struct Kind {
    bool any, part, behind, ahead;
    float bc;
  };
  auto kind_of = [&](int kt) __attribute__((always_inline)) {
    const int key0 = kt * kRows;
    Kind x;
    x.any = bits && !(a.causal && key0 > first + 31);
    x.part = bits != ~0ull || (a.causal && key0 + kRows - 1 > first);
    x.behind = BIAS && key0 + kRows - 1 - first <= -reach;
    x.ahead = BIAS && !x.behind && key0 - first - 31 >= (a.bias.ahead ? reach : 0);
    x.bc = x.behind ? far_behind : x.ahead ? far_ahead : 0.0f;
    return x;
  };
  // dS of 32 keys.
  auto scores = [&](const uint8_t *ks, int kt, int kb, const Kind &x) __attribute__((always_inline)) {
    const uint8_t *vs = ks + T::kBytes;
    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int i = 0; i < D / 16; ++i) s = mfma<BF>(rows.read(ks, kb, i), q.f[i], s);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) dp = mfma<BF>(rows.read(vs, kb, i), dO.f[i], dp);
    if (BIAS && !x.behind && !x.ahead) {
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        float bv[8];
        bias_run(table, pitch, reach, kt * kRows + 32 * kb + 16 * t2 + 8 * h - pos, bv);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[8 * t2 + e] += bv[e];
      }
    }
    if (x.part) {
      const uint64_t seen = (a.causal ? bits & up_to(pos - kt * kRows) : bits) >> (8 * h);
      const uint32_t word = static_cast<uint32_t>(kb ? seen >> 32 : seen);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = (word >> (16 * (r >> 3) + (r & 7))) & 1 ? s[r] : -__builtin_inff();
    }
    const float base = nl + x.bc;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = materialize(__builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c2, base)) * (dp[r] - dd));
    return s;
  };
  auto compute = [&](int stage, int kt, const Kind &x) __attribute__((always_inline)) {
    uint8_t *ks = stage ? smem1 : smem0;
    float add = 0.0f;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const f32x16 s = scores(ks, kt, kb, x);
      const bool near = !x.behind && !x.ahead;
      if (BIAS && near) {
        Diagonals diagonals;
        diagonals.add(0, s, lane);
        diagonals.add(1, s, lane);
        diagonals.store(mine + kt * kRows + 32 * kb + 8 * h - pos + reach + kSpill);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        add += s[r];
        size += fabsf(s[r]);
      }
      uint4 sb[2];
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        float ds[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) ds[e] = BF ? s[8 * t2 + e] : materialize(s[8 * t2 + e] * ds_mul);
        sb[t2] = pack8<BF>(ds);
      }
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
        for (int db = 0; db < D / 32; ++db) dq[db] = mfma<BF>(cols.read(ks, db, kb, t2), sb[t2], dq[db]);
    }
    missing += add;
    if constexpr (BIAS) {
      sum_behind += x.behind ? add : 0.0f;
      sum_ahead += x.ahead ? add : 0.0f;
    }
  };
  auto step = [&](int stage) __attribute__((always_inline)) {
    const uint64_t bits_next = keybits.word(kt + 1, byte);
    if (kt + 1 < end) issue(stage ^ 1, kt + 1, bits_next);
    byte = keybits.load(kt + 2);
    const Kind x = kind_of(kt);
    if (x.any) compute(stage, kt, x);
    bits = bits_next;
    wait_vmcnt<0>();
    __syncthreads();
  };
  auto begin = [&](int kt) {
    bits = keybits.word(kt, keybits.load(kt));
    issue(0, kt, bits);
    byte = keybits.load(kt + 1);
    wait_vmcnt<0>();
    __syncthreads();
    if constexpr (BIAS) {
      far_behind = table[0] * a.c2;
      far_ahead = table[2 * reach + 16] * a.c2;
    }
  };
  if (ntiles <= kRefine) {
    float lacks = 0.0f;
    for (int i = 0; i < ntiles; ++i) {
      begin(i);
      const Kind x = kind_of(i);
      if (x.any)
        for (int kb = 0; kb < 2; ++kb) {
          const f32x16 s = scores(smem0, i, kb, x);
#pragma unroll
          for (int r = 0; r < 16; ++r) lacks += s[r];
        }
      __syncthreads();
    }
    dd += pair_sum(lacks);
    size = __builtin_inff();
  }
  while (true) {
    if (kt < end) begin(kt);
    while (kt < end) {
      step(0);
      if (++kt >= end) break;
      step(1);
      ++kt;
    }
    missing = pair_sum(missing);
    size = pair_sum(size);
    if (cut.parts > 1) break;
    if (!any_off(missing, size)) break;  // no wave is at the tiles or the histograms any more
    dd += missing;
    size = __builtin_inff();
    kt = 0;
#pragma unroll
    for (int db = 0; db < D / 32; ++db) dq[db] = f32x16{};
    if constexpr (BIAS) {
      sum_behind = sum_ahead = 0.0f;
      clear_hist();
    }
  }
  if (h == 0 && row0 + c < w.Lqp) {
    if (cut.parts > 1 && !cut.again)
      cut.missing[part * (static_cast<int64_t>(a.B) * a.H * w.Lqp) + stat] = make_float2(missing, size);
    if (part == 0) {  // for key_kernel
      w.neg_lse[stat] = nl;
      w.dot[stat] = dd;
    }
  }

  if constexpr (BIAS) {
    __syncthreads();
    // The histograms added up, then each bucket by one wave.
    float *sums = hist + 2 * NW * span;
    sum_behind = wave_sum(sum_behind);
    sum_ahead = wave_sum(sum_ahead);
    if (lane == 0) {
      sums[2 * wave] = sum_behind;
      sums[2 * wave + 1] = sum_ahead;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < span; i += 64 * NW) {
      float x = 0.0f;
#pragma unroll
      for (int j = 0; j < 2 * NW; ++j) x += hist[j * span + i];
      hist[i] = x;
    }
    __syncthreads();
    const int n = a.bias.n, buckets = a.bias.ahead ? 2 * n : n;
    const int64_t bh = static_cast<int64_t>(b) * a.H + head;
    float *out = w.dtable_part + ((bh * cut.tiles + qt) * cut.parts + part) * buckets;
    for (int r = wave; r < buckets; r += NW) {
      const bool up = r >= n;  // keys after the query
      const int bt = up ? r - n : r;
      int lo = a.bias.edge[bt], hi = bt + 1 < n ? a.bias.edge[bt + 1] : reach + kSpill + 1;  // distances
      if (up) lo = max(lo, 1);
      float x = 0.0f;
      for (int i = lo + lane; i < hi; i += 64) x += hist[(up ? i : -i) + reach + kSpill];
      if (!a.bias.ahead && bt == 0)
        for (int i = 1 + lane; i <= reach + kSpill; i += 64) x += hist[i + reach + kSpill];
      x = wave_sum(x);
      if (lane == 0) {
        if (bt == n - 1 && !up)
          for (int j = 0; j < NW; ++j) x += sums[2 * j];
        if (a.bias.ahead ? up && bt == n - 1 : bt == 0)
          for (int j = 0; j < NW; ++j) x += sums[2 * j + 1];
        out[r] = x;
      }
    }
  }

  const int row = row0 + c;
  if (row >= a.Lq) return;
  const float mul = a.c2 * kLn2 * (BF ? 1.0f : __builtin_exp2f(-shift));
  const int64_t at = ((static_cast<int64_t>(b) * a.H + head) * a.Lq + row) * a.dh;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int ch = 32 * db + 8 * y + 4 * h;
      if (32 * db + 8 * y >= a.dh) continue;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = materialize(dq[db][4 * y + e] * mul);
      if (cut.parts > 1)
        *reinterpret_cast<float4 *>(cut.partial + static_cast<int64_t>(part) * a.B * a.H * a.Lq * a.dh + at + ch) =
            make_float4(x[0], x[1], x[2], x[3]);
      else
        *reinterpret_cast<uint2 *>(w.dq + at + ch) = make_uint2(pack<BF>(x[0], x[1]), pack<BF>(x[2], x[3]));
    }
}

// y = the sum of `parts` arrays of n floats, in their order; 4 values a thread. blockIdx.y: the second array of a pair.
template <bool BF>
__global__ __launch_bounds__(256) void sum_kernel(const float *__restrict__ partial, int parts, int64_t n, int arrays,
                                                  uint16_t *y0, uint16_t *y1) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const float *p = partial + blockIdx.y * n + i;
  float4 s = *reinterpret_cast<const float4 *>(p);
  for (int j = 1; j < parts; ++j) {
    const float4 x = *reinterpret_cast<const float4 *>(p + static_cast<int64_t>(j) * arrays * n);
    s.x += x.x;
    s.y += x.y;
    s.z += x.z;
    s.w += x.w;
  }
  *reinterpret_cast<uint2 *>((blockIdx.y ? y1 : y0) + i) =
      make_uint2(pack<BF>(materialize(s.x), materialize(s.y)), pack<BF>(materialize(s.z), materialize(s.w)));
}

// dk and dv of n values each where there are no queries; 4 values a thread. blockIdx.y: dv.
__global__ __launch_bounds__(256) void zero_kernel(int64_t n, uint16_t *dk, uint16_t *dv) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i < n) *reinterpret_cast<uint2 *>((blockIdx.y ? dv : dk) + i) = make_uint2(0, 0);
}

// dtable[r, head] = the sum over images and workgroups, in a fixed order. One workgroup per head.
__global__ __launch_bounds__(256) void dtable_kernel(const float *__restrict__ part, int B, int H, int each, int buckets,
                                                     void *dtable, int dtype) {
  __shared__ float red[256];
  const int head = blockIdx.x, rows = max(256 / buckets, 1), lane = threadIdx.x % buckets, row = threadIdx.x / buckets;
  float x = 0.0f;
  if (row < rows)
    for (int i = row; i < B * each; i += rows) {
      const int b = i / each, j = i - b * each;
      x += part[((static_cast<int64_t>(b) * H + head) * each + j) * buckets + lane];
    }
  red[threadIdx.x] = x;
  __syncthreads();
  if (threadIdx.x >= buckets) return;
  x = 0.0f;
  for (int j = 0; j < rows; ++j) x += red[j * buckets + threadIdx.x];
  const int64_t at = static_cast<int64_t>(threadIdx.x) * H + head;
  if (dtype == SELAS_F32) store_f<SELAS_F32>(dtable, at, x);
  else if (dtype == SELAS_F16) store_f<SELAS_F16>(dtable, at, x);
  else store_f<SELAS_BF16>(dtable, at, x);
}

// ------------------------------------------------------------------ host side

struct Plan {
  int D, qblocks, kblocks, buckets;
  Cut key, query;
  int64_t neg_lse, dot, g_norm, v_norm, dtable, key_partial, query_partial, missing, bytes;  // offsets into the workspace
  Threads threads;
};
constexpr int kNW = 4;

Plan plan_of(const Args &a, bool bf) {
  Plan p{};
  p.D = width_of(a.dh);
  p.qblocks = static_cast<int>(cdiv(a.Lq, kRows));
  p.kblocks = static_cast<int>(cdiv(a.Lk, kRows));
  p.buckets = a.bias.ahead ? 2 * a.bias.n : a.bias.n;
  const int64_t cu = cu_count();
  auto cut = [&](int64_t heads, int tiles, int64_t streamed, int64_t inner) {
    const int64_t whole = heads * tiles;
    // Workgroups for two to a CU, of four streamed tiles at least.
    const int64_t parts = std::max<int64_t>(1, std::min(2 * cu / std::max<int64_t>(whole, 1), streamed / 4));
    return Cut{tiles, static_cast<int>(parts), deal(whole * parts, inner, a.lengths || a.mask), fast_div(std::max(tiles, 1)),
               fast_div(static_cast<uint32_t>(parts)), fast_div(std::max(a.group, 1)), fast_div(std::max(a.Hk, 1)), nullptr, nullptr, 0};
  };
  const int ktiles = static_cast<int>(cdiv(a.Lk, 32 * kNW)), qtiles = static_cast<int>(cdiv(a.Lq, 32 * kNW));
  p.key = cut(static_cast<int64_t>(a.B) * a.Hk, ktiles, static_cast<int64_t>(a.group) * p.qblocks, ktiles);
  p.query = cut(static_cast<int64_t>(a.B) * a.H, qtiles, p.kblocks, static_cast<int64_t>(a.group) * qtiles);
  auto take = [&](int64_t floats) {
    const int64_t at = p.bytes;
    p.bytes += (floats * 4 + 255) / 256 * 256;
    return at;
  };
  const int64_t stats = static_cast<int64_t>(a.B) * a.H * p.qblocks * kRows;
  p.neg_lse = take(stats);
  p.dot = take(stats);
  if (!bf) {
    p.g_norm = take(static_cast<int64_t>(a.B) * a.H * p.qblocks);
    p.v_norm = take(static_cast<int64_t>(a.B) * a.Hk * p.kblocks);
  }
  if (a.bias.table) p.dtable = take(static_cast<int64_t>(a.B) * a.H * p.query.tiles * p.query.parts * p.buckets);
  if (p.key.parts > 1) p.key_partial = take(2ll * p.key.parts * a.B * a.Hk * a.Lk * a.dh);
  if (p.query.parts > 1) {
    p.query_partial = take(static_cast<int64_t>(p.query.parts) * a.B * a.H * a.Lq * a.dh);
    p.missing = take(2 * p.query.parts * stats);
  }
  const int64_t heads = static_cast<int64_t>(a.B) * a.H, key_heads = static_cast<int64_t>(a.B) * a.Hk;
  if (!bf) p.threads.add(heads * p.qblocks + key_heads * p.kblocks, 256);
  p.threads.add(p.query.deal.blocks, 64 * kNW);
  p.threads.add(p.key.deal.blocks, 64 * kNW);
  if (p.query.parts > 1) p.threads.add(cdiv(heads * a.Lq * a.dh, 1024), 256);
  if (p.key.parts > 1 || !a.Lq) p.threads.add(cdiv(key_heads * a.Lk * a.dh, 1024), 256);
  if (a.bias.table) p.threads.add(a.H, 256);
  return p;
}

void sum_table(const Args &a, const Grads &w, const Plan &p, hipStream_t st) {
  dtable_kernel<<<dim3(a.H), dim3(256), 0, st>>>(w.dtable_part, a.B, a.H, p.query.tiles * p.query.parts, p.buckets, w.dtable,
                                                 a.bias.dtype);
}

// Without queries every gradient is zero. q, k and v are not looked at (their pointers were not checked).
void launch_zeros(const Args &a, const Grads &w, const Plan &p, hipStream_t st) {
  const int64_t n = static_cast<int64_t>(a.B) * a.Hk * a.Lk * a.dh;
  if (n) zero_kernel<<<dim3(static_cast<uint32_t>(cdiv(n, 1024)), 2), dim3(256), 0, st>>>(n, w.dk, w.dv);
  if (a.bias.table) sum_table(a, w, p, st);
}

template <bool BF, int D, bool BIAS>
void launch(const Args &a, const Grads &w, const Plan &p, hipStream_t st) {
  const int reach = a.bias.reach;
  auto sum = [&](const Cut &cut, int64_t rows, int arrays, uint16_t *y0, uint16_t *y1) {
    const int64_t n = rows * a.dh;
    if (cut.parts > 1)
      sum_kernel<BF><<<dim3(static_cast<uint32_t>(cdiv(n, 1024)), arrays), dim3(256), 0, st>>>(cut.partial, cut.parts, n, arrays,
                                                                                               y0, y1);
  };
  const int norms = a.B * a.H * p.qblocks + a.B * a.Hk * p.kblocks;
  if (!BF && norms) norm_kernel<<<dim3(norms), dim3(256), 0, st>>>(a, w);
  if (p.query.deal.total) {
    const size_t lds = BIAS ? bias_bytes(reach) + 4 * (2 * kNW * hist_floats(reach) + 2 * kNW) : 0;
    Cut cut = p.query;
    query_kernel<BF, D, kNW, BIAS><<<dim3(cut.deal.blocks), dim3(64 * kNW), lds, st>>>(a, w, cut);
    cut.again = 1;
    if (cut.parts > 1) query_kernel<BF, D, kNW, BIAS><<<dim3(cut.deal.blocks), dim3(64 * kNW), lds, st>>>(a, w, cut);
    sum(p.query, static_cast<int64_t>(a.B) * a.H * a.Lq, 1, w.dq, nullptr);
  }
  if (p.key.deal.total) {
    key_kernel<BF, D, kNW, BIAS><<<dim3(p.key.deal.blocks), dim3(64 * kNW), BIAS ? 2 * bias_bytes(reach) : 0, st>>>(a, w, p.key);
    sum(p.key, static_cast<int64_t>(a.B) * a.Hk * a.Lk, 2, w.dk, w.dv);
  }
  if constexpr (BIAS) sum_table(a, w, p, st);
}

}  // namespace
}  // namespace textattn
}  // namespace selas

using namespace selas;
using namespace selas::textattn;

extern "C" int selas_text_attention_backward_workspace_bytes(const selas_text_attention_problem *problem, int dtype,
                                                             int64_t *bytes) {
  if (!bytes) return set_error(SELAS_EINVAL, "text_attention_backward_workspace_bytes: null pointer");
  *bytes = 0;
  Args a;
  if (int e = check_args("text_attention_backward_workspace_bytes", problem, dtype, false, a)) return e;
  if (!a.H) return ok();
  const Plan p = plan_of(a, dtype == SELAS_BF16);
  if (int e = p.threads.check("text_attention_backward_workspace_bytes")) return e;
  *bytes = p.bytes;
  return ok();
}

extern "C" int selas_text_attention_backward(const selas_text_attention_problem *problem, const void *grad, int64_t g_sb,
                                             int64_t g_sl, void *dq, void *dk, void *dv, void *dtable, int dtype,
                                             void *workspace, int64_t workspace_bytes, void *stream) {
  const char *what = "text_attention_backward";
  Args a;
  if (int e = check_args(what, problem, dtype, true, a)) return e;
  if (!a.H) return ok();
  const bool bf = dtype == SELAS_BF16;
  Grads w{};
  if (a.B && a.Lq) {
    if (!grad || !a.lse || !dq) return set_error(SELAS_EINVAL, "%s: null pointer (grad, lse or dq)", what);
    if (g_sb < 0 || g_sl < 0) return set_error(SELAS_EINVAL, "%s: grad has a negative stride", what);
    g_sl = stride_of(a.Lq, g_sl, a.dh);
    if (!aligned(grad, 16) || g_sb % 8 || g_sl % 8 || g_sl > (1 << 23))
      return set_error(SELAS_EUNSUPPORTED, "%s: grad must be 16-byte aligned with strides of whole 16 bytes, rows up to 2^23 elements", what);
  }
  if (a.B && a.Lk && (!dk || !dv)) return set_error(SELAS_EINVAL, "%s: null pointer (dk or dv)", what);
  if (a.bias.table && !dtable) return set_error(SELAS_EINVAL, "%s: null pointer (dtable)", what);
  if (!aligned(dq, 8) || !aligned(dk, 8) || !aligned(dv, 8))
    return set_error(SELAS_EUNSUPPORTED, "%s: dq, dk and dv must be 8-byte aligned", what);
  Plan p = plan_of(a, bf);
  if (int e = p.threads.check(what)) return e;
  if (p.bytes && (workspace_bytes < p.bytes || !workspace || !aligned(workspace, 16)))
    return set_error(SELAS_EINVAL, "%s: needs a 16-byte aligned workspace of %lld bytes", what, (long long)p.bytes);
  auto at = [&](int64_t offset) { return reinterpret_cast<float *>(static_cast<char *>(workspace) + offset); };
  w.g = {static_cast<const uint16_t *>(grad), g_sb, a.dh, g_sl};
  w.dq = static_cast<uint16_t *>(dq);
  w.dk = static_cast<uint16_t *>(dk);
  w.dv = static_cast<uint16_t *>(dv);
  w.neg_lse = at(p.neg_lse);
  w.dot = at(p.dot);
  w.Lqp = p.qblocks * kRows;
  w.qblocks = p.qblocks;
  w.kblocks = p.kblocks;
  w.g_norm = at(p.g_norm);
  w.v_norm = at(p.v_norm);
  w.dtable_part = at(p.dtable);
  w.dtable = dtable;
  p.key.partial = at(p.key_partial);
  p.query.partial = at(p.query_partial);
  p.query.missing = reinterpret_cast<float2 *>(at(p.missing));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (!a.B || !a.Lq) {
    launch_zeros(a, w, p, st);
    return check_launch(what);
  }
  auto go = [&](auto t, auto d) {
    constexpr bool kBf = decltype(t)::value;
    constexpr int kD = decltype(d)::value;
    if (a.bias.table) launch<kBf, kD, true>(a, w, p, st);
    else launch<kBf, kD, false>(a, w, p, st);
  };
  using I64 = std::integral_constant<int, 64>;
  using I96 = std::integral_constant<int, 96>;
  using I128 = std::integral_constant<int, 128>;
  auto width = [&](auto t) { p.D == 64 ? go(t, I64{}) : p.D == 96 ? go(t, I96{}) : go(t, I128{}); };
  if (bf) width(std::true_type{});
  else width(std::false_type{});
  return check_launch(what);
}
